"""What the operators on e4m3 pools refuse, before they touch a device: no GPU needed."""
import pytest

from navi_amd import abi
from test_kv_refusals import P, heads, pages, refused

F8 = abi.DT_F8E4M3


def _append(xt=0, ldx=4096, ld=1024, qt=0, ldq=2048, **kw):
    return abi.kv_append, pages(), heads(kv_dtype=F8, **kw), P, xt, ldx, P, P, ld, P, qt, ldq


def _attend(qt=0, ldq=2048, ld=1024, size=1 << 40, **kw):
    return abi.tree_attention, pages(), heads(kv_dtype=F8, **kw), P, qt, ldq, P, P, ld, 1.0, 4096, P, ldq, P, size


@pytest.mark.parametrize("kw,status", [(dict(k_scale=P + 2), 4), (dict(v_scale=P + 1), 4), (dict(ld=1032), 4), (dict(ld=1016), 4), (dict(head_dim=96), 6)], ids=str)
def test_both_refuse(kw, status):
    refused(status, *_append(**kw))
    refused(status, *_attend(**kw))


@pytest.mark.parametrize("t", [3, 4, F8, 7, -1])
def test_types_of_rows_and_queries(t):
    """f32, f16 and bf16 only: no rows or queries in 8 bits."""
    refused(6, *_append(xt=t))
    refused(6, *_append(qt=t))
    refused(6, *_attend(qt=t))


def test_strides_of_every_type():
    for t, per in ((0, 4), (1, 8), (2, 8)):
        refused(4, *_append(xt=t, ldx=4096 + per // 2))
        refused(4, *_attend(qt=t, ldq=2048 + per // 2))


def test_the_workspace_is_that_of_the_layout():
    """The type of the pool does not change how a call is cut."""
    assert abi.tree_workspace(pages(), heads(kv_dtype=F8), 4096) == abi.tree_workspace(pages(), heads(), 4096) > 0
    need = abi.tree_workspace(pages(), heads(kv_dtype=F8), 4096)
    assert "workspace" in refused(4, *_attend(size=need - 1))


def test_factors_of_other_pools_are_not_looked_at():
    """An f16 pool's layout may leave them unset."""
    assert abi.tree_workspace(pages(), heads(k_scale=P + 1, v_scale=P + 3), 4096) > 0
