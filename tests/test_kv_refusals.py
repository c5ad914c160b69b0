"""The paged K/V operators refuse bad arguments before they touch a device: no GPU needed."""
import ctypes as C

import pytest

from navi_amd import abi

P = 1 << 20                                    # an aligned address that no refused call reads


def pages(**kw):
    d = dict(n_requests=2, page_size=16, n_pages=8, max_blocks=4, n_rows=6, max_new=4, block_table=P, n_past=P, cu_rows=P, row_slot=P,
             row_pos=P, row_mask=P)
    d.update(kw)
    return abi.KvPages(**d)


def heads(**kw):
    d = dict(n_head=16, n_kv_head=8, head_dim=128, kv_dtype=abi.DT_F16)
    d.update(kw)
    return abi.KvHeads(**d)


def refused(code, fn, /, *a, **kw):
    with pytest.raises(abi.NaviError) as e:
        fn(*a, **kw)
    assert e.value.status == code, e.value
    return str(e.value)


PLAN = dict(n_new=P, table_in=P, held_in=P, free_in=P, free_pages=P, held=P, free=P, status=P, scratch=P)
BAD_PAGES = [dict(n_requests=0), dict(n_requests=65536), dict(page_size=0), dict(n_pages=0), dict(max_blocks=0), dict(n_rows=-1), dict(max_new=0),
             dict(n_pages=1 << 20, page_size=1 << 11), dict(block_table=None), dict(n_past=None), dict(cu_rows=None), dict(row_slot=None),
             dict(row_pos=None), dict(row_mask=None)]


@pytest.mark.parametrize("kw", BAD_PAGES, ids=str)
def test_every_operator_refuses_bad_pages(kw):
    p = pages(**kw)
    refused(abi.NAVI_ERR_INVALID, abi.kv_plan, p, **PLAN)
    refused(abi.NAVI_ERR_INVALID, abi.kv_append, p, heads(), P, 0, 4096, P, P, 1024, P, 0, 2048)
    refused(abi.NAVI_ERR_INVALID, abi.tree_attention, p, heads(), P, 0, 2048, P, P, 1024, 1.0, 64, P, 2048, P, 1 << 30)
    refused(abi.NAVI_ERR_INVALID, abi.kv_commit, p, [P], [P], 1024, P, 4, P, P + 64, P)
    assert abi.tree_workspace(p, heads(), 64) == 0


@pytest.mark.parametrize("name", sorted(PLAN))
def test_plan_refuses_null(name):
    refused(abi.NAVI_ERR_INVALID, abi.kv_plan, pages(), **{**PLAN, name: None})


def test_plan_refuses_wide_trees_and_misaligned_scratch():
    assert "64" in refused(abi.NAVI_ERR_INVALID, abi.kv_plan, pages(max_new=65, n_rows=130), **PLAN, parent=P)
    assert "aligned" in refused(abi.NAVI_ERR_INVALID, abi.kv_plan, pages(), **{**PLAN, "scratch": P + 4})


@pytest.mark.parametrize("kw,status", [(dict(n_head=15), 4), (dict(n_kv_head=0), 4), (dict(n_head=2048, n_kv_head=8), 4), (dict(head_dim=96), 6),
                                       (dict(kv_dtype=abi.DT_F32), 6), (dict(kv_dtype=7), 6)], ids=str)
def test_heads_are_checked(kw, status):
    refused(status, abi.kv_append, pages(), heads(**kw), P, 0, 1 << 20, P, P, 1 << 18, P, 0, 1 << 19)
    refused(status, abi.tree_attention, pages(), heads(**kw), P, kw.get("kv_dtype", 1), 1 << 19, P, P, 1 << 18, 1.0, 64, P, 1 << 19, P, 1 << 30)


def _append(pages_=None, heads_=None, x=P, xt=0, ldx=4096, k=P, v=P, ld=1024, q=P, qt=0, ldq=2048, **kw):
    return (abi.kv_append, pages_ or pages(), heads_ or heads(), x, xt, ldx, k, v, ld, q, qt, ldq), kw


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), 4), (dict(k=None), 4), (dict(v=None), 4), (dict(q=None), 4), (dict(x=P + 4), 4), (dict(k=P + 2), 4), (dict(q=P + 8), 4),
    (dict(ldx=4095), 4), (dict(ldx=4097), 4), (dict(ldq=2047), 4), (dict(ld=1023), 4), (dict(ld=1028), 4), (dict(xt=1, ldx=4100), 4),
    (dict(xt=2), 6), (dict(qt=2), 6), (dict(xt=3), 6), (dict(rot=P, n_rot=0), 4), (dict(rot=P + 4, n_rot=9), 4), (dict(q_norm=P + 4), 4),
    (dict(k_norm=P + 8), 4)], ids=str)
def test_append_refuses(kw, status):
    a, k = _append(**kw)
    refused(status, *a, **k)


def test_append_refuses_more_rows_than_a_grid_holds():
    a, k = _append(pages(n_rows=(1 << 31) // 32))
    refused(4, *a, **k)


@pytest.mark.parametrize("dim", [64, 128])
def test_launches_of_2_to_32_threads_are_refused(dim):
    """Append: dim / 8 threads a head; attention: 512 threads a request and head."""
    a, k = _append(pages(n_rows=(1 << 32) // (dim // 8) // 32), heads(head_dim=dim))
    assert "too many" in refused(4, *a, **k)
    assert "too many" in refused(4, *_attend(pages(n_requests=1 << 14), heads(n_head=512, n_kv_head=8, head_dim=dim), ldq=1 << 16, ldo=1 << 16))


def _attend(pages_=None, heads_=None, q=P, qt=0, ldq=2048, k=P, v=P, ld=1024, keys=64, out=P, ldo=2048, ws=P, size=1 << 40):
    return abi.tree_attention, pages_ or pages(), heads_ or heads(), q, qt, ldq, k, v, ld, 1.0, keys, out, ldo, ws, size


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 4), (dict(k=None), 4), (dict(v=None), 4), (dict(out=None), 4), (dict(q=P + 4), 4), (dict(out=P + 8), 4), (dict(k=P + 2), 4),
    (dict(ldq=2044), 4), (dict(ldq=2050), 4), (dict(ldo=2040), 4), (dict(ld=1016), 4), (dict(keys=0), 4), (dict(keys=2 ** 31 - 1), 4), (dict(qt=2), 6),
    (dict(qt=0, heads_=heads(kv_dtype=2)), 6), (dict(pages_=pages(max_new=65)), 4), (dict(pages_=pages(n_requests=65535), heads_=heads(n_head=1024, n_kv_head=8)), 4),
    (dict(pages_=pages(n_requests=65535), heads_=heads(n_head=1024, n_kv_head=8), ldq=1 << 17, ldo=1 << 17), 4)], ids=str)
def test_attention_refuses(kw, status):
    refused(status, *_attend(**kw))


def test_attention_refuses_a_small_workspace():
    need = abi.tree_workspace(pages(), heads(), 4096)
    assert need > 0
    for ws, size in ((None, need), (P, need - 1), (P + 4, need)):
        assert "workspace" in refused(4, *_attend(keys=4096, ws=ws, size=size))


def test_workspace_of_invalid_arguments_is_zero():
    assert abi.tree_workspace(pages(max_new=65), heads(), 4096) == 0
    assert abi.tree_workspace(pages(), heads(head_dim=80), 4096) == 0
    assert abi.tree_workspace(pages(), heads(), 0) == 0
    assert abi.lib().navi_tree_workspace(None, heads(), 64) == 0 and abi.lib().navi_tree_workspace(pages(), None, 64) == 0


@pytest.mark.parametrize("kw", [dict(path=None), dict(accept=None), dict(n_past=None), dict(status=None), dict(n_past=P), dict(max_path=0), dict(max_path=65),
                                dict(ld=1020), dict(ld=0), dict(k=[None]), dict(v=[P + 2]), dict(k=[], v=[])], ids=str)
def test_commit_refuses(kw):
    d = dict(k=[P], v=[P], ld=1024, path=P, max_path=4, accept=P, n_past=P + 64, status=P)
    d.update(kw)
    refused(4, abi.kv_commit, pages(), d["k"], d["v"], d["ld"], d["path"], d["max_path"], d["accept"], d["n_past"], d["status"])


@pytest.mark.parametrize("name,other", [(a, b) for a in ("n_past", "status") for b in ("past", "cu", "table", "path", "accept")] + [("n_past", "status")])
def test_commit_refuses_results_over_inputs(name, other):
    """Other blocks read the inputs until the launch ends: in place would be a race."""
    at = dict(table=P, past=P + 64, cu=P + 128, path=P + 192, accept=P + 256, n_past=P + 320, status=P + 384)
    at[name] = at[other]
    p = pages()
    p.block_table, p.n_past, p.cu_rows = at["table"], at["past"], at["cu"]
    assert "inputs" in refused(4, abi.kv_commit, p, [P], [P], 1024, at["path"], 4, at["accept"], at["n_past"], at["status"])


def test_commit_refuses_a_cache_smaller_than_the_pool():
    ptr = (C.c_void_p * 1)(P)
    view = abi.KvView(1, 8 * 16 - 1, 1024, C.cast(ptr, C.POINTER(C.c_void_p)), C.cast(ptr, C.POINTER(C.c_void_p)))
    err = C.create_string_buffer(256)
    assert abi.lib().navi_kv_commit(pages(), view, P, 4, P, P + 64, P, None, err, 256) == abi.NAVI_ERR_INVALID
    assert b"cache rows" in err.value


def test_struct_layouts_match_the_header(tmp_path):
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "navi_amd.h"', "int main(void) {"]
    for name, py in (("navi_kv_pages", abi.KvPages), ("navi_kv_heads", abi.KvHeads)):
        lines.append(f'printf("%zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f[0]}));' for f in py._fields_]
        lines.append('printf("\\n");')
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", str(root / "include"), "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    got = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, py in zip(got, (abi.KvPages, abi.KvHeads)):
        assert [int(x) for x in line.split()] == [C.sizeof(py)] + [getattr(py, f[0]).offset for f in py._fields_]


@pytest.mark.parametrize("name", ["n_past", "status"])
@pytest.mark.parametrize("field", ["status", "row_slot"])
def test_commit_refuses_results_over_the_plans(name, field):
    at = dict(n_past=P + 320, status=P + 384)
    p = pages(block_table=P + 64, n_past=P + 128, cu_rows=P + 192, row_slot=P + 256, status=P + 448)
    setattr(p, field, at[name])
    assert "inputs" in refused(4, abi.kv_commit, p, [P], [P + (1 << 20)], 1024, P, 4, P + 16, at["n_past"], at["status"])


ROWS = 8 * 16 * 1024 * 2                        # bytes of a layer's K or V in the pool of pages()


@pytest.mark.parametrize("k,v", [([P], [P + 256]), ([P], [P + ROWS - 16]), ([P + ROWS // 2], [P]), ([P, P + 512], [P + 2 * ROWS, P + 3 * ROWS]),
                                 ([P, P + 3 * ROWS], [P + ROWS, P + 2 * ROWS + 16])], ids=str)
def test_commit_refuses_rows_of_one_array_inside_another(k, v):
    """Rows are moved whole: K and V interleaved in one allocation (V's base inside K's row) would move into each other, and past its end."""
    assert "overlap" in refused(4, abi.kv_commit, pages(), k, v, 1024, P, 4, P, P + 64, P + 128)


def test_append_refuses_queries_over_rows_of_another_layout():
    """In place a head overwrites itself only with the same type and stride."""
    for kw in (dict(ldx=4096, ldq=2048), dict(ldx=4096, ldq=4096, xt=1), dict(ldx=4096, ldq=4096, qt=1)):
        a, k = _append(x=P, q=P, **kw)
        assert "over d_x" in refused(4, *a, **k)


def test_attention_refuses_results_over_queries_of_another_stride():
    assert "over d_q" in refused(4, *_attend(q=P, out=P, ldq=2048, ldo=4096))
    assert "over d_q" in refused(4, *_attend(q=P, out=P, ldq=4096, ldo=2048, keys=4096))


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_attention_refuses_a_scale_that_is_no_number(scale):
    assert "scale" in refused(4, abi.tree_attention, pages(), heads(), P, 0, 2048, P, P, 1024, scale, 64, P, 2048, P, 1 << 30)
