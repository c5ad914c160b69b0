"""What navi_sample_rows and navi_draft_accept refuse before they touch a device, and the definitions that their tests rest on: no GPU needed."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from navi_amd import abi
from sample_util import OFF, as_seen, token_of, weights, words_of, bits_of
from test_kv_refusals import BAD_PAGES, P, pages, refused

Q = P + (1 << 16)


def _sample(x=P, t=0, ld=2048, rows=4, vocab=2048, rules=Q, n_rules=4, u=Q + 256, token=Q + 512, **kw):
    return (abi.sample_rows, x, t, ld, rows, vocab, rules, n_rules, u, token), kw


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), 4), (dict(rules=None), 4), (dict(u=None), 4), (dict(token=None), 4), (dict(x=P + 2), 4), (dict(x=P + 1, t=1), 4), (dict(u=Q + 258), 4),
    (dict(rules=Q + 2), 4), (dict(token=Q + 513), 4), (dict(logprob=Q + 3), 4), (dict(allowed=Q + 1), 4), (dict(seen=Q + 2), 4), (dict(t=3), 6), (dict(t=5), 6),
    (dict(rows=-1), 4), (dict(vocab=0), 4), (dict(vocab=(1 << 20) + 1, ld=1 << 21), 4), (dict(ld=2047), 4), (dict(n_rules=0), 4), (dict(n_rules=3), 4), (dict(ld_token=0), 4),
    (dict(allowed=Q + 1024, ld_allowed=63), 4), (dict(seen=Q + 1024, ld_seen=63), 4), (dict(allowed=Q + 1024, ld_allowed=-1), 4),
    (dict(token=P), 4), (dict(token=Q + 256), 4), (dict(token=Q), 4), (dict(logprob=Q + 256), 4), (dict(logprob=Q + 512), 4), (dict(allowed=Q + 512), 4), (dict(seen=Q + 512), 4),
    (dict(vocab=20000, ld=20000), 4), (dict(vocab=20000, ld=20000, ws=P, ws_bytes=100), 4), (dict(vocab=20000, ld=20000, ws=P + 8, ws_bytes=1 << 30), 4),
    (dict(rows=1 << 22, n_rules=1), 4), (dict(rows=1 << 17, n_rules=1, vocab=1 << 20, ld=1 << 20, ws=P, ws_bytes=1 << 60), 4)], ids=str)
def test_sample_refuses(kw, status):
    a, k = _sample(**kw)
    refused(status, *a, **k)


def test_workspace():
    """None up to 16384 tokens and for arguments that are not valid; enough for a row's bins in any case."""
    assert all(abi.sample_workspace(r, v) == 0 for r, v in ((0, 30000), (-1, 30000), (4, 0), (4, 16384), (4, (1 << 20) + 1)))
    for rows, vocab in ((1, 16385), (1, 151936), (256, 151936), (3, 1 << 20)):
        need = abi.sample_workspace(rows, vocab)
        assert need >= rows * (-(-vocab // 16384) * 257 * 8 + 8192 * 8 + 4)
        a, k = _sample(rows=rows, n_rules=1, vocab=vocab, ld=vocab, ws=P, ws_bytes=need - 1)
        assert "workspace" in refused(4, *a, **k)


def _accept(p=None, drafted=Q, ld_drafted=16, sampled=Q + 64, ld_sampled=16, codes=16, path=Q + 128, most=8, accept=Q + 192, then=Q + 256, **kw):
    return (abi.draft_accept, p or pages(), drafted, ld_drafted, sampled, ld_sampled, codes, path, most, accept, then), kw


@pytest.mark.parametrize("kw", [dict(drafted=None), dict(sampled=None), dict(path=None), dict(accept=None), dict(then=None), dict(ld_drafted=15), dict(ld_sampled=15), dict(codes=0),
                                dict(codes=4097, ld_drafted=5000, ld_sampled=5000), dict(most=0), dict(most=65), dict(p=pages(max_new=65)), dict(path=Q), dict(accept=Q + 64),
                                dict(then=P), dict(path=Q + 192), dict(accept=Q + 256), dict(parent=Q + 128), dict(last=Q + 128), dict(last=Q + 192)], ids=str)
def test_accept_refuses(kw):
    a, k = _accept(**kw)
    refused(4, *a, **k)


@pytest.mark.parametrize("kw", BAD_PAGES, ids=str)
def test_accept_refuses_bad_pages(kw):
    a, k = _accept(pages(**kw))
    refused(4, *a, **k)


def test_accept_refuses_results_over_the_plans_status():
    p = pages(status=Q + 192)
    a, k = _accept(p)
    refused(4, *a, **k)


def test_rule_layout_matches_the_header(tmp_path):
    root = Path(__file__).resolve().parent.parent
    body = "".join(f'printf(" %zu", offsetof(navi_sample_rule, {f[0]}));' for f in abi.SampleRule._fields_)
    (tmp_path / "l.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "navi_amd.h"\nint main(void) { printf("%zu", sizeof(navi_sample_rule));' + body + "return 0; }")
    subprocess.run(["gcc", "-I", str(root / "include"), "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    got = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == [C.sizeof(abi.SampleRule)] + [getattr(abi.SampleRule, f[0]).offset for f in abi.SampleRule._fields_]


# ---- the definition itself, on cases small enough to know ---------------------------------------

def test_definition_of_the_cuts():
    x = np.log(np.array([0.1, 0.4, 0.4, 0.1], np.float32))
    keep = lambda *rule: list(np.flatnonzero(weights(x, rule)))
    assert keep(1, 0, 1, 0, 1) == [0, 1, 2, 3] and keep(1, 1, 1, 0, 1) == [1] and keep(1, 3, 1, 0, 1) == [0, 1, 2]
    assert keep(1, 0, 0.39, 0, 1) == [1] and keep(1, 0, 0.41, 0, 1) == [1, 2] and keep(1, 0, 0.85, 0, 1) == [0, 1, 2] and keep(1, 0, 0, 0, 1) == [1]
    assert keep(1, 0, 1, 0.3, 1) == [1, 2] and keep(1, 0, 1, 5, 1) == [1, 2] and keep(0, 0, 1, 0, 1) == [1]
    assert keep(1, 2, 0.6, 0, 1) == [1, 2] and keep(1, 2, 0.49, 0, 1) == [1]                     # top_p of what top_k leaves


def test_definition_of_the_draw_and_of_what_a_rule_sees():
    w = np.array([0, 0.25, 0, 0.5, 0.25])
    assert [token_of(w, u)[0] for u in (-1, 0, 0.2, 0.25, 0.7, 0.75, 0.99, 1, 3)] == [1, 1, 1, 3, 3, 4, 4, 4, 4]
    assert token_of(None, 0.3) == (-1, -np.inf) and abs(token_of(w, 0.3)[1] - np.log(0.5)) < 1e-15
    b = np.array([1, 0, 1, 1, 0] * 9, bool)
    assert (bits_of(words_of(b), 45) == b).all()
    x = as_seen([2.0, -2.0, np.nan, np.inf, -np.inf, 4.0], (1, 0, 1, 0, 2.0), np.array([1, 1, 1, 1, 1, 0], bool), np.array([1, 1, 1, 0, 1, 1], bool))
    assert x.tolist() == [1.0, -4.0, -np.inf, np.finfo(np.float32).max, -np.inf, -np.inf]
    assert weights(x[4:], OFF) is None
