"""navi_talker_verify over planned steps against the CPU oracle: a prompt prefilled into the talker's own cache and one
taken in as a chain of rows, trees of drafted rows on both, the accepted rows committed, and the next step on what
was committed. Bars as the prefill's: 2e-2 max abs and cosine > 0.9995 against the oracle's rows."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from gpu_util import compare, log
from kv_util import random_tree

pytestmark = pytest.mark.gpu
TOL_ABS, TOL_COS, PAGE = 2e-2, 0.9995, 16


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int64).astype(np.int32), dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def side(small_blob):
    from navi_amd import abi
    from oracle.model import Oracle
    abi.device_open()
    W = abi.DeviceWeights(small_blob, select=lambda t: t.name.startswith("talker."))
    return abi, Oracle(small_blob), abi.Talker(W, max_prompt_tokens=128, max_positions=512), W


class Pool:
    """The requests' state on the device, over the talker's own cache as pages of 16 rows."""

    def __init__(self, abi, talker, n, taken):
        self.abi, self.t, self.n, self.n_pages, self.blocks = abi, talker, n, 512 // PAGE, 12
        rest = list(range(self.n_pages - 1, -1, -1))
        table = [[-1] * self.blocks for _ in range(n)]
        for i, pages in taken.items():
            table[i][:len(pages)] = pages
            rest = [p for p in rest if p not in pages]
        self.table, self.held, self.free, self.stack = i32(table), i32([len(taken.get(i, [])) for i in range(n)]), i32([len(rest)]), i32(rest + [0] * (self.n_pages - len(rest)))
        self.past = i32([0] * n)

    def step(self, trees, rows, kv=None, logits=True, spare=0, spare_value=0., status=None):
        abi, new = self.abi, [len(t) for t in trees]
        R = sum(new) + spare
        self.cu, self.slot, self.pos, self.status = i32([0] * (self.n + 1)), i32([-1] * R), i32([0] * R), i32([0] * self.n)
        self.mask, scratch = torch.zeros(R, dtype=torch.int64, device="cuda"), i32([0] * 4 * self.n)
        d_new, d_par = i32(new), i32([p for t in trees for p in t] + [0] * spare)
        d_rows = torch.cat([torch.from_numpy(np.concatenate(rows).astype(np.float32)), torch.full((spare, 1024), spare_value)]).cuda()
        hid, lg = torch.zeros(R, 1024, device="cuda"), torch.zeros(R, self.t.params.talker.vocab, device="cuda")
        self.pages = abi.KvPages(self.n, PAGE, self.n_pages, self.blocks, R, 64, *(x.data_ptr() for x in (self.table, self.past, self.cu, self.slot, self.pos, self.mask)))
        torch.cuda.synchronize()
        abi.kv_plan(self.pages, n_new=d_new.data_ptr(), parent=d_par.data_ptr(), table_in=self.table.data_ptr(), held_in=self.held.data_ptr(),
                    free_in=self.free.data_ptr(), free_pages=self.stack.data_ptr(), held=self.held.data_ptr(), free=self.free.data_ptr(),
                    status=self.status.data_ptr(), scratch=scratch.data_ptr(), stream=abi.lib().navi_device_stream())
        self.t.verify(self.pages, self.blocks * PAGE, d_rows.data_ptr(), hid.data_ptr(), lg.data_ptr() if logits else None, kv=kv)
        assert self.status.tolist() == (status or [0] * self.n)
        return hid.cpu().numpy(), lg.cpu().numpy()

    def commit(self, paths, kv):
        st = self.abi.lib().navi_device_stream()
        path, acc, past, status = i32([p + [0] * (64 - len(p)) for p in paths]), i32([len(p) for p in paths]), i32([0] * self.n), i32([0] * self.n)
        torch.cuda.synchronize()
        self.abi.kv_commit(self.pages, list(kv.k), list(kv.v), kv.kv_dim, path.data_ptr(), 64, acc.data_ptr(), past.data_ptr(), status.data_ptr(), stream=st)
        torch.cuda.synchronize()
        assert status.tolist() == [0] * self.n
        self.past.copy_(past)


def oracle_rows(ora, history, x):
    """Post-norm hidden and logits of rows x after the rows of `history`."""
    kv = ora.new_kv(256)
    rows = np.concatenate([history, x]).astype(np.float32)
    h, lg = ora.talker_forward(torch.from_numpy(rows), kv, 0)
    return h.numpy()[len(history):], lg.numpy()[len(history):]


def chain_of(tree, j):
    out = []
    while j >= 0:
        out.insert(0, j)
        j = tree[j]
    return out


def check(ora, history, tree, x, hid, lg, what):
    for j in range(len(tree)):
        c = chain_of(tree, j)
        if j % 3 and j != len(tree) - 1 and len(tree) > 8:
            continue                                          # every third node of a larger tree
        h, l = oracle_rows(ora, history, x[c])
        for got, want, name in ((hid[j], h[-1], "hidden"), (lg[j], l[-1], "logits")):
            d, cos = compare(got, want)
            assert d < TOL_ABS and cos > TOL_COS, (what, j, name, d, cos)


@pytest.mark.parametrize("nodes", [1, 7, 40])
def test_verify_against_the_oracle(side, nodes):
    abi, ora, talker, _ = side
    rng = np.random.default_rng(nodes)
    prompt = [rng.standard_normal((n, 1024)).astype(np.float32) for n in (37, 21)]
    d = abi.DeviceBuffer(prompt[0].nbytes)
    d.upload(prompt[0])
    talker.prefill(d.ptr, 37)                                 # rows 0..36: pages 0, 1 and 2
    pool = Pool(abi, talker, 2, {0: [0, 1, 2]})
    pool.past.copy_(i32([37, 0]))
    # the second prompt goes in as a chain of 21 rows, beside one row of the first request
    first = rng.standard_normal((1, 1024)).astype(np.float32)
    trees, x = [[-1], [j - 1 for j in range(21)]], [first, prompt[1]]
    hid, lg = pool.step(trees, x)
    check(ora, prompt[0], trees[0], first, hid[:1], lg[:1], "one row")
    h, l = oracle_rows(ora, np.zeros((0, 1024), np.float32), prompt[1])
    for got, want in ((hid[1:], h), (lg[1:], l)):
        dmax, cos = compare(got, want)
        assert dmax < TOL_ABS and cos > TOL_COS, ("chain", dmax, cos)
    pool.commit([[0], list(range(21))], talker.kv)
    history = [np.concatenate([prompt[0], first]), prompt[1]]
    # trees on both, then one row each on what was accepted
    for step in range(2):
        trees = [random_tree(rng, nodes), random_tree(rng, max(1, nodes - 3))] if step == 0 else [[-1], [-1]]
        x = [rng.standard_normal((len(t), 1024)).astype(np.float32) for t in trees]
        hid, lg = pool.step(trees, x, spare=2)
        at = 0
        for i, t in enumerate(trees):
            check(ora, history[i], t, x[i], hid[at:at + len(t)], lg[at:at + len(t)], ("request", i, "step", step))
            at += len(t)
        paths = [chain_of(t, len(t) - 1) for t in trees]
        pool.commit(paths, talker.kv)
        history = [np.concatenate([h, xi[p]]) for h, xi, p in zip(history, x, paths)]
    log(f"verify {nodes} nodes: {talker.last_ms():.2f} ms for one row each")


def test_a_row_does_not_depend_on_the_other_requests(side):
    abi, _, talker, _ = side
    rng = np.random.default_rng(5)
    x = [rng.standard_normal((n, 1024)).astype(np.float32) for n in (5, 3, 8)]
    trees = [[-1, 0, 1, 1, 2], [-1, 0, 0], [-1, 0, 1, 2, 3, 4, 5, 6]]
    kv = abi.KvCache(talker.kv.n_layer, 512, 1024)            # a pool of the caller's
    all_h, all_l = Pool(abi, talker, 3, {}).step(trees, x, kv=kv)
    at = 0
    for t, xi in zip(trees, x):
        h, l = Pool(abi, talker, 1, {}).step([t], [xi], kv=kv)
        # (the attention may add a long request's keys in another order: f32 sums)
        assert np.abs(h - all_h[at:at + len(t)]).max() < 1e-3 and np.abs(l - all_l[at:at + len(t)]).max() < 1e-3
        h2, _ = Pool(abi, talker, 1, {}).step([t], [xi], kv=kv, logits=False)
        assert np.array_equal(h, h2)
        at += len(t)


def test_a_refused_request_and_padding_do_not_spoil_the_others(side):
    """A pool whose unwritten rows are NaN, a request that gets no page while it holds a part of one, rows of no request that are NaN:
    the other request's results are those it has alone, and the call succeeds."""
    abi, _, talker, _ = side
    L, rng = talker.kv.n_layer, np.random.default_rng(8)
    pool = torch.full((2, L, 512, 1024), float("nan"), dtype=torch.float16, device="cuda")
    pool[:, :, 16:19] = 0.25                                   # request 1: three cached rows on page 1
    kv = SimpleNamespace(view=abi.KvView(L, 512, 1024, *((C.c_void_p * L)(*(pool[i, l].data_ptr() for l in range(L))) for i in range(2))))
    x = [rng.standard_normal((n, 1024)).astype(np.float32) for n in (5, 20)]
    trees = [[-1, 0, 1, 1, 2], [j - 1 for j in range(20)]]
    p = Pool(abi, talker, 2, {1: [1]})
    p.past.copy_(i32([0, 3]))
    p.free.copy_(i32([1]))                                       # one page: the first request's
    h, l = p.step(trees, x, kv=kv, spare=3, spare_value=float("nan"), status=[0, 1])
    assert torch.isnan(pool[:, :, 19:32]).all() and p.slot.tolist()[5:25] == [-1] * 20
    alone_h, alone_l = Pool(abi, talker, 1, {}).step(trees[:1], x[:1], kv=abi.KvCache(L, 512, 1024))
    assert np.abs(h[:5] - alone_h).max() < 1e-3 and np.abs(l[:5] - alone_l).max() < 1e-3


def test_verify_of_the_most_rows(side):
    """128 rows, the handle's most: two requests' chains of 64, each against the chain's rows one request at a time."""
    abi, _, talker, _ = side
    rng = np.random.default_rng(9)
    x = [rng.standard_normal((64, 1024)).astype(np.float32) for _ in range(2)]
    kv, chain = abi.KvCache(talker.kv.n_layer, 512, 1024), [j - 1 for j in range(64)]
    h, l = Pool(abi, talker, 2, {}).step([chain, chain], x, kv=kv)
    for i in range(2):
        h1, l1 = Pool(abi, talker, 1, {}).step([chain], [x[i]], kv=kv)
        assert np.abs(h[64 * i:64 * i + 64] - h1).max() < TOL_ABS and np.abs(l[64 * i:64 * i + 64] - l1).max() < TOL_ABS


def test_verify_after_a_long_prefill_and_refusals(side):
    """A prefill above 64 rows leaves f16 pairs in the handle's buffers: rows of no request must not read them."""
    abi, _, talker, _ = side
    rng = np.random.default_rng(6)
    p = rng.standard_normal((100, 1024)).astype(np.float32)
    d = abi.DeviceBuffer(p.nbytes)
    d.upload(p)
    talker.prefill(d.ptr, 100)
    pool = Pool(abi, talker, 1, {0: list(range(7))})
    pool.past.copy_(i32([100]))
    hid, lg = pool.step([[-1, 0]], [p[:2]], spare=11)
    assert np.isfinite(hid[:2]).all() and np.isfinite(lg[:2]).all()
    g, b = pool.pages, torch.zeros(64, 1024, device="cuda").data_ptr()

    def refused(status, **kw):
        a = dict(pages=g, max_keys=192, d_rows=b, d_hidden=b, kv=None)
        a.update(kw)
        with pytest.raises(abi.NaviError) as e:
            talker.verify(**a)
        assert e.value.status == status, e.value

    def with_(**kw):
        q = type(g).from_buffer_copy(g)
        for k, v in kw.items():
            setattr(q, k, v)
        return q

    refused(4, d_rows=None)
    refused(4, d_hidden=None)
    refused(4, d_hidden=b + 4)
    refused(4, max_keys=0)
    refused(4, max_keys=513)
    refused(4, pages=with_(n_rows=129))
    refused(4, pages=with_(n_rows=0))
    refused(4, pages=with_(max_new=65))
    refused(4, pages=with_(n_pages=33))
    refused(4, kv=abi.KvCache(1, 512, 1024))
    refused(4, kv=abi.KvCache(talker.kv.n_layer, 511, 1024))
    x = np.full((1, 1024), 1e6, np.float32)                   # leaves the f16 range inside the layers
    x[0, ::2] = np.nan
    with pytest.raises(abi.NaviError) as e:
        pool.step([[-1]], [x])
    assert e.value.status == 4 and "f16 range" in str(e.value)


def nan_pool(abi, L, rows, kept=()):
    """A caller's pool whose rows are NaN but `kept` (rows of K and V that are 0.25), and its view."""
    pool = torch.full((2, L, rows, 1024), float("nan"), dtype=torch.float16, device="cuda")
    for r in kept:
        pool[:, :, r] = 0.25
    return pool, SimpleNamespace(view=abi.KvView(L, rows, 1024, *((C.c_void_p * L)(*(pool[i, l].data_ptr() for l in range(L))) for i in range(2))))


@pytest.mark.parametrize("past,tree,status", [(10000, [-1, 0, 1], 2), (2 ** 31 - 5, [-1, 0, 1], 2), (-5, [-1, 0], 2), (190, [-1, 0, 1], 2), (3, [-1, 0, 2, 1], 3),
                                              (3, [j - 1 for j in range(20)], 1)])
def test_no_refused_request_can_fail_the_call(side, past, tree, status):
    """Whatever a request holds that the plan refused (lengths out of range, bad parents, no pages): NaN in its held pages, cached
    positions included, stays its own, and another request's results are those it has alone."""
    abi, _, talker, _ = side
    L, rng = talker.kv.n_layer, np.random.default_rng(12)
    _, kv = nan_pool(abi, L, 512)
    x = [rng.standard_normal((n, 1024)).astype(np.float32) for n in (5, len(tree))]
    trees = [[-1, 0, 1, 1, 2], tree]
    p = Pool(abi, talker, 2, {1: [1]})
    p.past.copy_(i32([0, past]))
    p.free.copy_(i32([1]))
    h, l = p.step(trees, x, kv=kv, status=[0, status])
    alone_h, alone_l = Pool(abi, talker, 1, {}).step(trees[:1], x[:1], kv=abi.KvCache(L, 512, 1024))
    assert np.abs(h[:5] - alone_h).max() < 1e-3 and np.abs(l[:5] - alone_l).max() < 1e-3
    assert np.isfinite(h).all() and np.isfinite(l).all()


@pytest.mark.parametrize("past,inside", [(509, 3), (512, 0), (600, 0)])
def test_a_request_that_runs_past_the_last_position(side, past, inside):
    """Over a pool with more rows than the talker has positions (512), unwritten ones NaN: the rows past them get no K and V and no slot,
    a commit takes no path over them, and the rows before them and the other request are what they are alone."""
    abi, _, talker, _ = side
    L, rng, rows = talker.kv.n_layer, np.random.default_rng(past), 1024
    x = [rng.standard_normal((n, 1024)).astype(np.float32) for n in (5, 6)]
    trees = [[-1, 0, 1, 1, 2], [j - 1 for j in range(6)]]
    held = list(range(8, 8 + -(-past // PAGE)))

    def step(trees, x):
        pool, kv = nan_pool(abi, L, rows, [8 * PAGE + t for t in range(past)])
        p = Pool(abi, talker, 2, {})
        p.t = SimpleNamespace(params=talker.params, verify=lambda pages, keys, *a, **k: talker.verify(pages, 512, *a, **k))
        p.n_pages, p.blocks = rows // PAGE, 48
        p.table, p.held = i32([[-1] * 48, held + [-1] * (48 - len(held))]), i32([0, len(held)])
        p.free, p.stack = i32([6]), i32(list(range(6)) + [0] * (p.n_pages - 6))
        p.past.copy_(i32([0, past]))
        h, l = p.step(trees, x, kv=kv)
        return p, pool, kv, h, l

    p, pool, kv, h, l = step(trees, x)
    assert np.isfinite(h).all() and np.isfinite(l).all()
    slot = p.slot.tolist()
    assert all(s >= 0 for s in slot[:5 + inside]) and slot[5 + inside:] == [-1] * (6 - inside)
    alone_h, alone_l = Pool(abi, talker, 1, {}).step(trees[:1], x[:1], kv=abi.KvCache(L, 512, 1024))
    assert np.abs(h[:5] - alone_h).max() < 1e-3 and np.abs(l[:5] - alone_l).max() < 1e-3
    if inside:
        _, _, _, h1, l1 = step([[-1], trees[1][:inside]], [x[0][:1], x[1][:inside]])
        assert np.abs(h[5:5 + inside] - h1[1:]).max() < 1e-3 and np.abs(l[5:5 + inside] - l1[1:]).max() < 1e-3
    written = int(torch.isfinite(pool[0, 0, :, 0]).sum())
    assert written == past + 5 + inside
    p.pages.status = p.status.data_ptr()
    for accept, done in ((inside, 0), (inside + 1, 2)):
        path, acc, now, out = i32([list(range(8))] * 2), i32([1, accept]), i32([0, 0]), i32([9, 9])
        torch.cuda.synchronize()
        abi.kv_commit(p.pages, list(kv.view.k[:L]), list(kv.view.v[:L]), 1024, path.data_ptr(), 8, acc.data_ptr(), now.data_ptr(), out.data_ptr(),
                      stream=abi.lib().navi_device_stream())
        torch.cuda.synchronize()
        assert out.tolist() == [0, done] and now.tolist() == [1, past + (accept if done == 0 else 0)]


def test_verify_of_512_rows(side):
    """Eight requests' chains of 64, each against the chain one request at a time."""
    abi, _, _, W = side
    talker, rng = abi.Talker(W, max_prompt_tokens=512, max_positions=512), np.random.default_rng(10)
    x = [rng.standard_normal((64, 1024)).astype(np.float32) for _ in range(8)]
    kv, chain = abi.KvCache(talker.kv.n_layer, 512, 1024), [j - 1 for j in range(64)]
    h, l = Pool(abi, talker, 8, {}).step([chain] * 8, x, kv=kv)
    assert np.isfinite(h).all() and np.isfinite(l).all()
    for i in (0, 3, 7):
        h1, l1 = Pool(abi, talker, 1, {}).step([chain], [x[i]], kv=kv)
        assert np.abs(h[64 * i:64 * i + 64] - h1).max() < TOL_ABS and np.abs(l[64 * i:64 * i + 64] - l1).max() < TOL_ABS
