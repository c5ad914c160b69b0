"""The paged K/V operators on the GPU against their definitions in 64 bits (tests/kv_util.py)."""
import numpy as np
import pytest
import torch

from kv_util import HALF_STEP, TYPE, Step, ancestors, plan_reference, random_tree, signed, stream
from navi_amd import abi

pytestmark = pytest.mark.gpu
TOUCH = 2 ** 30 + 7                             # what an entry that nobody writes holds


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int64).astype(np.int32), dtype=torch.int32, device="cuda")


# ---- plan ----------------------------------------------------------------------------------------

def run_plan(past, new, parent, table, held, free, top, *, page, n_pages, n_rows, max_new, inplace=False, repeat=1):
    n, blocks = len(past), len(table[0])
    t_in, h_in, f_in, stack, n_past, n_new = i32(table), i32(held), i32([top]), i32(free), i32(past), i32(new)
    for _ in range(repeat):
        t, h, f = (t_in, h_in, f_in) if inplace else (torch.full_like(t_in, TOUCH), torch.full_like(h_in, TOUCH), torch.full_like(f_in, TOUCH))
        cu, status, scratch = i32([TOUCH] * (n + 1)), i32([TOUCH] * n), torch.empty(4 * n, dtype=torch.int32, device="cuda")
        slot, pos = i32([TOUCH] * n_rows), i32([TOUCH] * n_rows)
        mask = torch.full((n_rows,), TOUCH, dtype=torch.int64, device="cuda")
        par = None if parent is None else i32(parent)
        pages = abi.KvPages(n, page, n_pages, blocks, n_rows, max_new, t.data_ptr(), n_past.data_ptr(), cu.data_ptr(), slot.data_ptr(), pos.data_ptr(),
                            mask.data_ptr())
        abi.kv_plan(pages, n_new=n_new.data_ptr(), parent=None if par is None else par.data_ptr(), table_in=t_in.data_ptr(), held_in=h_in.data_ptr(),
                    free_in=f_in.data_ptr(), free_pages=stack.data_ptr(), held=h.data_ptr(), free=f.data_ptr(), status=status.data_ptr(),
                    scratch=scratch.data_ptr(), stream=stream())
        torch.cuda.synchronize()
    return {k: v.tolist() for k, v in dict(table=t, held=h, n_free=f, free=stack, cu=cu, slot=slot, pos=pos, mask=mask, status=status).items()}


def same_plan(got, want):
    for k, w in want.items():
        g = got[k]
        w = [TOUCH if x is None else x for x in w] if k in ("slot", "pos", "mask") else w
        assert g == w, (k, next((i, a, b) for i, (a, b) in enumerate(zip(g, w)) if a != b))


def plan_case(rng, n, page, most, tree, *, spare, past_most=300, spoil=0):
    past = [int(rng.integers(0, past_most)) for _ in range(n)]
    new = [int(rng.integers(-1, most + 1)) for _ in range(n)]
    held = [-(-p // page) + int(rng.integers(0, 2)) for p in past]
    blocks = max(max(held), max(-(-(p + max(c, 0)) // page) for p, c in zip(past, new))) + 1
    n_pages = sum(held) + spare
    order = rng.permutation(n_pages).tolist()
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-1] * (blocks - h))
        at += h
    free = order[at:] + [-7] * (n_pages - spare)
    parent = [p for c in new for p in random_tree(rng, max(c, 0), roots=int(rng.integers(1, 4)))] if tree else None
    for _ in range(spoil):
        i = int(rng.integers(0, n))
        what = int(rng.integers(0, 5 if tree else 4))
        if what == 0:
            past[i] = -1 - int(rng.integers(0, 5))
        elif what == 1:
            past[i] = blocks * page + 1 if rng.integers(0, 2) else 2 ** 31 - 1
        elif what == 2:
            held[i] = blocks + 1 if rng.integers(0, 2) else -1
        elif what == 3 and new[i] > 0:
            pass                                  # rows past n_rows come from the caller's n_rows
        elif parent:
            parent[int(rng.integers(0, len(parent)))] = int(rng.choice([-2, 63, 2 ** 31 - 1, 40]))
    rows = sum(max(c, 0) for c in new)
    return dict(past=past, new=new, parent=parent, table=table, held=held, free=free, top=spare, page=page, n_pages=n_pages, n_rows=rows + 5,
                max_new=max(most, 1))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("n,page,most,tree,spare,spoil", [
    (1, 16, 1, False, 4, 0), (1, 1, 64, True, 70, 0), (3, 7, 64, True, 40, 0), (5, 16, 20, False, 3, 0), (40, 16, 64, True, 300, 0), (40, 8, 9, True, 20, 4),
    (200, 16, 5, False, 1000, 9), (1100, 4, 3, True, 300, 30), (2500, 32, 2, False, 3000, 40), (6, 16, 3000, False, 1200, 0), (9, 64, 64, True, 0, 0)])
def test_plan(n, page, most, tree, spare, spoil, inplace):
    rng = np.random.default_rng(n * 1000 + page)
    c = plan_case(rng, n, page, most, tree, spare=spare, spoil=spoil)
    if spoil > 20 and c["parent"]:
        c["parent"] += [0] * 8
    same_plan(run_plan(inplace=inplace, **c), plan_reference(**c))


def test_plan_rows_past_the_arrays_are_refused_and_left():
    c = plan_case(np.random.default_rng(3), 12, 16, 9, False, spare=50)
    c["n_rows"] = sum(max(x, 0) for x in c["new"]) // 2
    same_plan(run_plan(**c), plan_reference(**c))
    c["n_rows"] = 0
    same_plan(run_plan(**c), plan_reference(**c))


def test_plan_more_rows_than_the_step_allows():
    c = plan_case(np.random.default_rng(4), 8, 16, 30, True, spare=50)
    c["max_new"] = 11
    want = plan_reference(**c)
    assert 2 in want["status"] and 0 in want["status"]
    same_plan(run_plan(**c), want)
    c["parent"] = None
    c["new"][2] = 2 ** 31 - 1                                    # its rows do not fit, nor do those after it
    same_plan(run_plan(**c), plan_reference(**c))


def test_plan_full_stack_and_bad_counts():
    c = plan_case(np.random.default_rng(5), 20, 8, 6, False, spare=9)
    for top in (-3, c["n_pages"] - 2, c["n_pages"] + 5):         # pushes past the stack's end are dropped
        c["top"] = min(max(top, 0), c["n_pages"])
        c["free"] = list(np.random.default_rng(1).permutation(c["n_pages"]))
        same_plan(run_plan(**{**c, "top": top}), plan_reference(**c))


def test_plan_page_of_everything_and_long_positions():
    top = 2 ** 31 - 1
    c = dict(past=[top - 3, 5, top - 3], new=[3, 2, 4], parent=None, table=[[0], [1], [0]], held=[1, 1, 1], free=[0], top=0, page=top, n_pages=1, n_rows=9, max_new=4)
    want = plan_reference(**c)
    assert want["status"] == [0, 0, 2] and want["slot"][3] == -1   # page 1 is not of the pool
    same_plan(run_plan(**c), want)


def test_plan_again_on_the_same_state_is_the_same():
    c = plan_case(np.random.default_rng(6), 30, 16, 64, True, spare=120)
    same_plan(run_plan(repeat=3, **c), plan_reference(**c))


# ---- append --------------------------------------------------------------------------------------

@pytest.mark.parametrize("x,q,cache", [("f32", "f32", "f16"), ("f32", "f16", "f16"), ("f16", "f16", "f16"), ("bf16", "bf16", "bf16"),
                                       ("f32", "f32", "bf16"), ("bf16", "f32", "bf16"), ("f32", "bf16", "bf16"), ("f16", "f32", "f16")])
@pytest.mark.parametrize("heads,kv,dim,rows,norm,rot,pad", [(16, 8, 128, 1, True, True, 0), (16, 16, 64, 37, True, True, 8), (8, 1, 128, 130, False, True, 16),
                                                          (3, 1, 64, 5, True, False, 0), (4, 2, 128, 9, False, False, 24)])
def test_append(x, q, cache, heads, kv, dim, rows, norm, rot, pad):
    g = torch.Generator().manual_seed(rows)
    n_slots, n_rot, w = 8 * 24, 50, (heads + 2 * kv) * dim
    xs = (torch.randn(rows + 2, w + pad, generator=g) * 3).to(TYPE[x][0])
    qn, kn = 1 + 0.2 * torch.randn(2, dim, generator=g)
    ang = torch.rand(n_rot, dim // 2, generator=g) * 6.3
    turn = torch.cat([ang.cos(), ang.sin()], 1)
    slot = torch.randperm(n_slots, generator=g)[:rows + 2].int()
    pos = torch.randint(0, n_rot, (rows + 2,), generator=g).int()
    if rows > 4:
        slot[1], slot[2], pos[3], pos[4] = -1, n_slots, n_rot, -1
    k0, v0 = (torch.randn(n_slots, kv * dim + pad, generator=g).to(TYPE[cache][0]) for _ in range(2))
    q0 = torch.full((rows + 2, heads * dim + pad), 5.0).to(TYPE[q][0])
    d = [t.cuda() for t in (xs, qn, kn, turn, slot, pos, k0, v0, q0)]
    dx, dqn, dkn, dt, ds, dp, dk, dv, dq = d
    one, cu, mask = i32([[0]]), i32([0, rows]), torch.zeros(rows + 2, dtype=torch.int64, device="cuda")
    pages = abi.KvPages(1, 24, 8, 1, rows + 2, rows, one.data_ptr(), one.data_ptr(), cu.data_ptr(), ds.data_ptr(), dp.data_ptr(), mask.data_ptr())
    abi.kv_append(pages, abi.KvHeads(heads, kv, dim, TYPE[cache][1]), dx.data_ptr(), TYPE[x][1], w + pad, dk.data_ptr(), dv.data_ptr(), kv * dim + pad,
                  dq.data_ptr(), TYPE[q][1], heads * dim + pad, q_norm=dqn.data_ptr() if norm else None, k_norm=dkn.data_ptr() if norm else None, eps=1e-6,
                  rot=dt.data_ptr() if rot else None, n_rot=n_rot if rot else 0, stream=stream())
    torch.cuda.synchronize()
    y = xs[:rows, :w].double().view(rows, heads + 2 * kv, dim)
    big = y.abs().amax(-1, keepdim=True)
    if norm:
        r = ((y * y).mean(-1, keepdim=True) + 1e-6).sqrt()
        wgt = torch.cat([qn.double().expand(heads, dim), kn.double().expand(kv, dim), torch.ones(kv, dim).double()])
        isv = torch.arange(heads + 2 * kv)[:, None] >= heads + kv
        y = torch.where(isv, y, y / r * wgt)
        big = torch.where(isv, big, big / r * wgt.abs().amax(-1, keepdim=True))
    inside = (pos[:rows] >= 0) & (pos[:rows] < n_rot) | (not rot)
    if rot:
        t = turn[pos[:rows].clamp(0, n_rot - 1).long()].double()[:, None]
        a, b = y.chunk(2, -1)
        c, s = t.chunk(2, -1)
        z = torch.cat([a * c - b * s, b * c + a * s], -1)
        y = torch.cat([z[:, :heads + kv], y[:, heads + kv:]], 1)
    # f32 steps: the sum of squares (dim roundings, halved by the root), the root, two products and two of the turn,
    # each 2^-24 of at most twice the row's largest value; then the stored type's half step of the value
    f32 = (dim / 2 + 16) * 2.0 ** -24 * 2 * big

    def near(got, want, extra, kind):
        err = (got.double() - want).abs()
        assert bool((err <= extra + HALF_STEP[kind] * want.abs() + 1e-30 + (2.0 ** -25 if kind == "f16" else 0)).all()), float(err.max())

    gq, gk, gv = dq.cpu(), dk.cpu(), dv.cpu()
    want_q = torch.where(inside[:, None, None], y[:, :heads], 0)
    near(gq[:rows, :heads * dim].view(rows, heads, dim), want_q, f32[:, :heads], q)
    assert bool((gq[rows:] == 5).all()) and bool((gq[:, heads * dim:] == 5).all())
    kept = [r for r in range(rows) if 0 <= slot[r] < n_slots and bool(inside[r])]
    s = slot[kept].long()
    near(gk[s, :kv * dim].view(-1, kv, dim), y[kept, heads:heads + kv], f32[kept, heads:heads + kv], cache)
    near(gv[s, :kv * dim].view(-1, kv, dim), y[kept, heads + kv:], 0, cache)
    rest = torch.ones(n_slots, dtype=torch.bool)
    rest[s] = False
    for got, before in ((gk, k0), (gv, v0)):
        assert torch.equal(got[rest], before[rest]) and torch.equal(got[:, kv * dim:], before[:, kv * dim:])


def test_append_over_its_own_input_and_without_rows():
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(6, 4 * 64, generator=g, device="cuda").half()
    k, v, q = torch.zeros(16, 64, device="cuda").half(), torch.zeros(16, 64, device="cuda").half(), torch.zeros(6, 128, device="cuda").half()
    slot, cu, one, mask = i32(range(6)), i32([0, 6]), i32([0]), torch.zeros(6, dtype=torch.int64, device="cuda")
    heads = abi.KvHeads(2, 1, 64, abi.DT_F16)
    pages = abi.KvPages(1, 16, 1, 1, 6, 6, one.data_ptr(), one.data_ptr(), cu.data_ptr(), slot.data_ptr(), slot.data_ptr(), mask.data_ptr())
    abi.kv_append(pages, heads, x.data_ptr(), 1, 256, k.data_ptr(), v.data_ptr(), 64, q.data_ptr(), 1, 128, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(q, x[:, :128]) and torch.equal(k[:6], x[:, 128:192]) and torch.equal(v[:6], x[:, 192:])
    before = x.clone()
    abi.kv_append(pages, heads, x.data_ptr(), 1, 256, k.data_ptr(), v.data_ptr(), 64, x.data_ptr(), 1, 256, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(x, before)                                # no norm, no rotation: the same values
    abi.kv_append(abi.KvPages(1, 16, 1, 1, 0, 6, one.data_ptr(), one.data_ptr(), cu.data_ptr(), None, None, None), heads, x.data_ptr(), 1, 256, k.data_ptr(),
                  v.data_ptr(), 64, q.data_ptr(), 1, 128, stream=stream())
    torch.cuda.synchronize()


def test_a_step_without_rows():
    """All requests have ended: their pages go back, the row arrays and the rows may be null, nothing else is written."""
    n, blocks = 3, 4
    table, held, free, stack = i32(range(12)), i32([4, 0, 2]), i32([0]), i32([TOUCH] * 12)
    past, new, cu, status, scratch = i32([60, 0, 17]), i32([-1, -1, -1]), i32([7] * 4), i32([7] * 3), i32([0] * 12)
    pages = abi.KvPages(n, 16, 12, blocks, 0, 8, table.data_ptr(), past.data_ptr(), cu.data_ptr(), None, None, None)
    abi.kv_plan(pages, n_new=new.data_ptr(), table_in=table.data_ptr(), held_in=held.data_ptr(), free_in=free.data_ptr(), free_pages=stack.data_ptr(),
                held=held.data_ptr(), free=free.data_ptr(), status=status.data_ptr(), scratch=scratch.data_ptr(), stream=stream())
    heads = abi.KvHeads(4, 2, 64, abi.DT_BF16)
    k = torch.ones(12 * 16, 128, device="cuda").bfloat16()
    abi.kv_append(pages, heads, None, 0, 512, k.data_ptr(), k.data_ptr(), 128, None, 0, 256, stream=stream())
    ws = torch.empty(max(16, abi.tree_workspace(pages, heads, 640)), dtype=torch.uint8, device="cuda")
    abi.tree_attention(pages, heads, None, abi.DT_BF16, 256, k.data_ptr(), k.data_ptr(), 128, 1.0, 640, None, 256, ws.data_ptr(), ws.numel(), stream=stream())
    path, accept, out, st = i32([0] * 3), i32([0] * 3), i32([-5] * 3), i32([9] * 3)
    abi.kv_commit(pages, [k.data_ptr()], [k.data_ptr()], 128, path.data_ptr(), 1, accept.data_ptr(), out.data_ptr(), st.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert table.tolist() == [-1] * 12 and held.tolist() == [0] * 3 and free.tolist() == [6]
    assert stack.tolist()[:6] == [0, 1, 2, 3, 8, 9] and cu.tolist() == [0] * 4 and status.tolist() == [0] * 3
    assert out.tolist() == past.tolist() and st.tolist() == [0] * 3 and bool((k == 1).all())


# ---- attention -------------------------------------------------------------------------------------

KINDS = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past", [0, 1, 15, 31, 32, 33, 63, 127, 128, 129, 300, 1000])
def test_single_token(kind, past):
    Step([(past, [-1])], kind=kind, seed=past).fill().check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim,page", [(16, 8, 128, 16), (16, 16, 64, 16), (8, 1, 128, 7), (12, 2, 64, 33), (5, 1, 64, 1), (32, 8, 128, 256)])
@pytest.mark.parametrize("nodes", [2, 8, 17, 40, 64])
def test_tree(kind, heads, kv, dim, page, nodes):
    rng = np.random.default_rng(nodes)
    Step([(45, random_tree(rng, nodes, roots=2))], kind=kind, heads=heads, kv_heads=kv, dim=dim, page=page, seed=nodes).fill().check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nodes,page", [(1, 16), (5, 24), (64, 64)])
def test_ragged_requests(kind, nodes, page):
    rng = np.random.default_rng(7)
    reqs = [(int(rng.integers(0, 500)), random_tree(rng, int(rng.integers(0, nodes + 1)))) for _ in range(7)]
    reqs = reqs[:3] + [(200, [])] + reqs[3:] + [(0, [-1])]
    s = Step(reqs, kind=kind, page=page, seed=nodes, pad_kv=8, spare_rows=3, spare_blocks=2, max_new=max(nodes, 2)).fill()
    s.check(pad_q=8, pad_o=16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past,nodes", [(4097, 1), (2500, 16), (1800, 64)])
def test_split_over_blocks(kind, past, nodes):
    rng = np.random.default_rng(past)
    s = Step([(past, random_tree(rng, nodes))], kind=kind, heads=4, kv_heads=2, seed=past).fill()
    s.device()
    assert abi.tree_workspace(s.pages(), s.layout(), s.max_keys) > 0
    a = s.check()
    assert torch.equal(a, s.attend(128 ** -0.5)), "the same call twice"


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2, 33, 255, 256, 257, 300])
def test_many_requests(kind, n):
    """Up to 256 requests are cut into chunks, more are not; some long, some short, some without rows."""
    rng = np.random.default_rng(n)
    reqs = [(int(np.exp(rng.uniform(0, 8))) if i % 50 == 1 else int(rng.integers(0, 60)), random_tree(rng, int(rng.integers(0, 4)))) for i in range(n)]
    reqs[0] = (4000, [-1, 0])
    Step(reqs, kind=kind, heads=2, kv_heads=1, dim=64, page=16, seed=n).fill().check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim,nodes,past", [(64, 2, 64, 5, 70), (32, 1, 128, 9, 600), (48, 1, 64, 64, 33), (8, 8, 64, 33, 4000), (6, 2, 128, 43, 1500)])
def test_large_groups_and_row_counts(kind, heads, kv, dim, nodes, past):
    """Query rows that fill several groups of 128, or leave the last of them nearly empty."""
    rng = np.random.default_rng(past)
    Step([(past, random_tree(rng, nodes)), (past // 3, random_tree(rng, 2))], kind=kind, heads=heads, kv_heads=kv, dim=dim, seed=past).fill().check()


@pytest.mark.parametrize("past", [40, 700])
def test_more_keys_than_announced(past):
    s = Step([(past, [-1, 0, 0]), (3, [-1])], heads=4, kv_heads=2, seed=past).fill()
    s.check(max_keys=1)
    s.check(max_keys=300)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past", [0, 50])
def test_rows_that_see_nothing(kind, past):
    s = Step([(past, [-1, 0, 1, 1]), (past, [-1, 0])], kind=kind, heads=4, kv_heads=2).fill()
    s.mask[1] = s.mask[4] = 0                                    # with past 0 those rows see nothing: zeros
    s.mask[2] |= 1 << 63 | 1 << 40                               # bits past the request's rows say nothing
    got = s.check()
    if past == 0:
        assert bool((got[1] == 0).all()) and bool((got[4] == 0).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("past,split", [(20, False), (3000, True)])
def test_what_a_row_does_not_see_has_no_influence(kind, what, past, split):
    parent = [-1, 0, 0, 2, 1]
    s = Step([(past, parent)], kind=kind, heads=4, kv_heads=2, seed=11).fill()
    clean = Step([(past, parent)], kind=kind, heads=4, kv_heads=2, seed=11).fill()
    at = s.slots(0)[past + 2]                                    # node 2: seen by nodes 2 and 3
    s.k[at], s.v[at] = what, what
    got, want = s.attend(0.1), clean.attend(0.1)
    for r in (0, 1, 4):
        assert torch.equal(got[r], want[r]), r
    s = Step([(past, parent)], kind=kind, heads=4, kv_heads=2, seed=11).fill()
    s.v[at, 5] = what                                            # one column of V: the others as they were
    got, col = s.attend(0.1).float().view(5, 4, 128), [c for c in range(128) if c != 5]
    want, tol = clean.expect(0.1)
    assert not bool(torch.isfinite(got[2:4, :2, 5]).any())
    err = np.abs(got[:, :, col].double().numpy() - want[:, :, col])
    assert (err <= tol[:, :, col]).all()
    assert bool(torch.isfinite(got[[0, 1, 4]]).all())


@pytest.mark.parametrize("kind", KINDS)
def test_missing_pages_are_not_seen(kind):
    for bad in (-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1):
        s = Step([(200, [-1, 0]), (30, [-1])], kind=kind, heads=4, kv_heads=2).fill()
        s.table[0, 2] = s.table[0, 7] = s.table[1, 0] = bad
        s.check()
    s = Step([(5, [-1])], kind=kind, heads=4, kv_heads=2).fill()
    s.table[0, 0] = -1
    assert bool((s.check()[0] == 0).all())


@pytest.mark.parametrize("scale", [1e4, 1e-6, 1.0, 1e30])
def test_f32_queries_of_any_size(scale):
    s = Step([(90, [-1, 0, 1])], kind="f32", heads=4, kv_heads=2).fill(scale=scale)
    s.check(scale=1 / (scale * 4))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [8.0, -1.0, 0.0])
def test_sharp_and_flat_scores(kind, scale):
    Step([(333, [-1, 0, 0, 1])], kind=kind, heads=4, kv_heads=2, seed=5).fill().check(scale=scale)


def test_lengths_out_of_range_stay_in_the_table():
    """n_past below zero counts as zero, past the table's columns as the columns' end; rows past max_new stay."""
    s = Step([(40, [-1, 0, 0, 0]), (10, [-1])], heads=4, kv_heads=2, max_new=2).fill()
    got = s.attend(0.1)
    want, tol = s.expect(0.1)
    got = got.double().numpy().reshape(5, 4, 128)
    assert (np.abs(got - want) <= tol)[[0, 1, 4]].all() and (got[2:4] == 7).all()
    s = Step([(40, [-1])], heads=4, kv_heads=2).fill().device()
    out = {}
    for past in (-5, 2 ** 31 - 1):
        s.d_past.fill_(past)
        o = torch.zeros(1, 512, dtype=torch.float16, device="cuda")
        q, k, v = s.q.cuda(), torch.nan_to_num(s.k).cuda(), torch.nan_to_num(s.v).cuda()
        size = abi.tree_workspace(s.pages(), s.layout(), 41)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        abi.tree_attention(s.pages(), s.layout(), q.data_ptr(), 1, 512, k.data_ptr(), v.data_ptr(), s.ld, 0.1, 41, o.data_ptr(), 512, ws.data_ptr(), size,
                           stream=stream())
        torch.cuda.synchronize()
        out[past] = o
    first = s.slots(0)[0]
    v0 = s.v[first].view(2, 1, 128).expand(2, 2, 128).reshape(-1)
    assert torch.equal(out[-5].cpu()[0], v0)                     # one position is left: its V
    assert bool(torch.isfinite(out[2 ** 31 - 1]).all())


def test_fewer_rows_than_the_requests_have():
    """n_rows below cu_rows' end: the rows past it are neither read nor written."""
    s = Step([(40, [-1, 0, 0, 0]), (10, [-1, 0, 1])], heads=4, kv_heads=2).fill()
    want, tol = s.expect(0.1)
    s.device()
    s.n_rows = 5
    q, k, v = s.q[:5].cuda(), s.k.cuda(), s.v.cuda()
    out = torch.full((7, 512), 7.0, dtype=torch.float16, device="cuda")
    abi.tree_attention(s.pages(), s.layout(), q.data_ptr(), 1, 512, k.data_ptr(), v.data_ptr(), s.ld, 0.1, s.max_keys, out.data_ptr(), 512, None, 0, stream=stream())
    torch.cuda.synchronize()
    got = out.cpu().double().numpy().reshape(7, 4, 128)
    assert (np.abs(got - want) <= tol)[:5].all() and (got[5:] == 7).all()


def test_rows_past_four_gigabytes():
    """Slots whose byte offset passes 32 bits and whose element offset passes 31."""
    heads, kv, dim, page, rows = 16, 8, 128, 16, 2_200_000 // 16 * 16
    free, _ = torch.cuda.mem_get_info()
    if free < 12 * 2 ** 30:
        pytest.skip("needs 9 GB of device memory")
    s = Step([(300, [-1, 0, 0])], heads=heads, kv_heads=kv, dim=dim, page=page, seed=2).fill()
    far = rows // page - s.n_pages                               # the same pages at the end of a large pool
    k, v = (torch.empty(rows, kv * dim, dtype=torch.float16, device="cuda") for _ in range(2))
    k[far * page:], v[far * page:] = s.k.cuda(), s.v.cuda()
    want = s.attend(0.09)
    table, n_pages = s.table + np.where(s.table >= 0, far, 0).astype(np.int32), rows // page
    d_table = torch.from_numpy(table).cuda()
    pages = s.pages()
    pages.block_table, pages.n_pages = d_table.data_ptr(), n_pages
    out = torch.zeros(3, heads * dim, dtype=torch.float16, device="cuda")
    size = abi.tree_workspace(pages, s.layout(), s.max_keys)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    abi.tree_attention(pages, s.layout(), s.d_q.data_ptr(), 1, heads * dim, k.data_ptr(), v.data_ptr(), kv * dim, 0.09, s.max_keys, out.data_ptr(),
                       heads * dim, ws.data_ptr(), size, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want)
    # append and commit reach the same rows
    x = torch.randn(3, (heads + 2 * kv) * dim, device="cuda")
    q = torch.empty(3, heads * dim, dtype=torch.float16, device="cuda")
    slot = i32(table[0, (300 + np.arange(3)) // page] * page + (300 + np.arange(3)) % page)
    pages.row_slot = slot.data_ptr()
    abi.kv_append(pages, s.layout(), x.data_ptr(), 0, x.shape[1], k.data_ptr(), v.data_ptr(), kv * dim, q.data_ptr(), 1, heads * dim, stream=stream())
    path, acc, past, status = i32([[0, 2]]), i32([2]), i32([0]), i32([9])
    abi.kv_commit(pages, [k.data_ptr()], [v.data_ptr()], kv * dim, path.data_ptr(), 2, acc.data_ptr(), past.data_ptr(), status.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    half = x.half()
    assert torch.equal(k[slot[1].item()], half[2, 2048:][:1024]) and torch.equal(v[slot[1].item()], half[2, 2048:][1024:])
    assert past.tolist() == [302] and status.tolist() == [0]


# ---- commit ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("layers,kvd,page,kind", [(1, 1024, 16, "f16"), (28, 1024, 16, "bf16"), (40, 64, 7, "f16"), (3, 1032, 1, "f16"), (2, 8, 64, "bf16")])
def test_commit(layers, kvd, page, kind):
    rng = np.random.default_rng(layers)
    reqs = [(int(rng.integers(0, 90)), random_tree(rng, int(c))) for c in (64, 1, 9, 30, 5, 6, 7, 8, 3, 4)]
    s = Step(reqs, page=page, kind=kind, heads=1, kv_heads=1, dim=64).device()
    pool = torch.randint(-2 ** 15, 2 ** 15, (layers, 2, s.n_pages * page, kvd), dtype=torch.int16)
    path, acc, want_past, want_status, want = [], [], [], [], pool.clone()
    for i, c in enumerate(s.count):
        a = int(rng.integers(0, c + 1)) if i else 40
        p = sorted(rng.permutation(c)[:a].tolist())
        row = p + [-9] * (64 - a)
        if i == 4:
            row, a = [1, 0, 2] + [0] * 61, 3                     # does not ascend
        elif i == 5:
            row, a = [1, 1] + [0] * 62, 2                        # the same row twice
        elif i == 6:
            row, a = [3, 7] + [0] * 62, 2                        # leaves the request's rows
        elif i == 7:
            a = 65
        elif i == 8:
            a = -1
        elif i == 9:
            s.table[i, (s.past[i] + 2) // page] = -1
            row, a = [0, 2] + [0] * 62, 2                        # a page that is not there
            s.d_table = i32(s.table)
        good = i not in (4, 5, 6, 7, 8, 9)
        path.append(row)
        acc.append(a)
        want_past.append(s.past[i] + (a if good else 0))
        want_status.append(0 if good else 2)
        if good:
            sl = s.slots(i)[s.past[i]:]
            for j in range(a):
                want[:, :, sl[j]] = pool[:, :, sl[row[j]]]
    d = pool.cuda()
    d_path, d_acc, past, status = i32(path), i32(acc), i32([0] * s.n), i32([-1] * s.n)
    size = pool[0, 0].numel() * 2
    k, v = ([d.data_ptr() + (2 * l + h) * size for l in range(layers)] for h in (0, 1))
    abi.kv_commit(s.pages(), k, v, kvd, d_path.data_ptr(), 64, d_acc.data_ptr(), past.data_ptr(), status.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert past.tolist() == want_past and status.tolist() == want_status
    assert torch.equal(d.cpu(), want)


# ---- streams, graphs, and a step as it is used -------------------------------------------------------

class Server:
    """Requests on one pool, as a program holds them: state on the device, one layer."""

    def __init__(self, n=5, page=8, n_pages=200, blocks=40, rows=160, kind="f16", seed=0):
        self.n, self.page, self.n_pages, self.blocks, self.rows, self.kind = n, page, n_pages, blocks, rows, kind
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.cache = g, TYPE["f16" if kind == "f32" else kind]
        self.k, self.v = (torch.full((n_pages * page, 256), float("nan"), dtype=self.cache[0], device="cuda") for _ in range(2))
        self.table, self.held, self.free, self.stack = i32([[-1] * blocks] * n), i32([0] * n), i32([n_pages]), i32(np.random.default_rng(seed).permutation(n_pages))
        self.past, self.new_past, self.n_new = i32([0] * n), i32([0] * n), i32([0] * n)
        self.cu, self.slot, self.pos, self.status, self.scratch = i32([0] * (n + 1)), i32([0] * rows), i32([0] * rows), i32([0] * n), i32([0] * 4 * n)
        self.mask, self.parent = torch.zeros(rows, dtype=torch.int64, device="cuda"), i32([0] * rows)
        self.path, self.accept, self.done = i32([[0] * 64] * n), i32([0] * n), i32([0] * n)
        angle = torch.arange(400., device="cuda")[:, None] * torch.rand(64, generator=g, device="cuda")
        self.turn = torch.cat([angle.cos(), angle.sin()], 1)
        self.norm = torch.rand(128, generator=g, device="cuda") + 0.5
        self.x = torch.zeros(rows, 8 * 128, device="cuda").to(TYPE[kind][0])
        self.q, self.out = (torch.zeros(rows, 512, device="cuda").to(TYPE[kind][0]) for _ in range(2))
        self.heads = abi.KvHeads(4, 2, 128, self.cache[1])
        self.pages = abi.KvPages(n, page, n_pages, blocks, rows, 64, *(t.data_ptr() for t in (self.table, self.past, self.cu, self.slot, self.pos, self.mask)))
        self.keys = blocks * page
        size = abi.tree_workspace(self.pages, self.heads, self.keys)
        self.ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def plan(self, st):
        abi.kv_plan(self.pages, n_new=self.n_new.data_ptr(), parent=self.parent.data_ptr(), table_in=self.table.data_ptr(), held_in=self.held.data_ptr(),
                    free_in=self.free.data_ptr(), free_pages=self.stack.data_ptr(), held=self.held.data_ptr(), free=self.free.data_ptr(),
                    status=self.status.data_ptr(), scratch=self.scratch.data_ptr(), stream=st)

    def layer(self, st):
        t = TYPE[self.kind][1]
        abi.kv_append(self.pages, self.heads, self.x.data_ptr(), t, 1024, self.k.data_ptr(), self.v.data_ptr(), 256, self.q.data_ptr(), t, 512,
                      q_norm=self.norm.data_ptr(), k_norm=self.norm.data_ptr(), rot=self.turn.data_ptr(), n_rot=400, stream=st)
        abi.tree_attention(self.pages, self.heads, self.q.data_ptr(), t, 512, self.k.data_ptr(), self.v.data_ptr(), 256, 128 ** -0.5, self.keys,
                           self.out.data_ptr(), 512, self.ws.data_ptr(), self.ws.numel(), stream=st)

    def commit(self, st):
        abi.kv_commit(self.pages, [self.k.data_ptr()], [self.v.data_ptr()], 256, self.path.data_ptr(), 64, self.accept.data_ptr(), self.new_past.data_ptr(),
                      self.done.data_ptr(), stream=st)


@pytest.mark.parametrize("kind", KINDS)
def test_steps_as_a_server_runs_them(kind):
    """Several steps of plan, append, attention and commit, with requests that end and start again: every row's
    output against dense attention over the K and V that its own token history gives."""
    rng, s = np.random.default_rng(1), Server(kind=kind)
    history = [[] for _ in range(s.n)]                            # per request: accepted q|k|v rows
    st = stream()
    norm, turn = s.norm.double().cpu(), s.turn.double().cpu()

    def head(x, pos):                                             # [heads][128] normed and turned
        x = x / ((x * x).mean(-1, keepdim=True) + 1e-6).sqrt() * norm
        c, sn = turn[pos].chunk(2)
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * sn, b * c + a * sn], -1)

    for step in range(7):
        trees = [random_tree(rng, int(rng.integers(1, 30)), roots=1) for _ in range(s.n)]
        new = [len(t) for t in trees]
        if step == 4:
            new[2], trees[2] = -1, []                             # ended: its pages go back
        cu = np.concatenate([[0], np.cumsum([len(t) for t in trees])])
        x = torch.randn(s.rows, 1024, generator=s.g, device="cuda").to(s.x.dtype)
        s.x.copy_(x)
        s.n_new.copy_(i32(new))
        s.parent[:cu[-1]] = i32([p for t in trees for p in t])
        s.out.fill_(7)
        s.plan(st)
        s.layer(st)
        path = [[] for _ in trees]
        for i, t in enumerate(trees):
            node = int(rng.integers(0, len(t))) if t else -1
            while node >= 0:
                path[i].insert(0, node)
                node = t[node]
        s.accept.copy_(i32([len(p) for p in path]))
        s.path.copy_(i32([p + [0] * (64 - len(p)) for p in path]))
        s.commit(st)
        torch.cuda.synchronize()
        assert s.status.tolist() == [0] * s.n and s.done.tolist() == [0] * s.n
        xs, out = x.double().cpu(), s.out.double().cpu()
        assert bool((out[cu[-1]:] == 7).all())
        u = HALF_STEP["f16" if kind == "f32" else kind]
        for i, t in enumerate(trees):
            for j in range(len(t)):
                chain, node = [], j
                while node >= 0:
                    chain.insert(0, xs[cu[i] + node])
                    node = t[node]
                seq = torch.stack(history[i] + chain).view(-1, 8, 128)
                q = head(seq[-1, :4], len(seq) - 1)
                q = q if kind == "f32" else q.to(s.x.dtype).double()
                k = torch.stack([head(r[4:6], p) for p, r in enumerate(seq)]).to(s.cache[0]).double()
                v = seq[:, 6:].to(s.cache[0]).double()
                for h in range(4):
                    sc = k[:, h // 2] @ q[h] * 128 ** -0.5
                    p = torch.softmax(sc, 0)
                    want = p @ v[:, h // 2]
                    got = out[cu[i] + j, h * 128:(h + 1) * 128]
                    # a K (or q) that the f32 steps of the append take over a rounding's border is a whole step off: 2u of
                    # each product, so scores 4u of |q| |k| / sqrt(128); p moves by twice that, and rounds by u; out by u
                    ds = 4 * u * float((k[:, h // 2].abs() @ q[h].abs()).max()) * 128 ** -0.5
                    A = p @ v[:, h // 2].abs()
                    assert bool(((got - want).abs() <= A * (2 * ds + u + 1e-5) + u * want.abs()).all()), (step, i, j, h)
        for i, p in enumerate(path):
            history[i] = [] if new[i] < 0 else history[i] + [xs[cu[i] + j] for j in p]
        s.past.copy_(s.new_past)
        if step == 4:
            s.past[2] = 0
            assert s.held.tolist()[2] == 0
        held = sum(s.held.tolist())
        assert held + s.free.item() == s.n_pages
        used = [p for row, h in zip(s.table.tolist(), s.held.tolist()) for p in row[:h]] + s.stack.tolist()[:s.free.item()]
        assert sorted(used) == list(range(s.n_pages)), "a page lost or given twice"


def seeded(s, seed, past):
    rng = np.random.default_rng(seed)
    trees = [random_tree(rng, int(rng.integers(1, 20))) for _ in range(s.n)]
    s.past.copy_(i32(past))
    s.held.zero_()
    s.table.fill_(-1)
    s.free.fill_(s.n_pages)
    s.n_new.copy_(i32([len(t) for t in trees]))
    s.parent.zero_()
    flat = [p for t in trees for p in t]
    s.parent[:len(flat)] = i32(flat)
    s.x.copy_(torch.randn(s.rows, 1024, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(s.x.dtype))
    for t in (s.k, s.v):
        t.copy_(torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda").to(t.dtype))
    s.accept.fill_(1)
    for t in (s.path, s.slot, s.pos, s.mask):                    # (entries past the step's rows stay as they are)
        t.zero_()
    s.out.fill_(7)


def test_on_another_stream_and_the_library_stream():
    want = None
    other = torch.cuda.Stream()
    for st in (stream(), other.cuda_stream, abi.lib().navi_device_stream()):
        abi.device_open()
        s = Server(seed=3)
        seeded(s, 5, [100] * s.n)
        torch.cuda.synchronize()
        st = abi.lib().navi_device_stream() if st is None else st
        s.plan(st)
        s.layer(st)
        s.commit(st)
        torch.cuda.synchronize()
        got = [t.clone() for t in (s.out, s.k, s.v, s.table, s.slot, s.new_past)]
        if want is not None:
            assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in zip(got, want))
        want = got


@pytest.mark.parametrize("kind", KINDS)
def test_over_its_own_queries(kind):
    """d_out = d_q: one row, groups of many, cut and uncut."""
    rng = np.random.default_rng(3)
    for reqs in ([(70, [-1])], [(40, random_tree(rng, 24)), (3, [-1])], [(2500, random_tree(rng, 9))], [(1800, random_tree(rng, 64)), (9, [-1, 0])]):
        s = Step(reqs, kind=kind, spare_rows=1).fill()
        want = s.check()
        s.device()
        q = torch.full((s.n_rows, s.heads * s.dim), 7.0, dtype=s.q.dtype)
        q[:s.rows] = s.q
        q = q.cuda()
        size = abi.tree_workspace(s.pages(), s.layout(), s.max_keys)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        abi.tree_attention(s.pages(), s.layout(), q.data_ptr(), TYPE[kind][1], q.shape[1], s.d_k.data_ptr(), s.d_v.data_ptr(), s.ld, s.dim ** -0.5, s.max_keys,
                           q.data_ptr(), q.shape[1], ws.data_ptr(), size, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(q.cpu(), want)


def test_two_streams_at_once():
    """Two servers' steps on a stream each, enqueued in turn without a wait, workspaces and scratch their own."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    servers = [Server(seed=i) for i in (11, 12)]
    alone = [Server(seed=i) for i in (11, 12)]
    for s in (*servers, *alone):
        seeded(s, 5, [60] * s.n)
    torch.cuda.synchronize()
    for s in alone:
        s.plan(streams[0].cuda_stream)
        for _ in range(6):
            s.layer(streams[0].cuda_stream)
        s.commit(streams[0].cuda_stream)
        torch.cuda.synchronize()
    for part in ("plan", *["layer"] * 6, "commit"):
        for s, st in zip(servers, streams):
            getattr(s, part)(st.cuda_stream)
    torch.cuda.synchronize()
    for a, b in zip(servers, alone):
        for name in ("out", "k", "v", "table", "held", "free", "slot", "pos", "mask", "cu", "new_past"):
            assert torch.equal(torch.nan_to_num(getattr(a, name).float()), torch.nan_to_num(getattr(b, name).float())), name


def test_graphs_replayed_between_eager_work():
    """Two captured graphs (a workspace each) replayed in turn, with eager steps and synchronizations between the replays."""
    eager, a, b = Server(seed=4), Server(seed=4), Server(seed=4)
    graphs = []
    for s in (a, b):
        seeded(s, 1, [30] * s.n)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.plan(stream())
            s.layer(stream())
            s.commit(stream())
        graphs.append(g)
    for seed in range(4):
        for s in (a, b, eager):
            seeded(s, seed + (s is b), [20 + 40 * seed] * s.n)
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for s, at in ((a, seed), (b, seed + 1)):
            seeded(eager, at, [20 + 40 * seed] * eager.n)
            eager.plan(stream())
            eager.layer(stream())
            eager.commit(stream())
            torch.cuda.synchronize()
            for name in ("out", "k", "v", "table", "held", "free", "slot", "pos", "mask", "cu", "new_past"):
                assert torch.equal(getattr(s, name)[:], getattr(eager, name)[:]), (seed, name)
