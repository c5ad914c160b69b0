"""Pools held in e4m3: navi_kv_append's rounding into them and navi_tree_attention's reading of them, against the definitions in
64 bits."""
import numpy as np
import pytest
import torch

from kv_util import HALF_STEP, TYPE, Step, random_tree, stream
from navi_amd import abi

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def codes_of(x):
    """Definition of the rounding: nearest code, past 448 the largest of its sign, NaN kept (as 0x7F)."""
    c = x.clamp(-448, 448).to(F8).view(torch.uint8)
    return torch.where(x.isnan(), torch.tensor(0x7F, dtype=torch.uint8), c)


class F8Step(Step):
    """A step on an e4m3 pool; `kind` is the queries' type, `factors` whether the kv heads have some."""

    def __init__(self, requests, *, factors=True, **kw):
        super().__init__(requests, **kw)
        self.factors = factors

    def fill(self, scale=1.0, spread=40.0):
        g = torch.Generator().manual_seed(int(self.rng.integers(1 << 30)))
        self.k, self.v = (torch.full((self.n_pages * self.page, self.ld), 0x7F, dtype=torch.uint8) for _ in range(2))
        w = self.kv_heads * self.dim
        if not self.factors:
            spread = 1.0
        self.fk, self.fv = (torch.ones(self.kv_heads) if not self.factors else (0.5 + torch.rand(self.kv_heads, generator=g)) / spread for _ in range(2))
        for i in range(self.n):
            s = torch.from_numpy(self.slots(i))
            for x in (self.k, self.v):
                x[s, :w] = codes_of(torch.randn(len(s), w, generator=g) * spread)
        self.q = (torch.randn(self.rows, self.heads * self.dim, generator=g) * scale).to(TYPE[self.kind][0])
        return self

    def layout(self):
        self.d_fk, self.d_fv = self.fk.cuda(), self.fv.cuda()
        return abi.KvHeads(self.heads, self.kv_heads, self.dim, abi.DT_F8E4M3, *((self.d_fk.data_ptr(), self.d_fv.data_ptr()) if self.factors else (None, None)))

    def expect(self, scale):
        """(out, bound) [rows][heads][dim]. With A = sum p |v| / sum p and n keys:
          scores: sums of `dim` f32 products, each rounding at most 2^-24 of sum |q k|; the products with scale and factor and the
            difference to the reference 3 2^-24 of |s| + 24 (in powers of two); an f32 q travels as an f16 pair, 2^-22 of its row's
            largest; p moves by twice that;
          p as a pair: bf16 2^-16, f16 2^-21 and never less than 2^-31 of |v| a key;
          exp2 and the sums over keys in f32: 2^-21 + (n / 8 + 64) 2^-24 of A; the sum's inverse, V's factor and the product 2^-22;
          out: half a step of its type."""
        d, g, u = self.dim, self.heads // self.kv_heads, HALF_STEP[self.kind]
        out, tol = np.zeros((self.rows, self.heads, d)), np.zeros((self.rows, self.heads, d))
        k, v = (x.view(F8).double().numpy() for x in (self.k, self.v))
        fk, fv = self.fk.double().numpy(), self.fv.double().numpy()
        for r in range(self.rows):
            i, t = self.visible(r)
            if not t:
                continue
            t = np.array(t)
            at = self.table[i, t // self.page].astype(np.int64) * self.page + t % self.page
            kk, vv = (x[at, :self.kv_heads * d].reshape(len(t), self.kv_heads, d) * f[:, None] for x, f in ((k, fk), (v, fv)))
            q = self.q[r].double().numpy().reshape(self.heads, d)
            for h in range(self.heads):
                kh, vh = kk[:, h // g], vv[:, h // g]
                sc = kh @ q[h] * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                mag = np.abs(kh) @ np.abs(q[h]) * abs(scale)
                ds = d * 2.0 ** -24 * mag.max() + 3 * 2.0 ** -24 * (np.abs(sc).max() + 24)
                if self.kind == "f32":
                    ds += 2.0 ** -22 * np.abs(q[h]).max() * np.abs(kh).sum(1).max() * abs(scale)
                A = p @ np.abs(vh)
                pair = A * 2.0 ** -16 if self.kind == "bf16" else A * 2.0 ** -21 + 2.0 ** -31 * np.abs(vh).sum(0)
                out[r, h] = p @ vh
                tol[r, h] = A * (2 * ds + 2.0 ** -21 + (len(t) / 8 + 64) * 2.0 ** -24 + 2.0 ** -22) + pair + u * np.abs(out[r, h]) + 1e-30
        return out, tol


def tree(n, seed=0):
    return random_tree(np.random.default_rng(seed), n)


# ---- attention ---------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (4, 2, 128), (6, 1, 128)])
@pytest.mark.parametrize("past,nodes", [(0, 1), (1, 1), (40, 1), (9, 12), (5, 24), (3, 64), (700, 1), (2500, 20), (1800, 64)])
def test_attention(kind, heads, kv, dim, past, nodes):
    """From a row that sees itself alone to 384 query rows a kv head; short calls and long ones that are cut."""
    F8Step([(past, tree(nodes, nodes))], kind=kind, heads=heads, kv_heads=kv, dim=dim, seed=past).fill().check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [1, 7, 24, 64])
def test_ragged_requests(kind, page):
    """Lengths of none and one, requests without rows, odd pages, rows behind the last, wider strides."""
    r = [(0, [-1]), (1, []), (130, tree(9)), (33, [-1]), (300, tree(3)), (0, tree(17)), (64, [])]
    F8Step(r, kind=kind, page=page, heads=8, kv_heads=2, dim=64, seed=page, pad_kv=32, spare_rows=3, spare_blocks=2).fill().check(pad_q=8, pad_o=16)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_no_factors(kind):
    F8Step([(200, tree(5)), (31, [-1])], kind=kind, heads=4, kv_heads=2, dim=128, factors=False).fill(scale=0.2).check()


@pytest.mark.parametrize("scale", [0.0, -0.06, 3.0])
def test_scales(scale):
    F8Step([(90, tree(7))], kind="f32", heads=4, kv_heads=2, dim=64).fill().check(scale=scale)


@pytest.mark.parametrize("nodes", [1, 20, 64])
def test_what_a_row_does_not_see_has_no_influence(nodes):
    """NaN in K and V of drafted rows reaches the rows that see it, in V's columns, and nobody else."""
    def step():
        return F8Step([(50, tree(nodes, 3)), (9, tree(2))], kind="f16", heads=4, kv_heads=2, dim=64, seed=5).fill()
    clean, s = step(), step()
    a = s.slots(0)[50 + nodes - 1]                                # the last node: seen by itself alone
    s.k[a], s.v[a, 3] = 0x7F, 0xFF
    got, want = s.attend(0.125), clean.attend(0.125)
    own = nodes - 1
    rest = [r for r in range(s.rows) if r != own]
    assert torch.equal(got[rest], want[rest])
    assert bool(got[own].isnan().all())
    s = step()
    s.v[a, 3] = 0x7F
    got = s.attend(0.125)
    head = got[own].view(4, 64)
    assert torch.equal(got[rest], want[rest]) and bool(head[:2, 3].isnan().all()) and not bool(head[2:].isnan().any()) and int(head.isnan().sum()) == 2


def test_pages_outside_the_pool_are_not_seen():
    s = F8Step([(200, tree(4))], kind="f32", heads=4, kv_heads=2, dim=128).fill()
    s.table[0, 3], s.table[0, 7] = -1, s.n_pages
    s.check()


def test_a_row_that_sees_nothing_gets_zeros():
    s = F8Step([(0, [-1, -1]), (20, [-1])], kind="f16", heads=4, kv_heads=2, dim=64).fill()
    s.mask[1] = 0
    got = s.check()
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("n,past", [(33, 100), (200, 60), (300, 40)])
def test_many_requests(n, past):
    F8Step([((i * 37) % past, [-1] if i % 3 else tree(2)) for i in range(n)], kind="bf16", heads=4, kv_heads=2, dim=64, seed=n).fill().check()


# ---- append ------------------------------------------------------------------------------------

class Rows:
    """Rows of q|k|v appended to an e4m3 pool whose bytes are 0xA5 before."""

    def __init__(self, x, *, heads, kv, dim, slots, n_slots, pad=0):
        rows = x.shape[0]
        self.i = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0] * 4], [0], [0, rows], slots, list(range(rows)))]
        self.mask = torch.zeros(rows, dtype=torch.int64, device="cuda")
        t, past, cu, slot, pos = (v.data_ptr() for v in self.i)
        self.pages = abi.KvPages(1, n_slots, 1, 4, rows, max(1, rows), t, past, cu, slot, pos, self.mask.data_ptr())
        self.x, self.layout = x.cuda(), (heads, kv, dim)
        self.k, self.v = (torch.full((n_slots, kv * dim + pad), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2))

    def append(self, kind, q_kind, factors=(None, None), **kw):
        heads, kv, dim = self.layout
        f = [None if t is None else t.cuda() for t in factors]
        lay = abi.KvHeads(heads, kv, dim, abi.DT_F8E4M3, *(None if t is None else t.data_ptr() for t in f))
        q = torch.full((self.x.shape[0], heads * dim), 7.0, dtype=TYPE[q_kind][0], device="cuda")
        kw = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
        abi.kv_append(self.pages, lay, self.x.data_ptr(), TYPE[kind][1], self.x.shape[1], self.k.data_ptr(), self.v.data_ptr(), self.k.shape[1], q.data_ptr(),
                      TYPE[q_kind][1], q.shape[1], stream=stream(), **{n: t.data_ptr() if isinstance(t, torch.Tensor) else t for n, t in kw.items()})
        torch.cuda.synchronize()
        return q.cpu(), self.k.cpu(), self.v.cpu()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_every_16_bit_value_rounds_to_its_code(kind):
    """No norm, no rotation, no factors: the codes are the values', infinities saturated, NaN kept."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = torch.cat([torch.zeros(256, 256, dtype=torch.int16), bits.view(256, 256), bits.flip(0).view(256, 256)], 1).view(TYPE[kind][0])
    q, k, v = Rows(x, heads=2, kv=2, dim=128, slots=list(range(256)), n_slots=256).append(kind, kind)
    for got, want in ((k, x[:, 256:512]), (v, x[:, 512:])):
        want = codes_of(want.float())
        nan = want == 0x7F
        assert torch.equal(got & torch.where(nan, 0x7F, 0xFF).to(torch.uint8), want)


def test_f32_values_next_to_every_border():
    """Both neighbours of every code's border and the border itself, each sign: ties go to the even code."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8).view(F8).double()
    edge = ((codes[1:] + codes[:-1]) / 2).float()
    x = torch.cat([edge, torch.nextafter(edge, torch.tensor(0.0)), torch.nextafter(edge, torch.tensor(1e9)),
                   torch.tensor([0.0, 2.0 ** -10, 2.0 ** -40, 1e-45, 448, 463.9, 464, 465, 1e30, float("inf"), float("nan")])])
    x = torch.cat([x, -x])
    n = -(-x.numel() // 64)
    flat = torch.zeros(n * 64)
    flat[:x.numel()] = x
    rows = torch.cat([torch.zeros(n, 64), flat.view(n, 64), flat.view(n, 64)], 1)
    q, k, v = Rows(rows, heads=1, kv=1, dim=64, slots=list(range(n)), n_slots=n).append("f32", "f32")
    want = codes_of(flat.view(n, 64))
    for got in (k, v):
        assert torch.equal(got & torch.where(want == 0x7F, 0x7F, 0xFF).to(torch.uint8), want)


@pytest.mark.parametrize("kind,q_kind", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("f16", "f32"), ("f16", "bf16"), ("bf16", "bf16"), ("bf16", "f32"),
                                         ("bf16", "f16")])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (3, 3, 64)])
def test_append_norms_turns_and_rounds(kind, q_kind, heads, kv, dim):
    """Every pair of types, strides wider than the rows, slots in any order, one row without."""
    g = torch.Generator().manual_seed(dim)
    rows, n_slots = 37, 50
    x = (torch.randn(rows, (heads + 2 * kv) * dim + 8, generator=g) * 2).to(TYPE[kind][0])
    slots = torch.randperm(n_slots, generator=g)[:rows].tolist()
    slots[5] = -1
    f = [(0.5 + torch.rand(kv, generator=g)) / 40 for _ in range(2)]
    qn, kn = (1 + 0.1 * torch.randn(dim, generator=g) for _ in range(2))
    angle = torch.rand(rows, dim // 2, generator=g, dtype=torch.float64) * 6
    rot = torch.cat([angle.cos(), angle.sin()], 1).float()
    q, k, v = Rows(x, heads=heads, kv=kv, dim=dim, slots=slots, n_slots=n_slots, pad=16).append(kind, q_kind, f, q_norm=qn, k_norm=kn, eps=1e-6, rot=rot, n_rot=rows)

    def head(a, w):
        a = a / (a.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        c, s = (t[:, None].double() for t in rot.chunk(2, 1))
        a0, a1 = a.chunk(2, -1)
        return torch.cat([a0 * c - a1 * s, a1 * c + a0 * s], -1)

    y = x[:, :(heads + 2 * kv) * dim].double().view(rows, -1, dim)
    # the norm: dim / 8 sums in a lane, 4 steps, an rsqrt of 2 units, two products; the rotation two products and a sum of
    # values up to twice the result's head: 2^-18 of the largest of the head
    f32 = 2.0 ** -18
    want = head(y[:, :heads], qn)
    off = (q.double().view(rows, heads, dim) - want).abs()
    assert bool((off <= HALF_STEP[q_kind] * want.abs() + f32 * want.abs().amax(-1, keepdim=True)).all())
    for got, full, fac in ((k, head(y[:, heads:heads + kv], kn), f[0]), (v, y[:, heads + kv:], f[1])):
        want = (full / fac.double()[:, None]).clamp(-448, 448)
        for r, s in enumerate(slots):
            if s < 0:
                continue
            c = got[s, :kv * dim].view(F8).double().view(kv, dim)
            # half a step: 2^-4 of the value, 2^-10 below the least normal one; the f32 value before it, and its quotient
            tol = want[r].abs() * 2.0 ** -4 + 2.0 ** -10 + 2 * f32 * want[r].abs().amax(-1, keepdim=True)
            assert bool(((c - want[r]).abs() <= tol).all()), (r, s)
        untouched = torch.ones(n_slots, dtype=torch.bool)
        untouched[[s for s in slots if s >= 0]] = False
        assert bool((got[untouched] == 0xA5).all()) and bool((got[:, kv * dim:] == 0xA5).all())


def test_append_in_place_and_rows_out_of_range():
    """q over x; a slot past the pool and a position past the rotation store nothing, and the latter loses its slot."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 4 * 64, generator=g)
    rot = torch.cat([torch.ones(3, 32), torch.zeros(3, 32)], 1).cuda()
    s = Rows(x, heads=2, kv=1, dim=64, slots=[2, 9, 0, 1], n_slots=4)
    lay = abi.KvHeads(2, 1, 64, abi.DT_F8E4M3, None, None)
    abi.kv_append(s.pages, lay, s.x.data_ptr(), 0, 256, s.k.data_ptr(), s.v.data_ptr(), 64, s.x.data_ptr(), 0, 256, rot=rot.data_ptr(), n_rot=3, stream=stream())
    torch.cuda.synchronize()
    k = s.k.cpu()
    assert torch.equal(k[[2, 0]], codes_of(x[[0, 2], 128:192])) and bool((k[[1, 3]] == 0xA5).all())
    assert s.i[3].tolist() == [2, 9, 0, -1]
    got = s.x.cpu()
    assert torch.equal(got[:3, :128], x[:3, :128]) and bool((got[3, :128] == 0).all()) and torch.equal(got[:, 128:], x[:, 128:])


# ---- a step ------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 128])
def test_append_attend_commit(dim):
    """Plan, append, attend, commit: what was appended is what is seen, and a commit moves it (rows of ld_kv bytes are ld_kv / 2 of the
    two-byte elements that it counts)."""
    g = torch.Generator().manual_seed(dim)
    heads, kv, page, past, parents = 4, 2, 8, 21, [-1, 0, 0, 1, 2, 4]
    rows, n_pages = past + len(parents), 6
    lay_f = [(0.5 + torch.rand(kv, generator=g)).cuda() / 40 for _ in range(2)]
    lay = abi.KvHeads(heads, kv, dim, abi.DT_F8E4M3, *(t.data_ptr() for t in lay_f))
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")
    t = dict(table=z(1, n_pages) - 1, past=z(1), cu=z(2), slot=z(rows), pos=z(rows), status=z(1), held=z(1), free=z(1) + n_pages,
             stack=torch.tensor([3, 0, 5, 1, 4, 2], dtype=torch.int32, device="cuda"), new=z(1), parent=z(rows), scratch=z(4), out=z(1), done=z(1))
    t["mask"] = torch.zeros(rows, dtype=torch.int64, device="cuda")
    p = {n: v.data_ptr() for n, v in t.items()}
    pages = abi.KvPages(1, page, n_pages, n_pages, rows, 64, *(p[n] for n in ("table", "past", "cu", "slot", "pos", "mask")), p["status"])
    w = kv * dim
    k, v = (torch.full((n_pages * page, w), 0x7F, dtype=torch.uint8, device="cuda") for _ in range(2))
    x = torch.randn(rows, (heads + 2 * kv) * dim, generator=g).half().cuda()
    out = torch.zeros(rows, heads * dim, dtype=torch.float16, device="cuda")

    def step(n, par, x):
        t["new"].fill_(n)
        if par is not None:
            t["parent"][:n] = torch.tensor(par, dtype=torch.int32)
        abi.kv_plan(pages, n_new=p["new"], parent=None if par is None else p["parent"], table_in=p["table"], held_in=p["held"], free_in=p["free"], free_pages=p["stack"],
                    held=p["held"], free=p["free"], status=p["status"], scratch=p["scratch"], stream=stream())
        q = torch.zeros(rows, heads * dim, dtype=torch.float16, device="cuda")
        abi.kv_append(pages, lay, x.data_ptr(), abi.DT_F16, x.shape[1], k.data_ptr(), v.data_ptr(), w, q.data_ptr(), abi.DT_F16, q.shape[1], stream=stream())
        ws = torch.empty(abi.tree_workspace(pages, lay, 64), dtype=torch.uint8, device="cuda")
        abi.tree_attention(pages, lay, q.data_ptr(), abi.DT_F16, q.shape[1], k.data_ptr(), v.data_ptr(), w, dim ** -0.5, 64, out.data_ptr(), out.shape[1],
                           ws.data_ptr(), ws.numel(), stream=stream())
        torch.cuda.synchronize()
        return q[:n].cpu(), out[:n].cpu()

    def want(q, keys):
        """A row over the rounded rows `keys` of x."""
        y = x.cpu().double().view(rows, -1, dim)[keys]
        kk, vv = (codes_of((y[:, a:b] / f.cpu().double()[:, None]).float()).view(F8).double() * f.cpu().double()[:, None]
                  for a, b, f in ((heads, heads + kv, lay_f[0]), (heads + kv, heads + 2 * kv, lay_f[1])))
        o = []
        for h in range(heads):
            s = torch.softmax(kk[:, h // 2] @ q.double().view(heads, dim)[h] * dim ** -0.5, 0)
            o.append(s @ vv[:, h // 2])
        return torch.cat(o)

    _, _ = step(past, None, x[:past].contiguous())                # a prompt
    t["past"].fill_(past)
    q, got = step(len(parents), parents, x[past:].contiguous())   # a tree
    # the f32 quotient may fall to the other side of a code's border than the 64-bit one: 2^-3 of one value of V or K in a few thousand
    for r, keys in ((0, [0]), (3, [0, 1, 3]), (5, [0, 2, 4, 5])):
        off = (got[r].double() - want(q[r], list(range(past)) + [past + a for a in keys])).abs().max()
        assert off <= 2.0 ** -8, (r, off)
    path, acc = torch.tensor([[0, 2, 4, 5]], dtype=torch.int32, device="cuda"), z(1) + 4
    abi.kv_commit(pages, [k.data_ptr()], [v.data_ptr()], w // 2, path.data_ptr(), 4, acc.data_ptr(), p["out"], p["done"], stream=stream())
    torch.cuda.synchronize()
    assert t["out"].tolist() == [past + 4] and t["done"].tolist() == [0]
    t["past"].fill_(past + 4)
    rows_of = list(range(past)) + [past + a for a in (0, 2, 4, 5)]
    q, got = step(1, [-1], x[:1].contiguous())
    assert (got[0].double() - want(q[0], rows_of + [0])).abs().max() <= 2.0 ** -8


def test_pages_past_32_bits():
    """The same step in pages at the start of a pool of 5 GB and at its end: K, V and the attention alike."""
    g = torch.Generator().manual_seed(5)
    heads, kv, dim, page, n_pages, rows = 16, 8, 128, 16, 330_000, 60
    w = kv * dim
    assert n_pages * page * w > 1 << 32
    k, v = (torch.empty(n_pages * page, w, dtype=torch.uint8, device="cuda") for _ in range(2))
    x = torch.randn(rows, (heads + 2 * kv) * dim, generator=g).bfloat16().cuda()
    lay = abi.KvHeads(heads, kv, dim, abi.DT_F8E4M3, None, None)
    got = []
    for table in ([0, 1, 2, 3], [n_pages - 1, n_pages - 3, n_pages - 2, n_pages - 4]):
        t = torch.tensor(table, dtype=torch.int32)
        at = torch.arange(rows)
        slot = (t[at // page] * page + at % page).int()
        d = [a.int().cuda() for a in (t, torch.tensor([0]), torch.tensor([0, rows]), slot, at)]
        mask = torch.tensor([(1 << (r + 1)) - 1 for r in range(rows)], dtype=torch.int64, device="cuda")
        pages = abi.KvPages(1, page, n_pages, 4, rows, 64, *(a.data_ptr() for a in d), mask.data_ptr())
        q = torch.zeros(rows, heads * dim, dtype=torch.bfloat16, device="cuda")
        out = torch.full_like(q, 7.0)
        abi.kv_append(pages, lay, x.data_ptr(), abi.DT_BF16, x.shape[1], k.data_ptr(), v.data_ptr(), w, q.data_ptr(), abi.DT_BF16, q.shape[1], stream=stream())
        ws = torch.empty(abi.tree_workspace(pages, lay, rows), dtype=torch.uint8, device="cuda")
        abi.tree_attention(pages, lay, q.data_ptr(), abi.DT_BF16, q.shape[1], k.data_ptr(), v.data_ptr(), w, dim ** -0.5, rows, out.data_ptr(), out.shape[1], ws.data_ptr(),
                           ws.numel(), stream=stream())
        path, acc, past, done = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[1, 4, 59]], [3], [9], [9]))
        abi.kv_commit(pages, [k.data_ptr()], [v.data_ptr()], w // 2, path.data_ptr(), 3, acc.data_ptr(), past.data_ptr(), done.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert past.tolist() == [3] and done.tolist() == [0]
        got.append([out.cpu()] + [c[slot.long().cuda()].cpu() for c in (k, v)])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    want = codes_of(x.cpu().float().view(rows, -1, dim)[:, heads:heads + kv].reshape(rows, w))
    order = [1, 4, 59] + list(range(3, rows))
    assert torch.equal(got[0][1], want[order])
