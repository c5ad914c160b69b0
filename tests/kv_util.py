"""Shared by the tests of the paged K/V operators: steps of requests on a pool of pages built on the
host, the operators' definitions in 64 bits, and the bounds their rounding allows."""
from __future__ import annotations

import numpy as np
import torch

from navi_amd import abi

TYPE = {"f32": (torch.float32, abi.DT_F32), "f16": (torch.float16, abi.DT_F16), "bf16": (torch.bfloat16, abi.DT_BF16)}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def stream():
    return torch.cuda.current_stream().cuda_stream


def ancestors(parent):
    bits = []
    for j, p in enumerate(parent):
        bits.append((bits[p] if p >= 0 else 0) | 1 << j)
    return bits


def signed(x):
    return x - (1 << 64) if x >> 63 else x


def random_tree(rng, n, roots=1):
    return [-1 if j < roots else int(rng.integers(max(0, j - 6), j)) for j in range(n)]


class Step:
    """Requests (n_past, parents) on a pool; every cache row that belongs to nobody is NaN."""

    def __init__(self, requests, *, page=16, heads=16, kv_heads=8, dim=128, kind="f16", seed=0, pad_kv=0, spare_rows=0, spare_blocks=0,
                 max_new=None, pages_extra=3):
        rng = np.random.default_rng(seed)
        self.rng, self.page, self.heads, self.kv_heads, self.dim, self.kind = rng, page, heads, kv_heads, dim, kind
        self.past, self.parents = [p for p, _ in requests], [t for _, t in requests]
        self.count = [len(t) for t in self.parents]
        self.n = len(requests)
        need = [-(-(p + c) // page) for p, c in zip(self.past, self.count)]
        self.n_pages = sum(need) + pages_extra
        self.blocks = max(max(need), 1) + spare_blocks
        order = rng.permutation(self.n_pages)
        self.table = np.full((self.n, self.blocks), -1, np.int32)
        at = 0
        for i, c in enumerate(need):
            self.table[i, :c] = order[at:at + c]
            at += c
        self.cu = np.concatenate([[0], np.cumsum(self.count)]).astype(np.int32)
        self.rows, self.n_rows = int(self.cu[-1]), int(self.cu[-1]) + spare_rows
        self.mask = [b for t in self.parents for b in ancestors(t)]
        self.max_new = max_new or max(1, max(self.count))
        self.max_keys = max(1, max(p + c for p, c in zip(self.past, self.count)))
        self.ld = kv_heads * dim + pad_kv
        self.cache = "f16" if kind == "f32" else kind

    def slots(self, i):
        t = np.arange(self.past[i] + self.count[i])
        return self.table[i, t // self.page].astype(np.int64) * self.page + t % self.page

    def fill(self, scale=1.0):
        """K, V (torch, CPU, cache type; NaN outside the requests) and q (f32 or cache type)."""
        t = TYPE[self.cache][0]
        g = torch.Generator().manual_seed(int(self.rng.integers(1 << 30)))
        self.k, self.v = (torch.full((self.n_pages * self.page, self.ld), float("nan"), dtype=t) for _ in range(2))
        w = self.kv_heads * self.dim
        for i in range(self.n):
            s = torch.from_numpy(self.slots(i))
            for x in (self.k, self.v):
                x[s, :w] = torch.randn(len(s), w, generator=g).to(t)
        self.q = (torch.randn(self.rows, self.heads * self.dim, generator=g) * scale).to(TYPE[self.kind][0])
        return self

    def device(self):
        self.d_table, self.d_past, self.d_cu = (torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()
                                                for a in (self.table, np.array(self.past), self.cu))
        extra = self.n_rows - self.rows
        self.d_mask = torch.tensor([signed(b) for b in self.mask] + [-1] * extra, dtype=torch.int64, device="cuda")
        self.d_slot = torch.full((self.n_rows,), -1, dtype=torch.int32, device="cuda")
        self.d_pos = torch.zeros(self.n_rows, dtype=torch.int32, device="cuda")
        return self

    def pages(self):
        return abi.KvPages(self.n, self.page, self.n_pages, self.blocks, self.n_rows, self.max_new, self.d_table.data_ptr(),
                           self.d_past.data_ptr(), self.d_cu.data_ptr(), self.d_slot.data_ptr(), self.d_pos.data_ptr(), self.d_mask.data_ptr())

    def layout(self):
        return abi.KvHeads(self.heads, self.kv_heads, self.dim, TYPE[self.cache][1])

    def attend(self, scale, *, pad_q=0, pad_o=0, max_keys=None, ws=None):
        """The operator on the GPU: [n_rows][heads * dim + pad_o], filled with 7 before."""
        self.device()
        w = self.heads * self.dim
        q = torch.full((self.n_rows, w + pad_q), 3.0, dtype=self.q.dtype)
        q[:self.rows, :w] = self.q
        self.d_q, self.d_k, self.d_v = q.cuda(), self.k.cuda(), self.v.cuda()
        out = torch.full((self.n_rows, w + pad_o), 7.0, dtype=self.q.dtype, device="cuda")
        pages, keys = self.pages(), max_keys or self.max_keys
        size = abi.tree_workspace(pages, self.layout(), keys)
        ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda") if ws is None else ws
        abi.tree_attention(pages, self.layout(), self.d_q.data_ptr(), TYPE[self.kind][1], w + pad_q, self.d_k.data_ptr(), self.d_v.data_ptr(),
                           self.ld, scale, keys, out.data_ptr(), w + pad_o, ws.data_ptr(), size, stream=stream())
        torch.cuda.synchronize()
        return out.cpu()

    def visible(self, r):
        """(request, positions that row r sees and whose page is in the pool)."""
        i = int(np.searchsorted(self.cu[1:], r, side="right"))
        t = list(range(self.past[i])) + [self.past[i] + a for a in range(min(self.count[i], 64)) if self.mask[r] >> a & 1]
        return i, [p for p in t if 0 <= self.table[i, p // self.page] < self.n_pages]

    def expect(self, scale):
        """(out, bound) [rows][heads][dim] in 64 bits: the definition, and how far the kernel's roundings
        may take it: with u half a step of q's type and A = sum p |v| / sum p,
          scores: f32 sums of `dim` products, each of the running sums' roundings at most 2^-24 of sum |q k|; the
            product with the scale and the difference to the reference, 2^-23 of |s| + 24 (in powers of two);
            f32 q travels as an f16 pair: 2^-22 of its row's largest value;
          p: u (a pair: 2^-22), exp2 2^-22; sums over keys: one rounding a product of 8 or more keys and 64 in joins;
          out: u."""
        d, g = self.dim, self.heads // self.kv_heads
        u = HALF_STEP[self.kind]
        out, tol = np.zeros((self.rows, self.heads, d)), np.zeros((self.rows, self.heads, d))
        k, v = self.k.double().numpy(), self.v.double().numpy()
        for r in range(self.rows):
            i, t = self.visible(r)
            if not t:
                continue
            t = np.array(t)
            s = self.table[i, t // self.page].astype(np.int64) * self.page + t % self.page
            kk, vv = (x[s, :self.kv_heads * d].reshape(len(t), self.kv_heads, d) for x in (k, v))
            q = self.q[r].double().numpy().reshape(self.heads, d)
            for h in range(self.heads):
                kh, vh = kk[:, h // g], vv[:, h // g]
                sc = kh @ q[h] * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                o = p @ vh
                mag = np.abs(kh) @ np.abs(q[h]) * abs(scale)
                ds = d * 2.0 ** -24 * mag.max() + 2.0 ** -23 * (np.abs(sc).max() + 24)
                if self.kind == "f32":
                    ds += 2.0 ** -22 * np.abs(q[h]).max() * np.abs(kh).sum(1).max() * abs(scale)
                pu = 2.0 ** -22 if self.kind == "f32" else u
                A = p @ np.abs(vh)
                out[r, h] = o
                tol[r, h] = A * (2 * ds + pu + 2.0 ** -21 + (len(t) / 8 + 64) * 2.0 ** -24) + u * np.abs(o) + 1e-30
        return out, tol

    def check(self, scale=None, **kw):
        scale = self.dim ** -0.5 if scale is None else scale
        got = self.attend(scale, **kw)
        want, tol = self.expect(scale)
        w = self.heads * self.dim
        rows = got[:self.rows, :w].double().numpy().reshape(want.shape)
        ok = np.abs(rows - want) <= tol                          # rows that see nothing: 0 within 0
        assert ok.all(), (np.argwhere(~ok)[:4], rows[~ok][:4], want[~ok][:4], tol[~ok][:4])
        assert bool((got[self.rows:] == 7).all()) and bool((got[:, w:] == 7).all()), "wrote outside its rows"
        return got


def plan_reference(past, new, parent, table, held, free, top, *, page, n_pages, n_rows, max_new):
    """navi_kv_plan's definition on the host: every result as a list, row_* with None where nothing is written."""
    n, blocks = len(past), len(table[0])
    table, held, free = [list(t) for t in table], list(held), list(free)
    status, cu, bad = [0] * n, [], []
    at = 0
    for i in range(n):
        count = max(new[i], 0)
        over = (past[i] < 0 or held[i] < 0 or held[i] > blocks or new[i] > max_new or at + count > n_rows or
                (new[i] >= 0 and past[i] + count > min(blocks * page, 2 ** 31 - 1)))
        cu.append(min(at, n_rows))
        at += count
        bad.append(over)
        status[i] = 2 if over else 0
    cu.append(min(at, n_rows))
    if parent is not None:
        for i in range(n):
            if not bad[i] and new[i] > 0 and any(not -1 <= parent[cu[i] + j] < j for j in range(new[i])):
                bad[i], status[i] = True, 3
    for i in range(n):
        if new[i] < 0 and not bad[i]:
            for b in range(held[i]):
                if top < n_pages:
                    free[top] = table[i][b]
                    top += 1
            table[i], held[i] = [-1] * blocks, 0
    short, left = False, top
    for i in range(n):
        if bad[i] or new[i] < 0:
            continue
        want = max(0, -(-(past[i] + new[i]) // page) - held[i])
        if want and (short or want > left):
            short, status[i] = True, 1
            want = 0
        for b in range(blocks):
            if b >= held[i] + want:
                table[i][b] = -1
            elif b >= held[i]:
                left -= 1
                table[i][b] = free[left]
        held[i] += want
    slot, pos, mask = [None] * n_rows, [None] * n_rows, [None] * n_rows
    for i in range(n):
        c = cu[i + 1] - cu[i]
        anc = ancestors([parent[cu[i] + j] for j in range(c)]) if parent is not None and not bad[i] else None
        for j in range(c):
            r = cu[i] + j
            m = 0 if bad[i] else anc[j] if anc else (1 << min(j + 1, 64)) - 1
            mask[r] = signed(m)
            pos[r] = 0 if bad[i] else past[i] + (bin(m).count("1") - 1 if anc else j)
            ok = status[i] == 0 and 0 <= table[i][(past[i] + j) // page] < n_pages
            slot[r] = table[i][(past[i] + j) // page] * page + (past[i] + j) % page if ok else -1
    return dict(table=table, held=held, n_free=[left], free=free, cu=cu, slot=slot, pos=pos, mask=mask, status=status)
