"""navi_draft_accept against its definition on the host, and the step that it closes: plan, append, attend, sample, accept, commit."""
import numpy as np
import pytest
import torch

from kv_util import random_tree, stream
from navi_amd import abi

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


class Drafts:
    """Requests' drafted rows, each with its parent's sampled codes or others."""

    def __init__(self, trees, codes, *, seed=0, hit=0.7, chain=False, last=True, pad=(0, 0), spare=0, max_path=64, max_new=64):
        rng = np.random.default_rng(seed)
        self.trees, self.codes, self.max_path, self.max_new = trees, codes, max_path, max_new
        self.chain = chain
        self.cu = np.concatenate([[0], np.cumsum([len(t) for t in trees])])
        self.rows = int(self.cu[-1]) + spare
        # few different codes, so that siblings are alike now and then
        self.sampled = rng.integers(0, 3, (self.rows, codes))
        self.drafted = rng.integers(0, 3, (self.rows, codes))
        self.last = rng.integers(0, 3, (len(trees), codes)) if last else None
        for i, t in enumerate(trees):
            for j, p in enumerate(t):
                if rng.random() < hit:
                    r = self.cu[i] + j
                    if p >= 0:
                        self.drafted[r] = self.sampled[self.cu[i] + p]
                    elif last:
                        self.drafted[r] = self.last[i]
        self.slot = np.arange(self.rows)
        self.status = np.zeros(len(trees), int)
        self.pad = pad

    def go(self, *, with_status=True, in_place=False, st=None):
        n, wide = len(self.trees), lambda a, p: i32(np.concatenate([a, np.full((a.shape[0], p), -9)], 1))
        self.d = dict(cu=i32(self.cu), slot=i32(self.slot), status=i32(self.status), drafted=wide(self.drafted, self.pad[0]), sampled=wide(self.sampled, self.pad[1]),
                      path=i32(np.full((n, self.max_path), -9)), accept=i32(np.full(n, -9)), next=i32(np.full((n, self.codes), -9)), other=i32(np.zeros(max(1, self.rows))))
        if not self.chain:
            flat = [p for t in self.trees for p in t]
            self.d["parent"] = i32(flat + [0] * (self.rows - len(flat)) + [0])
        if self.last is not None:
            self.d["last"] = i32(self.last)
            if in_place:
                self.d["next"] = self.d["last"]
        self.mask = torch.zeros(max(1, self.rows), dtype=torch.int64, device="cuda")
        p = {k: v.data_ptr() for k, v in self.d.items()}
        pages = abi.KvPages(n, 16, 1 << 12, 1, self.rows, self.max_new, p["other"], p["other"], p["cu"], p["slot"], p["other"], self.mask.data_ptr(),
                            p["status"] if with_status else None)
        abi.draft_accept(pages, p["drafted"], self.codes + self.pad[0], p["sampled"], self.codes + self.pad[1], self.codes, p["path"], self.max_path, p["accept"], p["next"],
                         parent=p.get("parent"), last=p.get("last"), stream=stream() if st is None else st)
        torch.cuda.synchronize()
        return [self.d[k].tolist() for k in ("path", "accept", "next")]

    def expect(self, with_status=True):
        path, accept, then = [], [], []
        for i, t in enumerate(self.trees):
            c0, got, at = self.cu[i], [], -1
            want = None if self.last is None else list(self.last[i])
            ok = len(t) <= self.max_new and not (with_status and self.status[i])
            while ok and len(got) < self.max_path:
                for j in range(len(t)):
                    parent = j - 1 if self.chain else t[j]
                    if parent != at or parent >= j or self.slot[c0 + j] < 0:
                        continue
                    if at < 0 and want is None or min(want) >= 0 and list(self.drafted[c0 + j]) == want:
                        break
                else:
                    break
                got.append(j)
                at, want = j, list(self.sampled[c0 + j])
            path.append(got + [0] * (self.max_path - len(got)))
            accept.append(len(got))
            then.append([-1] * self.codes if want is None else want)
        return [path, accept, [[int(c) for c in w] for w in then]]


def trees_of(rng, n, most):
    return [random_tree(rng, int(rng.integers(0, most + 1)), roots=int(rng.integers(1, 4))) for _ in range(n)]


@pytest.mark.parametrize("codes", [1, 2, 7, 16, 65])
@pytest.mark.parametrize("n,most", [(1, 1), (1, 8), (3, 64), (5, 20), (70, 64), (257, 12)])
@pytest.mark.parametrize("last", [True, False])
def test_trees(n, most, codes, last):
    """No rows to 64, several roots, siblings alike."""
    d = Drafts(trees_of(np.random.default_rng(n + most), n, most), codes, seed=codes, last=last, pad=(codes % 3, codes % 2))
    assert d.go() == d.expect()


@pytest.mark.parametrize("hit", [0.0, 0.9, 1.0])
@pytest.mark.parametrize("max_path", [1, 5, 64])
def test_chains(hit, max_path):
    """Without parents each row follows the one before it; 64 of them; a path that is cut short goes on from its last row."""
    d = Drafts([list(range(-1, k - 1)) for k in (64, 1, 0, 9, 33)], 3, hit=hit, chain=True, max_path=max_path)
    assert d.go() == d.expect()


def test_what_cannot_be_committed_is_not_taken():
    """Rows without a slot, requests that the plan refused or with more than max_new rows, parents that do not come before their rows."""
    d = Drafts([list(range(-1, 9)) for _ in range(6)] + [list(range(-1, 20))], 2, hit=1.0, max_new=12, spare=3)
    d.slot[d.cu[1] + 4] = d.slot[d.cu[2]] = -1
    d.status[3] = 1
    d.trees[4][5], d.trees[5][0] = 5, 3
    got = d.go()
    assert got == d.expect() and got[1] == [10, 4, 0, 0, 5, 0, 0]
    assert d.go(with_status=False) == d.expect(with_status=False)
    assert d.d["next"].tolist()[3] == list(map(int, d.sampled[d.cu[4] - 1]))


def test_codes_below_zero_equal_none():
    d = Drafts([[-1, 0, 1], [-1, 0, 1]], 2, hit=1.0)
    d.sampled[1, 1] = -1
    d.drafted[2] = d.sampled[1]
    d.last[1, 0] = d.drafted[3, 0] = -1
    got = d.go()
    assert got == d.expect() and got[1] == [2, 0]


def test_the_next_codes_over_the_last_ones_and_in_a_graph():
    d = Drafts(trees_of(np.random.default_rng(2), 9, 30), 16, seed=3)
    want = d.expect()
    assert d.go(in_place=True) == want
    d.go()
    graph = torch.cuda.CUDAGraph()
    p = {k: v.data_ptr() for k, v in d.d.items()}
    pages = abi.KvPages(9, 16, 1 << 12, 1, d.rows, 64, p["other"], p["other"], p["cu"], p["slot"], p["other"], d.mask.data_ptr(), p["status"])
    with torch.cuda.graph(graph):
        abi.draft_accept(pages, p["drafted"], 16, p["sampled"], 16, 16, p["path"], 64, p["accept"], p["next"], parent=p["parent"], last=p["last"], stream=stream())
    for seed in range(3):
        e = Drafts(d.trees, 16, seed=20 + seed)
        for k in ("drafted", "sampled", "last"):
            d.d[k].copy_(i32(getattr(e, k)))
        graph.replay()
        torch.cuda.synchronize()
        assert [d.d[k].tolist() for k in ("path", "accept", "next")] == e.expect()


def test_no_rows_at_all():
    d = Drafts([[], []], 4)
    assert d.go() == d.expect() and d.d["next"].tolist() == d.last.tolist()


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_a_server_that_checks_drafts_gives_the_tokens_of_one_that_does_not(cache):
    """Three requests of a one-layer model with a head, all on the device: ten tokens each, one a step; then by steps of drafted trees that hold some
    of the right tokens, accepted and committed. The same numbers of the draw belong to the same positions, so the tokens are the same."""
    heads, kv, dim, vocab, page, n, steps = 4, 2, 64, 97, 8, 3, 10
    width = (heads + 2 * kv) * dim
    g = torch.Generator().manual_seed(4)
    table_in = (torch.randn(vocab, width, generator=g)).half().cuda()                     # a token's q|k|v row
    head = (torch.randn(heads * dim, vocab, generator=g) * 0.7).cuda()
    draws = torch.rand(n, 64, generator=g).cuda()                                        # of the token at every position
    first = [5, 17, 60]
    f8 = cache == "e4m3"
    fac = [(torch.ones(kv) / 20).cuda() for _ in range(2)]
    lay = abi.KvHeads(heads, kv, dim, abi.DT_F8E4M3 if f8 else abi.DT_F16, *(t.data_ptr() for t in fac))
    rule = i32(np.array([(0.9, 20, 0.95, 0.0, 1.0)], dtype=[("t", "<f4"), ("k", "<i4"), ("p", "<f4"), ("m", "<f4"), ("r", "<f4")]).view(np.int32))

    def serve(trees_for):
        """trees_for(request, position) -> (parents, tokens) of the drafted nodes, the certain token as node 0."""
        pages_n, blocks, room = 24, 6, n * 8
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        t = dict(table=z(n, blocks) - 1, past=z(n), cu=z(n + 1), slot=z(room) - 1, pos=z(room), status=z(n), held=z(n), free=z(1) + pages_n,
                 stack=torch.randperm(pages_n, generator=torch.Generator().manual_seed(1)).int().cuda(), new=z(n), parent=z(room), scratch=z(4 * n), past_out=z(n), done=z(n),
                 drafted=z(room), sampled=z(room), last=i32(first), path=z(n, 8), accept=z(n))
        t["mask"] = torch.zeros(room, dtype=torch.int64, device="cuda")
        p = {k: v.data_ptr() for k, v in t.items()}
        k, v = (torch.zeros(pages_n * page, kv * dim, dtype=torch.uint8 if f8 else torch.float16, device="cuda") for _ in range(2))
        out = [[f] for f in first]
        calls = 0
        while min(map(len, out)) < steps:
            nodes = [trees_for(i, len(out[i]) - 1, out[i]) for i in range(n)]
            rows = sum(len(a) for a, _ in nodes)
            pages = abi.KvPages(n, page, pages_n, blocks, rows, 8, *(p[x] for x in ("table", "past", "cu", "slot", "pos", "mask", "status")))
            t["new"].copy_(i32([len(a) for a, _ in nodes]))
            t["parent"][:rows] = i32([x for a, _ in nodes for x in a])
            t["drafted"][:rows] = i32([x for _, b in nodes for x in b])
            s = stream()
            abi.kv_plan(pages, n_new=p["new"], parent=p["parent"], table_in=p["table"], held_in=p["held"], free_in=p["free"], free_pages=p["stack"], held=p["held"],
                        free=p["free"], status=p["status"], scratch=p["scratch"], stream=s)
            x = table_in[t["drafted"][:rows].long()].contiguous()
            q, o = (torch.zeros(rows, heads * dim, dtype=torch.float16, device="cuda") for _ in range(2))
            abi.kv_append(pages, lay, x.data_ptr(), abi.DT_F16, width, k.data_ptr(), v.data_ptr(), kv * dim, q.data_ptr(), abi.DT_F16, q.shape[1], stream=s)
            abi.tree_attention(pages, lay, q.data_ptr(), abi.DT_F16, q.shape[1], k.data_ptr(), v.data_ptr(), kv * dim, dim ** -0.5, 48, o.data_ptr(), o.shape[1], None, 0, stream=s)
            logits = torch.cat([o[r:r + 1].float() @ head for r in range(rows)])          # each row alone: the same sums in any company
            owner = torch.repeat_interleave(torch.arange(n, device="cuda"), t["new"].long())
            u = draws[owner, t["pos"][:rows].long()].contiguous()
            abi.sample_rows(logits.data_ptr(), 0, vocab, rows, vocab, rule.data_ptr(), 1, u.data_ptr(), p["sampled"], stream=s)
            abi.draft_accept(pages, p["drafted"], 1, p["sampled"], 1, 1, p["path"], 8, p["accept"], p["last"], parent=p["parent"], last=p["last"], stream=s)
            abi.kv_commit(pages, [k.data_ptr()], [v.data_ptr()], kv * dim // (2 if f8 else 1), p["path"], 8, p["accept"], p["past_out"], p["done"], stream=s)
            t["past"].copy_(t["past_out"])
            torch.cuda.synchronize()
            assert t["done"].tolist() == [0] * n
            cu = t["cu"].tolist()
            for i in range(n):
                path = t["path"][i, :int(t["accept"][i])].tolist()
                assert path[0] == 0
                out[i] += [int(t["sampled"][cu[i] + j]) for j in path]
                assert t["last"].tolist()[i] == out[i][-1] and int(t["past"][i]) == len(out[i]) - 1
            calls += 1
        return [o[:steps] for o in out], calls

    plain, one_a_step = serve(lambda i, at, out: ([-1], [out[-1]]))
    right = {(i, j): plain[i][j] for i in range(n) for j in range(steps)}
    rng = np.random.default_rng(0)

    def guess(i, at, out):
        """A wrong child, the right one, its right child, and a wrong one below that."""
        a, b = (right.get((i, at + d), 1) for d in (1, 2))
        wrong = lambda x: (x + 1 + int(rng.integers(0, vocab - 1))) % vocab if rng.random() < 0.8 else x
        return [-1, 0, 0, 2, 3], [out[-1], (a + 3) % vocab, a if rng.random() < 0.8 else wrong(a), b, (b + 1) % vocab]

    drafted, calls = serve(guess)
    assert drafted == plain and calls < one_a_step == steps - 1
