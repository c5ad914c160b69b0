"""A server's whole step on an e4m3 pool - plan, append, attend, sample, accept, commit - enqueued without a wait: on two streams at
once, and replayed from two graphs in turn, against the same steps one after another. The attention's rows serve as logits."""
import numpy as np
import pytest
import torch

from kv_util import random_tree, stream
from navi_amd import abi

pytestmark = pytest.mark.gpu
N, HEADS, KV, DIM, PAGE, BLOCKS, MOST, LONG = 3, 8, 2, 64, 16, 24, 12, 20000
ROWS, PAGES, W = N * MOST, N * BLOCKS, KV * DIM
WIDTH = HEADS * DIM


class Server:
    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")
        self.t = dict(table=z(N, BLOCKS) - 1, past=z(N), cu=z(N + 1), slot=z(ROWS), pos=z(ROWS), status=z(N), held=z(N), free=z(1) + PAGES,
                      stack=torch.from_numpy(rng.permutation(PAGES).astype(np.int32)).cuda(), new=z(N) + MOST, scratch=z(4 * N + 16), next_past=z(N), done=z(N),
                      parent=torch.tensor(sum((random_tree(rng, MOST) for _ in range(N)), []), dtype=torch.int32, device="cuda"),
                      drafted=z(ROWS, 2), sampled=z(ROWS, 2), last=z(N, 2), path=z(N, MOST), accept=z(N))
        self.t["mask"] = torch.zeros(ROWS, dtype=torch.int64, device="cuda")
        p = {n: v.data_ptr() for n, v in self.t.items()}
        self.pages = abi.KvPages(N, PAGE, PAGES, BLOCKS, ROWS, MOST, *(p[n] for n in ("table", "past", "cu", "slot", "pos", "mask")), p["status"])
        self.p = p
        self.factors = [(0.5 + torch.rand(KV, generator=g)).cuda() / 40 for _ in range(2)]
        self.heads = abi.KvHeads(HEADS, KV, DIM, abi.DT_F8E4M3, *(f.data_ptr() for f in self.factors))
        self.k, self.v = (torch.zeros(PAGES * PAGE, W, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.x = torch.zeros(ROWS, (HEADS + 2 * KV) * DIM, device="cuda")
        self.q, self.out = (torch.zeros(ROWS, WIDTH, device="cuda") for _ in range(2))
        self.long = torch.zeros(ROWS, LONG, dtype=torch.bfloat16, device="cuda")
        self.u = torch.zeros(2, ROWS, device="cuda")
        raw = np.array([(0.01, 4, 0.9, 0, 1)], dtype=[("t", "<f4"), ("k", "<i4"), ("p", "<f4"), ("m", "<f4"), ("r", "<f4")])
        self.rule = torch.from_numpy(raw.view(np.int32).copy()).cuda()
        self.ws = torch.full((abi.tree_workspace(self.pages, self.heads, BLOCKS * PAGE),), 0xFF, dtype=torch.uint8, device="cuda")
        self.sample_ws = torch.full((abi.sample_workspace(ROWS, LONG),), 0xFF, dtype=torch.uint8, device="cuda")

    def feed(self, seed):
        """The next step's inputs; drafted codes are few, so that some are sampled."""
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.x.shape, generator=g))
        self.long.copy_(torch.randn(self.long.shape, generator=g) * 3)
        self.u.copy_(torch.rand(self.u.shape, generator=g))
        self.t["drafted"].copy_(torch.randint(0, 2, (ROWS, 2), generator=g))

    def step(self, st):
        p, t = self.p, self.t
        abi.kv_plan(self.pages, n_new=p["new"], parent=p["parent"], table_in=p["table"], held_in=p["held"], free_in=p["free"], free_pages=p["stack"], held=p["held"],
                    free=p["free"], status=p["status"], scratch=p["scratch"], stream=st)
        abi.kv_append(self.pages, self.heads, self.x.data_ptr(), 0, self.x.shape[1], self.k.data_ptr(), self.v.data_ptr(), W, self.q.data_ptr(), 0, WIDTH, stream=st)
        abi.tree_attention(self.pages, self.heads, self.q.data_ptr(), 0, WIDTH, self.k.data_ptr(), self.v.data_ptr(), W, DIM ** -0.5, BLOCKS * PAGE, self.out.data_ptr(),
                           WIDTH, self.ws.data_ptr(), self.ws.numel(), stream=st)
        # a row's first code of two, from the attention's columns; its second from a long vocabulary
        abi.sample_rows(self.out.data_ptr(), 0, WIDTH, ROWS, 2, self.rule.data_ptr(), 1, self.u.data_ptr(), p["sampled"], ld_token=2, stream=st)
        abi.sample_rows(self.long.data_ptr(), abi.DT_BF16, LONG, ROWS, LONG, self.rule.data_ptr(), 1, self.u.data_ptr() + 4 * ROWS, p["sampled"] + 4, ld_token=2,
                        ws=self.sample_ws.data_ptr(), ws_bytes=self.sample_ws.numel(), stream=st)
        abi.draft_accept(self.pages, p["drafted"], 2, p["sampled"], 2, 1, p["path"], MOST, p["accept"], p["last"], parent=p["parent"], stream=st)
        abi.kv_commit(self.pages, [self.k.data_ptr()], [self.v.data_ptr()], W // 2, p["path"], MOST, p["accept"], p["next_past"], p["done"], stream=st)

    def turn(self):
        """What the next step starts from."""
        self.t["past"].copy_(self.t["next_past"])

    def state(self):
        return [self.t[n].cpu() for n in ("table", "held", "free", "slot", "pos", "mask", "cu", "status", "sampled", "path", "accept", "last", "next_past", "done")] + \
               [self.out.cpu(), self.k.cpu(), self.v.cpu()]


def check(a, b, what):
    for i, (x, y) in enumerate(zip(a.state(), b.state())):
        assert torch.equal(x, y), (what, i)


def test_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    servers, alone = [Server(1), Server(2)], [Server(1), Server(2)]
    for round_ in range(4):
        for pair in (servers, alone):
            for i, s in enumerate(pair):
                s.feed(10 * round_ + i)
        torch.cuda.synchronize()
        for s in alone:
            s.step(streams[0].cuda_stream)
            torch.cuda.synchronize()
        for s, st in zip(servers, streams):
            s.step(st.cuda_stream)
        torch.cuda.synchronize()
        for s, a in zip(servers, alone):
            check(s, a, round_)
        for s in (*servers, *alone):
            assert s.t["status"].tolist() == [0] * N and s.t["done"].tolist() == [0] * N and all(a >= 1 for a in s.t["accept"].tolist())
            s.turn()


def test_graphs_replayed_between_eager_steps():
    captured, eager, graphs = [Server(3), Server(4)], [Server(3), Server(4)], []
    for s in captured:
        s.feed(0)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.step(stream())
        graphs.append(g)
    for round_ in range(5):
        for pair in (captured, eager):
            for i, s in enumerate(pair):
                s.feed(100 + 10 * round_ + i)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        for s in eager:
            s.step(stream())
        torch.cuda.synchronize()
        for s, e in zip(captured, eager):
            check(s, e, round_)
            s.turn()
            e.turn()
