"""Rows that a plan refused, or that got no K and V, are not committed, and do not reach the other requests."""
import numpy as np
import pytest
import torch

from kv_util import random_tree, stream
from navi_amd import abi

pytestmark = pytest.mark.gpu
PAGE, LAYERS, WIDTH = 16, 3, 64


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int64).astype(np.int32), dtype=torch.int32, device="cuda")


class Planned:
    """A planned step of (n_past, parents) on a pool whose rows are numbered."""

    def __init__(self, requests, *, held=None, free=20, n_rows=None, max_new=16, blocks=8, spoil=()):
        past, trees = [p for p, _ in requests], [t for _, t in requests]
        n, new = len(past), [len(t) for t in trees]
        held = held or [-(-p // PAGE) for p in past]
        self.n, self.n_pages = n, 24
        order, table = list(range(self.n_pages)), []
        for h in held:
            h = max(0, min(h, blocks))
            table.append(order[:h] + [-1] * (blocks - h))
            order = order[h:]
        free = min(free, len(order))
        R = sum(new) if n_rows is None else n_rows
        for at, value in spoil:                                   # parents that do not come before their rows
            trees[at[0]][at[1]] = value
        z = lambda k: i32([0] * k)
        self.t = dict(table=i32(table), past=i32(past), cu=z(n + 1), slot=z(R), pos=z(R), status=z(n), held=i32(held), free=i32([free]),
                      stack=i32(order[:free] + [-1] * (self.n_pages - free)), new=i32(new), parent=i32([p for t in trees for p in t]), scratch=z(4 * n))
        self.t["mask"] = torch.zeros(R, dtype=torch.int64, device="cuda")
        self.pages = abi.KvPages(n, PAGE, self.n_pages, blocks, R, max_new, *(self.t[k].data_ptr() for k in ("table", "past", "cu", "slot", "pos", "mask")))
        p = {k: v.data_ptr() for k, v in self.t.items()}
        abi.kv_plan(self.pages, n_new=p["new"], parent=p["parent"], table_in=p["table"], held_in=p["held"], free_in=p["free"], free_pages=p["stack"],
                    held=p["held"], free=p["free"], status=p["status"], scratch=p["scratch"], stream=stream())
        self.pool = torch.arange(LAYERS * 2 * self.n_pages * PAGE * WIDTH, device="cuda").to(torch.int16).view(LAYERS, 2, -1, WIDTH)
        torch.cuda.synchronize()

    def commit(self, paths, with_status):
        """(n_past, status, moved rows' slots by request) of the commit of `paths`."""
        self.pages.status = self.t["status"].data_ptr() if with_status else None
        before, d = self.pool.cpu(), self.pool.clone()
        size = d[0, 0].numel() * 2
        k, v = ([d.data_ptr() + (2 * l + h) * size for l in range(LAYERS)] for h in (0, 1))
        path, acc, past, done = i32([p + [0] * (16 - len(p)) for p in paths]), i32([len(p) for p in paths]), i32([-9] * self.n), i32([-9] * self.n)
        abi.kv_commit(self.pages, k, v, WIDTH, path.data_ptr(), 16, acc.data_ptr(), past.data_ptr(), done.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        return past.tolist(), done.tolist(), before, d.cpu()

    def slots(self, i, k):
        t = int(self.t["past"][i]) + np.arange(k)
        return self.t["table"].cpu().numpy()[i, t // PAGE] * PAGE + t % PAGE


def check(s, paths, good, with_status):
    past, done, before, after = s.commit(paths, with_status)
    was, want = s.t["past"].tolist(), before.clone()
    for i, p in enumerate(paths):
        if good[i]:
            at = s.slots(i, max(p, default=-1) + 1)
            for j, x in enumerate(p):
                want[:, :, at[j]] = before[:, :, at[x]]
    assert done == [0 if g else 2 for g in good]
    assert past == [w + (len(p) if g else 0) for w, p, g in zip(was, paths, good)]
    assert torch.equal(after, want)


@pytest.mark.parametrize("with_status", [False, True])
def test_a_request_without_pages_is_not_committed(with_status):
    """Request 1 holds a part of a page and needs another; a path inside its held page does not advance it."""
    s = Planned([(3, [-1, 0, 1]), (18, [j - 1 for j in range(16)]), (40, [-1, 0])], free=0)
    assert s.t["status"].tolist() == [0, 1, 0] and s.t["slot"].tolist()[3:19] == [-1] * 16
    check(s, [[0, 2], [0, 1], [1]], [True, False, True], with_status)
    check(s, [[0, 2], [], [0]], [True, True, True], with_status)   # nothing accepted: nothing to refuse


@pytest.mark.parametrize("kw,status", [
    (dict(requests=[(3, [-1, 0]), (20, [-1, 0, 1])], spoil=[((1, 2), 2)]), 3),
    (dict(requests=[(3, [-1, 0]), (20, [-1, 0, 1])], n_rows=4), 2),                       # its last row has no place
    (dict(requests=[(3, [-1, 0]), (20, [-1, 0, 1, 1, 2, 3])], max_new=4), 2),
    (dict(requests=[(3, [-1, 0]), (20, [-1, 0, 1])], held=[1, 9]), 2),
    (dict(requests=[(3, [-1, 0]), (-4, [-1, 0, 1])], held=[1, 2]), 2),
    (dict(requests=[(3, [-1, 0]), (126, [-1, 0, 1])], held=[1, 8]), 2)], ids=str)
def test_what_the_plan_refused_is_not_committed(kw, status):
    s = Planned(**{**kw, "requests": [(p, list(t)) for p, t in kw["requests"]]})
    assert s.t["status"].tolist() == [0, status]
    check(s, [[1], [0, 1]], [True, False], True)
    check(s, [[0], []], [True, int(s.t["past"][1]) >= 0], True)


def test_a_row_without_a_slot_is_not_committed():
    """With the plan's status a slot taken away refuses the rows' paths, and theirs only."""
    s = Planned([(3, [-1, 0, 1]), (20, random_tree(np.random.default_rng(0), 9))])
    s.t["slot"][3 + 4] = -1
    check(s, [[0, 1], [0, 4]], [True, False], True)
    check(s, [[0, 1], [0, 5]], [True, True], True)
    check(s, [[0, 1], [0, 4]], [True, True], False)


def test_an_array_named_more_than_once_is_moved_once():
    """K and V one array, and layers that share theirs: a second move would start from rows that the first has moved."""
    s = Planned([(3, [j - 1 for j in range(12)]), (20, [-1])])
    size, want = s.pool[0, 0].numel() * 2, s.pool.cpu()
    a, b = (s.pool.data_ptr() + i * size for i in (0, 3))
    path, acc, past, done = i32([list(range(1, 12)) + [0] * 5, [0] * 16]), i32([11, 0]), i32([0, 0]), i32([-9, -9])
    abi.kv_commit(s.pages, [a, b, a], [a, b, b], WIDTH, path.data_ptr(), 16, acc.data_ptr(), past.data_ptr(), done.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    at = s.slots(0, 12)
    for i in ((0, 0), (1, 1)):
        want[i][at[:11]] = want[i][at[1:]].clone()
    assert torch.equal(s.pool.cpu(), want) and past.tolist() == [14, 20] and done.tolist() == [0, 0]


def test_append_takes_the_slot_of_a_row_without_a_rotation():
    """Its K and V are not stored, so a commit over it is refused; the rows before it commit."""
    s = Planned([(3, [-1, 0, 1]), (28, [-1, 0, 0, 1, 3, 4])])
    slots = s.t["slot"].tolist()
    heads, width = abi.KvHeads(2, 1, 64, abi.DT_F16), 64
    x, q = torch.ones(9, 256, device="cuda").half(), torch.ones(9, 128, device="cuda").half()
    k, v = torch.zeros(s.n_pages * PAGE, width, device="cuda").half(), torch.zeros(s.n_pages * PAGE, width, device="cuda").half()
    turn = torch.cat([torch.ones(31, 32), torch.zeros(31, 32)], 1).cuda()                  # positions 0 .. 30
    abi.kv_append(s.pages, heads, x.data_ptr(), abi.DT_F16, 256, k.data_ptr(), v.data_ptr(), width, q.data_ptr(), abi.DT_F16, 128, rot=turn.data_ptr(),
                  n_rot=31, stream=stream())
    torch.cuda.synchronize()
    pos, want = s.t["pos"].tolist(), list(slots)
    assert pos == [3, 4, 5, 28, 29, 29, 30, 31, 32]
    want[7] = want[8] = -1
    assert s.t["slot"].tolist() == want and q[7:].abs().max() == 0 and bool((q[:7] == 1).all())
    stored = torch.zeros(s.n_pages * PAGE, dtype=torch.bool)
    stored[slots[:7]] = True
    assert torch.equal((k[:, 0] == 1).cpu(), stored) and torch.equal((v[:, 5] == 1).cpu(), stored)
    check(s, [[0, 1], [0, 1, 3, 4]], [True, False], True)
    check(s, [[0, 1], [0, 1, 3]], [True, True], True)
