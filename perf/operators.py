"""The serving operators on a paged K/V cache that this library's speed is judged by: planning a step's pages and
slots, appending its keys and values, the attention of its drafted tokens, and committing the accepted ones.

A step of a server: every request has `n_past` rows in a pool of pages and takes `n_new` more, a chain (a prompt, one
token) or a tree of drafted tokens. The head layouts are the talker's (16 / 8 heads x 128), the codec transformer's
(16 / 16 x 64) and common grouped ones. Lengths follow from the case; values, page orders and trees from the seed.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS, THETA = 1e-6, 1e6


def listed():
    talker = {"heads": 16, "kv_heads": 8, "dim": 128}
    return [
        # One request takes its next token: the smallest plan.
        {"name": "plan_1", "op": "plan", "requests": 1, "ctx": 256, "new": 1, "page": 16, "ragged": False, "tree": False, "tight": False},
        # A full server verifies drafts: 256 requests of uneven length with trees of up to 64 nodes, some ended.
        {"name": "plan_256_trees", "op": "plan", "requests": 256, "ctx": 4000, "new": 64, "page": 16, "ragged": True, "tree": True, "tight": False},
        # Prompts of uneven length admitted together, into a pool that cannot hold the last of them.
        {"name": "plan_prompts", "op": "plan", "requests": 48, "ctx": 1, "new": 1001, "page": 64, "ragged": True, "tree": False, "tight": True},
        # The next token's row of a single stream, as the talker has it (f32 rows, f16 cache).
        {"name": "append_1", "op": "append", "requests": 1, "ctx": 256, "new": 1, "page": 16, "type": "f32", **talker},
        # A batch of prompts written into the pages.
        {"name": "append_prompts", "op": "append", "requests": 9, "ctx": 0, "new": 1001, "page": 16, "type": "bf16", **talker},
        # Single stream, single token at the benchmark's context, in the talker's own types.
        {"name": "decode_1_ctx256", "op": "attention", "requests": 1, "ctx": 256, "new": 1, "page": 16, "ragged": False, "type": "f32", **talker},
        # A server's decode step: 32 streams at context 1024.
        {"name": "decode_32_ctx1024", "op": "attention", "requests": 32, "ctx": 1024, "new": 1, "page": 16, "ragged": False, "type": "f16", **talker},
        # Drafts of up to 15 nodes for ragged requests, pages of an odd size, no grouped heads.
        {"name": "tree_12_ragged", "op": "attention", "requests": 12, "ctx": 3001, "new": 15, "page": 24, "ragged": True, "type": "bf16", "heads": 16, "kv_heads": 16, "dim": 64},
        # One request with the largest tree over a long cache.
        {"name": "tree_64_ctx32768", "op": "attention", "requests": 1, "ctx": 32768, "new": 64, "page": 64, "ragged": False, "type": "f32", **talker},
        # A full server with long contexts and drafts of 24 nodes.
        {"name": "tree_64x24_ctx8192", "op": "attention", "requests": 64, "ctx": 8192, "new": 24, "page": 16, "ragged": False, "type": "f16", **talker},
        # One request keeps 4 of 8 drafted tokens in the talker's 28 layers.
        {"name": "commit_1", "op": "commit", "requests": 1, "ctx": 256, "new": 8, "accept": 4, "page": 16, "layers": 28, "type": "f16", **talker},
        # A server's commit: 32 requests keep 7 of 40.
        {"name": "commit_32", "op": "commit", "requests": 32, "ctx": 200, "new": 40, "accept": 7, "page": 16, "layers": 28, "type": "bf16", **talker},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "attention", "commit"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256])
    heads, kv, dim = rng.choice([(16, 8, 128), (16, 8, 128), (16, 16, 64), (32, 8, 128), (8, 1, 128), (12, 2, 64)])
    layout = {"heads": heads, "kv_heads": kv, "dim": dim}
    if op == "plan":
        tree = rng.random() < 0.6
        return {"op": op, "requests": _log_int(rng, 1, 256), "ctx": _log_int(rng, 1, 4000), "new": _log_int(rng, 1, 64 if tree else 1000),
                "page": max(page, 8), "ragged": rng.random() < 0.7, "tree": tree, "tight": rng.random() < 0.2}
    if op == "append":
        n = _log_int(rng, 1, 64)
        return {"op": op, "requests": n, "ctx": _log_int(rng, 1, 4000), "new": _log_int(rng, 1, min(1000, max(1, 9000 // n))), "page": page,
                "type": rng.choice(["f32", "f16", "bf16"]), **layout}
    if op == "commit":
        new = rng.randint(1, 64)
        return {"op": op, "requests": _log_int(rng, 1, 32), "ctx": _log_int(rng, 1, 200), "new": new, "accept": rng.randint(1, min(new, 8)),
                "page": min(page, 64), "layers": rng.choice([2, 8, 28]), "type": rng.choice(["f16", "bf16"]), **layout}
    n = _log_int(rng, 1, 96)
    new = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, min(32768, 200000 // n))
    return {"op": op, "requests": n, "ctx": min(ctx, max(1, 4000000 // (n * new))), "new": new, "page": page, "ragged": rng.random() < 0.5,
            "type": rng.choice(["f32", "f16", "bf16"]), **layout}


# ---- lengths (from the case alone) -------------------------------------------------------------

def _lengths(case):
    """(cached rows, new rows) of each request; new < 0: the request has ended."""
    n, ctx, new = case["requests"], case["ctx"], case["new"]
    r = random.Random(n * 1000003 + ctx * 1009 + new)
    if case["op"] == "plan":
        past = [_log_int(r, 1, ctx) if case["ragged"] and i else ctx for i in range(n)]
        if not case["tree"] and case["ctx"] == 1:
            past = [0] * n                                     # prompts: nothing is cached yet
        add = [_log_int(r, 1, new) if case["ragged"] and i else new for i in range(n)]
        return past, [-1 if i % 16 == 7 and past[i] else a for i, a in enumerate(add)]
    if case["op"] == "attention" and case["ragged"]:
        return [_log_int(r, 1, ctx) if i else ctx for i in range(n)], [r.randint(1, new) if i else new for i in range(n)]
    return [ctx] * n, [new] * n


def _trees(rng, counts):
    """Parents of every row's node within its request: node 0 the root, the others below one of the eight before them."""
    out = []
    for c in counts:
        out += [-1 if j == 0 else rng.randrange(max(0, j - 8), j) for j in range(c)]
    return out


def _masks(parent, counts):
    """Ancestors (itself included) of every node as bits, as signed 64-bit numbers, and its depth."""
    bits, depth, at = [], [], 0
    for c in counts:
        b = []
        for j in range(c):
            p = parent[at + j]
            b.append((b[p] if p >= 0 else 0) | (1 << j))
        bits += [x - (1 << 64) if x >> 63 else x for x in b]
        depth += [bin(x).count("1") - 1 for x in b]
        at += c
    return bits, depth


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- what a program has in hand before the call ------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    past, new = _lengths(case)
    n, page = len(past), case["page"]
    counts = [max(c, 0) for c in new]
    rows = sum(counts)
    s = {"case": case, "rows": rows, "n_past": _i32(past), "most_new": max(1, max(counts)), "most_keys": max(p + c for p, c in zip(past, counts))}
    blocks = -(-s["most_keys"] // page)
    if case["op"] == "plan":
        held = [-(-p // page) for p in past]
        extra = [max(0, -(-(p + c) // page) - h) for p, c, h in zip(past, counts, held)]
        ended = sum(h for h, c in zip(held, new) if c < 0)
        spare = max(0, int(0.6 * sum(extra)) - ended) if case["tight"] else sum(extra) + 37
        used = sum(held)
        order = torch.randperm(used + spare, generator=g, device="cuda").int()
        table = torch.full((n, blocks), -1, dtype=torch.int32, device="cuda")
        at = torch.zeros(n + 1, dtype=torch.int64)
        at[1:] = torch.tensor(held).cumsum(0)
        col = torch.arange(blocks, device="cuda")
        inside = col < _i32(held)[:, None]
        table = torch.where(inside, order[(at[:-1].cuda()[:, None] + col).clamp(max=used + spare - 1)], table)
        free = torch.full((used + spare,), -1, dtype=torch.int32, device="cuda")
        free[:spare] = order[used:]
        s.update(n_new=_i32(new), table=table, held=_i32(held), free=free, n_free=_i32([spare]), pool_pages=used + spare,
                 parent=_i32(_trees(rng, counts)) if case["tree"] else None)
        return s
    need = [-(-(p + c) // page) for p, c in zip(past, counts)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((n, blocks), -1, dtype=torch.int32)
    host, at = order.cpu(), 0
    for i, c in enumerate(need):
        table[i, :c] = host[at:at + c]
        at += c
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    kvd = case["kv_heads"] * case["dim"]
    kind = DTYPE["f16" if case["type"] == "f32" else case["type"]]       # of the cache
    kept = {"device": "cuda", "generator": g}
    parent = _trees(rng, counts) if case["op"] == "attention" else list(range(-1, case["new"] - 1)) * n
    # a chain: only the first 64 rows' bits are looked at
    bits, depth = _masks(parent, counts) if case["op"] == "attention" else ([0] * rows, list(range(case["new"])) * n)
    s.update(table=table.cuda(), pool_pages=pages, cu=_i32(cu), row_mask=torch.tensor(bits, dtype=torch.int64, device="cuda"))
    slot, pos = [], []
    if case["op"] == "append":
        t = table.tolist()
        for i, c in enumerate(counts):
            for j in range(c):
                k = past[i] + j
                slot.append(t[i][k // page] * page + k % page)
                pos.append(k)
        s.update(row_slot=_i32(slot), row_pos=_i32(pos))
        d, width = case["dim"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        s["x"] = (torch.randn(rows, width, **kept) * 1.5).to(DTYPE[case["type"]])
        s["q_norm"], s["k_norm"] = (1 + 0.1 * torch.randn(d, **kept) for _ in range(2))
        inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        angle = torch.arange(s["most_keys"], device="cuda").double()[:, None] * inv
        s["rot"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["k"], s["v"] = (torch.randn(pages * page, kvd, **kept).to(kind) for _ in range(2))
    elif case["op"] == "attention":
        s.update(row_slot=torch.full((rows,), -1, dtype=torch.int32, device="cuda"), row_pos=_i32(depth))
        s["q"] = torch.randn(rows, case["heads"] * case["dim"], **kept).to(DTYPE[case["type"]])
        s["k"], s["v"] = (torch.randn(pages * page, kvd, device="cuda", generator=g, dtype=kind) for _ in range(2))
    else:
        path = []
        for c in counts:
            a = min(case["accept"], c)
            path.append([0] + sorted(rng.sample(range(1, c), a - 1)) + [0] * (case["accept"] - a))
        s.update(path=_i32(path), accept=_i32([min(case["accept"], c) for c in counts]), row_slot=_i32([-1] * rows), row_pos=_i32([0] * rows))
        s["pool"] = torch.randn(case["layers"], 2, pages * page, kvd, device="cuda", generator=g, dtype=kind)
    return s


# ---- one pass ----------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    with torch.no_grad():
        return {"plan": _plan, "append": _append, "attention": _attention, "commit": _commit}[op](s)


def _abi():
    at = str(Path(__file__).resolve().parent.parent / "navi-tts_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from navi_amd import abi
    return abi


def _stream():
    return torch.cuda.current_stream().cuda_stream


_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _pages(abi, s, table=None, cu=None, slot=None, pos=None, mask=None):
    c = s["case"]
    table, cu = s["table"] if table is None else table, s["cu"] if cu is None else cu
    slot, pos, mask = (s[k] if t is None else t for k, t in (("row_slot", slot), ("row_pos", pos), ("row_mask", mask)))
    return abi.KvPages(c["requests"], c["page"], s["pool_pages"], table.shape[1], s["rows"], s["most_new"], table.data_ptr(),
                       s["n_past"].data_ptr(), cu.data_ptr(), slot.data_ptr(), pos.data_ptr(), mask.data_ptr())


def _heads(abi, s):
    c = s["case"]
    return abi.KvHeads(c["heads"], c["kv_heads"], c["dim"], 2 if c["type"] == "bf16" else 1)


def _own_plan(s):
    abi, n, rows = _abi(), s["case"]["requests"], s["rows"]
    i32 = {"dtype": torch.int32, "device": "cuda"}
    table, held, n_free, status = torch.empty_like(s["table"]), torch.empty(n, **i32), torch.empty(1, **i32), torch.empty(n, **i32)
    cu, slot, pos, scratch = torch.empty(n + 1, **i32), torch.empty(rows, **i32), torch.empty(rows, **i32), torch.empty(4 * n, **i32)
    mask = torch.empty(rows, dtype=torch.int64, device="cuda")
    abi.kv_plan(_pages(abi, s, table, cu, slot, pos, mask), n_new=s["n_new"].data_ptr(), parent=None if s["parent"] is None else s["parent"].data_ptr(),
                table_in=s["table"].data_ptr(), held_in=s["held"].data_ptr(), free_in=s["n_free"].data_ptr(), free_pages=s["free"].data_ptr(),
                held=held.data_ptr(), free=n_free.data_ptr(), status=status.data_ptr(), scratch=scratch.data_ptr(), stream=_stream())
    return {"table": table, "held": held, "n_free": n_free, "free": s["free"], "cu": cu, "slot": slot, "pos": pos, "mask": mask, "status": status}


def _own_append(s):
    abi, c, x = _abi(), s["case"], s["x"]
    q = torch.empty(s["rows"], c["heads"] * c["dim"], dtype=x.dtype, device="cuda")
    abi.kv_append(_pages(abi, s), _heads(abi, s), x.data_ptr(), _TYPE[x.dtype], x.shape[1], s["k"].data_ptr(), s["v"].data_ptr(), s["k"].shape[1],
                  q.data_ptr(), _TYPE[x.dtype], q.shape[1], q_norm=s["q_norm"].data_ptr(), k_norm=s["k_norm"].data_ptr(), eps=EPS,
                  rot=s["rot"].data_ptr(), n_rot=s["rot"].shape[0], stream=_stream())
    return {"q": q, "k": s["k"], "v": s["v"]}


def _own_attention(s):
    abi, c, q = _abi(), s["case"], s["q"]
    pages, heads = _pages(abi, s), _heads(abi, s)
    out = torch.empty_like(q)
    ws = torch.empty(abi.tree_workspace(pages, heads, s["most_keys"]), dtype=torch.uint8, device="cuda")
    abi.tree_attention(pages, heads, q.data_ptr(), _TYPE[q.dtype], q.shape[1], s["k"].data_ptr(), s["v"].data_ptr(), s["k"].shape[1],
                       1 / math.sqrt(c["dim"]), s["most_keys"], out.data_ptr(), out.shape[1], ws.data_ptr(), ws.numel(), stream=_stream())
    return out


def _own_commit(s):
    abi, n = _abi(), s["case"]["requests"]
    n_past, status = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
    pool, size = s["pool"].data_ptr(), s["pool"][0, 0].numel() * 2
    layers = s["pool"].shape[0]
    abi.kv_commit(_pages(abi, s), [pool + 2 * l * size for l in range(layers)], [pool + (2 * l + 1) * size for l in range(layers)], s["pool"].shape[3],
                  s["path"].data_ptr(), s["path"].shape[1], s["accept"].data_ptr(), n_past.data_ptr(), status.data_ptr(), stream=_stream())
    return {"pool": s["pool"], "n_past": n_past, "status": status}


_OWN = {"plan": _own_plan, "append": _own_append, "attention": _own_attention, "commit": _own_commit}


# ---- the plain forms ---------------------------------------------------------------------------

def _rows_of(cu, rows):
    """Request and index in it of every row."""
    r = torch.arange(rows, device="cuda", dtype=torch.int32)
    req = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    return req, r - cu[req]


def _before(x):
    return x.cumsum(0, dtype=torch.int32) - x


def _plan(s):
    case, n, rows, page, past, new, held = s["case"], s["case"]["requests"], s["rows"], s["case"]["page"], s["n_past"], s["n_new"], s["held"]
    count, ended = new.clamp(min=0), new < 0
    cu = torch.cat([torch.zeros_like(new[:1]), count.cumsum(0, dtype=torch.int32)])
    req, j = _rows_of(cu, rows)
    # the pages that come back, then those that are taken from the stack's top
    back = torch.where(ended, held, 0)
    col = torch.arange(s["table"].shape[1], device="cuda", dtype=torch.int32)
    size = s["pool_pages"]
    to = torch.where(ended[:, None] & (col < held[:, None]), s["n_free"] + _before(back)[:, None] + col, size)
    free = torch.cat([s["free"], s["free"][:1]]).scatter(0, to.reshape(-1).long(), s["table"].reshape(-1))[:size]
    have = s["n_free"] + back.sum(dtype=torch.int32)
    extra = torch.where(ended, 0, ((past + count + page - 1) // page - held).clamp(min=0))
    off = _before(extra)
    refused = (extra > 0) & (off + extra > have)
    extra = torch.where(refused, 0, extra)
    taken = (col >= held[:, None]) & (col < (held + extra)[:, None])
    from_top = (have - 1 - off)[:, None] - (col - held[:, None])
    keep = (col < held[:, None]) & ~ended[:, None]
    table = torch.where(keep, s["table"], torch.where(taken, free[from_top.clamp(0, size - 1).long()], -1))
    at = past[req] + j
    slot = torch.where(refused[req], -1, table[req, torch.where(refused[req], 0, at // page)] * page + at % page)
    if s["parent"] is None:
        depth = j
        mask = torch.where(j >= 63, -1, (torch.ones_like(j, dtype=torch.int64) << (j.long() + 1).clamp(max=63)) - 1)
    else:
        # reach[i][a][b]: b is a or above it, by squaring the parent relation
        wide = s["most_new"]
        p = torch.full((n, wide + 1), -1, dtype=torch.int64, device="cuda")
        p[req, j] = s["parent"].long()
        node = torch.arange(wide, device="cuda")
        reach = ((p[:, :wide, None] == node) | (node[:, None] == node)).float()
        reach = _squared(_squared(_squared(_squared(_squared(_squared(reach))))))
        mask = (reach.long() << node).sum(-1)[req, j]
        depth = reach.sum(-1).int()[req, j] - 1
    return {"table": table, "held": torch.where(ended, 0, held + extra), "n_free": have - extra.sum(dtype=torch.int32), "free": free, "cu": cu,
            "slot": slot.int(), "pos": past[req] + depth, "mask": mask, "status": refused.int()}


def _squared(r):
    return ((r @ r) > 0).float()


def _append(s):
    c, d = s["case"], s["case"]["dim"]
    x = s["x"].float().view(s["rows"], -1, d)
    hq, hk = c["heads"], c["kv_heads"]
    cos, sin = s["rot"][s["row_pos"].long()].view(-1, 1, d).chunk(2, -1)
    w = torch.cat([s["q_norm"].expand(hq, d), s["k_norm"].expand(hk, d)])
    y = x[:, :hq + hk]
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
    y0, y1 = y.chunk(2, -1)
    y = torch.cat([y0 * cos - y1 * sin, y1 * cos + y0 * sin], -1)
    at = s["row_slot"].long()
    s["k"][at] = y[:, hq:].reshape(s["rows"], -1).to(s["k"].dtype)
    s["v"][at] = x[:, hq + hk:].reshape(s["rows"], -1).to(s["v"].dtype)
    return {"q": y[:, :hq].reshape(s["rows"], -1).to(s["x"].dtype), "k": s["k"], "v": s["v"]}


def _attention(s):
    c, n, d, hk = s["case"], s["case"]["requests"], s["case"]["dim"], s["case"]["kv_heads"]
    g, wide, page = c["heads"] // hk, s["most_new"], c["page"]
    req, j = _rows_of(s["cu"], s["rows"])
    at = torch.arange(s["most_keys"], device="cuda", dtype=torch.int32)
    slot = (s["table"][:, (at // page).long()].clamp(min=0) * page + at % page).long()
    k = s["k"][slot].view(n, -1, hk, d).permute(0, 2, 3, 1).float()                        # [n][kv head][dim][key]
    q = torch.zeros(n, wide, c["heads"] * d, device="cuda")
    q[req, j] = s["q"].float()
    q = q.view(n, wide, hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * wide, d)
    score = torch.matmul(q, k.contiguous()).view(n, hk, g, wide, -1) / math.sqrt(d)
    del k
    bits = torch.zeros(n, wide, dtype=torch.int64, device="cuda")
    bits[req, j] = s["row_mask"]
    ahead = at - s["n_past"][:, None]                                                     # [n][key]
    count = s["cu"][1:] - s["cu"][:-1]
    node = (bits[:, :, None] >> ahead.clamp(0, 63)[:, None]) & 1
    seen = (ahead < 0)[:, None] | ((ahead >= 0) & (ahead < count[:, None]))[:, None] & (node != 0)
    score = torch.where(seen[:, None, None], score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    del score
    v = s["v"][slot].view(n, -1, hk, d).permute(0, 2, 1, 3).float()
    o = torch.matmul(p.view(n, hk, g * wide, -1), v.contiguous()).view(n, hk, g, wide, d) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(n, wide, -1)[req, j].to(s["q"].dtype)


def _commit(s):
    page, k = s["case"]["page"], torch.arange(s["path"].shape[1], device="cuda", dtype=torch.int32)
    kept = k < s["accept"][:, None]

    def slot(node):
        at = s["n_past"][:, None] + torch.where(kept, node, 0)
        return (torch.gather(s["table"], 1, (at // page).long()) * page + at % page).long().reshape(-1)

    s["pool"][:, :, slot(k.expand_as(kept))] = s["pool"][:, :, slot(s["path"])]
    return {"pool": s["pool"], "n_past": s["n_past"] + s["accept"], "status": torch.zeros_like(s["accept"])}


# ---- the work, and the same in 64 bits ---------------------------------------------------------

def work(case):
    past, new = _lengths(case)
    n, counts = len(past), [max(c, 0) for c in new]
    rows, page = sum(counts), case["page"]
    if case["op"] == "plan":
        blocks = -(-max(p + c for p, c in zip(past, counts)) // page)
        # the table in and out, a request's lengths, held pages and results, a row's results (and its parent)
        return {"bytes": 8.0 * n * blocks + 28.0 * n + rows * (20.0 if case["tree"] else 16.0), "flops": 4.0 * (n * blocks + rows)}
    d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "append":
        reads = rows * ((hq + 2 * hk) * d * size + 8) + 4.0 * d * min(rows, case["ctx"] + case["new"])
        return {"bytes": reads + rows * d * (hq * size + 2 * hk * 2), "flops": 10.0 * rows * (hq + hk) * d}
    if case["op"] == "commit":
        moved = n * (min(case["accept"], case["new"]) - 1)
        return {"bytes": 2.0 * moved * hk * d * 2 * 2 * case["layers"] + 4.0 * n * (case["accept"] + 4), "flops": 0.0}
    keys = sum(p + c for p, c in zip(past, counts))
    pairs = sum((p + c / 2) * c for p, c in zip(past, counts))
    return {"bytes": 4.0 * keys * hk * d + 2.0 * rows * hq * d * size + 12.0 * rows + 4.0 * sum(-(-(p + c) // page) for p, c in zip(past, counts)),
            "flops": 4.0 * pairs * hq * d}


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return globals()["_exact_" + case["op"]](s, case)


def _exact_plan(s, case):
    past, new, held, table = (s[k].tolist() for k in ("n_past", "n_new", "held", "table"))
    parent = None if s["parent"] is None else s["parent"].tolist()
    stack, page, blocks = s["free"].tolist(), case["page"], s["table"].shape[1]
    top = int(s["n_free"])
    for i, c in enumerate(new):
        if c < 0:
            stack[top:top + held[i]] = table[i][:held[i]]
            top += held[i]
            table[i], held[i] = [-1] * blocks, 0
    left, cu, slot, pos, status, short = top, [0], [], [], [], False
    for i, c in enumerate(new):
        c, want = max(c, 0), max(0, -(-(past[i] + c) // page) - held[i]) if c >= 0 else 0
        refused = want > 0 and (short or want > left)
        short = short or refused
        if not refused:
            for _ in range(want):
                left -= 1
                table[i][held[i]] = stack[left]
                held[i] += 1
        slot += [-1 if refused else table[i][(past[i] + j) // page] * page + (past[i] + j) % page for j in range(c)]
        status.append(int(refused))
        cu.append(cu[-1] + c)
    counts = [max(c, 0) for c in new]
    if parent is not None:
        mask, depth = _masks(parent, counts)
    else:
        mask, depth = [-1 if j >= 63 else (2 << j) - 1 for c in counts for j in range(c)], [j for c in counts for j in range(c)]
    pos = [past[i] + depth[cu[i] + j] for i, c in enumerate(counts) for j in range(c)]
    return {"table": _i32(table), "held": _i32(held), "n_free": _i32([left]), "free": _i32(stack), "cu": _i32(cu), "slot": _i32(slot), "pos": _i32(pos),
            "mask": torch.tensor(mask, dtype=torch.int64), "status": _i32(status)}


def _exact_append(s, case):
    d, hq, hk, rows = case["dim"], case["heads"], case["kv_heads"], s["rows"]
    x = s["x"].double().view(rows, hq + 2 * hk, d)
    turn = torch.complex(s["rot"][:, :d // 2].double(), s["rot"][:, d // 2:].double())[s["row_pos"].long()][:, None]

    def head(a, w):
        a = a / (a.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        z = torch.complex(a[..., :d // 2].contiguous(), a[..., d // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1).reshape(rows, -1)

    k, v = s["k"].double(), s["v"].double()
    k[s["row_slot"].long()], v[s["row_slot"].long()] = head(x[:, hq:hq + hk], s["k_norm"]), x[:, hq + hk:].reshape(rows, -1)
    return {"q": head(x[:, :hq], s["q_norm"]), "k": k, "v": v}


def _exact_attention(s, case):
    d, hk, g, page = case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"], case["page"]
    cu, past, table, out = s["cu"].tolist(), s["n_past"].tolist(), s["table"].long(), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["requests"]):
        c, keys = cu[i + 1] - cu[i], past[i] + cu[i + 1] - cu[i]
        at = torch.arange(keys, device="cuda")
        slot = table[i, at // page] * page + at % page
        k, v = (s[x][slot].view(keys, hk, d) for x in ("k", "v"))
        node = torch.arange(c, device="cuda")
        seen = torch.ones(c, keys, dtype=torch.bool, device="cuda")
        seen[:, past[i]:] = ((s["row_mask"][cu[i]:cu[i + 1], None] >> node) & 1).bool()
        q = s["q"][cu[i]:cu[i + 1]].double().view(c, hk, g, d)
        for h in range(hk):
            a = (q[:, h].reshape(c * g, d) @ k[:, h].double().T / d ** 0.5).masked_fill(~seen.repeat_interleave(g, 0), -math.inf)
            out[cu[i]:cu[i + 1], h * g * d:(h + 1) * g * d] = (torch.softmax(a, -1) @ v[:, h].double()).view(c, g * d)
    return out


def _exact_commit(s, case):
    pool, page, table, past = s["pool"], case["page"], s["table"].tolist(), s["n_past"].tolist()

    def slot(i, node):
        return table[i][(past[i] + node) // page] * page + (past[i] + node) % page

    for i, (path, a) in enumerate(zip(s["path"].tolist(), s["accept"].tolist())):
        for k in range(a):
            pool[:, :, slot(i, k)] = pool[:, :, slot(i, path[k])]
        past[i] += a
    return {"pool": pool, "n_past": _i32(past), "status": _i32([0] * len(past))}
