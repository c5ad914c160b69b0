"""The operators of a server's step that this library's speed is judged by besides those of operators.py: a cache held in 8 bits
(keys and values rounded as they are written, and the attention that reads them back), the sampling of many rows of logits,
and the choice of the drafted rows that the sampled codes confirm.

The cache is a pool of pages as in operators.py, its elements e4m3 with one factor per kv head for K and for V. The head layouts
are the talker's (16 / 8 heads x 128), the codec transformer's (16 / 16 x 64) and common grouped ones; rows of logits are as wide
as the code predictor's 2048, the text vocabulary's 151936 and between. Lengths follow from the case; values, page orders, trees
and sampling rules from the seed.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
F8, F8_MOST = torch.float8_e4m3fn, 448.0
EPS, THETA = 1e-6, 1e6


def listed():
    talker = {"heads": 16, "kv_heads": 8, "dim": 128}
    return [
        # The next token's row of a single stream, as the talker has it (f32 rows), into an 8-bit cache.
        {"name": "append8_1", "op": "append", "requests": 1, "ctx": 256, "new": 1, "page": 16, "type": "f32", **talker},
        # A batch of prompts written into the pages.
        {"name": "append8_prompts", "op": "append", "requests": 9, "ctx": 0, "new": 1001, "page": 16, "type": "bf16", **talker},
        # Single stream, single token at the benchmark's context, queries in the talker's own type.
        {"name": "decode8_1_ctx256", "op": "attention", "requests": 1, "ctx": 256, "new": 1, "page": 16, "ragged": False, "type": "f32", **talker},
        # A server's decode step: 32 streams at context 1024.
        {"name": "decode8_32_ctx1024", "op": "attention", "requests": 32, "ctx": 1024, "new": 1, "page": 16, "ragged": False, "type": "f16", **talker},
        # Drafts of up to 15 nodes for ragged requests, pages of an odd size, no grouped heads.
        {"name": "tree8_12_ragged", "op": "attention", "requests": 12, "ctx": 3001, "new": 15, "page": 24, "ragged": True, "type": "bf16", "heads": 16, "kv_heads": 16, "dim": 64},
        # A full server with long contexts and drafts of 24 nodes.
        {"name": "tree8_64x24_ctx8192", "op": "attention", "requests": 64, "ctx": 8192, "new": 24, "page": 16, "ragged": False, "type": "f16", **talker},
        # One code of one stream, with the defaults of the framework's own sampler (temperature and top-k).
        {"name": "sample_1x2048", "op": "sample", "rows": 1, "vocab": 2048, "rule": "top_k", "masks": False, "type": "f32"},
        # The rows of a verified step: 32 requests with 16 drafted nodes, every request with rules of its own, repetitions penalised.
        {"name": "sample_512x2048", "op": "sample", "rows": 512, "vocab": 2048, "rule": "mixed", "masks": True, "type": "f32"},
        # The next token of one text stream: a nucleus over the whole text vocabulary.
        {"name": "sample_1x151936", "op": "sample", "rows": 1, "vocab": 151936, "rule": "top_p", "masks": False, "type": "bf16"},
        # A full server's text rows, every one with rules of its own.
        {"name": "sample_256x151936", "op": "sample", "rows": 256, "vocab": 151936, "rule": "mixed", "masks": False, "type": "f32"},
        # One request's eight drafted frames of 16 codes.
        {"name": "accept_1", "op": "accept", "requests": 1, "new": 8, "codes": 16, "ragged": False, "tree": True},
        # A full server's drafts, trees of up to 64 frames.
        {"name": "accept_256x64", "op": "accept", "requests": 256, "new": 64, "codes": 16, "ragged": True, "tree": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "sample", "sample", "accept"])
    if op == "sample":
        vocab = rng.choice([2048, 151936]) if rng.random() < 0.2 else _log_int(rng, 100, 151936)
        return {"op": op, "rows": _log_int(rng, 1, min(1024, 38000000 // vocab)), "vocab": vocab,
                "rule": rng.choice(["greedy", "plain", "top_k", "top_p", "min_p", "all", "mixed", "mixed"]), "masks": rng.random() < 0.4,
                "type": rng.choice(["f32", "f16", "bf16"])}
    if op == "accept":
        return {"op": op, "requests": _log_int(rng, 1, 256), "new": _log_int(rng, 1, 64), "codes": rng.choice([1, 1, 5, 16, 16]),
                "ragged": rng.random() < 0.7, "tree": rng.random() < 0.7}
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256])
    heads, kv, dim = rng.choice([(16, 8, 128), (16, 8, 128), (16, 16, 64), (32, 8, 128), (8, 1, 128), (12, 2, 64)])
    layout = {"heads": heads, "kv_heads": kv, "dim": dim}
    if op == "append":
        n = _log_int(rng, 1, 64)
        return {"op": op, "requests": n, "ctx": _log_int(rng, 1, 4000), "new": _log_int(rng, 1, min(1000, max(1, 9000 // n))), "page": page,
                "type": rng.choice(["f32", "f16", "bf16"]), **layout}
    n = _log_int(rng, 1, 96)
    new = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, min(32768, 200000 // n))
    return {"op": op, "requests": n, "ctx": min(ctx, max(1, 4000000 // (n * new))), "new": new, "page": page, "ragged": rng.random() < 0.5,
            "type": rng.choice(["f32", "f16", "bf16"]), **layout}


# ---- lengths (from the case alone) -------------------------------------------------------------

def _lengths(case):
    """(cached rows, new rows) of each request."""
    n, ctx, new = case["requests"], case.get("ctx", 100), case["new"]
    r = random.Random(n * 1000003 + ctx * 1009 + new)
    if case.get("ragged"):
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
    if case["op"] == "sample":
        return _prepare_sample(case, g, rng)
    past, counts = _lengths(case)
    n, rows = len(past), sum(counts)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    s = {"case": case, "rows": rows, "n_past": _i32(past), "cu": _i32(cu), "most_new": max(counts), "most_keys": max(p + c for p, c in zip(past, counts))}
    if case["op"] == "accept":
        return _prepare_accept(s, case, counts, g, rng)
    page = case["page"]
    need = [-(-(p + c) // page) for p, c in zip(past, counts)]
    pages, blocks = sum(need) + 3, -(-s["most_keys"] // page)
    host, table, at = torch.randperm(pages, generator=g, device="cuda").int().cpu(), torch.full((n, blocks), -1, dtype=torch.int32), 0
    for i, c in enumerate(need):
        table[i, :c] = host[at:at + c]
        at += c
    kvd = case["kv_heads"] * case["dim"]
    kept = {"device": "cuda", "generator": g}
    # a calibrated factor for each kv head: a standard deviation is 20 to 50 codes
    s["k_scale"], s["v_scale"] = (1 / (20 + 30 * torch.rand(case["kv_heads"], **kept)) for _ in range(2))
    s["k"], s["v"] = ((torch.randn(pages * page, kvd, device="cuda", generator=g, dtype=torch.float16) * 35).clamp(-F8_MOST, F8_MOST).to(F8) for _ in range(2))
    s.update(table=table.cuda(), pool_pages=pages)
    if case["op"] == "append":
        t, slot, pos = table.tolist(), [], []
        for i, c in enumerate(counts):
            for k in range(past[i], past[i] + c):
                slot.append(t[i][k // page] * page + k % page)
                pos.append(k)
        s.update(row_slot=_i32(slot), row_pos=_i32(pos), row_mask=torch.zeros(rows, dtype=torch.int64, device="cuda"))
        d, width = case["dim"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        s["x"] = (torch.randn(rows, width, **kept) * 1.5).to(DTYPE[case["type"]])
        s["q_norm"], s["k_norm"] = (1 + 0.1 * torch.randn(d, **kept) for _ in range(2))
        inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        angle = torch.arange(s["most_keys"], device="cuda").double()[:, None] * inv
        s["rot"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        return s
    bits, depth = _masks(_trees(rng, counts), counts)
    s.update(row_slot=torch.full((rows,), -1, dtype=torch.int32, device="cuda"), row_pos=_i32(depth), row_mask=torch.tensor(bits, dtype=torch.int64, device="cuda"))
    s["q"] = torch.randn(rows, case["heads"] * case["dim"], **kept).to(DTYPE[case["type"]])
    return s


def _rule(kind, rng):
    """(temperature, top_k, top_p, min_p, repetition penalty)"""
    if kind == "mixed":
        kind = rng.choice(["greedy", "plain", "top_k", "top_k", "top_p", "top_p", "min_p", "all", "all"])
    t = 0.0 if kind == "greedy" else rng.choice([0.6, 0.7, 0.9, 1.0, 1.2])
    k = rng.choice([5, 20, 50, 50, 200]) if kind in ("top_k", "all") else 0
    p = rng.choice([0.8, 0.9, 0.95]) if kind in ("top_p", "all") else 1.0
    m = rng.choice([0.02, 0.05, 0.1]) if kind == "min_p" or kind == "all" and rng.random() < 0.5 else 0.0
    return t, k, p, m, rng.choice([1.0, 1.05, 1.1])


def _prepare_sample(case, g, rng):
    rows, vocab = case["rows"], case["vocab"]
    kept = {"device": "cuda", "generator": g}
    # a bell of unlikely tokens and, as far as there are that many, a few dozen likely ones whose logits fall off
    x = torch.randn(rows, vocab, **kept) * 2
    likely = min(40, vocab // 4)
    at = (torch.randint(0, vocab, (rows, 1), **kept) + torch.arange(likely, device="cuda") * (vocab // likely)) % vocab   # each once
    lift = 12 + 3 * torch.rand(rows, 1, **kept) - torch.arange(likely, device="cuda") * torch.rand(rows, 1, **kept) * 0.4
    x.scatter_(1, at, lift + 0.5 * torch.randn(rows, likely, **kept))
    rule = [_rule(case["rule"], rng) for _ in range(rows)]
    s = {"case": case, "x": x.to(DTYPE[case["type"]]), "u": torch.rand(rows, **kept), "temperature": torch.tensor([r[0] for r in rule], device="cuda"),
         "top_k": _i32([r[1] for r in rule]), "top_p": torch.tensor([r[2] for r in rule], device="cuda"), "min_p": torch.tensor([r[3] for r in rule], device="cuda"),
         "penalty": torch.tensor([r[4] for r in rule], device="cuda")}
    # as the library takes them: five 4-byte fields a row
    s["rules"] = torch.stack([s["temperature"].view(torch.int32), s["top_k"], *(s[k].view(torch.int32) for k in ("top_p", "min_p", "penalty"))], 1).contiguous()
    if case["masks"]:
        words = -(-vocab // 32)
        def bits(share):                                       # every bit set with probability `share`
            b = torch.rand(rows, words * 32, **kept) < share
            w = (b.view(rows, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
            return torch.where(w >= 1 << 31, w - (1 << 32), w).int()
        s["allowed"], s["seen"] = bits(0.7), bits(0.05)
        s["allowed"][:, :1] |= 1                               # one at least
    return s


def _prepare_accept(s, case, counts, g, rng):
    rows, codes = s["rows"], case["codes"]
    parent = _trees(rng, counts) if case["tree"] else [j - 1 for c in counts for j in range(c)]
    s["sampled"] = torch.randint(0, 2048, (rows, codes), device="cuda", generator=g).int()
    start = torch.repeat_interleave(s["cu"][:-1], _i32(counts))
    before = torch.where(_i32(parent) < 0, 0, _i32(parent)) + start
    # a draft is what the row before was found to give, or differs in one code
    hit = torch.rand(rows, device="cuda", generator=g) < 0.7
    s["drafted"] = s["sampled"][before.long()].clone()
    s["drafted"][:, -1] += torch.where(hit, 0, 1).int()
    s["last"] = s["drafted"][s["cu"][:-1].long()].clone()      # the first row is what the cached ones gave
    s.update(parent=_i32(parent) if case["tree"] else None, row_slot=torch.arange(rows, device="cuda").int(), row_pos=torch.zeros_like(start),
             row_mask=torch.zeros(rows, dtype=torch.int64, device="cuda"), table=torch.zeros(len(counts), 16, dtype=torch.int32, device="cuda"), pool_pages=max(16, -(-rows // 16)))
    return s


# ---- one pass ----------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    with torch.no_grad():
        return {"append": _append, "attention": _attention, "sample": _sample, "accept": _accept}[op](s)


def _abi():
    at = str(Path(__file__).resolve().parent.parent / "navi-tts_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from navi_amd import abi
    return abi


def _stream():
    return torch.cuda.current_stream().cuda_stream


_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _handles(s):
    """The library's descriptions of the pool and the step, made once as a program keeps them, and the library."""
    if "handles" not in s:
        abi, c = _abi(), s["case"]
        pages = abi.KvPages(c["requests"], c.get("page", 16), s["pool_pages"], s["table"].shape[1], s["rows"], s["most_new"], s["table"].data_ptr(),
                            s["n_past"].data_ptr(), s["cu"].data_ptr(), s["row_slot"].data_ptr(), s["row_pos"].data_ptr(), s["row_mask"].data_ptr())
        heads = None if c["op"] == "accept" else abi.KvHeads(c["heads"], c["kv_heads"], c["dim"], abi.DT_F8E4M3, s["k_scale"].data_ptr(), s["v_scale"].data_ptr())
        s["handles"] = abi, pages, heads
    return s["handles"]


def _own_append(s):
    (abi, pages, heads), c, x = _handles(s), s["case"], s["x"]
    q = torch.empty(s["rows"], c["heads"] * c["dim"], dtype=x.dtype, device="cuda")
    abi.kv_append(pages, heads, x.data_ptr(), _TYPE[x.dtype], x.shape[1], s["k"].data_ptr(), s["v"].data_ptr(), s["k"].shape[1], q.data_ptr(), _TYPE[x.dtype],
                  q.shape[1], q_norm=s["q_norm"].data_ptr(), k_norm=s["k_norm"].data_ptr(), eps=EPS, rot=s["rot"].data_ptr(), n_rot=s["rot"].shape[0], stream=_stream())
    return {"q": q, "k": s["k"], "v": s["v"]}


def _own_attention(s):
    (abi, pages, heads), c, q = _handles(s), s["case"], s["q"]
    out = torch.empty_like(q)
    ws = torch.empty(abi.tree_workspace(pages, heads, s["most_keys"]), dtype=torch.uint8, device="cuda")
    abi.tree_attention(pages, heads, q.data_ptr(), _TYPE[q.dtype], q.shape[1], s["k"].data_ptr(), s["v"].data_ptr(), s["k"].shape[1],
                       1 / math.sqrt(c["dim"]), s["most_keys"], out.data_ptr(), out.shape[1], ws.data_ptr(), ws.numel(), stream=_stream())
    return out


def _own_sample(s):
    abi, x, rows, masks = _abi(), s["x"], s["case"]["rows"], s["case"]["masks"]
    token, logprob = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
    ws = torch.empty(abi.sample_workspace(rows, x.shape[1]), dtype=torch.uint8, device="cuda")
    abi.sample_rows(x.data_ptr(), _TYPE[x.dtype], x.shape[1], rows, x.shape[1], s["rules"].data_ptr(), rows, s["u"].data_ptr(), token.data_ptr(),
                    logprob=logprob.data_ptr(), allowed=s["allowed"].data_ptr() if masks else None, ld_allowed=s["allowed"].shape[1] if masks else 0,
                    seen=s["seen"].data_ptr() if masks else None, ld_seen=s["seen"].shape[1] if masks else 0, ws=ws.data_ptr(), ws_bytes=ws.numel(), stream=_stream())
    return {"token": token, "logprob": logprob}


def _own_accept(s):
    (abi, pages, _), n, codes = _handles(s), s["case"]["requests"], s["case"]["codes"]
    i32 = {"dtype": torch.int32, "device": "cuda"}
    path, accept, then = torch.empty(n, s["most_new"], **i32), torch.empty(n, **i32), torch.empty(n, codes, **i32)
    abi.draft_accept(pages, s["drafted"].data_ptr(), codes, s["sampled"].data_ptr(), codes, codes, path.data_ptr(), s["most_new"], accept.data_ptr(), then.data_ptr(),
                     parent=None if s["parent"] is None else s["parent"].data_ptr(), last=s["last"].data_ptr(), stream=_stream())
    return {"path": path, "accept": accept, "next": then}


_OWN = {"append": _own_append, "attention": _own_attention, "sample": _own_sample, "accept": _own_accept}


# ---- the plain forms ---------------------------------------------------------------------------

def _rows_of(cu, rows):
    """Request and index in it of every row."""
    r = torch.arange(rows, device="cuda", dtype=torch.int32)
    req = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    return req, r - cu[req]


def _to_f8(x, scale):
    """[rows][kv heads][dim] in units of each head's factor, rounded to 8 bits; past the largest: the largest."""
    return (x / scale[:, None]).clamp(-F8_MOST, F8_MOST).to(F8).reshape(x.shape[0], -1)


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
    s["k"].view(torch.uint8)[at] = _to_f8(y[:, hq:], s["k_scale"]).view(torch.uint8)
    s["v"].view(torch.uint8)[at] = _to_f8(x[:, hq + hk:], s["v_scale"]).view(torch.uint8)
    return {"q": y[:, :hq].reshape(s["rows"], -1).to(s["x"].dtype), "k": s["k"], "v": s["v"]}


def _attention(s):
    c, n, d, hk = s["case"], s["case"]["requests"], s["case"]["dim"], s["case"]["kv_heads"]
    g, wide, page = c["heads"] // hk, s["most_new"], c["page"]
    req, j = _rows_of(s["cu"], s["rows"])
    at = torch.arange(s["most_keys"], device="cuda", dtype=torch.int32)
    slot = (s["table"][:, (at // page).long()].clamp(min=0) * page + at % page).long()

    def cached(x, scale):
        x = x.view(torch.uint8)[slot].view(F8).view(n, -1, hk, d).float()
        return x * scale[:, None]

    k = cached(s["k"], s["k_scale"]).permute(0, 2, 3, 1)                                  # [n][kv head][dim][key]
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
    v = cached(s["v"], s["v_scale"]).permute(0, 2, 1, 3)
    o = torch.matmul(p.view(n, hk, g * wide, -1), v.contiguous()).view(n, hk, g, wide, d) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(n, wide, -1)[req, j].to(s["q"].dtype)


def _set(words, vocab):
    """Bits of [rows][words] as truth values [rows][vocab]."""
    return ((words[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().reshape(words.shape[0], -1)[:, :vocab]


def _sample(s):
    """The order is that of the logits, the lowest index first among equals; weights and their sums in 64 bits, since a
    number of the draw may lie next to a border."""
    x, vocab = s["x"].float(), s["case"]["vocab"]
    if s["case"]["masks"]:
        pen = s["penalty"][:, None]
        x = torch.where(_set(s["seen"], vocab), torch.where(x > 0, x / pen, x * pen), x)
        x = torch.where(_set(s["allowed"], vocab), x, -math.inf)
    v, at = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    w = torch.exp((v.double() - v[:, :1].double()) / t)
    k = torch.where(s["top_k"] < 1, vocab, s["top_k"])[:, None]
    w = torch.where(torch.arange(vocab, device="cuda") < k, w, 0.0)
    p = torch.where(s["top_p"] < 1, s["top_p"], math.inf).double()[:, None]
    before = w.cumsum(1) - w
    keep = (before < p * w.sum(1, keepdim=True)) & (w >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, at, torch.where(keep, w, 0.0))                    # back in the tokens' order
    upto = w.cumsum(1)
    total = upto[:, -1:]
    token = (upto <= s["u"].double()[:, None] * total).sum(1).clamp(max=vocab - 1)
    logprob = torch.log(w.gather(1, token[:, None]) / total)[:, 0]
    return {"token": torch.where(greedy, at[:, 0], token).int(), "logprob": torch.where(greedy, 0.0, logprob).float()}


def _accept(s):
    """A row is taken if the row before it is, its codes are those sampled there, and no earlier sibling has the same."""
    n, wide, rows = s["case"]["requests"], s["most_new"], s["rows"]
    req, j = _rows_of(s["cu"], rows)
    start = s["cu"][req]
    parent = s["parent"] if s["parent"] is not None else j - 1
    given = torch.where((parent < 0)[:, None], s["last"][req], s["sampled"][(start + parent.clamp(min=0)).long()])
    fits = (s["drafted"] == given).all(1)
    p = torch.full((n, wide), -2, dtype=torch.int64, device="cuda")                       # -2: no such row, or not as sampled
    p[req, j.long()] = torch.where(fits, parent, -2).long()
    node = torch.arange(wide, device="cuda")
    first = ((p[:, :, None] == p[:, None, :]) & (node < node[:, None])).any(-1)           # an earlier sibling fits
    p = torch.where(first, -2, p)
    # every row's ancestors by squaring; a row counts if its topmost one is a root
    link = ((p[:, :, None] == node) | (node[:, None] == node)).float()
    reach = _squared(_squared(_squared(_squared(_squared(_squared(link))))))
    taken = ((reach > 0) & (p == -1)[:, None, :]).any(-1)
    accept = taken.sum(1, dtype=torch.int32)
    order = torch.sort(torch.where(taken, node, wide), dim=1).values
    path = torch.where(node < accept[:, None], order, 0).int()
    end = torch.where(accept > 0, s["cu"][:-1] + path.gather(1, (accept - 1).clamp(min=0).long()[:, None])[:, 0], 0)
    then = torch.where((accept > 0)[:, None], s["sampled"][end.long()], s["last"])
    return {"path": path, "accept": accept, "next": then}


def _squared(r):
    return ((r @ r) > 0).float()


# ---- the work, and the same in 64 bits ---------------------------------------------------------

def work(case):
    if case["op"] == "sample":
        size = 4 if case["type"] == "f32" else 2
        masks = 2 * 4 * -(-case["vocab"] // 32) if case["masks"] else 0
        # the logits, a row's rules, number and results; the exponential and two sums of a weight
        return {"bytes": case["rows"] * (case["vocab"] * size + masks + 32.0), "flops": 4.0 * case["rows"] * case["vocab"]}
    past, counts = _lengths(case)
    n, rows = len(past), sum(counts)
    if case["op"] == "accept":
        return {"bytes": rows * (8.0 * case["codes"] + 8) + n * (8.0 * case["codes"] + 4.0 * max(counts) + 8), "flops": rows * (case["codes"] + 2.0)}
    d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "append":
        reads = rows * ((hq + 2 * hk) * d * size + 8) + 4.0 * d * min(rows, case["ctx"] + case["new"])
        return {"bytes": reads + rows * d * (hq * size + 2 * hk), "flops": 10.0 * rows * (hq + hk) * d}
    keys = sum(p + c for p, c in zip(past, counts))
    pairs = sum((p + c / 2) * c for p, c in zip(past, counts))
    return {"bytes": 2.0 * keys * hk * d + 2.0 * rows * hq * d * size + 12.0 * rows + 4.0 * sum(-(-(p + c) // case["page"]) for p, c in zip(past, counts)),
            "flops": 4.0 * pairs * hq * d}


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return globals()["_exact_" + case["op"]](s, case)


def _exact_append(s, case):
    """The cache's new rows before they are rounded."""
    d, hq, hk, rows = case["dim"], case["heads"], case["kv_heads"], s["rows"]
    x = s["x"].double().view(rows, hq + 2 * hk, d)
    turn = torch.complex(s["rot"][:, :d // 2].double(), s["rot"][:, d // 2:].double())[s["row_pos"].long()][:, None]

    def head(a, w):
        a = a / (a.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        z = torch.complex(a[..., :d // 2].contiguous(), a[..., d // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    k, v, at = s["k"].double(), s["v"].double(), s["row_slot"].long()
    k[at] = (head(x[:, hq:hq + hk], s["k_norm"]) / s["k_scale"].double()[:, None]).reshape(rows, -1).clamp(-F8_MOST, F8_MOST)
    v[at] = (x[:, hq + hk:] / s["v_scale"].double()[:, None]).reshape(rows, -1).clamp(-F8_MOST, F8_MOST)
    return {"q": head(x[:, :hq], s["q_norm"]).reshape(rows, -1), "k": k, "v": v}


def _exact_attention(s, case):
    d, hk, g, page = case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"], case["page"]
    cu, past, table, out = s["cu"].tolist(), s["n_past"].tolist(), s["table"].long(), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["requests"]):
        c, keys = cu[i + 1] - cu[i], past[i] + cu[i + 1] - cu[i]
        at = torch.arange(keys, device="cuda")
        slot = table[i, at // page] * page + at % page
        k, v = (s[x].view(torch.uint8)[slot].view(F8).double().view(keys, hk, d) for x in ("k", "v"))
        node = torch.arange(c, device="cuda")
        seen = torch.ones(c, keys, dtype=torch.bool, device="cuda")
        seen[:, past[i]:] = ((s["row_mask"][cu[i]:cu[i + 1], None] >> node) & 1).bool()
        q = s["q"][cu[i]:cu[i + 1]].double().view(c, hk, g, d)
        for h in range(hk):
            a = (q[:, h].reshape(c * g, d) @ k[:, h].T * (s["k_scale"][h].double() / d ** 0.5)).masked_fill(~seen.repeat_interleave(g, 0), -math.inf)
            out[cu[i]:cu[i + 1], h * g * d:(h + 1) * g * d] = (torch.softmax(a, -1) @ v[:, h] * s["v_scale"][h].double()).view(c, g * d)
    return out


def _exact_sample(s, case):
    """Row by row on the host: what is left is found by value, without sorting the tokens' order away."""
    x, vocab = s["x"].float().cpu().numpy(), case["vocab"]
    token, logprob = [], []
    for r in range(case["rows"]):
        a, (t, k, p, m, pen), u = x[r].copy(), (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "penalty")), float(s["u"][r])
        if case["masks"]:
            words = [np.unpackbits(s[n][r].cpu().numpy().view(np.uint8), bitorder="little")[:vocab].astype(bool) for n in ("seen", "allowed")]
            a = np.where(words[0], np.where(a > 0, a / np.float32(pen), a * np.float32(pen)), a).astype(np.float32)
            a[~words[1]] = -np.inf
        if t <= 0:
            token.append(int(a.argmax()))
            logprob.append(0.0)
            continue
        w = np.exp((a.astype(np.float64) - float(a.max())) / t)
        if 1 <= k < vocab:
            edge = np.partition(a, vocab - int(k))[vocab - int(k)]                        # the k-th largest
            tied = np.flatnonzero(a == edge)
            w[a < edge] = 0
            w[tied[int(k) - int((a > edge).sum()):]] = 0
        largest = a.argmax()
        if p < 1:
            order = np.lexsort((np.arange(vocab), -a.astype(np.float64)))
            run = np.cumsum(w[order])
            last = int(np.searchsorted(run, p * math.fsum(w)))                            # the first whose mass reaches it
            w[order[last + 1:]] = 0
        first = w[largest]
        w[w < m] = 0
        w[largest] = first
        upto = np.cumsum(w)
        i = int(np.searchsorted(upto, u * upto[-1], side="right"))
        token.append(min(i, vocab - 1))
        logprob.append(math.log(w[token[-1]] / math.fsum(w)))
    return {"token": torch.tensor(token, dtype=torch.int32), "logprob": torch.tensor(logprob, dtype=torch.float64)}


def _exact_accept(s, case):
    cu, drafted, sampled, last = (s[k].tolist() for k in ("cu", "drafted", "sampled", "last"))
    parent = None if s["parent"] is None else s["parent"].tolist()
    paths, accept, then = [], [], []
    for i in range(case["requests"]):
        at, want, path = -1, last[i], []
        while True:
            fit = [j for j in range(cu[i + 1] - cu[i]) if (parent[cu[i] + j] if parent else j - 1) == at and drafted[cu[i] + j] == want]
            if not fit:
                break
            at, want = fit[0], sampled[cu[i] + fit[0]]
            path.append(at)
        paths.append(path + [0] * (s["most_new"] - len(path)))
        accept.append(len(path))
        then.append(want)
    return {"path": _i32(paths), "accept": _i32(accept), "next": _i32(then)}
