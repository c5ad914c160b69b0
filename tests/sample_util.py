"""Shared by the tests of navi_sample_rows: its definition in 64 bits, row by row, and calls of it."""
from __future__ import annotations

import numpy as np
import torch

from navi_amd import abi

TYPE = {"f32": (torch.float32, abi.DT_F32), "f16": (torch.float16, abi.DT_F16), "bf16": (torch.bfloat16, abi.DT_BF16)}
OFF = (1.0, 0, 1.0, 0.0, 1.0)          # temperature, top_k, top_p, min_p, repetition penalty


def bits_of(words, vocab):
    return np.unpackbits(np.ascontiguousarray(words).view(np.uint8), bitorder="little")[:vocab].astype(bool)


def words_of(bits, n_words=None):
    b = np.zeros(32 * (n_words or -(-len(bits) // 32)), bool)
    b[:len(bits)] = bits
    return np.packbits(b, bitorder="little").view(np.uint32)


def as_seen(x, rule, allowed=None, seen=None):
    """Logits as the rule sees them (f32)."""
    x = np.asarray(x, np.float32).copy()
    pen = np.float32(rule[4])
    with np.errstate(all="ignore"):
        if seen is not None and pen > 0:
            x = np.where(seen, np.where(x > 0, x / pen, x * pen), x).astype(np.float32)
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, np.finfo(np.float32).max)
    if allowed is not None:
        x[~allowed] = -np.inf
    return x


def weights(x, rule):
    """Kept weights over the largest, 0 for what is left out: None without a token."""
    t, k, p, m, _ = (float(np.float32(r)) if i != 1 else int(r) for i, r in enumerate(rule))
    if not np.isfinite(x).any():
        return None
    order = np.lexsort((np.arange(len(x)), -x.astype(np.float64)))
    order = order[np.isfinite(x[order])]
    w = np.zeros(len(x))
    if not t > 0:
        w[order[0]] = 1
        return w
    s = np.exp((x[order].astype(np.float64) - float(x[order[0]])) / t)
    if k >= 1:
        s[k:] = 0
    if p < 1:
        upto = np.cumsum(s)
        last = int(np.searchsorted(upto, p * upto[-1]))
        s[max(last, 0) + 1:] = 0
    if m > 0:
        s[s < min(m, 1.0)] = 0
    w[order] = s
    return w


def token_of(w, u):
    """(token, log probability) of the number u."""
    if w is None:
        return -1, -np.inf
    u = float(np.float32(u))
    u = min(u, 1 - 2.0 ** -24) if u > 0 else 0.0
    upto = np.cumsum(w)
    i = int(np.searchsorted(upto, u * upto[-1], side="right"))
    i = min(i, int(np.flatnonzero(w)[-1]))
    return i, float(np.log(w[i] / upto[-1]))


class Call:
    """Rows of logits (torch, CPU) on the GPU, `ld` and `offset` elements of padding as given, and what a call gives for them."""

    def __init__(self, x, rules, u, *, pad=0, offset=0, allowed=None, seen=None, ld_token=1, shared=False, want_logprob=True):
        self.rows, self.vocab = x.shape
        self.kind = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[x.dtype]
        self.x, self.rules, self.u = x, rules, u
        self.ld, self.ld_token, self.offset = self.vocab + pad, ld_token, offset
        flat = torch.full((offset + self.rows * self.ld,), float("nan"), dtype=x.dtype)
        flat[offset:].view(self.rows, self.ld)[:, :self.vocab] = x
        self.d_x = flat.cuda()
        raw = np.array([tuple(r) for r in rules], dtype=[("t", "<f4"), ("k", "<i4"), ("p", "<f4"), ("m", "<f4"), ("r", "<f4")])
        self.d_rules = torch.from_numpy(raw.view(np.int32).copy()).cuda()
        self.d_u = torch.tensor(np.asarray(u, np.float32)).cuda()
        self.allowed, self.seen = allowed, seen                  # [rows or 1][words] uint32, or None
        self.d_allowed, self.d_seen = (None if b is None else torch.from_numpy(np.ascontiguousarray(b).view(np.int32)).cuda() for b in (allowed, seen))
        self.token = torch.full((self.rows * ld_token,), -77, dtype=torch.int32, device="cuda")
        self.logprob = torch.full((self.rows,), 7.0, device="cuda") if want_logprob else None
        self.ws = torch.full((abi.sample_workspace(self.rows, self.vocab),), 0xFF, dtype=torch.uint8, device="cuda")

    def go(self, stream=None):
        ld = lambda b: 0 if b is None or b.shape[0] == 1 else b.shape[1]
        ptr = lambda t: None if t is None else t.data_ptr()
        abi.sample_rows(self.d_x.data_ptr() + self.offset * self.d_x.element_size(), TYPE[self.kind][1], self.ld, self.rows, self.vocab, self.d_rules.data_ptr(),
                        len(self.rules), self.d_u.data_ptr(), self.token.data_ptr(), ld_token=self.ld_token, logprob=ptr(self.logprob),
                        allowed=ptr(self.d_allowed), ld_allowed=ld(self.allowed), seen=ptr(self.d_seen), ld_seen=ld(self.seen),
                        ws=ptr(self.ws), ws_bytes=self.ws.numel(), stream=torch.cuda.current_stream().cuda_stream if stream is None else stream)
        return self

    def expect(self):
        at = lambda b, r: None if b is None else bits_of(b[r % b.shape[0]], self.vocab)
        out = []
        for r in range(self.rows):
            rule = self.rules[r % len(self.rules)]
            x = as_seen(self.x[r].float().numpy(), rule, at(self.allowed, r), at(self.seen, r))
            out.append(token_of(weights(x, rule), self.u[r]))
        return out

    def check(self):
        """Tokens as the definition's, log probabilities within half a step of f32 and 2^-28: a weight's unit is 2^-31 of it, and sums of
        them are at most that far off."""
        self.go()
        torch.cuda.synchronize()
        want = self.expect()
        got = self.token.cpu().view(self.rows, self.ld_token)
        bad = [(r, int(got[r, 0]), want[r], self.rules[r % len(self.rules)], float(self.u[r])) for r in range(self.rows) if int(got[r, 0]) != want[r][0]]
        assert not bad, bad[:4]
        assert bool((got[:, 1:] == -77).all()), "wrote beside its tokens"
        if self.logprob is not None:
            lp = np.array([w[1] for w in want])
            with np.errstate(invalid="ignore"):
                off = np.abs(self.logprob.cpu().double().numpy() - lp)
            ok = (off <= np.abs(lp) * 2.0 ** -24 + 2.0 ** -28) | (np.isneginf(lp) & np.isneginf(self.logprob.cpu().numpy()))
            assert ok.all(), (np.flatnonzero(~ok)[:4], off[~ok][:4])
        return got[:, 0].tolist()
