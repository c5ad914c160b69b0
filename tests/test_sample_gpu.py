"""navi_sample_rows against its definition in 64 bits: the same token for every row."""
import numpy as np
import pytest
import torch

from navi_amd import abi
from sample_util import OFF, TYPE, Call, token_of, weights, words_of

pytestmark = pytest.mark.gpu

RULES = [OFF, (0.0, 0, 1, 0, 1), (0.7, 50, 1, 0, 1), (0.9, 0, 0.9, 0, 1), (1.2, 0, 1, 0.05, 1), (0.8, 40, 0.95, 0.02, 1), (1.0, 1, 1, 0, 1), (1.0, 0, 0.0, 0, 1),
         (1.0, 0, 1, 1.0, 1), (2.0, 1000, 0.5, 0, 1), (0.3, 5, 0.99, 0.5, 1), (1.0, 0, 0.999, 1e-4, 1)]


def logits(rows, vocab, seed, kind="f32", spread=2.0):
    """A bell, and a few likely tokens."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    n = min(vocab, 12)
    for r in range(rows):
        x[r, torch.randperm(vocab, generator=g)[:n]] += 4 + 6 * torch.rand(n, generator=g)
    return x.to(TYPE[kind][0]), torch.rand(rows, generator=g).numpy()


SIZES = [1, 2, 3, 5, 63, 64, 65, 255, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4097, 8192, 8193, 16383, 16384, 16385, 20001, 65537, 151936]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", SIZES)
def test_sizes_and_rules(vocab, kind):
    """Every rule at every size: a token to the text vocabulary, on both sides of each border between kernels."""
    x, u = logits(len(RULES), vocab, vocab, kind)
    Call(x, RULES, u).check()


@pytest.mark.parametrize("vocab,rows", [(262144, 3), (262145, 2), (1 << 20, 2), (30000, 140), (5000, 300)])
def test_largest_vocabularies_and_many_rows(vocab, rows):
    """Chunks of 4096 and of 16384 tokens, 64 of each."""
    x, u = logits(rows, vocab, rows)
    Call(x, [RULES[i % len(RULES)] for i in range(rows)], u).check()


@pytest.mark.parametrize("vocab", [37, 1000, 2048, 9000, 16384, 20000, 70000])
@pytest.mark.parametrize("levels", [1, 2, 5])
def test_ties(vocab, levels):
    """Few different logits, so that the border falls among equal ones and the indexes decide; one level: all equal, and more tokens
    in a bin than LDS holds."""
    g = torch.Generator().manual_seed(vocab + levels)
    x = torch.randint(0, levels, (10, vocab), generator=g).float() * 0.1
    k = max(1, vocab // 3)
    rules = [(1.0, k, 1, 0, 1), (1.0, k, 0.7, 0, 1), (1.0, 0, 0.37, 0, 1), (1.0, 0, 1, 0.97, 1), (0.01, k, 0.6, 0, 1), (5.0, vocab - 1, 0.999, 0, 1), (1.0, 1, 1, 0, 1),
             (1.0, vocab, 1, 0, 1), (1.0, vocab + 5, 0.123, 0, 1), (1.0, 2, 0.9, 0.5, 1)]
    Call(x, rules, torch.rand(10, generator=g).numpy()).check()


@pytest.mark.parametrize("vocab", [100, 2048, 12000, 40000])
def test_values_that_are_no_ordinary_numbers(vocab):
    """Infinities, NaN, both zeros, the largest and the smallest numbers; temperatures from the least to infinity."""
    inf, nan, big = float("inf"), float("nan"), float(np.finfo(np.float32).max)
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(12, vocab, generator=g)
    x[0, ::2], x[0, 1::3] = -inf, nan
    x[1, 5], x[1, vocab - 1] = inf, inf
    x[2, :], x[2, vocab // 2] = -inf, -3.0
    x[3, :] = -inf
    x[4, :] = nan
    x[5, ::3], x[5, 1::3], x[5, 2::3] = 0.0, -0.0, -1e-45
    x[6, 7], x[6, 8], x[6, 9] = big, big, -big
    x[7] = -x[7].abs() * 1e30
    x[8] *= 1e-40
    x[9, 3] = 3e38
    x[10, :] = -big
    rules = [(1.0, 0, 0.9, 0, 1), (1.0, 5, 0.9, 0.1, 1), (1.0, 0, 0.5, 0.5, 1), OFF, (0.5, 3, 1, 0, 1), (1.0, 0, 0.6, 0, 1), (1e-30, 2, 0.9, 0.1, 1), (1e30, 0, 0.4, 0, 1),
             (1e-45, 7, 0.9, 0, 1), (inf, 0, 0.3, 0, 1), (3e38, 9, 1, 0.2, 1), (nan, 4, nan, nan, nan)]
    for shift in range(3):
        Call(x, rules[shift:] + rules[:shift], torch.rand(12, generator=g).numpy()).check()


@pytest.mark.parametrize("vocab", [2048, 20000])
def test_zeros_of_both_signs_are_equal_where_bins_are_narrow(vocab):
    """At temperatures near the least, a bin holds few float keys, and 0 and -0 are neighbours among them: more than can be ranked at once."""
    x = torch.full((6, vocab), -1.0)
    x[:, 3:900:2], x[:, 4:900:2] = -0.0, 0.0
    u = np.array([0.0, 0.3, 0.9, 0.999, 0.5, 1.0], np.float32)
    for t in (1e-43, 1e-44, 1e-41):
        Call(x, [(t, k, 1, 0, 1) for k in (300, 65, 600, 880, 1, 897)], u).check()
        Call(x, [(t, 0, p, 0, 1) for p in (0.3, 0.08, 0.6, 0.97, 1e-6, 0.5)], u).check()


@pytest.mark.parametrize("vocab", [300, 2048, 33333])
def test_numbers_at_and_past_the_ends(vocab):
    """0 is the first kept token, what is not below 1 the last quantile, NaN and below 0 as 0."""
    x, _ = logits(7, vocab, 3)
    u = np.array([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, np.nan, 1e-38], np.float32)
    for rule in (OFF, (0.9, 20, 0.9, 0, 1), (1, 0, 1, 0.3, 1)):
        got = Call(x, [rule], np.where(np.isnan(u), 0, u)).check()
        c = Call(x, [rule], u).go()
        torch.cuda.synchronize()
        assert c.token.tolist() == got


@pytest.mark.parametrize("vocab", [64, 100, 2049, 16384, 40001])
def test_allowed_and_seen_tokens(vocab):
    """Sets a row and one for all, wider strides, bits past the last token set, a row with one allowed token and one with none; the penalty on
    both signs, off for 0, 1 and NaN."""
    rng = np.random.default_rng(vocab)
    x, u = logits(9, vocab, 5)
    n = -(-vocab // 32)
    allow = np.stack([words_of(rng.random(vocab) < 0.6, n + 3) for _ in range(9)])
    allow[2] = 0
    allow[3] = words_of(np.arange(vocab) == vocab - 1, n + 3)
    allow[4] = words_of(np.zeros(vocab, bool), n + 3)
    allow[:, n - 1] |= np.uint32(~((1 << ((vocab - 1) % 32 + 1)) - 1) & 0xFFFFFFFF)             # past the last token
    allow[:, n:] = 0xFFFFFFFF
    seen = np.stack([words_of(rng.random(vocab) < 0.3, n) for _ in range(9)])
    pens = [1.05, 1.5, 1.1, 1.0, 2.0, 0.7, 0.0, float("nan"), float("inf")]
    rules = [(0.8, [0, 30][i % 2], [1, 0.9][i // 2 % 2], 0, p) for i, p in enumerate(pens)]
    rules[5] = (0.0, 0, 1, 0, 1.3)
    got = Call(x, rules, u, allowed=allow, seen=seen).check()
    assert got[2] == got[4] == -1 and got[3] == vocab - 1
    Call(x, rules, u, allowed=allow[:1], seen=seen[1:2]).check()
    Call(x, rules, u, seen=seen).check()
    Call(x, rules, u, allowed=allow).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,pad,offset", [(1000, 1, 0), (1000, 0, 1), (2048, 3, 2), (2046, 2, 4), (20001, 7, 3), (20000, 8, 1)])
def test_strides_and_alignment(kind, vocab, pad, offset):
    x, u = logits(5, vocab, pad, kind)
    Call(x, [(0.9, 40, 0.95, 0.01, 1)], u, pad=pad, offset=offset, ld_token=16, want_logprob=pad != 3).check()


@pytest.mark.parametrize("vocab", [2048, 20000])
def test_a_row_does_not_depend_on_the_others(vocab):
    """One row alone, among few and among enough that longer chunks are taken."""
    x, u = logits(300, vocab, 11)
    rules = [RULES[i % len(RULES)] for i in range(300)]
    both = lambda c: (c.go(), torch.cuda.synchronize(), (c.token.tolist(), c.logprob.tolist()))[2]
    tokens, lps = both(Call(x, rules, u))
    for i in (0, 3, 5, 137, 299):
        t, lp = both(Call(x[i:i + 1], rules[i:i + 1], u[i:i + 1]))
        assert t[0] == tokens[i] and abs(lp[0] - lps[i]) <= 2.0 ** -23 * abs(lps[i]) + 2.0 ** -27   # both within check()'s bound
    assert both(Call(x, rules, u)) == (tokens, lps)


@pytest.mark.parametrize("vocab", [600, 20000])
@pytest.mark.parametrize("rule", [OFF, (0.7, 30, 1, 0, 1), (1.0, 0, 0.8, 0, 1), (0.9, 50, 0.9, 0.05, 1)])
def test_evenly_spread_numbers_give_the_distribution(vocab, rule):
    """4096 numbers, one in the middle of every 4096th: a token of probability p comes p 4096 times, one more or less."""
    n = 4096
    x, _ = logits(1, vocab, 21)
    c = Call(x.expand(n, vocab).contiguous(), [rule], (np.arange(n) + 0.5) / n).go()
    torch.cuda.synchronize()
    w = weights(x[0].numpy(), rule)
    count = np.bincount(c.token.cpu().numpy(), minlength=vocab)
    assert np.abs(count - n * w / w.sum()).max() <= 1.001


def test_random_calls():
    """Sizes, rules, types and masks drawn together."""
    rng = np.random.default_rng(8)
    for _ in range(40):
        vocab, rows = int(np.exp(rng.uniform(0, np.log(60000)))), int(rng.integers(1, 9))
        x, u = logits(rows, vocab, int(rng.integers(1 << 30)), ["f32", "f16", "bf16"][rng.integers(3)], float(rng.choice([0.3, 2, 8])))
        rules = [(float(rng.choice([0, 0.1, 0.7, 1, 3])), int(rng.choice([0, 1, 7, 50, 3000])), float(rng.choice([1, 0.99, 0.9, 0.5, 0.1])),
                  float(rng.choice([0, 0.001, 0.1])), float(rng.choice([1, 1.1, 0.9]))) for _ in range(rows)]
        n = -(-vocab // 32)
        allow = np.stack([words_of(rng.random(vocab) < 0.8, n) for _ in range(rows)]) if rng.random() < 0.5 else None
        seen = np.stack([words_of(rng.random(vocab) < 0.2, n) for _ in range(rows)]) if rng.random() < 0.5 else None
        Call(x, rules, u, allowed=allow, seen=seen, pad=int(rng.integers(0, 5))).check()


@pytest.mark.parametrize("vocab", [2048, 40000])
def test_replayed_from_a_graph(vocab):
    """The captured call on new logits, numbers and rules, with eager calls between the replays."""
    rows = 6
    x, u = logits(rows, vocab, 1)
    c = Call(x, RULES[:rows], u)
    c.go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.go()
    for i in range(4):
        x, u = logits(rows, vocab, 50 + i)
        new = Call(x, RULES[i:i + rows], u)
        c.d_x.copy_(new.d_x)
        c.d_u.copy_(new.d_u)
        c.d_rules.copy_(new.d_rules)
        c.token.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        assert c.token.tolist() == new.check() and torch.equal(c.logprob, new.logprob)


def test_two_streams_at_once():
    """Each with its own workspace."""
    calls = [Call(*logits(4, 50000, i)[:1], RULES[2:6], logits(4, 50000, i)[1]) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s in zip(calls, streams):
            c.go(s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        assert c.token.tolist() == [w[0] for w in c.expect()]


def test_no_rows_and_the_librarys_stream():
    abi.sample_rows(0, 0, 8, 0, 8, 0, 0, 0, 0, stream=None)
    x, u = logits(3, 500, 2)
    c = Call(x, [RULES[5]], u)
    torch.cuda.synchronize()
    c.go(abi.lib().navi_device_stream())
    abi.lib().navi_device_synchronize()
    assert c.token.tolist() == [w[0] for w in c.expect()]


@pytest.mark.parametrize("vocab", [500, 2048, 20000])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_every_kind_of_nan_is_left_out(vocab, kind):
    """Signalling and quiet ones of both signs, among the likely tokens and instead of the likeliest."""
    x, u = logits(len(RULES), vocab, 77, kind)
    bits = {"f32": (np.int32, [0x7F800001, 0x7FC00000, 0x7FFFFFFF, -0x7FFFFF, -1, 0x7FBFFFFF]),
            "f16": (np.int16, [0x7C01, 0x7E00, 0x7FFF, -0x3FF, -1, 0x7DFF]), "bf16": (np.int16, [0x7F81, 0x7FC0, 0x7FFF, -0x7F, -1, 0x7FBF])}[kind]
    raw = x.view(torch.int32 if kind == "f32" else torch.int16)
    for r in range(len(RULES)):
        top = x[r].float().topk(3).indices
        raw[r, top[::2]] = bits[1][r % 6]
        raw[r, r::7] = bits[1][(r + 3) % 6]
    Call(x, RULES, u).check()


@pytest.mark.parametrize("vocab", [2048, 20000])
def test_rows_past_32_bits(vocab):
    """Three rows 2^31 - 1 elements apart, the last from the 2^32nd on."""
    x, u = logits(3, vocab, 17, "bf16")
    rules = [(0.9, 40, 0.95, 0, 1), (1.0, 0, 0.8, 0, 1), (1.1, 60, 1, 0.02, 1)]
    c = Call(x, rules, u)
    ld = (1 << 31) - 1
    far = torch.empty(2 * ld + vocab, dtype=torch.bfloat16, device="cuda")
    for r in range(3):
        far[r * ld:r * ld + vocab] = x[r].cuda()
    want = c.check()
    c.d_x, c.ld = far, ld
    c.token.fill_(-5)
    c.go()
    torch.cuda.synchronize()
    assert c.token.tolist() == want
