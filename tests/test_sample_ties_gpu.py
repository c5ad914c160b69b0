"""navi_sample_rows where the kept tokens are equal and the number lies on a border between them: numbers that sums in floating point meet
from either side."""
import numpy as np
import pytest
import torch

from sample_util import Call, weights, words_of

pytestmark = pytest.mark.gpu

# temperature, logit, 64 u, and which pieces of 256 tokens hold one allowed token: rows in which an empty piece's running sum, whose additions
# are associated in another way, lies above the border that its neighbour's meets
PIECES = [(16, 0.8, -2.0, 40, [0, 3, 5, 6, 9, 12, 13, 15]), (16, 0.9, 4.0, 40, [0, 1, 2, 3, 4, 9, 13, 15]), (16, 1.2, 2.0, 48, [3, 5, 7, 8, 9, 10, 12, 15]),
          (16, 0.9, 6.0, 48, [0, 1, 2, 3, 4, 5, 6, 7, 8, 10, 11, 12]), (64, 0.7, -4.0, 48, [5, 18, 19, 20, 22, 29, 49, 54]),
          (64, 1.2, -0.5, 32, [0, 7, 10, 11, 13, 19, 22, 29, 31, 50]), (64, 1.0, -3.0, 48, [6, 19, 22, 23, 32, 35, 38, 39, 44, 49, 52, 53]),
          (64, 0.9, 2.0, 56, [0, 4, 11, 16, 21, 22, 28, 31, 35, 38, 40, 44, 46, 47, 48, 50, 51, 53, 55, 56, 57, 59, 60, 62])]
# the same of chunks, with two logits in each that is not empty: tokens of a chunk, chunks, temperature, the logits, 64 u, the chunks
CHUNKS = [(4096, 17, 0.9, 3.0, 2.75, 32, [0, 1, 3, 4, 5, 7, 8, 10, 11, 12, 13, 14, 15, 16]), (4096, 17, 0.7, -2.5, -3.25, 32, [1, 3, 5, 7, 8, 10, 12, 13, 14, 16]),
          (4096, 38, 0.8, 4.5, 3.25, 28, [0, 1, 2, 4, 5, 7, 10, 14, 17, 23, 26, 27, 28, 34, 35, 36]),
          (4096, 64, 0.9, -3.5, -4.5, 20, [1, 5, 7, 9, 10, 14, 19, 21, 25, 36, 37, 39, 47, 49, 55, 63]),
          (16384, 38, 0.9, -5.5, -5.75, 52, [1, 4, 7, 9, 10, 11, 15, 16, 17, 20, 21, 23, 24, 35, 36, 37])]


@pytest.mark.parametrize("case", PIECES, ids=str)
def test_a_piece_without_a_kept_token_is_not_drawn_from(case):
    n, t, x, u, at = case
    allow = np.zeros(256 * n, bool)
    allow[[256 * p + (37 * p + 11) % 256 for p in at]] = True
    Call(torch.full((1, 256 * n), x), [(t, 0, 1, 0, 1)], [u / 64], allowed=words_of(allow)[None]).check()


@pytest.mark.parametrize("case", CHUNKS, ids=str)
def test_a_chunk_without_a_kept_token_is_not_drawn_from(case):
    """On a border between two pairs, the last token before it or the first behind it, but one of the two, and its log probability."""
    size, n, t, a, b, u, at = case
    x = torch.full((1, size * n), -float("inf"))
    for c in at:
        x[0, size * c + 100], x[0, size * c + 300] = a, b
    call = Call(x, [(t, 0, 1, 0, 1)], [u / 64]).go()
    torch.cuda.synchronize()
    i = u * len(at) // 64
    assert u * len(at) % 64 == 0
    assert call.token.item() in (size * at[i - 1] + 300, size * at[i] + 100)
    w = weights(x[0].numpy(), call.rules[0])
    assert abs(call.logprob.item() - np.log(w[call.token.item()] / w.sum())) <= 8 * 2.0 ** -24 + 2.0 ** -28


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("vocab", [2048, 16384, 20000, 151936])
def test_a_number_on_a_border_between_equal_tokens(vocab, kind):
    """2, 3, 4, 8 and 12 equal tokens, near each other and far apart, under u = j / 64: the first one at which the sum passes u, j n / 64 whole or not, is token
    floor(j n / 64) of the n. All rows in one call, and a few a call: the same."""
    rng = np.random.default_rng(vocab)
    rows = 240
    x = torch.full((rows, vocab), -float("inf"))
    u, want, rules = [], [], []
    for r in range(rows):
        n, j = int(rng.choice([2, 3, 4, 8, 12])), int(rng.integers(1, 64))
        if r % 3 < 2:
            j = int(rng.integers(1, 4)) * 16 if n % 3 else 48                                # on a border, but for 3 tokens
        width = vocab if r % 2 else 64
        at = np.sort(rng.integers(0, vocab - width + 1) + rng.permutation(width)[:n])
        x[r, at] = float(rng.integers(-400, 400)) / 16
        u.append(j / 64)
        want.append(int(at[j * n // 64]))
        rules.append((float(rng.choice([0.7, 0.9, 1.0, 1.3])), int(rng.choice([0, n, 50])), float(rng.choice([1.0, 0.9999])), 0, 1))
    x = x.to(kind)
    call = Call(x, rules, u).go()
    torch.cuda.synchronize()
    assert call.token.tolist() == want
    for r in range(0, rows, 6):
        few = Call(x[r:r + 6], rules[r:r + 6], u[r:r + 6]).go()
        torch.cuda.synchronize()
        assert few.token.tolist() == want[r:r + 6]
        assert torch.equal(few.logprob, call.logprob[r:r + 6])
