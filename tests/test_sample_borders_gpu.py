"""navi_sample_rows where a rule's border lies among many close logits: the kept tokens, seen in the drawn one and its log probability, are the
definition's. (A log probability shows one token too many or too few: the kept weights' sum goes with it.)"""
import numpy as np
import pytest
import torch

from sample_util import TYPE, Call

pytestmark = pytest.mark.gpu

BIN = np.log(2) / 4                    # of the logits that the kernel's sums take together, at temperature 1: multiples of it are where they meet


def check(x, rules, kind="f32"):
    """One row under every rule, each with a number near the start, in the middle and near the end."""
    x = torch.as_tensor(np.asarray(x), dtype=torch.float32).to(TYPE[kind][0])
    u = np.tile([0.03, 0.5, 0.97], len(rules))
    Call(x.expand(len(u), len(x)).contiguous(), [r for r in rules for _ in range(3)], u).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,sigma", [(20000, 0.3), (40000, 0.1), (40000, 1.0), (151936, 0.3)])
def test_flat_rows(vocab, sigma, kind):
    """Normal logits so flat that a border is one of thousands of tokens of a bin, next to 0 among them."""
    x = np.random.default_rng(vocab).standard_normal(vocab) * sigma
    rules = [(1.0, 0, p, 0, 1) for p in (0.4, 0.42, 0.44, 0.45, 0.9)] + [(3.0, 0, 0.43, 0, 1), (0.5, 0, 0.3, 0, 1)]
    rules += [(1.0, int(vocab * k), 1, 0, 1) for k in (0.01, 0.29, 0.3, 0.31, 0.32, 0.33)] + [(1.0, vocab // 3, 0.9, 0.3, 1), (2.5, vocab // 4, 0.99, 0, 1)]
    # the first few tokens of the bin below 0.1733 and of that below 0
    rules += [(1.0, int((x >= e * BIN).sum()) + n, 1, 0, 1) for e in (1, 0) for n in (1, 2, 70)]
    check(x, rules, kind)


@pytest.mark.parametrize("vocab", [2048, 20000])
def test_two_marked_bins_side_by_side(vocab):
    """100 logits at the lower end of a bin, 100 in the upper part of the bin below it: top_k ends in the one, top_p in the one or the other."""
    x = np.full(vocab, -100.0)
    at = np.random.default_rng(1).permutation(vocab)
    x[at[:100]], x[at[100:200]] = np.linspace(0.1738, 0.1868, 100), np.linspace(0.1255, 0.1725, 100)
    for kind in ("f32", "f16", "bf16"):
        check(x, [(1.0, k, p, 0, 1) for k in (101, 110, 150, 190) for p in (1.0, 0.6, 0.95, 0.999)], kind)
        check(x, [(1.0, 0, p, m, 1) for p in (0.51, 0.53, 0.6, 0.8, 0.97) for m in (0.0, 0.98)], kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("temperature,edge", [(1.0, 1), (1.0, 0), (1.0, -1), (1.0, 7), (1.0, -31), (1.0, 400), (1.0, -3000), (0.7, 2), (3.0, -2), (200.0, 5), (1e-3, 3)])
@pytest.mark.parametrize("vocab", [5000, 30000])
def test_dense_on_both_sides_of_a_bins_end(vocab, temperature, edge, kind):
    """Close logits on both sides of an end between two bins, and rules that end just below it, next to rules that mark the bin above."""
    rng = np.random.default_rng(abs(edge) + vocab)
    width, e = BIN * temperature, edge * BIN * temperature
    x = np.full(vocab, e - 90 * width)
    at = rng.permutation(vocab)
    near, low, high = 1500, 300, 40
    x[at[:near]] = e + (rng.random(near) - 0.5) * 0.01 * width
    x[at[near:near + low]] = e - rng.random(low) * width
    x[at[near + low:near + low + high]] = e + rng.random(high) * 2 * width
    x = x.astype(np.float32)
    above = int((torch.as_tensor(x).to(TYPE[kind][0]).double().numpy() >= e).sum())
    t = temperature
    ks = [k for k in (above - 70, above - 1, above, above + 1, above + 2, above + 30, above + 65, above + 300, above + 800) if k > 0]
    check(x, [(t, k, 1, 0, 1) for k in ks] + [(t, k, 0.999, 0, 1) for k in ks] + [(t, 0, p, 0, 1) for p in (0.3, 0.47, 0.5, 0.53, 0.8)], kind)


@pytest.mark.parametrize("vocab", [16384, 20000, 151936])
def test_borders_at_many_places(vocab):
    """A bell's borders one by one: the first and the last tokens of its bins, by top_k."""
    x = np.random.default_rng(3).standard_normal(vocab) * 2.5
    x = x.astype(np.float32)
    edges = np.arange(-4, 12) * BIN
    ks = sorted({max(1, int((x >= e).sum()) + n) for e in edges for n in (-1, 0, 1, 9, 70)})
    check(x, [(1.0, k, 1, 0, 1) for k in ks[::2]] + [(1.0, k, 0.9, 0, 1) for k in ks[1::2]])
