"""navi_tree_attention of 16-bit queries is off by its output's rounding, not by its probabilities': these travel as hi + lo
pairs of the cache's type whatever the queries' type. Scores nearly flat, so that the scores' own f32 roundings stay small."""
import numpy as np
import pytest

from kv_util import HALF_STEP, Step, random_tree

pytestmark = pytest.mark.gpu
SCALE = 0.01


def bound(s):
    """(out, bound) [rows][heads][dim] in 64 bits. With A = sum p |v| / sum p and n keys:
      scores: sums of `dim` f32 products, each rounding at most 2^-24 of sum |q k|, the scale's product and the difference to
        the reference 2^-23 of |s| + 24 (in powers of two); p moves by twice that;
      p as a pair: bf16 2^-8 of a rest of 2^-8, so 2^-16; f16 (hi truncated) 2^-11 of a rest of 2^-10, so 2^-21, and never less
        than half of its least step, 2^-25, where the sum of p is at least 2^6: 2^-31 of |v| a key;
      exp2 and the sums over keys in f32: 2^-21 + (n / 8 + 64) 2^-24 of A;
      out: half a step of its type."""
    d, g, u = s.dim, s.heads // s.kv_heads, HALF_STEP[s.kind]
    out, tol = np.zeros((s.rows, s.heads, d)), np.zeros((s.rows, s.heads, d))
    k, v = s.k.double().numpy(), s.v.double().numpy()
    for r in range(s.rows):
        i, t = s.visible(r)
        t = np.array(t)
        at = s.table[i, t // s.page].astype(np.int64) * s.page + t % s.page
        kk, vv = (x[at, :s.kv_heads * d].reshape(len(t), s.kv_heads, d) for x in (k, v))
        q = s.q[r].double().numpy().reshape(s.heads, d)
        for h in range(s.heads):
            kh, vh = kk[:, h // g], vv[:, h // g]
            sc = kh @ q[h] * SCALE
            p = np.exp(sc - sc.max())
            p /= p.sum()
            ds = d * 2.0 ** -24 * SCALE * (np.abs(kh) @ np.abs(q[h])).max() + 2.0 ** -23 * (np.abs(sc).max() + 24)
            pair = (p @ np.abs(vh)) * 2.0 ** -16 if s.kind == "bf16" else (p @ np.abs(vh)) * 2.0 ** -21 + 2.0 ** -31 * np.abs(vh).sum(0)
            out[r, h] = p @ vh
            tol[r, h] = (p @ np.abs(vh)) * (2 * ds + 2.0 ** -21 + (len(t) / 8 + 64) * 2.0 ** -24) + pair + u * np.abs(out[r, h]) + 1e-30
    return out, tol


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (4, 2, 128)])
@pytest.mark.parametrize("past,nodes", [(7, 1), (40, 1), (9, 12), (5, 24), (3, 64), (700, 1), (2500, 20), (1800, 64)])
def test_probabilities_keep_their_bits(kind, heads, kv, dim, past, nodes):
    """One row, 24, 48 and 128 query rows a kv head; short calls and long ones that are cut."""
    s = Step([(past, random_tree(np.random.default_rng(nodes), nodes))], kind=kind, heads=heads, kv_heads=kv, dim=dim, seed=past).fill()
    got = s.attend(SCALE).double().numpy().reshape(s.rows, heads, dim)
    want, tol = bound(s)
    off = np.abs(got - want)
    assert (off <= tol).all(), (int((off > tol).sum()), off.size, float((off / tol).max()))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_two_keys_of_unequal_weight(kind):
    """p = 1 and 1 / 3 over values 1 and -3: the products cancel, so that a rounded p would be all that is left."""
    s = Step([(1, [-1])], kind=kind, heads=2, kv_heads=1, dim=64).fill()
    a, b = s.slots(0)
    s.k[[a, b]] = 0
    s.q[:] = 1
    s.k[a, 0] = 1
    s.v[a], s.v[b] = 1, -3
    got = s.attend(float(np.float32(np.log(3.0)))).double().numpy()
    # the scale log 3 is off by 2^-24 of itself as f32; f32 steps of the scores, exp2 and sums: 2^-20 of A = 1.5
    assert np.abs(got).max() <= 1.5 * (2.0 ** -20 + (2.0 ** -16 if kind == "bf16" else 2.0 ** -21)), np.abs(got).max()
