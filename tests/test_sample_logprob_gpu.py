"""navi_sample_rows' log probabilities at their upper end."""
import numpy as np
import pytest
import torch

from sample_util import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [1000, 16384, 20000, 151936])
def test_a_log_probability_is_not_above_0(vocab):
    """The only kept token's, whatever the roundings of its weight and of the sum: 0 to 2^-28, from below."""
    rng = np.random.default_rng(vocab)
    x = torch.from_numpy((rng.standard_normal((64, vocab)) * 3).astype(np.float32))
    rules = [[(0.8, 1, 1, 0, 1), (1.3, 0, 0.0, 0, 1), (0.7, 0, 1, 1.0, 1), (0.01, 0, 1, 0, 1)][i % 4] for i in range(64)]
    call = Call(x, rules, rng.random(64))
    call.check()
    lp = call.logprob.cpu()
    assert bool((lp <= 0).all()), lp.max()
    assert bool((lp[0::4] >= -2.0 ** -28).all()) and bool((lp[1::4] >= -2.0 ** -28).all())
