"""The bounds of dense_bounds are narrow enough to tell a sum that leaves something out."""
import numpy as np

from dense_bounds import sum_bounds
from dense_reference import log_probs

LOWEST = -3.4028235e38


def test_the_bounds_tell_what_is_left_out():
    """A tail that is dropped, or counted twice, lies outside of them."""
    x = np.random.default_rng(1).standard_normal(50257) * 3
    x[np.random.default_rng(2).random(x.size) < 0.2] = LOWEST
    (lse,), (entropy,), _, _, _ = log_probs(x[None], 1.0)
    b_lse, b_entropy, _ = sum_bounds(x, 1.0)
    assert b_lse < 3e-5 and b_entropy < 2e-4
    for cut in (x.max() - 8, np.sort(x)[-500]):
        part = np.where(x < cut, -np.inf, x)
        (lse2,), (entropy2,), _, _, _ = log_probs(part[None], 1.0)
        assert abs(lse2 - lse) > b_lse and abs(entropy2 - entropy) > b_entropy
