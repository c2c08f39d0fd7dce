"""Norms, 8-bit products and log probabilities in calls at the ends of their ranges: logits far apart,
long rows cut over workgroups, every form of the product with weights past the caches and rows copied
or far apart, sums held to what contributes to them, and FP8 codes read by the products they are for."""
import numpy as np
import pytest

from attn_reference import U, from_type, to_type
from dense_reference import log_probs, norm
from oracle import oracle as orc
from test_gpu_dense import LOWEST, Rows, blank, check_log_probs, check_product, dense, given, hard_rows, run_norm  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,far", [("f32", 3e38), ("bf16", 3e38), ("f32", 1.9e38)])
@pytest.mark.parametrize("scale", [0.5, 0.001, 1e-37, 1.0])
@pytest.mark.parametrize("vocab", [100, 70000])
def test_log_probs_of_logits_whose_difference_is_past_a_float(backend, dense, t, far, scale, vocab):
    """Finite logits have a finite ln p wherever a float holds it, however far apart they are."""
    x = np.full((2, vocab), -far)
    x[0, 7] = far
    x[1, 1::2] = far
    check_log_probs(backend, dense, x, t, 5, np.array([[7, 0, 8]] * 2), scale)


@pytest.mark.parametrize("t,vocab", [("f32", 163841), ("f32", 262144), ("f32", 1000003), ("bf16", 700001)])
@pytest.mark.parametrize("n_top", [0, 20])
def test_log_probs_of_long_hard_rows(backend, dense, t, vocab, n_top):
    """Rows cut into as many parts as their join takes: masks, ties, NaN, the best in few places."""
    x = hard_rows(vocab, LOWEST[t])
    for rows in (range(7, 8), range(0, 4), range(4, 7), range(8, 12), range(12, 18)):
        check_log_probs(backend, dense, x[rows], t, n_top, given(np.random.default_rng(14), len(rows), vocab, 2))
