"""Norms, 8-bit products and log probabilities in calls at the ends of their ranges: logits far apart,
long rows cut over workgroups, every form of the product with weights past the caches and rows copied
or far apart, sums held to what contributes to them, and FP8 codes read by the products they are for."""
import numpy as np
import pytest

from attn_reference import U, from_type, to_type
from dense_bounds import sum_bounds
from dense_reference import log_probs, norm
from objeta_amd import QuantBackend
from objeta_amd.workloads import fp4_random_split, fp8_random_tiles
from oracle import oracle as orc
from test_gpu_dense import LOWEST, Rows, blank, check_log_probs, check_product, dense, given, hard_rows, run_norm  # noqa: F401
from test_gpu_official import assert_gemv_close

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


def check_sums(be, dense, x, t, scale=1.0, n_top=4):
    n, vocab = x.shape
    x = to_type(x, t)
    x64 = from_type(x, t)
    tokens = given(np.random.default_rng(3), n, vocab, 6)
    out = {k: blank(be, n, w, "f32") for k, w in dict(lse=1, entropy=1, lp=6, top=n_top).items()}
    ids = blank(be, n, n_top, None, dtype=np.int32)
    d_tokens = be.to_device(tokens.astype(np.int32))
    dense.log_probs_device(n, vocab, t, Rows(be, x, t).ptr, scale=scale, d_tokens=d_tokens, n_given=6, d_token_log_probs=out["lp"].ptr,
                           d_lse=out["lse"].ptr, d_entropy=out["entropy"].ptr, n_top=n_top, d_top_ids=ids.ptr, d_top_log_probs=out["top"].ptr)
    be.synchronize()
    got = {k: v.get().astype(np.float64) for k, v in out.items()}
    want = dict(zip(("lse", "entropy", "lp", "ids", "top"), log_probs(x64, scale, tokens, n_top)))
    assert np.array_equal(ids.get(), want["ids"])
    for r in range(n):
        b_lse, b_entropy, b_lp = sum_bounds(x64[r], scale)
        assert abs(got["lse"][r, 0] - want["lse"][r]) <= b_lse, (r, got["lse"][r, 0], want["lse"][r], b_lse)
        assert abs(got["entropy"][r, 0] - want["entropy"][r]) <= b_entropy, (r, got["entropy"][r, 0], want["entropy"][r], b_entropy)
        for k in ("lp", "top"):
            g, w = got[k][r], want[k][r]
            near = np.isfinite(w)
            assert np.array_equal(g[~near], w[~near])
            assert np.all(np.abs(g[near] - w[near]) <= b_lp(w[near])), (r, k, g, w, b_lp(w))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,vocab", [(1, 9), (3, 257), (5, 4097), (2, 50257), (300, 30000), (130, 60001), (1, 151936), (1, 262144)])
@pytest.mark.parametrize("spread,scale", [(3.0, 1.0), (0.05, 1.0), (6.0, 0.7)])
def test_log_probs_within_what_contributes(backend, dense, t, n, vocab, spread, scale):
    """Rows with a sure answer, with few and with all their tokens near one another."""
    x = np.random.default_rng(vocab).standard_normal((n, vocab), dtype=np.float32) * spread
    check_sums(backend, dense, x, t, scale)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [40, 3000, 33000, 100003])
def test_log_probs_of_masked_rows_within_what_contributes(backend, dense, t, vocab):
    """The rows of hard_rows that have a number for an answer; masked tokens do not widen the bounds."""
    x = hard_rows(vocab, LOWEST[t])
    good = [r for r in range(len(x)) if np.any(np.isfinite(x[r])) and not np.any(np.isnan(x[r]) | (x[r] == np.inf))]
    check_sums(backend, dense, x[good], t)


# ------------------------------------------------------------------------- product
@pytest.mark.parametrize("n,rows,cols", [(33, 33000, 1024), (5, 33000, 1024), (64, 14336, 4096), (64, 4096, 14336), (40, 7170, 8192),
                                         (5, 7168, 8192), (256, 8200, 4112)])
def test_product_of_weights_past_the_caches(backend, dense, n, rows, cols):
    """Every tile that asks the caches not to keep its weights, in matrices of 32 MiB and more."""
    check_product(backend, dense, n, rows, cols, "bf16" if n % 2 else "f32")


@pytest.mark.parametrize("n,rows,cols", [(1000, 7168, 4095), (2000, 7168, 33), (300, 14336, 1000)])
def test_product_of_copied_rows_on_the_large_tiles(backend, dense, n, rows, cols):
    check_product(backend, dense, n, rows, cols, "bf16")


@pytest.mark.parametrize("n,rows,a_pad,w_pad", [(20, 24, (1 << 22) - 48, 0), (40, 20, 0, (1 << 22) - 48), (18, 17, (1 << 22) - 47, (1 << 22) - 41)])
def test_product_of_rows_far_apart(backend, dense, n, rows, a_pad, w_pad):
    """Strides of 4 MiB are past what a tile's loads span: sixteen tokens at a time."""
    check_product(backend, dense, n, rows, 48, "f32", pads=(a_pad, w_pad, 0))


# ---------------------------------------------------------------------------- norm
@pytest.mark.parametrize("rt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hidden", [100, 4096])
def test_norm_keeps_rows_without_a_residual(backend, dense, rt, hidden):
    """d_residual_out alone: the rows rounded to its type, and it is these that are normed."""
    rng = np.random.default_rng(31)
    x, w = to_type(rng.standard_normal((5, hidden)), "f32"), to_type(np.ones((1, hidden)), "f32")
    dx, dw, dh, dy = Rows(backend, x, "f32"), Rows(backend, w, "f32"), blank(backend, 5, hidden, rt), blank(backend, 5, hidden, "f32")
    dense.rms_norm_device(5, hidden, "f32", dx.ptr, dw.ptr, eps=1e-6, d_residual_out=dh.ptr, residual_dtype=rt, d_out=dy.ptr)
    backend.synchronize()
    h = to_type(x, rt)
    assert np.array_equal(dh.get(), h)
    _, y = norm(from_type(h, rt), np.ones((1, hidden)), 1e-6)
    assert np.all(np.abs(dy.get() - y) <= np.abs(y) * U * 1.01 + 2.0 ** -150)


@pytest.mark.parametrize("n,hidden,rows", [(1, 1024, 384), (3, 7168, 300)])
@pytest.mark.parametrize("weights", ["fp4", "fp8"])
def test_fp8_codes_of_the_norm_through_the_official_product(backend, dense, n, hidden, rows, weights):
    """The norm's FP8 codes and scales as the activations of the official products, against the oracle's
    product of the oracle's codes."""
    quant = QuantBackend(backend)
    codes, scales = run_norm(backend, dense, hidden, n, "bf16", "f32", "f32", "fp8", kept=True, seed=41)
    y = blank(backend, n, rows, "f32")
    w, ws = (fp4_random_split if weights == "fp4" else fp8_random_tiles)(rows, hidden, 43)
    call, ref = ((quant.fp8_act_fp4_weight_gemv_device, orc.fp8_act_fp4_gemv) if weights == "fp4"
                 else (quant.fp8_act_fp8_weight_gemv_device, orc.fp8_act_fp8_gemv))
    call(None, codes.ptr, scales.ptr, backend.to_device(w), backend.to_device(ws), y.ptr, rows, hidden, n)
    backend.synchronize()
    q, s, got = codes.get(), scales.get(), y.get()
    for i in range(n):
        assert_gemv_close(got[i], ref(q[i], s[i], w, ws, rows, hidden))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hidden", [128, 2048, 20480])
def test_fp8_codes_of_rows_that_are_not_numbers(backend, dense, t, hidden):
    """Zeros over eps 0, infinities and NaN: the bytes that the activation quantizer gives the float norm."""
    x = np.random.default_rng(51).standard_normal((6, hidden))
    x[0] = 0
    x[1, hidden // 2] = np.inf
    x[2, 3] = np.nan
    x[3, 100] = -np.inf
    x[4] = np.inf
    dx, dw = Rows(backend, to_type(x, t), t), Rows(backend, to_type(np.ones((1, hidden)), t), t)
    dy = blank(backend, 6, hidden, "f32")
    out = [(blank(backend, 6, hidden, None, dtype=np.uint8), blank(backend, 6, hidden // 128, None, dtype=np.uint8)) for _ in range(2)]
    dense.rms_norm_device(6, hidden, t, dx.ptr, dw.ptr, eps=0.0, d_out=dy.ptr, out_dtype="f32", codes="fp8", d_codes=out[0][0].ptr,
                          d_scales=out[0][1].ptr)
    QuantBackend(backend).act_quant_device(None, dy.ptr, 6, hidden, out[1][0].ptr, out[1][1].ptr)
    backend.synchronize()
    assert np.isnan(dy.get()[0]).all()
    assert np.array_equal(out[0][0].get(), out[1][0].get()) and np.array_equal(out[0][1].get(), out[1][1].get())
