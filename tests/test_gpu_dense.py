"""Norms with 8-bit output, rows to int8, products in 8-bit integers and log probabilities against
the plain 64-bit forms of dense_reference, within the bounds derived there. Codes, whole sums and
the order of the best are held to equality."""
import numpy as np
import pytest

from attn_reference import HALF_STEP, NP, from_type, to_type
from dense_reference import TINY, log_prob_bounds, log_probs, norm, norm_bound, product, rows_i8
from objeta_amd import DenseBackend, MoeExecutor, QuantBackend

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


@pytest.fixture
def dense(backend):
    MoeExecutor(backend).device_error()
    yield DenseBackend(backend)
    assert MoeExecutor(backend).device_error() == 0


class Rows:
    """Device rows of `t` that begin `skew` elements behind an aligned address, `stride` apart, with
    a filling between and behind them that nothing may change."""

    def __init__(self, be, x, t, stride=None, skew=0, dtype=None):
        self.n, self.width = x.shape
        self.stride, self.skew = stride or self.width, skew
        self.kind = dtype or NP[t]
        self.host = np.full(skew + self.n * self.stride + 8, 77).astype(self.kind)
        self.view(self.host)[:, :self.width] = x
        self.buf = be.to_device(self.host)
        self.ptr = self.buf.ptr + skew * np.dtype(self.kind).itemsize

    def view(self, a):
        return a[self.skew:self.skew + self.n * self.stride].reshape(self.n, self.stride)

    def get(self):
        """The rows; what lies around them is as it was."""
        a = self.buf.download(self.kind, self.host.size)
        rows = self.view(a)[:, :self.width].copy()
        self.view(a)[:, :self.width] = self.view(self.host)[:, :self.width]
        assert np.array_equal(a, self.host), "elements around the rows were written"
        return rows


def blank(be, n, width, t, stride=None, skew=0, dtype=None):
    return Rows(be, np.full((n, width), 33, dtype or NP[t]), t, stride, skew, dtype)


# ------------------------------------------------------------------------- norm
def run_norm(be, dense, hidden, n, t, rt=None, ot=None, codes=None, kept=False, skew=0, pad=0, eps=1e-6, offset=0.0, seed=0, x=None,
             r=None, wt=None, stream=None):
    rng = np.random.default_rng(seed + hidden)
    wt = wt or t
    x = to_type(rng.standard_normal((n, hidden)) * 3 if x is None else x, t)
    w = to_type(1 + 0.3 * rng.standard_normal((1, hidden)), wt)
    r = None if rt is None else to_type(rng.standard_normal((n, hidden)) * 5 if r is None else r, rt)
    s = hidden + pad
    dx, dw = Rows(be, x, t, s, skew), Rows(be, w, wt, skew=skew)
    dr = None if rt is None else Rows(be, r, rt, s, skew)
    dh = blank(be, n, hidden, rt, s, skew) if kept else None
    dy = None if ot is None else blank(be, n, hidden, ot, s, skew)
    dq = ds = None
    if codes:
        dq = blank(be, n, hidden, None, s, skew, np.int8 if codes == "i8" else np.uint8)
        ds = blank(be, n, 1, "f32") if codes == "i8" else blank(be, n, hidden // 128, None, dtype=np.uint8)
    dense.rms_norm_device(n, hidden, t, dx.ptr, dw.ptr, eps=eps, weight_dtype=wt, weight_offset=offset, d_residual=dr and dr.ptr,
                          d_residual_out=dh and dh.ptr, residual_dtype=rt, d_out=dy and dy.ptr, out_dtype=ot, codes=codes,
                          d_codes=dq and dq.ptr, d_scales=ds and ds.ptr, x_stride=s, residual_stride=s, residual_out_stride=s,
                          out_stride=s, codes_stride=s, stream=stream)
    be.synchronize(stream)
    h, y = norm(from_type(x, t), from_type(w, wt), eps, None if r is None else from_type(r, rt), rt, kept, offset)
    if kept:
        assert np.array_equal(from_type(dh.get(), rt), h, equal_nan=True)
    if ot:
        got = from_type(dy.get(), ot)
        finite = np.isfinite(y)
        assert np.array_equal(np.isnan(got), np.isnan(y))
        assert np.all((np.abs(got - y) <= norm_bound(y, ot))[finite])
    with np.errstate(over="ignore"):
        y32 = y.astype(np.float32)
    if codes == "i8":
        want_q, want_s = rows_i8(y32)
        assert np.array_equal(ds.get()[:, 0], want_s, equal_nan=True)
        assert np.array_equal(dq.get(), want_q)
    if codes == "fp8":
        values, scales = QuantBackend(be).act_quant(None, y32, n, hidden)
        assert np.array_equal(dq.get().ravel(), values) and np.array_equal(ds.get().ravel(), scales)
    return dq, ds


@pytest.mark.parametrize("hidden", [1, 7, 8, 9, 63, 64, 511, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 4096, 4100, 8191, 8192, 8193,
                                    16384, 16385, 32767, 32768])
@pytest.mark.parametrize("n", [1, 5])
def test_norm_widths(backend, dense, hidden, n):
    run_norm(backend, dense, hidden, n, "bf16", "f32", "f32", "i8", kept=True)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rt,kept", [(None, False), ("f32", False), ("f32", True), ("f16", True), ("bf16", True), ("bf16", False)])
@pytest.mark.parametrize("ot,codes", [(None, "i8"), ("f32", None), ("bf16", "i8"), ("f16", "fp8"), (None, "fp8")])
def test_norm_types(backend, dense, t, rt, kept, ot, codes):
    run_norm(backend, dense, 1280, 6, t, rt, ot, codes, kept=kept)


@pytest.mark.parametrize("hidden", [256, 777, 2048, 5000])
@pytest.mark.parametrize("skew,pad", [(0, 3), (1, 0), (3, 5), (8, 8), (5, 1)])
@pytest.mark.parametrize("t", ["f32", "f16"])
def test_norm_rows_anywhere(backend, dense, hidden, skew, pad, t):
    run_norm(backend, dense, hidden, 9, t, t, t, "i8", kept=True, skew=skew, pad=pad)


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("eps", [1e-5, 0.0, 3.0])
def test_norm_weights_and_eps(backend, dense, wt, offset, eps):
    run_norm(backend, dense, 640, 3, "bf16", None, "f32", "i8", wt=wt, offset=offset, eps=eps)


@pytest.mark.parametrize("hidden", [128, 1024, 4096, 20480])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_norm_odd_values(backend, dense, hidden, eps):
    """Rows of zeros, of one value, of tiny and of huge ones, and with an infinity or NaN."""
    x = np.random.default_rng(4).standard_normal((8, hidden))
    x[0] = 0
    x[1] = 0
    x[1, -1] = 1
    x[2] *= 1e-38
    x[3] *= 1e37
    x[4, 5] = np.inf
    x[5, hidden // 2] = np.nan
    x[6] = -3.25
    run_norm(backend, dense, hidden, 8, "f32", None, "f32", "i8", x=x, eps=eps)
    if eps:  # (a block's codes of what a row of zeros over eps 0 gives are NaN's)
        run_norm(backend, dense, hidden, 8, "f32", None, "f32", "fp8", x=x, eps=eps)


def test_norm_sums_that_overflow_a_half(backend, dense):
    """The residual stream in f16 goes to infinity where its sum does."""
    x = np.full((2, 512), 60000.0)
    run_norm(backend, dense, 512, 2, "f16", "f16", "f32", "i8", kept=True, x=x, r=x)
    run_norm(backend, dense, 512, 2, "f16", "f16", "f32", "i8", kept=False, x=x, r=x)


@pytest.mark.parametrize("n,hidden", [(3001, 96), (70001, 64), (1030, 3200)])
def test_norm_many_tokens_on_another_stream(backend, dense, n, hidden):
    run_norm(backend, dense, hidden, n, "bf16", "bf16", "bf16", None, kept=True, stream=backend.stream(1))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hidden", [100, 1536, 9000])
def test_norm_in_place(backend, dense, t, hidden):
    """The sum where the residual was, the norm where x was."""
    rng = np.random.default_rng(5)
    x, r = (to_type(rng.standard_normal((7, hidden)), t) for _ in range(2))
    w = to_type(np.ones((1, hidden)), t)
    dx, dr, dw = Rows(backend, x, t, hidden + 3), Rows(backend, r, t), Rows(backend, w, t)
    dense.rms_norm_device(7, hidden, t, dx.ptr, dw.ptr, eps=1e-6, d_residual=dr.ptr, d_residual_out=dr.ptr, d_out=dx.ptr,
                          x_stride=hidden + 3, out_stride=hidden + 3)
    backend.synchronize()
    h, y = norm(from_type(x, t), from_type(w, t), 1e-6, from_type(r, t), t, True)
    assert np.array_equal(from_type(dr.get(), t), h)
    assert np.all(np.abs(from_type(dx.get(), t) - y) <= norm_bound(y, t))


@pytest.mark.parametrize("hidden", [384, 2048, 7168])
def test_fused_codes_are_those_of_the_float_norm(backend, dense, hidden):
    """Norm, then the quantizer over its float output: the same bytes as in one call."""
    rng = np.random.default_rng(6)
    x, w = rng.standard_normal((33, hidden)).astype(np.float32), np.ones((1, hidden), np.float32)
    dx, dw, dy = Rows(backend, x, "f32"), Rows(backend, w, "f32"), blank(backend, 33, hidden, "f32")
    out = [(blank(backend, 33, hidden, None, dtype=np.int8), blank(backend, 33, 1, "f32")) for _ in range(2)]
    dense.rms_norm_device(33, hidden, "f32", dx.ptr, dw.ptr, d_out=dy.ptr, codes="i8", d_codes=out[0][0].ptr, d_scales=out[0][1].ptr)
    dense.quantize_rows_device(33, hidden, "f32", dy.ptr, out[1][0].ptr, out[1][1].ptr)
    backend.synchronize()
    assert np.array_equal(out[0][0].get(), out[1][0].get()) and np.array_equal(out[0][1].get(), out[1][1].get())


# --------------------------------------------------------------------- quantizer
def check_quantize(be, dense, x, t, skew=0, pad=0):
    n, cols = x.shape
    x = to_type(x, t)
    dx = Rows(be, x, t, cols + pad, skew)
    dq, ds = blank(be, n, cols, None, cols + pad, skew, np.int8), blank(be, n, 1, "f32")
    dense.quantize_rows_device(n, cols, t, dx.ptr, dq.ptr, ds.ptr, x_stride=cols + pad, codes_stride=cols + pad)
    be.synchronize()
    q, s = rows_i8(from_type(x, t))
    assert np.array_equal(ds.get()[:, 0], s, equal_nan=True)
    assert np.array_equal(dq.get(), q)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", [1, 3, 16, 100, 512, 520, 1024, 3000, 4096, 11008, 30000, 65536])
def test_quantize_rows(backend, dense, t, cols):
    check_quantize(backend, dense, np.random.default_rng(cols).standard_normal((6, cols)) * 0.02, t)


@pytest.mark.parametrize("skew,pad", [(1, 0), (3, 1), (2, 7)])
@pytest.mark.parametrize("cols", [33, 600, 4097])
def test_quantize_rows_anywhere(backend, dense, skew, pad, cols):
    check_quantize(backend, dense, np.random.default_rng(cols).standard_normal((11, cols)), "bf16", skew, pad)


@pytest.mark.parametrize("cols", [256, 2000, 16000])
def test_quantize_halves(backend, dense, cols):
    """Quotients that are halves exactly or off them by a float's last step, of scales that are
    powers of two and not."""
    rng, rows = np.random.default_rng(7), []
    for s in (1.0, 0.25, 3.0, 0.1, 7.77e-3, 1e30, 3e-37):
        s = np.float64(np.float32(s))
        x = (rng.integers(-126, 126, cols) + 0.5) * s
        x[0] = 127 * s
        x = x.astype(np.float32)
        rows += [x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf))]
    check_quantize(backend, dense, np.array(rows), "f32")


@pytest.mark.parametrize("cols", [64, 1000, 9001])
def test_quantize_tiny_and_odd_rows(backend, dense, cols):
    """Subnormal rows and scales, zeros, infinities and NaN, the largest floats."""
    x = np.random.default_rng(8).standard_normal((10, cols)).astype(np.float32)
    for i, f in enumerate((1e-37, 1e-39, 1e-42, 5e-44, 1.4e-45)):
        x[i] *= np.float32(f) if f > 1e-38 else 1
        if f <= 1e-38:
            x[i] = (x[i].astype(np.float64) * f).astype(np.float32)
    x[5] = 0
    x[6, cols // 3] = np.inf
    x[7, cols // 2] = np.nan
    x[8] = np.float32(3.4028235e38)
    x[9, 0] = -3.4028235e38
    check_quantize(backend, dense, x, "f32")


def test_quantize_many_rows(backend, dense):
    check_quantize(backend, dense, np.random.default_rng(9).standard_normal((9001, 72)), "f16")


@pytest.mark.parametrize("t,n,cols,pad,skew", [("f32", 4100, 4096, 0, 0), ("f16", 33000, 1025, 3, 1), ("bf16", 280000, 120, 0, 0),
                                               ("f32", 1025, 16384, 4, 0)])
def test_quantize_large_matrices(backend, dense, t, n, cols, pad, skew):
    x = np.random.default_rng(cols).standard_normal((n, cols), dtype=np.float32)
    check_quantize(backend, dense, x, t, pad=pad, skew=skew)


# ----------------------------------------------------------------------- product
def check_product(be, dense, n, rows, cols, ot="f32", bias=True, skews=(0, 0, 0), pads=(0, 0, 0), extreme=False, seed=0, stream=None):
    rng = np.random.default_rng(seed + 31 * n + rows + cols)
    a, w = (rng.integers(-128, 128, (m, cols)).astype(np.int8) for m in (n, rows))
    if extreme:
        a[:], w[:] = -128, -128
        w[::2] = 127
    sa, sw = (np.exp(rng.standard_normal(m)).astype(np.float32) * np.float32(f) for m, f in ((n, 0.02), (rows, 0.001)))
    b = rng.standard_normal(rows).astype(np.float32) if bias else None
    da, dw = Rows(be, a, None, cols + pads[0], skews[0], np.int8), Rows(be, w, None, cols + pads[1], skews[1], np.int8)
    dsa, dsw = Rows(be, sa[None], "f32"), Rows(be, sw[None], "f32")
    db = Rows(be, b[None], "f32") if bias else None
    out = blank(be, n, rows, ot, rows + pads[2], skews[2])
    dense.i8_product_device(n, rows, cols, da.ptr, dsa.ptr, dw.ptr, dsw.ptr, out.ptr, out_dtype=ot, d_bias=db and db.ptr,
                            a_stride=cols + pads[0], w_stride=cols + pads[1], out_stride=rows + pads[2], stream=stream)
    be.synchronize(stream)
    want = product(a, sa, w, sw, b)
    assert np.array_equal(out.get(), to_type(want, ot))


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 31, 33, 47, 64, 65, 100, 129, 200, 257, 300])
@pytest.mark.parametrize("rows,cols", [(16, 64), (1, 1), (7, 15), (100, 1000), (512, 2048), (300, 129), (1023, 4096)])
def test_product_sizes(backend, dense, n, rows, cols):
    check_product(backend, dense, n, rows, cols, ["f32", "f16", "bf16"][(n + rows) % 3], bias=n % 2 == 0)


@pytest.mark.parametrize("n", [1, 20, 70, 260])
@pytest.mark.parametrize("skews,pads", [((1, 0, 0), (0, 0, 0)), ((0, 3, 1), (0, 0, 0)), ((16, 16, 4), (16, 48, 4)), ((5, 7, 3), (1, 1, 1)),
                                        ((0, 0, 0), (13, 0, 0)), ((0, 0, 0), (0, 13, 0)), ((0, 0, 0), (0, 0, 5)), ((4, 8, 2), (4, 8, 2))])
@pytest.mark.parametrize("ot", TYPES)
def test_product_rows_anywhere(backend, dense, n, skews, pads, ot):
    check_product(backend, dense, n, 330, 528, ot, skews=skews, pads=pads)


@pytest.mark.parametrize("n,rows", [(1, 3), (17, 20), (300, 260)])
def test_product_of_the_largest_codes_and_columns(backend, dense, n, rows):
    check_product(backend, dense, n, rows, 131071, bias=False, extreme=True)


@pytest.mark.parametrize("n,rows,cols", [(1, 20000, 256), (33, 5000, 768), (520, 3000, 512), (1025, 1030, 1536), (4100, 96, 64), (700, 9000, 128)])
def test_product_of_many_rows_on_another_stream(backend, dense, n, rows, cols):
    check_product(backend, dense, n, rows, cols, "bf16", stream=backend.stream(1))


@pytest.mark.parametrize("n,rows,cols", [(5, 9000, 4096), (16, 7168, 64), (4, 7200, 80), (12, 8000, 33), (100, 9000, 4096), (32, 9000, 2048), (20, 9000, 4095),
                                         (100, 9000, 1001), (100, 20000, 4096), (600, 9000, 33), (1500, 9000, 512),
                                         (1000, 4097, 4096), (600, 7200, 4700)])
def test_product_of_every_tile(backend, dense, n, rows, cols):
    check_product(backend, dense, n, rows, cols, "bf16" if n % 3 else "f32", pads=(0, 0, n % 2 * 5))


@pytest.mark.parametrize("cols", [15, 16, 17, 35, 130])
@pytest.mark.parametrize("skews,pads", [((0, 0, 0), (0, 0, 0)), ((3, 0, 0), (1, 0, 0)), ((0, 2, 1), (13, 30, 1))])
def test_product_of_many_rows_that_begin_anywhere(backend, dense, cols, skews, pads):
    """Past some size such rows are copied to whole chunks first."""
    check_product(backend, dense, 1700, 1650, cols, "f32", skews=skews, pads=pads)


@pytest.mark.parametrize("n,rows,cols", [(1700, 1650, 37), (1700, 1650, 48), (5, 40, 130)])
def test_product_captured_without_a_call_ahead(n, rows, cols):
    """On a stream of its own that has no workspace: such rows are then read where they lie."""
    import ctypes as C
    from objeta_amd import HipBackend
    from objeta_amd.api import check as ok
    with HipBackend(0, 1) as be:
        rng = np.random.default_rng(21)
        a, w = (rng.integers(-128, 128, (m, cols)).astype(np.int8) for m in (n, rows))
        sa, sw = (np.exp(rng.standard_normal(m)).astype(np.float32) for m in (n, rows))
        d = [be.to_device(x) for x in (a, sa, w, sw)]
        out = be.alloc(4 * n * rows)
        st, g = be.stream(0), C.c_void_p()
        ok(be.L.objeta_hip_graph_begin_capture(be.ctx, st))
        DenseBackend(be).i8_product_device(n, rows, cols, d[0], d[1], d[2], d[3], out)
        ok(be.L.objeta_hip_graph_end_capture(be.ctx, st, C.byref(g)))
        want = product(a, sa, w, sw)
        for _ in range(3):
            ok(be.L.objeta_hip_zero_device(be.ctx, st, out.addr(), out.nbytes))
            ok(be.L.objeta_hip_graph_launch(be.ctx, g, st))
            be.synchronize()
            assert np.array_equal(out.download(np.float32, n * rows).reshape(n, rows), want)
        DenseBackend(be).i8_product_device(n, rows, cols, d[0], d[1], d[2], d[3], out)
        be.synchronize()
        assert np.array_equal(out.download(np.float32, n * rows).reshape(n, rows), want)
        ok(be.L.objeta_hip_graph_destroy(be.ctx, g))
        del d, out


def test_product_results_do_not_depend_on_the_batch(backend, dense):
    """A token's row is the same bits alone and in batches of any size."""
    rng, rows, cols = np.random.default_rng(11), 200, 640
    a, w = (rng.integers(-127, 128, (m, cols)).astype(np.int8) for m in (600, rows))
    sa, sw = (np.exp(rng.standard_normal(m)).astype(np.float32) for m in (600, rows))
    da, dw, dsa, dsw = (backend.to_device(x) for x in (a, w, sa, sw))
    want = None
    for n in (600, 300, 65, 17, 5, 1):
        out = blank(backend, n, rows, "f32")
        dense.i8_product_device(n, rows, cols, da, dsa, dw, dsw, out.ptr)
        backend.synchronize()
        want = out.get() if want is None else want
        assert np.array_equal(out.get(), want[:n])


# -------------------------------------------------------------- log probabilities
def check_log_probs(be, dense, x, t, n_top=0, tokens=None, scale=1.0, pad=0, skew=0, entropy=True, lse=True, stream=None):
    n, vocab = x.shape
    x = to_type(x, t)
    dx = Rows(be, x, t, vocab + pad, skew)
    if pad:  # what lies behind the vocabulary would win
        host = dx.view(dx.host)
        host[:, vocab:] = to_type(np.full(pad, 3e4), t)
        dx.buf.upload(dx.host)
    dl, de = (blank(be, n, 1, "f32") if f else None for f in (lse, entropy))
    dp = None if tokens is None else blank(be, *tokens.shape, "f32")
    di, dt = (blank(be, n, n_top, None, dtype=k) if n_top else None for k in (np.int32, np.float32))
    dense.log_probs_device(n, vocab, t, dx.ptr, scale=scale, d_tokens=None if tokens is None else be.to_device(tokens.astype(np.int32)),
                           n_given=0 if tokens is None else tokens.shape[1], d_token_log_probs=dp and dp.ptr, d_lse=dl and dl.ptr,
                           d_entropy=de and de.ptr, n_top=n_top, d_top_ids=di and di.ptr, d_top_log_probs=dt and dt.ptr,
                           stride=vocab + pad, stream=stream)
    be.synchronize(stream)
    x64 = from_type(x, t)
    want = log_probs(x64, scale, tokens, n_top)

    def near(got, want, which):
        for r in range(n):
            g, w = got[r].astype(np.float64).ravel(), np.asarray(want[r], np.float64).ravel()
            with np.errstate(over="ignore"):
                w = np.where(np.isfinite(w.astype(np.float32)), w, w.astype(np.float32))  # past a float's range
            same = np.isfinite(w)
            assert np.array_equal(g[~same], w[~same], equal_nan=True), (r, g, w)
            bound = np.broadcast_to(log_prob_bounds(x64[r], scale, want_lse[r], want_h[r], np.where(same, w, 0))[which], w.shape)
            assert np.all(np.abs(g[same] - w[same]) <= bound[same] + TINY["f32"]), (r, g, w, bound)
    want_lse, want_h = want[0], np.nan_to_num(want[1])
    if lse:
        near(dl.get(), want[0], 0)
    if entropy:
        near(de.get(), want[1], 1)
    if tokens is not None:
        near(dp.get(), want[2], 2)
    if n_top:
        assert np.array_equal(di.get(), want[3])
        near(dt.get(), want[4], 2)


def given(rng, n, vocab, k):
    t = rng.integers(0, vocab, (n, k))
    t[rng.random((n, k)) < 0.1] = -1
    return t


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 255, 1000, 4096, 8191, 8193, 16385, 50257])
@pytest.mark.parametrize("n", [1, 3])
def test_log_probs_sizes(backend, dense, t, vocab, n):
    rng = np.random.default_rng(vocab + n)
    check_log_probs(backend, dense, rng.standard_normal((n, vocab)) * 3, t, min(vocab, 20), given(rng, n, vocab, 3))


@pytest.mark.parametrize("n_top", [0, 1, 2, 5, 31, 32])
@pytest.mark.parametrize("n,vocab", [(1, 151936), (7, 40000), (1100, 3000), (2, 262144)])
def test_log_probs_of_the_best(backend, dense, n_top, n, vocab):
    rng = np.random.default_rng(n_top)
    check_log_probs(backend, dense, rng.standard_normal((n, vocab)) * 2.5, "bf16" if n > 1 else "f32", n_top, given(rng, n, vocab, 1),
                    entropy=n_top != 5, lse=n_top != 2)


@pytest.mark.parametrize("t,n,vocab,n_top", [("f32", 130, 130001, 3), ("f32", 300, 60000, 7), ("f16", 1300, 26003, 0), ("bf16", 1100, 31000, 5)])
def test_log_probs_of_large_batches(backend, dense, t, n, vocab, n_top):
    check_log_probs(backend, dense, np.random.default_rng(n).standard_normal((n, vocab), dtype=np.float32) * 3, t, n_top=n_top)


@pytest.mark.parametrize("scale", [0.01, 0.7, 5.0])
@pytest.mark.parametrize("pad,skew", [(0, 0), (1, 1), (3, 0), (8, 5)])
@pytest.mark.parametrize("t", TYPES)
def test_log_probs_rows_anywhere(backend, dense, scale, pad, skew, t):
    rng = np.random.default_rng(12)
    check_log_probs(backend, dense, rng.standard_normal((5, 10001)) * 4, t, 7, given(rng, 5, 10001, 4), scale, pad, skew,
                    stream=backend.stream(1))


def hard_rows(vocab, lowest):
    """Rows whose masks leave little or nothing, ties, and values that meet in few places."""
    rng = np.random.default_rng(13)
    x = rng.standard_normal((18, vocab)) * 2
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, vocab // 3] = 1.5
    x[2, rng.random(vocab) < 0.999] = -np.inf
    x[3] = lowest  # a mask of the type's lowest value that leaves nothing
    x[4, rng.random(vocab) < 0.999] = lowest
    x[5] = 0.25  # all alike
    x[6] = np.round(x[6])  # many ties
    x[7] = np.sort(x[7])
    x[8] = np.sort(x[8])[::-1]
    x[9, ::1024] += 50  # the best in a few threads' stretches
    x[10, :vocab // 5] += 40
    x[11, vocab // 2] = 60.0  # a sure answer
    x[12] *= 0
    x[12, 1::2] = -0.0  # zeros of both signs are alike
    x[13, 5] = np.nan
    x[14, vocab // 7] = np.inf
    x[15] = np.nan
    x[16] = -np.inf
    x[16, vocab - 1] = np.nan
    x[17, 8:16] = 30.0  # ties within a thread's load
    return x


LOWEST = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("vocab", [40, 3000, 33000, 100003])
@pytest.mark.parametrize("n_top", [0, 3, 32])
def test_log_probs_of_hard_rows(backend, dense, t, vocab, n_top):
    """Every row alone, cut over workgroups, and all at once, one workgroup each."""
    x = hard_rows(vocab, LOWEST[t])
    tokens = given(np.random.default_rng(14), len(x), vocab, 2)
    tokens[1, 0], tokens[11, 0] = vocab // 3, vocab // 2
    check_log_probs(backend, dense, x, t, n_top, tokens)
    if vocab != 40:
        many = np.concatenate([x] * 57)[:1024]  # one workgroup a row
        check_log_probs(backend, dense, many[-36:] if vocab > 3000 else many, t, n_top, None)


@pytest.mark.parametrize("value", [1e30, -1e30, 3e38, -3e38, 1e33, -2.0 ** 100, 1e-30])
@pytest.mark.parametrize("scale", [1.0, 0.001, 100.0])
def test_log_probs_of_huge_logits(backend, dense, value, scale):
    """All around one huge value, equal to it or a little off: the exponents' references leave the range."""
    x = np.full((3, 5000), np.float32(value), np.float64)
    x[1, 7] = np.float32(value * 1.0000005)
    x[2, 100:] = 1.0
    check_log_probs(backend, dense, x, "f32", 5, np.array([[7, 99]] * 3), scale)


@pytest.mark.parametrize("vocab", [100, 30000])
def test_log_probs_of_tokens_outside(backend, vocab):
    """Such tokens are NaN and set bit 2; -1 asks for none."""
    err = MoeExecutor(backend)
    err.device_error()
    d = DenseBackend(backend)
    x = np.zeros((2, vocab), np.float32)
    out = blank(backend, 2, 4, "f32")
    d.log_probs_device(2, vocab, "f32", backend.to_device(x), d_tokens=backend.to_device(np.array([[vocab, 0, -1, -2], [1, -1, 2, 2 ** 31 - 1]], np.int32)),
                       n_given=4, d_token_log_probs=out.ptr)
    backend.synchronize()
    got = out.get()
    assert err.device_error() == 4
    assert np.array_equal(np.isnan(got), [[True, False, False, True], [False, False, False, True]])
    assert got[0, 2] == 0 and got[1, 1] == 0 and np.allclose(got[[0, 1, 1], [1, 0, 2]], -np.log(vocab), rtol=1e-5)


# ------------------------------------------------------------- a run of them together
def scoring(be, dense, t, seed, n, hidden, vocab):
    """Norm with the residual, the answer head over its codes, and what is read off the logits."""
    rng = np.random.default_rng(seed)
    x, r = to_type(rng.standard_normal((n, hidden)), t), rng.standard_normal((n, hidden)).astype(np.float32) * 2
    w = to_type(1 + 0.1 * rng.standard_normal(hidden), t)
    head = rng.standard_normal((vocab, hidden)).astype(np.float32) * np.float32(2 * hidden ** -0.5)
    tokens = rng.integers(0, vocab, (n, 1)).astype(np.int32)
    d = {k: be.to_device(v) for k, v in dict(x=x, r=r, w=w, head=head, tokens=tokens).items()}
    for k, size in dict(h=4 * n * hidden, q=n * hidden, s=4 * n, hq=vocab * hidden, hs=4 * vocab, logits=4 * n * vocab, lp=4 * n, lse=4 * n,
                        entropy=4 * n, ids=4 * n * 5, top=4 * n * 5).items():
        d[k] = be.alloc(size)
    dense.quantize_rows_device(vocab, hidden, "f32", d["head"], d["hq"], d["hs"])

    def step(stream=None):
        dense.rms_norm_device(n, hidden, t, d["x"], d["w"], d_residual=d["r"], d_residual_out=d["h"], residual_dtype="f32", codes="i8",
                              d_codes=d["q"], d_scales=d["s"], stream=stream)
        dense.i8_product_device(n, vocab, hidden, d["q"], d["s"], d["hq"], d["hs"], d["logits"], stream=stream)
        dense.log_probs_device(n, vocab, "f32", d["logits"], d_tokens=d["tokens"], n_given=1, d_token_log_probs=d["lp"], d_lse=d["lse"],
                               d_entropy=d["entropy"], n_top=5, d_top_ids=d["ids"], d_top_log_probs=d["top"], stream=stream)

    def check():
        _, y = norm(from_type(x, t), from_type(w, t), 1e-6, r.astype(np.float64), "f32", True)
        q, s = rows_i8(y)
        hq, hs = rows_i8(head)
        logits = product(q, s, hq, hs)
        assert np.array_equal(d["logits"].download(np.float32, n * vocab).reshape(n, vocab), logits)
        want = log_probs(logits.astype(np.float64), 1.0, tokens, 5)
        assert np.array_equal(d["ids"].download(np.int32, 5 * n).reshape(n, 5), want[3])
        for i in range(n):
            b = log_prob_bounds(logits[i], 1.0, want[0][i], want[1][i], want[2][i])
            assert abs(d["lse"].download(np.float32, n)[i] - want[0][i]) <= b[0]
            assert abs(d["entropy"].download(np.float32, n)[i] - want[1][i]) <= b[1]
            assert np.all(np.abs(d["lp"].download(np.float32, n)[i] - want[2][i]) <= b[2])
        # what eight bits cost the answers: codes are off by half a step at most
        half = 0.5 * (np.abs(y).max(-1) / 127)[:, None] * np.abs(head).sum(-1) + 0.5 * (np.abs(head).max(-1) / 127) * np.abs(y).sum(-1)[:, None]
        rest = 0.25 * hidden * (np.abs(y).max(-1) / 127)[:, None] * (np.abs(head).max(-1) / 127)
        assert np.all(np.abs(logits - y @ head.astype(np.float64).T) <= (half + rest) * 1.001)
    return step, check, d


@pytest.mark.parametrize("t,n,hidden,vocab", [("bf16", 1, 512, 4001), ("f16", 6, 384, 2000), ("f32", 90, 200, 1111)])
def test_scoring_chain(backend, dense, t, n, hidden, vocab):
    step, check, _ = scoring(backend, dense, t, 15, n, hidden, vocab)
    step()
    backend.synchronize()
    check()


@pytest.mark.parametrize("n,vocab", [(1, 50000), (40, 3000)])
def test_scoring_chain_captured(backend, dense, n, vocab):
    """Replayed with eager calls and other work between, every replay checked."""
    st = backend.stream(1)
    step, check, d = scoring(backend, dense, "bf16", 16, n, 256, vocab)
    backend.synchronize()
    step(st)
    backend.synchronize(st)
    import ctypes as C
    from objeta_amd.api import check as ok
    L, ctx = backend.L, backend.ctx
    g = C.c_void_p()
    ok(L.objeta_hip_graph_begin_capture(ctx, st))
    step(st)
    ok(L.objeta_hip_graph_end_capture(ctx, st, C.byref(g)))
    try:
        for _ in range(4):
            for k in ("logits", "ids", "lp", "lse", "entropy", "q"):
                ok(L.objeta_hip_zero_device(ctx, st, d[k].addr(), d[k].nbytes))
            other = scoring(backend, dense, "f32", 17, 3, 128, 500)
            other[0](st)
            ok(L.objeta_hip_graph_launch(ctx, g, st))
            backend.synchronize(st)
            check()
            other[1]()
    finally:
        ok(L.objeta_hip_graph_destroy(ctx, g))


def test_two_streams_at_once(backend, dense):
    a, b = scoring(backend, dense, "bf16", 18, 2, 256, 40000), scoring(backend, dense, "f32", 19, 1, 128, 60000)
    backend.synchronize()
    for _ in range(20):
        a[0](backend.stream(0))
        b[0](backend.stream(1))
    backend.synchronize(backend.stream(0))
    backend.synchronize(backend.stream(1))
    a[1]()
    b[1]()
