"""Norms with 8-bit output, rows quantized to 8 bits, products in 8-bit integers and log
probabilities over the C ABI: what a decoder layer runs between its attention and its experts,
and what is read off its answers. The reference has none of these on its device path.

Arguments named d_* are device addresses (DeviceBuffer, int or c_void_p); element types are
"f32", "f16" or "bf16"; strides count elements from row to row and default to dense rows. Calls
are asynchronous on `stream` (None: the context's stream 0)."""
from __future__ import annotations

from .api import HipBackend, check
from .attention import _at, _choice, _dtype

CODES = {"i8": 1, "fp8": 2}


class DenseBackend:
    """The dense calls of a decoder layer (objeta_hip.h says what each computes)."""

    def __init__(self, backend: HipBackend):
        self.backend = backend
        self.L = backend.L

    def rms_norm_device(self, n_tokens: int, hidden: int, dtype: str, d_x, d_weight, eps: float = 1e-6,
                        weight_dtype: str | None = None, weight_offset: float = 0.0, d_residual=None, d_residual_out=None,
                        residual_dtype: str | None = None, d_out=None, out_dtype: str | None = None, codes: str | None = None,
                        d_codes=None, d_scales=None, x_stride: int | None = None, residual_stride: int | None = None,
                        residual_out_stride: int | None = None, out_stride: int | None = None,
                        codes_stride: int | None = None, stream=None) -> None:
        """RMS norm of x + residual; any of: the sum (d_residual_out), the norm (d_out), its codes
        ("i8" with a float scale a token, "fp8" in the official blocks). Types default to `dtype`."""
        x = _dtype(dtype)
        check(self.L.objeta_hip_rms_norm_device(
            self.backend.ctx, stream, n_tokens, hidden, x, _at(d_x), hidden if x_stride is None else x_stride,
            x if weight_dtype is None else _dtype(weight_dtype), _at(d_weight), weight_offset, eps,
            x if residual_dtype is None else _dtype(residual_dtype), _at(d_residual),
            hidden if residual_stride is None else residual_stride, _at(d_residual_out),
            hidden if residual_out_stride is None else residual_out_stride, x if out_dtype is None else _dtype(out_dtype),
            _at(d_out), hidden if out_stride is None else out_stride, 0 if codes is None else _choice(CODES, codes, "codes"), _at(d_codes),
            hidden if codes_stride is None else codes_stride, _at(d_scales)))

    def quantize_rows_device(self, n_rows: int, cols: int, dtype: str, d_x, d_codes, d_scales, x_stride: int | None = None,
                             codes_stride: int | None = None, stream=None) -> None:
        """Rows (a weight's channels, tokens) to int8 with a float scale a row."""
        check(self.L.objeta_hip_quantize_rows_i8_device(
            self.backend.ctx, stream, n_rows, cols, _dtype(dtype), _at(d_x), cols if x_stride is None else x_stride,
            _at(d_codes), cols if codes_stride is None else codes_stride, _at(d_scales)))

    def i8_product_device(self, n_tokens: int, rows: int, cols: int, d_a, d_a_scales, d_w, d_w_scales, d_out,
                          out_dtype: str = "f32", d_bias=None, a_stride: int | None = None, w_stride: int | None = None,
                          out_stride: int | None = None, stream=None) -> None:
        """out[t][r] = (a[t] . w[r]) a_scales[t] w_scales[r] (+ bias[r]) of int8 rows."""
        check(self.L.objeta_hip_i8_product_device(
            self.backend.ctx, stream, n_tokens, rows, cols, _at(d_a), cols if a_stride is None else a_stride, _at(d_a_scales),
            _at(d_w), cols if w_stride is None else w_stride, _at(d_w_scales), _at(d_bias), _dtype(out_dtype), _at(d_out),
            rows if out_stride is None else out_stride))

    def log_probs_device(self, n_rows: int, vocab: int, dtype: str, d_logits, scale: float = 1.0, d_tokens=None,
                         n_given: int = 0, d_token_log_probs=None, d_lse=None, d_entropy=None, n_top: int = 0, d_top_ids=None,
                         d_top_log_probs=None, stride: int | None = None, stream=None) -> None:
        """ln softmax(scale * logits) of n_given tokens a row, each row's log-sum, entropy and n_top best."""
        check(self.L.objeta_hip_log_probs_device(
            self.backend.ctx, stream, n_rows, vocab, _dtype(dtype), _at(d_logits), vocab if stride is None else stride, scale,
            _at(d_tokens), n_given, _at(d_token_log_probs), _at(d_lse), _at(d_entropy), n_top, _at(d_top_ids),
            _at(d_top_log_probs)))
