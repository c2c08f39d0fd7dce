"""The attention half of a decoder layer over the C ABI: rotary positions, attention over
packed prompts, and a paged key/value cache with the attention that reads it.

The reference has the place but nothing in it: AttentionBackend answers Unsupported
(crates/objeta-cuda/src/attention.rs:1-21). Arguments named d_* are device addresses
(DeviceBuffer, int or c_void_p); element types are "f32", "f16" or "bf16"; strides count
elements from token to token and default to densely packed heads. Calls are asynchronous on
`stream` (None: the context's stream 0)."""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import KvCacheDesc, RopeParams, RopePlan
from .api import HipBackend, _addr, check

ELEMENT_TYPES = {"f32": 0, "f16": 1, "bf16": 2}
ELEMENT_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_LAYOUTS = {"interleaved": 0, "half": 1}
_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}


def _choice(table: dict, name, what: str) -> int:
    if name not in table:
        raise ValueError(f"{what} {name!r} must be one of {sorted(table)}")
    return table[name]


def _dtype(name) -> int:
    code = ELEMENT_TYPES.get(name)
    return _choice(ELEMENT_TYPES, name, "element type") if code is None else code


def _at(v):
    """An address as the C call takes it; integers and None go as they are, which is cheapest."""
    return v if type(v) is int or v is None else _addr(v)


class Rope:
    """Rotary positions of a model, made once: base `theta`, the head's first `rotary_dim`
    dimensions in "half" (i, i + rotary_dim / 2) or "interleaved" (2i, 2i + 1) pairs, and
    the scaling for contexts beyond the trained one (objeta_hip_rope_params). `amplitude`
    None takes the scaling's own (YaRN: 0.1 ln factor + 1, otherwise 1). Needs no device."""

    def __init__(self, rotary_dim: int, theta: float = 10000.0, layout: str = "half", scaling: str = "none",
                 factor: float = 1.0, original_context: float = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 amplitude: float | None = None):
        if amplitude is not None and amplitude == 0.0:
            raise ValueError("amplitude 0 would erase the rotated dimensions")
        p = RopeParams(theta, rotary_dim, _choice(_LAYOUTS, layout, "layout"), _choice(_SCALINGS, scaling, "scaling"), 0,
                       factor, original_context, beta_fast, beta_slow, 0.0 if amplitude is None else amplitude)
        self.plan = RopePlan()
        self._ref = C.byref(self.plan)
        check(_lib.load().objeta_hip_rope_init(C.byref(p), self._ref))
        self.rotary_dim = rotary_dim

    def turns(self) -> np.ndarray:
        """Each pair's turn per position as a 64-bit fraction of a full turn."""
        return np.array(self.plan.turn[:self.rotary_dim // 2], np.uint64)


class KvCache:
    """A paged key/value cache of a stack of layers (objeta_hip_kv_cache): k and v
    [n_layers][n_pages][n_kv_heads][page_size][head_dim] of `dtype`, page tables
    [n_seqs][max_pages], lengths and page counts, all on the device. Buffers not passed in
    are allocated, the tables empty. The page operations run on the device without a host
    round trip; device_error() of the MoeExecutor reports bad indices (bit 2) and a lack of
    free pages (bit 3)."""

    def __init__(self, backend: HipBackend, n_layers: int, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int,
                 n_seqs: int, max_pages: int, dtype: str = "bf16", d_k=None, d_v=None, d_page_table=None,
                 d_seq_lens=None, d_ref_counts=None):
        self.backend, self.L, self.dtype = backend, backend.L, dtype
        self.n_layers, self.n_pages, self.n_kv_heads = n_layers, n_pages, n_kv_heads
        self.page_size, self.head_dim, self.n_seqs, self.max_pages = page_size, head_dim, n_seqs, max_pages
        code = _dtype(dtype)
        nbytes = n_layers * n_pages * n_kv_heads * page_size * head_dim * ELEMENT_BYTES[dtype]

        def tables(n, value):
            return backend.to_device(np.full(n, value, np.int32))
        self.d_k = backend.alloc(nbytes) if d_k is None else d_k
        self.d_v = backend.alloc(nbytes) if d_v is None else d_v
        self.d_page_table = tables(n_seqs * max_pages, -1) if d_page_table is None else d_page_table
        self.d_seq_lens = tables(n_seqs, 0) if d_seq_lens is None else d_seq_lens
        self.d_ref_counts = tables(n_pages, 0) if d_ref_counts is None else d_ref_counts
        self.desc = KvCacheDesc(_addr(self.d_k), _addr(self.d_v), _addr(self.d_page_table), _addr(self.d_seq_lens),
                                _addr(self.d_ref_counts), code, n_layers, n_pages, n_kv_heads, page_size, head_dim, n_seqs,
                                max_pages)
        self._ref = C.byref(self.desc)

    def append_device(self, layer: int, d_seqs, d_cu_rows, n_batch: int, n_rows: int, dtype: str, d_k, d_v,
                      rope: Rope | None = None, d_positions=None, d_q=None, d_q_out=None, n_q_heads: int = 0,
                      q_out_dtype: str | None = None, k_stride: int | None = None, v_stride: int | None = None,
                      q_stride: int | None = None, q_out_stride: int | None = None, stream=None) -> None:
        """Keys and values of new tokens to the last slots of their sequences (made by
        extend_device), keys and, with d_q, queries rotated on the way."""
        row, q_row = self.n_kv_heads * self.head_dim, n_q_heads * self.head_dim
        check(self.L.objeta_hip_kv_append_device(
            self.backend.ctx, stream, self._ref, layer, _at(d_seqs), _at(d_cu_rows), n_batch, n_rows,
            _dtype(dtype), _at(d_k), row if k_stride is None else k_stride, _at(d_v),
            row if v_stride is None else v_stride, None if rope is None else rope._ref,
            _at(d_positions), _at(d_q), q_row if q_stride is None else q_stride, n_q_heads,
            _dtype(dtype if q_out_dtype is None else q_out_dtype), _at(d_q_out),
            q_row if q_out_stride is None else q_out_stride))

    def extend_device(self, d_seqs, d_counts, n: int, stream=None) -> None:
        """Room for d_counts[i] more tokens of sequence d_seqs[i]; a shared last page is copied."""
        check(self.L.objeta_hip_kv_extend_device(self.backend.ctx, stream, self._ref, _at(d_seqs),
                                                 _at(d_counts), n))

    def fork_device(self, d_src, d_dst, n: int, stream=None) -> None:
        """Sequence d_dst[i] becomes d_src[i] as it was before the call, on shared pages."""
        check(self.L.objeta_hip_kv_fork_device(self.backend.ctx, stream, self._ref, _at(d_src), _at(d_dst),
                                               n))

    def compact_device(self, d_seqs, d_drafts, d_keep, d_kept, n: int, max_keep: int, stream=None) -> None:
        """Of the last d_drafts[i] tokens of sequence d_seqs[i], those with the d_kept[i] ascending
        indices d_keep[i] stay and move together; the others are dropped."""
        check(self.L.objeta_hip_kv_compact_device(self.backend.ctx, stream, self._ref, _at(d_seqs),
                                                  _at(d_drafts), _at(d_keep), _at(d_kept), n, max_keep))

    def free_device(self, d_seqs, n: int, stream=None) -> None:
        """Sequence d_seqs[i] releases its pages and is empty."""
        check(self.L.objeta_hip_kv_free_device(self.backend.ctx, stream, self._ref, _at(d_seqs), n))


class AttentionBackend:
    """The calls the reference's AttentionBackend (attention.rs:1-21) leaves Unsupported."""

    def __init__(self, backend: HipBackend):
        self.backend = backend
        self.L = backend.L

    def rope_device(self, rope: Rope, d_positions, n_tokens: int, head_dim: int, d_q, d_q_out, n_q_heads: int, d_k=None,
                    d_k_out=None, n_k_heads: int = 0, dtype: str = "f32", out_dtype: str | None = None,
                    q_stride: int | None = None, q_out_stride: int | None = None, k_stride: int | None = None,
                    k_out_stride: int | None = None, stream=None) -> None:
        """Rotary positions for queries and (n_k_heads > 0) keys in one launch."""
        q_row, k_row = n_q_heads * head_dim, n_k_heads * head_dim
        check(self.L.objeta_hip_rope_device(
            self.backend.ctx, stream, rope._ref, _at(d_positions), n_tokens, head_dim, _dtype(dtype),
            _dtype(dtype if out_dtype is None else out_dtype), _at(d_q), q_row if q_stride is None else q_stride,
            _at(d_q_out), q_row if q_out_stride is None else q_out_stride, n_q_heads, _at(d_k),
            k_row if k_stride is None else k_stride, _at(d_k_out),
            k_row if k_out_stride is None else k_out_stride, n_k_heads))

    def prompt_device(self, dtype: str, d_q, d_k, d_v, d_out, n_q_heads: int, n_kv_heads: int, head_dim: int,
                      n_tokens: int, d_cu_seqlens, n_seqs: int, causal: bool = True, scale: float | None = None,
                      d_lse=None, q_stride: int | None = None, k_stride: int | None = None, v_stride: int | None = None,
                      out_stride: int | None = None, stream=None) -> None:
        """Attention over packed sequences; scale None is head_dim ** -0.5."""
        q_row, kv_row = n_q_heads * head_dim, n_kv_heads * head_dim
        check(self.L.objeta_hip_attn_prompt_device(
            self.backend.ctx, stream, _dtype(dtype), _at(d_q), q_row if q_stride is None else q_stride, n_q_heads,
            _at(d_k), kv_row if k_stride is None else k_stride, _at(d_v), kv_row if v_stride is None else v_stride,
            n_kv_heads, head_dim, n_tokens, _at(d_cu_seqlens), n_seqs, 1 if causal else 0,
            head_dim ** -0.5 if scale is None else scale, _at(d_out), q_row if out_stride is None else out_stride,
            _at(d_lse)))

    def cached_device(self, cache: KvCache, layer: int, d_seqs, d_cu_rows, n_batch: int, n_rows: int, max_rows: int,
                      max_len: int, dtype: str, d_q, d_out, n_q_heads: int, d_tree=None, scale: float | None = None,
                      d_lse=None, q_stride: int | None = None, out_stride: int | None = None, stream=None) -> None:
        """Attention of each sequence's last rows over the cache: causal, or by the 64-bit masks
        d_tree among an entry's own rows. scale None is head_dim ** -0.5."""
        q_row = n_q_heads * cache.head_dim
        check(self.L.objeta_hip_attn_cached_device(
            self.backend.ctx, stream, cache._ref, layer, _at(d_seqs), _at(d_cu_rows), n_batch, n_rows,
            max_rows, max_len, _dtype(dtype), _at(d_q), q_row if q_stride is None else q_stride, n_q_heads,
            _at(d_tree), cache.head_dim ** -0.5 if scale is None else scale, _at(d_out),
            q_row if out_stride is None else out_stride, _at(d_lse)))
