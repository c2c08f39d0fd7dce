"""Rotary positions, prompt attention and attention over the cache against the plain 64-bit
forms of attn_reference, within the error bounds derived there."""
import ctypes as C

import numpy as np
import pytest

from attn_reference import (NP, attend, download, frequencies, from_type, lse_bound, rotate, rotate_bound, to_type)
from objeta_amd import AttentionBackend, KvCache, MoeExecutor, Rope
from objeta_amd.api import check

pytestmark = pytest.mark.gpu

FILL = 7.0  # what untouched output rows hold


@pytest.fixture
def att(backend):
    MoeExecutor(backend).device_error()
    yield AttentionBackend(backend)
    assert MoeExecutor(backend).device_error() == 0


# ---------------------------------------------------------------------- rotary
@pytest.mark.parametrize("tin,tout", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary,nq,nk", [(64, 64, 5, 2), (128, 64, 32, 4), (8, 2, 1, 1), (80, 80, 3, 0), (256, 250, 2, 7), (40, 6, 70, 3)])
def test_rope(backend, att, tin, tout, layout, dim, rotary, nq, nk):
    rng = np.random.default_rng(1)
    n = 9
    pos = np.array([0, 1, -1, 4095, 131072, 1 << 20, 2 ** 31 - 1, -2 ** 31, 12345], np.int32)
    q, k = (to_type(rng.standard_normal((n, h, dim)), tin) for h in (nq, max(nk, 1)))
    rope = Rope(rotary, theta=500000.0, layout=layout, scaling="yarn", factor=8.0, original_context=2048)
    amp = float(rope.plan.amplitude)
    dq, dk, dp = (backend.to_device(x) for x in (q, k, pos))
    qo, ko = (backend.to_device(np.zeros(x.shape, NP[tout])) for x in (q, k))
    att.rope_device(rope, dp, n, dim, dq, qo, nq, dk if nk else None, ko if nk else None, nk, dtype=tin, out_dtype=tout)
    backend.synchronize()
    f = frequencies(rotary, 500000.0, "yarn", 8.0, 2048)
    for x, o, h in ((q, qo, nq),) + (((k, ko, nk),) if nk else ()):
        x64 = from_type(x, tin)
        want = rotate(x64, pos, f, layout, amp)
        # the angle's own: frequencies as doubles (14 half steps of 2^-53) times the position
        far = np.abs(pos.astype(np.float64))[:, None, None] * 3e-15 * amp * np.abs(x64).max() * 2
        assert np.all(np.abs(download(o, tout, x.shape) - want) <= rotate_bound(x64, rotary, layout, tout, amp, want) + far)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad", [0, 4, 1])
def test_rope_in_place_in_a_packed_buffer(backend, att, dtype, pad):
    """q and k rotated where they lie in rows of q | k | v; odd row lengths take single elements."""
    rng = np.random.default_rng(2)
    n, dim, nq, nk = 33, 64, 4, 2
    row = dim * (nq + 2 * nk) + pad
    x = to_type(rng.standard_normal((n, row)), dtype)
    pos = np.arange(n, dtype=np.int32) + 70000
    d, es = backend.to_device(x), x.itemsize
    q_at, k_at = d.ptr, d.ptr + nq * dim * es
    rope = Rope(dim, layout="interleaved")
    att.rope_device(rope, backend.to_device(pos), n, dim, q_at, q_at, nq, k_at, k_at, nk, dtype=dtype, q_stride=row,
                    q_out_stride=row, k_stride=row, k_out_stride=row)
    backend.synchronize()
    got = download(d, dtype, x.shape)
    x64 = from_type(x, dtype)
    heads = x64[:, :dim * (nq + nk)].reshape(n, nq + nk, dim)
    want = rotate(heads, pos, frequencies(dim, 10000.0), "interleaved")
    bound = rotate_bound(heads, dim, "interleaved", dtype, 1.0, want) + 70033 * 3e-15 * 10
    assert np.all(np.abs(got[:, :dim * (nq + nk)].reshape(heads.shape) - want) <= bound)
    assert np.array_equal(got[:, dim * (nq + nk):], x64[:, dim * (nq + nk):])


def test_rope_many_tokens_on_another_stream(backend, att):
    n, dim = 3001, 32
    x = np.random.default_rng(3).standard_normal((n, 2, dim)).astype(np.float32)
    pos = np.arange(n, dtype=np.int32)
    st = backend.stream(1)
    d, p = backend.to_device(x, st), backend.to_device(pos, st)
    att.rope_device(Rope(dim), p, n, dim, d, d, 2, stream=st)
    backend.synchronize(st)
    want = rotate(x.astype(np.float64), pos, frequencies(dim, 10000.0), "half")
    assert np.all(np.abs(d.download(np.float32, x.size, st).reshape(x.shape) - want) <= rotate_bound(x, dim, "half", "f32", 1.0, want) + 1e-10)


# --------------------------------------------------------------------- prompts
def check_heads(got, lse, q, k, v, seen_of, rows_of, scale, dtype, group):
    """Every row of every head within its bound; seen_of(rows) gives the mask of a sequence."""
    for lo, hi, klo, khi in rows_of:
        if lo == hi:
            continue
        seen = seen_of(lo, hi, klo, khi)
        for h in range(q.shape[1]):
            g = h // group
            out, want_lse, bound = attend(q[lo:hi, h], k[klo:khi, g], v[klo:khi, g], seen, scale, dtype, dtype)
            err = np.abs(got[lo:hi, h] - out)
            assert np.all(err <= bound), (lo, hi, h, float(np.max(err / np.maximum(bound, 1e-300))))
            some = np.isfinite(want_lse)
            mag = scale * (np.abs(np.nan_to_num(q[lo:hi, h], posinf=0, neginf=0)) @ np.abs(np.nan_to_num(k[klo:khi, g], posinf=0, neginf=0)).T).max()
            assert np.all(np.abs(lse[lo:hi, h] - want_lse)[some] <= lse_bound(want_lse, q.shape[2], mag)[some])
            assert np.array_equal(np.isneginf(lse[lo:hi, h]), ~some)


def run_prompt(backend, att, q, k, v, lens, dtype, causal, scale=None, before=0, strides=None, stream=None):
    """q, k, v as uploaded arrays [n][heads][dim]; the sequences start at row `before`."""
    n, nq, dim = q.shape
    nk = k.shape[1]
    cu = np.concatenate(([before], before + np.cumsum(lens))).astype(np.int32)
    dq, dk, dv = (backend.to_device(x, stream) for x in (q, k, v))
    fill = to_type(np.full(q.shape, FILL), dtype)
    out, lse = backend.to_device(fill, stream), backend.to_device(np.full((n, nq), FILL, np.float32), stream)
    att.prompt_device(dtype, dq, dk, dv, out, nq, nk, dim, n, backend.to_device(cu, stream), len(lens), causal=causal,
                      scale=scale, d_lse=lse, stream=stream)
    backend.synchronize(stream)
    return download(out, dtype, q.shape), lse.download(np.float32, n * nq, stream).reshape(n, nq).astype(np.float64), cu


def prompt_case(backend, att, dtype, nq, nk, dim, lens, causal, pad=3, before=0, scale=None, seed=0, size=1.0):
    rng = np.random.default_rng(seed)
    n = before + sum(lens) + pad
    q, k, v = (to_type(size * rng.standard_normal((n, h, dim)), dtype) for h in (nq, nk, nk))
    got, lse, cu = run_prompt(backend, att, q, k, v, lens, dtype, causal, scale, before)
    q64, k64, v64 = (from_type(x, dtype) for x in (q, k, v))
    s = dim ** -0.5 if scale is None else scale

    def seen(lo, hi, klo, khi):
        m = np.ones((hi - lo, khi - klo), bool)
        return np.tril(m) if causal else m
    check_heads(got, lse, q64, k64, v64, seen, [(a, b, a, b) for a, b in zip(cu[:-1], cu[1:])], np.float64(np.float32(s)), dtype, nq // nk)
    for r in list(range(before)) + list(range(cu[-1], n)):
        assert np.all(got[r] == FILL) and np.all(lse[r] == FILL)


TYPES = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk,dim", [(1, 1, 8), (4, 2, 64), (3, 3, 40), (8, 1, 128), (5, 1, 80), (2, 2, 256), (6, 2, 136)])
def test_prompt_heads(backend, att, dtype, causal, nq, nk, dim):
    prompt_case(backend, att, dtype, nq, nk, dim, [1, 0, 33, 64, 97, 2], causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [2], [31], [32], [63], [64], [65], [127], [128], [129], [300], [0], [0, 0, 5, 0], [1] * 70,
                                  [128, 128], [129, 127, 1]])
def test_prompt_lengths(backend, att, dtype, lens):
    prompt_case(backend, att, dtype, 2, 1, 64, lens, True, before=len(lens) % 3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompt_long(backend, att, dtype):
    prompt_case(backend, att, dtype, 2, 2, 128, [1111, 700], True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,size", [(0.02, 1.0), (1.0, 1.0), (0.3, 4.0)])
def test_prompt_scales(backend, att, dtype, scale, size):
    """Flat and very peaked softmaxes (scores to several hundred)."""
    prompt_case(backend, att, dtype, 2, 1, 64, [150], True, scale=scale, size=size)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_growing_scores(backend, att, dtype):
    """Every key's score above all before it, so that the running maximum moves in each tile."""
    n, dim = 400, 64
    rng = np.random.default_rng(4)
    k = rng.standard_normal((n, 1, dim)) * 0.05
    k[:, 0, 0] = np.arange(n) * 0.25
    q = rng.standard_normal((n, 1, dim)) * 0.05
    q[:, 0, 0] = 1.0
    v = rng.standard_normal((n, 1, dim))
    for sign in (1.0, -1.0):  # and below all before it
        a = [to_type(x, dtype) for x in (q, k * sign, v)]
        got, lse, cu = run_prompt(backend, att, *a, [n], dtype, False, scale=1.0)
        q64, k64, v64 = (from_type(x, dtype) for x in a)
        check_heads(got, lse, q64, k64, v64, lambda *r: np.ones((n, n), bool), [(0, n, 0, n)], 1.0, dtype, 1)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_strides(backend, att, dtype):
    """Queries, keys and values in one packed buffer, outputs in wider rows."""
    rng = np.random.default_rng(5)
    n, nq, nk, dim, wide = 77, 4, 2, 64, 4 * 64 + 8
    row = dim * (nq + 2 * nk)
    x = to_type(rng.standard_normal((n, row)), dtype)
    es = x.itemsize
    d = backend.to_device(x)
    out = backend.to_device(to_type(np.full((n, wide), FILL), dtype))
    cu = backend.to_device(np.array([0, 50, 77], np.int32))
    att.prompt_device(dtype, d.ptr, d.ptr + nq * dim * es, d.ptr + (nq + nk) * dim * es, out, nq, nk, dim, n, cu, 2,
                      q_stride=row, k_stride=row, v_stride=row, out_stride=wide)
    backend.synchronize()
    got = download(out, dtype, (n, wide))
    assert np.all(got[:, nq * dim:] == FILL)
    x64 = from_type(x, dtype)
    q, k, v = (x64[:, a * dim:b * dim].reshape(n, -1, dim) for a, b in ((0, nq), (nq, nq + nk), (nq + nk, nq + 2 * nk)))
    got = got[:, :nq * dim].reshape(n, nq, dim)
    for lo, hi in ((0, 50), (50, 77)):
        for h in range(nq):
            o, _, bound = attend(q[lo:hi, h], k[lo:hi, h // 2], v[lo:hi, h // 2], np.tril(np.ones((hi - lo, hi - lo), bool)),
                                 np.float64(np.float32(0.125)), dtype, dtype)
            assert np.all(np.abs(got[lo:hi, h] - o) <= bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_prompt_unseen_places_do_not_matter(backend, att, dtype, what):
    """Infinities and NaN in later tokens, in the sequence behind and in padding."""
    rng = np.random.default_rng(6)
    n, nq, nk, dim = 120, 4, 2, 64
    q, k, v = (rng.standard_normal((n, h, dim)) for h in (nq, nk, nk))
    bad_from, lens = 70, [40, 60]  # tokens 70.. of the second sequence see them, nobody before does
    a = [to_type(x, dtype) for x in (q, k, v)]
    base, base_lse, _ = run_prompt(backend, att, *a, lens, dtype, True)
    k[bad_from:], v[bad_from:] = what, what
    q[100:] = what
    b = [to_type(x, dtype) for x in (q, k, v)]
    got, lse, cu = run_prompt(backend, att, *b, lens, dtype, True)
    q64, k64, v64 = (from_type(x, dtype) for x in a)
    check_heads(got, lse, q64, k64, v64, lambda lo, hi, klo, khi: np.tril(np.ones((hi - lo, khi - klo), bool)),
                [(0, 40, 0, 40), (40, 70, 40, 70)], np.float64(np.float32(0.125)), dtype, 2)
    assert not np.any(np.isfinite(got[70:100]))
    assert np.all(got[100:] == FILL)
    assert np.all(np.isfinite(base[:100]))


def test_prompt_a_seen_infinity(backend, att):
    """A value of infinity that a row sees is its result there and leaves other dimensions alone."""
    n, dim = 70, 16
    rng = np.random.default_rng(7)
    q, k, v = (rng.standard_normal((n, 1, dim)).astype(np.float32) for _ in range(3))
    v[10, 0, 3] = np.inf
    got, lse, _ = run_prompt(backend, att, q, k, v, [n], "f32", True)
    assert np.all(np.isinf(got[10:, 0, 3])) and np.all(np.isfinite(got[:10, 0, 3]))
    v2 = v.copy()
    v2[10, 0, 3] = 0
    want, want_lse, _ = run_prompt(backend, att, q, k, v2, [n], "f32", True)
    keep = [d for d in range(dim) if d != 3]
    # both are within the bound of the exact result, one of them summed in another order
    assert np.max(np.abs(got[:, 0, keep] - want[:, 0, keep])) <= 1e-5
    assert np.max(np.abs(lse - want_lse)) <= 1e-5


def test_prompt_scores_of_minus_infinity(backend, att):
    """Keys of the type's lowest value and of -inf: rows whose every score is -inf come out 0."""
    n, dim = 40, 32
    q = np.ones((n, 1, dim), np.float32)
    k = np.zeros((n, 1, dim), np.float32)
    v = np.random.default_rng(8).standard_normal((n, 1, dim)).astype(np.float32)
    k[:5] = -np.inf
    k[5:9] = np.finfo(np.float32).min
    got, lse, _ = run_prompt(backend, att, q, k, v, [n], "f32", True)
    assert np.all(got[:9] == 0) and np.all(np.isneginf(lse[:9]))
    for i in range(9, n):
        assert np.allclose(got[i, 0], v[9:i + 1, 0].mean(0), atol=1e-5)


def test_prompt_bad_indices(backend):
    """Indices out of order or range leave rows untouched; ends past the tokens are reported."""
    att, err = AttentionBackend(backend), MoeExecutor(backend)
    err.device_error()
    rng = np.random.default_rng(9)
    q = rng.standard_normal((20, 1, 16)).astype(np.float32)
    d = backend.to_device(q)
    for cu, ok_rows, bit in (([0, 10, 25], range(10), 4), ([-5, 10, 20], range(10, 20), 4), ([30, 40, 50], [], 0)):
        out = backend.to_device(np.full(q.shape, FILL, np.float32))
        att.prompt_device("f32", d, d, d, out, 1, 1, 16, 20, backend.to_device(np.array(cu, np.int32)), 2)
        backend.synchronize()
        got = out.download(np.float32, q.size).reshape(q.shape)
        touched = [r for r in range(20) if not np.all(got[r] == FILL)]
        assert touched == list(ok_rows), cu
        assert err.device_error() == bit


def test_prompt_same_bits_again(backend, att):
    rng = np.random.default_rng(10)
    a = [to_type(rng.standard_normal((700, h, 128)), "bf16") for h in (8, 2, 2)]
    first, l1, _ = run_prompt(backend, att, *a, [300, 400], "bf16", True)
    second, l2, _ = run_prompt(backend, att, *a, [300, 400], "bf16", True, stream=backend.stream(1))
    assert np.array_equal(first, second) and np.array_equal(l1, l2)


# ----------------------------------------------------------------- cached decode
class Cached:
    """A cache filled with random keys and values for sequences of the given lengths."""

    def __init__(self, backend, lens, kv="bf16", heads=2, page=16, dim=64, layers=1, seed=0, spare=3):
        rng = self.rng = np.random.default_rng(seed)
        self.be, self.lens, self.kv, self.page, self.heads, self.dim = backend, lens, kv, page, heads, dim
        pages = [-(-n // page) for n in lens]
        total, top = sum(pages) + spare, max(pages + [1]) + 2
        order = rng.permutation(total)
        self.table = np.full((len(lens), top), -1, np.int32)
        at = 0
        for s, p in enumerate(pages):
            self.table[s, :p] = order[at:at + p]
            at += p
        self.k, self.v = (to_type(rng.standard_normal((layers, total, heads, page, dim)), kv) for _ in range(2))
        self.cache = KvCache(backend, layers, total, heads, page, dim, len(lens), top, dtype=kv)
        self.upload()

    def upload(self):
        self.cache.d_k.upload(self.k)
        self.cache.d_v.upload(self.v)
        self.cache.d_page_table.upload(self.table)
        self.cache.d_seq_lens.upload(np.array(self.lens, np.int32))

    def rows_of(self, which, layer, s):
        a = from_type(getattr(self, which)[layer], self.kv)
        pages = self.table[s][:-(-self.lens[s] // self.page)]
        return a[pages].transpose(1, 0, 2, 3).reshape(self.heads, -1, self.dim)[:, :self.lens[s]]

    def set_slot(self, which, s, slot, value):
        getattr(self, which)[:, self.table[s, slot // self.page], :, slot % self.page] = value


def run_cached(att, c, seqs, rows, dtype, nq, tree=None, layer=0, max_rows=None, max_len=None, pad=2, seed=1, stream=None, q=None,
               scale=None):
    be = c.be
    n = sum(rows) + pad
    rng = np.random.default_rng(seed)
    if q is None:
        q = to_type(rng.standard_normal((n, nq, c.dim)), dtype)
    cu = np.concatenate(([0], np.cumsum(rows))).astype(np.int32)
    out = be.to_device(to_type(np.full(q.shape, FILL), dtype), stream)
    lse = be.to_device(np.full((n, nq), FILL, np.float32), stream)
    masks = None if tree is None else be.to_device(np.array(list(tree) + [0] * pad, np.uint64), stream)
    att.cached_device(c.cache, layer, be.to_device(np.array(seqs, np.int32), stream), be.to_device(cu, stream), len(seqs), n,
                      max(rows + [1]) if max_rows is None else max_rows, max(c.lens) if max_len is None else max_len, dtype,
                      be.to_device(q, stream), out, nq, d_tree=masks, d_lse=lse, stream=stream, scale=scale)
    be.synchronize(stream)
    got = from_type(out.download(NP[dtype], q.size, stream).reshape(q.shape), dtype)
    l = lse.download(np.float32, n * nq, stream).reshape(n, nq).astype(np.float64)
    assert np.all(got[n - pad:] == FILL) and np.all(l[n - pad:] == FILL)
    return q, got, l, cu


def check_cached(c, seqs, q, got, lse, cu, dtype, nq, tree=None, layer=0):
    group = nq // c.heads
    scale = np.float64(np.float32(c.dim ** -0.5))
    for b, s in enumerate(seqs):
        lo, hi = cu[b], cu[b + 1]
        if lo == hi:
            continue
        n, m = c.lens[s], hi - lo
        k, v = c.rows_of("k", layer, s), c.rows_of("v", layer, s)
        seen = np.ones((m, n), bool)
        for i in range(m):
            if tree is None:
                seen[i, n - m + i + 1:] = False
            else:
                seen[i, n - m:] = [(int(tree[lo + i]) >> j) & 1 for j in range(m)]
        for h in range(nq):
            # float queries: neither the scores nor the probabilities are rounded to the cache's type
            out, want_lse, bound = attend(from_type(q[lo:hi, h], dtype), k[h // group], v[h // group], seen, scale, dtype, dtype)
            err = np.abs(got[lo:hi, h] - out)
            assert np.all(err <= bound), (b, s, h, float(np.max(err / np.maximum(bound, 1e-300))))
            some = np.isfinite(want_lse)
            assert np.array_equal(np.isneginf(lse[lo:hi, h]), ~some)
            mag = scale * (np.abs(from_type(q[lo:hi, h], dtype)) @ np.abs(k[h // group]).T).max()
            assert np.all(np.abs(lse[lo:hi, h] - want_lse)[some] <= lse_bound(want_lse, c.dim, mag)[some])


PAIRS = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


@pytest.mark.parametrize("dtype,kv", PAIRS)
@pytest.mark.parametrize("page,dim,nq,nk", [(8, 64, 4, 2), (16, 128, 8, 1), (32, 256, 2, 2), (64, 40, 3, 3), (256, 136, 7, 1), (16, 8, 40, 1)])
def test_cached_decode(backend, att, dtype, kv, page, dim, nq, nk):
    c = Cached(backend, [1, 37, 300, 64, 5], kv, nk, page, dim)
    seqs, rows = [3, 0, 4, 1, 2, 2], [1, 1, 1, 1, 1, 0]
    q, got, lse, cu = run_cached(att, c, seqs, rows, dtype, nq)
    check_cached(c, seqs, q, got, lse, cu, dtype, nq)


@pytest.mark.parametrize("dtype,kv", PAIRS)
@pytest.mark.parametrize("rows", [[1, 3, 2], [8, 8, 8], [33, 5, 64], [200, 1, 130]])
def test_cached_chunks(backend, att, dtype, kv, rows):
    """The causal chain: chunks of a prompt over what is cached, chunk and context of one length too."""
    c = Cached(backend, [200, 77, 700], kv, 2, 16, 64)
    q, got, lse, cu = run_cached(att, c, [0, 1, 2], rows, dtype, 8)
    check_cached(c, [0, 1, 2], q, got, lse, cu, dtype, 8)


def tree_masks(rng, n):
    bits = []
    for i in range(n):
        parent = int(rng.integers(max(0, i - 5), i + 1)) - 1
        bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
    return bits


@pytest.mark.parametrize("dtype,kv", PAIRS)
@pytest.mark.parametrize("rows,nq,nk", [([1, 2, 7], 4, 2), ([64, 33, 64], 2, 1), ([64, 1, 20], 8, 1), ([5, 4, 3], 3, 3)])
def test_cached_trees(backend, att, dtype, kv, rows, nq, nk):
    c = Cached(backend, [64, 100, 515], kv, nk, 16, 64, seed=2)
    rng = np.random.default_rng(3)
    tree = sum([tree_masks(rng, n) for n in rows], [])
    q, got, lse, cu = run_cached(att, c, [0, 1, 2], rows, dtype, nq, tree=tree)
    check_cached(c, [0, 1, 2], q, got, lse, cu, dtype, nq, tree=tree)


@pytest.mark.parametrize("dtype,kv", [("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("rows", [[4], [40]])
def test_cached_tree_rows_that_see_nothing(backend, att, dtype, kv, rows):
    """Drafts at the very start of a sequence, with masks of 0: no key at all; and any other mask."""
    n = rows[0]
    c = Cached(backend, [n], kv, 1, 8, 64, seed=4)
    rng = np.random.default_rng(5)
    tree = [0 if i % 3 == 0 else int(rng.integers(0, 1 << n, dtype=np.uint64)) for i in range(n)]
    q, got, lse, cu = run_cached(att, c, [0], rows, dtype, 2, tree=tree)
    check_cached(c, [0], q, got, lse, cu, dtype, 2, tree=tree)
    assert np.all(got[0] == 0) and np.all(np.isneginf(lse[0]))


@pytest.mark.parametrize("dtype,kv", PAIRS)
@pytest.mark.parametrize("rows", [1, 48])
def test_cached_long_contexts_are_cut(backend, att, dtype, kv, rows):
    """Keys over many workgroups and the join of their parts, lengths around the cuts."""
    c = Cached(backend, [5000, 256, 257, 4999, 255, 511], kv, 1, 64, 64, seed=6)
    seqs, r = [0, 1, 2, 3, 4, 5], [rows] * 6
    q, got, lse, cu = run_cached(att, c, seqs, r, dtype, 2)
    check_cached(c, seqs, q, got, lse, cu, dtype, 2)


@pytest.mark.parametrize("rows", [[1, 2], [70, 3]])
def test_cached_bounds_only_cut_the_work(backend, att, rows):
    """max_len below and far above the truth, and max_rows above it, give the same results."""
    c = Cached(backend, [1500, 900], "bf16", 2, 16, 64, seed=7)
    for mr, ml in ((70, 1), (70, 100000), (75, 300), (1000, 1500), (72, 257)):
        q, got, lse, cu = run_cached(att, c, [0, 1], rows, "bf16", 8, max_rows=mr, max_len=ml)
        check_cached(c, [0, 1], q, got, lse, cu, "bf16", 8)


@pytest.mark.parametrize("rows,max_rows,group", [([4, 9], 4, 4), ([50, 3], 40, 8), ([20, 70], 1, 16)])
@pytest.mark.parametrize("max_len", [200, 3000])
def test_cached_more_rows_than_said(backend, rows, max_rows, group, max_len):
    """Rows past max_rows come out right or NaN and are reported; those within it are right."""
    att, err = AttentionBackend(backend), MoeExecutor(backend)
    err.device_error()
    c = Cached(backend, [1500, 900], "f16", 1, 16, 64, seed=7)
    q, got, lse, cu = run_cached(att, c, [0, 1], rows, "f16", group, max_rows=max_rows, max_len=max_len)
    assert err.device_error() == 4
    full, full_lse = run_cached(att, c, [0, 1], rows, "f16", group, q=q, max_len=max_len)[1:3]
    for b in range(2):
        for r in range(cu[b], cu[b + 1]):
            for h in range(group):
                gone = np.isnan(got[r, h]).all() and np.isnan(lse[r, h])
                # the same sums, the keys cut elsewhere: half a step of the output and of p each
                near = np.all(np.abs(got[r, h] - full[r, h]) <= 4 * 2.0 ** -11) and abs(lse[r, h] - full_lse[r, h]) <= 1e-5
                assert near or (gone and r - cu[b] >= max_rows), (b, r, h)


def test_cached_layers(backend, att):
    c = Cached(backend, [50, 20], "f16", 2, 8, 32, layers=3, seed=8)
    for layer in range(3):
        q, got, lse, cu = run_cached(att, c, [0, 1], [1, 1], "f16", 2, layer=layer)
        check_cached(c, [0, 1], q, got, lse, cu, "f16", 2, layer=layer)


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f32", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("rows", [4, 50])
@pytest.mark.parametrize("long", [False, True])
def test_cached_unseen_places_do_not_matter(backend, att, dtype, kv, rows, long):
    """NaN and infinities in slots past a sequence, in pages of nobody, in drafts masked out and
    later in the chain."""
    c = Cached(backend, [2500 if long else 100, 90], kv, 1, 16, 64, seed=9)
    rng = np.random.default_rng(10)
    n = [rows, rows]
    tree = sum([tree_masks(rng, m) for m in n], [])
    hidden = rows - 2  # draft nobody but itself sees
    for b in range(2):
        for i in range(rows):
            if i != hidden:
                tree[b * rows + i] &= ~(1 << hidden)
    q, want, want_lse, cu = run_cached(att, c, [0, 1], n, dtype, 2, tree=tree)
    nan = to_type(np.array(np.nan), kv)
    used = set(c.table[c.table >= 0].tolist())
    for x in (c.k, c.v):
        for p in range(x.shape[1]):
            if p not in used:
                x[:, p] = nan
    for s in range(2):
        for slot in range(c.lens[s], -(-c.lens[s] // 16) * 16):
            c.set_slot("k", s, slot, nan)
            c.set_slot("v", s, slot, to_type(np.array(np.inf), kv))
        c.set_slot("k", s, c.lens[s] - rows + hidden, nan)
        c.set_slot("v", s, c.lens[s] - rows + hidden, nan)
    c.upload()
    _, got, lse, _ = run_cached(att, c, [0, 1], n, dtype, 2, tree=tree)
    rest = [r for r in range(2 * rows) if r % rows != hidden]
    assert np.all(np.isnan(got[[hidden, rows + hidden]]))
    for b in range(2):  # the plain form over what is seen: the hidden draft's place filled with zeros
        s = b
        c.set_slot("k", s, c.lens[s] - rows + hidden, 0)
        c.set_slot("v", s, c.lens[s] - rows + hidden, 0)
    got[[hidden, rows + hidden]], lse[[hidden, rows + hidden]] = 0, 0
    for b in range(2):
        lo, m, L = b * rows, rows, c.lens[b]
        k, v = c.rows_of("k", 0, b)[0], c.rows_of("v", 0, b)[0]
        seen = np.ones((m, L), bool)
        for i in range(m):
            seen[i, L - m:] = [(int(tree[lo + i]) >> j) & 1 for j in range(m)]
        for h in range(2):
            out, _, bound = attend(from_type(q[lo:lo + m, h], dtype), k, v, seen, np.float64(np.float32(0.125)), dtype, dtype)
            ok = [i for i in range(m) if i != hidden]
            assert np.all(np.abs(got[lo:lo + m, h] - out)[ok] <= bound[ok])


@pytest.mark.parametrize("rows", [1, 40])
def test_cached_bad_indices(backend, rows):
    """Bad sequences, lengths and pages: NaN for the entry, the rest right, the error word set."""
    att, err = AttentionBackend(backend), MoeExecutor(backend)
    err.device_error()
    c = Cached(backend, [600, 50, 45], "f16", 1, 16, 64, seed=11)
    q, got, lse, cu = run_cached(att, c, [0, 9, 1, -1], [rows] * 4, "f16", 2)
    check_cached(c, [0], q, got, lse, cu[:2], "f16", 2)
    assert np.all(np.isnan(got[rows:2 * rows])) and np.all(np.isnan(got[3 * rows:4 * rows])) and np.all(np.isnan(lse[rows:2 * rows]))
    assert np.all(np.isfinite(got[2 * rows:3 * rows])) and err.device_error() == 4
    good = c.table.copy()
    for bad in (-1, c.k.shape[1], 1 << 30):
        c.table[0, 20] = bad
        c.cache.d_page_table.upload(c.table)
        _, got, lse, _ = run_cached(att, c, [0, 1], [rows] * 2, "f16", 2)
        assert np.all(np.isnan(got[:rows])) and np.all(np.isfinite(got[rows:2 * rows])) and err.device_error() == 4
    c.table = good
    c.upload()
    for lens in ([-3, 50, 45], [1 << 30, 50, 45], [rows - 1, 50, 45]):
        c.cache.d_seq_lens.upload(np.array(lens, np.int32))
        _, got, lse, _ = run_cached(att, c, [0, 1], [rows] * 2, "f16", 2, max_len=600)
        assert np.all(np.isnan(got[:rows])) and np.all(np.isfinite(got[rows:2 * rows])) and err.device_error() == 4
    c.upload()
    # more than 64 rows under masks
    _, got, _, _ = run_cached(att, c, [0, 1], [65, 3], "f16", 2, tree=[1] * 68)
    assert np.all(np.isnan(got[:65])) and np.all(np.isfinite(got[65:68])) and err.device_error() == 4
    # row indices out of range or order name no rows
    be = backend
    for cu in ([-1, 2, 4], [0, 5, 4], [0, 2, 99]):
        q = be.to_device(np.zeros((4, 2, 64), np.float16))
        out = be.to_device(np.full((4, 2, 64), FILL, np.float16))
        att.cached_device(c.cache, 0, be.to_device(np.array([1, 2], np.int32)), be.to_device(np.array(cu, np.int32)), 2, 4, rows, 600,
                          "f16", q, out, 2)
        be.synchronize()
        assert err.device_error() == 4
        got = out.download(np.float16, 512).reshape(4, 128)
        named = {r for a, b in zip(cu[:-1], cu[1:]) if 0 <= a <= b <= 4 for r in range(a, b)}
        for r in range(4):
            if r not in named:
                assert np.all(got[r] == FILL)


def test_cached_two_streams_and_graph(backend, att):
    """Calls in flight on two streams have workspaces of their own; a captured call replays on
    lengths and contents that changed since."""
    c = Cached(backend, [3000, 2000], "bf16", 2, 16, 64, seed=12)
    d = Cached(backend, [2500, 1000], "bf16", 2, 16, 64, seed=13)
    st = [backend.stream(0), backend.stream(1)]
    ref = [run_cached(att, x, [0, 1], [1, 1], "bf16", 8, stream=s) for x, s in ((c, st[0]), (d, st[1]))]
    be, bufs = backend, []
    for x, s, r in ((c, st[0], ref[0]), (d, st[1], ref[1])):
        bufs.append([be.to_device(np.array([0, 1], np.int32), s), be.to_device(r[3], s), be.to_device(r[0], s), be.alloc(r[0].nbytes)])

    def call(x, b, s):
        att.cached_device(x.cache, 0, b[0], b[1], 2, 4, 1, 3000, "bf16", b[2], b[3], 8, stream=s)
    for _ in range(20):
        call(c, bufs[0], st[0])
        call(d, bufs[1], st[1])
    for i in range(2):
        be.synchronize(st[i])
        got = from_type(bufs[i][3].download(np.uint16, ref[i][0].size, st[i]).reshape(ref[i][0].shape), "bf16")
        assert np.array_equal(got[:2], ref[i][1][:2])
    check(be.L.objeta_hip_graph_begin_capture(be.ctx, st[0]))
    call(c, bufs[0], st[0])
    g = C.c_void_p()
    check(be.L.objeta_hip_graph_end_capture(be.ctx, st[0], C.byref(g)))
    for lens in ([3000, 2000], [17, 1999], [1, 2]):
        c.lens = lens
        c.upload()
        want = run_cached(att, c, [0, 1], [1, 1], "bf16", 8, stream=st[0], q=ref[0][0], max_len=3000)
        check(be.L.objeta_hip_graph_launch(be.ctx, g, st[0]))
        be.synchronize(st[0])
        got = from_type(bufs[0][3].download(np.uint16, ref[0][0].size, st[0]).reshape(ref[0][0].shape), "bf16")
        assert np.array_equal(got[:2], want[1][:2])
        check_cached(c, [0, 1], want[0], want[1], want[2], want[3], "bf16", 8)
    check(be.L.objeta_hip_graph_destroy(be.ctx, g))


@pytest.mark.parametrize("rows", [1, 12])
def test_cached_offsets_past_32_bits(backend, att, rows):
    """A pool of more than 2^32 elements: the last layer's last pages."""
    layers, pages, heads, page, dim = 2, 33000, 4, 256, 64  # 4.3e9 elements of k and of v
    c = KvCache(backend, layers, pages, heads, page, dim, 1, 4, dtype="bf16")
    rng = np.random.default_rng(14)
    k, v = (to_type(rng.standard_normal((3, heads, page, dim)), "bf16") for _ in range(2))
    size = heads * page * dim * 2
    for d, x in ((c.d_k, k), (c.d_v, v)):
        d.upload(x, offset=(layers * pages - 3) * size)
    table = np.array([pages - 1, pages - 3, pages - 2, -1], np.int32)
    c.d_page_table.upload(table)
    c.d_seq_lens.upload(np.array([600], np.int32))
    q = to_type(rng.standard_normal((rows, 8, dim)), "bf16")
    out = backend.alloc(q.nbytes)
    att.cached_device(c, 1, backend.to_device(np.array([0], np.int32)), backend.to_device(np.array([0, rows], np.int32)), 1, rows,
                      rows, 600, "bf16", backend.to_device(q), out, 8)
    backend.synchronize()
    got, order = download(out, "bf16", q.shape), [2, 0, 1]
    k64, v64 = (from_type(x, "bf16")[order].transpose(1, 0, 2, 3).reshape(heads, -1, dim)[:, :600] for x in (k, v))
    seen = np.ones((rows, 600), bool)
    for i in range(rows):
        seen[i, 600 - rows + i + 1:] = False
    for h in range(8):
        o, _, bound = attend(from_type(q[:, h], "bf16"), k64[h // 2], v64[h // 2], seen, 0.125, "bf16", "bf16")
        assert np.all(np.abs(got[:, h] - o) <= bound)


# ------------------------------------------------------------------ a run of them
def test_generate_with_drafts(backend, att):
    """A prompt, its cache, a fork, a tree of drafts verified, the accepted branch kept, and decode
    from there: the attention of every step equals the plain form over the tokens themselves."""
    be, rng = backend, np.random.default_rng(15)
    nq, nk, dim, page, dt = 4, 2, 64, 16, "f32"
    rope = Rope(dim, theta=10000.0)
    f = frequencies(dim, 10000.0)
    c = KvCache(be, 1, 64, nk, page, dim, 4, 16, dtype="f32")
    ints = lambda v: be.to_device(np.array(v, np.int32).ravel())  # noqa: E731
    kept = {}  # sequence -> rotated keys, values on the host (float64), token by token

    def step(seqs, rows, depth, tree=None):
        """New tokens through extend, append (rotation) and attention; returns nothing, checks all."""
        n = sum(rows)
        q, k, v = (rng.standard_normal((n, h, dim)).astype(np.float32) for h in (nq, nk, nk))
        pos = np.array(sum([[len(kept[s][0]) + x for x in d] for s, d in zip(seqs, depth)], []), np.int32)
        cu = np.concatenate(([0], np.cumsum(rows)))
        d_seqs, d_cu = ints(seqs), ints(cu)
        c.extend_device(d_seqs, ints(rows), len(seqs))
        dq, out = be.to_device(q), be.alloc(q.nbytes)
        c.append_device(0, d_seqs, d_cu, len(seqs), n, dt, be.to_device(k), be.to_device(v), rope=rope, d_positions=ints(pos),
                        d_q=dq, d_q_out=dq, n_q_heads=nq)
        masks = None if tree is None else be.to_device(np.array(tree, np.uint64))
        att.cached_device(c, 0, d_seqs, d_cu, len(seqs), n, max(rows), 256, dt, dq, out, nq, d_tree=masks)
        be.synchronize()
        got = out.download(np.float32, q.size).reshape(q.shape)
        qr, kr = rotate(q.astype(np.float64), pos, f, "half"), rotate(k.astype(np.float64), pos, f, "half")
        for b, s in enumerate(seqs):
            lo, hi = cu[b], cu[b + 1]
            base = len(kept[s][0])
            kept[s] = [np.concatenate((kept[s][0], kr[lo:hi])), np.concatenate((kept[s][1], v[lo:hi].astype(np.float64)))]
            seen = np.ones((hi - lo, base + hi - lo), bool)
            for i in range(hi - lo):
                seen[i, base:] = [j <= i if tree is None else (tree[lo + i] >> j) & 1 for j in range(hi - lo)]
            for h in range(nq):
                o, _, bound = attend(qr[lo:hi, h], kept[s][0][:, h // 2], kept[s][1][:, h // 2], seen, 0.125, dt, dt)
                # q and k are rotated in float: 8 half steps of (|x| + |y|) each, which move a score by
                # at most 2 * 8 * 2 U scale |q| |k| and a result by twice that of its size
                move = 64 * 2.0 ** -24 * 0.125 * np.linalg.norm(qr[lo:hi, h], axis=1).max() * np.linalg.norm(kept[s][0][:, h // 2], axis=1).max()
                assert np.all(np.abs(got[lo:hi, h] - o) <= bound + move * np.abs(kept[s][1][:, h // 2]).max())

    empty = [np.zeros((0, nk, dim)), np.zeros((0, nk, dim))]
    kept = {0: list(empty), 1: list(empty)}
    step([0, 1], [37, 16], [list(range(37)), list(range(16))])            # two prompts
    c.fork_device(ints([0, 1]), ints([2, 3]), 2)
    kept[2], kept[3] = list(kept[0]), list(kept[1])
    step([2, 0, 3, 1], [1, 1, 1, 1], [[0]] * 4)                            # each branch goes its own way
    parents = [-1, 0, 0, 1, 3, 2]                                          # drafts
    masks, depth = [], []
    for i, p in enumerate(parents):
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    step([0, 2], [6, 6], [depth, depth], tree=masks * 2)
    accepted = {0: [0, 2, 5], 2: [0, 1, 3, 4]}
    keep = [accepted[0] + [-1] * 3, accepted[2] + [-1] * 2]
    c.compact_device(ints([0, 2]), ints([6, 6]), ints(keep), ints([3, 4]), 2, 6)
    for s in (0, 2):
        n = len(kept[s][0]) - 6
        at = list(range(n)) + [n + x for x in accepted[s]]
        kept[s] = [x[at] for x in kept[s]]
    c.free_device(ints([3]), 1)
    for _ in range(14):                                                    # over a page's end
        step([2, 1, 0], [1, 1, 1], [[0]] * 3)
    be.synchronize()
    assert c.d_seq_lens.download(np.int32, 4).tolist() == [len(kept[0][0]), len(kept[1][0]), len(kept[2][0]), 0]
    refs = c.d_ref_counts.download(np.int32, 64)
    table = c.d_page_table.download(np.int32, 64).reshape(4, 16)
    assert np.array_equal(np.bincount(table[table >= 0], minlength=64), refs)
