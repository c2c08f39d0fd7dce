"""Attention over queries, keys and values that hold infinities and NaN which rows see, against the
64-bit form with their own arithmetic: a score of NaN or inf makes a row NaN, one of -inf leaves its
key out (times an infinity: NaN), rows of which every score is -inf come out 0; an infinity or NaN
among the values reaches the dimensions that it lies in and no other. And what such calls cost."""
import ctypes as C
import zlib

import numpy as np
import pytest

from attn_reference import attend, from_type, lse_bound, to_type
from objeta_amd import AttentionBackend, MoeExecutor
from objeta_amd.api import check
from test_gpu_attention import PAIRS, TYPES, Cached, run_cached, run_prompt, tree_masks

pytestmark = pytest.mark.gpu


@pytest.fixture
def att(backend):
    MoeExecutor(backend).device_error()
    yield AttentionBackend(backend)
    assert MoeExecutor(backend).device_error() == 0


def check_head(got, lse, q, k, v, seen, scale, dtype, what):
    """One head's rows: q [rows][dim], k, v [keys][dim] in 64 bits."""
    odd_keys, odd_rows = ~np.isfinite(k).all(1), ~np.isfinite(q).all(1)
    with np.errstate(all="ignore"):
        s = scale * (np.where(odd_rows[:, None], 0, q) @ np.where(odd_keys[:, None], 0, k).T)
        for j in np.nonzero(odd_keys)[0]:  # term by term: inf and NaN as they come
            s[:, j] = scale * (q * k[j]).sum(1)
        for i in np.nonzero(odd_rows)[0]:
            s[i] = scale * (q[i] * k).sum(1)
        lost = np.any(seen & (np.isnan(s) | (s == np.inf)), 1)
        counted = seen & (s > -np.inf) & ~lost[:, None]
        none = ~lost & ~counted.any(1)
        # what of each kind a row sees in each dimension; a key left out by its score makes NaN of them
        kinds = [(seen & ~lost[:, None]).astype(np.float64) @ x.astype(np.float64) > 0 for x in (v == np.inf, v == -np.inf, np.isnan(v))]
        out_key = ((seen & (s == -np.inf)).astype(np.float64) @ (~np.isfinite(v)).astype(np.float64)) > 0
    nan = kinds[2] | (kinds[0] & kinds[1]) | out_key | lost[:, None]
    special = np.where(nan, np.nan, np.where(kinds[0], np.inf, np.where(kinds[1], -np.inf, 0.0)))
    k0, v0 = np.where(odd_keys[:, None], 0, k), np.where(np.isfinite(v), v, 0)
    fine = ~lost & ~odd_rows
    assert not np.any(counted[fine][:, odd_keys]), "an infinite key with a finite score"
    out, want_lse, bound = attend(np.where(fine[:, None], q, 0), k0, v0, counted, scale, dtype, dtype)
    plain = ~nan & ~kinds[0] & ~kinds[1]
    here = plain & fine[:, None]
    assert np.all(np.abs(got - out)[here] <= bound[here]), (what, float(np.max((np.abs(got - out) / np.maximum(bound, 1e-300))[here])))
    assert np.array_equal(got[~plain], special[~plain], equal_nan=True), what
    assert np.all(np.isnan(lse[lost])) and np.all(lse[none] == -np.inf), what
    rows = fine & ~none
    mag = scale * (np.abs(np.where(fine[:, None], q, 0)) @ np.abs(k0).T).max()
    assert np.all(np.abs(lse - want_lse)[rows] <= lse_bound(want_lse, q.shape[1], mag)[rows]), what


SPECIALS = [np.inf, -np.inf, np.nan]
WHERE = ["value", "values", "key", "keys away", "query", "all of it"]


def spoil(rng, where, q, k, v, seq):
    """Puts infinities and NaN into q, k, v [tokens][heads][dim] (float64); seq: the tokens they go to."""
    pick = lambda n: rng.choice(seq, min(n, len(seq)), replace=False)  # noqa: E731
    dims = k.shape[2]
    if where in ("value", "all of it"):  # one element
        v[pick(1), rng.integers(v.shape[1]), rng.integers(dims)] = SPECIALS[rng.integers(3)]
    if where in ("values", "all of it"):  # many, each dimension for itself
        for t in pick(12):
            v[t, rng.integers(v.shape[1]), rng.choice(dims, 3, replace=False)] = [SPECIALS[x] for x in rng.integers(0, 3, 3)]
    if where in ("key", "all of it"):  # rows that see it are NaN
        k[pick(1), rng.integers(k.shape[1]), rng.integers(dims)] = np.nan
    if where == "keys away":  # dimension 0 of queries is positive: scores of -inf
        q[..., 0] = np.abs(q[..., 0]) + 0.5
        k[pick(20), :, 0] = -np.inf
        v[pick(2), 0, 1 % dims] = np.inf
    if where in ("query", "all of it"):
        q[pick(1), rng.integers(q.shape[1]), rng.integers(dims)] = SPECIALS[rng.integers(3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", WHERE)
@pytest.mark.parametrize("lens,nq,nk,dim,causal", [([200, 90], 4, 2, 64, True), ([150], 2, 1, 40, False), ([131, 70], 2, 2, 128, True),
                                                   ([129], 3, 1, 192, True), ([100, 30], 1, 1, 256, False), ([1100], 1, 1, 64, True),
                                                   ([700, 600], 1, 1, 128, False)])
def test_prompt_specials(backend, att, dtype, where, lens, nq, nk, dim, causal):
    rng = np.random.default_rng(zlib.crc32(f"{dtype} {where} {lens} {dim}".encode()))
    n = sum(lens)
    q, k, v = (rng.standard_normal((n, h, dim)) for h in (nq, nk, nk))
    spoil(rng, where, q, k, v, np.arange(0, lens[0]))
    a = [to_type(x, dtype) for x in (q, k, v)]
    got, lse, cu = run_prompt(backend, att, *a, lens, dtype, causal)
    q, k, v = (from_type(x, dtype) for x in a)
    for lo, hi in zip(cu[:-1], cu[1:]):
        seen = np.ones((hi - lo, hi - lo), bool)
        seen = np.tril(seen) if causal else seen
        for h in range(nq):
            g = h * nk // nq
            check_head(got[lo:hi, h], lse[lo:hi, h], q[lo:hi, h], k[lo:hi, g], v[lo:hi, g], seen, np.float64(np.float32(dim ** -0.5)), dtype,
                       (lo, h))


@pytest.mark.parametrize("dtype,kv", PAIRS)
@pytest.mark.parametrize("where", WHERE)
@pytest.mark.parametrize("rows,tree,nq,nk,dim,long", [(1, False, 4, 2, 64, 700), (1, False, 8, 1, 128, 150), (1, False, 2, 1, 256, 300),
                                                      (1, False, 2, 2, 64, 5000), (9, True, 3, 1, 64, 200), (12, False, 2, 1, 128, 300),
                                                      (11, True, 2, 1, 256, 150), (50, True, 2, 1, 64, 300), (40, False, 2, 1, 128, 900),
                                                      (64, True, 1, 1, 192, 200), (70, False, 1, 1, 256, 300)])
def test_cached_specials(backend, att, dtype, kv, where, rows, tree, nq, nk, dim, long):
    """The 16-, 32- and 128-row forms, in one piece and cut, causal and by masks."""
    rng = np.random.default_rng(zlib.crc32(f"{dtype} {kv} {where} {rows} {dim} {long}".encode()))
    c = Cached(backend, [long, rows + 30], kv, nk, 16, dim, seed=60)
    n = 2 * rows
    q = rng.standard_normal((n + 2, nq, dim))
    # the first sequence's tokens as they lie in the cache, spoiled there, the last rows among them
    page, row = c.table[0, np.arange(long) // 16], np.arange(long) % 16
    k, v = (from_type(x[0, page, :, row], kv) for x in (c.k, c.v))
    q_all = np.zeros((long, nq, dim))
    q_all[long - rows:] = q[:rows]
    at = np.unique(np.concatenate((rng.integers(0, long, 12), rng.integers(long - rows, long, 12))))
    spoil(rng, where, q_all, k, v, at)
    if where in ("query", "all of it"):  # (of the rows there are)
        q_all[long - 1 - int(rng.integers(rows)), 0, 0] = np.inf
    q[:rows] = q_all[long - rows:]
    if where == "keys away":
        q[..., 0] = np.abs(q[..., 0]) + 0.5
    c.k[0, page, :, row], c.v[0, page, :, row] = to_type(k, kv), to_type(v, kv)
    c.upload()
    masks = sum([tree_masks(rng, rows) for _ in range(2)], []) if tree else None
    q = to_type(q, dtype)
    _, got, lse, cu = run_cached(att, c, [0, 1], [rows, rows], dtype, nq, tree=masks, q=q)
    for b in range(2):
        lo, hi, total = cu[b], cu[b + 1], c.lens[b]
        kb, vb = c.rows_of("k", 0, b), c.rows_of("v", 0, b)
        seen = np.ones((rows, total), bool)
        for i in range(rows):
            seen[i, total - rows:] = [(int(masks[lo + i]) >> j) & 1 if tree else j <= i for j in range(rows)]
        for h in range(nq):
            g = h * nk // nq
            check_head(got[lo:hi, h], lse[lo:hi, h], from_type(q[lo:hi, h], dtype), kb[g], vb[g], seen, np.float64(np.float32(dim ** -0.5)),
                       dtype, (b, h))


@pytest.mark.parametrize("dtype,kv", [("f32", "f32"), ("f32", "bf16")])
def test_cached_large_finite_values(backend, att, dtype, kv):
    """Values near the type's largest: their weighted sums stay finite."""
    c = Cached(backend, [300, 90], kv, 1, 16, 64, seed=61)
    k, v = from_type(c.k, kv), from_type(c.v, kv)
    v[..., 5] = np.where(np.arange(16) % 2 == 0, 3.0e38, -3.0e38)
    k *= 0.01
    c.k, c.v = to_type(k, kv), to_type(v, kv)
    c.upload()
    for rows in (1, 9, 40):
        q, got, lse, cu = run_cached(att, c, [0, 1], [rows, rows], dtype, 1)
        for b in range(2):
            lo, hi, total = cu[b], cu[b + 1], c.lens[b]
            seen = np.tril(np.ones((rows, total), bool), total - rows)
            out, _, bound = attend(from_type(q[lo:hi, 0], dtype), c.rows_of("k", 0, b)[0], c.rows_of("v", 0, b)[0], seen, 0.125, dtype, dtype)
            assert np.all(np.abs(got[lo:hi, 0] - out) <= bound)


@pytest.mark.parametrize("rows", [1, 9, 40])
def test_cached_large_values_of_unlikely_keys(backend, att, rows):
    """A key 2^-100 as likely as the others still counts where its value is 2^126, in a pass that was not
    finite for another dimension's sake."""
    n, dim = 200, 64
    c = Cached(backend, [n], "f32", 1, 16, dim, seed=63)
    at = np.arange(n)
    place = (0, c.table[0, at // 16], slice(None), at % 16)
    k, v = np.zeros((n, 1, dim), np.float32), np.random.default_rng(64).standard_normal((n, 1, dim)).astype(np.float32)
    k[7, 0, 0] = -100 * np.log(2) * 8  # times 1/8 and a query of 1: e^-69.3 = 2^-100
    v[7, 0, 3], v[9, 0, 5] = 2.0 ** 126, np.inf
    c.k[place], c.v[place] = k, v
    c.upload()
    q = np.ones((rows + 2, 1, dim), np.float32)
    _, got, lse, _ = run_cached(att, c, [0], [rows], "f32", 1, q=q)
    for i in range(rows):
        seen = n - rows + i + 1
        s = np.zeros(seen)
        s[7] = 0.125 * float(k[7, 0, 0])
        p = np.exp(s)
        want = (p @ np.where(np.isfinite(v[:seen, 0]), v[:seen, 0], 0).astype(np.float64)) / p.sum()
        # the score's roundings (72 of its 69.3, and its logarithm's) and the sums over up to 200 keys
        size = (p @ np.abs(np.where(np.isfinite(v[:seen, 0]), v[:seen, 0], 0)).astype(np.float64)) / p.sum()
        bound = size * 2.0 ** -24 * (2 * (80 * 70 + 4 * 70 + seen + 16))
        ok = np.arange(dim) != 5
        assert np.all(np.abs(got[i, 0] - want)[ok] <= bound[ok]) and got[i, 0, 5] == np.inf


@pytest.mark.parametrize("dtype,n,dim", [("bf16", 8192, 128), ("f16", 8192, 64), ("f32", 4096, 128), ("f32", 4096, 256)])
@pytest.mark.parametrize("what", ["one value", "all values", "one key"])
def test_specials_cost_a_few_passes(backend, att, dtype, n, dim, what):
    """A long prompt of which every row sees an infinity or NaN takes a small multiple of a finite one's
    time: a second pass over tiles, with marks where values have them. (A row's keys one after the
    other, as a plain loop, are some thousand times as long.)"""
    rng, nq, st = np.random.default_rng(62), 8, backend.stream(0)
    q, k, v = (rng.standard_normal((n, h, dim)) for h in (nq, 2, 2))
    cu, out = backend.to_device(np.array([0, n], np.int32)), backend.alloc(n * nq * dim * 4)
    begin, end = C.c_void_p(), C.c_void_p()
    for e in (begin, end):
        check(backend.L.objeta_hip_event_create(backend.ctx, C.byref(e)))

    def took():
        bufs = [backend.to_device(to_type(x, dtype)) for x in (q, k, v)]
        times = []
        for _ in range(4):
            check(backend.L.objeta_hip_event_record(backend.ctx, begin, st))
            att.prompt_device(dtype, *bufs, out, nq, 2, dim, n, cu, 1, stream=st)
            check(backend.L.objeta_hip_event_record(backend.ctx, end, st))
            ms = C.c_float()
            check(backend.L.objeta_hip_event_elapsed_ms(backend.ctx, begin, end, C.byref(ms)))
            times.append(ms.value)
        return min(times)
    finite = took()
    if what == "one value":
        v[0, :, 0] = np.inf
    elif what == "all values":
        v[:] = np.nan
    else:
        k[0, :, 0] = -np.inf
    odd = took()
    for e in (begin, end):
        check(backend.L.objeta_hip_event_destroy(backend.ctx, e))
    assert odd <= 20 * finite, (finite, odd)
