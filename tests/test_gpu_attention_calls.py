"""Calls of rotary positions, appends and attention at the edges of what they take: strides of one
row, batches with empty entries, batches without entries, more workgroups than one launch holds, and
row indices out of order."""
import numpy as np
import pytest

from attn_reference import attend, download, frequencies, from_type, lse_bound, rotate, rotate_bound, to_type
from objeta_amd import AttentionBackend, KvCache, MoeExecutor, Rope
from test_gpu_attention import FILL, TYPES, Cached, check_cached, run_cached

pytestmark = pytest.mark.gpu


@pytest.fixture
def att(backend):
    MoeExecutor(backend).device_error()
    yield AttentionBackend(backend)
    assert MoeExecutor(backend).device_error() == 0


def ints(be, v):
    return be.to_device(np.array(v, np.int32).ravel())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 200, 256])
@pytest.mark.parametrize("q_stride,k_stride,v_stride,out_stride", [(0, 0, 0, 0), (8, 8, 4, 12), (1, 2, 24, 7), (1 << 22, 1 << 22, 1 << 23, 5),
                                                                   (9, (1 << 23) + 8, 1 << 24, 1 << 30)])
def test_prompt_of_one_token_has_no_strides(backend, att, dtype, dim, q_stride, k_stride, v_stride, out_stride):
    """There is no second row for a stride to lead to."""
    rng, nq, nk = np.random.default_rng(40), 4, 2
    q, k, v = (to_type(rng.standard_normal((1, h, dim)), dtype) for h in (nq, nk, nk))
    out = backend.to_device(to_type(np.full(q.shape, FILL), dtype))
    lse = backend.to_device(np.full((1, nq), FILL, np.float32))
    att.prompt_device(dtype, *(backend.to_device(x) for x in (q, k, v)), out, nq, nk, dim, 1, ints(backend, [0, 1]), 1, d_lse=lse,
                      q_stride=q_stride, k_stride=k_stride, v_stride=v_stride, out_stride=out_stride)
    backend.synchronize()
    got, got_lse = download(out, dtype, q.shape), lse.download(np.float32, nq)
    scale = np.float64(np.float32(dim ** -0.5))
    for h in range(nq):
        q64, k64, v64 = (from_type(x, dtype) for x in (q[:, h], k[:, h // 2], v[:, h // 2]))
        want, want_lse, bound = attend(q64, k64, v64, np.ones((1, 1), bool), scale, dtype, dtype)
        assert np.all(np.abs(got[:, h] - want) <= bound)
        assert abs(got_lse[h] - want_lse[0]) <= lse_bound(want_lse, dim, scale * (np.abs(q64) @ np.abs(k64).T).max())[0]


@pytest.mark.parametrize("batch", [2, 5, 62, 63, 64, 65, 130])
@pytest.mark.parametrize("dim", [16, 40])
def test_append_with_empty_entries_of_named_sequences(backend, att, batch, dim):
    """Entries without rows write nothing, so they take nothing from an entry ahead that names their
    sequence: a batch padded to a fixed count, and one that repeats a sequence with rows and without."""
    be, rng = backend, np.random.default_rng(batch)
    page, used = 8, (batch + 1) // 2
    c = KvCache(be, 1, used, 2, page, dim, used, 1, dtype="f32")
    table = rng.permutation(used).astype(np.int32).reshape(used, 1)
    lens = rng.integers(2, page + 1, used).astype(np.int32)
    pool = np.full((used, 2, page, dim), FILL, np.float32)
    for d, x in ((c.d_page_table, table), (c.d_seq_lens, lens), (c.d_ref_counts, np.ones(used, np.int32)), (c.d_k, pool), (c.d_v, pool)):
        d.upload(x)
    again = batch - used  # empty entries: of every sequence in turn, the first one's among them
    for seqs, rows in ((list(range(used)) + list(range(again)), [1] * used + [0] * again),
                       (list(range(used)) + [0] * again, [2] * used + [0] * again),
                       ([0] + list(range(1, used)) + [0] + [0] * (again - 1), [2] * used + [1] + [0] * (again - 1))):
        n, cu = sum(rows), np.concatenate(([0], np.cumsum(rows)))
        k, v = (rng.standard_normal((n, 2, dim)).astype(np.float32) for _ in range(2))
        c.d_k.upload(pool)
        c.d_v.upload(pool)
        c.append_device(0, ints(be, seqs), ints(be, cu), batch, n, "f32", be.to_device(k), be.to_device(v))
        be.synchronize()
        want_k, want_v = pool.copy(), pool.copy()
        last = {s: b for b, s in enumerate(seqs) if rows[b]}  # the last entry with rows
        for s, b in last.items():
            for i in range(rows[b]):
                at = lens[s] - rows[b] + i
                want_k[table[s, 0], :, at], want_v[table[s, 0], :, at] = k[cu[b] + i], v[cu[b] + i]
        assert np.array_equal(c.d_k.download(np.float32, pool.size).reshape(pool.shape), want_k)
        assert np.array_equal(c.d_v.download(np.float32, pool.size).reshape(pool.shape), want_v)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rotated", [True, False])
def test_append_of_no_entries_rotates_queries(backend, att, dtype, rotated):
    """Queries of every row are written, also where no entry names any."""
    rng, n, nq, dim = np.random.default_rng(41), 5, 3, 32
    c = KvCache(backend, 1, 2, 1, 8, dim, 1, 2, dtype="f16")
    pool = rng.standard_normal((2, 8, dim)).astype(np.float16)
    c.d_k.upload(pool)
    c.d_v.upload(pool)
    q, k = (to_type(rng.standard_normal((n, h, dim)), dtype) for h in (nq, 1))
    pos = np.arange(n, dtype=np.int32) + 900
    out, d_k = backend.to_device(to_type(np.full(q.shape, FILL), dtype)), backend.to_device(k)
    c.append_device(0, None, None, 0, n, dtype, d_k, d_k, rope=Rope(dim) if rotated else None, d_positions=ints(backend, pos),
                    d_q=backend.to_device(q), d_q_out=out, n_q_heads=nq)
    backend.synchronize()
    q64 = from_type(q, dtype)
    want = rotate(q64, pos, frequencies(dim, 10000.0), "half") if rotated else q64
    bound = rotate_bound(q64, dim, "half", dtype, 1.0, want) + 905 * 3e-15 * 10 if rotated else 0
    assert np.all(np.abs(download(out, dtype, q.shape) - want) <= bound)
    for d in (c.d_k, c.d_v):
        assert np.array_equal(d.download(np.float16, pool.size).reshape(pool.shape), pool)


@pytest.mark.parametrize("rows,long", [(40, False), (40, True), (2, False), (2, True)])
@pytest.mark.parametrize("at,value", [(0, -1), (1, 1 << 20), (63, 1 << 20), (64, -4), (65, 1 << 30), (100, 1 << 20), (129, -1), (130, 1 << 20)])
def test_cached_bad_row_indices_anywhere_are_reported(backend, rows, long, at, value):
    """A row index out of range, in any place of a batch past a wave's lanes, sets the bit; the entries
    ahead of it are computed."""
    att, err = AttentionBackend(backend), MoeExecutor(backend)
    err.device_error()
    c = Cached(backend, [3000 if long else 90, 60], "f16", 1, 16, 64, seed=42)
    seqs = [b % 2 for b in range(130)]
    cu = np.arange(131) * rows
    n = int(cu[-1])
    q = to_type(np.random.default_rng(43).standard_normal((n, 1, 64)), "f16")
    bad = cu.copy()
    bad[at] = value
    out = backend.to_device(np.full(q.shape, FILL, np.float16))
    lse = backend.to_device(np.full((n, 1), FILL, np.float32))
    att.cached_device(c.cache, 0, ints(backend, seqs), ints(backend, bad), 130, n, rows, max(c.lens), "f16", backend.to_device(q), out,
                      1, d_lse=lse)
    backend.synchronize()
    assert err.device_error() == 4
    if value >= 0:  # (starts below all rows move the ones behind up by one entry)
        got, l = download(out, "f16", q.shape), lse.download(np.float32, n).reshape(n, 1).astype(np.float64)
        for b in {0, at // 2, at - 2} & set(range(max(at - 1, 0))):
            lo, hi = cu[b], cu[b + 1]
            check_cached(c, [seqs[b]], q[lo:hi], got[lo:hi], l[lo:hi], [0, rows], "f16", 1)


def sequence_of(cu, i):
    """The sequence that holds token i: the first, by bisection, whose end is past it."""
    lo, hi = 0, len(cu) - 1
    while lo < hi:
        mid = (lo + hi) // 2
        if cu[mid + 1] <= i:
            lo = mid + 1
        else:
            hi = mid
    return lo if lo < len(cu) - 1 and cu[lo] <= i < cu[lo + 1] else None


@pytest.mark.parametrize("n,heads,dim", [(6000, 1, 64), (40, 1, 64)])  # in parts, and whole
@pytest.mark.parametrize("cu", [[1, 0, 1, 0, 6001], [-2, 0, -1, 0, 39], [5, 2, 30, 10, 38], [0, 30, 10, 20, 35],
                                [0, 7, 3, 1, 20, 2, 30, 33, 12], [9, 1, 5, 2, 7], [0, 5, -3, 10, 20, 30], [2, 1] * 40 + [0, 33],
                                [0, 39] + [12] * 70 + [30, 8] * 3])
def test_prompt_indices_out_of_order(backend, n, heads, dim, cu):
    """Rows that belong to no sequence are left as they were, whether the keys are cut over workgroups
    or not, and whatever an earlier call left behind."""
    att, err = AttentionBackend(backend), MoeExecutor(backend)
    rng = np.random.default_rng(44)
    q = to_type(rng.standard_normal((n, heads, dim)), "bf16")
    d = backend.to_device(q)

    def call(cu):
        out = backend.to_device(to_type(np.full(q.shape, FILL), "bf16"))
        lse = backend.to_device(np.full((n, heads), FILL, np.float32))
        att.prompt_device("bf16", d, d, d, out, heads, heads, dim, n, ints(backend, cu), len(cu) - 1, causal=False, d_lse=lse)
        backend.synchronize()
        return download(out, "bf16", q.shape), lse.download(np.float32, n * heads)
    call(np.linspace(0, n, 5).astype(int))
    err.device_error()
    got, lse = call(cu)
    of = [sequence_of(cu, i) for i in range(n)]
    real = [i for i in range(n) if of[i] is not None and cu[of[i]] >= 0 and cu[of[i] + 1] <= n]
    touched = [i for i in range(n) if not np.all(got[i] == FILL)]
    assert touched == real and [i for i in range(n) if lse[i] != FILL] == real
    assert err.device_error() == (4 if any(of[i] is not None for i in set(range(n)) - set(real)) else 0)
    x = from_type(q, "bf16")[:, 0]
    for s in sorted({of[i] for i in real}):
        lo, hi = cu[s], cu[s + 1]
        mine = [i for i in real if of[i] == s]
        want, _, bound = attend(x[mine], x[lo:hi], x[lo:hi], np.ones((len(mine), hi - lo), bool), 0.125, "bf16", "bf16")
        assert np.all(np.abs(got[mine, 0] - want) <= bound)


MANY = (1 << 24) + 5  # tokens: a workgroup of 256 threads each is past 2^32 threads


def places_of(n):
    """Rows at the ends and around where a launch may end."""
    at = {0, 1, n - 1, n - 2, n // 2}
    for p in (1 << 20, 1 << 22, 1 << 23, 1 << 24):
        at |= {p - 1, p, p + 1}
    return sorted(x for x in at if 0 <= x < n)


def test_rope_of_more_tokens_than_a_launch_holds(backend, att):
    rng, dim = np.random.default_rng(45), 8
    x = np.resize(rng.standard_normal((4099, dim)).astype(np.float16), (MANY, dim))
    pos = np.arange(MANY, dtype=np.int32)
    d = backend.to_device(x)
    att.rope_device(Rope(dim), backend.to_device(pos), MANY, dim, d, d, 1, dtype="f16")
    backend.synchronize()
    at = places_of(MANY)
    got = np.stack([d.download(np.float16, dim, offset=p * dim * 2) for p in at]).astype(np.float64)[:, None]
    x64 = x[at].astype(np.float64)[:, None]
    want = rotate(x64, pos[at], frequencies(dim, 10000.0), "half")
    assert np.all(np.abs(got - want) <= rotate_bound(x64, dim, "half", "f16", 1.0, want) + MANY * 3e-15 * 10)


def test_append_of_more_tokens_than_a_launch_holds(backend, att):
    rng, dim, page = np.random.default_rng(46), 8, 256
    x = np.resize(rng.standard_normal((4099, 1, dim)).astype(np.float16), (MANY, 1, dim))
    n_pages = -(-MANY // page)
    c = KvCache(backend, 1, n_pages + 1, 1, page, dim, 2, n_pages, dtype="f16")
    c.d_page_table.upload(np.arange(n_pages + 1, dtype=np.int32))  # the second sequence's one page behind the first's
    c.d_seq_lens.upload(np.array([MANY - 3, 2], np.int32))
    d = backend.to_device(x)
    c.append_device(0, ints(backend, [0, 1]), ints(backend, [0, MANY - 3, MANY - 1]), 2, MANY, "f16", d, d)  # the last row is nobody's
    backend.synchronize()
    for p in (p for p in places_of(MANY) if p < MANY - 1):
        slot = p if p < MANY - 3 else n_pages * page + p - (MANY - 3)
        for pool in (c.d_k, c.d_v):
            assert np.array_equal(pool.download(np.float16, dim, offset=slot * dim * 2), x[p, 0]), p


@pytest.mark.parametrize("rows", [1, 40])
def test_cached_more_workgroups_than_a_launch_holds(backend, att, rows):
    """65535 entries over 300 key/value heads, nearly all of them empty."""
    batch, heads, dim = 65535, 300, 8
    c = Cached(backend, [50, 41], "f16", heads, 8, dim, seed=47)
    seqs = np.zeros(batch, np.int32)
    counts = np.zeros(batch, np.int64)
    seqs[-1], seqs[70] = 1, 1
    counts[0], counts[70], counts[-1] = rows, 1, rows
    cu = np.concatenate(([0], np.cumsum(counts)))
    n = int(cu[-1])
    q = to_type(np.random.default_rng(48).standard_normal((n, heads, dim)), "f16")
    out = backend.to_device(np.full(q.shape, FILL, np.float16))
    lse = backend.to_device(np.full((n, heads), FILL, np.float32))
    att.cached_device(c.cache, 0, backend.to_device(seqs), ints(backend, cu), batch, n, rows, 50, "f16", backend.to_device(q), out, heads,
                      d_lse=lse)
    backend.synchronize()
    got, l = download(out, "f16", q.shape), lse.download(np.float32, n * heads).reshape(n, heads).astype(np.float64)
    for b in (0, 70, batch - 1):
        lo, hi = cu[b], cu[b + 1]
        check_cached(c, [seqs[b]], q[lo:hi], got[lo:hi], l[lo:hi], [0, hi - lo], "f16", heads)


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("batch", [24, 90])
def test_cached_chunk_beside_decode(backend, att, dtype, kv, batch):
    """One chunk of a prompt and single tokens of other sequences, some of them long, in one call."""
    rng = np.random.default_rng(batch)
    lens = [2300, 9000, 6100] + rng.integers(1, 700, 9).tolist()
    c = Cached(backend, lens, kv, 1, 16, 64, seed=49)
    seqs = [0] + [1 + b % 11 for b in range(batch - 1)]
    rows = [1000] + [1] * (batch - 1)
    q, got, lse, cu = run_cached(att, c, seqs, rows, dtype, 2)
    check_cached(c, seqs[:14] + seqs[-3:], np.concatenate([q[:1013], q[cu[-4]:cu[-1]]]), np.concatenate([got[:1013], got[cu[-4]:cu[-1]]]),
                 np.concatenate([lse[:1013], lse[cu[-4]:cu[-1]]]), list(cu[:15]) + [1014, 1015, 1016], dtype, 2)


def test_cached_many_entries_and_padding(backend, att):
    """A million rows of room, of which few entries of many have some: no more workgroups are asked
    for than there can be work for."""
    batch, heads, dim, n = 2048, 128, 8, 1 << 20
    c = Cached(backend, [300, 41], "f16", heads, 8, dim, seed=50)
    seqs, counts = np.zeros(batch, np.int32), np.zeros(batch, np.int64)
    seqs[70], counts[0], counts[70], counts[-1] = 1, 40, 35, 200
    cu = np.concatenate(([0], np.cumsum(counts)))
    used = int(cu[-1])
    q = to_type(np.random.default_rng(51).standard_normal((used, heads, dim)), "f16")
    d_q, out = backend.alloc(n * heads * dim * 2), backend.alloc(n * heads * dim * 2)
    edge = np.full((used + 8, heads, dim), FILL, np.float16)
    d_q.upload(q)
    out.upload(edge)
    lse = backend.to_device(np.full((n, heads), FILL, np.float32))
    att.cached_device(c.cache, 0, backend.to_device(seqs), ints(backend, cu), batch, n, n, 300, "f16", d_q, out, heads, d_lse=lse)
    backend.synchronize()
    got = from_type(out.download(np.float16, edge.size).reshape(edge.shape), "f16")
    l = lse.download(np.float32, n * heads).reshape(n, heads)
    for b in (0, 70, batch - 1):
        lo, hi = cu[b], cu[b + 1]
        check_cached(c, [seqs[b]], q[lo:hi], got[lo:hi], l[lo:hi].astype(np.float64), [0, hi - lo], "f16", heads)
    assert np.all(got[used:] == FILL) and np.all(l[used:] == FILL)
