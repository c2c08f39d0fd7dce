"""Attention where 128 rows share the tiles and where keys are cut over workgroups: head sizes, many
entries, cuts that the kernel chooses, prompts in parts, and floats in parts, against the plain form
in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from attn_reference import attend, from_type, lse_bound, to_type
from objeta_amd import AttentionBackend, HipBackend, HipError, KvCache, MoeExecutor
from objeta_amd.api import check
from test_gpu_attention import FILL, PAIRS, TYPES, Cached, check_cached, prompt_case, run_cached, run_prompt, tree_masks

pytestmark = pytest.mark.gpu


@pytest.fixture
def att(backend):
    MoeExecutor(backend).device_error()
    yield AttentionBackend(backend)
    assert MoeExecutor(backend).device_error() == 0


@pytest.mark.parametrize("dtype,kv", PAIRS)
@pytest.mark.parametrize("dim", [8, 72, 80, 96, 104, 128, 136, 192, 200, 256])
def test_cached_many_rows_head_sizes(backend, att, dtype, kv, dim):
    c = Cached(backend, [300, 70, 64, 513], kv, 1, 16, dim, seed=20)
    rows, seqs = [40, 33, 64, 1], [0, 1, 2, 3]
    q, got, lse, cu = run_cached(att, c, seqs, rows, dtype, 2)
    check_cached(c, seqs, q, got, lse, cu, dtype, 2)
    rng = np.random.default_rng(21)
    tree = sum([tree_masks(rng, n) for n in rows], [])
    q, got, lse, cu = run_cached(att, c, seqs, rows, dtype, 2, tree=tree)
    check_cached(c, seqs, q, got, lse, cu, dtype, 2, tree=tree)


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f32", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("batch", [63, 64, 65, 150])
def test_cached_many_entries(backend, dtype, kv, batch):
    """Entries past a wave's lanes, empty and bad ones among them, one sequence named several times."""
    att, err = AttentionBackend(backend), MoeExecutor(backend)
    err.device_error()
    rng = np.random.default_rng(batch)
    c = Cached(backend, [2600] + rng.integers(40, 200, 11).tolist(), kv, 1, 16, 64, seed=22)
    seqs = rng.integers(0, 12, batch).tolist()
    seqs[0], seqs[-1], seqs[batch // 2], seqs[7] = 0, 0, -1, 12
    rows = [int(r) for r in rng.choice([0, 1, 2, 40], batch)]
    rows[0], rows[-1], rows[7], rows[batch // 2], rows[3], rows[-2] = 40, 33, 2, 40, 0, 0
    q, got, lse, cu = run_cached(att, c, seqs, rows, dtype, 1)
    assert err.device_error() == 4
    good = [b for b in range(batch) if 0 <= seqs[b] < 12]
    for b in good:
        check_cached(c, [seqs[b]], q[cu[b]:cu[b + 1]], got[cu[b]:cu[b + 1]], lse[cu[b]:cu[b + 1]], [0, rows[b]], dtype, 1)
    for b in (7, batch // 2):
        assert np.all(np.isnan(got[cu[b]:cu[b + 1]])) and np.all(np.isnan(lse[cu[b]:cu[b + 1]]))


@pytest.mark.parametrize("dtype,kv", PAIRS)
@pytest.mark.parametrize("lens,rows,heads", [
    ([4100, 300, 90, 2000], [50, 3, 64, 33], 1), ([9001], [64], 1), ([9001], [700], 2), ([3000, 64, 1, 2999], [33, 64, 1, 0], 4),
    ([700] * 40, [34] * 40, 1), ([257, 256, 255, 512], [64, 64, 64, 64], 2)])
def test_cached_cuts_that_fill_the_card(backend, att, dtype, kv, lens, rows, heads):
    c = Cached(backend, lens, kv, heads, 16, 64, seed=23)
    seqs = list(range(len(lens)))
    q, got, lse, cu = run_cached(att, c, seqs, rows, dtype, heads)
    check_cached(c, seqs, q, got, lse, cu, dtype, heads)
    again = run_cached(att, c, seqs, rows, dtype, heads, q=q)
    assert np.array_equal(got, again[1]) and np.array_equal(lse, again[2])


@pytest.mark.parametrize("dtype,kv,dim", [(*p, 64) for p in PAIRS] + [("f32", "f32", 128), ("f32", "f32", 256), ("f16", "f16", 256)])
@pytest.mark.parametrize("lens,heads,group", [([767], 1, 4), ([769, 768], 2, 1), ([255, 256, 257], 1, 16), ([127, 128, 129, 385], 1, 1),
                                              ([1023, 1024] * 10, 4, 2), ([1025] * 16 + [3], 4, 1), ([500, 20] * 35, 4, 1),
                                              ([513, 385], 2, 20)])
def test_cached_decode_around_the_cuts(backend, att, dtype, kv, dim, lens, heads, group):
    """One piece or several, workgroups of one or both sizes, 16 or 32 rows a tile."""
    c = Cached(backend, lens, kv, heads, 16, dim, seed=19)
    seqs = list(range(len(lens)))
    q, got, lse, cu = run_cached(att, c, seqs, [1] * len(lens), dtype, heads * group)
    check_cached(c, seqs, q, got, lse, cu, dtype, heads * group)


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("rows", [1, 40])
def test_cached_more_parts_than_lanes(backend, att, dtype, kv, rows):
    c = Cached(backend, [20000, 16640, 16385, 16384, 90], kv, 1, 64, 40, seed=27)
    for seqs in ([0, 1, 2, 3, 4], [2], [3, 4]):
        q, got, lse, cu = run_cached(att, c, seqs, [rows] * len(seqs), dtype, 1)
        check_cached(c, seqs, q, got, lse, cu, dtype, 1)


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("batch,rows", [(130, 1), (300, 2), (70, 16)])
def test_cached_joins_of_many_rows(backend, att, dtype, kv, batch, rows):
    """Few parts of thousands of (row, head)s, which a wave each joins, and entries past the lanes."""
    rng = np.random.default_rng(24)
    c = Cached(backend, rng.integers(700, 1100, 8).tolist(), kv, 1, 16, 64, seed=25)
    seqs = rng.integers(0, 8, batch).tolist()
    nq = 16
    q, got, lse, cu = run_cached(att, c, seqs, [rows] * batch, dtype, nq)
    for b in list(range(0, batch, 17)) + [batch - 1]:
        check_cached(c, [seqs[b]], q[cu[b]:cu[b + 1]], got[cu[b]:cu[b + 1]], lse[cu[b]:cu[b + 1]], [0, rows], dtype, nq)


@pytest.mark.parametrize("rows", [1, 40])
def test_cached_batch_padded_far(backend, att, rows):
    """100 thousand rows of which one entry has a few: the padding is left alone."""
    be, n, nq = backend, 100000, 16
    c = Cached(backend, [3000], "f16", 1, 16, 64, seed=28)
    q = to_type(np.random.default_rng(29).standard_normal((rows, nq, 64)), "f16")
    d_q, out = be.alloc(n * nq * 64 * 2), be.alloc(n * nq * 64 * 2)
    d_q.upload(q)
    edge = np.full((rows + 8, nq, 64), FILL, np.float16)
    out.upload(edge)
    lse = be.to_device(np.full((n, nq), FILL, np.float32))
    att.cached_device(c.cache, 0, be.to_device(np.array([0], np.int32)), be.to_device(np.array([0, rows], np.int32)), 1, n, rows, 3000,
                      "f16", d_q, out, nq, d_lse=lse)
    be.synchronize()
    got = out.download(np.float16, edge.size).reshape(edge.shape).astype(np.float64)
    l = lse.download(np.float32, n * nq).reshape(n, nq)
    check_cached(c, [0], q, got[:rows], l[:rows].astype(np.float64), [0, rows], "f16", nq)
    assert np.all(got[rows:] == FILL) and np.all(l[rows:] == FILL)


def test_cached_replays_choose_their_own_cuts(backend, att):
    """A captured call of many rows on lengths that changed since: each replay as an eager call."""
    be, st = backend, backend.stream(1)
    c = Cached(backend, [3000, 2000], "bf16", 2, 16, 64, seed=26)
    ref = run_cached(att, c, [0, 1], [64, 40], "bf16", 4, stream=st)
    b = [be.to_device(np.array([0, 1], np.int32), st), be.to_device(ref[3], st), be.to_device(ref[0], st), be.alloc(ref[0].nbytes)]
    be.synchronize(st)
    check(be.L.objeta_hip_graph_begin_capture(be.ctx, st))
    att.cached_device(c.cache, 0, b[0], b[1], 2, 106, 64, 3000, "bf16", b[2], b[3], 4, stream=st)
    g = C.c_void_p()
    check(be.L.objeta_hip_graph_end_capture(be.ctx, st, C.byref(g)))
    for lens in ([3000, 2000], [64, 1999], [2999, 40], [3000, 2000]):
        c.lens = lens
        c.upload()
        want = run_cached(att, c, [0, 1], [64, 40], "bf16", 4, stream=st, q=ref[0], max_len=3000)
        check(be.L.objeta_hip_graph_launch(be.ctx, g, st))
        be.synchronize(st)
        got = from_type(b[3].download(np.uint16, ref[0].size, st).reshape(ref[0].shape), "bf16")
        assert np.array_equal(got[:104], want[1][:104])
        check_cached(c, [0, 1], want[0], want[1], want[2], want[3], "bf16", 4)
    check(be.L.objeta_hip_graph_destroy(be.ctx, g))


# ------------------------------------------------------------------- prompts in parts
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,nq,nk,dim", [([1300], 1, 1, 64), ([700, 5, 0, 900], 2, 1, 128), ([1100], 3, 3, 192), ([600, 601], 1, 1, 256),
                                            ([2000], 1, 1, 96), ([40] * 30, 1, 1, 80), ([513], 4, 1, 200)])
def test_prompt_in_parts(backend, att, dtype, causal, lens, nq, nk, dim):
    """Few tiles of rows whose keys are cut over workgroups, rows before and behind left alone."""
    prompt_case(backend, att, dtype, nq, nk, dim, lens, causal, before=3, seed=30)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", [np.inf, np.nan])
def test_prompt_in_parts_unseen_places(backend, att, dtype, what):
    """Later tokens and another sequence of infinities or NaN, in every part of the keys."""
    rng = np.random.default_rng(31)
    lens, dim = [900, 400], 64
    n = sum(lens)
    a = [to_type(rng.standard_normal((n, 1, dim)), dtype) for _ in range(3)]
    good, good_lse, _ = run_prompt(backend, att, *a, lens, dtype, True)
    b = [from_type(x, dtype) for x in a]
    for x in b[1:]:
        x[500:900] = what
        x[905:] = what
    got, lse, _ = run_prompt(backend, att, *(to_type(x, dtype) for x in b), lens, dtype, True)
    rows = list(range(500)) + list(range(900, 905))
    q, k, v = (from_type(x, dtype)[:, 0] for x in a)
    for lo, hi in ((0, 500), (900, 905)):
        out, want, bound = attend(q[lo:hi], k[lo:hi], v[lo:hi], np.tril(np.ones((hi - lo, hi - lo), bool)), 0.125, dtype, dtype)
        assert np.all(np.abs(got[lo:hi, 0] - out) <= bound)
        mag = 0.125 * (np.abs(q[lo:hi]) @ np.abs(k[lo:hi]).T).max()
        assert np.all(np.abs(lse[lo:hi, 0] - want) <= lse_bound(want, dim, mag))
    assert not np.any(np.isfinite(got[[r for r in range(n) if r not in rows]]))
    assert np.all(np.isfinite(good)) and np.all(np.isfinite(good_lse))


def test_prompt_in_parts_replays_from_a_graph(backend, att):
    """Captured with the workspace that an eager call left, replayed on other tokens and other cuts
    of the batch; refused on a stream that has no workspace of that size yet."""
    be, st = backend, backend.stream(0)
    rng = np.random.default_rng(32)
    n, dim = 1200, 64
    q, k, v = (to_type(rng.standard_normal((n, 1, dim)), "f16") for _ in range(3))
    run_prompt(backend, att, q, k, v, [700, 500], "f16", True, stream=st)
    bufs = [be.to_device(x, st) for x in (q, k, v)]
    cu, out = be.to_device(np.array([0, 700, 1200], np.int32), st), be.alloc(q.nbytes)
    be.synchronize(st)
    check(be.L.objeta_hip_graph_begin_capture(be.ctx, st))
    att.prompt_device("f16", *bufs, out, 1, 1, dim, n, cu, 2, stream=st)
    g = C.c_void_p()
    check(be.L.objeta_hip_graph_end_capture(be.ctx, st, C.byref(g)))
    for lens in ([700, 500], [1, 1199], [1100, 100], [700, 500]):
        x = [to_type(rng.standard_normal((n, 1, dim)), "f16") for _ in range(3)]
        for d, h in zip(bufs, x):
            d.upload(h, st)
        cu.upload(np.array([0, lens[0], n], np.int32), st)
        want = run_prompt(backend, att, *x, lens, "f16", True, stream=st)[0]
        check(be.L.objeta_hip_graph_launch(be.ctx, g, st))
        be.synchronize(st)
        assert np.array_equal(from_type(out.download(np.float16, out.nbytes // 2, st).reshape(q.shape), "f16"), want)
    check(be.L.objeta_hip_graph_destroy(be.ctx, g))


def test_prompts_in_parts_on_two_streams(backend, att):
    """Calls in flight on two streams join parts of their own."""
    rng = np.random.default_rng(33)
    n, dim, st = 1500, 64, [backend.stream(0), backend.stream(1)]
    x = [[to_type(rng.standard_normal((n, 1, dim)), "bf16") for _ in range(3)] for _ in range(2)]
    want = [run_prompt(backend, att, *x[i], [n], "bf16", False, stream=st[i])[0] for i in range(2)]
    dev = [[backend.to_device(a, s) for a in y] for y, s in zip(x, st)]
    cu = [backend.to_device(np.array([0, n], np.int32), s) for s in st]
    out = [backend.alloc(n * dim * 2) for _ in st]
    for _ in range(20):
        for i in range(2):
            att.prompt_device("bf16", *dev[i], out[i], 1, 1, dim, n, cu[i], 1, causal=False, stream=st[i])
    for i in range(2):
        backend.synchronize(st[i])
        got = from_type(out[i].download(np.uint16, n * dim, st[i]).reshape(n, 1, dim), "bf16")
        assert np.array_equal(got, want[i])


# ------------------------------------------------------------------- floats in parts
def test_prompt_floats_at_the_limits(backend, att):
    """Keys past bf16's largest value (their first part is infinite), small ones, and values of every
    size: floats in three parts give what floats give."""
    rng = np.random.default_rng(34)
    n, dim = 70, 64
    q, k, v = (rng.standard_normal((n, 1, dim)).astype(np.float32) for _ in range(3))
    k[5, 0, 9], k[33, 0, 2], q[:, 0, 9], q[:, 0, 2] = 3.4e38, -3.4e38, 2e-38, 2e-38
    k[:, 0, 20:30] *= np.float32(1e-25)
    v[:, 0, :8] *= np.float32(1e30)
    v[:, 0, 8:16] *= np.float32(1e-28)
    for at_limit in (True, False):
        if not at_limit:
            k[5, 0, 9], k[33, 0, 2] = 1.0, -1.0
        got, lse, _ = run_prompt(backend, att, q, k, v, [n], "f32", True)
        q64, k64, v64 = (x[:, 0].astype(np.float64) for x in (q, k, v))
        out, want, bound = attend(q64, k64, v64, np.tril(np.ones((n, n), bool)), 0.125, "f32", "f32")
        assert np.all(np.abs(got[:, 0] - out) <= bound)
        mag = 0.125 * (np.abs(q64) @ np.abs(k64).T).max()
        assert np.all(np.abs(lse[:, 0] - want) <= lse_bound(want, dim, mag))
    one = np.full((1, 1, dim), 3.4e38, np.float32)  # a single key: its value itself
    got, _, _ = run_prompt(backend, att, q[:1], k[:1], one, [1], "f32", True)
    assert np.all(np.abs(got - 3.4e38) <= 3.4e38 * 2.0 ** -22)


# ------------------------------------------------------------------- appends of many entries
@pytest.mark.parametrize("batch", [62, 63, 64, 65, 130])
def test_append_many_entries(backend, batch):
    """One token each into as many sequences, two of them named again later: the last entry's row stays."""
    be, rng = backend, np.random.default_rng(batch)
    n_seqs, page, dim = batch, 8, 16
    c = KvCache(be, 1, n_seqs, 2, page, dim, n_seqs, 1, dtype="f32")
    table = rng.permutation(n_seqs).astype(np.int32).reshape(n_seqs, 1)
    lens = rng.integers(1, page + 1, n_seqs).astype(np.int32)
    c.d_page_table.upload(table)
    c.d_seq_lens.upload(lens)
    c.d_ref_counts.upload(np.ones(n_seqs, np.int32))
    pool = np.full((n_seqs, 2, page, dim), FILL, np.float32)
    c.d_k.upload(pool)
    c.d_v.upload(pool)
    seqs = rng.permutation(n_seqs).astype(np.int32)
    seqs[batch - 1], seqs[batch - 2] = seqs[3], seqs[batch - 3]
    k, v = (rng.standard_normal((batch, 2, dim)).astype(np.float32) for _ in range(2))
    c.append_device(0, be.to_device(seqs), be.to_device(np.arange(batch + 1, dtype=np.int32)), batch, batch, "f32", be.to_device(k),
                    be.to_device(v))
    be.synchronize()
    want_k, want_v = pool.copy(), pool.copy()
    for b, s in enumerate(seqs):
        want_k[table[s, 0], :, lens[s] - 1], want_v[table[s, 0], :, lens[s] - 1] = k[b], v[b]
    assert np.array_equal(c.d_k.download(np.float32, pool.size).reshape(pool.shape), want_k)
    assert np.array_equal(c.d_v.download(np.float32, pool.size).reshape(pool.shape), want_v)


def test_capture_without_a_workspace_is_refused():
    """A call that would have to allocate while its stream is captured says so; the capture ends
    cleanly, and the call goes in once an eager one has left the workspace."""
    be = HipBackend(0, 1)
    att, st = AttentionBackend(be), be.stream(0)
    n, dim = 1200, 64
    x = np.random.default_rng(35).standard_normal((n, 1, dim)).astype(np.float32)
    d, cu, out, want = be.to_device(x), be.to_device(np.array([0, n], np.int32)), be.alloc(n * dim * 4), be.alloc(n * dim * 4)

    def call(to):
        att.prompt_device("f32", d, d, d, to, 1, 1, dim, n, cu, 1, stream=st)
    be.synchronize()
    g = C.c_void_p()
    check(be.L.objeta_hip_graph_begin_capture(be.ctx, st))
    with pytest.raises(HipError, match="captur"):
        call(out)
    check(be.L.objeta_hip_graph_end_capture(be.ctx, st, C.byref(g)))
    check(be.L.objeta_hip_graph_destroy(be.ctx, g))
    call(want)
    check(be.L.objeta_hip_graph_begin_capture(be.ctx, st))
    call(out)
    check(be.L.objeta_hip_graph_end_capture(be.ctx, st, C.byref(g)))
    for _ in range(3):
        out.upload(np.zeros((n, dim), np.float32))
        check(be.L.objeta_hip_graph_launch(be.ctx, g, st))
        be.synchronize(st)
        assert np.array_equal(out.download(np.float32, n * dim), want.download(np.float32, n * dim))
    check(be.L.objeta_hip_graph_destroy(be.ctx, g))
