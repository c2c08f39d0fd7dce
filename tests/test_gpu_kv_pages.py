"""The page operations and the cache writes against the bookkeeping on lists and copies on the
host (attn_reference.Pages): tables, lengths and counts equal, keys and values byte for byte."""
import numpy as np
import pytest

from attn_reference import NP, Pages, from_type, frequencies, rotate, rotate_bound, to_type
from objeta_amd import HipBackend, KvCache, MoeExecutor, Rope
from objeta_amd.api import check

import ctypes as C

pytestmark = pytest.mark.gpu


class Rig:
    """A cache on the device with random contents and its image on the host."""

    def __init__(self, backend, seed, dtype="bf16", layers=2, pages=40, heads=2, page=8, dim=16, seqs=8, max_pages=12):
        self.be, self.rng = backend, np.random.default_rng(seed)
        self.cache = KvCache(backend, layers, pages, heads, page, dim, seqs, max_pages, dtype=dtype)
        shape = (layers, pages, heads, page, dim)
        self.k, self.v = (to_type(self.rng.standard_normal(shape), dtype) for _ in range(2))
        self.cache.d_k.upload(self.k)
        self.cache.d_v.upload(self.v)
        self.m = Pages(seqs, max_pages, pages, page)
        self.err = MoeExecutor(backend)
        self.err.device_error()

    def ints(self, v):
        return self.be.to_device(np.array(v, np.int32).ravel())

    def extend(self, seqs, counts, stream=None):
        for s, old, new, rows in self.m.extend(seqs, counts):
            self.k[:, new, :, :rows], self.v[:, new, :, :rows] = self.k[:, old, :, :rows], self.v[:, old, :, :rows]
        self.cache.extend_device(self.ints(seqs), self.ints(counts), len(seqs), stream)

    def fork(self, src, dst):
        self.m.fork(src, dst)
        self.cache.fork_device(self.ints(src), self.ints(dst), len(src))

    def free(self, seqs):
        self.m.free(seqs)
        self.cache.free_device(self.ints(seqs), len(seqs))

    def compact(self, seqs, drafts, keep, kept, width=None):
        width = max([len(r) for r in keep] + [1]) if width is None else width
        rows = [list(r) + [-1] * (width - len(r)) for r in keep]
        p = self.m.page
        for s, a, b, t in self.m.compact(seqs, drafts, rows, kept):
            for x in (self.k, self.v):
                x[:, t[b // p], :, b % p] = x[:, t[a // p], :, a % p]
        self.cache.compact_device(self.ints(seqs), self.ints(drafts), self.ints(rows), self.ints(kept), len(seqs), width)

    def compare(self, what=""):
        c = self.cache
        t, lens, refs = self.m.arrays()
        self.be.synchronize()
        assert np.array_equal(c.d_page_table.download(np.int32, t.size).reshape(t.shape), t), what
        assert np.array_equal(c.d_seq_lens.download(np.int32, lens.size), lens), what
        assert np.array_equal(c.d_ref_counts.download(np.int32, refs.size), refs), what
        raw = np.uint16 if self.k.dtype.itemsize == 2 else np.uint32
        for d, h in ((c.d_k, self.k), (c.d_v, self.v)):
            assert np.array_equal(d.download(raw, h.size), h.view(raw).ravel()), what
        assert self.err.device_error() == self.m.error, what
        self.m.error = 0


@pytest.mark.parametrize("dtype,page,dim", [("bf16", 8, 8), ("f16", 16, 40), ("f32", 32, 72), ("bf16", 256, 128)])
def test_extend_fork_compact_free(backend, dtype, page, dim):
    r = Rig(backend, 1, dtype=dtype, page=page, dim=dim)
    r.extend([3, 0, 5], [page + 1, 0, 2 * page])
    r.compare("first pages")
    r.fork([3, 3, 5], [1, 2, 7])
    r.compare("fork")
    r.extend([3, 1, 2], [1, page, 1])  # the last holder keeps the page, the others copy it
    r.compare("copy on write")
    r.compact([1, 2], [page, 1], [[0, page - 1] if page > 2 else [0], []], [2, 0])
    r.compare("compact")
    r.fork([1, 3], [3, 1])  # two sequences change places
    r.compare("exchange")
    r.free([3, 7, 0])
    r.compare("free")
    r.extend([4], [3])
    r.compare("pages come back, lowest first")


@pytest.mark.parametrize("seed", range(6))
def test_random_operations(backend, seed):
    r = Rig(backend, seed + 10, pages=45, seqs=10, max_pages=9)
    rng, page = r.rng, r.m.page
    for step in range(40):
        n = int(rng.integers(1, 6))
        op = rng.integers(0, 4)
        seqs = [int(x) for x in rng.integers(-1, 11, n)]  # out of range and repeated ones among them
        if op == 0:
            r.extend(seqs, [int(x) for x in rng.integers(-1, 3 * page, n)])
        elif op == 1:
            r.fork(seqs, [int(x) for x in rng.integers(-1, 11, n)])
        elif op == 2:
            drafts = [int(rng.integers(0, r.m.lens[s] + 2)) if r.m.ok(s) else 3 for s in seqs]
            keep, kept = [], []
            for d in drafts:
                k = int(rng.integers(0, min(max(d, 0), 20) + 1))
                row = sorted(rng.choice(max(d, 1), k, replace=False).tolist()) if k else []
                if k > 1 and rng.random() < 0.1:
                    row[0] = row[1]
                keep.append(row)
                kept.append(len(row))
            r.compact(seqs, drafts, keep, kept)
        else:
            r.free(seqs[:2])
        r.compare(f"step {step} op {op} {seqs}")


def test_no_pages_left(backend):
    r = Rig(backend, 3, pages=10, max_pages=12, page=8)
    r.extend([0, 1, 2, 3], [40, 30, 24, 1])  # 5 + 4 pages fit, 3 do not, nor does what comes behind
    r.compare()
    assert r.m.lens == [40, 30, 0, 0, 0, 0, 0, 0]
    r.extend([2, 3], [8, 0])
    r.compare("the last page, and an entry without a need")
    r.extend([3, 0], [0, 8])
    r.compare()


def test_longest_sequence_and_lists(backend):
    r = Rig(backend, 4, pages=1500, seqs=1100, max_pages=3, layers=1, heads=1)
    seqs = [int(x) for x in r.rng.permutation(1024)]
    r.extend(seqs, [int(x) for x in r.rng.integers(0, 12, 1024)])
    r.compare("1024 entries")
    r.extend([5, 6], [24 - r.m.lens[5], 25 - r.m.lens[6]])  # full to the last slot; one more is refused
    r.compare("the last slot")
    r.fork(list(range(512)), list(range(512, 1024)))
    r.compare("512 forks")
    r.extend(seqs, [1] * 1024)
    r.compare("512 copies at once")
    r.compact(seqs, [1] * 1024, [[0] if s % 2 else [] for s in seqs], [s % 2 for s in seqs])
    r.compare("compact all")
    r.free(seqs)
    r.compare("free all")


def test_many_pages(backend):
    """Free pages are found in order across every wave's part of a large table."""
    r = Rig(backend, 5, pages=70001, seqs=4, max_pages=20000, layers=1, heads=1, page=8, dim=8)
    r.extend([0, 1], [8 * 9999 + 1, 8 * 20000])
    r.extend([2], [8 * 20000])
    r.compare("three")
    r.free([1])
    r.extend([3, 0], [8 * 19990 + 3, 9])
    r.compare("into the gap")


def test_compact_boundaries(backend):
    r = Rig(backend, 6, pages=60, page=8, max_pages=14)
    r.extend([0, 1, 2, 3], [101, 64, 70, 5])
    keep64 = sorted(r.rng.choice(100, 64, replace=False).tolist())
    r.compact([0, 1, 2, 3], [100, 64, 1, 5], [keep64, list(range(64)), [0], []], [64, 64, 1, 0], width=64)
    r.compare("64 kept; all kept; none")
    r.compact([1, 2], [64, 30], [[], []], [0, 0], width=1)
    r.compare("taken back")
    r.fork([0], [4])
    r.compact([0, 4], [10, 10], [[3], [0]], [1, 1])  # one would write into a shared page, the other only cuts
    r.compare("shared pages")
    r.cache.compact_device(r.ints([2]), r.ints([2]), None, r.ints([0]), 1, 0)  # no list at all
    r.m.compact([2], [2], [[]], [0])
    r.compare("cut without a list")


def test_page_operations_replay_from_a_graph(backend):
    r = Rig(backend, 7)
    st = backend.stream(0)
    r.extend([0, 1], [13, 5])
    r.fork([0], [2])
    r.compare()
    seqs, counts, src, dst = r.ints([0, 2]), r.ints([1, 2]), r.ints([0]), r.ints([2])
    keep, drafts, kept = r.ints([[1], [1]]), r.ints([2, 2]), r.ints([1, 1])
    check(backend.L.objeta_hip_graph_begin_capture(backend.ctx, st))
    r.cache.free_device(dst, 1, st)
    r.cache.fork_device(src, dst, 1, st)
    r.cache.extend_device(seqs, counts, 2, st)
    r.cache.compact_device(seqs, drafts, keep, kept, 2, 1, st)
    g = C.c_void_p()
    check(backend.L.objeta_hip_graph_end_capture(backend.ctx, st, C.byref(g)))
    p = r.m.page
    for rep in range(4):
        check(backend.L.objeta_hip_graph_launch(backend.ctx, g, st))
        r.m.free([2])
        r.m.fork([0], [2])
        for s, old, new, rows in r.m.extend([0, 2], [1, 2]):
            r.k[:, new, :, :rows], r.v[:, new, :, :rows] = r.k[:, old, :, :rows], r.v[:, old, :, :rows]
        for s, a, b, t in r.m.compact([0, 2], [2, 2], [[1], [1]], [1, 1]):
            for x in (r.k, r.v):
                x[:, t[b // p], :, b % p] = x[:, t[a // p], :, a % p]
        r.compare(f"replay {rep}")
        r.extend([1], [3])  # an eager call on the same workspace between the replays
        r.compare()
    check(backend.L.objeta_hip_graph_destroy(backend.ctx, g))


# ---------------------------------------------------------------------- append
@pytest.mark.parametrize("src,dst", [("f32", "bf16"), ("f32", "f16"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("layout,rotary,dim", [("half", 16, 16), ("interleaved", 24, 40), ("half", 6, 72), ("interleaved", 2, 128)])
def test_append(backend, src, dst, layout, rotary, dim):
    r = Rig(backend, 8, dtype=dst, dim=dim, heads=3, page=8)
    r.extend([4, 2, 7, 1], [9, 5, 1, 20])
    rows, seqs = [3, 5, 1, 0, 17], [4, 2, 7, 0, 1]
    cu = np.concatenate(([2], 2 + np.cumsum(rows)))  # the first two rows belong to nobody, nor do the last three
    n, nq = int(cu[-1]) + 3, 5
    k, v, q = (to_type(r.rng.standard_normal((n, h, dim)), src) for h in (3, 3, nq))
    pos = r.rng.integers(-5, 1 << 20, n).astype(np.int32)
    rope = Rope(rotary, theta=10000.0, layout=layout)
    be = backend
    d = [be.to_device(x) for x in (k, v, q, pos)]
    d_qo = be.to_device(np.zeros((n, nq, dim), NP[src]))
    r.cache.append_device(1, r.ints(seqs), r.ints(cu), 5, n, src, d[0], d[1], rope=rope, d_positions=d[3], d_q=d[2],
                          d_q_out=d_qo, n_q_heads=nq)
    be.synchronize()
    f = frequencies(rotary, 10000.0)
    k64, v64, q64 = (from_type(x, src) for x in (k, v, q))
    want_k, want_q = rotate(k64, pos, f, layout), rotate(q64, pos, f, layout)
    got_q = from_type(d_qo.download(NP[src], q.size).reshape(q.shape), src)
    assert np.all(np.abs(got_q - want_q) <= rotate_bound(q64, rotary, layout, src, 1.0, want_q))
    shape = r.k.shape
    got_k, got_v = (x.download(NP[dst], r.k.size).reshape(shape) for x in (r.cache.d_k, r.cache.d_v))
    bound = rotate_bound(k64, rotary, layout, dst, 1.0, want_k)
    vt = to_type(v64, dst)
    for b, s in enumerate(seqs):
        for row in range(cu[b], cu[b + 1]):
            slot = r.m.lens[s] - (cu[b + 1] - row)
            page, at = r.m.tables[s][slot // 8], slot % 8
            assert np.all(np.abs(from_type(got_k[1, page, :, at], dst) - want_k[row]) <= bound[row])
            assert np.array_equal(got_v[1, page, :, at], vt[row])
            r.k[1, page, :, at], r.v[1, page, :, at] = got_k[1, page, :, at], got_v[1, page, :, at]
    r.compare("nothing else is written")


def test_append_without_rotation_or_queries(backend):
    r = Rig(backend, 9, dtype="f16", dim=24)
    r.extend([0], [11])
    k, v = (r.rng.standard_normal((11, 2, 24)).astype(np.float32) for _ in range(2))
    r.cache.append_device(0, r.ints([0]), r.ints([0, 11]), 1, 11, "f32", backend.to_device(k), backend.to_device(v))
    for j in range(11):
        page = r.m.tables[0][j // 8]
        r.k[0, page, :, j % 8], r.v[0, page, :, j % 8] = k[j].astype(np.float16), v[j].astype(np.float16)
    r.compare()


def test_append_bad_indices_and_repeats(backend):
    """A sequence named twice takes its last entry's rows; sequences that are none, rows that no
    slot is left for, and tables with bad pages write nothing and are reported."""
    r = Rig(backend, 11, dtype="f32", dim=8, heads=1, layers=1)
    r.extend([0, 1, 2], [6, 2, 9])
    table, lens, refs = r.m.arrays()
    k = r.rng.standard_normal((12, 1, 8)).astype(np.float32)
    v = r.rng.standard_normal((12, 1, 8)).astype(np.float32)
    dk, dv = backend.to_device(k), backend.to_device(v)

    def append(seqs, cu):
        r.cache.append_device(0, r.ints(seqs), r.ints(cu), len(seqs), 12, "f32", dk, dv)

    append([0, 1, 0], [0, 4, 6, 9])
    for row, slot in ((6, 3), (7, 4), (8, 5)):
        r.k[0, table[0, 0], 0, slot], r.v[0, table[0, 0], 0, slot] = k[row, 0], v[row, 0]
    for row, slot in ((4, 0), (5, 1)):
        r.k[0, table[1, 0], 0, slot], r.v[0, table[1, 0], 0, slot] = k[row, 0], v[row, 0]
    r.compare("repeat")
    append([8, -1, 3], [0, 1, 2, 3])  # out of range; a sequence without tokens
    r.m.error = 4
    r.compare("sequences")
    append([1], [0, 3])  # three rows, two slots: the first has none
    for row, slot in ((1, 0), (2, 1)):
        r.k[0, table[1, 0], 0, slot], r.v[0, table[1, 0], 0, slot] = k[row, 0], v[row, 0]
    r.m.error = 4
    r.compare("too many rows")
    append([1], [5, 3])  # indices out of order name no row
    append([1], [20, 30])
    r.compare("cu")
    bad = table.copy()
    bad[2, 1] = 40  # one past the pool
    r.cache.d_page_table.upload(bad)
    append([2], [0, 2])  # slots 7 (first page) and 8 (the bad one)
    r.k[0, table[2, 0], 0, 7], r.v[0, table[2, 0], 0, 7] = k[0, 0], v[0, 0]
    r.cache.d_page_table.upload(table)
    r.m.error = 4
    r.compare("pages")


@pytest.mark.parametrize("max_pages", [2730, 2731, 8192, 8193])
def test_fork_of_long_tables(backend, max_pages):
    """Around the size up to which one workgroup holds all tables: shared, exchanged, onto one that
    held pages of its own, an entry refused among them."""
    r = Rig(backend, 7, pages=14000, page=8, seqs=6, max_pages=max_pages, layers=1, heads=1, dim=8)
    r.extend([0, 1, 2], [8 * 2700 + 3, 8 * 2000, 17])
    r.fork([0, 1, 2], [3, 4, 1])
    r.compare("three")
    r.fork([0, 3, 9], [1, 0, 2])
    r.compare("onto pages of its own, back, and a bad one")
    r.fork([1, 4, 0], [4, 1, 4])
    r.compare("exchange, and one destination twice")
    r.fork([2], [2])
    r.compare("itself")
