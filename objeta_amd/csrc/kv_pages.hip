// kv_pages.hip — the page operations of the key/value cache, on the device without a host
// round trip: extend (with copy on write), fork, compact, free.
//
// The bookkeeping is integers in small tables: bound by launches and dependent reads, not by
// bytes. Every result is a function of the tables alone: a page is free when its count is 0,
// and free pages are taken in index order, so no list's history matters; counts change by
// integer atomics, whose order does not either. What moves keys and values (the rows of a
// copied page, accepted drafts) is bound by HBM, one launch for all layers.
#include "kernels.hpp"
#include "kv_common.hpp"

namespace objeta {
namespace dev {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef int32_t i4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kExtThreads = 1024;

// One copy of extend: the first `rows` rows of page `from` to page `to`.
struct PageCopy {
    int32_t from, to, rows, pad;
};

// Sum over the threads below this one, and the total; 1024 threads, `sh` of 17 words.
__device__ __forceinline__ uint64_t scan_1024(uint64_t v, uint64_t* sh, uint64_t& total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(s, d, 64);
        if (lane >= static_cast<uint32_t>(d)) s += o;
    }
    __syncthreads();  // sh may still be read from a scan before
    if (lane == 63) sh[wave] = s;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
    for (uint32_t w = 0; w < kExtThreads / 64; ++w) {
        if (w < wave) before += sh[w];
        total += sh[w];
    }
    return before + s - v;
}

// extend's bookkeeping in one workgroup, a thread an entry:
//   1. what each entry needs (copy on write included), summed over the entries before it;
//   2. the free pages in index order, counted by waves that each own a part of the counts;
//   3. table entries, counts and lengths of the entries that the free pages cover: the thread
//      that finds the f'th free page finds the entry that takes it.
// Bound by dependent reads: sequence, length, last page and its count, each some 0.7 us away.
// The counts of the first kHeld * 1024 pages are read beside them and held as masks; only
// larger pools are read twice.
__global__ __launch_bounds__(kExtThreads) void kv_extend_kernel(KvView kv, const int32_t* __restrict__ seqs,
                                                                const int32_t* __restrict__ counts, uint32_t n,
                                                                PageCopy* __restrict__ copies,
                                                                uint32_t* __restrict__ n_copies, uint32_t* err) {
    constexpr uint32_t kWaves = kExtThreads / 64, kHeld = 8;
    __shared__ alignas(16) int32_t sh_seq[kExtThreads], sh_last[kExtThreads];
    __shared__ uint64_t sh_start[kExtThreads + 1];
    __shared__ int32_t sh_have[kExtThreads];    // first table slot an entry's new pages go to
    __shared__ int32_t sh_filled[kExtThreads];  // rows of the page that its first new page is a copy of; 0: of none
    __shared__ uint64_t sh_scan[kWaves];
    __shared__ uint32_t sh_free[kWaves], sh_n_copies;
    const uint32_t i = threadIdx.x, lane = i & 63, wave = i >> 6;
    const uint32_t page = 1u << kv.shift;
    if (i == 0) sh_n_copies = 0;

    const int32_t seq = i < n ? seqs[i] : -1;
    const int32_t count = i < n ? counts[i] : 0;
    // the counts of this wave's part of the pages
    const uint64_t part_pages = ((static_cast<uint64_t>(kv.n_pages) + kExtThreads - 1) / kExtThreads) * 64;
    const uint64_t p0 = wave * part_pages;
    const uint64_t p1 = p0 + part_pages < kv.n_pages ? p0 + part_pages : kv.n_pages;
    int32_t ref[kHeld];
    auto read = [&](uint64_t p) {  // 64 kHeld of them at once
#pragma unroll
        for (uint32_t x = 0; x < kHeld; ++x) {
            const uint64_t at = p + x * 64 + lane;
            ref[x] = at < p1 ? kv.refs[at] : -1;
        }
    };
    read(p0);
    const int32_t len0 = i < n && seq_ok(kv, seq) ? kv.lens[seq] : 0;
    sh_seq[i] = seq;
    __syncthreads();
    // the entries ahead, four at a time: one that names the sequence again is refused
    bool ok = i < n && seq_ok(kv, seq);
    auto ahead = [&](const int32_t* sh, int32_t what) {
        int32_t found = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < n; j += 4) {
            const i4 x = *reinterpret_cast<const i4*>(sh + j);
#pragma unroll
            for (uint32_t y = 0; y < 4; ++y) found += (j + y < i) & (x[y] == what);
        }
        return found;
    };
    if (wave * 64 < n) ok = ahead(sh_seq, seq) == 0 && ok;
    const int32_t len = ok ? len0 : 0;
    ok = ok && count >= 0 && len_ok(kv, len) &&
         static_cast<int64_t>(len) + count <= (static_cast<int64_t>(kv.max_pages) << kv.shift);
    const uint32_t filled = static_cast<uint32_t>(len) & (page - 1);
    const bool part = ok && filled && count > 0;
    const int32_t last =
        part ? kv.table[static_cast<uint64_t>(seq) * kv.max_pages + (static_cast<uint32_t>(len) >> kv.shift)] : -1;
    if (part && !page_ok(kv, last)) ok = false;
    if (i < n && !ok) atomicOr(err, kErrIndex);
    const bool shares = part && ok;
    const int32_t last_refs = shares ? kv.refs[last] : 0;
    sh_last[i] = shares ? last : -1;
    __syncthreads();
    // entries ahead that hold the same page: each took one count from it
    const bool copy = __any(last_refs > 1) && last_refs - ahead(sh_last, last) > 1;
    const uint32_t have = (static_cast<uint32_t>(len) + page - 1) >> kv.shift;
    const uint32_t want = (static_cast<uint32_t>(len) + static_cast<uint32_t>(count) + page - 1) >> kv.shift;
    const uint64_t need = ok ? want - have + (copy ? 1 : 0) : 0;
    sh_have[i] = static_cast<int32_t>(copy ? have - 1 : have);
    sh_filled[i] = copy ? static_cast<int32_t>(filled) : 0;
    uint64_t held[kHeld];
    uint32_t mine = 0;
    auto masks = [&](uint64_t* free) {
#pragma unroll
        for (uint32_t x = 0; x < kHeld; ++x) {
            free[x] = __ballot(ref[x] == 0);
            mine += __popcll(free[x]);
        }
    };
    masks(held);
    uint64_t total;
    const uint64_t start = scan_1024(need, sh_scan, total);
    sh_start[i] = start;
    if (i == 0) sh_start[kExtThreads] = total;
    if (total) {
        uint64_t free[kHeld];
        for (uint64_t p = p0 + kHeld * 64; p < p1; p += kHeld * 64) {
            read(p);
            masks(free);
        }
    }
    if (lane == 0) sh_free[wave] = mine;
    __syncthreads();
    uint64_t at = 0, n_free = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w < wave) at += sh_free[w];
        n_free += sh_free[w];
    }
    const bool fits = ok && start + need <= n_free;
    if (ok && !fits) atomicOr(err, kErrNoPages);

    // Page p, the f'th free one, to the entry whose part of the list f lies in: the last start
    // <= f (entries that need nothing lie behind the one that does), if it fits. Only this
    // wave reads its part of the counts from here on, before it writes them.
    auto give = [&](uint64_t p, uint64_t f) {
        uint32_t lo = 0, hi = n;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (sh_start[mid] <= f) lo = mid;
            else hi = mid;
        }
        if (sh_start[lo + 1] > n_free) return;
        const uint64_t slot = f - sh_start[lo];
        kv.table[static_cast<uint64_t>(sh_seq[lo]) * kv.max_pages + static_cast<uint64_t>(sh_have[lo]) + slot] =
            static_cast<int32_t>(p);
        kv.refs[p] = 1;
        if (slot == 0 && sh_filled[lo]) {
            atomicSub(&kv.refs[sh_last[lo]], 1);
            copies[atomicAdd(&sh_n_copies, 1u)] = PageCopy{sh_last[lo], static_cast<int32_t>(p), sh_filled[lo], 0};
        }
    };
    auto give_all = [&](uint64_t p, const uint64_t* free) {
#pragma unroll
        for (uint32_t x = 0; x < kHeld; ++x) {
            const uint64_t to = at + __popcll(free[x] & ((uint64_t(1) << lane) - 1));
            if ((free[x] >> lane & 1) && to < total) give(p + x * 64 + lane, to);
            at += __popcll(free[x]);
        }
    };
    if (at < total) give_all(p0, held);
    for (uint64_t p = p0 + kHeld * 64; p < p1 && at < total; p += kHeld * 64) {
        uint64_t free[kHeld];
        read(p);
        masks(free);
        give_all(p, free);
    }
    if (fits) kv.lens[seq] = len + count;
    __syncthreads();
    if (i == 0) *n_copies = sh_n_copies;
}

// The listed copies in every layer, keys and values: one wave for a page's rows of one head.
__global__ __launch_bounds__(256) void kv_copy_pages_kernel(const PageCopy* __restrict__ copies,
                                                            const uint32_t* __restrict__ n_copies, u4* k, u4* v,
                                                            uint32_t n_layers, uint32_t n_pages, uint32_t n_heads,
                                                            uint32_t row16, uint32_t page) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t per = static_cast<uint64_t>(n_layers) * 2 * n_heads;
    const uint64_t units = *n_copies * per;
    const uint64_t head16 = static_cast<uint64_t>(row16) * page;
    for (uint64_t u = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); u < units; u += gridDim.x * 4ull) {
        const PageCopy c = copies[u / per];
        const uint64_t r = u % per;
        const uint64_t layer = r / (2 * n_heads), head = r % (2 * n_heads);
        u4* pool = head < n_heads ? k : v;
        const uint64_t h = head < n_heads ? head : head - n_heads;
        const u4* from = pool + ((layer * n_pages + static_cast<uint32_t>(c.from)) * n_heads + h) * head16;
        u4* to = pool + ((layer * n_pages + static_cast<uint32_t>(c.to)) * n_heads + h) * head16;
        const uint32_t n16 = static_cast<uint32_t>(c.rows) * row16;
#pragma unroll 4
        for (uint32_t x = lane; x < n16; x += 64) to[x] = from[x];
    }
}

// Whether an entry below `e` names the same sequence; asked by a whole workgroup of 256.
__device__ __forceinline__ bool named_before(const int32_t* __restrict__ ids, uint32_t e, int32_t id) {
    bool same = false;
    for (uint32_t j = threadIdx.x; j < e; j += 256) same |= ids[j] == id;
    return __syncthreads_or(same);
}

// fork in two launches: with everything held in registers by one workgroup it is one, and no
// faster (24 x 2 sequences of 94 pages: 6.0 us against 3.3 and 2.6).
// First half: counts of the pages that change hands, and the sources' tables as they
// are now (rows [n][max_pages], then lengths [n]; -1 for an entry that is left out).
__global__ __launch_bounds__(256) void kv_fork_stage_kernel(KvView kv, const int32_t* __restrict__ src,
                                                            const int32_t* __restrict__ dst, int32_t* __restrict__ rows,
                                                            int32_t* __restrict__ lens, uint32_t* err) {
    const uint32_t e = blockIdx.y;
    const int32_t s = src[e], d = dst[e];
    const bool again = named_before(dst, e, d);
    bool ok = seq_ok(kv, s) && seq_ok(kv, d) && !again;
    const int32_t len = ok ? kv.lens[s] : -1;
    ok = ok && len_ok(kv, len);
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i == 0) {
        lens[e] = ok ? len : -1;
        if (!ok) atomicOr(err, kErrIndex);
    }
    if (!ok || i >= kv.max_pages) return;
    int32_t p = kv.table[static_cast<uint64_t>(s) * kv.max_pages + i];
    if (p != -1 && !page_ok(kv, p)) {
        atomicOr(err, kErrIndex);
        p = -1;
    }
    rows[static_cast<uint64_t>(e) * kv.max_pages + i] = p;
    if (p >= 0) atomicAdd(&kv.refs[p], 1);
    const int32_t old = kv.table[static_cast<uint64_t>(d) * kv.max_pages + i];
    if (page_ok(kv, old)) atomicSub(&kv.refs[old], 1);
}

__global__ __launch_bounds__(256) void kv_fork_write_kernel(KvView kv, const int32_t* __restrict__ dst,
                                                            const int32_t* __restrict__ rows,
                                                            const int32_t* __restrict__ lens) {
    const uint32_t e = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
    const int32_t len = lens[e];
    if (len < 0 || i >= kv.max_pages) return;
    const int32_t d = dst[e];
    kv.table[static_cast<uint64_t>(d) * kv.max_pages + i] = rows[static_cast<uint64_t>(e) * kv.max_pages + i];
    if (i == 0) kv.lens[d] = len;
}

__global__ __launch_bounds__(256) void kv_free_kernel(KvView kv, const int32_t* __restrict__ seqs, uint32_t* err) {
    const uint32_t e = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
    const int32_t s = seqs[e];
    const bool again = named_before(seqs, e, s);
    if (!seq_ok(kv, s) || again) {
        if (i == 0) atomicOr(err, kErrIndex);
        return;
    }
    if (i >= kv.max_pages) return;
    int32_t* at = kv.table + static_cast<uint64_t>(s) * kv.max_pages + i;
    const int32_t p = *at;
    if (page_ok(kv, p)) atomicSub(&kv.refs[p], 1);
    *at = -1;
    if (i == 0) kv.lens[s] = 0;
}

constexpr uint32_t kMaxKeep = 64;

// compact, first half: checks an entry and moves its kept rows down. A thread owns one
// 16-byte column of one (layer, keys or values, head) and moves it row after row: row j goes
// to a place at or below its own and below every later row's, and eight rows are read before
// the eight are written, so nothing is overwritten before it was read.
__global__ __launch_bounds__(256) void kv_compact_move_kernel(KvView kv, const int32_t* __restrict__ seqs,
                                                              const int32_t* __restrict__ drafts,
                                                              const int32_t* __restrict__ keep,
                                                              const int32_t* __restrict__ kept, uint32_t max_keep,
                                                              u4* k, u4* v, uint32_t n_layers, uint32_t n_heads,
                                                              uint32_t row16, int32_t* __restrict__ new_lens,
                                                              uint32_t* err) {
    __shared__ uint64_t sh_from[kMaxKeep], sh_to[kMaxKeep];  // 16-byte units from (layer 0, head 0)
    const uint32_t e = blockIdx.y, page = 1u << kv.shift;
    const int32_t seq = seqs[e], nd = drafts[e], nk = kept[e];
    const bool again = named_before(seqs, e, seq);
    bool ok = seq_ok(kv, seq) && !again;
    const int32_t len = ok ? kv.lens[seq] : 0;
    ok = ok && len_ok(kv, len) && nd >= 0 && nd <= len && nk >= 0 && nk <= nd && static_cast<uint32_t>(nk) <= max_keep;
    const uint64_t page16 = static_cast<uint64_t>(n_heads) * page * row16;
    bool bad = false;
    const uint32_t j = threadIdx.x;
    if (ok && j < static_cast<uint32_t>(nk)) {
        const int32_t* row = keep + static_cast<uint64_t>(e) * max_keep;
        const int32_t x = row[j];
        bad = x < 0 || x >= nd || (j > 0 && row[j - 1] >= x);
        if (!bad) {
            const int32_t* table = kv.table + static_cast<uint64_t>(seq) * kv.max_pages;
            const uint32_t a = static_cast<uint32_t>(len - nd + x), b = static_cast<uint32_t>(len - nd) + j;
            const int32_t pa = table[a >> kv.shift], pb = table[b >> kv.shift];
            bad = !page_ok(kv, pa) || !page_ok(kv, pb) || (a != b && kv.refs[pb] != 1);
            sh_from[j] = static_cast<uint32_t>(pa) * page16 + (a & (page - 1)) * row16;
            sh_to[j] = static_cast<uint32_t>(pb) * page16 + (b & (page - 1)) * row16;
        }
    }
    ok = !__syncthreads_or(bad) && ok;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        new_lens[e] = ok ? len - nd + nk : -1;
        if (!ok) atomicOr(err, kErrIndex);
    }
    if (!ok) return;
    const uint64_t columns = static_cast<uint64_t>(n_layers) * 2 * n_heads * row16;
    for (uint64_t c = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; c < columns; c += gridDim.x * 256ull) {
        const uint32_t x = static_cast<uint32_t>(c % row16);
        const uint64_t unit = c / row16, layer = unit / (2 * n_heads);
        const uint32_t hh = static_cast<uint32_t>(unit % (2 * n_heads)), h = hh < n_heads ? hh : hh - n_heads;
        u4* base = (hh < n_heads ? k : v) + layer * kv.n_pages * page16 + static_cast<uint64_t>(h) * page * row16 + x;
        for (uint32_t j0 = 0; j0 < static_cast<uint32_t>(nk); j0 += 8) {
            u4 t[8];
#pragma unroll
            for (uint32_t y = 0; y < 8; ++y)
                if (j0 + y < static_cast<uint32_t>(nk)) t[y] = base[sh_from[j0 + y]];
#pragma unroll
            for (uint32_t y = 0; y < 8; ++y)
                if (j0 + y < static_cast<uint32_t>(nk)) base[sh_to[j0 + y]] = t[y];
        }
    }
}

// compact, second half: the new lengths, and pages past them released.
__global__ __launch_bounds__(256) void kv_compact_cut_kernel(KvView kv, const int32_t* __restrict__ seqs,
                                                             const int32_t* __restrict__ new_lens) {
    const uint32_t e = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
    const int32_t len = new_lens[e];
    if (len < 0 || i >= kv.max_pages) return;
    const int32_t s = seqs[e];
    if (i == 0) kv.lens[s] = len;
    if (i < (static_cast<uint32_t>(len) + (1u << kv.shift) - 1) >> kv.shift) return;
    int32_t* at = kv.table + static_cast<uint64_t>(s) * kv.max_pages + i;
    const int32_t p = *at;
    if (page_ok(kv, p)) atomicSub(&kv.refs[p], 1);
    if (p != -1) *at = -1;
}

}  // namespace dev

using namespace dev;

namespace {

// Checks shared by the page operations.
int32_t begin(objeta_hip_context* ctx, const objeta_hip_kv_cache* cache, uint64_t n, const char* action) {
    OBJ_TRY(check_ctx(ctx, action));
    OBJ_TRY(check_kv(cache, action));
    if (n > kMaxPageOps)
        OBJ_FAIL(kInvalidInput, action, strf("%llu entries, at most %llu a call", (unsigned long long)n,
                                             (unsigned long long)kMaxPageOps));
    return 0;
}

dim3 table_grid(const objeta_hip_kv_cache& c, uint64_t n) {
    return dim3((c.max_pages + 255) / 256, static_cast<uint32_t>(n));
}

}  // namespace

}  // namespace objeta

using namespace objeta;

extern "C" {

int32_t objeta_hip_kv_extend_device(objeta_hip_context* ctx, objeta_hip_stream stream, const objeta_hip_kv_cache* cache,
                                    const int32_t* d_seqs, const int32_t* d_counts, uint64_t n) {
    OBJ_GUARD_BEGIN
    const char* action = "kv_extend_device";
    OBJ_TRY(begin(ctx, cache, n, action));
    if (n == 0) return 0;
    if (!d_seqs || !d_counts) OBJ_FAIL(kInvalidInput, action, "sequences or counts are NULL");
    OBJ_HIP(hipSetDevice(ctx->device), "hipSetDevice");
    const objeta_hip_kv_cache& c = *cache;
    const hipStream_t s = resolve_stream(ctx, stream);
    void* ws = nullptr;
    const size_t copies = 256;
    OBJ_TRY(ensure_workspace(ctx, s, kWsPages, copies + kMaxPageOps * sizeof(PageCopy), &ws));
    char* w = static_cast<char*>(ws);
    uint32_t* n_copies = reinterpret_cast<uint32_t*>(w);
    PageCopy* pc = reinterpret_cast<PageCopy*>(w + copies);
    hipLaunchKernelGGL(kv_extend_kernel, dim3(1), dim3(kExtThreads), 0, s, kv_view(c), d_seqs, d_counts,
                       static_cast<uint32_t>(n), pc, n_copies, ctx->err_word);
    OBJ_HIP(hipGetLastError(), action);
    // most calls copy nothing and the rest few pages: enough workgroups to fill the device
    // once, fewer where even n copies need fewer
    const uint64_t waves = n * c.n_layers * 2 * c.n_kv_heads;
    const uint32_t grid = static_cast<uint32_t>(waves < 4096 ? (waves + 3) / 4 : 1024);
    const uint32_t row16 = c.head_dim * static_cast<uint32_t>(dtype_size(c.dtype)) / 16;
    hipLaunchKernelGGL(kv_copy_pages_kernel, dim3(grid), dim3(256), 0, s, pc, n_copies, static_cast<u4*>(c.k),
                       static_cast<u4*>(c.v), c.n_layers, c.n_pages, c.n_kv_heads, row16, c.page_size);
    OBJ_HIP(hipGetLastError(), action);
    return 0;
    OBJ_GUARD_END
}

int32_t objeta_hip_kv_fork_device(objeta_hip_context* ctx, objeta_hip_stream stream, const objeta_hip_kv_cache* cache,
                                  const int32_t* d_src, const int32_t* d_dst, uint64_t n) {
    OBJ_GUARD_BEGIN
    const char* action = "kv_fork_device";
    OBJ_TRY(begin(ctx, cache, n, action));
    if (n == 0) return 0;
    if (!d_src || !d_dst) OBJ_FAIL(kInvalidInput, action, "sources or destinations are NULL");
    OBJ_HIP(hipSetDevice(ctx->device), "hipSetDevice");
    const objeta_hip_kv_cache& c = *cache;
    const hipStream_t s = resolve_stream(ctx, stream);
    void* ws = nullptr;
    OBJ_TRY(ensure_workspace(ctx, s, kWsPages, (kMaxPageOps + static_cast<size_t>(n) * c.max_pages) * 4, &ws));
    int32_t* lens = static_cast<int32_t*>(ws);
    int32_t* rows = lens + kMaxPageOps;
    hipLaunchKernelGGL(kv_fork_stage_kernel, table_grid(c, n), dim3(256), 0, s, kv_view(c), d_src, d_dst, rows, lens,
                       ctx->err_word);
    OBJ_HIP(hipGetLastError(), action);
    hipLaunchKernelGGL(kv_fork_write_kernel, table_grid(c, n), dim3(256), 0, s, kv_view(c), d_dst, rows, lens);
    OBJ_HIP(hipGetLastError(), action);
    return 0;
    OBJ_GUARD_END
}

int32_t objeta_hip_kv_compact_device(objeta_hip_context* ctx, objeta_hip_stream stream, const objeta_hip_kv_cache* cache,
                                     const int32_t* d_seqs, const int32_t* d_drafts, const int32_t* d_keep,
                                     const int32_t* d_kept, uint64_t n, uint64_t max_keep) {
    OBJ_GUARD_BEGIN
    const char* action = "kv_compact_device";
    OBJ_TRY(begin(ctx, cache, n, action));
    if (max_keep > kMaxKeep)
        OBJ_FAIL(kInvalidInput, action, strf("max_keep %llu exceeds %u", (unsigned long long)max_keep, kMaxKeep));
    if (n == 0) return 0;
    if (!d_seqs || !d_drafts || !d_kept || (max_keep && !d_keep))
        OBJ_FAIL(kInvalidInput, action, "sequences, drafts, keep or kept are NULL");
    OBJ_HIP(hipSetDevice(ctx->device), "hipSetDevice");
    const objeta_hip_kv_cache& c = *cache;
    const hipStream_t s = resolve_stream(ctx, stream);
    void* ws = nullptr;
    OBJ_TRY(ensure_workspace(ctx, s, kWsPages, kMaxPageOps * 4, &ws));
    int32_t* lens = static_cast<int32_t*>(ws);
    const uint32_t row16 = c.head_dim * static_cast<uint32_t>(dtype_size(c.dtype)) / 16;
    const uint64_t blocks = (static_cast<uint64_t>(c.n_layers) * 2 * c.n_kv_heads * row16 + 255) / 256;
    const uint32_t grid = max_keep ? static_cast<uint32_t>(blocks < 256 ? blocks : 256) : 1;
    hipLaunchKernelGGL(kv_compact_move_kernel, dim3(grid, static_cast<uint32_t>(n)), dim3(256), 0, s, kv_view(c), d_seqs,
                       d_drafts, d_keep, d_kept, static_cast<uint32_t>(max_keep), static_cast<u4*>(c.k),
                       static_cast<u4*>(c.v), c.n_layers, c.n_kv_heads, row16, lens, ctx->err_word);
    OBJ_HIP(hipGetLastError(), action);
    hipLaunchKernelGGL(kv_compact_cut_kernel, table_grid(c, n), dim3(256), 0, s, kv_view(c), d_seqs, lens);
    OBJ_HIP(hipGetLastError(), action);
    return 0;
    OBJ_GUARD_END
}

int32_t objeta_hip_kv_free_device(objeta_hip_context* ctx, objeta_hip_stream stream, const objeta_hip_kv_cache* cache,
                                  const int32_t* d_seqs, uint64_t n) {
    OBJ_GUARD_BEGIN
    const char* action = "kv_free_device";
    OBJ_TRY(begin(ctx, cache, n, action));
    if (n == 0) return 0;
    if (!d_seqs) OBJ_FAIL(kInvalidInput, action, "sequences are NULL");
    OBJ_HIP(hipSetDevice(ctx->device), "hipSetDevice");
    hipLaunchKernelGGL(kv_free_kernel, table_grid(*cache, n), dim3(256), 0, resolve_stream(ctx, stream), kv_view(*cache),
                       d_seqs, ctx->err_word);
    OBJ_HIP(hipGetLastError(), action);
    return 0;
    OBJ_GUARD_END
}

}  // extern "C"
