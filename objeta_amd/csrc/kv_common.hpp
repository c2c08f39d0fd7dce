// kv_common.hpp — what the rotary, paged-cache and attention translation units share:
// element types, host checks of a cache descriptor and of overlapping rows, and the
// device view of a cache with its bounds checks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "host_common.hpp"

namespace objeta {

enum : int { kDtF32 = OBJETA_HIP_DT_F32, kDtF16 = OBJETA_HIP_DT_F16, kDtBF16 = OBJETA_HIP_DT_BF16 };
constexpr uint32_t kErrIndex = 4u;    // device error word, bit 2: an index outside its table
constexpr uint32_t kErrNoPages = 8u;  // bit 3: not enough free pages
constexpr uint64_t kMaxHeadDim = 256;
constexpr uint64_t kMaxPageOps = 1024;  // entries of one page operation
constexpr uint64_t kMaxTokens = 0x7FFF0000u;  // of a sequence: 32-bit sums of a key's index and a tile's keys stay below 2^31

// Workgroups of one launch: a grid of 2^32 threads and more in a dimension runs fewer workgroups
// than asked for, without an error. More go in several launches, each told its first one; a
// multiple of the XCDs.
constexpr uint64_t kMostGroups = uint64_t(1) << 22;

inline bool dtype_ok(int32_t t) { return t == kDtF32 || t == kDtF16 || t == kDtBF16; }
inline uint64_t dtype_size(int32_t t) { return t == kDtF32 ? 4 : 2; }
inline bool head_dim_ok(uint64_t d) { return d >= 8 && d <= kMaxHeadDim && d % 8 == 0; }

// n rows of `width` bytes, `stride` bytes apart.
struct RowSet {
    const void* p;
    uint64_t stride, width, n;
};
// Whether two row sets share a byte. Sets of one stride are compared row by row (columns of
// one packed buffer do not overlap), others by their whole extents.
inline bool rows_overlap(const RowSet& a, const RowSet& b) {
    if (!a.p || !b.p || !a.n || !b.n || !a.width || !b.width) return false;
    const uint64_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    const uint64_t ea = pa + (a.n - 1) * a.stride + a.width, eb = pb + (b.n - 1) * b.stride + b.width;
    if (ea <= pb || eb <= pa) return false;
    if (a.n > 1 && b.n > 1 && a.stride == b.stride && a.stride >= a.width && a.stride >= b.width) {
        const uint64_t d = (pb >= pa ? pb - pa : a.stride - (pa - pb) % a.stride) % a.stride;  // b's column in a's rows
        return d < a.width || d + b.width > a.stride;
    }
    return true;
}
// (n - 1) * stride + width elements of `size` bytes without a 64-bit overflow.
inline bool extent_ok(uint64_t n, uint64_t stride, uint64_t width, uint64_t size) {
    return n < (uint64_t(1) << 31) && stride < (uint64_t(1) << 31) && width < (uint64_t(1) << 31) && size <= 8;
}

// Checks a cache descriptor (sizes, pointers, alignment).
int32_t check_kv(const objeta_hip_kv_cache* c, const char* action);
int32_t check_rope(const objeta_hip_rope* r, uint64_t head_dim, const char* action);

#if defined(__HIPCC__)
namespace dev {

// The cache's tables as kernels read them. Every index is checked here before use.
struct KvView {
    int32_t* table;
    int32_t* lens;
    int32_t* refs;
    uint32_t n_seqs, max_pages, n_pages, shift;  // page size 1 << shift
};

__device__ __forceinline__ bool seq_ok(const KvView& kv, int32_t s) {
    return static_cast<uint32_t>(s) < kv.n_seqs;
}
__device__ __forceinline__ bool page_ok(const KvView& kv, int32_t p) {
    return static_cast<uint32_t>(p) < kv.n_pages;
}
__device__ __forceinline__ bool len_ok(const KvView& kv, int32_t len) {
    return len >= 0 && static_cast<uint64_t>(len) <= (static_cast<uint64_t>(kv.max_pages) << kv.shift);
}

// How many of cu[0 .. n) are <= r, by one wave; with ascending cu the batch entry that
// holds row r is this less one.
__device__ __forceinline__ uint32_t count_le(const int32_t* __restrict__ cu, uint32_t n, int64_t r) {
    uint32_t c = 0;
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t i = 0; i < n; i += 64) c += __popcll(__ballot(i + lane < n && cu[i + lane] <= r));
    return c;
}

// The sequence of packed prompts that holds a token: the first of n whose end is past it, where
// `ended(b)` tells that sequence b's is not. The attention kernel and the join of its parts ask the
// same questions, so that they agree where the indices are in no order too.
template <class Ended>
__device__ __forceinline__ uint32_t first_unended(uint32_t n, Ended ended) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (ended(mid)) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// That sequence's tokens [lo, hi), found for token r by a whole wave; up to 63 sequences lie in the
// lanes after one read. `any`: it holds r, and its tokens are among the n_rows.
struct TokenRange {
    int32_t lo, hi;
    bool any;
    __device__ __forceinline__ TokenRange(const int32_t* __restrict__ cu, uint32_t n, uint32_t n_rows, int32_t r) {
        const uint32_t lane = threadIdx.x & 63;
        uint32_t b;
        lo = hi = 0;
        if (n < 64) {
            const int32_t start = cu[lane <= n ? lane : n];
            const uint64_t past = __ballot(start <= r) >> 1;
            b = first_unended(n, [&](uint32_t x) { return (past >> x & 1) != 0; });
            if (b < n) lo = __builtin_amdgcn_readlane(start, b), hi = __builtin_amdgcn_readlane(start, b + 1);
        } else {
            b = first_unended(n, [&](uint32_t x) { return cu[x + 1] <= r; });
            if (b < n) lo = cu[b], hi = cu[b + 1];
        }
        any = b < n && 0 <= lo && lo <= r && r < hi && static_cast<uint32_t>(hi) <= n_rows;
    }
};

// The batch entry that holds row r, found by a whole wave. `any`: there is one; `again` (where
// LATER): a later entry that has rows names the same sequence. Up to 63 entries lie in the lanes
// after one read, since such reads are what small kernels wait for (a join of 32 rows: 4.4 us, with
// a search and reads of its own for the entry's bounds 4.9).
template <bool LATER>
struct RowEntry {
    int32_t lo, hi, seq;
    bool any, again;
    __device__ __forceinline__ RowEntry(const int32_t* __restrict__ cu, const int32_t* __restrict__ seqs, uint32_t n_batch,
                                        int64_t r) {
        const uint32_t lane = threadIdx.x & 63;
        uint32_t b;
        lo = hi = 0, seq = -1, again = false;
        if (n_batch < 64) {
            const int32_t start = cu[lane <= n_batch ? lane : n_batch], s = seqs[lane < n_batch ? lane : n_batch - 1];
            int32_t end = 0;  // read beside the starts, so that no wait is added
            if (LATER) end = cu[lane < n_batch ? lane + 1 : n_batch];
            const uint32_t le = __popcll(__ballot(lane <= n_batch && start <= r));
            any = le != 0 && le <= n_batch;
            if (!any) return;
            b = le - 1;
            lo = __builtin_amdgcn_readlane(start, b), hi = __builtin_amdgcn_readlane(start, le);
            seq = __builtin_amdgcn_readlane(s, b);
            if (LATER) again = __ballot(lane > b && lane < n_batch && s == seq && end > start) != 0;
        } else {
            const uint32_t le = count_le(cu, n_batch + 1, r);
            any = le != 0 && le <= n_batch;
            if (!any) return;
            b = le - 1;
            lo = cu[b], hi = cu[le], seq = seqs[b];
            for (uint32_t i = b + 1; LATER && i < n_batch; i += 64)
                again |= __ballot(i + lane < n_batch && seqs[i + lane] == seq && cu[i + lane + 1] > cu[i + lane]) != 0;
        }
        any = lo <= r && r < hi;
    }
};

}  // namespace dev

inline dev::KvView kv_view(const objeta_hip_kv_cache& c) {
    uint32_t shift = 0;
    while ((1u << shift) < c.page_size) ++shift;
    return dev::KvView{c.page_table, c.seq_lens, c.ref_counts, c.n_seqs, c.max_pages, c.n_pages, shift};
}
#endif

}  // namespace objeta
