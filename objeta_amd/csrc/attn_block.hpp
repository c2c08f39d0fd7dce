// attn_block.hpp — attention of 128 rows by one workgroup of four waves, the tiles of keys
// and values shared in LDS: prompts, and many rows (trees of drafts, chunks) over the cache.
//
// A row is a (token, query head) pair of one key/value head, token by token, so that grouped
// heads share every tile, and short sequences packed behind one another share a workgroup: a
// row carries the range of keys that it sees, and a workgroup walks the keys that any of its
// rows sees. Tiles that all rows of a wave see whole take no mask; those none sees are
// skipped. Keys and values of tile t + 1 travel in registers during the products of tile t
// and go to the other LDS buffer behind them: one barrier a tile.
#pragma once

#include "attn_tile.hpp"

namespace objeta {
namespace dev {

template <int KT, int DT>
struct Block {
    typedef Rows<KT, DT, 32> R;
    static constexpr int kKeys = R::kBytes <= 512 ? 64 : 32;
    static constexpr int kSub = kKeys / 32;
    static constexpr int kLoads = kKeys * R::kUnits / 256;  // 16-byte units of K (and of V) a thread stages
    static constexpr int kTile = kKeys * R::kBytes;
    static_assert(kKeys * R::kUnits % 256 == 0, "whole units a thread");
    static constexpr int kLds = 4 * kTile;
    // two workgroups a CU where LDS and registers allow it
    static constexpr int kPerCu = kLds <= 65536 ? 2 : 1;
};

template <int QT, int KT, int DT, bool PAGED>
__global__ __launch_bounds__(256, (QT == kDtF32 ? 1 : Block<KT, DT>::kPerCu)) void attn_block_kernel(AttnArgs a) {
    typedef Math<QT, KT, DT, 32> M;
    typedef Rows<KT, DT, 32> R;
    typedef Block<KT, DT> B;
    constexpr int kKeys = B::kKeys;
    __shared__ alignas(16) char lds[2][2][B::kTile];
    __shared__ int32_t sh_lo[4], sh_hi[4];
    __shared__ int32_t ring[4][8];  // page ids of a tile's groups of eight keys
    __shared__ int32_t sh_bad;

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    uint32_t tile, head, split = 0;
    int32_t row0 = 0, n_q = static_cast<int32_t>(a.n_rows), len = 0;
    KvRows<PAGED, KT> kv;
    bool usable = true;
    if constexpr (PAGED) {
        const CachedItem item(a, blockIdx.x);
        if (!item.any) return;
        split = item.split, tile = item.tile, head = item.head;
        const uint32_t b = item.b;
        row0 = a.cu[b];
        const int32_t end = a.cu[b + 1];
        n_q = end - row0;
        if (row0 < 0 || end < row0 || static_cast<uint32_t>(end) > a.n_rows) {
            if (tid == 0) atomicOr(a.err, kErrIndex);
            return;
        }
        const int32_t seq = a.seqs[b];
        usable = seq_ok(a.kv, seq);
        len = usable ? a.kv.lens[seq] : 0;
        usable = usable && len_ok(a.kv, len) && n_q <= len && (!a.tree || n_q <= 64);
        if (!usable) len = 0;
        if (!usable && tid == 0 && n_q) atomicOr(a.err, kErrIndex);
        if (split && static_cast<uint64_t>(split) * a.chunk >= static_cast<uint64_t>(len)) return;
        kv.kv = a.kv;
        kv.table = a.kv.table + static_cast<uint64_t>(usable ? seq : 0) * a.kv.max_pages;
        kv.page_step = (static_cast<uint64_t>(a.n_kv) * a.dim) << a.kv.shift;
        const uint64_t off = a.layer_off + ((static_cast<uint64_t>(head) * a.dim) << a.kv.shift);
        kv.k = static_cast<const typename M::kelem*>(a.k) + off;
        kv.v = static_cast<const typename M::kelem*>(a.v) + off;
    } else {
        // the last tiles see the most keys: they start first
        head = blockIdx.x % a.n_kv;
        tile = a.n_tiles - 1 - blockIdx.x / a.n_kv;
        kv.k = static_cast<const typename M::kelem*>(a.k) + static_cast<uint64_t>(head) * a.dim;
        kv.v = static_cast<const typename M::kelem*>(a.v) + static_cast<uint64_t>(head) * a.dim;
        kv.k_stride = a.k_stride, kv.v_stride = a.v_stride;
    }
    kv.dim = a.dim;
    const uint32_t n_m = static_cast<uint32_t>(n_q) * a.group;

    for (; static_cast<uint64_t>(tile) * 128 < n_m; tile += a.n_tiles) {
        // ---- this lane's row
        const uint32_t m = tile * 128 + wave * 32 + (lane & 31);
        bool real = m < n_m;
        const uint32_t i = m / a.group, q_head = head * a.group + m % a.group;
        const uint64_t row = static_cast<uint64_t>(row0) + (real ? i : 0);
        RowView view{0, -1, 0x7FFFFFFF, 0};
        if constexpr (PAGED) {
            if (real && usable) {
                const int32_t base = len - n_q;
                if (a.tree) view = RowView{0, len - 1, base, a.tree[row]};
                else view.hi = base + static_cast<int32_t>(i);
            }
        } else {
            if (real) {
                // the sequence that holds token i: the last start that is <= i
                uint32_t lo = 0, hi = a.n_batch;  // cu[lo] <= i < cu[hi] once both are known to hold
                while (lo < hi) {
                    const uint32_t mid = (lo + hi) >> 1;
                    if (a.cu[mid + 1] <= static_cast<int32_t>(i)) lo = mid + 1;
                    else hi = mid;
                }
                int32_t s = 0, e = 0;
                if (lo < a.n_batch) s = a.cu[lo], e = a.cu[lo + 1];
                const bool in = lo < a.n_batch && s <= static_cast<int32_t>(i) && static_cast<int32_t>(i) < e;
                if (in && (s < 0 || static_cast<uint32_t>(e) > a.n_rows)) atomicOr(a.err, kErrIndex);
                real = in && s >= 0 && static_cast<uint32_t>(e) <= a.n_rows;
                if (real) view.lo = s, view.hi = a.causal ? static_cast<int32_t>(i) : e - 1;
            }
        }
        typename M::Query q;
        float scale = a.scale_log2;
        M::load_q(q, static_cast<const typename M::qelem*>(a.q) + row * a.q_stride + static_cast<uint64_t>(q_head) * a.dim, real,
                  a.dim, lane, scale);
        // ---- what the wave and the workgroup see
        const bool sees_any = view.lo <= view.hi;
        int32_t w_lo = sees_any ? view.lo : 0x7FFFFFFF, w_hi = sees_any ? view.hi : -1;
        int32_t all_lo = sees_any || !real ? view.lo : 0x7FFFFFFF;  // from here to all_hi every real row sees all
        int32_t all_hi = real ? (view.base - 1 < view.hi ? view.base - 1 : view.hi) : 0x7FFFFFFF;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) {
            const int32_t x = __shfl_xor(w_lo, s, 64), y = __shfl_xor(w_hi, s, 64);
            const int32_t z = __shfl_xor(all_lo, s, 64), w = __shfl_xor(all_hi, s, 64);
            w_lo = x < w_lo ? x : w_lo, w_hi = y > w_hi ? y : w_hi;
            all_lo = z > all_lo ? z : all_lo, all_hi = w < all_hi ? w : all_hi;
        }
        if (tid == 0) sh_bad = 0;
        if (lane == 0) sh_lo[wave] = w_lo, sh_hi[wave] = w_hi;
        __syncthreads();
        int32_t k_lo = sh_lo[0], k_hi = sh_hi[0];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            k_lo = sh_lo[w] < k_lo ? sh_lo[w] : k_lo;
            k_hi = sh_hi[w] > k_hi ? sh_hi[w] : k_hi;
        }
        int32_t k_end = k_hi + 1;
        if constexpr (PAGED) {
            const int64_t c0 = static_cast<int64_t>(split) * a.chunk, c1 = c0 + a.chunk;
            if (k_lo < c0) k_lo = static_cast<int32_t>(c0);
            if (split + 1 < a.n_splits && k_end > c1) k_end = static_cast<int32_t>(c1);
        }
        RowState<M> st;
        st.clear();
        const int32_t k_begin = k_lo & ~(kKeys - 1);
        const int32_t n_tiles = k_begin < k_end ? (k_end - k_begin + kKeys - 1) / kKeys : 0;

        // ---- staging
        u32x4a rk[B::kLoads], rv[B::kLoads];
        bool bad = false;
        auto load_pages = [&](int32_t t) -> int32_t {  // threads 0 .. kKeys / 8
            int32_t p = 0;
            if constexpr (PAGED) {
                const int32_t slot = k_begin + t * kKeys + static_cast<int32_t>(tid) * 8;
                if (tid < kKeys / 8 && slot < k_end) p = kv.page_of(static_cast<uint32_t>(slot), bad);
            }
            return p;
        };
        auto load_tile = [&](int32_t t) {
#pragma unroll
            for (int x = 0; x < B::kLoads; ++x) {
                const uint32_t u = x * 256 + tid, key = u / R::kUnits, c = u % R::kUnits;
                const int32_t slot = k_begin + t * kKeys + static_cast<int32_t>(key);
                const bool in = slot < k_end && c * (16 / R::kEs) < a.dim;
                rk[x] = u32x4a{0, 0, 0, 0};
                rv[x] = u32x4a{0, 0, 0, 0};
                if (in) {
                    if constexpr (PAGED) {
                        const uint64_t at = kv.paged_at(ring[t & 3][key >> 3], static_cast<uint32_t>(slot));
                        rk[x] = *reinterpret_cast<const u32x4a*>(kv.k + at + c * (16 / R::kEs));
                        rv[x] = *reinterpret_cast<const u32x4a*>(kv.v + at + c * (16 / R::kEs));
                    } else {
                        rk[x] = *reinterpret_cast<const u32x4a*>(kv.k + static_cast<uint32_t>(slot) * kv.k_stride +
                                                                 c * (16 / R::kEs));
                        rv[x] = *reinterpret_cast<const u32x4a*>(kv.v + static_cast<uint32_t>(slot) * kv.v_stride +
                                                                 c * (16 / R::kEs));
                    }
                }
            }
        };
        auto store_tile = [&](int buf) {
#pragma unroll
            for (int x = 0; x < B::kLoads; ++x) {
                const uint32_t u = x * 256 + tid, key = u / R::kUnits, c = u % R::kUnits;
                *reinterpret_cast<u32x4a*>(&lds[buf][0][key * R::kBytes + ((c ^ R::swz_k(key)) << 4)]) = rk[x];
                *reinterpret_cast<u32x4a*>(&lds[buf][1][key * R::kBytes + ((c ^ R::swz_v(key)) << 4)]) = rv[x];
            }
        };
        if (n_tiles) {
            if constexpr (PAGED) {
                const int32_t p0 = load_pages(0), p1 = load_pages(1);
                if (tid < kKeys / 8) ring[0][tid] = p0, ring[1][tid] = p1;
                __syncthreads();
            }
            load_tile(0);
            store_tile(0);
        }
        __syncthreads();
        const uint32_t kx = M::k_first(lane), vx = M::v_first(lane);
        for (int32_t t = 0; t < n_tiles; ++t) {
            int32_t ahead = 0;
            if (PAGED && t + 2 < n_tiles) ahead = load_pages(t + 2);
            if (t + 1 < n_tiles) load_tile(t + 1);
            const int32_t k0 = k_begin + t * kKeys;
            if (k0 <= w_hi && k0 + kKeys > w_lo) {
                const char* kb = lds[t & 1][0];
                Scores<M> s[B::kSub];
#pragma unroll
                for (int n = 0; n < B::kSub; ++n) scores<M>(s[n], q, kb + n * 32 * R::kBytes, lane, kx);
                if (k0 < all_lo || k0 + kKeys - 1 > all_hi || k0 < k_lo || k0 + kKeys > k_end) {
#pragma unroll
                    for (int n = 0; n < B::kSub; ++n)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int32_t key = k0 + 32 * n + static_cast<int32_t>(M::key_of(0, r, h));
                            if (!(view.sees(key) && key >= k_lo && key < k_end)) s[n].s[0][r] = -kInf;
                        }
                }
                accumulate<M, B::kSub>(st, s, scale, lds[t & 1][1], vx);
            }
            if (t + 1 < n_tiles) store_tile((t + 1) & 1);
            if constexpr (PAGED) {
                if (t + 2 < n_tiles && tid < kKeys / 8) ring[(t + 2) & 3][tid] = ahead;
            }
            __syncthreads();
        }
        if constexpr (PAGED) {
            if (bad) sh_bad = 1;
            __syncthreads();
            if (!usable || sh_bad) {
                if (tid == 0 && sh_bad) atomicOr(a.err, kErrIndex);
                st.l = __builtin_nanf("");
#pragma unroll
                for (int d = 0; d < DT / 32; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) st.o[d][r] = st.l;
                write_rows<M, QT>(a, st, real, row, q_head, split, lane);
                __syncthreads();
                continue;
            }
        }
        if (not_finite<M>(st)) {
            for (int r = 0; r < 32; ++r) {
                if (!__builtin_amdgcn_readlane(real, r)) continue;
                const uint32_t r_m = tile * 128 + wave * 32 + r, r_head = head * a.group + r_m % a.group;
                const uint64_t r_row = static_cast<uint64_t>(row0) + r_m / a.group;
                RowView rv1{__builtin_amdgcn_readlane(view.lo, r), __builtin_amdgcn_readlane(view.hi, r),
                            __builtin_amdgcn_readlane(view.base, r), 0};
                rv1.mask = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int32_t>(view.mask), r)) |
                           static_cast<uint64_t>(static_cast<uint32_t>(
                               __builtin_amdgcn_readlane(static_cast<int32_t>(view.mask >> 32), r)))
                               << 32;
                float rm, rl, ro[4];
                row_by_row<M, PAGED, KT>(kv,
                                         static_cast<const typename M::qelem*>(a.q) + r_row * a.q_stride +
                                             static_cast<uint64_t>(r_head) * a.dim,
                                         rv1, k_lo, k_end, a.scale_log2, a.dim, rm, rl, ro);
                write_row<M>(a, rm, rl, ro, r_row, r_head, split, lane);
            }
        } else {
            write_rows<M, QT>(a, st, real, row, q_head, split, lane);
        }
        if constexpr (!PAGED) break;
        __syncthreads();  // the next tile's ranges go where this one's were read
    }
}

}  // namespace dev
}  // namespace objeta
