// attn_block.hpp — attention of 128 rows by one workgroup of four waves, the tiles of keys
// and values shared in LDS: prompts, and many rows (trees of drafts, chunks) over the cache.
//
// A row is a (token, query head) pair of one key/value head, token by token, so that grouped
// heads share every tile, and short sequences packed behind one another share a workgroup: a
// row carries the range of keys that it sees, and a workgroup walks the keys that any of its
// rows sees. Tiles that all rows of a wave see whole take no mask. Keys and values of the next
// tile but one travel in registers.
#pragma once

#include "attn_careful.hpp"

namespace objeta {
namespace dev {

template <int KT, int DT>
struct Block {
    typedef Rows<KT, DT, 32> R;
    static constexpr int kKeys = KT != kDtF32x3 && R::kBytes <= 512 ? 64 : 32;
    static constexpr int kSub = kKeys / 32;
    static constexpr int kLoads = kKeys / (4 * R::kPer);  // 16-byte units of K (and of V) a thread stages
    static constexpr int kTileK = kKeys * R::kK, kTileV = kKeys * R::kV;
    static_assert(R::kEs == 4 || kSub == 2, "16-bit tiles are two steps");
    static constexpr int kLds = 2 * (kTileK + kTileV);
    // two workgroups a CU where LDS and registers allow it
    static constexpr int kPerCu = kLds <= 73728 ? 2 : 1;
};

// How float keys and values are taken: in parts where two tiles of them fit LDS.
template <int KT, int DT>
constexpr int block_type = KT == kDtF32 && DT <= 192 ? kDtF32x3 : KT;

template <int QT, int KT, int DT, bool PAGED>
__global__ __launch_bounds__(256, (QT == kDtF32 ? 1 : Block<KT, DT>::kPerCu)) void attn_block_kernel(AttnArgs a) {
    typedef Math<QT, KT, DT, 32> M;
    typedef Rows<KT, DT, 32> R;
    typedef Block<KT, DT> B;
    constexpr int kKeys = B::kKeys;
    __shared__ alignas(16) char lds_k[2][B::kTileK], lds_v[2][B::kTileV];
    __shared__ int32_t sh_lo[4], sh_hi[4];
    __shared__ int32_t ring[4][8];  // page ids of a tile's groups of eight keys
    __shared__ int32_t sh_bad;       // bit 0: a bad page; bit 1: a result that is not finite
    __shared__ uint32_t sh_odd[3];   // second pass: keys of a tile without parts; whether values are marked

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    uint32_t tile, head, split = 0;
    int32_t row0 = 0, n_q = static_cast<int32_t>(a.n_rows), len = 0;
    KvRows<PAGED, KT> kv;
    uint32_t part = 0;
    bool usable = true, last_part = true;
    if constexpr (PAGED) {
        const BlockItem item(a, a.first + blockIdx.x, 256 * (QT == kDtF32 ? 1 : B::kPerCu));
        if (!item.any) return;
        split = item.split, tile = item.tile, head = item.head;
        row0 = item.row0, n_q = item.n_q, len = item.len;
        usable = item.usable;
        part = ((static_cast<uint32_t>(len) + item.splits - 1) / item.splits + kKeys - 1) / kKeys * kKeys;
        last_part = split + 1 == item.splits;
        const int32_t seq = item.seq;
        if (!usable && tid == 0) atomicOr(a.err, kErrIndex);
        kv.kv = a.kv;
        kv.table = a.kv.table + static_cast<uint64_t>(usable ? seq : 0) * a.kv.max_pages;
        kv.page_step = (static_cast<uint64_t>(a.n_kv) * a.dim) << a.kv.shift;
        const uint64_t off = a.layer_off + ((static_cast<uint64_t>(head) * a.dim) << a.kv.shift);
        kv.k = static_cast<const typename M::kelem*>(a.k) + off;
        kv.v = static_cast<const typename M::kelem*>(a.v) + off;
    } else {
        // the last tiles see the most keys: they start first
        const uint32_t id = a.first + blockIdx.x, piece = id / a.n_kv;
        head = id % a.n_kv;
        split = piece % a.n_splits;
        tile = a.n_tiles - 1 - piece / a.n_splits;
        kv.k = static_cast<const typename M::kelem*>(a.k) + static_cast<uint64_t>(head) * a.dim;
        kv.v = static_cast<const typename M::kelem*>(a.v) + static_cast<uint64_t>(head) * a.dim;
        kv.k_stride = a.k_stride, kv.v_stride = a.v_stride;
    }
    kv.dim = a.dim;
    const uint32_t n_m = static_cast<uint32_t>(n_q) * a.group;

    if constexpr (PAGED) past_rows<M>(a, tile, 128, n_m, row0, head, split);
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
            const uint32_t lo = first_unended(a.n_batch, [&](uint32_t x) { return a.cu[x + 1] <= static_cast<int32_t>(i); });
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
    // ---- what the workgroup sees, [k_lo, k_end), and what every real row of the wave sees whole
    int32_t k_lo, k_end, all_lo, all_hi;
    if (tid == 0) sh_bad = 0;
    if constexpr (PAGED) {
        const uint32_t m0 = tile * 128 + __builtin_amdgcn_readfirstlane(wave) * 32;
        const uint32_t m1 = tile * 128 + 128 < n_m ? tile * 128 + 127 : n_m - 1;
        const int64_t c0 = static_cast<int64_t>(split) * part, c1 = c0 + part;
        const int32_t base = len - n_q;
        k_lo = static_cast<int32_t>(c0 < len ? c0 : len);
        k_end = usable ? (a.tree ? len : base + static_cast<int32_t>(m1 / a.group) + 1) : 0;
        if (!last_part && k_end > c1) k_end = static_cast<int32_t>(c1);
        all_lo = 0;
        all_hi = a.tree ? base - 1 : base + static_cast<int32_t>(m0 / a.group);
    } else {
        const bool sees_any = view.lo <= view.hi;
        int32_t w_lo = sees_any ? view.lo : 0x7FFFFFFF, w_hi = sees_any ? view.hi : -1;
        all_lo = sees_any || !real ? view.lo : 0x7FFFFFFF;
        all_hi = real ? view.hi : 0x7FFFFFFF;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) {
            const int32_t x = __shfl_xor(w_lo, s, 64), y = __shfl_xor(w_hi, s, 64);
            const int32_t z = __shfl_xor(all_lo, s, 64), w = __shfl_xor(all_hi, s, 64);
            w_lo = x < w_lo ? x : w_lo, w_hi = y > w_hi ? y : w_hi;
            all_lo = z > all_lo ? z : all_lo, all_hi = w < all_hi ? w : all_hi;
        }
        if (lane == 0) sh_lo[wave] = w_lo, sh_hi[wave] = w_hi;
        __syncthreads();
        int32_t lo = sh_lo[0], hi = sh_hi[0];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            lo = sh_lo[w] < lo ? sh_lo[w] : lo;
            hi = sh_hi[w] > hi ? sh_hi[w] : hi;
        }
        k_lo = __builtin_amdgcn_readfirstlane(lo), k_end = __builtin_amdgcn_readfirstlane(hi) + 1;
        all_lo = __builtin_amdgcn_readfirstlane(all_lo), all_hi = __builtin_amdgcn_readfirstlane(all_hi);
        if (a.n_splits > 1 && k_lo < k_end) {
            const uint32_t n = static_cast<uint32_t>(k_end - k_lo);
            part = ((n + a.n_splits - 1) / a.n_splits + kKeys - 1) / kKeys * kKeys;
            const int64_t p0 = static_cast<int64_t>(k_lo & ~(kKeys - 1)) + static_cast<int64_t>(split) * part;
            const int64_t p1 = split + 1 < a.n_splits ? p0 + part : k_end;
            k_lo = p0 > k_lo ? static_cast<int32_t>(p0 < k_end ? p0 : k_end) : k_lo;
            k_end = p1 < k_end ? static_cast<int32_t>(p1) : k_end;
        }
    }
    RowState<M> st;
    st.clear();
    const int32_t k_begin = k_lo & ~(kKeys - 1);
    const int32_t n_tiles = k_begin < k_end ? (k_end - k_begin + kKeys - 1) / kKeys : 0;

    // ---- staging
    u32x4a rk[B::kLoads], rv[B::kLoads];
    bool bad = false;
    auto load_pages = [&](int32_t t) -> int32_t {  // threads 0 .. kKeys / 8: of eight keys each
        int32_t p = 0;
        if constexpr (PAGED) {
            const int32_t slot = k_begin + t * kKeys + static_cast<int32_t>(tid) * 8;
            if (tid < kKeys / 8 && slot < k_end) p = kv.entry_of(static_cast<uint32_t>(slot));
        }
        return p;
    };
    auto store_pages = [&](int32_t t, int32_t p) {
        if constexpr (PAGED)
            if (tid < kKeys / 8) ring[t & 3][tid] = kv.checked(p, bad);
    };
    // Load x of a wave takes kPer keys of a tile, which lie in one group of eight: the address is
    // uniform in the wave but for the lane's place, the same for all x.
    const uint32_t w_key = __builtin_amdgcn_readfirstlane(wave) * R::kPer;
    const uint32_t k_row = static_cast<uint32_t>(PAGED ? a.dim : kv.k_stride) * R::kEs;  // bytes
    const uint32_t v_row = static_cast<uint32_t>(PAGED ? a.dim : kv.v_stride) * R::kEs;
    // lanes past a row's last unit take one again, and store it again
    const uint32_t l_unit = lane % R::kLanes, l_key = lane / R::kLanes;
    const uint32_t unit = l_unit < R::kUnits ? l_unit : l_unit - (R::kLanes - R::kUnits);
    // a unit behind the head's last dimension reads nothing, wherever its row is
    const bool inside = unit * (16 / R::kEs) < a.dim;
    const uint32_t k_place = inside ? l_key * k_row + unit * 16 : kNowhere;
    const uint32_t v_place = inside ? l_key * v_row + unit * 16 : kNowhere;
    // K (V) of tile t to registers; zeros behind the last key
    auto load = [&](u32x4a* r, const typename M::kelem* base, uint64_t stride, uint32_t row, uint32_t at_lane, int32_t t) {
        const int32_t t0 = k_begin + t * kKeys;
        if constexpr (PAGED) {
#pragma unroll
            for (int x = 0; x < B::kLoads; ++x) {
                const uint32_t key = x * 4 * R::kPer + w_key;
                const int32_t left = k_end - t0 - static_cast<int32_t>(key);  // keys from this one on
                const uint32_t bytes = __builtin_amdgcn_readfirstlane(left < 0 ? 0 : (left > 8 ? 8 : left)) * row;
                const uint64_t at = kv.paged_at(__builtin_amdgcn_readfirstlane(ring[t & 3][key >> 3]),
                                                static_cast<uint32_t>(t0) + key);
                r[x] = buffer_unit(buffer_of(base + at, bytes), at_lane);
            }
        } else {
            const int32_t left = k_end - t0;
            // (to a scalar register: the clamp is a vector instruction)
            const uint32_t rows = __builtin_amdgcn_readfirstlane(left < 0 ? 0 : (left > kKeys ? kKeys : left));
            const auto b = buffer_of(base + static_cast<uint64_t>(t0) * stride, rows * row);
#pragma unroll
            for (int x = 0; x < B::kLoads; ++x) r[x] = buffer_unit(b, at_lane + (x * 4 * R::kPer + w_key) * row);
        }
    };
    auto load_k = [&](int32_t t) { load(rk, kv.k, kv.k_stride, k_row, k_place, t); };
    auto load_v = [&](int32_t t) { load(rv, kv.v, kv.v_stride, v_row, v_place, t); };
    auto load_tile = [&](int32_t t) {  // both of a tile that there is
        const int32_t t0 = k_begin + t * kKeys;
        if constexpr (PAGED) {
#pragma unroll
            for (int x = 0; x < B::kLoads; ++x) {
                const uint32_t key = x * 4 * R::kPer + w_key;
                const int32_t left = k_end - t0 - static_cast<int32_t>(key);
                const uint32_t bytes = left > 0 ? (left < 8 ? left : 8) * k_row : 0;
                const uint64_t at = kv.paged_at(__builtin_amdgcn_readfirstlane(ring[t & 3][key >> 3]),
                                                static_cast<uint32_t>(t0) + key);
                rk[x] = buffer_unit(buffer_of(kv.k + at, bytes), k_place);
                rv[x] = buffer_unit(buffer_of(kv.v + at, bytes), k_place);
            }
        } else {
            const int32_t left = k_end - t0;
            const uint32_t rows = left > kKeys ? kKeys : left;
            const auto kb = buffer_of(kv.k + static_cast<uint64_t>(t0) * kv.k_stride, rows * k_row);
            const auto vb = buffer_of(kv.v + static_cast<uint64_t>(t0) * kv.v_stride, rows * v_row);
#pragma unroll
            for (int x = 0; x < B::kLoads; ++x) {
                const uint32_t key = x * 4 * R::kPer + w_key;
                rk[x] = buffer_unit(kb, k_place + key * k_row);
                rv[x] = buffer_unit(vb, v_place + key * v_row);
            }
        }
    };
    const uint32_t place = unit * (16 / R::kEs * R::kLs);
    const uint32_t k_at = (wave * R::kPer + l_key) * R::kK + place, v_at = (wave * R::kPer + l_key) * R::kV + place;
    auto store_unit = [&](char* to, u32x4a x) {
        if constexpr (KT == kDtF32x3) {
            const f32x4 y = __builtin_bit_cast(f32x4, x);
            float rest[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const uint32_t a = take_bf16(rest[0], rest[1]), b = take_bf16(rest[2], rest[3]);
                *reinterpret_cast<uint2*>(to + p * R::kPart) = uint2{a, b};
            }
        } else {
            *reinterpret_cast<u32x4a*>(to) = x;
        }
    };
    auto store_k = [&](int buf, int x) { store_unit(lds_k[buf] + k_at + x * 4 * R::kPer * R::kK, rk[x]); };
    auto store_v = [&](int buf, int x) { store_unit(lds_v[buf] + v_at + x * 4 * R::kPer * R::kV, rv[x]); };
    auto store_tile = [&](int buf) {
#pragma unroll
        for (int x = 0; x < B::kLoads; ++x) {
            store_k(buf, x);
            store_v(buf, x);
        }
    };
    const uint32_t k_first = M::k_first(lane), v_first = M::v_first(lane);
    Scores<M> sc[2];
    auto mask = [&](Scores<M>& cur, int32_t key0) {
        uint32_t hh = h;
        asm volatile("" : "+v"(hh));  // nothing of the few masked tiles is kept over the turns
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int32_t key = key0 + static_cast<int32_t>(M::key_of(0, r, hh));
            if (!(view.sees(key) & (key >= k_lo) & (key < k_end))) cur.s[0][r] = -kInf;
        }
    };
    // One softmax step: 32 keys' scores `cur` weighted and multiplied with their values, and the
    // next 32 keys' scores computed on the way, so that arithmetic runs in the shadow of products.
    // 16-bit fragments are read well ahead of the products that take them, keys a step (`keys`
    // holds the next 32's, and then those at k_after), values half a step; without the scheduling
    // barriers the compiler moves the reads back to their products, and each waits for LDS. The
    // workgroup meets where the step's last values have been read.
    constexpr bool kAhead = !M::kFloat && M::kKvParts == 1 && (M::kParts == 1 || DT <= 128);
    Keys<M> keys;
    auto step = [&](Scores<M>& cur, Scores<M>& next, const char* v, const char* k) {
        Weights<M> w0, w1;
        if constexpr (kAhead) {
            Values<M> v0, v1;
            take_top<M>(st, cur, scale);
            const float off = M::kShift - st.reference();
            read_values<M>(v0, v, 0);
            __builtin_amdgcn_sched_barrier(0);
            score<M>(next, q, keys);
            weigh<M>(w0, st, cur, 0, scale, off);
            __builtin_amdgcn_sched_barrier(0);
            read_values<M>(v1, v, 1);
            add_values<M>(st, w0, v0);
            weigh<M>(w1, st, cur, 1, scale, off);
            __syncthreads();
            read_keys<M>(keys, k);
            __builtin_amdgcn_sched_barrier(0);
            add_values<M>(st, w1, v1);
        } else {
            take_top<M>(st, cur, scale);
            const float off = M::kShift - st.reference();
            score_rows<M>(next, q, k);
            weigh<M>(w0, st, cur, 0, scale, off);
            value_rows<M>(st, w0, v, 0);
            weigh<M>(w1, st, cur, 1, scale, off);
            value_rows<M>(st, w1, v, 1);
        }
    };
    if constexpr (M::kKvParts == 3) {
        // K runs a tile ahead of V: a turn multiplies tile t's values and tile t + 1's keys, and
        // writes the parts of tile t + 1's values and tile t + 2's keys, all of it independent,
        // so that it meets once. The turn goes by groups of the six products of three fragments,
        // the next group's fragments read ahead; splitting and softmax are dealt out between
        // the groups, in the shadow of their products. A turn of 192 dimensions takes 8470 cycles of
        // which the products are 4608: a wave alone on its SIMD issues some 1000 instructions in it,
        // and waits for loads (1300 less without them). Float products would take 12288.
        if (n_tiles) {
            if constexpr (PAGED) {
                int32_t p[4];
#pragma unroll
                for (int32_t t = 0; t < 4; ++t) p[t] = load_pages(t);
#pragma unroll
                for (int32_t t = 0; t < 4; ++t) store_pages(t, p[t]);
                __syncthreads();
            }
            load_tile(0);
            M::settle(q);
            store_tile(0);
            load_k(1);
#pragma unroll
            for (int x = 0; x < B::kLoads; ++x) store_k(1, x);
            load_k(2);
            load_v(1);
        }
        __syncthreads();
        if (n_tiles) score_rows<M>(sc[0], q, lds_k[0] + k_first);
        constexpr int kGroups = M::kSteps + 2 * M::kOut;
        for (int32_t t = 0; t < n_tiles; ++t) {
            const int32_t k0 = k_begin + t * kKeys;
            if (k0 < all_lo || k0 + kKeys - 1 > all_hi || k0 < k_lo || k0 + kKeys > k_end) mask(sc[0], k0);
            const int32_t ahead = load_pages(t + 4);
            const char* k = lds_k[(t + 1) & 1] + k_first;
            const char* v = lds_v[t & 1] + v_first;
            typename M::frag f[2][3];
            auto read = [&](typename M::frag* to, int g) {
                const int d = (g - M::kSteps) % M::kOut, half = (g - M::kSteps) / M::kOut;
#pragma unroll
                for (int x = 0; x < 3; ++x)
                    to[x] = g < M::kSteps ? M::lds_k(k, g, x) : M::lds_v(v + M::kStep * half * R::kV, d, x);
            };
            Weights<M> w[2];
            read(f[0], 0);
            take_top<M>(st, sc[0], scale);
            const float off = M::kShift - st.reference();
            sc[1].s[0] = M::zero();
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                if (g + 1 < kGroups) read(f[(g + 1) & 1], g + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 2; x >= 0; --x)
#pragma unroll
                    for (int p = 2 - x; p >= 0; --p) {
                        if (g < M::kSteps) sc[1].s[0] = M::mma(f[g & 1][x], q.f[p][g], sc[1].s[0]);
                        else st.o[(g - M::kSteps) % M::kOut] = M::mma(f[g & 1][x], w[(g - M::kSteps) / M::kOut].f[p],
                                                                     st.o[(g - M::kSteps) % M::kOut]);
                    }
#pragma unroll
                for (int x = 0; x < B::kLoads; ++x) {
                    if (g == x * M::kSteps / B::kLoads) store_k(t & 1, x);
                    if (g == M::kSteps + x * 2 * M::kOut / B::kLoads) store_v((t + 1) & 1, x);
                }
                if (g == M::kSteps / 2) weigh<M>(w[0], st, sc[0], 0, scale, off);
                if (g == M::kSteps - 1) load_k(t + 3);
                if (g == M::kSteps) weigh<M>(w[1], st, sc[0], 1, scale, off);
                __builtin_amdgcn_sched_barrier(0);
            }
            sc[0] = sc[1];
            load_v(t + 2);
            store_pages(t + 4, ahead);
            __syncthreads();
        }
    } else {
        // Tile t lies in LDS buffer t % 2, tile t + 1 in registers, and the scores of tile t's first
        // 32 keys are there.
        if (n_tiles) {
            if constexpr (PAGED) {
                const int32_t p0 = load_pages(0), p1 = load_pages(1), p2 = load_pages(2);
                store_pages(0, p0);
                store_pages(1, p1);
                store_pages(2, p2);
                __syncthreads();
            }
            load_tile(0);
            M::settle(q);
            store_tile(0);
            if (n_tiles > 1) load_tile(1);
        }
        __syncthreads();
        if (n_tiles) {
            const char* k = lds_k[0] + k_first;
            if constexpr (kAhead) {
                read_keys<M>(keys, k);
                score<M>(sc[0], q, keys);
                read_keys<M>(keys, k + 32 * R::kK);
            } else {
                score_rows<M>(sc[0], q, k);
            }
        }
        for (int32_t t = 0; t < n_tiles; ++t) {
            int32_t ahead = 0;
            if (PAGED && t + 3 < n_tiles) ahead = load_pages(t + 3);
            if (t + 1 < n_tiles) store_tile((t + 1) & 1);
            if (t + 2 < n_tiles) load_tile(t + 2);
            const int32_t k0 = k_begin + t * kKeys;
            const bool masked = k0 < all_lo || k0 + kKeys - 1 > all_hi || k0 < k_lo || k0 + kKeys > k_end;
            const char* v = lds_v[t & 1] + v_first;
            const char* kn = lds_k[(t + 1) & 1] + k_first;  // behind the last tile: whatever is there, for scores nobody uses
            if constexpr (kAhead) {
                // the first step's meeting: tile t + 1 is in LDS; the second's: tile t is read
                if (masked) mask(sc[0], k0);
                step(sc[0], sc[1], v, kn);
                if (masked) mask(sc[1], k0 + 32);
                if constexpr (PAGED) {
                    if (t + 3 < n_tiles) store_pages(t + 3, ahead);
                }
                step(sc[1], sc[0], v + 32 * R::kV, kn + 32 * R::kK);
            } else {
                if constexpr (B::kSub == 2) {
                    if (masked) mask(sc[0], k0);
                    step(sc[0], sc[1], v, lds_k[t & 1] + k_first + 32 * R::kK);
                }
                __syncthreads();  // tile t + 1 is in LDS
                constexpr int last = B::kSub - 1, other = 1 - last;
                if (masked) mask(sc[last], k0 + 32 * last);
                step(sc[last], sc[other], v + last * 32 * R::kV, kn);
                if constexpr (B::kSub == 1) sc[0] = sc[1];
                if constexpr (PAGED) {
                    if (t + 3 < n_tiles) store_pages(t + 3, ahead);
                }
                __syncthreads();  // tile t is read
            }
        }
    }
    const AttnArgs& e = args_again();
    if (PAGED && bad) atomicOr(&sh_bad, 1);
    if (not_finite<M>(st) && lane == 0) atomicOr(&sh_bad, 2);
    __syncthreads();
    const int32_t state = sh_bad;
    if (PAGED && (!usable || (state & 1))) {
        if (tid == 0 && (state & 1)) atomicOr(e.err, kErrIndex);
        st.l = __builtin_nanf("");
#pragma unroll
        for (int d = 0; d < DT / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[d][r] = st.l;
    } else if (state) {
        // some product met an infinity or NaN: the tiles again, one at a time (see attn_careful.hpp)
        const auto* q_row = static_cast<const typename M::qelem*>(e.q) + row * e.q_stride + static_cast<uint64_t>(q_head) * e.dim;
        const bool q_odd = query_without_parts<M, KT>(q_row, e.dim);
        const float lift = lift_of<KT>(static_cast<uint32_t>(PAGED ? len : n_q));
        Specials<M> specials{};
        st.clear();
        for (int32_t t = 0; t < n_tiles; ++t) {
            __syncthreads();  // the tile before is read
            if (tid < 3) sh_odd[tid] = 0;
            store_pages(t, load_pages(t));
            __syncthreads();
            load_tile(t);
#pragma unroll
            for (int x = 0; x < B::kLoads; ++x) {
                const uint32_t key = x * 4 * R::kPer + wave * R::kPer + l_key;
                store_k(0, x);
                if (M::kParts > 1 && key_without_parts<KT>(rk[x]) != 0) atomicOr(&sh_odd[key >> 5], 1u << (key & 31));
                u32x4a marks;
                if (take_specials<KT>(rv[x], marks) != 0) sh_odd[2] = 1;
                store_values<M, KT>(lds_v[0] + v_at + x * 4 * R::kPer * R::kV, rv[x]);
                store_marks<M, KT>(lds_v[1] + v_at + x * 4 * R::kPer * R::kV, marks);
            }
            __syncthreads();
#pragma unroll 1
            for (int sub = 0; sub < kKeys / 32; ++sub) {
                const Seen seen =
                    careful_step<M>(st, q, q_row, q_odd, kv, view, k_begin + t * kKeys + 32 * sub, k_lo, k_end, sh_odd[sub], scale, lift, e.dim,
                                    lds_k[0] + k_first + sub * 32 * R::kK, lds_v[0] + v_first + sub * 32 * R::kV);
                if (sh_odd[2]) add_specials<M>(specials, seen, lds_v[1] + v_first + sub * 32 * R::kV);
            }
        }
        apply_specials<M>(st, specials);
    }
    write_rows<M, QT>(e, st, real, row, q_head, split, lane);
}

}  // namespace dev
}  // namespace objeta
