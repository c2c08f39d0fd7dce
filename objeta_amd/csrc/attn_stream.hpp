// attn_stream.hpp — attention of up to 16 or 32 rows of one sequence and key/value head over
// the cache: decode, and small trees of drafts. Bound by reading keys and values once.
//
// Every wave walks key tiles of its own (the chunk's tiles dealt out in turn) with its own
// part of LDS, so no barrier holds a wave's loads up: the next tile is in flight in registers
// while the present one is multiplied. The waves' running softmaxes are joined at the end
// through LDS. The matrix units multiply 16 or 32 rows whether or not there are as many; at
// 16 bits they would keep up with ten times the memory's rate.
#pragma once

#include "attn_careful.hpp"

namespace objeta {
namespace dev {

// WIDE: twice the waves, for few workgroups that each have a CU to themselves (517 keys of one
// sequence in one piece, bf16: 8.9 us against 10.4), where more would wait for one another (32
// sequences of 301 to 8192: 46.5 against 42.6).
template <int KT, int DT, int ROWS, bool WIDE>
struct Stream {
    typedef Rows<KT, DT, ROWS> R;
    static constexpr int kLoads = 32 / R::kPer;                // 16-byte units of K (and of V) a lane stages
    static constexpr int kWave = 32 * (R::kK + R::kV);         // LDS of a wave: a tile of K and one of V
    static constexpr int kWaves = stream_waves(DT * R::kEs) * (WIDE ? 2 : 1);
    static_assert(kWave >= ROWS * DT * 4, "o of a wave's rows in its part");
    // waves a SIMD: two where a wave's part of LDS lets eight be on a CU
    static constexpr int kPerSimd = DT * R::kEs <= 256 ? 2 : 1;
};

__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// (32 rows of 64 f16 dimensions fit three waves a SIMD, 168 registers, only if told to: 170 else)
template <int QT, int KT, int DT, int ROWS, bool WIDE>
__global__ __launch_bounds__((64 * Stream<KT, DT, ROWS, WIDE>::kWaves),
                             (ROWS == 32 ? (KT == kDtF16 && DT == 64 ? 3 : 1) : Stream<KT, DT, ROWS, WIDE>::kPerSimd)) void attn_stream_kernel(AttnArgs a) {
    typedef Math<QT, KT, DT, ROWS> M;
    typedef Rows<KT, DT, ROWS> R;
    typedef Stream<KT, DT, ROWS, WIDE> S;
    constexpr int kWaves = S::kWaves;
    __shared__ alignas(16) char lds[kWaves][S::kWave];
    __shared__ float sh_m[kWaves][ROWS], sh_l[kWaves][ROWS];
    __shared__ int32_t sh_bad;

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane / ROWS, mine = lane % ROWS;
    const StreamItem item(a, a.first + blockIdx.x);
    if (!item.any) return;
    const uint32_t split = item.split, head = item.head, b = item.b, tile = 0;
    const int32_t row0 = a.cu[b], end = a.cu[b + 1], n_q = end - row0;
    if (row0 < 0 || end < row0 || static_cast<uint32_t>(end) > a.n_rows) {
        if (tid == 0) atomicOr(a.err, kErrIndex);
        return;
    }
    const int32_t seq = a.seqs[b];
    bool usable = seq_ok(a.kv, seq);
    int32_t len = usable ? a.kv.lens[seq] : 0;
    usable = usable && len_ok(a.kv, len) && n_q <= len && (!a.tree || n_q <= 64);
    if (!usable) len = 0;
    if (!usable && tid == 0 && n_q) atomicOr(a.err, kErrIndex);
    if (split && static_cast<uint64_t>(split) * a.chunk >= static_cast<uint64_t>(len)) return;
    KvRows<true, KT> kv;
    kv.kv = a.kv;
    kv.table = a.kv.table + static_cast<uint64_t>(usable ? seq : 0) * a.kv.max_pages;
    kv.page_step = (static_cast<uint64_t>(a.n_kv) * a.dim) << a.kv.shift;
    kv.dim = a.dim;
    const uint64_t off = a.layer_off + ((static_cast<uint64_t>(head) * a.dim) << a.kv.shift);
    kv.k = static_cast<const typename M::kelem*>(a.k) + off;
    kv.v = static_cast<const typename M::kelem*>(a.v) + off;
    const uint32_t n_m = static_cast<uint32_t>(n_q) * a.group;
    const int64_t c0 = static_cast<int64_t>(split) * a.chunk;
    const int32_t k_lo = static_cast<int32_t>(c0);
    const int32_t k_end = split + 1 < a.n_splits && c0 + a.chunk < len ? static_cast<int32_t>(c0 + a.chunk) : len;
    char* k_lds = lds[wave];
    char* v_lds = lds[wave] + 32 * R::kK;

    past_rows<M>(a, tile, ROWS, n_m, row0, head, split);
    if (static_cast<uint64_t>(tile) * ROWS >= n_m) return;
    const uint32_t m = tile * ROWS + mine;
    const bool real = m < n_m;
    const uint32_t i = real ? m / a.group : 0, q_head = head * a.group + (real ? m % a.group : 0);
    const uint64_t row = static_cast<uint64_t>(row0) + i;
    const int32_t base = len - n_q;
    RowView view{0, -1, 0x7FFFFFFF, 0};
    if (real && usable) {
        if (a.tree) view = RowView{0, len - 1, base, a.tree[row]};
        else view.hi = base + static_cast<int32_t>(i);
    }
    typename M::Query q;
    float scale = a.scale_log2;
    M::load_q(q, static_cast<const typename M::qelem*>(a.q) + row * a.q_stride + static_cast<uint64_t>(q_head) * a.dim, real,
              a.dim, lane, scale);
    M::settle(q);
    if (tid == 0) sh_bad = 0;
    RowState<M> st;
    st.clear();

    // tiles k_lo + 32 (wave + kWaves t)
    u32x4a rk[S::kLoads], rv[S::kLoads];
    bool bad = false;
    auto load_pages = [&](int32_t k0) -> int32_t {  // lane x < 4: the page of keys k0 + 8 x ..
        int32_t p = 0;
        const int32_t slot = k0 + static_cast<int32_t>(lane) * 8;
        if (lane < 4 && slot < k_end) p = kv.entry_of(static_cast<uint32_t>(slot));
        return p;
    };
    // Load x takes the keys x kPer .. of a tile, which lie in one group of eight, so in one page:
    // the address is uniform but for the lane's place, the same for all x.
    const uint32_t row_bytes = a.dim * R::kEs, unit = lane % R::kLanes;
    const uint32_t place = unit * (16 / R::kEs) < a.dim ? lane / R::kLanes * row_bytes + unit * 16 : kNowhere;
    auto load_tile = [&](int32_t k0, int32_t pages) {
#pragma unroll
        for (int x = 0; x < S::kLoads; ++x) {
            const uint32_t key = x * R::kPer;
            const int32_t left = k_end - k0 - static_cast<int32_t>(key);  // keys from this one on
            const uint32_t bytes = left > 0 ? (left < 8 ? left : 8) * row_bytes : 0;
            const uint64_t at = kv.paged_at(__builtin_amdgcn_readlane(pages, key >> 3), static_cast<uint32_t>(k0) + key);
            rk[x] = buffer_unit(buffer_of(kv.k + at, bytes), place);
            rv[x] = buffer_unit(buffer_of(kv.v + at, bytes), place);
        }
    };
    const uint32_t k_at = lane / R::kLanes * R::kK + unit * 16, v_at = lane / R::kLanes * R::kV + unit * 16;
    const int32_t step = 32 * kWaves;
    int32_t k0 = k_lo + 32 * static_cast<int32_t>(__builtin_amdgcn_readfirstlane(wave));
    int32_t pages = 0;
    if (k0 < k_end) {
        pages = load_pages(k0);
        const int32_t first = kv.checked(pages, bad);
        if (k_end - k0 > step) pages = load_pages(k0 + step);
        load_tile(k0, first);
    }
    for (; k0 < k_end; k0 = k_end - k0 > step ? k0 + step : k_end) {
        if (R::kLanes == R::kUnits || unit < R::kUnits) {
#pragma unroll
            for (int x = 0; x < S::kLoads; ++x) {
                *reinterpret_cast<u32x4a*>(k_lds + k_at + x * R::kPer * R::kK) = rk[x];
                *reinterpret_cast<u32x4a*>(v_lds + v_at + x * R::kPer * R::kV) = rv[x];
            }
        }
        if (k_end - k0 > step) {
            const int32_t now = kv.checked(pages, bad);
            if (k_end - k0 > 2 * step) pages = load_pages(k0 + 2 * step);
            load_tile(k0 + step, now);
        }
        wave_lds_fence();
        Scores<M> s;
        score_rows<M>(s, q, k_lds + M::k_first(lane));
        if (a.tree || k0 + 32 > base + 1 || k0 + 32 > k_end) {
#pragma unroll
            for (int n = 0; n < M::kKeyTiles; ++n)
#pragma unroll
                for (int r = 0; r < M::kRegs; ++r) {
                    const int32_t key = k0 + static_cast<int32_t>(M::key_of(n, r, h));
                    if (!(view.sees(key) & (key < k_end))) s.s[n][r] = -kInf;
                }
        }
        take_top<M>(st, s, scale);
        const float off = M::kShift - st.reference();
#pragma unroll
        for (int g = 0; g < kGroups<M>; ++g) {
            Weights<M> w;
            weigh<M>(w, st, s, g, scale, off);
            value_rows<M>(st, w, v_lds + M::v_first(lane), g);
        }
        wave_lds_fence();
    }

    const AttnArgs& e = args_again();
    // ---- the waves' results into one: a wave's o goes to its own part of LDS
    float top, l;
    auto meet = [&]() -> int32_t {
        st.l = row_sum<ROWS>(st.l);
        if (h == 0) sh_m[wave][mine] = st.m, sh_l[wave][mine] = st.l;
        __syncthreads();
        if (bad) atomicOr(&sh_bad, 1);
        top = sh_m[0][mine];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, sh_m[w][mine]);
        const float ref = top == -kInf ? 0.0f : top;
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) l += sh_l[w][mine] * exp2_hw(sh_m[w][mine] - ref);
        const float f = exp2_hw(st.m - ref);
        if (not_finite<M>(st) && lane == 0) atomicOr(&sh_bad, 2);
        float* o_lds = reinterpret_cast<float*>(lds[wave]);  // [dimension / 4][row][4]
#pragma unroll
        for (int d = 0; d < M::kOut; ++d)
#pragma unroll
            for (int r = 0; r < M::kRegs / 4; ++r)
                *reinterpret_cast<f32x4*>(o_lds + (out_dim<M>(d, r, h) / 4 * ROWS + mine) * 4) =
                    f32x4{st.o[d][4 * r] * f, st.o[d][4 * r + 1] * f, st.o[d][4 * r + 2] * f, st.o[d][4 * r + 3] * f};
        __syncthreads();
        return sh_bad;
    };
    const int32_t state = meet();
    if (usable && state == 2) {
        // some product met an infinity or NaN: the wave's tiles again, one at a time (see
        // attn_careful.hpp). The others' parts of LDS are not read before the next meeting.
        const auto* q_row = static_cast<const typename M::qelem*>(e.q) + row * e.q_stride + static_cast<uint64_t>(q_head) * e.dim;
        const bool q_odd = query_without_parts<M, KT>(q_row, e.dim);
        const float lift = lift_of<KT>(static_cast<uint32_t>(len));
        Specials<M> specials{};
        st.clear();
        for (int32_t t0 = k_lo + 32 * static_cast<int32_t>(__builtin_amdgcn_readfirstlane(wave)); t0 < k_end;
             t0 = k_end - t0 > step ? t0 + step : k_end) {
            const int32_t t_pages = kv.checked(load_pages(t0), bad);
            // two units of K and V at a time, for the registers' sake
            auto unit_of = [&](const typename M::kelem* pool, uint32_t x) {
                const uint32_t key = x * R::kPer;
                const int32_t left = k_end - t0 - static_cast<int32_t>(key);
                const uint32_t bytes = left > 0 ? (left < 8 ? left : 8) * row_bytes : 0;
                const uint64_t at = kv.paged_at(__builtin_amdgcn_readlane(t_pages, key >> 3), static_cast<uint32_t>(t0) + key);
                return buffer_unit(buffer_of(pool + at, bytes), place);
            };
            uint32_t odd = 0, marked = 0;
            wave_lds_fence();  // the tile before is read
#pragma unroll 1
            for (uint32_t x = 0; x < static_cast<uint32_t>(S::kLoads); x += 2) {
                u32x4a uk[2], uv[2], marks;
#pragma unroll
                for (uint32_t y = 0; y < 2; ++y) uk[y] = unit_of(kv.k, x + y), uv[y] = unit_of(kv.v, x + y);
#pragma unroll
                for (uint32_t y = 0; y < 2; ++y) {
                    if constexpr (M::kParts > 1)
                        odd |= static_cast<uint32_t>(key_without_parts<KT>(uk[y]) != 0) << ((x + y) * R::kPer + lane / R::kLanes);
                    marked |= take_specials<KT>(uv[y], marks);
                    *reinterpret_cast<u32x4a*>(k_lds + k_at + (x + y) * R::kPer * R::kK) = uk[y];
                    *reinterpret_cast<u32x4a*>(v_lds + v_at + (x + y) * R::kPer * R::kV) = uv[y];
                }
            }
#pragma unroll
            for (int y = 1; y < 64; y <<= 1) odd |= __shfl_xor(odd, y, 64);
            wave_lds_fence();
            const Seen seen = careful_step<M>(st, q, q_row, q_odd, kv, view, t0, k_lo, k_end, __builtin_amdgcn_readfirstlane(odd),
                                              scale, lift, e.dim, k_lds + M::k_first(lane), v_lds + M::v_first(lane));
            if (__any(marked != 0)) {  // the values' marks in their place
                wave_lds_fence();
#pragma unroll 1
                for (uint32_t x = 0; x < static_cast<uint32_t>(S::kLoads); x += 2) {
                    u32x4a uv[2], marks;
#pragma unroll
                    for (uint32_t y = 0; y < 2; ++y) uv[y] = unit_of(kv.v, x + y);
#pragma unroll
                    for (uint32_t y = 0; y < 2; ++y) {
                        take_specials<KT>(uv[y], marks);
                        *reinterpret_cast<u32x4a*>(v_lds + v_at + (x + y) * R::kPer * R::kV) = marks;
                    }
                }
                wave_lds_fence();
                add_specials<M>(specials, seen, v_lds + M::v_first(lane));
            }
        }
        wave_lds_fence();
        apply_specials<M>(st, specials);
        meet();
    }
    if (tid == 0 && (state & 1)) atomicOr(e.err, kErrIndex);
    const bool poison = !usable || (state & 1);
    if (poison) l = __builtin_nanf("");
    const float inv = e.n_splits > 1 ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
    // this thread: its row, groups of four dimensions
    for (uint32_t g = wave * (64 / ROWS) + h; g * 4 < e.dim; g += kWaves * (64 / ROWS)) {
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[w]) +
                                                   (g * ROWS + mine) * 4);
        sum *= inv;
        if (poison) sum = f32x4{l, l, l, l};
        if (!real) continue;
        if (e.n_splits > 1)
            *reinterpret_cast<f32x4*>(e.part + part_at(e, split, row, q_head) * e.dim + 4 * g) = sum;
        else
            store_out<QT>(static_cast<typename M::qelem*>(e.out) + row * e.out_stride +
                              static_cast<uint64_t>(q_head) * e.dim + 4 * g, sum);
    }
    if (real && wave == 0 && h == 0) {
        if (e.n_splits > 1) {
            const uint64_t at = part_at(e, split, row, q_head);
            e.part_ml[2 * at] = top - M::kShift;
            e.part_ml[2 * at + 1] = l;
        } else if (e.lse) {
            e.lse[row * e.n_heads + q_head] =
                l == 0.0f ? -kInf : (top - M::kShift + __builtin_amdgcn_logf(l)) * kLn2;
        }
    }
}

}  // namespace dev
}  // namespace objeta
