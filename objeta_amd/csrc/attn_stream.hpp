// attn_stream.hpp — attention of up to 32 rows of one sequence and key/value head over the
// cache: decode, and small trees of drafts. Bound by reading keys and values once.
//
// Every wave walks key tiles of its own (the chunk's tiles dealt out in turn) with its own
// part of LDS, so no barrier holds a wave's loads up: the next tile is in flight in registers
// while the present one is multiplied. The waves' running softmaxes are joined at the end
// through LDS. The matrix units multiply 32 rows whether or not there are as many; at 16 bits
// they would keep up with ten times the memory's rate.
#pragma once

#include "attn_tile.hpp"

namespace objeta {
namespace dev {

template <int KT, int DT>
struct Stream {
    typedef Rows<KT, DT> R;
    static constexpr int kLoads = 32 * R::kUnits / 64;  // 16-byte units of K (and of V) a lane stages
    static constexpr int kWave = 2 * 32 * R::kBytes;    // LDS of a wave: a tile of K and one of V
    static constexpr int kWaves = kWave <= 16384 ? 4 : (kWave <= 32768 ? 2 : 1);
    static_assert(kWave >= 32 * DT * 4, "o of 32 rows in a wave's part");
};

__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int QT, int KT, int DT>
__global__ __launch_bounds__((64 * Stream<KT, DT>::kWaves)) void attn_stream_kernel(AttnArgs a) {
    typedef Math<QT, KT, DT> M;
    typedef Rows<KT, DT> R;
    typedef Stream<KT, DT> S;
    constexpr int kWaves = S::kWaves;
    __shared__ alignas(16) char lds[kWaves][S::kWave];
    __shared__ float sh_m[kWaves][32], sh_l[kWaves][32];
    __shared__ int32_t sh_bad;

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const uint32_t split = blockIdx.x % a.n_splits, head = blockIdx.y, b = blockIdx.z;
    uint32_t tile = blockIdx.x / a.n_splits;
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
    char* v_lds = lds[wave] + 32 * R::kBytes;
    const uint32_t kx = M::k_first(lane), vx = M::v_first(lane);

    for (; static_cast<uint64_t>(tile) * 32 < n_m; tile += a.n_tiles) {
        const uint32_t m = tile * 32 + (lane & 31);
        const bool real = m < n_m;
        const uint32_t i = real ? m / a.group : 0, q_head = head * a.group + (real ? m % a.group : 0);
        const uint64_t row = static_cast<uint64_t>(row0) + i;
        const int32_t base = len - n_q;
        RowView view{0, -1, 0x7FFFFFFF, 0};
        if (real && usable) {
            if (a.tree) view = RowView{0, len - 1, base, a.tree[row]};
            else view.hi = base + static_cast<int32_t>(i);
        }
        typename M::frag q[DT / 16];
        const typename M::qelem* qp =
            static_cast<const typename M::qelem*>(a.q) + row * a.q_stride + static_cast<uint64_t>(q_head) * a.dim;
#pragma unroll
        for (int s = 0; s < DT / 16; ++s) {
            const uint32_t d = 16 * s + 8 * h;
            q[s] = (real && d < a.dim) ? M::load_q(qp + d) : M::zero();
        }
        if (tid == 0) sh_bad = 0;
        RowState<DT> st;
        st.clear();

        // tiles k_lo + 32 (wave + kWaves t)
        u32x4a rk[S::kLoads], rv[S::kLoads];
        bool bad = false;
        auto load_pages = [&](int32_t k0) -> int32_t {  // lane x < 4: the page of keys k0 + 8 x ..
            int32_t p = 0;
            const int32_t slot = k0 + static_cast<int32_t>(lane) * 8;
            if (lane < 4 && slot < k_end) p = kv.page_of(static_cast<uint32_t>(slot), bad);
            return p;
        };
        auto load_tile = [&](int32_t k0, int32_t pages) {
#pragma unroll
            for (int x = 0; x < S::kLoads; ++x) {
                const uint32_t u = x * 64 + lane, key = u / R::kUnits, c = u % R::kUnits;
                const int32_t page = __shfl(pages, static_cast<int>(key >> 3), 64);
                const int32_t slot = k0 + static_cast<int32_t>(key);
                rk[x] = u32x4a{0, 0, 0, 0};
                rv[x] = u32x4a{0, 0, 0, 0};
                if (slot < k_end && c * (16 / R::kEs) < a.dim) {
                    const uint64_t at = kv.paged_at(page, static_cast<uint32_t>(slot)) + c * (16 / R::kEs);
                    rk[x] = *reinterpret_cast<const u32x4a*>(kv.k + at);
                    rv[x] = *reinterpret_cast<const u32x4a*>(kv.v + at);
                }
            }
        };
        const int32_t step = 32 * kWaves;
        int32_t k0 = k_lo + 32 * static_cast<int32_t>(wave);
        int32_t pages = 0;
        if (k0 < k_end) {
            load_tile(k0, load_pages(k0));
            if (k_end - k0 > step) pages = load_pages(k0 + step);
        }
        for (; k0 < k_end; k0 = k_end - k0 > step ? k0 + step : k_end) {
#pragma unroll
            for (int x = 0; x < S::kLoads; ++x) {
                const uint32_t u = x * 64 + lane, key = u / R::kUnits, c = u % R::kUnits;
                *reinterpret_cast<u32x4a*>(k_lds + key * R::kBytes + ((c ^ R::swz_k(key)) << 4)) = rk[x];
                *reinterpret_cast<u32x4a*>(v_lds + key * R::kBytes + ((c ^ R::swz_v(key)) << 4)) = rv[x];
            }
            if (k_end - k0 > step) {
                load_tile(k0 + step, pages);
                if (k_end - k0 > 2 * step) pages = load_pages(k0 + 2 * step);
            }
            wave_lds_fence();
            f32x16 s[1];
            s[0] = scores<M, DT>(q, k_lds, lane, kx);
            if (a.tree || k0 + 32 > base + 1 || k0 + 32 > k_end) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int32_t key = k0 + (r & 3) + 8 * (r >> 2) + 4 * static_cast<int32_t>(h);
                    if (!(view.sees(key) && key < k_end)) s[0][r] = -kInf;
                }
            }
            accumulate<M, DT, 1>(st, s, a.scale_log2, v_lds, vx);
            wave_lds_fence();
        }

        // ---- the waves' results into one: a wave's o goes to its own part of LDS
        st.l += other_half(st.l);
        if (h == 0) sh_m[wave][lane] = st.m, sh_l[wave][lane] = st.l;
        __syncthreads();
        if (bad) atomicOr(&sh_bad, 1);
        float top = sh_m[0][lane & 31];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, sh_m[w][lane & 31]);
        const float ref = top == -kInf ? 0.0f : top;
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) l += sh_l[w][lane & 31] * exp2_hw(sh_m[w][lane & 31] - ref);
        const float f = exp2_hw(st.m - ref);
        const bool odd = not_finite<DT>(st);
        if (odd && lane == 0) atomicOr(&sh_bad, 2);
        float* o_lds = reinterpret_cast<float*>(lds[wave]);  // [dimension / 4][row][4]
#pragma unroll
        for (int d = 0; d < DT / 32; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f32x4*>(o_lds + ((8 * d + 2 * r + h) * 32 + (lane & 31)) * 4) =
                    f32x4{st.o[d][4 * r] * f, st.o[d][4 * r + 1] * f, st.o[d][4 * r + 2] * f, st.o[d][4 * r + 3] * f};
        __syncthreads();
        const int32_t state = sh_bad;
        if (usable && state == 2) {
            // some product met an infinity or NaN: the rows again, key by key (see row_by_row)
            for (uint32_t r = wave; r < 32; r += kWaves) {
                const uint32_t r_m = tile * 32 + r;
                if (r_m >= n_m) break;
                const uint32_t r_head = head * a.group + r_m % a.group, r_i = r_m / a.group;
                const uint64_t r_row = static_cast<uint64_t>(row0) + r_i;
                RowView rv1{0, base + static_cast<int32_t>(r_i), 0x7FFFFFFF, 0};
                if (a.tree) rv1 = RowView{0, len - 1, base, a.tree[r_row]};
                float rm, rl, ro[4];
                row_by_row<M, true, KT>(kv,
                                        static_cast<const typename M::qelem*>(a.q) + r_row * a.q_stride +
                                            static_cast<uint64_t>(r_head) * a.dim,
                                        rv1, k_lo, k_end, a.scale_log2, a.dim, rm, rl, ro);
                write_row<M>(a, rm, rl, ro, r_row, r_head, split, lane);
            }
        } else {
            if (tid == 0 && (state & 1)) atomicOr(a.err, kErrIndex);
            const bool poison = !usable || (state & 1);
            if (poison) l = __builtin_nanf("");
            const float inv = a.n_splits > 1 ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
            // this thread: row lane % 32, groups of four dimensions
            for (uint32_t g = wave * 2 + h; g * 4 < a.dim; g += 2 * kWaves) {
                f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kWaves; ++w)
                    sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[w]) +
                                                           (g * 32 + (lane & 31)) * 4);
                sum *= inv;
                if (poison) sum = f32x4{l, l, l, l};
                if (!real) continue;
                if (a.n_splits > 1)
                    *reinterpret_cast<f32x4*>(a.part + part_at(a, split, row, q_head) * a.dim + 4 * g) = sum;
                else
                    store_out<QT>(static_cast<typename M::qelem*>(a.out) + row * a.out_stride +
                                      static_cast<uint64_t>(q_head) * a.dim + 4 * g, sum);
            }
            if (real && wave == 0 && h == 0) {
                if (a.n_splits > 1) {
                    const uint64_t at = part_at(a, split, row, q_head);
                    a.part_ml[2 * at] = top - M::kShift;
                    a.part_ml[2 * at + 1] = l;
                } else if (a.lse) {
                    a.lse[row * a.n_heads + q_head] =
                        l == 0.0f ? -kInf : (top - M::kShift + __builtin_amdgcn_logf(l)) * kLn2;
                }
            }
        }
        __syncthreads();  // LDS is used again
    }
}

}  // namespace dev
}  // namespace objeta
