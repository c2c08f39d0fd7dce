// attn_careful.hpp — the second pass of attention over keys or values that hold infinities or NaN,
// taken by a workgroup whose first pass is not finite.
//
// The matrix products multiply a value that a row does not see by a probability of 0, which an
// infinity or NaN there turns into NaN, and take a float as parts, of which an infinity has none.
// So the second pass stages such values as zeros and marks them in a matrix of their own (1 for
// inf, 64 for -inf, 4096 for NaN): its product with the rows' masks counts, for each row and
// dimension, what of each kind the row sees among 32 keys, exactly. Scores of a key or a query that
// has no parts are computed in floats, a row a lane. m is kept above the largest score by the
// logarithm of the keys' number (values of f16, whose sums have the room: at it), so that sums of
// large finite values stay finite too, over all parts and waves.
//
// It walks the same tiles, one at a time; what it costs over the first pass is bounded by that, and
// by one row's dot product a lane for each key without parts.
#pragma once

#include "attn_tile.hpp"

namespace objeta {
namespace dev {

// The infinities and NaN of a 16-byte unit to zeros in `x` and marks in `mark`, of the same type
// (float values: floats). Not 0 where there are any. By arithmetic on whole words: a condition for
// each element would be a register pair of the few scalar ones.
template <int KT>
__device__ __forceinline__ uint32_t take_specials(u32x4a& x, u32x4a& mark) {
    constexpr bool k32 = KT == kDtF32 || KT == kDtF32x3;
    constexpr uint32_t kExp = k32 ? 0x7F800000u : (KT == kDtF16 ? 0x7C007C00u : 0x7F807F80u);
    constexpr uint32_t kSign = k32 ? 0x80000000u : 0x80008000u, kRest = ~(kExp | kSign);
    constexpr uint32_t kOne = k32 ? 0x3F800000u : (KT == kDtF16 ? 0x3C003C00u : 0x3F803F80u);
    constexpr uint32_t k64 = k32 ? 0x42800000u : (KT == kDtF16 ? 0x54005400u : 0x42804280u);
    constexpr uint32_t k4096 = k32 ? 0x45800000u : (KT == kDtF16 ? 0x6C006C00u : 0x45804580u);
    // all ones in an element whose sign bit is set
    auto whole = [](uint32_t s) { return k32 ? 0u - (s >> 31) : (s >> 15 & 0x00010001u) * 0xFFFFu; };
    // the sign bit of an element below it that is not 0
    auto some = [](uint32_t w) { return (w + ~kSign) & kSign; };
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = x[i];
        const uint32_t special = ~some((b & kExp) ^ kExp) & kSign, nan = some(b & kRest) & special, minus = b & special & ~nan;
        mark[i] = (whole(nan) & k4096) | (whole(minus) & k64) | (whole(special & ~nan & ~minus) & kOne);
        x[i] = b & ~whole(special);
        any |= special;
    }
    return any;
}

// Whether a float has no parts: infinities, NaN, and (bf16 parts) what rounds to an infinity.
template <int KT>
__device__ __forceinline__ bool no_parts(float x) {
    return (__builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu) >= (KT == kDtF16 ? 0x7F800000u : 0x7F7F8000u);
}
// Not 0 where a 16-byte unit of a key holds an element without parts.
template <int KT>
__device__ __forceinline__ uint32_t key_without_parts(const u32x4a& x) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (KT == kDtF32 || KT == kDtF32x3) {
            any |= (x[i] & 0x7FFFFFFFu) + (0x80000000u - 0x7F7F8000u);
        } else {
            constexpr uint32_t kExp = KT == kDtF16 ? 0x7C007C00u : 0x7F807F80u;
            any |= ~(((x[i] & kExp) ^ kExp) + 0x7FFF7FFFu);
        }
    }
    return any & (KT == kDtF32 || KT == kDtF32x3 ? 0x80000000u : 0x80008000u);
}

// A finite float's first bf16 part: the nearest, but for what would round to an infinity.
__device__ __forceinline__ uint32_t first_part(float x) {
    uint32_t b = __builtin_bit_cast(uint32_t, x);
    if ((b & 0x7FFFFFFFu) < 0x7F7F8000u) b += 0x7FFFu + (b >> 16 & 1);
    return b & 0xFFFF0000u;
}

// Stages a unit of finite values (marks) at `to`; float ones of the parts' kind as three bf16 parts
// (the first alone).
template <class M, int KT>
__device__ __forceinline__ void store_values(char* to, u32x4a x) {
    if constexpr (KT == kDtF32x3) {
        const f32x4 y = __builtin_bit_cast(f32x4, x);
        float rest[4];
        uint32_t top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            top[i] = first_part(y[i]);
            rest[i] = y[i] - __builtin_bit_cast(float, top[i]);
        }
        *reinterpret_cast<uint2*>(to) = uint2{top[0] >> 16 | top[1], top[2] >> 16 | top[3]};
#pragma unroll
        for (int p = 1; p < 3; ++p) {
            const uint32_t a = take_bf16(rest[0], rest[1]), b = take_bf16(rest[2], rest[3]);
            *reinterpret_cast<uint2*>(to + p * M::R::kPart) = uint2{a, b};
        }
    } else {
        *reinterpret_cast<u32x4a*>(to) = x;
    }
}
template <class M, int KT>
__device__ __forceinline__ void store_marks(char* to, u32x4a x) {
    if constexpr (KT == kDtF32x3) *reinterpret_cast<uint2*>(to) = uint2{x[0] >> 16 | x[1], x[2] >> 16 | x[3]};
    else *reinterpret_cast<u32x4a*>(to) = x;
}

// Whether this lane's row has a query without parts; asked by a whole wave.
template <class M, int KT>
__device__ __forceinline__ bool query_without_parts(const typename M::qelem* q, uint32_t dim) {
    if constexpr (M::kParts == 1) return false;
    const uint32_t lane = threadIdx.x & 63;
    bool odd = false;
#pragma unroll 4
    for (uint32_t d = lane / M::kRows; d < dim; d += 64 / M::kRows) odd |= no_parts<KT>(static_cast<float>(q[d]));
    const uint64_t rows = __ballot(odd);
    uint64_t any = 0;
#pragma unroll
    for (int y = 0; y < 64; y += M::kRows) any |= rows >> y;
    return any >> (lane % M::kRows) & 1;
}

// Scores of what has no parts: of the keys `odd` (a bit each of the 32 from key0 on, the same in all
// lanes), and of all keys for a row that is odd itself.
template <class M, bool PAGED, int KT>
__device__ __forceinline__ void patch_scores(Scores<M>& s, const KvRows<PAGED, KT>& kv, const typename M::qelem* q, bool q_odd,
                                             uint32_t dim, int32_t key0, int32_t k_end, uint32_t odd) {
    if constexpr (M::kParts > 1) {
        uint32_t h = (threadIdx.x & 63) / M::kRows;
        asm volatile("" : "+v"(h));
        bool bad = false;
        for (uint32_t todo = __any(q_odd) ? ~0u : odd; todo; todo &= todo - 1) {
            const uint32_t at = static_cast<uint32_t>(__builtin_ctz(todo));
            const int32_t key = key0 + static_cast<int32_t>(at);
            if (key < 0 || key >= k_end) continue;
            const auto* k = kv.k_row(static_cast<uint32_t>(key), bad);
            float dot = 0.0f;
#pragma unroll 1
            for (uint32_t d = 8 * h; d < dim; d += 8 * (64 / M::kRows)) {
                typedef typename M::kelem k4 __attribute__((ext_vector_type(4)));
#pragma unroll
                for (int y = 0; y < 8; y += 4) {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(q + d + y);
                    const k4 b = *reinterpret_cast<const k4*>(k + d + y);
#pragma unroll
                    for (int i = 0; i < 4; ++i) dot = __builtin_fmaf(a[i], static_cast<float>(b[i]), dot);
                }
            }
            dot = row_sum<M::kRows>(dot);
            const bool take = q_odd || (odd >> at & 1);
#pragma unroll
            for (int n = 0; n < M::kKeyTiles; ++n)
#pragma unroll
                for (int r = 0; r < M::kRegs; ++r)
                    if (take && M::key_of(n, r, h) == at) s.s[n][r] = dot;
        }
    }
}

// What of infinities and NaN a lane's row has seen: for accumulator register r of o[d] the bits
// 3 r (inf), 3 r + 1 (-inf), 3 r + 2 (NaN).
template <class M>
struct Specials {
    uint64_t f[M::kOut];
};

// Of a lane's scores of 32 keys (bit kRegs n + r): the keys that its row sees, and of these the ones
// whose score is -inf. By words: kept as conditions they would take a register pair of the few scalar
// ones each.
struct Seen {
    uint32_t keys, dead;
};

// The row's mask over group t of the keys as an operand: 1 for a key that it sees, 4096 for one whose
// score is -inf (its probability is 0, and 0 times an infinity NaN).
template <class M>
__device__ __forceinline__ void seen_weights(typename M::frag& w, const Seen& seen, int t) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int at = M::kRows == 32 ? 8 * t + j : M::kRegs * (j / 4) + j % 4;
        const float x = static_cast<float>((seen.keys >> at & 1) + (seen.dead >> at & 1) * 4095u);
        if constexpr (M::kFloat) w.v[j] = x;
        else w[j] = static_cast<typename M::pelem>(x);
    }
}
// `v`: the first row of 32 keys' marks plus v_first.
template <class M>
__device__ __forceinline__ void add_specials(Specials<M>& sp, const Seen& seen, const char* v) {
    typename M::frag w[kGroups<M>];
#pragma unroll
    for (int g = 0; g < kGroups<M>; ++g) seen_weights<M>(w[g], seen, g);
#pragma unroll
    for (int d = 0; d < M::kOut; ++d) {
        typename M::acc c = M::zero();
#pragma unroll
        for (int g = 0; g < kGroups<M>; ++g) c = M::mma(M::lds_v(v + M::kStep * g * M::R::kV, d), w[g], c);
#pragma unroll
        for (int r = 0; r < M::kRegs; ++r) {
            const uint32_t n = static_cast<uint32_t>(c[r]);  // at most 32 of each kind
            const uint32_t plus = n & 63u, minus = n >> 6 & 63u, nan = n >> 12;
            const uint32_t bits = (plus < 1 ? plus : 1u) | (minus < 1 ? minus : 1u) << 1 | (nan < 1 ? nan : 1u) << 2;
            sp.f[d] |= static_cast<uint64_t>(bits) << (3 * r);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}
template <class M>
__device__ __forceinline__ void apply_specials(RowState<M>& st, const Specials<M>& sp) {
#pragma unroll
    for (int d = 0; d < M::kOut; ++d)
#pragma unroll
        for (int r = 0; r < M::kRegs; ++r) {
            const uint32_t bits = static_cast<uint32_t>(sp.f[d] >> (3 * r));
            const uint32_t plus = 0u - (bits & 1u), minus = 0u - (bits >> 1 & 1u), nan = 0u - (bits >> 2 & 1u);
            st.o[d][r] += __builtin_bit_cast(float, plus & 0x7F800000u);
            st.o[d][r] += __builtin_bit_cast(float, minus & 0xFF800000u);
            st.o[d][r] += __builtin_bit_cast(float, nan & 0x7FC00000u);
        }
}

// How far above the largest score m is kept where a row sees at most `keys` keys.
template <int KT>
__device__ __forceinline__ float lift_of(uint32_t keys) {
    return KT == kDtF16 || keys == 0 ? 0.0f : static_cast<float>(32 - __builtin_clz(keys));
}

// 32 keys of the second pass: `k` and `v` are their staged rows plus k_first and v_first.
template <class M, bool PAGED, int KT>
__device__ __forceinline__ Seen careful_step(RowState<M>& st, const typename M::Query& q, const typename M::qelem* q_row, bool q_odd,
                                             const KvRows<PAGED, KT>& kv, const RowView& view, int32_t key0, int32_t k_lo,
                                             int32_t k_end, uint32_t odd, float scale, float lift, uint32_t dim, const char* k, const char* v) {
    uint32_t h = (threadIdx.x & 63) / M::kRows;
    asm volatile("" : "+v"(h));  // nothing of this pass is computed ahead of it
    Scores<M> s;
    Seen seen{0, 0};
    score_rows<M>(s, q, k);
    __builtin_amdgcn_sched_barrier(0);
    patch_scores<M>(s, kv, q_row, q_odd, dim, key0, k_end, odd);
#pragma unroll
    for (int n = 0; n < M::kKeyTiles; ++n)
#pragma unroll
        for (int r = 0; r < M::kRegs; ++r) {
            const int32_t key = key0 + static_cast<int32_t>(M::key_of(n, r, h));
            const uint32_t sees = view.sees(key) & (key >= k_lo) & (key < k_end);
            const uint32_t dead = s.s[n][r] == -kInf ? sees : 0u;
            seen.keys |= sees << (M::kRegs * n + r);
            seen.dead |= dead << (M::kRegs * n + r);
            if (!sees) s.s[n][r] = -kInf;
            __builtin_amdgcn_sched_barrier(0);
        }
    take_top<M>(st, s, scale, 0.0f, lift);
    const float off = M::kShift - st.reference();
#pragma unroll
    for (int g = 0; g < kGroups<M>; ++g) {
        Weights<M> w;
        weigh<M>(w, st, s, g, scale, off);
#pragma unroll
        for (int d = 0; d < M::kOut; ++d) {
            __builtin_amdgcn_sched_barrier(0);  // one dimension's fragments at a time: the pass needs no more registers than the first
#pragma unroll
            for (int x = 0; x < M::kKvParts; ++x) {
                const typename M::frag f = M::lds_v(v + M::kStep * g * M::R::kV, d, x);
#pragma unroll
                for (int p = 0; p < M::kParts; ++p)
                    if (M::counts(x, p)) st.o[d] = M::mma(f, w.f[p], st.o[d]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    return seen;
}

}  // namespace dev
}  // namespace objeta
