// attn_tile.hpp — the tile of attention that all its kernels share: 32 query rows of a wave
// against 32 keys on the matrix cores, with the running softmax.
//
// Mathematics, for a row's scores s_j = scale q . k_j in units of log 2: with m a running
// reference near the largest score, l = sum 2^(s_j - m) and o = sum 2^(s_j - m) v_j; when m
// grows, l and o take the factor 2^(m - m'). The result is o / l, and ln 2 (m + log2 l).
//
// Layout. The scores are computed transposed, S^T = K Q^T: the 32 x 32 result then holds
// query row n = lane % 32 in its columns, and a lane 16 keys of its one row (the other 16 in
// lane ^ 32), so that maxima and sums are taken within a lane and across one swap, and
// rescaling o^T is a factor of the lane. The same registers are the product O^T += V^T P^T's
// second operand without any exchange: the sum over keys may run in any order, so its index
// (lane half h, element j) stands for the key 16 t + 8 (j / 4) + 4 h + j % 4 that the lane
// holds. V^T comes from V's rows in LDS by the transposing 64-bit read, whose 4 x 16 blocks
// are those four keys.
//
// LDS rows are the keys' rows of 16-byte units; a unit's place within its row is exchanged
// by an exclusive or with bits of the key (swz_k, swz_v), so that the 16 lanes of a read
// phase fall into different banks.
//
// f16 and bf16 use the 32x32x16 products of their type. With float queries each of these
// becomes eight 32x32x2 float products over the same fragments (16-bit keys and values
// converted when read): 1/16 of the rate, but no rounding of q or of the probabilities.
#pragma once

#include "kv_common.hpp"

namespace objeta {
namespace dev {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
struct f32x8 {
    float v[8];
};
typedef __attribute__((address_space(3))) char lds_char;

constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

template <int T> struct ElemOf { typedef float type; };
template <> struct ElemOf<kDtF16> { typedef _Float16 type; };
template <> struct ElemOf<kDtBF16> { typedef __bf16 type; };

// Rows of DT elements of type KT in LDS.
template <int KT, int DT>
struct Rows {
    static constexpr int kEs = KT == kDtF32 ? 4 : 2;
    static constexpr int kBytes = DT * kEs;
    static constexpr int kUnits = kBytes / 16;
    // the units of 16 consecutive keys at one column spread over the 16 units of 64 banks
    static __device__ __forceinline__ uint32_t swz_k(uint32_t key) {
        if constexpr (kUnits % 16 == 0) return key & 15;
        else if constexpr (kUnits % 8 == 0) return (key >> 1) & 7;
        else return (key >> 2) & 3;
    }
    // 16-bit: the 64-byte parts that one transposing read takes from four keys; float: the
    // 128-byte parts of keys four apart
    static __device__ __forceinline__ uint32_t swz_v(uint32_t key) {
        if constexpr (KT == kDtF32) return kUnits % 16 == 0 ? ((key >> 2) & 1) << 3 : 0;
        else if constexpr (kUnits % 16 == 0) return (key & 3) << 2;
        else if constexpr (kUnits % 8 == 0) return ((key >> 1) & 1) << 2;
        else return 0;
    }
};

// The products of one type of queries (QT) with one type of keys and values (KT).
template <int QT, int KT, int DT>
struct Math {
    static_assert(QT == KT || QT == kDtF32, "float queries, or queries of the cache's type");
    typedef Rows<KT, DT> R;
    static constexpr bool kFloat = QT == kDtF32;
    typedef typename ElemOf<QT>::type qelem;
    typedef typename ElemOf<KT>::type kelem;
    template <int T> struct FragOf { typedef f32x8 type; };
    typedef typename std::conditional<kFloat, f32x8,
                                      typename std::conditional<KT == kDtF16, h16x8, b16x8>::type>::type frag;
    // f16 probabilities are scaled by 2^7 (with m's slack of 2^8 still below the largest
    // value), which keeps those down to 2^-21 of the largest in its normal range
    static constexpr float kShift = (!kFloat && KT == kDtF16) ? 7.0f : 0.0f;

    static __device__ __forceinline__ frag zero() {
        frag f{};
        return f;
    }
    static __device__ __forceinline__ frag load_q(const qelem* p) {
        if constexpr (kFloat) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
            return f32x8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
        } else {
            return *reinterpret_cast<const frag*>(p);
        }
    }
    static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, f32x16 c) {
        if constexpr (kFloat) {
#pragma unroll
            for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
            return c;
        } else if constexpr (KT == kDtF16) {
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
        } else {
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
        }
    }
    template <class V>
    static __device__ __forceinline__ frag widen(const V& x) {
        f32x8 f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f.v[j] = static_cast<float>(x[j]);
        return f;
    }
    // Dimensions 16 s + 8 h .. + 8 of this lane's key (lane % 32 of the tile): K as the first
    // operand. `row` is the key's LDS row, `x0` its swizzled first unit in bytes.
    static __device__ __forceinline__ uint32_t k_first(uint32_t lane) {
        const uint32_t h = lane >> 5, key = lane & 31;
        return ((KT == kDtF32 ? 2 * h : h) ^ R::swz_k(key)) * 16;
    }
    static __device__ __forceinline__ frag lds_k(const char* row, uint32_t x0, int s) {
        if constexpr (KT == kDtF32) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(row + (x0 ^ (64 * s)));
            const f32x4 b = *reinterpret_cast<const f32x4*>(row + (x0 ^ (64 * s) ^ 16));
            return f32x8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
        } else if constexpr (kFloat) {
            typedef typename std::conditional<KT == kDtF16, h16x8, b16x8>::type v8;
            return widen(*reinterpret_cast<const v8*>(row + (x0 ^ (32 * s))));
        } else {
            return *reinterpret_cast<const frag*>(row + (x0 ^ (32 * s)));
        }
    }
    // This lane's place for V: byte offset from a group of 16 keys' first row to the first
    // of its reads at dimensions 0..31.
    static __device__ __forceinline__ uint32_t v_first(uint32_t lane) {
        const uint32_t h = lane >> 5;
        if constexpr (KT == kDtF32) {
            return 4 * h * R::kBytes + (R::swz_v(4 * h) * 16) + (lane & 31) * 4;
        } else {
            const uint32_t l = lane & 15, ds = (lane >> 4) & 1, key = 4 * h + (l >> 2);
            const uint32_t unit = 2 * ds + ((l & 3) >> 1);
            return key * R::kBytes + ((unit ^ R::swz_v(key)) * 16) + (l & 1) * 8;
        }
    }
    // V^T of 16 keys (rows from `rows` on) at dimensions 32 dd + lane % 32.
    static __device__ __forceinline__ frag lds_v(const char* rows, uint32_t v0, int dd) {
        if constexpr (KT == kDtF32) {
            f32x8 f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                f.v[j] = *reinterpret_cast<const float*>(rows + (v0 ^ (128 * dd)) + (8 * (j / 4) + j % 4) * R::kBytes);
            return f;
        } else {
            const char* p = rows + (v0 ^ (64 * dd));
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_char*)(p));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(lds_char*)(p + 8 * R::kBytes));
            const s16x8 v = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            if constexpr (kFloat) {
                typedef typename std::conditional<KT == kDtF16, h16x8, b16x8>::type v8;
                return widen(__builtin_bit_cast(v8, v));
            } else {
                return __builtin_bit_cast(frag, v);
            }
        }
    }
    // Eight probabilities as the second operand: rounded to nearest, as the output is.
    static __device__ __forceinline__ frag pack(const float* p) {
        if constexpr (kFloat) {
            return f32x8{{p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]}};
        } else {
            frag f;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = static_cast<kelem>(p[j]);
            return f;
        }
    }
};

// A value and its counterpart 32 lanes away.
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Running softmax of this lane's row (m and, over this lane's keys only, l), and o^T.
template <int DT>
struct RowState {
    float m = -kInf, l = 0.0f;
    f32x16 o[DT / 32];
    __device__ __forceinline__ void clear() {
        m = -kInf, l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    }
    __device__ __forceinline__ float reference() const { return m == -kInf ? 0.0f : m; }
    // Takes the factor of a new reference.
    __device__ __forceinline__ void raise(float to) {
        const float f = exp2_hw(m - (to == -kInf ? 0.0f : to));
        m = to;
        l *= f;
#pragma unroll
        for (int d = 0; d < DT / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
};

// How far the scores may outgrow m before o is rescaled (factor 2^8: far from any limit of
// the types, and rare after the first keys).
constexpr float kSlack = 8.0f;

// S^T of 32 keys at `rows` (LDS).
template <class M, int DT>
__device__ __forceinline__ f32x16 scores(const typename M::frag (&q)[DT / 16], const char* rows, uint32_t lane, uint32_t k0) {
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
    const char* row = rows + (lane & 31) * M::R::kBytes;
#pragma unroll
    for (int i = 0; i < DT / 16; ++i) s = M::mma(M::lds_k(row, k0, i), q[i], s);
    return s;
}

// The softmax step over NS tiles of raw (unscaled, masked to -inf) scores and their values.
template <class M, int DT, int NS>
__device__ __forceinline__ void accumulate(RowState<DT>& st, f32x16 (&s)[NS], float scale, const char* v_rows, uint32_t v0) {
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, s[n][r]);
    top = __builtin_fmaxf(top, other_half(top)) * scale;
    if (__any(top > st.m + kSlack)) st.raise(__builtin_fmaxf(st.m, top));
    const float off = M::kShift - st.reference();
#pragma unroll
    for (int n = 0; n < NS; ++n) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = exp2_hw(__builtin_fmaf(s[n][8 * t + j], scale, off));
                st.l += p[j];
            }
            const typename M::frag pf = M::pack(p);
            const char* rows = v_rows + (32 * n + 16 * t) * M::R::kBytes;
#pragma unroll
            for (int d = 0; d < DT / 32; ++d) st.o[d] = M::mma(M::lds_v(rows, v0, d), pf, st.o[d]);
        }
    }
}

struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;
    uint64_t q_stride, k_stride, v_stride, out_stride;  // elements; k and v of packed prompts
    const int32_t* cu;
    uint32_t n_batch, n_rows, n_heads, n_kv, group, dim;
    float scale, scale_log2;
    int32_t causal;
    // paged
    KvView kv;
    const int32_t* seqs;
    const uint64_t* tree;
    uint64_t layer_off;  // elements
    // keys cut over workgroups
    uint32_t chunk, n_splits, n_tiles;
    float *part, *part_ml;  // [n_splits][n_rows * n_heads][dim], [..][2]
    uint32_t* err;
};

// What one row sees: keys lo .. hi, and among those from `base` on only the set bits of mask.
struct RowView {
    int32_t lo, hi, base;
    uint64_t mask;
    __device__ __forceinline__ bool sees(int32_t key) const {
        const uint32_t bit = static_cast<uint32_t>(key - base);
        return key >= lo && key <= hi && (key < base || bit > 63 || ((mask >> bit) & 1));
    }
};

// The rows of K and V of one (sequence, head): packed rows, or pages.
template <bool PAGED, int KT>
struct KvRows {
    typedef typename ElemOf<KT>::type elem;
    const elem *k, *v;
    uint64_t k_stride, v_stride;
    const int32_t* table;
    KvView kv;
    uint64_t page_step;  // elements from page to page
    uint32_t dim;
    // the page of a slot; 0 for one that is none, and *bad
    __device__ __forceinline__ int32_t page_of(uint32_t slot, bool& bad) const {
        const int32_t p = table[slot >> kv.shift];
        if (page_ok(kv, p)) return p;
        bad = true;
        return 0;
    }
    __device__ __forceinline__ uint64_t paged_at(int32_t page, uint32_t slot) const {
        return static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_step + (slot & ((1u << kv.shift) - 1)) * dim;
    }
    __device__ __forceinline__ const elem* k_row(uint32_t key, bool& bad) const {
        if constexpr (PAGED) return k + paged_at(page_of(key, bad), key);
        else return k + key * k_stride;
    }
    __device__ __forceinline__ const elem* v_row(uint32_t key, bool& bad) const {
        if constexpr (PAGED) return v + paged_at(page_of(key, bad), key);
        else return v + key * v_stride;
    }
};

// One row computed key by key over the keys it sees in [k0, k1), by a whole wave (a lane has
// dimensions lane, lane + 64, ...). The matrix products multiply unseen values by a
// probability of 0, which an infinity or NaN there turns into NaN; a wave whose result is
// not finite comes here, where unseen places are not touched.
template <class M, bool PAGED, int KT>
__device__ __forceinline__ void row_by_row(const KvRows<PAGED, KT>& kv, const typename M::qelem* q, const RowView& view,
                                           int32_t k0, int32_t k1, float scale, uint32_t dim, float& m, float& l,
                                           float (&o)[4]) {
    const uint32_t lane = threadIdx.x & 63;
    float qv[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const uint32_t d = lane + 64 * x;
        qv[x] = d < dim ? static_cast<float>(q[d]) : 0.0f;
        o[x] = 0.0f;
    }
    m = -kInf, l = 0.0f;
    bool bad = false;
    for (int32_t j = k0; j < k1; ++j) {
        if (!view.sees(j)) continue;
        const auto* kr = kv.k_row(static_cast<uint32_t>(j), bad);
        const auto* vr = kv.v_row(static_cast<uint32_t>(j), bad);
        float dot = 0.0f, vv[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint32_t d = lane + 64 * x;
            vv[x] = 0.0f;
            if (d < dim) {
                dot = __builtin_fmaf(qv[x], static_cast<float>(kr[d]), dot);
                vv[x] = static_cast<float>(vr[d]);
            }
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) dot += __shfl_xor(dot, s, 64);
        const float sc = dot * scale;
        const float top = __builtin_fmaxf(m, sc), ref = top == -kInf ? 0.0f : top;
        const float f = exp2_hw(m - ref), p = exp2_hw(sc - ref);
        l = l * f + p;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] = o[x] * f + p * vv[x];
        m = top;
    }
}

// Writes four consecutive output values.
template <int QT>
__device__ __forceinline__ void store_out(typename ElemOf<QT>::type* p, f32x4 v) {
    if constexpr (QT == kDtF32) {
        *reinterpret_cast<f32x4*>(p) = v;
    } else {
        typedef typename ElemOf<QT>::type e4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<e4*>(p) = __builtin_convertvector(v, e4);
    }
}

// Where one (row, head)'s partial result of a split lies.
__device__ __forceinline__ uint64_t part_at(const AttnArgs& a, uint32_t split, uint64_t row, uint32_t head) {
    return (static_cast<uint64_t>(split) * a.n_rows + row) * a.n_heads + head;
}

// A wave's 32 rows done: normalised output and lse, or (several splits) the parts. Lanes 0-31
// and 32-63 hold the same rows with different dimensions.
template <class M, int QT, int DT>
__device__ __forceinline__ void write_rows(const AttnArgs& a, const RowState<DT>& st, bool real, uint64_t row, uint32_t head,
                                           uint32_t split, uint32_t lane) {
    const float l = st.l + other_half(st.l);
    if (!real) return;
    const uint32_t h = lane >> 5;
    if (a.n_splits > 1) {
        const uint64_t at = part_at(a, split, row, head);
        float* p = a.part + at * a.dim;
#pragma unroll
        for (int d = 0; d < DT / 32; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t x = 32 * d + 8 * r + 4 * h;
                if (x < a.dim)
                    *reinterpret_cast<f32x4*>(p + x) =
                        f32x4{st.o[d][4 * r], st.o[d][4 * r + 1], st.o[d][4 * r + 2], st.o[d][4 * r + 3]};
            }
        if (h == 0) {
            a.part_ml[2 * at] = st.m - M::kShift;
            a.part_ml[2 * at + 1] = l;
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    typename M::qelem* p = static_cast<typename M::qelem*>(a.out) + row * a.out_stride + static_cast<uint64_t>(head) * a.dim;
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t x = 32 * d + 8 * r + 4 * h;
            if (x < a.dim)
                store_out<QT>(p + x, f32x4{st.o[d][4 * r] * inv, st.o[d][4 * r + 1] * inv, st.o[d][4 * r + 2] * inv,
                                           st.o[d][4 * r + 3] * inv});
        }
    if (a.lse && h == 0)
        a.lse[row * a.n_heads + head] = l == 0.0f ? -kInf : (st.m - M::kShift + __builtin_amdgcn_logf(l)) * kLn2;
}

// The same for one row of row_by_row, by a whole wave (`poison`: NaN instead).
template <class M>
__device__ __forceinline__ void write_row(const AttnArgs& a, float m, float l, const float (&o)[4], uint64_t row,
                                          uint32_t head, uint32_t split, uint32_t lane) {
    if (a.n_splits > 1) {
        const uint64_t at = part_at(a, split, row, head);
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (lane + 64 * x < a.dim) a.part[at * a.dim + lane + 64 * x] = o[x];
        if (lane == 0) a.part_ml[2 * at] = m, a.part_ml[2 * at + 1] = l;
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    typename M::qelem* p = static_cast<typename M::qelem*>(a.out) + row * a.out_stride + static_cast<uint64_t>(head) * a.dim;
#pragma unroll
    for (int x = 0; x < 4; ++x)
        if (lane + 64 * x < a.dim) p[lane + 64 * x] = static_cast<typename M::qelem>(o[x] * inv);
    if (a.lse && lane == 0) a.lse[row * a.n_heads + head] = l == 0.0f ? -kInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <int DT>
__device__ __forceinline__ bool not_finite(const RowState<DT>& st) {
    float x = 0.0f;
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) x = __builtin_fmaf(st.o[d][r], 0.0f, x);
    return __any(!(x == 0.0f));
}

}  // namespace dev
}  // namespace objeta
