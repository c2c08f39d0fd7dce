// attn_tile.hpp — the tile of attention that all its kernels share: kRows = 32 or 16 query
// rows of a wave against 32 keys on the matrix cores, with the running softmax.
//
// Mathematics, for a row's scores s_j = scale q . k_j in units of log 2: with m a running
// reference near the largest score, l = sum 2^(s_j - m) and o = sum 2^(s_j - m) v_j; when m
// grows, l and o take the factor 2^(m - m'). The result is o / l, and ln 2 (m + log2 l).
//
// Layout. The scores are computed transposed, S^T = K Q^T: a lane then holds keys of one query
// row (lane % kRows), and the row's other keys lie in the lanes of the same remainder, so that
// maxima and sums are taken within a lane and across one or two exchanges, and rescaling o^T
// is a factor of the lane. The same registers are the product O^T += V^T P^T's second operand
// without any exchange: the sum over keys may run in any order, so its index (lane part h =
// lane / kRows, element j) stands for the key that the lane holds there. V^T comes from V's
// rows in LDS by the transposing 64-bit read, whose blocks of 4 keys x 16 dimensions are what
// a lane's four consecutive elements name.
//
// Types. f16 and bf16 use the products of their type, probabilities rounded to it. Float
// queries on a 16-bit cache are split into parts of the cache's type whose sum holds 22 (f16,
// two parts of the row times a power of two) or 24 bits (bf16, three), each product is exact,
// and so are the probabilities split: a float result at two or three 16-bit products instead
// of the eight float ones that a 16-bit product's worth of float products takes at a
// sixteenth of the rate. So are float keys and values where 128 rows share the work (three
// parts by three of bf16, without the three products below 2^-24: six 16-bit ones; a value
// below 2^-102 loses its last part); else floats use the float products.
#pragma once

#include "kv_common.hpp"

#include <type_traits>

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
// Float keys and values that lie in LDS as three bf16 parts each.
constexpr int kDtF32x3 = 3;
static_assert(kDtF32x3 != kDtF32 && kDtF32x3 != kDtF16 && kDtF32x3 != kDtBF16, "a type of its own");

// Rows of DT elements of type KT in LDS, read by tiles of ROWS query rows. A key's row is
// padded: by 16 bytes, the 16-byte reads of 16 consecutive keys at one column fall into 16
// different groups of four banks (of 64); by 32 bytes, the 32-byte parts that a transposing
// read takes from four consecutive keys, and the 32 (ROWS = 16: by 16, the 16) floats of keys
// four apart, into different banks.
template <int KT, int DT, int ROWS>
struct Rows {
    static constexpr int kEs = KT == kDtF32 || KT == kDtF32x3 ? 4 : 2;  // of an element in memory
    static constexpr int kBytes = DT * kEs;
    static constexpr int kUnits = kBytes / 16;
    static constexpr int kLs = KT == kDtF32 ? 4 : 2;  // of an element of a part in LDS
    static constexpr int kParts = KT == kDtF32x3 ? 3 : 1;
    static constexpr int kPart = DT * kLs;  // bytes from part to part of a row in LDS
    static constexpr int kK = kParts * kPart + 16;
    static constexpr int kV = kParts * kPart + (KT == kDtF32 && ROWS == 16 ? 16 : 32);
    // lanes that load one row: a power of two, so that a wave's load lies within eight keys
    static constexpr int kLanes = kUnits <= 8 ? 8 : (kUnits <= 16 ? 16 : (kUnits <= 32 ? 32 : 64));
    static constexpr int kPer = 64 / kLanes;  // keys of a wave's load
};

// Two floats rounded to bf16, side by side; x and y keep the rest. By words: left to
// conversions of single values, the compiler makes each of them twice.
__device__ __forceinline__ uint32_t take_bf16(float& x, float& y) {
    typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const uint32_t pair = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, b16x2));
    x -= __builtin_bit_cast(float, pair << 16);
    y -= __builtin_bit_cast(float, pair & 0xFFFF0000u);
    return pair;
}

template <int ROWS> struct AccOf { typedef f32x16 type; };
template <> struct AccOf<16> { typedef f32x4 type; };

// The products of one type of queries (QT) with one type of keys and values (KT).
template <int QT, int KT, int DT, int ROWS>
struct Math {
    static_assert(QT == KT || QT == kDtF32, "float queries, or queries of the cache's type");
    typedef Rows<KT, DT, ROWS> R;
    typedef typename AccOf<ROWS>::type acc;
    static constexpr int kRows = ROWS;
    static constexpr int kRegs = ROWS == 32 ? 16 : 4;   // of an accumulator
    static constexpr int kKeyTiles = 32 / ROWS;         // accumulators that hold 32 keys' scores
    static constexpr int kStep = 8 * (64 / ROWS);       // dimensions (keys) of one product
    static constexpr int kSteps = DT / kStep;
    static constexpr int kOut = DT / ROWS;              // accumulators of o
    static constexpr bool kFloat = KT == kDtF32;
    static constexpr int kParts = QT == KT ? 1 : (KT == kDtF16 ? 2 : 3);  // of a query's and a probability's
    static constexpr int kKvParts = R::kParts;                            // of a key's and a value's
    // whether the product of these parts counts: of three and three, those above 2^-24
    static constexpr bool counts(int kv, int q) { return kKvParts == 1 || kv + q < 3; }
    typedef typename ElemOf<QT>::type qelem;
    typedef typename ElemOf<KT>::type kelem;
    typedef typename std::conditional<KT == kDtF16, _Float16, __bf16>::type pelem;  // of parts
    typedef typename std::conditional<kFloat, f32x8,
                                      typename std::conditional<KT == kDtF16, h16x8, b16x8>::type>::type frag;
    struct Query {
        frag f[kParts][kSteps];
    };
    // f16 probabilities are scaled by 2^7 (with m's slack of 2^8 still below the largest
    // value), which keeps those down to 2^-21 of the largest in its normal range
    static constexpr float kShift = KT == kDtF16 ? 7.0f : 0.0f;

    static __device__ __forceinline__ acc zero() {
        acc c;
#pragma unroll
        for (int r = 0; r < kRegs; ++r) c[r] = 0.0f;
        return c;
    }
    static __device__ __forceinline__ acc mma(const frag& a, const frag& b, acc c) {
        if constexpr (kFloat) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (ROWS == 32) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
                else c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
            }
            return c;
        } else if constexpr (KT == kDtF16) {
            if constexpr (ROWS == 32) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
            else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
        } else {
            if constexpr (ROWS == 32) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
            else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
        }
    }
    // Splits eight floats into the parts of an operand, each the rest's nearest value.
    template <class Put>
    static __device__ __forceinline__ void split(const float* x, Put put) {
        float rest[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            frag f;
            if constexpr (kParts == 3) {
                u32x4a words;
#pragma unroll
                for (int j = 0; j < 4; ++j) words[j] = take_bf16(rest[2 * j], rest[2 * j + 1]);
                put(p, __builtin_bit_cast(frag, words));
                continue;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f[j] = static_cast<pelem>(rest[j]);
                if (p + 1 < kParts) rest[j] -= static_cast<float>(f[j]);
            }
            put(p, f);
        }
    }
    // This lane's part of its row's query: dimensions kStep i + 8 h .. + 8. `scale` takes the
    // power of two that the row was multiplied by.
    static __device__ __forceinline__ void load_q(Query& q, const qelem* p, bool real, uint32_t dim, uint32_t lane,
                                                  float& scale) {
        const uint32_t h = lane / ROWS;
        if constexpr (QT != kDtF32) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const uint32_t d = kStep * i + 8 * h;
                frag z{};
                q.f[0][i] = real && d < dim ? *reinterpret_cast<const frag*>(p + d) : z;
            }
        } else {
            float x[kSteps][8];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const uint32_t d = kStep * i + 8 * h;
                f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f}, b = a;
                if (real && d < dim) {
                    a = *reinterpret_cast<const f32x4*>(p + d);
                    b = *reinterpret_cast<const f32x4*>(p + d + 4);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = a[j], x[i][4 + j] = b[j];
            }
            if constexpr (KT == kDtF16) {
                // the row's largest value to [2^13, 2^14): f16's range, with its sums' room
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = __builtin_fmaxf(top, __builtin_fabsf(x[i][j]));
#pragma unroll
                for (int s = ROWS; s < 64; s <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, s, 64));
                int e = 0;
                if (top > 0.0f && top < kInf) e = 14 - __builtin_amdgcn_frexp_expf(top);
                e = e > 120 ? 120 : e;
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[i][j] = __builtin_amdgcn_ldexpf(x[i][j], e);
                scale = __builtin_amdgcn_ldexpf(scale, -e);
            }
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if constexpr (kFloat) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) q.f[0][i].v[j] = x[i][j];
                } else {
                    split(x[i], [&](int part, const frag& f) { q.f[part][i] = f; });
                }
            }
        }
    }
    // Waits for the query here. Left in flight into a loop, its first use there would wait
    // in every turn for whatever loads the turn has on their way.
    static __device__ __forceinline__ void settle(Query& q) {
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if constexpr (kFloat) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(q.f[p][i].v[j]));
                } else {
                    u32x4a x = __builtin_bit_cast(u32x4a, q.f[p][i]);
                    asm volatile("" : "+v"(x));
                    q.f[p][i] = __builtin_bit_cast(frag, x);
                }
            }
    }
    // Dimensions kStep i + 8 h .. + 8 of this lane's key (lane % ROWS of the tile): K as the
    // first operand. `p` is the tile's first row plus k_first.
    static __device__ __forceinline__ uint32_t k_first(uint32_t lane) {
        return lane % ROWS * R::kK + lane / ROWS * (8 * R::kLs);
    }
    static __device__ __forceinline__ frag lds_k(const char* p, int i, int part = 0) {
        p += part * R::kPart;
        if constexpr (kFloat) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p + 4 * kStep * i);
            const f32x4 b = *reinterpret_cast<const f32x4*>(p + 4 * kStep * i + 16);
            return f32x8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
        } else {
            return *reinterpret_cast<const frag*>(p + 2 * kStep * i);
        }
    }
    // The key of score register r of tile n, and the keys of element j of a group of kStep
    // keys (offset from the lane part's first).
    static __device__ __forceinline__ uint32_t key_of(int n, int r, uint32_t h) {
        return ROWS == 32 ? (r & 3) + 8 * (r >> 2) + 4 * h : 16 * n + r + 4 * h;
    }
    static constexpr int kFar = ROWS == 32 ? 8 : 16;  // elements 4 .. 7 lie this many keys behind 0 .. 3
    // V^T of kStep keys at dimensions ROWS dd + lane % ROWS; `p` is the first key's row plus
    // v_first.
    static __device__ __forceinline__ uint32_t v_first(uint32_t lane) {
        const uint32_t h = lane / ROWS;
        if constexpr (kFloat) {
            return 4 * h * R::kV + (lane % ROWS) * 4;
        } else {
            const uint32_t l = lane & 15, ds = ROWS == 32 ? (lane >> 4) & 1 : 0;
            return (4 * h + (l >> 2)) * R::kV + ds * 32 + (l & 3) * 8;
        }
    }
    static __device__ __forceinline__ frag lds_v(const char* p, int dd, int part = 0) {
        p += part * R::kPart + ROWS * R::kLs * dd;
        if constexpr (kFloat) {
            f32x8 f;
#pragma unroll
            for (int j = 0; j < 8; ++j) f.v[j] = *reinterpret_cast<const float*>(p + (kFar * (j / 4) + j % 4) * R::kV);
            return f;
        } else {
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_char*)(p));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(lds_char*)(p + kFar * R::kV));
            const s16x8 v = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            return __builtin_bit_cast(frag, v);
        }
    }
};

// x of this lane and of its counterpart 32 (16) lanes away, in either order.
struct Pair {
    float a, b;
};
__device__ __forceinline__ Pair with_32(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];  // a bit cast of a vector's element takes its first
    return Pair{__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ Pair with_16(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return Pair{__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
// A maximum or sum over the lanes that hold one row.
template <int ROWS>
__device__ __forceinline__ float row_max(float x) {
    if constexpr (ROWS == 16) {
        const Pair p = with_16(x);
        x = __builtin_fmaxf(p.a, p.b);
    }
    const Pair p = with_32(x);
    return __builtin_fmaxf(p.a, p.b);
}
template <int ROWS>
__device__ __forceinline__ float row_sum(float x) {
    if constexpr (ROWS == 16) {
        const Pair p = with_16(x);
        x = p.a + p.b;
    }
    const Pair p = with_32(x);
    return p.a + p.b;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Running softmax of this lane's row (m and, over this lane's keys only, l), and o^T.
template <class M>
struct RowState {
    float m, l;
    typename M::acc o[M::kOut];
    __device__ __forceinline__ void clear() {
        m = -kInf, l = 0.0f;
#pragma unroll
        for (int d = 0; d < M::kOut; ++d) o[d] = M::zero();
    }
    __device__ __forceinline__ float reference() const { return m == -kInf ? 0.0f : m; }
    // Takes the factor of a new reference.
    __device__ __forceinline__ void raise(float to) {
        const float f = exp2_hw(m - (to == -kInf ? 0.0f : to));
        m = to;
        l *= f;
#pragma unroll
        for (int d = 0; d < M::kOut; ++d)
#pragma unroll
            for (int r = 0; r < M::kRegs; ++r) o[d][r] *= f;
    }
};

// How far the scores may outgrow m before o is rescaled (factor 2^8: far from any limit of
// the types, and rare after the first keys).
constexpr float kSlack = 8.0f;

// The scores (unscaled) of 32 keys.
template <class M>
struct Scores {
    typename M::acc s[M::kKeyTiles];
};

// S^T of 32 keys; `k` is their first row in LDS plus k_first.
template <class M>
__device__ __forceinline__ void score_rows(Scores<M>& s, const typename M::Query& q, const char* k) {
#pragma unroll
    for (int n = 0; n < M::kKeyTiles; ++n) {
        s.s[n] = M::zero();
#pragma unroll
        for (int i = 0; i < M::kSteps; ++i) {
#pragma unroll
            for (int x = 0; x < M::kKvParts; ++x) {
                const typename M::frag f = M::lds_k(k + n * M::kRows * M::R::kK, i, x);
#pragma unroll
                for (int p = 0; p < M::kParts; ++p)
                    if (M::counts(x, p)) s.s[n] = M::mma(f, q.f[p][i], s.s[n]);
            }
        }
    }
}

// The probabilities of group t of kStep keys as an operand.
template <class M>
struct Weights {
    typename M::frag f[M::kParts];
};

// The fragments of 32 keys (kRows == 32) for all steps of their scores.
template <class M>
struct Keys {
    typename M::frag f[M::kSteps];
};
template <class M>
__device__ __forceinline__ void read_keys(Keys<M>& k, const char* p) {
#pragma unroll
    for (int i = 0; i < M::kSteps; ++i) k.f[i] = M::lds_k(p, i);
}
template <class M>
__device__ __forceinline__ void score(Scores<M>& s, const typename M::Query& q, const Keys<M>& k) {
    s.s[0] = M::zero();
#pragma unroll
    for (int i = 0; i < M::kSteps; ++i)
#pragma unroll
        for (int p = 0; p < M::kParts; ++p) s.s[0] = M::mma(k.f[i], q.f[p][i], s.s[0]);
}
// The fragments of the values of group t (`v`: 32 keys' first row plus v_first), and their
// products.
template <class M>
struct Values {
    typename M::frag f[M::kOut];
};
template <class M>
__device__ __forceinline__ void read_values(Values<M>& f, const char* v, int t) {
#pragma unroll
    for (int d = 0; d < M::kOut; ++d) f.f[d] = M::lds_v(v + M::kStep * t * M::R::kV, d);
}
template <class M>
__device__ __forceinline__ void add_values(RowState<M>& st, const Weights<M>& w, const Values<M>& v) {
#pragma unroll
    for (int d = 0; d < M::kOut; ++d)
#pragma unroll
        for (int part = 0; part < M::kParts; ++part) st.o[d] = M::mma(v.f[d], w.f[part], st.o[d]);
}

// The largest score of 32 keys, scaled, over the lanes of a row; raises the reference, `lift` above
// the largest, where that has outgrown it by more than `slack`.
template <class M>
__device__ __forceinline__ void take_top(RowState<M>& st, const Scores<M>& s, float scale, float slack = kSlack, float lift = 0.0f) {
    float top = -kInf;
#pragma unroll
    for (int t = 0; t < M::kKeyTiles; ++t)
#pragma unroll
        for (int r = 0; r < M::kRegs; ++r) top = __builtin_fmaxf(top, s.s[t][r]);
    top = row_max<M::kRows>(top) * scale + lift;
    if (__any(top > st.m + slack)) st.raise(__builtin_fmaxf(st.m, top));
}

template <class M>
__device__ __forceinline__ void weigh(Weights<M>& w, RowState<M>& st, const Scores<M>& s, int t, float scale, float off) {
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = M::kRows == 32 ? s.s[0][8 * t + j] : s.s[j / 4 % M::kKeyTiles][j % 4];
        p[j] = exp2_hw(__builtin_fmaf(x, scale, off));
        st.l += p[j];
    }
    if constexpr (M::kFloat) w.f[0] = f32x8{{p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]}};
    else M::split(p, [&](int part, const typename M::frag& x) { w.f[part] = x; });  // rounded to nearest, as the output is
}

// o^T += V^T P^T of group t.
template <class M>
__device__ __forceinline__ void value_rows(RowState<M>& st, const Weights<M>& w, const char* v, int t) {
#pragma unroll
    for (int d = 0; d < M::kOut; ++d) {
#pragma unroll
        for (int x = 0; x < M::kKvParts; ++x) {
            const typename M::frag f = M::lds_v(v + M::kStep * t * M::R::kV, d, x);
#pragma unroll
            for (int p = 0; p < M::kParts; ++p)
                if (M::counts(x, p)) st.o[d] = M::mma(f, w.f[p], st.o[d]);
        }
    }
}
template <class M>
constexpr int kGroups = 32 / M::kStep;  // of kStep keys in 32: two of 16, or one of 32

struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;
    uint64_t q_stride, k_stride, v_stride, out_stride;  // elements; k and v of packed prompts
    const int32_t* cu;
    uint32_t n_batch, n_rows, n_heads, n_kv, group, dim;
    float scale_log2;  // times log2 e
    int32_t causal;
    // paged
    KvView kv;
    const int32_t* seqs;
    const uint64_t* tree;
    uint64_t layer_off;  // elements
    // keys cut over workgroups: of cached sequences in equal parts of about `chunk`, of a prompt's
    // tile of rows in n_splits equal ones. pick: the kernel takes a chunk that fills the card,
    // and leaves it in *picked for the join. wide: workgroups of twice the waves.
    uint32_t chunk, n_splits, n_tiles, tile_rows, pick, wide;
    uint32_t first;  // the launch's first workgroup
    uint32_t* picked;
    float *part, *part_ml;  // [n_splits][n_rows * n_heads][dim], [..][2]
    uint32_t* err;
};

// Waves of a workgroup of 16 or 32 rows, by the bytes of a head's row: as many as LDS lets two such
// workgroups have on a CU (one, of the largest rows of 32).
constexpr int stream_waves(int row_bytes) { return row_bytes <= 256 ? 4 : (row_bytes <= 512 ? 2 : 1); }

// Which (entry, head, split) a workgroup of 16 or 32 rows takes. The splits are the slowest
// index: short sequences have only the first ones, and workgroups go to the eight XCDs in
// turn, so a fast split index would give the first XCDs most of the work. The groups are
// turned by one place from split to split, so that no XCD keeps the longest sequences.
struct StreamItem {
    uint32_t b, head, split;
    bool any;
    __device__ __forceinline__ StreamItem(const AttnArgs& a, uint32_t id) {
        const uint32_t per = a.n_batch * a.n_kv, g = (id & ~7u) + ((id + (id & ~7u) / per) & 7);
        split = g / per;
        any = split < a.n_splits;
        head = g % per % a.n_kv;
        b = g % per / a.n_kv;
    }
};

// The sum over the lanes up to this one, by moves within rows of 16 and broadcasts of their last
// lanes: a few cycles each, where an exchange through LDS takes some sixty.
template <class T>
__device__ __forceinline__ T sum_to_lane(T v) {
    auto add = [&](auto move) {
        const int x = move(__builtin_bit_cast(int, v));
        v += __builtin_bit_cast(T, x);
    };
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false); });  // row_shr:1
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false); });
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false); });
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false); });
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false); });  // row_bcast:15 to rows 1 and 3
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false); });  // row_bcast:31 to rows 2 and 3
    return v;
}

// Into how many parts a sequence's keys are cut.
__device__ __forceinline__ uint32_t splits_of(int32_t len, uint32_t chunk, uint32_t most) {
    const uint32_t n = (static_cast<uint32_t>(len) + chunk - 1) / chunk;
    return n < 1 ? 1 : (n < most ? n : most);
}

// Which piece of work a workgroup of 128 rows takes, counted over the pieces that there are:
// entries differ in rows and lengths, and a grid over the largest of both would be mostly
// empty workgroups, unevenly over the XCDs (8 trees of 9 to 64 drafts: 39 to 64 workgroups on
// an XCD, the kernel 80 us for 44 us of work on every CU). Each wave reads 64 entries at a
// time, a lane an entry, and finds the id'th piece in their running sum; what it read of the
// entry need not be read again. Up to 64 entries it also chooses the chunk, which the host
// could only choose for the longest (8 trees over 2000 to 7001 tokens: parts of at most 896 keys
// instead of 1024, the kernel 52.5 us instead of 55.5, the join 10 instead of 11.4).
struct BlockItem {
    uint32_t head, split, tile, splits;
    int32_t row0, n_q, len, seq;
    bool any, usable;
    static __device__ __forceinline__ uint32_t total(uint32_t v) { return __builtin_amdgcn_readlane(sum_to_lane(v), 63); }
    // `slots` workgroups run at a time.
    __device__ __forceinline__ BlockItem(const AttnArgs& a, uint32_t id, uint32_t slots) {
        const uint32_t lane = threadIdx.x & 63;
        uint32_t chunk = a.chunk;
        const bool first = id == 0;
        any = false;
        if (first && a.n_batch > 64) {  // it finds its piece early: row ranges behind are its to check too
            bool bad = false;
            for (uint32_t b = 64 + threadIdx.x; b < a.n_batch; b += blockDim.x) {
                const int32_t lo = a.cu[b], hi = a.cu[b + 1];
                bad |= lo < 0 || hi < lo || static_cast<uint32_t>(hi) > a.n_rows;
            }
            if (bad) atomicOr(a.err, kErrIndex);
        }
        for (uint32_t b0 = 0; b0 < a.n_batch; b0 += 64) {
            const uint32_t b = b0 + lane;
            int32_t lo = 0, n = 0, s = 0, l = 0;
            bool ok = true;
            uint32_t tiles = 0;
            if (b < a.n_batch) {
                lo = a.cu[b];
                const int32_t hi = a.cu[b + 1];
                s = a.seqs[b];
                const bool rows = lo >= 0 && hi >= lo && static_cast<uint32_t>(hi) <= a.n_rows;
                if (!rows && first) atomicOr(a.err, kErrIndex);
                n = rows ? hi - lo : 0;
                ok = seq_ok(a.kv, s);
                l = ok ? a.kv.lens[s] : 0;
                ok = ok && len_ok(a.kv, l) && n <= l && (!a.tree || n <= 64);
                if (!ok) l = 0;
                tiles = (static_cast<uint32_t>(n) * a.group + 127) / 128;
                tiles = tiles < a.n_tiles ? tiles : a.n_tiles;
            }
            if (a.pick) {
                // pieces of `chunk` keys are to be at most what runs at once, or a multiple of
                // it where the tiles alone are more than three quarters
                const uint32_t one = total(tiles * a.n_kv);
                const uint32_t room = (one * 4 / 3 + slots) / slots * slots;
                float keys = static_cast<float>(tiles * a.n_kv) * static_cast<float>((static_cast<uint32_t>(l) + 63) / 64);
                keys = sum_to_lane(keys);
                const uint32_t least = __builtin_amdgcn_readlane(static_cast<uint32_t>(keys / static_cast<float>(room)), 63) + 1;
                for (uint32_t k = 8; k <= 16; k += k < 12 ? 1 : 2) {
                    chunk = least * 8 * k;
                    chunk = chunk < 256 ? 256 : chunk;
                    if (total(tiles * a.n_kv * splits_of(l, chunk, a.n_splits)) <= room) break;
                }
                if (first && threadIdx.x == 0) *a.picked = chunk;
            }
            const uint32_t parts = splits_of(l, chunk, a.n_splits), pieces = tiles * parts * a.n_kv;
            const uint32_t sum = sum_to_lane(pieces);
            const uint64_t past = __ballot(sum > id);
            if (past) {
                const int at = __builtin_ctzll(past);
                const uint32_t in = id - (__builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(pieces, at));
                const uint32_t n_tiles = __builtin_amdgcn_readlane(tiles, at), rest = in / a.n_kv;
                head = in % a.n_kv, tile = rest % n_tiles, split = rest / n_tiles;
                splits = __builtin_amdgcn_readlane(parts, at);
                row0 = __builtin_amdgcn_readlane(lo, at), n_q = __builtin_amdgcn_readlane(n, at);
                len = __builtin_amdgcn_readlane(l, at), seq = __builtin_amdgcn_readlane(s, at);
                usable = __builtin_amdgcn_readlane(static_cast<int32_t>(ok), at) != 0;
                any = true;
                return;
            }
            id -= __builtin_amdgcn_readlane(sum, 63);
        }
    }
};

// The kernel's arguments read anew from where the launch left them (each of these kernels has
// one argument). Used behind a loop, they need no registers during it.
__device__ __forceinline__ const AttnArgs& args_again() {
    auto p = (const __attribute__((address_space(4))) AttnArgs*)(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+s"(p));
    return *(const AttnArgs*)p;
}

// What one row sees: keys lo .. hi, and among those from `base` on (64 at most up to hi) only
// the set bits of mask.
struct RowView {
    int32_t lo, hi, base;
    uint64_t mask;
    __device__ __forceinline__ bool sees(int32_t key) const {
        // no short-cut operators: a branch for each of a tile's scores costs more than the tests
        const uint32_t bit = static_cast<uint32_t>(key - base);
        const uint32_t word = static_cast<uint32_t>(bit & 32 ? mask >> 32 : mask);
        return (key >= lo) & (key <= hi) & ((key < base) | ((word >> (bit & 31)) & 1));
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
    // A table entry as it stands: read ahead, it is checked when it is used, so that nothing
    // waits for it before.
    __device__ __forceinline__ int32_t entry_of(uint32_t slot) const { return table[slot >> kv.shift]; }
    // A page that an entry names; 0 for one that is none, and `bad`.
    __device__ __forceinline__ int32_t checked(int32_t p, bool& bad) const {
        if (page_ok(kv, p)) return p;
        bad = true;
        return 0;
    }
    __device__ __forceinline__ int32_t page_of(uint32_t slot, bool& bad) const { return checked(entry_of(slot), bad); }
    __device__ __forceinline__ uint64_t paged_at(int32_t page, uint32_t slot) const {
        return static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_step + (slot & ((1u << kv.shift) - 1)) * dim;
    }
    __device__ __forceinline__ const elem* k_row(uint32_t key, bool& bad) const {
        if constexpr (PAGED) return k + paged_at(page_of(key, bad), key);
        else return k + key * k_stride;
    }
};

// Loads through a buffer descriptor: a unit at or past `bytes` comes back as zeros with no
// test and no branch, so a tile's loads are one straight run. `p` is the same in all lanes.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(bytes), 0x00027000);
}
__device__ __forceinline__ u32x4a buffer_unit(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
    return __builtin_bit_cast(u32x4a, __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(offset), 0, 0));
}
constexpr uint32_t kNowhere = 0xC0000000u;   // a lane's place past every buffer, with room for the tile's offsets
constexpr uint64_t kMaxKvStride = 1u << 23;  // elements: 64 rows below kNowhere bytes

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

// The first of the four dimensions that accumulator registers 4 r .. 4 r + 3 of o[d] hold.
template <class M>
__device__ __forceinline__ uint32_t out_dim(int d, int r, uint32_t h) {
    return M::kRows * d + (M::kRows == 32 ? 8 * r : 0) + 4 * h;
}

// A wave's rows done: normalised output and lse, or (several splits) the parts. The lanes of
// one row hold different dimensions.
template <class M, int QT>
__device__ __forceinline__ void write_rows(const AttnArgs& a, const RowState<M>& st, bool real, uint64_t row, uint32_t head,
                                           uint32_t split, uint32_t lane) {
    const float l = row_sum<M::kRows>(st.l);
    if (!real) return;
    const uint32_t h = lane / M::kRows;
    const bool parts = a.n_splits > 1;
    const uint64_t at = parts ? part_at(a, split, row, head) : 0;
    const float inv = parts ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
    float* pp = a.part + at * a.dim;
    typename M::qelem* p = static_cast<typename M::qelem*>(a.out) + row * a.out_stride + static_cast<uint64_t>(head) * a.dim;
#pragma unroll
    for (int d = 0; d < M::kOut; ++d)
#pragma unroll
        for (int r = 0; r < M::kRegs / 4; ++r) {
            const uint32_t x = out_dim<M>(d, r, h);
            const f32x4 v = {st.o[d][4 * r] * inv, st.o[d][4 * r + 1] * inv, st.o[d][4 * r + 2] * inv, st.o[d][4 * r + 3] * inv};
            if (x < a.dim) {
                if (parts) *reinterpret_cast<f32x4*>(pp + x) = v;
                else store_out<QT>(p + x, v);
            }
        }
    if (h == 0) {
        if (parts) a.part_ml[2 * at] = st.m - M::kShift, a.part_ml[2 * at + 1] = l;
        else if (a.lse)
            a.lse[row * a.n_heads + head] = l == 0.0f ? -kInf : (st.m - M::kShift + __builtin_amdgcn_logf(l)) * kLn2;
    }
}

// Rows of an entry past what max_rows allows for (n_tiles of `rows`): NaN, reported. By the last
// tile's workgroup; a join writes its own.
template <class M>
__device__ __forceinline__ void past_rows(const AttnArgs& a, uint32_t tile, uint32_t rows, uint32_t n_m, int32_t row0,
                                          uint32_t head, uint32_t split) {
    const uint64_t room = static_cast<uint64_t>(a.n_tiles) * rows;
    if (n_m <= room || tile + 1 != a.n_tiles || split) return;
    if (threadIdx.x == 0) atomicOr(a.err, kErrIndex);
    if (a.n_splits > 1) return;
    const float nan = __builtin_nanf("");
    for (uint64_t m = room; m < n_m; ++m) {
        const uint64_t row = static_cast<uint64_t>(row0) + m / a.group;
        const uint32_t q_head = head * a.group + static_cast<uint32_t>(m % a.group);
        typename M::qelem* p = static_cast<typename M::qelem*>(a.out) + row * a.out_stride + static_cast<uint64_t>(q_head) * a.dim;
        for (uint32_t d = threadIdx.x; d < a.dim; d += blockDim.x) p[d] = static_cast<typename M::qelem>(nan);
        if (a.lse && threadIdx.x == 0) a.lse[row * a.n_heads + q_head] = nan;
    }
}

template <class M>
__device__ __forceinline__ bool not_finite(const RowState<M>& st) {
    float x = 0.0f;
#pragma unroll
    for (int d = 0; d < M::kOut; ++d)
#pragma unroll
        for (int r = 0; r < M::kRegs; ++r) x = __builtin_fmaf(st.o[d][r], 0.0f, x);
    return __any(!(x == 0.0f));
}

}  // namespace dev
}  // namespace objeta
