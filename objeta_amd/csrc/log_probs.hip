// log_probs.hip — log probabilities of given tokens, with the entropy and the best alternatives.
//
// With z = scale x, m = max z: S = sum exp(z - m), lse = m + ln S, log p_i = z_i - lse and
// H = ln S - sum exp(z - m) (z - m) / S, in one pass: a thread keeps a reference R (its largest z so
// far, in units of ln 2), s = sum 2^(z - R) and t = sum 2^(z - R) (z - R), and moves both when R grows:
// with d = R - R', s' = 2^d s and t' = 2^d (t + d s).
//
// The best N: a thread also keeps the largest x of each stretch it read (up to 8; of a cut row four threads
// keep one for their part). The N-th largest of 64 maxima, each of every 64th thread's values (in the join every
// 64th block's), bounds the N-th best from below, so only the few stretches that reach it are read again, and
// what reaches it there is ranked. A value's key is its bits in their order above the
// complement of its index: equal values go by the lowest index. Where too many values reach the bound
// (ties, all of the best in few threads), the N-th value is found bit by bit over the row instead.
//
// Bound: rows that are many by HBM, 16-bit ones by the instructions of an element, some ten, too (2048 rows of
// 151936 floats with the best five 194 us, 6.4 TB/s; bf16 105, 5.9 TB/s); few rows are cut over workgroups, whose parts a
// second launch joins (one row of 151936 floats with the best twenty 9.8 us, two launches).
#include "dense_common.hpp"
#include "kernels.hpp"

namespace objeta {
namespace dev {

constexpr uint32_t kLpJoin = 256;    // threads that join a row's parts; as many parts at most
constexpr uint32_t kLpBlocks = 64;  // of a part
constexpr uint32_t kLpKept = 20;    // blocks' largest that a thread of the join holds
constexpr uint32_t kLpMostParts = kLpKept * kLpJoin / kLpBlocks;  // of a row whose best are asked for
constexpr uint32_t kLpVecs = 2;      // 16-byte loads of a turn; the next turn's are in flight
constexpr uint32_t kLpStretches = 8;  // (with 16, LDS held five workgroups a CU in place of eight)
constexpr uint32_t kLpMostTop = 32;
constexpr uint32_t kLpMostCandidates = 1024;
constexpr uint32_t kLpMostHits = 512;
// References lie between -2^24 and 2^24, where rounding one moves its largest term by a factor of two
// at most. Threads whose values are all lower add nothing to a row within; a row whose largest is
// outside is summed a second time about that value itself.
constexpr float kLpFar = 16777216.0f;

struct LpArgs {
    const void* x;
    uint64_t stride;
    uint64_t first;  // the launch's first row
    uint32_t n_rows, vocab, n_given, n_top, parts, part_size;
    float scale, c;  // c = scale / ln 2
    const int32_t* tokens;
    float *lp, *lse, *entropy, *top;
    int32_t* ids;
    float4* stats;  // [rows][parts]: m, R, s, t
    float* blocks;  // [rows][parts][kLpBlocks]: the largest of what four neighbouring threads read
    uint32_t* err;
};

// A float's bits in the order of floats; NaN below all.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
    if (x != x) return 0;
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o >> 31 ? o & 0x7FFFFFFFu : ~o); }
constexpr uint32_t kOrderedInf = 0x007FFFFFu;  // of -infinity

template <int TYPE> struct LpElem { static constexpr uint32_t kPer = TYPE == kDtF32 ? 4 : 8; };  // elements of 16 bytes

template <int TYPE>
__device__ __forceinline__ float lp_at(const void* row, uint64_t i) {
    if constexpr (TYPE == kDtF32) return static_cast<const float*>(row)[i];
    const uint16_t b = static_cast<const uint16_t*>(row)[i];
    return TYPE == kDtBF16 ? __uint_as_float(static_cast<uint32_t>(b) << 16) : static_cast<float>(__builtin_bit_cast(_Float16, b));
}
template <int TYPE>
__device__ __forceinline__ void lp_floats(const reg_u32x4& r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == kDtF32) x[i] = __uint_as_float(r[i]);
        else if constexpr (TYPE == kDtBF16) x[2 * i] = __uint_as_float(r[i] << 16), x[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
        else {
            x[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r[i])));
            x[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r[i] >> 16)));
        }
    }
}
// 16 bytes from element i on, -infinity behind `end`.
template <int TYPE>
__device__ __forceinline__ reg_u32x4 lp_load(const void* row, uint32_t i, uint32_t end) {
    constexpr uint32_t kPer = LpElem<TYPE>::kPer;
    const char* p = static_cast<const char*>(row) + static_cast<uint64_t>(i) * (16 / kPer);
    if (i + kPer <= end) return *reinterpret_cast<const any_u32x4*>(p);
    reg_u32x4 r;
    if constexpr (TYPE == kDtF32) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) r[j] = i + j < end ? reinterpret_cast<const uint32_t*>(p)[j] : 0xFF800000u;
    } else {
        constexpr uint32_t inf = TYPE == kDtBF16 ? 0xFF80u : 0xFC00u;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t a = i + 2 * j < end ? reinterpret_cast<const uint16_t*>(p)[2 * j] : inf;
            const uint32_t b = i + 2 * j + 1 < end ? reinterpret_cast<const uint16_t*>(p)[2 * j + 1] : inf;
            r[j] = a | b << 16;
        }
    }
    return r;
}

// Sums about a reference, and their join.
struct LpSums {
    float m, ref, s, t;
    __device__ __forceinline__ void move(float to) {
        const float d = __builtin_fmaxf(ref - to, -1000.0f);
        const float f = __builtin_amdgcn_exp2f(d);
        t = f * __builtin_fmaf(d, s, t);
        s *= f;
        ref = to;
    }
};

template <int THREADS>
struct LpShared {
    LpSums sums[THREADS / 64];
    uint32_t max[THREADS];
    uint64_t keys[kLpMostCandidates + 8];
    uint64_t best[kLpMostTop];
    uint16_t hit[kLpMostHits];
    uint32_t hist[256];
    uint32_t count, bound, digit, hits, wave[THREADS / 64];
};

// A row's given token that falls to this thread, read ahead of the rest.
struct LpGiven {
    int32_t token;
    float x;
};
__device__ __forceinline__ int32_t lp_token(const LpArgs& a, uint64_t r, uint32_t g) { return g < a.n_given ? a.tokens[r * a.n_given + g] : -1; }
template <int TYPE>
__device__ __forceinline__ LpGiven lp_given(const LpArgs& a, uint64_t r, int32_t token) {
    LpGiven n{token, 0.0f};
    if (static_cast<uint32_t>(token) < a.vocab) n.x = lp_at<TYPE>(static_cast<const char*>(a.x) + r * a.stride * (16 / LpElem<TYPE>::kPer), token);
    return n;
}

template <int THREADS>
__device__ __forceinline__ LpSums lp_join_all(LpSums v, LpShared<THREADS>& sh) {
    auto over_wave = [](LpSums u) {
        u.move(max_of_wave(u.ref));
        return LpSums{max_of_wave(u.m), u.ref, sum_of_wave(u.s), sum_of_wave(u.t)};
    };
    v = over_wave(v);
    const uint32_t lane = threadIdx.x & 63;
    if (lane == 0) sh.sums[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lane < THREADS / 64 ? sh.sums[lane] : LpSums{-__builtin_inff(), -kLpFar, 0.0f, 0.0f};
    v = over_wave(v);
    __syncthreads();
    return v;
}

// sh.keys[0 .. n) to sh.best, the n_top largest in order, 0 behind the last; keys differ (but for zeros).
template <int THREADS>
__device__ __forceinline__ void lp_rank(LpShared<THREADS>& sh, uint32_t n, uint32_t n_top) {
    if (threadIdx.x < kLpMostTop) sh.best[threadIdx.x] = 0;
    if (threadIdx.x < 8) sh.keys[n + threadIdx.x] = 0;  // whole turns of eight
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
        const uint64_t k = sh.keys[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; j += 8) {
            uint64_t o[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) o[u] = sh.keys[j + u];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) rank += o[u] > k;
        }
        if (rank < n_top) sh.best[rank] = k;
    }
    __syncthreads();
}

__device__ __forceinline__ uint64_t lp_key(uint32_t value, uint32_t index) {
    return static_cast<uint64_t>(value) << 32 | static_cast<uint32_t>(~index);
}

// Appends to sh.keys the elements of [lo, hi) whose ordered value is `value`, the lowest indices
// first, until there are `want` keys.
template <int TYPE, int THREADS>
__device__ void lp_fill(const void* row, uint32_t lo, uint32_t hi, uint32_t value, uint32_t want, LpShared<THREADS>& sh) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t i = lo; i < hi; i += THREADS) {
        const uint32_t have = sh.count;
        if (have >= want) break;
        const uint32_t at = i + threadIdx.x;
        const bool hit = at < hi && ordered(lp_at<TYPE>(row, at)) == value;
        const uint64_t hits = __ballot(hit);
        if (lane == 0) sh.wave[wave] = __popcll(hits);
        __syncthreads();
        uint32_t place = have + __popcll(hits & ((uint64_t(1) << lane) - 1)), all = have;
        for (uint32_t w = 0; w < THREADS / 64; ++w) {
            if (w < wave) place += sh.wave[w];
            all += sh.wave[w];
        }
        if (hit && place < want) sh.keys[place] = lp_key(value, at);
        __syncthreads();
        if (threadIdx.x == 0) sh.count = all < want ? all : want;
        __syncthreads();
    }
}

// The n_top best above -infinity of [lo, hi) by the digits of their values; there are more than n_top.
template <int TYPE, int THREADS>
__device__ void lp_by_digits(const void* row, uint32_t lo, uint32_t hi, uint32_t n_top, LpShared<THREADS>& sh) {
    uint32_t prefix = 0, want = n_top;  // values whose upper digits are the prefix's: `want` of them are among the best
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) sh.hist[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = lo + threadIdx.x; i < hi; i += THREADS) {
            const uint32_t o = ordered(lp_at<TYPE>(row, i));
            if (o > kOrderedInf && (shift == 24 || o >> (shift + 8) == prefix >> (shift + 8))) atomicAdd(&sh.hist[o >> shift & 255], 1u);
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            uint32_t above = 0;
            for (uint32_t d = threadIdx.x + 1; d < 256; ++d) above += sh.hist[d];
            if (above < want && above + sh.hist[threadIdx.x] >= want) sh.digit = threadIdx.x, sh.bound = want - above;
        }
        __syncthreads();
        prefix |= sh.digit << shift;
        want = sh.bound;
        __syncthreads();
    }
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (uint32_t i = lo + threadIdx.x; i < hi; i += THREADS) {
        const uint32_t o = ordered(lp_at<TYPE>(row, i));
        if (o > prefix) sh.keys[atomicAdd(&sh.count, 1u)] = lp_key(o, i);  // n_top - want of them
    }
    __syncthreads();
    lp_fill<TYPE>(row, lo, hi, prefix, n_top, sh);
}

// Bounds the n_top-th best from below by the n_top-th largest of 64 maxima of `mine`, lane by lane over
// the waves; above -infinity. Clears the counts.
template <int THREADS>
__device__ __forceinline__ uint32_t lp_bound(uint32_t mine, uint32_t n_top, LpShared<THREADS>& sh) {
    const uint32_t tid = threadIdx.x;
    sh.max[tid] = mine;
    if (tid == 0) sh.count = sh.hits = 0;
    __syncthreads();
    if (tid < 64) {
        uint32_t most = mine;
#pragma unroll
        for (uint32_t i = 64; i < THREADS; i += 64) most = larger(most, sh.max[tid + i]);
        most = (most & ~63u) | tid;  // all different, and none above what it was but by those bits
        uint32_t rank = 0;
#pragma unroll
        for (uint32_t i = 0; i < 64; ++i) rank += lane_of(most, i) > most;
        if (rank == n_top - 1) sh.bound = larger(most & ~63u, kOrderedInf + 1);
    }
    __syncthreads();
    return sh.bound;
}

template <int THREADS>
__device__ __forceinline__ void lp_hit(uint32_t what, LpShared<THREADS>& sh) {
    const uint32_t place = atomicAdd(&sh.hits, 1u);
    if (place < kLpMostHits) sh.hit[place] = static_cast<uint16_t>(what);
}

// Keys of the values of 16 bytes that reach the bound.
template <int TYPE, int THREADS>
__device__ __forceinline__ void lp_search(const void* row, uint32_t from, uint32_t hi, uint32_t bound, LpShared<THREADS>& sh) {
    float x[LpElem<TYPE>::kPer];
    lp_floats<TYPE>(lp_load<TYPE>(row, from, hi), x);
#pragma unroll
    for (uint32_t u = 0; u < LpElem<TYPE>::kPer; ++u) {
        const uint32_t o = ordered(x[u]);
        if (o < bound) continue;
        const uint32_t place = atomicAdd(&sh.count, 1u);
        if (place < kLpMostCandidates) sh.keys[place] = lp_key(o, from + u);
    }
}

// What a row's sums and best come to.
template <int TYPE, int THREADS>
__device__ void lp_finish(const LpArgs& a, uint64_t r, LpSums v, LpGiven first, LpShared<THREADS>& sh) {
    const void* row = static_cast<const char*>(a.x) + r * a.stride * (16 / LpElem<TYPE>::kPer);
    const uint32_t tid = threadIdx.x;
    const bool none = v.m == -__builtin_inff() && v.s == v.s;  // (the sum is NaN where the row holds one)
    const bool again = v.m != -__builtin_inff() && !(v.ref > -kLpFar && v.ref < kLpFar);
    if (again) {
        LpSums u{v.m, 0.0f, 0.0f, 0.0f};
        for (uint32_t i = tid; i < a.vocab; i += THREADS) {
            const float d = (lp_at<TYPE>(row, i) - v.m) * a.c, e = __builtin_amdgcn_exp2f(d);
            u.s += e;
            u.t = __builtin_fmaf(e, __builtin_fmaxf(d, -200.0f), u.t);
        }
        v = lp_join_all(u, sh);
    }
    constexpr float kLn2 = 0.693147180559945309f;
    const float log_s = __builtin_amdgcn_logf(v.s);  // of base 2
    const float more = (again ? log_s : log_s + __builtin_fmaf(-v.m, a.c, v.ref)) * kLn2;  // ln sum exp(z - m)
    auto not_above_0 = [](float p) { return p > 0.0f ? 0.0f : p; };  // NaN stays
    auto log_prob = [&](float x) {
        if (none) return -__builtin_inff();
        const float d = x - v.m;
        // (logits so far apart that a float does not hold their difference: it may hold the scaled one)
        const float z = d == -__builtin_inff() ? __builtin_fmaf(x, a.scale, -v.m * a.scale) - more : __builtin_fmaf(d, a.scale, -more);
        return not_above_0(z);
    };
    if (tid == 0) {
        if (a.lse) a.lse[r] = none ? -__builtin_inff() : __builtin_fmaf(v.m, a.scale, more);
        if (a.entropy) a.entropy[r] = none ? 0.0f : -not_above_0((v.t / v.s - log_s) * kLn2);
    }
    for (uint32_t g = tid; g < a.n_given; g += THREADS) {
        if (g != tid) first = lp_given<TYPE>(a, r, lp_token(a, r, g));
        float p = 0.0f;
        if (static_cast<uint32_t>(first.token) < a.vocab) {
            p = log_prob(first.x);
        } else if (first.token != -1) {
            p = __builtin_nanf("");
            atomicOr(a.err, kErrIndex);
        }
        a.lp[r * a.n_given + g] = p;
    }
    if (a.n_top) {
        // sh.best holds the values above -infinity; the others by their indices
        if (sh.best[a.n_top - 1] == 0) {
            if (tid == 0) {
                uint32_t n = 0;
                while (n < a.n_top && sh.best[n]) sh.keys[n] = sh.best[n], ++n;
                sh.count = n;
            }
            __syncthreads();
            lp_fill<TYPE>(row, 0, a.vocab, kOrderedInf, a.n_top, sh);
            lp_fill<TYPE>(row, 0, a.vocab, 0, a.n_top, sh);
            if (tid < a.n_top) sh.best[tid] = sh.keys[tid];
            __syncthreads();
        }
        if (tid < a.n_top) {
            const uint64_t k = sh.best[tid];
            const uint32_t index = ~static_cast<uint32_t>(k);
            if (a.ids) a.ids[r * a.n_top + tid] = static_cast<int32_t>(index);
            if (a.top) a.top[r * a.n_top + tid] = k >> 32 ? log_prob(unordered(static_cast<uint32_t>(k >> 32))) : __builtin_nanf("");
        }
    }
}

enum : int { kTopNone = 0, kTopHere = 1, kTopJoin = 2 };  // who finds the best: nobody, this workgroup, the join

// ONCE: logits are not kept in the caches.
template <int TYPE, int TOP, bool ENTROPY, bool ONCE, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS == 256 ? 8 : 4) void lp_part_kernel(LpArgs a) {
    constexpr uint32_t kPer = LpElem<TYPE>::kPer, kStep = THREADS * kPer, kTurn = kLpVecs * kStep;
    __shared__ LpShared<THREADS> sh;
    __shared__ float stretch[TOP == kTopHere ? kLpStretches : 1][THREADS];
    const uint64_t r = a.first + blockIdx.x;
    const uint32_t part = blockIdx.y, tid = threadIdx.x;
    const uint32_t lo = part * a.part_size, hi = a.vocab - lo < a.part_size ? a.vocab : lo + a.part_size;
    const void* row = static_cast<const char*>(a.x) + r * a.stride * (16 / kPer);
    const uint32_t turns = (hi - lo + kTurn - 1) / kTurn, per = (turns + kLpStretches - 1) / kLpStretches;
    const uint32_t whole = (hi - lo) / kTurn;  // turns without an end inside

    const int32_t token = a.parts == 1 ? lp_token(a, r, tid) : -1;
    const float ninf = -__builtin_inff();
    LpSums v{ninf, -kLpFar, 0.0f, 0.0f};
    float longest = ninf;
    uint32_t left = per, g = 0;  // turns until the stretch ends; its index
    reg_u32x4 next[kLpVecs];
    const char* mine_at = static_cast<const char*>(row) + (static_cast<uint64_t>(lo) + tid * kPer) * (16 / kPer);
    auto load = [&](uint32_t turn) {
        if (turn < whole) {
            const any_u32x4* at = reinterpret_cast<const any_u32x4*>(mine_at + static_cast<uint64_t>(turn) * kLpVecs * THREADS * 16);
#pragma unroll
            for (uint32_t u = 0; u < kLpVecs; ++u) next[u] = ONCE ? __builtin_nontemporal_load(at + u * THREADS) : at[u * THREADS];
        } else if (turn < turns) {
#pragma unroll
            for (uint32_t u = 0; u < kLpVecs; ++u) next[u] = lp_load<TYPE>(row, lo + turn * kTurn + u * kStep + tid * kPer, hi);
        }
    };
    load(0);
    const LpGiven given = lp_given<TYPE>(a, r, token);
    for (uint32_t turn = 0; turn < turns; ++turn) {
        float x[kLpVecs][kPer];
#pragma unroll
        for (uint32_t u = 0; u < kLpVecs; ++u) lp_floats<TYPE>(next[u], x[u]);
        load(turn + 1);
        float m = ninf;
#pragma unroll
        for (uint32_t u = 0; u < kLpVecs; ++u)
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) m = __builtin_fmaxf(m, x[u][i]);
        if constexpr (TOP == kTopHere) {
            longest = __builtin_fmaxf(longest, m);
            if (--left == 0 || turn + 1 == turns) {
                stretch[g++][tid] = longest;
                longest = ninf;
                left = per;
            }
        }
        if (m > v.m) {
            v.m = m;
            v.move(__builtin_fmaxf(m * a.c, -kLpFar));
        }
        float s2 = 0.0f, t2 = 0.0f;  // every other one apart: shorter chains
#pragma unroll
        for (uint32_t u = 0; u < kLpVecs; ++u)
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) {
                const float d = __builtin_fmaf(x[u][i], a.c, -v.ref), e = __builtin_amdgcn_exp2f(d);
                (i & 1 ? s2 : v.s) += e;
                if (ENTROPY) (i & 1 ? t2 : v.t) = __builtin_fmaf(e, __builtin_fmaxf(d, -200.0f), i & 1 ? t2 : v.t);
            }
        v.s += s2;
        v.t += t2;
    }
    const float mine = v.m;
    v = lp_join_all(v, sh);

    if constexpr (TOP == kTopHere) {
        const uint32_t key = ordered(mine), bound = lp_bound(key, a.n_top, sh);
        if (key >= bound)
            for (uint32_t j = 0; j < g; ++j)
                if (ordered(stretch[j][tid]) >= bound) lp_hit(tid * kLpStretches + j, sh);
        __syncthreads();
        // Every thread takes 16 bytes of a stretch that was hit.
        const uint32_t each = per * kLpVecs, items = sh.hits <= kLpMostHits ? sh.hits * each : 0;
        for (uint32_t i = tid; i < items; i += THREADS) {
            const uint32_t h = sh.hit[i / each], in = i % each, turn = h % kLpStretches * per + in / kLpVecs;
            if (turn < turns) lp_search<TYPE>(row, lo + turn * kTurn + in % kLpVecs * kStep + h / kLpStretches * kPer, hi, bound, sh);
        }
        __syncthreads();
        if (sh.count > kLpMostCandidates || sh.hits > kLpMostHits) lp_by_digits<TYPE>(row, lo, hi, a.n_top, sh);
        lp_rank(sh, sh.count, a.n_top);
    }
    if (a.parts == 1) {
        lp_finish<TYPE>(a, r, v, given, sh);
        return;
    }
    const uint64_t at = r * a.parts + part;
    if (tid == 0) a.stats[at] = make_float4(v.m, v.ref, v.s, v.t);
    if constexpr (TOP == kTopJoin) {
        static_assert(THREADS == 4 * kLpBlocks, "four threads a block");
        const float m = larger(mine, max_moved<0xB1>(mine));  // of pairs, then of fours
        const float m4 = larger(m, max_moved<0x4E>(m));
        if ((tid & 3) == 0) a.blocks[at * kLpBlocks + tid / 4] = m4;
    }
}

template <int TYPE>
__global__ __launch_bounds__(kLpJoin) void lp_join_kernel(LpArgs a) {
    __shared__ LpShared<kLpJoin> sh;
    const uint64_t r = a.first + blockIdx.x;
    const uint32_t tid = threadIdx.x;
    const int32_t token = lp_token(a, r, tid);
    float4 sums = make_float4(-__builtin_inff(), -kLpFar, 0.0f, 0.0f);
    if (tid < a.parts) sums = a.stats[r * a.parts + tid];
    float kept[kLpKept], mine = -__builtin_inff();  // read beside the sums
    if (a.n_top) {
        const uint32_t all = a.parts * kLpBlocks;
#pragma unroll
        for (uint32_t u = 0; u < kLpKept; ++u) {
            const uint32_t i = tid + u * kLpJoin;
            kept[u] = i < all ? a.blocks[r * all + i] : -__builtin_inff();
        }
    }
    const LpGiven given = lp_given<TYPE>(a, r, token);
    LpSums v{sums.x, sums.y, sums.z, sums.w};
    v = lp_join_all(v, sh);
    if (a.n_top) {
        constexpr uint32_t kPer = LpElem<TYPE>::kPer, kStep = 4 * kLpBlocks * kPer, kTurn = kLpVecs * kStep;
        const void* row = static_cast<const char*>(a.x) + r * a.stride * (16 / kPer);
        const uint32_t turns = a.part_size / kTurn, each = turns * kLpVecs * 4;
#pragma unroll
        for (uint32_t u = 0; u < kLpKept; ++u) mine = larger(mine, kept[u]);
        const uint32_t key = ordered(mine), bound = lp_bound(key, a.n_top, sh);
        if (key >= bound)
#pragma unroll
            for (uint32_t u = 0; u < kLpKept; ++u)
                if (ordered(kept[u]) >= bound) lp_hit(tid + u * kLpJoin, sh);
        __syncthreads();
        const uint32_t items = sh.hits <= kLpMostHits ? sh.hits * each : 0;
        for (uint32_t i = tid; i < items; i += kLpJoin) {
            const uint32_t h = sh.hit[i / each], in = i % each, vec = in / 4;
            const uint32_t from = h / kLpBlocks * a.part_size + vec * kStep + (h % kLpBlocks * 4 + in % 4) * kPer;
            if (from < a.vocab) lp_search<TYPE>(row, from, a.vocab, bound, sh);
        }
        __syncthreads();
        if (sh.count > kLpMostCandidates || sh.hits > kLpMostHits) lp_by_digits<TYPE>(row, 0, a.vocab, a.n_top, sh);
        lp_rank(sh, sh.count, a.n_top);
    }
    lp_finish<TYPE>(a, r, v, given, sh);
}

}  // namespace dev

using namespace dev;

namespace {

template <int TYPE, int TOP, int THREADS>
void launch_part(hipStream_t s, dim3 grid, bool once, const LpArgs& a) {
    if (a.entropy && once) hipLaunchKernelGGL((lp_part_kernel<TYPE, TOP, true, true, THREADS>), grid, dim3(THREADS), 0, s, a);
    else if (a.entropy) hipLaunchKernelGGL((lp_part_kernel<TYPE, TOP, true, false, THREADS>), grid, dim3(THREADS), 0, s, a);
    else if (once) hipLaunchKernelGGL((lp_part_kernel<TYPE, TOP, false, true, THREADS>), grid, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((lp_part_kernel<TYPE, TOP, false, false, THREADS>), grid, dim3(THREADS), 0, s, a);
}
template <int TYPE>
void launch_typed(hipStream_t s, dim3 grid, uint32_t threads, bool once, const LpArgs& a) {
    if (a.parts > 1) {
        if (a.n_top) launch_part<TYPE, kTopJoin, 256>(s, grid, once, a);
        else launch_part<TYPE, kTopNone, 256>(s, grid, once, a);
        hipLaunchKernelGGL((lp_join_kernel<TYPE>), dim3(grid.x), dim3(kLpJoin), 0, s, a);
    } else if (threads == 256) {
        if (a.n_top) launch_part<TYPE, kTopHere, 256>(s, grid, once, a);
        else launch_part<TYPE, kTopNone, 256>(s, grid, once, a);
    } else {
        if (a.n_top) launch_part<TYPE, kTopHere, 1024>(s, grid, once, a);
        else launch_part<TYPE, kTopNone, 1024>(s, grid, once, a);
    }
}

int32_t launch_lp(hipStream_t s, int32_t type, uint32_t threads, bool once, LpArgs a, const char* action) {
    for (a.first = 0; a.first < a.n_rows; a.first += kMostGroups / 4) {
        const uint64_t n = a.n_rows - a.first;
        const dim3 grid(static_cast<uint32_t>(n < kMostGroups / 4 ? n : kMostGroups / 4), a.parts);
        if (type == kDtF32) launch_typed<kDtF32>(s, grid, threads, once, a);
        else if (type == kDtF16) launch_typed<kDtF16>(s, grid, threads, once, a);
        else launch_typed<kDtBF16>(s, grid, threads, once, a);
        OBJ_HIP(hipGetLastError(), action);
    }
    return 0;
}

}  // namespace

}  // namespace objeta

using namespace objeta;

extern "C" {

int32_t objeta_hip_log_probs_device(objeta_hip_context* ctx, objeta_hip_stream stream, uint64_t n_rows, uint64_t vocab,
                                    int32_t dtype, const void* d_logits, uint64_t stride, float scale, const int32_t* d_tokens,
                                    uint64_t n_given, float* d_token_log_probs, float* d_lse, float* d_entropy, uint64_t n_top,
                                    int32_t* d_top_ids, float* d_top_log_probs) {
    OBJ_GUARD_BEGIN
    const char* action = "log_probs_device";
    OBJ_TRY(check_ctx(ctx, action));
    if (vocab == 0 || vocab > kMaxTokens) OBJ_FAIL(kInvalidInput, action, "vocab must be 1 to 2^31 - 2^16");
    if (!dtype_ok(dtype)) OBJ_FAIL(kInvalidInput, action, "dtype must be F32, F16 or BF16");
    if (!(scale > 0.0f && scale < 1e30f)) OBJ_FAIL(kInvalidInput, action, "scale must be positive and finite");
    if (n_given > 1024) OBJ_FAIL(kInvalidInput, action, "at most 1024 given tokens a row");
    if (n_top > kLpMostTop || n_top > vocab) OBJ_FAIL(kInvalidInput, action, "n_top must be at most 32 and the vocab");
    if (n_rows >= (uint64_t(1) << 31)) OBJ_FAIL(kInvalidInput, action, "too many rows");
    if ((n_given != 0) != (d_token_log_probs != nullptr) || (n_given != 0) != (d_tokens != nullptr))
        OBJ_FAIL(kInvalidInput, action, "given tokens and their log probabilities come together with n_given");
    if (n_top != 0 && !d_top_ids) OBJ_FAIL(kInvalidInput, action, "top ids are NULL");
    if (n_top == 0 && (d_top_ids || d_top_log_probs)) OBJ_FAIL(kInvalidInput, action, "top outputs with n_top 0");
    if (!n_given && !n_top && !d_lse && !d_entropy) OBJ_FAIL(kInvalidInput, action, "no output is given");
    if (n_rows == 0) return 0;
    const uint64_t es = dtype_size(dtype);
    OBJ_TRY(check_dense_rows(action, "logits", d_logits, n_rows, stride, vocab, es));
    RowSet sets[7] = {row_set(d_logits, n_rows, stride, vocab, es), row_set(d_tokens, 1, 0, n_rows * n_given, 4)};
    int n_sets = 2;
    const struct { const char* what; const void* p; uint64_t n; } outs[5] = {
        {"token log probs", d_token_log_probs, n_given}, {"lse", d_lse, 1}, {"entropy", d_entropy, 1},
        {"top ids", d_top_ids, n_top}, {"top log probs", d_top_log_probs, n_top}};
    if (d_tokens) OBJ_TRY(check_dense_rows(action, "tokens", d_tokens, 1, 0, n_given, 4));
    for (const auto& o : outs) {
        if (!o.p) continue;
        OBJ_TRY(check_dense_rows(action, o.what, o.p, 1, 0, o.n, 4));
        const RowSet set = row_set(o.p, 1, 0, n_rows * o.n, 4);
        OBJ_TRY(check_dense_apart(action, o.what, set, sets, n_sets, -1));
        sets[n_sets++] = set;
    }
    const OnDevice on(ctx->device);
    OBJ_HIP(on.status(), action);
    const hipStream_t s = resolve_stream(ctx, stream);
    LpArgs a{};
    a.x = d_logits, a.stride = n_rows > 1 ? stride : 0;
    a.n_rows = static_cast<uint32_t>(n_rows), a.vocab = static_cast<uint32_t>(vocab);
    a.n_given = static_cast<uint32_t>(n_given), a.n_top = static_cast<uint32_t>(n_top);
    a.scale = scale, a.c = static_cast<float>(scale * 1.4426950408889634074);
    a.tokens = d_tokens, a.lp = d_token_log_probs, a.lse = d_lse, a.entropy = d_entropy, a.ids = d_top_ids, a.top = d_top_log_probs;
    a.err = ctx->err_word;
    // One workgroup a row where rows fill the card or are short (of 1024 threads while there is a CU for
    // each), otherwise rows are cut and joined. us, 1024 threads / cut: 1 row of 32000 floats 8.3 / 10.5,
    // of 151936 18.3 / 10.8; 64 rows of 50000 in 16 bits 12.0 / 12.9, of 151936 19.8 / 17.5; 200 rows of 151936
    // 20.5 / 24.1. 256 threads / cut: 300 rows of 32000 in 16 bits 14.6 / 16.1, of 151936 42 / 30.
    const uint64_t row_bytes = vocab * es;
    // Logits of 64 MiB and more (held / not kept, us: 2048 rows of 151936 bf16 117 / 105, floats 219 / 194, 8192
    // of 32000 bf16 104 / 94; 64 rows of 151936, 19 MB, 16.4 / 17.6).
    const bool once = n_rows * row_bytes >= (uint64_t(64) << 20);
    const bool large = n_rows <= 256 && (row_bytes <= 200000 || n_rows >= 128);
    const uint32_t threads = large ? 1024 : 256, turn = threads * kLpVecs * (dtype == kDtF32 ? 4 : 8);
    const uint64_t most = (vocab + turn - 1) / turn, want = large || row_bytes <= 100000 ? 1 : 1024 / n_rows;
    uint64_t parts = want < 1 ? 1 : (want < most ? want : most);
    // The join holds the largest of as many parts as it has registers for, since reading them a second time costs
    // more than longer parts up to some 8 million logits: one row with the best twenty in 80 parts / up to 256, us:
    // 200000 floats 11.0 / 13.3, 262144 11.3 / 16.7, a million 15.5 / 29.6, 4 million 23 / 33, 16 million 67 / 49. (With
    // 32 or 64 held in place of 20 a row of 151936 takes 11.3 or 14.5 for 10.6, shorter ones the same.)
    const uint64_t most_parts = n_top ? kLpMostParts : kLpJoin;
    if (parts > most_parts) parts = most_parts;
    const uint64_t size = ((vocab + parts - 1) / parts + turn - 1) / turn * turn;
    a.part_size = static_cast<uint32_t>(size);
    a.parts = static_cast<uint32_t>((vocab + size - 1) / size);
    if (a.parts > 1) {
        void* ws = nullptr;
        const size_t n = static_cast<size_t>(n_rows) * a.parts;
        OBJ_TRY(ensure_workspace(ctx, s, kWsLogProbs, n * (sizeof(float4) + (n_top ? 4 * kLpBlocks : 0)), &ws));
        a.stats = static_cast<float4*>(ws);
        a.blocks = reinterpret_cast<float*>(a.stats + n);
    }
    return launch_lp(s, dtype, threads, once, a, action);
    OBJ_GUARD_END
}

}  // extern "C"
