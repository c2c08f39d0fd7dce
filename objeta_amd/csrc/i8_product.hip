// i8_product.hip — products in 8-bit integers with a scale for each token and each channel:
//
//   out[t][r] = fl(fl(float(sum_k a[t][k] w[r][k]) sa[t]) sw[r]) (+ bias[r])
//
// The sums are whole numbers in 32 bits, exact in any order (at most 131071 columns), so that
// results do not depend on how the work is cut.
//
// Bound: up to some 100 tokens by the channels' codes from HBM (one token of 4096 columns to 151936
// channels 102 us, 6.1 TB/s; 32 tokens 124, 5.2 TB/s), beyond by the matrix cores, whose clock real codes draw down
// (4099 tokens of 4096 to 14336 228 to 236 us, 2.04 to 2.11 POP/s); small products by a workgroup's chain of loads,
// products and their join.
#include "dense_common.hpp"
#include "kernels.hpp"

#include <cmath>
#include <type_traits>

namespace objeta {
namespace dev {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

struct I8Args {
    const int8_t *a, *w;
    const float *sa, *sw, *bias;
    void* out;
    uint64_t a_stride, w_stride, out_stride;
    uint32_t n_tokens, rows, cols;
    int32_t out_type;
    bool once;  // channels' codes are not kept in the caches
};

typedef uint32_t word_u32x4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ i32x4 load16(const int8_t* p) { return __builtin_bit_cast(i32x4, *reinterpret_cast<const word_u32x4*>(p)); }

// Rows that begin anywhere: loads off a word's boundary take twice as long, so that the whole words
// around sixteen codes are read and moved together when they are used.
struct Raw16 {
    i32x4 v;
    uint32_t w;
};
// The words of the sixteen codes at base + off, base a multiple of 4; a fifth one where they reach into it.
__device__ __forceinline__ Raw16 load_raw16(const int8_t* base, uint32_t off) {
    const int8_t* p = base + (off & ~3u);
    return Raw16{load16(p), *reinterpret_cast<const uint32_t*>(base + ((off & ~3u) + (off & 3 ? 16 : 12)))};
}
__device__ __forceinline__ i32x4 straight(const Raw16& r, uint32_t off) {
    const uint32_t a = r.v[0], b = r.v[1], c = r.v[2], d = r.v[3], n = off & 3;
    return i32x4{static_cast<int32_t>(__builtin_amdgcn_alignbyte(b, a, n)), static_cast<int32_t>(__builtin_amdgcn_alignbyte(c, b, n)),
                 static_cast<int32_t>(__builtin_amdgcn_alignbyte(d, c, n)), static_cast<int32_t>(__builtin_amdgcn_alignbyte(r.w, d, n))};
}
// Sixteen codes moved down by n, zeros behind them.
__device__ __forceinline__ i32x4 moved(const i32x4& v, uint32_t n) {
    uint64_t lo = static_cast<uint32_t>(v[0]) | static_cast<uint64_t>(static_cast<uint32_t>(v[1])) << 32;
    uint64_t hi = static_cast<uint32_t>(v[2]) | static_cast<uint64_t>(static_cast<uint32_t>(v[3])) << 32;
    const uint32_t bits = 8 * (n & 7);
    if (n >= 16) lo = hi = 0;
    if (n >= 8) lo = hi, hi = 0;
    if (bits) lo = lo >> bits | hi << (64 - bits), hi >>= bits;
    return i32x4{static_cast<int32_t>(lo), static_cast<int32_t>(lo >> 32), static_cast<int32_t>(hi), static_cast<int32_t>(hi >> 32)};
}
// Where a row's sixteen codes from column k on are read: past its last sixteen, there (and moved down).
__device__ __forceinline__ uint32_t read_at(uint32_t k, uint32_t cols) { return k + 16 <= cols ? k : cols - 16; }
// Codes of a row of fewer than sixteen.
__device__ __forceinline__ i32x4 load_few(const int8_t* row, uint32_t k, uint32_t cols) {
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 15; ++i)
        if (k + i < cols) v[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i % 4));
    return i32x4{static_cast<int32_t>(v[0]), static_cast<int32_t>(v[1]), static_cast<int32_t>(v[2]), static_cast<int32_t>(v[3])};
}

__device__ __forceinline__ float scaled(int32_t sum, float sa, float sw, bool add, float bias) {
#pragma clang fp contract(off)
    const float x = static_cast<float>(sum) * sa * sw;
    return add ? x + bias : x;
}

__device__ __forceinline__ void store_one(int32_t type, void* out, uint64_t at, float x) {
    if (type == kDtF32) static_cast<float*>(out)[at] = x;
    else static_cast<uint16_t*>(out)[at] = static_cast<uint16_t>(bits_of(type, x));
}

// Few tokens: a workgroup takes 16 channels and 16 tokens, its eight waves share the columns. The
// matrix instruction's operands are sixteen codes of a channel (lane % 16) and of a token, columns
// 16 (lane / 16) on; channels' codes come straight from memory, each once, four loads ahead. (One token:
// 4096 of 14336 columns 12.9 us, 4.6 TB/s; 151936 of 4096 103 us, 6.0 TB/s. Loads past the caches
// changed nothing here. 32 channels a workgroup read tokens' codes half as often, but 4096 channels
// are then 128 workgroups: 18 us; the 151936 take 111.)
constexpr int kStreamWaves = 8, kStreamAhead = 4;
template <bool WHOLE>
__global__ __launch_bounds__(64 * kStreamWaves) void i8_stream_kernel(I8Args a) {
    __shared__ i32x4 part[kStreamWaves][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r0 = 16 * blockIdx.x, t0 = 16 * blockIdx.y, r = r0 + (lane & 15), t = t0 + (lane & 15);
    // (past the last channel and token: these again)
    const int8_t* const row[2] = {a.w + (r < a.rows ? r : a.rows - 1) * a.w_stride, a.a + (t < a.n_tokens ? t : a.n_tokens - 1) * a.a_stride};
    typedef typename std::conditional<WHOLE, i32x4, Raw16>::type Raw;
    typedef Raw Stage[kStreamAhead][2];
    auto load = [&](Stage& v, uint32_t k) {
#pragma unroll
        for (int u = 0; u < kStreamAhead; ++u)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint32_t at = k + 64 * u + 16 * (lane >> 4);
                if constexpr (WHOLE) {
                    v[u][n] = load16(row[n] + (at < a.cols ? at : 0));
                } else if (a.cols >= 16) {
                    const uint64_t p = reinterpret_cast<uint64_t>(row[n]);
                    v[u][n] = load_raw16(reinterpret_cast<const int8_t*>(p & ~uint64_t(3)), static_cast<uint32_t>(p & 3) + read_at(at, a.cols));
                } else {
                    v[u][n] = Raw16{load_few(row[n], at, a.cols), 0};
                }
            }
    };
    // past the last column: channels' codes 0, tokens' any
    auto codes = [&](const Raw& v, int n, uint32_t k, uint32_t at) {
        if constexpr (WHOLE) {
            return n == 0 && at >= a.cols ? i32x4{0, 0, 0, 0} : v;
        } else {
            if (a.cols < 16) return v.v;
            const uint32_t from = read_at(at, a.cols);
            const i32x4 x = straight(v, static_cast<uint32_t>(reinterpret_cast<uint64_t>(row[n])) + from);
            return k + 64 <= a.cols ? x : moved(x, at - from);
        }
    };
    i32x4 sum = {};
    constexpr uint32_t kEach = 64 * kStreamAhead, kStep = kEach * kStreamWaves;
    Stage next;
    load(next, kEach * wave);
    for (uint32_t k = kEach * wave; k < a.cols; k += kStep) {
        Stage now;
#pragma unroll
        for (int u = 0; u < kStreamAhead; ++u) now[u][0] = next[u][0], now[u][1] = next[u][1];
        if (k + kStep < a.cols) load(next, k + kStep);
#pragma unroll
        for (int u = 0; u < kStreamAhead; ++u) {
            const uint32_t at = k + 64 * u + 16 * (lane >> 4);
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(codes(now[u][0], 0, k + 64 * u, at), codes(now[u][1], 1, k + 64 * u, at), sum, 0, 0, 0);
        }
    }
    part[wave][lane] = sum;
    __syncthreads();
    if (wave || t >= a.n_tokens) return;
    i32x4 s = part[0][lane];
#pragma unroll
    for (int v = 1; v < kStreamWaves; ++v) s += part[v][lane];
    const float sa = a.sa[t];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t c = r0 + 4 * (lane >> 4) + j;
        if (c < a.rows) store_one(a.out_type, a.out, t * a.out_stride + c, scaled(s[j], sa, a.sw[c], a.bias, a.bias ? a.bias[c] : 0.0f));
    }
}

constexpr int kOnce = 2;  // a buffer load that asks the caches not to keep its lines

// More tokens: a workgroup computes 32 TC WC channels by 32 TT WT tokens, 128 KG columns a step; each
// of KG groups of WC WT waves takes 128 of these, and the groups' sums are added at the end. A group's
// columns lie twice in LDS, rows of 128 bytes whose 16-byte chunks are exchanged by the row (chunk c of
// row r at c ^ (r / 2 % 8)), so that sixteen lanes that read one chunk of sixteen rows, or write two rows, touch all
// 64 banks (a read of a wave: 4.4 cycles; exchanged by r % 8 it took 8.1, of rows as they are 32; a
// write 13). The next AHEAD steps' columns travel in registers: the first of them
// is written to the other half midway, and those behind the last are asked for in its place.
template <int WC, int WT, int TC, int TT, int KG, int AHEAD, bool WHOLE>
__global__ __launch_bounds__(64 * WC * WT * KG, 2) void i8_tile_kernel(I8Args a, uint32_t tiles_c, uint32_t tiles_t) {
    constexpr uint32_t kGroup = 64 * WC * WT, kC = 32 * TC * WC, kT = 32 * TT * WT;
    constexpr uint32_t kPer = kGroup / 8, kLoads = (kC + kT) / kPer, kLoadsC = kC / kPer;
    constexpr uint32_t kHalf = (kC + kT) * 128;
    constexpr uint32_t kPitch = TC > 1 ? 68 : 36;  // words of a row of results
    // Eight waves, two of a SIMD: they take turns, one multiplying while the other moves operands.
    constexpr bool kTurns = WC * WT * KG == 8;
    constexpr uint32_t kSums = (KG - 1) * kGroup * TC * TT * 64, kPieces = WC * WT * 32 * kPitch * 4;
    constexpr uint32_t kBytes = 2 * KG * kHalf > kSums + kPieces ? 2 * KG * kHalf : kSums + kPieces;
    static_assert(kC % kPer == 0 && kT % kPer == 0, "whole loads");
    __shared__ __attribute__((aligned(16))) char lds[kBytes];
    __shared__ float sh_sw[kC], sh_bias[kC], sh_sa[kT];

    // Workgroups of one XCD take tiles next to one another: eight tiles of tokens by some of channels.
    const uint32_t tiles = tiles_c * tiles_t, each = (tiles + 7) / 8;
    const uint32_t index = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if (index >= tiles || (blockIdx.x >> 3) >= each) return;
    const uint32_t group = index / (8 * tiles_c), in = index % (8 * tiles_c);
    const uint32_t high = tiles_t - 8 * group < 8 ? tiles_t - 8 * group : 8;
    const uint32_t c0 = in / high * kC, t0 = (8 * group + in % high) * kT;

    const uint32_t tid = threadIdx.x % kGroup, lane = tid & 63, wave = tid >> 6;
    const uint32_t kg = __builtin_amdgcn_readfirstlane(threadIdx.x / kGroup);
    const uint32_t wc = wave % WC, wt = wave / WC;
    const uint32_t chunk = tid & 7, first = tid >> 3;

    const uint32_t rows_c = a.rows - c0 < kC ? a.rows - c0 : kC, rows_t = a.n_tokens - t0 < kT ? a.n_tokens - t0 : kT;
    const int8_t* base_c = a.w + c0 * a.w_stride;
    const int8_t* base_t = a.a + t0 * a.a_stride;
    const auto rs_c = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base_c), 0,
                                                        static_cast<int>((rows_c - 1) * a.w_stride + a.cols), 0x00027000);
    const auto rs_t = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base_t), 0,
                                                        static_cast<int>((rows_t - 1) * a.a_stride + a.cols), 0x00027000);
    uint32_t from[kLoads];  // of this thread's rows (the last one again past it), their chunk
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
        const uint32_t r = first + kPer * (j < kLoadsC ? j : j - kLoadsC), n = j < kLoadsC ? rows_c : rows_t;
        from[j] = (r < n ? r : n - 1) * static_cast<uint32_t>(j < kLoadsC ? a.w_stride : a.a_stride);
    }
    typedef typename std::conditional<WHOLE, i32x4, Raw16>::type Raw;
    typedef Raw Stage[kLoads];
    Stage stage[AHEAD];
    // (rows that begin anywhere are addressed from the word ahead of the first)
    const uint32_t low_c = reinterpret_cast<uint64_t>(base_c) & 3, low_t = reinterpret_cast<uint64_t>(base_t) & 3;
    const uint32_t last = a.cols < 16 ? 0 : a.cols - 16;
    auto load = [&](Stage& v, uint32_t step, uint32_t j0, uint32_t j1) {
        const uint32_t k = 128 * (step * KG + kg) + 16 * chunk;
        // (Larger tiles have no registers for it; 64 x 64 takes 172 with the choice, 164 without, and two workgroups a CU for three.)
        if constexpr (WHOLE && kC * kT <= 8192) {
            if (a.once) {
#pragma unroll
                for (uint32_t j = j0; j < j1; ++j) {
                    const int at = k < a.cols ? static_cast<int>(from[j] + k) : -1;
                    v[j] = __builtin_bit_cast(i32x4, j < kLoadsC ? __builtin_amdgcn_raw_buffer_load_b128(rs_c, at, 0, kOnce)
                                                                 : __builtin_amdgcn_raw_buffer_load_b128(rs_t, at, 0, 0));
                }
                return;
            }
        }
#pragma unroll
        for (uint32_t j = j0; j < j1; ++j) {
            if constexpr (WHOLE) {  // columns past the last are out of the buffer's range: zeros
                const int at = k < a.cols ? static_cast<int>(from[j] + k) : -1;
                v[j] = __builtin_bit_cast(i32x4, j < kLoadsC ? __builtin_amdgcn_raw_buffer_load_b128(rs_c, at, 0, 0)
                                                             : __builtin_amdgcn_raw_buffer_load_b128(rs_t, at, 0, 0));
            } else {
                const uint32_t low = j < kLoadsC ? low_c : low_t;
                v[j] = load_raw16((j < kLoadsC ? base_c : base_t) - low, low + from[j] + (k < last ? k : last));
            }
        }
    };
    char* const mine = lds + kg * 2 * kHalf;
    auto put = [&](const Stage& v, uint32_t step, uint32_t j0, uint32_t j1) {
#pragma unroll
        for (uint32_t j = j0; j < j1; ++j) {
            const uint32_t turn = kPer % 16 ? (first + kPer * j) / 2 % 8 : first / 2 % 8;
            i32x4 x;
            if constexpr (WHOLE) {
                x = v[j];
            } else {
                const uint32_t k0 = 128 * (step * KG + kg), k = k0 + 16 * chunk, at = k < last ? k : last;
                x = straight(v[j], (j < kLoadsC ? low_c : low_t) + from[j] + at);
                if (k0 + 128 > a.cols) x = moved(x, k - at);
            }
            *reinterpret_cast<i32x4*>(mine + (step & 1) * kHalf + (first + kPer * j) * 128 + 16 * (chunk ^ turn)) = x;
        }
    };

    const uint32_t at_c = (wc * 32 * TC + (lane & 31)) * 128 + 16 * ((lane >> 5) ^ (lane / 2 % 8));
    const uint32_t at_t = (kC + wt * 32 * TT + (lane & 31)) * 128 + 16 * ((lane >> 5) ^ (lane / 2 % 8));
    i32x16 sum[TC][TT] = {};
    const uint32_t steps = (a.cols + 128 * KG - 1) / (128 * KG);
    load(stage[0], 0, 0, kLoads);
    for (uint32_t i = threadIdx.x; i < kC; i += kGroup * KG) {
        const bool there = i < rows_c;
        sh_sw[i] = there ? a.sw[c0 + i] : 0.0f;
        sh_bias[i] = there && a.bias ? a.bias[c0 + i] : 0.0f;
    }
    for (uint32_t i = threadIdx.x; i < kT; i += kGroup * KG) sh_sa[i] = i < rows_t ? a.sa[t0 + i] : 0.0f;
    put(stage[0], 0, 0, kLoads);
    // (Loads keep their order, so that a wait for one step's leaves the later ones in flight.)
#pragma unroll
    for (uint32_t d = 0; d < AHEAD; ++d) {
        load(stage[d], 1 + d, 0, kLoads);
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    i32x4 c[2][TC], t[2][TT];  // operands of two quarters
    auto take = [&](uint32_t half, uint32_t q) {
#pragma unroll
        for (uint32_t i = 0; i < TC; ++i) c[q & 1][i] = *reinterpret_cast<const i32x4*>(mine + half * kHalf + (at_c ^ (32 * q)) + i * 4096);
#pragma unroll
        for (uint32_t i = 0; i < TT; ++i) t[q & 1][i] = *reinterpret_cast<const i32x4*>(mine + half * kHalf + (at_t ^ (32 * q)) + i * 4096);
    };
    auto multiply = [&](uint32_t q) {
#pragma unroll
        for (uint32_t i = 0; i < TC; ++i)
#pragma unroll
            for (uint32_t n = 0; n < TT; ++n)
                sum[i][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(c[q & 1][i], t[q & 1][n], sum[i][n], 0, 0, 0);
    };
    auto meet = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto step = [&](Stage& v, uint32_t s) {
        const uint32_t half = s & 1;
        if constexpr (kTurns) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                take(half, 2 * h);
                take(half, 2 * h + 1);
                put(v, s + 1, h * kLoads / 2, (h + 1) * kLoads / 2);
                load(v, s + 1 + AHEAD, h * kLoads / 2, (h + 1) * kLoads / 2);
                meet();
                __builtin_amdgcn_s_setprio(1);
                multiply(0);
                multiply(1);
                __builtin_amdgcn_s_setprio(0);
                meet();
            }
        } else {
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {
                if (q < 3) {
                    take(half, q + 1);
                } else {
                    __syncthreads();
                    take(half ^ 1, 0);
                }
                if (q == 1) {
                    put(v, s + 1, 0, kLoads);
                    __builtin_amdgcn_sched_barrier(0);
                    load(v, s + 1 + AHEAD, 0, kLoads);
                }
                __builtin_amdgcn_sched_barrier(0);
                multiply(q);
            }
        }
    };
    const bool second = kTurns && __builtin_amdgcn_readfirstlane(threadIdx.x) >= 256;
    if (second) meet();
    if constexpr (!kTurns) take(0, 0);
    // Whole groups of AHEAD steps, then what is left: a way out of the loop's middle would leave the
    // order of loads unknown at its top.
    uint32_t s = 0;
    for (; s + AHEAD <= steps; s += AHEAD)
#pragma unroll
        for (uint32_t d = 0; d < AHEAD; ++d) step(stage[d], s + d);
#pragma unroll
    for (uint32_t d = 0; d + 1 < AHEAD; ++d)
        if (s + d < steps) step(stage[d], s + d);
    if (kTurns && !second) meet();
    __syncthreads();

    if constexpr (KG > 1) {
        i32x4* others = reinterpret_cast<i32x4*>(lds + kPieces);
        auto at = [&](uint32_t g, uint32_t i, uint32_t n, uint32_t v) { return ((((g - 1) * TC + i) * TT + n) * 4 + v) * kGroup + tid; };
#pragma unroll
        for (uint32_t i = 0; i < TC; ++i)
#pragma unroll
            for (uint32_t n = 0; n < TT; ++n)
#pragma unroll
                for (uint32_t v = 0; v < 4; ++v)
                    if (kg) others[at(kg, i, n, v)] = i32x4{sum[i][n][4 * v], sum[i][n][4 * v + 1], sum[i][n][4 * v + 2], sum[i][n][4 * v + 3]};
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (uint32_t g = 1; g < KG; ++g)
#pragma unroll
            for (uint32_t i = 0; i < TC; ++i)
#pragma unroll
                for (uint32_t n = 0; n < TT; ++n)
#pragma unroll
                    for (uint32_t v = 0; v < 4; ++v) {
                        const i32x4 o = others[at(g, i, n, v)];
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) sum[i][n][4 * v + e] += o[e];
                    }
    }

    // Results by way of LDS, 32 tokens by 64 (32) channels of a wave at a time, so that eight (four)
    // lanes write neighbouring channels of a token. (A lane of the product holds channels
    // 8 g + 4 (lane / 32) + 0 .. 3 of token lane % 32.)
    int32_t* piece = reinterpret_cast<int32_t*>(lds) + wave * 32 * kPitch;
#pragma unroll
    for (uint32_t n = 0; n < TT; ++n)
#pragma unroll
        for (uint32_t p = 0; p < TC; p += 2) {
            const uint32_t tiles_here = p + 1 < TC ? 2 : 1, lanes = 4 * tiles_here;  // of a token's row
#pragma unroll
            for (uint32_t i = 0; i < tiles_here; ++i)
#pragma unroll
                for (uint32_t g = 0; g < 4; ++g)
                    *reinterpret_cast<i32x4*>(piece + (lane & 31) * kPitch + 32 * i + 8 * g + 4 * (lane >> 5)) =
                        i32x4{sum[p + i][n][4 * g], sum[p + i][n][4 * g + 1], sum[p + i][n][4 * g + 2], sum[p + i][n][4 * g + 3]};
            const uint32_t at = 8 * (lane % lanes), in_c = wc * 32 * TC + 32 * p + at;
            const uint32_t left = in_c < rows_c ? (rows_c - in_c < 8 ? rows_c - in_c : 8) : 0;
            float sw[8], bias[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) sw[i] = sh_sw[in_c + i], bias[i] = sh_bias[in_c + i];
#pragma unroll
            for (uint32_t j = 0; j < lanes / 2; ++j) {
                const uint32_t row = j * (64 / lanes) + lane / lanes, in_t = wt * 32 * TT + 32 * n + row;
                const i32x4 u = *reinterpret_cast<const i32x4*>(piece + row * kPitch + at);
                const i32x4 v = *reinterpret_cast<const i32x4*>(piece + row * kPitch + at + 4);
                const float sa = sh_sa[in_t];
                float y[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) y[i] = scaled(i < 4 ? u[i & 3] : v[i & 3], sa, sw[i], a.bias, bias[i]);
                if (in_t < rows_t && left) store_floats(a.out_type, a.out, (t0 + in_t) * a.out_stride + c0 + in_c, left, y);
            }
        }
}

// Rows that begin anywhere copied to multiples of 16 bytes, zeros up to these behind them.
__global__ __launch_bounds__(256) void i8_straighten_kernel(const int8_t* from, uint64_t stride, uint32_t rows, uint32_t cols, int8_t* to) {
    const uint32_t chunks = (cols + 15) / 16;
    const uint64_t all = static_cast<uint64_t>(rows) * chunks;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<uint64_t>(gridDim.x) * 256) {
        const uint32_t r = static_cast<uint32_t>(i / chunks), k = 16 * static_cast<uint32_t>(i % chunks), at = read_at(k, cols);
        const uint64_t p = reinterpret_cast<uint64_t>(from + r * stride);
        const uint32_t off = static_cast<uint32_t>(p & 3) + at;
        const i32x4 v = straight(load_raw16(reinterpret_cast<const int8_t*>(p & ~uint64_t(3)), off), off);
        reinterpret_cast<i32x4*>(to)[i] = at == k ? v : moved(v, k - at);
    }
}

}  // namespace dev

using namespace dev;

namespace {

constexpr uint64_t kMaxCols = 131071;  // sums of products of codes from -128 on stay below 2^31

void launch_stream(hipStream_t s, const I8Args& a, bool whole) {
    const dim3 grid((a.rows + 15) / 16, (a.n_tokens + 15) / 16), block(64 * kStreamWaves);
    if (whole) hipLaunchKernelGGL((i8_stream_kernel<true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((i8_stream_kernel<false>), grid, block, 0, s, a);
}

template <int WC, int WT, int TC, int TT, int KG, int AHEAD, bool WHOLE>
void launch_tile(hipStream_t s, const I8Args& a) {
    const uint32_t tc = (a.rows + 32 * TC * WC - 1) / (32 * TC * WC), tt = (a.n_tokens + 32 * TT * WT - 1) / (32 * TT * WT);
    hipLaunchKernelGGL((i8_tile_kernel<WC, WT, TC, TT, KG, AHEAD, WHOLE>), dim3((tc * tt + 7) / 8 * 8), dim3(64 * WC * WT * KG), 0, s, a, tc, tt);
}
// (Rows that begin anywhere need registers for moving them and load one step ahead.)
template <int WC, int WT, int TC, int TT, int KG, int AHEAD>
void launch_either(hipStream_t s, const I8Args& a, bool whole) {
    if (whole) launch_tile<WC, WT, TC, TT, KG, AHEAD, true>(s, a);
    else launch_tile<WC, WT, TC, TT, KG, 1, false>(s, a);
}

// What a tile costs, in us, measured over batches of 5 to 8192 tokens and matrices of 512 to 160000
// channels by 64 to 14336 columns: `fixed` around the columns; for 128 columns `low` where a CU has one
// workgroup and few others run, `full` a workgroup of a full card, where the products of real codes
// draw the clock down (8192^3: 450 us, of zeros 318). `resident` workgroups share a CU, as far as registers go and, of
// rows that begin anywhere (fewer loads ahead, 90 to 178 registers for 172 to 246), LDS; eight waves have it to
// themselves. `again` is what each further round of them adds, whose loads begin beside the last one's products (300
// tokens of 4096 to 14336: five 64 x 64 tiles a CU 49.0 us, 128 x 256 38.5; 8192 of 1024 to 28672: 28 of 128 x 128 390,
// 14 of 256 x 256 345; 15 of 328 to 52105, anywhere: four of 64 x 64 9.9, two of 128 x 128 11.5).
struct TileCost {
    uint32_t channels, tokens, resident, resident_anywhere;
    double fixed, again, low, full;
};
enum : int { kTile256, kTile128x256, kTile128, kTile64x128, kTile64, kTile32x64, kTile32, kTiles };
constexpr TileCost kTileCosts[kTiles] = {
    {256, 256, 1, 1, 6.7, 6.7, 1.03, 1.70}, {128, 256, 1, 1, 5.1, 5.1, 0.85, 1.15}, {128, 128, 2, 2, 3.7, 2.6, 0.65, 0.60},
    {64, 128, 2, 3, 3.9, 2.6, 0.42, 0.39},  {64, 64, 2, 4, 3.6, 1.6, 0.30, 0.23},   {32, 64, 1, 1, 4.2, 4.2, 0.21, 0.22},
    {32, 32, 1, 1, 4.9, 4.9, 0.15, 0.16},
};

// The tile that would take the least time: large ones do the most products for what they load, but
// few of them leave CUs idle, and rounds of them the last one part empty (2048 tokens of 4096 to
// 4096: 256 x 256 47 us, 128 x 256 43; 4096 tokens: 65 and 84. 64 tokens of 14336 to 4096: 64 x 64 38,
// 32 x 32 with eight groups along the columns 22; 64 of 4096 to 14336: 18 and 37).
int best_tile(const I8Args& a, bool whole) {
    const double steps = (a.cols + 127) / 128;
    const int first = whole ? kTile256 : kTile128x256;
    int best = first;
    double least = 0;
    for (int i = first; i < kTiles; ++i) {
        const TileCost& c = kTileCosts[i];
        const double tiles = static_cast<double>((a.rows + c.channels - 1) / c.channels) * ((a.n_tokens + c.tokens - 1) / c.tokens);
        const double each = ceil(tiles / 256);  // of the CU with most
        const double rounds = ceil(each / (whole ? c.resident : c.resident_anywhere));
        double us = c.fixed + (rounds - 1) * c.again;
        if (c.resident > 1) {
            us += steps * (each * c.full > c.low ? each * c.full : c.low);
        } else {
            const double busy = tiles < 256 ? tiles / 256 : 1;
            us += steps * each * (c.low + (c.full - c.low) * busy);
        }
        if (i == first || us < least) best = i, least = us;
    }
    return best;
}

// Whole chunks of 16 codes, each at a multiple of 16 bytes.
bool whole_chunks(const I8Args& a) {
    return (a.cols | a.a_stride | a.w_stride | reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.w)) % 16 == 0;
}

// Rows that begin anywhere cost the tiles moves of all they load: where tokens and channels are many,
// both are copied to a workspace first (4000 tokens and channels of 4003 columns: 131 us, with the
// copies 85; 512 tokens, 14336 channels of 4095: 71 with them, 65 without).
constexpr uint64_t kMostStraight = uint64_t(1) << 30;
int32_t straighten(objeta_hip_context* ctx, hipStream_t s, I8Args& a, const char* action) {
    const uint64_t pitch = (static_cast<uint64_t>(a.cols) + 15) / 16 * 16, n = a.n_tokens, r = a.rows;
    if (n * r < 800 * (n + r) || a.cols < 16 || (n + r) * pitch > kMostStraight) return 0;
    // Powers of two, so that the workspace stays within the largest copies and the regions that it
    // outgrew (kept for graphs that use them) come to less than it together.
    uint64_t bytes = uint64_t(1) << 20;
    while (bytes < (n + r) * pitch) bytes *= 2;
    // Captured without a workspace, or with no memory for one: read as they are.
    if (!workspace_ready(ctx, s, kWsCodes, bytes)) return 0;
    void* ws = nullptr;
    if (ensure_workspace(ctx, s, kWsCodes, bytes, &ws) != 0) return 0;
    int8_t* to = static_cast<int8_t*>(ws);
    hipLaunchKernelGGL(i8_straighten_kernel, dim3(2048), dim3(256), 0, s, a.a, a.a_stride, a.n_tokens, a.cols, to);
    hipLaunchKernelGGL(i8_straighten_kernel, dim3(2048), dim3(256), 0, s, a.w, a.w_stride, a.rows, a.cols, to + n * pitch);
    OBJ_HIP(hipGetLastError(), action);
    a.a = to, a.w = to + n * pitch, a.a_stride = a.w_stride = pitch, a.cols = static_cast<uint32_t>(pitch);
    return 0;
}

int32_t launch_i8(objeta_hip_context* ctx, hipStream_t s, I8Args a, const char* action) {
    if (!whole_chunks(a)) OBJ_TRY(straighten(ctx, s, a, action));
    const bool whole = whole_chunks(a);
    // Codes of channels past what the last-level cache keeps from one layer's turn to the next: 64 tokens of
    // 4096 to 14336 19.1 and 17.3 us, 17 of 4096 to 32000 33.0 and 30.2; 64 of 2048 to 5120 (which it keeps)
    // 7.6 and 8.7.
    a.once = static_cast<uint64_t>(a.rows) * a.cols >= (uint64_t(32) << 20) && a.n_tokens <= 256;
    const bool near = a.a_stride < (1u << 22) && a.w_stride < (1u << 22);  // a tile's rows within a buffer's 32-bit range
    // Tiles load tokens' codes once for more channels, and pass large matrices by the caches: 8 tokens of
    // 4096 to 14336 14.4 us, streamed 16.7 (one: 14.5 and 14.6), of 4096 to 151936 106 and 128 (one: 103 and
    // 102), of 4095 to 14336 20.6 and 27.2, of 14336 to 4096 19.1 and 14.5 (16 tokens: 19.7 and 18.0).
    const uint32_t few = a.rows >= 7168 ? 2 : 16;
    if (a.n_tokens <= few || !near || a.cols < 16) {
        launch_stream(s, a, whole);
    } else {
        switch (best_tile(a, whole)) {
            case kTile256: launch_tile<2, 4, 4, 2, 1, 1, true>(s, a); break;
            case kTile128x256: launch_either<2, 4, 2, 2, 1, 2>(s, a, whole); break;
            case kTile128: launch_either<2, 2, 2, 2, 1, 2>(s, a, whole); break;
            case kTile64x128: launch_either<2, 2, 1, 2, 1, 3>(s, a, whole); break;
            case kTile64:
                // Up to 32 tokens a tile half as high, two groups along the columns: 32 tokens of 4096 to 14336
                // 16.8 -> 14.8 us, to 151936 139 -> 126, 20 of 4095 to 14336 28.7 -> 21.5; of 1024 to
                // 32000 9.3 and 10.5.
                if (a.n_tokens <= 32 && a.cols >= 2048) launch_either<2, 1, 1, 1, 2, 4>(s, a, whole);
                else launch_either<2, 2, 1, 1, 1, 3>(s, a, whole);
                break;
            case kTile32x64: launch_either<1, 2, 1, 1, 4, 2>(s, a, whole); break;
            default: launch_either<1, 1, 1, 1, 8, 3>(s, a, whole); break;
        }
    }
    OBJ_HIP(hipGetLastError(), action);
    return 0;
}

}  // namespace

}  // namespace objeta

using namespace objeta;

extern "C" {

int32_t objeta_hip_i8_product_device(objeta_hip_context* ctx, objeta_hip_stream stream, uint64_t n_tokens, uint64_t rows,
                                     uint64_t cols, const int8_t* d_a, uint64_t a_stride, const float* d_a_scales,
                                     const int8_t* d_w, uint64_t w_stride, const float* d_w_scales, const float* d_bias,
                                     int32_t out_dtype, void* d_out, uint64_t out_stride) {
    OBJ_GUARD_BEGIN
    const char* action = "i8_product_device";
    OBJ_TRY(check_ctx(ctx, action));
    if (cols == 0 || cols > kMaxCols)
        OBJ_FAIL(kInvalidInput, action, strf("cols %llu must be 1 to 131071", (unsigned long long)cols));
    if (rows >= (uint64_t(1) << 24)) OBJ_FAIL(kInvalidInput, action, "too many rows");
    if (n_tokens > 65535 * 16) OBJ_FAIL(kInvalidInput, action, "too many tokens");
    if (!dtype_ok(out_dtype)) OBJ_FAIL(kInvalidInput, action, "out dtype must be F32, F16 or BF16");
    if (n_tokens == 0 || rows == 0) return 0;
    const uint64_t os = dtype_size(out_dtype);
    OBJ_TRY(check_dense_rows(action, "a", d_a, n_tokens, a_stride, cols, 1));
    OBJ_TRY(check_dense_rows(action, "a scales", d_a_scales, n_tokens, 1, 1, 4));
    OBJ_TRY(check_dense_rows(action, "w", d_w, rows, w_stride, cols, 1));
    OBJ_TRY(check_dense_rows(action, "w scales", d_w_scales, rows, 1, 1, 4));
    if (d_bias) OBJ_TRY(check_dense_rows(action, "bias", d_bias, rows, 1, 1, 4));
    OBJ_TRY(check_dense_rows(action, "out", d_out, n_tokens, out_stride, rows, os));
    const RowSet in[5] = {row_set(d_a, n_tokens, a_stride, cols, 1), row_set(d_w, rows, w_stride, cols, 1),
                          row_set(d_a_scales, n_tokens, 1, 1, 4), row_set(d_w_scales, rows, 1, 1, 4), row_set(d_bias, rows, 1, 1, 4)};
    OBJ_TRY(check_dense_apart(action, "out", row_set(d_out, n_tokens, out_stride, rows, os), in, 5, -1));
    I8Args a{};
    a.a = d_a, a.w = d_w, a.sa = d_a_scales, a.sw = d_w_scales, a.bias = d_bias, a.out = d_out;
    a.a_stride = n_tokens > 1 ? a_stride : 0, a.w_stride = rows > 1 ? w_stride : 0, a.out_stride = n_tokens > 1 ? out_stride : 0;
    a.n_tokens = static_cast<uint32_t>(n_tokens), a.rows = static_cast<uint32_t>(rows), a.cols = static_cast<uint32_t>(cols);
    a.out_type = out_dtype;
    const OnDevice on(ctx->device);
    OBJ_HIP(on.status(), action);
    return launch_i8(ctx, resolve_stream(ctx, stream), a, action);
    OBJ_GUARD_END
}

}  // extern "C"
