// i8_product.hip — products in 8-bit integers with a scale for each token and each channel:
//
//   out[t][r] = fl(fl(float(sum_k a[t][k] w[r][k]) sa[t]) sw[r]) (+ bias[r])
//
// The sums are whole numbers in 32 bits, exact in any order (at most 131071 columns), so that
// results do not depend on how the work is cut.
#include "dense_common.hpp"
#include "kernels.hpp"

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
};

// Sixteen codes of a row from column k on; columns past the last are 0.
__device__ __forceinline__ i32x4 load_codes(const int8_t* row, uint32_t k, uint32_t cols) {
    if (k + 16 <= cols) return __builtin_bit_cast(i32x4, *reinterpret_cast<const any_u32x4*>(row + k));
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
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

// Few tokens: a workgroup takes 16 channels and 16 NT tokens, its waves share the columns. The
// matrix instruction's operands are sixteen codes of a channel (lane % 16) and of a token, columns
// 16 (lane / 16) on; channels' codes come straight from memory, each once, U loads ahead.
template <int WAVES, int NT, int U, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES) void i8_stream_kernel(I8Args a) {
    __shared__ i32x4 part[WAVES][NT][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r0 = 16 * blockIdx.x, t0 = 16 * NT * blockIdx.y;
    const uint32_t r = r0 + (lane & 15) < a.rows ? r0 + (lane & 15) : a.rows - 1;
    const int8_t* w = a.w + r * a.w_stride;
    const int8_t* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint32_t t = t0 + 16 * n + (lane & 15);
        x[n] = a.a + (t < a.n_tokens ? t : a.n_tokens - 1) * a.a_stride;
    }
    i32x4 nw[U], nx[U][NT];
    auto load = [&](uint32_t k) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t at = k + 64 * u + 16 * (lane >> 4);
            if constexpr (WHOLE) {  // past the last column: channels' codes 0, tokens' any
                const bool in = at < a.cols;
                const i32x4 v = __builtin_bit_cast(i32x4, *reinterpret_cast<const any_u32x4*>(w + (in ? at : 0)));
                nw[u] = in ? v : i32x4{0, 0, 0, 0};
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    nx[u][n] = __builtin_bit_cast(i32x4, *reinterpret_cast<const any_u32x4*>(x[n] + (in ? at : 0)));
            } else {
                nw[u] = load_codes(w, at, a.cols);
#pragma unroll
                for (int n = 0; n < NT; ++n) nx[u][n] = load_codes(x[n], at, a.cols);
            }
        }
    };
    i32x4 sum[NT] = {};
    constexpr uint32_t kStep = 64 * U * WAVES;
    load(64 * U * wave);
    for (uint32_t k = 64 * U * wave; k < a.cols; k += kStep) {
        i32x4 cw[U], cx[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            cw[u] = nw[u];
#pragma unroll
            for (int n = 0; n < NT; ++n) cx[u][n] = nx[u][n];
        }
        if (k + kStep < a.cols) load(k + kStep);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n) sum[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(cw[u], cx[u][n], sum[n], 0, 0, 0);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) part[wave][n][lane] = sum[n];
    __syncthreads();
    for (uint32_t n = wave; n < NT; n += WAVES) {
        i32x4 s = part[0][n][lane];
        for (int i = 1; i < WAVES; ++i) s += part[i][n][lane];
        const uint32_t t = t0 + 16 * n + (lane & 15);
        if (t >= a.n_tokens) continue;
        const float sa = a.sa[t];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t c = r0 + 4 * (lane >> 4) + i;
            if (c < a.rows) store_one(a.out_type, a.out, t * a.out_stride + c, scaled(s[i], sa, a.sw[c], a.bias, a.bias ? a.bias[c] : 0.0f));
        }
    }
}

// Many tokens: a workgroup computes 32 TC WC channels by 32 TT WT tokens over 128 columns at a time.
// These lie twice in LDS, rows of 128 bytes whose 16-byte chunks are exchanged by the row's last three
// bits (chunk c of row r at c ^ (r & 7)), so that eight lanes that read one chunk of eight rows, or
// write a row, touch all banks. The next columns travel through registers: written to the other
// half midway, while those behind them are asked for.
template <int WC, int WT, int TC, int TT, bool WHOLE>
__global__ __launch_bounds__(64 * WC * WT) void i8_tile_kernel(I8Args a, uint32_t tiles_c, uint32_t tiles_t) {
    constexpr uint32_t kThreads = 64 * WC * WT, kC = 32 * TC * WC, kT = 32 * TT * WT;
    constexpr uint32_t kPer = kThreads / 8, kLoads = (kC + kT) / kPer, kLoadsC = kC / kPer;
    constexpr uint32_t kHalf = (kC + kT) * 128;
    static_assert(kC % kPer == 0 && kT % kPer == 0 && TC % 2 == 0, "whole loads, pairs of channel tiles");
    static_assert(2 * kHalf >= WC * WT * 32 * 68 * 4, "a wave's piece of the results fits");
    __shared__ __attribute__((aligned(16))) char lds[2 * kHalf];

    // Workgroups of one XCD take tiles next to one another: eight tiles of tokens by some of channels.
    const uint32_t tiles = tiles_c * tiles_t, each = (tiles + 7) / 8;
    const uint32_t index = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if (index >= tiles || (blockIdx.x >> 3) >= each) return;
    const uint32_t group = index / (8 * tiles_c), in = index % (8 * tiles_c);
    const uint32_t high = tiles_t - 8 * group < 8 ? tiles_t - 8 * group : 8;
    const uint32_t c0 = in / high * kC, t0 = (8 * group + in % high) * kT;

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
    i32x4 stage[kLoads];
    auto load = [&](uint32_t k0) {
        const uint32_t k = k0 + 16 * chunk;
#pragma unroll
        for (uint32_t j = 0; j < kLoads; ++j) {
            if constexpr (WHOLE) {  // columns past the last are out of the buffer's range: zeros
                const int at = k < a.cols ? static_cast<int>(from[j] + k) : -1;
                stage[j] = __builtin_bit_cast(i32x4, j < kLoadsC ? __builtin_amdgcn_raw_buffer_load_b128(rs_c, at, 0, 0)
                                                                 : __builtin_amdgcn_raw_buffer_load_b128(rs_t, at, 0, 0));
            } else {
                stage[j] = load_codes((j < kLoadsC ? base_c : base_t) + from[j], k, a.cols);
            }
        }
    };
    const uint32_t to = first * 128 + 16 * (chunk ^ (first & 7));
    auto put = [&](uint32_t half) {
#pragma unroll
        for (uint32_t j = 0; j < kLoads; ++j) *reinterpret_cast<i32x4*>(lds + half * kHalf + to + j * kPer * 128) = stage[j];
    };

    const uint32_t at_c = (wc * 32 * TC + (lane & 31)) * 128 + 16 * ((lane >> 5) ^ (lane & 7));
    const uint32_t at_t = (kC + wt * 32 * TT + (lane & 31)) * 128 + 16 * ((lane >> 5) ^ (lane & 7));
    i32x16 sum[TC][TT] = {};
    const uint32_t steps = (a.cols + 127) / 128;
    load(0);
    put(0);
    if (steps > 1) load(128);
    __syncthreads();
    for (uint32_t s = 0; s < steps; ++s) {
        const uint32_t half = s & 1;
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
            i32x4 c[TC], t[TT];
#pragma unroll
            for (uint32_t i = 0; i < TC; ++i) c[i] = *reinterpret_cast<const i32x4*>(lds + half * kHalf + (at_c ^ (32 * q)) + i * 4096);
#pragma unroll
            for (uint32_t i = 0; i < TT; ++i) t[i] = *reinterpret_cast<const i32x4*>(lds + half * kHalf + (at_t ^ (32 * q)) + i * 4096);
#pragma unroll
            for (uint32_t i = 0; i < TC; ++i)
#pragma unroll
                for (uint32_t n = 0; n < TT; ++n) sum[i][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(c[i], t[n], sum[i][n], 0, 0, 0);
            if (q == 1 && s + 1 < steps) {
                put(half ^ 1);
                if (s + 2 < steps) load(128 * (s + 2));
            }
        }
        __syncthreads();
    }

    // Results by way of LDS, 32 tokens by 64 channels of a wave at a time, so that eight lanes write
    // 64 neighbouring channels of a token. (A lane of the product holds channels 8 g + 4 (lane / 32) +
    // 0 .. 3 of token lane % 32.)
    int32_t* piece = reinterpret_cast<int32_t*>(lds) + wave * 32 * 68;
#pragma unroll
    for (uint32_t n = 0; n < TT; ++n)
#pragma unroll
        for (uint32_t p = 0; p < TC / 2; ++p) {
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                for (uint32_t g = 0; g < 4; ++g)
                    *reinterpret_cast<i32x4*>(piece + (lane & 31) * 68 + 32 * i + 8 * g + 4 * (lane >> 5)) =
                        i32x4{sum[2 * p + i][n][4 * g], sum[2 * p + i][n][4 * g + 1], sum[2 * p + i][n][4 * g + 2], sum[2 * p + i][n][4 * g + 3]};
            const uint32_t c = c0 + wc * 32 * TC + 64 * p + 8 * (lane & 7);
            const uint32_t left = c < a.rows ? (a.rows - c < 8 ? a.rows - c : 8) : 0;
            float sw[8], bias[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                sw[i] = i < left ? a.sw[c + i] : 0.0f;
                bias[i] = i < left && a.bias ? a.bias[c + i] : 0.0f;
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t row = 8 * j + (lane >> 3), t = t0 + wt * 32 * TT + 32 * n + row;
                if (t >= a.n_tokens || !left) continue;
                const i32x4 u = *reinterpret_cast<const i32x4*>(piece + row * 68 + 8 * (lane & 7));
                const i32x4 v = *reinterpret_cast<const i32x4*>(piece + row * 68 + 8 * (lane & 7) + 4);
                const float sa = a.sa[t];
                float y[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) y[i] = scaled(i < 4 ? u[i & 3] : v[i & 3], sa, sw[i], a.bias, bias[i]);
                store_floats(a.out_type, a.out, t * a.out_stride + c, left, y);
            }
        }
}

}  // namespace dev

using namespace dev;

namespace {

constexpr uint64_t kMaxCols = 131071;  // sums of products of codes from -128 on stay below 2^31

template <int NT, int U>
void launch_stream(hipStream_t s, const I8Args& a, bool whole) {
    const dim3 grid((a.rows + 15) / 16, (a.n_tokens + 16 * NT - 1) / (16 * NT));
    if (whole) hipLaunchKernelGGL((i8_stream_kernel<4, NT, U, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((i8_stream_kernel<4, NT, U, false>), grid, dim3(256), 0, s, a);
}

template <int WC, int WT, int TC, int TT>
void launch_tile(hipStream_t s, const I8Args& a, bool whole) {
    const uint32_t tc = (a.rows + 32 * TC * WC - 1) / (32 * TC * WC), tt = (a.n_tokens + 32 * TT * WT - 1) / (32 * TT * WT);
    const dim3 grid((tc * tt + 7) / 8 * 8), block(64 * WC * WT);
    if (whole) hipLaunchKernelGGL((i8_tile_kernel<WC, WT, TC, TT, true>), grid, block, 0, s, a, tc, tt);
    else hipLaunchKernelGGL((i8_tile_kernel<WC, WT, TC, TT, false>), grid, block, 0, s, a, tc, tt);
}

int32_t launch_i8(hipStream_t s, const I8Args& a, const char* action) {
    // Whole chunks of 16 codes, each at a multiple of 16 bytes.
    const bool whole = (a.cols | a.a_stride | a.w_stride | reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.w)) % 16 == 0;
    const bool near = a.a_stride < (1u << 22) && a.w_stride < (1u << 22);  // a tile's rows within a buffer's 32-bit range
    const uint64_t big = static_cast<uint64_t>((a.rows + 255) / 256) * ((a.n_tokens + 255) / 256);
    if (!near || a.n_tokens <= 64) {
        if (a.n_tokens <= 16) launch_stream<1, 4>(s, a, whole);
        else if (a.n_tokens <= 32) launch_stream<2, 4>(s, a, whole);
        else if (a.n_tokens <= 48) launch_stream<3, 2>(s, a, whole);
        else launch_stream<4, 2>(s, a, whole);
    } else if (big >= 128) {
        launch_tile<2, 4, 4, 2>(s, a, whole);
    } else {
        launch_tile<2, 2, 2, 2>(s, a, whole);
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
    return launch_i8(resolve_stream(ctx, stream), a, action);
    OBJ_GUARD_END
}

}  // extern "C"
