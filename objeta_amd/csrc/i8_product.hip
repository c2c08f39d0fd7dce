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

__device__ __forceinline__ float scaled(int32_t sum, float sa, float sw, const float* bias, uint32_t r) {
#pragma clang fp contract(off)
    const float x = static_cast<float>(sum) * sa * sw;
    return bias ? x + bias[r] : x;
}

__device__ __forceinline__ void store_one(int32_t type, void* out, uint64_t at, float x) {
    if (type == kDtF32) static_cast<float*>(out)[at] = x;
    else static_cast<uint16_t*>(out)[at] = static_cast<uint16_t>(bits_of(type, x));
}

// Few tokens: a workgroup takes 16 channels and 16 NT tokens, its waves share the columns. The
// matrix instruction's operands are sixteen codes of a channel (lane % 16) and of a token, columns
// 16 (lane / 16) on; channels' codes come straight from memory, each once.
template <int WAVES, int NT>
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
    i32x4 sum[NT] = {};
    for (uint32_t k = 64 * wave; k < a.cols; k += 64 * WAVES) {
        const uint32_t at = k + 16 * (lane >> 4);
        const i32x4 b = load_codes(w, at, a.cols);
#pragma unroll
        for (int n = 0; n < NT; ++n)
            sum[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, load_codes(x[n], at, a.cols), sum[n], 0, 0, 0);
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
            if (c < a.rows) store_one(a.out_type, a.out, t * a.out_stride + c, scaled(s[i], sa, a.sw[c], a.bias, c));
        }
    }
}

}  // namespace dev

using namespace dev;

namespace {

constexpr uint64_t kMaxCols = 131071;  // sums of products of codes from -128 on stay below 2^31

int32_t launch_i8(hipStream_t s, const I8Args& a, const char* action) {
    const dim3 grid((a.rows + 15) / 16, (a.n_tokens + 63) / 64);
    hipLaunchKernelGGL((i8_stream_kernel<4, 4>), grid, dim3(256), 0, s, a);
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
