// dense_common.hpp — what the norm, the 8-bit product and the log probabilities share: host
// checks of their tensors, the context's device made current, element loads and wave sums.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_common.hpp"

namespace objeta {

// Makes the context's device current for a call and gives the caller's back.
class OnDevice {
public:
    explicit OnDevice(int device) {
        if (hipGetDevice(&before_) != hipSuccess || before_ == device) before_ = -1;
        else status_ = hipSetDevice(device);
    }
    ~OnDevice() {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    hipError_t status() const { return status_; }

private:
    int before_ = -1;
    hipError_t status_ = hipSuccess;
};

// Rows of `width` elements of `size` bytes, `stride` elements apart (one row: unused).
inline RowSet row_set(const void* p, uint64_t n, uint64_t stride, uint64_t width, uint64_t size) {
    return RowSet{p, (n > 1 ? stride : width) * size, width * size, n};
}
int32_t check_dense_rows(const char* action, const char* what, const void* p, uint64_t n, uint64_t stride, uint64_t width,
                         uint64_t size);
// That `out` overlaps none of the others; it may be others[own] itself (own -1: none).
int32_t check_dense_apart(const char* action, const char* what, const RowSet& out, const RowSet* others, int n, int own);

#if defined(__HIPCC__)
namespace dev {

// Sixteen and eight bytes at an address of any alignment: this target's global loads take them.
typedef uint32_t any_u32x4 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t any_u32x2 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t reg_u32x4 __attribute__((ext_vector_type(4)));

// Eight elements as they lie in memory; 16-bit types fill `a` alone.
struct Raw8 {
    reg_u32x4 a, b;
};

// Eight elements of row `p` from element i on, of which n are there (others 0).
template <class E>
__device__ __forceinline__ Raw8 load_some(const E* p, uint32_t n) {
    Raw8 r{};
    E* x = reinterpret_cast<E*>(&r);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if (i < n) x[i] = p[i];
    return r;
}
__device__ __forceinline__ Raw8 load_raw8(int32_t type, const void* base, uint64_t at, uint32_t n) {
    if (type == kDtF32) {
        const uint32_t* p = static_cast<const uint32_t*>(base) + at;
        if (n < 8) return load_some(p, n);
        return Raw8{*reinterpret_cast<const any_u32x4*>(p), *reinterpret_cast<const any_u32x4*>(p + 4)};
    }
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if (n < 8) return load_some(p, n);
    return Raw8{*reinterpret_cast<const any_u32x4*>(p), reg_u32x4{0, 0, 0, 0}};
}
// The same of rows that the caches need not keep.
__device__ __forceinline__ Raw8 load_raw8_once(int32_t type, const void* base, uint64_t at, uint32_t n) {
    if (n < 8) return load_raw8(type, base, at, n);
    if (type == kDtF32) {
        const any_u32x4* p = reinterpret_cast<const any_u32x4*>(static_cast<const uint32_t*>(base) + at);
        return Raw8{__builtin_nontemporal_load(p), __builtin_nontemporal_load(p + 1)};
    }
    return Raw8{__builtin_nontemporal_load(reinterpret_cast<const any_u32x4*>(static_cast<const uint16_t*>(base) + at)), reg_u32x4{0, 0, 0, 0}};
}
__device__ __forceinline__ void to_floats(int32_t type, const Raw8& r, float (&x)[8]) {
    if (type == kDtF32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r.a[i]), x[4 + i] = __uint_as_float(r.b[i]);
    } else if (type == kDtBF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(r.a[i] << 16), x[2 * i + 1] = __uint_as_float(r.a[i] & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r.a[i])));
            x[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r.a[i] >> 16)));
        }
    }
}
__device__ __forceinline__ uint32_t bits_of(int32_t type, float x) {  // a 16-bit type's bits, rounded to nearest even
    return type == kDtBF16 ? static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<__bf16>(x)))
                           : static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(x)));
}
__device__ __forceinline__ float rounded_to(int32_t type, float x) {
    if (type == kDtF32) return x;
    return type == kDtBF16 ? static_cast<float>(static_cast<__bf16>(x)) : static_cast<float>(static_cast<_Float16>(x));
}
__device__ __forceinline__ void store_floats(int32_t type, void* base, uint64_t at, uint32_t n, const float (&x)[8]) {
    if (type == kDtF32) {
        float* p = static_cast<float*>(base) + at;
        if (n >= 8) {
            reg_u32x4 a, b;
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(x[i]), b[i] = __float_as_uint(x[4 + i]);
            *reinterpret_cast<any_u32x4*>(p) = a;
            *reinterpret_cast<any_u32x4*>(p + 4) = b;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if (i < n) p[i] = x[i];
        }
        return;
    }
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    reg_u32x4 a;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = bits_of(type, x[2 * i]) | bits_of(type, x[2 * i + 1]) << 16;
    if (n >= 8) {
        *reinterpret_cast<any_u32x4*>(p) = a;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (i < n) p[i] = static_cast<uint16_t>(a[i / 2] >> (16 * (i & 1)));
    }
}

// Over a wave, by moves within its rows of 16 lanes and four reads (a third of the time of six
// exchanges of lanes through LDS). The order of sums is fixed.
template <int CTRL> __device__ __forceinline__ uint32_t moved_or_0(uint32_t v) {
    return __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true);
}
template <int CTRL> __device__ __forceinline__ uint32_t moved_or_same(uint32_t v) {
    return __builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v), CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int l) { return __builtin_amdgcn_readlane(static_cast<int>(v), l); }
__device__ __forceinline__ double lane_of(double v, int l) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, static_cast<uint64_t>(lane_of(static_cast<uint32_t>(u >> 32), l)) << 32 | lane_of(static_cast<uint32_t>(u), l));
}
__device__ __forceinline__ float lane_of(float v, int l) { return __uint_as_float(lane_of(__float_as_uint(v), l)); }
template <int CTRL> __device__ __forceinline__ float add_moved(float v) { return v + __uint_as_float(moved_or_0<CTRL>(__float_as_uint(v))); }
template <int CTRL> __device__ __forceinline__ double add_moved(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t m = static_cast<uint64_t>(moved_or_0<CTRL>(static_cast<uint32_t>(u >> 32))) << 32 | moved_or_0<CTRL>(static_cast<uint32_t>(u));
    return v + __builtin_bit_cast(double, m);
}
template <class T> __device__ __forceinline__ T sum_of_wave(T v) {
    v = add_moved<0x111>(v);
    v = add_moved<0x112>(v);
    v = add_moved<0x114>(v);
    v = add_moved<0x118>(v);
    return (lane_of(v, 15) + lane_of(v, 31)) + (lane_of(v, 47) + lane_of(v, 63));
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }
template <int CTRL> __device__ __forceinline__ uint32_t max_moved(uint32_t v) { return larger(v, moved_or_same<CTRL>(v)); }
template <int CTRL> __device__ __forceinline__ float max_moved(float v) {
    return larger(v, __uint_as_float(moved_or_same<CTRL>(__float_as_uint(v))));
}
template <class T> __device__ __forceinline__ T max_of_wave(T v) {
    v = max_moved<0x111>(v);
    v = max_moved<0x112>(v);
    v = max_moved<0x114>(v);
    v = max_moved<0x118>(v);
    return larger(larger(lane_of(v, 15), lane_of(v, 31)), larger(lane_of(v, 47), lane_of(v, 63)));
}

// A value of the lane that a turn of the row of 16 lanes brings here.
template <int CTRL> __device__ __forceinline__ uint32_t turned(uint32_t v) { return moved_or_same<CTRL>(v); }
template <int CTRL> __device__ __forceinline__ float turned(float v) { return __uint_as_float(moved_or_same<CTRL>(__float_as_uint(v))); }
template <int CTRL> __device__ __forceinline__ double turned(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, static_cast<uint64_t>(moved_or_same<CTRL>(static_cast<uint32_t>(u >> 32))) << 32 | moved_or_same<CTRL>(static_cast<uint32_t>(u)));
}

}  // namespace dev
#endif

}  // namespace objeta
