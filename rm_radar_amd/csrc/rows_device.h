// rows_device.h -- device pieces that feature_cache.hip and linear.hip share: typed loads / stores of a few consecutive values at
// any alignment, and the arithmetic of a block-scaled value.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "rows.h"

namespace rmr {
namespace rowsdev {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
// global memory takes 16-byte accesses at any alignment of the element type
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

struct F16 {
    unsigned short b;
};
struct BF16 {
    unsigned short b;
};

__device__ __forceinline__ float to_f32(F16 v) { return (float)__builtin_bit_cast(_Float16, v.b); }
__device__ __forceinline__ float to_f32(BF16 v) { return __uint_as_float((unsigned)v.b << 16); }
__device__ __forceinline__ float to_f32(float v) { return v; }

// one rounding, to nearest even
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ F16 from_f32<F16>(float v) {
    return F16{__builtin_bit_cast(unsigned short, (_Float16)v)};
}
template <>
__device__ __forceinline__ BF16 from_f32<BF16>(float v) {
    return BF16{__builtin_bit_cast(unsigned short, (__bf16)v)};
}
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}

// V = 16 / sizeof(T) consecutive values, the first `have` of them there (the others read as zero)
template <class T, int V = 16 / (int)sizeof(T)>
__device__ __forceinline__ void load_values(const T* p, int have, float (&v)[V]) {
    union {
        u32x4 u;
        T t[V];
    } w;
    if (have >= V) {
        w.u = *(const u32x4_any*)p;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f32(w.t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < have ? to_f32(p[i]) : 0.0f;
    }
}

template <class T, int V = 16 / (int)sizeof(T)>
__device__ __forceinline__ void store_values(T* p, int have, const float (&v)[V]) {
    union {
        u32x4 u;
        T t[V];
    } w;
#pragma unroll
    for (int i = 0; i < V; ++i) w.t[i] = from_f32<T>(v[i]);
    if (have >= V) {
        *(u32x4_any*)p = w.u;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < have) p[i] = w.t[i];
    }
}

__device__ __forceinline__ bool is_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// the block's exponent from its largest finite magnitude: the smallest e >= -127 with top <= 448 * 2^e (448 = 1.75 * 2^8)
__device__ __forceinline__ int mx8_exponent(float top) {
    const unsigned b = __float_as_uint(top);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -127 ? -127 : e;
}
// 2^-e for e in [-127, 120] (an f32's largest exponent needs no more)
__device__ __forceinline__ float mx8_inverse(int e) { return __uint_as_float((unsigned)(127 - e) << 23); }
// 2^e from the stored byte e + 127 (byte 0: the subnormal 2^-127)
__device__ __forceinline__ float mx8_scale(unsigned byte) { return __uint_as_float(byte ? byte << 23 : 0x400000u); }
// where the scale byte of block b of a row sits
__device__ __forceinline__ int mx8_scale_at(int b) { return (b >> 4) * 16 + (b & 3) * 4 + ((b >> 2) & 3); }

// 4 values times `inv` to 4 e4m3 bytes.  The product with a power of two is exact wherever it is not far below the smallest
// e4m3 value, so this is the one rounding.
__device__ __forceinline__ unsigned to_e4m3x4(const float* v, float inv) {
    float u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = is_finite(v[i]) ? v[i] * inv : __uint_as_float(0x7fc00000u);
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], w, true);
    return (unsigned)w;
}

}  // namespace rowsdev
}  // namespace rmr
