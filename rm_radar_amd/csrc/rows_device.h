// rows_device.h -- device pieces that feature_cache.hip and linear.hip share: typed loads / stores of a few consecutive values at
// any alignment, and the arithmetic of a block-scaled value.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

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

// the same as 4 words
template <class T>
__device__ __forceinline__ u32x4 load_words(const T* p, int have) {
    constexpr int V = 16 / (int)sizeof(T);
    if (have >= V) return *(const u32x4_any*)p;
    union {
        u32x4 u;
        T t[V];
    } o;
    o.u = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < have) o.t[i] = p[i];
    return o.u;
}

template <class T, int V = 16 / (int)sizeof(T)>
__device__ __forceinline__ u32x4 pack_values(const float (&v)[V]) {
    union {
        u32x4 u;
        T t[V];
    } w;
#pragma unroll
    for (int i = 0; i < V; ++i) w.t[i] = from_f32<T>(v[i]);
    return w.u;
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

// the magnitude of the largest of some values as f32 bits: monotonic, infinities and NaN above all others
template <class T, int W>
__device__ __forceinline__ unsigned words_top(const unsigned (&w)[W]) {
    if constexpr (sizeof(T) == 4) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) m = max(m, w[i] & 0x7fffffffu);
        return m;
    } else {
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < W; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, w[i] & 0x7fff7fffu));
        const unsigned short t = m[0] > m[1] ? m[0] : m[1];
        if constexpr (std::is_same_v<T, BF16>) return (unsigned)t << 16;
        return __float_as_uint((float)__builtin_bit_cast(_Float16, t));
    }
}

// W words of a block (all of its values that this lane holds) to e4m3 bytes; exchange(bits) is the maximum over the block's lanes.
// The usual block costs one packed maximum and half a conversion per value: the scaled conversions divide by 2^e and round once.
// Blocks with infinities or NaN, and those of e = -127 (their power of two is an f32 subnormal), go value by value.
template <class T, int W, class Exchange>
__device__ __forceinline__ int quantise_words(const unsigned (&w)[W], unsigned (&q)[W * (int)sizeof(unsigned) / (int)sizeof(T) / 4], const Exchange& exchange) {
    constexpr int N = W * 4 / (int)sizeof(T);   // values
    unsigned top = exchange(words_top<T>(w));
    const bool odd = top >= 0x7f800000u || (top > 0 && top < 0x08000000u);   // 2^-111 and less: e may be -127
    if (__builtin_expect(__any(odd), 0)) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (sizeof(T) == 4)
                v[i] = __uint_as_float(w[i]);
            else
                v[i] = to_f32(T{(unsigned short)(w[i / 2] >> (i & 1) * 16)});
        }
        unsigned t = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) t = is_finite(v[i]) ? max(t, __float_as_uint(v[i]) & 0x7fffffffu) : t;
        top = exchange(t);
        const int e = mx8_exponent(__uint_as_float(top));
        const float inv = mx8_inverse(e);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) q[i] = to_e4m3x4(v + 4 * i, inv);
        return e;
    }
    const int e = mx8_exponent(__uint_as_float(top));
    const float scale = top ? __uint_as_float((unsigned)(e + 127) << 23) : 1.0f;
    typedef short s2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        s2 d = {0, 0};
        if constexpr (std::is_same_v<T, F16>) {
            d = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(d, __builtin_bit_cast(h2, w[2 * i]), scale, false);
            d = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(d, __builtin_bit_cast(h2, w[2 * i + 1]), scale, true);
        } else if constexpr (std::is_same_v<T, BF16>) {
            d = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(d, __builtin_bit_cast(b2, w[2 * i]), scale, false);
            d = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(d, __builtin_bit_cast(b2, w[2 * i + 1]), scale, true);
        } else {
            d = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(d, __uint_as_float(w[4 * i]), __uint_as_float(w[4 * i + 1]), scale, false);
            d = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(d, __uint_as_float(w[4 * i + 2]), __uint_as_float(w[4 * i + 3]), scale, true);
        }
        q[i] = __builtin_bit_cast(unsigned, d);
    }
    return e;
}

}  // namespace rowsdev
}  // namespace rmr
