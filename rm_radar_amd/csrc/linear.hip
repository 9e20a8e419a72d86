// linear.hip -- y = act(x W^T + b) + residual on the matrix pipe, f32 accumulation, one rounding to y's type.
//
// All three formats (f16, bf16, block-scaled e4m3) are moved the same way, in K steps of 128 bytes along a row = eight chunks
// of 16 bytes.  Lane (slot = lane & 15, g = lane >> 4) of a 16-row MFMA operand needs chunks g and g + 4 of its row: two operands
// of 16x16x32 (16-bit types: chunk h * 4 + g is k = 32 h + 8 g ... + 7) or the two halves of one 16x16x128 (e4m3).
//
// Operands are swapped (D = W x): a lane ends with output features of ONE row.  The features of a group of 64 are dealt to the
// four 16-row operands j as feature = 16 g + 4 j + i for D row 4 g + i, so that lane group g holds the 16 CONSECUTIVE features
// 16 g ... 16 g + 15 of its row: bias, residual and y move in whole 16-byte pieces without any exchange between lanes.
//
// Weights are laid out once, in the order of the operand registers: [group of 64][K step][j][half][lane][16 bytes], zeros behind
// the last feature and the last k.  A group's step is 8 KiB contiguous, copied to LDS as it is and read back at lane * 16:
// no bank conflicts, no address arithmetic.  x is copied to LDS by rows of 128 bytes, chunk c of row r at position c ^ (r >> 1 & 7),
// which spreads the 16 rows of a fragment read over all 64 banks.
#include <type_traits>
#include <utility>

#include "rows_device.h"

namespace rmr {
namespace {

using namespace rowsdev;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// what the kernels multiply: the three formats, and mx8 rows expanded to bf16 on their way into the matrix pipe.  Inside one
// instruction the 8-bit products are lined up to the largest of their group and cut 13 bits below it (measured with two cancelling
// products and a third).  On rows and weights of random blocks that leaves the sums 1.5e-5 (at most 1.3e-4) of the norm of their
// products off, for K of 576 to 4300.  Half a step of a 16-bit y is 2^-9 or 2^-11 of y: it hides that unless the sum cancels to a few
// per cent of its products.  That is the 8-bit rate's price, and a caller who does not want to pay it asks for an f32 y.  That call
// takes kMx8Wide: an e4m3 value times its power of two IS a bf16 value (but for values below 2^-126, which get bf16's subnormal
// steps), and bf16 products are summed in full f32, at half the rate: 1.3e-7 (at most 1.4e-6) of the norm.
enum { kF16 = RMR_LINEAR_F16, kBf16 = RMR_LINEAR_BF16, kMx8 = RMR_LINEAR_MX8, kMx8Wide };

constexpr int kStepBytes = 128;      // of a row, per K step
constexpr int kGroupStep = 8192;     // bytes of one K step of 64 output features

// f(integral_constant<K>) ... f(integral_constant<N - 1>)
template <int K, int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (K < N) {
        f(std::integral_constant<int, K>{});
        static_for<K + 1, N>(std::forward<F>(f));
    }
}

// ------------------------------------------------------------------------------------------------ laying out the weights

// feature of the group of 64 that sits in slot `slot` of operand j
__device__ __forceinline__ int feature_of(int j, int slot) { return (slot >> 2) * 16 + j * 4 + (slot & 3); }

struct PackArgs {
    const void* w;
    int64_t ldw;
    int n, k, ksteps, groups;
    unsigned char* out;
};

template <class S, class T>
__global__ __launch_bounds__(256) void pack_weight_kernel(PackArgs a) {
    const int64_t pieces = (int64_t)a.groups * a.ksteps * (kGroupStep / 16);
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < pieces; p += (int64_t)gridDim.x * 256) {
        const int lane = (int)(p & 63), h = (int)(p >> 6) & 1, j = (int)(p >> 7) & 3;
        const int64_t gs = p >> 9;
        const int step = (int)(gs % a.ksteps), group = (int)(gs / a.ksteps);
        const int64_t n = (int64_t)group * 64 + feature_of(j, lane & 15);
        const int k = step * 64 + (h * 4 + (lane >> 4)) * 8;
        union {
            u32x4 u;
            T t[8];
        } o;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o.t[i] = from_f32<T>(n < a.n && k + i < a.k ? to_f32(((const S*)a.w)[n * a.ldw + k + i]) : 0.0f);
        *(u32x4*)(a.out + p * 16) = o.u;
    }
}

struct PackMx8Args {
    Mx8Rows rows;
    int n, ksteps, groups;
    unsigned char* out;
    unsigned* scale;
};

__global__ __launch_bounds__(256) void pack_mx8_kernel(PackMx8Args a) {
    const int64_t pieces = (int64_t)a.groups * a.ksteps * (kGroupStep / 16);
    const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, stride = (int64_t)gridDim.x * 256;
    for (int64_t p = first; p < pieces; p += stride) {
        const int lane = (int)(p & 63), h = (int)(p >> 6) & 1, j = (int)(p >> 7) & 3;
        const int64_t gs = p >> 9;
        const int step = (int)(gs % a.ksteps), group = (int)(gs / a.ksteps);
        const int64_t n = (int64_t)group * 64 + feature_of(j, lane & 15);
        u32x4 v = {0, 0, 0, 0};
        if (n < a.n) v = *(const u32x4*)(a.rows.data + n * a.rows.pitch + step * kStepBytes + (h * 4 + (lane >> 4)) * 16);
        *(u32x4*)(a.out + p * 16) = v;
    }
    const int quads = (a.ksteps + 3) / 4;
    const int64_t words = (int64_t)a.groups * quads * 256;
    for (int64_t p = first; p < words; p += stride) {
        const int lane = (int)(p & 63), j = (int)(p >> 6) & 3;
        const int64_t gq = p >> 8;
        const int quad = (int)(gq % quads), group = (int)(gq / quads);
        const int64_t n = (int64_t)group * 64 + feature_of(j, lane & 15);
        a.scale[p] = n < a.n ? *(const unsigned*)(a.rows.scale + n * a.rows.scale_pitch + quad * 16 + (lane >> 4) * 4) : 0u;
    }
}

// rows of 16-bit values to rows of `pitch` bytes, zeros behind the last value: for rows whose length or alignment does not
// allow 16-byte pieces
struct AlignArgs {
    const void* x;
    int64_t ld, n;
    int width, per_row;   // 16-byte pieces of a row
    unsigned magic;       // ceil(2^31 / per_row): i / per_row = i magic >> 31
    int rows;             // rows of a workgroup
    unsigned char* out;
};

__global__ __launch_bounds__(256) void align_rows_kernel(AlignArgs a) {
    const int64_t groups = (a.n + a.rows - 1) / a.rows;
    for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        const int64_t r0 = g * a.rows;
        const int pieces = (int)(a.n - r0 < a.rows ? a.n - r0 : a.rows) * a.per_row;
        for (int i = threadIdx.x; i < pieces; i += 256) {
            const int r = (int)(((uint64_t)(unsigned)i * a.magic) >> 31), c = (i - r * a.per_row) * 8;
            const F16* src = (const F16*)a.x + (r0 + r) * a.ld + c;   // (any 16-bit type)
            *(u32x4*)(a.out + (r0 * a.per_row + i) * 16) = load_words<F16>(src, a.width - c);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------- the epilogue

// the activation of a result that is rounded to T behind it
template <class T, int ACT>
__device__ __forceinline__ float activate(float v) {
    constexpr float kLog2e = 1.44269504f;
    if constexpr (ACT == RMR_ACT_RELU) return v < 0.0f ? 0.0f : v;
    if constexpr (ACT == RMR_ACT_SILU) return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * v));
    if constexpr (ACT == RMR_ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * v));
    if constexpr (ACT == RMR_ACT_GELU) {
        // v / 2 erfc(-v / sqrt 2) = v Phi(v), with Phi(-z) = e^(-z z / 2) g(z) for z = |v|, so that the negative side keeps its relative
        // precision however small it gets.  g(z) = erfcx(z / sqrt 2) / 2 is t P(t), t = 1 / (1 + p z): the coefficients minimise the
        // largest relative error for z <= 14.5, behind which the power is zero.  Degree 8 for an f32 result (2e-8; 4.5e-7 evaluated in
        // f32); degree 5 is off by 5e-6, a hundredth of half a step of f16 (8192^3 bf16: 2 % less time than with degree 8).
        constexpr bool kLong = sizeof(T) == 4;
        const float t = __builtin_amdgcn_rcpf(fmaf(kLong ? 0.21f : 0.31f, fabsf(v), 1.0f));
        float q;
        if constexpr (kLong) {
            q = fmaf(-0.0712944732f, t, 0.2818030221f);
            q = fmaf(q, t, -0.3264901234f);
            q = fmaf(q, t, 0.3449831350f);
            q = fmaf(q, t, -0.0907701970f);
            q = fmaf(q, t, 0.1234710871f);
            q = fmaf(q, t, 0.0695700082f);
            q = fmaf(q, t, 0.0850123999f);
            q = fmaf(q, t, 0.0837151507f);
        } else {
            q = fmaf(-0.0739291299f, t, 0.1804503092f);
            q = fmaf(q, t, 0.0157447480f);
            q = fmaf(q, t, 0.1334297684f);
            q = fmaf(q, t, 0.1204412802f);
            q = fmaf(q, t, 0.1238607030f);
        }
        q *= t * __builtin_amdgcn_exp2f(-0.5f * kLog2e * (v * v));
        return v * (v < 0.0f ? q : 1.0f - q);
    }
    return v;
}

struct LinearArgs {
    // rows: chunk c of row i at x + (slots ? slots[i] : i) * x_pitch + c * 16
    const unsigned char* x;
    int64_t x_pitch;
    const unsigned char* x_scale;   // mx8
    int64_t x_scale_pitch;
    const int64_t* slots;
    int64_t n_slots;
    int64_t rows;
    int last_chunks;   // 16-byte chunks of a row that the last K step has
    const unsigned char* zero;
    const unsigned char* w;
    const unsigned* w_scale;
    const float* bias;
    int ksteps, groups, out_features;
    const void* residual;
    int64_t ldr;
    void* y;
    int64_t ldy;
    int y_type, act;
    int64_t row_tiles;
    int col_tiles;
    // K split over workgroups: split i multiplies steps [i * split_steps, ...) and leaves its f32 sums in
    // partial[i][rows][64 groups]; a second launch joins them in order.  0: one workgroup does all of K
    int split_steps;
    float* partial;
};

// One operand row of the epilogue: 16 features c0 ... c0 + 15 of one row of x, v[j][i] = feature c0 + 4 j + i before the bias.  A wave
// whose rows and features are all there takes the straight path: residual loads of a batch of rows first, then arithmetic and
// stores, 16 bytes each.
template <class T, int ACT, int MT, int Q, bool PRE, class Acc>
__device__ __forceinline__ void finish_full(const LinearArgs& a, Acc&& acc, const u32x4 (&pre)[PRE ? MT : 1][4], const f32x4 (&bias)[4], int64_t row0, int c0) {
    constexpr int V = 16 / (int)sizeof(T), P = 16 / V;   // values of a piece, pieces of 16 features
    constexpr int B = MT < 4 ? MT : 4;                   // rows of a batch
    T* y = (T*)a.y + row0 * a.ldy + c0;
    const T* r = a.residual ? (const T*)a.residual + row0 * a.ldr + c0 : nullptr;
    const int64_t ystep = 16 * a.ldy, rstep = 16 * a.ldr;
    static_for<0, MT / B>([&](auto batch) {
        u32x4 rv[B][P];
        if constexpr (PRE) {
#pragma unroll
            for (int m = 0; m < B; ++m)
#pragma unroll
                for (int p = 0; p < P; ++p) rv[m][p] = pre[decltype(batch)::value * B + m][p];
        } else if (r) {
#pragma unroll
            for (int m = 0; m < B; ++m) {
#pragma unroll
                for (int p = 0; p < P; ++p) rv[m][p] = *(const u32x4_any*)(r + p * V);
                r += rstep;
            }
        }
        static_for<0, B>([&](auto in) {
            constexpr int b = decltype(in)::value, m = decltype(batch)::value * B + b;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                union {
                    u32x4 u;
                    T t[V];
                } w;
                w.u = r ? rv[b][p] : u32x4{0, 0, 0, 0};
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int k = p * V + i;
                    o[i] = activate<T, ACT>(acc(std::integral_constant<int, m>{})[Q * 4 + (k >> 2)][k & 3] + bias[k >> 2][k & 3]);
                    if (r) o[i] += to_f32(w.t[i]);
                }
                store_values<T>(y + p * V, V, o);
            }
            y += ystep;
        });
    });
}

// a wave at an edge: its MT x 16 values per lane wait in LDS (`spill`, 64 bytes a lane and row, pitch 1024 floats), so that the loop over
// the rows is one piece of code
template <class T>
__device__ __forceinline__ void finish_edge(const LinearArgs& a, const float* spill, int mt, int64_t row, int c0) {
    constexpr int V = 16 / (int)sizeof(T);
    const int have = a.out_features - c0;
    if (have <= 0) return;
    f32x4 bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[j] = *(const f32x4*)(a.bias + c0 + j * 4);
#pragma unroll 1
    for (int m = 0; m < mt; ++m, row += 16, spill += 1024) {
        if (row >= a.rows) return;
        T* y = (T*)a.y + row * a.ldy + c0;
        float rv[16 / V][V];
        if (a.residual) {
            const T* r = (const T*)a.residual + row * a.ldr + c0;
#pragma unroll
            for (int p = 0; p < 16 / V; ++p) load_values<T>(r + p * V, have - p * V, rv[p]);
        }
        float o[16 / V][V];
        const auto fill = [&](auto act) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 v = *(const f32x4*)(spill + 4 * j) + bias[j];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[(4 * j + i) / V][(4 * j + i) % V] = activate<T, decltype(act)::value>(v[i]);
            }
        };
        switch (a.act) {
            case RMR_ACT_RELU: fill(std::integral_constant<int, RMR_ACT_RELU>{}); break;
            case RMR_ACT_SILU: fill(std::integral_constant<int, RMR_ACT_SILU>{}); break;
            case RMR_ACT_GELU: fill(std::integral_constant<int, RMR_ACT_GELU>{}); break;
            case RMR_ACT_SIGMOID: fill(std::integral_constant<int, RMR_ACT_SIGMOID>{}); break;
            default: fill(std::integral_constant<int, RMR_ACT_NONE>{}); break;
        }
#pragma unroll
        for (int p = 0; p < 16 / V; ++p) {
            if (a.residual)
#pragma unroll
                for (int i = 0; i < V; ++i) o[p][i] += rv[p][i];
            if (have > p * V) store_values<T>(y + p * V, have - p * V, o[p]);
        }
    }
}

// a wave's 16 MT rows x 64 features: operand set Q of acc(m)
template <int MT>
__device__ __forceinline__ bool all_there(const LinearArgs& a, int64_t row0, int n0) {
    return row0 + 16 * MT <= a.rows && n0 + 64 <= a.out_features;
}

template <class T, int MT, int Q, bool PRE, class Acc>
__device__ __forceinline__ void finish_typed(const LinearArgs& a, Acc&& acc, const u32x4 (&pre)[PRE ? MT : 1][4], float* spill, int64_t row0, int n0, int lane) {
    const int c0 = n0 + (lane >> 4) * 16;
    const int64_t row = row0 + (lane & 15);
    if (all_there<MT>(a, row0, n0)) {
        f32x4 bias[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) bias[j] = *(const f32x4*)(a.bias + c0 + j * 4);
        switch (a.act) {
            case RMR_ACT_RELU: finish_full<T, RMR_ACT_RELU, MT, Q, PRE>(a, acc, pre, bias, row, c0); break;
            case RMR_ACT_SILU: finish_full<T, RMR_ACT_SILU, MT, Q, PRE>(a, acc, pre, bias, row, c0); break;
            case RMR_ACT_GELU: finish_full<T, RMR_ACT_GELU, MT, Q, PRE>(a, acc, pre, bias, row, c0); break;
            case RMR_ACT_SIGMOID: finish_full<T, RMR_ACT_SIGMOID, MT, Q, PRE>(a, acc, pre, bias, row, c0); break;
            default: finish_full<T, RMR_ACT_NONE, MT, Q, PRE>(a, acc, pre, bias, row, c0); break;
        }
    } else {
        static_for<0, MT>([&](auto mm) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *(f32x4*)(spill + decltype(mm)::value * 1024 + 4 * j) = acc(mm)[Q * 4 + j];
        });
        finish_edge<T>(a, spill, MT, row, c0);
    }
}

template <int MT, int Q, bool PRE, class Acc>
__device__ __forceinline__ void finish_group(const LinearArgs& a, Acc&& acc, const u32x4 (&pre)[PRE ? MT : 1][4], float* spill, int64_t row0, int n0, int lane) {
    if (a.y_type == RMR_TYPE_F16)
        finish_typed<F16, MT, Q, PRE>(a, acc, pre, spill, row0, n0, lane);
    else if (a.y_type == RMR_TYPE_BF16)
        finish_typed<BF16, MT, Q, PRE>(a, acc, pre, spill, row0, n0, lane);
    else
        finish_typed<float, MT, Q, PRE>(a, acc, pre, spill, row0, n0, lane);
}

// ------------------------------------------------------------------------------------------------------- the tile kernel

// 64 lanes x 16 bytes of global memory to LDS at lds + lane * 16 where `mask` is -1, nothing where it is 0 (uniform; the wave's 64
// lanes are all active here)
__device__ __forceinline__ uint64_t lanes_of(int mask) {
    const unsigned m = (unsigned)__builtin_amdgcn_readfirstlane(mask);
    return (uint64_t)m << 32 | m;
}
__device__ __forceinline__ void dma_lane(unsigned lds, const unsigned char* p, int mask) {
    asm volatile("s_mov_b32 m0, %0\n\ts_mov_b64 exec, %2\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b64 exec, -1"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p), "s"(lanes_of(mask))
                 : "memory");
}
// two KiB in a row: an instruction's offset counts on both sides, so the second address is given 1024 less
__device__ __forceinline__ void dma_lane_pair(unsigned lds, const unsigned char* p, const unsigned char* q, int mask) {
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_mov_b64 exec, %3\n\tglobal_load_lds_dwordx4 %1, off\n\tglobal_load_lds_dwordx4 %2, off offset:1024\n\ts_mov_b64 exec, -1"
        :
        : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p), "v"(q), "s"(lanes_of(mask))
        : "memory");
}
// the same from a uniform address + lane offset, OFFSET bytes further on both sides
template <int OFFSET>
__device__ __forceinline__ void dma_uniform_pair(unsigned lds, const unsigned char* base, unsigned off, int mask) {
    const uint64_t b = (uint64_t)base;
    const uint64_t u = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(b >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((unsigned)b);
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_mov_b64 exec, %3\n\tglobal_load_lds_dwordx4 %1, %2 offset:%4\n\tglobal_load_lds_dwordx4 %1, %2 offset:%5\n\ts_mov_b64 exec, -1"
        :
        : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(u), "s"(lanes_of(mask)), "n"(OFFSET), "n"(OFFSET + 1024)
        : "memory");
}

// 16 e4m3 values times 2^(byte - 127) as two bf16 operands, values 0 ... 7 and 8 ... 15
__device__ __forceinline__ void widen(u32x4 v, unsigned byte, bf16x8 (&o)[2]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const float scale = __uint_as_float(byte << 23);   // the conversion takes the exponent field only
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], scale, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], scale, true);
        o[i >> 1][(i & 1) * 4 + 0] = lo[0], o[i >> 1][(i & 1) * 4 + 1] = lo[1];
        o[i >> 1][(i & 1) * 4 + 2] = hi[0], o[i >> 1][(i & 1) * 4 + 3] = hi[1];
    }
}

// one operand of a K step in the registers it is multiplied from
template <int FORMAT>
struct Operand {
    u32x4 h[2];
    unsigned scale;
    __device__ __forceinline__ void set(const u32x4 (&v)[2], const unsigned (&s)[2]) { h[0] = v[0], h[1] = v[1], scale = s[0]; }
};
template <>
struct Operand<kMx8Wide> {
    bf16x8 b[2][2];
    __device__ __forceinline__ void set(const u32x4 (&v)[2], const unsigned (&s)[2]) { widen(v[0], s[0] & 255, b[0]), widen(v[1], s[1] & 255, b[1]); }
};

template <int FORMAT>
__device__ __forceinline__ f32x4 step_product(const Operand<FORMAT>& w, const Operand<FORMAT>& x, f32x4 c) {
    if constexpr (FORMAT == kF16) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, w.h[h]), __builtin_bit_cast(half8, x.h[h]), c, 0, 0, 0);
    } else if constexpr (FORMAT == kBf16) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.h[h]), __builtin_bit_cast(bf16x8, x.h[h]), c, 0, 0, 0);
    } else if constexpr (FORMAT == kMx8) {
        struct Two {
            u32x4 h[2];
        };
        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(i32x8, Two{{w.h[0], w.h[1]}}),
                                                             __builtin_bit_cast(i32x8, Two{{x.h[0], x.h[1]}}), c, 0, 0, 0, (int)w.scale, 0, (int)x.scale);
    } else {
        // both operands deal their 128 values to the four instructions alike, so the order along k does not matter
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.b[h][i], x.b[h][i], c, 0, 0, 0);
    }
    return c;
}

// scale dwords a lane holds per row: its own block's, or -- widened -- those of the blocks its two chunks lie in
template <int FORMAT>
constexpr int kScales = FORMAT == kMx8Wide ? 2 : 1;
template <int FORMAT>
__device__ __forceinline__ int scale_block(int h, int g) {
    return FORMAT == kMx8Wide ? h * 2 + (g >> 1) : g;
}

// One tile of 16 MT WM rows x 64 G WN features; a wave computes 16 MT x 64 G.
//
// NB LDS buffers of one K step each.  A step has two (or four) phases, parts of its rows.  While one part multiplies, the next part's
// fragments are read from LDS; before the last part every read of the buffer is done, one barrier, and while the last part
// multiplies the copies of step t + NB go out into this buffer and the first fragments of step t + 1 come in from the next one.  So
// a copy has NB - 1 steps to land, a fragment a phase, and a step costs one barrier.  Everything that is not a product is dealt
// evenly over the products of its phase (sched_barrier keeps it there): the matrix pipe runs while the rest issues in its shadow.
template <int FORMAT, int MT, int G, int WM, int WN, int NB>
__global__ __launch_bounds__(64 * WM * WN, MT * G >= 16 || NB > 3 ? 1 : 2) void linear_tile_kernel(LinearArgs a) {
    constexpr bool kScaled = FORMAT == kMx8 || FORMAT == kMx8Wide;
    constexpr int S = kScales<FORMAT>;
    constexpr int NP = FORMAT == kMx8 && MT == 8 ? 4 : 2;   // phases of a step (four: half the registers for rows)
    constexpr int kWaves = WM * WN, MH = MT / NP, J = 4 * G;
    constexpr int BM = 16 * MT * WM, BG = G * WN;
    constexpr int kXBytes = BM * kStepBytes, kWBytes = BG * kGroupStep;
    constexpr int kXPer = BM / 8 / kWaves;               // copies of 8 rows per wave and step
    constexpr int kWPer = BG * 8 / kWaves;               // copies of 1 KiB of weights per wave and step
    constexpr int kXScale = (BM + 63) / 64 * 1024, kWScale = BG * 1024;   // bytes of four steps' scales
    constexpr int kScalePieces = kXScale / 1024 + BG;
    constexpr int kScalePer = kScaled ? (kScalePieces + kWaves - 1) / kWaves : 0;
    constexpr int kCopies = kXPer + kWPer + kScalePer;   // per wave and step; the scales' do something every fourth step
    static_assert(BM % (8 * kWaves) == 0 && (BG * 8) % kWaves == 0 && MT % NP == 0, "copies divide over the waves");
    static_assert(NB >= 2 && NB <= 4 && (NB - 1) * kCopies < 64, "the copies in flight fit the counter, the scales two buffers");
    constexpr int kW0 = NB * kXBytes, kS0 = kW0 + NB * kWBytes;   // LDS: the buffers' rows, their weights, two quads of scales
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kS0 + (kScaled ? 2 * (kXScale + kWScale) : 0)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    // consecutive workgroups go to the eight XCDs in turn: each XCD takes a run of tiles, walked in bands of kBand row tiles, so that
    // the tiles that run on it at one time share rows and weights in its L2
    constexpr int kBand = 8;
    int64_t mt;
    int nt;
    {
        const unsigned tiles = gridDim.x, xcd = blockIdx.x & 7, q = tiles >> 3, r = tiles & 7;
        const unsigned tile = xcd * q + (xcd < r ? xcd : r) + (blockIdx.x >> 3);
        const unsigned band = tile / (kBand * a.col_tiles), in = tile - band * (kBand * a.col_tiles);
        const unsigned left = (unsigned)a.row_tiles - band * kBand, high = left < kBand ? left : kBand;
        mt = band * kBand + in % high, nt = (int)(in / high);
    }
    const int64_t m0 = mt * BM;
    const int g0 = nt * BG;   // first group of 64 features
    const int s0 = blockIdx.y * a.split_steps;   // first step (a multiple of 4)
    const int steps = a.split_steps && a.ksteps - s0 > a.split_steps ? a.split_steps : a.ksteps - s0;
    const int last_chunks = s0 + steps == a.ksteps ? a.last_chunks : 8;

    const auto source_row = [&](int lr, bool& there) {
        int64_t row = m0 + lr;
        if (row >= a.rows) row = a.rows - 1;   // rows behind the end repeat the last one, nothing of them is stored
        there = true;
        if (a.slots) {
            row = a.slots[row];
            there = row >= 0 && row < a.n_slots;
        }
        return row;
    };
    // ---- what this lane copies: rows (wave * kXPer + i) * 8 + lane / 8, chunk (lane & 7) ^ (row >> 1 & 7)
    const unsigned char* xp[kXPer];
    int xinc[kXPer];
    unsigned tail = 0;   // bit i: copy i's chunk lies behind the row's end in the last step
#pragma unroll
    for (int i = 0; i < kXPer; ++i) {
        const int lr = (wave * kXPer + i) * 8 + (lane >> 3);
        const int chunk = (lane & 7) ^ ((lr >> 1) & 7);
        bool there;
        const int64_t row = source_row(lr, there);
        xp[i] = (there ? a.x + row * a.x_pitch + (int64_t)s0 * kStepBytes + chunk * 16 : a.zero + chunk * 16) - (i & 1) * 1024;
        xinc[i] = there ? kStepBytes : 0;
        tail |= chunk >= last_chunks ? 1u << i : 0u;
    }
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
    const unsigned ldsx = __builtin_amdgcn_readfirstlane(lds0 + wave * kXPer * 1024), ldsw = __builtin_amdgcn_readfirstlane(lds0 + kW0 + wave * kWPer * 1024);
    const unsigned woff = lane * 16;
    // a wave's pieces of 1 KiB of weights: a run of kWPer, inside one group
    static_assert(kXPer % 2 == 0 && kWPer % 2 == 0 && 8 % kWPer == 0, "the copies go out in pairs, a wave's weight pieces lie in one group");
    const unsigned char* wp;
    {
        int gr = g0 + wave * kWPer / 8;
        if (gr >= a.groups) gr = a.groups - 1;
        wp = a.w + (((int64_t)gr * a.ksteps + s0) * 8 + wave * kWPer % 8) * 1024;
    }
    // the steps' copies go out in order: the pointers walk along.  A step behind the last one copies nothing.
    const auto copy_x = [&](auto pair, int buf, int mask) {
        constexpr int i = decltype(pair)::value * 2;
        dma_lane_pair(ldsx + buf * kXBytes + i * 1024, xp[i], xp[i + 1], mask);
        xp[i] += xinc[i], xp[i + 1] += xinc[i + 1];
    };
    const auto copy_w = [&](auto pair, int buf, int mask) {   // (an offset reaches 4095: two pairs from one address)
        constexpr int i = decltype(pair)::value * 2;
        dma_uniform_pair<i % 4 * 1024>(ldsw + buf * kWBytes + i / 4 * 4096, wp + i / 4 * 4096, woff, mask);
        if (i + 2 == kWPer) wp += kGroupStep;
    };
    const auto before_copies = [&](int t) {   // the last step of rows that end inside it: what lies behind is read as zero
        // (held rows are padded; and without this branch the loop is one block, in which the products stay where they are put)
        if (!kScaled && t == steps - 1 && last_chunks < 8) {
#pragma unroll
            for (int i = 0; i < kXPer; ++i)
                if (tail >> i & 1) xp[i] = a.zero - (i & 1) * 1024;
        }
    };
    // four steps' scales, with the first of them: 64 rows' 16 bytes, or a group's 1 KiB, per copy; piece wave + k * kWaves
    const int quads = (a.ksteps + 3) / 4;
    const unsigned char* sp[kScaled ? kScalePer : 1];
    int sinc[kScaled ? kScalePer : 1];
    if constexpr (kScaled) {
#pragma unroll
        for (int k = 0; k < kScalePer; ++k) {
            const int piece = wave + k * kWaves;
            if (piece < kXScale / 1024) {
                bool there;
                const int lr = piece * 64 + lane;
                const int64_t row = source_row(lr < BM ? lr : BM - 1, there);
                sp[k] = there ? a.x_scale + row * a.x_scale_pitch + (s0 >> 2) * 16 : a.zero;
                sinc[k] = there ? 16 : 0;
            } else {
                int gr = g0 + piece - kXScale / 1024;
                if (gr >= a.groups) gr = a.groups - 1;
                sp[k] = (const unsigned char*)(a.w_scale + ((int64_t)gr * quads + (s0 >> 2)) * 256 + lane * 4);
                sinc[k] = 1024;
            }
        }
    }
    const auto copy_scales = [&](int t) {
        if constexpr (kScaled) {
            const int mask = (t & 3) == 0 && t < steps ? -1 : 0;
#pragma unroll
            for (int k = 0; k < kScalePer; ++k) {
                const int piece = wave + k * kWaves;
                dma_lane(lds0 + kS0 + ((t >> 2) & 1) * (kXScale + kWScale) + piece * 1024, sp[k], piece < kScalePieces ? mask : 0);
                sp[k] += mask & sinc[k];
            }
        }
    };

    // ---- fragments and their scales
    u32x4 wr[J][2], xr[2][MH][2];
    unsigned ws[kScaled ? J : 1][2], xs[kScaled ? 2 * MH : 1][2];
    const int xlane = (wm * MT * 16 + (lane & 15)) * kStepBytes, swz = ((lane & 15) >> 1) & 7;
    int xl0 = xlane + ((g ^ swz) * 16), xl1 = xlane + (((4 + g) ^ swz) * 16);   // in the buffer that is read
    int wl = kW0 + wn * G * kGroupStep + lane * 16;
    const auto read_x = [&](int m, int h) { return *(const u32x4*)(smem + (h ? xl1 : xl0) + m * 16 * kStepBytes); };
    const auto read_w = [&](int j, int h) { return *(const u32x4*)(smem + wl + (j >> 2) * kGroupStep + ((j & 3) * 2 + h) * 1024); };
    // (a scale is one byte: its block's dword, the byte of the step)
    int xsl[2], wsl[2];
#pragma unroll
    for (int h = 0; h < S; ++h) {
        const int b = scale_block<FORMAT>(h, g);
        xsl[h] = kS0 + (wm * MT * 16 + (lane & 15)) * 16 + b * 4;
        wsl[h] = kS0 + kXScale + wn * G * 1024 + (b * 16 + (lane & 15)) * 4;
    }
    const auto scale_at = [&](int t) { return ((t >> 2) & 1) * (kXScale + kWScale) + (t & 3); };
    const auto read_xs = [&](int at, int to, int m) {
        if constexpr (kScaled)
#pragma unroll
            for (int h = 0; h < S; ++h) xs[to][h] = *(smem + xsl[h] + at + m * 256);
    };
    const auto read_ws = [&](int at, int j) {
        if constexpr (kScaled)
#pragma unroll
            for (int h = 0; h < S; ++h) ws[j][h] = *(smem + wsl[h] + at + (j >> 2) * 1024 + (j & 3) * 256);
    };

    f32x4 acc[MT][J];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < J; ++j) acc[m][j] = f32x4{0, 0, 0, 0};

    // ---- the first NB steps' copies, the first fragments
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        before_copies(b);
        copy_scales(b);
        const int mask = b < steps ? -1 : 0;
        static_for<0, kXPer / 2>([&](auto pair) { copy_x(pair, b, mask); });
        static_for<0, kWPer / 2>([&](auto pair) { copy_w(pair, b, mask); });
    }
    // A small tile has registers to spare: its residual comes in while it multiplies, and waits there.
    constexpr bool kPre = MT * G <= (FORMAT == kMx8Wide ? 2 : 4);
    u32x4 pre[kPre ? MT : 1][4];
    if constexpr (kPre) {
        const int64_t row0 = m0 + wm * MT * 16;
        const int n0 = (g0 + wn) * 64;
        if (a.residual && !a.split_steps && all_there<MT>(a, row0, n0)) {
            const int size = a.y_type == RMR_TYPE_F32 ? 4 : 2;
            const unsigned char* r = (const unsigned char*)a.residual + ((row0 + (lane & 15)) * a.ldr + n0 + g * 16) * size;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int p = 0; p < 2; ++p) pre[m][p] = *(const u32x4_any*)(r + p * 16);
                if (size == 4)
#pragma unroll
                    for (int p = 2; p < 4; ++p) pre[m][p] = *(const u32x4_any*)(r + p * 16);
                r += 16 * a.ldr * size;
            }
        }
    }
    // (only copies that surely went out are counted: an empty one need not be, and the residual's loads only make the waits stricter)
    if (steps >= NB)
        asm volatile("s_waitcnt vmcnt(%0)" : : "n"((NB - 1) * (kXPer + kWPer)) : "memory");
    else
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    asm volatile("s_barrier" : : : "memory");
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < J; ++j) wr[j][h] = read_w(j, h);
#pragma unroll
        for (int m = 0; m < MH; ++m) xr[0][m][h] = read_x(m, h);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) read_ws(0, j);
#pragma unroll
    for (int m = 0; m < MH; ++m) read_xs(0, m, m);

    // one step an iteration: every accumulator is updated once, and stays in its registers
    int buf = 0;
    for (int t = 0; t < steps; ++t) {
        constexpr int kSlots = MH * J;   // products of a phase, the features outside, the rows inside
        const int now = kScaled ? scale_at(t) : 0, next = kScaled ? scale_at(t + 1) : 0;
        const auto product = [&](auto phase, auto slot) {
            constexpr int PH = decltype(phase)::value, m = decltype(slot)::value % MH, j = decltype(slot)::value / MH;
            Operand<FORMAT> wf, xf;
            const unsigned none[2] = {0, 0};
            if constexpr (kScaled) {
                wf.set(wr[j], ws[j]), xf.set(xr[PH & 1][m], xs[(PH & 1) * MH + m]);
            } else {
                wf.set(wr[j], none), xf.set(xr[PH & 1][m], none);
            }
            acc[PH * MH + m][j] = step_product<FORMAT>(wf, xf, acc[PH * MH + m][j]);
        };
        // the rows' fragments of phase `to`, dealt over the first half of the phase before it
        const auto read_rows = [&](auto to, auto slot, int at) {
            constexpr int T = decltype(to)::value, s = decltype(slot)::value;
            static_for<0, 2 * MH>([&](auto act) {
                constexpr int i = decltype(act)::value;
                if constexpr (i * (kSlots / 2) / (2 * MH) == s) {
                    xr[T & 1][i >> 1][i & 1] = read_x(T * MH + (i >> 1), i & 1);
                    if constexpr (i % 2) read_xs(at, (T & 1) * MH + (i >> 1), T * MH + (i >> 1));
                }
            });
        };
        static_for<0, NP - 1>([&](auto phase) {
            static_for<0, kSlots>([&](auto slot) {
                product(phase, slot);
                read_rows(std::integral_constant<int, decltype(phase)::value + 1>{}, slot, now);
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        // step t + 1 has landed for every wave, and every wave has read all of step t
        if (NB > 2 && t + NB <= steps)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((NB - 2) * (kXPer + kWPer)) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
        asm volatile("s_barrier" : : : "memory");
        const int more = t + NB < steps ? -1 : 0;
        const bool wrap = buf == NB - 1;
        xl0 += wrap ? -(NB - 1) * kXBytes : kXBytes, xl1 += wrap ? -(NB - 1) * kXBytes : kXBytes, wl += wrap ? -(NB - 1) * kWBytes : kWBytes;
        before_copies(t + NB);
        copy_scales(t + NB);
        // last phase: the next step's first fragments -- a weight fragment right behind the last product of the one it replaces -- and
        // the copies of the step after it
        static_for<0, kSlots>([&](auto slot) {
            constexpr int s = decltype(slot)::value;
            product(std::integral_constant<int, NP - 1>{}, slot);
            read_rows(std::integral_constant<int, 0>{}, slot, next);
            if constexpr (s % MH == MH - 1) {
#pragma unroll
                for (int h = 0; h < 2; ++h) wr[s / MH][h] = read_w(s / MH, h);
                read_ws(next, s / MH);
            }
            static_for<0, (kXPer + kWPer) / 2>([&](auto act) {
                constexpr int i = decltype(act)::value;
                if constexpr (i * kSlots / ((kXPer + kWPer) / 2) == s) {
                    if constexpr (i < kXPer / 2)
                        copy_x(std::integral_constant<int, i>{}, buf, more);
                    else
                        copy_w(std::integral_constant<int, i - kXPer / 2>{}, buf, more);
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        buf = wrap ? 0 : buf + 1;
    }
    // (no copy is in flight any more: the last step waited for all of them)
    if (a.split_steps) {
        static_for<0, G>([&](auto group) {
            constexpr int q = decltype(group)::value;
            const int gr = g0 + wn * G + q;
            if (gr >= a.groups) return;
            const int64_t row0 = m0 + wm * MT * 16 + (lane & 15);
            float* to = a.partial + (((int64_t)blockIdx.y * a.rows + row0) * a.groups + gr) * 64 + g * 16;
            static_for<0, MT>([&](auto mm) {
                constexpr int m = decltype(mm)::value;
                if (row0 + m * 16 < a.rows)
#pragma unroll
                    for (int j = 0; j < 4; ++j) *(f32x4*)(to + (int64_t)m * 16 * a.groups * 64 + j * 4) = acc[m][q * 4 + j];
            });
        });
        return;
    }
    // (the LDS that a lane of an edge tile writes may still be read by a slower wave's last fragment loads, whose values nobody uses)
    float* spill = (float*)smem + wave * MT * 1024 + lane * 16;
    static_assert(kWaves * MT * 4096 <= kS0, "the edge waves' values fit the buffers");
    static_for<0, G>([&](auto group) {
        constexpr int q = decltype(group)::value;
        const int gr = g0 + wn * G + q;
        if (gr < a.groups)
            finish_group<MT, q, kPre>(a, [&](auto m) -> f32x4(&)[J] { return acc[decltype(m)::value]; }, pre, spill, m0 + wm * MT * 16, gr * 64, lane);
    });
}

// ---------------------------------------------------------------------------------------------------- the few-rows kernel
//
// Up to 16 MT rows: the weights' bytes are the work, and every one of them goes from memory straight into the registers it is
// multiplied from -- no LDS, no barrier until the end.  A workgroup owns 16 JN features; its eight waves deal the K steps among
// themselves (wave v takes steps v, v + 8, ...) and their sums are joined through LDS in wave order, so the result does not depend on
// timing.  One step's loads a wave are in flight: two or four gained nothing (within 4 % on one row of 4096 -> 4096, which takes 9.5 us with
// its weights in the last-level cache and 11.7 from memory, 3.5 and 2.9 TB/s).  x is read as it is -- any alignment and length -- and quantised in
// registers where the format asks for it: no launch in front, no workspace.

constexpr int kFewWaves = 8;

// where a lane's chunk of 16 bytes (of the operand) comes from
enum { kRaw, kFromF16, kFromBf16, kFromF32, kHeld };
template <int SRC>
struct SourceType {
    typedef unsigned short T;
};
template <>
struct SourceType<kFromF16> {
    typedef F16 T;
};
template <>
struct SourceType<kFromBf16> {
    typedef BF16 T;
};
template <>
struct SourceType<kFromF32> {
    typedef float T;
};

struct FewArgs {
    LinearArgs a;
    const void* x;   // kRaw, kFrom*: the caller's rows
    int64_t ldx;
    int in_features;
};

// 16 values of a row as e4m3, and their block's exponent byte.  The block's other half is in lane ^ 16.
template <class T>
__device__ __forceinline__ u32x4 quantised_chunk(const u32x4 (&raw)[sizeof(T)], unsigned& byte) {
    unsigned w[4 * sizeof(T)], q[4];
#pragma unroll
    for (int p = 0; p < (int)sizeof(T); ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[p * 4 + i] = raw[p][i];
    byte = (unsigned)(quantise_words<T>(w, q, [](unsigned t) { return max(t, (unsigned)__shfl_xor((int)t, 16)); }) + 127);
    return u32x4{q[0], q[1], q[2], q[3]};
}

template <class T>
__device__ __forceinline__ void finish_quad(const LinearArgs& a, f32x4 v, int64_t row, int c0) {
    const int have = a.out_features - c0;
    if (row >= a.rows || have <= 0) return;
    const f32x4 b = *(const f32x4*)(a.bias + c0);
    v += b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        switch (a.act) {
            case RMR_ACT_RELU: v[i] = activate<T, RMR_ACT_RELU>(v[i]); break;
            case RMR_ACT_SILU: v[i] = activate<T, RMR_ACT_SILU>(v[i]); break;
            case RMR_ACT_GELU: v[i] = activate<T, RMR_ACT_GELU>(v[i]); break;
            case RMR_ACT_SIGMOID: v[i] = activate<T, RMR_ACT_SIGMOID>(v[i]); break;
            default: break;
        }
    }
    T* y = (T*)a.y + row * a.ldy + c0;
    const T* r = a.residual ? (const T*)a.residual + row * a.ldr + c0 : nullptr;
    if (have >= 4 && sizeof(T) == 4) {
        if (r) {
            float rv[4];
            load_values<float, 4>((const float*)r, 4, rv);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += rv[i];
        }
        const float o[4] = {v[0], v[1], v[2], v[3]};
        store_values<float, 4>((float*)y, 4, o);
        return;
    }
    if (have >= 4) {
        union {
            u32x2 u;
            T t[4];
        } w;
        if (r) {
            w.u = *(const u32x2_any*)r;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += to_f32(w.t[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) w.t[i] = from_f32<T>(v[i]);
        *(u32x2_any*)y = w.u;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < have) y[i] = from_f32<T>(v[i] + (r ? to_f32(r[i]) : 0.0f));
}

template <int FORMAT, int SRC, int MT, int JN>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few_kernel(FewArgs f) {
    const LinearArgs& a = f.a;
    constexpr bool kScaled = FORMAT == kMx8 || FORMAT == kMx8Wide;
    constexpr int S = kScales<FORMAT>;
    __shared__ f32x4 part[kFewWaves][MT * JN][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4;
    const int group = blockIdx.x / (4 / JN), j0 = (blockIdx.x % (4 / JN)) * JN;
    const unsigned char* w = a.w + ((int64_t)group * a.ksteps * 8 + j0 * 2) * 1024 + lane * 16;
    const int quads = (a.ksteps + 3) / 4;
    const unsigned* wsp = kScaled ? a.w_scale + (int64_t)group * quads * 256 + j0 * 64 + (lane & 15) : nullptr;
    typedef typename SourceType<SRC>::T T;
    constexpr bool kQuantise = SRC == kFromF16 || SRC == kFromBf16 || SRC == kFromF32;
    constexpr int R = kQuantise ? (int)sizeof(T) : 1;   // pieces of 16 bytes that a chunk of the operand is made of
    const T* xrow[MT];
    const unsigned char* held[MT];
    const unsigned char* hscale[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        int64_t row = m * 16 + (lane & 15);
        if (row >= a.rows) row = a.rows - 1;
        if constexpr (SRC == kHeld) {
            row = a.slots[row];
            const bool there = row >= 0 && row < a.n_slots;
            held[m] = there ? a.x + row * a.x_pitch : nullptr;
            hscale[m] = a.x_scale + row * a.x_scale_pitch;
        } else {
            xrow[m] = (const T*)f.x + row * f.ldx;
        }
    }
    f32x4 acc[MT][JN];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < JN; ++j) acc[m][j] = f32x4{0, 0, 0, 0};

    for (int t = wave; t < a.ksteps; t += kFewWaves) {
        u32x4 wv[JN][2], xv[MT][2][R];
        unsigned wsv[JN][2], xsv[MT][2];
#pragma unroll
        for (int j = 0; j < JN; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h) wv[j][h] = *(const u32x4*)(w + (int64_t)t * kGroupStep + (j * 2 + h) * 1024);
            if constexpr (kScaled)
#pragma unroll
                for (int h = 0; h < S; ++h) wsv[j][h] = wsp[(t >> 2) * 256 + j * 64 + scale_block<FORMAT>(h, g) * 16] >> ((t & 3) * 8);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int chunk = h * 4 + g;
                if constexpr (SRC == kRaw) {
                    const int k0 = t * 64 + chunk * 8;
                    xv[m][h][0] = load_words<T>(xrow[m] + k0, f.in_features - k0);
                } else if constexpr (SRC == kHeld) {
                    xv[m][h][0] = u32x4{0, 0, 0, 0};
                    if (held[m]) xv[m][h][0] = *(const u32x4*)(held[m] + t * kStepBytes + chunk * 16);
                } else {
#pragma unroll
                    for (int p = 0; p < R; ++p) {
                        const int k0 = t * kStepBytes + chunk * 16 + p * (16 / R);
                        xv[m][h][p] = load_words<T>(xrow[m] + k0, f.in_features - k0);
                    }
                }
            }
            if constexpr (SRC == kHeld)
#pragma unroll
                for (int h = 0; h < S; ++h)
                    xsv[m][h] = held[m] ? *(const unsigned*)(hscale[m] + (t >> 2) * 16 + scale_block<FORMAT>(h, g) * 4) >> ((t & 3) * 8) : 0u;
        }
        Operand<FORMAT> wf[JN];
#pragma unroll
        for (int j = 0; j < JN; ++j) wf[j].set(wv[j], wsv[j]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            u32x4 v[2];
            unsigned xs[2] = {0, 0};
            if constexpr (kQuantise) {
                unsigned b[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) v[h] = quantised_chunk<T>(xv[m][h], b[h]);
                if constexpr (FORMAT == kMx8Wide) {
                    xs[0] = b[0], xs[1] = b[1];
                } else {
                    // lane group g scales block g, whose two chunks 2 g and 2 g + 1 lie in half g / 2 of groups 2 g % 4 and one more
                    const unsigned both = __shfl(b[0] | b[1] << 8, (lane & 15) + ((g & 1) << 5));
                    xs[0] = g >> 1 ? both >> 8 : both & 255;
                }
            } else {
                v[0] = xv[m][0][0], v[1] = xv[m][1][0];
                if constexpr (kScaled) xs[0] = xsv[m][0], xs[1] = xsv[m][S - 1];
            }
            Operand<FORMAT> xf;
            xf.set(v, xs);
#pragma unroll
            for (int j = 0; j < JN; ++j) acc[m][j] = step_product<FORMAT>(wf[j], xf, acc[m][j]);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < JN; ++j) part[wave][m * JN + j][lane] = acc[m][j];
    __syncthreads();
    for (int p = wave; p < MT * JN; p += kFewWaves) {
        f32x4 v = part[0][p][lane];
#pragma unroll
        for (int k = 1; k < kFewWaves; ++k) v += part[k][p][lane];
        const int64_t row = (p / JN) * 16 + (lane & 15);
        const int c0 = group * 64 + g * 16 + (j0 + p % JN) * 4;
        if (a.y_type == RMR_TYPE_F16)
            finish_quad<F16>(a, v, row, c0);
        else if (a.y_type == RMR_TYPE_BF16)
            finish_quad<BF16>(a, v, row, c0);
        else
            finish_quad<float>(a, v, row, c0);
    }
}

// rows up to which the few-rows kernel takes a call
constexpr int64_t kFewRows = RMR_LINEAR_FEW_ROWS;

template <int FORMAT, int SRC>
void launch_few(const FewArgs& f, int cus, hipStream_t s) {
    // 32 features a workgroup instead of 16 where that still leaves work for half the chip (all of it for more than 16 rows): 8192 -> 8192
    // bf16 on one row 27 us against 38, 4096 -> 8192 mx8 on 16 rows 9.7 against 15; 4096 -> 1024 on one row 6.5 against 4.4
    const bool one = f.a.rows <= 16;
    const bool wide = f.a.groups * 2 >= (one ? cus / 2 : cus);
    const unsigned grid = (unsigned)f.a.groups * (wide ? 2 : 4);
    if (one && wide)
        linear_few_kernel<FORMAT, SRC, 1, 2><<<grid, 64 * kFewWaves, 0, s>>>(f);
    else if (one)
        linear_few_kernel<FORMAT, SRC, 1, 1><<<grid, 64 * kFewWaves, 0, s>>>(f);
    else if (wide)
        linear_few_kernel<FORMAT, SRC, 2, 2><<<grid, 64 * kFewWaves, 0, s>>>(f);
    else
        linear_few_kernel<FORMAT, SRC, 2, 1><<<grid, 64 * kFewWaves, 0, s>>>(f);
    RMR_HIP(hipGetLastError());
}

template <int FORMAT>
void launch_few_mx8(const FewArgs& f, bool kept, int type, int cus, hipStream_t s) {
    if (kept)
        launch_few<FORMAT, kHeld>(f, cus, s);
    else if (type == RMR_TYPE_F16)
        launch_few<FORMAT, kFromF16>(f, cus, s);
    else if (type == RMR_TYPE_BF16)
        launch_few<FORMAT, kFromBf16>(f, cus, s);
    else
        launch_few<FORMAT, kFromF32>(f, cus, s);
}

// joins the splits' sums, in order, and finishes the rows: four features of one row a thread
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a, int splits) {
    const int64_t quads = a.rows * a.groups * 16, stride = a.rows * a.groups * 64;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < quads; p += (int64_t)gridDim.x * 256) {
        const int64_t row = p / (a.groups * 16);
        const int c0 = (int)(p - row * (a.groups * 16)) * 4;
        const float* from = a.partial + p * 4;
        f32x4 v = *(const f32x4*)from;
        for (int k = 1; k < splits; ++k) v += *(const f32x4*)(from + k * stride);
        if (a.y_type == RMR_TYPE_F16)
            finish_quad<F16>(a, v, row, c0);
        else if (a.y_type == RMR_TYPE_BF16)
            finish_quad<BF16>(a, v, row, c0);
        else
            finish_quad<float>(a, v, row, c0);
    }
}

template <int FORMAT, int MT, int G, int WM, int WN, int NB>
void launch_tile(LinearArgs a, int splits, hipStream_t s) {
    a.row_tiles = (a.rows + 16 * MT * WM - 1) / (16 * MT * WM);
    a.col_tiles = (a.groups + G * WN - 1) / (G * WN);
    const int64_t tiles = a.row_tiles * a.col_tiles;
    if (tiles >= 1 << 24) fail(RMR_ERR_INVALID_ARGUMENT, "linear: %lld tiles in one call", (long long)tiles);
    linear_tile_kernel<FORMAT, MT, G, WM, WN, NB><<<dim3((unsigned)tiles, (unsigned)splits), 64 * WM * WN, 0, s>>>(a);
    RMR_HIP(hipGetLastError());
}

// what a call of more than kFewRows rows runs: a tile shape and how many workgroups share a tile's K
enum { kTileBig, kTileMid, kTileSmall };
struct Choice {
    int tile, splits, split_steps;
};

// Time of a call in us from what the shapes were measured at: a round of tiles costs its steps and what a tile has besides (first
// copies, epilogue).  A CU holds one big tile or two of the others; one alone runs faster than two together.
//   us a step (bf16 8192^3 and 64 x 4096 x 4096)   big 1.52   mid 1.0, alone 0.64   small 0.62, alone 0.36
//   us besides (8192 x 512 x 8192, 4096 x 1024^2)  big 8      mid 4                 small 3
// 2048 x 4096^2 bf16: big 80, mid 63, small 82; 1000 x 4096^2: 81, 46, 43; 102400 x 384^2 f16: 69, 60, 75; 8192 x 512 x 8192: 82, 87, 101.
// The mx8 steps (twice the values) differ from these by less than the shapes do, but for f32 y: widened rows take 2.1 a step in the mid
// shape and 1.35 in the small one (kept 2048 and 1000 x 4096^2), the same ratio, and have no big one.
double tile_time(int64_t tiles, int ksteps, int cus, int per_cu, double step, double alone, double besides) {
    const int64_t full = tiles / (per_cu * (int64_t)cus), rest = tiles % (per_cu * (int64_t)cus);
    return full * (ksteps * step + besides) + (rest > cus ? ksteps * step + besides : rest ? ksteps * alone + besides : 0.0);
}

Choice choose(int format, int64_t rows, int groups, int ksteps, int cus) {
    const int64_t big = ((rows + 255) / 256) * ((groups + 3) / 4);
    const int64_t mid = ((rows + 127) / 128) * ((groups + 1) / 2);
    const int64_t small = ((rows + 63) / 64) * ((groups + 1) / 2);
    Choice c{kTileSmall, 1, 0};
    const double t_small = tile_time(small, ksteps, cus, 2, 0.62, 0.36, 3), t_mid = tile_time(mid, ksteps, cus, 2, 1.0, 0.64, 4);
    const double t_big = format == kMx8Wide ? 1e30 : tile_time(big, ksteps, cus, 1, 1.52, 1.52, 8);
    if (t_mid <= t_small && t_mid <= t_big)
        c.tile = kTileMid;
    else if (t_big < t_small)
        c.tile = kTileBig;
    // Few tiles and a long K: workgroups share a tile's steps.  The partial sums travel through memory and cost a launch, about as much as
    // 16 steps, so only from 32 steps on, at least 8 each, and with no more than 6 MB of sums: 64 x 4096 x 4096 bf16 26 us in one
    // piece, 19 / 15 / 17 us in 2 / 4 / 8; 256 x 1024 x 4096 (16 steps) 9.7 us in one piece, 17 in two.
    if (small <= cus / 2 && ksteps >= 32) {
        c.tile = kTileSmall;
        int64_t splits = cus / small;
        const int64_t room = (6 << 20) / (rows * groups * 64 * 4), steps = ksteps / 8;
        if (splits > room) splits = room;
        if (splits > steps) splits = steps;
        if (splits > 1) {
            c.split_steps = (int)((ksteps + splits - 1) / splits + 3) / 4 * 4;   // the scales come by fours
            c.splits = (ksteps + c.split_steps - 1) / c.split_steps;
            if (c.splits == 1) c.split_steps = 0;
        }
    }
    return c;
}

template <int FORMAT>
void launch_format(LinearArgs a, const Choice& c, hipStream_t s) {
    a.split_steps = c.split_steps;
    if (c.tile == kTileBig) {
        if constexpr (FORMAT != kMx8Wide) launch_tile<FORMAT, 8, 2, 2, 2, 2>(a, 1, s);
    } else if (c.tile == kTileMid) {
        launch_tile<FORMAT, 4, 1, 2, 2, 2>(a, 1, s);
    } else {
        launch_tile<FORMAT, 2, 1, 2, 2, 3>(a, c.splits, s);
        if (c.splits > 1) {
            const int64_t blocks = (a.rows * a.groups * 16 + 255) / 256;
            linear_join_kernel<<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, s>>>(a, c.splits);
            RMR_HIP(hipGetLastError());
        }
    }
}

}  // namespace

// -------------------------------------------------------------------------------------------------------------- Linear

Linear::Linear(const rmr_linear_cfg& cfg, const void* weight, int weight_type, int64_t ldw, const float* bias, int mem, hipStream_t s)
    : ctx_(device_ctx(cfg.device)), cfg_(cfg) {
    const int n = cfg.out_features, k = cfg.in_features;
    const bool mx8 = cfg.format == RMR_LINEAR_MX8;
    ksteps_ = mx8 ? (k + 127) / 128 : (k + 63) / 64;
    groups_ = (n + 63) / 64;
    w_.alloc((size_t)groups_ * ksteps_ * kGroupStep);
    bias_.alloc((size_t)groups_ * 64);
    zero_.alloc(kStepBytes);
    RMR_HIP(hipMemsetAsync(bias_.p, 0, bias_.n * sizeof(float), s));
    RMR_HIP(hipMemsetAsync(zero_.p, 0, zero_.n, s));
    if (bias)
        RMR_HIP(hipMemcpyAsync(bias_.p, bias, (size_t)n * sizeof(float), mem == RMR_MEM_DEVICE ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice, s));
    DevBuf<unsigned char> staged, q, qs;
    const void* w = weight;
    if (mem != RMR_MEM_DEVICE) {
        const size_t row = (size_t)k * type_bytes(weight_type);
        staged.alloc(row * n);
        RMR_HIP(hipMemcpy2DAsync(staged.p, row, weight, (size_t)ldw * type_bytes(weight_type), row, n, hipMemcpyHostToDevice, s));
        w = staged.p, ldw = k;
    }
    const int64_t pieces = (int64_t)groups_ * ksteps_ * (kGroupStep / 16);
    const unsigned grid = (unsigned)((pieces + 255) / 256 < 65536 ? (pieces + 255) / 256 : 65536);
    if (mx8) {
        Mx8Rows rows{nullptr, nullptr, mx8_pitch(k), mx8_scale_pitch(k)};
        q.alloc((size_t)(rows.pitch * n));
        qs.alloc((size_t)(rows.scale_pitch * n));
        wscale_.alloc((size_t)groups_ * ((ksteps_ + 3) / 4) * 256);
        rows.data = q.p, rows.scale = qs.p;
        RMR_HIP(hipMemsetAsync(qs.p, 0, qs.n, s));
        launch_quantise_rows(ctx_, s, RowSource{w, weight_type, ldw}, k, n, rows);
        pack_mx8_kernel<<<grid, 256, 0, s>>>(PackMx8Args{rows, n, ksteps_, groups_, w_.p, wscale_.p});
    } else {
        const PackArgs pa{w, ldw, n, k, ksteps_, groups_, w_.p};
        const bool bf = cfg.format == RMR_LINEAR_BF16;
        if (weight_type == RMR_TYPE_F16)
            bf ? pack_weight_kernel<F16, BF16><<<grid, 256, 0, s>>>(pa) : pack_weight_kernel<F16, F16><<<grid, 256, 0, s>>>(pa);
        else if (weight_type == RMR_TYPE_BF16)
            bf ? pack_weight_kernel<BF16, BF16><<<grid, 256, 0, s>>>(pa) : pack_weight_kernel<BF16, F16><<<grid, 256, 0, s>>>(pa);
        else
            bf ? pack_weight_kernel<float, BF16><<<grid, 256, 0, s>>>(pa) : pack_weight_kernel<float, F16><<<grid, 256, 0, s>>>(pa);
    }
    RMR_HIP(hipGetLastError());
    RMR_HIP(hipStreamSynchronize(s));   // any stream may use the layer from here on, and the caller's weights are free
}

struct Linear::Plan {
    size_t x_bytes = 0, scale_bytes = 0;   // staged rows in the workspace: aligned 16-bit rows, or quantised ones
    size_t partial_bytes = 0;              // sums of the workgroups that share a tile's K
    Choice choice{};
    size_t total() const { return x_bytes + scale_bytes + partial_bytes; }
};

Linear::Plan Linear::plan(const Call& c) const {
    Plan p;
    if (c.rows <= kFewRows) return p;
    const int format = cfg_.format != RMR_LINEAR_MX8 ? cfg_.format : c.y_type != RMR_TYPE_F32 ? kMx8 : kMx8Wide;
    p.choice = choose(format, c.rows, groups_, ksteps_, ctx_.num_cus);
    if (p.choice.splits > 1) p.partial_bytes = (size_t)p.choice.splits * c.rows * groups_ * 64 * sizeof(float);
    if (c.kept) {
        // read where they lie
    } else if (cfg_.format == RMR_LINEAR_MX8) {
        p.x_bytes = (size_t)(c.rows * mx8_pitch(cfg_.in_features));
        p.scale_bytes = (size_t)(c.rows * mx8_scale_pitch(cfg_.in_features));
    } else if (cfg_.in_features % 8 || (c.ld_bytes() % 16 && c.rows > 1) || (uintptr_t)c.x.p % 16) {
        p.x_bytes = (size_t)(c.rows * ksteps_ * kStepBytes);
    }
    return p;
}

size_t Linear::workspace_bytes(const Call& c) const { return plan(c).total(); }

void Linear::run(const Call& c) {
    if (c.rows <= 0) return;
    const Plan p = plan(c);
    if (p.total() > c.workspace_bytes || (p.total() && !c.workspace))
        fail(RMR_ERR_CAPACITY, "linear: the call needs %zu bytes of workspace, %zu given", p.total(), c.workspace_bytes);
    if (p.total() && (uintptr_t)c.workspace % 16) fail(RMR_ERR_INVALID_ARGUMENT, "linear: the workspace must be 16-byte aligned");
    DeviceGuard guard(ctx_.device);
    LinearArgs a{};
    a.rows = c.rows, a.last_chunks = 8, a.zero = zero_.p;
    a.w = w_.p, a.w_scale = wscale_.p, a.bias = bias_.p;
    a.ksteps = ksteps_, a.groups = groups_, a.out_features = cfg_.out_features;
    a.residual = c.residual, a.ldr = c.ldr, a.y = c.y, a.ldy = c.ldy, a.y_type = c.y_type, a.act = cfg_.activation;
    if (c.kept) {
        const Mx8Rows r = c.cache->rows();
        a.x = r.data, a.x_pitch = r.pitch, a.x_scale = r.scale, a.x_scale_pitch = r.scale_pitch;
        a.slots = c.slots, a.n_slots = c.cache->slots();
    } else if (c.rows <= kFewRows) {
        // read as it is
    } else if (cfg_.format == RMR_LINEAR_MX8) {
        const Mx8Rows r{(unsigned char*)c.workspace, (unsigned char*)c.workspace + p.x_bytes, mx8_pitch(cfg_.in_features), mx8_scale_pitch(cfg_.in_features)};
        launch_quantise_rows(ctx_, c.stream, c.x, cfg_.in_features, c.rows, r);
        a.x = r.data, a.x_pitch = r.pitch, a.x_scale = r.scale, a.x_scale_pitch = r.scale_pitch;
    } else if (p.x_bytes) {
        // a workgroup's pieces: four a thread, one where that would leave much of the chip idle (1777 rows of 1001 to 1237: 23.0 us, 24.5 with four)
        const int per_row = ksteps_ * 8, pieces = c.rows * per_row >= (int64_t)ctx_.num_cus * 4096 ? 1024 : 256;
        const int rows = per_row < pieces ? pieces / per_row : 1;
        const AlignArgs al{c.x.p, c.x.ld, c.rows, cfg_.in_features, per_row, (unsigned)(((1ull << 31) + per_row - 1) / per_row), rows, (unsigned char*)c.workspace};
        const int64_t groups = (c.rows + rows - 1) / rows;
        ProfScope align(ctx_.prof, c.stream, "align_rows", 0, 2.0 * c.rows * ksteps_ * kStepBytes);
        align_rows_kernel<<<(unsigned)(groups < 65536 ? groups : 65536), 256, 0, c.stream>>>(al);
        RMR_HIP(hipGetLastError());
        a.x = (const unsigned char*)c.workspace, a.x_pitch = (int64_t)ksteps_ * kStepBytes;
    } else {
        a.x = (const unsigned char*)c.x.p, a.x_pitch = c.ld_bytes();
        a.last_chunks = (cfg_.in_features - (ksteps_ - 1) * 64) / 8;
    }
    a.partial = (float*)((unsigned char*)c.workspace + p.x_bytes + p.scale_bytes);
    const double out = (double)c.rows * cfg_.out_features;
    ProfScope prof(ctx_.prof, c.stream, "linear", 2.0 * out * cfg_.in_features,
                   (double)w_.n + (double)c.rows * ksteps_ * kStepBytes + out * type_bytes(c.y_type) * (c.residual ? 2 : 1));
    if (c.rows <= kFewRows) {
        const FewArgs f{a, c.x.p, c.x.ld, cfg_.in_features};
        if (cfg_.format == RMR_LINEAR_F16)
            launch_few<kF16, kRaw>(f, ctx_.num_cus, c.stream);
        else if (cfg_.format == RMR_LINEAR_BF16)
            launch_few<kBf16, kRaw>(f, ctx_.num_cus, c.stream);
        else if (c.y_type != RMR_TYPE_F32)
            launch_few_mx8<kMx8>(f, c.kept, c.x.type, ctx_.num_cus, c.stream);
        else
            launch_few_mx8<kMx8Wide>(f, c.kept, c.x.type, ctx_.num_cus, c.stream);
        return;
    }
    if (cfg_.format == RMR_LINEAR_F16)
        launch_format<kF16>(a, p.choice, c.stream);
    else if (cfg_.format == RMR_LINEAR_BF16)
        launch_format<kBf16>(a, p.choice, c.stream);
    else if (c.y_type != RMR_TYPE_F32)
        launch_format<kMx8>(a, p.choice, c.stream);
    else
        launch_format<kMx8Wide>(a, p.choice, c.stream);
}

}  // namespace rmr
