// feature_cache.hip -- rows quantised as they enter a cache, and read back (formats: rows.h).
//
// Both directions are copies that change the element type: bound by memory, one pass, no value touched twice.  A thread owns 16
// bytes of the 16- or 32-bit side (8 or 4 values), so a wave's accesses there are 1 KiB contiguous at any row pitch and alignment;
// a block of 32 is 4 or 8 neighbouring lanes, whose largest magnitude crosses by 2 or 3 lane exchanges.  One chunk of a thread in flight
// and full occupancy beat two or four chunks and fewer waves (200000 rows of 1024 f32, scattered: 278 us reading, 240 writing against
// 276 / 289 and 240 / 251).
#include "rows_device.h"

namespace rmr {
namespace {

using namespace rowsdev;

constexpr int kThreads = 256;
constexpr int kMaxRows = 64;          // rows a workgroup takes at a time
constexpr int64_t kMaxGrid = 65536;   // more row groups than this are walked
// up to so many rows a workgroup looks through the slot list itself for a later row of the same slot; above, the rows claim
// their slots in two passes over the list beforehand
constexpr int64_t kScanRows = 4096;

// The wide side of a call of more bytes than this passes the caches by (non-temporal), the cache's rows do not.  Three states in turn:
// 262144 scattered rows of 1024 bf16 read in 169 us (182 without), 200000 of 1001 f32 in 261 (301), written and read 363 (380) and 480
// (531).  Most of that is the reads'.  A write alone gains where the rows fit the last-level cache (100000 x 576 f16 47 us, 56 without)
// and loses where they do not (the first two cases 213 and 239, 200 and 225 without); with the read behind it that is made up for
// (361 and 476, 361 and 482 without).  Smaller calls stay where the next operator finds them.
constexpr int64_t kStreamBytes = 64 << 20;

enum { DEST_RUN, DEST_SCAN, DEST_OWNER };

struct WriteArgs {
    const void* x;
    int64_t ld, n;
    int width;
    unsigned char *data, *scale;
    int64_t pitch, scale_pitch;
    const int64_t* slots;
    const int* owner;
    int64_t first, n_slots;
    int per_row;     // threads' chunks per row: pitch / values of a chunk
    unsigned magic;  // ceil(2^31 / per_row): i / per_row = i magic >> 31 while i per_row < 2^31
    int rows;        // rows of a group
    bool stream;     // pass the caches by
};

template <class T, int DEST>
__global__ __launch_bounds__(kThreads) void quantise_rows_kernel(WriteArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ int64_t dest[kMaxRows];
    __shared__ int later[kMaxRows];
    const int tid = threadIdx.x;
    const int64_t groups = (a.n + a.rows - 1) / a.rows;
    for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        const int64_t r0 = g * a.rows;
        const int rows = (int)(a.n - r0 < a.rows ? a.n - r0 : a.rows);
        if constexpr (DEST != DEST_RUN) {
            __syncthreads();   // the last group's destinations are read
            if (tid < rows) {
                int64_t s = a.slots[r0 + tid];
                if (s < 0 || s >= a.n_slots) s = -1;
                if (DEST == DEST_OWNER && s >= 0 && a.owner[s] != (int)(r0 + tid)) s = -1;
                dest[tid] = s;
                later[tid] = 0;
            }
            __syncthreads();
            if constexpr (DEST == DEST_SCAN) {
                for (int64_t j = r0 + 1 + tid; j < a.n; j += kThreads) {
                    const int64_t s = a.slots[j];
                    for (int r = 0; r < rows; ++r)
                        if (dest[r] == s && j > r0 + r) later[r] = 1;
                }
                __syncthreads();
            }
        }
        const int chunks = rows * a.per_row;
        for (int i = tid; i < chunks; i += kThreads) {
            const int r = (int)(((uint64_t)(unsigned)i * a.magic) >> 31);
            const int c = (i - r * a.per_row) * V;   // first value of the chunk
            int64_t to = a.first + r0 + r;
            if constexpr (DEST != DEST_RUN) to = later[r] ? -1 : dest[r];
            if (to < 0) continue;   // lanes of one block share their row
            const T* from = (const T*)a.x + (r0 + r) * a.ld + c;
            const u32x4 x = a.stream && a.width - c >= V ? __builtin_nontemporal_load((const u32x4_any*)from) : load_words<T>(from, a.width - c);
            const unsigned w[4] = {x[0], x[1], x[2], x[3]};
            unsigned q[V / 4];
            const int e = quantise_words<T>(w, q, [](unsigned t) {
#pragma unroll
                for (int k = 1; k < 32 / V; k *= 2) t = max(t, (unsigned)__shfl_xor((int)t, k));
                return t;
            });
            unsigned char* p = a.data + to * a.pitch + c;
            if constexpr (V == 8)
                *(u32x2*)p = u32x2{q[0], q[1]};
            else
                *(unsigned*)p = q[0];
            if ((c & 31) == 0) a.scale[to * a.scale_pitch + mx8_scale_at(c >> 5)] = (unsigned char)(e + 127);
        }
    }
}

__global__ __launch_bounds__(kThreads) void clear_owner_kernel(const int64_t* slots, int64_t n, int64_t n_slots, int* owner) {
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
        const int64_t s = slots[i];
        if (s >= 0 && s < n_slots) owner[s] = -1;
    }
}

__global__ __launch_bounds__(kThreads) void claim_owner_kernel(const int64_t* slots, int64_t n, int64_t n_slots, int* owner) {
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
        const int64_t s = slots[i];
        if (s >= 0 && s < n_slots) atomicMax(owner + s, (int)i);   // a maximum: the same in any order
    }
}

struct ReadArgs {
    const unsigned char *data, *scale;
    int64_t pitch, scale_pitch;
    const int64_t* slots;
    int64_t n, n_slots;
    void* out;
    int64_t ld;
    int width;
    int per_row;
    unsigned magic;
    int rows;
    bool stream;
};

template <class T>
__global__ __launch_bounds__(kThreads) void read_rows_kernel(ReadArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    const int64_t groups = (a.n + a.rows - 1) / a.rows;
    for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        const int64_t r0 = g * a.rows;
        const int rows = (int)(a.n - r0 < a.rows ? a.n - r0 : a.rows);
        const int chunks = rows * a.per_row;
        for (int i = threadIdx.x; i < chunks; i += kThreads) {
            const int r = (int)(((uint64_t)(unsigned)i * a.magic) >> 31);
            const int c = (i - r * a.per_row) * V;
            const int64_t s = a.slots[r0 + r];
            float v[V];
            if (s >= 0 && s < a.n_slots) {
                unsigned q[V / 4];
                const unsigned char* p = a.data + s * a.pitch + c;
                if constexpr (V == 8) {
                    const u32x2 w = *(const u32x2*)p;
                    q[0] = w[0], q[1] = w[1];
                } else {
                    q[0] = *(const unsigned*)p;
                }
                const float scale = mx8_scale(a.scale[s * a.scale_pitch + mx8_scale_at(c >> 5)]);
#pragma unroll
                for (int k = 0; k < V / 4; ++k) {
                    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[k], false);
                    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[k], true);
                    v[4 * k + 0] = lo[0] * scale, v[4 * k + 1] = lo[1] * scale;
                    v[4 * k + 2] = hi[0] * scale, v[4 * k + 3] = hi[1] * scale;
                }
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = 0.0f;
            }
            T* to = (T*)a.out + (r0 + r) * a.ld + c;
            if (a.stream && a.width - c >= V)
                __builtin_nontemporal_store(pack_values<T>(v), (u32x4_any*)to);
            else
                store_values<T>(to, a.width - c, v);
        }
    }
}

// rows per group: about `chunks` threads' chunks, and enough groups to fill the chip
int rows_per_group(int64_t n, int per_row, int cus) {
    int rows = 1024 / per_row;
    if (n / (rows > 1 ? rows : 1) < 4 * cus) rows = kThreads / per_row;
    return rows < 1 ? 1 : rows > kMaxRows ? kMaxRows : rows;
}

unsigned magic_of(int per_row) { return (unsigned)(((1ull << 31) + per_row - 1) / per_row); }

template <int DEST>
void launch_write(DeviceCtx& ctx, hipStream_t s, int type, WriteArgs& a) {
    const int v = type == RMR_TYPE_F32 ? 4 : 8;
    a.per_row = (int)(a.pitch / v);
    a.magic = magic_of(a.per_row);
    a.rows = rows_per_group(a.n, a.per_row, ctx.num_cus);
    a.stream = a.n * a.width * (int64_t)type_bytes(type) > kStreamBytes;
    const int64_t groups = (a.n + a.rows - 1) / a.rows;
    const unsigned grid = (unsigned)(groups < kMaxGrid ? groups : kMaxGrid);
    ProfScope prof(ctx.prof, s, "quantise_rows", 0,
                   (double)a.n * (a.width * (double)type_bytes(type) + a.width + (a.width + 31) / 32));
    if (type == RMR_TYPE_F16)
        quantise_rows_kernel<F16, DEST><<<grid, kThreads, 0, s>>>(a);
    else if (type == RMR_TYPE_BF16)
        quantise_rows_kernel<BF16, DEST><<<grid, kThreads, 0, s>>>(a);
    else
        quantise_rows_kernel<float, DEST><<<grid, kThreads, 0, s>>>(a);
    RMR_HIP(hipGetLastError());
}

WriteArgs write_args(const RowSource& x, int width, int64_t n, const Mx8Rows& to) {
    WriteArgs a{};
    a.x = x.p, a.ld = x.ld, a.n = n, a.width = width;
    a.data = to.data, a.scale = to.scale, a.pitch = to.pitch, a.scale_pitch = to.scale_pitch;
    return a;
}

unsigned list_grid(int64_t n) {
    const int64_t g = (n + kThreads - 1) / kThreads;
    return (unsigned)(g < kMaxGrid ? g : kMaxGrid);
}

}  // namespace

void launch_quantise_rows(DeviceCtx& ctx, hipStream_t s, const RowSource& x, int width, int64_t n, const Mx8Rows& to) {
    if (n <= 0) return;
    WriteArgs a = write_args(x, width, n, to);
    launch_write<DEST_RUN>(ctx, s, x.type, a);
}

FeatureCache::FeatureCache(int device, int64_t slots, int width) : ctx_(device_ctx(device)), slots_(slots), width_(width) {
    data_.alloc((size_t)(slots * mx8_pitch(width)));
    scale_.alloc((size_t)(slots * mx8_scale_pitch(width)));
    owner_.alloc((size_t)slots);
    RMR_HIP(hipMemset(data_.p, 0, data_.n));
    RMR_HIP(hipMemset(scale_.p, 0, scale_.n));
    RMR_HIP(hipDeviceSynchronize());   // any stream may use it from here on
}

void FeatureCache::write(const RowSource& x, const int64_t* slots, int64_t n, hipStream_t s) {
    if (n <= 0) return;
    DeviceGuard guard(ctx_.device);
    WriteArgs a = write_args(x, width_, n, rows());
    a.slots = slots, a.n_slots = slots_, a.owner = owner_.p;
    if (n <= kScanRows) {
        launch_write<DEST_SCAN>(ctx_, s, x.type, a);
        return;
    }
    clear_owner_kernel<<<list_grid(n), kThreads, 0, s>>>(slots, n, slots_, owner_.p);
    claim_owner_kernel<<<list_grid(n), kThreads, 0, s>>>(slots, n, slots_, owner_.p);
    launch_write<DEST_OWNER>(ctx_, s, x.type, a);
}

void FeatureCache::write_run(const RowSource& x, int64_t first, int64_t n, hipStream_t s) {
    if (n <= 0) return;
    DeviceGuard guard(ctx_.device);
    WriteArgs a = write_args(x, width_, n, rows());
    a.first = first;
    launch_write<DEST_RUN>(ctx_, s, x.type, a);
}

void FeatureCache::read(const int64_t* slots, int64_t n, void* out, int type, int64_t ld, hipStream_t s) {
    if (n <= 0) return;
    DeviceGuard guard(ctx_.device);
    const Mx8Rows rw = rows();
    ReadArgs a{};
    a.data = rw.data, a.scale = rw.scale, a.pitch = rw.pitch, a.scale_pitch = rw.scale_pitch;
    a.slots = slots, a.n = n, a.n_slots = slots_, a.out = out, a.ld = ld, a.width = width_;
    const int v = type == RMR_TYPE_F32 ? 4 : 8;
    a.per_row = (width_ + v - 1) / v;
    a.magic = magic_of(a.per_row);
    a.rows = rows_per_group(n, a.per_row, ctx_.num_cus);
    a.stream = n * width_ * (int64_t)type_bytes(type) > kStreamBytes;
    const int64_t groups = (n + a.rows - 1) / a.rows;
    const unsigned grid = (unsigned)(groups < kMaxGrid ? groups : kMaxGrid);
    ProfScope prof(ctx_.prof, s, "read_rows", 0, (double)n * (width_ * (double)type_bytes(type) + width_ + (width_ + 31) / 32));
    if (type == RMR_TYPE_F16)
        read_rows_kernel<F16><<<grid, kThreads, 0, s>>>(a);
    else if (type == RMR_TYPE_BF16)
        read_rows_kernel<BF16><<<grid, kThreads, 0, s>>>(a);
    else
        read_rows_kernel<float><<<grid, kThreads, 0, s>>>(a);
    RMR_HIP(hipGetLastError());
}

}  // namespace rmr
