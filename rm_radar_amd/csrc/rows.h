// rows.h -- dense operators on rows of features: a cache of block-scaled 8-bit rows (feature_cache.hip) and a linear layer
// with bias, activation and residual in its epilogue (linear.hip).
//
// A block-scaled ("mx8") row keeps blocks of 32 values: one power of two 2^e per block (the byte e + 127) and 32 OCP e4m3
// values.  e is the smallest exponent in [-127, 127] with max|v| <= 448 * 2^e over the block's finite values, so nothing saturates
// and every value is off by at most half an e4m3 step.  The matrix pipe multiplies such blocks itself
// (v_mfma_scale_f32_16x16x128_f8f6f4), the scales cost no arithmetic.
//
// Storage of a row: width bytes of e4m3 padded with zeros to a multiple of 128 (one K step of the product), and 16 scale bytes
// per 512 values: the byte of block 4 t + g sits at 4 g + t, so that lane group g of the MFMA finds the scales of its block in
// four consecutive steps in ONE dword.
#pragma once
#include "common.h"

namespace rmr {

// makes a device current for one call and gives the caller's back afterwards
class DeviceGuard {
   public:
    explicit DeviceGuard(int device) {
        RMR_HIP(hipGetDevice(&before_));
        if (before_ != device) RMR_HIP(hipSetDevice(device));
        device_ = device;
    }
    ~DeviceGuard() {
        if (before_ != device_) (void)hipSetDevice(before_);
    }
    DeviceGuard(const DeviceGuard&) = delete;
    DeviceGuard& operator=(const DeviceGuard&) = delete;

   private:
    int before_ = 0, device_ = 0;
};

// gives the caller's device back whatever became current meanwhile: around the making of a handle, whose device_ctx() checks a device
// and makes it current.  (Without a device there is none to give back.)
class DeviceKeeper {
   public:
    DeviceKeeper() {
        if (hipGetDevice(&before_) != hipSuccess) before_ = -1;
    }
    ~DeviceKeeper() {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }
    DeviceKeeper(const DeviceKeeper&) = delete;
    DeviceKeeper& operator=(const DeviceKeeper&) = delete;

   private:
    int before_ = -1;
};

inline size_t type_bytes(int type) { return type == RMR_TYPE_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == RMR_TYPE_F16 || type == RMR_TYPE_BF16 || type == RMR_TYPE_F32; }
inline int64_t mx8_pitch(int64_t width) { return (width + 127) / 128 * 128; }
inline int64_t mx8_scale_pitch(int64_t width) { return (width + 511) / 512 * 16; }

// rows of `width` elements, `ld` elements apart
struct RowSource {
    const void* p;
    int type;
    int64_t ld;
};

// mx8 rows: data[row][pitch], scale[row][scale_pitch]
struct Mx8Rows {
    unsigned char* data;
    unsigned char* scale;
    int64_t pitch, scale_pitch;
};

// rows i = 0 .. n-1 of x into row i of `to`
void launch_quantise_rows(DeviceCtx& ctx, hipStream_t s, const RowSource& x, int width, int64_t n, const Mx8Rows& to);

class FeatureCache {
   public:
    FeatureCache(int device, int64_t slots, int width);
    void write(const RowSource& x, const int64_t* slots, int64_t n, hipStream_t s);
    // rows into slots first .. first + n - 1
    void write_run(const RowSource& x, int64_t first, int64_t n, hipStream_t s);
    void read(const int64_t* slots, int64_t n, void* out, int type, int64_t ld, hipStream_t s);
    int64_t slots() const { return slots_; }
    int width() const { return width_; }
    int device() const { return ctx_.device; }
    size_t bytes() const { return data_.n + scale_.n + owner_.n * sizeof(int); }
    Mx8Rows rows() { return {data_.p, scale_.p, mx8_pitch(width_), mx8_scale_pitch(width_)}; }

   private:
    DeviceCtx& ctx_;
    int64_t slots_;
    int width_;
    DevBuf<unsigned char> data_, scale_;
    DevBuf<int> owner_;  // per slot: the highest row of the running write that names it
};

class Linear {
   public:
    Linear(const rmr_linear_cfg& cfg, const void* weight, int weight_type, int64_t ldw, const float* bias, int mem, hipStream_t s);
    // where the layer's rows come from: x, or slots of a cache
    struct Call {
        int64_t ld_bytes() const { return x.ld * (int64_t)type_bytes(x.type); }
        RowSource x{nullptr, 0, 0};
        FeatureCache* cache = nullptr;
        const int64_t* slots = nullptr;
        bool kept = false;   // the rows are a cache's
        int64_t rows = 0;
        const void* residual = nullptr;
        int64_t ldr = 0;
        void* y = nullptr;
        int y_type = 0;
        int64_t ldy = 0;
        void* workspace = nullptr;
        size_t workspace_bytes = 0;
        hipStream_t stream = nullptr;
    };
    size_t workspace_bytes(const Call& c) const;
    void run(const Call& c);
    int in_features() const { return cfg_.in_features; }
    int out_features() const { return cfg_.out_features; }
    const rmr_linear_cfg& cfg() const { return cfg_; }

   private:
    struct Plan;
    Plan plan(const Call& c) const;

    DeviceCtx& ctx_;
    rmr_linear_cfg cfg_;
    int ksteps_ = 0;   // steps of 128 bytes along a row
    int groups_ = 0;   // groups of 64 output features
    DevBuf<unsigned char> w_;       // [group][step][j][half][lane][16 bytes], see linear.hip
    DevBuf<unsigned> wscale_;       // mx8: [group][ceil(steps / 4)][j][lane], four steps' scale bytes of a lane's block
    DevBuf<float> bias_;            // [64 groups]
    DevBuf<unsigned char> zero_;    // 128 bytes of zeros: what lanes behind a row's end, or without a row, read
};

}  // namespace rmr

struct rmr_feature_cache {
    rmr::FeatureCache impl;
    rmr_feature_cache(int device, int64_t slots, int width) : impl(device, slots, width) {}
};
struct rmr_linear {
    rmr::Linear impl;
    rmr_linear(const rmr_linear_cfg& c, const void* w, int wt, int64_t ldw, const float* b, int mem, hipStream_t s)
        : impl(c, w, wt, ldw, b, mem, s) {}
};
