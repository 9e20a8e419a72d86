// rows.h -- radar::FeatureCache and radar::Linear: rows of features behind the detector, on the device (no counterpart in the
// reference).  Thin owners of the C-ABI's handles; errors throw as the reference's constructors do.  Pointers are device
// pointers, streams are hipStream_t (nullptr = the default stream); calls are enqueued and return.
#pragma once
#include <cstddef>
#include <cstdint>
#include <utility>

#include "../rmr.h"
#include "detector.h"

namespace radar {

class FeatureCache {
   public:
    FeatureCache() = delete;
    FeatureCache(std::int64_t slots, int width, int device = 0) {
        if (rmr_status s = rmr_feature_cache_create(device, slots, width, &h_); s != RMR_OK) detail::throw_status(s);
    }
    ~FeatureCache() { rmr_feature_cache_destroy(h_); }
    FeatureCache(const FeatureCache&) = delete;
    FeatureCache& operator=(const FeatureCache&) = delete;
    FeatureCache(FeatureCache&& o) noexcept : h_(std::exchange(o.h_, nullptr)) {}
    FeatureCache& operator=(FeatureCache&& o) noexcept {
        std::swap(h_, o.h_);
        return *this;
    }

    void write(const void* x, int type, std::int64_t ld, const std::int64_t* slots, std::int64_t n, void* stream = nullptr) {
        if (rmr_status s = rmr_feature_cache_write(h_, x, type, ld, slots, n, stream); s != RMR_OK) detail::throw_status(s);
    }
    void read(const std::int64_t* slots, std::int64_t n, void* out, int type, std::int64_t ld, void* stream = nullptr) {
        if (rmr_status s = rmr_feature_cache_read(h_, slots, n, out, type, ld, stream); s != RMR_OK) detail::throw_status(s);
    }
    std::size_t bytes() const { return rmr_feature_cache_bytes(h_); }
    rmr_feature_cache* handle() const { return h_; }

   private:
    rmr_feature_cache* h_ = nullptr;
};

class Linear {
   public:
    Linear() = delete;
    // weight [out_features][in_features] of weight_type, bias f32 or nullptr, both in `mem` (RMR_MEM_HOST / RMR_MEM_DEVICE)
    Linear(int in_features, int out_features, int format, int activation, const void* weight, int weight_type, const float* bias,
           int mem = RMR_MEM_HOST, void* stream = nullptr, int device = 0) {
        const rmr_linear_cfg c{device, in_features, out_features, format, activation};
        if (rmr_status s = rmr_linear_create(&c, weight, weight_type, in_features, bias, mem, stream, &h_); s != RMR_OK)
            detail::throw_status(s);
    }
    ~Linear() { rmr_linear_destroy(h_); }
    Linear(const Linear&) = delete;
    Linear& operator=(const Linear&) = delete;
    Linear(Linear&& o) noexcept : h_(std::exchange(o.h_, nullptr)) {}
    Linear& operator=(Linear&& o) noexcept {
        std::swap(h_, o.h_);
        return *this;
    }

    // bytes of workspace that the call needs; kept: through the form that takes a cache
    std::size_t workspace(const rmr_linear_call& call, bool kept = false) const {
        std::size_t n = 0;
        if (rmr_status s = rmr_linear_workspace(h_, &call, kept, &n); s != RMR_OK) detail::throw_status(s);
        return n;
    }
    void run(const rmr_linear_call& call, void* stream = nullptr) const {
        if (rmr_status s = rmr_linear_run(h_, &call, stream); s != RMR_OK) detail::throw_status(s);
    }
    void run(const FeatureCache& cache, const std::int64_t* slots, const rmr_linear_call& call, void* stream = nullptr) const {
        if (rmr_status s = rmr_linear_run_kept(h_, cache.handle(), slots, &call, stream); s != RMR_OK) detail::throw_status(s);
    }

   private:
    rmr_linear* h_ = nullptr;
};

}  // namespace radar
