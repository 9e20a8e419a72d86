// radar::FeatureCache and radar::Linear from C++: without a GPU the constructors throw; with one, rows written by the test go through
// a cache and two layers, and the results go back for comparison with the ctypes path.  argv: in.bin out.bin
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <vector>

#include "radar/rows.h"

static std::vector<float> load(FILE* f, size_t n) {
    std::vector<float> v(n);
    if (std::fread(v.data(), 4, n, f) != n) std::exit(2);
    return v;
}

template <class T>
static T* to_device(const std::vector<T>& v) {
    void* p = nullptr;
    if (hipMalloc(&p, v.size() * sizeof(T)) != hipSuccess || hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) std::exit(3);
    return (T*)p;
}

int main(int argc, char** argv) {
    if (rmr_device_count() == 0) {
        int thrown = 0;
        const float w[6] = {};
        try {
            radar::FeatureCache c(0, 8);
        } catch (const std::invalid_argument&) { ++thrown; }
        try {
            radar::FeatureCache c(8, 8);
        } catch (const std::runtime_error&) { ++thrown; }
        try {
            radar::Linear l(3, 2, 9, RMR_ACT_NONE, w, RMR_TYPE_F32, nullptr);
        } catch (const std::invalid_argument&) { ++thrown; }
        try {
            radar::Linear l(3, 2, RMR_LINEAR_MX8, RMR_ACT_NONE, w, RMR_TYPE_F32, nullptr);
        } catch (const std::runtime_error&) { ++thrown; }
        std::printf(thrown == 4 ? "api_rows ok\n" : "api_rows: %d of 4 thrown\n", thrown);
        return thrown == 4 ? 0 : 1;
    }
    if (argc < 3) return 2;
    constexpr int kRows = 70, kIn = 200, kMid = 96, kOut = 40;
    FILE* f = std::fopen(argv[1], "rb");
    if (!f) return 2;
    const auto x = load(f, kRows * kIn), w1 = load(f, kMid * kIn), b1 = load(f, kMid), w2 = load(f, kOut * kMid);
    std::fclose(f);
    std::vector<std::int64_t> slots(kRows);
    for (int i = 0; i < kRows; ++i) slots[i] = (i * 37) % 101;
    float* dx = to_device(x);
    std::int64_t* ds = to_device(slots);
    float* mid = to_device(std::vector<float>(kRows * kMid));
    float* out = to_device(std::vector<float>(kRows * kOut));
    radar::FeatureCache cache(101, kIn);
    cache.write(dx, RMR_TYPE_F32, kIn, ds, kRows);
    radar::Linear up(kIn, kMid, RMR_LINEAR_MX8, RMR_ACT_SILU, w1.data(), RMR_TYPE_F32, b1.data());
    radar::Linear down(kMid, kOut, RMR_LINEAR_MX8, RMR_ACT_NONE, w2.data(), RMR_TYPE_F32, nullptr);
    rmr_linear_call call{};
    call.rows = kRows, call.y = mid, call.y_type = RMR_TYPE_F32, call.ldy = kMid;
    if (up.workspace(call, true) != 0) return 4;
    up.run(cache, ds, call);
    rmr_linear_call second{};
    second.x = mid, second.x_type = RMR_TYPE_F32, second.ldx = kMid, second.rows = kRows;
    second.y = out, second.y_type = RMR_TYPE_F32, second.ldy = kOut;
    unsigned char* ws = to_device(std::vector<unsigned char>(down.workspace(second) + 16));
    second.workspace = ws, second.workspace_bytes = down.workspace(second);
    down.run(second);
    std::vector<float> back(kRows * (kMid + kOut));
    if (hipMemcpy(back.data(), mid, kRows * kMid * 4, hipMemcpyDeviceToHost) != hipSuccess) return 5;
    if (hipMemcpy(back.data() + kRows * kMid, out, kRows * kOut * 4, hipMemcpyDeviceToHost) != hipSuccess) return 5;
    f = std::fopen(argv[2], "wb");
    std::fwrite(back.data(), 4, back.size(), f);
    std::fclose(f);
    std::printf("api_rows ran\n");
    return 0;
}
