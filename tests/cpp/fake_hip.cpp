// fake_hip.cpp -- a HIP runtime of two devices without a GPU, for tests of host code: device memory is host memory, a kernel launch
// does nothing, streams, events and graphs are names.  Loaded with global visibility before librmr.so, whose calls it takes.
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <cstring>

namespace {

constexpr int kDevices = 2;
thread_local int current = 0;
std::atomic<long> synced[kDevices], launches, urgent;
char names[64];   // what handles point at

}  // namespace

extern "C" {

// for the tests: waits for the whole device, kernel launches, streams of another priority than the default so far
long fake_hip_synced(int device) { return synced[device]; }
long fake_hip_launches() { return launches; }
long fake_hip_priority_streams() { return urgent; }

hipError_t hipGetDeviceCount(int* n) { return *n = kDevices, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = current, hipSuccess; }
hipError_t hipSetDevice(int d) {
    if (d < 0 || d >= kDevices) return hipErrorInvalidDevice;
    return current = d, hipSuccess;
}
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    std::memset(p, 0, sizeof(*p));
    std::snprintf(p->gcnArchName, sizeof(p->gcnArchName), "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return ++synced[current], hipSuccess; }
hipError_t hipDeviceGetStreamPriorityRange(int* least, int* greatest) { return *least = 1, *greatest = -1, hipSuccess; }

hipError_t hipMalloc(void** p, size_t n) { return (*p = std::calloc(1, n + 256)) ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return hipMalloc(p, n); }
hipError_t hipHostFree(void* p) { return hipFree(p); }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { return std::memcpy(d, s, n), hipSuccess; }
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) { return std::memcpy(d, s, n), hipSuccess; }
hipError_t hipMemcpy2DAsync(void* d, size_t dp, const void* s, size_t sp, size_t w, size_t h, hipMemcpyKind, hipStream_t) {
    for (size_t i = 0; i < h; ++i) std::memcpy((char*)d + i * dp, (const char*)s + i * sp, w);
    return hipSuccess;
}
hipError_t hipMemset(void* p, int v, size_t n) { return std::memset(p, v, n), hipSuccess; }
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) { return std::memset(p, v, n), hipSuccess; }

hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = (hipStream_t)names, hipSuccess; }
hipError_t hipStreamCreateWithPriority(hipStream_t* s, unsigned, int priority) { return urgent += priority != 0, *s = (hipStream_t)names, hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamBeginCapture(hipStream_t, hipStreamCaptureMode) { return hipSuccess; }
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* g) { return *g = (hipGraph_t)names, hipSuccess; }
hipError_t hipGraphInstantiate(hipGraphExec_t* e, hipGraph_t, hipGraphNode_t*, char*, size_t) { return *e = (hipGraphExec_t)names, hipSuccess; }
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) { return hipSuccess; }
hipError_t hipGraphDestroy(hipGraph_t) { return hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t) { return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { return *e = (hipEvent_t)names, hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return *e = (hipEvent_t)names, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { return *ms = 1.0f, hipSuccess; }

const char* hipGetErrorString(hipError_t) { return "an error of the stand-in runtime"; }
hipError_t hipGetLastError() { return hipSuccess; }

hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) { return ++launches, hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* s) { return *g = dim3(1), *b = dim3(1), *lds = 0, *s = nullptr, hipSuccess; }
void** __hipRegisterFatBinary(const void*) { return (void**)names; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}

}  // extern "C"
