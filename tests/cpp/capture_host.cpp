// What va_adamw_list_create asks of the HIP runtime while its stream is captured: whether it is, and nothing else.  The runtime's functions
// that a context and a list call are defined here, over host memory, so no device is needed and none is touched.
#define __HIP_PLATFORM_AMD__
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "va_hip.h"

static int allocations, copies, frees;
static hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
static hipError_t asked = hipSuccess;

extern "C" {
hipError_t hipGetDeviceCount(int* n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    std::memset(p, 0, sizeof(*p));
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = reinterpret_cast<hipStream_t>(&capture), hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) { return *s = capture, asked; }
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return *p = std::calloc(1, n), hipSuccess; }
hipError_t hipHostFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetSymbolAddress(void**, const void*) { return hipErrorInvalidValue; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) { return ++allocations, *p = std::malloc(n), hipSuccess; }
hipError_t hipFree(void* p) { return ++frees, std::free(p), hipSuccess; }
hipError_t hipMemcpy(void* to, const void* from, size_t n, hipMemcpyKind) { return ++copies, std::memcpy(to, from, n), hipSuccess; }
}

static int failures = 0;
#define CHECK(cond)                                             \
    do {                                                        \
        if (!(cond)) {                                          \
            std::printf("FAIL line %d: %s\n", __LINE__, #cond); \
            ++failures;                                         \
        }                                                       \
    } while (0)

int main() {
    va_context* ctx = nullptr;
    if (va_context_create(0, &ctx) != VA_OK) return std::printf("no context\n"), 1;
    static float param[300], grad[300], first[300], second[300];
    va_adamw_tensor t{};
    t.param = t.out_param = param, t.grad = grad, t.first = t.out_first = first, t.second = t.out_second = second;
    t.size = 300, t.rate_factor = t.decay_factor = 1.0f;
    va_adamw_list* list = nullptr;
    allocations = copies = frees = 0;
    CHECK(va_adamw_list_create(ctx, &t, 1, 32, &list) == VA_OK && list && allocations == 1 && copies == 2);
    CHECK(va_adamw_list_destroy(list) == VA_OK && frees == 1);
    for (hipStreamCaptureStatus s : {hipStreamCaptureStatusActive, hipStreamCaptureStatusInvalidated}) {
        capture = s;
        allocations = copies = frees = 0;
        list = reinterpret_cast<va_adamw_list*>(&t);
        CHECK(va_adamw_list_create(ctx, &t, 1, 32, &list) == VA_ERR_INVALID_ARG && !list);
        CHECK(!allocations && !copies && !frees);
        CHECK(std::strstr(va_last_error_message(ctx), "captured"));
    }
    capture = hipStreamCaptureStatusNone;
    asked = hipErrorStreamCaptureImplicit;  // (the legacy stream while another is captured)
    allocations = copies = frees = 0;
    CHECK(va_adamw_list_create(ctx, &t, 1, 32, &list) == VA_ERR_HIP && !list && !allocations && !copies && !frees);
    asked = hipSuccess;
    CHECK(va_adamw_list_create(ctx, &t, 1, 32, &list) == VA_OK && list);
    CHECK(va_adamw_list_destroy(list) == VA_OK);
    CHECK(va_context_destroy(ctx) == VA_OK);
    std::printf("capture_host: %s\n", failures ? "failed" : "ok");
    return failures != 0;
}
