// The CUDA runtime as the host side of one kernel file sees it, for tests without a
// GPU: several devices, launches that are written down and never run. Linked with
// the file's object (its kernels are not registered anywhere).
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <map>
#include <set>
#include <string>
#include <utility>

namespace {
int g_device = 0, g_open_timings = 0, g_unbound_launches = 0;
unsigned g_last_grid = 0;
int g_launches = 0;
std::set<std::pair<int, const void*>> g_opted;   // device, kernel
char g_message[512];
int g_err = 0;

// what the driver would say to a launch
cudaError_t launch(const void* f, dim3 grid, size_t shared) {
    if (shared > 48 * 1024 && !g_opted.count({g_device, f})) {
        ++g_unbound_launches;
        return cudaErrorInvalidValue;
    }
    g_last_grid = grid.x;
    ++g_launches;
    return cudaSuccess;
}
CUresult encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}
}  // namespace

// ------------------------------------------------ what the tests ask and set
#define TEST_API extern "C" __attribute__((visibility("default")))
TEST_API void fake_set_device(int d) { g_device = d; }
TEST_API int fake_open_timings() { return g_open_timings; }
TEST_API int fake_launches() { return g_launches; }
TEST_API int fake_refused_launches() { return g_unbound_launches; }
TEST_API unsigned fake_last_grid() { return g_last_grid; }
TEST_API const char* fake_message() { return g_message; }

// ------------------------------------------------ the runtime's own helpers
bool sb_op_begin(void* stream, cudaStream_t* st, int** err) {
    *st = (cudaStream_t)stream;
    *err = &g_err;
    return true;
}
void sb_set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_message, sizeof(g_message), fmt, ap);
    va_end(ap);
}
bool sb_cuda_ok(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return true;
    sb_set_error("%s: error %d", what, (int)e);
    return false;
}
int sb_timing_begin(const char*, cudaStream_t) { return g_open_timings++; }
void sb_timing_end(int, cudaStream_t) { --g_open_timings; }

// ------------------------------------------------ the CUDA runtime
extern "C" {
cudaError_t CUDARTAPI cudaGetDevice(int* d) {
    *d = g_device;
    return cudaSuccess;
}
cudaError_t CUDARTAPI cudaGetLastError(void) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int dev) {   // SM counts that tell devices apart
    *v = dev == 0 ? 148 : 100 + dev;
    return cudaSuccess;
}
cudaError_t CUDARTAPI cudaFuncSetAttribute(const void* f, cudaFuncAttribute, int) {
    g_opted.insert({g_device, f});
    return cudaSuccess;
}
cudaError_t CUDARTAPI cudaGetDriverEntryPoint(const char*, void** f, unsigned long long, cudaDriverEntryPointQueryResult* found) {
    *f = (void*)encode;
    *found = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
cudaError_t CUDARTAPI cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) {
    return launch(f, c->gridDim, c->dynamicSmemBytes);
}
cudaError_t CUDARTAPI cudaLaunchKernel(const void* f, dim3 grid, dim3, void**, size_t shared, cudaStream_t) {
    return launch(f, grid, shared);
}
unsigned CUDARTAPI __cudaPushCallConfiguration(dim3, dim3, size_t, cudaStream_t) { return 1; }   // <<< >>> launches nothing
cudaError_t CUDARTAPI __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
void** CUDARTAPI __cudaRegisterFatBinary(void*) { return nullptr; }
void CUDARTAPI __cudaRegisterFatBinaryEnd(void**) {}
void CUDARTAPI __cudaUnregisterFatBinary(void**) {}
void CUDARTAPI __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
}
