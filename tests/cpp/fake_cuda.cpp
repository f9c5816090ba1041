// A CUDA runtime for the host side of the candidate operators: device memory is host memory, kernels do not run, and
// what was asked of streams and events is counted.  Linked with the objects of their sources into a
// library of its own (tests/test_candidates_host.py), so that page lists, plans, launch shapes and the order of
// device work are tested without a GPU.
#include "../../include/t2sx.h"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

namespace {

std::string g_error;
long long g_launches, g_synced, g_fail_at;   // g_fail_at: the launch that fails, counted from 1; 0: none
std::map<cudaStream_t, long long> g_recorded;
dim3 g_grid;
cudaError_t g_last = cudaSuccess;
struct { dim3 grid, block; size_t smem; cudaStream_t stream; } g_config;

cudaError_t launched(dim3 grid) {
    g_grid = grid;
    if (++g_launches == g_fail_at) return g_last = cudaErrorLaunchFailure;
    return cudaSuccess;
}

CUresult CUDAAPI encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
               CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}

}  // namespace

// ---- what the operators take from other parts of the library ----
int t2sx_set_error(int code, const char* msg) {
    g_error = msg;
    return code;
}
extern "C" T2SX_API const char* t2sx_last_error(void) { return g_error.c_str(); }
namespace t2sx {
long long tc_test_wait_cycles() { return 0; }
namespace tc {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() { return encode; }
}  // namespace tc
}  // namespace t2sx

// ---- for the tests ----
extern "C" {
T2SX_API void fake_reset(void) {
    g_launches = g_synced = g_fail_at = 0;
    g_recorded.clear();
    g_last = cudaSuccess;
}
T2SX_API void fake_fail_launch(long long nth) { g_fail_at = g_launches + nth; }
T2SX_API long long fake_launches(void) { return g_launches; }
T2SX_API long long fake_grid_x(void) { return g_grid.x; }
T2SX_API long long fake_synced(void) { return g_synced; }
T2SX_API long long fake_recorded(void* stream) { return g_recorded[(cudaStream_t)stream]; }
}

// ---- the runtime ----
extern "C" {
void** __cudaRegisterFatBinary(void*) { static void* h; return &h; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
unsigned __cudaPushCallConfiguration(dim3 grid, dim3 block, size_t smem, void* stream) {
    g_config = {grid, block, smem, (cudaStream_t)stream};
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* grid, dim3* block, size_t* smem, void* stream) {
    *grid = g_config.grid;
    *block = g_config.block;
    *smem = g_config.smem;
    *(cudaStream_t*)stream = g_config.stream;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void*, dim3 grid, dim3, void**, size_t, cudaStream_t) { return launched(grid); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void*, void**) { return launched(c->gridDim); }
cudaError_t cudaGetLastError() {
    const cudaError_t e = g_last;
    g_last = cudaSuccess;
    return e;
}
const char* cudaGetErrorString(cudaError_t) { return "a failure made by the test"; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { *e = (cudaEvent_t)malloc(1); return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t e) { free(e); return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t s) { ++g_recorded[s]; return cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { ++g_synced; return cudaSuccess; }
cudaError_t cudaStreamWaitEvent(cudaStream_t, cudaEvent_t, unsigned) { return cudaSuccess; }
cudaError_t cudaMalloc(void** p, size_t n) { return (*p = malloc(n)) ? cudaSuccess : cudaErrorMemoryAllocation; }
cudaError_t cudaFree(void* p) { free(p); return cudaSuccess; }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) { return cudaMalloc(p, n); }
cudaError_t cudaMallocHost(void** p, size_t n) { return cudaMalloc(p, n); }
cudaError_t cudaFreeHost(void* p) { return cudaFree(p); }
cudaError_t cudaHostGetDevicePointer(void** d, void* h, unsigned) { *d = h; return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) { memcpy(d, s, n); return cudaSuccess; }
}
