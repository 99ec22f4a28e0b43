// fake_device.cpp -- the CUDA runtime calls that the serving-step operators' host code makes, without a
// device: memory is the host's, launches are recorded, and a call can be made to fail.  Linked with
// the sources of those operators and of the kernels beside them it shows what they ask of the runtime.
#include <cuda.h>
#include <cuda_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <set>
#include <string>
#include <utility>
#include <vector>

#include "fake_device.h"

namespace {

constexpr int kDefaultSmem = 48 * 1024;   // what a kernel may take a CTA without having been allowed more

int device = 0;
cudaError_t last = cudaSuccess;
int fail_launch = -1, fail_attribute = -1;   // which one from now on fails (0: the next)
std::vector<Launch> launches;
std::map<const void *, std::string> &names() {  // (filled before this file's own objects are made)
    static std::map<const void *, std::string> m;
    return m;
}
std::map<std::pair<int, const void *>, int> smem;
std::set<void *> memory;
struct { dim3 grid, block; size_t bytes; } call;   // between a launch's <<<>>> and its stub

bool hit(int &countdown) { return countdown >= 0 && countdown-- == 0; }

CUresult encode(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}

cudaError_t launched(const void *f, dim3 grid, dim3 block, size_t bytes, void **args) {
    if (hit(fail_launch)) return cudaErrorLaunchOutOfResources;
    Launch l{};
    const std::string &n = names()[f];
    l.kind = n.find("rotate") != n.npos ? ROTATE : n.find("prefix_kernel") != n.npos ? PREFIX
             : n.find("stream_kernel") != n.npos ? STREAM : n.find("combine_kernel") != n.npos ? COMBINE : OTHER;
    l.device = device;
    l.grid = int32_t(grid.x * grid.y);
    l.threads = int32_t(block.x);
    l.smem = int32_t(bytes);
    const auto a = smem.find({device, f});
    l.allowed = a == smem.end() ? kDefaultSmem : a->second;
    if (l.smem > l.allowed) return cudaErrorInvalidValue;
    if (l.kind == PREFIX || l.kind == STREAM || l.kind == COMBINE) fake_paged(args[0], &l);
    launches.push_back(l);
    return cudaSuccess;
}

}  // namespace

// ---- the runtime --------------------------------------------------------------------------------------

extern "C" {

cudaError_t cudaGetDevice(int *d) {
    *d = device;
    return cudaSuccess;
}
cudaError_t cudaMalloc(void **p, size_t n) {
    // (large scratch is never touched: the pages are not there before they are)
    *p = std::calloc(1, n > 0 ? n : 1);
    if (*p == nullptr) return cudaErrorMemoryAllocation;
    memory.insert(*p);
    return cudaSuccess;
}
cudaError_t cudaFree(void *p) {
    if (p != nullptr && memory.erase(p) == 0) return cudaErrorInvalidValue;
    std::free(p);
    return cudaSuccess;
}
cudaError_t cudaMemset(void *p, int v, size_t n) {
    std::memset(p, v, n);
    return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void *p, int v, size_t n, cudaStream_t) { return cudaMemset(p, v, n); }
cudaError_t cudaDeviceSynchronize() { return cudaSuccess; }
cudaError_t cudaGetLastError() {
    const cudaError_t e = last;
    last = cudaSuccess;
    return e;
}
const char *cudaGetErrorString(cudaError_t) { return "an error"; }
cudaError_t cudaFuncSetAttribute(const void *f, cudaFuncAttribute a, int v) {
    if (hit(fail_attribute)) return cudaErrorInvalidValue;
    if (a == cudaFuncAttributeMaxDynamicSharedMemorySize) smem[{device, f}] = v;
    return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char *, void **p, unsigned long long, cudaDriverEntryPointQueryResult *q) {
    *p = reinterpret_cast<void *>(&encode);
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void *f, dim3 grid, dim3 block, void **args, size_t bytes, cudaStream_t) {
    return last = launched(f, grid, block, bytes, args);
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *c, const void *f, void **args) {
    return launched(f, c->gridDim, c->blockDim, c->dynamicSmemBytes, args);
}

// what the compiler's registration code of a translation unit calls
void **__cudaRegisterFatBinary(void *) {
    static void *handle = nullptr;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
char __cudaInitModule(void **) { return 1; }
void __cudaRegisterFunction(void **, const char *f, char *, const char *name, int, uint3 *, uint3 *, dim3 *, dim3 *, int *) {
    names()[f] = name;
}
unsigned __cudaPushCallConfiguration(dim3 grid, dim3 block, size_t bytes, struct CUstream_st *) {
    call = {grid, block, bytes};
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3 *grid, dim3 *block, size_t *bytes, void *stream) {
    *grid = call.grid, *block = call.block, *bytes = call.bytes;
    *static_cast<cudaStream_t *>(stream) = nullptr;
    return cudaSuccess;
}

// ---- for the tests ---------------------------------------------------------------------------------------

void fake_reset() {
    device = 0;
    fail_launch = fail_attribute = -1;
    launches.clear();
}
void fake_set_device(int d) { device = d; }
void fake_fail_launch(int n) { fail_launch = n; }
void fake_fail_attribute(int n) { fail_attribute = n; }
int fake_live_allocations() { return int(memory.size()); }
int fake_launches(Launch *out, int most) {
    const int n = int(launches.size()) < most ? int(launches.size()) : most;
    std::memcpy(out, launches.data(), size_t(n) * sizeof(Launch));
    launches.clear();
    return n;
}

}  // extern "C"
