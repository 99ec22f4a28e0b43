// host.cuh -- host-side helpers shared by the C ABI's source files (defined in api.cu).
#pragma once

#include <atomic>
#include <string>

#include "common.cuh"

namespace kvx {

// Set the thread's last error and return `code`.
int fail(int code, const std::string &msg);
// Clear the thread's last error.
void clear_error();
// KVX_OK on an sm_100 device, else KVX_ERR_RUNTIME.
int check_device();
int sm_count();
// The message of a device-side error (status word [0] = code, [1] = detail).
const char *detail_message(int code, int detail);
// Read (and optionally reset) a device status pair; synchronous.
int read_status(int *dev_status, bool reset);

// Lets one kernel take `bytes` of dynamic shared memory a CTA on the current device, where this object
// has not done so yet: the limit belongs to a device.  A failure is returned and tried again.
class SmemLimit {
public:
    template <class K> cudaError_t allow(K kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
        if (e != cudaSuccess || (done_.load(std::memory_order_relaxed) & bit) != 0) return e;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) done_.fetch_or(bit, std::memory_order_relaxed);
        return e;
    }

private:
    std::atomic<uint64_t> done_{0};   // devices
};

#define KVX_CUDA(call)                                                                         \
    do {                                                                                       \
        cudaError_t e_ = (call);                                                               \
        if (e_ != cudaSuccess)                                                                 \
            return kvx::fail(KVX_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_)); \
    } while (0)

}  // namespace kvx
