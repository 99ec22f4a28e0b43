// host.cuh -- host-side helpers shared by the C ABI's source files (defined in api.cu).
#pragma once

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

#define KVX_CUDA(call)                                                                         \
    do {                                                                                       \
        cudaError_t e_ = (call);                                                               \
        if (e_ != cudaSuccess)                                                                 \
            return kvx::fail(KVX_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_)); \
    } while (0)

}  // namespace kvx
