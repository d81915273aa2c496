// What the translation units that define C entries share: status mapping, device facts, argument tests.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/lloom_b200.h"

namespace lloom {

// LLOOM_OK, or LLOOM_ERR_LAUNCH with the error kept for lloom_b200_last_cuda_error (lloom_b200.cu)
int launch_status(cudaError_t e);

struct DeviceInfo {
    int sm_count = 0;
    int max_smem_optin = 0;   // per block
    int smem_per_sm = 0;      // per multiprocessor
    int smem_reserved = 0;    // per block, taken by the driver
    int cc_major = 0;
    bool ok = false;
};
// Of the current device, queried once per device; LLOOM_ERR_DEVICE if this code cannot run on it
int device_info(DeviceInfo &out);

inline bool aligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline bool elem_type_ok(int t) { return t == LLOOM_F32 || t == LLOOM_F16 || t == LLOOM_BF16; }

}  // namespace lloom
