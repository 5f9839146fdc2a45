// Host-side helpers of the C entry points: argument checks and status mapping.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/iqk_b200.h"

namespace iqk {

inline bool dtype_ok(int d) { return d == IQK_F32 || d == IQK_F16 || d == IQK_BF16; }
inline bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

inline int cuda_status(cudaError_t err) {
    if (err == cudaSuccess) return IQK_OK;
    cudaGetLastError();  // clear a sticky launch error for the caller
    return IQK_ERR_CUDA;
}

// SM count of the current device, queried once per device.
inline int num_sms_current() {
    static std::atomic<int> cached[64];
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev >= 0 && dev < 64 && (sms = cached[dev].load()) > 0) return sms;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
        sms = 148;
    if (dev >= 0 && dev < 64) cached[dev].store(sms);
    return sms;
}

// Launch configuration with programmatic stream serialization (the kernel
// waits with griddepcontrol.wait, see grid_dep_wait).
struct PdlLaunch {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    PdlLaunch(unsigned grid, unsigned block, size_t smem, cudaStream_t stream) {
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(block);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
};

}  // namespace iqk
