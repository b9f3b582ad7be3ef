// A kernel's launch attributes, set when a launch needs more than any before it.
#pragma once

#include <cuda_runtime_api.h>

#include <mutex>

namespace rfx {

// The dynamic shared memory that one kernel may ask for, raised when a launch asks for more than any before
// it, and, where asked for, clusters of more than eight blocks: one static object a kernel, so that a call does not
// pay for the attributes again.  Host threads take turns: an attribute set between another's check and
// its own would leave less than `have` says.
struct SmemLimit {
    static constexpr int DEVICES = 64;
    int have[DEVICES] = {};
    bool wide[DEVICES] = {};
    std::mutex turn;
    template <typename K>
    cudaError_t raise(K kernel, size_t bytes, bool wide_clusters = false) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev < 0 || dev >= DEVICES) return cudaErrorInvalidDevice;
        std::lock_guard<std::mutex> mine(turn);
        if (wide_clusters && !wide[dev]) {
            e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            wide[dev] = true;
        }
        if (have[dev] >= (int)bytes) return cudaSuccess;
        e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess) have[dev] = (int)bytes;
        return e;
    }
};

}  // namespace rfx
