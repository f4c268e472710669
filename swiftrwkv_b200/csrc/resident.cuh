// How many blocks of a kernel run at once.
#pragma once

#include <atomic>

#include "common.cuh"

namespace rwkv {

// Blocks of one kernel that an SM holds, by device and warps per block, asked for once.
// The kernel may take `most` bytes of dynamic shared memory, the same whatever this
// call needs: the attribute is the kernel's, and another host thread may be between
// its own setting and its launch with rows of another length.
class ResidentBlocks {
    static constexpr int DEVICES = 64, WARPS = 16;
    std::atomic<int> n_[DEVICES][WARPS + 1] = {};

public:
    template <typename K>
    cudaError_t get(K kern, int threads, int smem, int most, int* per_sm) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
        int dev;
        if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
        std::atomic<int>* kept = dev < DEVICES ? &n_[dev][threads / 32] : nullptr;
        *per_sm = kept ? kept->load(std::memory_order_relaxed) : 0;
        if (*per_sm > 0) return cudaSuccess;
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kern, threads, smem);
        if (e != cudaSuccess) return e;
        if (*per_sm < 1) return cudaErrorInvalidConfiguration;
        if (kept) kept->store(*per_sm, std::memory_order_relaxed);
        return cudaSuccess;
    }
};

}  // namespace rwkv
