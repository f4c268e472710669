// Gradients of parameters that many rows share: each block of a row kernel leaves
// its partial sums in a row of `part`; their join adds them in a fixed order, so
// that results repeat bit for bit.
#pragma once

#include "ckpt8.cuh"

namespace rwkv {

struct ParamJoin {
    const float* part;  // [blocks][width]
    int blocks;
    int64_t width, D;  // column c goes to element c % D of out[c / D]
    void* out[3];
    int dtype;
};

// 32 columns per block, 32 interleaved slices of the partials.  Launched to start
// beside the row kernel's end (pdl_wait).
static __global__ void __launch_bounds__(1024) param_join_kernel(const ParamJoin a) {
    __shared__ float red[32][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + col;
    pdl_wait();
    float s = 0.f;
    if (c < a.width) {
#pragma unroll 4
        for (int b = slice; b < a.blocks; b += 32) s += a.part[b * a.width + c];
    }
    red[slice][col] = s;
    __syncthreads();
    // warp w sums column w over the slices
    const float t = warp_sum(red[col][slice]);
    const int64_t o = (int64_t)blockIdx.x * 32 + slice;
    if (col == 0 && o < a.width) {
        const int64_t k = o / a.D;
        store_param(a.out[k], a.dtype, o - k * a.D, t);
    }
}

inline int launch_param_join(const ParamJoin& a, cudaStream_t st) {
    const cudaError_t e =
        launch_pdl(param_join_kernel, dim3((unsigned)((a.width + 31) / 32)), dim3(1024), 0, st, a);
    if (e != cudaSuccess) return fail(RWKV_E_CUDA, "param_join_kernel: %s", cudaGetErrorString(e));
    return ok();
}

}  // namespace rwkv
