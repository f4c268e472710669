// Gradients of parameters that many rows share: each block of a row kernel leaves
// its partial sums in a row of `part`; their join adds them in a fixed order, so
// that results repeat bit for bit.
#pragma once

#include "ckpt8.cuh"

namespace rwkv {

struct ParamJoin {
    const float* part;  // [blocks][width]
    int blocks;
    int64_t width, D;  // even; column c goes to element c % D of out[c / D]
    void* out[3];
    int dtype;
};

constexpr int PJ_SLICES = 16;

// 64 columns per block, two to a lane, PJ_SLICES interleaved slices of the partials.
// Launched to start beside the row kernel's end (pdl_wait).
static __global__ void __launch_bounds__(32 * PJ_SLICES) param_join_kernel(const ParamJoin a) {
    __shared__ float2 red[PJ_SLICES][32];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 64 + 2 * lane;
    pdl_wait();
    float2 s = make_float2(0.f, 0.f);
    if (c < a.width) {
        // eight loads at a time in flight, also of the last few
        for (int b0 = slice; b0 < a.blocks; b0 += 8 * PJ_SLICES) {
            float2 v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int b = b0 + i * PJ_SLICES;
                v[i] = b < a.blocks ? *reinterpret_cast<const float2*>(a.part + b * a.width + c) : make_float2(0.f, 0.f);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) s.x += v[i].x, s.y += v[i].y;
        }
    }
    red[slice][lane] = s;
    __syncthreads();
    const int64_t o = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x < 64 && o < a.width) {
        const float* r = &red[0][0].x + threadIdx.x;
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < PJ_SLICES; i++) t += r[64 * i];
        const int k = a.width == a.D ? 0 : (int)(o / a.D);
        store_param(a.out[k], a.dtype, o - k * a.D, t);
    }
}

inline int launch_param_join(const ParamJoin& a, cudaStream_t st) {
    const cudaError_t e =
        launch_pdl(param_join_kernel, dim3((unsigned)((a.width + 63) / 64)), dim3(32 * PJ_SLICES), 0, st, a);
    if (e != cudaSuccess) return fail(RWKV_E_CUDA, "param_join_kernel: %s", cudaGetErrorString(e));
    return ok();
}

}  // namespace rwkv
