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

// 64 columns per block, two to a lane, SLICES interleaved slices of the partials.
// Launched to start beside the row kernel's end (pdl_wait).
template <int SLICES, int LOADS>
__global__ void __launch_bounds__(32 * SLICES) param_join_kernel(const ParamJoin a) {
    __shared__ float2 red[SLICES][32];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 64 + 2 * lane;
    pdl_wait();
    float2 s = make_float2(0.f, 0.f);
    if (c < a.width) {
        // LOADS at a time in flight, also of the last few (a loop whose last ones follow one
        // another: 8.3 instead of 4.8 us for 236 partials of 7680 columns; a column to a lane
        // and twice the blocks: 1 us more for 444 of 5120)
        for (int b0 = slice; b0 < a.blocks; b0 += LOADS * SLICES) {
            float2 v[LOADS];
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int b = b0 + i * SLICES;
                v[i] = b < a.blocks ? *reinterpret_cast<const float2*>(a.part + b * a.width + c) : make_float2(0.f, 0.f);
            }
#pragma unroll
            for (int i = 0; i < LOADS; i++) s.x += v[i].x, s.y += v[i].y;
        }
    }
    red[slice][lane] = s;
    __syncthreads();
    const int64_t o = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x < 64 && o < a.width) {
        const float* r = &red[0][0].x + threadIdx.x;
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < SLICES; i++) t += r[64 * i];
        const int k = a.width == a.D ? 0 : (int)(o / a.D);
        store_param(a.out[k], a.dtype, o - k * a.D, t);
    }
}

inline int launch_param_join(const ParamJoin& a, cudaStream_t st) {
    const dim3 grid((unsigned)((a.width + 63) / 64));
    // as many threads and loads as reach all partials in one or two rounds: 444 of 5120
    // columns by 8 loads 0.8 us more, 236 of 7680 0.8 more, 118 of 15360 by 16 0.8 more
    const cudaError_t e = a.blocks > 256   ? launch_pdl(param_join_kernel<32, 16>, grid, dim3(1024), 0, st, a)
                          : a.blocks > 128 ? launch_pdl(param_join_kernel<16, 16>, grid, dim3(512), 0, st, a)
                                           : launch_pdl(param_join_kernel<16, 8>, grid, dim3(512), 0, st, a);
    if (e != cudaSuccess) return fail(RWKV_E_CUDA, "param_join_kernel: %s", cudaGetErrorString(e));
    return ok();
}

}  // namespace rwkv
