// The projection forward for a few rows (decode): y = act(x W^T + bias) + residual
// for up to 16 rows of x, bound by streaming W from HBM once.
//
// A block takes 16 outputs over all of K (32, a checkpoint group, where a
// checkpoint is kept; an output's sum is the same either way).  Its warps take 32-wide pieces of K in
// turn and multiply on mma.sync m16n8k16 (16 weight rows x 8 activation rows): at
// one fragment per 16-byte load the tensor pipe is far from a limit, and a row
// count below 8 costs nothing extra.  Lane (g, t) = (lane / 4, lane % 4) loads 8
// consecutive k of weight rows g and g + 8 and of activation row g, and the two
// MMAs of the piece take words (0, 1) and (2, 3) of all three: the same permutation
// of k on both sides, so that every load is 16 bytes and no shuffle is needed.
// GP_U pieces are in flight per warp; the launch bound of one block per SM is what
// makes the compiler keep them in registers (without it 2048 outputs of 8192 take
// 13.8 us).  Measured, weights from HBM, in a graph, 1 row: 8192 outputs of 2048
// 7.8 us (4.3 TB/s), 2048 of 8192 8.8 us, 65536 of 2048 41 us (6.5 TB/s); the tile
// kernel takes 19 us for the first.  The warps' sums meet in shared memory and
// are added in warp order (deterministic).
#pragma once

#include "gemm_proj.cuh"

namespace rwkv {

constexpr int GP_ROWS = 16;  // rows of x at most
constexpr int GP_IN = 8 * PJ_CHAIN;  // terms at most: PJ_CHAIN for each of 8 warps
constexpr int GP_U = 4;

struct GemvProjArgs {
    const void* x;
    const void* w;
    void* y;
    ProjEpi e;
    int rows, OUT, IN;
};

template <bool BF16>
__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: groups of 8 activation rows; NW warps; MT groups of 16 outputs.
template <bool BF16, int NT, int NW, int MT, bool FAST>
__global__ void __launch_bounds__(NW * 32, 1) gemv_proj_kernel(const GemvProjArgs a) {
    constexpr int O = 16 * MT, U = GP_U;
    __shared__ float red[NW][8 * NT][O + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int o0 = blockIdx.x * O;
    const uint16_t* w = static_cast<const uint16_t*>(a.w) + (int64_t)(o0 + g) * a.IN;
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + (int64_t)g * a.IN;
    float c[MT][NT][4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int k0 = warp * 32; k0 < a.IN; k0 += NW * 32 * U) {
        uint4 f[U][MT][2], fx[U][NT];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + u * NW * 32 + 8 * t;
            const bool in = k < a.IN;
#pragma unroll
            for (int m = 0; m < 2 * MT; m++)
                f[u][m / 2][m % 2] = in && o0 + g + 8 * m < a.OUT
                                         ? __ldcs(reinterpret_cast<const uint4*>(w + 8 * m * (int64_t)a.IN + k))
                                         : zero;
#pragma unroll
            for (int n = 0; n < NT; n++)
                fx[u][n] = in && g + 8 * n < a.rows ? *reinterpret_cast<const uint4*>(x + 8 * n * (int64_t)a.IN + k) : zero;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint4 p = f[u][m][0], q = f[u][m][1];
                    mma_16816<BF16>(c[m][n], p.x, q.x, p.y, q.y, fx[u][n].x, fx[u][n].y);
                    mma_16816<BF16>(c[m][n], p.z, q.z, p.w, q.w, fx[u][n].z, fx[u][n].w);
                }
    }
    // lane (g, t) holds outputs g and g + 8 of rows 2t and 2t + 1
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) red[warp][8 * n + 2 * t + (i & 1)][16 * m + g + 8 * (i >> 1)] = c[m][n][i];
    __syncthreads();
    for (int i = threadIdx.x; i < O * a.rows; i += NW * 32) {
        const int row = i / O, o = i % O, col = o0 + o;
        float z = 0.f;
#pragma unroll
        for (int k = 0; k < NW; k++) z += red[k][row][o];
        if (a.e.bias && col < a.OUT) z += load_param(a.e.bias, a.e.bias_dtype, col);
        if constexpr (MT == 2) {  // a warp holds one group of one row
            const uint32_t e = ck_exponent(__reduce_max_sync(0xffffffffu, col < a.OUT ? abs_bits(z) : 0u));
            if (col < a.OUT) a.e.codes[(int64_t)row * a.OUT + col] = (int8_t)ck_code(z, ck_inv_scale(e));
            if (o == 0) a.e.exps[row * (int64_t)((a.OUT + CK_GROUP - 1) / CK_GROUP) + blockIdx.x] = (uint8_t)e;
        }
        if (col >= a.OUT) continue;
        const int64_t at = (int64_t)row * a.OUT + col;
        auto store = [&](void* p, float v) {
            if (BF16) static_cast<__nv_bfloat16*>(p)[at] = from_f<__nv_bfloat16>(v);
            else static_cast<__half*>(p)[at] = from_f<__half>(v);
        };
        if (a.e.z) store(a.e.z, z);
        float y = z;
        with_act(a.e.act, [&]<int ACT>() { y = act_t<ACT, FAST>(z); });
        if (a.e.add) y += load_param(a.e.add, a.e.out_f32 ? RWKV_F32 : BF16 ? RWKV_BF16 : RWKV_F16, at);
        if (a.e.out_f32) static_cast<float*>(a.y)[at] = y;
        else store(a.y, y);
    }
}

// 8 warps where that already gives an SM two blocks, else 16.
template <bool BF16, int NT, int MT, bool FAST>
inline void launch_gemv_proj_t(const GemvProjArgs& a, int sm_count, cudaStream_t st) {
    const int grid = ceil_div(a.OUT, 16 * MT);
    if (ceil_div(a.OUT, 16) < 2 * sm_count) gemv_proj_kernel<BF16, NT, 16, MT, FAST><<<grid, 512, 0, st>>>(a);
    else gemv_proj_kernel<BF16, NT, 8, MT, FAST><<<grid, 256, 0, st>>>(a);
}
template <bool BF16, bool FAST>
inline void launch_gemv_proj_f(const GemvProjArgs& a, int sm_count, cudaStream_t st) {
    const bool two = a.rows > 8, ck = a.e.codes != nullptr;
    if (two && ck) launch_gemv_proj_t<BF16, 2, 2, FAST>(a, sm_count, st);
    else if (two) launch_gemv_proj_t<BF16, 2, 1, FAST>(a, sm_count, st);
    else if (ck) launch_gemv_proj_t<BF16, 1, 2, FAST>(a, sm_count, st);
    else launch_gemv_proj_t<BF16, 1, 1, FAST>(a, sm_count, st);
}
inline cudaError_t launch_gemv_proj(const GemvProjArgs& a, int sm_count, cudaStream_t st) {
    if (a.e.bf16 && a.e.fast()) launch_gemv_proj_f<true, true>(a, sm_count, st);
    else if (a.e.bf16) launch_gemv_proj_f<true, false>(a, sm_count, st);
    else if (a.e.fast()) launch_gemv_proj_f<false, true>(a, sm_count, st);
    else launch_gemv_proj_f<false, false>(a, sm_count, st);
    return cudaGetLastError();
}

}  // namespace rwkv
