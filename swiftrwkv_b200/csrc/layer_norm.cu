// Layer norm over the last dimension, forward and backward, with the 8-bit
// checkpoint of its input written or read in the same pass.
//
//   forward   y = (x - mean) rstd w + b; mean and the centred sum of squares in
//             fp32, two passes over the row
//   backward  h = (x - mean) rstd, g = dy w:
//             dx = rstd (g - mean(g) - h mean(g h)) [+ dres]
//             dw = sum_n dy h, db = sum_n dy
//
// Both are bound by HBM: each element is read and written once, and a row stays
// in registers between its passes.  Rows are read in 16-byte vectors; the raw
// vectors are kept (half the registers of fp32 for 16-bit types) and unpacked
// in each pass.
#include "ckpt8.cuh"

namespace rwkv {
namespace {

// ------------------------------------------------------------------- forward

struct LnFwdArgs {
    const void* x;
    const void* w;
    const void* b;
    void* y;
    float* mean;
    float* rstd;
    int8_t* codes;
    uint8_t* exps;
    int wdtype, rows, D, G;
    float eps;
};

// Sum over the TPR threads of a row: a warp, or the whole block.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = warp_sum(v);
    if constexpr (TPR > 32) {
        const int w = threadIdx.x >> 5;
        __syncthreads();  // the previous sum's readers are done
        if ((threadIdx.x & 31) == 0) red[w] = v;
        __syncthreads();
        v = (threadIdx.x & 31) < TPR / 32 ? red[threadIdx.x & 31] : 0.f;
        v = warp_sum(v);
    }
    return v;
}

// TPR threads per row (32: a warp, several rows per block; else one block per
// row), at most NV vectors per thread: vector j of thread t is t + j TPR.
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) ln_fwd_kernel(const LnFwdArgs a) {
    constexpr int VE = Vec16<T>::N;
    __shared__ float red[32];
    const int t = threadIdx.x & (TPR - 1);
    const int64_t row = TPR == 32 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;  // whole rows of threads leave
    const int nvec = a.D / VE;
    const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.D);
    uint4 raw[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int v = t + j * TPR;
        raw[j] = v < nvec ? xr[v] : make_uint4(0, 0, 0, 0);
    }
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        float f[VE];
        Vec16<T>::unpack(raw[j], f);
#pragma unroll
        for (int k = 0; k < VE; k++) s += f[k];
    }
    const float mean = row_sum<TPR>(s, red) / (float)a.D;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        float f[VE];
        Vec16<T>::unpack(raw[j], f);
        if (t + j * TPR < nvec) {
#pragma unroll
            for (int k = 0; k < VE; k++) {
                const float d = f[k] - mean;
                q = fmaf(d, d, q);
            }
        }
    }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(q, red) / (float)a.D + a.eps);
    if (t == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    uint4* yr = reinterpret_cast<uint4*>(static_cast<T*>(a.y) + row * a.D);
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int v = t + j * TPR;
        float f[VE];
        Vec16<T>::unpack(raw[j], f);
        if (a.codes) {
            // a group of 32 channels is 32 / VE neighbouring threads
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < VE; k++) top = max(top, abs_bits(f[k]));
#pragma unroll
            for (int o = 1; o < CK_GROUP / VE; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const uint32_t e = ck_exponent(top);
            const float inv = ck_inv_scale(e);
            if (v < nvec) {
                uint32_t* c = reinterpret_cast<uint32_t*>(a.codes + row * a.D + (int64_t)v * VE);
#pragma unroll
                for (int k = 0; k < VE; k += 4) c[k / 4] = ck_pack4(f[k], f[k + 1], f[k + 2], f[k + 3], inv);
                if (v % (CK_GROUP / VE) == 0) a.exps[row * a.G + v / (CK_GROUP / VE)] = (uint8_t)e;
            }
        }
        if (v < nvec) {
#pragma unroll
            for (int k = 0; k < VE; k++)
                f[k] = fmaf((f[k] - mean) * rstd, load_param(a.w, a.wdtype, v * VE + k),
                            load_param(a.b, a.wdtype, v * VE + k));
            yr[v] = Vec16<T>::pack(f);
        }
    }
}

// Any length and alignment: a block per row, single elements, the row re-read
// (from L1 / L2) in each pass.  y may be x: every element is read for the last
// time by the thread that writes it, after the sums.
template <typename T>
__global__ void __launch_bounds__(256) ln_fwd_any_kernel(const LnFwdArgs a) {
    __shared__ float red[32];
    const int64_t row = blockIdx.x;
    const T* xr = static_cast<const T*>(a.x) + row * a.D;
    T* yr = static_cast<T*>(a.y) + row * a.D;
    float s = 0.f;
    for (int i = threadIdx.x; i < a.D; i += 256) s += to_f<T>(xr[i]);
    const float mean = row_sum<256>(s, red) / (float)a.D;
    float q = 0.f;
    for (int i = threadIdx.x; i < a.D; i += 256) {
        const float d = to_f<T>(xr[i]) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(row_sum<256>(q, red) / (float)a.D + a.eps);
    if (threadIdx.x == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    // whole warps: a warp's 32 elements are one group
    for (int i0 = 0; i0 < a.D; i0 += 256) {
        const int i = i0 + threadIdx.x;
        const float x = i < a.D ? to_f<T>(xr[i]) : 0.f;
        if (a.codes) {
            const uint32_t e = ck_exponent(__reduce_max_sync(0xffffffffu, abs_bits(x)));
            if (i < a.D) {
                a.codes[row * a.D + i] = (int8_t)ck_code(x, ck_inv_scale(e));
                if (i % CK_GROUP == 0) a.exps[row * a.G + i / CK_GROUP] = (uint8_t)e;
            }
        }
        if (i < a.D)
            yr[i] = from_f<T>(fmaf((x - mean) * rstd, load_param(a.w, a.wdtype, i), load_param(a.b, a.wdtype, i)));
    }
}

template <typename T>
int launch_ln_fwd(const LnFwdArgs& a, bool vec, cudaStream_t st) {
    const int nvec = a.D / Vec16<T>::N;
    if (vec && nvec <= 32 * 16) {
        const int grid = ceil_div(a.rows, 4);
        if (nvec <= 32 * 4) ln_fwd_kernel<T, 32, 4><<<grid, 128, 0, st>>>(a);
        else if (nvec <= 32 * 8) ln_fwd_kernel<T, 32, 8><<<grid, 128, 0, st>>>(a);
        else ln_fwd_kernel<T, 32, 16><<<grid, 128, 0, st>>>(a);
    } else if (vec && nvec <= 512 * 8) {
        ln_fwd_kernel<T, 512, 8><<<a.rows, 512, 0, st>>>(a);
    } else {
        ln_fwd_any_kernel<T><<<a.rows, 256, 0, st>>>(a);
    }
    return check_launch("ln_fwd_kernel");
}

// ------------------------------------------------------------------ backward

struct LnBwdArgs {
    const void* dy;
    const void* x;
    const int8_t* codes;
    const uint8_t* exps;
    const void* w;
    const float* mean;
    const float* rstd;
    const void* dres;
    void* dx;
    float* part;  // [blocks][2][D] sums of dy h and dy over the block's rows, or NULL
    int wdtype, rows, D, G;
};

// A block takes R rows at a time, blockIdx.x R + i, with stride gridDim.x R;
// thread t owns the vectors t + j blockDim.x of every row, so its sums over
// rows of dy h and dy stay in registers until the end.  One barrier per R rows
// (the two row sums of R rows in one exchange, buffers alternating).
template <typename T, bool CK, int NV, int R>
__global__ void __launch_bounds__(512) ln_bwd_kernel(const LnBwdArgs a) {
    constexpr int VE = Vec16<T>::N;
    __shared__ float2 red[2][R][16];
    const int t = threadIdx.x, nt = blockDim.x, warp = t >> 5, lane = t & 31, nw = nt >> 5;
    const int nvec = a.D / VE;
    const float inv_d = 1.f / (float)a.D;
    float w[NV][VE], sw[NV][VE], sb[NV][VE];
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int k = 0; k < VE; k++) {
            const int v = t + j * nt;
            w[j][k] = v < nvec ? load_param(a.w, a.wdtype, v * VE + k) : 0.f;
            sw[j][k] = sb[j][k] = 0.f;
        }
    int buf = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < a.rows; r0 += (int64_t)gridDim.x * R, buf ^= 1) {
        uint4 rdy[R][NV], rx[R][NV];
        float mean[R], rstd[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int64_t row = r0 + r;
            const bool ok = row < a.rows;
            mean[r] = ok ? a.mean[row] : 0.f;
            rstd[r] = ok ? a.rstd[row] : 0.f;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int v = t + j * nt;
                rdy[r][j] = rx[r][j] = make_uint4(0, 0, 0, 0);
                if (ok && v < nvec) {
                    const int64_t at = row * a.D + (int64_t)v * VE;
                    rdy[r][j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.dy) + at);
                    if constexpr (CK) {
                        const uint32_t* c = reinterpret_cast<const uint32_t*>(a.codes + at);
                        rx[r][j].x = c[0];
                        if constexpr (VE == 8) rx[r][j].y = c[1];
                        rx[r][j].z = a.exps[row * a.G + v / (CK_GROUP / VE)];
                    } else {
                        rx[r][j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + at);
                    }
                }
            }
        }
        // h of a vector (0 beyond the row's end)
        auto normed = [&](int r, int j, float* h) {
            if constexpr (CK) {
                const float s = ck_scale(rx[r][j].z);
                ck_unpack4(rx[r][j].x, s, h);
                if constexpr (VE == 8) ck_unpack4(rx[r][j].y, s, h + 4);
            } else {
                Vec16<T>::unpack(rx[r][j], h);
            }
#pragma unroll
            for (int k = 0; k < VE; k++) h[k] = (h[k] - mean[r]) * rstd[r];
        };
#pragma unroll
        for (int r = 0; r < R; r++) {
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                float dy[VE], h[VE];
                Vec16<T>::unpack(rdy[r][j], dy);
                normed(r, j, h);
#pragma unroll
                for (int k = 0; k < VE; k++) {
                    const float g = dy[k] * w[j][k];
                    s1 += g;
                    s2 = fmaf(g, h[k], s2);
                    sw[j][k] = fmaf(dy[k], h[k], sw[j][k]);
                    sb[j][k] += dy[k];
                }
            }
            s1 = warp_sum(s1);
            s2 = warp_sum(s2);
            if (lane == 0) red[buf][r][warp] = make_float2(s1, s2);
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int64_t row = r0 + r;
            float2 p = lane < nw ? red[buf][r][lane] : make_float2(0.f, 0.f);
            const float m1 = warp_sum(p.x) * inv_d, m2 = warp_sum(p.y) * inv_d;
            if (row >= a.rows) continue;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int v = t + j * nt;
                if (v >= nvec) continue;
                float dy[VE], h[VE], o[VE];
                Vec16<T>::unpack(rdy[r][j], dy);
                normed(r, j, h);
                const int64_t at = row * a.D + (int64_t)v * VE;
                if (a.dres) Vec16<T>::unpack(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.dres) + at), o);
#pragma unroll
                for (int k = 0; k < VE; k++) {
                    const float d = rstd[r] * (dy[k] * w[j][k] - m1 - h[k] * m2);
                    o[k] = a.dres ? o[k] + d : d;
                }
                *reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + at) = Vec16<T>::pack(o);
            }
        }
    }
    if (!a.part) return;
    float* p = a.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int v = t + j * nt;
        if (v >= nvec) continue;
#pragma unroll
        for (int k = 0; k < VE; k += 4) {
            *reinterpret_cast<float4*>(p + v * VE + k) = make_float4(sw[j][k], sw[j][k + 1], sw[j][k + 2], sw[j][k + 3]);
            *reinterpret_cast<float4*>(p + a.D + v * VE + k) =
                make_float4(sb[j][k], sb[j][k + 1], sb[j][k + 2], sb[j][k + 3]);
        }
    }
}

template <typename T, bool CK>
__device__ __forceinline__ float bwd_x(const LnBwdArgs& a, int64_t row, int i) {
    if constexpr (CK) return (float)a.codes[row * a.D + i] * ck_scale(a.exps[row * a.G + i / CK_GROUP]);
    else return to_f<T>(static_cast<const T*>(a.x)[row * a.D + i]);
}

// Any length and alignment.  dx: a block per row, single elements.  dx may be
// dy, so the column sums (ln_bwd_cols_any_kernel) are launched first.
template <typename T, bool CK>
__global__ void __launch_bounds__(256) ln_bwd_any_kernel(const LnBwdArgs a) {
    __shared__ float red[32];
    const int64_t row = blockIdx.x;
    const float mean = a.mean[row], rstd = a.rstd[row];
    const T* dyr = static_cast<const T*>(a.dy) + row * a.D;
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < a.D; i += 256) {
        const float g = to_f<T>(dyr[i]) * load_param(a.w, a.wdtype, i);
        s1 += g;
        s2 = fmaf(g, (bwd_x<T, CK>(a, row, i) - mean) * rstd, s2);
    }
    const float m1 = row_sum<256>(s1, red) / (float)a.D, m2 = row_sum<256>(s2, red) / (float)a.D;
    for (int i = threadIdx.x; i < a.D; i += 256) {
        const float g = to_f<T>(dyr[i]) * load_param(a.w, a.wdtype, i);
        float d = rstd * (g - m1 - (bwd_x<T, CK>(a, row, i) - mean) * rstd * m2);
        if (a.dres) d += to_f<T>(static_cast<const T*>(a.dres)[row * a.D + i]);
        static_cast<T*>(a.dx)[row * a.D + i] = from_f<T>(d);
    }
}
// Column sums over the rows blockIdx.y, blockIdx.y + gridDim.y, ...
template <typename T, bool CK>
__global__ void __launch_bounds__(256) ln_bwd_cols_any_kernel(const LnBwdArgs a) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.D) return;
    float sw = 0.f, sb = 0.f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float dy = to_f<T>(static_cast<const T*>(a.dy)[row * a.D + i]);
        sw = fmaf(dy, (bwd_x<T, CK>(a, row, i) - a.mean[row]) * a.rstd[row], sw);
        sb += dy;
    }
    float* p = a.part + (int64_t)blockIdx.y * 2 * a.D;
    p[i] = sw;
    p[a.D + i] = sb;
}

// out[c] = sum over the blocks of part[block][c], c < 2D (dweight, dbias): 32
// columns per block, 8 interleaved slices of the partials, in a fixed order.
__global__ void __launch_bounds__(256) ln_bwd_params_kernel(const float* __restrict__ part, int blocks, int D,
                                                            void* dw, void* db, int wdtype) {
    __shared__ float red[8][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + col, width = 2 * (int64_t)D;
    float s = 0.f;
    if (c < width)
        for (int b = slice; b < blocks; b += 8) s += part[b * width + c];
    red[slice][col] = s;
    __syncthreads();
    if (slice == 0 && c < width) {
#pragma unroll
        for (int k = 1; k < 8; k++) s += red[k][col];
        if (c < D) store_param(dw, wdtype, c, s);
        else store_param(db, wdtype, c - D, s);
    }
}

constexpr int LN_BWD_BLOCKS = 148 * 2;  // at most: two resident blocks per SM

// Blocks of the row kernel and rows it takes at a time, from the vectors of a
// row (16-byte ones; the 16-bit types have half as many).
inline int bwd_rows_at_once(int nvec) { return nvec <= 512 ? 4 : nvec <= 1024 ? 2 : 1; }
inline int bwd_blocks(int rows, int R) { return std::min(ceil_div(rows, R), LN_BWD_BLOCKS); }

template <typename T, bool CK>
int launch_ln_bwd(LnBwdArgs a, bool vec, void* dw, void* db, cudaStream_t st) {
    const int nvec = a.D / Vec16<T>::N;
    int blocks;
    if (vec && nvec <= 2048) {
        const int NV = nvec <= 512 ? 1 : nvec <= 1024 ? 2 : 4;
        const int nt = ceil_div(ceil_div(nvec, NV), 32) * 32;
        blocks = bwd_blocks(a.rows, bwd_rows_at_once(nvec));
        if (NV == 1) ln_bwd_kernel<T, CK, 1, 4><<<blocks, nt, 0, st>>>(a);
        else if (NV == 2) ln_bwd_kernel<T, CK, 2, 2><<<blocks, nt, 0, st>>>(a);
        else ln_bwd_kernel<T, CK, 4, 1><<<blocks, nt, 0, st>>>(a);
    } else {
        blocks = std::min(a.rows, 64);
        if (a.part) {
            ln_bwd_cols_any_kernel<T, CK><<<dim3(ceil_div(a.D, 256), blocks), 256, 0, st>>>(a);
            if (int rc = check_launch("ln_bwd_cols_kernel")) return rc;
        }
        ln_bwd_any_kernel<T, CK><<<a.rows, 256, 0, st>>>(a);
    }
    if (int rc = check_launch("ln_bwd_kernel")) return rc;
    if (!a.part) return ok();
    ln_bwd_params_kernel<<<ceil_div(2 * (int64_t)a.D, 32), 256, 0, st>>>(a.part, blocks, a.D, dw, db, a.wdtype);
    return check_launch("ln_bwd_params_kernel");
}

bool al(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
uintptr_t elem(int dtype) { return dtype == RWKV_F32 ? 4 : 2; }

int check_rows(int rows, int D, const char* fn) {
    RWKV_REQUIRE(rows >= 1 && D >= 1 && D <= 1 << 30, RWKV_E_SHAPE, "%s: rows=%d D=%d (rows >= 1, D in 1..2^30)", fn,
                 rows, D);
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

using namespace rwkv;

extern "C" int rwkv_layer_norm_forward(int dtype, const void* x, int wdtype, const void* weight, const void* bias,
                                       float eps, void* y, float* mean, float* rstd, int8_t* codes, uint8_t* exps,
                                       int rows, int D, rwkv_stream_t stream) {
    const char* fn = "rwkv_layer_norm_forward";
    RWKV_REQUIRE(valid_dtype(dtype) && valid_dtype(wdtype), RWKV_E_DTYPE, "%s: dtypes x=%d w=%d", fn, dtype, wdtype);
    RWKV_REQUIRE(x && weight && bias && y, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(!mean == !rstd, RWKV_E_NULL, "%s: give both mean and rstd or neither", fn);
    RWKV_REQUIRE(!codes == !exps, RWKV_E_NULL, "%s: give both codes and exps or neither", fn);
    if (int rc = check_rows(rows, D, fn)) return rc;
    RWKV_REQUIRE(eps >= 0.f, RWKV_E_SHAPE, "%s: eps=%g must be >= 0", fn, eps);
    RWKV_REQUIRE(al(x, elem(dtype)) && al(y, elem(dtype)) && al(weight, elem(wdtype)) && al(bias, elem(wdtype)) &&
                     al(mean, 4) && al(rstd, 4),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not aligned to its element type", fn);
    const LnFwdArgs a{x, weight, bias, y, mean, rstd, codes, exps, wdtype, rows, D, ceil_div(D, CK_GROUP), eps};
    const bool vec = D % 8 == 0 && al(x, 16) && al(y, 16) && al(codes, 8);
    return dispatch_dtype(dtype, [&]<typename T>() { return launch_ln_fwd<T>(a, vec, (cudaStream_t)stream); });
}

extern "C" int64_t rwkv_layer_norm_backward_workspace_size(int rows, int D) {
    if (rows < 1 || D < 1) return 0;
    return (int64_t)std::min(rows, LN_BWD_BLOCKS) * 2 * D * (int64_t)sizeof(float);
}

extern "C" int rwkv_layer_norm_backward(int dtype, const void* dy, const void* x, const int8_t* codes,
                                        const uint8_t* exps, int wdtype, const void* weight, const float* mean,
                                        const float* rstd, const void* dres, void* dx, void* dweight, void* dbias,
                                        int rows, int D, void* workspace, int64_t workspace_bytes,
                                        rwkv_stream_t stream) {
    const char* fn = "rwkv_layer_norm_backward";
    RWKV_REQUIRE(valid_dtype(dtype) && valid_dtype(wdtype), RWKV_E_DTYPE, "%s: dtypes x=%d w=%d", fn, dtype, wdtype);
    RWKV_REQUIRE(dy && weight && mean && rstd && dx, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(x ? !codes && !exps : codes && exps, RWKV_E_NULL, "%s: give either x or codes and exps", fn);
    RWKV_REQUIRE(!dweight == !dbias, RWKV_E_NULL, "%s: give both dweight and dbias or neither", fn);
    if (int rc = check_rows(rows, D, fn)) return rc;
    RWKV_REQUIRE(al(dy, elem(dtype)) && al(x, elem(dtype)) && al(dres, elem(dtype)) && al(dx, elem(dtype)) &&
                     al(weight, elem(wdtype)) && al(dweight, elem(wdtype)) && al(dbias, elem(wdtype)) &&
                     al(mean, 4) && al(rstd, 4),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not aligned to its element type", fn);
    if (dweight) {
        const int64_t need = rwkv_layer_norm_backward_workspace_size(rows, D);
        RWKV_REQUIRE(workspace && workspace_bytes >= need, RWKV_E_WORKSPACE, "%s: workspace of %lld bytes, need %lld",
                     fn, (long long)workspace_bytes, (long long)need);
        RWKV_REQUIRE(al(workspace, 16), RWKV_E_UNSUPPORTED, "%s: workspace not 16-byte aligned", fn);
    }
    const LnBwdArgs a{dy,   x,  codes, exps, weight, mean, rstd, dres, dx, dweight ? static_cast<float*>(workspace) : nullptr,
                      wdtype, rows, D, ceil_div(D, CK_GROUP)};
    const bool vec = D % 8 == 0 && al(dy, 16) && al(x, 16) && al(codes, 8) && al(dres, 16) && al(dx, 16);
    return dispatch_dtype(dtype, [&]<typename T>() {
        return codes ? launch_ln_bwd<T, true>(a, vec, dweight, dbias, (cudaStream_t)stream)
                     : launch_ln_bwd<T, false>(a, vec, dweight, dbias, (cudaStream_t)stream);
    });
}
