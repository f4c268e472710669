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
// in registers between its passes.  Rows are read in 16-byte vectors.  The forward
// keeps short rows in fp32 and long ones as read (half the registers for 16-bit
// types), unpacked in each pass.
#include <algorithm>

#include "ckpt8.cuh"
#include "copy_async.cuh"
#include "resident.cuh"

namespace rwkv {
namespace {

constexpr int LN_STAGES = 3;

// Rows of any length in aligned vectors.  Row r starts r D mod VE elements into a
// 16-byte vector, so rows a multiple of VE apart start at the same place: a block
// whose rows are has its columns fixed to its threads.  A row's vectors are those
// that it touches; of the first `head` elements and of the last those from `tail` on
// belong to other rows.  They are read as zeros and never written (the tensor's end
// bounds the last vector, its 16-byte aligned start the first).
template <typename T>
__device__ __forceinline__ void drop_head(uint4& r, int head) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
    constexpr int E = sizeof(T) == 2 ? 2 : 1;  // elements per word
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (E * i + E <= head) w[i] = 0;
        else if (E == 2 && E * i < head) w[i] &= 0xffff0000u;
    }
    r = make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void drop_tail(uint4& r, int tail) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
    constexpr int E = sizeof(T) == 2 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (E * i >= tail) w[i] = 0;
        else if (E == 2 && E * i + 1 == tail) w[i] &= 0xffffu;
    }
    r = make_uint4(w[0], w[1], w[2], w[3]);
}
// elements lo .. hi of a vector at p
template <typename T>
__device__ __forceinline__ void store_part(T* p, const float* v, int lo, int hi) {
#pragma unroll
    for (int k = 0; k < Vec16<T>::N; k++)
        if (k >= lo && k < hi) p[k] = from_f<T>(v[k]);
}

// vectors that a row of D elements touches at most
template <typename T>
int most_vectors(int D) {
    return (int)(((int64_t)D + 2 * Vec16<T>::N - 2) / Vec16<T>::N);
}

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

// Sums over the TPR threads of a row (a warp, or the whole block) of R values.
template <int TPR, int R>
__device__ __forceinline__ void row_sums(float* v, float* red) {
#pragma unroll
    for (int r = 0; r < R; r++) v[r] = warp_sum(v[r]);
    if constexpr (TPR > 32) {
        const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
        __syncthreads();  // the previous sums' readers are done
#pragma unroll
        for (int r = 0; r < R; r++)
            if (lane == 0) red[r * 32 + w] = v[r];
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) {
            if constexpr (TPR == 64) {
                v[r] = red[r * 32] + red[r * 32 + 1];
            } else {
                v[r] = lane < TPR / 32 ? red[r * 32 + lane] : 0.f;
                v[r] = warp_sum(v[r]);
            }
        }
    }
}
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    row_sums<TPR, 1>(&v, red);
    return v;
}

// A block of TPR threads takes R rows, at most NV vectors of a row per thread:
// vector j of thread t is t + j TPR.  The R rows share the loads of weight and
// bias, which in fp32 are four times a bf16 row's own bytes from L1.  Up to 80
// elements per thread are held in fp32, more as read.  WF32: weight and bias in
// fp32 (no branch between their loads); CK: write the checkpoint.
template <typename T, int TPR, int NV, int R, bool WF32, bool CK>
__global__ void __launch_bounds__(TPR, 1) ln_fwd_kernel(const LnFwdArgs a) {
    constexpr int VE = Vec16<T>::N;
    constexpr bool F32 = R * NV * VE <= 80;
    __shared__ float red[32 * R];
    const int t = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * R;
    const int nvec = a.D / VE;
    const uint4* xr = static_cast<const uint4*>(a.x) + row0 * nvec + t;
    uint4 raw[R][NV];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < NV; j++)
            raw[r][j] = row0 + r < a.rows && t + j * TPR < nvec ? __ldcs(xr + (int64_t)r * nvec + j * TPR)
                                                               : make_uint4(0, 0, 0, 0);
    if constexpr (CK) {
        // a group of 32 channels is 32 / VE neighbouring threads
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int v = t + j * TPR;
                uint32_t top = top_bits<T>(raw[r][j]);
#pragma unroll
                for (int o = 1; o < CK_GROUP / VE; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                const uint32_t e = ck_exponent(top_f32<T>(top));
                const float inv = ck_inv_scale(e);
                if (row0 + r < a.rows && v < nvec) {
                    float f[VE];
                    Vec16<T>::unpack(raw[r][j], f);
                    int8_t* c = a.codes + (row0 + r) * a.D + (int64_t)v * VE;
                    if constexpr (VE == 8)
                        *reinterpret_cast<uint2*>(c) = make_uint2(ck_pack4(f[0], f[1], f[2], f[3], inv),
                                                                  ck_pack4(f[4], f[5], f[6], f[7], inv));
                    else
                        *reinterpret_cast<uint32_t*>(c) = ck_pack4(f[0], f[1], f[2], f[3], inv);
                    if (v % (CK_GROUP / VE) == 0) a.exps[(row0 + r) * a.G + v / (CK_GROUP / VE)] = (uint8_t)e;
                }
            }
    }
    float x[F32 ? R : 1][F32 ? NV : 1][VE];
    auto vec = [&](int r, int j) -> float* { return x[F32 ? r : 0][F32 ? j : 0]; };
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        mean[r] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float* f = vec(r, j);
            Vec16<T>::unpack(raw[r][j], f);
#pragma unroll
            for (int k = 0; k < VE; k++) mean[r] += f[k];
        }
    }
    row_sums<TPR, R>(mean, red);
#pragma unroll
    for (int r = 0; r < R; r++) {
        mean[r] /= (float)a.D;
        rstd[r] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float* f = vec(r, j);
            if constexpr (!F32) Vec16<T>::unpack(raw[r][j], f);
            if (t + j * TPR < nvec) {
#pragma unroll
                for (int k = 0; k < VE; k++) {
                    const float d = f[k] - mean[r];
                    rstd[r] = fmaf(d, d, rstd[r]);
                }
            }
        }
    }
    row_sums<TPR, R>(rstd, red);
#pragma unroll
    for (int r = 0; r < R; r++) {
        rstd[r] = 1.f / sqrtf(rstd[r] / (float)a.D + a.eps);
        if (t == 0 && a.mean && row0 + r < a.rows) {
            a.mean[row0 + r] = mean[r];
            a.rstd[row0 + r] = rstd[r];
        }
    }
    uint4* yr = static_cast<uint4*>(a.y) + row0 * nvec + t;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int v = t + j * TPR;
        if (v < nvec) {
            float w[VE], b[VE];
            load_params<VE>(a.w, WF32 ? RWKV_F32 : a.wdtype, v * VE, w);
            load_params<VE>(a.b, WF32 ? RWKV_F32 : a.wdtype, v * VE, b);
#pragma unroll
            for (int r = 0; r < R; r++) {
                float* f = vec(r, j);
                if constexpr (!F32) Vec16<T>::unpack(raw[r][j], f);
                float o[VE];
#pragma unroll
                for (int k = 0; k < VE; k++) o[k] = fmaf((f[k] - mean[r]) * rstd[r], w[k], b[k]);
                if (row0 + r < a.rows) __stcs(yr + (int64_t)r * nvec + j * TPR, Vec16<T>::pack(o));
            }
        }
    }
}

// Rows that need not start on a vector: a block walks rows a multiple of VE apart,
// so that its columns, and with them weight and bias, stay in registers; x runs
// LN_STAGES - 1 rows ahead in a ring private to each thread.  A group of a
// checkpoint ends inside a vector, so that the groups' largest |x| meet in shared
// memory.  16384 x 2411 bf16: 60 us (single elements 144), with checkpoint 110
// (190); bound by the step of a row (two barriers, two sums), whatever the number
// of resident blocks.
template <typename T, int NV, bool CK, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) ln_fwd_shift_kernel(const LnFwdArgs a) {
    constexpr int VE = Vec16<T>::N, MAXG = 512 * 3 * 8 / CK_GROUP + 8;
    extern __shared__ uint4 ring[];  // [stage][NV][thread]
    __shared__ float red[2][16];
    __shared__ uint32_t tops[CK ? 2 : 1][CK ? MAXG : 1];
    const int t = threadIdx.x, nt = blockDim.x, warp = t >> 5, lane = t & 31, nw = nt >> 5;
    const int head = (int)((int64_t)blockIdx.x * a.D % VE), nvec = (a.D + head + VE - 1) / VE;
    auto column = [&](int j) { return (t + j * nt) * VE - head; };  // of a vector's first element
    float w[NV][VE], b[NV][VE];
    bool has[NV];
    int tail[NV], lo[NV];  // its elements lo .. tail are the row's
#pragma unroll
    for (int j = 0; j < NV; j++) {
        has[j] = t + j * nt < nvec;
        tail[j] = min(VE, a.D - column(j));
        lo[j] = max(0, -column(j));
#pragma unroll
        for (int k = 0; k < VE; k++) {
            const bool in = has[j] && k >= lo[j] && k < tail[j];
            w[j][k] = in ? load_param(a.w, a.wdtype, column(j) + k) : 0.f;
            b[j][k] = in ? load_param(a.b, a.wdtype, column(j) + k) : 0.f;
        }
    }
    if constexpr (CK)
        for (int g = t; g < a.G; g += nt) tops[0][g] = tops[1][g] = 0;
    const int64_t vstep = (int64_t)gridDim.x * a.D / VE;  // in vectors
    int64_t at = (int64_t)blockIdx.x * a.D / VE, fat = at;
    const uint4* const x = static_cast<const uint4*>(a.x) + t;
    const int stage_n = NV * nt;
    auto fetch = [&](int64_t row, int base) {
        if (row < a.rows) {
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (has[j]) copy_async_n<16>(ring + base + j * nt, x + fat + j * nt, tail[j] * (int)sizeof(T));
        }
        copy_commit();
        fat += vstep;
    };
#pragma unroll
    for (int i = 0; i < LN_STAGES - 1; i++) fetch(blockIdx.x + (int64_t)i * gridDim.x, t + i * stage_n);
    if constexpr (CK) __syncthreads();
    // the block's sum of v over its threads, in every thread
    auto total = [&](float v, float* r) {
        v = warp_sum(v);
        if (lane == 0) r[warp] = v;
        __syncthreads();
        return warp_sum(lane < nw ? r[lane] : 0.f);
    };
    int cur = t, put = t + (LN_STAGES - 1) * stage_n, buf = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, at += vstep, buf ^= 1) {
        fetch(row + (int64_t)(LN_STAGES - 1) * gridDim.x, put);
        copy_wait<LN_STAGES - 1>();
        uint4 raw[NV];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            raw[j] = has[j] ? ring[cur + j * nt] : make_uint4(0, 0, 0, 0);
            if (j == 0 && t == 0) drop_head<T>(raw[j], head);
            float f[VE];
            Vec16<T>::unpack(raw[j], f);
#pragma unroll
            for (int k = 0; k < VE; k++) s += f[k];
            if (CK && has[j]) {
                const int c = max(column(j), 0), g = c / CK_GROUP, other = CK_GROUP - c % CK_GROUP + lo[j];
                uint4 first = raw[j];
                if (other < VE) {
                    uint4 second = raw[j];
                    drop_head<T>(second, other);
                    drop_tail<T>(first, other);
                    if (g + 1 < a.G) atomicMax(&tops[buf][g + 1], top_bits<T>(second));
                }
                atomicMax(&tops[buf][g], top_bits<T>(first));
            }
        }
        const float mean = total(s, red[0]) / (float)a.D;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float f[VE];
            Vec16<T>::unpack(raw[j], f);
#pragma unroll
            for (int k = 0; k < VE; k++) {
                const float d = has[j] && k >= lo[j] && k < tail[j] ? f[k] - mean : 0.f;
                q = fmaf(d, d, q);
            }
        }
        if constexpr (CK) {
            // the groups' exponents, and the codes
            for (int g = t; g < a.G; g += nt) {
                a.exps[row * a.G + g] = (uint8_t)ck_exponent(top_f32<T>(tops[buf][g]));
                tops[buf ^ 1][g] = 0;  // read before this row's first barrier, added to after its second
            }
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (!has[j]) continue;
                const int c = max(column(j), 0), g = c / CK_GROUP, other = CK_GROUP - c % CK_GROUP + lo[j];
                const float i0 = ck_inv_scale(ck_exponent(top_f32<T>(tops[buf][g])));
                const float i1 = ck_inv_scale(ck_exponent(top_f32<T>(tops[buf][min(g + 1, a.G - 1)])));
                float f[VE];
                Vec16<T>::unpack(raw[j], f);
                uint32_t q8[VE / 4];
#pragma unroll
                for (int i = 0; i < VE / 4; i++) {  // codes of either group, without a branch (a branch: 5 us more)
                    const uint32_t p0 = ck_pack4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3], i0);
                    const uint32_t p1 = ck_pack4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3], i1);
                    const int n = min(max(other - 4 * i, 0), 4);
                    const uint32_t m = n == 4 ? ~0u : (1u << 8 * n) - 1;
                    q8[i] = (p0 & m) | (p1 & ~m);
                }
                int8_t* out = a.codes + VE * (at + t + j * nt);
                if (lo[j] > 0 || tail[j] < VE) {
#pragma unroll
                    for (int k = 0; k < VE; k++)
                        if (k >= lo[j] && k < tail[j]) out[k] = (int8_t)(q8[k / 4] >> 8 * (k % 4));
                } else if constexpr (VE == 8) {
                    *reinterpret_cast<uint2*>(out) = make_uint2(q8[0], q8[VE / 4 - 1]);
                } else {
                    *reinterpret_cast<uint32_t*>(out) = q8[0];
                }
            }
        }
        const float rstd = 1.f / sqrtf(total(q, red[1]) / (float)a.D + a.eps);
        if (t == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (!has[j]) continue;
            float o[VE];
            Vec16<T>::unpack(raw[j], o);
#pragma unroll
            for (int k = 0; k < VE; k++) o[k] = fmaf((o[k] - mean) * rstd, w[j][k], b[j][k]);
            uint4* out = static_cast<uint4*>(a.y) + at + t + j * nt;
            if (lo[j] > 0 || tail[j] < VE) store_part<T>(reinterpret_cast<T*>(out), o, lo[j], tail[j]);
            else __stcs(out, Vec16<T>::pack(o));
        }
        put = cur;
        cur = cur == t + (LN_STAGES - 1) * stage_n ? t : cur + stage_n;
    }
    copy_wait<0>();
}

// Tensors off a 16-byte boundary, short odd rows, and rows of more vectors than the
// kernels above take: single elements, element j of thread t is t + j TPR (a warp's 32 elements
// are a checkpoint group), at most NE per thread, in registers.
template <typename T, int TPR, int NE>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR, 1) ln_fwd_any_kernel(const LnFwdArgs a) {
    __shared__ float red[32];
    const int t = threadIdx.x & (TPR - 1);
    const int64_t row = TPR == 32 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    const T* xr = static_cast<const T*>(a.x) + row * a.D;
    T* yr = static_cast<T*>(a.y) + row * a.D;
    float x[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) x[j] = t + j * TPR < a.D ? to_f<T>(xr[t + j * TPR]) : 0.f;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NE; j++) s += x[j];
    const float mean = row_sum<TPR>(s, red) / (float)a.D;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NE; j++) {
        const float d = t + j * TPR < a.D ? x[j] - mean : 0.f;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(q, red) / (float)a.D + a.eps);
    if (t == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NE; j++) {
        const int i = t + j * TPR;
        if (a.codes) {
            const uint32_t e = ck_exponent(__reduce_max_sync(0xffffffffu, abs_bits(x[j])));
            if (i < a.D) {
                a.codes[row * a.D + i] = (int8_t)ck_code(x[j], ck_inv_scale(e));
                if (i % CK_GROUP == 0) a.exps[row * a.G + i / CK_GROUP] = (uint8_t)e;
            }
        }
        if (i < a.D)
            yr[i] = from_f<T>(fmaf((x[j] - mean) * rstd, load_param(a.w, a.wdtype, i), load_param(a.b, a.wdtype, i)));
    }
}

// Any length: a block per row, the row re-read (from L1 / L2) in each pass.  y
// may be x: every element is read for the last time by the thread that writes
// it, after the sums.
template <typename T>
__global__ void __launch_bounds__(256) ln_fwd_long_kernel(const LnFwdArgs a) {
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

template <typename T, int TPR, int NV, int R, bool CK>
void launch_ln_fwd_t(const LnFwdArgs& a, cudaStream_t st) {
    const int grid = ceil_div(a.rows, R);
    if (a.wdtype == RWKV_F32) ln_fwd_kernel<T, TPR, NV, R, true, CK><<<grid, TPR, 0, st>>>(a);
    else ln_fwd_kernel<T, TPR, NV, R, false, CK><<<grid, TPR, 0, st>>>(a);
}

template <typename T, int NV, bool CK, int MAXT, int MINB>
cudaError_t launch_ln_fwd_shift(const LnFwdArgs& a, cudaStream_t st) {
    auto kern = ln_fwd_shift_kernel<T, NV, CK, MAXT, MINB>;
    constexpr int VE = Vec16<T>::N, PER_T = LN_STAGES * NV * 16;  // shared memory of a thread
    const int nt = ceil_div(ceil_div(most_vectors<T>(a.D), NV), 32) * 32;
    const int smem = PER_T * nt;
    static ResidentBlocks resident;
    int per_sm;
    const cudaError_t e = resident.get(kern, nt, smem, PER_T * MAXT, &per_sm);
    if (e != cudaSuccess) return e;
    kern<<<std::min(a.rows, 148 * per_sm / VE * VE), nt, smem, st>>>(a);
    return cudaGetLastError();
}

// whole: rows of whole vectors, with weight and bias on 16-byte boundaries
template <typename T, bool CK>
int launch_ln_fwd(const LnFwdArgs& a, bool vec, bool whole, cudaStream_t st) {
    const int nvec = a.D / Vec16<T>::N, touched = most_vectors<T>(a.D);
    // Threads and vectors per thread by length, two rows at a time (16384 x
    // 2560 bf16: 36 us against 40 us one by one, 16384 x 1024: 16 against 19);
    // with a checkpoint, above 256 vectors, one row (44 against 50 us), since the
    // packing hides the parameters' loads and two rows leave fewer threads.  A
    // row's sums run the same way with and without a checkpoint.
    constexpr int R = CK ? 1 : 2;
    // Lengths that are not whole vectors take vectors too, above 256 elements; below, a
    // warp per row of single elements is faster (16384 x 250 bf16: 9.5 against 14.7 us).
    if (vec && whole && nvec <= 512 * 8) {
        if (nvec <= 64) launch_ln_fwd_t<T, 64, 1, 2, CK>(a, st);
        else if (nvec <= 64 * 2) launch_ln_fwd_t<T, 64, 2, 2, CK>(a, st);
        else if (nvec <= 64 * 3) launch_ln_fwd_t<T, 64, 3, 2, CK>(a, st);
        else if (nvec <= 128 * 2) launch_ln_fwd_t<T, 128, 2, 2, CK>(a, st);
        else if (nvec <= 64 * 5) launch_ln_fwd_t<T, 64, 5, R, CK>(a, st);
        else if (nvec <= 256 * 2) launch_ln_fwd_t<T, 256, 2, R, CK>(a, st);
        else if (nvec <= 256 * 5) launch_ln_fwd_t<T, 256, 5, R, CK>(a, st);
        else launch_ln_fwd_t<T, 512, 8, 1, CK>(a, st);
    } else if (vec && !whole && a.D > 32 * 8 && touched <= 512 * 3) {
        const cudaError_t e = touched > 1024  ? launch_ln_fwd_shift<T, 3, CK, 512, 1>(a, st)
                              : touched > 512 ? launch_ln_fwd_shift<T, 2, CK, 512, 1>(a, st)
                              : touched > 320 ? launch_ln_fwd_shift<T, 1, CK, 512, 1>(a, st)
                                              : launch_ln_fwd_shift<T, 1, CK, 320, 2>(a, st);
        if (e != cudaSuccess) return fail(RWKV_E_CUDA, "ln_fwd_shift_kernel: %s", cudaGetErrorString(e));
    } else if (a.D <= 32 * 8) {
        ln_fwd_any_kernel<T, 32, 8><<<ceil_div(a.rows, 4), 128, 0, st>>>(a);
    } else if (a.D <= 512 * 20) {
        if (a.D <= 128 * 4) ln_fwd_any_kernel<T, 128, 4><<<a.rows, 128, 0, st>>>(a);
        else if (a.D <= 128 * 8) ln_fwd_any_kernel<T, 128, 8><<<a.rows, 128, 0, st>>>(a);
        else if (a.D <= 256 * 8) ln_fwd_any_kernel<T, 256, 8><<<a.rows, 256, 0, st>>>(a);
        else if (a.D <= 512 * 8) ln_fwd_any_kernel<T, 512, 8><<<a.rows, 512, 0, st>>>(a);
        else if (a.D <= 512 * 12) ln_fwd_any_kernel<T, 512, 12><<<a.rows, 512, 0, st>>>(a);
        else ln_fwd_any_kernel<T, 512, 20><<<a.rows, 512, 0, st>>>(a);
    } else {
        ln_fwd_long_kernel<T><<<a.rows, 256, 0, st>>>(a);
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

// A block takes R rows at a time, R (blockIdx.x + i gridDim.x); thread t owns
// the vectors t + j blockDim.x of every row, so its sums over rows of dy h and
// dy stay in registers until the end.  dy, x (or its codes) and dres run
// LN_STAGES - 1 steps ahead through a ring in shared memory; a thread copies
// (cp.async) and reads only its own vectors, so the ring needs no barrier, and
// HBM stays busy while the block computes and waits at its barrier: one per R
// rows, for the two row sums (buffers alternating).
//
// SH: rows that need not start on a vector, one at a time, gridDim.x a multiple of VE
// (or no block with a second row).
template <typename T, bool CK, int NV, int R, int MAXT, int MINB, bool SH>
__global__ void __launch_bounds__(MAXT, MINB) ln_bwd_kernel(const LnBwdArgs a) {
    constexpr int VE = Vec16<T>::N;
    static_assert(!SH || R == 1, "neighbouring rows start at different places");
    extern __shared__ uint4 ring[];  // [stage][row][dy | x | dres][NV][thread]
    __shared__ float red[2][16][2 * R];
    const int t = threadIdx.x, nt = blockDim.x, warp = t >> 5, lane = t & 31, nw = nt >> 5;
    const int head = SH ? (int)((int64_t)blockIdx.x * a.D % VE) : 0;
    const int nvec = (a.D + head + VE - 1) / VE;
    const float inv_d = 1.f / (float)a.D;
    float w[NV][VE], sw[NV][VE], sb[NV][VE];
    bool has[NV];
    int tail[NV];                                                  // of each vector, VE in the row's midst
    auto column = [&](int j) { return (t + j * nt) * VE - head; };  // of a vector's first element
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int v = t + j * nt;
        has[j] = v < nvec;
        tail[j] = SH ? min(VE, a.D - column(j)) : VE;
#pragma unroll
        for (int k = 0; k < VE; k++) w[j][k] = sw[j][k] = sb[j][k] = 0.f;
        if constexpr (SH) {
#pragma unroll
            for (int k = 0; k < VE; k++)
                if (has[j] && column(j) + k >= 0 && k < tail[j]) w[j][k] = load_param(a.w, a.wdtype, column(j) + k);
        } else {
            if (has[j]) load_params<VE>(a.w, a.wdtype, (int64_t)v * VE, w[j]);
        }
    }
    const int step = (int)gridDim.x * R;
    const int64_t vstep = SH ? (int64_t)step * a.D / VE : (int64_t)step * nvec;  // in vectors
    const uint4* const dy = static_cast<const uint4*>(a.dy) + t;
    const uint4* const xs = static_cast<const uint4*>(a.x) + t;
    const uint4* const dres = static_cast<const uint4*>(a.dres) + t;
    using Codes = std::conditional_t<VE == 8, uint2, uint32_t>;  // of one vector
    const Codes* const cs = reinterpret_cast<const Codes*>(a.codes) + t;
    // one row at a time always exists inside the loop
    auto exists = [&](int64_t r0, int r) { return R == 1 || r0 + r < a.rows; };
    // ring slot of (row, part, vector) in the stage that starts at `base`
    auto slot = [&](int base, int r, int part, int j) { return ring + base + ((r * 3 + part) * NV + j) * nt; };
    const int stage_n = R * 3 * NV * nt;
    auto fetch = [&](int64_t r0, int64_t at, int base) {
        if (r0 < a.rows) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int j = 0; j < NV; j++)
                    if (exists(r0, r) && has[j]) {
                        const int64_t o = at + r * nvec + j * nt;
                        if constexpr (SH) {
                            const int n = tail[j] * (int)sizeof(T);
                            copy_async_n<16>(slot(base, r, 0, j), dy + o, n);
                            if constexpr (CK) copy_async_n<VE>(slot(base, r, 1, j), cs + o, tail[j]);
                            else copy_async_n<16>(slot(base, r, 1, j), xs + o, n);
                            if (a.dres) copy_async_n<16>(slot(base, r, 2, j), dres + o, n);
                        } else {
                            copy_async<16>(slot(base, r, 0, j), dy + o);
                            if constexpr (CK) copy_async<VE>(slot(base, r, 1, j), cs + o);
                            else copy_async<16>(slot(base, r, 1, j), xs + o);
                            if (a.dres) copy_async<16>(slot(base, r, 2, j), dres + o);
                        }
                    }
        }
        copy_commit();
    };
    // the rows' statistics and exponents, one step ahead in registers
    float mean[R], rstd[R], nmean[R], nrstd[R];
    uint32_t ex[R][NV], nex[R][NV];
    auto fetch_small = [&](int64_t r0) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int64_t row = min(r0 + r, (int64_t)a.rows - 1);  // of no use past the end
            nmean[r] = a.mean[row];
            nrstd[r] = a.rstd[row];
            if constexpr (CK) {
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    if constexpr (SH) {  // a vector may lie in two groups
                        const uint8_t* e = a.exps + row * a.G;
                        const int c = column(j);
                        nex[r][j] = has[j] ? e[max(c, 0) / CK_GROUP] | (uint32_t)e[min(c + VE, a.D) - 1 >> 5] << 8 : 0u;
                    } else {
                        nex[r][j] = has[j] ? a.exps[row * a.G + (t + j * nt) / (CK_GROUP / VE)] : 0u;
                    }
                }
            }
        }
    };
    const int64_t first = (int64_t)blockIdx.x * R;
    int64_t at = SH ? first * a.D / VE : first * nvec, fat = at;
#pragma unroll
    for (int i = 0; i < LN_STAGES - 1; i++, fat += vstep) fetch(first + (int64_t)i * step, fat, t + i * stage_n);
    fetch_small(first);
    int cur = t, put = t + (LN_STAGES - 1) * stage_n, buf = 0;
    for (int64_t r0 = first; r0 < a.rows; r0 += step, at += vstep, fat += vstep, buf ^= 1) {
        fetch(r0 + (int64_t)(LN_STAGES - 1) * step, fat, put);
        copy_wait<LN_STAGES - 1>();
#pragma unroll
        for (int r = 0; r < R; r++) {
            mean[r] = nmean[r];
            rstd[r] = nrstd[r];
            if constexpr (CK)
#pragma unroll
                for (int j = 0; j < NV; j++) ex[r][j] = nex[r][j];
        }
        fetch_small(r0 + step);
        // pass 1: h, the sums over the row (g, g h) and over the rows (dy h, dy)
        float h[R][NV][VE], rs[2 * R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            rs[2 * r] = rs[2 * r + 1] = 0.f;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (!exists(r0, r) || !has[j]) continue;
                float dy[VE];
                if constexpr (SH) {
                    if (j == 0 && t == 0) {
                        drop_head<T>(*slot(cur, r, 0, j), head);
                        if constexpr (!CK) drop_head<T>(*slot(cur, r, 1, j), head);
                    }
                }
                Vec16<T>::unpack(*slot(cur, r, 0, j), dy);
                // x - mean in one rounding: no multiple of rstd cancels where |mean| is large
                if constexpr (CK) {
                    const uint32_t* c = reinterpret_cast<const uint32_t*>(slot(cur, r, 1, j));
                    ck_codes4(c[0], h[r][j]);
                    if constexpr (VE == 8) ck_codes4(c[1], h[r][j] + 4);
                    if constexpr (SH) {
                        const float s0 = ck_scale(ex[r][j] & 255u), s1 = ck_scale(ex[r][j] >> 8);
                        const int other = CK_GROUP - (max(column(j), 0) & (CK_GROUP - 1)) + (column(j) < 0 ? head : 0);
#pragma unroll
                        for (int k = 0; k < VE; k++) h[r][j][k] = fmaf(h[r][j][k], k < other ? s0 : s1, -mean[r]);
                    } else {
                        const float s = ck_scale(ex[r][j]);
#pragma unroll
                        for (int k = 0; k < VE; k++) h[r][j][k] = fmaf(h[r][j][k], s, -mean[r]);
                    }
                } else {
                    Vec16<T>::unpack(*slot(cur, r, 1, j), h[r][j]);
#pragma unroll
                    for (int k = 0; k < VE; k++) h[r][j][k] -= mean[r];
                }
#pragma unroll
                for (int k = 0; k < VE; k++) {
                    h[r][j][k] *= rstd[r];
                    const float g = dy[k] * w[j][k];
                    rs[2 * r] += g;
                    rs[2 * r + 1] = fmaf(g, h[r][j][k], rs[2 * r + 1]);
                    sw[j][k] = fmaf(dy[k], h[r][j][k], sw[j][k]);
                    sb[j][k] += dy[k];
                }
            }
        }
        // over the warp: value i ends up in lanes 16 i / R .. (32 / 2R lanes each)
        constexpr int N = 2 * R, L = 32 / N;
        const float p = lanes_sum<N>(rs, lane);
        if (lane % L == 0) red[buf][warp][lane / L] = p;
        __syncthreads();
        float tot = 0.f;
#pragma unroll
        for (int i = 0; i < 16 / L + (16 % L != 0); i++) {
            const int k = lane % L + i * L;
            if (k < nw) tot += red[buf][k][lane / L];
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, o);
        tot *= inv_d;
        // pass 2: dx = rstd (g - m1 - h m2) + dres
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float c0 = -rstd[r] * __shfl_sync(0xffffffffu, tot, 2 * r * L);
            const float c1 = -rstd[r] * __shfl_sync(0xffffffffu, tot, (2 * r + 1) * L);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (!exists(r0, r) || !has[j]) continue;
                float dy[VE], o[VE];
                Vec16<T>::unpack(*slot(cur, r, 0, j), dy);
                if (a.dres) {
                    Vec16<T>::unpack(*slot(cur, r, 2, j), o);
#pragma unroll
                    for (int k = 0; k < VE; k++) o[k] += c0;
                } else {
#pragma unroll
                    for (int k = 0; k < VE; k++) o[k] = c0;
                }
#pragma unroll
                for (int k = 0; k < VE; k++) o[k] = fmaf(dy[k] * w[j][k], rstd[r], fmaf(h[r][j][k], c1, o[k]));
                uint4* out = static_cast<uint4*>(a.dx) + t + at + r * nvec + j * nt;
                const int lo = j == 0 && t == 0 ? head : 0;
                if (SH && (lo > 0 || tail[j] < VE)) store_part<T>(reinterpret_cast<T*>(out), o, lo, tail[j]);
                else __stcs(out, Vec16<T>::pack(o));
            }
        }
        put = cur;
        cur = cur == t + (LN_STAGES - 1) * stage_n ? t : cur + stage_n;
    }
    copy_wait<0>();
    if (!a.part) return;
    float* p = a.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int v = t + j * nt;
        if (v >= nvec) continue;
        if constexpr (SH) {
#pragma unroll
            for (int k = 0; k < VE; k++)
                if (column(j) + k >= 0 && k < tail[j]) {
                    p[column(j) + k] = sw[j][k];
                    p[a.D + column(j) + k] = sb[j][k];
                }
            continue;
        }
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

// Tensors off a 16-byte boundary, and rows of more vectors than ln_bwd_kernel
// takes: a block per row at a time, single elements, element t + j NT of thread t,
// at most NE; the sums over rows stay in registers (10326 x 2412 fp16: 220 us, in
// vectors 54).
template <typename T, bool CK, int NT, int NE>
__global__ void __launch_bounds__(NT) ln_bwd_any_kernel(const LnBwdArgs a) {
    __shared__ float2 red[2][NT / 32];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const float inv_d = 1.f / (float)a.D;
    float w[NE], sw[NE], sb[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) {
        w[j] = t + j * NT < a.D ? load_param(a.w, a.wdtype, t + j * NT) : 0.f;
        sw[j] = sb[j] = 0.f;
    }
    // the next row is read while this one is computed
    float ndy[NE], nx[NE], nmean = 0.f, nrstd = 0.f;
    auto fetch = [&](int64_t row) {
        if (row >= a.rows) return;
        const T* dyr = static_cast<const T*>(a.dy) + row * a.D;
        nmean = a.mean[row];
        nrstd = a.rstd[row];
#pragma unroll
        for (int j = 0; j < NE; j++) {
            const int i = t + j * NT;
            ndy[j] = i < a.D ? to_f<T>(dyr[i]) : 0.f;
            nx[j] = i < a.D ? bwd_x<T, CK>(a, row, i) : 0.f;
        }
    };
    fetch(blockIdx.x);
    int buf = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, buf ^= 1) {
        const float mean = nmean, rstd = nrstd;
        float dy[NE], h[NE], res[NE];
#pragma unroll
        for (int j = 0; j < NE; j++) {
            const int i = t + j * NT;
            dy[j] = ndy[j];
            h[j] = nx[j];
            res[j] = a.dres && i < a.D ? to_f<T>(static_cast<const T*>(a.dres)[row * a.D + i]) : 0.f;
        }
        fetch(row + gridDim.x);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NE; j++) {
            h[j] = t + j * NT < a.D ? (h[j] - mean) * rstd : 0.f;
            const float g = dy[j] * w[j];
            s1 += g;
            s2 = fmaf(g, h[j], s2);
            sw[j] = fmaf(dy[j], h[j], sw[j]);
            sb[j] += dy[j];
        }
        s1 = warp_sum(s1);
        s2 = warp_sum(s2);
        if (lane == 0) red[buf][warp] = make_float2(s1, s2);
        __syncthreads();
        const float2 p = lane < NT / 32 ? red[buf][lane] : make_float2(0.f, 0.f);
        const float m1 = warp_sum(p.x) * inv_d, m2 = warp_sum(p.y) * inv_d;
#pragma unroll
        for (int j = 0; j < NE; j++) {
            const int i = t + j * NT;
            if (i >= a.D) break;
            const float d = rstd * (dy[j] * w[j] - m1 - h[j] * m2);
            static_cast<T*>(a.dx)[row * a.D + i] = from_f<T>(res[j] + d);
        }
    }
    if (!a.part) return;
    float* p = a.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int j = 0; j < NE; j++) {
        const int i = t + j * NT;
        if (i >= a.D) break;
        p[i] = sw[j];
        p[a.D + i] = sb[j];
    }
}

// Any length.  dx: a block per row, the row re-read (from L1 / L2).  dx may be dy, so
// the column sums (ln_bwd_cols_kernel) are launched first.
template <typename T, bool CK>
__global__ void __launch_bounds__(256) ln_bwd_long_kernel(const LnBwdArgs a) {
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
__global__ void __launch_bounds__(256) ln_bwd_cols_kernel(const LnBwdArgs a) {
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
// columns per block, 32 interleaved slices of the partials, in a fixed order.
// Launched to start beside the row kernel's end (pdl_wait).
__global__ void __launch_bounds__(1024) ln_bwd_params_kernel(const float* part, int blocks, int D,
                                                             void* dw, void* db, int wdtype) {
    __shared__ float red[32][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + col, width = 2 * (int64_t)D;
    pdl_wait();
    float s = 0.f;
    if (c < width) {
#pragma unroll 4
        for (int b = slice; b < blocks; b += 32) s += part[b * width + c];
    }
    red[slice][col] = s;
    __syncthreads();
    // warp w sums column w over the slices
    const float t = warp_sum(red[col][slice]);
    const int64_t o = (int64_t)blockIdx.x * 32 + slice;
    if (col == 0 && o < width) {
        if (o < D) store_param(dw, wdtype, o, t);
        else store_param(db, wdtype, o - D, t);
    }
}

constexpr int LN_BWD_BLOCKS = 148 * 4;  // at most: four resident blocks per SM
constexpr int LN_LONG_BLOCKS = 64;      // column sums of the rows that only the long kernels take
// 512 threads with three vectors of 8 each, or 20 single elements
constexpr int LN_BWD_VECTORS = 512 * 3, LN_BWD_ELEMENTS = 512 * 20;

template <typename T, bool CK, int NV, int R, int MAXT, int MINB, bool SH>
cudaError_t launch_ln_bwd_t(const LnBwdArgs& a, int* blocks, cudaStream_t st) {
    auto kern = ln_bwd_kernel<T, CK, NV, R, MAXT, MINB, SH>;
    constexpr int VE = Vec16<T>::N;
    const int nt = ceil_div(ceil_div(SH ? most_vectors<T>(a.D) : a.D / VE, NV), 32) * 32;
    constexpr int PER_T = LN_STAGES * R * 3 * NV * 16;  // shared memory of a thread
    const int smem = PER_T * nt;
    // as many blocks as are resident, so that they all run in one wave
    static ResidentBlocks resident;
    int per_sm;
    const cudaError_t e = resident.get(kern, nt, smem, PER_T * MAXT, &per_sm);
    if (e != cudaSuccess) return e;
    const int most = std::min(148 * per_sm, LN_BWD_BLOCKS);
    *blocks = std::min(ceil_div(a.rows, R), SH ? most / VE * VE : most);
    kern<<<*blocks, nt, smem, st>>>(a);
    return cudaGetLastError();
}

// SH: lengths that are not a multiple of 8
template <typename T, bool CK, bool SH>
int launch_ln_bwd(LnBwdArgs a, bool vec, void* dw, void* db, cudaStream_t st) {
    const int nvec = SH ? most_vectors<T>(a.D) : a.D / Vec16<T>::N;
    int blocks;
    if (vec && nvec <= LN_BWD_VECTORS) {
        // vectors per thread: the fewest with at most 512 threads.  Two rows
        // at a time from a dense x (16384 x 2048 bf16: 50 us, one row 65 us), one
        // from a checkpoint, whose decoding takes more registers (2560 channels: 68
        // us, two rows 77).  Up to 320 threads with registers for two blocks per
        // SM (2560 channels: dense 62 us, unbounded 72; 2048 from a checkpoint 54
        // and 60; for three: 2560 from a checkpoint 87 us)
        constexpr int R = CK || SH ? 1 : 2;
        const cudaError_t e = nvec > 1024  ? launch_ln_bwd_t<T, CK, 3, 1, 512, 1, SH>(a, &blocks, st)
                              : nvec > 512 ? launch_ln_bwd_t<T, CK, 2, 1, 512, 1, SH>(a, &blocks, st)
                              : nvec > 320 ? launch_ln_bwd_t<T, CK, 1, R, 512, 1, SH>(a, &blocks, st)
                                           : launch_ln_bwd_t<T, CK, 1, R, 320, 2, SH>(a, &blocks, st);
        if (e != cudaSuccess) return fail(RWKV_E_CUDA, "ln_bwd_kernel: %s", cudaGetErrorString(e));
    } else if (a.D <= LN_BWD_ELEMENTS) {
        blocks = std::min(a.rows, LN_BWD_BLOCKS);
        if (a.D <= 256) ln_bwd_any_kernel<T, CK, 256, 1><<<blocks, 256, 0, st>>>(a);
        else if (a.D <= 256 * 2) ln_bwd_any_kernel<T, CK, 256, 2><<<blocks, 256, 0, st>>>(a);
        else if (a.D <= 256 * 4) ln_bwd_any_kernel<T, CK, 256, 4><<<blocks, 256, 0, st>>>(a);
        else if (a.D <= 512 * 3) ln_bwd_any_kernel<T, CK, 512, 3><<<blocks, 512, 0, st>>>(a);
        else if (a.D <= 512 * 4) ln_bwd_any_kernel<T, CK, 512, 4><<<blocks, 512, 0, st>>>(a);
        else if (a.D <= 512 * 8) ln_bwd_any_kernel<T, CK, 512, 8><<<blocks, 512, 0, st>>>(a);
        else if (a.D <= 512 * 12) ln_bwd_any_kernel<T, CK, 512, 12><<<blocks, 512, 0, st>>>(a);
        else ln_bwd_any_kernel<T, CK, 512, 20><<<blocks, 512, 0, st>>>(a);
    } else {
        blocks = std::min(a.rows, LN_LONG_BLOCKS);
        if (a.part) {
            ln_bwd_cols_kernel<T, CK><<<dim3(ceil_div(a.D, 256), blocks), 256, 0, st>>>(a);
            if (int rc = check_launch("ln_bwd_cols_kernel")) return rc;
        }
        ln_bwd_long_kernel<T, CK><<<a.rows, 256, 0, st>>>(a);
    }
    if (int rc = check_launch("ln_bwd_kernel")) return rc;
    if (!a.part) return ok();
    const cudaError_t e = launch_pdl(ln_bwd_params_kernel, dim3(ceil_div(2 * (int64_t)a.D, 32)), dim3(1024), 0, st,
                                     (const float*)a.part, blocks, a.D, dw, db, a.wdtype);
    if (e != cudaSuccess) return fail(RWKV_E_CUDA, "ln_bwd_params_kernel: %s", cudaGetErrorString(e));
    return ok();
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
    const bool whole = D % 8 == 0 && al(weight, 16) && al(bias, 16);
    const bool vec = al(x, 16) && al(y, 16) && al(codes, 8);
    return dispatch_dtype(dtype, [&]<typename T>() {
        return codes ? launch_ln_fwd<T, true>(a, vec, whole, (cudaStream_t)stream)
                     : launch_ln_fwd<T, false>(a, vec, whole, (cudaStream_t)stream);
    });
}

extern "C" int64_t rwkv_layer_norm_backward_workspace_size(int rows, int D) {
    if (rows < 1 || D < 1) return 0;
    // (whatever the type and the alignment)
    const int blocks = D > std::max(LN_BWD_VECTORS * 8, LN_BWD_ELEMENTS) ? LN_LONG_BLOCKS : LN_BWD_BLOCKS;
    return (int64_t)std::min(rows, blocks) * 2 * D * (int64_t)sizeof(float);
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
    const bool whole = D % 8 == 0 && al(weight, 16);
    const bool vec = al(dy, 16) && al(x, 16) && al(codes, 8) && al(dres, 16) && al(dx, 16);
    return dispatch_dtype(dtype, [&]<typename T>() {
        auto st = (cudaStream_t)stream;
        if (whole)
            return codes ? launch_ln_bwd<T, true, false>(a, vec, dweight, dbias, st)
                         : launch_ln_bwd<T, false, false>(a, vec, dweight, dbias, st);
        return codes ? launch_ln_bwd<T, true, true>(a, vec, dweight, dbias, st)
                     : launch_ln_bwd<T, false, true>(a, vec, dweight, dbias, st);
    });
}
