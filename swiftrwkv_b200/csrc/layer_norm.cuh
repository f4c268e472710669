// What the layer norm (layer_norm.cu) and the residual norm (residual_norm.cu) share:
// the kernels of rows in 16-byte vectors and their launches.
#pragma once

#include <algorithm>
#include <atomic>

#include "ckpt8.cuh"
#include "philox.cuh"

namespace rwkv {

template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}
// the first n bytes, zeros behind them
template <int BYTES>
__device__ __forceinline__ void copy_async_n(void* dst, const void* src, int n) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
    // the residual norm's: what is normed is x + drop(branch), and goes to `sum` too
    const void* branch;
    void* sum;
    Dropout drop;
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
// fp32 (no branch between their loads); CK: write the checkpoint; BR: the residual
// norm, whose sums are held, normed and checkpointed in fp32 and rounded where they
// are stored.
template <typename T, int TPR, int NV, int R, bool WF32, bool CK, bool BR = false>
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
    float x[F32 ? R : 1][F32 ? NV : 1][VE];
    auto vec = [&](int r, int j) -> float* { return x[F32 ? r : 0][F32 ? j : 0]; };
    if constexpr (BR) {
        static_assert(F32, "the sums stay in fp32 registers");
        const uint4* br = static_cast<const uint4*>(a.branch) + row0 * nvec + t;
        uint4* sr = static_cast<uint4*>(a.sum) + row0 * nvec + t;
        uint4 add[R][NV];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NV; j++)
                add[r][j] = row0 + r < a.rows && t + j * TPR < nvec ? __ldcs(br + (int64_t)r * nvec + j * TPR)
                                                                   : make_uint4(0, 0, 0, 0);
        const DropKey key = drop_key(a.drop);
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                float* f = vec(r, j);
                float q[VE];
                Vec16<T>::unpack(raw[r][j], f);
                Vec16<T>::unpack(add[r][j], q);
                drop_at<VE>(q, key, (uint64_t)((row0 + r) * nvec + t + j * TPR) * VE, a.drop.threshold, a.drop.scale);
#pragma unroll
                for (int k = 0; k < VE; k++) f[k] = __fadd_rn(f[k], q[k]);
                const bool in = row0 + r < a.rows && t + j * TPR < nvec;
                if (in) __stcs(sr + (int64_t)r * nvec + j * TPR, Vec16<T>::pack(f));
                if constexpr (CK) {
                    uint32_t top = 0;
#pragma unroll
                    for (int k = 0; k < VE; k++) top = max(top, abs_bits(f[k]));
#pragma unroll
                    for (int o = 1; o < CK_GROUP / VE; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const uint32_t e = ck_exponent(top);
                    const float inv = ck_inv_scale(e);
                    const int v = t + j * TPR;
                    if (in) {
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
    }
    if constexpr (CK && !BR) {
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
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        mean[r] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float* f = vec(r, j);
            if constexpr (!BR) Vec16<T>::unpack(raw[r][j], f);
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

template <typename T, int TPR, int NV, int R, bool CK, bool BR = false>
void launch_ln_fwd_t(const LnFwdArgs& a, cudaStream_t st) {
    const int grid = ceil_div(a.rows, R);
    if (a.wdtype == RWKV_F32) ln_fwd_kernel<T, TPR, NV, R, true, CK, BR><<<grid, TPR, 0, st>>>(a);
    else ln_fwd_kernel<T, TPR, NV, R, false, CK, BR><<<grid, TPR, 0, st>>>(a);
}

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
    // the residual norm's: dbranch = drop(dx), from dx before its rounding
    void* dbranch;
    Dropout drop;
};

// The sums over a warp of N values per lane (N a power of two), value i in the
// lanes i 32 / N .. : each exchange halves the values a lane holds, so that N
// sums take N - 1 + log2(32 / N) shuffles instead of 5 N.
template <int N>
__device__ __forceinline__ float lanes_sum(float* v, int lane) {
#pragma unroll
    for (int n = N, o = 16; n > 1; n /= 2, o /= 2) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < n / 2; i++) {
            const float keep = up ? v[i + n / 2] : v[i], send = up ? v[i] : v[i + n / 2];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    float s = v[0];
#pragma unroll
    for (int o = 16 / N; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// A block takes R rows at a time, R (blockIdx.x + i gridDim.x); thread t owns
// the vectors t + j blockDim.x of every row, so its sums over rows of dy h and
// dy stay in registers until the end.  dy, x (or its codes) and dres run
// LN_STAGES - 1 steps ahead through a ring in shared memory; a thread copies
// (cp.async) and reads only its own vectors, so the ring needs no barrier, and
// HBM stays busy while the block computes and waits at its barrier: one per R
// rows, for the two row sums (buffers alternating).
//
// SH: rows that need not start on a vector, one at a time, gridDim.x a multiple of VE
// (or no block with a second row).  BR: the residual norm, with the branch's gradient.
template <typename T, bool CK, int NV, int R, int MAXT, int MINB, bool SH, bool BR = false>
__global__ void __launch_bounds__(MAXT, MINB) ln_bwd_kernel(const LnBwdArgs a) {
    constexpr int VE = Vec16<T>::N;
    static_assert(!SH || R == 1, "neighbouring rows start at different places");
    static_assert(!SH || !BR, "a vector's bits are one block's");
    extern __shared__ uint4 ring[];  // [stage][row][dy | x | dres][NV][thread]
    __shared__ float red[2][16][2 * R];
    const int t = threadIdx.x, nt = blockDim.x, warp = t >> 5, lane = t & 31, nw = nt >> 5;
    const int head = SH ? (int)((int64_t)blockIdx.x * a.D % VE) : 0;
    const int nvec = (a.D + head + VE - 1) / VE;
    const float inv_d = 1.f / (float)a.D;
    [[maybe_unused]] DropKey key;
    if constexpr (BR) key = drop_key(a.drop);
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
                if constexpr (BR) {
                    const int64_t i = t + at + r * nvec + j * nt;
                    drop_at<VE>(o, key, (uint64_t)i * VE, a.drop.threshold, a.drop.scale);
                    __stcs(static_cast<uint4*>(a.dbranch) + i, Vec16<T>::pack(o));
                }
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

// out[c] = sum over the blocks of part[block][c], c < 2D (dweight, dbias): 32
// columns per block, 32 interleaved slices of the partials, in a fixed order.
// Launched to start beside the row kernel's end (pdl_wait).
static __global__ void __launch_bounds__(1024) ln_bwd_params_kernel(const float* part, int blocks, int D,
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

template <typename T, bool CK, int NV, int R, int MAXT, int MINB, bool SH, bool BR = false>
cudaError_t launch_ln_bwd_t(const LnBwdArgs& a, int* blocks, cudaStream_t st) {
    auto kern = ln_bwd_kernel<T, CK, NV, R, MAXT, MINB, SH, BR>;
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

inline bool al(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline uintptr_t elem(int dtype) { return dtype == RWKV_F32 ? 4 : 2; }

}  // namespace rwkv
