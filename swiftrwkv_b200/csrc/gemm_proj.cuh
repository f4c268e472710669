// The three matrix products of a trainable projection on the tcgen05 tensor
// cores, one kernel:
//
//     D[m, n] = epilogue( sum_k A[m, k] B[n, k] )            (fp32 accumulation)
//
//   forward  y[row, o]  = act(x W^T + bias) + residual     A = x (K-major), B = W (K-major)
//   dX       dx[row, i] = (dY W) act'(z) + addend          A = dY (K-major), B = W^T (MN-major)
//   dW       dw[o, i]   = dY^T X                           A = dY^T (MN-major), B = X^T (MN-major)
//
// A and B are both bf16 or both fp16 and are read in place by TMA: an operand
// whose rows run along K lands K-major, one whose rows run along M / N lands
// MN-major, both with the 128-byte swizzle, and the instruction descriptor says
// which.  Boxes that reach past a tensor's end read zeros, so no size has to be
// a multiple of a tile; row pitches must be multiples of 16 bytes (IN and OUT
// multiples of 8).
//
// Tile = 128 rows of D (TMEM lanes) x BN columns, K in stages of 64.  A persistent
// CTA walks its tiles; the accumulator of tile t lives in TMEM half (t & 1), so
// the epilogue of one tile runs beside the MMAs of the next.
//   warp 0      TMA producer, ST stages
//   warp 1      TMEM owner; one thread issues 4 tcgen05.mma (M=128, N=BN, K=16)
//               per stage and commits the stage / the tile
//   warps 2-9   epilogue: TMEM lane quadrant (warp & 3) = 32 rows of D, column half
//               (warp - 2) / 4; 32 columns at a time.  A thread holds 32 consecutive
//               columns of one row, exactly a checkpoint group, so a group's largest
//               |z| needs no exchange.  Results go through a swizzled 32 x 32 tile in
//               shared memory and leave by TMA store (full 64-byte row pieces, clipped
//               at the tensor's end).
// Tiles are walked in groups of 8 row blocks, so that the CTAs at work at one
// time share a few row blocks of A and a few of B in L2.
//
// Split-K (S > 1, when there are fewer tiles than SMs): split z of a tile sums its
// share of the stages into a fp32 partial tile in the workspace, and
// proj_join_kernel adds the partials in split order (deterministic) and runs
// the epilogue.
//
// Every mbarrier wait is bounded (tc::mbar_wait); a wait that gives up sets the
// shared error flag, every role winds down, the producer waits (bounded) for its
// copies in flight and TMEM is freed after the final MMA commit.
#pragma once

#include "ckpt8.cuh"
#include "gemm_dx.cuh"

namespace rwkv {

constexpr int PJ_BK = 64;
constexpr int PJ_GROUP_M = 8;      // row blocks walked together
constexpr int PJ_EPI_WARPS = 8;
constexpr int PJ_THREADS = 64 + 32 * PJ_EPI_WARPS;
constexpr int PJ_STAGE_OUT = 4096;  // staging bytes per epilogue warp: 32 x 32 fp32, or two 32 x 32 of 16 bits

// What happens to the sums; all tensors are row-major [M, N].
struct ProjEpi {
    int bf16;           // operand type: bf16 (else fp16)
    int out_f32;        // D in fp32 (else in the operand type)
    int act;            // forward: act(z); grad: times act'(pre)
    int grad;
    const void* bias;   // [N] or NULL, bias_dtype
    int bias_dtype;
    const void* add;    // residual / addend in D's type, or NULL
    int8_t* codes;      // forward: 8-bit checkpoint of z, or NULL
    uint8_t* exps;
    void* z;            // forward: z in the operand type, or NULL
    const void* pre;    // grad: pre-activation in the operand type, or
    const int8_t* pre_codes;  // its checkpoint
    const uint8_t* pre_exps;
};

struct ProjArgs {
    CUtensorMap amap, bmap;
    CUtensorMap dmap;   // D, box {32, 32}; split-K: the partials {N, M, S} fp32, box {32, 32, 1}
    ProjEpi e;
    int M, N, nk;       // D's size, K stages
    int mt, nt, S;      // tiles along M and N, splits
    uint32_t idesc;
    int* err;           // device flag: a wait gave up
    int* err_host;      // mapped host record
};

// Two 16-bit values of the operand type as floats, and back.
__device__ __forceinline__ float2 unpack2(uint32_t w, int bf16) {
    if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, int bf16) {
    if (bf16) return tc::pack_bf16x2(lo, hi);
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void load8_16(const void* p, int64_t at, int bf16, float* v) {
    const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = unpack2(w[i], bf16);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack8_16(const float* v, int bf16) {
    return make_uint4(pack2(v[0], v[1], bf16), pack2(v[2], v[3], bf16), pack2(v[4], v[5], bf16),
                      pack2(v[6], v[7], bf16));
}

// The epilogue of columns col .. col + 31 of one row, of which the first nv (a
// multiple of 8) exist; v holds the sums, 0 in columns that do not exist.
__device__ __forceinline__ void proj_epilogue32(float* v, const ProjEpi& e, int64_t row, int col, int nv, int N) {
    const int64_t at = row * N + col;
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (8 * i < nv) {
                float b[8];
                load_params<8>(e.bias, e.bias_dtype, col + 8 * i, b);
#pragma unroll
                for (int k = 0; k < 8; k++) v[8 * i + k] += b[k];
            }
    }
    if (e.codes) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) top = max(top, abs_bits(v[i]));
        const uint32_t x = ck_exponent(top);
        const float inv = ck_inv_scale(x);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (8 * i < nv)
                *reinterpret_cast<uint2*>(e.codes + at + 8 * i) =
                    make_uint2(ck_pack4(v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3], inv),
                               ck_pack4(v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7], inv));
        e.exps[row * ((N + CK_GROUP - 1) / CK_GROUP) + col / CK_GROUP] = (uint8_t)x;
    }
    if (e.z) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (8 * i < nv)
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(e.z) + at + 8 * i) = pack8_16(v + 8 * i, e.bf16);
    }
    if (e.grad) {
        float p[32];
        if (e.pre_codes) {
            const float s = ck_scale(e.pre_exps[row * ((N + CK_GROUP - 1) / CK_GROUP) + col / CK_GROUP]);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (8 * i < nv) {
                    const uint2 w = *reinterpret_cast<const uint2*>(e.pre_codes + at + 8 * i);
                    ck_unpack4(w.x, s, p + 8 * i);
                    ck_unpack4(w.y, s, p + 8 * i + 4);
                }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (8 * i < nv) load8_16(e.pre, at + 8 * i, e.bf16, p + 8 * i);
        }
        with_act(e.act, [&]<int ACT>() {
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (i < nv) v[i] *= act_grad_t<ACT, true>(p[i]);
        });
    } else {
        with_act(e.act, [&]<int ACT>() {
#pragma unroll
            for (int i = 0; i < 32; i++) v[i] = act_t<ACT, true>(v[i]);
        });
    }
    if (e.add) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (8 * i >= nv) break;
            float a[8];
            if (e.out_f32) {
                const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(e.add) + at + 8 * i);
                const float4 lo = p[0], hi = p[1];
                a[0] = lo.x, a[1] = lo.y, a[2] = lo.z, a[3] = lo.w;
                a[4] = hi.x, a[5] = hi.y, a[6] = hi.z, a[7] = hi.w;
            } else {
                load8_16(e.add, at + 8 * i, e.bf16, a);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) v[8 * i + k] += a[k];
        }
    }
}

namespace tc {
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src),
                 "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                 "r"(src), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// at most N of this thread's bulk stores still read their shared memory
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory"); }
}  // namespace tc

template <int BN>
struct PjCfg {
    static constexpr int A_BYTES = 128 * 128;       // 128 rows x 64 k, 16 bits
    static constexpr int B_BYTES = BN * 128;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int OUT_BYTES = PJ_EPI_WARPS * PJ_STAGE_OUT;
    static constexpr int ST = 192 * 1024 / STAGE;
    static constexpr int NBAR = 2 * ST + 5;
    static constexpr int O_OFF = ST * STAGE;        // output staging
    static constexpr int B_OFF = O_OFF + OUT_BYTES;
    static constexpr int T_OFF = B_OFF + NBAR * 8;
    static constexpr int TOTAL = T_OFF + 16 + 1024;
    static constexpr int TMC = 2 * BN;
    static_assert(TOTAL <= 227 * 1024, "shared memory per CTA");
    static_assert(BN == 64 || BN == 128 || BN == 256, "TMEM allocation is a power of two; halves in 32s");
};

// AMN / BMN: the operand is MN-major.
template <int BN, bool AMN, bool BMN>
__global__ void __launch_bounds__(PJ_THREADS, 1) proj_kernel(const __grid_constant__ ProjArgs a) {
    using C = PjCfg<BN>;
    constexpr int ST = C::ST;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::B_OFF);
    uint64_t* empty = full + ST;   // the stage's MMAs are done
    uint64_t* accf = empty + ST;   // [2] the tile's accumulator is complete
    uint64_t* acce = accf + 2;     // [2] the epilogue has drained it
    uint64_t* done = acce + 2;     // every MMA is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::T_OFF);
    int* skip_slot = reinterpret_cast<int*>(smem + C::T_OFF + 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int ntiles = a.mt * a.nt * a.S;
    const int my_tiles = (int)blockIdx.x < ntiles ? (ntiles - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
    int* err = a.err;

    if (tid == 0) {
        for (int s = 0; s < ST; s++) {
            tc::mbar_init(full + s, 1);
            tc::mbar_init(empty + s, 1);
        }
        for (int b = 0; b < 2; b++) {
            tc::mbar_init(accf + b, 1);
            tc::mbar_init(acce + b, PJ_EPI_WARPS);
        }
        tc::mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        // an earlier wait gave up and nobody cleared the flag: skip the work
        *skip_slot = *(volatile int*)err;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(tc::saddr(tmem_slot)), "r"(C::TMC));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc::tc_before();
    __syncthreads();
    tc::tc_after();
    const uint32_t tmem = *tmem_slot;
    const bool skip = *skip_slot != 0;
    bool ok = !skip;
    const int tiles = skip ? 0 : my_tiles;

    // tile i of this CTA: first row and column, split, stages [k0, k1)
    struct Tile {
        int m0, n0, z, k0, k1;
    };
    auto tile_at = [&](int i) {
        int t = (int)blockIdx.x + i * (int)gridDim.x;
        Tile r;
        r.z = t % a.S;
        t /= a.S;
        const int per = PJ_GROUP_M * a.nt, g = t / per, rem = t - g * per;
        const int gm = min(PJ_GROUP_M, a.mt - g * PJ_GROUP_M);
        r.m0 = (g * PJ_GROUP_M + rem % gm) * 128;
        r.n0 = rem / gm * BN;
        r.k0 = (int)((int64_t)a.nk * r.z / a.S);
        r.k1 = (int)((int64_t)a.nk * (r.z + 1) / a.S);
        return r;
    };

    if (warp == 0) {
        if (lane == 0) {  // ---- TMA producer
            int g = 0;
            for (int i = 0; i < tiles && ok; i++) {
                const Tile t = tile_at(i);
                for (int ks = t.k0; ks < t.k1; ks++, g++) {
                    const int s = g % ST;
                    if (g >= ST && !tc::mbar_wait(empty + s, ((g / ST) - 1) & 1, err)) {
                        ok = false;
                        break;
                    }
                    unsigned char* sa = smem + s * C::STAGE;
                    unsigned char* sb = sa + C::A_BYTES;
                    tc::mbar_expect_tx(full + s, C::STAGE);
                    if constexpr (AMN) {
                        tc::tma_2d(sa, &a.amap, full + s, t.m0, ks * PJ_BK);
                        tc::tma_2d(sa + 8192, &a.amap, full + s, t.m0 + 64, ks * PJ_BK);
                    } else {
                        tc::tma_2d(sa, &a.amap, full + s, ks * PJ_BK, t.m0);
                    }
                    if constexpr (BMN) {
#pragma unroll
                        for (int c = 0; c < BN / 64; c++)
                            tc::tma_2d(sb + c * 8192, &a.bmap, full + s, t.n0 + 64 * c, ks * PJ_BK);
                    } else {
                        tc::tma_2d(sb, &a.bmap, full + s, ks * PJ_BK, t.n0);
                    }
                }
            }
            // the copies issued here land before the CTA may exit
            for (int j = max(0, g - ST); j < g; j++)
                if (!tc::mbar_wait_own(full + (j % ST), (j / ST) & 1, err)) ok = false;
        }
    } else if (warp == 1) {
        if (lane == 0) {  // ---- MMA issuer
            int g = 0;
            for (int i = 0; i < tiles && ok; i++) {
                const Tile t = tile_at(i);
                const int b = i & 1;
                if (i >= 2 && !tc::mbar_wait(acce + b, ((i >> 1) - 1) & 1, err)) {
                    ok = false;
                    break;
                }
                tc::tc_after();
                const uint32_t d = tmem + b * BN;
                for (int ks = t.k0; ks < t.k1; ks++, g++) {
                    const int s = g % ST;
                    if (!tc::mbar_wait(full + s, (g / ST) & 1, err)) {
                        ok = false;
                        break;
                    }
                    tc::tc_after();
                    const uint32_t sa = tc::saddr(smem + s * C::STAGE), sb = sa + C::A_BYTES;
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) {
                        const uint64_t ad = AMN ? tc::mn_sw128_desc(sa + kk * 2048, 8192) : tc::sw128_desc(sa) + 2 * kk;
                        const uint64_t bd = BMN ? tc::mn_sw128_desc(sb + kk * 2048, 8192) : tc::sw128_desc(sb) + 2 * kk;
                        tc::umma_ss(d, ad, bd, a.idesc, (ks > t.k0 || kk) ? 1u : 0u);
                    }
                    tc::umma_commit(empty + s);
                }
                if (!ok) break;
                tc::umma_commit(accf + b);
            }
            tc::umma_commit(done);  // also after an early exit: TMEM is freed after the MMAs
            if (!tc::mbar_wait_own(done, 0, err)) ok = false;
        }
    } else {
        // ---- epilogue
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lane_base = (uint32_t)(32 * q) << 16;
        const uint32_t stage = tc::saddr(smem + C::O_OFF + (warp - 2) * PJ_STAGE_OUT);
        const bool wide = a.S > 1 || a.e.out_f32;  // 4-byte results
        int nst = 0;                                // stores issued by this warp
        for (int i = 0; i < tiles; i++) {
            const Tile t = tile_at(i);
            const int b = i & 1;
            if (!tc::mbar_wait(accf + b, (i >> 1) & 1, err)) {
                ok = false;
                break;
            }
            tc::tc_after();
            const int row = t.m0 + 32 * q + lane;
            for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
                const int col = t.n0 + c;
                if (col >= a.N || t.m0 + 32 * q >= a.M) break;  // whole warps
                uint32_t r[32];
                tc::tmem_ld32_async(tmem + lane_base + b * BN + c, r);
                tc::tmem_ld_wait();
                float v[32];
#pragma unroll
                for (int k = 0; k < 32; k++) v[k] = __uint_as_float(r[k]);
                if (a.S == 1 && row < a.M) proj_epilogue32(v, a.e, row, col, min(32, a.N - col), a.N);
                // the staging tile is free once the store that read it last is done
                if (lane == 0) {
                    if (wide) tc::bulk_wait_read<0>();
                    else tc::bulk_wait_read<1>();
                }
                __syncwarp();
                uint32_t base = stage;
                if (wide) {  // 128-byte rows, 16-byte chunks swizzled by the row (mod 8)
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        tc::st_shared_v4(base + lane * 128 + ((k ^ (lane & 7)) << 4), __float_as_uint(v[4 * k]),
                                         __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]),
                                         __float_as_uint(v[4 * k + 3]));
                } else {     // 64-byte rows, chunks swizzled by row / 2 (mod 4)
                    base += (nst & 1) * 2048;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint4 p = pack8_16(v + 8 * k, a.e.bf16);
                        tc::st_shared_v4(base + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4), p.x, p.y, p.z, p.w);
                    }
                }
                tc::fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (a.S > 1) tc::tma_store_3d(&a.dmap, base, col, t.m0 + 32 * q, t.z);
                    else tc::tma_store_2d(&a.dmap, base, col, t.m0 + 32 * q);
                    tc::bulk_commit();
                }
                nst++;
            }
            tc::tc_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(acce + b);
        }
        if (lane == 0) tc::bulk_wait<0>();
    }
    tc::tc_before();
    const int bad = __syncthreads_or(!ok && (warp >= 2 || lane == 0));
    if (warp == 1) {
        tc::tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMC));
    }
    if (tid == 0 && bad) {
        *(volatile int*)a.err_host = 1;
        __threadfence_system();
    }
}

// Joins split-K partials: part [S][M][N] fp32.  A thread takes 32 columns of a row.
static __global__ void __launch_bounds__(128) proj_join_kernel(const float* __restrict__ part, const ProjEpi e, void* d, int M,
                                                        int N, int S) {
    const int per = (N + 31) / 32;
    const int64_t i = blockIdx.x * (int64_t)128 + threadIdx.x;
    if (i >= (int64_t)M * per) return;
    const int64_t row = i / per;
    const int col = (int)(i - row * per) * 32, nv = min(32, N - col);
    const int64_t at = row * N + col;
    float v[32];
#pragma unroll
    for (int k = 0; k < 32; k++) v[k] = 0.f;
    for (int z = 0; z < S; z++) {
        const float4* p = reinterpret_cast<const float4*>(part + (int64_t)z * M * N + at);
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (4 * k < nv) {
                const float4 f = p[k];
                v[4 * k] += f.x, v[4 * k + 1] += f.y, v[4 * k + 2] += f.z, v[4 * k + 3] += f.w;
            }
    }
    proj_epilogue32(v, e, row, col, nv, N);
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (8 * k < nv) {
            if (e.out_f32) {
                float4* o = reinterpret_cast<float4*>(static_cast<float*>(d) + at + 8 * k);
                o[0] = make_float4(v[8 * k], v[8 * k + 1], v[8 * k + 2], v[8 * k + 3]);
                o[1] = make_float4(v[8 * k + 4], v[8 * k + 5], v[8 * k + 6], v[8 * k + 7]);
            } else {
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(d) + at + 8 * k) = pack8_16(v + 8 * k, e.bf16);
            }
        }
}

// ------------------------------------------------------------------ host side

// Tile width and splits for an M x N product over nk stages, from the sizes
// alone (the workspace query has to agree with the call).
struct ProjPlan {
    int BN, mt, nt, S;
    int64_t ws_bytes;  // split-K partials
};
inline ProjPlan proj_plan(int64_t M, int64_t N, int64_t K) {
    ProjPlan p{};
    const int nk = (int)((K + PJ_BK - 1) / PJ_BK);
    p.mt = (int)((M + 127) / 128);
    p.BN = 256;
    while (p.BN > 64 && (int64_t)p.mt * ((N + p.BN - 1) / p.BN) < 148) p.BN /= 2;
    p.nt = (int)((N + p.BN - 1) / p.BN);
    const int64_t tiles = (int64_t)p.mt * p.nt;
    // split K until every SM has a tile, with at least 4 stages per split
    p.S = (int)std::max<int64_t>(1, std::min<int64_t>(148 / std::max<int64_t>(1, tiles), nk / 4));
    p.ws_bytes = p.S > 1 ? (int64_t)p.S * M * N * 4 : 0;
    return p;
}

inline bool proj_map_2d(CUtensorMap* m, CUtensorMapDataType type, int esize, const void* p, int64_t inner,
                        int64_t outer, int box_inner, int box_outer, CUtensorMapSwizzle sw) {
    auto enc = tensor_map_encoder();
    if (!enc) return false;
    cuuint32_t es[2] = {1, 1};
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    cuuint64_t strides[1] = {(cuuint64_t)(inner * esize)};
    cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer};
    return enc(m, type, 2, const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, bool AMN, bool BMN>
inline cudaError_t proj_launch_t(const ProjArgs& a, int sm_count, cudaStream_t st) {
    using C = PjCfg<BN>;
    auto kern = proj_kernel<BN, AMN, BMN>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::TOTAL);
    if (e != cudaSuccess) return e;
    const int64_t tiles = (int64_t)a.mt * a.nt * a.S;
    kern<<<(int)std::min<int64_t>(tiles, sm_count), PJ_THREADS, C::TOTAL, st>>>(a);
    return cudaGetLastError();
}

// D [M, N] = epilogue(A B^T), A [M, K] (AMN: stored [K, M]), B [N, K] (BMN: stored [K, N]).
template <bool AMN, bool BMN>
inline cudaError_t proj_gemm(const void* A, const void* B, void* D, int64_t M, int64_t N, int64_t K, const ProjEpi& e,
                             float* ws, int* err, int* err_host, int sm_count, cudaStream_t st) {
    const ProjPlan p = proj_plan(M, N, K);
    ProjArgs a{};
    a.e = e;
    a.M = (int)M;
    a.N = (int)N;
    a.nk = (int)((K + PJ_BK - 1) / PJ_BK);
    a.mt = p.mt;
    a.nt = p.nt;
    a.S = p.S;
    a.idesc = tc::idesc_f16(128, p.BN, e.bf16 != 0) | (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u);
    a.err = err;
    a.err_host = err_host;
    const CUtensorMapDataType t16 = e.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const auto sw128 = CU_TENSOR_MAP_SWIZZLE_128B;
    bool ok = AMN ? proj_map_2d(&a.amap, t16, 2, A, M, K, 64, PJ_BK, sw128)
                  : proj_map_2d(&a.amap, t16, 2, A, K, M, PJ_BK, 128, sw128);
    ok = ok && (BMN ? proj_map_2d(&a.bmap, t16, 2, B, N, K, 64, PJ_BK, sw128)
                    : proj_map_2d(&a.bmap, t16, 2, B, K, N, PJ_BK, p.BN, sw128));
    if (p.S > 1) {
        auto enc = tensor_map_encoder();
        cuuint32_t es[3] = {1, 1, 1}, box[3] = {32, 32, 1};
        cuuint64_t dims[3] = {(cuuint64_t)N, (cuuint64_t)M, (cuuint64_t)p.S};
        cuuint64_t strides[2] = {(cuuint64_t)N * 4, (cuuint64_t)(M * N) * 4};
        ok = ok && enc(&a.dmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, ws, dims, strides, box, es,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, sw128, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    } else if (e.out_f32) {
        ok = ok && proj_map_2d(&a.dmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, D, N, M, 32, 32, sw128);
    } else {
        ok = ok && proj_map_2d(&a.dmap, t16, 2, D, N, M, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
    }
    if (!ok) return cudaErrorInvalidValue;
    cudaError_t rc = p.BN == 64    ? proj_launch_t<64, AMN, BMN>(a, sm_count, st)
                     : p.BN == 128 ? proj_launch_t<128, AMN, BMN>(a, sm_count, st)
                                   : proj_launch_t<256, AMN, BMN>(a, sm_count, st);
    if (rc != cudaSuccess || p.S == 1) return rc;
    const int64_t threads = M * ((N + 31) / 32);
    proj_join_kernel<<<ceil_div(threads, 128), 128, 0, st>>>(ws, e, D, (int)M, (int)N, p.S);
    return cudaGetLastError();
}

}  // namespace rwkv
