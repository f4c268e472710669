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
// Tile = 128 rows of D (TMEM lanes) x 128 columns on one CTA, or 256 x 256 on a pair
// of CTAs (cta_group::2: each holds 128 rows of A and of B and its 128 rows of D; the
// first issues the MMAs for both), K in stages of 64.  A persistent CTA or pair
// walks its tiles; the accumulator of tile t lives in TMEM half (t & 1), so the
// epilogue of one tile runs beside the MMAs of the next.
//   warp 0      TMA producer, ST stages; a pair's loads count on the first CTA's
//               barriers
//   warp 1      TMEM owner; one thread issues 4 tcgen05.mma (K=16) per stage and
//               commits the stage / the tile (to both CTAs)
//   warps 2 ..  epilogue, 16 warps (a sigmoid over 4093 x 2048 sums of 96 takes 21 us
//               with 8): TMEM lane quadrant (warp & 3) = 32 rows of D, an equal share
//               of the columns per 4 warps, 32 columns at a time in two halves.
//               With a checkpoint 8 warps, a thread holding the 32 columns of a
//               group, so that its largest |z| needs no exchange (16 such warps
//               spill: 16384 x 8192 over 2048 takes 462 us, with 8 436).  Results go
//               through a swizzled 32 x 32 tile in shared memory and leave by TMA
//               store (full 64-byte row pieces, clipped at the tensor's end).
// Tiles are walked in groups of 8 row blocks, so that the CTAs at work at one
// time share a few row blocks of A and a few of B in L2.
//
// Whole waves of tiles (148 at a time, 74 on pairs) run as they are; the tiles of the last,
// partial wave are split S ways along K, so that the SMs left over share them
// (a product of fewer tiles than SMs is all last wave).  A split writes its fp32
// sums as a tile into the workspace, and the join kernel adds the splits in order
// (deterministic) and runs the epilogue.
//
// An accumulator takes 32768 terms at most; longer sums split every tile along K.  A
// step of the tensor core cuts its 16 products and the accumulator off at 2^-25 of the
// largest one's binade and their sum at 2^-23, toward zero (measured), so that a step
// may lose 5 2^-23 of the sum and sums of one sign drift: 2^19 terms in [1/4, 1] come
// out 3.0e-3 low from one accumulator, 1.6e-4 from 16.  The join's additions round to
// nearest.
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
constexpr int PJ_SMS = 148;
constexpr int PJ_CHAIN = 32768;    // terms that one accumulator takes
constexpr int PJ_OUT_BYTES = 32 * 1024;  // output staging, shared by the epilogue warps

// Which epilogue a kernel has, at compile time: one that can do everything keeps
// the registers of everything alive (16384 x 8192 over 96 takes 270 us with a
// plain result in it, 72 us in its own kernel).
enum : int {
    PJ_PLAIN = 0,  // the sums
    PJ_FWD = 1,    // bias, z, activation, residual
    PJ_FWD_CK = 2, // and the checkpoint of z
    PJ_GRAD = 3,   // times act'(pre), addend
};
// FAST, with tanh and sigmoid: the fast functions (act_t), for results of 16 bits.  In
// kernels of their own: both kinds of functions in one cost the 16-bit results (4093 x
// 2048 over 96, dX with tanh: 16.2 -> 19.8 us).  The exact ones take 24.3 us there, the
// forward's sigmoid 21.7 (fast 16.1), its tanh 17.5 (17.6).

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

    bool fast() const { return !out_f32 || (act != RWKV_ACT_TANH && act != RWKV_ACT_SIGMOID); }
    int kind() const {
        return grad ? PJ_GRAD : codes ? PJ_FWD_CK : bias || z || add || act != RWKV_ACT_NONE ? PJ_FWD : PJ_PLAIN;
    }
};

struct ProjArgs {
    CUtensorMap amap, bmap;
    CUtensorMap dmap;   // D, box {32, 32}, or {16, 32} in fp32
    CUtensorMap cmap;   // checkpoint codes, box {32, 32} (N % 16 == 0)
    CUtensorMap pmap;   // the splits' tiles {BN, 128 units} fp32, box {16, 32}
    ProjEpi e;
    int M, N, nk;       // D's size, K stages
    int mt, nt;         // tiles along M and N
    int full, F, S;     // tiles of whole waves, splits of each; splits of each of the others
    int ctma;           // codes leave by TMA
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

__device__ __forceinline__ int64_t proj_group(int64_t row, int col, int N) {
    return row * ((N + CK_GROUP - 1) / CK_GROUP) + col / CK_GROUP;
}
// 32 codes at p, the first nv (a multiple of 8) of which exist; one row in two
// starts 8 bytes off a 16-byte boundary where N % 16 == 8.
__device__ __forceinline__ void proj_load_codes(const int8_t* p, int nv, uint4* w) {
    if (nv == 32 && ((uintptr_t)p & 15) == 0) {
        w[0] = reinterpret_cast<const uint4*>(p)[0];
        w[1] = reinterpret_cast<const uint4*>(p)[1];
    } else {
        const uint2 z = make_uint2(0, 0), *q = reinterpret_cast<const uint2*>(p);
        const uint2 a = nv > 0 ? q[0] : z, b = nv > 8 ? q[1] : z, c = nv > 16 ? q[2] : z, d = nv > 24 ? q[3] : z;
        w[0] = make_uint4(a.x, a.y, b.x, b.y);
        w[1] = make_uint4(c.x, c.y, d.x, d.y);
    }
}
__device__ __forceinline__ void proj_store_codes(int8_t* p, int nv, const uint32_t* w) {
    uint2* q = reinterpret_cast<uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (8 * i < nv) q[i] = make_uint2(w[2 * i], w[2 * i + 1]);
}

// A warp's other inputs of 32 rows by 32 columns, as read.
struct ProjAux {
    uint4 add[4];  // residual / addend, 16 bits
    uint4 pre[4];  // pre-activation of row (lane), or its 32 codes in the first two
    uint32_t exp;  // and their exponent
    float bias;    // of column (lane)
};
__device__ __forceinline__ const uint4* proj_add16(const ProjEpi& e, int64_t row, int col, int N) {
    return reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(e.add) + row * N + col);
}
__device__ __forceinline__ const uint4* proj_pre16(const ProjEpi& e, int64_t row, int col, int N) {
    return reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(e.pre) + row * N + col);
}
// The rows row0 .. by the columns col ..: the pre-activation and its exponent by
// row; the bias by column, broadcast from there when it is added; and the residual
// as the rows (lane / 4) + 8 i, piece lane % 4 of 16 bytes, so that an instruction
// covers 8 rows' 64 bytes (a row per lane takes 4 times as many wavefronts from the
// port that also feeds the tensor core: 16384 x 8192 over 2048 with a residual 493
// us, this way 451, without 391).
template <int KIND>
__device__ __forceinline__ void proj_load_aux(const ProjEpi& e, int row0, int col, int nv, int M, int N, int lane,
                                              ProjAux& x) {
    if constexpr (KIND == PJ_PLAIN) return;
    const int64_t row = row0 + lane;
    if (KIND == PJ_GRAD && row < M) {
        if (e.pre_codes) {
            proj_load_codes(e.pre_codes + row * N + col, nv, x.pre);
            x.exp = e.pre_exps[proj_group(row, col, N)];
        } else {
            const uint4* p = proj_pre16(e, row, col, N);
#pragma unroll
            for (int i = 0; i < 4; i++) x.pre[i] = 8 * i < nv ? p[i] : make_uint4(0, 0, 0, 0);
        }
    }
    if (KIND != PJ_GRAD && e.bias) x.bias = lane < nv ? load_param(e.bias, e.bias_dtype, col + lane) : 0.f;
    if (e.add && !e.out_f32) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = row0 + lane / 4 + 8 * i;
            x.add[i] = r < M && 8 * (lane % 4) < nv ? __ldcs(proj_add16(e, r, col, N) + lane % 4) : make_uint4(0, 0, 0, 0);
        }
    }
}
__device__ __forceinline__ void floats8_16(const uint4& r, int bf16, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = unpack2(w[i], bf16);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// The epilogue of W columns col .. of one row up to the residual; the first nv (a
// multiple of 8) columns exist; v holds the sums, 0 in columns that do not exist,
// with the bias added; pre / exp as in ProjAux.  PJ_FWD_CK: the codes go to w and the
// exponent byte is returned, for the caller to store; the group is the thread's own
// 32 columns, or (W = 8) those of four neighbouring lanes.
template <int KIND, bool FAST, int W>
__device__ __forceinline__ uint32_t proj_epilogue(float* v, const ProjEpi& e, const uint4* pre, uint32_t pexp,
                                                  int64_t row, int col, int nv, int N, uint32_t* w) {
    uint32_t exp = 0;
    if constexpr (KIND == PJ_FWD_CK) {
        static_assert(W == 32 || W == 8, "whole groups");
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < W; i++) top = max(top, abs_bits(v[i]));
        if constexpr (W == 8) {
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        }
        exp = ck_exponent(top);
        const float inv = ck_inv_scale(exp);
#pragma unroll
        for (int i = 0; i < W / 4; i++) w[i] = ck_pack4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv);
    }
    if ((KIND == PJ_FWD || KIND == PJ_FWD_CK) && e.z) {
#pragma unroll
        for (int i = 0; i < W / 8; i++)
            if (8 * i < nv)
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(e.z) + row * N + col + 8 * i) =
                    pack8_16(v + 8 * i, e.bf16);
    }
    if constexpr (KIND == PJ_GRAD) {
        const float s = e.pre_codes ? ck_scale(pexp) : 0.f;
        with_act(e.act, [&]<int ACT>() {
#pragma unroll
            for (int i = 0; i < W / 8; i++) {
                float p[8];
                if (e.pre_codes) {
                    const uint4 c = pre[i / 2];
                    ck_unpack4(i % 2 ? c.z : c.x, s, p);
                    ck_unpack4(i % 2 ? c.w : c.y, s, p + 4);
                } else {
                    floats8_16(pre[i], e.bf16, p);
                }
#pragma unroll
                for (int k = 0; k < 8; k++) v[8 * i + k] *= act_grad_t<ACT, FAST>(p[k]);
            }
        });
    } else if constexpr (KIND != PJ_PLAIN) {
        if (e.act != RWKV_ACT_NONE)
            with_act(e.act, [&]<int ACT>() {
#pragma unroll
                for (int i = 0; i < W; i++) v[i] = act_t<ACT, FAST>(v[i]);
            });
    }
    return exp;
}
// fp32 residual, read where it is added (a residual stream kept in fp32)
template <int W>
__device__ __forceinline__ void proj_add_f32(float* v, const ProjEpi& e, int64_t at, int nv) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(e.add) + at);
#pragma unroll
    for (int i = 0; i < W / 4; i++)
        if (4 * i < nv) {
            const float4 f = p[i];
            v[4 * i] += f.x, v[4 * i + 1] += f.y, v[4 * i + 2] += f.z, v[4 * i + 3] += f.w;
        }
}

namespace tc {
template <int W>
__device__ __forceinline__ void tmem_ld_async(uint32_t taddr, uint32_t* r) {
    if constexpr (W == 32)
        tmem_ld32_async(taddr, r);
    else
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src),
                 "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
    return r;
}
__device__ __forceinline__ void st_shared_u4(uint32_t addr, const uint4& v) { st_shared_v4(addr, v.x, v.y, v.z, v.w); }
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// at most N of this thread's bulk stores still read their shared memory
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
// Two SMs on one tile (cta_group::2).  The loads are plain ones into this CTA's own
// shared memory; their bytes are counted on the barrier at `bar` (a shared::cluster
// address), the first CTA's.
__device__ __forceinline__ void tma_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(saddr(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void umma_ss_pair(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// arrives at the same barrier of both CTAs once the MMAs issued so far are done
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            saddr(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
}  // namespace tc

// CG: CTAs on a tile of 128 CG rows; each holds 128 rows of A and BN / CG of B.
template <int BN, int CG, int KIND>
struct PjCfg {
    static constexpr int A_BYTES = 128 * 128;       // 128 rows x 64 k, 16 bits
    static constexpr int B_BYTES = BN / CG * 128;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int EW = KIND == PJ_FWD_CK ? 8 : 16;  // epilogue warps
    static constexpr int W = KIND == PJ_FWD_CK ? 32 : 16;  // columns a thread holds
    static constexpr int EC = BN / (EW / 4);               // columns of each warp
    static constexpr int THREADS = 64 + 32 * EW;
    static constexpr int SLOT = PJ_OUT_BYTES / EW;         // staging bytes per warp
    static constexpr int ST = 192 * 1024 / STAGE;
    static constexpr int NBAR = 2 * ST + 5;
    static constexpr int O_OFF = ST * STAGE;        // output staging
    static constexpr int B_OFF = O_OFF + PJ_OUT_BYTES;
    static constexpr int T_OFF = B_OFF + NBAR * 8;
    static constexpr int TOTAL = T_OFF + 16 + 1024;
    static constexpr int TMC = 2 * BN;
    static_assert(TOTAL <= 227 * 1024, "shared memory per CTA");
    static_assert(BN == 128 || BN == 256, "TMEM allocation is a power of two; shares of 32 columns");
    static_assert(ST >= 3, "pipeline depth");
    static_assert(CG == 1 || BN == 256, "a pair of CTAs takes 256 x 256");
};

// AMN / BMN: the operand is MN-major.
template <int BN, int CG, bool AMN, bool BMN, int KIND, bool FAST>
__global__ void __launch_bounds__(PjCfg<BN, CG, KIND>::THREADS, 1) proj_kernel(const __grid_constant__ ProjArgs a) {
    using C = PjCfg<BN, CG, KIND>;
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
    const int rank = CG == 2 ? (int)blockIdx.x & 1 : 0;  // within the pair; rank 0 issues the MMAs
    const int first = (int)blockIdx.x / CG, stride = (int)gridDim.x / CG;
    const int whole = a.full * a.F, units = whole + (a.mt * a.nt - a.full) * a.S;
    const int my_tiles = first < units ? (units - 1 - first) / stride + 1 : 0;
    int* err = a.err;
    // rank 0's barriers, as both CTAs address them
    auto lead = [&](uint64_t* bar) { return CG == 2 ? tc::map_rank(tc::saddr(bar), 0) : tc::saddr(bar); };

    if (tid == 64) {
        tc::prefetch_map(&a.amap);
        tc::prefetch_map(&a.bmap);
        tc::prefetch_map(&a.dmap);
    }
    if (tid == 0) {
        for (int s = 0; s < ST; s++) {
            tc::mbar_init(full + s, 1);
            tc::mbar_init(empty + s, 1);
        }
        for (int b = 0; b < 2; b++) {
            tc::mbar_init(accf + b, 1);
            tc::mbar_init(acce + b, CG * C::EW);
        }
        tc::mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        // an earlier wait gave up and nobody cleared the flag: skip the work
        *skip_slot = *(volatile int*)err;
    }
    if (warp == 1) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(tc::saddr(tmem_slot)), "r"(C::TMC));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(tc::saddr(tmem_slot)), "r"(C::TMC));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    tc::tc_before();
    __syncthreads();
    if constexpr (CG == 2) tc::cluster_sync();  // both CTAs' barriers exist
    tc::tc_after();
    pdl_wait();  // everything before read only this kernel's arguments and the flag
    const uint32_t tmem = *tmem_slot;
    const bool skip = *skip_slot != 0;
    bool ok = !skip;
    const int tiles = skip ? 0 : my_tiles;

    // unit i of this CTA: first row and column, stages [k0, k1), and for a split
    // the row of its tile in the workspace (-1: a whole tile)
    struct Tile {
        int m0, n0, k0, k1, part;
    };
    auto tile_at = [&](int i) {
        const int u = first + i * stride;
        Tile r;
        int t = u, z = 0, S = 1, slot = -1;
        if (u < whole) {
            if (a.F > 1) {  // a split of every tile, then the next: neighbours share their K
                S = a.F;
                z = u / a.full;
                t = u - z * a.full;
                slot = u;
            }
        } else {
            S = a.S;
            const int j = (u - whole) / S;
            z = u - whole - j * S;
            t = a.full + j;
            slot = a.F > 1 ? u : u - whole;
        }
        r.k0 = 0;
        r.k1 = a.nk;
        r.part = -1;
        if (slot >= 0) {
            r.k0 = (int)((int64_t)a.nk * z / S);
            r.k1 = (int)((int64_t)a.nk * (z + 1) / S);
            r.part = (slot * CG + rank) * 128;
        }
        const int per = PJ_GROUP_M * a.nt, g = t / per, rem = t - g * per;
        const int gm = min(PJ_GROUP_M, a.mt - g * PJ_GROUP_M);
        r.m0 = ((g * PJ_GROUP_M + rem % gm) * CG + rank) * 128;
        r.n0 = rem / gm * BN;
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
                    const uint32_t bar = lead(full + s);
                    if (rank == 0) tc::mbar_expect_tx(full + s, CG * C::STAGE);
                    auto load = [&](void* dst, const CUtensorMap* map, int x, int y) {
                        if constexpr (CG == 2) tc::tma_2d_pair(dst, map, bar, x, y);
                        else tc::tma_2d(dst, map, full + s, x, y);
                    };
                    const int nb = t.n0 + rank * (BN / CG);
                    if constexpr (AMN) {
                        load(sa, &a.amap, t.m0, ks * PJ_BK);
                        load(sa + 8192, &a.amap, t.m0 + 64, ks * PJ_BK);
                    } else {
                        load(sa, &a.amap, ks * PJ_BK, t.m0);
                    }
                    if constexpr (BMN) {
#pragma unroll
                        for (int c = 0; c < BN / CG / 64; c++) load(sb + c * 8192, &a.bmap, nb + 64 * c, ks * PJ_BK);
                    } else {
                        load(sb, &a.bmap, ks * PJ_BK, nb);
                    }
                }
            }
            // the copies issued here land before the CTA may exit (a pair's second CTA
            // counts them on the first's barriers: its own are done when every MMA is,
            // and after a wait that gave up it allows them 2 ms)
            if (rank == 0) {
                for (int j = max(0, g - ST); j < g; j++)
                    if (!tc::mbar_wait_own(full + (j % ST), (j / ST) & 1, err)) ok = false;
            } else if (!ok) {
                for (const uint64_t t0 = tc::gtime(); tc::gtime() - t0 < 2000000;) __nanosleep(1000);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {  // ---- MMA issuer (of a pair, the first CTA's)
            auto commit = [&](uint64_t* bar) {
                if constexpr (CG == 2) tc::umma_commit_pair(bar);
                else tc::umma_commit(bar);
            };
            int g = 0;
            for (int i = 0; i < tiles && ok && rank == 0; i++) {
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
                        if constexpr (CG == 2) tc::umma_ss_pair(d, ad, bd, a.idesc, (ks > t.k0 || kk) ? 1u : 0u);
                        else tc::umma_ss(d, ad, bd, a.idesc, (ks > t.k0 || kk) ? 1u : 0u);
                    }
                    commit(empty + s);
                }
                if (!ok) break;
                commit(accf + b);
            }
            if (rank == 0) {
                commit(done);  // also after an early exit: TMEM is freed after the MMAs
                if (!tc::mbar_wait_own(done, 0, err)) ok = false;
            }
        }
    } else {
        // ---- epilogue
        const int q = warp & 3, c0 = (warp - 2) / 4 * C::EC;
        const uint32_t lane_base = (uint32_t)(32 * q) << 16;
        const uint32_t base = tc::saddr(smem + C::O_OFF + (warp - 2) * C::SLOT);
        constexpr int W = C::W;
        // 64-byte rows (32 values of 16 bits, or 16 fp32), 16-byte chunks swizzled by row / 2
        auto slot = [&](int r, int k) { return base + r * 64 + ((k ^ ((r >> 1) & 3)) << 4); };
        for (int i = 0; i < tiles; i++) {
            const Tile t = tile_at(i);
            const int b = i & 1, row0 = t.m0 + 32 * q, row = row0 + lane;
            const bool part = t.part >= 0, wide = part || a.e.out_f32;  // 4-byte results
            const bool epi = KIND != PJ_PLAIN && !part, add16 = epi && a.e.add && !a.e.out_f32;
            // this warp's columns c0 .. c1 of the tile that exist, in whole steps of 32
            const int c1 = row0 >= a.M ? c0 : min(c0 + C::EC, a.N - t.n0);
            ProjAux aux;
            if (epi && c0 < c1) proj_load_aux<KIND>(a.e, row0, t.n0 + c0, min(32, a.N - t.n0 - c0), a.M, a.N, lane, aux);
            if (!tc::mbar_wait(accf + b, (i >> 1) & 1, err)) {
                ok = false;
                break;
            }
            tc::tc_after();
            uint32_t exps = 0;
            for (int c = c0; c < c1; c += 32) {
                const int col = t.n0 + c, nv = min(32, a.N - col);
                if (epi && c > c0) proj_load_aux<KIND>(a.e, row0, col, nv, a.M, a.N, lane, aux);
                uint32_t codes[8];
#pragma unroll
                for (int h = 0; h < 32 / W; h++) {
                    uint32_t r[W];
                    tc::tmem_ld_async<W>(tmem + lane_base + b * BN + c + h * W, r);
                    if (h == 0 || wide) {
                        // the staging tile is free once the store that read it last is done
                        if (lane == 0) tc::bulk_wait_read<0>();
                        __syncwarp();
                    }
                    if (h == 0 && add16) {
#pragma unroll
                        for (int k = 0; k < 4; k++) tc::st_shared_u4(slot(lane / 4 + 8 * k, lane % 4), aux.add[k]);
                        __syncwarp();
                    }
                    tc::tmem_ld_wait();
                    float v[W];
#pragma unroll
                    for (int k = 0; k < W; k++) v[k] = __uint_as_float(r[k]);
                    if (epi) {
                        if (KIND != PJ_GRAD && a.e.bias) {
#pragma unroll
                            for (int k = 0; k < W; k++) v[k] += __shfl_sync(0xffffffffu, aux.bias, h * W + k);
                        }
                        if (row < a.M) {
                            // W / 8 vectors of a dense pre-activation, half as many of codes
                            const uint4 p[2] = {a.e.pre_codes ? aux.pre[h * W / 16] : aux.pre[h * W / 8],
                                                aux.pre[(h * W / 8 + 1) % 4]};
                            exps |= proj_epilogue<KIND, FAST, W>(v, a.e, p, aux.exp, row, col + h * W, nv - h * W, a.N, codes)
                                    << ((c - c0) / 4);
                            if (a.e.add && a.e.out_f32)
                                proj_add_f32<W>(v, a.e, (int64_t)row * a.N + col + h * W, nv - h * W);
                        }
                    }
                    if (wide) {  // 16 columns to a box
#pragma unroll
                        for (int k = 0; k < W / 4; k++)
                            tc::st_shared_v4(slot(lane, k % 4) + k / 4 * 2048, __float_as_uint(v[4 * k]),
                                             __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]),
                                             __float_as_uint(v[4 * k + 3]));
                        tc::fence_async_smem();
                        __syncwarp();
                        if (lane == 0) {
#pragma unroll
                            for (int k = 0; k < W / 16; k++) {
                                if (part) tc::tma_store_2d(&a.pmap, base + k * 2048, c + h * W + 16 * k, t.part + 32 * q);
                                else if (h * W + 16 * k < nv) tc::tma_store_2d(&a.dmap, base + k * 2048, col + h * W + 16 * k, row0);
                            }
                            tc::bulk_commit();
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < W / 8; k++) {
                            const uint32_t at = slot(lane, h * W / 8 + k);
                            if (add16) {
                                float f[8];
                                floats8_16(tc::ld_shared_v4(at), a.e.bf16, f);
#pragma unroll
                                for (int j = 0; j < 8; j++) v[8 * k + j] += f[j];
                            }
                            tc::st_shared_u4(at, pack8_16(v + 8 * k, a.e.bf16));
                        }
                    }
                }
                if constexpr (KIND == PJ_FWD_CK) {
                    // codes: 32-byte rows behind a 16-bit tile, or straight to memory
                    if (epi && a.ctma && !wide) {
                        tc::st_shared_v4(base + 2048 + lane * 32, codes[0], codes[1], codes[2], codes[3]);
                        tc::st_shared_v4(base + 2048 + lane * 32 + 16, codes[4], codes[5], codes[6], codes[7]);
                    } else if (epi && row < a.M) {
                        proj_store_codes(a.e.codes + (int64_t)row * a.N + col, nv, codes);
                    }
                }
                if (!wide) {
                    tc::fence_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tc::tma_store_2d(&a.dmap, base, col, row0);
                        if (KIND == PJ_FWD_CK && a.ctma) tc::tma_store_2d(&a.cmap, base + 2048, col, row0);
                        tc::bulk_commit();
                    }
                }
            }
            tc::tc_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) tc::mbar_arrive_cluster(lead(acce + b));
                else tc::mbar_arrive(acce + b);
            }
            if (KIND == PJ_FWD_CK && epi && row < a.M && c0 < c1) {
                // the exponents of this warp's groups, together where they are a word
                uint8_t* p = a.e.exps + proj_group(row, t.n0 + c0, a.N);
                const int n = (c1 - c0 + 31) / 32;
                if (n == 4 && ((uintptr_t)p & 3) == 0) {
                    *reinterpret_cast<uint32_t*>(p) = exps;
                } else {
                    for (int k = 0; k < n; k++) p[k] = (uint8_t)(exps >> (8 * k));
                }
            }
        }
        if (lane == 0) tc::bulk_wait_read<0>();  // the staging tiles may go; the stores end with the grid
    }
    tc::tc_before();
    const int bad = __syncthreads_or(!ok && (warp >= 2 || lane == 0));
    if constexpr (CG == 2) {
        // the second CTA's epilogue has seen its last tile: the MMAs are as good as done
        if (rank == 1 && warp == 1 && lane == 0) tc::mbar_wait_own(done, 0, err);
        __syncwarp();
        tc::cluster_sync();  // neither CTA's memory is in use by the other
    }
    if (warp == 1) {
        tc::tc_after();
        if constexpr (CG == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMC));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMC));
    }
    if (tid == 0 && bad) {
        *(volatile int*)a.err_host = 1;
        __threadfence_system();
    }
}

struct ProjJoin {
    const float* part;  // [F > 1: split full + tile, behind them][(tile - full) S + split][BM][BN]
    ProjEpi e;
    void* d;
    int M, N, mt, nt, full, F, S, BM, BN;
};
// Joins the splits of the tiles full .., with F > 1 of all: thread i takes 8 columns of a row of a
// tile (four neighbouring lanes hold a checkpoint group), the splits' loads all in
// flight, 16 at most.
template <int KIND, bool FAST>
__device__ __forceinline__ void proj_join(const ProjJoin& a, int64_t i) {
    const int per = a.BN / 8;
    const int piece = (int)(i % per), r = (int)(i / per % a.BM);
    const int64_t j = i / per / a.BM;  // the grid covers whole tiles
    const int t = (a.F > 1 ? 0 : a.full) + (int)j;
    const int pg = PJ_GROUP_M * a.nt, g = t / pg, rem = t - g * pg;
    const int gm = min(PJ_GROUP_M, a.mt - g * PJ_GROUP_M);
    const int64_t row = (int64_t)(g * PJ_GROUP_M + rem % gm) * a.BM + r;
    const int col = rem / gm * a.BN + 8 * piece;
    const bool in = row < a.M && col < a.N;
    if (__all_sync(0xffffffffu, !in)) return;
    const int64_t at = row * a.N + col;
    float v[8] = {};
    if (in) {
        // n splits, the first in `slot`, the others `step` further each
        auto add = [&](int64_t slot, int n, int step) {
            const float* p = a.part + (slot * a.BM + r) * a.BN + 8 * piece;
#pragma unroll 8
            for (int z = 0; z < n; z++) {
                const float4* q = reinterpret_cast<const float4*>(p + (int64_t)z * step * a.BM * a.BN);
                const float4 x = q[0], y = q[1];
                v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
                v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
            }
        };
        if (a.F == 1) add(j * a.S, a.S, 1);
        else if (t < a.full) add(t, a.F, a.full);
        else add((int64_t)a.full * a.F + (int64_t)(t - a.full) * a.S, a.S, 1);
    }
    if ((KIND == PJ_FWD || KIND == PJ_FWD_CK) && a.e.bias && in) {
        float b[8];
        load_params<8>(a.e.bias, a.e.bias_dtype, col, b);
#pragma unroll
        for (int m = 0; m < 8; m++) v[m] += b[m];
    }
    uint4 pre[1] = {};
    uint32_t pexp = 0, codes[2];
    if (KIND == PJ_GRAD && in) {
        if (a.e.pre_codes) {
            const uint2 w = *reinterpret_cast<const uint2*>(a.e.pre_codes + at);
            pre[0] = make_uint4(w.x, w.y, 0, 0);
            pexp = a.e.pre_exps[proj_group(row, col, a.N)];
        } else {
            pre[0] = *proj_pre16(a.e, row, col, a.N);
        }
    }
    if (KIND != PJ_FWD_CK && !in) return;
    const uint32_t exp = proj_epilogue<KIND, FAST, 8>(v, a.e, pre, pexp, row, col, in ? 8 : 0, a.N, codes);
    if (!in) return;
    if constexpr (KIND == PJ_FWD_CK) {
        *reinterpret_cast<uint2*>(a.e.codes + at) = make_uint2(codes[0], codes[1]);
        if (piece % 4 == 0) a.e.exps[proj_group(row, col, a.N)] = (uint8_t)exp;
    }
    if (KIND != PJ_PLAIN && a.e.add) {
        if (a.e.out_f32) {
            proj_add_f32<8>(v, a.e, at, 8);
        } else {
            float f[8];
            floats8_16(*proj_add16(a.e, row, col, a.N), a.e.bf16, f);
#pragma unroll
            for (int m = 0; m < 8; m++) v[m] += f[m];
        }
    }
    if (a.e.out_f32) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.d) + at);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.d) + at) = pack8_16(v, a.e.bf16);
    }
}
// Column sums of dY beside the joined tiles (rwkv_projection_dw's db): blocks from
// `first` on take 32 columns each, warp w the slices (or, of a short dY, its rows) w, w +
// 4, ...; fixed order.
struct ColJoin {
    const float* part;  // [slices][N], or NULL:
    const void* dy;     // [slices][N] in 16 bits, the rows themselves
    float* out;
    int N, slices, bf16;
};
constexpr int PJ_JOIN_T = 128;
template <int KIND, bool FAST>
__global__ void __launch_bounds__(PJ_JOIN_T) proj_join_kernel(const ProjJoin a, const ColJoin c, int first) {
    pdl_wait();
    if ((int)blockIdx.x < first) {
        proj_join<KIND, FAST>(a, blockIdx.x * (int64_t)PJ_JOIN_T + threadIdx.x);
        return;
    }
    __shared__ float red[PJ_JOIN_T / 32][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, col = ((int)blockIdx.x - first) * 32 + lane;
    float s = 0.f;
    if (col < c.N) {
        if (c.part) {
#pragma unroll 8
            for (int k = w; k < c.slices; k += PJ_JOIN_T / 32) s += c.part[(int64_t)k * c.N + col];
        } else {
#pragma unroll 8
            for (int k = w; k < c.slices; k += PJ_JOIN_T / 32)
                s += load_param(c.dy, c.bf16 ? RWKV_BF16 : RWKV_F16, (int64_t)k * c.N + col);
        }
    }
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && col < c.N) c.out[col] = red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane];
}

// ------------------------------------------------------------------ host side

// Tile, whole tiles and splits of the others for an M x N product, from the sizes
// alone (the workspace query has to agree with the call).
//  - 256 x 256 on a pair of CTAs where such tiles fill the pairs: half the shared
//    memory traffic per product of 128 x 256 on one CTA (dX 8192 x 8192 over 2048
//    186 us against 204, dW 2048 x 8192 over 8192 165 against 190).
//  - 128 x 128 otherwise, and for products too short to hide a wide tile's epilogue
//    (K <= 512).
//  - The tiles past the last whole wave are split the way that the estimate below
//    finds shortest: a stage of 64 takes 0.45 us on a pair and 0.27 us on a CTA (an SM's
//    share of L2 bandwidth); joining takes 3.5 us and writes and reads each split's
//    tile once in L2 (8 TB/s).
//  - More than PJ_CHAIN terms: the tiles of whole waves are split too, into as few as
//    that takes (2304 x 2304 over 65536: 416 us, in one drifting accumulator 408; over
//    2^19 3340 and 3179).
struct ProjPlan {
    int CG, BN, mt, nt, full, F, S;
    int64_t ws_bytes;  // the splits' tiles
    int BM() const { return 128 * CG; }
    int64_t parts() const { return (F > 1 ? (int64_t)full * F : 0) + (S > 1 ? ((int64_t)mt * nt - full) * S : 0); }
    // the parts' rows in the workspace are counted in 31 bits
    bool ok() const { return parts() * BM() < 1ll << 31; }
};
inline ProjPlan proj_plan(int64_t M, int64_t N, int64_t K) {
    ProjPlan p{};
    const int nk = (int)((K + PJ_BK - 1) / PJ_BK);
    const bool pair = K > 512 && (M + 255) / 256 * ((N + 255) / 256) >= PJ_SMS / 2;
    p.CG = pair ? 2 : 1;
    p.BN = pair ? 256 : 128;
    p.mt = (int)((M + p.BM() - 1) / p.BM());
    p.nt = (int)((N + p.BN - 1) / p.BN);
    const int wave = PJ_SMS / p.CG, tiles = p.mt * p.nt, rem = tiles % wave;
    p.full = tiles - rem;
    p.F = p.S = (int)((K + PJ_CHAIN - 1) / PJ_CHAIN);
    double best = 0.0;
    for (int S = p.F; rem && S <= std::max(p.F, 16) && (S == p.F || nk / S >= 2); S++) {
        const double stage = pair ? 0.45 : 0.27, bytes = 2.0 * rem * S * p.BM() * p.BN * 4;
        const double us = (double)(((int64_t)rem * S + wave - 1) / wave) * ((nk + S - 1) / S) * stage +
                          (S > 1 ? 3.5 + bytes / 8e6 : 0.0);
        if (S == p.F || us < best) best = us, p.S = S;
    }
    if (p.S == 1) p.full = tiles;
    p.ws_bytes = p.parts() * p.BM() * p.BN * 4;
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

template <int BN, int CG, bool AMN, bool BMN, int KIND, bool FAST>
inline cudaError_t proj_launch_t(const ProjArgs& a, int sm_count, bool after_own, cudaStream_t st) {
    using C = PjCfg<BN, CG, KIND>;
    auto kern = proj_kernel<BN, CG, AMN, BMN, KIND, FAST>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::TOTAL);
    if (e != cudaSuccess) return e;
    const int units = a.full * a.F + (a.mt * a.nt - a.full) * a.S;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min(units, sm_count / CG) * CG);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::TOTAL;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    cfg.attrs = at;
    if (CG == 2) {
        at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[cfg.numAttrs].val.clusterDim.x = 2;
        at[cfg.numAttrs].val.clusterDim.y = 1;
        at[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    if (after_own) {
        at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    return cudaLaunchKernelEx(&cfg, kern, a);
}

// D [M, N] = epilogue(A B^T), A [M, K] (AMN: stored [K, M]), B [N, K] (BMN: stored
// [K, N]); with `cols` the column sums beside it.  after_own: the launch before
// this one on the stream is this call's own, of a kernel without TMEM, so that this
// one may start its set-up beside it.
template <bool AMN, bool BMN, int KIND, bool FAST>
inline cudaError_t proj_gemm(const void* A, const void* B, void* D, int64_t M, int64_t N, int64_t K, const ProjEpi& e,
                             float* ws, int* err, int* err_host, int sm_count, cudaStream_t st, bool after_own = false,
                             const ColJoin* cols = nullptr) {
    const ProjPlan p = proj_plan(M, N, K);
    if (!p.ok()) return cudaErrorInvalidValue;
    ProjArgs a{};
    a.e = e;
    a.M = (int)M;
    a.N = (int)N;
    a.nk = (int)((K + PJ_BK - 1) / PJ_BK);
    a.mt = p.mt;
    a.nt = p.nt;
    a.full = p.full;
    a.F = p.F;
    a.S = p.S;
    a.idesc = tc::idesc_f16(p.BM(), p.BN, e.bf16 != 0) | (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u);
    a.err = err;
    a.err_host = err_host;
    const CUtensorMapDataType t16 = e.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const auto sw128 = CU_TENSOR_MAP_SWIZZLE_128B;
    bool ok = AMN ? proj_map_2d(&a.amap, t16, 2, A, M, K, 64, PJ_BK, sw128)
                  : proj_map_2d(&a.amap, t16, 2, A, K, M, PJ_BK, 128, sw128);
    ok = ok && (BMN ? proj_map_2d(&a.bmap, t16, 2, B, N, K, 64, PJ_BK, sw128)
                    : proj_map_2d(&a.bmap, t16, 2, B, K, N, PJ_BK, 128, sw128));
    ok = ok && (e.out_f32 ? proj_map_2d(&a.dmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, D, N, M, 16, 32, CU_TENSOR_MAP_SWIZZLE_64B)
                          : proj_map_2d(&a.dmap, t16, 2, D, N, M, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B));
    a.ctma = KIND == PJ_FWD_CK && N % 16 == 0;
    if (a.ctma)
        ok = ok && proj_map_2d(&a.cmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, e.codes, N, M, 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (p.ws_bytes)
        ok = ok && proj_map_2d(&a.pmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, ws, p.BN, p.parts() * p.BM(), 16, 32,
                               CU_TENSOR_MAP_SWIZZLE_64B);
    if (!ok) return cudaErrorInvalidValue;
    const cudaError_t rc = p.CG == 2 ? proj_launch_t<256, 2, AMN, BMN, KIND, FAST>(a, sm_count, after_own, st)
                                     : proj_launch_t<128, 1, AMN, BMN, KIND, FAST>(a, sm_count, after_own, st);
    if (rc != cudaSuccess || (!p.ws_bytes && !cols)) return rc;
    const ProjJoin j{ws, e, D, (int)M, (int)N, p.mt, p.nt, p.full, p.F, p.S, p.BM(), p.BN};
    const int joined = p.mt * p.nt - (p.F > 1 ? 0 : p.full);
    const int first = ceil_div((int64_t)joined * p.BM() * (p.BN / 8), PJ_JOIN_T);
    const ColJoin c = cols ? *cols : ColJoin{};
    return launch_pdl(proj_join_kernel<KIND, FAST>, dim3(first + ceil_div(c.N, 32)), dim3(PJ_JOIN_T), 0, st, j, c, first);
}

}  // namespace rwkv
