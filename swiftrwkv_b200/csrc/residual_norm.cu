// The residual norm: a branch added to the residual stream, through dropout and
// scaled, and the sum normed for the next branch, in one pass.
//
//   forward   s = x + scale drop(branch), y = (s - mean) rstd w + b
//   backward  h = (s - mean) rstd, g = dy w:
//             dx = rstd (g - mean(g) - h mean(g h)) + dres, dbranch = scale drop(dx),
//             dw = sum_n dy h, db = sum_n dy
//
// HBM's part is 4 tensors forward (x, branch, s, y) and 5 backward (dy, s, dres, dx,
// dbranch), 1 + 1/32 bytes per element for s as a checkpoint.  s is normed and
// checkpointed in fp32, before its rounding.  Beside that both are bound by the issue
// of instructions: a vector of 8 elements takes 16 bytes per tensor, and dropout 72
// (forward) to 94 instructions (58 draw its bits, the others apply them), so that the kernels
// count them: pairs of fp32 in one instruction, several vectors or rows to a thread's share of
// a row's sums.
#include <algorithm>

#include "ckpt8.cuh"
#include "copy_async.cuh"
#include "f32x2.cuh"
#include "param_join.cuh"
#include "philox.cuh"
#include "resident.cuh"

namespace rwkv {
namespace {

template <int MODE, typename T>
__device__ __forceinline__ void branch_part(Pairs<T>& v, const DropKey& key, uint64_t i, const Dropout& d) {
    if constexpr (MODE == DROP_NONE) {
#pragma unroll
        for (int k = 0; k < Pairs<T>::P; k++) v[k] = mul2(v[k], both(d.scale));
    } else {
        drop_vector<MODE, Pairs<T>::VE>(v.floats(), key, i, d);
    }
}

// ------------------------------------------------------------------- forward

struct RnFwdArgs {
    const void *x, *branch, *w, *b;
    void *sum, *y;
    float *mean, *rstd;
    int8_t* codes;
    uint8_t* exps;
    int wdtype, rows, D, G;
    float eps;
    Dropout drop;
};

// the largest magnitude of three, NaN if one is
__device__ __forceinline__ float top3(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// four codes as ck_pack4, where none is clipped and the group holds no NaN
__device__ __forceinline__ uint32_t pack4_within(const float2& a, const float2& b, float inv) {
    const float2 m = both(12582912.f), p = fma2(a, both(inv), m), q = fma2(b, both(inv), m);
    return __byte_perm(__byte_perm(__float_as_uint(p.x), __float_as_uint(p.y), 0x0040),
                       __byte_perm(__float_as_uint(q.x), __float_as_uint(q.y), 0x0040), 0x5410);
}

// The codes of a vector, and its group's exponent byte (32 / VE neighbouring threads).
// Clipping takes a third of the packing; only groups whose largest rounds up to 128 (or
// that stand for NaN) need it.
template <typename T>
__device__ __forceinline__ void checkpoint(const Pairs<T>& s, int8_t* codes, uint8_t* exps, bool in, bool first) {
    constexpr int VE = Pairs<T>::VE;
    float t = top3(s[0].x, s[0].y, s[1].x);
    if constexpr (VE == 8) t = top3(top3(t, s[1].y, s[2].x), top3(s[2].y, s[3].x, s[3].y), t);
    else t = top3(t, s[1].y, t);
    uint32_t top = __float_as_uint(t);
#pragma unroll
    for (int o = 1; o < CK_GROUP / VE; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t e = ck_exponent(top);
    const float inv = ck_inv_scale(e);
    uint32_t c[VE / 4];
    if (__uint_as_float(top) * inv < 127.5f) {
#pragma unroll
        for (int k = 0; k < VE / 4; k++) c[k] = pack4_within(s[2 * k], s[2 * k + 1], inv);
    } else {
#pragma unroll
        for (int k = 0; k < VE / 4; k++) c[k] = ck_pack4(s[2 * k].x, s[2 * k].y, s[2 * k + 1].x, s[2 * k + 1].y, inv);
    }
    if (!in) return;
    if constexpr (VE == 8) *reinterpret_cast<uint2*>(codes) = make_uint2(c[0], c[VE / 4 - 1]);
    else *reinterpret_cast<uint32_t*>(codes) = c[0];
    if (first) *exps = (uint8_t)e;
}

// the sum of a vector, in halves, so that equal values add exactly
template <typename T>
__device__ __forceinline__ float vector_sum(const Pairs<T>& v) {
    float2 h = add2(v[0], v[1]);
    if constexpr (Pairs<T>::P == 4) h = add2(h, add2(v[2], v[3]));
    return h.x + h.y;
}

// Which of two means a row takes: that of its values, whose sum rounds by the size of
// the partial sums, or one from the values' distances to a pivot, exact for constant rows
// and better than the other where the mean is large against the spread.
__device__ __forceinline__ bool is_far(float mean, float variance) { return variance * 64.f < mean * mean; }

// TPR threads take R rows, at most NV vectors of a row per thread: vector j of thread t
// is t + j TPR.  A block is TPR threads, or 128 where a row is a warp's or a part's of one:
// its statistics then are sums between lanes, the pivot the values' mean.
//
// Otherwise statistics of a row come from one round of sums and one barrier: each warp
// takes the mean of its first lane's first vector as a pivot p and leaves p, sum(s - p),
// sum (s - p)^2 and sum(s); around the first warp's pivot these join to mean and variance.
// A pivot is the mean of VE elements of the row, so that (p - mean)^2 <= M / VE with M the
// row's centred sum of squares: what cancels in a warp's share of n elements is n M / VE at
// most, a fraction of M for rows without outliers.  A row in which more than 3 M cancels
// (whose pivots hold outliers: up to 400 2^-24 of M were lost), or whose sums are past fp32, is
// summed once more around its mean, by its own sums alone: the same next to any other row.
// 42 M elements bf16, 1024 to 6144 channels: within 0.5 us of the kernel without it, 3 to 8 us
// more where every row starts with outliers.
template <typename T, int TPR, int NV, int R, bool CK, int MODE>
__global__ void __launch_bounds__(TPR > 32 ? TPR : 128, 1) rn_fwd_kernel(const __grid_constant__ RnFwdArgs a) {
    constexpr int VE = Vec16<T>::N, P = VE / 2;
    const int t = threadIdx.x % TPR, lane = threadIdx.x & 31;
    const int nvec = a.D / VE;
    const int64_t row0 = (TPR > 32 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (128 / TPR) + threadIdx.x / TPR) * R;
    const int64_t at = row0 * nvec;  // in vectors
    const uint4* const x = static_cast<const uint4*>(a.x) + at;
    const uint4* const br = static_cast<const uint4*>(a.branch) + at;
    Pairs<T> s[R][NV];
    {
        uint4 rx[R][NV], rb[R][NV];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int v = t + j * TPR;
                const bool in = v < nvec && row0 + r < a.rows;
                rx[r][j] = in ? __ldcs(x + r * nvec + v) : make_uint4(0, 0, 0, 0);
                rb[r][j] = in ? __ldcs(br + r * nvec + v) : make_uint4(0, 0, 0, 0);
            }
        const DropKey key = drop_key<MODE>(a.drop);
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int v = t + j * TPR;
                const bool in = v < nvec && row0 + r < a.rows;
                Pairs<T> q;
                s[r][j].unpack(rx[r][j]);
                q.unpack(rb[r][j]);
                branch_part<MODE>(q, key, (uint64_t)(at + r * nvec + v), a.drop);
#pragma unroll
                for (int k = 0; k < P; k++) s[r][j][k] = add2(s[r][j][k], q[k]);
                if (in) __stcs(static_cast<uint4*>(a.sum) + at + r * nvec + v, s[r][j].pack());
                if constexpr (CK)
                    checkpoint(s[r][j], a.codes + (at + r * nvec + v) * VE,
                               a.exps + (row0 + r) * a.G + v / (CK_GROUP / VE), in, lane % (CK_GROUP / VE) == 0);
            }
    }
    float mean[R], rstd[R];
    const float inv_d = 1.f / (float)a.D;
    if constexpr (TPR <= 32) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            float2 sum = both(0.f), d1 = both(0.f), d2 = both(0.f);
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int k = 0; k < P; k++) sum = add2(sum, s[r][j][k]);
            const float m = group_sum<TPR>(sum.x + sum.y) * inv_d;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const float2 n = both(t + j * TPR < nvec ? -m : 0.f);  // zeros beyond the row's end
#pragma unroll
                for (int k = 0; k < P; k++) {
                    const float2 d = add2(s[r][j][k], n);
                    d1 = add2(d1, d);
                    d2 = fma2(d, d, d2);
                }
            }
            const float u = group_sum<TPR>(d1.x + d1.y) * inv_d, q = group_sum<TPR>(d2.x + d2.y);
            const bool far = is_far(m, q * inv_d);
            mean[r] = far ? m + u : m;
            rstd[r] = far ? fmaxf(q - u * u * (float)a.D, 0.f) : q;
        }
    } else {
        constexpr int NW = TPR / 32;
        __shared__ alignas(16) float red[R][NW][4];  // of each warp: pivot p, sums of s - p, (s - p)^2, s
        const int warp = t >> 5;
        float sums[4 * R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float pivot = __shfl_sync(0xffffffffu, vector_sum(s[r][0]), 0) * (1.f / VE);
            if (lane == 0) red[r][warp][0] = pivot;
            float2 sum = both(0.f), d1 = both(0.f), d2 = both(0.f);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const float2 n = both(t + j * TPR < nvec ? -pivot : 0.f);  // zeros beyond the row's end
#pragma unroll
                for (int k = 0; k < P; k++) {
                    const float2 d = add2(s[r][j][k], n);
                    sum = add2(sum, s[r][j][k]);
                    d1 = add2(d1, d);
                    d2 = fma2(d, d, d2);
                }
            }
            sums[4 * r] = 0.f;
            sums[4 * r + 1] = d1.x + d1.y;
            sums[4 * r + 2] = d2.x + d2.y;
            sums[4 * r + 3] = sum.x + sum.y;
        }
        const float p = lanes_sum<4 * R>(sums, lane);
        const int which = lane / (8 / R) % 4;
        if (lane % (8 / R) == 0 && which) red[lane / (32 / R)][warp][which] = p;
        __syncthreads();
        // elements of warp w's share of a row
        auto count = [&](int w) {
            int n = 0;
#pragma unroll
            for (int j = 0; j < NV; j++) n += max(0, min(32, nvec - w * 32 - j * TPR));
            return (float)(n * VE);
        };
        // of the sum of squares around the pivots, beside one around the mean of q
        auto most = [](float q) { return fminf(4.f * q, 3.4e38f); };
        bool far[R], again[R], any = false;  // alike in all threads, which join the same sums in the same order
#pragma unroll
        for (int r = 0; r < R; r++) {
            float u = 0.f, q = 0.f, sum = 0.f;
            bool within;
            const float p0 = red[r][0][0];
            if constexpr (NW <= 5) {  // every thread joins the warps' sums
                float e[NW], d1[NW], c[NW];
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const float4 f = *reinterpret_cast<const float4*>(red[r][w]);
                    e[w] = f.x - p0, d1[w] = f.y, q += f.z, sum += f.w, c[w] = count(w);
                    u += fmaf(c[w], e[w], d1[w]);
                }
                u *= inv_d;
                const float around = q;
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const float f = e[w] - u;
                    q = fmaf(f, fmaf(c[w], f, 2.f * d1[w]), q);
                }
                within = around <= most(q);
            } else {  // lane % NW has a warp's
                const float4 f = *reinterpret_cast<const float4*>(red[r][lane % NW]);
                const float e = f.x - p0, c = count(lane % NW);
                u = fmaf(c, e, f.y);
                sum = f.w;
#pragma unroll
                for (int m = NW / 2; m > 0; m >>= 1) {
                    u += __shfl_xor_sync(0xffffffffu, u, m);
                    sum += __shfl_xor_sync(0xffffffffu, sum, m);
                }
                u *= inv_d;
                q = fmaf(e - u, fmaf(c, e - u, 2.f * f.y), f.z);
#pragma unroll
                for (int m = NW / 2; m > 0; m >>= 1) q += __shfl_xor_sync(0xffffffffu, q, m);
                within = !__any_sync(0xffffffffu, !(f.z * (float)NW <= most(q)));
            }
            far[r] = is_far(p0 + u, q * inv_d);
            mean[r] = far[r] ? p0 + u : sum * inv_d;
            rstd[r] = q < 0.f ? 0.f : q;  // (a NaN passes)
            again[r] = !within;
            any |= again[r];
        }
        if (any) {
            __shared__ float around[R][NW][2];  // of each warp: sums of s - mean, (s - mean)^2
#pragma unroll
            for (int r = 0; r < R; r++) {
                float2 d1 = both(0.f), d2 = both(0.f);
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    const float2 n = both(t + j * TPR < nvec ? -mean[r] : 0.f);
#pragma unroll
                    for (int k = 0; k < P; k++) {
                        const float2 d = add2(s[r][j][k], n);
                        d1 = add2(d1, d);
                        d2 = fma2(d, d, d2);
                    }
                }
                sums[2 * r] = d1.x + d1.y;
                sums[2 * r + 1] = d2.x + d2.y;
            }
            const float p = lanes_sum<2 * R>(sums, lane);
            if (lane % (16 / R) == 0) around[lane / (32 / R)][warp][lane / (16 / R) % 2] = p;
            __syncthreads();
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (!again[r]) continue;
                float u = 0.f, q = 0.f;
#pragma unroll 1
                for (int w = 0; w < NW; w++) u += around[r][w][0], q += around[r][w][1];
                u *= inv_d;
                if (far[r]) mean[r] += u;
                q = fmaf(-u * u, (float)a.D, q);
                rstd[r] = q < 0.f ? 0.f : q;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        rstd[r] = 1.f / sqrtf(rstd[r] * inv_d + a.eps);
        if (t == 0 && a.mean && row0 + r < a.rows) {
            a.mean[row0 + r] = mean[r];
            a.rstd[row0 + r] = rstd[r];
        }
    }
    uint4* const y = static_cast<uint4*>(a.y) + at;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int v = t + j * TPR;
        if (v >= nvec) continue;
        Pairs<T> w, b;
        load_params<VE>(a.w, a.wdtype, v * VE, w.floats());
        load_params<VE>(a.b, a.wdtype, v * VE, b.floats());
#pragma unroll
        for (int r = 0; r < R; r++) {
            Pairs<T> o;
#pragma unroll
            for (int k = 0; k < P; k++) o[k] = fma2(mul2(add2(s[r][j][k], both(-mean[r])), both(rstd[r])), w[k], b[k]);
            if (row0 + r < a.rows) __stcs(y + r * nvec + v, o.pack());
        }
    }
}

// ------------------------------------------------------------------ backward

struct RnBwdArgs {
    const void *dy, *s;
    const int8_t* codes;
    const uint8_t* exps;
    const void* w;
    const float *mean, *rstd;
    const void* dres;
    void *dx, *dbranch;
    float* part;  // [blocks][2][D] sums of dy h and dy over the block's rows, or NULL
    int wdtype, rows, D, G;
    Dropout drop;
};

constexpr int RN_STAGES = 3;

// A block walks over rows; thread t owns the vectors t + j blockDim.x of every row, so
// that the sums over rows stay in registers until the end.  dy, s (or its codes) and dres
// run RN_STAGES - 1 rows ahead through a ring in shared memory that is private to each
// thread (cp.async); one barrier per row, for its two sums (buffers alternating).
//
// 16384 x 2560 bf16: 65 us without dropout, dense or from a checkpoint (floors 64 and 58),
// 74 and 81 with it.  Bound then by issue: 281 to 305 instructions per vector (187 to 217
// without dropout), at 56 % of the slots with the 13 warps per SM that the registers leave (one
// vector a thread, 20 warps: 83 with a checkpoint and dropout, 73 dense without; more warps of
// fewer registers load the weights again and again: 81 to 100).
template <typename T, bool CK, int MODE, int NV, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) rn_bwd_kernel(const __grid_constant__ RnBwdArgs a) {
    constexpr int VE = Vec16<T>::N, P = VE / 2;
    extern __shared__ uint4 ring[];  // [stage][dy | s | dres][NV][thread]
    __shared__ float red[2][16][2];
    using Codes = std::conditional_t<VE == 8, uint2, uint32_t>;  // of one vector
    const int t = threadIdx.x, nt = blockDim.x, warp = t >> 5, lane = t & 31, nw = nt >> 5;
    const int nvec = a.D / VE;
    pdl_trigger();
    const float inv_d = 1.f / (float)a.D;
    const DropKey key = drop_key<MODE>(a.drop);
    Pairs<T> w[NV], sw[NV], sb[NV];
    bool has[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int v = t + j * nt;
        has[j] = v < nvec;
        load_params<VE>(a.w, a.wdtype, (int64_t)(has[j] ? v : 0) * VE, w[j].floats());
#pragma unroll
        for (int k = 0; k < P; k++) sw[j][k] = sb[j][k] = both(0.f);
    }
    const int stage_n = 3 * NV * nt;
    auto slot = [&](int base, int part, int j) { return ring + base + (part * NV + j) * nt; };
    const int64_t vstep = (int64_t)gridDim.x * nvec;  // in vectors
    int64_t at = (int64_t)blockIdx.x * nvec + t, fat = at;
    auto fetch = [&](int64_t row, int base) {
        if (row < a.rows) {
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (has[j]) {
                    const int64_t i = fat + j * nt;
                    copy_async<16>(slot(base, 0, j), static_cast<const uint4*>(a.dy) + i);
                    if constexpr (CK) copy_async<VE>(slot(base, 1, j), reinterpret_cast<const Codes*>(a.codes) + i);
                    else copy_async<16>(slot(base, 1, j), static_cast<const uint4*>(a.s) + i);
                    if (a.dres) copy_async<16>(slot(base, 2, j), static_cast<const uint4*>(a.dres) + i);
                }
        }
        copy_commit();
        fat += vstep;
    };
    // a row's statistics and exponents, one row ahead in registers (as 4-byte copies
    // into the ring they cost 10 us of 70)
    float nmean, nrstd;
    uint32_t ex[NV], nex[NV];
    auto fetch_small = [&](int64_t next) {
        const uint32_t row = min((uint32_t)next, (uint32_t)a.rows - 1);  // of no use past the end
        nmean = a.mean[row];
        nrstd = a.rstd[row];
        if constexpr (CK)
#pragma unroll
            for (int j = 0; j < NV; j++)
                nex[j] = has[j] ? a.exps[(int64_t)row * a.G + (t + j * nt) / (CK_GROUP / VE)] : 0u;
    };
#pragma unroll
    for (int i = 0; i < RN_STAGES - 1; i++) fetch(blockIdx.x + (int64_t)i * gridDim.x, t + i * stage_n);
    fetch_small(blockIdx.x);
    int cur = t, put = t + (RN_STAGES - 1) * stage_n, buf = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, at += vstep, buf ^= 1) {
        fetch(row + (int64_t)(RN_STAGES - 1) * gridDim.x, put);
        copy_wait<RN_STAGES - 1>();
        const float mean = nmean, rstd = nrstd;
        if constexpr (CK)
#pragma unroll
            for (int j = 0; j < NV; j++) ex[j] = nex[j];
        fetch_small(row + gridDim.x);
        // pass 1: h, the sums over the row (g, g h) and over the rows (dy h, dy)
        Pairs<T> h[NV];
        float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (!has[j]) continue;
            Pairs<T> d;
            d.unpack(*slot(cur, 0, j));
            // s - mean in one rounding: no multiple of rstd cancels where |mean| is large
            if constexpr (CK) {
                const uint32_t* c = reinterpret_cast<const uint32_t*>(slot(cur, 1, j));
                ck_codes4(c[0], h[j].floats());
                if constexpr (VE == 8) ck_codes4(c[1], h[j].floats() + 4);
                const float2 scale = both(ck_scale(ex[j]));
#pragma unroll
                for (int k = 0; k < P; k++) h[j][k] = fma2(h[j][k], scale, both(-mean));
            } else {
                h[j].unpack(*slot(cur, 1, j));
#pragma unroll
                for (int k = 0; k < P; k++) h[j][k] = add2(h[j][k], both(-mean));
            }
#pragma unroll
            for (int k = 0; k < P; k++) {
                h[j][k] = mul2(h[j][k], both(rstd));
                const float2 g = mul2(d[k], w[j][k]);
                s1 = add2(s1, g);
                s2 = fma2(g, h[j][k], s2);
                sw[j][k] = fma2(d[k], h[j][k], sw[j][k]);
                sb[j][k] = add2(sb[j][k], d[k]);
            }
        }
        // over the warp: the sum of g ends up in lanes 0..15, that of g h in 16..31
        float sums[2] = {s1.x + s1.y, s2.x + s2.y};
        const float p = lanes_sum<2>(sums, lane);
        if ((lane & 15) == 0) red[buf][warp][lane >> 4] = p;
        __syncthreads();
        float tot = (lane & 15) < nw ? red[buf][lane & 15][lane >> 4] : 0.f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, o);
        tot *= inv_d * -rstd;
        // pass 2: dx = rstd (g - m1 - h m2) + dres
        const float2 c0 = both(__shfl_sync(0xffffffffu, tot, 0)), c1 = both(__shfl_sync(0xffffffffu, tot, 16));
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (!has[j]) continue;
            Pairs<T> d, o;
            d.unpack(*slot(cur, 0, j));
            if (a.dres) {
                o.unpack(*slot(cur, 2, j));
#pragma unroll
                for (int k = 0; k < P; k++) o[k] = add2(o[k], c0);
            } else {
#pragma unroll
                for (int k = 0; k < P; k++) o[k] = c0;
            }
#pragma unroll
            for (int k = 0; k < P; k++) o[k] = fma2(mul2(d[k], w[j][k]), both(rstd), fma2(h[j][k], c1, o[k]));
            const int64_t i = at + j * nt;
            __stcs(static_cast<uint4*>(a.dx) + i, o.pack());
            branch_part<MODE>(o, key, (uint64_t)i, a.drop);
            __stcs(static_cast<uint4*>(a.dbranch) + i, o.pack());
        }
        put = cur;
        cur = cur == t + (RN_STAGES - 1) * stage_n ? t : cur + stage_n;
    }
    copy_wait<0>();
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (!has[j]) continue;
        float* o = part + (int64_t)(t + j * nt) * VE;
#pragma unroll
        for (int k = 0; k < P; k += 2) {
            *reinterpret_cast<float4*>(o + 2 * k) = make_float4(sw[j][k].x, sw[j][k].y, sw[j][k + 1].x, sw[j][k + 1].y);
            *reinterpret_cast<float4*>(o + a.D + 2 * k) = make_float4(sb[j][k].x, sb[j][k].y, sb[j][k + 1].x, sb[j][k + 1].y);
        }
    }
}

// Short rows (at most 32 NV vectors): TPR lanes a row, 128 / TPR rows of a block at a time,
// the next ones read ahead into registers; no barrier until the columns' sums of a block's
// rows meet.
template <typename T, bool CK, int MODE, int TPR, int NV>
__global__ void __launch_bounds__(128) rn_bwd_short_kernel(const __grid_constant__ RnBwdArgs a) {
    constexpr int VE = Vec16<T>::N, P = VE / 2;
    using Codes = std::conditional_t<VE == 8, uint2, uint32_t>;
    extern __shared__ float2 sums[];  // [warp][dy h | dy][NV][P][TPR]
    const int t = threadIdx.x % TPR, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nvec = a.D / VE;
    pdl_trigger();
    const float inv_d = 1.f / (float)a.D;
    const DropKey key = drop_key<MODE>(a.drop);
    Pairs<T> w[NV], sw[NV], sb[NV];
    bool has[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        has[j] = t + j * TPR < nvec;
        load_params<VE>(a.w, a.wdtype, (has[j] ? t + j * TPR : 0) * VE, w[j].floats());
#pragma unroll
        for (int k = 0; k < P; k++) sw[j][k] = sb[j][k] = both(0.f);
    }
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4 ndy[NV], ns[NV], nres[NV];
    float nmean = 0.f, nrstd = 0.f;
    uint32_t nex[NV];
    // what lies beyond a row's or the tensor's end reads as zeros
    auto fetch = [&](int64_t row) {
        const bool in = row < a.rows;
        nmean = in ? a.mean[row] : 0.f;
        nrstd = in ? a.rstd[row] : 0.f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t i = row * nvec + t + j * TPR;
            const bool h = in && has[j];
            ndy[j] = h ? __ldcs(static_cast<const uint4*>(a.dy) + i) : zero;
            nres[j] = h && a.dres ? __ldcs(static_cast<const uint4*>(a.dres) + i) : zero;
            ns[j] = zero;
            if constexpr (CK) {
                nex[j] = h ? a.exps[row * a.G + (t + j * TPR) / (CK_GROUP / VE)] : 0u;
                if (h) *reinterpret_cast<Codes*>(&ns[j]) = __ldcs(reinterpret_cast<const Codes*>(a.codes) + i);
            } else {
                if (h) ns[j] = __ldcs(static_cast<const uint4*>(a.s) + i);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * (128 / TPR);
    int64_t row = (int64_t)blockIdx.x * (128 / TPR) + threadIdx.x / TPR;
    const int steps = (int)((a.rows + step - 1) / step);  // of every row's lanes alike, for the shuffles
    fetch(row);
    for (int n = 0; n < steps; n++, row += step) {
        const float mean = nmean, rstd = nrstd;
        uint4 dy[NV], res[NV];
        Pairs<T> h[NV];
        float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            Pairs<T> d;
            const float sub = has[j] ? -mean : 0.f;  // h is 0 beyond the row's end: no -mean rstd that overflows
            dy[j] = ndy[j], res[j] = nres[j];
            d.unpack(dy[j]);
            if constexpr (CK) {
                ck_codes4(ns[j].x, h[j].floats());
                if constexpr (VE == 8) ck_codes4(ns[j].y, h[j].floats() + 4);
                const float2 scale = both(ck_scale(nex[j]));
#pragma unroll
                for (int k = 0; k < P; k++) h[j][k] = fma2(h[j][k], scale, both(sub));
            } else {
                h[j].unpack(ns[j]);
#pragma unroll
                for (int k = 0; k < P; k++) h[j][k] = add2(h[j][k], both(sub));
            }
#pragma unroll
            for (int k = 0; k < P; k++) {  // (dy is 0 beyond the row's end, and adds nothing)
                h[j][k] = mul2(h[j][k], both(rstd));
                const float2 g = mul2(d[k], w[j][k]);
                s1 = add2(s1, g);
                s2 = fma2(g, h[j][k], s2);
                sw[j][k] = fma2(d[k], h[j][k], sw[j][k]);
                sb[j][k] = add2(sb[j][k], d[k]);
            }
        }
        fetch(row + step);
        const float2 c0 = both(group_sum<TPR>(s1.x + s1.y) * inv_d * -rstd);
        const float2 c1 = both(group_sum<TPR>(s2.x + s2.y) * inv_d * -rstd);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (!has[j] || row >= a.rows) continue;
            Pairs<T> d, o;
            d.unpack(dy[j]);
            o.unpack(res[j]);
#pragma unroll
            for (int k = 0; k < P; k++)
                o[k] = fma2(mul2(d[k], w[j][k]), both(rstd), fma2(h[j][k], c1, add2(o[k], c0)));
            const int64_t i = row * nvec + t + j * TPR;
            __stcs(static_cast<uint4*>(a.dx) + i, o.pack());
            branch_part<MODE>(o, key, (uint64_t)i, a.drop);
            __stcs(static_cast<uint4*>(a.dbranch) + i, o.pack());
        }
    }
    if (!a.part) return;
    // over the warp's rows, then the block's warps, in a fixed order
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int k = 0; k < P; k++)
#pragma unroll
            for (int o = TPR; o < 32; o <<= 1) {
                const float2 f = make_float2(__shfl_xor_sync(0xffffffffu, sw[j][k].x, o), __shfl_xor_sync(0xffffffffu, sw[j][k].y, o));
                const float2 g = make_float2(__shfl_xor_sync(0xffffffffu, sb[j][k].x, o), __shfl_xor_sync(0xffffffffu, sb[j][k].y, o));
                sw[j][k] = add2(sw[j][k], f);
                sb[j][k] = add2(sb[j][k], g);
            }
    constexpr int N = NV * P * TPR;  // pairs of one sum
    if (lane < TPR) {
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int k = 0; k < P; k++) {
                sums[warp * 2 * N + (j * P + k) * TPR + t] = sw[j][k];
                sums[(warp * 2 + 1) * N + (j * P + k) * TPR + t] = sb[j][k];
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * N; i += 128) {
        float2 f = sums[i];
#pragma unroll
        for (int v = 1; v < 4; v++) f = add2(f, sums[v * 2 * N + i]);
        const int which = i / N, jk = i % N / TPR, lane_of = i % TPR, v = lane_of + jk / P * TPR;
        if (v < nvec)
            *reinterpret_cast<float2*>(a.part + ((int64_t)blockIdx.x * 2 + which) * a.D + v * VE + jk % P * 2) = f;
    }
}

// ------------------------------------------------------------------- launches

constexpr int RN_VECTORS = 512 * 3;
// Blocks of the backward at most (the partial sums of the parameters are as many rows):
// four per SM, more of fewer threads (40960 x 1024 bf16 with dropout: 74 us, four per SM 89).
int most_blocks(int D) { return 148 * std::min(8, std::max(4, 8192 / D)); }

template <typename T, int TPR, int NV, int R, bool CK, int MODE>
void launch_fwd(const RnFwdArgs& a, cudaStream_t st) {
    constexpr int BT = TPR > 32 ? TPR : 128;
    rn_fwd_kernel<T, TPR, NV, R, CK, MODE><<<ceil_div(a.rows, R * (BT / TPR)), BT, 0, st>>>(a);
}

template <typename T, bool CK, int MODE>
int forward(const RnFwdArgs& a, cudaStream_t st) {
    const int nvec = a.D / Vec16<T>::N;
    // As few threads as hold a row in registers: a row's sums and the weights' loads are
    // shared by more of its vectors.  42 M elements bf16 with dropout (floor 51 us), 64 to
    // 6144 channels: 52 to 57 us.  On the other sides of these borders: 64 channels by 64
    // threads a row 389 us, 256 99, 768 by 64 of two vectors 62, 6144 by 256 of four 66.  2560
    // channels by 64 threads of five and 160 of two: 62 and 60, with a checkpoint 65 and 67,
    // without dropout 55 and 56 (by a warp of ten 57, 71 with dropout).  A checkpoint changes
    // none of them: results are the same with and without.
    if (nvec <= 8) launch_fwd<T, 8, 1, 2, CK, MODE>(a, st);
    else if (nvec <= 16) launch_fwd<T, 16, 1, 2, CK, MODE>(a, st);
    else if (nvec <= 32) launch_fwd<T, 32, 1, 2, CK, MODE>(a, st);
    else if (nvec <= 32 * 2) launch_fwd<T, 32, 2, 2, CK, MODE>(a, st);
    else if (nvec <= 32 * 3) launch_fwd<T, 32, 3, 1, CK, MODE>(a, st);
    else if (nvec <= 64 * 2) launch_fwd<T, 64, 2, 2, CK, MODE>(a, st);
    else if (nvec <= 64 * 3) launch_fwd<T, 64, 3, 2, CK, MODE>(a, st);
    else if (nvec <= 64 * 4) launch_fwd<T, 64, 4, 1, CK, MODE>(a, st);
    else if (nvec <= 64 * 5) launch_fwd<T, 64, 5, 1, CK, MODE>(a, st);
    else if (nvec <= 128 * 4) launch_fwd<T, 128, 4, 1, CK, MODE>(a, st);
    else if (nvec <= 256 * 3) launch_fwd<T, 256, 3, 1, CK, MODE>(a, st);
    else if (nvec <= 256 * 4) launch_fwd<T, 256, 4, 1, CK, MODE>(a, st);
    else launch_fwd<T, 512, 3, 1, CK, MODE>(a, st);
    return check_launch("rn_fwd_kernel");
}

template <typename T, bool CK, int MODE, int NV, int MAXT, int MINB>
cudaError_t launch_bwd(const RnBwdArgs& a, int* blocks, cudaStream_t st) {
    auto kern = rn_bwd_kernel<T, CK, MODE, NV, MAXT, MINB>;
    const int nt = ceil_div(ceil_div(a.D / Vec16<T>::N, NV), 32) * 32;
    constexpr int PER_T = RN_STAGES * 3 * NV * 16;  // shared memory of a thread
    // as many blocks as are resident, so that they all run in one wave
    static ResidentBlocks resident;
    int per_sm;
    const cudaError_t e = resident.get(kern, nt, PER_T * nt, PER_T * MAXT, &per_sm);
    if (e != cudaSuccess) return e;
    // and two rows each, but 128 blocks, whose sums are quickly joined: 257 x 2560 bf16 6.4 us with
    // its join, one row each 7.5, four 7.7; 64 rows by one each 4.5, by two 5.4
    const int busy = std::max(std::min(a.rows, 128), ceil_div(a.rows, 2));
    *blocks = std::min(busy, std::min(148 * per_sm, most_blocks(a.D)));
    kern<<<*blocks, nt, PER_T * nt, st>>>(a);
    return cudaGetLastError();
}

template <typename T, bool CK, int MODE, int TPR, int NV>
cudaError_t launch_short(const RnBwdArgs& a, int* blocks, cudaStream_t st) {
    // four rows or more for each row's lanes
    *blocks = std::min(ceil_div(a.rows, 4 * (128 / TPR)), 148 * 4);
    rn_bwd_short_kernel<T, CK, MODE, TPR, NV>
        <<<*blocks, 128, 4 * 2 * NV * (Vec16<T>::N / 2) * TPR * sizeof(float2), st>>>(a);
    return cudaGetLastError();
}

template <typename T, bool CK, int MODE>
int backward(const RnBwdArgs& a, void* dw, void* db, cudaStream_t st) {
    const int nvec = a.D / Vec16<T>::N;
    // rows of a warp up to 96 vectors with dropout (768 channels, 42 M elements bf16: 82 us, of
    // a block 90; 520 channels 98 and 127), up to 64 without (768: 87 and 75 us)
    constexpr int SHORT = MODE == DROP_NONE ? 64 : 96;
    int blocks;
    const cudaError_t e = nvec > 1024    ? launch_bwd<T, CK, MODE, 3, 512, 1>(a, &blocks, st)
                          : nvec > 512   ? launch_bwd<T, CK, MODE, 2, 512, 1>(a, &blocks, st)
                          : nvec > 320   ? launch_bwd<T, CK, MODE, 2, 256, 2>(a, &blocks, st)
                          : nvec > SHORT ? launch_bwd<T, CK, MODE, 2, 160, 3>(a, &blocks, st)
                          : nvec > 64    ? launch_short<T, CK, MODE, 32, SHORT / 32>(a, &blocks, st)
                          : nvec > 32    ? launch_short<T, CK, MODE, 32, 2>(a, &blocks, st)
                          : nvec > 16    ? launch_short<T, CK, MODE, 32, 1>(a, &blocks, st)
                          : nvec > 8     ? launch_short<T, CK, MODE, 16, 1>(a, &blocks, st)
                                         : launch_short<T, CK, MODE, 8, 1>(a, &blocks, st);
    if (e != cudaSuccess) return fail(RWKV_E_CUDA, "rn_bwd_kernel: %s", cudaGetErrorString(e));
    return a.part ? launch_param_join(ParamJoin{a.part, blocks, 2 * (int64_t)a.D, a.D, {dw, db, nullptr}, a.wdtype}, st) : ok();
}

bool al(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
uintptr_t elem(int dtype) { return dtype == RWKV_F32 ? 4 : 2; }

int check_sizes(int dtype, int wdtype, int rows, int D, double p, double scale, const char* fn) {
    RWKV_REQUIRE(valid_dtype(dtype) && valid_dtype(wdtype), RWKV_E_DTYPE, "%s: dtypes x=%d w=%d", fn, dtype, wdtype);
    const int most = dtype == RWKV_F32 ? RN_VECTORS * 4 : RN_VECTORS * 8;
    RWKV_REQUIRE(rows >= 1 && D >= 1, RWKV_E_SHAPE, "%s: rows=%d D=%d", fn, rows, D);
    RWKV_REQUIRE(D % 8 == 0 && D <= most, RWKV_E_UNSUPPORTED, "%s: D=%d must be a multiple of 8, at most %d", fn, D, most);
    RWKV_REQUIRE(p >= 0.0 && p <= 1.0, RWKV_E_SHAPE, "%s: p=%g must be in 0..1", fn, p);
    // (where everything is dropped the factor is 0 whatever scale is)
    RWKV_REQUIRE(std::isfinite((float)scale) && std::isfinite(make_dropout(p, scale, 0, 0, nullptr).scale), RWKV_E_SHAPE,
                 "%s: scale=%g and scale over 1 - p must be finite in fp32", fn, scale);
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

using namespace rwkv;

extern "C" int rwkv_residual_norm_forward(int dtype, const void* x, const void* branch, double scale, double p,
                                          uint64_t seed, uint64_t offset, const int64_t* state, int wdtype,
                                          const void* weight, const void* bias, float eps, void* sum, void* y,
                                          float* mean, float* rstd, int8_t* codes, uint8_t* exps, int rows, int D,
                                          rwkv_stream_t stream) {
    const char* fn = "rwkv_residual_norm_forward";
    if (int rc = check_sizes(dtype, wdtype, rows, D, p, scale, fn)) return rc;
    RWKV_REQUIRE(x && branch && weight && bias && sum && y, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(!mean == !rstd, RWKV_E_NULL, "%s: give both mean and rstd or neither", fn);
    RWKV_REQUIRE(!codes == !exps, RWKV_E_NULL, "%s: give both codes and exps or neither", fn);
    RWKV_REQUIRE(eps >= 0.f, RWKV_E_SHAPE, "%s: eps=%g must be >= 0", fn, eps);
    RWKV_REQUIRE(al(x, 16) && al(branch, 16) && al(weight, 16) && al(bias, 16) && al(sum, 16) && al(y, 16) &&
                     al(codes, 8) && al(state, 8) && al(mean, 4) && al(rstd, 4),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned (codes, state: 8; mean, rstd: 4)", fn);
    const RnFwdArgs a{x,    branch, weight, bias, sum, y, mean, rstd, codes, exps, wdtype, rows, D, ceil_div(D, CK_GROUP),
                      eps, make_dropout(p, scale, seed, offset, state)};
    return dispatch_dtype(dtype, [&]<typename T>() {
        return dispatch_drop(a.drop, [&]<int MODE>() {
            return codes ? forward<T, true, MODE>(a, (cudaStream_t)stream) : forward<T, false, MODE>(a, (cudaStream_t)stream);
        });
    });
}

extern "C" int64_t rwkv_residual_norm_backward_workspace_size(int rows, int D) {
    if (rows < 1 || D < 1 || D > RN_VECTORS * 8) return 0;
    return (int64_t)std::min(rows, most_blocks(D)) * 2 * D * (int64_t)sizeof(float);
}

extern "C" int rwkv_residual_norm_backward(int dtype, const void* dy, const void* sum, const int8_t* codes,
                                           const uint8_t* exps, int wdtype, const void* weight, const float* mean,
                                           const float* rstd, const void* dres, double scale, double p, uint64_t seed,
                                           uint64_t offset, const int64_t* state, void* dx, void* dbranch,
                                           void* dweight, void* dbias, int rows, int D, void* workspace,
                                           int64_t workspace_bytes, rwkv_stream_t stream) {
    const char* fn = "rwkv_residual_norm_backward";
    if (int rc = check_sizes(dtype, wdtype, rows, D, p, scale, fn)) return rc;
    RWKV_REQUIRE(dy && weight && mean && rstd && dx && dbranch, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(sum ? !codes && !exps : codes && exps, RWKV_E_NULL, "%s: give either sum or codes and exps", fn);
    RWKV_REQUIRE(!dweight == !dbias, RWKV_E_NULL, "%s: give both dweight and dbias or neither", fn);
    RWKV_REQUIRE(al(dy, 16) && al(sum, 16) && al(codes, 8) && al(dres, 16) && al(dx, 16) && al(dbranch, 16) &&
                     al(weight, 16) && al(dweight, elem(wdtype)) && al(dbias, elem(wdtype)) && al(state, 8) &&
                     al(mean, 4) && al(rstd, 4),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned (codes, state: 8; others: their element)", fn);
    if (dweight) {
        const int64_t need = rwkv_residual_norm_backward_workspace_size(rows, D);
        RWKV_REQUIRE(workspace && workspace_bytes >= need, RWKV_E_WORKSPACE, "%s: workspace of %lld bytes, need %lld",
                     fn, (long long)workspace_bytes, (long long)need);
        RWKV_REQUIRE(al(workspace, 16), RWKV_E_UNSUPPORTED, "%s: workspace not 16-byte aligned", fn);
    }
    const RnBwdArgs a{dy,   sum,  codes, exps, weight, mean, rstd, dres, dx, dbranch,
                      dweight ? static_cast<float*>(workspace) : nullptr, wdtype, rows, D, ceil_div(D, CK_GROUP),
                      make_dropout(p, scale, seed, offset, state)};
    return dispatch_dtype(dtype, [&]<typename T>() {
        return dispatch_drop(a.drop, [&]<int MODE>() {
            return codes ? backward<T, true, MODE>(a, dweight, dbias, (cudaStream_t)stream)
                         : backward<T, false, MODE>(a, dweight, dbias, (cudaStream_t)stream);
        });
    });
}
