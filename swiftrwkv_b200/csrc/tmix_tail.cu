// The end of the time mix in training: a norm by head of the WKV output a, the
// bonus and the gate, and their gradient.  Per row and head of S channels:
//
//   n = (a - mean) rstd, rstd = 1 / sqrt(var + eps);  c = sum r k rk
//   z = n w + b + c v,  out = z g
//   dz = dout g, dg = dout z, dv = c dz, dc = sum dz v, dr = dc k rk, dk = dc r rk
//   e = dz w:  da = rstd (e - mean(e) - n mean(e n))
//   dw = sum_rows dz n, db = sum_rows dz, drk = sum_rows dc r k
//
// Both are bound by HBM: 6 and 11 tensors (16384 x 2048 bf16 65 us of a floor of 61;
// backward, 16384 x 2560, 156 and 5 for the parameters' join of 140).  A thread owns 8
// channels, S / 8 neighbouring lanes a head, whose sums are shuffles between them; nothing
// crosses a warp.  Threads are laid over [slots, D / 8] and walk over the rows of their slot,
// so that their channels are fixed: the parameters and the sums of their gradients
// stay in registers.  The statistics are not kept by the forward pass: the backward
// reads a whole anyway.
#include <algorithm>

#include "ckpt8.cuh"
#include "copy_async.cuh"
#include "param_join.cuh"

namespace rwkv {
namespace {

constexpr int TAIL_T = 128;

struct TailArgs {
    const void *a, *r, *k, *v, *g;  // [rows, D]
    const void *rk, *w, *b;         // [D]
    int wdtype, units, slots, rows;  // units: D / 8
    float eps;
};
struct TailGrad {
    const void* dout;
    void *da, *dr, *dk, *dv, *dg;
    float* part;  // [slots][drk, dw, db][D], or NULL
};

// The 8 channels of a thread: one 16-byte vector, or of fp32 two, L vectors apart, so
// that a head's lanes read and write whole sectors (neighbouring vectors: 109 us instead
// of 66 at 8192 x 2048).
template <typename T, int L>
struct Own8 {
    static constexpr int VE = Vec16<T>::N, W = 8 / VE, STEP = VE * L;
    // the first one's channel, for unit u of a row
    static __device__ __forceinline__ int channel(int u) { return u / L * (8 * L) + u % L * VE; }
    static __device__ __forceinline__ void params(const void* p, int dtype, int c, float* v) {
#pragma unroll
        for (int w = 0; w < W; w++) load_params<VE>(p, dtype, c + w * STEP, v + w * VE);
    }
    static __device__ __forceinline__ void store(T* p, const float* v) {
#pragma unroll
        for (int w = 0; w < W; w++) __stcs(reinterpret_cast<uint4*>(p + w * STEP), Vec16<T>::pack(v + w * VE));
    }
    static __device__ __forceinline__ void sums(float* p, const float* v) {
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
            for (int k = 0; k < VE; k += 4)
                *reinterpret_cast<float4*>(p + w * STEP + k) =
                    make_float4(v[w * VE + k], v[w * VE + k + 1], v[w * VE + k + 2], v[w * VE + k + 3]);
    }
};

// The vectors of a row that a thread owns run ahead of their use by a stage or two
// through a ring in shared memory that is private to the thread (cp.async, no
// barrier), so that HBM stays busy through a head's sums (loads at the head of each row's
// work: 90 us forward, 183 backward).  Two stages of fp32, which fill 48 KB in
// the backward (40 forward).
template <typename T, int L, int N>
struct TailRing {
    static constexpr int W = Own8<T, L>::W, STAGES = sizeof(T) == 2 ? 3 : 2;
    uint4 r[STAGES][N * W][TAIL_T];

    // N tensors' 8 elements at `at`, or zeros
    __device__ __forceinline__ void fetch(int stage, const void* const* p, int64_t at, bool in) {
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int w = 0; w < W; w++)
                copy_async_n<16>(&r[stage][i * W + w][threadIdx.x],
                                 static_cast<const T*>(p[i]) + at + w * Own8<T, L>::STEP, in ? 16 : 0);
        copy_commit();
    }
    __device__ __forceinline__ void floats(int stage, int i, float* v) const {
#pragma unroll
        for (int w = 0; w < W; w++) Vec16<T>::unpack(r[stage][i * W + w][threadIdx.x], v + w * Vec16<T>::N);
    }
};

// L lanes a head.  All threads of a warp take the same number of steps, with or
// without a row, for the shuffles.
template <typename T, int L>
__global__ void __launch_bounds__(TAIL_T) tmix_tail_kernel(const TailArgs a, T* out) {
    const int64_t id = blockIdx.x * (int64_t)TAIL_T + threadIdx.x;
    const int slot = (int)(id / a.units), u = (int)(id - (int64_t)slot * a.units);
    const int64_t D = 8 * (int64_t)a.units;
    constexpr float inv = 1.f / (8 * L);
    float rk[8], w[8], b[8];
    using Own = Own8<T, L>;
    const int first = Own::channel(u);
    Own::params(a.rk, a.wdtype, first, rk);
    Own::params(a.w, a.wdtype, first, w);
    Own::params(a.b, a.wdtype, first, b);
    using Ring = TailRing<T, L, 5>;
    __shared__ Ring ring;
    const void* const from[5] = {a.a, a.r, a.k, a.v, a.g};
    const uint32_t rows = slot < a.slots ? a.rows : 0;  // unsigned: a step past 2^31 - 1 rows
    const int steps = ceil_div(a.rows, a.slots);
    const int64_t step = a.slots * D;
    int64_t at = slot * D + first, next = at;
    uint32_t fetched = slot;
    auto fetch = [&](int stage) {
        const bool in = fetched < rows;
        ring.fetch(stage, from, in ? next : 0, in);
        fetched += a.slots;
        next += step;
    };
#pragma unroll
    for (int i = 0; i < Ring::STAGES - 1; i++) fetch(i);
    int stage = 0, put = Ring::STAGES - 1;
    uint32_t row = slot;
    for (int i = 0; i < steps; i++, row += a.slots, at += step) {
        fetch(put);
        copy_wait<Ring::STAGES - 1>();
        float x[8], y[8], c = 0.f, s = 0.f, q = 0.f;
        ring.floats(stage, 1, x);
        ring.floats(stage, 2, y);
#pragma unroll
        for (int j = 0; j < 8; j++) c = fmaf(x[j] * y[j], rk[j], c);
        ring.floats(stage, 0, x);
#pragma unroll
        for (int j = 0; j < 8; j++) s += x[j];
        c = group_sum<L>(c);
        const float mean = group_sum<L>(s) * inv;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] -= mean;
            q = fmaf(x[j], x[j], q);
        }
        const float rstd = 1.f / sqrtf(group_sum<L>(q) * inv + a.eps);
        ring.floats(stage, 3, y);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = fmaf(c, y[j], fmaf(x[j] * rstd, w[j], b[j]));
        ring.floats(stage, 4, y);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] *= y[j];
        if (row < rows) Own::store(out + at, x);
        put = stage;
        stage = stage == Ring::STAGES - 1 ? 0 : stage + 1;
    }
    copy_wait<0>();
}

template <typename T, int L>
__global__ void __launch_bounds__(TAIL_T) tmix_tail_backward_kernel(const TailArgs a, const TailGrad o) {
    pdl_trigger();
    const int64_t id = blockIdx.x * (int64_t)TAIL_T + threadIdx.x;
    const int slot = (int)(id / a.units), u = (int)(id - (int64_t)slot * a.units);
    const int64_t D = 8 * (int64_t)a.units;
    constexpr float inv = 1.f / (8 * L);
    float rk[8], w[8], b[8], srk[8], sw[8], sb[8];
    using Own = Own8<T, L>;
    const int first = Own::channel(u);
    Own::params(a.rk, a.wdtype, first, rk);
    Own::params(a.w, a.wdtype, first, w);
    Own::params(a.b, a.wdtype, first, b);
#pragma unroll
    for (int j = 0; j < 8; j++) srk[j] = sw[j] = sb[j] = 0.f;
    using Ring = TailRing<T, L, 6>;
    __shared__ Ring ring;
    const void* const from[6] = {a.a, a.r, a.k, a.v, a.g, o.dout};
    const uint32_t rows = slot < a.slots ? a.rows : 0;  // unsigned: a step past 2^31 - 1 rows
    const int steps = ceil_div(a.rows, a.slots);
    const int64_t step = a.slots * D;
    int64_t at = slot * D + first, next = at;
    uint32_t fetched = slot;
    auto fetch = [&](int stage) {
        const bool in = fetched < rows;
        ring.fetch(stage, from, in ? next : 0, in);
        fetched += a.slots;
        next += step;
    };
#pragma unroll
    for (int i = 0; i < Ring::STAGES - 1; i++) fetch(i);
    int stage = 0, put = Ring::STAGES - 1;
    uint32_t row = slot;
    for (int i = 0; i < steps; i++, row += a.slots, at += step) {
        const bool in = row < rows;
        fetch(put);
        copy_wait<Ring::STAGES - 1>();
        float r[8], k[8], x[8], v[8], g[8], d[8], c = 0.f, s = 0.f;
        ring.floats(stage, 1, r);
        ring.floats(stage, 2, k);
        ring.floats(stage, 0, x);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            c = fmaf(r[j] * k[j], rk[j], c);
            s += x[j];
        }
        c = group_sum<L>(c);
        const float mean = group_sum<L>(s) * inv;
        ring.floats(stage, 3, v);
        ring.floats(stage, 4, g);
        ring.floats(stage, 5, d);
        // sums over the head: (a - mean)^2, dz v, e, e (a - mean)
        float q = 0.f, dc = 0.f, e1 = 0.f, e2 = 0.f, dz[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] -= mean;
            dz[j] = d[j] * g[j];
            q = fmaf(x[j], x[j], q);
            dc = fmaf(dz[j], v[j], dc);
            const float e = dz[j] * w[j];
            e1 += e;
            e2 = fmaf(e, x[j], e2);
        }
        q = group_sum<L>(q);
        dc = group_sum<L>(dc);
        const float m1 = group_sum<L>(e1) * inv;
        // 0 without a row, whose zeros at eps = 0 would make n NaN and with it the sums over rows
        const float rstd = in ? 1.f / sqrtf(q * inv + a.eps) : 0.f;
        const float m2 = group_sum<L>(e2) * inv * rstd;
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] *= rstd;
            t[j] = d[j] * fmaf(c, v[j], fmaf(x[j], w[j], b[j]));
        }
        if (in) Own::store(static_cast<T*>(o.dg) + at, t);
#pragma unroll
        for (int j = 0; j < 8; j++) t[j] = rstd * (fmaf(dz[j], w[j], -m1) - x[j] * m2);
        if (in) Own::store(static_cast<T*>(o.da) + at, t);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            sw[j] = fmaf(dz[j], x[j], sw[j]);
            sb[j] += dz[j];
            t[j] = c * dz[j];
        }
        if (in) Own::store(static_cast<T*>(o.dv) + at, t);
#pragma unroll
        for (int j = 0; j < 8; j++) t[j] = dc * rk[j] * k[j];
        if (in) Own::store(static_cast<T*>(o.dr) + at, t);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            t[j] = dc * rk[j] * r[j];
            srk[j] = fmaf(dc * r[j], k[j], srk[j]);
        }
        if (in) Own::store(static_cast<T*>(o.dk) + at, t);
        put = stage;
        stage = stage == Ring::STAGES - 1 ? 0 : stage + 1;
    }
    copy_wait<0>();
    if (!o.part || slot >= a.slots) return;
    float* p = o.part + (int64_t)slot * 3 * D + first;
    Own::sums(p, srk);
    Own::sums(p + D, sw);
    Own::sums(p + 2 * D, sb);
}

template <typename F>
int dispatch_head(int S, F&& f) {
    switch (S) {
        case 32: return f.template operator()<4>();
        case 64: return f.template operator()<8>();
        case 128: return f.template operator()<16>();
        default: return f.template operator()<32>();
    }
}

// six and four blocks per SM: five and three 65 and 168 us, seven and four with two
// stages 64 and 174, at the sizes above
constexpr int64_t FWD_THREADS = 148 * 6 * TAIL_T, BWD_THREADS = 148 * 4 * TAIL_T;

// Slots of a call: enough threads for every SM, at least `least` rows each.
int plan(int rows, int units, int64_t threads, int least) {
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows + least - 1) / least, threads / units));
}
constexpr int BWD_LEAST = 4;

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_args(int dtype, const TailArgs& a, int rows, int H, int S, const char* fn) {
    RWKV_REQUIRE(valid_dtype(dtype) && valid_dtype(a.wdtype), RWKV_E_DTYPE, "%s: dtypes x=%d w=%d", fn, dtype, a.wdtype);
    RWKV_REQUIRE(a.a && a.r && a.k && a.v && a.g && a.rk && a.w && a.b, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(rows >= 1 && H >= 1 && H <= 1 << 16, RWKV_E_SHAPE, "%s: rows=%d H=%d (rows >= 1, H in 1..2^16)", fn,
                 rows, H);
    RWKV_REQUIRE(S == 32 || S == 64 || S == 128 || S == 256, RWKV_E_UNSUPPORTED, "%s: S=%d (32, 64, 128 or 256)", fn, S);
    RWKV_REQUIRE(a.eps >= 0.f, RWKV_E_SHAPE, "%s: eps=%g must be >= 0", fn, a.eps);
    RWKV_REQUIRE(al16(a.a) && al16(a.r) && al16(a.k) && al16(a.v) && al16(a.g) && al16(a.rk) && al16(a.w) && al16(a.b),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned", fn);
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

using namespace rwkv;

extern "C" int rwkv_tmix_tail_forward(int dtype, const void* wkv, const void* r, const void* k, const void* v,
                                      const void* g, int wdtype, const void* rk, const void* weight, const void* bias,
                                      float eps, void* out, int rows, int H, int S, rwkv_stream_t stream) {
    const char* fn = "rwkv_tmix_tail_forward";
    TailArgs a{wkv, r, k, v, g, rk, weight, bias, wdtype, 0, 0, rows, eps};
    RWKV_REQUIRE(out, RWKV_E_NULL, "%s: NULL argument", fn);
    if (int rc = check_args(dtype, a, rows, H, S, fn)) return rc;
    RWKV_REQUIRE(al16(out), RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned", fn);
    a.units = H * (S / 8);
    a.slots = plan(rows, a.units, FWD_THREADS, 1);
    return dispatch_dtype(dtype, [&]<typename T>() {
        return dispatch_head(S, [&]<int L>() {
            const int64_t threads = (int64_t)a.slots * a.units;
            tmix_tail_kernel<T, L>
                <<<(unsigned)((threads + TAIL_T - 1) / TAIL_T), TAIL_T, 0, (cudaStream_t)stream>>>(a, (T*)out);
            return check_launch("tmix_tail_kernel");
        });
    });
}

extern "C" int64_t rwkv_tmix_tail_backward_workspace_size(int rows, int H, int S) {
    if (rows < 1 || H < 1 || H > 1 << 16 || (S != 32 && S != 64 && S != 128 && S != 256)) return 0;
    return (int64_t)plan(rows, H * (S / 8), BWD_THREADS, BWD_LEAST) * 3 * H * S * (int64_t)sizeof(float);
}

extern "C" int rwkv_tmix_tail_backward(int dtype, const void* dout, const void* wkv, const void* r, const void* k,
                                       const void* v, const void* g, int wdtype, const void* rk, const void* weight,
                                       const void* bias, float eps, void* dwkv, void* dr, void* dk, void* dv, void* dg,
                                       void* drk, void* dweight, void* dbias, int rows, int H, int S, void* workspace,
                                       int64_t workspace_bytes, rwkv_stream_t stream) {
    const char* fn = "rwkv_tmix_tail_backward";
    TailArgs a{wkv, r, k, v, g, rk, weight, bias, wdtype, 0, 0, rows, eps};
    TailGrad o{dout, dwkv, dr, dk, dv, dg, nullptr};
    RWKV_REQUIRE(dout && dwkv && dr && dk && dv && dg, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(!drk == !dweight && !drk == !dbias, RWKV_E_NULL, "%s: give drk, dweight and dbias or none of them", fn);
    if (int rc = check_args(dtype, a, rows, H, S, fn)) return rc;
    RWKV_REQUIRE(al16(dout) && al16(dwkv) && al16(dr) && al16(dk) && al16(dv) && al16(dg) && al16(drk) && al16(dweight) &&
                     al16(dbias),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned", fn);
    if (drk) {
        const int64_t need = rwkv_tmix_tail_backward_workspace_size(rows, H, S);
        RWKV_REQUIRE(workspace && workspace_bytes >= need, RWKV_E_WORKSPACE, "%s: workspace of %lld bytes, need %lld",
                     fn, (long long)workspace_bytes, (long long)need);
        RWKV_REQUIRE(al16(workspace), RWKV_E_UNSUPPORTED, "%s: workspace not 16-byte aligned", fn);
        o.part = static_cast<float*>(workspace);
    }
    a.units = H * (S / 8);
    a.slots = plan(rows, a.units, BWD_THREADS, BWD_LEAST);
    return dispatch_dtype(dtype, [&]<typename T>() {
        return dispatch_head(S, [&]<int L>() {
            const cudaStream_t st = (cudaStream_t)stream;
            const int64_t threads = (int64_t)a.slots * a.units;
            tmix_tail_backward_kernel<T, L><<<(unsigned)((threads + TAIL_T - 1) / TAIL_T), TAIL_T, 0, st>>>(a, o);
            if (int rc = check_launch("tmix_tail_backward_kernel")) return rc;
            if (!drk) return ok();
            const int64_t D = (int64_t)H * S;
            return launch_param_join(ParamJoin{o.part, a.slots, 3 * D, D, {drk, dweight, dbias}, wdtype}, st);
        });
    });
}
