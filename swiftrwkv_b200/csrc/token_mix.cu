// Token mix: each token interpolated with the one before it, J ways (the inputs of
// the time mix's projections; J = 1: the channel mix's), and its gradient.
//
//   y_j[t] = x[t] + (x[t-1] - x[t]) m_j,  x[-1] = prev (or 0)
//   dx[t]  = sum_j (1 - m_j) dy_j[t] + sum_j m_j dy_j[t+1]  (+ dlast at the last token)
//   dm_j   = sum over tokens of dy_j[t] (x[t-1] - x[t]),  dprev = sum_j m_j dy_j[0]
//
// Both are bound by HBM: 1 + J and 2 + J tensors.  A thread owns one 16-byte vector
// of channels and walks over consecutive tokens of the flattened [B, T], so that a
// token is read once, the interpolations' weights stay in registers and the
// gradient of the weights is summed there.  `slots` threads share a vector's tokens;
// each reads one token beyond its own (the one before in the forward, the one after
// in the backward).  Tokens from a sequence's length on are not read: they give y =
// 0 and dx = 0, whatever they and their gradients hold.
#include <algorithm>

#include "ckpt8.cuh"
#include "param_join.cuh"

namespace rwkv {
namespace {

constexpr int MIX_WAYS = 6, MIX_T = 128;

struct MixArgs {
    const void* x;
    const void* mix;   // [J, D]
    const void* prev;  // [B, D] or NULL
    const int32_t* lengths;  // [B] or NULL
    int mdtype, B, T, nvec, slots;
    int64_t rows, chunk;  // B T, and the tokens of a slot
};
struct MixOut {
    void* y[MIX_WAYS];
    void* last;
};
struct MixGrad {
    const void* dy[MIX_WAYS];  // NULL: zero
    const void* dlast;
    void* dx;
    void* dprev;
    float* part;  // [slots][J][D], or NULL
};

// A place in the flattened tokens.
struct Token {
    int b, t, len;
    __device__ __forceinline__ void length(const MixArgs& a) {
        len = a.lengths && b < a.B ? max(0, min(a.lengths[b], a.T)) : a.T;
    }
    __device__ __forceinline__ void start(const MixArgs& a, int64_t n) {
        b = (int)(n / a.T);
        t = (int)(n - (int64_t)b * a.T);
        length(a);
    }
    __device__ __forceinline__ void next(const MixArgs& a) {
        if (++t == a.T) {
            t = 0;
            b++;
            length(a);
        }
    }
};

template <typename T, int J>
__global__ void __launch_bounds__(MIX_T) token_mix_kernel(const MixArgs a, const MixOut o) {
    constexpr int VE = Vec16<T>::N;
    const int64_t id = blockIdx.x * (int64_t)MIX_T + threadIdx.x;
    const int slot = (int)(id / a.nvec), v = (int)(id - (int64_t)slot * a.nvec);
    int64_t n = slot * a.chunk;
    const int64_t end = min(n + a.chunk, a.rows);
    if (slot >= a.slots || n >= end) return;
    const uint4* const x = static_cast<const uint4*>(a.x) + v;
    const uint4* const prev = static_cast<const uint4*>(a.prev) + v;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    float m[J][VE];
#pragma unroll
    for (int j = 0; j < J; j++) load_params<VE>(a.mix, a.mdtype, ((int64_t)j * a.nvec + v) * VE, m[j]);
    Token k;
    k.start(a, n);
    uint4 before = k.t && k.t < k.len ? x[(n - 1) * a.nvec] : zero;
    uint4 ahead = k.t < k.len ? x[n * a.nvec] : zero;
    while (n < end) {
        const uint4 cur = ahead;
        const Token here = k;
        k.next(a);
        if (n + 1 < end && k.t < k.len) ahead = x[(n + 1) * a.nvec];
        if (here.t == 0) {
            before = a.prev ? prev[(int64_t)here.b * a.nvec] : zero;
            if (here.len == 0) static_cast<uint4*>(o.last)[(int64_t)here.b * a.nvec + v] = before;
        }
        if (here.t == here.len - 1) static_cast<uint4*>(o.last)[(int64_t)here.b * a.nvec + v] = cur;
        float f[VE], d[VE];
        Vec16<T>::unpack(cur, f);
        Vec16<T>::unpack(before, d);
#pragma unroll
        for (int i = 0; i < VE; i++) d[i] -= f[i];
#pragma unroll
        for (int j = 0; j < J; j++) {
            float y[VE];
#pragma unroll
            for (int i = 0; i < VE; i++) y[i] = fmaf(d[i], m[j][i], f[i]);
            __stcs(static_cast<uint4*>(o.y[j]) + n * a.nvec + v, here.t < here.len ? Vec16<T>::pack(y) : zero);
        }
        before = cur;
        n++;
    }
}

template <typename T, int J>
__global__ void __launch_bounds__(MIX_T) token_mix_backward_kernel(const MixArgs a, const MixGrad g) {
    constexpr int VE = Vec16<T>::N;
    const int64_t id = blockIdx.x * (int64_t)MIX_T + threadIdx.x;
    const int slot = (int)(id / a.nvec), v = (int)(id - (int64_t)slot * a.nvec);
    int64_t n = slot * a.chunk;
    const int64_t end = min(n + a.chunk, a.rows);
    if (slot >= a.slots) return;
    const uint4* const x = static_cast<const uint4*>(a.x) + v;
    const uint4* const prev = static_cast<const uint4*>(a.prev) + v;
    const uint4* const dlast = static_cast<const uint4*>(g.dlast) + v;
    uint4* const dx = static_cast<uint4*>(g.dx) + v;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    float m[J][VE], dm[J][VE];
#pragma unroll
    for (int j = 0; j < J; j++) {
        load_params<VE>(a.mix, a.mdtype, ((int64_t)j * a.nvec + v) * VE, m[j]);
#pragma unroll
        for (int i = 0; i < VE; i++) dm[j][i] = 0.f;
    }
    auto load = [&](int64_t at, const Token& k, uint4* r) {
#pragma unroll
        for (int j = 0; j < J; j++)
            r[j] = k.t < k.len && g.dy[j] ? __ldcs(static_cast<const uint4*>(g.dy[j]) + at * a.nvec + v) : zero;
    };
    Token k;
    k.start(a, n);
    float before[VE], own[VE];  // x of the token before; the gradient so far of the token before
    bool open = false;          // whether that is still to be stored
    if (n < end) {
        Vec16<T>::unpack(k.t && k.t < k.len ? x[(n - 1) * a.nvec] : zero, before);
        for (; n < end; n++, k.next(a)) {
            const bool real = k.t < k.len;
            uint4 r[J];
            load(n, k, r);
            float f[VE], back[VE], rest[VE], d[VE];
            Vec16<T>::unpack(real ? __ldcs(x + n * a.nvec) : zero, f);
            if (k.t == 0) Vec16<T>::unpack(real && a.prev ? prev[(int64_t)k.b * a.nvec] : zero, before);
#pragma unroll
            for (int i = 0; i < VE; i++) back[i] = rest[i] = 0.f, d[i] = before[i] - f[i];
#pragma unroll
            for (int j = 0; j < J; j++) {
                float dy[VE];
                Vec16<T>::unpack(r[j], dy);
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    back[i] = fmaf(m[j][i], dy[i], back[i]);
                    rest[i] += fmaf(-m[j][i], dy[i], dy[i]);  // (1 - m) dy, rounded once
                    dm[j][i] = fmaf(dy[i], real ? d[i] : 0.f, dm[j][i]);
                }
            }
            if (open) {
                if (k.t)
#pragma unroll
                    for (int i = 0; i < VE; i++) own[i] += back[i];
                __stcs(dx + (n - 1) * a.nvec, Vec16<T>::pack(own));
            }
            if (g.dlast && (k.t == k.len - 1 || (k.t == 0 && k.len == 0))) {
                float l[VE];
                Vec16<T>::unpack(dlast[(int64_t)k.b * a.nvec], l);
#pragma unroll
                for (int i = 0; i < VE; i++) (k.len ? rest[i] : back[i]) += l[i];
            }
            if (k.t == 0 && g.dprev) static_cast<uint4*>(g.dprev)[(int64_t)k.b * a.nvec + v] = Vec16<T>::pack(back);
#pragma unroll
            for (int i = 0; i < VE; i++) own[i] = rest[i], before[i] = f[i];
            open = true;
        }
        if (n < a.rows && k.t) {  // the next slot's first token goes on with this sequence
            uint4 r[J];
            load(n, k, r);
            float back[VE] = {};
#pragma unroll
            for (int j = 0; j < J; j++) {
                float dy[VE];
                Vec16<T>::unpack(r[j], dy);
#pragma unroll
                for (int i = 0; i < VE; i++) back[i] = fmaf(m[j][i], dy[i], back[i]);
            }
#pragma unroll
            for (int i = 0; i < VE; i++) own[i] += back[i];
        }
        __stcs(dx + (n - 1) * a.nvec, Vec16<T>::pack(own));
    }
    if (!g.part) return;
    float* p = g.part + (int64_t)slot * J * a.nvec * VE + (int64_t)v * VE;
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < VE; i += 4)
            *reinterpret_cast<float4*>(p + (int64_t)j * a.nvec * VE + i) =
                make_float4(dm[j][i], dm[j][i + 1], dm[j][i + 2], dm[j][i + 3]);
}

template <typename F>
int dispatch_ways(int J, F&& f) {
    switch (J) {
        case 1: return f.template operator()<1>();
        case 2: return f.template operator()<2>();
        case 3: return f.template operator()<3>();
        case 4: return f.template operator()<4>();
        case 5: return f.template operator()<5>();
        default: return f.template operator()<6>();
    }
}

// Slots of a call: enough threads for every SM, at least `least` tokens each.
void plan(MixArgs& a, int64_t threads, int least) {
    const int64_t most = std::max<int64_t>(1, threads / a.nvec);
    const int64_t slots = std::max<int64_t>(1, std::min((a.rows + least - 1) / least, most));
    a.chunk = (a.rows + slots - 1) / slots;
    a.slots = (int)((a.rows + a.chunk - 1) / a.chunk);
}
constexpr int64_t FWD_THREADS = 148 * 8 * 128, BWD_THREADS = 148 * 2 * 128;
constexpr int FWD_LEAST = 1, BWD_LEAST = 4;

int vectors(int dtype, int D) { return dtype == RWKV_F32 ? D / 4 : D / 8; }

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_sizes(int dtype, int mdtype, int B, int T, int D, int J, const char* fn) {
    RWKV_REQUIRE(valid_dtype(dtype) && valid_dtype(mdtype), RWKV_E_DTYPE, "%s: dtypes x=%d mix=%d", fn, dtype, mdtype);
    RWKV_REQUIRE(B >= 1 && T >= 1 && D >= 1 && D <= 1 << 20, RWKV_E_SHAPE, "%s: B=%d T=%d D=%d (B, T >= 1, D in 1..2^20)",
                 fn, B, T, D);
    RWKV_REQUIRE((int64_t)B * T <= 1ll << 40 && (int64_t)B * T * D <= 1ll << 44, RWKV_E_SHAPE, "%s: B=%d T=%d D=%d", fn,
                 B, T, D);
    RWKV_REQUIRE(J >= 1 && J <= MIX_WAYS, RWKV_E_SHAPE, "%s: J=%d (1..%d)", fn, J, MIX_WAYS);
    RWKV_REQUIRE(D % 8 == 0, RWKV_E_UNSUPPORTED, "%s: D=%d must be a multiple of 8", fn, D);
    return RWKV_OK;
}

MixArgs make_args(int dtype, const void* x, int mdtype, const void* mix, const void* prev, const int32_t* lengths, int B,
                  int T, int D) {
    return MixArgs{x, mix, prev, lengths, mdtype, B, T, vectors(dtype, D), 0, (int64_t)B * T, 0};
}

}  // namespace
}  // namespace rwkv

using namespace rwkv;

extern "C" int rwkv_token_mix_forward(int dtype, const void* x, int mdtype, const void* mix, const void* prev,
                                      const int32_t* lengths, void* const* y, void* last, int B, int T, int D, int J,
                                      rwkv_stream_t stream) {
    const char* fn = "rwkv_token_mix_forward";
    if (int rc = check_sizes(dtype, mdtype, B, T, D, J, fn)) return rc;
    RWKV_REQUIRE(x && mix && y && last, RWKV_E_NULL, "%s: NULL argument", fn);
    MixOut o{};
    for (int j = 0; j < J; j++) {
        RWKV_REQUIRE(y[j], RWKV_E_NULL, "%s: y[%d] is NULL", fn, j);
        RWKV_REQUIRE(al16(y[j]), RWKV_E_UNSUPPORTED, "%s: y[%d] not 16-byte aligned", fn, j);
        o.y[j] = y[j];
    }
    o.last = last;
    RWKV_REQUIRE(al16(x) && al16(mix) && al16(prev) && al16(last) && ((uintptr_t)lengths & 3) == 0, RWKV_E_UNSUPPORTED,
                 "%s: a tensor is not 16-byte aligned (lengths: 4)", fn);
    MixArgs a = make_args(dtype, x, mdtype, mix, prev, lengths, B, T, D);
    plan(a, FWD_THREADS, FWD_LEAST);
    return dispatch_dtype(dtype, [&]<typename T_>() {
        return dispatch_ways(J, [&]<int J_>() {
            const int64_t threads = (int64_t)a.slots * a.nvec;
            token_mix_kernel<T_, J_><<<(unsigned)((threads + MIX_T - 1) / MIX_T), MIX_T, 0, (cudaStream_t)stream>>>(a, o);
            return check_launch("token_mix_kernel");
        });
    });
}

extern "C" int64_t rwkv_token_mix_backward_workspace_size(int dtype, int B, int T, int D, int J) {
    if (!valid_dtype(dtype) || B < 1 || T < 1 || D < 8 || D % 8 || D > 1 << 20 || J < 1 || J > MIX_WAYS) return 0;
    MixArgs a = make_args(dtype, nullptr, 0, nullptr, nullptr, nullptr, B, T, D);
    plan(a, BWD_THREADS, BWD_LEAST);
    return (int64_t)a.slots * J * D * (int64_t)sizeof(float);
}

extern "C" int rwkv_token_mix_backward(int dtype, const void* const* dy, const void* x, int mdtype, const void* mix,
                                       const void* prev, const int32_t* lengths, const void* dlast, void* dx, void* dmix,
                                       void* dprev, int B, int T, int D, int J, void* workspace,
                                       int64_t workspace_bytes, rwkv_stream_t stream) {
    const char* fn = "rwkv_token_mix_backward";
    if (int rc = check_sizes(dtype, mdtype, B, T, D, J, fn)) return rc;
    RWKV_REQUIRE(dy && x && mix && dx, RWKV_E_NULL, "%s: NULL argument", fn);
    MixGrad g{};
    for (int j = 0; j < J; j++) {
        RWKV_REQUIRE(al16(dy[j]), RWKV_E_UNSUPPORTED, "%s: dy[%d] not 16-byte aligned", fn, j);
        g.dy[j] = dy[j];
    }
    RWKV_REQUIRE(al16(x) && al16(mix) && al16(prev) && al16(dlast) && al16(dx) && al16(dmix) && al16(dprev) &&
                     ((uintptr_t)lengths & 3) == 0,
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned (lengths: 4)", fn);
    MixArgs a = make_args(dtype, x, mdtype, mix, prev, lengths, B, T, D);
    plan(a, BWD_THREADS, BWD_LEAST);
    g.dlast = dlast;
    g.dx = dx;
    g.dprev = dprev;
    if (dmix) {
        const int64_t need = rwkv_token_mix_backward_workspace_size(dtype, B, T, D, J);
        RWKV_REQUIRE(workspace && workspace_bytes >= need, RWKV_E_WORKSPACE, "%s: workspace of %lld bytes, need %lld",
                     fn, (long long)workspace_bytes, (long long)need);
        RWKV_REQUIRE(al16(workspace), RWKV_E_UNSUPPORTED, "%s: workspace not 16-byte aligned", fn);
        g.part = static_cast<float*>(workspace);
    }
    return dispatch_dtype(dtype, [&]<typename T_>() {
        return dispatch_ways(J, [&]<int J_>() {
            const cudaStream_t st = (cudaStream_t)stream;
            const int64_t threads = (int64_t)a.slots * a.nvec;
            token_mix_backward_kernel<T_, J_><<<(unsigned)((threads + MIX_T - 1) / MIX_T), MIX_T, 0, st>>>(a, g);
            if (int rc = check_launch("token_mix_backward_kernel")) return rc;
            if (!dmix) return ok();
            const int64_t width = (int64_t)J * D;
            return launch_param_join(ParamJoin{g.part, a.slots, width, width, {dmix, nullptr, nullptr}, mdtype}, st);
        });
    });
}
