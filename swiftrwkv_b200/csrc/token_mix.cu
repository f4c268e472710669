// Token mix: each token interpolated with the one before it, J ways (the inputs of
// the time mix's projections; J = 1: the channel mix's), and its gradient.
//
//   y_j[t] = x[t] + (x[t-1] - x[t]) m_j,  x[-1] = prev (or 0)
//   dx[t]  = sum_j (1 - m_j) dy_j[t] + sum_j m_j dy_j[t+1]  (+ dlast at the last token)
//   dm_j   = sum over tokens of dy_j[t] (x[t-1] - x[t]),  dprev = sum_j m_j dy_j[0]
//
// Both are bound by HBM: 1 + J and 2 + J tensors (16384 x 2560 bf16, six ways: 91 us
// of a floor of 89 forward, 113 with the weights' join of 102 backward, the kernels alone).  A thread owns
// one 16-byte vector of channels of consecutive tokens of the flattened [B, T], so that
// a token is read about once and the interpolations' weights stay in registers.  The
// forward takes four tokens a thread: what is left to do are stores, and many short
// threads keep them coming (walks over 110 tokens with x read ahead: 119 us).  The
// backward walks over as many tokens as there are threads for, since it sums the
// weights' gradient in registers; each thread reads one token beyond its own, for its part
// in the last one's gradient.  Tokens from a sequence's length on are not read: they
// give y = 0 and dx = 0, whatever they and their gradients hold.
#include <algorithm>

#include "ckpt8.cuh"
#include "copy_async.cuh"
#include "f32x2.cuh"
#include "param_join.cuh"

namespace rwkv {
namespace {

constexpr int MIX_WAYS = 6, MIX_T = 128, MIX_STAGES = 3;

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

// A thread takes U consecutive tokens, their loads first.
template <typename T, int J, int U>
__global__ void __launch_bounds__(MIX_T) token_mix_kernel(const MixArgs a, const MixOut o) {
    constexpr int VE = Vec16<T>::N, P = VE / 2;
    const int64_t id = blockIdx.x * (int64_t)MIX_T + threadIdx.x;
    const int64_t slot = id / a.nvec;
    const int v = (int)(id - slot * a.nvec);
    const int64_t first = slot * U;
    if (first >= a.rows) return;
    const uint4* const x = static_cast<const uint4*>(a.x) + first * a.nvec + v;
    const uint4* const prev = static_cast<const uint4*>(a.prev) + v;
    uint4* const last = static_cast<uint4*>(o.last) + v;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int n = (int)min((int64_t)U, a.rows - first);
    Token start, k;
    start.start(a, first);
    k = start;
    uint4 cur[U];  // zeros from a sequence's length on
    uint4 before = zero;
    if (start.t == 0) {
        if (a.prev) before = prev[(int64_t)start.b * a.nvec];
    } else if (start.t < start.len) {
        before = x[-a.nvec];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        cur[u] = u < n && k.t < k.len ? x[u * a.nvec] : zero;
        k.next(a);
    }
    float2 m[J][P];
#pragma unroll
    for (int j = 0; j < J; j++)
        load_params<VE>(a.mix, a.mdtype, ((int64_t)j * a.nvec + v) * VE, reinterpret_cast<float*>(m[j]));
    k = start;
    int64_t at = first * a.nvec + v;
    const float2 minus = both(-1.f);
#pragma unroll
    for (int u = 0; u < U; u++, at += a.nvec, k.next(a)) {
        if (u >= n) break;
        if (k.t == 0) {
            if (u > 0) before = a.prev ? prev[(int64_t)k.b * a.nvec] : zero;
            if (k.len == 0) last[(int64_t)k.b * a.nvec] = before;
        }
        if (k.t == k.len - 1) last[(int64_t)k.b * a.nvec] = cur[u];
        if (k.t >= k.len) {  // zeros whatever the weights hold
#pragma unroll
            for (int j = 0; j < J; j++) __stcs(static_cast<uint4*>(o.y[j]) + at, zero);
            continue;
        }
        Pairs<T> f, d;
        f.unpack(cur[u]);
        d.unpack(before);
#pragma unroll
        for (int i = 0; i < P; i++) d[i] = fma2(f[i], minus, d[i]);
#pragma unroll
        for (int j = 0; j < J; j++) {
            Pairs<T> y;
#pragma unroll
            for (int i = 0; i < P; i++) y[i] = fma2(d[i], m[j][i], f[i]);
            __stcs(static_cast<uint4*>(o.y[j]) + at, y.pack());
        }
        before = cur[u];
    }
}

// The gradient.  The J + 1 vectors of a token run MIX_STAGES - 1 tokens ahead through
// a ring in shared memory that is private to the thread (cp.async, no barrier; loads of
// each token as it is needed: 181 us).  Products and sums in pairs of fp32.  J = 6 in 16
// bits takes 184 registers, of them 96 for the weights and their gradient.
template <typename T, int J>
__global__ void __launch_bounds__(MIX_T) token_mix_backward_kernel(const MixArgs a, const MixGrad g) {
    constexpr int VE = Vec16<T>::N, P = VE / 2;
    __shared__ uint4 ring[MIX_STAGES][J + 1][MIX_T];  // dy_j, x
    pdl_trigger();
    const int64_t id = blockIdx.x * (int64_t)MIX_T + threadIdx.x;
    const int slot = (int)(id / a.nvec), v = (int)(id - (int64_t)slot * a.nvec);
    if (slot >= a.slots) return;
    const int64_t first = slot * a.chunk, end = min(first + a.chunk, a.rows);
    const uint4* const x = static_cast<const uint4*>(a.x) + v;
    const uint4* const prev = static_cast<const uint4*>(a.prev) + v;
    uint4* dx = static_cast<uint4*>(g.dx) + first * a.nvec + v;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    float2 nm[J][P], dm[J][P];  // -m_j and dm_j, in pairs
#pragma unroll
    for (int j = 0; j < J; j++) {
        float m[VE];
        load_params<VE>(a.mix, a.mdtype, ((int64_t)j * a.nvec + v) * VE, m);
#pragma unroll
        for (int i = 0; i < P; i++) nm[j][i] = make_float2(-m[2 * i], -m[2 * i + 1]), dm[j][i] = make_float2(0.f, 0.f);
    }
    Token k, ahead;
    k.start(a, first);
    ahead = k;
    // the token after the slot's last is read too, for its part in the last one's gradient
    int64_t left = end - first + 1, at = first * a.nvec;
    // what is not read is filled with zeros
    auto fetch = [&](int stage) {
        const bool real = left > 0 && ahead.t < ahead.len;
#pragma unroll
        for (int j = 0; j < J; j++) {
            const bool read = real && g.dy[j];
            const uint4* p = static_cast<const uint4*>(g.dy[j]) + v;
            copy_async_n<16>(&ring[stage][j][threadIdx.x], read ? p + at : x, read ? 16 : 0);
        }
        copy_async_n<16>(&ring[stage][J][threadIdx.x], real && left > 1 ? x + at : x, real && left > 1 ? 16 : 0);
        copy_commit();
        at += a.nvec;
        left--;
        ahead.next(a);
        if (ahead.b == a.B) left = 0;
    };
#pragma unroll
    for (int i = 0; i < MIX_STAGES - 1; i++) fetch(i);
    auto pairs = [](const uint4& r, float2* f) { Vec16<T>::unpack(r, reinterpret_cast<float*>(f)); };
    auto store = [&](uint4* p, const float2* f) { __stcs(p, Vec16<T>::pack(reinterpret_cast<const float*>(f))); };
    float2 before[P], own[P];  // x of the token before; its gradient so far
    pairs(k.t && k.t < k.len ? x[(first - 1) * a.nvec] : zero, before);
    int stage = 0, put = MIX_STAGES - 1;
    const float2 minus = make_float2(-1.f, -1.f);
    for (int64_t n = end - first, i0 = 0;; n--, i0 = 1, k.next(a)) {
        if (n == 0 && (k.b == a.B || k.t == 0)) break;
        fetch(put);
        copy_wait<MIX_STAGES - 1>();
        float2 back[P], rest[P], f[P], d[P];  // back: -sum m dy
        if (k.t == 0) pairs(k.len > 0 && a.prev ? prev[(int64_t)k.b * a.nvec] : zero, before);
        pairs(ring[stage][J][threadIdx.x], f);
#pragma unroll
        for (int i = 0; i < P; i++) {
            back[i] = rest[i] = make_float2(0.f, 0.f);
            d[i] = fma2(f[i], minus, before[i]);
        }
        const bool real = k.t < k.len;  // no products of what is not, which infinite weights or x would make NaN
        if (n == 0) {  // the next slot's first token goes on with this sequence
            if (!real) break;
#pragma unroll
            for (int j = 0; j < J; j++) {
                float2 dy[P];
                pairs(ring[stage][j][threadIdx.x], dy);
#pragma unroll
                for (int i = 0; i < P; i++) back[i] = fma2(nm[j][i], dy[i], back[i]);
            }
#pragma unroll
            for (int i = 0; i < P; i++) own[i] = fma2(back[i], minus, own[i]);
            break;
        }
        if (real) {
#pragma unroll
            for (int j = 0; j < J; j++) {
                float2 dy[P];
                pairs(ring[stage][j][threadIdx.x], dy);
#pragma unroll
                for (int i = 0; i < P; i++) {
                    back[i] = fma2(nm[j][i], dy[i], back[i]);
                    rest[i] = add2(rest[i], fma2(nm[j][i], dy[i], dy[i]));  // (1 - m) dy, rounded once
                    dm[j][i] = fma2(dy[i], d[i], dm[j][i]);
                }
            }
        }
        if (i0) {
            if (k.t)
#pragma unroll
                for (int i = 0; i < P; i++) own[i] = fma2(back[i], minus, own[i]);
            store(dx, own);
            dx += a.nvec;
        }
        if (k.t == 0 || k.t == k.len - 1) {  // an end of its sequence
            float2 l[P];
            const bool last = g.dlast && (k.t == k.len - 1 || k.len == 0);
            pairs(last ? static_cast<const uint4*>(g.dlast)[(int64_t)k.b * a.nvec + v] : zero, l);
            if (k.len) {
#pragma unroll
                for (int i = 0; i < P; i++) rest[i] = add2(rest[i], l[i]);
            }
            if (k.t == 0 && g.dprev) {
#pragma unroll
                for (int i = 0; i < P; i++) back[i] = k.len ? mul2(back[i], minus) : l[i];
                store(static_cast<uint4*>(g.dprev) + (int64_t)k.b * a.nvec + v, back);
            }
        }
#pragma unroll
        for (int i = 0; i < P; i++) own[i] = rest[i], before[i] = f[i];
        put = stage;
        stage = stage == MIX_STAGES - 1 ? 0 : stage + 1;
    }
    store(dx, own);
    copy_wait<0>();
    if (!g.part) return;
    float* p = g.part + (int64_t)slot * J * a.nvec * VE + (int64_t)v * VE;
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < P; i += 2)
            *reinterpret_cast<float4*>(p + (int64_t)j * a.nvec * VE + 2 * i) =
                make_float4(dm[j][i].x, dm[j][i].y, dm[j][i + 1].x, dm[j][i + 1].y);
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

// Slots of a backward call: 256 threads per SM for six and five ways, 384 for four, 512 for
// fewer (more threads than these are slower: 16384 x 2560 bf16, whole calls with the join and the host's
// part, one way, 512 45 us, 896 53; six ways, 256 118 us, 384 121), four tokens each at least.  By the sizes alone: results repeat.
void plan(MixArgs& a, int J) {
    const int64_t threads = 148 * MIX_T * std::min(4, (14 + (J + 1) / 2) / (J + 1));
    const int64_t most = std::max<int64_t>(1, threads / a.nvec);
    const int64_t slots = std::max<int64_t>(1, std::min((a.rows + 3) / 4, most));
    a.chunk = (a.rows + slots - 1) / slots;
    a.slots = (int)((a.rows + a.chunk - 1) / a.chunk);
}

int vectors(int dtype, int D) { return dtype == RWKV_F32 ? D / 4 : D / 8; }

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_sizes(int dtype, int mdtype, int B, int T, int D, int J, const char* fn) {
    RWKV_REQUIRE(valid_dtype(dtype) && valid_dtype(mdtype), RWKV_E_DTYPE, "%s: dtypes x=%d mix=%d", fn, dtype, mdtype);
    RWKV_REQUIRE(B >= 1 && T >= 1 && D >= 1 && D <= 1 << 20, RWKV_E_SHAPE, "%s: B=%d T=%d D=%d (B, T >= 1, D in 1..2^20)",
                 fn, B, T, D);
    RWKV_REQUIRE((int64_t)B * T <= (1ll << 40) / D, RWKV_E_SHAPE, "%s: B=%d T=%d D=%d (at most 2^40 elements)",
                 fn, B, T, D);
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
    const MixArgs a = make_args(dtype, x, mdtype, mix, prev, lengths, B, T, D);
    return dispatch_dtype(dtype, [&]<typename T_>() {
        return dispatch_ways(J, [&]<int J_>() {
            auto launch = [&]<int U>() {
                const int64_t threads = (a.rows + U - 1) / U * a.nvec;
                token_mix_kernel<T_, J_, U>
                    <<<(unsigned)((threads + MIX_T - 1) / MIX_T), MIX_T, 0, (cudaStream_t)stream>>>(a, o);
            };
            // Few vectors are spread over threads (16384: 2.9 us, by four tokens 3.5), more
            // share a token before and the weights (65536: 4.3 and 3.6 us; 16384 x 2560
            // bf16, six ways: 92 us by four or eight tokens, 97 by two, floor 89).
            if (a.rows * a.nvec > 1 << 15) launch.template operator()<4>();
            else launch.template operator()<1>();
            return check_launch("token_mix_kernel");
        });
    });
}

extern "C" int64_t rwkv_token_mix_backward_workspace_size(int dtype, int B, int T, int D, int J) {
    if (!valid_dtype(dtype) || B < 1 || T < 1 || D < 8 || D % 8 || D > 1 << 20 || J < 1 || J > MIX_WAYS) return 0;
    MixArgs a = make_args(dtype, nullptr, 0, nullptr, nullptr, nullptr, B, T, D);
    plan(a, J);
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
    plan(a, J);
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
