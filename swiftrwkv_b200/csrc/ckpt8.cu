// 8-bit activation checkpoints: packing, restoring (optionally through an
// activation), and the activation's gradient from a checkpoint or from the
// pre-activation itself.
//
// All three are one pass over memory and bound by HBM.  The unit of work is 8
// channels (16-byte accesses of the tensors, two for fp32, 8 bytes of codes); a
// thread takes CU units CT apart, all loads first, and four neighbouring
// threads find the largest |x| of their group of 32 with two shuffles.  Where
// D % 32 == 0 the whole tensor is one long row of groups and nothing is
// divided.  The uses read any D in units (groups looked up by element where D %
// 32 != 0); packing takes rows of D % 8 == 0 in units and others a warp per
// group.
#include <algorithm>

#include "ckpt8.cuh"

namespace rwkv {
namespace {

constexpr int CT = 256;

// 8 elements of a row as read and as floats, 16-byte accesses
template <typename T>
struct Raw8 {
    static constexpr int W = 8 / Vec16<T>::N;
    uint4 r[W];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < W; i++) r[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < W; i++) r[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void floats(float* v) const {
#pragma unroll
        for (int i = 0; i < W; i++) Vec16<T>::unpack(r[i], v + i * Vec16<T>::N);
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t t = top_bits<T>(r[0]);
        if constexpr (W == 2) t = max(t, top_bits<T>(r[1]));
        return t;
    }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
#pragma unroll
    for (int i = 0; i < 8 / Vec16<T>::N; i++)
        __stcs(reinterpret_cast<uint4*>(p) + i, Vec16<T>::pack(v + i * Vec16<T>::N));
}

constexpr int CU = 4;

// FLAT: D % 32 == 0, rows run on.  Otherwise units are counted in rows padded
// to whole groups (4 units), so that a group's units are neighbours in a warp.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(CT, 1) ckpt8_pack_kernel(const T* __restrict__ x, int8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ exps, int64_t units, int D, int G) {
    const int64_t i0 = blockIdx.x * (int64_t)(CT * CU) + threadIdx.x;
    Raw8<T> raw[CU];
    int64_t at[CU];
    bool in[CU];
#pragma unroll
    for (int j = 0; j < CU; j++) {
        const int64_t i = i0 + j * CT;
        in[j] = i < units;
        at[j] = 8 * i;
        if constexpr (!FLAT) {
            const int64_t row = units < (1ll << 32) ? (uint32_t)i / (uint32_t)(4 * G) : i / (4 * G);
            const int u = (int)(i - row * (4 * G));
            in[j] = in[j] && 8 * u < D;
            at[j] = row * D + 8 * u;
        }
        raw[j].zero();
        if (in[j]) raw[j].load(x + at[j]);
    }
#pragma unroll
    for (int j = 0; j < CU; j++) {
        uint32_t top = raw[j].top();
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = ck_exponent(top_f32<T>(top));
        const float inv = ck_inv_scale(e);
        if (in[j]) {
            float v[8];
            raw[j].floats(v);
            __stcs(reinterpret_cast<uint2*>(codes + at[j]), make_uint2(ck_pack4(v[0], v[1], v[2], v[3], inv),
                                                                       ck_pack4(v[4], v[5], v[6], v[7], inv)));
            if (((i0 + j * CT) & 3) == 0) exps[(i0 + j * CT) >> 2] = (uint8_t)e;
        }
    }
}

// Any D and alignment: a warp per group, 8 groups at a time.
template <typename T>
__global__ void __launch_bounds__(CT, 1) ckpt8_pack_any_kernel(const T* __restrict__ x, int8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ exps, int64_t groups, int D, int G) {
    const int lane = threadIdx.x & 31;
    const int64_t g0 = ((blockIdx.x * (int64_t)CT + threadIdx.x) >> 5) * 8;
    float v[8];
    int64_t at[8];
    bool in[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int64_t g = g0 + j;
        const int64_t row = groups < (1ll << 32) ? (uint32_t)g / (uint32_t)G : g / G;
        const int c = (int)(g - row * G) * CK_GROUP + lane;
        in[j] = g < groups && c < D;
        at[j] = row * D + c;
        v[j] = in[j] ? to_f<T>(x[at[j]]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t e = ck_exponent(__reduce_max_sync(0xffffffffu, abs_bits(v[j])));
        if (in[j]) codes[at[j]] = (int8_t)ck_code(v[j], ck_inv_scale(e));
        if (lane == 0 && g0 + j < groups) exps[g0 + j] = (uint8_t)e;
    }
}

// MODE 0: out = act(value).  MODE 1: out = dy * act'(value), MODE 2: out =
// dy * act'(z), z dense.  Elementary functions in fp32 precision where the result
// is fp32.
template <int MODE, int ACT, typename T, bool FLAT>
__global__ void __launch_bounds__(CT, 1) ckpt8_use_kernel(const T* dy, const T* __restrict__ z,
                                                       const int8_t* __restrict__ codes,
                                                       const uint8_t* __restrict__ exps, T* out, int64_t n, int D,
                                                       int G) {
    constexpr bool FAST = sizeof(T) == 2, HAS_DY = MODE != 0;
    const int64_t i0 = blockIdx.x * (int64_t)(CT * CU) + threadIdx.x, units = n / 8;
    Raw8<T> rz[CU], rd[CU];
    uint2 w[CU];
    uint32_t e[CU];
#pragma unroll
    for (int j = 0; j < CU; j++) {
        const int64_t i = i0 + j * CT;
        if (i >= units) continue;
        if constexpr (MODE == 2) rz[j].load(z + 8 * i);
        else w[j] = __ldcs(reinterpret_cast<const uint2*>(codes + 8 * i));
        if constexpr (MODE < 2 && FLAT) e[j] = exps[i >> 2];
        if constexpr (HAS_DY) rd[j].load(dy + 8 * i);
    }
#pragma unroll
    for (int j = 0; j < CU; j++) {
        const int64_t i = i0 + j * CT;
        if (i >= units) continue;
        float v[8], d[8];
        if constexpr (MODE == 2) {
            rz[j].floats(v);
        } else {
            if constexpr (FLAT) {
                const float s = ck_scale(e[j]);
                ck_unpack4(w[j].x, s, v);
                ck_unpack4(w[j].y, s, v + 4);
            } else {
                ck_codes4(w[j].x, v);
                ck_codes4(w[j].y, v + 4);
                int64_t row = n < (1ll << 32) ? (uint32_t)(8 * i) / (uint32_t)D : 8 * i / D;
                int c = (int)(8 * i - row * D);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    v[k] *= ck_scale(exps[row * G + c / CK_GROUP]);
                    if (++c == D) c = 0, row++;
                }
            }
        }
        if constexpr (HAS_DY) rd[j].floats(d);
#pragma unroll
        for (int k = 0; k < 8; k++)
            v[k] = HAS_DY ? d[k] * act_grad_t<ACT, FAST>(v[k]) : act_t<ACT, FAST>(v[k]);
        store8(out + 8 * i, v);
    }
    // the tensor's last n % 8 elements
    const int64_t t = 8 * units + threadIdx.x;
    if (blockIdx.x == 0 && t < n) {
        float f;
        if constexpr (MODE == 2) f = to_f<T>(z[t]);
        else f = (float)codes[t] * ck_scale(exps[t / D * G + (int)(t % D) / CK_GROUP]);
        if constexpr (HAS_DY) out[t] = from_f<T>(to_f<T>(dy[t]) * act_grad_t<ACT, FAST>(f));
        else out[t] = from_f<T>(act_t<ACT, FAST>(f));
    }
}

// Misaligned tensors: single elements.
template <int MODE, int ACT, typename T>
__global__ void __launch_bounds__(CT, 1) ckpt8_use_any_kernel(const T* dy, const T* __restrict__ z,
                                                           const int8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ exps, T* out, int64_t n, int D,
                                                           int G) {
    constexpr bool FAST = sizeof(T) == 2;
    for (int64_t i = blockIdx.x * (int64_t)CT + threadIdx.x; i < n; i += (int64_t)gridDim.x * CT) {
        const int64_t row = i / D;
        float v;
        if constexpr (MODE == 2) v = to_f<T>(z[i]);
        else v = (float)codes[i] * ck_scale(exps[row * G + (int)(i - row * D) / CK_GROUP]);
        if constexpr (MODE == 0) out[i] = from_f<T>(act_t<ACT, FAST>(v));
        else out[i] = from_f<T>(to_f<T>(dy[i]) * act_grad_t<ACT, FAST>(v));
    }
}

bool al(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int units_grid(int64_t units) { return std::max(1, ceil_div(units, CT * CU)); }

template <typename F>
int dispatch_act(int act, F&& f) {
    switch (act) {
        case RWKV_ACT_RELU2: return f.template operator()<RWKV_ACT_RELU2>();
        case RWKV_ACT_TANH: return f.template operator()<RWKV_ACT_TANH>();
        case RWKV_ACT_SIGMOID: return f.template operator()<RWKV_ACT_SIGMOID>();
        default: return f.template operator()<RWKV_ACT_NONE>();
    }
}

template <int MODE>
int launch_use(int dtype, const void* dy, const void* z, const int8_t* codes, const uint8_t* exps, int act, void* out,
               int rows, int D, cudaStream_t st, const char* fn) {
    const int G = ceil_div(D, CK_GROUP);
    const int64_t n = (int64_t)rows * D;
    const bool vec = al(dy, 16) && al(z, 16) && al(codes, 8) && al(out, 16), flat = D % CK_GROUP == 0;
    return dispatch_dtype(dtype, [&]<typename T>() {
        return dispatch_act(act, [&]<int ACT>() {
            const T *d = (const T*)dy, *x = (const T*)z;
            T* o = (T*)out;
            if (!vec)
                ckpt8_use_any_kernel<MODE, ACT, T>
                    <<<(int)std::min<int64_t>((n + CT - 1) / CT, 148 * 16), CT, 0, st>>>(d, x, codes, exps, o, n, D, G);
            else if (flat || MODE == 2)  // dense z needs no groups
                ckpt8_use_kernel<MODE, ACT, T, true><<<units_grid(n / 8), CT, 0, st>>>(d, x, codes, exps, o, n, D, G);
            else
                ckpt8_use_kernel<MODE, ACT, T, false><<<units_grid(n / 8), CT, 0, st>>>(d, x, codes, exps, o, n, D, G);
            return check_launch(fn);
        });
    });
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

static int check_rows(int rows, int D, const char* fn) {
    RWKV_REQUIRE(rows >= 1 && D >= 1 && D <= 1 << 30 && (int64_t)rows * D <= 1ll << 40, RWKV_E_SHAPE,
                 "%s: rows=%d D=%d (rows >= 1, D in 1..2^30, at most 2^40 elements)", fn, rows, D);
    return RWKV_OK;
}

static bool aligned_to(const void* p, int dtype) {
    return ((uintptr_t)p & (dtype == RWKV_F32 ? 3u : 1u)) == 0;
}

extern "C" int rwkv_ckpt8_pack(int dtype, const void* x, int8_t* codes, uint8_t* exps, int rows, int D,
                               rwkv_stream_t stream) {
    const char* fn = "rwkv_ckpt8_pack";
    RWKV_REQUIRE(valid_dtype(dtype), RWKV_E_DTYPE, "%s: dtype %d", fn, dtype);
    RWKV_REQUIRE(x && codes && exps, RWKV_E_NULL, "%s: NULL argument", fn);
    if (int rc = check_rows(rows, D, fn)) return rc;
    RWKV_REQUIRE(aligned_to(x, dtype), RWKV_E_UNSUPPORTED, "%s: x not aligned to its element type", fn);
    const int G = ceil_div(D, CK_GROUP);
    const int64_t groups = (int64_t)rows * G;
    cudaStream_t st = (cudaStream_t)stream;
    const bool vec = D % 8 == 0 && al(x, 16) && al(codes, 8);
    return dispatch_dtype(dtype, [&]<typename T>() {
        if (vec && D % CK_GROUP == 0)
            ckpt8_pack_kernel<T, true><<<units_grid(4 * groups), CT, 0, st>>>((const T*)x, codes, exps, 4 * groups, D, G);
        else if (vec)
            ckpt8_pack_kernel<T, false><<<units_grid(4 * groups), CT, 0, st>>>((const T*)x, codes, exps, 4 * groups, D, G);
        else
            ckpt8_pack_any_kernel<T><<<ceil_div(groups, CT / 32 * 8), CT, 0, st>>>((const T*)x, codes, exps, groups, D, G);
        return check_launch(fn);
    });
}

extern "C" int rwkv_ckpt8_values(const int8_t* codes, const uint8_t* exps, int act, int odtype, void* out, int rows,
                                 int D, rwkv_stream_t stream) {
    const char* fn = "rwkv_ckpt8_values";
    RWKV_REQUIRE(valid_dtype(odtype), RWKV_E_DTYPE, "%s: dtype %d", fn, odtype);
    RWKV_REQUIRE(valid_act(act), RWKV_E_UNSUPPORTED, "%s: activation %d", fn, act);
    RWKV_REQUIRE(codes && exps && out, RWKV_E_NULL, "%s: NULL argument", fn);
    if (int rc = check_rows(rows, D, fn)) return rc;
    RWKV_REQUIRE(aligned_to(out, odtype), RWKV_E_UNSUPPORTED, "%s: out not aligned to its element type", fn);
    return launch_use<0>(odtype, nullptr, nullptr, codes, exps, act, out, rows, D, (cudaStream_t)stream, fn);
}

extern "C" int rwkv_act_backward(int dtype, const void* dy, const void* z, const int8_t* codes, const uint8_t* exps,
                                 int act, void* dz, int rows, int D, rwkv_stream_t stream) {
    const char* fn = "rwkv_act_backward";
    RWKV_REQUIRE(valid_dtype(dtype), RWKV_E_DTYPE, "%s: dtype %d", fn, dtype);
    RWKV_REQUIRE(valid_act(act), RWKV_E_UNSUPPORTED, "%s: activation %d", fn, act);
    RWKV_REQUIRE(dy && dz, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(z ? !codes && !exps : codes && exps, RWKV_E_NULL, "%s: give either z or codes and exps", fn);
    if (int rc = check_rows(rows, D, fn)) return rc;
    RWKV_REQUIRE(aligned_to(dy, dtype) && aligned_to(z, dtype) && aligned_to(dz, dtype), RWKV_E_UNSUPPORTED,
                 "%s: a tensor is not aligned to its element type", fn);
    return z ? launch_use<2>(dtype, dy, z, nullptr, nullptr, act, dz, rows, D, (cudaStream_t)stream, fn)
             : launch_use<1>(dtype, dy, nullptr, codes, exps, act, dz, rows, D, (cudaStream_t)stream, fn);
}
