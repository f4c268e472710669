// 8-bit activation checkpoints: packing, restoring (optionally through an
// activation), and the activation's gradient from a checkpoint or from the
// pre-activation itself.
//
// All three are one pass over memory and bound by HBM: every thread moves 8
// channels with 16-byte accesses (two for fp32) and 8-byte accesses of the
// codes, and the four threads of a group of 32 find its largest |x| with two
// shuffles.  Rows whose length is not a multiple of 8, or pointers that are not
// 16-byte aligned, take a kernel with a warp per group and single elements.
#include "ckpt8.cuh"

namespace rwkv {
namespace {

constexpr int CT = 256;

// 8 elements of a row as floats and back, 16-byte accesses
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
#pragma unroll
    for (int i = 0; i < 8 / Vec16<T>::N; i++)
        Vec16<T>::unpack(reinterpret_cast<const uint4*>(p)[i], v + i * Vec16<T>::N);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
#pragma unroll
    for (int i = 0; i < 8 / Vec16<T>::N; i++)
        reinterpret_cast<uint4*>(p)[i] = Vec16<T>::pack(v + i * Vec16<T>::N);
}

// Unit of work: 8 channels.  A row is padded to whole groups (4 units), so
// that a group's four units are four consecutive threads of one warp.
struct Unit {
    int64_t row;
    int u;
    bool in;
};
__device__ __forceinline__ Unit unit_at(int64_t i, int D, int G) {
    Unit r;
    r.row = i / (4 * G);
    r.u = (int)(i - r.row * (4 * G));
    r.in = 8 * r.u < D;
    return r;
}

template <typename T>
__global__ void __launch_bounds__(CT) ckpt8_pack_kernel(const T* __restrict__ x, int8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ exps, int64_t units, int D, int G) {
    // the loop runs whole warps: units is a multiple of 4 and i differs by lane only
    for (int64_t i0 = blockIdx.x * (int64_t)CT; i0 < units; i0 += (int64_t)gridDim.x * CT) {
        const int64_t i = i0 + threadIdx.x;
        const Unit t = unit_at(i < units ? i : 0, D, G);
        const bool in = i < units && t.in;
        float v[8] = {};
        const int64_t at = t.row * D + 8 * t.u;
        if (in) load8(x + at, v);
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) top = max(top, abs_bits(v[k]));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = ck_exponent(top);
        const float inv = ck_inv_scale(e);
        if (in) {
            const uint2 w = {ck_pack4(v[0], v[1], v[2], v[3], inv), ck_pack4(v[4], v[5], v[6], v[7], inv)};
            *reinterpret_cast<uint2*>(codes + at) = w;
            if ((t.u & 3) == 0) exps[t.row * G + (t.u >> 2)] = (uint8_t)e;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(CT) ckpt8_pack_any_kernel(const T* __restrict__ x, int8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ exps, int64_t groups, int D, int G) {
    const int lane = threadIdx.x & 31;
    for (int64_t g = (blockIdx.x * (int64_t)CT + threadIdx.x) >> 5; g < groups; g += ((int64_t)gridDim.x * CT) >> 5) {
        const int64_t row = g / G;
        const int c = (int)(g - row * G) * CK_GROUP + lane;
        const float v = c < D ? to_f<T>(x[row * D + c]) : 0.f;
        const uint32_t e = ck_exponent(__reduce_max_sync(0xffffffffu, abs_bits(v)));
        if (c < D) codes[row * D + c] = (int8_t)ck_code(v, ck_inv_scale(e));
        if (lane == 0) exps[g] = (uint8_t)e;
    }
}

// MODE 0: out = act(value).  MODE 1: out = dy * act'(value), MODE 2: out =
// dy * act'(z), z dense.  MODE 3: out = act(z).
template <int MODE, int ACT, typename T>
__global__ void __launch_bounds__(CT) ckpt8_use_kernel(const T* dy, const T* __restrict__ z,
                                                       const int8_t* __restrict__ codes,
                                                       const uint8_t* __restrict__ exps, T* out, int64_t units, int D,
                                                       int G) {
    const int per = D / 8;
    for (int64_t i = blockIdx.x * (int64_t)CT + threadIdx.x; i < units; i += (int64_t)gridDim.x * CT) {
        const int64_t row = i / per, at = 8 * i;
        float v[8], o[8];
        if constexpr (MODE >= 2) {
            load8(z + at, v);
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(codes + at);
            const float s = ck_scale(exps[row * G + ((int)(i - row * per) >> 2)]);
            ck_unpack4(w.x, s, v);
            ck_unpack4(w.y, s, v + 4);
        }
        if constexpr (MODE == 0 || MODE == 3) {
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = act_t<ACT>(v[k]);
        } else {
            load8(dy + at, o);
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] *= act_grad_t<ACT>(v[k]);
        }
        store8(out + at, o);
    }
}

template <int MODE, int ACT, typename T>
__global__ void __launch_bounds__(CT) ckpt8_use_any_kernel(const T* dy, const T* __restrict__ z,
                                                           const int8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ exps, T* out, int64_t n, int D,
                                                           int G) {
    for (int64_t i = blockIdx.x * (int64_t)CT + threadIdx.x; i < n; i += (int64_t)gridDim.x * CT) {
        const int64_t row = i / D;
        float v;
        if constexpr (MODE >= 2) v = to_f<T>(z[i]);
        else v = (float)codes[i] * ck_scale(exps[row * G + (int)(i - row * D) / CK_GROUP]);
        if constexpr (MODE == 0 || MODE == 3) out[i] = from_f<T>(act_t<ACT>(v));
        else out[i] = from_f<T>(to_f<T>(dy[i]) * act_grad_t<ACT>(v));
    }
}

bool al(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int grid_for(int64_t threads) {
    const int64_t g = (threads + CT - 1) / CT;
    return (int)std::max<int64_t>(1, std::min<int64_t>(g, 148 * 16));
}

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
    const bool vec = D % 8 == 0 && al(dy, 16) && al(z, 16) && al(codes, 8) && al(out, 16);
    return dispatch_dtype(dtype, [&]<typename T>() {
        return dispatch_act(act, [&]<int ACT>() {
            if (vec)
                ckpt8_use_kernel<MODE, ACT, T><<<grid_for(n / 8), CT, 0, st>>>((const T*)dy, (const T*)z, codes, exps,
                                                                              (T*)out, n / 8, D, G);
            else
                ckpt8_use_any_kernel<MODE, ACT, T><<<grid_for(n), CT, 0, st>>>((const T*)dy, (const T*)z, codes, exps,
                                                                              (T*)out, n, D, G);
            return check_launch(fn);
        });
    });
}

}  // namespace

int launch_ckpt8_values(const int8_t* codes, const uint8_t* exps, int act, int odtype, void* out, int rows, int D,
                        cudaStream_t st) {
    return launch_use<0>(odtype, nullptr, nullptr, codes, exps, act, out, rows, D, st, "ckpt8_values_kernel");
}
int launch_act(int dtype, const void* z, int act, void* out, int rows, int D, cudaStream_t st) {
    return launch_use<3>(dtype, nullptr, z, nullptr, nullptr, act, out, rows, D, st, "act_kernel");
}

}  // namespace rwkv

using namespace rwkv;

static int check_rows(int rows, int D, const char* fn) {
    RWKV_REQUIRE(rows >= 1 && D >= 1 && D <= 1 << 30, RWKV_E_SHAPE, "%s: rows=%d D=%d (rows >= 1, D in 1..2^30)", fn,
                 rows, D);
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
        if (vec)
            ckpt8_pack_kernel<T><<<grid_for(4 * groups), CT, 0, st>>>((const T*)x, codes, exps, 4 * groups, D, G);
        else
            ckpt8_pack_any_kernel<T><<<grid_for(32 * groups), CT, 0, st>>>((const T*)x, codes, exps, groups, D, G);
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
    return launch_ckpt8_values(codes, exps, act, odtype, out, rows, D, (cudaStream_t)stream);
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
