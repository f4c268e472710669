// 8-bit activation checkpoints and the activations of the projection epilogue,
// shared by the layer-norm, projection and checkpoint kernels.
//
// Checkpoint of a row-major [rows, D] tensor: per row and group of 32
// consecutive channels one scale s = 2^E, the power of two with
// max|x| / s in [64, 128) (E >= -126), and int8 codes q = round(x / s), ties
// to even, clipped to [-127, 127].  x / s and s q are exact in fp32 and s q is
// exact in bf16 (7 significant bits), so decoding into a bf16 tensor-core
// operand loses nothing; |x - s q| <= max|x| / 127.5.  (A scale max|x| / 127
// would gain up to one bit where max|x| / s is near 64, and would cost an
// inexact product in every decode and four bytes per group instead of one.)
// A group that holds an infinity or a NaN stands for NaN: exponent byte 255
// with codes 0.  Scales are stored as E + 127 in one byte: 1 + 1/32 bytes per
// element.
#pragma once

#include "common.cuh"

namespace rwkv {

constexpr int CK_GROUP = 32;

// Bits of |x|: as unsigned integers they order like |x|, infinity above every
// finite value and NaN above infinity, so a group's largest needs no float max
// (which would drop NaN).
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The stored exponent byte of a group from the bits of its largest |x|.
__device__ __forceinline__ uint32_t ck_exponent(uint32_t top) {
    const int b = (int)(top >> 23);
    return b == 255 ? 255u : (uint32_t)max(b - 6, 1);
}
// 1 / s for exponent byte e (0 for a NaN group, whose codes are 0)
__device__ __forceinline__ float ck_inv_scale(uint32_t e) {
    return e == 255 ? 0.f : __uint_as_float((254u - e) << 23);
}
// s; infinity for a NaN group, so that 0 * s is NaN
__device__ __forceinline__ float ck_scale(uint32_t e) { return __uint_as_float(e << 23); }

// The code of x.  In a NaN group (inv == 0) the product is 0 or NaN and
// __float2int_rn turns NaN into 0.
__device__ __forceinline__ int ck_code(float x, float inv) {
    return max(-127, min(127, __float2int_rn(__fmul_rn(x, inv))));
}
__device__ __forceinline__ uint32_t ck_pack4(float a, float b, float c, float d, float inv) {
    return (uint32_t)(ck_code(a, inv) & 255) | ((uint32_t)(ck_code(b, inv) & 255) << 8) |
           ((uint32_t)(ck_code(c, inv) & 255) << 16) | ((uint32_t)(ck_code(d, inv) & 255) << 24);
}
// The four values of a word of codes.  Byte ^ 0x80 is q + 128; placed in the
// low mantissa of 2^23 it reads 2^23 + q + 128 exactly.
__device__ __forceinline__ void ck_unpack4(uint32_t w, float s, float* v) {
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; i++)
        v[i] = (__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u | (uint32_t)i)) - 8388736.f) * s;
}

// ---------------------------------------------------------------- activations

// act(z).  Comparisons are written so that a NaN passes through.
template <int ACT>
__device__ __forceinline__ float act_t(float z) {
    if constexpr (ACT == RWKV_ACT_RELU2) {
        const float m = z < 0.f ? 0.f : z;
        return m * m;
    } else if constexpr (ACT == RWKV_ACT_TANH) {
        return tanhf(z);
    } else if constexpr (ACT == RWKV_ACT_SIGMOID) {
        return 1.f / (1.f + expf(-z));
    }
    return z;
}
// act'(z).  tanh' = 4 e / (1 + e)^2 with e = exp(-2|z|) and sigmoid' =
// e / (1 + e)^2 with e = exp(-|z|): no cancellation for large |z|.
template <int ACT>
__device__ __forceinline__ float act_grad_t(float z) {
    if constexpr (ACT == RWKV_ACT_RELU2) {
        return z < 0.f ? 0.f : 2.f * z;
    } else if constexpr (ACT == RWKV_ACT_TANH) {
        const float e = expf(-2.f * fabsf(z)), d = 1.f + e;
        return 4.f * e / (d * d);
    } else if constexpr (ACT == RWKV_ACT_SIGMOID) {
        const float e = expf(-fabsf(z)), d = 1.f + e;
        return e / (d * d);
    }
    return 1.f;
}
// The activation as a run-time value: f.template operator()<ACT>().
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
    if (act == RWKV_ACT_RELU2) f.template operator()<RWKV_ACT_RELU2>();
    else if (act == RWKV_ACT_TANH) f.template operator()<RWKV_ACT_TANH>();
    else if (act == RWKV_ACT_SIGMOID) f.template operator()<RWKV_ACT_SIGMOID>();
    else f.template operator()<RWKV_ACT_NONE>();
}
inline bool valid_act(int a) { return a >= RWKV_ACT_NONE && a <= RWKV_ACT_SIGMOID; }

// --------------------------------------------------- 16-byte vectors of T

template <typename T>
struct Vec16 {
    static constexpr int N = 16 / (int)sizeof(T);
    static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
        const T* p = reinterpret_cast<const T*>(&r);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = to_f<T>(p[i]);
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        uint4 r;
        T* p = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = from_f<T>(v[i]);
        return r;
    }
};

// One element of a parameter vector kept in fp32, bf16 or fp16.
__device__ __forceinline__ float load_param(const void* p, int dtype, int64_t i) {
    if (dtype == RWKV_F32) return static_cast<const float*>(p)[i];
    if (dtype == RWKV_BF16) return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
    return to_f(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
    if (dtype == RWKV_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == RWKV_BF16) static_cast<__nv_bfloat16*>(p)[i] = from_f<__nv_bfloat16>(v);
    else static_cast<__half*>(p)[i] = from_f<__half>(v);
}

}  // namespace rwkv
