// 8-bit activation checkpoints and the activations of the projection epilogue,
// shared by the layer-norm, projection and checkpoint kernels.
//
// Checkpoint of a row-major [rows, D] tensor: per row and group of 32
// consecutive channels one scale s = 2^E, the power of two with
// max|x| / s in [64, 128) (E >= -126), and int8 codes q = round(x / s), ties
// to even, clipped to [-127, 127].  x / s and s q are exact in fp32 and s q is
// exact in bf16 (7 significant bits), so decoding into a bf16 tensor-core
// operand loses nothing; |x - s q| <= max|x| / 127.5, or 2^-127 where max|x| < 2^-120
// and E stays at -126.  (A scale max|x| / 127
// would gain up to one bit where max|x| / s is near 64, and would cost an
// inexact product in every decode and four bytes per group instead of one.)
// A group that holds an infinity or a NaN stands for NaN: exponent byte 255
// with codes 0.  Scales are stored as E + 127 in one byte: 1 + 1/32 bytes per
// element.
#pragma once

#include <type_traits>

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
// Four codes as a word.  x / s + 1.5 2^23 is rounded once, to the integer round(x
// / s) above 1.5 2^23, whose low byte is the code; clipping is on that scale.
// One fused multiply-add and two min / max per code, where a conversion to
// integer runs at a quarter of the rate.
__device__ __forceinline__ uint32_t ck_pack4(float a, float b, float c, float d, float inv) {
    constexpr float M = 12582912.f;
    auto code = [inv](float x) {
        return __float_as_uint(fminf(fmaxf(fmaf(x, inv, M), M - 127.f), M + 127.f));
    };
    const uint32_t w = __byte_perm(__byte_perm(code(a), code(b), 0x0040), __byte_perm(code(c), code(d), 0x0040), 0x5410);
    return inv == 0.f ? 0u : w;  // a NaN group
}
// Bits of the largest |x| of a 16-byte vector of T, comparable across a group
// (for 16-bit types in 16 bits, compared two at a time), and its fp32 form.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const uint4& r) {
    if constexpr (sizeof(T) == 4) {
        return max(max(r.x & 0x7fffffffu, r.y & 0x7fffffffu), max(r.z & 0x7fffffffu, r.w & 0x7fffffffu));
    } else {
        const uint32_t m = __vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu),
                                    __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
        return max(m >> 16, m & 0xffffu);
    }
}
template <typename T>
__device__ __forceinline__ uint32_t top_f32(uint32_t top) {
    if constexpr (sizeof(T) == 4) return top;
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return top << 16;
    else return abs_bits(__half2float(__ushort_as_half((unsigned short)top)));
}
// The four codes of a word as floats.  Byte ^ 0x80 is q + 128; placed in the low
// mantissa of 2^23 it reads 2^23 + q + 128 exactly.
__device__ __forceinline__ void ck_codes4(uint32_t w, float* q) {
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u | (uint32_t)i)) - 8388736.f;
}
__device__ __forceinline__ void ck_unpack4(uint32_t w, float s, float* v) {
    ck_codes4(w, v);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] *= s;
}

// ---------------------------------------------------------------- activations

// act(z) and act'(z).  Comparisons are written so that a NaN passes through.
// tanh and sigmoid and their derivatives come from e = exp(-2|z|) or exp(-|z|),
// which is at most 1, so that nothing overflows and no derivative cancels:
//   tanh = (1 - e) / (1 + e) with z's sign, tanh' = 4 e / (1 + e)^2
//   sigmoid = (1 or e) / (1 + e) by z's sign, sigmoid' = e / (1 + e)^2
// FAST: __expf (2 + |1.16 x| ulp) and __fdividef (2 ulp), for results that are rounded
// to 16 bits: tanh within 2^-18 relative (at |z| = 2^-6, where 1 - e = 2^-5 is off by
// 2^-23 from e), sigmoid and the derivatives as e, 2^-18 at |z| = 10 and 2^-16 where
// bf16 ends; below |z| = 2^-6, where 1 - e cancels further, tanh z = z - z^3 / 3 (next
// term z^5 2/15 < 2^-26 z).  Otherwise expf, tanhf and IEEE division.
template <int ACT, bool FAST>
__device__ __forceinline__ float act_t(float z) {
    if constexpr (ACT == RWKV_ACT_RELU2) {
        const float m = z < 0.f ? 0.f : z;
        return m * m;
    } else if constexpr (ACT == RWKV_ACT_TANH) {
        if constexpr (!FAST) return tanhf(z);
        const float e = __expf(-2.f * fabsf(z));
        const float t = copysignf(__fdividef(1.f - e, 1.f + e), z);
        return fabsf(z) < 0.015625f ? fmaf(z * z * z, -1.f / 3.f, z) : t;
    } else if constexpr (ACT == RWKV_ACT_SIGMOID) {
        const float e = FAST ? __expf(-fabsf(z)) : expf(-fabsf(z)), n = z < 0.f ? e : 1.f;
        return FAST ? __fdividef(n, 1.f + e) : n / (1.f + e);
    }
    return z;
}
template <int ACT, bool FAST>
__device__ __forceinline__ float act_grad_t(float z) {
    if constexpr (ACT == RWKV_ACT_RELU2) {
        return z < 0.f ? 0.f : 2.f * z;
    } else if constexpr (ACT == RWKV_ACT_TANH || ACT == RWKV_ACT_SIGMOID) {
        constexpr float k = ACT == RWKV_ACT_TANH ? 2.f : 1.f;
        if constexpr (!FAST) {
            const float e = expf(-k * fabsf(z)), d = 1.f + e;
            return k * k * e / (d * d);
        }
        const float e = __expf(-k * fabsf(z)), r = __fdividef(k, 1.f + e);
        return e * r * r;
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
struct Vec16;
template <>
struct Vec16<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
        v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y);
        v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
// Two 16-bit values in a word: one instruction each way for bf16 where element
// access through the vector's address takes two.
template <typename T>
__device__ __forceinline__ float2 word_floats(uint32_t w) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t floats_word(float lo, float hi) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
template <typename T>
struct Vec16 {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = word_floats<T>(w[i]);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        return make_uint4(floats_word<T>(v[0], v[1]), floats_word<T>(v[2], v[3]), floats_word<T>(v[4], v[5]),
                          floats_word<T>(v[6], v[7]));
    }
};

// 8 elements as read and as floats, 16-byte accesses
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

// VE (4 or 8) consecutive elements of a parameter vector kept in fp32, bf16 or
// fp16, from a 16-byte aligned vector; one element of it.
template <int VE>
__device__ __forceinline__ void load_params(const void* p, int dtype, int64_t i, float* v) {
    if (dtype == RWKV_F32) {
#pragma unroll
        for (int k = 0; k < VE; k += 4) {
            const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + k);
            v[k] = f.x, v[k + 1] = f.y, v[k + 2] = f.z, v[k + 3] = f.w;
        }
        return;
    }
    uint32_t w[VE / 2];
    const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
    if constexpr (VE == 8) {
        const uint4 r = *reinterpret_cast<const uint4*>(q);
        w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
    } else {
        const uint2 r = *reinterpret_cast<const uint2*>(q);
        w[0] = r.x, w[1] = r.y;
    }
#pragma unroll
    for (int k = 0; k < VE / 2; k++) {
        const float2 f = dtype == RWKV_BF16 ? make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u))
                                            : __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
    }
}
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
