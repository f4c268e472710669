// Pairs of fp32 in one instruction (sm_100a): each half as fmaf and + round it.
#pragma once

#include "ckpt8.cuh"

namespace rwkv {

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
        "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// A 16-byte vector of T as pairs.
template <typename T>
struct Pairs {
    static constexpr int VE = Vec16<T>::N, P = VE / 2;
    float2 f[P];
    __device__ __forceinline__ void unpack(const uint4& r) { Vec16<T>::unpack(r, reinterpret_cast<float*>(f)); }
    __device__ __forceinline__ uint4 pack() const { return Vec16<T>::pack(reinterpret_cast<const float*>(f)); }
    __device__ __forceinline__ float* floats() { return reinterpret_cast<float*>(f); }
    __device__ __forceinline__ float2& operator[](int i) { return f[i]; }
    __device__ __forceinline__ const float2& operator[](int i) const { return f[i]; }
};

}  // namespace rwkv
