// Dropout from a counter-based generator: whether an element is dropped follows
// from its place in the tensor, a seed and an offset, so that no mask is stored and
// the backward pass draws the same one again.
//
// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", SC 2011): ten rounds of two 32 x 32 -> 64 bit products over a
// 128-bit counter under a 64-bit key give four words.  Counter: the element's block
// (64 bits) and the offset (64 bits); key: the seed.  A block is 8 elements of the
// tensor in row-major order, 16 bits each (element i: half i % 2, low half first, of
// word (i % 8) / 2): 16 bits halve the products per element against 32, which would
// bound the kernels instead of HBM, and round p to a multiple of 2^-16.  What is kept
// is scaled by the inverse of the rounded probability, so that the mean is kept.
#pragma once

#include <cmath>

#include "common.cuh"

namespace rwkv {

struct Dropout {
    uint64_t seed, offset;
    const int64_t* state;  // device [2], or NULL: seed, and what is added to offset
    uint32_t threshold;    // dropped where the 16 bits are below it: 0 none, 65536 all
    float scale;           // of what is kept
};

// p in [0, 1]; scale: a factor of the kept values beside 1 / (1 - p)
inline Dropout make_dropout(double p, double scale, uint64_t seed, uint64_t offset, const int64_t* state) {
    Dropout d{seed, offset, state, (uint32_t)std::nearbyint(p * 65536.0), 0.f};
    d.scale = d.threshold < 65536 ? (float)(scale * (65536.0 / (65536.0 - d.threshold))) : 0.f;
    return d;
}

struct DropKey {
    uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ DropKey drop_key(const Dropout& d) {
    uint64_t seed = d.seed, offset = d.offset;
    if (d.state) {
        seed = (uint64_t)d.state[0];
        offset += (uint64_t)d.state[1];
    }
    return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
}

__device__ __forceinline__ uint4 philox(const DropKey& key, uint64_t block) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = key.o0, c3 = key.o1, k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// v[k] of the 2 N elements that N words stand for: scaled, or 0 where dropped (also
// an infinity or a NaN)
template <int N>
__device__ __forceinline__ void drop(float* v, const uint32_t* words, uint32_t threshold, float scale) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[2 * i] = (words[i] & 0xffffu) < threshold ? 0.f : __fmul_rn(v[2 * i], scale);
        v[2 * i + 1] = (words[i] >> 16) < threshold ? 0.f : __fmul_rn(v[2 * i + 1], scale);
    }
}
// N (4 or 8) consecutive elements from element i on, i a multiple of N
template <int N>
__device__ __forceinline__ void drop_at(float* v, const DropKey& key, uint64_t i, uint32_t threshold, float scale) {
    if (threshold == 0) {
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = __fmul_rn(v[k], scale);
        return;
    }
    const uint4 r = philox(key, i >> 3);
    if constexpr (N == 8) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        drop<4>(v, w, threshold, scale);
    } else {
        const uint32_t w[2] = {i & 4 ? r.z : r.x, i & 4 ? r.w : r.y};
        drop<2>(v, w, threshold, scale);
    }
}

}  // namespace rwkv
