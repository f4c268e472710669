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
    const int64_t* state;  // device [2], or NULL: the seed, and what is added to offset
    uint64_t offset;
    uint32_t keys[20];     // without state: the rounds' keys (in constant memory, where they cost nothing)
    uint32_t threshold;    // dropped where the 16 bits are below it: 0 none, 65536 all
    float scale;           // of what is kept
};

constexpr uint32_t PHILOX_K0 = 0x9E3779B9u, PHILOX_K1 = 0xBB67AE85u;  // added to the key's words each round

// p in [0, 1]; scale: a factor of the kept values beside 1 / (1 - p)
inline Dropout make_dropout(double p, double scale, uint64_t seed, uint64_t offset, const int64_t* state) {
    Dropout d{state, offset, {}, (uint32_t)std::nearbyint(p * 65536.0), 0.f};
    for (int i = 0; i < 10; i++) {
        d.keys[2 * i] = (uint32_t)seed + i * PHILOX_K0;
        d.keys[2 * i + 1] = (uint32_t)(seed >> 32) + i * PHILOX_K1;
    }
    d.scale = d.threshold < 65536 ? (float)(scale * (65536.0 / (65536.0 - d.threshold))) : 0.f;
    return d;
}

// What a kernel does: nothing is dropped (p below 2^-17), or by a key of the launch's or
// of the device's.
enum : int { DROP_NONE = 0, DROP_KEY = 1, DROP_STATE = 2 };
template <typename F>
int dispatch_drop(const Dropout& d, F&& f) {
    if (d.threshold == 0) return f.template operator()<DROP_NONE>();
    return d.state ? f.template operator()<DROP_STATE>() : f.template operator()<DROP_KEY>();
}

// The key and the offset of a launch, as each thread holds them (the key with `state` only).
struct DropKey {
    uint32_t k0, k1, o0, o1;
};

template <int MODE>
__device__ __forceinline__ DropKey drop_key(const Dropout& d) {
    uint64_t seed = 0, offset = d.offset;
    if constexpr (MODE == DROP_STATE) {
        seed = (uint64_t)d.state[0];
        offset += (uint64_t)d.state[1];
    }
    return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
}

// The four words of a block.  58 instructions: the rounds' keys in constant memory (20
// more where each thread adds them up), a product's halves as two instructions (2 fewer than
// one 64-bit product, whose register pairs are moved about).
template <int MODE>
__device__ __forceinline__ uint4 philox(const Dropout& d, const DropKey& key, uint32_t block_lo, uint32_t block_hi) {
    uint32_t c0 = block_lo, c1 = block_hi, c2 = key.o0, c3 = key.o1;
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint32_t h0 = __umulhi(0xD2511F53u, c0), l0 = 0xD2511F53u * c0;
        const uint32_t h1 = __umulhi(0xCD9E8D57u, c2), l1 = 0xCD9E8D57u * c2;
        c0 = h1 ^ c1 ^ (MODE == DROP_KEY ? d.keys[2 * i] : key.k0 + i * PHILOX_K0);
        c1 = l1;
        c2 = h0 ^ c3 ^ (MODE == DROP_KEY ? d.keys[2 * i + 1] : key.k1 + i * PHILOX_K1);
        c3 = l0;
    }
    return make_uint4(c0, c1, c2, c3);
}

// v[k] of the 2 N elements that N words stand for: scaled, or 0 where dropped (also
// an infinity or a NaN).  A half is below the threshold where it is at most `bound` =
// 65536 threshold - 1 in the upper bits of a word, whatever lies below it: no
// extraction, and a threshold of 65536 drops everything.  threshold >= 1.
template <int N>
__device__ __forceinline__ void drop(float* v, const uint32_t* words, uint32_t threshold, float scale) {
    const uint32_t bound = (threshold << 16) - 1;
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[2 * i] = words[i] << 16 <= bound ? 0.f : __fmul_rn(v[2 * i], scale);
        v[2 * i + 1] = words[i] <= bound ? 0.f : __fmul_rn(v[2 * i + 1], scale);
    }
}
// the 8 elements of a block from its words
__device__ __forceinline__ void drop_block(float* v, const uint4& r, const Dropout& d) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    drop<4>(v, w, d.threshold, d.scale);
}
// The N (4 or 8) elements of vector i of the tensor, what is kept of them scaled.
template <int MODE, int N>
__device__ __forceinline__ void drop_vector(float* v, const DropKey& key, uint64_t i, const Dropout& d) {
    if constexpr (MODE == DROP_NONE) {
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = __fmul_rn(v[k], d.scale);
    } else if constexpr (N == 8) {
        drop_block(v, philox<MODE>(d, key, (uint32_t)i, (uint32_t)(i >> 32)), d);
    } else {
        const uint4 r = philox<MODE>(d, key, (uint32_t)(i >> 1), (uint32_t)(i >> 33));
        const uint32_t w[2] = {i & 1 ? r.z : r.x, i & 1 ? r.w : r.y};
        drop<2>(v, w, d.threshold, d.scale);
    }
}

}  // namespace rwkv
