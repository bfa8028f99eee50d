// Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011): the counter-based generator of the block operators' draws (include/nbx.h).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace nbx {

// One call's stream of draws: key = seed, counter = (q, call, step).
struct DrawKey {
    uint32_t k0, k1, call, step;
};

__device__ __forceinline__ DrawKey draw_key(const int64_t* rng, uint32_t call) {
    const uint64_t seed = (uint64_t)rng[0], step = (uint64_t)rng[1];
    return {(uint32_t)seed, (uint32_t)(seed >> 32), call, (uint32_t)step};
}

// The four words of block q; draws 8 q .. 8 q + 7 are their halfwords, low half first.
__device__ __forceinline__ uint4 draw_block(const DrawKey& key, uint64_t q) {
    uint32_t a = (uint32_t)q, b = (uint32_t)(q >> 32), c = key.call, d = key.step, k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t x = (uint64_t)a * 0xD2511F53u, y = (uint64_t)c * 0xCD9E8D57u;
        a = (uint32_t)(y >> 32) ^ b ^ k0;
        b = (uint32_t)y;
        c = (uint32_t)(x >> 32) ^ d ^ k1;
        d = (uint32_t)x;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(a, b, c, d);
}

// Bit j: whether draw 8 q + j keeps (its halfword is at least the threshold).
__device__ __forceinline__ uint32_t keep_bits(const DrawKey& key, uint64_t q, uint32_t threshold) {
    const uint4 w = draw_block(key, q);
    uint32_t m = 0;
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        m |= (uint32_t)((v[i] & 0xFFFFu) >= threshold) << (2 * i) | (uint32_t)((v[i] >> 16) >= threshold) << (2 * i + 1);
    return m;
}

// The same as eight truth values (lane masks in scalar registers: one select per use).
struct Keep8 {
    bool k[8];
};
__device__ __forceinline__ Keep8 keep_all(bool k) {
    Keep8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.k[i] = k;
    return r;
}
__device__ __forceinline__ Keep8 keep_eight(const DrawKey& key, uint64_t q, uint32_t threshold) {
    const uint4 w = draw_block(key, q);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    Keep8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.k[2 * i] = (v[i] & 0xFFFFu) >= threshold;
        r.k[2 * i + 1] = (v[i] >> 16) >= threshold;
    }
    return r;
}

__device__ __forceinline__ bool keep_one(const DrawKey& key, uint64_t draw, uint32_t threshold) {
    return keep_bits(key, draw >> 3, threshold) >> (draw & 7) & 1;
}

inline float keep_scale(uint32_t threshold) { return (float)(65536.0 / (65536.0 - (double)threshold)); }

}  // namespace nbx
