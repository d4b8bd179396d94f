// philox.hpp — the counter-based generator of the dropout masks.
#pragma once

#include "common.hpp"

namespace tdgs {

struct PhiloxKey {
    uint32_t k0, k1;
    PhiloxKey() = default;
    explicit PhiloxKey(uint64_t seed) : k0((uint32_t)seed), k1((uint32_t)(seed >> 32)) {}
};

struct Philox4 {
    uint32_t w[4];
};

// Philox4x32-10 of the counter (lo, hi): ten rounds of two products of 32 bits, whose upper halves are mixed
// with the other words and the round's key, which grows by fixed steps.
__device__ __forceinline__ Philox4 philox(PhiloxKey key, uint64_t lo, uint64_t hi) {
    uint32_t c0 = (uint32_t)lo, c1 = (uint32_t)(lo >> 32), c2 = (uint32_t)hi, c3 = (uint32_t)(hi >> 32);
    uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// Elements are kept where their word is at least floor(p 2^32), and then multiplied by 1 / (1 - p).
struct DropRule {
    uint32_t least;
    bool none;      // p = 1: nothing is kept
    float scale;
    DropRule() = default;
    explicit DropRule(double p) : least(0), none(p >= 1.0), scale(0.0f) {
        if (!none) {
            least = (uint32_t)(uint64_t)(p * 4294967296.0);
            scale = (float)(1.0 / (1.0 - p));
        }
    }
    __device__ __forceinline__ bool keeps(uint32_t word) const { return word >= least && !none; }
};

}  // namespace tdgs
