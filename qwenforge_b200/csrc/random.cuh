// The sampler's random numbers: a counter-based integer hash of (seed, sequence, step, token).
#pragma once
#include <stdint.h>

__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7FEB352Du;
    x ^= x >> 15;
    x *= 0x846CA68Bu;
    x ^= x >> 16;
    return x;
}

__device__ __forceinline__ uint32_t row_key(unsigned long long seed, long long seq_id, int step) {
    uint32_t key = mix32((uint32_t)seed ^ 0x9E3779B9u);
    key = mix32(key ^ (uint32_t)(seed >> 32));
    key = mix32(key ^ (uint32_t)seq_id);
    key = mix32(key ^ (uint32_t)((unsigned long long)seq_id >> 32) ^ 0x85EBCA6Bu);
    key = mix32(key ^ (uint32_t)step);
    return key;
}

// 23 random bits of token i under a row's key; the uniform number is (bits + 1/2) / 2^23.
__device__ __forceinline__ uint32_t token_bits(uint32_t key, uint32_t i) { return mix32(key ^ mix32(i ^ 0x27D4EB2Fu)) >> 9; }
