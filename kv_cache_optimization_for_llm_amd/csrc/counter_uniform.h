// The sampler's random numbers: one in [0, 1) for (seed, key, step), splitmix64's finaliser over the three and its top 24 bits.
#pragma once
#include <hip/hip_runtime.h>

__host__ __device__ inline float counter_uniform(unsigned int seed, unsigned int key, unsigned int step) {
    unsigned long long z = ((unsigned long long)key << 32) ^ (unsigned long long)step;
    z ^= (unsigned long long)seed * 0x9E3779B97F4A7C15ULL;
    z += 0x9E3779B97F4A7C15ULL;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
    z = z ^ (z >> 31);
    return (float)(z >> 40) * (1.0f / 16777216.0f);
}
