// What the sampling kernels share: the counter-based uniform numbers, the rule for the better of two scores, and the words that a
// step's kernels leave behind its tokens.
#pragma once

#include "common.cuh"

__device__ __forceinline__ uint32_t mix32(uint32_t v) {
    v ^= v >> 16;
    v *= 0x7FEB352Du;
    v ^= v >> 15;
    v *= 0x846CA68Bu;
    v ^= v >> 16;
    return v;
}

__device__ __forceinline__ float uniform_for(uint64_t seed, uint32_t step, uint32_t index) {
    uint32_t word = mix32((uint32_t)seed ^ 0x9E3779B9u);
    word = mix32(word ^ (uint32_t)(seed >> 32));
    word = mix32(word ^ step);
    word = mix32(word ^ index);
    return ((float)(word >> 9) + 0.5f) * (1.0f / 8388608.0f);  // exact in 32-bit, never 0 or 1
}

// Keeps the larger score; equal scores keep the lower index.
__device__ __forceinline__ void take_better(float& best, int& best_index, float score, int index) {
    if (score > best || (score == best && index < best_index)) {
        best = score;
        best_index = index;
    }
}

// The words that a step's kernels report errors in, behind the tokens: what a step reads back is then one piece of memory (the
// kernels in front are complete).
__device__ __forceinline__ void leave_flags(int* behind, const int* flag_a, const int* flag_b) {
    if (flag_a == nullptr || flag_b == nullptr) return;
    behind[0] = *flag_a;
    behind[1] = *flag_b;
}
