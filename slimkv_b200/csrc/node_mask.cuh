// Which keys a drafted node sees (ancestor words of slimkv_tree_masks).
#pragma once

#include "common.cuh"

namespace slimkv {

__device__ __forceinline__ uint32_t mask_word(const int32_t* row, int words, int w) {
    return w >= 0 && w < words ? uint32_t(__ldg(row + w)) : 0u;
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// Which of the 32 keys from node `first` on (below 0: context) node t sees:
// the context, and the nodes of its words (without words: up to itself).
__device__ __forceinline__ uint32_t seen_keys(const int32_t* row, int words, int t, int nodes, int first) {
    const uint32_t context = low_bits(-first);
    uint32_t bits;
    if (row) {
        const int w = first >> 5;               // floor
        bits = __funnelshift_r(mask_word(row, words, w), mask_word(row, words, w + 1), first & 31);
    } else {
        bits = low_bits(t + 1 - first);
    }
    return context | (bits & low_bits(nodes - first));
}

}  // namespace slimkv
