// What the kernels of tree attention share: their parameters and the bits of a row's mask.
#pragma once
#include "kernels.cuh"

namespace b200 {

constexpr int kTreeMaxWords = 4;     // 64-bit words of a node's mask: trees of up to 256 nodes

struct TreeParams {
  const __nv_bfloat16* q;
  long long q_row_stride;
  __nv_bfloat16* out;                // (total_q, H, 128) contiguous
  const int* cu_q;
  const int* context_lens;
  const int* block_tables;
  long long bt_row_stride;
  int bt_cols, block_size;
  long long num_blocks;
  const uint32_t* masks;             // (total_q, mask_words) 32-bit words; nullptr: each node sees those before it and itself
  int mask_words;                    // 32-bit words of a row
  int batch, total_q, H, Hkv, G;
  float scale_log2;
  struct TreePieces* pieces;         // records of cut units
  float* partials;                   // [2 * CTAs] partial results
};

// Which of 32 keys a row sees.  `d`: index of the first of them among the step's nodes (negative: that many lie in front of
// them), `left`: how many of the 32 the sequence has, `node`: the row's own index.  `mask`: the row's words, nullptr: in order.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }
__device__ __forceinline__ uint32_t tree_keep32(const uint32_t* mask, int words, int node, int d, int left) {
  uint32_t m = 0xffffffffu;
  if (d + 32 > 0) {
    if (!mask) {
      m = low_bits(node - d + 1);
    } else if (d < 0) {
      m = (words > 0 ? mask[0] : 0u) << -d | low_bits(-d);
    } else {
      const int w = d >> 5;
      m = __funnelshift_r(w < words ? mask[w] : 0u, w + 1 < words ? mask[w + 1] : 0u, d & 31);
    }
  }
  return m & low_bits(left);
}

}  // namespace b200
