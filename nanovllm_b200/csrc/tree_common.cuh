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
  int above, upto;                   // sequences with more than `above` and at most `upto` nodes are this launch's
  float scale_log2;
  // The tcgen05 kernel takes the maximum of unscaled scores, which wants a positive scale: it is scale_abs (of 0 the least number
  // above, so that -inf stays -inf), and of a negative one `negate`, a bit of the instruction descriptor, turns Q.
  float scale_abs;
  uint32_t negate;
  int cluster_log;                   // where a cluster has a unit: log2 of its CTAs
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

// What a cut unit's pieces are, for the join.  A CTA's share can begin within a unit (its partial results go to place 2 * CTA) and end
// within one that it began (place 2 * CTA + 1).  Every CTA writes its entries.
constexpr int kTrMaxCtas = 160;               // (a B200 has 148 multiprocessors)
struct TreePieces {
  // x: nodes of the unit that the share ends within, 0: none; z, w: that unit's first row, its kv head.  y: the share begins within a
  // unit: 1, or 2 if it has the unit's last tile, too; 0: it does not
  int4 of[kTrMaxCtas];
};

// Partial results of one piece: 8 groups of 32 rows, each [128 dims][32 rows] and [max, sum][32 rows] in fp32, so that both kernels
// move whole lines with a row per lane.
constexpr int kTrGroup = 130 * 32;
constexpr int kTrPartial = 8 * kTrGroup;      // floats
constexpr int kSmPartial = kTrGroup;          // (tree_small.cu has at most 16 rows)

// One sequence as the line sees it.
struct TreeSeq {
  int q_begin, nodes, Lk, tiles, blocks;     // blocks: of a unit's most nodes
  bool last_split;                           // the last block has at most half of that
};
template <typename L>
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int block_nodes, int i) {
  TreeSeq s;
  s.q_begin = max(0, min(p.cu_q[i], p.total_q));
  s.nodes = max(0, min(p.cu_q[i + 1], p.total_q) - s.q_begin);
  if (s.nodes <= p.above || s.nodes > p.upto) s.nodes = 0;
  s.Lk = max(0, min(p.context_lens[i], p.bt_cols * p.block_size));
  s.tiles = (s.Lk + L::kKeys - 1) / L::kKeys;
  s.blocks = s.tiles > 0 ? (s.nodes + block_nodes - 1) / block_nodes : 0;
  s.last_split = s.nodes - (s.blocks - 1) * block_nodes <= block_nodes / 2;
  return s;
}
// (32 bits: the host refuses geometries whose line might be longer)
template <typename L>
__device__ __forceinline__ unsigned tree_cost(const TreeSeq& s, int Hkv) {
  if (s.blocks == 0) return 0;
  return Hkv * ((s.blocks - s.last_split) * (s.tiles * L::kTilePair + L::kUnitPair) + s.last_split * (s.tiles * L::kTileSplit + L::kUnitSplit));
}
// Place `off` of a sequence's part of the line: unit (block * Hkv + head) and key tile.
template <typename L>
__device__ __forceinline__ void tree_locate(const TreeSeq& s, int Hkv, unsigned off, int& unit, int& tile) {
  const unsigned pair = s.tiles * L::kTilePair + L::kUnitPair;
  const unsigned block = s.blocks == 1 ? 0 : min(off / (pair * Hkv), static_cast<unsigned>(s.blocks - 1));
  off -= block * pair * Hkv;
  const bool split = block == s.blocks - 1 && s.last_split;
  const unsigned w = split ? L::kTileSplit : L::kTilePair, start = split ? L::kUnitSplit : L::kUnitPair;
  const unsigned one = s.tiles * w + start;
  const unsigned h = off / one;
  off -= h * one;
  unit = static_cast<int>(block * Hkv + h);
  tile = static_cast<int>(off < start ? 0 : (off - start) / w);
}

// Walks along a sequence's key tiles: the cache row of each, far below zero (TMA reads zeros there) where its block is none of
// the cache.
template <typename L>
struct TreeRows {
  const int* blocks;
  int row, in_block;
  __device__ __forceinline__ void start(const TreeParams& p, int seq, int tile) {
    const int col = tile * L::kKeys / p.block_size;
    blocks = p.block_tables + seq * p.bt_row_stride + col;
    in_block = -(tile * L::kKeys - col * p.block_size);        // (not looked up yet)
  }
  __device__ __forceinline__ int next(const TreeParams& p) {
    if (in_block <= 0) {
      const int blk = *blocks++;
      row = blk >= 0 && blk < p.num_blocks ? blk * p.block_size - in_block : -(1 << 30);
      in_block += p.block_size;
    }
    const int r = row;
    row += L::kKeys;
    in_block -= L::kKeys;
    return r;
  }
};

// A CTA's share of the line of all units' key tiles, which is cut into equal ones: s_at[0] its first place (sequence, unit, tile),
// s_at[1] the one behind its last; both start out as {batch, 0, 0}.  `s_bare` is set where some sequence has nodes but no keys.
// Lengths are read ahead of the wait for the kernel in front: none that lets this one start early writes them.  With up to a
// block of sequences one sum over them gives the total and every sequence's place; larger batches take two.  All threads take part.
template <typename L, int kThreads>
__device__ __forceinline__ void tree_share(const TreeParams& p, int block_nodes, unsigned* s_scan /* [kThreads / 32] */, int (*s_at)[3], int* s_bare) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned total = 0;
  TreeSeq s = {};
  const int rounds = (p.batch + kThreads - 1) / kThreads;
#pragma unroll 1
  for (int pass = rounds > 1 ? 0 : 1; pass < 2; ++pass) {
    unsigned upto = 0;
#pragma unroll 1
    for (int r = 0; r < rounds; ++r) {
      const int i = r * kThreads + tid;
      unsigned mine = 0;
      if (i < p.batch) {
        s = tree_seq<L>(p, block_nodes, i);
        mine = tree_cost<L>(s, p.Hkv);
        if (s.nodes > 0 && s.tiles == 0) *s_bare = 1;
      }
      unsigned x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_scan[warp] = x;
      __syncthreads();
      unsigned w = lane < kThreads / 32 ? s_scan[lane] : 0;
#pragma unroll
      for (int o = 1; o < kThreads / 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
      }
      const unsigned all = __shfl_sync(0xffffffffu, w, kThreads / 32 - 1), front = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
      const unsigned before = upto + (warp ? front : 0) + x - mine;
      upto += all;
      if (rounds == 1) total = upto;
      else __syncthreads();
      if (pass == 1 && mine > 0) {
        // (any function of the CTA that grows from 0 to the total will do)
        const unsigned one = 0xffffffffu / gridDim.x;
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {
          const unsigned at = __umulhi(total, one * (blockIdx.x + e));
          if (at >= before && at < before + mine && blockIdx.x + e < gridDim.x) {
            int unit, tile;
            tree_locate<L>(s, p.Hkv, at - before, unit, tile);
            s_at[e][0] = i;
            s_at[e][1] = unit;
            s_at[e][2] = tile;
          }
        }
      }
    }
    total = upto;
  }
}

// Cost of a tile and of a unit in the line of tree_small.cu: a unit, with its rows, its last accumulators and its part in the join, weighs as much as 4.5
// tiles.  Us with 0 | 2.25 | 4.5 | 9, calls on end in a graph: 256 chains of 4 nodes on 100 .. 2048 tokens at 16/8 heads 221 | 198 | 190 | 190, 64 of 2 .. 10 on
// 500 .. 3000 at 4/2 40.1 | 36.4 | 34.4 | 33.8, 256 of 3 .. 9 on 100 .. 1000 at 8/4 94.5 | 81.0 | 81.1 | 81.7, 64 of 3 on 500 .. 3000 at 4/2 31.0 | 30.7 | 29.8 | 30.5.
struct SmLine {
  static constexpr int kKeys = 64;
  static constexpr int kTileSplit = 4, kUnitSplit = 18, kTilePair = 4, kUnitPair = 18;
};
// 1-D bulk copy global -> shared, completion counted on an mbarrier (addresses and size multiples of 16).
__device__ __forceinline__ void tree_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// Few nodes (tree_small.cu): up to 16 rows to a unit, G <= 16; K/V maps with boxes of 64 and of 16 tokens.
int launch_tree_small(const TreeParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, const CUtensorMap& map_k16,
                      const CUtensorMap& map_v16, int ctas, cudaStream_t stream);
// What a kernel of `ctas` CTAs leaves for the join (tree_attn.cu): records, partial results, floats from one of these to the next.
struct TreeCuts {
  const TreePieces* pieces;
  const float* partials;
  int stride;
};
struct TreeJoin {
  TreeCuts of[2];
  int kernels;
};
int launch_tree_join(const TreeParams& p, const TreeJoin& join, int ctas, cudaStream_t stream);

}  // namespace b200
