// Attention of drafted tokens over the paged cache: every sequence brings the nodes of a tree (or a chain), whose keys and values
// are already in the cache behind its context.  A node sees the context, and of the nodes those that its mask names.
//
// Bytes: K and V once per (sequence, kv head), whatever the number of nodes: rows = nodes x query heads of the group share them.
// At 8 rows that is 8 flops a byte, at 256 it is 256, where tensor throughput and HBM balance.  tcgen05 carries all of it: a tile
// of 128 rows costs the tensor core the same however few of them are nodes, and that is less time than its bytes take.
//
// One persistent CTA per SM.  A unit is (sequence, block of up to 2 * QT nodes, kv head), QT = 128 / G.  All units' key tiles (128
// keys) stand in one line, which is cut into equal shares, one per CTA; a unit that a cut runs through leaves partial
// results (maximum, sum, unnormalised output in fp32), which a second kernel joins in order.  Roles of the 16 warps:
//   warp 0        TMA producer: walks the CTA's share, publishes items, loads Q tiles and a ring of K and V tiles
//   warp 1        one thread issues tcgen05.mma: S_X = Q_X K^T, O_X += P_X V (P read from TMEM)
//   warps 4-7, 8-11   softmax warpgroups of the halves A and B: a thread owns a row; P goes back over S
//   warps 12-15   output warpgroup: finished accumulators out of TMEM, to `out` or to the partials
// The halves are the two chains S -> softmax -> P V that TMEM has room for.  Up to 128 rows, they take the key tiles of a unit in
// turn and the output warpgroup joins them; with more, each has a Q tile of its own and both use every key tile.
// TMEM: S_A [0,128)  S_B [128,256)  O_A [256,384)  O_B [384,512).  Every mbarrier wait is bounded.
#include <atomic>

#include "../../include/b200_attn.h"
#include "tc_wait.cuh"
#include "tcgen05.cuh"
#include "tree_common.cuh"

namespace b200 {
extern std::atomic<long long> g_launches;

constexpr int kTrKv = 128;
constexpr int kTrSub = 128 * 128;             // one 64-column sub-tile of a 128-row tile (bytes)
constexpr int kTrTile = 2 * kTrSub;           // 128 rows x 128 dims bf16 = 32 KiB
constexpr int kTrThreads = 512;
constexpr int kTrRing = 5;                    // K and V tiles, one ring in the order in which they are used
constexpr int kTrItems = 4;                   // items in flight
constexpr float kTrRescale = 8.0f;
// The line's measure: cost of a key tile with the halves sharing it out, with a Q tile each, and of a unit by itself.
constexpr int kTrCostSplit = 4, kTrCostPair = 5, kTrCostUnit = 3;
// Partial results of one piece: 8 groups of 32 rows, each [128 dims][32 rows] and [max, sum][32 rows] in fp32, so that both kernels
// move whole lines with a row per lane.
constexpr int kTrGroup = 130 * 32;
constexpr int kTrPartial = 8 * kTrGroup;      // floats

static __device__ int g_status_tree = 0;

struct TreeItem {
  int seq;              // -1: no more work
  int h;
  int q_row;            // global row of the unit's first node
  int node0, nodes;     // that node's index in its sequence, and how many the unit has
  int first, Lk;        // position of the sequence's node 0; its keys
  int t0, n;            // key tiles of this piece
  int split;            // the halves share the key tiles out
  int partial;          // -1: the whole unit, else where its partial results go
};

// What a cut unit's pieces are: a record for each place of partial results, written by every CTA.
struct TreePiece {
  int state;            // 0: none, 1: more of the unit follows, 2: its last
  int q_row, h, nodes;
};

// One sequence as the line sees it.
struct TreeSeq {
  int q_begin, nodes, Lk, tiles, blocks;     // blocks: of 2 * QT nodes
  bool last_split;                           // the last block has at most QT nodes
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int QT, int i) {
  TreeSeq s;
  s.q_begin = max(0, min(__ldg(p.cu_q + i), p.total_q));
  s.nodes = max(0, min(__ldg(p.cu_q + i + 1), p.total_q) - s.q_begin);
  s.Lk = max(0, min(__ldg(p.context_lens + i), p.bt_cols * p.block_size));
  s.tiles = (s.Lk + kTrKv - 1) / kTrKv;
  s.blocks = s.tiles > 0 ? (s.nodes + 2 * QT - 1) / (2 * QT) : 0;
  s.last_split = s.nodes - (s.blocks - 1) * 2 * QT <= QT;
  return s;
}
__device__ __forceinline__ long long tree_cost(const TreeSeq& s, int Hkv) {
  if (s.blocks == 0) return 0;
  return Hkv * (static_cast<long long>(s.blocks) * (s.tiles * kTrCostPair + kTrCostUnit) -
                (s.last_split ? static_cast<long long>(s.tiles) * (kTrCostPair - kTrCostSplit) : 0));
}
// Place `off` of a sequence's part of the line: unit (block * Hkv + head) and key tile.
__device__ __forceinline__ void tree_locate(const TreeSeq& s, int Hkv, long long off, int& unit, int& tile) {
  const long long pair = static_cast<long long>(s.tiles) * kTrCostPair + kTrCostUnit;
  const long long block = min(off / (pair * Hkv), static_cast<long long>(s.blocks - 1));
  off -= block * pair * Hkv;
  const int w = block == s.blocks - 1 && s.last_split ? kTrCostSplit : kTrCostPair;
  const long long one = static_cast<long long>(s.tiles) * w + kTrCostUnit;
  const long long h = off / one;
  off -= h * one;
  unit = static_cast<int>(block * Hkv + h);
  tile = static_cast<int>(max(off - kTrCostUnit, 0LL) / w);
}

__global__ void __launch_bounds__(kTrThreads, 1)
tree_attn_kernel(const TreeParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k16,
                 const __grid_constant__ CUtensorMap map_v16) {
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* const sQ = smem;                      // [2][32 KiB]
  unsigned char* const sKV = smem + 2 * kTrTile;       // [kTrRing][32 KiB]
  __shared__ __align__(8) uint64_t bar_item_full[kTrItems], bar_item_empty[kTrItems];
  __shared__ __align__(8) uint64_t bar_q_full[2], bar_q_empty[2], bar_kv_full[kTrRing], bar_kv_empty[kTrRing];
  __shared__ __align__(8) uint64_t bar_s_full[2], bar_p_full[2], bar_o_final[2], bar_o_free[2], bar_l_full[2], bar_l_empty[2];
  __shared__ float s_max[2][128], s_sum[2][128];       // a half's rows: maximum (log2 units) and sum
  __shared__ __align__(16) TreeItem s_item[kTrItems];
  __shared__ long long s_scan[kTrThreads / 32];
  __shared__ int s_at[2][3];                           // the share's first place and the one behind its last: sequence, unit, tile
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort, s_bare;                      // s_bare: some sequence has nodes but no keys

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.G, QT = 128 / p.G;
  if (tid == 0) {
    s_abort = 0;
    s_bare = 0;
    for (int i = 0; i < kTrItems; ++i) { mbar_init(&bar_item_full[i], 1); mbar_init(&bar_item_empty[i], 13); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_q_full[i], 1);
      mbar_init(&bar_q_empty[i], 1);
      mbar_init(&bar_s_full[i], 1);
      mbar_init(&bar_p_full[i], 4);
      mbar_init(&bar_o_final[i], 1);
      mbar_init(&bar_o_free[i], 4);
      mbar_init(&bar_l_full[i], 4);
      mbar_init(&bar_l_empty[i], 4);
    }
    for (int i = 0; i < kTrRing; ++i) { mbar_init(&bar_kv_full[i], 1); mbar_init(&bar_kv_empty[i], 1); }
    mbar_fence_init();
    s_at[0][0] = s_at[1][0] = p.batch;
    s_at[0][1] = s_at[0][2] = s_at[1][1] = s_at[1][2] = 0;
  }
  __syncthreads();
  // The CTA's share of the line.  (Lengths ahead of the wait below: no kernel that lets this one start early writes them.)
  // With up to a block of sequences one sum over them gives the total and every sequence's place; larger batches take two.
  {
    long long total = 0, mine = 0, before = 0;
    TreeSeq s = {};
    const int rounds = (p.batch + kTrThreads - 1) / kTrThreads;
    for (int pass = rounds > 1 ? 0 : 1; pass < 2; ++pass) {
      long long upto = 0, lo = 0, hi = 0;
      for (int r = 0; r < rounds; ++r) {
        const int i = r * kTrThreads + tid;
        mine = 0;
        if (i < p.batch) {
          s = tree_seq(p, QT, i);
          mine = tree_cost(s, p.Hkv);
          if (s.nodes > 0 && s.tiles == 0) s_bare = 1;
        }
        long long x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (lane == 31) s_scan[warp] = x;
        __syncthreads();
        long long all = 0;
        before = upto;
#pragma unroll
        for (int w = 0; w < kTrThreads / 32; ++w) {
          const long long v = s_scan[w];
          if (w < warp) before += v;
          all += v;
        }
        __syncthreads();
        before += x - mine;
        upto += all;
        if (rounds == 1) total = upto;
        if (pass == 1 && i < p.batch && mine > 0) {
          lo = total * blockIdx.x / gridDim.x;
          hi = total * (blockIdx.x + 1) / gridDim.x;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const long long at = e ? hi : lo;
            if (at >= before && at < before + mine) {
              int unit, tile;
              tree_locate(s, p.Hkv, at - before, unit, tile);
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
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (s_bare) {
    // sequences with nodes and no keys: zeros
    for (int i = blockIdx.x; i < p.batch; i += gridDim.x) {
      const TreeSeq s = tree_seq(p, QT, i);
      if (s.tiles > 0) continue;
      uint4* const dst = reinterpret_cast<uint4*>(p.out + static_cast<long long>(s.q_begin) * p.H * 128);
      for (long long e = tid; e < static_cast<long long>(s.nodes) * p.H * 16; e += kTrThreads) dst[e] = make_uint4(0, 0, 0, 0);
    }
  }
  if (warp == 1) {
    tc::tmem_alloc(&s_tmem_base, 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem_base;
  volatile int* abort_flag = &s_abort;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;" ::: "memory");
    if (warp == 0 && lane == 0) {
      // ================================ TMA producer ================================
      tma_prefetch_desc(&map_q);
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
      TreePiece pieces[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      int seq = s_at[0][0], unit = s_at[0][1], t0 = s_at[0][2];
      const int end_seq = s_at[1][0], end_unit = s_at[1][1], end_tile = s_at[1][2];
      int n_pub = 0, kv = 0, kv_ph = 1, q_use = 0;
      bool ok = true;
      TreeSeq s = {};
      int have = -1;
      while (ok && seq < p.batch && seq <= end_seq) {
        if (have != seq) {
          s = tree_seq(p, QT, seq);
          have = seq;
        }
        if (unit >= s.blocks * p.Hkv) {
          ++seq;
          unit = t0 = 0;
          continue;
        }
        const bool at_end = seq == end_seq && unit >= end_unit;
        const int t1 = at_end ? (unit == end_unit ? end_tile : 0) : s.tiles;
        if (t1 > t0) {
          const int block = unit / p.Hkv, h = unit - block * p.Hkv, node0 = block * 2 * QT;
          const int nodes = min(2 * QT, s.nodes - node0), n = t1 - t0;
          const bool split = nodes <= QT;
          const bool whole = t0 == 0 && t1 == s.tiles;
          const int place = t0 > 0 ? 0 : 1;
          if (!whole) pieces[place] = {t1 < s.tiles ? 1 : 2, s.q_begin + node0, h, nodes};
          const int is = n_pub % kTrItems;
          if (!t2_wait_timed(&bar_item_empty[is], ((n_pub / kTrItems) & 1) ^ 1, abort_flag)) { ok = false; break; }
          s_item[is] = {seq, h, s.q_begin + node0, node0, nodes, s.Lk - s.nodes, s.Lk, t0, n, split, whole ? -1 : 2 * static_cast<int>(blockIdx.x) + place};
          mbar_arrive(&bar_item_full[is]);
          ++n_pub;
          // Q tiles: one, or two in turn
          for (int x = 0; x < (split ? 1 : 2) && ok; ++x, ++q_use) {
            const int b = q_use & 1;
            if (!t2_wait_timed(&bar_q_empty[b], ((q_use >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
            mbar_expect_tx(&bar_q_full[b], QT * G * 256);
            tma_load_3d(sQ + b * kTrTile, &map_q, &bar_q_full[b], 0, h * G, s.q_begin + node0 + x * QT);
            tma_load_3d(sQ + b * kTrTile + kTrSub, &map_q, &bar_q_full[b], 64, h * G, s.q_begin + node0 + x * QT);
          }
          if (!ok) break;
          // K and V tiles in the order of their use: K runs ahead of V by the tiles that are in the halves
          const int* const bt_row = p.block_tables + seq * p.bt_row_stride;
          auto row_of = [&](int t) -> int {
            const int key0 = (t0 + t) * kTrKv, col = key0 / p.block_size;
            const long long blk = __ldg(bt_row + col);
            return blk >= 0 && blk < p.num_blocks ? static_cast<int>(blk * p.block_size + (key0 - col * p.block_size)) : -(1 << 30);      // (nowhere: zeros)
          };
          auto load = [&](const CUtensorMap* map, const CUtensorMap* map16, int t) -> bool {
            if (!t2_wait_timed(&bar_kv_empty[kv], kv_ph, abort_flag)) return false;
            unsigned char* const dst = sKV + kv * kTrTile;
            const int row0 = row_of(t), left = s.Lk - (t0 + t) * kTrKv;
            if (left > kTrKv - 16) {
              mbar_expect_tx(&bar_kv_full[kv], kTrTile);
              tma_load_3d(dst, map, &bar_kv_full[kv], 0, h, row0);
              tma_load_3d(dst + kTrSub, map, &bar_kv_full[kv], 64, h, row0);
            } else {
              // the sequence's last tile: only what it has of it
              const int boxes = (left + 15) >> 4;
              mbar_expect_tx(&bar_kv_full[kv], boxes * 4096);
              for (int b = 0; b < boxes; ++b) {
                tma_load_3d(dst + b * 2048, map16, &bar_kv_full[kv], 0, h, row0 + b * 16);
                tma_load_3d(dst + kTrSub + b * 2048, map16, &bar_kv_full[kv], 64, h, row0 + b * 16);
              }
            }
            if (++kv == kTrRing) { kv = 0; kv_ph ^= 1; }
            return true;
          };
          const int ahead = split ? 2 : 1;
          for (int j = 0; j < ahead && j < n && ok; ++j) ok = load(&map_k, &map_k16, j);
          for (int j = 0; j < n && ok; ++j) {
            ok = load(&map_v, &map_v16, j);
            if (ok && j + ahead < n) ok = load(&map_k, &map_k16, j + ahead);
          }
        }
        if (at_end) break;
        ++unit;
        t0 = 0;
      }
      reinterpret_cast<int4*>(p.pieces)[2 * blockIdx.x] = make_int4(pieces[0].state, pieces[0].q_row, pieces[0].h, pieces[0].nodes);
      reinterpret_cast<int4*>(p.pieces)[2 * blockIdx.x + 1] = make_int4(pieces[1].state, pieces[1].q_row, pieces[1].h, pieces[1].nodes);
      if (ok) {
        const int is = n_pub % kTrItems;
        if (t2_wait_timed(&bar_item_empty[is], ((n_pub / kTrItems) & 1) ^ 1, abort_flag)) {
          s_item[is].seq = -1;
          mbar_arrive(&bar_item_full[is]);
          t2_wait_timed(&bar_item_empty[is], (n_pub / kTrItems) & 1, abort_flag);      // every role has taken it
        }
      }
    } else if (warp == 1 && lane == 0) {
      // ================================ MMA issuer ================================
      constexpr uint32_t idesc_qk = tc::idesc_bf16_f32(128, 128, false, false);
      constexpr uint32_t idesc_pv = tc::idesc_bf16_f32(128, 128, false, true);
      constexpr uint32_t desc_hi = tc::smem_desc_sw128_hi(1024);
      const uint32_t q_lo = tc::smem_desc_sw128_lo(smem_u32(sQ), 16), k_lo = tc::smem_desc_sw128_lo(smem_u32(sKV), 16);
      const uint32_t v_lo = tc::smem_desc_sw128_lo(smem_u32(sKV), kTrSub);
      int n_item = 0, kv = 0, kv_ph = 0, q_use = 0;
      int np[2] = {0, 0}, no[2] = {0, 0};       // P tiles taken and accumulators finished per half
      bool ok = true;
      auto next_kv = [&]() { if (++kv == kTrRing) { kv = 0; kv_ph ^= 1; } };
      auto issue_s = [&](int hx, int q, int slot) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t off = ((ks >> 2) * kTrSub + (ks & 3) * 32) >> 4;
          tc::mma_ss_lo(tmem + hx * 128, q_lo + q * (kTrTile >> 4) + off, k_lo + slot * (kTrTile >> 4) + off, desc_hi, idesc_qk, ks > 0);
        }
        tc::commit(&bar_s_full[hx]);
      };
      auto issue_pv = [&](int hx, int slot, bool accumulate) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          tc::mma_ts_lo(tmem + 256 + hx * 128, tmem + hx * 128 + ks * 8, v_lo + slot * (kTrTile >> 4) + ks * (2048 >> 4), desc_hi, idesc_pv,
                        accumulate || ks > 0);
      };
      while (ok) {
        const int is = n_item % kTrItems;
        if (!t2_wait(&bar_item_full[is], (n_item / kTrItems) & 1, abort_flag)) break;
        const int seq = s_item[is].seq, n = s_item[is].n;
        const bool split = s_item[is].split;
        mbar_arrive(&bar_item_empty[is]);
        if (seq < 0) break;
        ++n_item;
        const int qa = q_use & 1, qb = split ? qa : qa ^ 1;
        if (!t2_wait(&bar_q_full[qa], (q_use >> 1) & 1, abort_flag)) break;
        ++q_use;
        if (!split) {
          if (!t2_wait(&bar_q_full[qb], (q_use >> 1) & 1, abort_flag)) break;
          ++q_use;
        }
        // the first S of either half
        if (!t2_wait_hot(&bar_kv_full[kv], kv_ph, abort_flag)) break;
        tc::fence_after_sync();
        issue_s(0, qa, kv);
        if (split) {
          tc::commit(&bar_kv_empty[kv]);
          next_kv();
          if (n > 1) {
            if (!t2_wait_hot(&bar_kv_full[kv], kv_ph, abort_flag)) break;
            tc::fence_after_sync();
            issue_s(1, qa, kv);
            tc::commit(&bar_kv_empty[kv]);
            next_kv();
          }
          if (n <= 2) tc::commit(&bar_q_empty[qa]);
        } else {
          issue_s(1, qb, kv);
          tc::commit(&bar_kv_empty[kv]);
          next_kv();
          if (n == 1) { tc::commit(&bar_q_empty[qa]); tc::commit(&bar_q_empty[qb]); }
        }
        // then P V of a tile, and the half's next S
        const int ahead = split ? 2 : 1;
#pragma unroll 1
        for (int j = 0; j < n && ok; ++j) {
          const int v_slot = kv;
          if (!t2_wait_hot(&bar_kv_full[kv], kv_ph, abort_flag)) { ok = false; break; }
          next_kv();
          const bool more = j + ahead < n;
          const int k_slot = kv;
          if (more) {
            if (!t2_wait_hot(&bar_kv_full[kv], kv_ph, abort_flag)) { ok = false; break; }
            next_kv();
          }
          const int h0 = split ? j & 1 : 0, h1 = split ? h0 : 1;
#pragma unroll 1
          for (int hx = h0; hx <= h1; ++hx) {
            // (the output warpgroup has taken the previous accumulator)
            if (j < ahead && !t2_wait_hot(&bar_o_free[hx], (no[hx] & 1) ^ 1, abort_flag)) { ok = false; break; }
            if (!t2_wait_hot(&bar_p_full[hx], np[hx] & 1, abort_flag)) { ok = false; break; }
            ++np[hx];
            tc::fence_after_sync();
            issue_pv(hx, v_slot, j >= ahead);
            if (more) {
              issue_s(hx, hx && !split ? qb : qa, k_slot);
            } else {
              tc::commit(&bar_o_final[hx]);
              ++no[hx];
            }
          }
          if (!ok) break;
          tc::commit(&bar_kv_empty[v_slot]);
          if (more) {
            tc::commit(&bar_kv_empty[k_slot]);
            if (j + ahead + 1 == n) {       // the unit's last S
              tc::commit(&bar_q_empty[qa]);
              if (!split) tc::commit(&bar_q_empty[qb]);
            }
          }
        }
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;" ::: "memory");
    // ================================ softmax ================================
    const int hx = (warp - 4) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;                  // row of the tile
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tmem_s = tmem + hx * 128 + lane_base, tmem_o = tmem + 256 + hx * 128 + lane_base;
    const float c = p.scale_log2;
    int n_item = 0, ns = 0, n_fin = 0;
    int kv = 0, kv_ph = 0;                              // the ring's place behind the unit
    bool ok = true;
    while (ok) {
      const int is = n_item % kTrItems;
      if (!t2_wait(&bar_item_full[is], (n_item / kTrItems) & 1, abort_flag)) break;
      const TreeItem it = s_item[is];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_item_empty[is]);
      if (it.seq < 0) break;
      ++n_item;
      const int nx = it.split ? (hx ? it.n >> 1 : (it.n + 1) >> 1) : it.n;
      const int tile_nodes = it.split || !hx ? min(it.nodes, QT) : it.nodes - QT;
      const bool active = quarter * 32 < tile_nodes * G;         // this warp has rows
      const int in_tile = r / G + (it.split || !hx ? 0 : QT);    // the row's node within the unit
      const bool row_ok = in_tile < it.nodes && r < QT * G;
      const uint32_t* const mask = p.masks && row_ok ? p.masks + static_cast<long long>(it.q_row + in_tile) * p.mask_words : nullptr;
      // (rows that are none see nothing: a chain's row of index -1 - nodes)
      const int node = row_ok ? it.node0 + in_tile : -0x40000000;
      const bool chain = p.masks == nullptr;
      // place of the unit's last V tile in the ring, for its ragged tile
      int last_kv = kv + 2 * it.n - 1;
      int last_ph = kv_ph;
      { const int turns = last_kv / kTrRing; last_kv -= turns * kTrRing; last_ph ^= turns & 1; }
      { const int behind = kv + 2 * it.n, turns = behind / kTrRing; kv = behind - turns * kTrRing; kv_ph ^= turns & 1; }
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < nx; ++j) {
        if (!t2_wait_hot(&bar_s_full[hx], ns & 1, abort_flag)) { ok = false; break; }
        ++ns;
        const int key0 = (it.t0 + (it.split ? 2 * j + hx : j)) * kTrKv;
        if (active) {
          tc::fence_after_sync();
          uint32_t sv[4][32];
#pragma unroll
          for (int cch = 0; cch < 4; ++cch) tc::ld_32x32b_x32(tmem_s + cch * 32, sv[cch]);
          tc::wait_ld();
          if (key0 + kTrKv > min(it.first, it.Lk)) {
#pragma unroll
            for (int cch = 0; cch < 4; ++cch) {
              const int d = key0 + cch * 32 - it.first, left = it.Lk - key0 - cch * 32;
              const uint32_t keep = chain || row_ok ? tree_keep32(chain ? nullptr : mask, p.mask_words, node, d, left) : 0u;
              if (keep != 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!((keep >> i) & 1)) sv[cch][i] = 0xff800000u;   // -inf
              }
            }
          }
          // eight independent chains of 3-input max
          float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
          float mx4 = -INFINITY, mx5 = -INFINITY, mx6 = -INFINITY, mx7 = -INFINITY;
#pragma unroll
          for (int cch = 0; cch < 4; ++cch) {
#pragma unroll
            for (int i = 0; i < 32; i += 16) {
              mx0 = fmax3(mx0, __uint_as_float(sv[cch][i]), __uint_as_float(sv[cch][i + 1]));
              mx1 = fmax3(mx1, __uint_as_float(sv[cch][i + 2]), __uint_as_float(sv[cch][i + 3]));
              mx2 = fmax3(mx2, __uint_as_float(sv[cch][i + 4]), __uint_as_float(sv[cch][i + 5]));
              mx3 = fmax3(mx3, __uint_as_float(sv[cch][i + 6]), __uint_as_float(sv[cch][i + 7]));
              mx4 = fmax3(mx4, __uint_as_float(sv[cch][i + 8]), __uint_as_float(sv[cch][i + 9]));
              mx5 = fmax3(mx5, __uint_as_float(sv[cch][i + 10]), __uint_as_float(sv[cch][i + 11]));
              mx6 = fmax3(mx6, __uint_as_float(sv[cch][i + 12]), __uint_as_float(sv[cch][i + 13]));
              mx7 = fmax3(mx7, __uint_as_float(sv[cch][i + 14]), __uint_as_float(sv[cch][i + 15]));
            }
          }
          const float mx = fmax3(fmax3(mx0, mx1, mx2), fmax3(mx3, mx4, mx5), fmaxf(mx6, mx7));
          const float m_new = fmaxf(m_used, mx);
          if (j == 0) {
            m_used = m_new;
          } else {
            const bool grow = (m_new - m_used) * c > kTrRescale;
            if (__any_sync(0xffffffffu, grow)) {
              const float alpha = grow ? fast_exp2((m_used - m_new) * c) : 1.f;
              if (grow) { m_used = m_new; l *= alpha; }
#pragma unroll 1
              for (int cch = 0; cch < 8; ++cch) {
                uint32_t v[16];
                tc::ld_32x32b_x16(tmem_o + cch * 16, v);
                tc::wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                tc::st_32x32b_x16(tmem_o + cch * 16, v);
              }
            }
          }
          // P = exp2(c * (s - m)), masked entries -inf -> 0; rounded to bf16 as the product takes it, the sum is of the unrounded ones
          const float mc = (m_used == -INFINITY ? 0.f : m_used) * c;
          const unsigned long long c2 = f32x2_pack(c, c), nmc2 = f32x2_pack(-mc, -mc);
          unsigned long long ls0 = 0ull, ls1 = 0ull, ls2 = 0ull, ls3 = 0ull;
#pragma unroll
          for (int cch = 0; cch < 4; ++cch) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              float p0, p1, p2, p3, p4, p5, p6, p7;
              f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(sv[cch][2 * i]), __uint_as_float(sv[cch][2 * i + 1])), c2, nmc2), p0, p1);
              f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(sv[cch][2 * i + 2]), __uint_as_float(sv[cch][2 * i + 3])), c2, nmc2), p2, p3);
              f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(sv[cch][2 * i + 4]), __uint_as_float(sv[cch][2 * i + 5])), c2, nmc2), p4, p5);
              f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(sv[cch][2 * i + 6]), __uint_as_float(sv[cch][2 * i + 7])), c2, nmc2), p6, p7);
              p0 = fast_exp2(p0); p1 = fast_exp2(p1); p2 = fast_exp2(p2); p3 = fast_exp2(p3);
              p4 = fast_exp2(p4); p5 = fast_exp2(p5); p6 = fast_exp2(p6); p7 = fast_exp2(p7);
              ls0 = f32x2_add(ls0, f32x2_pack(p0, p1));
              ls1 = f32x2_add(ls1, f32x2_pack(p2, p3));
              ls2 = f32x2_add(ls2, f32x2_pack(p4, p5));
              ls3 = f32x2_add(ls3, f32x2_pack(p6, p7));
              pk[i] = pack_bf16(p0, p1);
              pk[i + 1] = pack_bf16(p2, p3);
              pk[i + 2] = pack_bf16(p4, p5);
              pk[i + 3] = pack_bf16(p6, p7);
            }
            tc::st_32x32b_x16(tmem_s + cch * 16, pk);
          }
          float a0, a1;
          f32x2_unpack(f32x2_add(f32x2_add(ls0, ls1), f32x2_add(ls2, ls3)), a0, a1);
          l += a0 + a1;
          tc::wait_st();
        }
        if (key0 + kTrKv > it.Lk) {
          // The sequence's last tile: V rows behind its end are stale or foreign; zero them, so that 0 * garbage cannot turn into
          // NaN in the tensor core.  (It is the unit's last V tile.)
          if (!t2_wait_hot(&bar_kv_full[last_kv], last_ph, abort_flag)) { ok = false; break; }
          unsigned char* const rows = sKV + last_kv * kTrTile;
#pragma unroll 1
          for (int i = (it.Lk - key0) * 128 + r * 16; i < kTrSub; i += 128 * 16) {
            *reinterpret_cast<uint4*>(rows + i) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(rows + kTrSub + i) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_p_full[hx]);   // one arrival per warp
      }
      if (!ok) break;
      if (nx > 0) {
        if (!t2_wait(&bar_l_empty[hx], (n_fin & 1) ^ 1, abort_flag)) { ok = false; break; }
        s_max[hx][r] = m_used == -INFINITY ? -INFINITY : m_used * c;
        s_sum[hx][r] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_l_full[hx]);
        ++n_fin;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;" ::: "memory");
    // ================================ output warpgroup ================================
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    int n_item = 0;
    int nf[2] = {0, 0};                                  // accumulators drained so far
    bool ok = true;
    while (ok) {
      const int is = n_item % kTrItems;
      if (!t2_wait(&bar_item_full[is], (n_item / kTrItems) & 1, abort_flag)) break;
      const TreeItem it = s_item[is];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_item_empty[is]);
      if (it.seq < 0) break;
      ++n_item;
      // one turn for the joined halves, or one for each
#pragma unroll 1
      for (int turn = 0; turn < (it.split ? 1 : 2) && ok; ++turn) {
        const bool joined = it.split && it.n > 1;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (e == 1 && !joined) continue;
          const int hx = turn + e;
          if (!t2_wait(&bar_l_full[hx], nf[hx] & 1, abort_flag)) { ok = false; break; }
          m[e] = s_max[hx][r];
          l[e] = s_sum[hx][r];
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_l_empty[hx]);
          if (!t2_wait(&bar_o_final[hx], nf[hx] & 1, abort_flag)) { ok = false; break; }
          ++nf[hx];
        }
        if (!ok) break;
        tc::fence_after_sync();
        const int tile_nodes = turn == 0 ? min(it.nodes, QT) : it.nodes - QT;
        if (quarter * 32 < tile_nodes * G) {
          const float M = fmaxf(m[0], m[1]);
          float wa = M == -INFINITY ? 0.f : fast_exp2(m[0] - M), wb = M == -INFINITY ? 0.f : fast_exp2(m[1] - M);
          const float sum = l[0] * wa + l[1] * wb;
          const bool row_ok = r < tile_nodes * G;
          const int t = r / G;
          __nv_bfloat16* const dst = p.out + (static_cast<long long>(it.q_row + turn * QT + t) * p.H + it.h * G + (r - t * G)) * 128;
          float* const part = it.partial < 0 ? nullptr : p.partials + static_cast<long long>(it.partial) * kTrPartial + (turn * 4 + quarter) * kTrGroup + lane;
          if (part) {
            part[128 * 32] = M;
            part[129 * 32] = sum;
          } else {
            const float inv = sum > 0.f ? 1.f / sum : 0.f;      // (a row that sees nothing: zeros)
            wa *= inv;
            wb *= inv;
          }
          const uint32_t ta = tmem + 256 + turn * 128 + lane_base;
#pragma unroll 1
          for (int cch = 0; cch < 8; ++cch) {
            uint32_t a[16];
            tc::ld_32x32b_x16(ta + cch * 16, a);
            if (joined) {
              uint32_t b[16];
              tc::ld_32x32b_x16(ta + 128 + cch * 16, b);
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) a[i] = __float_as_uint(fmaf(__uint_as_float(b[i]), wb, __uint_as_float(a[i]) * wa));
            } else {
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) a[i] = __float_as_uint(__uint_as_float(a[i]) * wa);
            }
            if (part) {
#pragma unroll
              for (int i = 0; i < 16; ++i) part[(cch * 16 + i) * 32] = __uint_as_float(a[i]);
            } else if (row_ok) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint4 w;
                w.x = pack_bf16(__uint_as_float(a[8 * i]), __uint_as_float(a[8 * i + 1]));
                w.y = pack_bf16(__uint_as_float(a[8 * i + 2]), __uint_as_float(a[8 * i + 3]));
                w.z = pack_bf16(__uint_as_float(a[8 * i + 4]), __uint_as_float(a[8 * i + 5]));
                w.w = pack_bf16(__uint_as_float(a[8 * i + 6]), __uint_as_float(a[8 * i + 7]));
                reinterpret_cast<uint4*>(dst)[cch * 2 + i] = w;
              }
            }
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar_o_free[turn]);
          if (joined) mbar_arrive(&bar_o_free[1]);
        }
      }
    }
  }

  // ---- teardown: everyone meets, then the allocating warp frees TMEM ----
  tc::fence_before_sync();
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
  if (tid == 0 && s_abort) atomicExch(&g_status_tree, 1);
}

// Units that a cut ran through: a CTA per (cut, group of 32 rows), the cut that is a unit's first joins all of its pieces, in their
// order.  A warp takes 8 of the 128 dims, a lane a row.
constexpr int kTrJoinThreads = 512;
__global__ void __launch_bounds__(kTrJoinThreads)
tree_join_kernel(const TreeParams p, int ctas) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cut = blockIdx.x + 1, group = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4* const pieces = reinterpret_cast<const int4*>(p.pieces);
  const int4 head = __ldcg(pieces + 2 * (cut - 1) + 1);
  if (head.x != 1) return;
  const int G = p.G, QT = 128 / G, half = group >> 2, r = (group & 3) * 32 + lane;
  const int nodes = min(head.w - half * QT, QT);      // of this half
  if ((group & 3) * 32 >= nodes * G) return;
  const float* const mine = p.partials + static_cast<long long>(group) * kTrGroup + lane;
  auto part = [&](int place) { return mine + static_cast<long long>(place) * kTrPartial; };
  // the pieces: the first one's place, then the next CTAs' first places until the last
  float M = ld_cg_f32(part(2 * (cut - 1) + 1) + 128 * 32);
  int last = cut;
  for (;; ++last) {
    const int state = __ldcg(pieces + 2 * last).x;
    if (state) M = fmaxf(M, ld_cg_f32(part(2 * last) + 128 * 32));
    if (state == 2 || last + 1 >= ctas) break;
  }
  float sum = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int c = cut - 1; c <= last; ++c) {
    if (c >= cut && !__ldcg(pieces + 2 * c).x) continue;
    const float* const from = part(c < cut ? 2 * c + 1 : 2 * c);
    const float w = M == -INFINITY ? 0.f : fast_exp2(ld_cg_f32(from + 128 * 32) - M);
    sum = fmaf(ld_cg_f32(from + 129 * 32), w, sum);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fmaf(ld_cg_f32(from + (warp * 8 + i) * 32), w, o[i]);
  }
  if (r >= nodes * G) return;
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  const int t = r / G;
  uint4 v;
  v.x = pack_bf16(o[0] * inv, o[1] * inv);
  v.y = pack_bf16(o[2] * inv, o[3] * inv);
  v.z = pack_bf16(o[4] * inv, o[5] * inv);
  v.w = pack_bf16(o[6] * inv, o[7] * inv);
  reinterpret_cast<uint4*>(p.out + (static_cast<long long>(head.y + half * QT + t) * p.H + head.z * G + (r - t * G)) * 128)[warp] = v;
}

// Workspace: the pieces' records, then two places of partial results per CTA.
static int64_t tree_pieces_bytes(int ctas) { return (static_cast<int64_t>(ctas) * 2 * sizeof(TreePiece) + 255) / 256 * 256; }
static int64_t tree_workspace(int ctas) { return tree_pieces_bytes(ctas) + static_cast<int64_t>(ctas) * 2 * kTrPartial * 4; }

int read_status_tree() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_status_tree, sizeof(int));
  return v;
}
int reset_state_tree() {
  const int zero = 0;
  return check_cuda(cudaMemcpyToSymbol(g_status_tree, &zero, sizeof(int)), "device_status: clearing the tree attention status word");
}

}  // namespace b200

extern "C" int64_t b200_tree_workspace_bytes(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  using namespace b200;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim != 128 || num_heads / num_kv_heads > 128)
    return set_error(kErrBadShape, "tree_workspace_bytes: bad geometry (H=%d Hkv=%d D=%d)", num_heads, num_kv_heads, head_dim);
  const int grid = sm_count();
  if (grid <= 0) return set_error(kErrNoDriver, "tree_workspace_bytes: no CUDA device");
  return tree_workspace(grid);
}

extern "C" int b200_tree_attn(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache, int64_t num_blocks,
                              int32_t block_size, const int32_t* block_tables, int64_t bt_row_stride, int32_t bt_cols,
                              const int32_t* cu_seqlens_q, const int32_t* context_lens, const uint64_t* tree_masks,
                              int32_t mask_words, void* out, void* workspace, int64_t workspace_bytes, int32_t batch, int32_t total_q,
                              int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float scale, void* stream) {
  using namespace b200;
  if (batch < 0 || total_q < 0) return set_error(kErrBadShape, "tree_attn: negative batch or total_q");
  if (head_dim != 128) return set_error(kErrBadShape, "tree_attn: head_dim must be 128 (got %d)", head_dim);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads)
    return set_error(kErrBadShape, "tree_attn: num_heads (%d) must be a positive multiple of num_kv_heads (%d)", num_heads, num_kv_heads);
  const int G = num_heads / num_kv_heads;
  if (G > 128) return set_error(kErrBadShape, "tree_attn: at most 128 query heads per kv head");
  if (tree_masks && (mask_words < 1 || mask_words > kTreeMaxWords))
    return set_error(kErrBadShape, "tree_attn: mask_words must be in [1, %d] (got %d)", kTreeMaxWords, mask_words);
  if (block_size <= 0 || block_size % 256) return set_error(kErrBadShape, "tree_attn: block_size must be a positive multiple of 256 (got %d)", block_size);
  if (num_blocks <= 0 || num_blocks * block_size >= (1LL << 31)) return set_error(kErrBadShape, "tree_attn: num_blocks * block_size must be in (0, 2^31)");
  if (bt_cols <= 0 || bt_row_stride < bt_cols || static_cast<long long>(bt_cols) * block_size >= (1LL << 30))
    return set_error(kErrBadShape, "tree_attn: bad block table geometry (cols=%d stride=%lld)", bt_cols, (long long)bt_row_stride);
  if (batch == 0 || total_q == 0) return kOk;
  if (!q || !k_cache || !v_cache || !block_tables || !cu_seqlens_q || !context_lens || !out)
    return set_error(kErrNullPointer, "tree_attn: null pointer argument");
  if (q_row_stride < static_cast<long long>(num_heads) * 128 || q_row_stride % 8)
    return set_error(kErrMisaligned, "tree_attn: q_row_stride must be >= H*128 and a multiple of 8 elements");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15)
    return set_error(kErrMisaligned, "tree_attn: q, out and the caches must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(tree_masks) & 7) return set_error(kErrMisaligned, "tree_attn: tree_masks must be 8-byte aligned");
  if (!workspace || workspace_bytes < b200_tree_workspace_bytes(num_heads, num_kv_heads, head_dim) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return set_error(kErrWorkspace, "tree_attn: workspace missing, too small or not 16-byte aligned");
  TreeParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_row_stride = q_row_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu_q = cu_seqlens_q;
  p.context_lens = context_lens;
  p.block_tables = block_tables;
  p.bt_row_stride = bt_row_stride;
  p.bt_cols = bt_cols;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.masks = reinterpret_cast<const uint32_t*>(tree_masks);
  p.mask_words = 2 * mask_words;
  p.batch = batch;
  p.total_q = total_q;
  p.H = num_heads;
  p.Hkv = num_kv_heads;
  p.G = G;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int grid = sm_count();
  p.pieces = static_cast<int*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + tree_pieces_bytes(grid));
  CUtensorMap map_q, map_k, map_v, map_k16, map_v16;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * block_size, row = static_cast<uint64_t>(num_kv_heads) * 128;
  int rc = make_tokens_heads_map(&map_q, q, static_cast<uint64_t>(total_q), num_heads, static_cast<uint64_t>(q_row_stride), 128 / G, G);
  if (!rc) rc = make_tokens_heads_map(&map_k, k_cache, rows, num_kv_heads, row, kTrKv);
  if (!rc) rc = make_tokens_heads_map(&map_v, v_cache, rows, num_kv_heads, row, kTrKv);
  if (!rc) rc = make_tokens_heads_map(&map_k16, k_cache, rows, num_kv_heads, row, 16);
  if (!rc) rc = make_tokens_heads_map(&map_v16, v_cache, rows, num_kv_heads, row, 16);
  if (rc) return rc;
  const size_t smem = static_cast<size_t>(2 + kTrRing) * kTrTile;
  static std::atomic<size_t> configured[kMaxDevices];
  rc = ensure_dynamic_smem(reinterpret_cast<const void*>(tree_attn_kernel), smem, configured, "tree_attn: cudaFuncSetAttribute");
  if (rc) return rc;
  cudaError_t le = launch_early(tree_attn_kernel, grid, kTrThreads, smem, static_cast<cudaStream_t>(stream), p, map_q, map_k, map_v, map_k16, map_v16);
  g_launches.fetch_add(1);
  rc = check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "tree_attn launch");
  if (rc || grid < 2) return rc;
  // rows of the largest unit there can be, in groups of 32; a unit of two tiles has its second tile's rows from group 4 on
  const long long most = total_q <= 128 / G ? (static_cast<long long>(total_q) * G + 31) / 32 : 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid - 1, static_cast<unsigned>(most));
  cfg.blockDim = dim3(kTrJoinThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  le = cudaLaunchKernelEx(&cfg, tree_join_kernel, p, grid);
  g_launches.fetch_add(1);
  return check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "tree_attn join launch");
}
