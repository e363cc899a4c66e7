// Attention of drafted tokens over the paged cache: every sequence brings the nodes of a tree (or a chain), whose keys and values
// are already in the cache behind its context.  A node sees the context, and of the nodes those that its mask names.
//
// Bytes: K and V once per (sequence, kv head), whatever the number of nodes: rows = nodes x query heads of the group share them.
// At 8 rows that is 8 flops a byte, at 256 it is 256, where tensor throughput and HBM balance.  A tile of 128 rows costs tcgen05 the
// same however few of them are nodes, and that is less time than its bytes take (but power: batches with few nodes to a sequence
// go to tree_small.cu, which leaves this kernel the large trees among them).
//
// One persistent CTA per SM.  A unit is (sequence, block of up to 2 * QT nodes, kv head), QT = 128 / G.  All units' key tiles (128
// keys) stand in one line, which is cut into equal shares, one per CTA; a unit that a cut runs through leaves partial
// results (maximum, sum, unnormalised output in fp32), which a second kernel joins in order.  Roles of the 16 warps:
//   warps 0, 3    a thread each loads through TMA: 0 walks the CTA's share, publishes items, loads Q tiles and a ring of K tiles,
//                 3 a ring of V tiles
//   warps 1, 2    a thread each issues tcgen05.mma: 1 S_X = Q_X K^T, 2 O_X += P_X V (P read from TMEM)
//   warps 4-7, 8-11   softmax warpgroups of the halves A and B: a thread owns a row
//   warps 12-15   output warpgroup: finished accumulators out of TMEM, to `out` or to the partials
// The halves are two softmax chains.  Work is a row of steps that they take in strict turn, across the units' borders: a step is a
// key tile of a unit with at most 128 rows (the output warpgroup joins what the halves have of it), or a key tile for one of the
// two Q tiles of a larger unit.
// kCluster, for few units: a thread-block cluster of 2, 4 or 8 CTAs has a unit and shares its key tiles out; their partial results are
// joined through distributed shared memory, each CTA joining and writing its part of the dims, so there is no second launch.
// TMEM: S [0,128)  P_A [128,192)  P_B [192,256)  O_A [256,384)  O_B [384,512).  Both halves' scores go through one S: a row is in
// its thread's registers 200 cycles after the product, and then the next step's product may run.  With an S of its own in
// which P replaced the scores, a half's next S had to wait for its P V: a chain of 3740 cycles a tile at 256 rows, of which the
// softmax is 1990.
// Every mbarrier wait is bounded.
// Calls on end in a graph (with the join): 1 sequence of 1037 tokens, 9 nodes, 16/8 heads 9.7 us, in a cluster of 8 (of these 5 are the chain of
// loads, a tile's S, softmax and P V, and 3 the two meetings and the join); 13 of 203 .. 3001, 5 .. 33 nodes, 32/8 31.9 us
// (2.8 TB/s: 6 us until the first tiles are there, 7 the join); 4 of 24000 .. 40960, 33 .. 64 nodes, 8/2 45.8 us (2.9 TB/s, 560 TFLOP/s);
// 128 of 512 .. 4096, 64 nodes, 32/8 336 to 349 us (3.8 to 4.0 TB/s, 890 to 920 TFLOP/s) in bursts of 20 calls between rests, at 1965 MHz, and 405 to 412 on end, at the power
// cap and 1390 to 1460 MHz, eagerly as in graphs: the softmax chain of a tile, about 3100 cycles for both halves against 2048 of tensor work.
#include <atomic>
#include <climits>
#include <cmath>
#include <limits>

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
constexpr int kTrRingK = 2, kTrRingV = 3;     // tiles of K and V in shared memory
constexpr int kTrItems = 4;                   // items in flight
constexpr float kTrRescale = 8.0f;
// The line's measure: cost of a key tile and of a unit by itself, with at most QT nodes (a step per tile) and with more (two).  Between
// the cycles that a CTA's P V thread took: 256 chains of 4 nodes, bound by memory, 2210 a tile and 2380 a unit (their steps no longer come here by themselves,
// but among larger trees); 13 ragged trees about 1300 and 3300 a tile of either kind; 128 trees of 64 nodes 3090 a tile and 11300 a unit.
struct TcLine {
  static constexpr int kKeys = kTrKv;
  static constexpr int kTileSplit = 4, kUnitSplit = 5, kTilePair = 7, kUnitPair = 24;
};

static __device__ int g_status_tree = 0;

struct TreeItem {
  int seq;              // -1: no more work
  int h;
  int q_row;            // global row of the unit's first node
  int node0, nodes;     // that node's index in its sequence, and how many the unit has
  int first, Lk;        // position of the sequence's node 0; its keys
  int t0, n;            // key tiles of this piece
  int split;            // at most QT nodes: a step per key tile, else two
  int turn;             // the half that takes the unit's first step
  int partial;          // -1: the whole unit, else where its partial results go
};

// A key tile of K or V into its place: in one box per half of the dims; of a sequence's last tile only what it has (`left` keys), in
// boxes of 16 rows.
__device__ __forceinline__ void tree_load(const CUtensorMap* whole, const CUtensorMap* map16, uint64_t* full, unsigned char* dst, int h, int row,
                                          int left) {
  if (left > kTrKv - 16) {
    mbar_expect_tx(full, kTrTile);
    tma_load_3d(dst, whole, full, 0, h, row);
    tma_load_3d(dst + kTrSub, whole, full, 64, h, row);
    return;
  }
  const int boxes = (left + 15) >> 4;
  mbar_expect_tx(full, boxes * 4096);
#pragma unroll 1
  for (int b = 0; b < boxes; ++b) {
    tma_load_3d(dst + b * 2048, map16, full, 0, h, row + b * 16);
    tma_load_3d(dst + kTrSub + b * 2048, map16, full, 64, h, row + b * 16);
  }
}
__device__ __forceinline__ void tree_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-memory address of CTA `rank` of the cluster that corresponds to this CTA's `addr`.
__device__ __forceinline__ uint32_t tree_cluster_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void tree_cluster_store(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void tree_cluster_store4(uint32_t addr, const uint32_t* v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// What the CTAs of a cluster send one another, in the room of the rings: from each of them 128 / CTAs dims (4 of a row side by
// side, so that a store or load of a warp moves 512 bytes), then maxima and sums, of 256 rows.
constexpr int kTrClusterLog = 3, kTrClusterMax = 1 << kTrClusterLog;
static_assert(2 * (64 + 2) * 256 * 4 <= 7 * kTrTile && kTrClusterMax * (16 + 2) * 256 * 4 <= 7 * kTrTile, "inbox");

template <bool kCluster>
__global__ void __launch_bounds__(kTrThreads, 1)
tree_attn_kernel(const TreeParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k16,
                 const __grid_constant__ CUtensorMap map_v16) {
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* const sQ = smem;                      // [2][32 KiB]
  unsigned char* const sK = smem + 2 * kTrTile;        // [kTrRingK][32 KiB]
  unsigned char* const sV = sK + kTrRingK * kTrTile;   // [kTrRingV][32 KiB]
  __shared__ __align__(8) uint64_t bar_item_full[kTrItems], bar_item_empty[kTrItems];
  __shared__ __align__(8) uint64_t bar_q_full[2], bar_q_empty[2];
  __shared__ __align__(8) uint64_t bar_k_full[kTrRingK], bar_k_empty[kTrRingK], bar_v_full[kTrRingV], bar_v_empty[kTrRingV];
  __shared__ __align__(8) uint64_t bar_s_full[2], bar_s_free, bar_p_full[2], bar_pv[2], bar_o_final[2], bar_o_free[2], bar_l_full[2], bar_l_empty[2];
  __shared__ float s_max[2][128], s_sum[2][128];       // a half's rows: maximum (log2 units) and sum
  __shared__ __align__(16) TreeItem s_item[kTrItems];
  __shared__ unsigned s_scan[kTrThreads / 32];
  __shared__ int s_at[2][3];                           // the share's first place and the one behind its last: sequence, unit, tile
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort, s_bare;                      // s_bare: some sequence has nodes but no keys

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.G, QT = 128 / p.G;
  // (the join comes in as CTAs of this kernel leave: beside one there is no room)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!kCluster && p.above > 0) {
    // behind the kernel for few nodes, which as a rule has taken all there is
    int left = 0;
#pragma unroll 1
    for (int i = tid; i < p.batch; i += kTrThreads) left |= min(p.cu_q[i + 1], p.total_q) - max(0, p.cu_q[i]) > p.above;
    if (!__syncthreads_or(left)) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      if (tid == 0) p.pieces->of[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
  }
  if (tid == 0) {
    s_abort = 0;
    s_bare = 0;
    for (int i = 0; i < kTrItems; ++i) { mbar_init(&bar_item_full[i], 1); mbar_init(&bar_item_empty[i], 15); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_q_full[i], 1);
      mbar_init(&bar_q_empty[i], 1);
      mbar_init(&bar_s_full[i], 1);
      mbar_init(&bar_p_full[i], 4);
      mbar_init(&bar_pv[i], 1);
      mbar_init(&bar_o_final[i], 1);
      mbar_init(&bar_o_free[i], 4);
      mbar_init(&bar_l_full[i], 4);
      mbar_init(&bar_l_empty[i], 4);
    }
    mbar_init(&bar_s_free, 4);
    for (int i = 0; i < kTrRingK; ++i) { mbar_init(&bar_k_full[i], 1); mbar_init(&bar_k_empty[i], 1); }
    for (int i = 0; i < kTrRingV; ++i) { mbar_init(&bar_v_full[i], 1); mbar_init(&bar_v_empty[i], 1); }
    mbar_fence_init();
    s_at[0][0] = s_at[1][0] = p.batch;
    s_at[0][1] = s_at[0][2] = s_at[1][1] = s_at[1][2] = 0;
  }
  __syncthreads();
  int c_nodes = 0, c_row = 0, c_head = 0, c_tiles = 0;       // kCluster: the cluster's unit
  const int c_log = kCluster ? p.cluster_log : 0, c_size = 1 << c_log, c_rank = blockIdx.x & (c_size - 1);
  const int c_dims = 128 >> c_log, c_inbox = (c_dims + 2) * 256;                        // floats of one sender
  if constexpr (kCluster) {
    // sequence i owns blocks of nodes [cu_q[i] / (2 * QT) + i, ...); there are few sequences
    const int x = static_cast<int>(blockIdx.x) >> c_log, slot = x / p.Hkv;
    c_head = x - slot * p.Hkv;
    int seq = 0;
#pragma unroll 1
    for (int i = 1; i < p.batch; ++i)
      if (max(0, min(p.cu_q[i], p.total_q)) / (2 * QT) + i <= slot) seq = i;
    const TreeSeq s = tree_seq<TcLine>(p, 2 * QT, seq);
    const int block = slot - (s.q_begin / (2 * QT) + seq), node0 = block * 2 * QT;
    c_nodes = block >= 0 ? min(s.nodes - node0, 2 * QT) : 0;
    c_row = s.q_begin + node0;
    c_tiles = s.tiles;
    if (c_nodes > 0 && tid == 0) {
      s_bare = c_rank == 0 && c_tiles == 0;
      s_at[0][0] = s_at[1][0] = c_tiles > 0 ? seq : p.batch;
      s_at[0][1] = s_at[1][1] = block * p.Hkv + c_head;
      // (what is left over goes to the CTAs in front: the last has the tile with the masks)
      s_at[0][2] = (c_tiles * c_rank + c_size - 1) >> c_log;
      s_at[1][2] = (c_tiles * (c_rank + 1) + c_size - 1) >> c_log;
    }
  } else
    tree_share<TcLine, kTrThreads>(p, 2 * QT, s_scan, s_at, &s_bare);
  __syncthreads();
  volatile int* abort_flag = &s_abort;
  uint32_t tmem = 0;
  bool met = false;               // kCluster: this thread has been through the first meeting
  if (warp > 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (kCluster && s_bare) {
      for (int e = tid - 32; e < c_nodes * G * 16; e += kTrThreads - 32)
        reinterpret_cast<uint4*>(p.out + (static_cast<long long>(c_row + e / (G * 16)) * p.H + c_head * G) * 128)[e % (G * 16)] = make_uint4(0, 0, 0, 0);
    } else if (s_bare) {
      // sequences with nodes and no keys: zeros
#pragma unroll 1
      for (int i = blockIdx.x; i < p.batch; i += gridDim.x) {
        const TreeSeq s = tree_seq<TcLine>(p, 2 * QT, i);
        if (s.tiles > 0) continue;
        uint4* const dst = reinterpret_cast<uint4*>(p.out + static_cast<long long>(s.q_begin) * p.H * 128);
        for (long long e = tid - 32; e < static_cast<long long>(s.nodes) * p.H * 16; e += kTrThreads - 32) dst[e] = make_uint4(0, 0, 0, 0);
      }
    }
    if (warp == 1) {
      tc::tmem_alloc(&s_tmem_base, 512);
      tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    named_bar_sync(1, kTrThreads - 32);         // (the producer is on its way already)
    tc::fence_after_sync();
    tmem = s_tmem_base;
  }

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;" ::: "memory");
    if (tid == 0) {
      // ================================ items, Q and K ================================
      tma_prefetch_desc(&map_q);
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
      int cont = 0, head = 0;
      int2 head_unit = make_int2(0, 0);
      int seq = s_at[0][0], unit = s_at[0][1], from = s_at[0][2], have = -1;
      TreeSeq s = {};
      TreeRows<TcLine> rows = {};
      const int end_seq = s_at[1][0], end_unit = s_at[1][1], end_tile = s_at[1][2];
      int n_pub = 0, q_use = 0, turn = 0, k_at = 0, k_ph = 1;
      int halves = 0;                 // kCluster: halves with work
      bool ok = true, started = false;
#pragma unroll 1
      while (ok && seq < p.batch) {
        // the next unit that has tiles here
        if (have != seq) {
          s = tree_seq<TcLine>(p, 2 * QT, seq);
          have = seq;
        }
        if (unit >= s.blocks * p.Hkv) {
          seq = seq < end_seq ? seq + 1 : p.batch;
          unit = from = 0;
          continue;
        }
        const bool at_end = seq == end_seq && unit >= end_unit;
        const int t0 = from, t1 = !at_end ? s.tiles : unit == end_unit ? max(end_tile, from) : from;
        const int block = unit / p.Hkv, h = unit - block * p.Hkv, node0 = block * 2 * QT, nodes = min(2 * QT, s.nodes - node0);
        const int owner = seq;
        ++unit;
        from = 0;
        if (at_end) seq = p.batch;
        if (t0 == t1) continue;
        const int split = nodes <= QT, q_row = s.q_begin + node0;
        const bool whole = t0 == 0 && t1 == s.tiles;
        const int place = t0 > 0 ? 0 : 1;
        if (t0 > 0) {
          cont = t1 < s.tiles ? 1 : 2;
        } else if (!whole) {
          head = nodes;
          head_unit = make_int2(q_row, h);
        }
        const int is = n_pub % kTrItems;
        if (!t2_wait_timed(&bar_item_empty[is], ((n_pub / kTrItems) & 1) ^ 1, abort_flag)) { ok = false; break; }
        s_item[is] = {owner, h, q_row, node0, nodes, s.Lk - s.nodes, s.Lk, t0, t1 - t0, split, turn, whole ? -1 : 2 * static_cast<int>(blockIdx.x) + place};
        mbar_arrive(&bar_item_full[is]);
        ++n_pub;
        if (split) turn ^= (t1 - t0) & 1;
        if constexpr (kCluster) halves = split && t1 - t0 == 1 ? 1 : 2;     // (a CTA has one item)
        rows.start(p, owner, t0);
        int row = rows.next(p), left = s.Lk - t0 * kTrKv;
        if (!started) {
          // everything so far overlaps the end of the kernel in front: lengths and tables, which it does not write
          tma_prefetch_l2_3d(&map_k, 0, h, row);
          tma_prefetch_l2_3d(&map_k, 64, h, row);
          asm volatile("griddepcontrol.wait;" ::: "memory");
          started = true;
        }
#pragma unroll 1
        for (int t = t0; t < t1; ++t) {
          if (!t2_wait_timed(&bar_k_empty[k_at], k_ph, abort_flag)) { ok = false; break; }
          tree_load(&map_k, &map_k16, &bar_k_full[k_at], sK + k_at * kTrTile, h, row, left);
          if (++k_at == kTrRingK) { k_at = 0; k_ph ^= 1; }
          if (t == t0) {
            // its Q tile, or two
#pragma unroll 1
            for (int x = 0; x < (split ? 1 : 2); ++x, ++q_use) {
              const int b = q_use & 1;
              if (!t2_wait_timed(&bar_q_empty[b], ((q_use >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
              mbar_expect_tx(&bar_q_full[b], QT * G * 256);
              tma_load_3d(sQ + b * kTrTile, &map_q, &bar_q_full[b], 0, h * G, q_row + x * QT);
              tma_load_3d(sQ + b * kTrTile + kTrSub, &map_q, &bar_q_full[b], 64, h * G, q_row + x * QT);
            }
          }
          if (t + 1 < t1) {
            row = rows.next(p);
            left -= kTrKv;
          }
        }
      }
      if (!started) asm volatile("griddepcontrol.wait;" ::: "memory");
      if constexpr (!kCluster) {
        p.pieces->of[blockIdx.x] = make_int4(head, cont, head_unit.x, head_unit.y);
      }
      if (ok) {
        const int is = n_pub % kTrItems;
        if (t2_wait_timed(&bar_item_empty[is], ((n_pub / kTrItems) & 1) ^ 1, abort_flag)) {
          s_item[is].seq = -1;
          mbar_arrive(&bar_item_full[is]);
          // Every role has taken it, so all their waits have ended.  (kCluster: the output warps take it behind the meeting that this
          // warp is to come to; in front of it their last wait is for the accumulators.)
          if constexpr (kCluster) {
            for (int i = 0; i < halves; ++i) t2_wait_timed(&bar_o_final[i], 0, abort_flag);
          } else
            t2_wait_timed(&bar_item_empty[is], (n_pub / kTrItems) & 1, abort_flag);
        }
      }
    } else if (warp == 1 && lane == 0) {
      // ================================ S = Q K^T ================================
      // (the sign of a negative scale: in the softmax, a pass of its own over S, it cost every call up to 1 %)
      const uint32_t idesc_qk = tc::idesc_bf16_f32(128, 128, false, false) | p.negate;
      constexpr uint32_t desc_hi = tc::smem_desc_sw128_hi(1024);
      const uint32_t q_lo = tc::smem_desc_sw128_lo(smem_u32(sQ), 16), k_lo = tc::smem_desc_sw128_lo(smem_u32(sK), 16);
      int n_item = 0, q_use = 0, k_at = 0, k_ph = 0, n_step = 0;
      bool ok = true;
      while (ok) {
        const int is = n_item % kTrItems;
        if (!t2_wait(&bar_item_full[is], (n_item / kTrItems) & 1, abort_flag)) break;
        const int seq = s_item[is].seq, split = s_item[is].split, steps = split ? s_item[is].n : 2 * s_item[is].n;
        mbar_arrive(&bar_item_empty[is]);
        if (seq < 0) break;
        ++n_item;
#pragma unroll 1
        for (int at = 0; at < steps; ++at, ++n_step) {
          const int hx = n_step & 1, second = !split && (at & 1);      // second: of the unit's two Q tiles
          const int q = q_use + second;
          if (at <= second && !t2_wait(&bar_q_full[q & 1], (q >> 1) & 1, abort_flag)) { ok = false; break; }
          if (!t2_wait_hot(&bar_k_full[k_at], k_ph, abort_flag)) { ok = false; break; }
          // (the scores of the step in front are in registers)
          if (!t2_wait_hot(&bar_s_free, (n_step & 1) ^ 1, abort_flag)) { ok = false; break; }
          tc::fence_after_sync();
          const uint32_t d = tmem, qd = q_lo + (q & 1) * (kTrTile >> 4), kd = k_lo + k_at * (kTrTile >> 4);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t off = ((ks >> 2) * kTrSub + (ks & 3) * 32) >> 4;
            tc::mma_ss_lo(d, qd + off, kd + off, desc_hi, idesc_qk, ks > 0);
          }
          tc::commit(&bar_s_full[hx]);
          if (split || second) {
            tc::commit(&bar_k_empty[k_at]);
            if (++k_at == kTrRingK) { k_at = 0; k_ph ^= 1; }
          }
          if (at + (split ? 1 : 2) >= steps) tc::commit(&bar_q_empty[q & 1]);
        }
        q_use += split ? 1 : 2;
      }
    } else if (warp == 2 && lane == 0) {
      // ================================ O += P V ================================
      // (A thread of its own: next to the softmax warps of its scheduler a single thread retires an instruction in 10 cycles, and
      // what stands around the 16 products of a step took as long as they did.)
      constexpr uint32_t idesc_pv = tc::idesc_bf16_f32(128, 128, false, true);
      constexpr uint32_t desc_hi = tc::smem_desc_sw128_hi(1024);
      const uint32_t v_lo = tc::smem_desc_sw128_lo(smem_u32(sV), kTrSub);
      int n_item = 0, v_at = 0, v_ph = 0, n_step = 0, o_ph = 3;
      bool ok = true;
      while (ok) {
        const int is = n_item % kTrItems;
        if (!t2_wait(&bar_item_full[is], (n_item / kTrItems) & 1, abort_flag)) break;
        const int seq = s_item[is].seq, split = s_item[is].split, steps = split ? s_item[is].n : 2 * s_item[is].n;
        mbar_arrive(&bar_item_empty[is]);
        if (seq < 0) break;
        ++n_item;
#pragma unroll 1
        for (int at = 0; at < steps; ++at, ++n_step) {
          const int hx = n_step & 1;
          if (!t2_wait_hot(&bar_v_full[v_at], v_ph, abort_flag)) { ok = false; break; }
          if (at < 2) {
            // the output warpgroup has taken the accumulator of the unit in front
            if (!t2_wait_hot(&bar_o_free[hx], (o_ph >> hx) & 1, abort_flag)) { ok = false; break; }
            o_ph ^= 1 << hx;
          }
          if (!t2_wait_hot(&bar_p_full[hx], (n_step >> 1) & 1, abort_flag)) { ok = false; break; }
          tc::fence_after_sync();
          const uint32_t d = tmem + 256 + hx * 128, a = tmem + 128 + hx * 64, v = v_lo + v_at * (kTrTile >> 4);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) tc::mma_ts_lo(d, a + ks * 8, v + ks * (2048 >> 4), desc_hi, idesc_pv, at >= 2 || ks > 0);
          tc::commit(&bar_pv[hx]);
          if (at + 2 >= steps) tc::commit(&bar_o_final[hx]);
          if (split || (at & 1)) {
            tc::commit(&bar_v_empty[v_at]);
            if (++v_at == kTrRingV) { v_at = 0; v_ph ^= 1; }
          }
        }
      }
    } else if (warp == 3 && lane == 0) {
      // ================================ V ================================
      TreeRows<TcLine> rows = {};
      int n_item = 0, v_at = 0, v_ph = 1;
      bool ok = true;
      while (ok) {
        const int is = n_item % kTrItems;
        if (!t2_wait(&bar_item_full[is], (n_item / kTrItems) & 1, abort_flag)) break;
        const int seq = s_item[is].seq, h = s_item[is].h, t0 = s_item[is].t0, n = s_item[is].n;
        int left = s_item[is].Lk - t0 * kTrKv;
        mbar_arrive(&bar_item_empty[is]);
        if (seq < 0) break;
        ++n_item;
        rows.start(p, seq, t0);
#pragma unroll 1
        for (int j = 0; j < n; ++j, left -= kTrKv) {
          const int row = rows.next(p);
          if (!t2_wait(&bar_v_empty[v_at], v_ph, abort_flag)) { ok = false; break; }
          tree_load(&map_v, &map_v16, &bar_v_full[v_at], sV + v_at * kTrTile, h, row, left);
          if (++v_at == kTrRingV) { v_at = 0; v_ph ^= 1; }
        }
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;" ::: "memory");
    // ================================ softmax ================================
    const int hx = (warp - 4) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;                  // row of the tile
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tmem_s = tmem + lane_base, tmem_p = tmem + 128 + hx * 64 + lane_base, tmem_o = tmem + 256 + hx * 128 + lane_base;
    const float c = p.scale_abs;
    int n_item = 0, ns = 0, n_fin = 0;
    int v_at = 0, v_ph = 0;                             // place and phase in the V ring of the unit's last tile
    int v_next = 0;                                     // (tiles so far, modulo the ring's two turns)
    bool ok = true;
    while (ok) {
      const int is = n_item % kTrItems;
      if (!t2_wait(&bar_item_full[is], (n_item / kTrItems) & 1, abort_flag)) break;
      const TreeItem it = s_item[is];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_item_empty[is]);
      if (it.seq < 0) break;
      ++n_item;
      const int mine = hx ^ it.turn;                             // 0: this half takes the unit's first step
      const int nx = it.split ? (it.n + 1 - mine) >> 1 : it.n;
      const int tile = it.split ? 0 : mine;                      // the Q tile
      const int tile_nodes = tile ? it.nodes - QT : min(it.nodes, QT);
      const bool active = quarter * 32 < tile_nodes * G;         // this warp has rows
      const int in_tile = r / G + tile * QT;                     // the row's node within the unit
      const bool row_ok = in_tile < it.nodes && r < QT * G;
      const bool chain = p.masks == nullptr;
      const uint32_t* const mask = !chain && row_ok ? p.masks + static_cast<long long>(it.q_row + in_tile) * p.mask_words : nullptr;
      if (mask && (it.t0 + it.n) * kTrKv > it.first) asm volatile("prefetch.global.L1 [%0];" ::"l"(mask));
      // (rows that are none see nothing: a chain's row of an index below all)
      const int node = row_ok ? it.node0 + in_tile : -0x40000000;
      v_next = (v_next + it.n) % (2 * kTrRingV);
      { const int last = v_next ? v_next - 1 : 2 * kTrRingV - 1; v_at = last % kTrRingV; v_ph = last / kTrRingV; }
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < nx; ++j) {
        if (!t2_wait_hot(&bar_s_full[hx], ns & 1, abort_flag)) { ok = false; break; }
        ++ns;
        const int key0 = (it.t0 + (it.split ? 2 * j + mine : j)) * kTrKv;
        if (active) {
          tc::fence_after_sync();
          if (key0 + kTrKv > min(it.first, it.Lk)) {
            // the tile reaches the nodes: masked scores go back over S first (rolled: the hot code stays short)
#pragma unroll 1
            for (int cch = 0; cch < 4; ++cch) {
              const int col = key0 + cch * 32;
              const uint32_t keep = chain || row_ok ? tree_keep32(mask, p.mask_words, node, col - it.first, it.Lk - col) : 0u;
              if (__all_sync(0xffffffffu, keep == 0xffffffffu)) continue;
              uint32_t v[32];
              tc::ld_32x32b_x32(tmem_s + cch * 32, v);
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((keep >> i) & 1)) v[i] = 0xff800000u;   // -inf
              tc::st_32x32b_x32(tmem_s + cch * 32, v);
            }
            tc::wait_st();
          }
          // the whole S row in registers: four TMEM loads in flight, one wait; eight independent chains of 3-input max
          uint32_t sv[4][32];
#pragma unroll
          for (int cch = 0; cch < 4; ++cch) tc::ld_32x32b_x32(tmem_s + cch * 32, sv[cch]);
          tc::wait_ld();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_s_free);
          float m8[8] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int cch = 0; cch < 4; ++cch)
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              m8[(i >> 1) & 7] = fmax3(m8[(i >> 1) & 7], __uint_as_float(sv[cch][i]), __uint_as_float(sv[cch][i + 1]));
          const float mx = fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]));
          const float m_new = fmaxf(m_used, mx);
          if (j == 0) {
            m_used = m_new;
          } else {
            const bool grow = (m_new - m_used) * c > kTrRescale;
            if (__any_sync(0xffffffffu, grow)) {
              if (!t2_wait_hot(&bar_pv[hx], ns & 1, abort_flag)) { ok = false; break; }
              tc::fence_after_sync();
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
            if (cch == 0 && ns > 1) {
              // the P of the half's step in front has been used
              if (!t2_wait_hot(&bar_pv[hx], ns & 1, abort_flag)) { ok = false; break; }
              tc::fence_after_sync();
            }
            tc::st_32x32b_x16(tmem_p + cch * 16, pk);
          }
          if (!ok) break;
          float a0, a1;
          f32x2_unpack(f32x2_add(f32x2_add(ls0, ls1), f32x2_add(ls2, ls3)), a0, a1);
          l += a0 + a1;
          tc::wait_st();
        } else {
          if (lane == 0) mbar_arrive(&bar_s_free);
          // (no rows, but in step with the others: the next S comes ahead of this one's P V, and its arrival below must not count
          // for the step in front)
          if (ns > 1 && !t2_wait(&bar_pv[hx], ns & 1, abort_flag)) { ok = false; break; }
        }
        if (key0 + kTrKv > it.Lk) {
          // The sequence's last tile: V rows behind its end are stale or foreign; zero them, so that 0 * garbage cannot turn into
          // NaN in the tensor core.  (It is the unit's last V tile.)
          if (!t2_wait_hot(&bar_v_full[v_at], v_ph, abort_flag)) { ok = false; break; }
          unsigned char* const rows = sV + v_at * kTrTile;
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
        const int h0 = it.turn ^ turn;                   // the half that has it; joined: the other, too
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (e == 1 && !joined) continue;
          const int hx = h0 ^ e;
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
        if constexpr (kCluster) {
          // (the last turn waited for is the CTA's last product: nothing reads the rings any more)
          if (turn == 0) {
            if (!it.split) {
              if (!t2_wait(&bar_o_final[it.turn ^ 1], nf[it.turn ^ 1] & 1, abort_flag)) { ok = false; break; }
            }
            tree_cluster_sync();
            met = true;
          }
        }
        if (quarter * 32 < tile_nodes * G) {
          const float M = fmaxf(m[0], m[1]);
          float wa = M == -INFINITY ? 0.f : fast_exp2(m[0] - M), wb = M == -INFINITY ? 0.f : fast_exp2(m[1] - M);
          const float sum = l[0] * wa + l[1] * wb;
          const bool row_ok = r < tile_nodes * G;
          const int t = r / G;
          __nv_bfloat16* const dst = p.out + (static_cast<long long>(it.q_row + turn * QT + t) * p.H + it.h * G + (r - t * G)) * 128;
          float* const part = kCluster || it.partial < 0 ? nullptr : p.partials + static_cast<long long>(it.partial) * kTrPartial + (turn * 4 + quarter) * kTrGroup + lane;
          const uint32_t inbox = smem_u32(smem) + c_rank * c_inbox * 4, in_row = turn * 128 + r;
          if constexpr (kCluster) {
#pragma unroll 1
            for (int x = 0; x < c_size; ++x) {
              tree_cluster_store(tree_cluster_addr(inbox + c_dims * 1024 + in_row * 4, x), M);
              tree_cluster_store(tree_cluster_addr(inbox + (c_dims + 1) * 1024 + in_row * 4, x), sum);
            }
          } else if (part) {
            part[128 * 32] = M;
            part[129 * 32] = sum;
          } else {
            const float inv = sum > 0.f ? 1.f / sum : 0.f;      // (a row that sees nothing: zeros)
            wa *= inv;
            wb *= inv;
          }
          const uint32_t ta = tmem + 256 + h0 * 128 + lane_base, tb = tmem + 384 - h0 * 128 + lane_base;
#pragma unroll 1
          for (int cch = 0; cch < 8; ++cch) {
            uint32_t a[16];
            tc::ld_32x32b_x16(ta + cch * 16, a);
            uint32_t b[16];
            if (joined) {
              tc::ld_32x32b_x16(tb + cch * 16, b);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) b[i] = 0;
            }
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) a[i] = __float_as_uint(fmaf(__uint_as_float(b[i]), wb, __uint_as_float(a[i]) * wa));
            if constexpr (kCluster) {
              const uint32_t to = tree_cluster_addr(inbox + (cch * 16 & (c_dims - 1)) * 1024 + in_row * 16, cch * 16 >> (7 - c_log));
#pragma unroll
              for (int i = 0; i < 16; i += 4) tree_cluster_store4(to + i * 1024, a + i);
            } else if (part) {
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
          mbar_arrive(&bar_o_free[h0]);
          if (joined) mbar_arrive(&bar_o_free[h0 ^ 1]);
        }
      }
    }
  }

  if constexpr (kCluster) {
    if (!met) tree_cluster_sync();             // (output warps that had an item have been here before)
    tree_cluster_sync();
    // all partial results are here: a thread joins a row, 8 of this CTA's dims at a time
    const float* const inbox = reinterpret_cast<const float*>(smem);
    const int row = tid & 255, half = row >> 7, r = row & 127, t = r / G, node = half * QT + t;
    if (r < QT * G && node < c_nodes && c_tiles > 0) {
      // (with fewer tiles than CTAs some have sent nothing)
      float m[kTrClusterMax], l[kTrClusterMax], M = -INFINITY;
#pragma unroll
      for (int x = 0; x < kTrClusterMax; ++x) {
        const bool sent = x < c_size && (c_tiles * (x + 1) + c_size - 1) >> c_log > (c_tiles * x + c_size - 1) >> c_log;
        m[x] = sent ? inbox[x * c_inbox + c_dims * 256 + row] : -INFINITY;
        l[x] = sent ? inbox[x * c_inbox + (c_dims + 1) * 256 + row] : 0.f;
        M = fmaxf(M, m[x]);
      }
      const float ref = M == -INFINITY ? 0.f : M;
      float sum = 0.f;
#pragma unroll
      for (int x = 0; x < kTrClusterMax; ++x) {
        m[x] = fast_exp2(m[x] - ref);
        sum = fmaf(l[x], m[x], sum);
      }
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
      __nv_bfloat16* const dst = p.out + (static_cast<long long>(c_row + node) * p.H + c_head * G + (r - t * G)) * 128 + c_rank * c_dims;
#pragma unroll 1
      for (int d = (tid >> 8) * 8; d < c_dims; d += 16) {
        float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < kTrClusterMax; ++x) {
          if (m[x] == 0.f) continue;             // (nothing sent, or nothing that counts)
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(inbox + x * c_inbox + (d + i) * 256 + row * 4);
            o[i] = fmaf(v.x, m[x], o[i]);
            o[i + 1] = fmaf(v.y, m[x], o[i + 1]);
            o[i + 2] = fmaf(v.z, m[x], o[i + 2]);
            o[i + 3] = fmaf(v.w, m[x], o[i + 3]);
          }
        }
        uint4 v;
        v.x = pack_bf16(o[0] * inv, o[1] * inv);
        v.y = pack_bf16(o[2] * inv, o[3] * inv);
        v.z = pack_bf16(o[4] * inv, o[5] * inv);
        v.w = pack_bf16(o[6] * inv, o[7] * inv);
        *reinterpret_cast<uint4*>(dst + d) = v;
      }
    }
  }
  // ---- teardown: everyone meets, then the allocating warp frees TMEM ----
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
  if (tid == 0 && s_abort) atomicExch(&g_status_tree, 1);
}

// Units that a cut ran through.  A task is (unit, group of 32 rows, some of the dims: the fewer units, the fewer); its partial results
// come as bulk copies, all under way at once.  What takes time here is round trips to L2 (records 0.4 us, pieces 1.4, of 6.6 at 4 long
// contexts, of 4 at 13 trees) and fetching the code, which is new for every launch (going through it once ahead of the wait: the same):
// so every warp reads all records (five a lane) and finds its unit and pieces by bits of ballots.
constexpr int kTrJoinThreads = 128;
constexpr int kTrJoinCtas = 5;                // per SM
constexpr int kTrJoinPieces = 16;             // of 16 dims; 2 of 128
constexpr int kTrJoinFloats = kTrJoinPieces * (16 * 32 + 64);
constexpr int kTrJoinWords = kTrMaxCtas / 32;

// kTwo: of two kernels (a form of its own: as one, with 128 registers for 95, it cost 128 trees of 64 nodes 2.4 of 341 us).
template <bool kTwo>
__global__ void __launch_bounds__(kTrJoinThreads) tree_join_kernel(const TreeParams p, const TreeJoin join_of, int ctas) {
  __shared__ __align__(128) float s_buf[kTrJoinFloats];
  __shared__ float s_weight[kTrJoinPieces][32];
  __shared__ short s_list[kTrMaxCtas + 1];    // places of the unit's pieces
  __shared__ __align__(8) uint64_t s_bar;
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.G, QT = 128 / G;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    s_abort = 0;
    mbar_init(&s_bar, 1);
    mbar_fence_init();
  }
  int loads = 0;                              // phases of the barrier
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // (the second kernel's are looked at along with the first's: mostly there are none)
  bool second = false;
  if constexpr (kTwo) {
    int any = 0;
#pragma unroll
    for (int w = 0; w < kTrJoinWords; ++w)
      if (w * 32 + lane < ctas) any |= join_of.of[1].pieces->of[w * 32 + lane].x;
    second = __any_sync(0xffffffffu, any);
  }
#pragma unroll 1
  for (int kernel = 0; kernel < (kTwo && second ? 2 : 1); ++kernel) {
    const TreeCuts cuts = {kTwo && kernel ? join_of.of[1].pieces : join_of.of[0].pieces, kTwo && kernel ? join_of.of[1].partials : join_of.of[0].partials,
                           kTwo && kernel ? join_of.of[1].stride : join_of.of[0].stride};
    int4 piece[kTrJoinWords];                   // nodes of the unit that begins (0: none), how the share begins, that unit
#pragma unroll
    for (int w = 0; w < kTrJoinWords; ++w) {
      const int c = w * 32 + lane;
      piece[w] = c < ctas ? cuts.pieces->of[c] : make_int4(0, 0, 0, 0);
    }
    unsigned heads[kTrJoinWords];
    int units = 0;
#pragma unroll
    for (int w = 0; w < kTrJoinWords; ++w) {
      heads[w] = __ballot_sync(0xffffffffu, piece[w].x > 0);
      units += __popc(heads[w]);
    }
    // tasks of a unit: 8 groups x 1, 2, 4 or 8 slices of the dims, so that there are about as many as CTAs
    const int shift = units > 111 ? 0 : units > 55 ? 1 : units > 27 ? 2 : 3;
#pragma unroll 1
    for (int task = blockIdx.x; task < units << (3 + shift); task += gridDim.x) {
      // the unit: the CTA that has its first piece, and how many nodes
      int k = task >> (3 + shift), c0 = 0, nodes_all = 0;
      int2 unit = make_int2(0, 0);
#pragma unroll
      for (int w = 0; w < kTrJoinWords; ++w) {
        const unsigned found = __ballot_sync(0xffffffffu, piece[w].x > 0 && __popc(heads[w] & ((1u << lane) - 1)) == k);
        if (found) {
          c0 = w * 32 + __ffs(found) - 1;
          nodes_all = __shfl_sync(0xffffffffu, piece[w].x, __ffs(found) - 1);
          unit.x = __shfl_sync(0xffffffffu, piece[w].z, __ffs(found) - 1);
          unit.y = __shfl_sync(0xffffffffu, piece[w].w, __ffs(found) - 1);
        }
        k -= __popc(heads[w]);
      }
      const int at = task & ((8 << shift) - 1), group = at >> shift, half = group >> 2;
      const int nodes = half ? nodes_all - QT : min(nodes_all, QT);
      if ((group & 3) * 32 >= nodes * G) continue;
      __syncthreads();                          // (the list and the buffer of the task in front have been read)
      // its pieces: that CTA's second place, then first places up to the unit's last
      int n = 1;
      bool open = true;
      if (tid == 0) s_list[0] = static_cast<short>(2 * c0 + 1);
#pragma unroll
      for (int w = 0; w < kTrJoinWords; ++w) {
        const int c = w * 32 + lane;
        const unsigned after = __ballot_sync(0xffffffffu, c > c0), last = __ballot_sync(0xffffffffu, piece[w].y == 2) & after;
        unsigned mine = __ballot_sync(0xffffffffu, piece[w].y != 0) & after;
        if (last) mine &= last ^ (last - 1);    // up to the first of them
        if (!open) mine = 0;
        if (warp == 0 && (mine >> lane) & 1) s_list[n + __popc(mine & ((1u << lane) - 1))] = static_cast<short>(2 * c);
        n += __popc(mine);
        open = open && !last;
      }
      __syncthreads();
      const int r = (group & 3) * 32 + lane, t = r / G;
      const int dims_all = 128 >> shift, first_dim = (at & ((1 << shift) - 1)) * dims_all;
      __nv_bfloat16* const dst = p.out + (static_cast<long long>(unit.x + half * QT + t) * p.H + unit.y * G + (r - t * G)) * 128;
      // as many dims at a time as let all pieces into the buffer, at least 16
      const int dims = min(dims_all, n <= 2 ? 128 : n <= 4 ? 64 : n <= 8 ? 32 : 16), stride = dims * 32 + 64;
#pragma unroll 1
      for (int dim0 = first_dim; dim0 < first_dim + dims_all; dim0 += dims) {
        float M = -INFINITY, sum = 0.f, o[16];
#pragma unroll 1
        for (int base = 0; base < n; base += kTrJoinPieces) {
          const int m = min(n - base, kTrJoinPieces);
          if (loads) __syncthreads();           // the buffer has been read
          if (tid == 0) mbar_expect_tx(&s_bar, m * stride * 4);
          __syncwarp();
          if (tid < m) {
            // of a piece: its dims, then maxima and sums
            const float* const from = cuts.partials + s_list[base + tid] * static_cast<long long>(cuts.stride) + group * kTrGroup;
            tree_bulk_load(s_buf + tid * stride, from + dim0 * 32, dims * 128, &s_bar);
            tree_bulk_load(s_buf + tid * stride + dims * 32, from + 128 * 32, 256, &s_bar);
          }
          // (a wait that gave up leaves the barriers below complete: nobody leaves)
          if (!mbar_wait(&s_bar, loads & 1, &s_abort)) atomicExch(&g_status_tree, 1);
          ++loads;
          // every warp for itself: the new maximum and sum; the weights are shared out
          float top = M;
#pragma unroll 4
          for (int x = 0; x < m; ++x) top = fmaxf(top, s_buf[x * stride + dims * 32 + lane]);
          const float ref = top == -INFINITY ? 0.f : top, was = fast_exp2(M - ref);
          M = top;
          sum *= was;
#pragma unroll 4
          for (int x = 0; x < m; ++x) {
            const float w = fast_exp2(s_buf[x * stride + dims * 32 + lane] - ref);
            sum = fmaf(s_buf[x * stride + dims * 32 + 32 + lane], w, sum);
            if ((x & 3) == warp) s_weight[x][lane] = w;
          }
          __syncthreads();
          const float inv = sum > 0.f ? 1.f / sum : 0.f;
          // a row's dims are a quarter to each warp, up to 16 at a time: two stores then fill a sector (more pieces follow with
          // 16 dims only)
          const auto join = [&](auto width) {
            constexpr int N = decltype(width)::value;
#pragma unroll 1
            for (int d = warp * N; d < dims; d += 4 * N) {
#pragma unroll
              for (int i = 0; i < N; ++i) o[i] = N == 4 && base ? o[i] * was : 0.f;
#pragma unroll 2
              for (int x = 0; x < m; ++x) {
                const float w = s_weight[x][lane];
#pragma unroll
                for (int i = 0; i < N; ++i) o[i] = fmaf(s_buf[x * stride + (d + i) * 32 + lane], w, o[i]);
              }
              if (base + m == n && r < nodes * G) {
#pragma unroll
                for (int i = 0; i < N; i += 8) {
                  const uint2 a = make_uint2(pack_bf16(o[i] * inv, o[i + 1] * inv), pack_bf16(o[i + 2] * inv, o[i + 3] * inv));
                  if constexpr (N == 4)
                    *reinterpret_cast<uint2*>(dst + dim0 + d) = a;
                  else
                    *reinterpret_cast<uint4*>(dst + dim0 + d + i) =
                        make_uint4(a.x, a.y, pack_bf16(o[i + 4] * inv, o[i + 5] * inv), pack_bf16(o[i + 6] * inv, o[i + 7] * inv));
                }
              }
            }
          };
          if (dims == 16) join(std::integral_constant<int, 4>{});
          else if (dims == 32) join(std::integral_constant<int, 8>{});
          else join(std::integral_constant<int, 16>{});
        }
      }
    }
  }
}

constexpr size_t kTrSmem = static_cast<size_t>(2 + kTrRingK + kTrRingV) * kTrTile;
// Sizes of clusters, and how wide (in key tiles) the table may be for each: what the host knows of the lengths.  Us with the join |
// with clusters, calls on end in a graph:
//   8   1 sequence of 300, 4000, 12000 tokens, 9 nodes, 16/8 heads   13.0, 16.9, 21.5 | 9.5, 12.0, 18.4; 60 nodes, 8/2 heads
//       15.4, 20.5, 29.9 | 13.1, 20.3, 29.8, and of 16000 30.0 | 37.5
//   4   4 of 500, 2000, 4000, 20 nodes, 32/8   16.6, 20.1, 26.2 | 10.1, 15.6, 23.4; of 200 .. 4000   19.4 | 21.8
//   2   9 of 500, 2000, 4000, 9 nodes, 16/8    15.8, 24.7, 36.4 | 12.8, 20.8, 31.7; 6 of 200 .. 4000   21.0 | 22.4
// (What clusters lose, they lose where lengths differ; wider tables make that worse: 4 of 300 .. 8000 lost 8 us, 6 of them 5.)
constexpr int kTrClusterSizes = 3;
constexpr int kTrClusterTiles[kTrClusterSizes] = {128, 40, 32};
// Blocks of 16 / G nodes that a sequence may have in the kernel for few nodes, which reads its keys once for each.  Us with 1 | 2 | 4 | without a limit (and
// the launch behind it), calls on end in a graph at 16/8 heads: 48 sequences of 1 node and 16 of 16 (2 blocks), all of 500 .. 3000 tokens 96 | 111 | 112 | 113; 56
// of 1 and 8 of 32 (4 blocks) on 4000 110 | 110 | 127 | 134; 200 of 2 and 56 of 18 (3), 100 .. 2048 200 | 200 | 282 | 279; 64 of 1 and one of 256 (32) on
// 40000 166 | 167 | 167 | 660; 256 of 4 (1) 189 | 189 | 188 | 186; 64 of 2 .. 10 (up to 2) at 4/2 heads 45.5 | 36.0 | 35.7 | 33.3.
constexpr int kSmMostBlocks = 2;

template <bool kCluster>
static int tree_configure() {
  static std::atomic<size_t> configured[kMaxDevices];
  return ensure_dynamic_smem(reinterpret_cast<const void*>(tree_attn_kernel<kCluster>), kTrSmem, configured, "tree_attn: cudaFuncSetAttribute");
}
static void tree_cluster_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, unsigned clusters, unsigned size, cudaStream_t stream) {
  cfg->gridDim = dim3(clusters * size);
  cfg->blockDim = dim3(kTrThreads);
  cfg->dynamicSmemBytes = kTrSmem;
  cfg->stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg->attrs = attr;
  cfg->numAttrs = 2;
}
// How many clusters of 8 >> i CTAs the current device holds at a time (0: not known).
static int tree_clusters_on_chip(int i) {
  static std::atomic<int> known[kMaxDevices][kTrClusterSizes];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  if ((n = known[dev][i].load(std::memory_order_acquire)) > 0) return n;
  if (tree_configure<true>()) return 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  tree_cluster_config(&cfg, attr, 1, kTrClusterMax >> i, nullptr);
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, tree_attn_kernel<true>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  known[dev][i].store(n, std::memory_order_release);
  return n;
}

// Workspace: the records of this kernel's pieces and of those of tree_small.cu, then two places of partial results per CTA for each.
constexpr int64_t kTrPiecesBytes = (sizeof(TreePieces) + 255) / 256 * 256;
static int64_t tree_workspace(int ctas) { return 2 * kTrPiecesBytes + static_cast<int64_t>(ctas) * 2 * (kTrPartial + kSmPartial) * 4; }

int launch_tree_join(const TreeParams& p, const TreeJoin& join, int ctas, cudaStream_t stream) {
  if (ctas < 2) return kOk;
  const cudaError_t le = launch_early(join.kernels > 1 ? tree_join_kernel<true> : tree_join_kernel<false>, ctas * kTrJoinCtas, kTrJoinThreads, 0, stream, p, join, ctas);
  g_launches.fetch_add(1);
  return check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "tree_attn join launch");
}

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
  p.scale_abs = scale == 0.f ? std::numeric_limits<float>::denorm_min() : std::fabs(p.scale_log2);
  p.negate = scale < 0.f ? tc::kIdescNegateA : 0u;
  const int grid = sm_count();
  if (grid > kTrMaxCtas) return set_error(kErrDevice, "tree_attn: more than %d multiprocessors", kTrMaxCtas);
  char* const ws = static_cast<char*>(workspace);
  p.above = 0;
  p.upto = INT_MAX;
  p.pieces = reinterpret_cast<TreePieces*>(ws);
  p.partials = reinterpret_cast<float*>(ws + 2 * kTrPiecesBytes);
  CUtensorMap map_q, map_k, map_v, map_k16, map_v16, map_k64, map_v64;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * block_size, row = static_cast<uint64_t>(num_kv_heads) * 128;
  int rc = make_tokens_heads_map(&map_q, q, static_cast<uint64_t>(total_q), num_heads, static_cast<uint64_t>(q_row_stride), 128 / G, G);
  if (!rc) rc = make_tokens_heads_map(&map_k, k_cache, rows, num_kv_heads, row, kTrKv);
  if (!rc) rc = make_tokens_heads_map(&map_v, v_cache, rows, num_kv_heads, row, kTrKv);
  if (!rc) rc = make_tokens_heads_map(&map_k16, k_cache, rows, num_kv_heads, row, 16);
  if (!rc) rc = make_tokens_heads_map(&map_v16, v_cache, rows, num_kv_heads, row, 16);
  if (rc) return rc;
  // few units: a cluster each, one launch
  const long long units = (static_cast<long long>(total_q) / (2 * (128 / G)) + batch) * num_kv_heads;
  for (int i = 0; i < kTrClusterSizes; ++i) {
    if (static_cast<long long>(bt_cols) * (block_size / kTrKv) > kTrClusterTiles[i] || units > tree_clusters_on_chip(i)) continue;
    rc = tree_configure<true>();
    if (rc) return rc;
    p.cluster_log = kTrClusterLog - i;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    tree_cluster_config(&cfg, attr, static_cast<unsigned>(units), 1u << p.cluster_log, static_cast<cudaStream_t>(stream));
    const cudaError_t le = cudaLaunchKernelEx(&cfg, tree_attn_kernel<true>, p, map_q, map_k, map_v, map_k16, map_v16);
    g_launches.fetch_add(1);
    return check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "tree_attn(cluster) launch");
  }
  // the longest that either kernel's line can be (table widths are all that the host knows of the lengths), in 31 bits
  const auto line = [&](int block_nodes, int keys, int tile, int unit) {
    return static_cast<double>(num_kv_heads) * (total_q / block_nodes + static_cast<double>(batch)) *
           (static_cast<double>(bt_cols) * (block_size / keys) * tile + unit);
  };
  if (line(2 * (128 / G), TcLine::kKeys, TcLine::kTilePair, TcLine::kUnitPair) >= 2147483648.0)
    return set_error(kErrBadShape, "tree_attn: %d sequences with tables of %d blocks are too many for one call", batch, bt_cols);
  const bool small_fits = G <= 16 && line(16 / G, SmLine::kKeys, SmLine::kTilePair, SmLine::kUnitPair) < 2147483648.0;
  TreeJoin join = {{{p.pieces, p.partials, kTrPartial}, {}}, 1};
  // Few nodes to a sequence: tree_small.cu, up to 12 rows on average.  Us of this kernel | that one with the launch behind it, calls on end in a graph:
  // 256 sequences of 100 .. 2048 tokens at 16/8 heads, 1 node 213 | 180, 4 nodes 212 to 226 | 190, 6 nodes (12 rows) 219 to 229 | 200, 8 nodes (16 rows)
  // 221 to 231 | 217, 12 nodes 238 | 398; 128 of 500 .. 4096 at 32/8, 1 node 209 | 192; 256 of 100 .. 1000 at 8/4, 3 .. 9 nodes (12 rows) 106 | 78; 64 of
  // 500 .. 3000 at 4/2, 3 nodes 32.2 | 30.5, 2 .. 10 nodes (12 rows) 32.2 | 35.4, 2 .. 14 nodes (16 rows) 31.8 | 38.5; 20 of 300 .. 2000 at 32/8, 3 nodes
  // (12 rows) 29.7 | 30.9, 4 nodes (16 rows) 29.9 | 33.4.  (Lengths are not known here, so some short calls pay 1 to 3 us for what long ones gain.)
  // A sequence has its keys read once for every 16 / G of its nodes there, so those with more than kSmMostBlocks times that are left to this kernel, in
  // a launch behind that one (which leaves at once where there are none).
  if (small_fits && static_cast<long long>(total_q) * G <= 12LL * batch) {
    rc = make_tokens_heads_map(&map_k64, k_cache, rows, num_kv_heads, row, 64);
    if (!rc) rc = make_tokens_heads_map(&map_v64, v_cache, rows, num_kv_heads, row, 64);
    TreeParams few = p;
    few.upto = kSmMostBlocks * (16 / G);
    few.pieces = reinterpret_cast<TreePieces*>(ws + kTrPiecesBytes);
    few.partials = p.partials + static_cast<int64_t>(grid) * 2 * kTrPartial;
    if (!rc) rc = launch_tree_small(few, map_k64, map_v64, map_k16, map_v16, grid, static_cast<cudaStream_t>(stream));
    if (rc) return rc;
    p.above = few.upto;
    join = {{{few.pieces, few.partials, kSmPartial}, join.of[0]}, total_q > p.above ? 2 : 1};
  }
  if (total_q > p.above) {
    rc = tree_configure<false>();
    if (rc) return rc;
    const cudaError_t le = launch_early(tree_attn_kernel<false>, grid, kTrThreads, kTrSmem, static_cast<cudaStream_t>(stream), p, map_q, map_k, map_v, map_k16, map_v16);
    g_launches.fetch_add(1);
    rc = check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "tree_attn launch");
    if (rc) return rc;
  }
  return launch_tree_join(p, join, grid, static_cast<cudaStream_t>(stream));
}
