// Tree attention for sequences with few nodes: up to 16 rows (nodes x query heads of the group) to a unit, on mma.sync.
//
// The tcgen05 kernel (tree_attn.cu) multiplies 128 rows whatever the number of nodes.  That costs less time than the bytes take, but
// a third of the power: at 8 rows it ran into the 1000 W cap and at 1500 MHz.  Here the tensor core works on 16 rows, and
// what bounds it is HBM.
//
// One persistent CTA per SM takes its share of the line of all units' key tiles (64 keys); a unit is (sequence, block of 16 / G
// nodes, kv head).  A producer thread feeds a ring of 6 stages (K and V of a tile, 32 KB, through TMA).  8 consumer warps in two
// groups take the tiles in turn, 16 keys of a tile to a warp: a byte of shared memory is read by one warp only.  At the end of
// a unit a group leaves its accumulators in the stage of its last tile, which goes back to the ring when the epilogue warps have
// joined them: the consumers go on with the next unit meanwhile, and the room costs nothing.
//
// 256 chains of 4 nodes on 100 .. 2048 tokens at 16/8 heads: 188 us with the launch for large trees and the join, 6.0 TB/s (a copy: 6.55); 1 node 180.
#include <atomic>

#include "../../include/b200_attn.h"
#include "tree_common.cuh"

namespace b200 {
extern std::atomic<long long> g_launches;

constexpr int kSmSub = 64 * 128;                 // 64 keys x 64 dims bf16
constexpr int kSmStage = 4 * kSmSub;             // K lo, K hi, V lo, V hi
constexpr int kSmStages = 6;
constexpr int kSmItems = 4;
constexpr int kSmProducer = 8, kSmEpilogue = 9;  // warps: 0-3 and 4-7 consumers, 9-11 epilogue (with 13 warps a scheduler had four, and
constexpr int kSmThreads = 12 * 32;              // each only 128 registers)
constexpr int kSmQRow = 256 + 16, kSmQ = 16 * kSmQRow;      // a unit's rows, apart by 4 banks
static __device__ int g_status_tree_small = 0;

struct SmallItem {
  int seq;              // -1: no more work
  int h, q_row, node0, nodes;
  int first, Lk;        // position of the sequence's node 0; its keys
  int t0, n;            // key tiles of this piece
  int count;            // tiles of the CTA in front of it
  int partial;          // -1: the whole unit, else where its partial results go
};

// A consumer warp's running state: rows lane / 4 and lane / 4 + 8.
struct SmallAcc {
  float o[16][4];
  float m0, m1, l0, l1;
};

// One warp's 16 keys of a tile in shared memory: S = Q K^T, mask, online softmax in the log2 domain, O += P V.  keep0, keep1: which of
// the 16 keys the thread's two rows see; valid: how many of them the sequence has.
__device__ __forceinline__ void small_tile(unsigned char* stage, int slab, int lane, int valid, uint32_t keep0, uint32_t keep1, float scale_log2,
                                           const uint32_t (&qa)[8][4], SmallAcc& a) {
  const int quad = lane & 3;
  const uint32_t k_base = smem_u32(stage), v_base = k_base + 2 * kSmSub;
  if (valid < 16) {
    // V rows behind the sequence's end are stale or foreign: zero, so that 0 * garbage cannot turn into NaN
    unsigned char* const vb = stage + 2 * kSmSub;
#pragma unroll 1
    for (int e = lane; e < 16 * 16; e += 32) {
      const int r = slab * 16 + (e >> 4), c = e & 15;
      if ((e >> 4) >= valid) *reinterpret_cast<uint4*>(vb + (c >> 3) * kSmSub + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
    __syncwarp();
  }
  float s[2][4];
#pragma unroll
  for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
  {
    const int tok = slab * 16 + ((lane >> 4) << 3) + (lane & 7), dsel = ((lane >> 3) & 1) << 3;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t b0, b1, b2, b3;
      ldmatrix_x4(k_base + tile_offset(tok, ks * 16 + dsel, 64), b0, b1, b2, b3);
      mma_bf16_16816(s[0], qa[ks], b0, b1);
      mma_bf16_16816(s[1], qa[ks], b2, b3);
    }
  }
  float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int bit = j * 8 + quad * 2 + e;
      s[j][e] = (keep0 >> bit) & 1 ? s[j][e] * scale_log2 : -INFINITY;
      s[j][2 + e] = (keep1 >> bit) & 1 ? s[j][2 + e] * scale_log2 : -INFINITY;
      mx0 = fmaxf(mx0, s[j][e]);
      mx1 = fmaxf(mx1, s[j][2 + e]);
    }
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
  const float mn0 = fmaxf(a.m0, mx0), mn1 = fmaxf(a.m1, mx1);
  const float ms0 = mn0 == -INFINITY ? 0.f : mn0, ms1 = mn1 == -INFINITY ? 0.f : mn1;
  const float a0 = fast_exp2(a.m0 - ms0), a1 = fast_exp2(a.m1 - ms1);
  a.m0 = mn0;
  a.m1 = mn1;
  float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      s[j][e] = fast_exp2(s[j][e] - ms0);
      s[j][2 + e] = fast_exp2(s[j][2 + e] - ms1);
      ps0 += s[j][e];
      ps1 += s[j][2 + e];
    }
  a.l0 = a.l0 * a0 + ps0;
  a.l1 = a.l1 * a1 + ps1;
  if (a0 != 1.f || a1 != 1.f) {
#pragma unroll
    for (int n = 0; n < 16; ++n) { a.o[n][0] *= a0; a.o[n][1] *= a0; a.o[n][2] *= a1; a.o[n][3] *= a1; }
  }
  // (P rounded to bf16 as the product takes it; the sum is of the unrounded ones)
  const uint32_t pa[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
  const int tok = slab * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), dsel = (lane >> 4) << 3;
#pragma unroll
  for (int n2 = 0; n2 < 8; ++n2) {
    uint32_t b0, b1, b2, b3;
    ldmatrix_x4_trans(v_base + tile_offset(tok, n2 * 16 + dsel, 64), b0, b1, b2, b3);
    mma_bf16_16816(a.o[2 * n2], pa, b0, b1);
    mma_bf16_16816(a.o[2 * n2 + 1], pa, b2, b3);
  }
}

__global__ void __launch_bounds__(kSmThreads, 1)
tree_small_kernel(const TreeParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ CUtensorMap map_k16, const __grid_constant__ CUtensorMap map_v16) {
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* const stages = smem;                               // [kSmStages][32 KiB]
  unsigned char* const sQ = smem + kSmStages * kSmStage;            // [2][4 KiB]
  __shared__ __align__(8) uint64_t bar_full[kSmStages], bar_empty[kSmStages];
  __shared__ __align__(8) uint64_t bar_item_full[kSmItems], bar_item_empty[kSmItems], bar_q_full[2], bar_q_empty[2];
  __shared__ __align__(8) uint64_t bar_state_full[2], bar_state_free[2], bar_read[2];
  __shared__ float s_ml[8][16][2];                                  // consumer warps' maxima (log2 units) and sums
  __shared__ __align__(16) SmallItem s_item[kSmItems];
  __shared__ unsigned s_scan[kSmThreads / 32];
  __shared__ int s_at[2][3];
  __shared__ int s_abort, s_bare;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.G, block_nodes = 16 / p.G;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    s_abort = 0;
    s_bare = 0;
    for (int i = 0; i < kSmStages; ++i) { mbar_init(&bar_full[i], 1); mbar_init(&bar_empty[i], 4); }
    for (int i = 0; i < kSmItems; ++i) { mbar_init(&bar_item_full[i], 1); mbar_init(&bar_item_empty[i], 11); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_q_full[i], 1);
      mbar_init(&bar_q_empty[i], 8);
      mbar_init(&bar_state_full[i], 4);
      mbar_init(&bar_state_free[i], 3);
      mbar_init(&bar_read[i], 4);
    }
    mbar_fence_init();
    s_at[0][0] = s_at[1][0] = p.batch;
    s_at[0][1] = s_at[0][2] = s_at[1][1] = s_at[1][2] = 0;
  }
  __syncthreads();
  tree_share<SmLine, kSmThreads>(p, block_nodes, s_scan, s_at, &s_bare);
  __syncthreads();
  volatile int* abort_flag = &s_abort;

  if (warp == kSmProducer) {
    if (lane != 0) return;
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
    int cont = 0, head = 0;
    int2 head_unit = make_int2(0, 0);
    int seq = s_at[0][0], unit = s_at[0][1], from = s_at[0][2], have = -1;
    TreeSeq s = {};
    TreeRows<SmLine> rows = {};
    const int end_seq = s_at[1][0], end_unit = s_at[1][1], end_tile = s_at[1][2];
    int n_pub = 0, count = 0, stage = 0, ph = 1;
    bool ok = true, started = false;
#pragma unroll 1
    while (ok && seq < p.batch) {
      if (have != seq) {
        s = tree_seq<SmLine>(p, block_nodes, seq);
        have = seq;
      }
      if (unit >= s.blocks * p.Hkv) {
        seq = seq < end_seq ? seq + 1 : p.batch;
        unit = from = 0;
        continue;
      }
      const bool at_end = seq == end_seq && unit >= end_unit;
      const int t0 = from, t1 = !at_end ? s.tiles : unit == end_unit ? max(end_tile, from) : from;
      const int block = unit / p.Hkv, h = unit - block * p.Hkv, node0 = block * block_nodes, nodes = min(block_nodes, s.nodes - node0);
      const int owner = seq, q_row = s.q_begin + node0;
      ++unit;
      from = 0;
      if (at_end) seq = p.batch;
      if (t0 == t1) continue;
      const bool whole = t0 == 0 && t1 == s.tiles;
      if (t0 > 0) {
        cont = t1 < s.tiles ? 1 : 2;
      } else if (!whole) {
        head = nodes;
        head_unit = make_int2(q_row, h);
      }
      const int is = n_pub % kSmItems;
      if (!mbar_wait(&bar_item_empty[is], ((n_pub / kSmItems) & 1) ^ 1, abort_flag)) { ok = false; break; }
      s_item[is] = {owner, h, q_row, node0, nodes, s.Lk - s.nodes, s.Lk, t0, t1 - t0, count, whole ? -1 : 2 * static_cast<int>(blockIdx.x) + (t0 > 0 ? 0 : 1)};
      mbar_arrive(&bar_item_full[is]);
      rows.start(p, owner, t0);
      int left = s.Lk - t0 * SmLine::kKeys;
#pragma unroll 1
      for (int t = t0; t < t1; ++t, left -= SmLine::kKeys) {
        const int row = rows.next(p);
        if (!started) {
          // everything so far overlaps the end of the kernel in front: lengths and tables, which it does not write
          for (int x = 0; x < 128; x += 64) {
            tma_prefetch_l2_3d(&map_k, x, h, row);
            tma_prefetch_l2_3d(&map_v, x, h, row);
          }
          asm volatile("griddepcontrol.wait;" ::: "memory");
          started = true;
        }
        if (!mbar_wait(&bar_empty[stage], ph, abort_flag)) { ok = false; break; }
        unsigned char* const st = stages + stage * kSmStage;
        uint64_t* const full = &bar_full[stage];
        if (left > SmLine::kKeys - 16) {
          mbar_expect_tx(full, kSmStage);
          tma_load_3d(st, &map_k, full, 0, h, row);
          tma_load_3d(st + kSmSub, &map_k, full, 64, h, row);
          tma_load_3d(st + 2 * kSmSub, &map_v, full, 0, h, row);
          tma_load_3d(st + 3 * kSmSub, &map_v, full, 64, h, row);
        } else {
          // the sequence's last tile: only what it has of it, in boxes of 16 keys
          const int boxes = (left + 15) >> 4;
          mbar_expect_tx(full, boxes * 8192);
#pragma unroll 1
          for (int b = 0; b < boxes; ++b) {
            tma_load_3d(st + b * 2048, &map_k16, full, 0, h, row + b * 16);
            tma_load_3d(st + kSmSub + b * 2048, &map_k16, full, 64, h, row + b * 16);
            tma_load_3d(st + 2 * kSmSub + b * 2048, &map_v16, full, 0, h, row + b * 16);
            tma_load_3d(st + 3 * kSmSub + b * 2048, &map_v16, full, 64, h, row + b * 16);
          }
        }
        if (++stage == kSmStages) { stage = 0; ph ^= 1; }
        if (t == t0) {
          // the unit's rows
          const int b = n_pub & 1;
          if (!mbar_wait(&bar_q_empty[b], ((n_pub >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&bar_q_full[b], nodes * G * 256);
#pragma unroll 1
          for (int x = 0, r = 0; x < nodes; ++x) {
            const __nv_bfloat16* const from = p.q + static_cast<long long>(q_row + x) * p.q_row_stride + h * G * 128;
#pragma unroll 1
            for (int g = 0; g < G; ++g, ++r) tree_bulk_load(sQ + b * kSmQ + r * kSmQRow, from + g * 128, 256, &bar_q_full[b]);
          }
        }
      }
      count += t1 - t0;
      ++n_pub;
    }
    if (!started) asm volatile("griddepcontrol.wait;" ::: "memory");
    p.pieces->of[blockIdx.x] = make_int4(head, cont, head_unit.x, head_unit.y);
    if (ok) {
      const int is = n_pub % kSmItems;
      if (mbar_wait(&bar_item_empty[is], ((n_pub / kSmItems) & 1) ^ 1, abort_flag)) {
        s_item[is].seq = -1;
        mbar_arrive(&bar_item_full[is]);
      }
    }
    if (s_abort) atomicExch(&g_status_tree_small, 1);
    return;
  }

  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp < kSmProducer) {
    // ================================ consumers ================================
    const int group = warp >> 2, slab = warp & 3;
    const int r0 = lane >> 2, quad = lane & 3;
    const int n0 = r0 / G, n1 = (r0 + 8) / G;           // nodes of the thread's rows
    int n_item = 0, n_state = 0;
    SmallAcc a;
#pragma unroll 1
    while (true) {
      const int is = n_item % kSmItems;
      if (!mbar_wait(&bar_item_full[is], (n_item / kSmItems) & 1, abort_flag)) break;
      const SmallItem it = s_item[is];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_item_empty[is]);
      if (it.seq < 0) break;
      const int qb = n_item & 1;
      if (!mbar_wait(&bar_q_full[qb], (n_item >> 1) & 1, abort_flag)) break;
      const bool ok0 = n0 < it.nodes && r0 < it.nodes * G, ok1 = n1 < it.nodes && r0 + 8 < it.nodes * G;
      uint32_t qa[8][4];
      {
        const uint32_t* const q0 = reinterpret_cast<const uint32_t*>(sQ + qb * kSmQ + r0 * kSmQRow);
        const uint32_t* const q1 = q0 + 8 * kSmQRow / 4;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          qa[ks][0] = ok0 ? q0[ks * 8 + quad] : 0u;
          qa[ks][1] = ok1 ? q1[ks * 8 + quad] : 0u;
          qa[ks][2] = ok0 ? q0[ks * 8 + 4 + quad] : 0u;
          qa[ks][3] = ok1 ? q1[ks * 8 + 4 + quad] : 0u;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_q_empty[qb]);
      ++n_item;
      const uint32_t* const mask0 = p.masks && ok0 ? p.masks + static_cast<long long>(it.q_row + n0) * p.mask_words : nullptr;
      const uint32_t* const mask1 = p.masks && ok1 ? p.masks + static_cast<long long>(it.q_row + n1) * p.mask_words : nullptr;
#pragma unroll
      for (int n = 0; n < 16; ++n) a.o[n][0] = a.o[n][1] = a.o[n][2] = a.o[n][3] = 0.f;
      a.m0 = a.m1 = -INFINITY;
      a.l0 = a.l1 = 0.f;
      int last = -1;
      bool gave_up = false;
#pragma unroll 1
      for (int j = (it.count ^ group) & 1; j < it.n; j += 2) {
        const int at = it.count + j, stage = at % kSmStages;
        if (!mbar_wait(&bar_full[stage], (at / kSmStages) & 1, abort_flag)) { gave_up = true; break; }
        const int key0 = (it.t0 + j) * SmLine::kKeys + slab * 16, valid = it.Lk - key0;
        if (valid > 0) {
          uint32_t keep0 = 0xffffu, keep1 = 0xffffu;
          if (key0 + 16 > min(it.first, it.Lk)) {
            const int d = key0 - it.first;
            keep0 = p.masks && !ok0 ? 0u : tree_keep32(mask0, p.mask_words, it.node0 + n0, d, valid);
            keep1 = p.masks && !ok1 ? 0u : tree_keep32(mask1, p.mask_words, it.node0 + n1, d, valid);
          }
          small_tile(stages + stage * kSmStage, slab, lane, valid, keep0, keep1, p.scale_log2, qa, a);
        }
        __syncwarp();
        if (j + 2 < it.n) {
          if (lane == 0) mbar_arrive(&bar_empty[stage]);
        } else {
          if (lane == 0) mbar_arrive(&bar_read[group]);
          last = stage;
        }
      }
      if (gave_up) break;
      if (last < 0) continue;
      // The group's accumulators into the stage of its last tile, which every warp of it has read; maxima and sums where the
      // epilogue has taken the last unit's.
      a.l0 += __shfl_xor_sync(0xffffffffu, a.l0, 1);
      a.l0 += __shfl_xor_sync(0xffffffffu, a.l0, 2);
      a.l1 += __shfl_xor_sync(0xffffffffu, a.l1, 1);
      a.l1 += __shfl_xor_sync(0xffffffffu, a.l1, 2);
      if (!mbar_wait(&bar_state_free[group], (n_state & 1) ^ 1, abort_flag)) break;
      if (!mbar_wait(&bar_read[group], n_state & 1, abort_flag)) break;
      // ([16 rows][128 dims], groups of 8 dims in another order in each row, so that a store meets no bank twice)
      float* const state = reinterpret_cast<float*>(stages + last * kSmStage + slab * kSmSub);
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        *reinterpret_cast<float2*>(state + r0 * 128 + ((n ^ r0) * 8) + quad * 2) = make_float2(a.o[n][0], a.o[n][1]);
        *reinterpret_cast<float2*>(state + (r0 + 8) * 128 + ((n ^ r0) * 8) + quad * 2) = make_float2(a.o[n][2], a.o[n][3]);
      }
      if (quad == 0) {
        s_ml[warp][r0][0] = a.m0;
        s_ml[warp][r0][1] = a.l0;
        s_ml[warp][r0 + 8][0] = a.m1;
        s_ml[warp][r0 + 8][1] = a.l1;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_state_full[group]);
      ++n_state;
    }
    if (*abort_flag) atomicExch(&g_status_tree_small, 1);
    return;
  }

  // ================================ epilogue ================================
  const int ew = warp - kSmEpilogue;                     // rows ew, ew + 3, ..
  if (s_bare) {
    // sequences with nodes and no keys: zeros
#pragma unroll 1
    for (int i = blockIdx.x; i < p.batch; i += gridDim.x) {
      const TreeSeq s = tree_seq<SmLine>(p, block_nodes, i);
      if (s.tiles > 0) continue;
      uint4* const dst = reinterpret_cast<uint4*>(p.out + static_cast<long long>(s.q_begin) * p.H * 128);
      for (long long e = ew * 32 + lane; e < static_cast<long long>(s.nodes) * p.H * 16; e += 96) dst[e] = make_uint4(0, 0, 0, 0);
    }
  }
  int n_item = 0, n_state[2] = {0, 0};
#pragma unroll 1
  while (true) {
    const int is = n_item % kSmItems;
    if (!mbar_wait(&bar_item_full[is], (n_item / kSmItems) & 1, abort_flag)) break;
    const SmallItem it = s_item[is];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar_item_empty[is]);
    if (it.seq < 0) break;
    ++n_item;
    // last tiles of the groups: n - 1 and n - 2
    const int at1 = it.count + it.n - 1, groups = min(it.n, 2);
    int stage[2];
    bool gave_up = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (x >= groups) continue;
      const int g = (at1 - x) & 1;
      stage[x] = (at1 - x) % kSmStages;
      if (!mbar_wait(&bar_state_full[g], (g ? n_state[1] : n_state[0]) & 1, abort_flag)) { gave_up = true; break; }
      if (g) ++n_state[1]; else ++n_state[0];
    }
    if (gave_up) break;
    const int rows = it.nodes * G;
#pragma unroll 1
    for (int r = ew; r < rows; r += 3) {
      // lane x < 8: state of consumer warp x
      const int g_of = (lane >> 2) & 1;
      const bool there = lane < 8 && (groups == 2 || g_of == (at1 & 1));
      const float m = there ? s_ml[lane][r][0] : -INFINITY, l = there ? s_ml[lane][r][1] : 0.f;
      float M = m;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      M = __shfl_sync(0xffffffffu, M, 0);
      const float w = M == -INFINITY ? 0.f : fast_exp2(m - M);
      float sum = l * w;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      sum = __shfl_sync(0xffffffffu, sum, 0);
      float4 o4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x >= groups) continue;
        const int g = (at1 - x) & 1;
#pragma unroll
        for (int sl = 0; sl < 4; ++sl) {
          const float ws = __shfl_sync(0xffffffffu, w, g * 4 + sl);
          const float4 v = *reinterpret_cast<const float4*>(stages + stage[x] * kSmStage + sl * kSmSub + r * 512 + ((lane >> 1) ^ (r & 7)) * 32 + (lane & 1) * 16);
          o4.x = fmaf(v.x, ws, o4.x);
          o4.y = fmaf(v.y, ws, o4.y);
          o4.z = fmaf(v.z, ws, o4.z);
          o4.w = fmaf(v.w, ws, o4.w);
        }
      }
      if (it.partial < 0) {
        const float inv = sum > 0.f ? 1.f / sum : 0.f;      // (a row that sees nothing: zeros)
        const int t = r / G;
        *reinterpret_cast<uint2*>(p.out + (static_cast<long long>(it.q_row + t) * p.H + it.h * G + (r - t * G)) * 128 + lane * 4) =
            make_uint2(pack_bf16(o4.x * inv, o4.y * inv), pack_bf16(o4.z * inv, o4.w * inv));
      } else {
        float* const part = p.partials + static_cast<long long>(it.partial) * kSmPartial + r;
        part[(lane * 4) * 32] = o4.x;
        part[(lane * 4 + 1) * 32] = o4.y;
        part[(lane * 4 + 2) * 32] = o4.z;
        part[(lane * 4 + 3) * 32] = o4.w;
        if (lane == 0) {
          part[128 * 32] = M;
          part[129 * 32] = sum;
        }
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x >= groups) continue;
        mbar_arrive(&bar_empty[stage[x]]);
        if (ew == 0) mbar_arrive(&bar_empty[stage[x]]);       // (a stage wants four arrivals)
        mbar_arrive(&bar_state_free[(at1 - x) & 1]);
      }
    }
  }
  if (*abort_flag) atomicExch(&g_status_tree_small, 1);
}

int launch_tree_small(const TreeParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, const CUtensorMap& map_k16, const CUtensorMap& map_v16,
                      int ctas, cudaStream_t stream) {
  constexpr size_t smem = kSmStages * kSmStage + 2 * kSmQ;
  static std::atomic<size_t> configured[kMaxDevices];
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(tree_small_kernel), smem, configured, "tree_attn(small): cudaFuncSetAttribute");
  if (rc) return rc;
  const cudaError_t le = launch_early(tree_small_kernel, ctas, kSmThreads, smem, stream, p, map_k, map_v, map_k16, map_v16);
  g_launches.fetch_add(1);
  return check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "tree_attn(small) launch");
}

int read_status_tree_small() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_status_tree_small, sizeof(int));
  return v;
}
int reset_state_tree_small() {
  const int zero = 0;
  return check_cuda(cudaMemcpyToSymbol(g_status_tree_small, &zero, sizeof(int)), "device_status: clearing the tree attention (small) status word");
}

}  // namespace b200
