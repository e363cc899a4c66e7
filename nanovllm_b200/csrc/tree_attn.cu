// Attention of drafted tokens over the paged cache: every sequence brings the nodes of a tree (or a chain), whose keys and values
// are already in the cache behind its context.  A node sees the context, and of the nodes those that its mask names.
//
// One CTA owns 64 rows of the (node, query head of the group) product of one sequence and kv head, 16 to a warp, so a K/V tile is
// loaded once for all of them.  K/V arrive as 64-token TMA tiles through a 4-stage mbarrier ring fed by a producer warp; the
// consumer warps run Q K^T, online softmax and P V in registers on mma.sync.
#include <atomic>

#include "../../include/b200_attn.h"
#include "tree_common.cuh"

namespace b200 {
extern std::atomic<long long> g_launches;

constexpr int kTaTile = 64;
constexpr int kTaSub = kTaTile * 128;
constexpr int kTaStageBytes = 4 * kTaSub;
constexpr int kTaStages = 4;
constexpr int kTaWarps = 4;
constexpr int kTaRows = 16 * kTaWarps;

static __device__ int g_status_tree = 0;

__global__ void __launch_bounds__(kTaWarps * 32 + 32, 1)
tree_attn_kernel(const TreeParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bar_full[kTaStages], bar_empty[kTaStages];
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.G;
  if (tid == 0) {
    s_abort = 0;
    for (int s = 0; s < kTaStages; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], kTaWarps);
    }
    mbar_fence_init();
  }
  // sequence i owns row tiles [cu_q[i] * G / 64 + i, ...)
  const int h = blockIdx.x % p.Hkv, x = static_cast<int>(blockIdx.x / p.Hkv);
  int seq = 0, hi = p.batch;
  while (hi - seq > 1) {
    const int mid = (seq + hi) >> 1;
    if (static_cast<int>(static_cast<long long>(p.cu_q[mid]) * G / kTaRows) + mid <= x) seq = mid; else hi = mid;
  }
  const int q_begin = max(p.cu_q[seq], 0), nodes = min(p.cu_q[seq + 1], p.total_q) - q_begin;
  const int rt = x - (static_cast<int>(static_cast<long long>(q_begin) * G / kTaRows) + seq);
  if (rt < 0 || nodes <= 0 || rt * kTaRows >= nodes * G) return;
  const int Lk = max(0, min(p.context_lens[seq], p.bt_cols * p.block_size)), first = Lk - nodes;    // position of node 0
  const int n_tiles = (Lk + kTaTile - 1) / kTaTile;
  __syncthreads();
  volatile int* abort_flag = &s_abort;

  if (warp == kTaWarps) {
    if (lane == 0) {
      const int* bt_row = p.block_tables + seq * p.bt_row_stride;
      for (int t = 0; t < n_tiles; ++t) {
        const int stage = t % kTaStages;
        if (!mbar_wait(&bar_empty[stage], ((t / kTaStages) & 1) ^ 1, abort_flag)) { atomicExch(&g_status_tree, 1); break; }
        const int tok0 = t * kTaTile, col = tok0 / p.block_size;
        const long long blk = bt_row[col];
        const int row0 = blk >= 0 && blk < p.num_blocks ? static_cast<int>(blk * p.block_size + (tok0 - col * p.block_size)) : -kTaTile;
        unsigned char* st = stages + stage * kTaStageBytes;
        mbar_expect_tx(&bar_full[stage], kTaStageBytes);
        tma_load_3d(st, &map_k, &bar_full[stage], 0, h, row0);
        tma_load_3d(st + kTaSub, &map_k, &bar_full[stage], 64, h, row0);
        tma_load_3d(st + 2 * kTaSub, &map_v, &bar_full[stage], 0, h, row0);
        tma_load_3d(st + 3 * kTaSub, &map_v, &bar_full[stage], 64, h, row0);
      }
    }
    return;
  }

  const int quad = lane & 3;
  const int r0 = rt * kTaRows + warp * 16 + (lane >> 2), r1 = r0 + 8;      // rows of the (node, head) product
  const int n0 = r0 / G, n1 = r1 / G;
  const bool ok0 = n0 < nodes, ok1 = n1 < nodes;
  const uint32_t* mask0 = p.masks && ok0 ? p.masks + static_cast<long long>(q_begin + n0) * p.mask_words : nullptr;
  const uint32_t* mask1 = p.masks && ok1 ? p.masks + static_cast<long long>(q_begin + n1) * p.mask_words : nullptr;
  uint32_t qa[8][4];
  {
    const uint32_t* q0 = reinterpret_cast<const uint32_t*>(p.q + static_cast<long long>(q_begin + n0) * p.q_row_stride + (h * G + r0 % G) * 128);
    const uint32_t* q1 = reinterpret_cast<const uint32_t*>(p.q + static_cast<long long>(q_begin + n1) * p.q_row_stride + (h * G + r1 % G) * 128);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      qa[ks][0] = ok0 ? ld_u32(q0 + ks * 8 + quad) : 0u;
      qa[ks][1] = ok1 ? ld_u32(q1 + ks * 8 + quad) : 0u;
      qa[ks][2] = ok0 ? ld_u32(q0 + ks * 8 + 4 + quad) : 0u;
      qa[ks][3] = ok1 ? ld_u32(q1 + ks * 8 + 4 + quad) : 0u;
    }
  }
  float o[16][4];
#pragma unroll
  for (int n = 0; n < 16; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

  for (int t = 0; t < n_tiles; ++t) {
    const int stage = t % kTaStages;
    if (!mbar_wait(&bar_full[stage], (t / kTaStages) & 1, abort_flag)) { if (lane == 0) atomicExch(&g_status_tree, 1); return; }
    const int key0 = t * kTaTile;
    if (key0 + kTaTile > Lk) {
      // ragged last tile: rows behind the sequence's end are foreign data; zero V there
      unsigned char* vb = stages + stage * kTaStageBytes + 2 * kTaSub;
      const int end = Lk - key0;
      for (int e = tid; e < (kTaTile - end) * 16; e += kTaWarps * 32) {
        const int r = end + (e >> 4), c = e & 15;
        *reinterpret_cast<uint4*>(vb + (c >> 3) * kTaSub + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
      }
      named_bar_sync(1, kTaWarps * 32);
    }
    const uint32_t st = smem_u32(stages + stage * kTaStageBytes);
    const uint32_t k_base = st, v_base = st + 2 * kTaSub;
    float s[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    {
      const int trow = ((lane >> 4) << 3) + (lane & 7);
      const int dsel = ((lane >> 3) & 1) << 3;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int j2 = 0; j2 < 4; ++j2) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4(k_base + tile_offset(j2 * 16 + trow, ks * 16 + dsel, kTaTile), b0, b1, b2, b3);
          mma_bf16_16816(s[2 * j2], qa[ks], b0, b1);
          mma_bf16_16816(s[2 * j2 + 1], qa[ks], b2, b3);
        }
    }
    uint32_t keep0[2] = {0xffffffffu, 0xffffffffu}, keep1[2] = {0xffffffffu, 0xffffffffu};
    if (key0 + kTaTile > first)                                             // the tile reaches the nodes
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int d = key0 + c * 32 - first, left = Lk - key0 - c * 32;
        keep0[c] = tree_keep32(mask0, p.mask_words, n0, d, left);
        keep1[c] = tree_keep32(mask1, p.mask_words, n1, d, left);
      }
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int bit = (j & 3) * 8 + quad * 2 + e;
        s[j][e] = (keep0[j >> 2] >> bit) & 1 ? s[j][e] * p.scale_log2 : -INFINITY;
        s[j][2 + e] = (keep1[j >> 2] >> bit) & 1 ? s[j][2 + e] * p.scale_log2 : -INFINITY;
        mx0 = fmaxf(mx0, s[j][e]);
        mx1 = fmaxf(mx1, s[j][2 + e]);
      }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
    const float ms0 = mn0 == -INFINITY ? 0.f : mn0, ms1 = mn1 == -INFINITY ? 0.f : mn1;
    const float a0 = fast_exp2(m0 - ms0), a1 = fast_exp2(m1 - ms1);
    m0 = mn0; m1 = mn1;
    float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[j][e] = fast_exp2(s[j][e] - ms0);
        s[j][2 + e] = fast_exp2(s[j][2 + e] - ms1);
        ps0 += s[j][e];
        ps1 += s[j][2 + e];
      }
    l0 = l0 * a0 + ps0;
    l1 = l1 * a1 + ps1;
#pragma unroll
    for (int n = 0; n < 16; ++n) { o[n][0] *= a0; o[n][1] *= a0; o[n][2] *= a1; o[n][3] *= a1; }
    {
      const int trow = (((lane >> 3) & 1) << 3) + (lane & 7);
      const int dsel = (lane >> 4) << 3;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t pa[4];
        pa[0] = pack_bf16(s[2 * kk][0], s[2 * kk][1]);
        pa[1] = pack_bf16(s[2 * kk][2], s[2 * kk][3]);
        pa[2] = pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]);
        pa[3] = pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
        for (int n2 = 0; n2 < 8; ++n2) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4_trans(v_base + tile_offset(kk * 16 + trow, n2 * 16 + dsel, kTaTile), b0, b1, b2, b3);
          mma_bf16_16816(o[2 * n2], pa, b0, b1);
          mma_bf16_16816(o[2 * n2 + 1], pa, b2, b3);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar_empty[stage]);
  }
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  const float inv0 = l0 > 0.f ? 1.f / l0 : 0.f, inv1 = l1 > 0.f ? 1.f / l1 : 0.f;      // nothing visible: zeros
  if (ok0) {
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + (static_cast<long long>(q_begin + n0) * p.H + h * G + r0 % G) * 128);
#pragma unroll
    for (int n = 0; n < 16; ++n) dst[n * 4 + quad] = pack_bf16(o[n][0] * inv0, o[n][1] * inv0);
  }
  if (ok1) {
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + (static_cast<long long>(q_begin + n1) * p.H + h * G + r1 % G) * 128);
#pragma unroll
    for (int n = 0; n < 16; ++n) dst[n * 4 + quad] = pack_bf16(o[n][2] * inv1, o[n][3] * inv1);
  }
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
  return 16;
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
  CUtensorMap map_k, map_v;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * block_size;
  int rc = make_tokens_heads_map(&map_k, k_cache, rows, num_kv_heads, static_cast<uint64_t>(num_kv_heads) * 128, kTaTile);
  if (rc) return rc;
  rc = make_tokens_heads_map(&map_v, v_cache, rows, num_kv_heads, static_cast<uint64_t>(num_kv_heads) * 128, kTaTile);
  if (rc) return rc;
  const size_t smem = 1024 + static_cast<size_t>(kTaStages) * kTaStageBytes;
  static std::atomic<size_t> configured[kMaxDevices];
  rc = ensure_dynamic_smem(reinterpret_cast<const void*>(tree_attn_kernel), smem, configured, "tree_attn: cudaFuncSetAttribute");
  if (rc) return rc;
  const long long blocks = (static_cast<long long>(total_q) * G / kTaRows + batch) * num_kv_heads;
  if (blocks > 0x7fffffffLL) return set_error(kErrBadShape, "tree_attn: too many query rows");
  tree_attn_kernel<<<static_cast<unsigned>(blocks), kTaWarps * 32 + 32, smem, static_cast<cudaStream_t>(stream)>>>(p, map_k, map_v);
  g_launches.fetch_add(1);
  return check_cuda(cudaGetLastError(), "tree_attn launch");
}
