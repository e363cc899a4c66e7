// What a step with drafted trees does behind the model: the walk along the sampled tokens, and the accepted nodes' cache rows to
// their places.
#include "../../include/b200_attn.h"
#include "kernels.cuh"

namespace b200 {
extern std::atomic<long long> g_launches;

// ---- the walk ------------------------------------------------------------------------------------------------------
// target[r] is what the target model sampled behind node r, so the path from the root along children whose drafted token equals
// their parent's sample is made of the target's own samples, at any temperature.  One warp per tree: the nodes' parents and
// tokens go to shared memory once, and each level is a ballot over the nodes behind the current one.  2.6 us for 13 trees, 3.9 for 512
// (launches on end in a graph): the launch and two trips to memory.
constexpr int kAcceptWarps = 4;
constexpr int kAcceptNodes = 256;        // nodes of a tree that are kept in shared memory; later ones are read where they lie

struct AcceptParams {
  const long long *draft, *target;
  const int *parents, *cu, *cached, *context;
  int batch, num_tokens, max_path;
  int *accepted, *path, *cached_out;
  long long* tokens;
};

__global__ void __launch_bounds__(kAcceptWarps * 32) accept_tree_kernel(const AcceptParams p) {
  __shared__ long long s_draft[kAcceptWarps][kAcceptNodes], s_target[kAcceptWarps][kAcceptNodes];
  __shared__ int s_parent[kAcceptWarps][kAcceptNodes];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x * kAcceptWarps + warp;
  if (i >= p.batch) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int start = max(0, min(p.cu[i], p.num_tokens)), nodes = max(0, min(p.cu[i + 1], p.num_tokens) - start);
  const int cached = p.cached[i];
  int count = 0;
  if (p.context[i] > 0 && nodes > 0) {
#pragma unroll 4
    for (int n = lane; n < min(nodes, kAcceptNodes); n += 32) {
      s_draft[warp][n] = p.draft[start + n];
      s_target[warp][n] = p.target[start + n];
      s_parent[warp][n] = p.parents[start + n];
    }
    __syncwarp();
    int cur = 0;
    while (true) {
      const long long want = cur < kAcceptNodes ? s_target[warp][cur] : p.target[start + cur];
      if (lane == 0) {
        p.path[static_cast<long long>(i) * p.max_path + count] = cur;
        p.tokens[static_cast<long long>(i) * p.max_path + count] = want;
      }
      if (++count == p.max_path) break;
      int next = -1;
      for (int base = (cur + 1) & ~31; base < nodes; base += 32) {       // children come behind their parent
        const int n = base + lane;
        bool hit = false;
        if (n > cur && n < nodes)
          hit = n < kAcceptNodes ? s_parent[warp][n] == cur && s_draft[warp][n] == want
                                 : p.parents[start + n] == cur && p.draft[start + n] == want;
        const unsigned found = __ballot_sync(0xffffffffu, hit);
        if (found) {
          next = base + __ffs(found) - 1;
          break;
        }
      }
      if (next < 0) break;
      cur = next;
    }
  }
  for (int k = count + lane; k < p.max_path; k += 32) {
    p.path[static_cast<long long>(i) * p.max_path + k] = -1;
    p.tokens[static_cast<long long>(i) * p.max_path + k] = -1;
  }
  if (lane == 0) {
    p.accepted[i] = count;
    p.cached_out[i] = cached + count;
  }
}

// ---- the cache ------------------------------------------------------------------------------------------------------
// Row start + path[k] of every plane goes to start + k.  Entries below their place (path[k] < k) are not moved, so a row that is
// written (k) is read by later moves only where path[k'] = k < k', which that excludes: a thread may have the loads of
// several moves in flight, and keeps to one 16-byte column of a row.  A few MB at most move, so what counts is the way there: lengths
// and path, then the table, then the rows, a round trip each.  Every warp goes it by itself, a move to a lane: no shared memory, no
// barrier (with a list of the moves in shared memory 3.35 and 7.06 us where this takes 2.8 and 6.1).  2.5 us for 5 sequences (2.5 MB), 5.7 for 128
// (22 MB, 3.9 TB/s), started early.
constexpr int kCompactThreads = 256;

struct CompactParams {
  char* cache;
  long long plane_stride, row_bytes;
  unsigned vecs;                         // 16-byte columns of a row
  unsigned columns;                      // of all planes
  int num_blocks, block_size;
  const int *path, *accepted, *start, *block_tables;
  int path_cols;
  long long bt_row_stride;
  int bt_cols;
};

__device__ __forceinline__ long long compact_row(const CompactParams& p, const int* table, int at) {
  const int col = at / p.block_size;
  if (at < 0 || col >= p.bt_cols) return -1;
  const int id = table[col];
  return id >= 0 && id < p.num_blocks ? static_cast<long long>(id) * p.block_size + (at - col * p.block_size) : -1;
}

__global__ void __launch_bounds__(kCompactThreads) compact_kvcache_kernel(const CompactParams p) {
  const int i = blockIdx.y, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int* const table = p.block_tables + i * p.bt_row_stride;
  const int* const path = p.path + static_cast<long long>(i) * p.path_cols;
  int node = lane < p.path_cols ? path[lane] : -1;
  const int start = p.start[i], n = min(p.accepted[i], p.path_cols);
  const unsigned column = blockIdx.x * kCompactThreads + threadIdx.x;
  const bool live = column < p.columns;
  const unsigned plane = column / p.vecs;
  char* const mine = p.cache + plane * p.plane_stride + (column - plane * p.vecs) * 16;
  for (int base = 0; base < n; base += 32) {
    const int k = base + lane;
    if (base > 0) node = k < n ? path[k] : -1;
    long long src = -1, dst = -1;
    if (k < n && start >= 0 && node > k && node <= 0x7fffffff - start) {
      src = compact_row(p, table, start + node);
      dst = compact_row(p, table, start + k);
    }
    unsigned moves = __ballot_sync(0xffffffffu, src >= 0 && dst >= 0);
    src *= p.row_bytes;
    dst *= p.row_bytes;
    while (moves) {
      uint4 v[8];
      long long to[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int from = __ffs(moves) - 1;             // (-1: none left)
        moves &= moves - 1;
        const long long at = __shfl_sync(0xffffffffu, src, from & 31);
        to[u] = from >= 0 ? __shfl_sync(0xffffffffu, dst, from & 31) : -1;
        if (live && from >= 0) v[u] = *reinterpret_cast<const uint4*>(mine + at);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (live && to[u] >= 0) *reinterpret_cast<uint4*>(mine + to[u]) = v[u];
    }
  }
}

}  // namespace b200

extern "C" int b200_accept_tree(const int64_t* draft_tokens, const int64_t* target_tokens, const int32_t* parents,
                                const int32_t* cu_seqlens_q, const int32_t* cached_lens, const int32_t* context_lens, int32_t batch,
                                int32_t num_tokens, int32_t max_path, int32_t* accepted, int32_t* path, int64_t* tokens,
                                int32_t* new_cached_lens, void* stream) {
  using namespace b200;
  if (batch < 0 || num_tokens < 0 || max_path < 1) return set_error(kErrBadShape, "accept_tree: batch (%d) and num_tokens (%d) must not be negative, max_path (%d) at least 1", batch, num_tokens, max_path);
  if (batch == 0) return kOk;
  if (!cu_seqlens_q || !cached_lens || !context_lens || !accepted || !path || !tokens || !new_cached_lens ||
      (num_tokens > 0 && (!draft_tokens || !target_tokens || !parents)))
    return set_error(kErrNullPointer, "accept_tree: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(draft_tokens) | reinterpret_cast<uintptr_t>(target_tokens) | reinterpret_cast<uintptr_t>(tokens)) & 7)
    return set_error(kErrMisaligned, "accept_tree: tokens must be 8-byte aligned");
  AcceptParams p;
  p.draft = reinterpret_cast<const long long*>(draft_tokens);
  p.target = reinterpret_cast<const long long*>(target_tokens);
  p.parents = parents;
  p.cu = cu_seqlens_q;
  p.cached = cached_lens;
  p.context = context_lens;
  p.batch = batch;
  p.num_tokens = num_tokens;
  p.max_path = max_path;
  p.accepted = accepted;
  p.path = path;
  p.cached_out = new_cached_lens;
  p.tokens = reinterpret_cast<long long*>(tokens);
  const cudaError_t le = launch_early(accept_tree_kernel, (static_cast<unsigned>(batch) + kAcceptWarps - 1) / kAcceptWarps, kAcceptWarps * 32, 0,
                                      static_cast<cudaStream_t>(stream), p);
  g_launches.fetch_add(1);
  return check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "accept_tree launch");
}

extern "C" int b200_compact_kvcache(void* cache, int32_t planes, int64_t plane_stride_bytes, int64_t row_bytes, int64_t num_blocks,
                                    int32_t block_size, const int32_t* path, int32_t path_cols, const int32_t* accepted,
                                    const int32_t* start_lens, const int32_t* block_tables, int64_t bt_row_stride, int32_t bt_cols,
                                    int32_t batch, void* stream) {
  using namespace b200;
  if (batch < 0 || batch > 65535 || planes < 0 || path_cols < 0) return set_error(kErrBadShape, "compact_kvcache: batch must be in [0, 65535], planes and path_cols not negative (got %d, %d, %d)", batch, planes, path_cols);
  if (batch == 0 || planes == 0 || path_cols <= 1) return kOk;
  if (!cache || !path || !accepted || !start_lens || !block_tables) return set_error(kErrNullPointer, "compact_kvcache: null pointer argument");
  if (block_size <= 0 || num_blocks <= 0 || num_blocks * block_size >= (1LL << 31)) return set_error(kErrBadShape, "compact_kvcache: num_blocks * block_size must be in (0, 2^31)");
  if (bt_cols <= 0 || bt_row_stride < bt_cols) return set_error(kErrBadShape, "compact_kvcache: bad block table geometry");
  if (row_bytes <= 0 || row_bytes > (1 << 20) || plane_stride_bytes < num_blocks * block_size * row_bytes) return set_error(kErrBadShape, "compact_kvcache: rows of 1 to 2^20 bytes, planes that do not overlap");
  if ((reinterpret_cast<uintptr_t>(cache) | row_bytes | plane_stride_bytes) & 15) return set_error(kErrMisaligned, "compact_kvcache: cache, rows and planes must be multiples of 16 bytes");
  const long long columns = planes * (row_bytes / 16);
  if (columns >= 0x7fffffffLL) return set_error(kErrBadShape, "compact_kvcache: too many planes");
  CompactParams p;
  p.cache = static_cast<char*>(cache);
  p.plane_stride = plane_stride_bytes;
  p.row_bytes = row_bytes;
  p.vecs = static_cast<unsigned>(row_bytes / 16);
  p.columns = static_cast<unsigned>(columns);
  p.num_blocks = static_cast<int>(num_blocks);
  p.block_size = block_size;
  p.path = path;
  p.accepted = accepted;
  p.start = start_lens;
  p.block_tables = block_tables;
  p.path_cols = path_cols;
  p.bt_row_stride = bt_row_stride;
  p.bt_cols = bt_cols;
  const unsigned blocks = (p.columns + kCompactThreads - 1) / kCompactThreads;
  const cudaError_t le = launch_early(compact_kvcache_kernel, dim3(blocks, static_cast<unsigned>(batch)), kCompactThreads, 0,
                                      static_cast<cudaStream_t>(stream), p);
  g_launches.fetch_add(1);
  return check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "compact_kvcache launch");
}
