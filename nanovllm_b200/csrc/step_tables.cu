// A step's tables from request lengths, on the GPU: blocks out of the free list, block-table rows, slots, positions, cumulative
// lengths and, for a step that brings drafted trees, each node's ancestors; and the way back, blocks into the free list.
//
// The reference keeps its free list and its tables in Python (nanovllm/engine/block_manager.py:26-112) and prepares a step on
// the host (nanovllm/engine/model_runner.py:119-179).  Where the lengths are known on the GPU only (what the walk through a
// drafted tree accepts is), that costs a round trip; here they never leave it.
//
// With need_i = ceil((cached_i + new_i) / block_size), want_i = max(0, need_i - owned_i) and E_i the sum of want_j over j < i,
// sequence i's j-th new block is free[n - 1 - (E_i + j)]: the list is a stack, and giving the same blocks back in the same order
// leaves it as it was.  A few KB move, so the time is that of the dependent steps (lengths -> owned -> scan -> ids -> slots):
// one cluster of 8 CTAs does all of them.  Each CTA scans the whole batch for itself and fills an eighth of the outputs; the
// cluster's barrier stands between the last read of the old state and the first write of the new one.  Us for 512 decodes, 40 prompts
// and 96 trees, launches on end in a graph: 1 CTA 9.3, 24.6, 24.6; 2 CTAs 7.3, 16.2, 14.9; 4 6.3, 10.5, 9.9; 8 5.9, 7.5, 7.3, and started
// early 5.6, 7.1, 6.6 (release 2.3).  Of the 4.9 on the device for the decodes 1.1 are the hash of the rows, 1.5 the two sums; of
// the 5.9 for prompts 3.5 the tokens (four of a thread's tokens at a time: the same).
#include <climits>

#include "../../include/b200_attn.h"
#include "kernels.cuh"

namespace b200 {
extern std::atomic<long long> g_launches;

constexpr int kStepThreads = 512;
constexpr int kStepCtas = 8;
constexpr int kStepMaxBatch = 4096;      // what the scan keeps in shared memory
constexpr int kStepMaxWords = 4;         // trees of up to 256 nodes

struct StepParams {
  const int *rows, *cached, *fresh, *parents;      // rows, parents: may be null
  int batch, num_tokens, block_size;
  int* tables;
  long long table_stride;
  int table_cols, max_requests, num_blocks;
  int *owned, *free_blocks, *pool;
  int buffer_rows;
  int *cu_q, *cu_k, *context, *slots, *out_tables;
  long long* positions;
  unsigned long long* masks;
  int mask_words;
  int hash_slots;                                  // power of two, 0 without rows
};

// Sums over the block of two numbers: each thread's own prefixes (exclusive) and the totals.  All threads take part.
struct StepSum {
  long long a;
  int b;
};
__device__ __forceinline__ StepSum block_scan(StepSum v, StepSum* scratch /* [kStepThreads / 32] */, StepSum& total) {
  constexpr int kWarps = kStepThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  StepSum x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, x.a, o);
    const int b = __shfl_up_sync(0xffffffffu, x.b, o);
    if (lane >= o) { x.a += a; x.b += b; }
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  StepSum w = lane < kWarps ? scratch[lane] : StepSum{0, 0};      // (every warp for itself: one barrier less)
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, w.a, o);
    const int b = __shfl_up_sync(0xffffffffu, w.b, o);
    if (lane >= o) { w.a += a; w.b += b; }
  }
  const int front = max(warp - 1, 0);
  const long long fa = __shfl_sync(0xffffffffu, w.a, front);
  const int fb = __shfl_sync(0xffffffffu, w.b, front);
  total.a = __shfl_sync(0xffffffffu, w.a, kWarps - 1);
  total.b = __shfl_sync(0xffffffffu, w.b, kWarps - 1);
  return {(warp ? fa : 0) + x.a - v.a, (warp ? fb : 0) + x.b - v.b};
}

// Marks, for each row that occurs in rows[0 .. batch), its first place: open addressing with as many slots as twice the batch.
// (The table has been cleared.)
__device__ __forceinline__ void hash_clear(int hash_slots, int* keys, int* firsts) {
  for (int i = threadIdx.x; i < hash_slots; i += kStepThreads) {
    keys[i] = INT_MIN;
    firsts[i] = INT_MAX;
  }
}
__device__ __forceinline__ void hash_rows(const int* rows, int batch, int hash_slots, int* keys, int* firsts) {
  __syncthreads();
  for (int i = threadIdx.x; i < batch; i += kStepThreads) {
    const int r = rows[i];
    if (r < 0) continue;
    for (unsigned s = static_cast<unsigned>(r) * 2654435761u >> 7;; ++s) {
      const int at = static_cast<int>(s & (hash_slots - 1));
      const int was = atomicCAS(&keys[at], INT_MIN, r);
      if (was == INT_MIN || was == r) {
        atomicMin(&firsts[at], i);
        break;
      }
    }
  }
  __syncthreads();
}
__device__ __forceinline__ bool first_place(int r, int i, int hash_slots, const int* keys, const int* firsts) {
  unsigned s = static_cast<unsigned>(r) * 2654435761u >> 7;
  while (keys[s & (hash_slots - 1)] != r) ++s;       // (it is there: hash_rows put it there)
  return firsts[s & (hash_slots - 1)] == i;
}

__global__ void __cluster_dims__(kStepCtas, 1, 1) __launch_bounds__(kStepThreads, 1) step_tables_kernel(const StepParams p) {
  // (No early trigger of dependent launches: attention reads these tables ahead of its own wait.)
  extern __shared__ int smem[];
  int* const s_cu = smem;                       // [batch + 1] first token
  int* const s_cached = s_cu + p.batch + 1;     // [batch]
  int* const s_held = s_cached + p.batch;       // [batch] blocks the request had
  int* const s_need = s_held + p.batch;         // [batch] blocks it needs; -1: left out
  int* const s_top = s_need + p.batch;          // [batch] where in the list its first new block stands
  int* const s_row = s_top + p.batch;           // [batch]
  int* const s_keys = s_row + p.batch;          // [hash_slots]
  int* const s_firsts = s_keys + p.hash_slots;  // [hash_slots]
  __shared__ StepSum scratch[2][kStepThreads / 32];
  __shared__ int s_granted;
  const int tid = threadIdx.x, rank = blockIdx.x;
  hash_clear(p.hash_slots, s_keys, s_firsts);
  if (tid == 0) s_granted = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");     // from here on: what the kernel in front may have written
  // What stands in the way is one load behind the other, so the first ones go out together: the thread's sequence, and the
  // parents of its tokens on their way into L1.
  const int n_free = max(0, min(p.pool[0], p.num_blocks));
  const bool live0 = tid < p.batch;
  const int row0 = live0 ? (p.rows ? p.rows[tid] : tid) : -1, cached0 = live0 ? p.cached[tid] : 0, fresh0 = live0 ? p.fresh[tid] : 0;
  if (p.masks)
    for (int t = rank * kStepThreads + tid; t < p.num_tokens; t += kStepCtas * kStepThreads)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(p.parents + t));
  const int owned0 = row0 >= 0 && row0 < p.max_requests ? p.owned[row0] : 0;
  if (p.rows) hash_rows(p.rows, p.batch, p.hash_slots, s_keys, s_firsts);
  else __syncthreads();
  long long tokens = 0, keys_so_far = 0;
  int wanted = 0, left_out = 0;
#pragma unroll 1
  for (int base = 0; base < p.batch; base += kStepThreads) {
    const int i = base + tid;
    const bool live = i < p.batch;
    const int row = base == 0 ? row0 : live ? (p.rows ? p.rows[i] : i) : -1;
    const int cached = max(base == 0 ? cached0 : live ? p.cached[i] : 0, 0), fresh = max(base == 0 ? fresh0 : live ? p.fresh[i] : 0, 0);
    const long long len = static_cast<long long>(cached) + fresh;
    bool ok = live && row >= 0 && row < p.max_requests && len <= INT_MAX - p.block_size;
    if (ok && p.rows) ok = first_place(row, i, p.hash_slots, s_keys, s_firsts);
    const int held = ok ? max(0, min(base == 0 ? owned0 : p.owned[row], p.table_cols)) : 0;
    const int need = ok ? (static_cast<int>(len) + p.block_size - 1) / p.block_size : 0;
    ok = ok && need <= p.table_cols && !(p.masks && fresh > 64 * p.mask_words);
    // (whether a sequence's tokens fit is known with the first sum only; what it would have wanted must not count then, so
    // those behind the last token that fits are cut off: the sums grow)
    StepSum total;
    const StepSum at = block_scan({fresh, ok ? max(need - held, 0) : 0}, scratch[0], total);
    const long long t0 = tokens + at.a;
    const int want = ok ? max(need - held, 0) : 0, before = wanted + at.b;
    tokens += total.a;
    wanted += total.b;
    ok = ok && t0 + fresh <= p.num_tokens && (want == 0 || before + want <= n_free);
    if (live) {
      s_cu[i] = static_cast<int>(min(t0, static_cast<long long>(p.num_tokens)));
      s_cached[i] = cached;
      s_held[i] = held;
      s_need[i] = ok ? need : -1;
      s_top[i] = n_free - 1 - before;
      s_row[i] = row;
    }
    if (rank == 0) {
      // (what is granted is what comes first of what is wanted)
      const int context = ok ? static_cast<int>(len) : 0;
      const StepSum k = block_scan({context, live && !ok ? 1 : 0}, scratch[1], total);
      if (live) {
        p.cu_q[i] = s_cu[i];
        p.cu_k[i] = static_cast<int>(keys_so_far + k.a);
        p.context[i] = context;
      }
      keys_so_far += total.a;
      left_out += total.b;
      if (ok && want > 0) atomicMax(&s_granted, before + want);
    }
    __syncthreads();
  }
  const int all = static_cast<int>(min(tokens, static_cast<long long>(p.num_tokens)));
  if (tid == 0) s_cu[p.batch] = all;
  if (rank == 0)
    for (int i = p.batch + tid; i <= p.buffer_rows; i += kStepThreads) {
      p.cu_q[i] = all;
      p.cu_k[i] = static_cast<int>(keys_so_far);
      if (i < p.buffer_rows) p.context[i] = 0;
    }
  __syncthreads();
  // owned and the list's length have been read
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  for (int t = rank * kStepThreads + tid; t < p.num_tokens; t += kStepCtas * kStepThreads) {
    int slot = -1;
    long long position = 0;
    unsigned long long m[kStepMaxWords] = {0, 0, 0, 0};
    if (t < all) {
      int lo = 0, hi = p.batch;                 // the last sequence that starts at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid; else hi = mid;
      }
      if (s_need[lo] >= 0) {
        const int start = s_cu[lo], j = t - start, at = s_cached[lo] + j;
        const int col = at / p.block_size, held = s_held[lo];
        const int id = col < held ? p.tables[s_row[lo] * p.table_stride + col] : p.free_blocks[s_top[lo] - (col - held)];
        if (id >= 0 && id < p.num_blocks) slot = id * p.block_size + (at - col * p.block_size);
        position = at;
        if (p.masks) {
          // up to the root: parents come before their children, anything else ends the walk
          int depth = 0;
          for (int n = j;; ++depth) {
#pragma unroll
            for (int w = 0; w < kStepMaxWords; ++w)
              if (n >> 6 == w) m[w] |= 1ull << (n & 63);
            const int up = p.parents[start + n];
            if (up < 0 || up >= n) break;
            n = up;
          }
          position = s_cached[lo] + depth;
        }
      }
    }
    p.slots[t] = slot;
    p.positions[t] = position;
    if (p.masks)
#pragma unroll
      for (int w = 0; w < kStepMaxWords; ++w)
        if (w < p.mask_words) p.masks[static_cast<long long>(t) * p.mask_words + w] = m[w];
  }
  const int cells = p.batch * p.table_cols;     // (batch and columns are bounded on the host)
  for (int e = rank * kStepThreads + tid; e < cells; e += kStepCtas * kStepThreads) {
    const int i = e / p.table_cols, col = e - i * p.table_cols;
    const int held = s_held[i], need = s_need[i];
    int id = -1;
    if (col < need) {
      int* const mine = p.tables + s_row[i] * p.table_stride + col;
      if (col < held) {
        id = *mine;
      } else {
        id = p.free_blocks[s_top[i] - (col - held)];
        *mine = id;                              // (no other CTA reads columns that were not held)
      }
    }
    p.out_tables[e] = id;
  }
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0) {
    for (int i = tid; i < p.batch; i += kStepThreads)
      if (s_need[i] > s_held[i]) p.owned[s_row[i]] = s_need[i];
    if (tid == 0) {
      p.pool[0] = n_free - s_granted;
      p.pool[1] = left_out;
    }
  }
}

// Requests keep the blocks of their first keep_lens[i] tokens; the others go back, sequence i's first to where step_tables took
// its first from.
struct ReleaseParams {
  const int *rows, *keep_lens;
  int batch, block_size;
  int* tables;
  long long table_stride;
  int table_cols, max_requests, num_blocks;
  int *owned, *free_blocks, *pool;
  int hash_slots;
};

__global__ void __launch_bounds__(kStepThreads, 1) release_blocks_kernel(const ReleaseParams p) {
  extern __shared__ int smem[];
  int* const s_before = smem;                   // [batch + 1] blocks that come before
  int* const s_keep = s_before + p.batch + 1;   // [batch]
  int* const s_row = s_keep + p.batch;          // [batch]
  int* const s_keys = s_row + p.batch;
  int* const s_firsts = s_keys + p.hash_slots;
  __shared__ StepSum scratch[kStepThreads / 32];
  const int tid = threadIdx.x;
  hash_clear(p.hash_slots, s_keys, s_firsts);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n_free = max(0, min(p.pool[0], p.num_blocks));
  const bool live0 = tid < p.batch;
  const int row0 = live0 ? (p.rows ? p.rows[tid] : tid) : -1, len0 = live0 ? p.keep_lens[tid] : 0;
  const int owned0 = row0 >= 0 && row0 < p.max_requests ? p.owned[row0] : 0;
  if (p.rows) hash_rows(p.rows, p.batch, p.hash_slots, s_keys, s_firsts);
  int back = 0;
#pragma unroll 1
  for (int base = 0; base < p.batch; base += kStepThreads) {
    const int i = base + tid;
    const bool live = i < p.batch;
    const int row = base == 0 ? row0 : live ? (p.rows ? p.rows[i] : i) : -1;
    bool ok = row >= 0 && row < p.max_requests;
    if (ok && p.rows) ok = first_place(row, i, p.hash_slots, s_keys, s_firsts);
    const int held = ok ? max(0, min(base == 0 ? owned0 : p.owned[row], p.table_cols)) : 0;
    const int len = max(base == 0 ? len0 : live ? p.keep_lens[i] : 0, 0);
    const int keep = min(len / p.block_size + (len % p.block_size != 0), held);
    StepSum total;
    const int before = back + block_scan({0, held - keep}, scratch, total).b;
    back += total.b;
    if (live) {
      s_before[i] = before;
      s_keep[i] = keep;
      s_row[i] = row;
      if (keep < held) p.owned[row] = keep;      // (rows are distinct where they release anything)
    }
    __syncthreads();
  }
  if (tid == 0) s_before[p.batch] = back;
  __syncthreads();
  for (int k = tid; k < back; k += kStepThreads) {
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_before[mid] <= k) lo = mid; else hi = mid;
    }
    int* const cell = p.tables + s_row[lo] * p.table_stride + s_keep[lo] + (k - s_before[lo]);
    const long long at = static_cast<long long>(n_free) + back - 1 - k;
    if (at < p.num_blocks) p.free_blocks[at] = *cell;
    *cell = -1;
  }
  if (tid == 0) p.pool[0] = static_cast<int>(min(static_cast<long long>(n_free) + back, static_cast<long long>(p.num_blocks)));
}

static int hash_size(int batch) {
  int n = 64;
  while (n < 2 * batch) n <<= 1;
  return n;
}

static int check_state(const char* what, const void* tables, int64_t table_stride, int32_t table_cols, int32_t max_requests,
                       const void* owned, const void* free_blocks, const void* pool, int64_t num_blocks, int32_t batch,
                       int32_t block_size) {
  if (batch < 0 || batch > kStepMaxBatch) return set_error(kErrBadShape, "%s: batch must be in [0, %d] (got %d)", what, kStepMaxBatch, batch);
  if (!tables || !owned || !free_blocks || !pool) return set_error(kErrNullPointer, "%s: null state pointer", what);
  if (block_size <= 0 || block_size % 256) return set_error(kErrBadShape, "%s: block_size must be a positive multiple of 256 (got %d)", what, block_size);
  if (num_blocks <= 0 || num_blocks * block_size >= (1LL << 31)) return set_error(kErrBadShape, "%s: num_blocks * block_size must be in (0, 2^31)", what);
  if (table_cols <= 0 || table_stride < table_cols || max_requests <= 0 || static_cast<int64_t>(table_cols) * kStepMaxBatch > (1LL << 30) ||
      static_cast<int64_t>(table_cols) * block_size >= (1LL << 31))
    return set_error(kErrBadShape, "%s: bad table geometry (%d requests x %d columns, stride %lld)", what, max_requests, table_cols,
                     (long long)table_stride);
  return kOk;
}

}  // namespace b200

extern "C" int b200_step_tables(const int32_t* rows, const int32_t* cached_lens, const int32_t* new_lens, const int32_t* parents,
                                int32_t batch, int32_t num_tokens, int32_t block_size, int32_t* tables, int64_t table_stride,
                                int32_t table_cols, int32_t max_requests, int32_t* owned, int32_t* free_blocks, int32_t* pool,
                                int64_t num_blocks, int32_t buffer_rows, int32_t* cu_seqlens_q, int32_t* cu_seqlens_k,
                                int32_t* context_lens, int32_t* slot_mapping, int64_t* positions, int32_t* block_tables,
                                uint64_t* tree_masks, int32_t mask_words, void* stream) {
  using namespace b200;
  int rc = check_state("step_tables", tables, table_stride, table_cols, max_requests, owned, free_blocks, pool, num_blocks, batch, block_size);
  if (rc) return rc;
  if (num_tokens < 0 || num_tokens > (1 << 30) || buffer_rows < batch) return set_error(kErrBadShape, "step_tables: num_tokens (%d) must be in [0, 2^30], buffer_rows (%d) not below batch (%d)", num_tokens, buffer_rows, batch);
  if (!cu_seqlens_q || !cu_seqlens_k || (buffer_rows > 0 && !context_lens) || (num_tokens > 0 && (!slot_mapping || !positions)) ||
      (batch > 0 && (!cached_lens || !new_lens || !block_tables)))
    return set_error(kErrNullPointer, "step_tables: null pointer argument");
  if ((tree_masks != nullptr) != (parents != nullptr) && num_tokens > 0) return set_error(kErrNullPointer, "step_tables: parents and tree_masks go together");
  if (tree_masks && (mask_words < 1 || mask_words > kStepMaxWords)) return set_error(kErrBadShape, "step_tables: mask_words must be in [1, %d] (got %d)", kStepMaxWords, mask_words);
  if ((reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(tree_masks)) & 7)
    return set_error(kErrMisaligned, "step_tables: positions and tree_masks must be 8-byte aligned");
  StepParams p;
  p.rows = rows;
  p.cached = cached_lens;
  p.fresh = new_lens;
  p.parents = parents;
  p.batch = batch;
  p.num_tokens = num_tokens;
  p.block_size = block_size;
  p.tables = tables;
  p.table_stride = table_stride;
  p.table_cols = table_cols;
  p.max_requests = max_requests;
  p.num_blocks = static_cast<int>(num_blocks);
  p.owned = owned;
  p.free_blocks = free_blocks;
  p.pool = pool;
  p.buffer_rows = buffer_rows;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.context = context_lens;
  p.slots = slot_mapping;
  p.out_tables = block_tables;
  p.positions = reinterpret_cast<long long*>(positions);
  p.masks = reinterpret_cast<unsigned long long*>(tree_masks);
  p.mask_words = mask_words;
  p.hash_slots = rows ? hash_size(batch) : 0;
  const size_t smem = (static_cast<size_t>(batch) * 6 + 1 + 2 * static_cast<size_t>(p.hash_slots)) * 4;
  static std::atomic<size_t> configured[kMaxDevices];
  if (smem > 48 * 1024) {
    rc = ensure_dynamic_smem(reinterpret_cast<const void*>(step_tables_kernel), smem, configured, "step_tables: cudaFuncSetAttribute");
    if (rc) return rc;
  }
  const cudaError_t le = launch_early(step_tables_kernel, kStepCtas, kStepThreads, smem, static_cast<cudaStream_t>(stream), p);
  g_launches.fetch_add(1);
  return check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "step_tables launch");
}

extern "C" int b200_release_blocks(const int32_t* rows, const int32_t* keep_lens, int32_t batch, int32_t block_size, int32_t* tables,
                                   int64_t table_stride, int32_t table_cols, int32_t max_requests, int32_t* owned,
                                   int32_t* free_blocks, int32_t* pool, int64_t num_blocks, void* stream) {
  using namespace b200;
  int rc = check_state("release_blocks", tables, table_stride, table_cols, max_requests, owned, free_blocks, pool, num_blocks, batch, block_size);
  if (rc) return rc;
  if (batch == 0) return kOk;
  if (!keep_lens) return set_error(kErrNullPointer, "release_blocks: null pointer argument");
  ReleaseParams p;
  p.rows = rows;
  p.keep_lens = keep_lens;
  p.batch = batch;
  p.block_size = block_size;
  p.tables = tables;
  p.table_stride = table_stride;
  p.table_cols = table_cols;
  p.max_requests = max_requests;
  p.num_blocks = static_cast<int>(num_blocks);
  p.owned = owned;
  p.free_blocks = free_blocks;
  p.pool = pool;
  p.hash_slots = rows ? hash_size(batch) : 0;
  const size_t smem = (static_cast<size_t>(batch) * 3 + 1 + 2 * static_cast<size_t>(p.hash_slots)) * 4;
  static std::atomic<size_t> configured[kMaxDevices];
  if (smem > 48 * 1024) {
    rc = ensure_dynamic_smem(reinterpret_cast<const void*>(release_blocks_kernel), smem, configured, "release_blocks: cudaFuncSetAttribute");
    if (rc) return rc;
  }
  const cudaError_t le = launch_early(release_blocks_kernel, 1, kStepThreads, smem, static_cast<cudaStream_t>(stream), p);
  g_launches.fetch_add(1);
  return check_cuda(le != cudaSuccess ? le : cudaGetLastError(), "release_blocks launch");
}
