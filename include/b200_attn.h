/* b200_attn.h -- C ABI of the B200 (sm_100a) paged-KV attention library, libb200attn.so.
 *
 * The entry points are what a binding for nano-vllm's attention layer calls in place of the
 * reference's Triton kernel and flash_attn calls.  File:line citations are relative to the
 * nano-vllm project root.
 *
 * Conventions
 *  - Every pointer is a device pointer on the current CUDA device unless stated otherwise.
 *    The compute entry points never allocate, free or copy device memory and never synchronise;
 *    every launch goes to `stream` (a cudaStream_t passed as void*; NULL = legacy default stream),
 *    so calls can be captured into CUDA graphs.  The exceptions say so in their own comments: the
 *    two status queries synchronise the device, b200_ipc_open maps another process's buffer.
 *  - Activations and caches are bf16 for the attention entry points.  head_dim must be 128.
 *  - Strides are in ELEMENTS.  Pointers and row strides must be 16-byte aligned.
 *  - The paged cache has the reference's layout (nanovllm/engine/model_runner.py:107-117): one
 *    contiguous array (num_blocks, block_size, num_kv_heads, head_dim) for K and one for V;
 *    flat slot = block_id * block_size + offset.  block_size must be a multiple of 256
 *    (nanovllm/config.py:22).
 *  - Block tables are int32 (batch, bt_cols) with row stride bt_row_stride; entries at columns
 *    >= ceil(len / block_size) may hold -1 or stale ids (nanovllm/engine/model_runner.py:119-123,
 *    :203) and are never dereferenced.
 *  - Early starts (programmatic dependent launch).  b200_store_kvcache, b200_qk_norm_rope_store, b200_decode_attn,
 *    b200_store_decode_attn, b200_prefill_attn / b200_store_prefill_attn, b200_tree_attn and the other entry points for
 *    steps with drafted tokens start early behind a kernel that lets its dependents do so (griddepcontrol.launch_dependents), and read part of their metadata before they wait for it:
 *      decode                 context_lens, block_tables; b200_store_decode_attn also slot_mapping
 *      prefill, tcgen05       cu_seqlens_q, cu_seqlens_k
 *      tree attention         cu_seqlens_q, context_lens, block_tables
 *      store, producer, prefill on mma.sync     nothing (what the first two read ahead they read again)
 *      step tables, release, accept, compaction     nothing
 *    So a kernel that lets its dependents start early must not write these arrays.  Of this library the store,
 *    producer, decode, tree attention and mma.sync prefill kernels do (they write cache rows, q, k, outputs and workspaces
 *    only); the metadata unpack, all-reduce and tcgen05 prefill kernels, and the step's tables, release, accept and
 *    compaction, which write such arrays, do not.  Behind any other kernel or copy there is nothing to observe.
 *  - Return value: 0 on success; negative = arguments rejected before any launch; positive = a
 *    cudaError_t from the launch.  b200_last_error() describes the last failure of the calling
 *    thread.  Nothing throws, aborts or traps.
 */
#ifndef B200_ATTN_H_
#define B200_ATTN_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B200_ATTN_VERSION 100

#define B200_OK 0
#define B200_ERR_NULL_POINTER (-1)
#define B200_ERR_BAD_SHAPE (-2)
#define B200_ERR_MISALIGNED (-3)
#define B200_ERR_WORKSPACE (-4)
#define B200_ERR_NO_DRIVER (-5)
#define B200_ERR_TENSOR_MAP (-6)
#define B200_ERR_DEVICE (-7)
#define B200_ERR_TIMEOUT (-8)

/* Library version (B200_ATTN_VERSION of the build). */
int b200_version(void);

/* Message for the last non-zero status returned to this thread ("" if none). Host pointer,
 * valid until the thread's next failing call. */
const char* b200_last_error(void);

/* Replaces store_kvcache_kernel + store_kvcache (nanovllm/layers/attention.py:10-40).
 * For token i in [0, n_tokens): slot = slot_mapping[i]; slot == -1 is skipped; otherwise the
 * row_elems elements of key row i (at key + i * key_row_stride) are copied to flat cache row
 * `slot` of k_cache, and likewise for value / v_cache.  Pure byte copy (any elem_bytes);
 * row_elems * elem_bytes and both row strides must be multiples of 16 bytes.  Offsets are
 * formed in 64 bits.  n_slots (= num_blocks * block_size) bounds the slot: an out-of-range
 * slot is skipped, never written.  n_tokens == 0 is a no-op. */
int b200_store_kvcache(const void* key, const void* value, int64_t key_row_stride, int64_t value_row_stride,
                       void* k_cache, void* v_cache, const int32_t* slot_mapping, int32_t n_tokens,
                       int32_t row_elems, int32_t elem_bytes, int64_t n_slots, void* stream);

/* Bytes of workspace b200_decode_attn needs for any batch up to `max_batch` with this head
 * geometry on the current device (depends on its multiprocessor count).  The caller allocates
 * it once, ZERO-FILLS it once, and passes it to every call; the kernels leave the parts that
 * must be zero as they found them.  Calls that share a workspace must not overlap on the GPU.
 * Returns a negative status on bad arguments. */
int64_t b200_decode_workspace_bytes(int32_t max_batch, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim);

/* Replaces flash_attn_with_kvcache as called for decode (nanovllm/layers/attention.py:71-74).
 * For sequence i: the single query token q[i] (num_heads x head_dim at q + i * q_row_stride)
 * attends the context_lens[i] cached tokens reached through block_tables[i, :]; GQA maps q head
 * h to kv head h / (num_heads / num_kv_heads); softmax(scale * q k^T) v with fp32 softmax and
 * accumulation; out[i] (num_heads x head_dim, contiguous rows of num_heads * head_dim) in bf16.
 * context_lens[i] <= 0 writes zeros and touches no cache.  The launch geometry depends only on
 * (batch, head geometry, bt_cols), never on device data; the same inputs give the same bits on every call.  Early start:
 * see above. */
int b200_decode_attn(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                     int64_t num_blocks, int32_t block_size, const int32_t* block_tables, int64_t bt_row_stride,
                     int32_t bt_cols, const int32_t* context_lens, void* out, void* workspace,
                     int64_t workspace_bytes, int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                     int32_t head_dim, float scale, void* stream);

/* b200_store_kvcache(k, v, ..) of one row per sequence and b200_decode_attn as one call, the layer's decode step
 * (nanovllm/layers/attention.py:59-74): row i of k and v goes to flat cache row slot_mapping[i] (-1 and slots outside the
 * cache are skipped), and attention sees the cache with all of the step's rows in place.  Up to 160 sequences, or few
 * (sequence, kv head) pairs, it is one launch, else the two kernels one after the other. */
int b200_store_decode_attn(const void* q, int64_t q_row_stride, const void* k, const void* v, int64_t k_row_stride,
                           int64_t v_row_stride, const int32_t* slot_mapping, void* k_cache, void* v_cache,
                           int64_t num_blocks, int32_t block_size, const int32_t* block_tables, int64_t bt_row_stride,
                           int32_t bt_cols, const int32_t* context_lens, void* out, void* workspace,
                           int64_t workspace_bytes, int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                           int32_t head_dim, float scale, void* stream);

/* No counterpart in the reference: decode attention for callers that cannot allocate.
 *
 * b200_decode_attn needs a caller-owned workspace.  Some callers have no way to provide one: an
 * engine that has already given all free device memory to its KV cache (a later cudaMalloc may
 * fail), a plugin interface that forbids allocating inside the call, code that must stay away from
 * the framework's allocator.  This variant computes exactly what b200_decode_attn computes, with
 * the same arguments minus the workspace, and keeps its scratch inside the library: a __device__
 * array of b200_decode_static_scratch_bytes() (8 249 600 bytes, about 7.9 MiB) that every GPU which loads the
 * library holds until the process exits.  It calls no cudaMalloc/cudaFree and no allocating
 * library routine.
 *
 * Limits (rejected with B200_ERR_WORKSPACE and a message, nothing launched): (persistent CTAs of
 * the device = 2 per multiprocessor) x (num_heads / num_kv_heads) may be at most 1280 -- on a
 * 148-SM B200 that is up to 4 query heads per kv head -- and num_kv_heads at most 128.  Beyond
 * that use b200_decode_attn.
 *
 * The first call on each device looks up the array's device address (cudaGetSymbolAddress, with
 * that device current); make that first call before any stream capture begins.  All calls on a
 * device share the one array: it keeps the previous call's contents (the entry point clears the
 * part that must start at zero, on `stream`, before launching), and two calls that overlap on
 * the GPU -- different streams, or different host threads -- race on it.  Serialise them. */
int64_t b200_decode_static_scratch_bytes(void);
int b200_decode_attn_static(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                            int64_t num_blocks, int32_t block_size, const int32_t* block_tables,
                            int64_t bt_row_stride, int32_t bt_cols, const int32_t* context_lens, void* out,
                            int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
                            void* stream);

/* Replaces flash_attn_varlen_func as called for prefill (nanovllm/layers/attention.py:64-70).
 * Sequence i owns query rows cu_seqlens_q[i] .. cu_seqlens_q[i+1] of q (total_q, num_heads, 128)
 * and keys 0 .. Lk_i - 1 with Lk_i = cu_seqlens_k[i+1] - cu_seqlens_k[i].  Causal mask aligned
 * bottom-right: query row r sees keys 0 .. Lk_i - Lq_i + r.
 *  - block_tables == NULL: dense K/V.  k, v are (total_k, num_kv_heads, 128) with row strides
 *    k_row_stride / v_row_stride, sequence i's keys at rows cu_seqlens_k[i] ...
 *  - block_tables != NULL (prefix cache): K/V for the whole key range come from k_cache/v_cache
 *    through block_tables[i, t / block_size]; k and v are ignored.
 * Sequences with Lq_i == 0 produce no rows.  out is (total_q, num_heads, 128) contiguous bf16.
 * max_seqlen_q / max_seqlen_k are the host-side bounds the caller already has
 * (nanovllm/utils/context.py:9-10).  kernel_variant: 0 = default (the persistent tcgen05 kernel
 * when 128 % (num_heads / num_kv_heads) == 0, the scale is positive and the batch is not so short that the mma.sync kernel is
 * through it sooner, else the mma.sync kernel), 1 = force the mma.sync
 * kernel, 2 = force the tcgen05 kernel (B200_ERR_BAD_SHAPE if it cannot take the shape or the scale).  Launches
 * of the tcgen05 kernel share one device-side ticket counter: do not overlap two of them on one
 * GPU.  The persistent kernel
 * writes `out` through TMA stores: out must be 16-byte aligned (as every tensor here). */
int b200_prefill_attn(const void* q, int64_t q_row_stride, const void* k, const void* v, int64_t k_row_stride,
                      int64_t v_row_stride, int64_t total_k, const void* k_cache, const void* v_cache,
                      int64_t num_blocks, int32_t block_size, const int32_t* block_tables, int64_t bt_row_stride,
                      int32_t bt_cols, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t batch,
                      int32_t total_q, int32_t max_seqlen_q, int32_t max_seqlen_k, void* out, int32_t num_heads,
                      int32_t num_kv_heads, int32_t head_dim, float scale, int32_t kernel_variant, void* stream);

/* b200_store_kvcache(k, v, ..) and dense b200_prefill_attn(q, k, v, ..) as one call, the layer's prefill step without a
 * cached prefix (nanovllm/layers/attention.py:59-70): token i's k and v rows also go to flat cache row slot_mapping[i]
 * (total_k entries; -1 and slots >= n_slots are skipped).  Attention does not read the cache here and does
 * not wait for it: both kernels do the copy on the side, in the same launch. */
int b200_store_prefill_attn(const void* q, int64_t q_row_stride, const void* k, const void* v, int64_t k_row_stride,
                            int64_t v_row_stride, int64_t total_k, void* k_cache, void* v_cache,
                            const int32_t* slot_mapping, int64_t n_slots, const int32_t* cu_seqlens_q,
                            const int32_t* cu_seqlens_k, int32_t batch, int32_t total_q, int32_t max_seqlen_q,
                            int32_t max_seqlen_k, void* out, int32_t num_heads, int32_t num_kv_heads,
                            int32_t head_dim, float scale, void* stream);

/* ---- producer side of the layer: QK-norm + rotary embedding + cache store in one launch -------------------
 * Replaces, for one decoder layer and one step, what the reference runs between its fused qkv projection
 * and its attention call (nanovllm/models/qwen3.py:75-79 and nanovllm/layers/attention.py:62-63):
 *   q_norm, k_norm   nanovllm/layers/layernorm.py:16-26       fp32 RMS normalisation over head_dim, cast to
 *                                                              bf16, times the bf16 weight
 *   rotary_emb       nanovllm/layers/rotary_embedding.py:6-14  rotate-half with cos/sin gathered by position
 *   store_kvcache    nanovllm/layers/attention.py:10-40        k (after norm and rotation) and v to their slots
 * qkv is the (n_tokens, (num_heads + 2 * num_kv_heads) * 128) bf16 output of the fused projection with row
 * stride qkv_row_stride (elements); positions are int64 as in the reference; cos_sin_cache is the reference's
 * (max_position, 1, 128) fp32 table (64 cos then 64 sin per position).  q_out (n_tokens, num_heads, 128) and
 * k_out (n_tokens, num_kv_heads, 128) are written contiguous (dense prefill reads k from there).  With
 * k_cache / v_cache given, token i's k and v rows also go to flat cache row slot_mapping[i] (-1 and slots
 * >= n_slots are skipped); both NULL = no store (the engine's warm-up pass).  v is never copied anywhere else:
 * the attention call keeps reading it as a view of qkv. */
int b200_qk_norm_rope_store(const void* qkv, int64_t qkv_row_stride, const int64_t* positions, const void* q_weight,
                            const void* k_weight, const float* cos_sin_cache, int32_t max_position, float eps,
                            void* q_out, void* k_out, void* k_cache, void* v_cache, const int32_t* slot_mapping,
                            int64_t n_slots, int32_t n_tokens, int32_t num_heads, int32_t num_kv_heads,
                            int32_t head_dim, void* stream);

/* ---- caller side of the decode path: a step's metadata into the graph's static buffers in one launch -----
 * Replaces, for one decode step, the seven device operations with which the reference's model runner moves
 * its freshly copied metadata into the buffers its CUDA graphs were captured on
 * (nanovllm/engine/model_runner.py:193-203), and lets its five host-to-device copies (:163-179, :119-123)
 * become one: the host packs the step into one record,
 *   int64 input_ids[batch] | int64 positions[batch] | int32 slot_mapping[batch] | int32 context_lens[batch] |
 *   int32 block_tables[batch][table_width]  (rows padded with -1)
 * copies it to the device (8-byte aligned), and this call scatters it with the reference's exact effect:
 * rows [0, batch) of input_ids and positions are written; slot_mapping is -1 and context_lens 0 on rows
 * [batch, buffer_rows); block_tables (row stride buffer_table_cols) gets columns [0, table_width) of rows
 * [0, batch) and keeps the rest.  batch <= buffer_rows and table_width <= buffer_table_cols. */
int b200_unpack_decode_metadata(const void* packed, int32_t batch, int32_t table_width, int32_t buffer_rows,
                                int32_t buffer_table_cols, int64_t* input_ids, int64_t* positions,
                                int32_t* slot_mapping, int32_t* context_lens, int32_t* block_tables, void* stream);

/* ---- steps with drafted tokens (speculative decoding) -------------------------------------------------------
 * No counterpart in the reference, which decodes one token per sequence and step.  A step in which every sequence brings
 * the nodes of a drafted tree: tables for it (b200_step_tables), its attention in every layer (b200_tree_attn, behind
 * b200_store_kvcache or b200_qk_norm_rope_store with the step's slots), the walk along the sampled tokens
 * (b200_accept_tree), the accepted nodes' cache rows to their places (b200_compact_kvcache), and what the sequences no
 * longer need back into the free list (b200_release_blocks).  Lengths and blocks need not come back to the host.
 *
 * A tree: node 0 is its root (the last token that was committed), parents[j] < j is the index of node j's parent within
 * the tree, anything else (-1, say) means that it has none.  Nodes lie in the cache one behind the other, from the cached
 * length on, whatever their depth. */

/* A step's tables from request lengths.  Requests own rows of `tables` (max_requests, table_cols; row stride table_stride)
 * and the first owned[r] ids of their row; free_blocks[0 .. pool[0]) is a stack of free ids.  Sequence i of the batch is
 * request rows[i] (NULL: i) with cached_lens[i] tokens in the cache and new_lens[i] in this step, whose token rows lie one
 * behind the other (num_tokens in all).  It takes ceil((cached + new) / block_size) - owned blocks (none below zero) from
 * the stack, which go into its row and owned; the sequences take theirs in the order of the batch.  Written:
 *   cu_seqlens_q, cu_seqlens_k (buffer_rows + 1), context_lens (buffer_rows): cumulative new and context lengths, and
 *                 cached + new; rows from `batch` on repeat the totals and have length 0
 *   slot_mapping, positions (num_tokens): cache slot and position of each token, -1 and 0 behind the last
 *   block_tables  (batch, table_cols): ids, -1 behind the last
 *   tree_masks    (num_tokens, mask_words), with `parents` (num_tokens) only: bit n of a node's mask says that it sees node
 *                 n, an ancestor or itself; its position is then the cached length plus its depth
 * A sequence is left out (context length 0, slots -1, positions and masks 0, nothing taken) if its row is outside
 * [0, max_requests) or stands in the batch before, if it needs more than table_cols blocks, has more than 64 * mask_words
 * nodes, if its tokens do not all fit into num_tokens, or if there are not enough free blocks when its turn comes (then
 * later ones get none either).  pool[1] is set to the number of sequences left out.  Negative lengths count as 0.
 * batch is at most 4096, mask_words at most 4.  Outputs must not overlap the inputs.  The launch lets nothing start early. */
int b200_step_tables(const int32_t* rows, const int32_t* cached_lens, const int32_t* new_lens, const int32_t* parents,
                     int32_t batch, int32_t num_tokens, int32_t block_size, int32_t* tables, int64_t table_stride,
                     int32_t table_cols, int32_t max_requests, int32_t* owned, int32_t* free_blocks, int32_t* pool,
                     int64_t num_blocks, int32_t buffer_rows, int32_t* cu_seqlens_q, int32_t* cu_seqlens_k,
                     int32_t* context_lens, int32_t* slot_mapping, int64_t* positions, int32_t* block_tables,
                     uint64_t* tree_masks, int32_t mask_words, void* stream);

/* Request rows[i] (NULL: i) keeps the blocks of its first keep_lens[i] tokens; the others go back onto the stack (their
 * columns become -1), in the order that undoes b200_step_tables.  A row that stands in the batch before, or outside
 * [0, max_requests), gives nothing back.  free_blocks has room for num_blocks ids; more are dropped.  Blocks that other
 * rows use as well must not be given back: keep them, and take them out of `owned`. */
int b200_release_blocks(const int32_t* rows, const int32_t* keep_lens, int32_t batch, int32_t block_size, int32_t* tables,
                        int64_t table_stride, int32_t table_cols, int32_t max_requests, int32_t* owned,
                        int32_t* free_blocks, int32_t* pool, int64_t num_blocks, void* stream);

/* Bytes of workspace that b200_tree_attn needs with this head geometry on the current device, whatever the batch.  It need
 * not be initialised and holds nothing between calls; calls that may overlap on the GPU need one each. */
int64_t b200_tree_workspace_bytes(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim);

/* Attention of a step's nodes over the paged cache, which has their keys and values already.  Sequence i's nodes are query
 * rows cu_seqlens_q[i] .. cu_seqlens_q[i+1] of q (total_q, num_heads, 128); node j lies at cache position context_lens[i] - T
 * + j, T their number.  Each sees all positions in front of the nodes, and of these node n where bit n of its row of
 * tree_masks (total_q, mask_words) is set; with tree_masks NULL those before it and itself (a drafted chain).  Bits of nodes
 * that the sequence does not have mean nothing; nodes from 64 * mask_words on are seen by none.  A row that sees nothing
 * (context_lens[i] <= 0 among them) gives zeros.  GQA, scale and numerics as b200_decode_attn; out (total_q, num_heads, 128)
 * contiguous; rows outside cu_seqlens_q are left as they are.  Keys and values of a sequence's positions must be finite, seen or
 * not.  At most 128 query heads per kv head, mask_words at most 4.  Where the call does not fit into thread-block clusters (few units and narrow
 * tables), num_kv_heads * (batch + total_q / (2 * (128 / G))) * (bt_cols * (block_size / 128) * 7 + 24) must be below 2^31, G = num_heads / num_kv_heads
 * (8 kv heads, 512 sequences of 64 nodes, G = 4: tables of 4.7 million tokens).  The same inputs give the same bits on every call. */
int b200_tree_attn(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache, int64_t num_blocks,
                   int32_t block_size, const int32_t* block_tables, int64_t bt_row_stride, int32_t bt_cols,
                   const int32_t* cu_seqlens_q, const int32_t* context_lens, const uint64_t* tree_masks, int32_t mask_words,
                   void* out, void* workspace, int64_t workspace_bytes, int32_t batch, int32_t total_q, int32_t num_heads,
                   int32_t num_kv_heads, int32_t head_dim, float scale, void* stream);

/* The walk through each tree: from the root to the child (the first, if there are several) whose draft token equals the
 * target token of the node it hangs on, and on from there, at most max_path nodes.  target_tokens[r] is what the target
 * model's sampler gave behind node r, so what comes out are its own samples.  Written per sequence: accepted (nodes on the
 * path), path (batch, max_path: their indices), tokens (batch, max_path: their target tokens, the step's result), both -1
 * behind the last, and new_cached_lens = cached_lens + accepted (may be the same array).  Sequences without nodes or with
 * context_lens[i] <= 0 (left out of the step) accept none. */
int b200_accept_tree(const int64_t* draft_tokens, const int64_t* target_tokens, const int32_t* parents,
                     const int32_t* cu_seqlens_q, const int32_t* cached_lens, const int32_t* context_lens, int32_t batch,
                     int32_t num_tokens, int32_t max_path, int32_t* accepted, int32_t* path, int64_t* tokens,
                     int32_t* new_cached_lens, void* stream);

/* The accepted nodes' rows to their places, in all planes of a cache (K and V of every layer; plane_stride_bytes apart,
 * each num_blocks * block_size rows of row_bytes): the row of position start_lens[i] + path[i][k] goes to start_lens[i] + k
 * for k < accepted[i], path (batch, path_cols) contiguous.  path ascends, from the root on (a path of one column is the root alone: nothing
 * is moved); entries below their place (path[i][k] < k) are not moved, nor is anything from or to a position without a block of the cache, or with a negative start length.  Pure byte copy.  Sequences must not share
 * the blocks behind their start lengths.  batch is at most 65535. */
int b200_compact_kvcache(void* cache, int32_t planes, int64_t plane_stride_bytes, int64_t row_bytes, int64_t num_blocks,
                         int32_t block_size, const int32_t* path, int32_t path_cols, const int32_t* accepted,
                         const int32_t* start_lens, const int32_t* block_tables, int64_t bt_row_stride, int32_t bt_cols,
                         int32_t batch, void* stream);

/* ---- behind the path: the all-reduce after the output projection, for decode-sized messages ---------------
 * Replaces `dist.all_reduce(y)` in RowParallelLinear.forward (nanovllm/layers/linear.py:149-153) when y is at
 * most b200_small_allreduce_max_bytes() (512 KiB) of bf16: a one-shot sum over plain peer loads and stores.
 * Set-up is the caller's: every rank allocates an exchange buffer of b200_small_allreduce_buffer_bytes(),
 * zero-filled, shares it with the other ranks of the node (CUDA IPC) and passes the `world` device pointers under
 * which IT sees the ranks' buffers (own buffer at index `rank`; a HOST array of pointers), plus a private,
 * zero-filled device block of b200_small_allreduce_state_bytes().  All ranks must make the same sequence of calls
 * with the same sizes.  inout (n_elems bf16, a multiple of 8, 16-byte aligned) is replaced by the sum over ranks,
 * accumulated in fp32 in rank order (every rank gets identical bits).  Every wait is bounded
 * (wait_limit_seconds, default 1 s when <= 0): a rank whose peers do not show up leaves its message unchanged
 * and sets a status word, read with b200_small_allreduce_status(); after that the ranks must zero their buffers
 * and state blocks together before the next call.  The launch can be captured in a CUDA graph. */
int64_t b200_small_allreduce_buffer_bytes(void);
int64_t b200_small_allreduce_state_bytes(void);
int64_t b200_small_allreduce_max_bytes(void);
int b200_small_allreduce(void* const* peer_buffers, int32_t rank, int32_t world, void* local_state, void* inout,
                         int64_t n_elems, double wait_limit_seconds, void* stream);
/* Synchronises the current device and returns B200_ERR_TIMEOUT if a wait of b200_small_allreduce gave up since the
 * state block was zero-filled, else 0. */
int b200_small_allreduce_status(const void* local_state);
/* Set-up helpers for the exchange buffers (no counterpart in the reference, which leaves this to NCCL): export a
 * device buffer of this process as a 64-byte CUDA IPC handle plus the buffer's offset inside its allocation, and map
 * a buffer exported by another process into the current device's address space.  The mapping lasts until the process
 * exits.  Host pointers for handle, offset and result. */
int b200_ipc_export(const void* ptr, void* handle_out_64_bytes, int64_t* offset_out);
int b200_ipc_open(const void* handle_64_bytes, int64_t offset, void** ptr_out);

/* Number of kernels this library has launched from the calling process so far (all threads).
 * Benchmarks use the difference across a timed region. */
int64_t b200_launch_count(void);

/* Diagnostic, not for the hot path: synchronises the current device and returns
 * B200_ERR_TIMEOUT if any kernel of this library gave up on a bounded wait since the last call
 * that reported one (the output of that launch is undefined), a positive cudaError_t if the
 * device reports an error, else 0.  A call that reports a timeout also recovers: it clears the
 * status words and the prefill kernel's ticket counter, so later launches start clean and the
 * next call speaks about them only.  What the library cannot reach is the caller-owned decode
 * workspace: if the failed launch was a decode, zero-fill that workspace again. */
int b200_device_status(void);

/* Test hook for the recovery path above, never called by the product: synchronises the device and
 * leaves the library's device-side state as a prefill launch that gave up on a wait would have
 * left it (status word set, ticket counter stale).  Nothing is launched and no GPU fault is
 * involved.  The next b200_device_status() must report B200_ERR_TIMEOUT and repair the state. */
int b200_test_inject_timeout(void);

/* Test hook, never called by the product: one thread waits on a barrier that nobody arrives on until the wait gives
 * up, once with each of the library's two kinds of timed wait (common; tcgen05 prefill), about a second each.  Fills
 * seconds[2] (host memory) with what they took, -1 where a wait did not report that it gave up. */
int b200_test_wait_limits(float* seconds);

/* Test hook, never called by the product, needs no device: CTAs per (sequence, kv head) that b200_decode_attn gives a batch of
 * `pairs` of them, with a block table of max_tiles x 64 tokens, on a chip that holds on_chip[0 .. 3] (host memory) clusters of
 * 8, 4, 2 and 1 CTAs at a time; 0: the general kernel. */
int b200_test_cluster_rule(int64_t pairs, int32_t heads_per_kv_head, int32_t max_tiles, const int32_t* on_chip);

#ifdef __cplusplus
}
#endif
#endif /* B200_ATTN_H_ */
