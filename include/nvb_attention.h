/*
 * nvb_attention.h — C ABI of the B200 (sm_100a) paged-attention library
 * `libnvb.so`. This is the drop-in boundary behind nano-vllm-rs's
 * `--attention-backend` seam.
 *
 * Every pointer except `stream` is a CUDA device pointer on the current
 * device. `stream` is a cudaStream_t owned by the caller. No attention entry
 * point allocates device memory, synchronizes the stream, or owns a context,
 * so their launches (nvb_paged_decode_static_scratch aside: see its own
 * comment) are safe inside CUDA-graph stream capture, with one exception:
 * the first launch that sees a new KV-cache base pointer encodes its TMA
 * descriptor on the host (no device work); do that first launch before
 * capture, as the reference engine does with its warm-up forward. The
 * multi-GPU set-up calls nvb_peer_buffer_* allocate and map memory (call
 * them once, outside capture), and nvb_paged_decode_gather takes a per-call
 * epoch, so a captured launch would replay a stale one: launch it directly.
 *
 * Layouts (identical to the reference):
 *   q, out           [total_q, q_heads, 128] bf16, contiguous
 *   k, v (per layer) [num_blocks, block_size, kv_heads, 128] bf16
 *   block_table      [batch, table_stride] int32, -1 marks an unused entry
 *   cu_q             [batch + 1] int32, cumulative query counts
 *   kv_lens          [batch] int32, NOT cumulative, includes this step
 *   slot_mapping     [rows] int32, slot = page * block_size + pos % block_size
 *
 * Return value: 0 on success, -1 on invalid host arguments, or a positive
 * cudaError_t for a launch error. The message is in a thread-local buffer
 * returned by nvb_last_error(). Asynchronous device faults surface at the
 * caller's next synchronization, as in the reference.
 */
#ifndef NVB_ATTENTION_H
#define NVB_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Paged-KV attention, call-compatible with the reference's FlashAttention
 * adapter `nvr_flash_fwd` (kernels/flash_native/flash_native.h:22-27,
 * implementation kernels/flash_native/flash_native.cu:40-121; Rust binding
 * src/gpu.rs:181-202, caller src/gpu.rs:890-995).
 *
 *  - max_q == 1: decode. Exactly one query per sequence (total_q == batch).
 *    One CTA per (sequence, kv head, split) streams the sequence's KV pages
 *    through TMA; the whole GQA query group shares each KV tile. With
 *    num_splits > 1 the split partials go to lse_accum
 *    [num_splits, batch, q_heads] and out_accum [num_splits, batch, q_heads,
 *    128] (FP32) and a combine kernel writes `out`.
 *  - max_q > 1: varlen / chunked causal prefill. Queries of sequence b are
 *    the contiguous suffix of its KV context (bottom-right causal mask).
 *    Runs on tcgen05 tensor cores with TMEM accumulators. num_splits must
 *    be 1.
 *  - lse (natural-log softmax LSE) is written at [(b * q_heads + h) * max_q
 *    + i] for query i of sequence b.
 *
 * Limits: head_dim 128, block_size a positive multiple of 256, q_heads a
 * multiple of kv_heads, q_heads <= 256 (any GQA group, as the reference:
 * flash_native.cu:48-52), 1 <= num_splits <= 128. Unlike the reference (max_k <= 4096) the
 * context is bounded only by block_size * table_stride < 2^31.
 * Like the reference, page ids are trusted: a negative page id masks its
 * tokens, a page id past the end of the cache is undefined behaviour. Use
 * nvb_paged_fwd_ex to have out-of-range page ids masked as well.
 */
int nvb_paged_fwd(void* stream, const void* q, const void* k, const void* v, void* out,
                  const int* cu_q, const int* kv_lens, const int* block_table, int batch,
                  int total_q, int max_q, int max_k, int q_heads, int kv_heads, int block_size,
                  int table_stride, int num_splits, float* lse, float* lse_accum,
                  float* out_accum);

/* nvb_paged_fwd with the cache extent `num_blocks`: the TMA descriptors are
 * bounded by the cache and page ids outside [0, num_blocks) mask their
 * tokens (as the reference's native kernel does, kernels/kernels.cu:281-282).
 * This is the entry point the library's own host wrappers use. */
int nvb_paged_fwd_ex(void* stream, const void* q, const void* k, const void* v, void* out,
                     const int* cu_q, const int* kv_lens, const int* block_table, int batch,
                     int total_q, int max_q, int max_k, int q_heads, int kv_heads,
                     int block_size, int table_stride, int num_splits, float* lse,
                     float* lse_accum, float* out_accum, int num_blocks);

/* Split-KV decode that allocates nothing, for callers that cannot call
 * cudaMalloc (a plugin inside a host process that owns the CUDA allocator, a
 * fixed device-memory budget): the split partials live in a fixed array in
 * this library's device memory instead of caller-provided lse_accum /
 * out_accum. No counterpart in the reference. Decode only (one query per
 * sequence, total_q == batch); other arguments as nvb_paged_fwd_ex.
 * Limit: num_splits * batch * q_heads <= 16384 (about 8.1 MB held per GPU
 * until exit); larger calls return -1. All calls on a device share the array,
 * so calls that overlap on the GPU race; the first call in each CUDA context
 * (normally one per device) looks up the array's address and should come
 * before any stream capture. */
int nvb_paged_decode_static_scratch(void* stream, const void* q, const void* k, const void* v,
                                    void* out, const int* cu_q, const int* kv_lens,
                                    const int* block_table, int batch, int max_k, int q_heads,
                                    int kv_heads, int block_size, int table_stride,
                                    int num_splits, float* lse, int num_blocks);

/* Split count for decode, replacing `nvr_flash_num_splits`
 * (kernels/flash_native/flash_native.h:31-32, flash_native.cu:17-38).
 * A B200 heuristic: the most (sequence, kv head, split) CTAs that fit one
 * wave of 2 CTAs per SM, with at least 256 KV tokens per split.
 * Pass the physical SM count. Invalid arguments return 0. */
int nvb_num_splits(int batch, int q_heads, int kv_heads, int max_k, int num_sms);

/* Multi-GPU decode over kv-head shards (no counterpart in the reference,
 * which is single-GPU). One process per GPU of a node; rank r holds kv
 * heads [r*kv_heads, (r+1)*kv_heads) of the cache and passes its q
 * [batch, q_heads, 128] (the query heads of those kv heads). The split-KV
 * combine stores each result into every rank's output
 * [batch, world*q_heads, 128] at head offset r*q_heads (peer stores over
 * NVLink), then a one-warp barrier exchanges `epoch` with every rank; when
 * the call's work on `stream` is done, every rank's contributions are in this
 * rank's output. Arguments as nvb_paged_fwd_ex (max_q = 1, no lse) plus:
 *   out_local   [batch, q_heads, 128] BF16 scratch (used when num_splits == 1)
 *   peer_out    host array of `world` device pointers: each rank's output
 *   peer_flag   host array of `world` device pointers: each rank's flags,
 *               at least `world` uint32 starting at 0 (one slot per rank)
 *   epoch       strictly increasing per call (1, 2, ...), the same on every rank
 * Every rank must make the call with the same epoch; a rank that does not
 * leaves the others' barrier to give up after about two seconds, recording
 * device error 7 (nvb_device_error). Output buffers are written by all
 * ranks: alternate two of them between steps, and read step n's output (or
 * enqueue its readers on `stream`) before this rank's next call. A peer one
 * step ahead stores step n + 2 into the same buffer as soon as this rank's
 * step n + 1 has exchanged its epoch, which is before work enqueued after
 * that call runs. The same holds for the two output sets of the capturable
 * form below. */
int nvb_paged_decode_gather(void* stream, const void* q, const void* k, const void* v, void* out_local,
                            const int* cu_q, const int* kv_lens, const int* block_table, int batch, int max_k,
                            int q_heads, int kv_heads, int block_size, int table_stride, int num_blocks,
                            int num_splits, float* lse_accum, float* out_accum, void* const* peer_out,
                            unsigned int* const* peer_flag, int world, int rank, unsigned int epoch);

/* The same step in a form that a CUDA graph can capture once and replay
 * (no host argument changes between steps; no counterpart in the reference).
 * The epoch lives in device memory: peer_flag[rank] needs world + 2 uint32
 * (starting at 0): slot `world` is this rank's step counter, advanced at the
 * end of each step, and slot world + 1 a count of finished combine CTAs (the
 * last one runs the epoch exchange, so a step is two launches, decode and
 * combine, and no separate barrier). Step n (n = 1, 2, ...)
 * writes its results into output set n & 1: peer_out1[p] for odd n,
 * peer_out0[p] for even n, each rank's [batch, world*q_heads, 128] BF16.
 * Every rank must run the same number of steps in the same order; do not
 * mix calls of this form and of nvb_paged_decode_gather on one flag set. */
int nvb_paged_decode_gather_capturable(void* stream, const void* q, const void* k, const void* v, void* out_local,
                                       const int* cu_q, const int* kv_lens, const int* block_table, int batch,
                                       int max_k, int q_heads, int kv_heads, int block_size, int table_stride,
                                       int num_blocks, int num_splits, float* lse_accum, float* out_accum,
                                       void* const* peer_out0, void* const* peer_out1,
                                       unsigned int* const* peer_flag, int world, int rank);

/* Device buffers shared between the ranks of a node through CUDA IPC (the
 * outputs and flags of nvb_paged_decode_gather). create: cudaMalloc `bytes`
 * (zeroed) and write its 64-byte IPC handle; open: map a peer's handle;
 * close: unmap a peer's mapping; free: release this rank's buffer. */
int nvb_peer_buffer_create(size_t bytes, void** ptr, void* ipc_handle);
int nvb_peer_buffer_open(const void* ipc_handle, void** ptr);
int nvb_peer_buffer_close(void* ptr);
int nvb_peer_buffer_free(void* ptr);

/* Attention of drafted trees over the paged cache, for steps that verify
 * several drafted tokens of a sequence at once (no counterpart in the
 * reference, which decodes one token per sequence and step).
 *
 * Sequence b's queries [cu_q[b], cu_q[b + 1]) are the n nodes of its tree in
 * any order; the last n of its kv_lens[b] keys are the same nodes' keys, in
 * the same order, and the keys before them (ctx = kv_lens[b] - n) are visible
 * to every node. tree_mask [total_q, mask_words] says which nodes a node sees:
 * bit (t & 63) of word t / 64 of row i is set where node i attends to node t
 * (itself and its ancestors; nvbh_tree_mask builds it from parents). Where a
 * chain's mask is given this is causal attention.
 *
 *  - max_q bounds every sequence's nodes (at most 64 * mask_words, mask_words
 *    in [1, 16]), max_k its kv_lens. Sequences without nodes, and rows of q
 *    and out before cu_q[0] and from cu_q[batch] on, are left alone.
 *  - lse (may be null) is [total_q, q_heads]. A node that sees no key has
 *    output 0 and lse -inf; so has a sequence with kv_lens < n or longer than
 *    its table.
 *  - num_splits cuts every sequence's keys into that many ranges. Where
 *    parts = nvb_tree_parts(num_splits) > 1 they need lse_accum [parts, total_q,
 *    q_heads] and out_accum [parts, total_q, q_heads, 128] (FP32); calls
 *    that may overlap need their own. nvb_tree_num_splits gives the count for
 *    a GPU of num_sms SMs.
 *  - a key that a node does not see has no part in its result, whatever
 *    values the cache holds there (infinities and NaN too).
 *  - scores, row maxima and sums are FP32; each probability is rounded to BF16
 *    for its product with V, as in this library's other tensor-core kernels:
 *    up to 2^-8 of sum p |v| beside the output's own rounding.
 *  - page ids outside [0, num_blocks) mask their tokens.
 * Other limits as nvb_paged_fwd_ex; batch at most 65535. */
int nvb_paged_tree_fwd(void* stream, const void* q, const void* k, const void* v, void* out,
                       const int* cu_q, const int* kv_lens, const int* block_table,
                       const uint64_t* tree_mask, int mask_words, int batch, int total_q, int max_q,
                       int max_k, int q_heads, int kv_heads, int block_size, int table_stride,
                       int num_splits, float* lse, float* lse_accum, float* out_accum,
                       int num_blocks);
/* Parts of a sequence that num_splits ranges leave in lse_accum / out_accum:
 * 1 where they are joined on chip and the two are not used (they may be null
 * then), else more; 0 for a count outside [1, 128]. */
int nvb_tree_parts(int num_splits);
int nvb_tree_num_splits(int batch, int max_q, int q_heads, int kv_heads, int max_k, int num_sms);

/* Copies within the cache over all layers at once (no counterpart in the
 * reference). k_layers and v_layers are HOST arrays of `layers` device
 * pointers, each a cache [num_blocks, block_size, kv_heads, head_dim] BF16;
 * they are read during the call. At most 1024 layers, 64 in one launch.
 *
 * nvb_cache_copy_pages copies page src_pages[i] to page dst_pages[i] for each
 * of `pairs` pairs (device arrays), the first rows[i] tokens of it where rows
 * is not null: the pages that forked sequences must not share
 * (nvbh_pool_fork). Pairs with a page outside [0, num_blocks) are skipped;
 * there are at most num_blocks pairs.
 * Pairs run in any order: no page may be the target of two pairs, nor the
 * target of one and the source of another.
 *
 * nvb_cache_compact_paths keeps the accepted path of a verified tree: with
 * ctx = kv_lens[b] - n as in nvb_paged_tree_fwd, the K and V rows at position
 * ctx + path[b, d] move to position ctx + d for d in [1, counts[b]), and
 * new_kv_lens[b] = ctx + counts[b] (path and counts as nvbe_layer_verify
 * writes them: strictly increasing from path[b, 0] = 0; path_stride is the
 * row length of path). The pages written must not be shared with another
 * sequence of the batch. */
int nvb_cache_copy_pages(void* stream, void* const* k_layers, void* const* v_layers, int layers,
                         const int* src_pages, const int* dst_pages, const int* rows, int pairs,
                         int kv_heads, int head_dim, int block_size, int num_blocks);
int nvb_cache_compact_paths(void* stream, void* const* k_layers, void* const* v_layers, int layers,
                            const int* cu_q, const int* kv_lens, const int* block_table,
                            const int* path, const int* counts, int* new_kv_lens, int batch,
                            int path_stride, int kv_heads, int head_dim, int block_size,
                            int table_stride, int num_blocks);

/* Latent attention: a cache with one latent vector a token (no counterpart
 * in the reference, whose models keep keys and values a head).
 *
 *   cache   [num_blocks, block_size, 576] bf16: 512 normalised latent values,
 *           then 64 rotated key values that all heads share
 *
 * nvb_latent_store appends a step's tokens. kv holds `rows` rows of 576 values
 * kv_stride elements apart (512 latent values, 64 key values); row r goes to
 * cache slot slots[r] as x * weight / sqrt(mean(x^2) + eps) over the first 512
 * (weight [512] bf16) and the last 64 rotated by position positions[r]. Slots
 * outside [0, block_size * num_blocks) are skipped; no two rows may have the
 * same slot. The rotary parts of the queries are rotated by the same call: q
 * and q_out are the first of `rows` x q_heads parts of 64 values, at row and
 * head strides of their own (in elements), so that they may be slices of
 * longer heads; q_out may be q itself, with the same strides, and must not
 * overlap it otherwise. kv and q_out may be slices of the same rows, beside one
 * another in each. kv may be null (queries only: weight, slots and cache are
 * not used), and so may q (q_heads, q_out and their strides are not used).
 * Pair i of a part is its elements (i, i + 32), or (2i, 2i + 1) with
 * `interleaved`, turned by (cos, sin) = rope_table[position, i] and [position,
 * 32 + i]; rope_table is [max_positions, 64] FP32 (nvbh_rope_table, or
 * nvb_rope_cache with head_dim 64); positions outside it turn by nothing.
 * Values are computed in FP32 and rounded to BF16 once.
 *
 * nvb_latent_gather makes the first cu_k[b + 1] - cu_k[b] cached rows of every
 * sequence contiguous, in order: row cu_k[b] + j of latent (512 values) and of
 * rope (64 values), at strides of their own. The projection that expands
 * latents into keys and values reads `latent`, nvb_latent_prefill_fwd `rope`.
 * Rows of pages outside [0, num_blocks), and behind the page table, are zero;
 * rows before cu_k[0] and from cu_k[batch] on are left alone. latent and rope
 * may be slices of the same rows, beside one another in each.
 *
 * Strides are multiples of 8 elements, all but the int arrays is 16-byte
 * aligned. What these four entry points write must not overlap anything else
 * that they are given (-1). */
int nvb_latent_store(void* stream, const void* kv, long long kv_stride, const void* weight,
                     const int* positions, const int* slots, void* cache, const void* q,
                     long long q_row_stride, long long q_head_stride, void* q_out,
                     long long out_row_stride, long long out_head_stride, int rows, int q_heads,
                     int interleaved, int block_size, int num_blocks, float eps,
                     const float* rope_table, int max_positions);
int nvb_latent_gather(void* stream, const void* cache, const int* block_table, const int* cu_k,
                      void* latent, long long latent_stride, void* rope, long long rope_stride,
                      int batch, int total_k, int block_size, int table_stride, int num_blocks);

/* Absorbed form: attention over the latent cache itself, for decode steps and
 * for short runs of queries (drafts, short chunks). Keys are the cache's rows
 * (576), values their first 512, for all heads the same:
 *
 *   o_i = sum_j p_ij c_j[:512] / sum_j p_ij,  p_ij = exp(scale q_i . c_j)
 *
 * q [total_q, q_heads, 576] has the queries times the expansion of the keys in
 * its first 512 values and the rotated part in its last 64; out [total_q,
 * q_heads, 512] awaits the expansion of the values. Sequence b's queries
 * [cu_q[b], cu_q[b + 1]) are the last of its kv_lens[b] tokens (bottom-right
 * causal mask): query i of n sees the first kv_lens[b] - n + i + 1 keys.
 *
 *  - lse (may be null) is [total_q, q_heads]. A query that sees no key (or
 *    none with a score above -inf) has output 0 and lse -inf; so have all of
 *    a sequence whose kv_lens is negative or longer than its table. Rows
 *    before cu_q[0] and from cu_q[batch] on are left alone. Page ids outside
 *    [0, num_blocks) mask their tokens.
 *  - max_q (the most queries of a sequence) only guides how the work is shared
 *    out; results do not depend on the order in which CTAs run.
 *  - a key that a query does not see has no part in its result, whatever the
 *    cache holds there. A seen key that is not finite makes the result NaN, or,
 *    where its score is -inf, those of its elements that are not finite.
 *  - scores, row maxima and sums are FP32; each probability is rounded to BF16
 *    for its product with the values: up to 2^-8 of sum p |c| beside the
 *    output's own rounding. Those below 2^-125 of a row's largest may count as 0.
 *  - scratch: FP32, nvb_latent_scratch_floats(num_sms) elements for a GPU of
 *    num_sms SMs, whatever the batch (fewer make the call use fewer SMs; at
 *    least nvb_latent_scratch_floats(1)). Nothing is kept in it from one call
 *    for the next; calls that may overlap need their own.
 * Limits: block_size a multiple of 64, q_heads at most 256, batch at most
 * 65535, block_size * table_stride and block_size * num_blocks below 2^31. */
int nvb_paged_latent_fwd(void* stream, const void* q, const void* cache, void* out, const int* cu_q,
                         const int* kv_lens, const int* block_table, int batch, int total_q,
                         int max_q, int q_heads, int block_size, int table_stride, int num_blocks,
                         float scale, float* lse, float* scratch, long long scratch_floats);
long long nvb_latent_scratch_floats(int num_sms);

/* Expanded form: causal attention of prompts and chunks over keys and values
 * that were expanded from latents.
 *
 *   q       [total_q, q_heads, 192]: 128 values, then the 64 rotated ones
 *   kv      [total_k, q_heads, 256]: a head's 128 key values, then its 128 values
 *   k_rope  [total_k] rows of 64 values, rope_stride elements apart: the rotated
 *           part of the keys, the same for all heads
 *   out     [total_q, q_heads, 128]
 *   score   scale * (q[:128] . kv[:128] + q[128:] . k_rope)
 *
 * Sequence b has queries [cu_q[b], cu_q[b + 1]) and keys [cu_k[b], cu_k[b + 1]);
 * its queries are the last of its keys (bottom-right causal mask), so a chunk
 * behind a cached part has that part's keys expanded before its own
 * (nvb_latent_gather). lse (may be null) is [total_q, q_heads]. A query that
 * sees no key has output 0 and lse -inf, so have all of a sequence whose keys
 * are not within [0, total_k]; rows that belong to no sequence are left alone.
 * max_q must be at least the most queries of a sequence: rows past it are left
 * alone too. Keys a query does not see have no part in its result, whatever
 * they hold; a seen value that is not finite makes its element of the output
 * infinite or NaN. Rounding as nvb_paged_latent_fwd. Limits: q_heads at most
 * 256, batch at most 65535. */
int nvb_latent_prefill_fwd(void* stream, const void* q, const void* kv, const void* k_rope,
                           long long rope_stride, void* out, const int* cu_q, const int* cu_k,
                           int batch, int total_q, int total_k, int max_q, int q_heads, float scale,
                           float* lse);

/* Thread-local message for the last failing call on this thread
 * (kernels/flash_native/flash_native.cu:15, kernels/kernels.cu:28). */
const char* nvb_last_error(void);

/* Native-backend-compatible causal paged GQA, replacing `nv_attention`
 * (kernels/kernels.cu:475-485; Rust wrapper src/gpu.rs:829-887) with an
 * explicit stream instead of the reference's Context*. Row r attends to
 * positions[r] + 1 keys of block-table row seq_indices[r]; rows whose
 * sequence or context is invalid get zero output, as in the reference.
 * head_dim 128 (block_size a multiple of 32) runs on the tiled decode;
 * other head sizes from 1 to 512 (any block size) run on a generic CUDA-core
 * kernel, as the reference dispatches head sizes (kernels.cu:226-271,
 * 475-485). Other values are rejected with -1. Requires no scratch. */
int nvb_attention(void* stream, const void* q, const void* kcache, const void* vcache,
                  const int* positions, const int* seq_indices, const int* tables, void* out,
                  int rows, int q_heads, int kv_heads, int head_dim, int block_size,
                  int num_blocks, int table_stride, int batch, int max_context);

/* nvb_attention with split-KV, argument-compatible with the reference's
 * research entry `nv_attention_splitkv_candidate`
 * (kernels/decode_candidate.cuh:111-202, 247): (scratch, partitions)
 * appended. scratch holds rows * q_heads * partitions * (128 + 2) floats;
 * 1 <= partitions <= 128; partitions > 1 needs head_dim 128. */
int nvb_attention_splitkv(void* stream, const void* q, const void* kcache, const void* vcache,
                          const int* positions, const int* seq_indices, const int* tables,
                          void* out, int rows, int q_heads, int kv_heads, int head_dim,
                          int block_size, int num_blocks, int table_stride, int batch,
                          int max_context, float* scratch, int partitions);

/* Fused per-head Q/K RMSNorm + rotate-half RoPE + paged KV store, replacing
 * `nv_qkv_rope_cached` (kernels/kernels.cu:166-211, 474; Rust wrapper
 * src/gpu.rs:775-825) with an explicit stream. qkv is [rows, qh + 2*kvh,
 * dim] bf16 (q heads, then k heads, then v heads). Q goes to qout [rows, qh,
 * dim]; rotated K and copied V go to cache slot slots[row] (slots outside
 * [0, block_size * num_blocks) are skipped). rope_cache is [max_positions,
 * dim] FP32 with cos in columns [0, dim/2) and sin in [dim/2, dim);
 * positions outside [0, max_positions) use cos 1, sin 0. Bit-identical to
 * the reference kernel. dim must be 128. */
int nvb_qkv_rope_cached(void* stream, const void* qkv, const void* q_weight,
                        const void* k_weight, const int* positions, const int* slots,
                        void* qout, void* kcache, void* vcache, int rows, int q_heads,
                        int kv_heads, int head_dim, int block_size, int num_blocks, float eps,
                        const float* rope_cache, int max_positions);

/* Same, computing the rotation angle in-kernel from theta, replacing
 * `nv_qkv_rope` (kernels/kernels.cu:472). */
int nvb_qkv_rope(void* stream, const void* qkv, const void* q_weight, const void* k_weight,
                 const int* positions, const int* slots, void* qout, void* kcache, void* vcache,
                 int rows, int q_heads, int kv_heads, int head_dim, int block_size,
                 int num_blocks, float eps, float theta);

/* Builds the FP32 cos/sin table [positions, dim] for nvb_qkv_rope_cached,
 * replacing `nv_rope_cache` (kernels/kernels.cu:213-224, 473). */
int nvb_rope_cache(void* stream, float* cache, int positions, int head_dim, float theta);

/* CUDA-graph helpers on a caller stream, replacing nv_capture_begin /
 * nv_capture_end / nv_capture_abort / nv_graph_replay / nv_graph_destroy
 * (kernels/kernels.cu:80-97). Capture mode is thread-local, as in the
 * reference. *graph receives a cudaGraphExec_t. */
int nvb_capture_begin(void* stream);
int nvb_capture_end(void* stream, void** graph);
void nvb_capture_abort(void* stream);
int nvb_graph_replay(void* graph, void* stream);
void nvb_graph_destroy(void* graph);

/* Device-side error word written by bounded pipeline waits (0 = none).
 * Reading it synchronizes the device; it is a diagnostic, not for the
 * step loop. No counterpart in the reference, whose kernels do not spin. */
int nvb_device_error(int* code);
int nvb_clear_device_error(void);

/* Library version string. */
const char* nvb_version(void);

#ifdef __cplusplus
}
#endif

#endif /* NVB_ATTENTION_H */
