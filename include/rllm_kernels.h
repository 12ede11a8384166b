/*
 * rllm_kernels.h — C ABI of the MI355X (gfx950) paged-attention library.
 *
 * The library is a drop-in for rLLM's `rllm-kernels` FFI: every symbol the
 * reference's Rust code binds is exported here with the same name, argument
 * order and meaning, and the same error convention:
 *   - return 0 on success, otherwise a non-zero hipError_t value;
 *   - empty work (num_seqs <= 0 / num_tokens <= 0 / nbytes <= 0) returns 0
 *     without launching;
 *   - `stream` is a hipStream_t passed as an integer, 0 = default stream;
 *   - `_sync` variants launch on stream 0 and then hipDeviceSynchronize();
 *   - all pointers are caller-owned DEVICE pointers (the callee never frees);
 *   - invalid arguments (null pointers, shapes outside the supported set) are
 *     rejected on the host with hipErrorInvalidValue (1) before any launch.
 *
 * Layouts (crates/rllm-kernels/src/cuda/paged_attention.cu:82-86,245-250):
 *   q, out        [num_seqs | num_tokens, num_q_heads, head_dim]
 *   K / V cache   [num_blocks, num_kv_heads, head_dim, block_size]   (NHD)
 *   block_tables  [num_seqs, max_num_blocks_per_seq] int32, -1 = unused
 *   seq_lens      [num_seqs] int32 (KV length including the new token)
 *   query_start_loc [num_seqs + 1] int32 prefix sum of query tokens
 *   slot_mapping  [num_tokens] int64, slot = block * block_size + offset, -1 = skip
 * GQA: q head qh reads kv head qh * num_kv_heads / num_q_heads
 * (crates/rllm-kernels/src/attention.rs:40-42).
 *
 * Attention entry points accept the shapes the reference kernels accept
 * (paged_attention.cu:199-200, 369-370): any head_dim up to 1024, any block
 * size up to 4096 and num_q_heads a multiple of num_kv_heads.  head_dim 64 /
 * 128 with block_size 16 and num_q_heads / num_kv_heads in {1, 2, 4, 8} run
 * the tuned kernels; every other shape runs the shape-general kernels
 * (partition_size is ignored).  They split long contexts over scratch, which
 * is library-owned per (device, stream), and run unsplit where there is none: a
 * decode captured on a stream that has no scratch yet, any captured prefill,
 * rllm_paged_attention_decode_noalloc, or no memory left.  A decode that is
 * given a workspace takes no library scratch: it splits over the workspace, past
 * the arrival counters at its start, or, where that is too small, not at all
 * (32 KiB + num_seqs * num_q_heads * 64 * (head_dim + 2) * 4 bytes always do;
 * any non-null one, however small, keeps the library's scratch out).
 * Cache writes accept any shape.
 *
 * Alignment in bytes for the tuned attention kernels: caches 16 (FP8: 8), prefill
 * queries 16 and outputs 8, decode queries 4 and outputs 2.  The shape-general
 * kernels take any; queries, outputs or caches short of 16 (FP8 caches: 8) leave
 * the matrix cores out.
 *
 * Differences from the reference kernels, all deliberate:
 *   - a sequence with seq_len <= 0 gets an all-zero output row (the reference
 *     leaves it unwritten, paged_attention.cu:110);
 *   - prefill masks causally at absolute positions: query i of a sequence with
 *     n new tokens attends keys 0 .. seq_len - n + i (the reference uses
 *     0 .. i, paged_attention.cu:285-286, which ignores cached context);
 *   - E4M3 encoding saturates inputs in [480, 512) to 0x7E (the reference text
 *     yields the NaN byte 0x7F, cache_ops.cu:44);
 *   - FP8 bytes decode per OCP E4M3FN / E5M2 (the reference decoder mis-scales
 *     E4M3 subnormals, cache_ops.cu:58; its encoder never emits them).
 */
#ifndef RLLM_KERNELS_H
#define RLLM_KERNELS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element type codes of the *_ex / *_scaled entry points
 * (crates/rllm-core/src/dtype.rs:3-26) */
#define RLLM_DTYPE_F16 0
#define RLLM_DTYPE_BF16 1
#define RLLM_DTYPE_FP8_E4M3 2
#define RLLM_DTYPE_FP8_E5M2 3

/* ======================================================================
 * Decode paged attention (one query token per sequence)
 * ==================================================================== */

/* Replaces rllm_paged_attention_decode_f16, paged_attention.cu:181-210;
 * bound at crates/rllm-kernels/src/attention.rs:268-283.  f16 Q/KV/out. */
int32_t rllm_paged_attention_decode_f16(uint16_t *output, const uint16_t *query,
                                        const uint16_t *key_cache, const uint16_t *value_cache,
                                        const int32_t *block_tables, const int32_t *seq_lens,
                                        int64_t num_seqs, int64_t num_q_heads,
                                        int64_t num_kv_heads, int64_t head_dim,
                                        int64_t block_size, int64_t max_num_blocks_per_seq,
                                        float scale, uintptr_t stream);
/* Replaces rllm_paged_attention_decode_f16_sync, paged_attention.cu:212-235;
 * bound at attention.rs:320-334. */
int32_t rllm_paged_attention_decode_f16_sync(uint16_t *output, const uint16_t *query,
                                             const uint16_t *key_cache,
                                             const uint16_t *value_cache,
                                             const int32_t *block_tables,
                                             const int32_t *seq_lens, int64_t num_seqs,
                                             int64_t num_q_heads, int64_t num_kv_heads,
                                             int64_t head_dim, int64_t block_size,
                                             int64_t max_num_blocks_per_seq, float scale);

/* Replaces rllm_paged_attention_decode_fp8, paged_attention.cu:603-633;
 * bound at attention.rs:285-301.  f16 Q/out, FP8 KV bytes (E4M3, or E5M2 when
 * is_e5m2 != 0), no scale (k_scale = v_scale = 1). */
int32_t rllm_paged_attention_decode_fp8(uint16_t *output, const uint16_t *query,
                                        const uint8_t *key_cache, const uint8_t *value_cache,
                                        const int32_t *block_tables, const int32_t *seq_lens,
                                        int64_t num_seqs, int64_t num_q_heads,
                                        int64_t num_kv_heads, int64_t head_dim,
                                        int64_t block_size, int64_t max_num_blocks_per_seq,
                                        float scale, int32_t is_e5m2, uintptr_t stream);
/* Replaces rllm_paged_attention_decode_fp8_sync, paged_attention.cu:635-659;
 * bound at attention.rs:303-318. */
int32_t rllm_paged_attention_decode_fp8_sync(uint16_t *output, const uint16_t *query,
                                             const uint8_t *key_cache,
                                             const uint8_t *value_cache,
                                             const int32_t *block_tables,
                                             const int32_t *seq_lens, int64_t num_seqs,
                                             int64_t num_q_heads, int64_t num_kv_heads,
                                             int64_t head_dim, int64_t block_size,
                                             int64_t max_num_blocks_per_seq, float scale,
                                             int32_t is_e5m2);

/* New: bf16 Q/KV/out, same arguments as rllm_paged_attention_decode_f16
 * (the reference converts bf16 K/V to f16 first, layers.rs:400-402). */
int32_t rllm_paged_attention_decode_bf16(uint16_t *output, const uint16_t *query,
                                         const uint16_t *key_cache, const uint16_t *value_cache,
                                         const int32_t *block_tables, const int32_t *seq_lens,
                                         int64_t num_seqs, int64_t num_q_heads,
                                         int64_t num_kv_heads, int64_t head_dim,
                                         int64_t block_size, int64_t max_num_blocks_per_seq,
                                         float scale, uintptr_t stream);
int32_t rllm_paged_attention_decode_bf16_sync(uint16_t *output, const uint16_t *query,
                                              const uint16_t *key_cache,
                                              const uint16_t *value_cache,
                                              const int32_t *block_tables,
                                              const int32_t *seq_lens, int64_t num_seqs,
                                              int64_t num_q_heads, int64_t num_kv_heads,
                                              int64_t head_dim, int64_t block_size,
                                              int64_t max_num_blocks_per_seq, float scale);

/* New: general decode.
 *   q_dtype   RLLM_DTYPE_F16 | RLLM_DTYPE_BF16 (the output has the same type)
 *   kv_dtype  q_dtype, RLLM_DTYPE_FP8_E4M3 or RLLM_DTYPE_FP8_E5M2
 *   k_scale, v_scale  per-tensor dequantisation scales of an FP8 cache
 *             (cache value = byte value * scale); ignored for 16-bit caches
 *   partition_size  0 = automatic (stream split: up to one wave per SIMD for
 *             a 16-bit cache, two for FP8, each taking an equal share of all
 *             sequences' cache blocks; a sequence cut
 *             between waves is merged by the last wave to finish a piece of
 *             it, in the same kernel, summing the pieces in a fixed order,
 *             so repeated calls on the same inputs return the same bits
 *             whichever wave merges), < 0 = single pass (one wave per
 *             sequence and kv head), > 0 = context tokens per split-K
 *             partition (a multiple of 512; a second kernel merges)
 *   workspace, workspace_bytes  split-K scratch of at least
 *             rllm_paged_attention_decode_workspace_size(...) bytes; NULL =
 *             use a library-owned buffer cached per (device, stream, mode).
 *             With partition_size 0 the buffer holds arrival counters: it must
 *             be zero-filled before its first such call (and again after any
 *             other use); each completed call leaves it ready for the next.
 *             Calls that share a workspace must not overlap in time. */
int32_t rllm_paged_attention_decode_ex(void *output, const void *query, const void *key_cache,
                                       const void *value_cache, const int32_t *block_tables,
                                       const int32_t *seq_lens, int64_t num_seqs,
                                       int64_t num_q_heads, int64_t num_kv_heads,
                                       int64_t head_dim, int64_t block_size,
                                       int64_t max_num_blocks_per_seq, float scale,
                                       int32_t q_dtype, int32_t kv_dtype, float k_scale,
                                       float v_scale, int64_t partition_size, void *workspace,
                                       int64_t workspace_bytes, uintptr_t stream);

/* New: decode of a batch whose block tables share a prefix, the cascade
 * form of rllm_paged_attention_decode_ex for the shared prefixes that
 * AttentionMetadata::detect_common_prefix_blocks (attention.rs:204-226)
 * finds.  The reference has the detection but no kernel that uses it.
 *   num_prefix_blocks  the first num_prefix_blocks entries of every table
 *             are the same physical blocks, and every sequence's context
 *             covers them (seq_lens[s] >= num_prefix_blocks * block_size).
 *             A shorter context is still attended correctly, but the prefix
 *             block's slots past every sequence's context must then hold
 *             finite values.  0 runs the plain decode.
 * The prefix's keys and values are read once per kv head for the whole
 * batch, with matrix cores; each sequence's blocks past the prefix are
 * attended separately (in the same kernel launch), and a reduction merges
 * the two in the log-sum-exp domain.  The result equals rllm_paged_attention_decode_ex's within
 * rounding.  Shapes outside the tuned set (head_dim 64 / 128, block size 16,
 * GQA 1 / 2 / 4 / 8), f16 queries whose scale * log2(e) (* k_scale)
 * exceeds 1, and batches whose prefix saves too little run the plain decode:
 * the cascade is used when (num_seqs - 1) * num_prefix_blocks is at least
 * 3/5 of num_seqs * (max_blocks_per_seq - num_prefix_blocks) and, times
 * num_kv_heads, at least 10000 (the environment variable RLLM_CASCADE=always
 * or =never overrides this, read on every call).  Scratch is library-owned per (device,
 * stream); calls on one stream must not be captured unless an eager call of
 * the same or a larger shape ran on that stream before (a capture with too
 * small a buffer runs the plain decode instead). */
int32_t rllm_paged_attention_decode_prefix_ex(void *output, const void *query, const void *key_cache,
                                              const void *value_cache, const int32_t *block_tables,
                                              const int32_t *seq_lens, int64_t num_seqs,
                                              int64_t num_q_heads, int64_t num_kv_heads,
                                              int64_t head_dim, int64_t block_size,
                                              int64_t max_num_blocks_per_seq, float scale,
                                              int32_t q_dtype, int32_t kv_dtype, float k_scale,
                                              float v_scale, int64_t num_prefix_blocks,
                                              uintptr_t stream);

/* New: one step's attention over a mixed batch, in place of the pair of
 * calls the reference's ModelRunner::run_paged_attention makes "depending on
 * the batch composition" (model_runner.rs:404-414): the prefill group is
 * rllm_paged_attention_prefill_ex's arguments (prefill_*), the decode group
 * rllm_paged_attention_decode_ex's with partition_size 0 and no workspace
 * (decode_*), over the same caches, heads and scales.  The two groups'
 * outputs and queries are separate arrays (they may be two row ranges of one
 * buffer).  With the tuned shapes both groups run in one kernel launch: the
 * prefill workgroups (256 query rows each: 64 tokens at GQA 4) on their own
 * CUs, the decode beside them on the other CUs, or, when the prefill takes
 * more than half of the CUs, on every CU as the prefill leaves it.  Shapes
 * outside the tuned set, f16 queries whose scale * log2(e) (* k_scale)
 * exceeds 1, and an empty group run the two entry points in series.  Results
 * equal the two entry points' within rounding (the prefill group is never
 * split over its KV range in the one launch).  Scratch is the decode's library-owned stream workspace, per
 * (device, stream); a capture on a stream without it runs in series. */
int32_t rllm_paged_attention_mixed_ex(void *prefill_output, const void *prefill_query,
                                      const int32_t *prefill_block_tables, const int32_t *prefill_seq_lens,
                                      const int32_t *prefill_query_start_loc, int64_t prefill_num_seqs,
                                      int64_t prefill_num_tokens, int64_t prefill_max_blocks,
                                      void *decode_output, const void *decode_query,
                                      const int32_t *decode_block_tables, const int32_t *decode_seq_lens,
                                      int64_t decode_num_seqs, int64_t decode_max_blocks,
                                      const void *key_cache, const void *value_cache,
                                      int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                      int64_t block_size, float scale, int32_t q_dtype, int32_t kv_dtype,
                                      float k_scale, float v_scale, uintptr_t stream);

/* New: bytes of split-K workspace rllm_paged_attention_decode_ex needs for
 * these shapes on the current device (0 when nothing is split); negative on
 * invalid arguments. */
int64_t rllm_paged_attention_decode_workspace_size(int64_t num_seqs, int64_t num_q_heads,
                                                   int64_t num_kv_heads, int64_t head_dim,
                                                   int64_t block_size,
                                                   int64_t max_num_blocks_per_seq,
                                                   int64_t partition_size);

/* New, no counterpart in the reference: rllm_paged_attention_decode_ex with
 * no workspace argument, for callers that cannot allocate device memory (code
 * under hipGraph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  It calls no hipMalloc, hipFree or allocating library routine:
 * its scratch is one fixed device array of RLLM_DECODE_NOALLOC_SCRATCH_BYTES
 * per GPU, held from library load until the process ends.  The array starts
 * with the stream mode's arrival counters (4 bytes per resident wave of the
 * device, rounded up to 256: 32 KiB on MI355X); split-K partials
 * (partition_size > 0) are placed after them, so calls of either mode may
 * follow each other in any order.  A call that would need more scratch than
 * the array holds (rllm_paged_attention_decode_workspace_size gives the
 * figure; split-K adds the counters' bytes to it) returns hipErrorOutOfMemory
 * (2) before any launch; the stream mode of every tuned shape fits.  All calls
 * on one GPU share the array, whatever their stream: calls that overlap in
 * time on one GPU race and must be serialised by the caller.  The first call
 * on a device clears the counters with a kernel on `stream` and must not be
 * made under stream capture (it returns hipErrorStreamCaptureUnsupported
 * then); later calls may be captured. */
#define RLLM_DECODE_NOALLOC_SCRATCH_BYTES (24ll << 20)
int32_t rllm_paged_attention_decode_noalloc(void *output, const void *query,
                                            const void *key_cache, const void *value_cache,
                                            const int32_t *block_tables, const int32_t *seq_lens,
                                            int64_t num_seqs, int64_t num_q_heads,
                                            int64_t num_kv_heads, int64_t head_dim,
                                            int64_t block_size, int64_t max_num_blocks_per_seq,
                                            float scale, int32_t q_dtype, int32_t kv_dtype,
                                            float k_scale, float v_scale, int64_t partition_size,
                                            uintptr_t stream);

/* ======================================================================
 * Prefill / chunked-prefill paged attention (MFMA)
 * ==================================================================== */

/* Replaces rllm_paged_attention_prefill_f16, paged_attention.cu:349-380;
 * bound at attention.rs:336-354.  The new tokens' K/V must already be in the
 * cache (the caller writes them first, layers.rs:414-447). */
int32_t rllm_paged_attention_prefill_f16(uint16_t *output, const uint16_t *query,
                                         const uint16_t *key_cache, const uint16_t *value_cache,
                                         const int32_t *block_tables, const int32_t *seq_lens,
                                         const int32_t *query_start_loc, int64_t num_seqs,
                                         int64_t num_tokens, int64_t num_q_heads,
                                         int64_t num_kv_heads, int64_t head_dim,
                                         int64_t block_size, int64_t max_num_blocks_per_seq,
                                         float scale, uintptr_t stream);
/* Replaces rllm_paged_attention_prefill_f16_sync, paged_attention.cu:382-407;
 * bound at attention.rs:377-393. */
int32_t rllm_paged_attention_prefill_f16_sync(uint16_t *output, const uint16_t *query,
                                              const uint16_t *key_cache,
                                              const uint16_t *value_cache,
                                              const int32_t *block_tables,
                                              const int32_t *seq_lens,
                                              const int32_t *query_start_loc, int64_t num_seqs,
                                              int64_t num_tokens, int64_t num_q_heads,
                                              int64_t num_kv_heads, int64_t head_dim,
                                              int64_t block_size,
                                              int64_t max_num_blocks_per_seq, float scale);
/* Replaces rllm_paged_attention_prefill_fp8, paged_attention.cu:661-693;
 * bound at attention.rs:356-374. */
int32_t rllm_paged_attention_prefill_fp8(uint16_t *output, const uint16_t *query,
                                         const uint8_t *key_cache, const uint8_t *value_cache,
                                         const int32_t *block_tables, const int32_t *seq_lens,
                                         const int32_t *query_start_loc, int64_t num_seqs,
                                         int64_t num_tokens, int64_t num_q_heads,
                                         int64_t num_kv_heads, int64_t head_dim,
                                         int64_t block_size, int64_t max_num_blocks_per_seq,
                                         float scale, int32_t is_e5m2, uintptr_t stream);
/* Replaces rllm_paged_attention_prefill_fp8_sync, paged_attention.cu:695-721;
 * bound at attention.rs:395-412. */
int32_t rllm_paged_attention_prefill_fp8_sync(uint16_t *output, const uint16_t *query,
                                              const uint8_t *key_cache,
                                              const uint8_t *value_cache,
                                              const int32_t *block_tables,
                                              const int32_t *seq_lens,
                                              const int32_t *query_start_loc, int64_t num_seqs,
                                              int64_t num_tokens, int64_t num_q_heads,
                                              int64_t num_kv_heads, int64_t head_dim,
                                              int64_t block_size,
                                              int64_t max_num_blocks_per_seq, float scale,
                                              int32_t is_e5m2);
/* New: bf16 Q/KV/out, same arguments as rllm_paged_attention_prefill_f16. */
int32_t rllm_paged_attention_prefill_bf16(uint16_t *output, const uint16_t *query,
                                          const uint16_t *key_cache,
                                          const uint16_t *value_cache,
                                          const int32_t *block_tables, const int32_t *seq_lens,
                                          const int32_t *query_start_loc, int64_t num_seqs,
                                          int64_t num_tokens, int64_t num_q_heads,
                                          int64_t num_kv_heads, int64_t head_dim,
                                          int64_t block_size, int64_t max_num_blocks_per_seq,
                                          float scale, uintptr_t stream);
int32_t rllm_paged_attention_prefill_bf16_sync(uint16_t *output, const uint16_t *query,
                                               const uint16_t *key_cache,
                                               const uint16_t *value_cache,
                                               const int32_t *block_tables,
                                               const int32_t *seq_lens,
                                               const int32_t *query_start_loc,
                                               int64_t num_seqs, int64_t num_tokens,
                                               int64_t num_q_heads, int64_t num_kv_heads,
                                               int64_t head_dim, int64_t block_size,
                                               int64_t max_num_blocks_per_seq, float scale);
/* New: general prefill with dtype codes and FP8 scales as in *_decode_ex. */
int32_t rllm_paged_attention_prefill_ex(void *output, const void *query, const void *key_cache,
                                        const void *value_cache, const int32_t *block_tables,
                                        const int32_t *seq_lens,
                                        const int32_t *query_start_loc, int64_t num_seqs,
                                        int64_t num_tokens, int64_t num_q_heads,
                                        int64_t num_kv_heads, int64_t head_dim,
                                        int64_t block_size, int64_t max_num_blocks_per_seq,
                                        float scale, int32_t q_dtype, int32_t kv_dtype,
                                        float k_scale, float v_scale, uintptr_t stream);

/* ======================================================================
 * KV cache write (reshape_and_cache), block copy, zero, allocation
 * ==================================================================== */

/* Replaces rllm_cache_write_f16, cache_ops.cu:202-225; bound at
 * crates/rllm-kernels/src/cache_ops.rs:22-34.  16-bit bit copy, so it is
 * equally correct for bf16 data. */
int32_t rllm_cache_write_f16(uint16_t *key_cache, uint16_t *value_cache, const uint16_t *new_key,
                             const uint16_t *new_value, const int64_t *slot_mapping,
                             int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
                             int64_t block_size, int64_t num_blocks, uintptr_t stream);
/* Replaces rllm_cache_write_f16_sync, cache_ops.cu:227-246; bound at
 * cache_ops.rs:51-62. */
int32_t rllm_cache_write_f16_sync(uint16_t *key_cache, uint16_t *value_cache,
                                  const uint16_t *new_key, const uint16_t *new_value,
                                  const int64_t *slot_mapping, int64_t num_tokens,
                                  int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                  int64_t num_blocks);
/* New: bf16 alias of rllm_cache_write_f16. */
int32_t rllm_cache_write_bf16(uint16_t *key_cache, uint16_t *value_cache, const uint16_t *new_key,
                              const uint16_t *new_value, const int64_t *slot_mapping,
                              int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
                              int64_t block_size, int64_t num_blocks, uintptr_t stream);
/* Replaces rllm_cache_write_fp8, cache_ops.cu:366-390; bound at
 * cache_ops.rs:36-49.  f16 input, unscaled FP8 bytes. */
int32_t rllm_cache_write_fp8(uint8_t *key_cache, uint8_t *value_cache, const uint16_t *new_key,
                             const uint16_t *new_value, const int64_t *slot_mapping,
                             int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
                             int64_t block_size, int64_t num_blocks, int32_t is_e5m2,
                             uintptr_t stream);
/* Replaces rllm_cache_write_fp8_sync, cache_ops.cu:392-412; bound at
 * cache_ops.rs:64-76. */
int32_t rllm_cache_write_fp8_sync(uint8_t *key_cache, uint8_t *value_cache,
                                  const uint16_t *new_key, const uint16_t *new_value,
                                  const int64_t *slot_mapping, int64_t num_tokens,
                                  int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                  int64_t num_blocks, int32_t is_e5m2);
/* New: FP8 write of x / scale with per-tensor scales; input_dtype is
 * RLLM_DTYPE_F16 or RLLM_DTYPE_BF16.  The quotient is correctly rounded fp32,
 * the byte follows the reference rounding contract (round toward zero). */
int32_t rllm_cache_write_fp8_scaled(uint8_t *key_cache, uint8_t *value_cache,
                                    const uint16_t *new_key, const uint16_t *new_value,
                                    const int64_t *slot_mapping, int64_t num_tokens,
                                    int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                    int64_t num_blocks, int32_t input_dtype, float k_scale,
                                    float v_scale, int32_t is_e5m2, uintptr_t stream);

/* New: FP8 write of x / scale with a choice of rounding.  cache_dtype is
 * RLLM_DTYPE_FP8_E4M3 or RLLM_DTYPE_FP8_E5M2; rounding is
 *   RLLM_FP8_ROUND_TOWARD_ZERO    the reference contract (cache_ops.cu:13-46,
 *                                 75-103), identical to rllm_cache_write_fp8_scaled;
 *   RLLM_FP8_ROUND_NEAREST_EVEN   OCP rounding to nearest, ties to even, with
 *                                 FP8 subnormals (gradual underflow); values
 *                                 at or above the largest finite value and
 *                                 infinities saturate to it, NaN -> 0x7F.
 * Round toward zero shrinks every stored magnitude (by about 4% on average
 * for E4M3); nearest-even removes that bias.  Both decode with the same
 * attention kernels.  Other arguments as rllm_cache_write_fp8_scaled. */
#define RLLM_FP8_ROUND_TOWARD_ZERO 0
#define RLLM_FP8_ROUND_NEAREST_EVEN 1
int32_t rllm_cache_write_fp8_ex(uint8_t *key_cache, uint8_t *value_cache, const uint16_t *new_key,
                                const uint16_t *new_value, const int64_t *slot_mapping,
                                int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
                                int64_t block_size, int64_t num_blocks, int32_t input_dtype,
                                float k_scale, float v_scale, int32_t cache_dtype,
                                int32_t rounding, uintptr_t stream);

/* New (additive): rotary position embedding fused with the cache write.  It
 * replaces the model-side sequence RotaryEmbedding::apply (rope.rs:34-43,
 * 57-82: q and k rotated by halves, x*cos + rotate_half(x)*sin in the
 * activation dtype) followed by rllm_cache_write_* (cache_ops.cu:161-200,
 * 322-364) with one launch.  fused.cu:168-256 (rllm_fused_rope_f16, an
 * interleaved-pair rotation no caller binds) is not what the model computes.
 *   q, q_out    [num_tokens, num_q_heads, head_dim] of dtype; q_out == q is
 *               allowed (in place); both may be NULL when num_q_heads == 0
 *   k, v        [num_tokens, num_kv_heads, head_dim] of dtype; the rotated k
 *               and v go to the caches, k and v are not modified
 *   positions   int32 [num_tokens], clamped to [0, max_position)
 *   cos_cache,  f32 [max_position, head_dim/2] as RotaryEmbedding::new builds
 *   sin_cache   them (rope.rs:13-33); cast to dtype before use
 *   dtype       RLLM_DTYPE_F16 | RLLM_DTYPE_BF16
 *   kv_dtype    dtype, RLLM_DTYPE_FP8_E4M3 or RLLM_DTYPE_FP8_E5M2 (FP8 bytes =
 *               encode(x / scale), as rllm_cache_write_fp8_scaled)
 * slot_mapping < 0 (padding) or a block >= num_blocks skips the cache write of
 * that token; q is still rotated.  head_dim must be a multiple of 16, and q,
 * q_out, k, v, cos_cache and sin_cache 16-byte aligned. */
int32_t rllm_rope_cache_write(void *q_out, const void *q, const void *k, const void *v,
                              void *key_cache, void *value_cache, const int64_t *slot_mapping,
                              const int32_t *positions, const float *cos_cache,
                              const float *sin_cache, int64_t num_tokens, int64_t num_q_heads,
                              int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                              int64_t num_blocks, int64_t max_position, int32_t dtype,
                              int32_t kv_dtype, float k_scale, float v_scale, uintptr_t stream);

/* New: rllm_rope_cache_write with a choice of FP8 rounding (fp8_rounding is
 * RLLM_FP8_ROUND_TOWARD_ZERO, which rllm_rope_cache_write uses, or
 * RLLM_FP8_ROUND_NEAREST_EVEN; see rllm_cache_write_fp8_ex).  Ignored for
 * 16-bit caches. */
int32_t rllm_rope_cache_write_ex(void *q_out, const void *q, const void *k, const void *v,
                                 void *key_cache, void *value_cache, const int64_t *slot_mapping,
                                 const int32_t *positions, const float *cos_cache,
                                 const float *sin_cache, int64_t num_tokens, int64_t num_q_heads,
                                 int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                 int64_t num_blocks, int64_t max_position, int32_t dtype,
                                 int32_t kv_dtype, float k_scale, float v_scale,
                                 int32_t fp8_rounding, uintptr_t stream);

/* New (additive), host only: fills the f32 cos / sin tables
 * [max_position, head_dim/2] that rllm_rope_cache_write reads, as
 * RotaryEmbedding::new computes them (rope.rs:13-33: f64 angles, f32 store).
 * Both pointers are HOST memory; no GPU call is made. */
int32_t rllm_rope_tables(float *cos_cache, float *sin_cache, int64_t max_position,
                         int64_t head_dim, float theta);

/* Replace rllm_fused_rmsnorm_f16(_sync) and rllm_fused_silu_mul_f16(_sync),
 * fused.cu:20-166; bound at fused.rs:18-51.  They compute the model's ops
 * rather than fused.cu's kernels (whose RMSNorm reduces per CUDA block, wrong
 * for rows longer than one block):
 *   RMSNorm  (layers.rs:128-140): per row of hidden_size elements,
 *            y = x / sqrt(mean(x^2) + eps) * weight in f32, rounded to the dtype
 *   SiLU-mul (layers.rs:214-220): out = silu(gate) * up in the dtype, silu(x)
 *            = x / (1 + exp(-x)) with each op rounded to the dtype
 * n_elements must be a multiple of hidden_size, hidden_size a multiple of 8
 * and the RMSNorm pointers 16-byte aligned (hipErrorInvalidValue otherwise). */
int32_t rllm_fused_rmsnorm_f16(uint16_t *output, const uint16_t *input, const uint16_t *weight,
                               int64_t hidden_size, int64_t n_elements, float eps, uintptr_t stream);
int32_t rllm_fused_rmsnorm_f16_sync(uint16_t *output, const uint16_t *input, const uint16_t *weight,
                                    int64_t hidden_size, int64_t n_elements, float eps);
int32_t rllm_fused_silu_mul_f16(uint16_t *output, const uint16_t *gate, const uint16_t *up,
                                int64_t n_elements, uintptr_t stream);
int32_t rllm_fused_silu_mul_f16_sync(uint16_t *output, const uint16_t *gate, const uint16_t *up,
                                     int64_t n_elements);
/* New: the same for dtype RLLM_DTYPE_F16 or RLLM_DTYPE_BF16. */
int32_t rllm_rmsnorm_ex(void *output, const void *input, const void *weight, int64_t hidden_size,
                        int64_t n_elements, float eps, int32_t dtype, uintptr_t stream);
int32_t rllm_silu_mul_ex(void *output, const void *gate, const void *up, int64_t n_elements,
                         int32_t dtype, uintptr_t stream);

/* Replaces rllm_cache_block_copy(_sync), cache_ops.cu:264-292; bound at
 * cache_ops.rs:80-94. */
int32_t rllm_cache_block_copy(const uint8_t *src, uint8_t *dst, int64_t block_nbytes,
                              int64_t num_blocks, uintptr_t stream);
int32_t rllm_cache_block_copy_sync(const uint8_t *src, uint8_t *dst, int64_t block_nbytes,
                                   int64_t num_blocks);
/* Replaces rllm_cache_zero(_sync), cache_ops.cu:304-320; bound at
 * cache_ops.rs:96-97. */
int32_t rllm_cache_zero(uint8_t *ptr, int64_t nbytes, uintptr_t stream);
int32_t rllm_cache_zero_sync(uint8_t *ptr, int64_t nbytes);

/* New (additive): batched block copy for copy-on-write.  BlockPool::
 * copy_on_write (crates/rllm-cache/src/block_pool.rs:286-302) hands the caller
 * a fresh block whose bytes must be copied from the shared one with
 * rllm_cache_block_copy, one contiguous range per layer and per K/V
 * (cache_ops.cu:252-292); this copies a whole list in one launch.
 *   key_caches, value_caches  DEVICE arrays of num_layers cache base addresses
 *                             (each [num_blocks, Hkv, D, bs], block_nbytes per block)
 *   block_pairs               DEVICE int64 [num_pairs, 2]: (src, dst) block ids
 * Pairs with an id outside [0, num_blocks) or src == dst are skipped.  The
 * destinations must be distinct and must not be sources of other pairs. */
int32_t rllm_cache_copy_blocks(const uint64_t *key_caches, const uint64_t *value_caches,
                               int64_t num_layers, const int64_t *block_pairs, int64_t num_pairs,
                               int64_t num_blocks, int64_t block_nbytes, uintptr_t stream);

/* New (additive): swap of whole blocks between the paged caches and pinned host
 * records, the data movement behind CpuKvOffloadStore::put / get
 * (crates/rllm-cache/src/offload.rs:28-74).  host_records holds num_records
 * records of num_layers * 2 * block_nbytes bytes (the store's
 * block_size_bytes), each [layer][K, V][block_nbytes]; block block_ids[i] goes
 * to / comes from record record_slots[i] (record i when record_slots is NULL,
 * then num_records >= num_ids).  host_records must be pinned host memory from
 * hipHostMalloc / rllm_gpu_alloc_host (the kernel reads or writes it
 * directly; any other pointer returns hipErrorInvalidValue before a launch);
 * block_ids and record_slots are DEVICE int64 arrays.  Ids outside
 * [0, num_blocks) and slots outside [0, num_records) are skipped.  Synchronise
 * the stream before the host reads swapped-out records. */
int32_t rllm_cache_swap_out(const uint64_t *key_caches, const uint64_t *value_caches,
                            int64_t num_layers, const int64_t *block_ids, int64_t num_ids,
                            int64_t num_blocks, int64_t block_nbytes, const int64_t *record_slots,
                            int64_t num_records, void *host_records, uintptr_t stream);
int32_t rllm_cache_swap_in(const uint64_t *key_caches, const uint64_t *value_caches,
                           int64_t num_layers, const int64_t *block_ids, int64_t num_ids,
                           int64_t num_blocks, int64_t block_nbytes, const int64_t *record_slots,
                           int64_t num_records, const void *host_records, uintptr_t stream);

/* ======================================================================
 * MXFP4 KV cache: 4-bit codes with a scale per 32 elements
 * ==================================================================== */

/* New (additive).  One layer's keys (and values) are uint8
 * [num_blocks, num_kv_heads, page], page = rllm_mxfp4_page_bytes(head_dim,
 * block_size) = block_size * head_dim * 17 / 32 bytes: block_size rows (one a
 * token) of head_dim / 2 code bytes, then block_size rows of head_dim / 32 scale
 * bytes.  Byte i of a code row holds elements 2i (low four bits) and 2i + 1: sign,
 * two exponent bits, one mantissa bit (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6).  Scale
 * byte j (E8M0) stands for 2^(e - 127), the factor of elements 32j .. 32j + 31; 255
 * makes them NaN.  A block is num_kv_heads * page contiguous bytes, so
 * rllm_cache_copy_blocks, rllm_cache_swap_out / _in, rllm_cache_block_copy and
 * rllm_cache_zero move these caches as they are (zeroed pages read as zeros).
 * Shapes: head_dim a multiple of 32 up to 256, block_size a multiple of 16 up to
 * 4096, at most 1024 kv heads and 1024 q heads, caches 16-byte aligned; anything
 * else returns hipErrorInvalidValue.  slot_mapping is as for the other cache
 * writes; a block id of a table outside [0, num_blocks) is an unused entry. */

/* Bytes of a (block, kv head) page; -1 for a shape outside the above. */
int64_t rllm_mxfp4_page_bytes(int64_t head_dim, int64_t block_size);

/* Slot-mapped write of new_key / new_value [num_tokens, num_kv_heads, head_dim]
 * (input_dtype RLLM_DTYPE_F16 or RLLM_DTYPE_BF16, 16-byte aligned), quantised as it
 * is written: of 32 elements with largest magnitude a, the scale byte is
 * clamp(floor(log2 a) - 2 + 127, 1, 254) (the OCP microscaling rule) and each code the
 * nearest to x / 2^(e - 127), ties to the even one, at most 6; 32 elements with an
 * infinity or a NaN among them become NaN (byte 255).  Slots < 0 or of a block
 * past the cache are skipped; the slots of one call must differ. */
int32_t rllm_cache_write_mxfp4(uint8_t *key_cache, uint8_t *value_cache, const uint16_t *new_key,
                               const uint16_t *new_value, const int64_t *slot_mapping,
                               int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
                               int64_t block_size, int64_t num_blocks, int32_t input_dtype,
                               uintptr_t stream);

/* Reads rows back: out_key / out_value [num_tokens, num_kv_heads, head_dim] of
 * output_dtype get the rows slot_mapping[t] of the caches, zeros where the slot is
 * < 0 or of a block past the cache; a slot may be listed more than once.  Exact
 * in bf16 up to its largest value; f16 rounds to nearest even (values past 65504
 * become infinities, below 2^-14 subnormal). */
int32_t rllm_cache_read_mxfp4(uint16_t *out_key, uint16_t *out_value, const uint8_t *key_cache,
                              const uint8_t *value_cache, const int64_t *slot_mapping,
                              int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim,
                              int64_t block_size, int64_t num_blocks, int32_t output_dtype,
                              uintptr_t stream);

/* Rotary embedding fused with the write: arguments as rllm_rope_cache_write.
 * The rotation is in f32 (cos / sin as given, each product and the sum rounded to
 * f32); q_out is rounded to dtype once, the rotated key is quantised from its f32
 * value.  (rllm_rope_cache_write rounds every step to dtype, as the model does: its
 * q_out differs from this one's by rounding.)  head_dim must be a multiple of 64. */
int32_t rllm_rope_cache_write_mxfp4(void *q_out, const void *q, const void *k, const void *v,
                                    uint8_t *key_cache, uint8_t *value_cache,
                                    const int64_t *slot_mapping, const int32_t *positions,
                                    const float *cos_cache, const float *sin_cache,
                                    int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                                    int64_t head_dim, int64_t block_size, int64_t num_blocks,
                                    int64_t max_position, int32_t dtype, uintptr_t stream);

/* Decode attention over the cache: arguments as rllm_paged_attention_decode_ex,
 * with the cache's num_blocks.  output and query 4-byte aligned, of q_dtype
 * (RLLM_DTYPE_F16 | RLLM_DTYPE_BF16).  Sums, maxima and weights are f32; the result
 * does not depend on the q type's range (keys and values are not converted to
 * it).  Keys or values that read as NaN make the outputs that see them NaN, and no
 * others (values with scale bytes 253 and 254, which no write makes, count as NaN).
 * workspace: at least rllm_paged_attention_decode_mxfp4_workspace_size(...) bytes,
 * 16-byte aligned, zero-filled before its first such call (each completed call
 * leaves it ready for the next, of any size it is large enough for); calls that
 * share it must not overlap in time.  The size for a batch and a table width (blocks
 * times block size) serves every call of the same heads and head_dim with no more
 * sequences and no wider tables.
 * NULL: a library-owned buffer per (device, stream), sized by the same rule; a capture
 * on a stream that has none of the size yet runs a workgroup a (sequence, kv head)
 * and needs none.
 * Graphs captured on one stream share its buffer with each other and with eager
 * calls there: run them in order, or give each its own workspace. */
int32_t rllm_paged_attention_decode_mxfp4(void *output, const void *query, const uint8_t *key_cache,
                                          const uint8_t *value_cache, const int32_t *block_tables,
                                          const int32_t *seq_lens, int64_t num_seqs,
                                          int64_t num_q_heads, int64_t num_kv_heads,
                                          int64_t head_dim, int64_t block_size,
                                          int64_t max_num_blocks_per_seq, int64_t num_blocks,
                                          float scale, int32_t q_dtype, void *workspace,
                                          int64_t workspace_bytes, uintptr_t stream);
int64_t rllm_paged_attention_decode_mxfp4_workspace_size(int64_t num_seqs, int64_t num_q_heads,
                                                         int64_t num_kv_heads, int64_t head_dim,
                                                         int64_t block_size,
                                                         int64_t max_num_blocks_per_seq);

/* Chunked-prefill attention over the cache: arguments as
 * rllm_paged_attention_prefill_ex (causal at absolute positions; the new tokens'
 * rows must be in the cache already), with the cache's num_blocks.  query 16-byte,
 * output 8-byte aligned.  bf16 queries: the weights are rounded to bf16 before they
 * meet the values, as for 16-bit caches (to 16 bits where a sequence has few new
 * tokens); f16: to 16 bits.  Rows of output that query_start_loc leaves out stay as
 * they are; its entries must not fall or pass num_tokens (a call with one that does
 * may leave any of its outputs unwritten).  Query tokens that see no key, those before
 * position 0 of a seq_len below its new tokens among them, get zeros.  Calls of few new tokens use library-owned buffers per
 * (device, stream), the decode call's among them, on its terms for captured graphs; a
 * capture on a stream that has none of the size yet runs without. */
int32_t rllm_paged_attention_prefill_mxfp4(void *output, const void *query,
                                           const uint8_t *key_cache, const uint8_t *value_cache,
                                           const int32_t *block_tables, const int32_t *seq_lens,
                                           const int32_t *query_start_loc, int64_t num_seqs,
                                           int64_t num_tokens, int64_t num_q_heads,
                                           int64_t num_kv_heads, int64_t head_dim,
                                           int64_t block_size, int64_t max_num_blocks_per_seq,
                                           int64_t num_blocks, float scale, int32_t q_dtype,
                                           uintptr_t stream);

/* Replace rllm_vector_add_f32(_sync) and rllm_block_copy(_sync),
 * smoke.cu:21-66; bound at cuda.rs:17-35.  out = a + b (f32); nbytes
 * contiguous bytes src -> dst. */
int32_t rllm_vector_add_f32(const float *a, const float *b, float *out, int64_t n, uintptr_t stream);
int32_t rllm_vector_add_f32_sync(const float *a, const float *b, float *out, int64_t n);
int32_t rllm_block_copy(const uint8_t *src, uint8_t *dst, int64_t nbytes, uintptr_t stream);
int32_t rllm_block_copy_sync(const uint8_t *src, uint8_t *dst, int64_t nbytes);

/* Replace rllm_fused_rope_f16(_sync), fused.cu:168-256; bound at fused.rs:54-76.
 * The kernel's own convention, kept for its callers: interleaved pairs
 * (2i, 2i+1), freq = 1 / theta^(2i / head_dim), angle = position * freq, cos /
 * sin in f32 on the device, f16 in and out; q [num_tokens, Hq, D] -> out_q,
 * k [num_tokens, Hkv, D] -> out_k (every kv head, also when Hkv > Hq, where
 * the reference leaves heads unwritten).  The model's rotate-half RoPE is
 * rllm_rope_cache_write. */
int32_t rllm_fused_rope_f16(uint16_t *out_q, uint16_t *out_k, const uint16_t *query,
                            const uint16_t *key, const int32_t *positions, int64_t num_tokens,
                            int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                            float rope_theta, uintptr_t stream);
int32_t rllm_fused_rope_f16_sync(uint16_t *out_q, uint16_t *out_k, const uint16_t *query,
                                 const uint16_t *key, const int32_t *positions, int64_t num_tokens,
                                 int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                 float rope_theta);

/* Replace rllm_gpu_alloc / _free / _alloc_host / _free_host,
 * cache_ops.cu:417-439; bound at cache_ops.rs:100-103. */
int32_t rllm_gpu_alloc(void **ptr, int64_t nbytes);
int32_t rllm_gpu_free(void *ptr);
int32_t rllm_gpu_alloc_host(void **ptr, int64_t nbytes);
int32_t rllm_gpu_free_host(void *ptr);

#ifdef __cplusplus
}
#endif
#endif /* RLLM_KERNELS_H */
