/*
 * paged_kv8_b200.h — C ABI of the 8-bit paged KV cache on B200 (sm_100a).
 *
 * Three operators that work together: a step's block tables and slot map built on the GPU
 * from request lengths, the append of new K/V rows quantised to 8 bits, and attention of a
 * chunk of new tokens (one token and more) over the 8-bit pools.  None has a counterpart in
 * akshajravi/llm-inference-server, whose pools hold the model's dtype and whose block
 * tables are host lists; the conventions (flat slots, 0-padded tables, causal rule, return
 * codes, pa_last_error, asynchronous launches on the caller's stream) are those of
 * paged_attention_b200.h, which this header includes.
 *
 * Cache format.  A row (one token of one KV head, head_dim values) is stored as e4m3
 * payload and one scale byte b that stands for 2^(b - 127), b in [113, 134]:
 *   b       = 127 + the least e in [-14, 7] with max|x| <= 448 * 2^e
 *   payload = e4m3(x * 2^-e), round to nearest even, saturating
 * so every cached value is exactly an fp16 number; magnitudes past 57,344 saturate, and rows
 * below 448 * 2^-15 keep e = -14, a step of 2^-23.  A row that holds a NaN is stored as zeros with b = 255, which stands for NaN.
 *   payload pool [num_blocks, block_size, num_kv_heads, head_dim]   1 byte each
 *   scale pool   [num_blocks, num_kv_heads, block_size]             1 byte each
 *
 * Every entry point validates what the host can see.  What only the GPU can see (lengths,
 * ids) is validated there: a violation sets a bit in the device's KV8 error word
 * (pa_kv8_read_error) and the kernels read and write nothing out of bounds.
 */
#ifndef PAGED_KV8_B200_H
#define PAGED_KV8_B200_H

#include "paged_attention_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bits of the KV8 error word. */
#define PA_KV8_ERR_BLOCK 1    /* a block id outside the pool; a reserved step that would use it was emptied */
#define PA_KV8_ERR_TIMEOUT 4  /* a bounded wait inside a kernel ran out */
#define PA_KV8_ERR_STEP 8     /* inconsistent lengths or ids: the step was emptied; or it was stale: not committed */
#define PA_KV8_ERR_NO_BLOCKS 16 /* the free list is too short; the step was emptied */

/* Further bits of pa_last_launches(). */
#define PA_LAUNCH_KV8_ROWS 128    /* KV8 attention, few rows per sequence (mma.sync) */
#define PA_LAUNCH_KV8_COMBINE 256 /* join of tiles that several CTAs worked on */
#define PA_LAUNCH_KV8_TILES 512   /* KV8 attention, 256-row tiles (tcgen05) */

/* Most rows (sequences) of a step and most request slots of a table set. */
#define PA_KV8_MAX_ROWS 4096
#define PA_KV8_MAX_REQUESTS 131072
/* int32 words of a step's num_free_out before its rows'. */
#define PA_KV8_STEP_WORDS 24

/*
 * How attention cuts a step into work: sequences of at most `small_max` new tokens are cut
 * into tiles of `small_tokens` tokens (the kernel for few rows), longer ones into tiles of
 * `large_tokens` (the tensor-memory kernel); small_max 0: all of them.  A step's `work` array holds, for each class,
 * the running sum over sequences of the keys that their tiles visit.
 */
typedef struct pa_kv8_tiling {
  int32_t small_tokens;
  int32_t small_max;
  int32_t large_tokens;
  int32_t row_groups; /* groups of 8 (token, head) rows that the kernel for few rows holds */
} pa_kv8_tiling;

/* The tiling for a step of num_seqs chunks of at most max_query_len tokens, num_tokens in
 * all, with `group` query heads per KV head.  No reference counterpart. */
int32_t pa_kv8_choose_tiling(int32_t group, int32_t max_query_len, int32_t num_seqs, int32_t num_tokens,
                             pa_kv8_tiling* tiling);

/*
 * Build one step's metadata on the GPU.  No reference counterpart (the host builds it in
 * inference_server/core/paged_executor.py: 211-263).
 *
 *   row_ids      device [num_rows]: the request slot of each row, -1 for a padding row; or
 *                NULL: row i is slot i
 *   lens         device: with `held`, tokens cached per slot before the step (the context is
 *                lens + query_lens); without, the context per slot with this step's tokens
 *   query_lens   device [num_rows]: new tokens
 *   tables       device [num_slots, table_stride]: block ids per slot, `width` of them used
 *   held         device [num_slots]: blocks each slot holds, or NULL (tables are complete)
 *   free_blocks  device [free_capacity], num_free device [1]: the free list, taken from its
 *                end in row order; the new ids are also written into `tables`.  A row takes
 *                ceil(context / block_size) - held blocks if that is positive
 *   num_tokens   tokens the per-token arrays hold; those past the step's get -1
 *
 * Outputs (device): out_tables [num_rows, width], 0-padded (NULL without `held`),
 * context_lens / query_lens_out / held_out [num_rows], cu_query_lens [num_rows + 1],
 * seq_idx / q_pos / slot_mapping [num_tokens], work int64 [2, num_rows + 1], num_free_out
 * [PA_KV8_STEP_WORDS + num_rows], 8-byte aligned: the free list's length once the step counts,
 * then what pa_kv8_commit has to know of it (without `held` the first word only).
 * Nothing but `tables` is updated in place, so a step can be built again; pa_kv8_commit
 * makes it count.  A step whose lengths or ids are inconsistent (a slot named twice, more
 * tokens than num_tokens, a chunk over max_query_len, a context over width * block_size, a
 * free list too short, with `held` a block id outside the pool where a new token goes) is
 * emptied: all lengths 0, tables untouched, num_free_out -1.
 */
int32_t pa_kv8_build_step(const int32_t* row_ids, const int32_t* lens, const int32_t* query_lens, int32_t* tables,
                          int64_t table_stride, const int32_t* held, const int32_t* free_blocks,
                          const int32_t* num_free, int32_t free_capacity, int32_t num_rows, int32_t num_slots,
                          int32_t width, int32_t block_size, int64_t pool_num_blocks, int32_t num_tokens,
                          int32_t max_query_len, const pa_kv8_tiling* tiling, int32_t* out_tables,
                          int32_t* context_lens, int32_t* query_lens_out, int32_t* held_out, int32_t* cu_query_lens,
                          int32_t* seq_idx, int32_t* q_pos, int32_t* slot_mapping, int32_t* num_free_out,
                          int64_t* work, void* stream);

/*
 * Make a step count that was built with `held`: lens += accepted (NULL: the step's query_lens;
 * clamped to them), held = held_out, its new blocks leave the free list and stand in the tables.
 * query_lens, held_out and num_free_out are the step's; its rows' slots are those that the step
 * was built with, whatever row_ids holds by now.  A step that was emptied changes
 * nothing, nor does one that no longer fits, which sets PA_KV8_ERR_STEP: one of other lens, held
 * or num_free, one whose slots have other lengths by now, or whose new blocks are not the free
 * list's last ones any more (another step took them, or blocks were released over them).  A slot
 * that was released and filled again, to the same length in the same blocks, looks the same:
 * drop the steps of slots that are released.
 * No reference counterpart.
 */
int32_t pa_kv8_commit(const int32_t* row_ids, const int32_t* query_lens, const int32_t* accepted,
                      const int32_t* held_out, const int32_t* num_free_out, int32_t num_rows, int32_t num_slots,
                      int32_t* lens, int32_t* held, int32_t* num_free, void* stream);

/*
 * Put the blocks of `count` request slots back on the free list, in the order given (a
 * slot's last block first), and empty the slots; ids of -1 are passed over.  Refused as a
 * whole when a slot is named twice or the list would overflow.  No reference counterpart.
 */
int32_t pa_kv8_release(const int32_t* ids, int32_t count, const int32_t* tables, int64_t table_stride, int32_t width,
                       int32_t num_slots, int32_t* lens, int32_t* held, int32_t* free_blocks, int32_t free_capacity,
                       int32_t* num_free, void* stream);

/*
 * Quantise new rows and write them into the pools at their flat slots, K and V in one
 * launch; the 8-bit form of pa_reshape_and_cache (inference_server/core/
 * paged_executor.py:116-125).  key / value [num_tokens, num_kv_heads, head_dim], unit stride
 * along head_dim, strides in elements; head_dim 64 or 128; dtype any of PA_DTYPE_*.  Slots
 * outside the pool (the -1 of padding tokens) are passed over; a slot named twice must get
 * the same row.
 */
int32_t pa_kv8_append(const void* key, int64_t k_stride_token, int64_t k_stride_head, const void* value,
                      int64_t v_stride_token, int64_t v_stride_head, int32_t num_tokens, int32_t num_kv_heads,
                      int32_t head_dim, int32_t dtype, void* k_pool, void* v_pool, void* k_scale, void* v_scale,
                      int64_t pool_num_blocks, int32_t block_size, const int32_t* slot_mapping, void* stream);

/* Bytes of scratch that pa_kv8_attention needs for these sizes, whatever the lengths.
 * No reference counterpart. */
uint64_t pa_kv8_workspace_bytes(int32_t num_seqs, int32_t num_tokens, int32_t num_heads, int32_t num_kv_heads,
                                int32_t head_dim, int32_t max_query_len);

/*
 * Causal attention of each sequence's new tokens over the 8-bit pools: token t of sequence
 * i stands at p = context_lens[i] - query_lens[i] + t and attends to keys 0 .. p through
 * the block table (the rule of inference_server/core/attention.py:19-58).  Lengths and
 * tables stay on the device; the launches depend on the host's sizes only, so a captured
 * call can be replayed with other lengths.  Sums are float32; softmax weights are rounded to fp16
 * for the product with V: 11 bits, and at most 2^-32 of a row's largest weight lost a key.  cu_query_lens and work come from
 * pa_kv8_build_step with the tiling of the same group, sizes and max_query_len; with both NULL
 * the call sums query_lens and the work up by itself (over 64 sequences in one more launch),
 * with pa_kv8_build_step's checks.  table_width blocks of a table row are used.  Rows past the
 * last sequence's are left as they were.  head_dim 64 or 128, block_size a power of two
 * times 16, query fp16 or bf16 (strides in elements, multiples of 8; rows 16-byte aligned).
 */
int32_t pa_kv8_attention(const void* query, int64_t q_stride_token, int64_t q_stride_head, int32_t num_tokens,
                         int32_t num_heads, int32_t head_dim, const void* k_pool, const void* v_pool,
                         const void* k_scale, const void* v_scale, int64_t pool_num_blocks, int32_t block_size,
                         int32_t num_kv_heads, int32_t dtype, float scale, int32_t num_seqs, int32_t max_query_len,
                         const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                         const int32_t* context_lens, const int32_t* query_lens, const int32_t* cu_query_lens,
                         const int64_t* work, void* out, int64_t out_stride_token, int64_t out_stride_head,
                         void* workspace, uint64_t workspace_bytes, void* stream);

/* Read (and, with `clear`, reset) the current device's KV8 error word.  Synchronises the
 * stream.  No reference counterpart. */
int32_t pa_kv8_read_error(int32_t clear, int32_t* error_word, void* stream);

#ifdef __cplusplus
}
#endif

#endif
