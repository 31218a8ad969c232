// Parameters and launchers of the 8-bit paged KV cache's kernels (kv8_*.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged_kv8_b200.h"

namespace pa {

// What a reserved step leaves in device memory, for the commit to see whether it still fits:
// num_free comes first, as the step's num_free_out; the rows' request slots follow.
struct Kv8StepRecord {
  int32_t num_free;  // the free list's length once the step counts; -1: the step was emptied
  int32_t rows, width, block_size, free_capacity, spare;
  const int32_t *lens, *held, *num_free_at, *free_blocks;  // what it was built from
  int32_t* tables;
  int64_t table_stride;
  const int32_t *out_tables, *context_lens, *held_out;  // the step's arrays
};
static_assert(sizeof(Kv8StepRecord) == 4 * PA_KV8_STEP_WORDS, "the header's size of num_free_out");

struct Kv8StepParams {
  const int32_t *row_ids, *lens, *query_lens;
  int32_t* tables;
  int64_t table_stride;
  const int32_t *held, *free_blocks, *num_free;
  int32_t free_capacity, num_rows, num_slots, width, block_size, num_tokens, max_query_len;
  int64_t pool_blocks;
  pa_kv8_tiling tiling;
  int32_t *out_tables, *context_lens, *query_out, *held_out, *cu_query, *seq_idx, *q_pos, *slots, *num_free_out;
  int64_t* work;
};

struct Kv8AppendParams {
  const void *key, *value;
  int64_t k_st, k_sh, v_st, v_sh;
  int32_t num_tokens, num_kv_heads, head_dim, block_size;
  uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
  int64_t num_slots;
  const int32_t* slots;
  bool vec16;  // every row starts on a 16-byte boundary
};

constexpr int kKv8Direct = 64;  // sequences up to which attention sums a step up for itself

// A tile that slices share: what joins its partials has to know.
struct Kv8Join {
  int64_t start, each;  // the tile's place on the work line; the line's cuts
  uint32_t rest;
  int32_t n, keys;
  int32_t row0, tokens;  // tokens 0: no such tile starts in the slice
  int32_t last;          // the last slice with a part of it
};

struct Kv8AttnParams {
  const void* q;
  int64_t q_st, q_sh;
  void* out;
  int64_t o_st, o_sh;
  const uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t *ctx_lens, *cu_q;
  const int64_t* work;  // this class's running sums [num_seqs + 1]; NULL: made from the lengths below
  const int32_t* query_lens;
  int32_t num_tokens, max_query_len, max_context, small_max;
  bool few;  // the class: sequences of at most small_max new tokens, or those of more
  int32_t num_seqs, num_heads, num_kv_heads, group, block_shift, tile_tokens, slices;
  int32_t pool_blocks;
  float qscale;  // softmax scale * log2(e)
  float* part_o;
  float2* part_ml;
  Kv8Join* joins;  // [slices], by the slice that a shared tile starts in
  bool first;  // tiles kernel: the call's first kernel
};

int* kv8_error_word();  // device address of the current device's error word

cudaError_t launch_kv8_step(const Kv8StepParams& p, int* err, cudaStream_t stream);
cudaError_t launch_kv8_commit(const int32_t* query_lens, const int32_t* accepted,
                              const int32_t* held_out, const Kv8StepRecord* record, int32_t rows, int32_t slots,
                              int32_t* lens, int32_t* held, int32_t* num_free, int* err, cudaStream_t stream);
cudaError_t launch_kv8_release(const int32_t* ids, int32_t count, const int32_t* tables, int64_t table_stride,
                               int32_t width, int32_t slots, int32_t* lens, int32_t* held, int32_t* free_blocks,
                               int32_t free_capacity, int32_t* num_free, int* err, cudaStream_t stream);
cudaError_t launch_kv8_append(int dtype, const Kv8AppendParams& p, cudaStream_t stream);

// Slices of the work line for the kernel for few rows, and the rows a partial holds.
int kv8_rows_slices(int row_groups, int num_kv_heads, int sms);
// `pair`: p.num_kv_heads counts pairs of KV heads of 64 dims, p.group the query heads of a pair.
// The kernels of a call, in this order: rows, tiles, then the joins.  The tiles kernel starts
// while the one for few rows runs, so it must directly follow it.
cudaError_t launch_kv8_rows(int dtype, int head_dim, bool pair, int row_groups, const CUtensorMap& tk,
                            const CUtensorMap& tv, const Kv8AttnParams& p, int* err, cudaStream_t stream);
constexpr int kKv8RowGroups = 3;  // most groups of 8 rows
cudaError_t launch_kv8_rows_combine(int dtype, int head_dim, int row_groups, const Kv8AttnParams& p,
                                    cudaStream_t stream);
int kv8_tiles_slices(int num_kv_heads, int sms);
cudaError_t launch_kv8_tiles(int dtype, int head_dim, const CUtensorMap& tk, const CUtensorMap& tv,
                             const Kv8AttnParams& p, int* err, cudaStream_t stream);
cudaError_t launch_kv8_tiles_combine(int dtype, int head_dim, const Kv8AttnParams& p, cudaStream_t stream);
constexpr int kKv8TileRows = 256;  // (token, head) rows of its tiles
cudaError_t launch_kv8_combine(int dtype, int head_dim, int rows, int key_step, const Kv8AttnParams& p,
                               cudaStream_t stream);

}  // namespace pa
