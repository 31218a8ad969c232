// extern "C" entry points declared in include/paged_kv8_b200.h: argument checks, tensor
// maps (encoded per call) and dispatch.
#include <cudaTypedefs.h>

#include <algorithm>

#include "kv8.h"
#include "pa_common.cuh"
#include "pa_host.h"

namespace pa {

static int32_t kv8_cuda_fail(cudaError_t e, const char* what) {
  return fail(PA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// A payload pool [NB, BS, Hkv, D] as the 3-D tensor (D, Hkv, NB * BS), box (D, 1, 16),
// swizzled over the row's width.
static int32_t payload_map(const void* pool, int64_t blocks, int bs, int hkv, int dim, CUtensorMap* out) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(PA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the CUDA driver");
  cuuint64_t gdim[3] = {cuuint64_t(dim), cuuint64_t(hkv), cuuint64_t(blocks) * cuuint64_t(bs)};
  cuuint64_t gstride[2] = {cuuint64_t(dim), cuuint64_t(hkv) * dim};
  cuuint32_t box[3] = {cuuint32_t(dim), 1u, 16u};
  cuuint32_t estride[3] = {1u, 1u, 1u};
  CUresult r = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn)(
      out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(pool), gdim, gstride, box, estride,
      CU_TENSOR_MAP_INTERLEAVE_NONE, dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(PA_ERR_CUDA, "cuTensorMapEncodeTiled (8-bit pool) failed (CUresult %d)", int(r));
  return PA_OK;
}

static int sm_count() {
  static int known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!known[dev] && cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return known[dev];
}

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Slices for which the workspace holds partials, for the SMs of any sm_100 part.
constexpr int kMaxSms = 160;

// How the kernel for few rows runs a call: KV heads of 64 dims in pairs where that fits.
struct Kv8Rows {
  bool pair;
  int row_groups, num_kv_heads, group;
};
static Kv8Rows rows_form(const pa_kv8_tiling& t, int num_kv_heads, int group, int head_dim, int max_query_len) {
  const int tokens = std::max(1, std::min(t.small_tokens, max_query_len));  // of a tile, at most
  const int paired = (2 * group * tokens + 7) / 8;
  if (head_dim == 64 && num_kv_heads % 2 == 0 && paired <= kKv8RowGroups)
    return {true, paired, num_kv_heads / 2, 2 * group};
  return {false, t.row_groups, num_kv_heads, group};
}

struct Kv8Scratch {
  uint64_t work, cu, joins, tile_joins, ml, o, tile_ml, tile_o, bytes;
};
static Kv8Scratch attention_scratch(const Kv8Rows& f, int32_t num_seqs, int32_t num_kv_heads, int32_t head_dim, int sms,
                                    bool tiles) {
  const uint64_t slices = kv8_rows_slices(f.row_groups, f.num_kv_heads, sms);
  const uint64_t tile_slices = tiles ? kv8_tiles_slices(num_kv_heads, sms) : 0;
  const uint64_t rows = slices * f.num_kv_heads * 2 * (8 * f.row_groups);
  const uint64_t tile_rows = tile_slices * num_kv_heads * 2 * kKv8TileRows;
  Kv8Scratch s;
  s.work = 0;
  s.cu = (uint64_t(num_seqs) + 1) * 2 * sizeof(int64_t);
  s.joins = (s.cu + (uint64_t(num_seqs) + 1) * sizeof(int32_t) + 255) / 256 * 256;
  s.tile_joins = s.joins + slices * sizeof(Kv8Join);
  s.ml = (s.tile_joins + tile_slices * sizeof(Kv8Join) + 255) / 256 * 256;
  s.o = (s.ml + rows * sizeof(float2) + 255) / 256 * 256;
  s.tile_ml = (s.o + rows * head_dim * sizeof(float) + 255) / 256 * 256;
  s.tile_o = (s.tile_ml + tile_rows * sizeof(float2) + 255) / 256 * 256;
  s.bytes = s.tile_o + tile_rows * head_dim * sizeof(float);
  return s;
}

static int32_t check_step_sizes(const Kv8StepParams& p, int64_t table_stride) {
  if (p.tiling.small_tokens < 1 || p.tiling.large_tokens < 1) return fail(PA_ERR_INVALID_ARGUMENT, "build_step: bad tiling");
  if (p.num_rows < 0 || p.num_slots < 0 || p.width < 0 || p.block_size <= 0 || p.num_tokens < 0 ||
      p.max_query_len < 0 || p.free_capacity < 0 || table_stride < p.width)
    return fail(PA_ERR_INVALID_ARGUMENT, "build_step: bad sizes");
  if (p.num_rows > PA_KV8_MAX_ROWS)
    return fail(PA_ERR_UNSUPPORTED, "build_step: %d rows, at most %d are supported", p.num_rows, PA_KV8_MAX_ROWS);
  if (p.num_slots > PA_KV8_MAX_REQUESTS)
    return fail(PA_ERR_UNSUPPORTED, "build_step: %d request slots, at most %d are supported", p.num_slots,
                PA_KV8_MAX_REQUESTS);
  if (p.max_query_len > (1 << 20) || p.width > (1 << 20) || int64_t(p.width) * p.block_size > (int64_t(1) << 30))
    return fail(PA_ERR_UNSUPPORTED, "build_step: chunks up to 2^20 tokens and contexts up to 2^30 are supported");
  if (p.pool_blocks < 0 || p.pool_blocks * int64_t(p.block_size) > (int64_t(1) << 31) - 1)
    return fail(PA_ERR_UNSUPPORTED, "pool has more than 2^31 slots");
  if (!p.row_ids && p.num_rows > p.num_slots) return fail(PA_ERR_INVALID_ARGUMENT, "build_step: more rows than slots");
  return PA_OK;
}

}  // namespace pa

extern "C" {

int32_t pa_kv8_choose_tiling(int32_t group, int32_t max_query_len, int32_t num_seqs, int32_t num_tokens,
                             pa_kv8_tiling* tiling) {
  using namespace pa;
  if (!tiling) return fail(PA_ERR_INVALID_ARGUMENT, "tiling must not be NULL");
  if (group < 1 || max_query_len < 0 || num_seqs < 0 || num_tokens < 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "bad group, max_query_len or sizes");
  if (group > 16) return fail(PA_ERR_UNSUPPORTED, "%d query heads per KV head: at most 16 are supported", group);
  // A sequence of up to 24 (token, head) rows goes to the kernel for few rows, one of more to
  // the 256-row tiles.  Where the sizes leave no room for a short chunk beside the longest ones
  // (one prompt, chunks of one length) the first class has none: its two launches are spared.
  const int few = std::max(1, 8 * kKv8RowGroups / group);
  const bool none = max_query_len > few && num_tokens - int64_t(num_seqs - 1) * max_query_len > few;
  const int rows = group * std::max(1, std::min(max_query_len, few));
  tiling->row_groups = (rows + 7) / 8;
  tiling->small_tokens = std::max(1, 8 * tiling->row_groups / group);
  tiling->small_max = none ? 0 : std::min(max_query_len, few);
  tiling->large_tokens = kKv8TileRows / group;
  return PA_OK;
}

int32_t pa_kv8_build_step(const int32_t* row_ids, const int32_t* lens, const int32_t* query_lens, int32_t* tables,
                          int64_t table_stride, const int32_t* held, const int32_t* free_blocks,
                          const int32_t* num_free, int32_t free_capacity, int32_t num_rows, int32_t num_slots,
                          int32_t width, int32_t block_size, int64_t pool_num_blocks, int32_t num_tokens,
                          int32_t max_query_len, const pa_kv8_tiling* tiling, int32_t* out_tables,
                          int32_t* context_lens, int32_t* query_lens_out, int32_t* held_out, int32_t* cu_query_lens,
                          int32_t* seq_idx, int32_t* q_pos, int32_t* slot_mapping, int32_t* num_free_out,
                          int64_t* work, void* stream_ptr) {
  using namespace pa;
  if (!tiling) return fail(PA_ERR_INVALID_ARGUMENT, "build_step: bad tiling");
  Kv8StepParams p{};
  p.row_ids = row_ids;
  p.lens = lens;
  p.query_lens = query_lens;
  p.tables = tables;
  p.table_stride = table_stride;
  p.held = held;
  p.free_blocks = free_blocks;
  p.num_free = num_free;
  p.free_capacity = free_capacity;
  p.num_rows = num_rows;
  p.num_slots = num_slots;
  p.width = width;
  p.block_size = block_size;
  p.num_tokens = num_tokens;
  p.max_query_len = max_query_len;
  p.pool_blocks = pool_num_blocks;
  p.tiling = *tiling;
  p.out_tables = out_tables;
  p.context_lens = context_lens;
  p.query_out = query_lens_out;
  p.held_out = held_out;
  p.cu_query = cu_query_lens;
  p.seq_idx = seq_idx;
  p.q_pos = q_pos;
  p.slots = slot_mapping;
  p.num_free_out = num_free_out;
  p.work = work;
  const int32_t st = check_step_sizes(p, table_stride);
  if (st != PA_OK) return st;
  if ((num_rows > 0 && (!lens || !query_lens || !context_lens || !query_lens_out || !held_out)) || !cu_query_lens ||
      !num_free_out || !work || (num_tokens > 0 && (!seq_idx || !q_pos || !slot_mapping)) ||
      (num_rows > 0 && width > 0 && !tables) ||
      (held && (!num_free || (free_capacity > 0 && !free_blocks) || (num_rows > 0 && width > 0 && !out_tables))))
    return fail(PA_ERR_INVALID_ARGUMENT, "build_step: NULL device pointer");
  if (reinterpret_cast<uintptr_t>(num_free_out) % 8)
    return fail(PA_ERR_INVALID_ARGUMENT, "build_step: num_free_out must be 8-byte aligned");
  int* err = kv8_error_word();
  if (!err) return fail(PA_ERR_CUDA, "build_step: no CUDA device");
  cudaError_t e = launch_kv8_step(p, err, static_cast<cudaStream_t>(stream_ptr));
  return e == cudaSuccess ? PA_OK : kv8_cuda_fail(e, "build_step launch");
}

int32_t pa_kv8_commit(const int32_t*, const int32_t* query_lens, const int32_t* accepted,
                      const int32_t* held_out, const int32_t* num_free_out, int32_t num_rows, int32_t num_slots,
                      int32_t* lens, int32_t* held, int32_t* num_free, void* stream_ptr) {
  using namespace pa;
  if (num_rows < 0 || num_slots < 0) return fail(PA_ERR_INVALID_ARGUMENT, "commit: bad sizes");
  if (num_rows > PA_KV8_MAX_ROWS)
    return fail(PA_ERR_UNSUPPORTED, "commit: %d rows, at most %d are supported", num_rows, PA_KV8_MAX_ROWS);
  if (!num_free_out || !num_free || (num_rows > 0 && (!query_lens || !held_out || !lens || !held)))
    return fail(PA_ERR_INVALID_ARGUMENT, "commit: NULL device pointer");
  if (reinterpret_cast<uintptr_t>(num_free_out) % 8)
    return fail(PA_ERR_INVALID_ARGUMENT, "commit: num_free_out must be 8-byte aligned");
  int* err = kv8_error_word();
  if (!err) return fail(PA_ERR_CUDA, "commit: no CUDA device");
  cudaError_t e = launch_kv8_commit(query_lens, accepted, held_out,
                                    reinterpret_cast<const Kv8StepRecord*>(num_free_out), num_rows, num_slots, lens,
                                    held, num_free, err, static_cast<cudaStream_t>(stream_ptr));
  return e == cudaSuccess ? PA_OK : kv8_cuda_fail(e, "commit launch");
}

int32_t pa_kv8_release(const int32_t* ids, int32_t count, const int32_t* tables, int64_t table_stride, int32_t width,
                       int32_t num_slots, int32_t* lens, int32_t* held, int32_t* free_blocks, int32_t free_capacity,
                       int32_t* num_free, void* stream_ptr) {
  using namespace pa;
  if (count < 0 || num_slots < 0 || width < 0 || free_capacity < 0 || table_stride < width)
    return fail(PA_ERR_INVALID_ARGUMENT, "release: bad sizes");
  if (count > PA_KV8_MAX_ROWS || num_slots > PA_KV8_MAX_REQUESTS)
    return fail(PA_ERR_UNSUPPORTED, "release: at most %d ids of at most %d slots", PA_KV8_MAX_ROWS,
                PA_KV8_MAX_REQUESTS);
  if (count == 0) return PA_OK;
  if (!ids || !tables || !lens || !held || !free_blocks || !num_free)
    return fail(PA_ERR_INVALID_ARGUMENT, "release: NULL device pointer");
  int* err = kv8_error_word();
  if (!err) return fail(PA_ERR_CUDA, "release: no CUDA device");
  cudaError_t e = launch_kv8_release(ids, count, tables, table_stride, width, num_slots, lens, held, free_blocks,
                                     free_capacity, num_free, err, static_cast<cudaStream_t>(stream_ptr));
  return e == cudaSuccess ? PA_OK : kv8_cuda_fail(e, "release launch");
}

int32_t pa_kv8_append(const void* key, int64_t k_stride_token, int64_t k_stride_head, const void* value,
                      int64_t v_stride_token, int64_t v_stride_head, int32_t num_tokens, int32_t num_kv_heads,
                      int32_t head_dim, int32_t dtype, void* k_pool, void* v_pool, void* k_scale, void* v_scale,
                      int64_t pool_num_blocks, int32_t block_size, const int32_t* slot_mapping, void* stream_ptr) {
  using namespace pa;
  if (dtype != PA_DTYPE_F32 && dtype != PA_DTYPE_F16 && dtype != PA_DTYPE_BF16)
    return fail(PA_ERR_UNSUPPORTED, "dtype code %d is not float32, float16 or bfloat16", dtype);
  if (num_tokens < 0 || num_kv_heads <= 0 || block_size <= 0 || pool_num_blocks < 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "bad append shape");
  if (head_dim != 64 && head_dim != 128)
    return fail(PA_ERR_UNSUPPORTED, "head_dim %d: the 8-bit cache supports 64 and 128", head_dim);
  if (num_tokens == 0) return PA_OK;
  if (!key || !value || !k_pool || !v_pool || !k_scale || !v_scale || !slot_mapping)
    return fail(PA_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (!aligned16(k_pool) || !aligned16(v_pool))
    return fail(PA_ERR_INVALID_ARGUMENT, "8-bit pools must be 16-byte aligned");
  if (int64_t(num_tokens) * num_kv_heads > (int64_t(1) << 31) - 1)
    return fail(PA_ERR_UNSUPPORTED, "append of more than 2^31 rows");
  const int64_t es = dtype == PA_DTYPE_F32 ? 4 : 2;
  Kv8AppendParams p{};
  p.key = key;
  p.k_st = k_stride_token;
  p.k_sh = k_stride_head;
  p.value = value;
  p.v_st = v_stride_token;
  p.v_sh = v_stride_head;
  p.num_tokens = num_tokens;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.k_pool = static_cast<uint8_t*>(k_pool);
  p.v_pool = static_cast<uint8_t*>(v_pool);
  p.k_scale = static_cast<uint8_t*>(k_scale);
  p.v_scale = static_cast<uint8_t*>(v_scale);
  p.num_slots = pool_num_blocks * block_size;
  p.slots = slot_mapping;
  p.vec16 = aligned16(key) && aligned16(value) && (k_stride_token * es) % 16 == 0 && (k_stride_head * es) % 16 == 0 &&
            (v_stride_token * es) % 16 == 0 && (v_stride_head * es) % 16 == 0;
  cudaError_t e = launch_kv8_append(dtype, p, static_cast<cudaStream_t>(stream_ptr));
  return e == cudaSuccess ? PA_OK : kv8_cuda_fail(e, "8-bit append launch");
}

uint64_t pa_kv8_workspace_bytes(int32_t num_seqs, int32_t num_tokens, int32_t num_heads, int32_t num_kv_heads,
                                int32_t head_dim, int32_t max_query_len) {
  using namespace pa;
  pa_kv8_tiling t;
  if (num_seqs < 0 || num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      num_heads % num_kv_heads ||
      pa_kv8_choose_tiling(num_heads / num_kv_heads, max_query_len, num_seqs, num_tokens, &t) != PA_OK)
    return 0;
  const Kv8Rows f = rows_form(t, num_kv_heads, num_heads / num_kv_heads, head_dim, max_query_len);
  return attention_scratch(f, num_seqs, num_kv_heads, head_dim, kMaxSms, max_query_len > t.small_max).bytes;
}

int32_t pa_kv8_attention(const void* query, int64_t q_stride_token, int64_t q_stride_head, int32_t num_tokens,
                         int32_t num_heads, int32_t head_dim, const void* k_pool, const void* v_pool,
                         const void* k_scale, const void* v_scale, int64_t pool_num_blocks, int32_t block_size,
                         int32_t num_kv_heads, int32_t dtype, float scale, int32_t num_seqs, int32_t max_query_len,
                         const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                         const int32_t* context_lens, const int32_t* query_lens, const int32_t* cu_query_lens,
                         const int64_t* work, void* out, int64_t out_stride_token, int64_t out_stride_head,
                         void* workspace, uint64_t workspace_bytes, void* stream_ptr) {
  using namespace pa;
  reset_last_launches();
  if (dtype != PA_DTYPE_F16 && dtype != PA_DTYPE_BF16)
    return fail(PA_ERR_UNSUPPORTED, "dtype code %d: the 8-bit cache takes float16 and bfloat16 queries", dtype);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_tokens < 0 || num_seqs < 0 || pool_num_blocks < 0)
    return fail(PA_ERR_INVALID_ARGUMENT, "heads must be positive and sizes non-negative");
  if (num_heads % num_kv_heads)
    return fail(PA_ERR_INVALID_ARGUMENT, "%d query heads not divisible by %d kv heads", num_heads, num_kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return fail(PA_ERR_UNSUPPORTED, "head_dim %d: the 8-bit cache supports 64 and 128", head_dim);
  int shift = 0;
  while (shift < 8 && (16 << shift) < block_size) ++shift;
  if (block_size != (16 << shift))
    return fail(PA_ERR_UNSUPPORTED, "block_size %d: the 8-bit cache supports 16, 32, ... 4096", block_size);
  if (pool_num_blocks * int64_t(block_size) > (int64_t(1) << 31) - 1)
    return fail(PA_ERR_UNSUPPORTED, "pool has more than 2^31 slots");
  pa_kv8_tiling t;
  const int group = num_heads / num_kv_heads;
  int32_t st = pa_kv8_choose_tiling(group, max_query_len, num_seqs, num_tokens, &t);
  if (st != PA_OK) return st;
  if (num_tokens == 0 || num_seqs == 0) return PA_OK;
  if (pool_num_blocks == 0) return fail(PA_ERR_INVALID_ARGUMENT, "the pool has no blocks");
  const bool build = !work && !cu_query_lens;
  if (!query || !k_pool || !v_pool || !k_scale || !v_scale || !block_tables || !context_lens || !out || !workspace ||
      (build ? !query_lens : (!cu_query_lens || !work)))
    return fail(PA_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (!aligned16(query) || q_stride_token % 8 || q_stride_head % 8 || !aligned16(out) || out_stride_token % 8 ||
      out_stride_head % 8)
    return fail(PA_ERR_INVALID_ARGUMENT, "query and out rows must be 16-byte aligned");
  if (!aligned16(k_pool) || !aligned16(v_pool) || !aligned16(k_scale) || !aligned16(v_scale))
    return fail(PA_ERR_INVALID_ARGUMENT, "8-bit pools and their scales must be 16-byte aligned");
  const int sms = std::min(sm_count(), kMaxSms);
  const Kv8Rows f = rows_form(t, num_kv_heads, group, head_dim, max_query_len);
  const Kv8Scratch s = attention_scratch(f, num_seqs, num_kv_heads, head_dim, sms, max_query_len > t.small_max);
  if (workspace_bytes < s.bytes)
    return fail(PA_ERR_BUFFER_TOO_SMALL, "workspace holds %llu bytes, %llu needed",
                (unsigned long long)workspace_bytes, (unsigned long long)s.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(PA_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  int* err = kv8_error_word();
  if (!err) return fail(PA_ERR_CUDA, "no CUDA device");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (build) {
    Kv8StepParams b{};
    b.lens = context_lens;
    b.query_lens = query_lens;
    b.num_rows = b.num_slots = num_seqs;
    b.width = table_width;
    b.block_size = block_size;
    b.num_tokens = num_tokens;
    b.max_query_len = max_query_len;
    b.pool_blocks = pool_num_blocks;
    b.tiling = t;
    st = check_step_sizes(b, table_stride);
    if (st != PA_OK) return st;
    if (num_seqs > kKv8Direct) {  // fewer the kernels sum up for themselves
      b.cu_query = reinterpret_cast<int32_t*>(ws + s.cu);
      b.work = reinterpret_cast<int64_t*>(ws + s.work);
      const cudaError_t eb = launch_kv8_step(b, err, stream);
      if (eb != cudaSuccess) return kv8_cuda_fail(eb, "8-bit attention's step launch");
      cu_query_lens = b.cu_query;
      work = b.work;
    }
  }
  CUtensorMap tk, tv;
  const int row_dim = f.pair ? 2 * head_dim : head_dim;
  st = payload_map(k_pool, pool_num_blocks, block_size, f.num_kv_heads, row_dim, &tk);
  if (st == PA_OK) st = payload_map(v_pool, pool_num_blocks, block_size, f.num_kv_heads, row_dim, &tv);
  if (st != PA_OK) return st;
  Kv8AttnParams p{};
  p.q = query;
  p.q_st = q_stride_token;
  p.q_sh = q_stride_head;
  p.out = out;
  p.o_st = out_stride_token;
  p.o_sh = out_stride_head;
  p.k_pool = static_cast<const uint8_t*>(k_pool);
  p.v_pool = static_cast<const uint8_t*>(v_pool);
  p.k_scale = static_cast<const uint8_t*>(k_scale);
  p.v_scale = static_cast<const uint8_t*>(v_scale);
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.ctx_lens = context_lens;
  p.cu_q = cu_query_lens;
  p.work = work;
  p.query_lens = query_lens;
  p.num_tokens = num_tokens;
  p.max_query_len = max_query_len;
  p.max_context = int32_t(std::min<int64_t>(int64_t(table_width) * block_size, 1 << 30));
  p.small_max = t.small_max;
  p.few = true;
  p.num_seqs = num_seqs;
  p.num_heads = num_heads;
  p.num_kv_heads = f.num_kv_heads;
  p.group = f.group;
  p.block_shift = shift;
  p.tile_tokens = t.small_tokens;
  p.slices = kv8_rows_slices(f.row_groups, f.num_kv_heads, sms);
  p.pool_blocks = int32_t(pool_num_blocks);
  p.qscale = scale * kLog2e;
  p.part_ml = reinterpret_cast<float2*>(ws + s.ml);
  p.part_o = reinterpret_cast<float*>(ws + s.o);
  p.joins = reinterpret_cast<Kv8Join*>(ws + s.joins);
  // Small_max 0 with longer chunks: the first class is empty.
  const bool tiles = max_query_len > t.small_max, rows = t.small_max > 0 || !tiles;
  int32_t launched = 0;
  cudaError_t e = cudaSuccess;
  if (rows) {
    e = launch_kv8_rows(dtype, head_dim, f.pair, f.row_groups, tk, tv, p, err, stream);
    if (e != cudaSuccess) return kv8_cuda_fail(e, "8-bit attention launch");
    launched |= PA_LAUNCH_KV8_ROWS;
  }
  Kv8AttnParams q = p;  // of the tiles kernel
  if (tiles) {
    q.work = work ? work + num_seqs + 1 : nullptr;
    q.few = false;
    q.num_kv_heads = num_kv_heads;
    q.group = group;
    q.tile_tokens = t.large_tokens;
    q.slices = kv8_tiles_slices(num_kv_heads, sms);
    q.part_ml = reinterpret_cast<float2*>(ws + s.tile_ml);
    q.part_o = reinterpret_cast<float*>(ws + s.tile_o);
    q.joins = reinterpret_cast<Kv8Join*>(ws + s.tile_joins);
    q.first = !rows;
    if (f.pair) {  // the rows kernel's maps were of pairs
      st = payload_map(k_pool, pool_num_blocks, block_size, num_kv_heads, head_dim, &tk);
      if (st == PA_OK) st = payload_map(v_pool, pool_num_blocks, block_size, num_kv_heads, head_dim, &tv);
      if (st != PA_OK) return st;
    }
    e = launch_kv8_tiles(dtype, head_dim, tk, tv, q, err, stream);
    if (e != cudaSuccess) return kv8_cuda_fail(e, "8-bit attention tiles launch");
    launched |= PA_LAUNCH_KV8_TILES;
  }
  if (rows) e = launch_kv8_rows_combine(dtype, head_dim, f.row_groups, p, stream);
  if (e == cudaSuccess && tiles) e = launch_kv8_tiles_combine(dtype, head_dim, q, stream);
  if (e != cudaSuccess) return kv8_cuda_fail(e, "8-bit attention join launch");
  if ((rows && p.slices > 1) || (tiles && q.slices > 1)) launched |= PA_LAUNCH_KV8_COMBINE;
  note_launches(launched);
  return PA_OK;
}

int32_t pa_kv8_read_error(int32_t clear, int32_t* error_word, void* stream_ptr) {
  using namespace pa;
  if (!error_word) return fail(PA_ERR_INVALID_ARGUMENT, "NULL pointer");
  int* err = kv8_error_word();
  if (!err) return fail(PA_ERR_CUDA, "no CUDA device");
  return pa_read_device_error(err, clear, error_word, stream_ptr);
}

}  // extern "C"
