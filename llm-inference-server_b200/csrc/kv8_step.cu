// A step's block tables, slot map and work sums built on the GPU from request lengths, and
// the two small kernels that keep the request slots (commit, release).
//
//   context_i = lens[r_i] + q_i,   need_i = max(0, ceil(context_i / block_size) - held[r_i])
//   new block k of row i = free[num_free - 1 - (need_0 + ... + need_{i-1}) - k]
//   slot of token t of row i = table_i[p / block_size] * block_size + p % block_size,
//                              p = context_i - q_i + t
//
// The prefix sums over rows are what every other output needs.  Rows are few (thousands at
// most) and a grid-wide wait or a second launch costs more than the sums, so every CTA
// computes them for itself in shared memory and then fills its share of the tables and of
// the per-token arrays; no CTA reads what another writes (a new block's id comes from the
// free list by arithmetic, not from the table that it is also written to).  What bounds it is
// latency, of the lengths' loads, of the scan and of the look at the new blocks' ids: 8 rows 6.2
// us, 500 rows with 2.6 MB of tables 12, 13 prompts of 2,047 tokens 8.2 (captured, one behind the
// other, 4.9, 9.2 and 5.9).
#include "kv8.h"
#include "kv8_launch.cuh"
#include "kv8_line.cuh"
#include "pa_common.cuh"

namespace pa {

constexpr int kStepThreads = 512;

// Sums over the block: each of v[N] becomes the sum of the threads' before this one; `total`
// gets the sums over all.  `scratch` holds N values per warp; one pair of barriers for all N.
template <int N>
__device__ __forceinline__ void block_scan(int64_t (&v)[N], int64_t (&total)[N], int64_t (*scratch)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t sum[N];
#pragma unroll
  for (int n = 0; n < N; ++n) sum[n] = v[n];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int64_t up = __shfl_up_sync(0xffffffffu, sum[n], d);
      if (lane >= d) sum[n] += up;
    }
  if (lane == 31)
#pragma unroll
    for (int n = 0; n < N; ++n) scratch[warp][n] = sum[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    // One warp's worth of partial sums, added up by every warp.
    int64_t w = lane < warps ? scratch[lane][n] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += up;
    }
    total[n] = __shfl_sync(0xffffffffu, w, warps - 1);
    const int64_t before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    v[n] = (warp > 0 ? before : 0) + sum[n] - v[n];
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kStepThreads) kv8_step_kernel(const Kv8StepParams p, int* err) {
  extern __shared__ int32_t sm[];
  const int rows = p.num_rows;
  int32_t* s_cu = sm;                 // [rows + 1] tokens before the row
  int32_t* s_ctx = s_cu + rows + 1;   // [rows]
  int32_t* s_new = s_ctx + rows;      // [rows] new blocks before the row
  int32_t* s_held = s_new + rows;     // [rows]
  int32_t* s_row = s_held + rows;     // [rows] request slot or -1
  uint32_t* s_seen = reinterpret_cast<uint32_t*>(s_row + rows);  // a bit per slot, with row_ids only
  __shared__ int64_t scan[kStepThreads / 32][4];
  const int tid = threadIdx.x;
  pdl_release();

  if (p.row_ids) {
    for (int i = tid; i < (p.num_slots + 31) / 32; i += blockDim.x) s_seen[i] = 0u;
    __syncthreads();
  }
  const int avail = p.held ? *p.num_free : 0;

  int bad = 0;
  int64_t tokens = 0, blocks = 0, small = 0, large = 0;  // totals so far
  for (int first = 0; first < rows; first += blockDim.x) {
    const int i = first + tid;
    int q = 0, ctx = 0, held = 0, need = 0, row = -1, into = 0;
    bool touches = false;
    if (i < rows) {
      row = p.row_ids ? p.row_ids[i] : i;
      if (row >= p.num_slots || row < -1) {
        bad |= PA_KV8_ERR_STEP;
        row = -1;
      }
      if (row >= 0) {
        if (p.row_ids && (atomicOr(&s_seen[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u)) bad |= PA_KV8_ERR_STEP;
        q = p.query_lens[i];
        const int64_t len = p.lens[row];
        const int64_t c = p.held ? len + q : len;
        held = p.held ? p.held[row] : 0;
        const int64_t most = int64_t(p.width) * p.block_size;
        if (q < 0 || q > p.max_query_len || len < 0 || c < q || c > most || held < 0 || held > p.width) {
          bad |= PA_KV8_ERR_STEP;
          q = held = 0;
        } else {
          ctx = int(c);
          if (p.held) {
            need = max(0, (ctx + p.block_size - 1) / p.block_size - held);
            // Blocks held before that take new tokens: a token without a place must not count.  The
            // first, mostly the only one, is looked at behind the sums, which hide its load.
            const int32_t* mine = p.tables + int64_t(row) * p.table_stride;
            const int last = q > 0 ? min(held, (ctx + p.block_size - 1) / p.block_size) : 0;
            int j = int(len) / p.block_size;
            touches = j < last;
            if (touches) into = mine[j];
            while (++j < last) bad |= mine[j] < 0 || mine[j] >= p.pool_blocks ? PA_KV8_ERR_BLOCK : 0;
          }
        }
      }
      s_ctx[i] = ctx;
      s_held[i] = held;
      s_row[i] = row;
    }
    const bool few = q <= p.tiling.small_max;
    const int tt = few ? p.tiling.small_tokens : p.tiling.large_tokens;
    const int64_t keys = q > 0 ? line_keys_before(ctx - q, q, tt, (q + tt - 1) / tt) : 0;
    int64_t v[4] = {q, need, few ? keys : 0, few ? 0 : keys}, total[4];
    block_scan(v, total, scan);
    if (touches && (into < 0 || into >= p.pool_blocks)) bad |= PA_KV8_ERR_BLOCK;
    if (i < rows) {
      s_cu[i] = int32_t(tokens + v[0]);
      s_new[i] = int32_t(blocks + v[1]);
      if (blockIdx.x == 0) {
        p.work[i] = small + v[2];
        p.work[rows + 1 + i] = large + v[3];
      }
    }
    tokens += total[0];
    blocks += total[1];
    small += total[2];
    large += total[3];
    if (tokens > p.num_tokens) bad |= PA_KV8_ERR_STEP;
  }
  if (p.held) {
    if (avail < 0 || avail > p.free_capacity)
      bad |= PA_KV8_ERR_STEP;
    else if (blocks > avail)
      bad |= PA_KV8_ERR_NO_BLOCKS;
    else {
#pragma unroll 4
      for (int b = tid; b < int(blocks); b += blockDim.x) {  // the new blocks: the list's last ones
        const int id = p.free_blocks[avail - 1 - b];
        if (id < 0 || id >= p.pool_blocks) bad |= PA_KV8_ERR_BLOCK;
      }
    }
  }
  if (tid == 0) s_cu[rows] = int32_t(tokens);
  const bool reject = __syncthreads_or(bad) != 0;
  if (blockIdx.x == 0) {
    if (bad) set_error(err, bad);
    for (int i = tid; i <= rows; i += blockDim.x) {
      p.cu_query[i] = reject ? 0 : s_cu[i];
      if (reject) p.work[i] = p.work[rows + 1 + i] = 0;
      if (i < rows) {
        const int need = (i + 1 < rows ? s_new[i + 1] : int32_t(blocks)) - s_new[i];
        if (p.held) p.num_free_out[PA_KV8_STEP_WORDS + i] = s_row[i];
        if (p.context_lens) {
          p.context_lens[i] = reject ? 0 : s_ctx[i];
          p.query_out[i] = reject ? 0 : s_cu[i + 1] - s_cu[i];
          p.held_out[i] = reject ? 0 : s_held[i] + need;
        }
      }
    }
    if (tid == 0) {
      if (!reject) {
        p.work[rows] = small;
        p.work[2 * rows + 1] = large;
      }
      const int left = reject ? -1 : avail - int32_t(blocks);
      if (p.held)
        *reinterpret_cast<Kv8StepRecord*>(p.num_free_out) = {
            left,     rows,          p.width,  p.block_size,   p.free_capacity, 0,            p.lens,    p.held,
            p.num_free, p.free_blocks, p.tables, p.table_stride, p.out_tables,    p.context_lens, p.held_out};
      else if (p.num_free_out)
        *p.num_free_out = left;
    }
  }

  // Block tables: what the row holds, then its new blocks, then zeros.
  const int64_t stride = int64_t(gridDim.x) * blockDim.x, me = int64_t(blockIdx.x) * blockDim.x + tid;
  auto block_of = [&](int i, int j) -> int {  // j below the row's blocks
    const int k = j - s_held[i];
    return k < 0 ? p.tables[int64_t(s_row[i]) * p.table_stride + j] : p.free_blocks[avail - 1 - s_new[i] - k];
  };
  if (p.held) {
    const int64_t cells = int64_t(rows) * p.width;
    for (int64_t c = me; c < cells; c += stride) {
      const int i = int(c / p.width), j = int(c - int64_t(i) * p.width);
      int id = 0;
      if (!reject && s_row[i] >= 0) {
        const int need = (i + 1 < rows ? s_new[i + 1] : int32_t(blocks)) - s_new[i];
        if (j < s_held[i] + need) {
          id = block_of(i, j);
          if (id < 0 || id >= p.pool_blocks) set_error(err, PA_KV8_ERR_BLOCK);
          if (j >= s_held[i]) p.tables[int64_t(s_row[i]) * p.table_stride + j] = id;
        }
      }
      p.out_tables[c] = id;
    }
  }
  if (!p.seq_idx) return;
  // Per-token arrays.
  for (int64_t t = me; t < p.num_tokens; t += stride) {
    int seq = -1, pos = -1, slot = -1;
    if (!reject && t < tokens) {
      int lo = 0, hi = rows;  // s_cu[lo] <= t < s_cu[hi]
      while (hi - lo > 1) {
        const int m = (lo + hi) / 2;
        if (s_cu[m] <= t)
          lo = m;
        else
          hi = m;
      }
      seq = lo;
      pos = s_ctx[lo] - s_cu[lo + 1] + int(t);
      const int j = pos / p.block_size;
      const int id = p.held ? block_of(lo, j) : p.tables[int64_t(s_row[lo]) * p.table_stride + j];
      if (id < 0 || id >= p.pool_blocks)
        set_error(err, PA_KV8_ERR_BLOCK);
      else
        slot = id * p.block_size + pos % p.block_size;
    }
    p.seq_idx[t] = seq;
    p.q_pos[t] = pos;
    p.slots[t] = slot;
  }
}

// Row of item b in running sums at[0 .. rows] (at[row] <= b < at[row + 1]).
__device__ __forceinline__ int row_of(const int32_t* at, int rows, int b) {
  int lo = 0, hi = rows;
  while (hi - lo > 1) {
    const int m = (lo + hi) / 2;
    if (at[m] <= b)
      lo = m;
    else
      hi = m;
  }
  return lo;
}

// One CTA.  A step is planned from the slots and the free list as they are then, and other steps
// may count or blocks come back before it does, so the plan is compared first: each slot's
// length, the blocks of its last token and of those that the step brings, and that the step's new
// blocks are still the free list's last ones.  Then all of it is written, or nothing.  (A slot that
// was released and filled again to the same length with the same blocks looks the same.)  What bounds it is latency: the
// rows, their slots, the new blocks are three dependent loads, so a block's thread has nothing
// else to look up in global memory (with its slot and place read there: 12 us for 8 prompts of
// 4,096 tokens, 2,048 blocks, instead of 4.5).
constexpr int kCommitThreads = 1024;
__global__ void __launch_bounds__(kCommitThreads)
    kv8_commit_kernel(const int32_t* query_lens, const int32_t* accepted, const int32_t* held_out,
                      const Kv8StepRecord* record, int rows, int slots, int32_t* lens, int32_t* held,
                      int32_t* num_free, int* err) {
  extern __shared__ int32_t sm[];
  int32_t* s_at = sm;              // [rows + 1] new blocks before the row
  int32_t* s_row = s_at + rows + 1;  // [rows] request slot or -1
  int32_t* s_held = s_row + rows;  // [rows]
  __shared__ int64_t scan[kCommitThreads / 32][1];
  const int tid = threadIdx.x;
  const Kv8StepRecord r = *record;
  const int32_t* rows_of_step = reinterpret_cast<const int32_t*>(record + 1);
  const int have = *num_free;
  if (r.num_free < 0) return;  // the step was emptied
  if (r.lens != lens || r.held != held || r.num_free_at != num_free || r.held_out != held_out || r.rows != rows) {
    if (tid == 0) set_error(err, PA_KV8_ERR_STEP);  // of other tables
    return;
  }
  int bad = 0;
  int64_t blocks = 0;
  for (int first = 0; first < rows; first += blockDim.x) {
    const int i = first + tid;
    int need = 0;
    if (i < rows) {
      int row = rows_of_step[i], mine = 0;
      if (row >= slots) row = -1;
      if (row >= 0) {
        const int q = query_lens[i], ctx = r.context_lens[i], base = lens[row];
        mine = held[row];
        need = held_out[i] - mine;
        if (mine < 0 || need < 0 || held_out[i] > r.width || base < 0 || base + q != ctx) {
          bad = 1;
          need = 0;
        } else if (q > 0) {
          const int32_t *now = r.tables + int64_t(row) * r.table_stride, *then = r.out_tables + int64_t(i) * r.width;
          for (int j = max(base - 1, 0) / r.block_size; j < mine && j * r.block_size < ctx; ++j) bad |= now[j] != then[j];
        }
      }
      s_row[i] = row;
      s_held[i] = mine;
    }
    int64_t at[1] = {need}, sum[1];
    block_scan(at, sum, scan);
    if (i < rows) s_at[i] = int32_t(blocks + at[0]);
    blocks += sum[0];
  }
  if (tid == 0) s_at[rows] = int32_t(blocks);
  if (have > r.free_capacity || blocks > have) bad = 1;
  bool stale = __syncthreads_or(bad) != 0, other = false;
  // A new block's place in its slot's table, of which `other` learns that another plan, one that
  // was dropped, has been written there.
  auto place = [&](int i, int b) { return r.tables + int64_t(s_row[i]) * r.table_stride + s_held[i] + b - s_at[i]; };
  if (!stale && blocks > 0) {
    for (int b = tid; b < int(blocks); b += blockDim.x) {
      const int i = row_of(s_at, rows, b), id = r.out_tables[int64_t(i) * r.width + s_held[i] + b - s_at[i]];
      bad |= r.free_blocks[have - 1 - b] != id;
      other |= *place(i, b) != id;
    }
    stale = __syncthreads_or(bad) != 0;
  }
  if (stale) {
    if (tid == 0) set_error(err, PA_KV8_ERR_STEP);
    return;
  }
  if (other)
    for (int b = tid; b < int(blocks); b += blockDim.x) *place(row_of(s_at, rows, b), b) = r.free_blocks[have - 1 - b];
  for (int i = tid; i < rows; i += blockDim.x) {
    const int row = s_row[i];
    if (row < 0) continue;
    const int q = query_lens[i];
    lens[row] += accepted ? max(0, min(accepted[i], q)) : q;
    held[row] = held_out[i];
  }
  if (tid == 0) *num_free = have - int(blocks);
}

// One CTA: a release is rare and short, and its places on the free list depend on one
// another through the running sum.  8 slots of 256 blocks 6 us, 64 of 64 8, 4,096 of 32 235.
__global__ void __launch_bounds__(kStepThreads) kv8_release_kernel(const int32_t* ids, int count, const int32_t* tables,
                                                                   int64_t table_stride, int width, int slots,
                                                                   int32_t* lens, int32_t* held, int32_t* free_blocks,
                                                                   int free_capacity, int32_t* num_free, int* err) {
  extern __shared__ int32_t sm[];
  int32_t* s_at = sm;            // [count + 1] blocks before the id
  uint32_t* s_seen = reinterpret_cast<uint32_t*>(s_at + count + 1);
  __shared__ int64_t scan[kStepThreads / 32][1];
  const int tid = threadIdx.x;
  for (int i = tid; i < (slots + 31) / 32; i += blockDim.x) s_seen[i] = 0u;
  __syncthreads();
  int bad = 0;
  int64_t blocks = 0;
  for (int first = 0; first < count; first += blockDim.x) {
    const int i = first + tid;
    int n = 0;
    if (i < count) {
      const int row = ids[i];
      if (row >= slots || row < -1) {
        bad = 1;
      } else if (row >= 0) {
        if (atomicOr(&s_seen[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u) bad = 1;
        n = held[row];
        if (n < 0 || n > width) {
          bad = 1;
          n = 0;
        }
      }
    }
    int64_t at[1] = {n}, sum[1];
    block_scan(at, sum, scan);
    if (i < count) s_at[i] = int32_t(blocks + at[0]);
    blocks += sum[0];
  }
  const int have = *num_free;
  if (have < 0 || have + blocks > free_capacity) bad = 1;
  if (tid == 0) s_at[count] = int32_t(blocks);
  if (__syncthreads_or(bad)) {
    if (tid == 0) set_error(err, PA_KV8_ERR_STEP);
    return;
  }
  for (int b = tid; b < int(blocks); b += blockDim.x) {
    const int i = row_of(s_at, count, b);
    free_blocks[have + b] = tables[int64_t(ids[i]) * table_stride + (s_at[i + 1] - 1 - b)];
  }
  for (int i = tid; i < count; i += blockDim.x)
    if (ids[i] >= 0) lens[ids[i]] = held[ids[i]] = 0;
  if (tid == 0) *num_free = have + int(blocks);
}

// ------------------------------------------------------------------ launch
static __device__ int g_kv8_error;

int* kv8_error_word() {
  static int* known[64] = {};  // a device's word stays where it is
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (!known[dev]) {
    void* at = nullptr;
    if (cudaGetSymbolAddress(&at, g_kv8_error) != cudaSuccess) return nullptr;
    known[dev] = static_cast<int*>(at);
  }
  return known[dev];
}

// Asked for once per device and for the largest call: a request per call, of its own size, took
// back what another host thread had just asked for.
static cudaError_t allow_smem(const void* kern, size_t most, bool (&asked)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (asked[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(most));
  if (e == cudaSuccess) asked[dev] = true;
  return e;
}
static constexpr size_t step_smem(size_t rows, size_t slots) { return 4 * (5 * rows + 1) + 4 * ((slots + 31) / 32); }
static constexpr size_t commit_smem(size_t rows) { return 4 * (3 * rows + 1); }
static constexpr size_t release_smem(size_t count, size_t slots) { return 4 * (count + 1) + 4 * ((slots + 31) / 32); }

cudaError_t launch_kv8_step(const Kv8StepParams& p, int* err, cudaStream_t stream) {
  const size_t smem = step_smem(size_t(p.num_rows), p.row_ids ? size_t(p.num_slots) : 0);
  static bool asked[64];
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kv8_step_kernel),
                             step_smem(PA_KV8_MAX_ROWS, PA_KV8_MAX_REQUESTS), asked);
  if (e != cudaSuccess) return e;
  // As many threads as rows or new blocks, within limits: a sum over fewer warps is quicker.
  const int threads = p.num_rows <= 128 && p.num_tokens <= 128 * p.block_size ? 128 : kStepThreads;
  const int64_t cells = (p.held ? int64_t(p.num_rows) * p.width : 0) + (p.seq_idx ? p.num_tokens : 0);
  const int64_t want = (cells + threads - 1) / threads;
  const int grid = int(want < 1 ? 1 : (want < 148 ? want : 148));
  kv8_step_kernel<<<grid, threads, smem, stream>>>(p, err);
  return cudaGetLastError();
}

cudaError_t launch_kv8_commit(const int32_t* query_lens, const int32_t* accepted,
                              const int32_t* held_out, const Kv8StepRecord* record, int32_t rows, int32_t slots,
                              int32_t* lens, int32_t* held, int32_t* num_free, int* err, cudaStream_t stream) {
  const size_t smem = commit_smem(size_t(rows));
  static bool asked[64];
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kv8_commit_kernel), commit_smem(PA_KV8_MAX_ROWS), asked);
  if (e != cudaSuccess) return e;
  kv8_commit_kernel<<<1, kCommitThreads, smem, stream>>>(query_lens, accepted, held_out, record, rows, slots, lens, held,
                                                         num_free, err);
  return cudaGetLastError();
}

cudaError_t launch_kv8_release(const int32_t* ids, int32_t count, const int32_t* tables, int64_t table_stride,
                               int32_t width, int32_t slots, int32_t* lens, int32_t* held, int32_t* free_blocks,
                               int32_t free_capacity, int32_t* num_free, int* err, cudaStream_t stream) {
  const size_t smem = release_smem(size_t(count), size_t(slots));
  static bool asked[64];
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kv8_release_kernel),
                             release_smem(PA_KV8_MAX_ROWS, PA_KV8_MAX_REQUESTS), asked);
  if (e != cudaSuccess) return e;
  kv8_release_kernel<<<1, kStepThreads, smem, stream>>>(ids, count, tables, table_stride, width, slots, lens, held,
                                                        free_blocks, free_capacity, num_free, err);
  return cudaGetLastError();
}

}  // namespace pa
