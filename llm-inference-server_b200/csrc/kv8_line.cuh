// The work line of the KV8 attention kernels.
//
// A tile is `tile_tokens` consecutive new tokens of one sequence (all query heads of a KV
// head); it visits keys 0 .. its last token's position.  All tiles of a class laid end to
// end, each as long as its number of keys, form a line that is cut into equal slices, one
// per CTA and KV head: every CTA streams the same number of keys whatever the lengths are,
// and the launch does not depend on them.  A cut inside a tile is moved up to the next
// multiple of the kernel's key step, the same for both of its neighbours.
#pragma once

#include <stdint.h>

namespace pa {

// Keys of tile i of a sequence with q new tokens behind `base` cached ones.
__host__ __device__ __forceinline__ int64_t line_tile_keys(int64_t base, int64_t q, int64_t tt, int64_t i) {
  const int64_t last = (i + 1) * tt;
  return base + (last < q ? last : q);
}

// Keys of the first n tiles: full tiles visit base + tt, base + 2 tt, ...
__host__ __device__ __forceinline__ int64_t line_keys_before(int64_t base, int64_t q, int64_t tt, int64_t n) {
  const int64_t full = n < q / tt ? n : q / tt;
  return full * base + tt * (full * (full + 1) / 2) + (n > full ? base + q : 0);
}

struct LineTile {
  int seq;          // -1: past the end of the line
  int index;        // tile of the sequence
  int64_t start;    // place of its first key on the line
  int keys;
};

// End of slice s - 1 / start of slice s out of n over a line of `total` keys.
__device__ __forceinline__ int64_t line_cut(int64_t total, int n, int s) { return total * s / n; }

// Slices that a line of `total` keys is worth: at least `min_keys` each.
__device__ __forceinline__ int line_slices(int64_t total, int most, int min_keys) {
  const int64_t n = (total + min_keys - 1) / min_keys;
  return n < 1 ? 1 : (n < most ? int(n) : most);
}

// A place x of the line as a key of the tile, moved up to a multiple of `step`.
__device__ __forceinline__ int line_key(const LineTile& t, int64_t x, int step) {
  const int64_t d = x - t.start;
  if (d <= 0) return 0;
  const int64_t k = (d + step - 1) / step * step;
  return k < t.keys ? int(k) : t.keys;
}

// The tile that holds place x.  Called by a whole warp; `work` is the class's running sum.
__device__ __forceinline__ LineTile line_find(const int64_t* work, int num_seqs, const int32_t* ctx_lens,
                                              const int32_t* cu_q, int tt, int64_t x, int hint) {
  const int lane = threadIdx.x & 31;
  LineTile t;
  t.seq = -1;
  if (x >= work[num_seqs]) return t;
  // Largest i with work[i] <= x; the next 32 sequences first, then a 32-way search.
  int lo = 0, hi = num_seqs;  // work[lo] <= x < work[hi]
  {
    const int i = min(hint + 1 + lane, num_seqs);
    const unsigned above = __ballot_sync(0xffffffffu, work[i] > x);
    if (above) {
      hi = min(hint + __ffs(above), num_seqs);
      lo = hi - 1;
    } else {
      lo = min(hint + 32, num_seqs - 1);
    }
  }
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int i = min(lo + step * (lane + 1), hi);
    const unsigned above = __ballot_sync(0xffffffffu, work[i] > x);
    const int f = __ffs(above) - 1;  // lane 31 probes hi
    hi = min(lo + step * (f + 1), hi);
    lo = lo + step * f;
  }
  const int q = cu_q[lo + 1] - cu_q[lo], ctx = ctx_lens[lo];
  const int64_t base = ctx - q, rest = x - work[lo];
  int a = 0, b = (q + tt - 1) / tt;  // keys_before(a) <= rest < keys_before(b)
  while (b - a > 1) {
    const int m = (a + b) / 2;
    if (line_keys_before(base, q, tt, m) <= rest)
      a = m;
    else
      b = m;
  }
  t.seq = lo;
  t.index = a;
  t.start = work[lo] + line_keys_before(base, q, tt, a);
  t.keys = int(line_tile_keys(base, q, tt, a));
  return t;
}

}  // namespace pa
