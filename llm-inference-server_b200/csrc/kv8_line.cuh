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

#include "kv8.h"
#include "pa_common.cuh"

namespace pa {

// Keys of tile i of a sequence with q new tokens behind `base` cached ones.
__host__ __device__ __forceinline__ int line_tile_keys(int base, int q, int tt, int i) {
  const int64_t last = int64_t(i + 1) * tt;
  return base + (last < q ? int(last) : q);
}

// Keys of the first n tiles: full tiles visit base + tt, base + 2 tt, ...
__host__ __device__ __forceinline__ int64_t line_keys_before(int base, int q, int tt, int n) {
  const int whole = q / tt, full = n < whole ? n : whole;
  return int64_t(full) * base + int64_t(tt) * (int64_t(full) * (full + 1) / 2) + (n > full ? int64_t(base) + q : 0);
}

struct LineTile {
  int seq;          // -1: past the end of the line
  int index;        // tile of the sequence
  int64_t start;    // place of its first key on the line
  int keys;
  int first, q, ctx;  // of the sequence: packed index of its first token, new tokens, context
};

// The line's cuts: at least `min_keys` keys a slice (a power of two times 32 or so), at most
// `most` slices; slice s is [at(s), at(s + 1)).  Divisions of 64 bits are worth avoiding: they
// stand before a CTA's first load.
struct LineCuts {
  int64_t each;
  uint32_t rest;
  int n;

  __device__ __forceinline__ LineCuts(int64_t total, int most, int min_keys) {
    if (total >> 32) {
      n = most;  // 2^32 keys are worth any number of slices
      each = total / n;
      rest = uint32_t(total % n);
    } else {
      const uint32_t t = uint32_t(total), worth = t / uint32_t(min_keys) + (t % uint32_t(min_keys) ? 1 : 0);
      n = worth < 1 ? 1 : (worth < uint32_t(most) ? int(worth) : most);
      each = t / uint32_t(n);
      rest = t % uint32_t(n);
    }
  }
  __device__ __forceinline__ explicit LineCuts(const Kv8Join& j) : each(j.each), rest(j.rest), n(j.n) {}
  __device__ __forceinline__ int64_t at(int s) const { return each * s + rest * uint32_t(s) / uint32_t(n); }
};

// A place x of the line as a key of the tile, moved up to a multiple of `step`, a power of two.
__device__ __forceinline__ int line_key(const LineTile& t, int64_t x, int step) {
  const int64_t d = x - t.start;
  if (d <= 0) return 0;
  if (d >= t.keys) return t.keys;
  return min((int(d) + step - 1) & ~(step - 1), t.keys);
}

// Looks tiles up by place; a whole warp's.  Finding one is a chain of dependent loads, which is
// most of what a short call costs, so lane i keeps what belongs to sequence hint + i: loaded
// in one go, before the first place is even known, and enough for any batch of up to 32
// sequences and for walking from a sequence to the next.
//
// Without a step's sums (p.work NULL, at most kKv8Direct sequences) every warp makes them from
// the lengths by scans over its lanes, with the step kernel's checks: with a launch for them
// 48 x ~700 keys took 26.7 us instead of 23.7, 50 chunks of 50 over ~700 95 instead of 90.  A
// lane then has two sequences, i and i + 32; places only grow, so the second 32 take the
// first's registers when a place lies behind those.
struct LineFinder {
  const int64_t* work;
  const int32_t *ctx_lens, *cu_q;
  int num_seqs, tt, hint;
  int64_t total;       // keys on the line
  int64_t begin, end;  // of the lane's sequence on the line
  int first, next, ctx;
  int64_t begin2, end2;  // without a step's sums: of sequence 32 + lane
  int first2, next2, ctx2;

  __device__ __forceinline__ void load(int from) {
    hint = from;
    const int i = min(from + int(threadIdx.x & 31), num_seqs - 1);
    begin = work[i];
    end = work[i + 1];
    first = cu_q[i];
    next = cu_q[i + 1];
    ctx = ctx_lens[i];
  }

  __device__ __forceinline__ LineFinder(const Kv8AttnParams& p, int* err)
      : work(p.work), ctx_lens(p.ctx_lens), cu_q(p.cu_q), num_seqs(p.num_seqs), tt(p.tile_tokens) {
    if (work) {
      load(0);
      total = work[num_seqs];
      return;
    }
    hint = 0;
    const int lane = threadIdx.x & 31;
    int q = 0, q2 = 0;
    ctx = ctx2 = 0;
    if (lane < num_seqs) {
      ctx = ctx_lens[lane];
      q = p.query_lens[lane];
    }
    if (lane + 32 < num_seqs) {
      ctx2 = ctx_lens[lane + 32];
      q2 = p.query_lens[lane + 32];
    }
    bool bad = false;
    const int n1 = sum_up(p, q, 0, 0, begin, end, first, next, ctx, bad);
    total = __shfl_sync(0xffffffffu, end, 31);
    int n2 = n1;
    if (num_seqs > 32) {
      n2 = sum_up(p, q2, total, n1, begin2, end2, first2, next2, ctx2, bad);
      total = __shfl_sync(0xffffffffu, end2, 31);
    }
    // 64 chunks of at most 2^20 tokens: the sum fits 32 bits.
    if (__any_sync(0xffffffffu, bad) || n2 > p.num_tokens) {
      total = 0;
      if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) set_error(err, PA_KV8_ERR_STEP);
    }
  }

  // The sums of 32 sequences, the lane's with q new tokens and ctx keys, behind `keys0` keys and
  // `tokens0` tokens; gives the tokens of all so far.
  __device__ __forceinline__ static int sum_up(const Kv8AttnParams& p, int q, int64_t keys0, int tokens0,
                                               int64_t& begin, int64_t& end, int& first, int& next, int& ctx,
                                               bool& bad) {
    const int lane = threadIdx.x & 31, tt = p.tile_tokens;
    if (q < 0 || q > p.max_query_len || ctx < q || ctx > p.max_context) {
      bad = true;
      q = ctx = 0;
    }
    const bool mine = (q <= p.small_max) == p.few;
    const int64_t keys = q > 0 && mine ? line_keys_before(ctx - q, q, tt, (q + tt - 1) / tt) : 0;
    next = q;
    end = keys;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, next, d);
      const int64_t up_keys = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) {
        next += up;
        end += up_keys;
      }
    }
    next += tokens0;
    end += keys0;
    first = next - q;
    begin = end - keys;
    return __shfl_sync(0xffffffffu, next, 31);
  }

  // The tile that holds place x, with work[hint] <= x < total.
  __device__ __forceinline__ LineTile find(int64_t x) {
    const int lane = threadIdx.x & 31;
    unsigned above = __ballot_sync(0xffffffffu, end > x);
    if (!above && !work) {
      hint = 32;
      begin = begin2;
      end = end2;
      first = first2;
      next = next2;
      ctx = ctx2;
      above = __ballot_sync(0xffffffffu, end > x);
    } else if (!above) {
      // Largest i with work[i] <= x: a 32-way search, then the sequences from there.
      int lo = min(hint + 32, num_seqs - 1), hi = num_seqs;  // work[lo] <= x < work[hi]
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const unsigned up = __ballot_sync(0xffffffffu, work[min(lo + step * (lane + 1), hi)] > x);
        const int f = __ffs(up) - 1;  // lane 31 probes hi
        hi = min(lo + step * (f + 1), hi);
        lo = lo + step * f;
      }
      load(lo);
      above = 1u;
    }
    const int f = __ffs(above) - 1;
    LineTile t;
    t.seq = hint + f;
    t.first = __shfl_sync(0xffffffffu, first, f);
    t.q = __shfl_sync(0xffffffffu, next, f) - t.first;
    t.ctx = __shfl_sync(0xffffffffu, ctx, f);
    const int base = t.ctx - t.q;
    const int64_t at = __shfl_sync(0xffffffffu, begin, f), rest = x - at;
    int a = 0, b = (t.q + tt - 1) / tt;  // keys_before(a) <= rest < keys_before(b)
    while (b - a > 1) {
      const int m = (a + b) / 2;
      if (line_keys_before(base, t.q, tt, m) <= rest)
        a = m;
      else
        b = m;
    }
    t.index = a;
    t.start = at + line_keys_before(base, t.q, tt, a);
    t.keys = line_tile_keys(base, t.q, tt, a);
    return t;
  }
};

// The pieces of a slice [x, end), in order: the parts of its tiles, cut at multiples of `step`.
struct LinePiece {
  LineTile t;
  int k0, k1;  // keys
};
__device__ __forceinline__ bool line_next_piece(LineFinder& f, int64_t& x, int64_t end, int step, LinePiece& d) {
  while (x < end) {
    d.t = f.find(x);
    d.k0 = line_key(d.t, x, step);
    d.k1 = line_key(d.t, end, step);
    x = d.t.start + d.t.keys;
    if (d.k1 > d.k0) return true;
  }
  return false;
}

// Tile t, which starts in slice s and does not end there: at most one a slice, so whoever works
// on it leaves word and nobody has to look for shared tiles.
__device__ __forceinline__ Kv8Join line_join(const LineTile& t, const LineCuts& cuts, int s, int tile_tokens) {
  const int64_t end = t.start + t.keys;
  // The last slice with a part: the largest i with at(i) < end; slices differ by one key at
  // most, so a guess by their length is next to it.
  int last = min(s + 1 + int((end - cuts.at(s + 1)) / max(cuts.each, int64_t(1))), cuts.n - 1);
  while (last + 1 < cuts.n && cuts.at(last + 1) < end) ++last;
  while (last > s + 1 && cuts.at(last) >= end) --last;
  const int t0 = t.index * tile_tokens;
  return {t.start, cuts.each, cuts.rest, cuts.n, t.keys, t.first + t0, min(tile_tokens, t.q - t0), last};
}

}  // namespace pa
