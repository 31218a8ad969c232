// Attention of few new tokens per sequence over the 8-bit paged cache (decode, and chunks
// whose (token, head) rows fit one or two groups of 8), on mma.sync.
//
// For each row r = (new token t, query head of the KV head):
//   s_j = scale * q_r . K_j,  out_r = sum_j softmax_j(s) V_j,  j <= position of t
// with K_j = k_j 2^a_j and V_j = v_j 2^b_j, where k, v are e4m3 and a, b the rows' exponents.
// e4m3 widens to fp16 exactly, so S runs over the payloads and column j is scaled by 2^a_j;
// the weight that multiplies v_j is exp2(s_j - m) 2^(b_j + 8), rounded to fp16 (11 bits; the
// shift keeps weights of rows with the smallest exponent, -14, out of fp16's subnormals down
// to 2^-8 of the maximum, the largest is 2^15).  bf16 queries are brought into fp16 by a
// power of two per row, which is exact but for elements 2^-28 below the row's largest.
// Maximum, sum and accumulators are float32.
//
// HBM-bound: each K/V byte is read once per tile of rows.  The sequences' keys laid end to
// end are cut into equal slices (kv8_line.cuh), a CTA per slice and KV head with the KV head
// fastest, so that the CTAs of one slice read a pool block's heads side by side.  A CTA has
// four consumer warps, which take blocks of 16 keys in turn, and a producer warp, which
// walks the slice's pieces, reads the block table and keeps each consumer's ring full: the
// rings run across pieces, so a new sequence costs no drain.  Per block: K and V tile by TMA
// (a 16-row box); the 16 + 16 scale bytes through a producer lane's registers, a round of 32
// blocks ahead (as bulk copies of 16 bytes they cost the copy engine as much as the tiles:
// 177 us for 64 sequences of about 4,096 keys, 8 heads of 128).
//
// Widening costs one conversion per two elements and the transpose of V one byte permute per
// four: with 16-byte chunks of head_dim dealt out to the MMA's k index as ldmatrix delivers
// bytes (lane 4g + i holds dims 4i .. 4i + 3), K needs no permute at all.
#include <cuda_fp16.h>

#include "kv8.h"
#include "kv8_line.cuh"
#include "pa_common.cuh"
#include "tc_softmax.cuh"

namespace pa {

constexpr int kRowsWarps = 4;                       // consumers
constexpr int kRowsThreads = 32 * (kRowsWarps + 1);
constexpr int kRowsKeys = 16;                       // keys a stage
constexpr int kRowsDescs = 4;
// Fewest keys a slice gets: below this a CTA's set-up and its partial cost more than the
// keys it takes over.
constexpr int kRowsMinKeys = 128;
constexpr float kWeightShift = 256.f;               // 2^8, see above

template <int D, int RG>
struct RowsCfg {
  static constexpr int STAGES = D == 128 ? 4 : 8;   // 16 KB in flight per warp
  static constexpr int TILE = kRowsKeys * D;
  static constexpr int STAGE = 2 * TILE;
  static constexpr int NO = RG * (D / 8) * 2;       // accumulator registers
  static constexpr int OFF_SCALE = kRowsWarps * STAGES * STAGE;
  static constexpr int OFF_MERGE = OFF_SCALE + kRowsWarps * STAGES * 32;
  static constexpr int OFF_ML = OFF_MERGE + 2 * NO * 32 * 4;
  static constexpr int OFF_DESC = OFF_ML + kRowsWarps * RG * 8 * 8;
  static constexpr int OFF_BAR = OFF_DESC + kRowsDescs * 32;
  static constexpr int SMEM = OFF_BAR + (2 * kRowsWarps * STAGES + 2 * kRowsDescs) * 8;
};

struct RowsPiece {      // part of a tile that a CTA works on
  int32_t row0;         // packed index of the tile's first token; -1: no more pieces
  int32_t tokens;       // of the tile
  int32_t pos0;         // position of the first token
  int32_t ctx;          // of the sequence
  int32_t kb0, kb1;     // blocks of 16 keys
  int32_t part;         // -1: the whole tile, else the CTA's partial slot
  int32_t pad;
};

__device__ __forceinline__ void rows_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void rows_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsWarps) : "memory"); }

__device__ __forceinline__ void ldm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Two e4m3 values (low or high half of a word) as two fp16 values, exactly.
__device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, l;\n}\n" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}\n" : "=r"(r) : "r"(w));
  return r;
}
// D += A B, m16n8k16, fp16 operands.  With one group of rows, rows 8..15 of A are zero.
template <int RG>
__device__ __forceinline__ void mma16(float* d, const uint32_t (&a)[2 * RG], uint32_t b0, uint32_t b1) {
  if constexpr (RG == 1) {
    float x, y;
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%9,%9};"
        : "+f"(d[0]), "+f"(d[1]), "=f"(x), "=f"(y)
        : "r"(a[0]), "r"(0u), "r"(a[1]), "r"(b0), "r"(b1), "f"(0.f));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Byte offset of 16-byte chunk c of row r in a TMA tile whose rows are D bytes, with the
// swizzle as wide as the row (128 or 64 bytes).
template <int D>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  if constexpr (D == 128) return uint32_t(r * 128 + ((c ^ (r & 7)) << 4));
  return uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// Four query elements as two fp16 pairs, times 2^shift; `factor` collects 2^-shift.
template <typename T>
__device__ __forceinline__ float row_scale(float big) {  // power of two that brings `big` to [2^14, 2^15)
  const uint32_t e = (__float_as_uint(big) >> 23) & 0xffu;
  if (sizeof(T) == 2 && DType<T>::code == PA_DTYPE_F16) return 1.f;
  if (e == 0 || e == 255) return 1.f;
  const int up = 14 - (int(e) - 127);
  return __uint_as_float(uint32_t(127 + max(-126, min(127, up))) << 23);
}

template <typename T, int D, int RG>
__global__ void __launch_bounds__(kRowsThreads, RG == 1 ? 3 : 2)
    kv8_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const Kv8AttnParams p, int* err) {
  using C = RowsCfg<D, RG>;
  constexpr int CH = D / 16;  // 16-byte chunks of a row = k steps of S
  extern __shared__ __align__(1024) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + C::OFF_MERGE);
  float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  RowsPiece* desc = reinterpret_cast<RowsPiece*>(smem + C::OFF_DESC);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + kRowsWarps * C::STAGES;
  uint64_t* d_full = empty + kRowsWarps * C::STAGES;
  uint64_t* d_empty = d_full + kRowsDescs;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x % p.num_kv_heads;
  const int64_t total = p.work[p.num_seqs];
  const int slices = line_slices(total, p.slices, kRowsMinKeys);
  if (total == 0 || slice >= slices) return;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRowsWarps * C::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kRowsDescs; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], kRowsWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();

  if (warp == kRowsWarps) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tmap(&tk);
      prefetch_tmap(&tv);
    }
    const int64_t x0 = line_cut(total, slices, slice), x1 = line_cut(total, slices, slice + 1);
    int64_t x = x0;
    int issued[kRowsWarps];
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) issued[w] = 0;
    int pieces = 0, hint = 0;
    bool ok = true;
    struct BlockRef {
      int slot;  // first slot of the 16 keys
      uint4 ks, vs;
    };
    auto look_up = [&](const int32_t* row, int kb, int end) {
      BlockRef r;
      r.slot = 0;
      if (kb < end) {
        int id = row[kb >> p.block_shift];
        if (id < 0 || id >= p.pool_blocks) {
          set_error(err, PA_KV8_ERR_BLOCK);
          id = 0;
        }
        const int sub = (kb & ((1 << p.block_shift) - 1)) * 16;
        const int64_t at = ((int64_t(id) * p.num_kv_heads + kvh) << (p.block_shift + 4)) + sub;
        r.slot = (id << (p.block_shift + 4)) + sub;
        r.ks = __ldg(reinterpret_cast<const uint4*>(p.k_scale + at));
        r.vs = __ldg(reinterpret_cast<const uint4*>(p.v_scale + at));
      }
      return r;
    };
    while (ok) {
      LineTile t;
      t.seq = -1;
      int k0 = 0, k1 = 0;
      while (x < x1) {
        t = line_find(p.work, p.num_seqs, p.ctx_lens, p.cu_q, p.tile_tokens, x, hint);
        if (t.seq < 0) break;
        hint = t.seq;
        k0 = line_key(t, x, kRowsKeys);
        k1 = line_key(t, x1, kRowsKeys);
        x = t.start + t.keys;
        if (k1 > k0) break;
        t.seq = -1;
      }
      const int slot = pieces % kRowsDescs;
      if (pieces >= kRowsDescs) ok = mbar_wait(&d_empty[slot], ((pieces / kRowsDescs) - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      int ctx = 0, kb0 = 0, kb1 = 0;
      if (t.seq >= 0) {
        ctx = p.ctx_lens[t.seq];
        kb0 = k0 / kRowsKeys;
        kb1 = (k1 + kRowsKeys - 1) / kRowsKeys;
      }
      if (lane == 0) {
        RowsPiece d;
        d.row0 = -1;
        d.pad = 0;
        if (t.seq >= 0) {
          const int first = p.cu_q[t.seq], q = p.cu_q[t.seq + 1] - first, t0 = t.index * p.tile_tokens;
          d.row0 = first + t0;
          d.tokens = min(p.tile_tokens, q - t0);
          d.pos0 = ctx - q + t0;
          d.ctx = ctx;
          d.kb0 = kb0;
          d.kb1 = kb1;
          d.part = k0 > 0 ? 0 : (k1 < t.keys ? 1 : -1);
        }
        desc[slot] = d;
        rows_arrive(&d_full[slot]);
      }
      ++pieces;
      if (t.seq < 0) break;
      const int32_t* row = p.tables + int64_t(t.seq) * p.table_stride;
      // Each lane looks up one of the next 32 blocks and reads its scales, one round ahead of
      // the round whose tiles are being issued, and then issues its own block in turn.
      BlockRef cur = look_up(row, kb0 + lane, kb1), nxt;
      for (int kb = kb0; kb < kb1 && ok; kb += 32) {
        if (kb + 32 < kb1) nxt = look_up(row, kb + 32 + lane, kb1);
        const int n = min(32, kb1 - kb);
        for (int j = 0; j < n && ok; j += kRowsWarps) {
#pragma unroll
          for (int w = 0; w < kRowsWarps; ++w) {
            if (j + w < n) {
              const int st = issued[w] % C::STAGES;
              if (issued[w] >= C::STAGES)
                ok = mbar_wait(&empty[w * C::STAGES + st], ((issued[w] / C::STAGES) - 1) & 1) && ok;
              if (ok && lane == j + w) {
                uint64_t* bar = &full[w * C::STAGES + st];
                uint8_t* stage = smem + (w * C::STAGES + st) * C::STAGE;
                uint4* sc = reinterpret_cast<uint4*>(smem + C::OFF_SCALE + (w * C::STAGES + st) * 32);
                sc[0] = cur.ks;
                sc[1] = cur.vs;
                mbar_arrive_expect_tx(bar, C::STAGE);  // releases the scales too
                tma_load_3d(stage, &tk, 0, kvh, cur.slot, bar);
                tma_load_3d(stage + C::TILE, &tv, 0, kvh, cur.slot, bar);
              }
              if (ok) ++issued[w];
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        cur = nxt;
      }
    }
    if (!ok) {
      if (lane == 0) set_error(err, PA_KV8_ERR_TIMEOUT);
      // Leave with no copy into this CTA's shared memory in flight.
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w)
        for (int i = max(0, issued[w] - C::STAGES); i < issued[w]; ++i)
          mbar_wait(&full[w * C::STAGES + i % C::STAGES], (i / C::STAGES) & 1);
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, tig = lane & 3;
  const int mi = lane >> 3, ri = lane & 7;
  int taken = 0;
  bool ok = true;
  for (int piece = 0;; ++piece) {
    const int slot = piece % kRowsDescs;
    if (ok) ok = mbar_wait(&d_full[slot], (piece / kRowsDescs) & 1);
    // A timeout anywhere ends every warp at the same piece: the vote is a barrier too.
    int all;
    {
      const int mine = ok ? 1 : 0;
      asm volatile("{\n .reg .pred p, q;\n setp.ne.s32 p, %1, 0;\n barrier.cta.red.and.pred q, 2, %2, p;\n"
                   " selp.s32 %0, 1, 0, q;\n}\n"
                   : "=r"(all)
                   : "r"(mine), "n"(32 * kRowsWarps)
                   : "memory");
    }
    if (!all) break;
    const RowsPiece d = desc[slot];
    __syncwarp();
    if (lane == 0) rows_arrive(&d_empty[slot]);
    if (d.row0 < 0) break;

    // Queries as A fragments: row r = 8 rr + g is (token r / group, head r % group).
    uint32_t qa[CH][2 * RG];
    float factor[RG];
    int limit[RG];
#pragma unroll
    for (int rr = 0; rr < RG; ++rr) {
      const int r = 8 * rr + g, tok = r / p.group, head = r - tok * p.group;
      const bool valid = tok < d.tokens;
      limit[rr] = valid ? d.pos0 + tok : -1;
      const T* src = static_cast<const T*>(p.q) + int64_t(d.row0 + (valid ? tok : 0)) * p.q_st +
                     int64_t(kvh * p.group + head) * p.q_sh + 4 * tig;
      // Two passes over the row (the second from L1) rather than a row in registers.
      float big = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (valid) VecLoad<T, 4>::run(src + 16 * c, x);
        big = fmaxf(fmaxf(fmaxf(big, fabsf(x[0])), fmaxf(fabsf(x[1]), fabsf(x[2]))), fabsf(x[3]));
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const float up = row_scale<T>(big);
      factor[rr] = p.qscale / up;  // exact: a power of two
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        // fragment order {row g: k 2i..2i+1, (row g + 8: same), row g: k 2i+8.., (row g + 8)}
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (valid) VecLoad<T, 4>::run(src + 16 * c, x);
        qa[c][0 * RG + rr] = pack2<__half>(x[0] * up, x[1] * up);
        qa[c][1 * RG + rr] = pack2<__half>(x[2] * up, x[3] * up);
      }
    }

    float o[CH][2][2 * RG];  // chunk, even / odd dims, fragment
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 2 * RG; ++e) o[c][0][e] = o[c][1][e] = 0.f;
    float m[RG], l[RG];
#pragma unroll
    for (int rr = 0; rr < RG; ++rr) {
      m[rr] = -INFINITY;
      l[rr] = 0.f;
    }

    for (int kb = d.kb0 + warp; kb < d.kb1; kb += kRowsWarps, ++taken) {
      const int st = taken % C::STAGES;
      if (ok) ok = mbar_wait(&full[warp * C::STAGES + st], (taken / C::STAGES) & 1);
      const uint32_t kt = smem_u32(smem + (warp * C::STAGES + st) * C::STAGE), vt = kt + C::TILE;
      const uint8_t* sc = smem + C::OFF_SCALE + (warp * C::STAGES + st) * 32;
      // Scales of keys 2 tig, 2 tig + 1, 8 + 2 tig, 9 + 2 tig.
      float ks[2][2], vs[2][2];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const uint32_t a = *reinterpret_cast<const uint16_t*>(sc + 8 * nt + 2 * tig);
        const uint32_t b = *reinterpret_cast<const uint16_t*>(sc + 16 + 8 * nt + 2 * tig);
        ks[nt][0] = __uint_as_float((a & 0xffu) << 23);
        ks[nt][1] = __uint_as_float((a >> 8) << 23);
        vs[nt][0] = __uint_as_float((b & 0xffu) << 23) * kWeightShift;
        vs[nt][1] = __uint_as_float((b >> 8) << 23) * kWeightShift;
      }

      // ---- S over the payloads
      float s[2][2 * RG];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
        for (int e = 0; e < 2 * RG; ++e) s[nt][e] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c += 4) {
          uint32_t w[4];
          ldm4(kt + tile_at<D>(8 * nt + ri, c + mi), w);
#pragma unroll
          for (int i = 0; i < 4; ++i) mma16<RG>(s[nt], qa[c + i], widen_lo(w[i]), widen_hi(w[i]));
        }
      }

      // ---- online softmax; fragment element 2 rr + e is row 8 rr + g, key 8 nt + 2 tig + e
      const int key0 = kb * kRowsKeys + 2 * tig;
      const bool masked = kb * kRowsKeys + kRowsKeys - 1 > d.pos0;  // spare rows compute, unmasked, and are not stored
      uint32_t pa[2 * RG];
      float alpha[RG];
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        float mx = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& v = s[nt][2 * rr + e];
            v *= ks[nt][e] * factor[rr];
            if (masked && key0 + 8 * nt + e > limit[rr]) v = -INFINITY;
            mx = fmaxf(mx, v);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[rr], mx);
        const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet
        alpha[rr] = ex2(m[rr] - ref);
        m[rr] = mn;
        float sum = 0.f;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float pr = ex2(s[nt][2 * rr + e] - ref);
            sum += pr;
            w[e] = pr * vs[nt][e];
            if (masked && key0 + 8 * nt + e > limit[rr]) w[e] = 0.f;  // a hidden row may stand for NaN
          }
          pa[nt * RG + rr] = pack2<__half>(w[0], w[1]);
        }
        l[rr] = l[rr] * alpha[rr] + sum;
      }
      bool grown = false;
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) grown |= alpha[rr] != 1.f;
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int e = 0; e < 2 * RG; ++e) {
            o[c][0][e] *= alpha[e >> 1];
            o[c][1][e] *= alpha[e >> 1];
          }
      }

      // ---- O += W V
      const int left = d.ctx - kb * kRowsKeys;  // keys of this block inside the context
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if (left < kRowsKeys) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          keep[hf] = (8 * hf + 2 * tig < left ? 0x0000ffffu : 0u) | (8 * hf + 2 * tig + 1 < left ? 0xffff0000u : 0u);
      }
#pragma unroll
      for (int c = 0; c < CH; c += 2) {
        uint32_t w[4];  // (keys 0-7, chunk c), (keys 8-15, c), (0-7, c + 1), (8-15, c + 1)
        ldm4t(vt + tile_at<D>(8 * (mi & 1) + ri, c + (mi >> 1)), w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a = __byte_perm(w[2 * i] & keep[0], 0, 0x3120), b = __byte_perm(w[2 * i + 1] & keep[1], 0, 0x3120);
          mma16<RG>(o[c + i][0], pa, widen_lo(a), widen_lo(b));
          mma16<RG>(o[c + i][1], pa, widen_hi(a), widen_hi(b));
        }
      }
      __syncwarp();
      if (lane == 0) rows_arrive(&empty[warp * C::STAGES + st]);
    }

    // ---- join the four warps: common maximum, then a tree over the accumulators
    float big[RG];
#pragma unroll
    for (int rr = 0; rr < RG; ++rr) {
      l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 1);
      l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 2);
      if (tig == 0) ml[warp * 8 * RG + 8 * rr + g] = make_float2(m[rr], l[rr]);
    }
    rows_sync();
#pragma unroll
    for (int rr = 0; rr < RG; ++rr) {
      float2 v[kRowsWarps];
      big[rr] = -INFINITY;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        v[w] = ml[w * 8 * RG + 8 * rr + g];
        big[rr] = fmaxf(big[rr], v[w].x);
      }
      const float ref = big[rr] == -INFINITY ? 0.f : big[rr];
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) sum += v[w].y * ex2(v[w].x - ref);
      const float f = ex2(m[rr] - ref);
      l[rr] = sum;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          o[c][0][2 * rr + e] *= f;
          o[c][1][2 * rr + e] *= f;
        }
    }
    auto put = [&](int half) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 4 * RG; ++e)
          merge[(half * C::NO + c * 4 * RG + e) * 32 + lane] = o[c][e / (2 * RG)][e % (2 * RG)];
    };
    auto add = [&](int half) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 4 * RG; ++e)
          o[c][e / (2 * RG)][e % (2 * RG)] += merge[(half * C::NO + c * 4 * RG + e) * 32 + lane];
    };
    if (warp >= 2) put(warp - 2);
    rows_sync();
    if (warp < 2) add(warp);
    if (warp == 1) put(1);
    rows_sync();
    if (warp != 0) continue;
    add(1);
#pragma unroll
    for (int rr = 0; rr < RG; ++rr) {
      const int r = 8 * rr + g, tok = r / p.group, head = kvh * p.group + (r - tok * p.group);
      if (tok >= d.tokens) continue;
      const float f = (d.part < 0 ? 1.f / l[rr] : 1.f) * (1.f / kWeightShift);
      if (d.part < 0) {
        T* dst = static_cast<T*>(p.out) + int64_t(d.row0 + tok) * p.o_st + int64_t(head) * p.o_sh + 4 * tig;
#pragma unroll
        for (int c = 0; c < CH; ++c)
          *reinterpret_cast<uint2*>(dst + 16 * c) =
              make_uint2(pack2<T>(o[c][0][2 * rr] * f, o[c][1][2 * rr] * f),
                         pack2<T>(o[c][0][2 * rr + 1] * f, o[c][1][2 * rr + 1] * f));
      } else {
        const int64_t at = ((int64_t(slice) * p.num_kv_heads + kvh) * 2 + d.part) * (8 * RG) + r;
#pragma unroll
        for (int c = 0; c < CH; ++c)
          *reinterpret_cast<float4*>(p.part_o + at * D + 16 * c + 4 * tig) = make_float4(
              o[c][0][2 * rr] * f, o[c][1][2 * rr] * f, o[c][0][2 * rr + 1] * f, o[c][1][2 * rr + 1] * f);
        if (tig == 0) p.part_ml[at] = make_float2(big[rr], l[rr]);
      }
    }
  }
  if (!ok && lane == 0) set_error(err, PA_KV8_ERR_TIMEOUT);
}

// Joins the partials of tiles that a cut fell into.  CTA (s, kvh): the tile that the end of
// slice s falls into, if this is the first cut inside it.  A warp takes a row.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv8_combine_kernel(const Kv8AttnParams p, int rows, int key_step, int min_keys) {
  constexpr int E = D / 32;  // elements a lane
  const int64_t total = p.work[p.num_seqs];
  const int slices = line_slices(total, p.slices, min_keys);
  const int s = blockIdx.x + 1, kvh = blockIdx.y;
  if (total == 0 || s >= slices) return;
  const int64_t x = line_cut(total, slices, s);
  const LineTile t = line_find(p.work, p.num_seqs, p.ctx_lens, p.cu_q, p.tile_tokens, x, 0);
  if (t.seq < 0 || x <= t.start || line_cut(total, slices, s - 1) > t.start) return;
  if (line_key(t, x, key_step) >= t.keys) return;  // the first slice did the whole tile
  const int first = p.cu_q[t.seq], q = p.cu_q[t.seq + 1] - first, t0 = t.index * p.tile_tokens;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.z * 4 + warp, tok = r / p.group, head = kvh * p.group + (r - tok * p.group);
  if (tok >= min(p.tile_tokens, q - t0)) return;
  const int64_t end = t.start + t.keys;
  int last = s;
  while (last + 1 < slices && line_cut(total, slices, last + 1) < end) ++last;

  // A slice's part of the tile is its slot 1 if it starts the tile, else slot 0; it is empty
  // where both of its cuts move up to the same key.  Lanes look after 32 parts at a time; the
  // parts' accumulators are then read with nothing between the loads.
  float acc[E], m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int i0 = s - 1; i0 <= last; i0 += 32) {
    const int i = i0 + lane;
    float2 v = make_float2(-INFINITY, 0.f);
    int64_t at = 0;
    if (i <= last &&
        line_key(t, line_cut(total, slices, i + 1), key_step) > line_key(t, line_cut(total, slices, i), key_step)) {
      at = ((int64_t(i) * p.num_kv_heads + kvh) * 2 + (i == s - 1 ? 1 : 0)) * rows + r;
      v = p.part_ml[at];
    }
    float mn = v.x;
#pragma unroll
    for (int d = 16; d; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
    mn = fmaxf(mn, m);
    const float ref = mn == -INFINITY ? 0.f : mn, old = ex2(m - ref), f = ex2(v.x - ref);
    m = mn;
    float part = v.y * f;
#pragma unroll
    for (int d = 16; d; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
    sum = sum * old + part;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= old;
    const int n = min(32, last + 1 - i0);
    for (int k0 = 0; k0 < n; k0 += 8) {
      float o[8][E], fk[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        fk[k] = __shfl_sync(0xffffffffu, f, k0 + k);
        const int64_t ak = __shfl_sync(0xffffffffu, at, k0 + k);
        const bool some = __shfl_sync(0xffffffffu, v.x, k0 + k) != -INFINITY;  // NaN counts
#pragma unroll
        for (int e = 0; e < E; ++e) o[k][e] = 0.f;
        if (some) VecLoad<float, E>::run(p.part_o + ak * D + E * lane, o[k]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += o[k][e] * fk[k];
    }
  }
  T* dst = static_cast<T*>(p.out) + int64_t(first + t0 + tok) * p.o_st + int64_t(head) * p.o_sh + E * lane;
  const float inv = 1.f / sum;
#pragma unroll
  for (int e = 0; e < E; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(acc[e] * inv, acc[e + 1] * inv);
}

// ------------------------------------------------------------------ dispatch
template <typename T, int D, int RG>
static cudaError_t rows_one(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int* err,
                            cudaStream_t stream) {
  using C = RowsCfg<D, RG>;
  auto kern = kv8_rows_kernel<T, D, RG>;
  int dev = 0;
  cudaGetDevice(&dev);
  static bool configured[64] = {};
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  kern<<<p.slices * p.num_kv_heads, kRowsThreads, C::SMEM, stream>>>(tk, tv, p, err);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t rows_by_shape(int head_dim, int row_groups, const CUtensorMap& tk, const CUtensorMap& tv,
                                 const Kv8AttnParams& p, int* err, cudaStream_t s) {
  if (head_dim == 64)
    return row_groups == 1 ? rows_one<T, 64, 1>(tk, tv, p, err, s) : rows_one<T, 64, 2>(tk, tv, p, err, s);
  return row_groups == 1 ? rows_one<T, 128, 1>(tk, tv, p, err, s) : rows_one<T, 128, 2>(tk, tv, p, err, s);
}

int kv8_rows_slices(int row_groups, int num_kv_heads, int sms) {
  // Resident CTAs per SM: three with one group of rows, two with two (registers).
  const int n = sms * (row_groups == 1 ? 3 : 2) / num_kv_heads;
  return n < 1 ? 1 : n;
}

cudaError_t launch_kv8_rows(int dtype, int head_dim, int row_groups, const CUtensorMap& tk, const CUtensorMap& tv,
                            const Kv8AttnParams& p, int* err, cudaStream_t stream) {
  cudaError_t e = dtype == PA_DTYPE_F16 ? rows_by_shape<__half>(head_dim, row_groups, tk, tv, p, err, stream)
                                        : rows_by_shape<__nv_bfloat16>(head_dim, row_groups, tk, tv, p, err, stream);
  if (e != cudaSuccess) return e;
  return launch_kv8_combine(dtype, head_dim, 8 * row_groups, kRowsKeys, kRowsMinKeys, p, stream);
}

cudaError_t launch_kv8_combine(int dtype, int head_dim, int rows, int key_step, int min_keys, const Kv8AttnParams& p,
                               cudaStream_t stream) {
  if (p.slices < 2) return cudaSuccess;
  const dim3 grid(p.slices - 1, p.num_kv_heads, (p.tile_tokens * p.group + 3) / 4);
  if (dtype == PA_DTYPE_F16) {
    if (head_dim == 64)
      kv8_combine_kernel<__half, 64><<<grid, 128, 0, stream>>>(p, rows, key_step, min_keys);
    else
      kv8_combine_kernel<__half, 128><<<grid, 128, 0, stream>>>(p, rows, key_step, min_keys);
  } else {
    if (head_dim == 64)
      kv8_combine_kernel<__nv_bfloat16, 64><<<grid, 128, 0, stream>>>(p, rows, key_step, min_keys);
    else
      kv8_combine_kernel<__nv_bfloat16, 128><<<grid, 128, 0, stream>>>(p, rows, key_step, min_keys);
  }
  return cudaGetLastError();
}

}  // namespace pa
