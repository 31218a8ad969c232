// Attention of few new tokens per sequence over the 8-bit paged cache (decode, and chunks
// whose (token, head) rows fit one to three groups of 8), on mma.sync.
//
// For each row r = (new token t, query head of the KV head):
//   s_j = scale * q_r . K_j,  out_r = sum_j softmax_j(s) V_j,  j <= position of t
// with K_j = k_j 2^a_j and V_j = v_j 2^b_j, where k, v are e4m3 and a, b the rows' exponents.
// e4m3 widens to fp16 exactly, so S runs over the payloads and column j is scaled by 2^a_j;
// v_j takes its 2^b_j as it is widened, exactly (b_j in [-14, 7]).  The weight that multiplies
// V_j is exp2(s_j - m + 15) rounded to fp16: 11 bits down to 2^-29 of the maximum, and at most
// 2^-40 of it lost below.  The sum takes the same shift, so it cancels.  (With 2^b_j in the
// weight, rows of small values lost whole keys: a weight of 2^-19 of the maximum was 0 for
// b_j = -14.)  bf16 queries are brought into fp16 by a power of two per row, which is exact but
// for elements 2^-28 below the row's largest.  Maximum, sum and accumulators are float32.
//
// HBM-bound: each K/V byte is read once per tile of rows.  The sequences' keys laid end to
// end are cut into equal slices (kv8_line.cuh), a CTA per slice and KV head with the KV head
// fastest, so that the CTAs of one slice read a pool block's heads side by side.  A CTA has
// consumer warps, which take stages of 32 keys in turn, and a producer warp, which walks the
// slice's pieces, reads the block table and keeps each consumer's ring full: the rings run
// across pieces, so a new sequence costs no drain.  With one group of 8 rows there are three
// CTAs on an SM, and HBM bounds them; with more rows a thread needs 168 registers, three groups
// of 128 dims spill 120 bytes of them (pairs of heads 188), and there are two (five consumers a
// CTA, or one CTA of eleven, are no faster).  Per 16 keys: K and V tile by
// TMA (a 16-row box); the 16 + 16 scale bytes through a producer lane's registers, a round
// of 32 blocks ahead (as bulk copies of 16 bytes they cost the copy engine as much as the
// tiles: 177 against 152 us for 64 sequences of about 4,096 keys, 8 heads of 128).
//
// Both products are computed transposed, S^T = K Q^T and O^T = V^T W^T, because an MMA has
// 16 rows and 8 columns and there are few query rows: 16 keys (or dims) fill the rows, 8
// query rows the columns, so one group of 8 rows wastes nothing; the other way round half of
// each MMA is zeros.  W moves from the accumulator's layout to the operand's by one
// movmatrix per 8 x 8.  Widening costs one conversion per two elements; with 16-byte chunks
// of head_dim dealt out to the MMA's k index as ldmatrix delivers bytes (lane 4g + i holds
// dims 4i .. 4i + 3) K needs no permute, and V's transpose needs one byte permute per four.
//
// head_dim 64 with an even number of KV heads runs two KV heads as one of 128 dims (PAIR): a
// pool row of 64 bytes costs the copy engine as much as one of 128.  A query row then has
// zeros in the other head's dims, its scores take its own head's scales, and of O^T its own
// head's dims are kept; the columns that this costs were zeros before.
//
// Measured with the join (8 heads of 128 and 32 query heads; floors at 6,535 GB/s): 64 x ~4,096
// keys 112 us (floor 98), 131,071 keys 55 (41): a slice of 2,400 keys, of which the first loads
// and the join are 12 us; 517 keys 9.1, all of it launches, first loads and the join; 24 chunks
// of five over ~6,000 keys 98 (50), bound by the latency of the consumers' arithmetic (20 rows,
// two CTAs an SM); 48 x ~700 keys of 12 heads of 64, one query head each, 25 (9).
#include <cuda_fp16.h>

#include <type_traits>

#include "kv8.h"
#include "kv8_launch.cuh"
#include "kv8_line.cuh"
#include "kv8_widen.cuh"
#include "pa_common.cuh"
#include "tc_softmax.cuh"

namespace pa {

constexpr int kRowsStage = 32;                      // keys a stage: two 16-key blocks
constexpr int kRowsKeys = 16;                       // keys a block; cuts fall on these
constexpr int kRowsDescs = 2;
__host__ __device__ constexpr int rows_warps(int) { return 4; }                    // consumers
__host__ __device__ constexpr int rows_ctas(int row_groups) { return row_groups == 1 ? 3 : 2; }  // on an SM
// Fewest keys a slice gets, a stage for each consumer: below this a CTA's set-up and its
// partial cost more than the keys it takes over.
__host__ __device__ constexpr int rows_min_keys(int row_groups) { return kRowsStage * rows_warps(row_groups); }
constexpr float kWeightLog2 = 15.f;                 // weights stand times 2^15, see above

// D: dims of the payload rows (two heads' with PAIR), RG: groups of 8 query rows.
template <int D, int RG, bool PAIR>
struct RowsCfg {
  static_assert(!PAIR || D == 128, "pairs of heads of 64");
  static constexpr int DO = PAIR ? 64 : D;          // dims of a query and an output row
  static constexpr int SUBS = PAIR ? 2 : 1;         // KV heads of a payload row
  static constexpr int W = rows_warps(RG), CTAS = rows_ctas(RG), THREADS = 32 * (W + 1);
  static constexpr int SCALES = 2 * SUBS * kRowsStage;  // bytes a stage: K then V
  // 16 KB in flight per consumer, or with fewer consumers 24.
  static constexpr int STAGES = (D == 128 ? 1 : 2) * (RG == 1 ? 2 : 3);
  static constexpr int TILE = kRowsKeys * D;        // K or V of a block
  static constexpr int BLOCK = 2 * TILE;
  static constexpr int STAGE = 2 * BLOCK;
  static constexpr int CH = D / 16;                 // 16-byte chunks of a row = k steps of S
  static constexpr int NO = CH * RG * 4;            // accumulator registers
  static constexpr int MERGES = RG == 1 ? 2 : 1;    // accumulators on their way between warps
  static constexpr int OFF_SCALE = W * STAGES * STAGE;
  static constexpr int OFF_Q = OFF_SCALE + W * STAGES * SCALES;
  static constexpr int OFF_MERGE = OFF_Q;           // the queries are no longer read by then
  static constexpr int OFF_ML = OFF_MERGE + MERGES * NO * 32 * 4;
  static_assert(MERGES * NO * 32 * 4 >= CH * RG * 32 * 8, "merge area holds the queries");
  static constexpr int OFF_FACTOR = OFF_ML + W * RG * 8 * 8;
  static constexpr int OFF_LIMIT = OFF_FACTOR + RG * 8 * 4;
  static constexpr int OFF_DESC = OFF_LIMIT + RG * 8 * 4;
  static constexpr int OFF_BAR = OFF_DESC + kRowsDescs * 32;
  static constexpr int SMEM = OFF_BAR + (2 * W * STAGES + 2 * kRowsDescs) * 8;
  static constexpr bool Q_IN_REGS = RG <= 2;
  // 228 KB of shared memory on an SM, 1 KB of it taken per CTA.
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory for the CTAs an SM is to hold");
};

struct RowsPiece {      // part of a tile that a CTA works on
  int32_t row0;         // packed index of the tile's first token; -1: no more pieces
  int32_t tokens;       // of the tile
  int32_t pos0;         // position of the first token
  int32_t ctx;          // of the sequence
  int32_t kb0, kb1;     // blocks of 16 keys
  int32_t part;         // -1: the whole tile, else the CTA's partial slot
  int32_t pair0;        // stages the CTA had before it
};

__device__ __forceinline__ void rows_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
template <int W>
__device__ __forceinline__ void rows_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * W) : "memory");
}

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
// D += A B, m16n8k16, fp16 operands.
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The 8 x 8 tile of 16-bit elements, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

template <typename T, int D, int RG, bool PAIR>
__global__ void __launch_bounds__(RowsCfg<D, RG, PAIR>::THREADS, RowsCfg<D, RG, PAIR>::CTAS)
    kv8_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const Kv8AttnParams p, int* err) {
  using C = RowsCfg<D, RG, PAIR>;
  constexpr int CH = C::CH, DO = C::DO, W = C::W;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint2* sq = reinterpret_cast<uint2*>(smem + C::OFF_Q);
  float* merge = reinterpret_cast<float*>(smem + C::OFF_MERGE);
  float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  float* factors = reinterpret_cast<float*>(smem + C::OFF_FACTOR);
  int* limits = reinterpret_cast<int*>(smem + C::OFF_LIMIT);
  RowsPiece* desc = reinterpret_cast<RowsPiece*>(smem + C::OFF_DESC);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + W * C::STAGES;
  uint64_t* d_full = empty + W * C::STAGES;
  uint64_t* d_empty = d_full + kRowsDescs;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x % p.num_kv_heads;
  if (threadIdx.x == 0) {
    for (int i = 0; i < W * C::STAGES; ++i) {
      mbar_init(&full[i], 4);  // per block: its tiles are on their way, its scales are there
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kRowsDescs; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], W);
    }
    fence_mbar_init();
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  __syncthreads();
  pdl_wait();
  pdl_release();
  LineFinder finder(p, err);
  const int64_t total = finder.total;
  const LineCuts cuts(total, p.slices, rows_min_keys(RG));
  const bool tells = warp == W && lane == 0 && kvh == 0;  // of the tile that its slice shares with the next ones
  if (tells) p.joins[slice].tokens = 0;
  if (total == 0 || slice >= cuts.n) return;

  if (warp == W) {
    // ------------------------------------------------------------ producer
    const int64_t x1 = cuts.at(slice + 1);
    int64_t x = cuts.at(slice);
    int pairs = 0;  // stages issued so far; the i-th is consumer (i % W)'s
    int pieces = 0;
    bool ok = true;
    struct BlockRef {
      int slot;  // first slot of the 16 keys
      uint4 ks[C::SUBS], vs[C::SUBS];
    };
    // A block's id, and with it its place and scales: in two steps, so that neither a round's
    // ids nor its scales are waited for before the round before it is on its way.
    auto read_id = [&](const int32_t* row, int kb, int end) { return kb < end ? __ldg(row + (kb >> p.block_shift)) : 0; };
    auto look_up = [&](int id, int kb, int end) {
      BlockRef r;
      r.slot = 0;
      if (kb < end) {
        if (id < 0 || id >= p.pool_blocks) {
          set_error(err, PA_KV8_ERR_BLOCK);
          id = 0;
        }
        const int sub = (kb & ((1 << p.block_shift) - 1)) * 16;
        r.slot = (id << (p.block_shift + 4)) + sub;
#pragma unroll
        for (int u = 0; u < C::SUBS; ++u) {
          const int64_t at = (((int64_t(id) * p.num_kv_heads + kvh) * C::SUBS + u) << (p.block_shift + 4)) + sub;
          r.ks[u] = __ldg(reinterpret_cast<const uint4*>(p.k_scale + at));
          r.vs[u] = __ldg(reinterpret_cast<const uint4*>(p.v_scale + at));
        }
      }
      return r;
    };
    while (ok) {
      LinePiece at;
      const bool more = line_next_piece(finder, x, x1, kRowsKeys, at);
      const int slot = pieces % kRowsDescs;
      if (pieces >= kRowsDescs) ok = mbar_wait(&d_empty[slot], ((pieces / kRowsDescs) - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const LineTile& t = at.t;
      const int kb0 = at.k0 / kRowsKeys, kb1 = (at.k1 + kRowsKeys - 1) / kRowsKeys;
      if (lane == 0) {
        RowsPiece d;
        d.row0 = -1;
        d.pair0 = pairs;
        if (more) {
          const int t0 = t.index * p.tile_tokens;
          d.row0 = t.first + t0;
          d.tokens = min(p.tile_tokens, t.q - t0);
          d.pos0 = t.ctx - t.q + t0;
          d.ctx = t.ctx;
          d.kb0 = kb0;
          d.kb1 = kb1;
          d.part = at.k0 > 0 ? 0 : (at.k1 < t.keys ? 1 : -1);
        }
        desc[slot] = d;
        rows_arrive(&d_full[slot]);
      }
      ++pieces;
      if (!more) break;
      if (tells && at.k0 == 0 && at.k1 < t.keys) p.joins[slice] = line_join(t, cuts, slice, p.tile_tokens);
      const int32_t* row = p.tables + int64_t(t.seq) * p.table_stride;
      // Each lane looks after one of the next 32 blocks: its id is read two rounds ahead of the
      // round whose tiles are being issued, its scales one round; lanes then issue their own
      // blocks, two (a stage) at a time.
      const int id = read_id(row, kb0 + lane, kb1);
      int id_next = read_id(row, kb0 + 32 + lane, kb1);
      BlockRef cur = look_up(id, kb0 + lane, kb1), nxt = cur;
      for (int kb = kb0; kb < kb1 && ok; kb += 32) {
        const int n = min(32, kb1 - kb);
        // As many stages at a time as have places of their own in the rings, each lane issuing
        // its block as soon as its place is free: one stage after the other took about 770
        // clocks each and held the whole kernel up.
        constexpr int ROUND = W * C::STAGES < 16 ? W * C::STAGES : 16;
        for (int b0 = 0; b0 < n && ok; b0 += 2 * ROUND) {
          const int i = pairs + (lane - b0) / 2, turn = i / W, st = (i % W) * C::STAGES + turn % C::STAGES;
          bool waiting = lane >= b0 && lane < b0 + 2 * ROUND && lane < ((n + 1) & ~1);
          for (uint32_t tries = 0; tries < kWaitLimit; ++tries) {
            if (waiting && (turn < C::STAGES || mbar_test(&empty[st], ((turn / C::STAGES) - 1) & 1))) {
              waiting = false;
              uint64_t* bar = &full[st];
              const int half = lane & 1;
              if (lane < n) {
                uint8_t* stage = smem + st * C::STAGE + half * C::BLOCK;
                mbar_arrive_expect_tx(bar, C::BLOCK);
                tma_load_3d(stage, &tk, 0, kvh, cur.slot, bar);
                tma_load_3d(stage + C::TILE, &tv, 0, kvh, cur.slot, bar);
                uint8_t* sc = smem + C::OFF_SCALE + st * C::SCALES + 16 * half;
#pragma unroll
                for (int u = 0; u < C::SUBS; ++u) {
                  *reinterpret_cast<uint4*>(sc + u * kRowsStage) = cur.ks[u];
                  *reinterpret_cast<uint4*>(sc + (C::SUBS + u) * kRowsStage) = cur.vs[u];
                }
                rows_arrive(bar);
              } else {
                rows_arrive(bar);  // the piece's last stage holds one block
                rows_arrive(bar);
              }
            }
            if (!__any_sync(0xffffffffu, waiting)) break;
          }
          ok = !__any_sync(0xffffffffu, waiting);
          pairs += min(ROUND, (n - b0 + 1) / 2);
          if (b0 == 0 && kb + 32 < kb1) {
            nxt = look_up(id_next, kb + 32 + lane, kb1);
            id_next = read_id(row, kb + 64 + lane, kb1);
          }
        }
        cur = nxt;
      }
    }
    if (!ok) {
      if (lane == 0) set_error(err, PA_KV8_ERR_TIMEOUT);
      // Leave with no copy into this CTA's shared memory in flight.
      for (int i = max(0, pairs - W * C::STAGES); i < pairs; ++i)
        mbar_wait(&full[(i % W) * C::STAGES + i / W % C::STAGES], (i / W / C::STAGES) & 1);
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, tig = lane & 3;
  const int mi = lane >> 3, ri = lane & 7;
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
                   : "r"(mine), "n"(32 * W)
                   : "memory");
    }
    if (!all) break;
    const RowsPiece d = desc[slot];
    __syncwarp();
    if (lane == 0) rows_arrive(&d_empty[slot]);
    if (d.row0 < 0) break;

    // Queries as B fragments in shared memory: row r = (token r / group, head r % group),
    // brought into fp16 by a power of two; a warp takes a row at a time, all of its rows' loads
    // (spare rows repeat the last token) before the first is used: one after the other cost
    // 1,000 clocks a row, with three groups 3 us a piece (100 chunks of five over ~300 keys 70 : 65 us).
    constexpr int E = DO / 32, PER = 8 * RG / W;
    static_assert(PER * W == 8 * RG, "rows a warp");
    float xs[PER][E];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = warp + W * i, tok = r / p.group, head = r - tok * p.group;
      VecLoad<T, E>::run(static_cast<const T*>(p.q) + int64_t(d.row0 + min(tok, d.tokens - 1)) * p.q_st +
                             int64_t(kvh * p.group + head) * p.q_sh + E * lane,
                         xs[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = warp + W * i, tok = r / p.group, head = r - tok * p.group;
      const float(&x)[E] = xs[i];
      float big = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) big = fmaxf(big, fabsf(x[e]));
      if (DType<T>::code == PA_DTYPE_BF16) {
#pragma unroll
        for (int s = 16; s; s >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
      }
      const float up = query_power<T>(big);
      // Fragment words of row r: chunk c, (r & 7, dims 4 t .. 4 t + 3) at lane 4 (r & 7) + t.
      auto word = [&](int c, int t, int half) -> uint32_t& {
        return reinterpret_cast<uint32_t*>(&sq[(c * RG + (r >> 3)) * 32 + (r & 7) * 4 + t])[half];
      };
      if constexpr (E == 4) {
        word(lane / 4, lane % 4, 0) = pack2<__half>(x[0] * up, x[1] * up);
        word(lane / 4, lane % 4, 1) = pack2<__half>(x[2] * up, x[3] * up);
      } else {
        const int own = PAIR && 2 * head >= p.group ? 4 : 0;  // first chunk of the row's head
        word(own + lane / 8, lane % 8 / 2, lane & 1) = pack2<__half>(x[0] * up, x[1] * up);
        if (PAIR) word((own ^ 4) + lane / 8, lane % 8 / 2, lane & 1) = 0u;
      }
      if (lane == 0) {
        factors[r] = p.qscale / up;  // exact: a power of two
        limits[r] = tok < d.tokens ? min(d.pos0 + tok, d.kb1 * kRowsKeys - 1) : -1;
      }
    }
    rows_sync<W>();
    uint2 qr[C::Q_IN_REGS ? CH : 1][RG];
    if constexpr (C::Q_IN_REGS) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg)
#pragma unroll
        for (int c = 0; c < CH; ++c) qr[c][rg] = sq[(c * RG + rg) * 32 + lane];
    }
    // Rows 8 rg + 2 tig + {0, 1} of this lane.
    const float2* my_factors = reinterpret_cast<const float2*>(factors) + tig;
    const int2* my_limits = reinterpret_cast<const int2*>(limits) + tig;
    bool second[RG][2];  // with PAIR: of the pair's second head
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * rg + 2 * tig + e;
        second[rg][e] = PAIR && 2 * (r % p.group) >= p.group;
      }

    float o[CH][RG][4];  // dims 16 c + 2 g (+1: elements 2, 3), rows 8 rg + 2 tig + {0, 1}
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int rg = 0; rg < RG; ++rg)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][rg][e] = 0.f;
    float m[RG][2], l[RG][2];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[rg][e] = -INFINITY;
        l[rg][e] = 0.f;
      }

    const int skip = (warp + W - d.pair0 % W) % W;  // stages of the piece before this warp's first
    int turn = (d.pair0 + skip) / W;
    // The piece's stages with the first LG groups of rows: a tile of fewer tokens than the
    // widest leaves groups empty.
    auto stages = [&](auto groups) {
      constexpr int LG = decltype(groups)::value;
      for (int kb = d.kb0 + 2 * skip; kb < d.kb1; kb += 2 * W, ++turn) {
        const int st = warp * C::STAGES + turn % C::STAGES;
        if (ok) ok = mbar_wait(&full[st], (turn / C::STAGES) & 1);
        const uint32_t stage = smem_u32(smem + st * C::STAGE);
        const uint8_t* sc = smem + C::OFF_SCALE + st * C::SCALES;
        const int key0 = kb * kRowsKeys;
        // Spare rows of the tile compute, unmasked, and are not stored.
        const bool masked = key0 + kRowsStage - 1 > d.pos0 || kb + 2 > d.kb1;
        const int end = min(d.ctx, d.kb1 * kRowsKeys) - key0;  // keys of the stage that are there
        // ---- S^T over the payloads: element 2 h + e is key 16 b + 8 h + g, row 8 rg + 2 tig + e
        float s[2][LG][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int rg = 0; rg < LG; ++rg)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][rg][e] = 0.f;
#pragma unroll
          for (int c = 0; c < CH; c += 2) {
            uint32_t w[4];  // (keys 0-7, chunk c), (keys 8-15, c), (0-7, c + 1), (8-15, c + 1)
            ldm4(stage + n * C::BLOCK + tile_at<D>(8 * (mi & 1) + ri, c + (mi >> 1)), w);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a0 = widen_lo(w[2 * i]), a1 = widen_lo(w[2 * i + 1]), a2 = widen_hi(w[2 * i]),
                             a3 = widen_hi(w[2 * i + 1]);
#pragma unroll
              for (int rg = 0; rg < LG; ++rg) {
                uint2 q;
                if constexpr (C::Q_IN_REGS)
                  q = qr[c + i][rg];
                else
                  q = sq[((c + i) * RG + rg) * 32 + lane];
                mma16(s[n][rg], a0, a1, a2, a3, q.x, q.y);
              }
            }
          }
        }

        // ---- online softmax
        // K scales of keys 16 n + 8 h + g, or NaN where the key's K or V row stands for it: a score
        // of NaN makes the whole output row NaN, and only of tokens that see the key.  (A branch of
        // its own for V's cost 20 us of 24 chunks of five over 6,000 keys.)
        float ks[2][2][C::SUBS];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < C::SUBS; ++u) {
              const int at = u * kRowsStage + 16 * n + 8 * h + g;
              const uint32_t kb = sc[at], vb = sc[C::SUBS * kRowsStage + at];
              ks[n][h][u] = __uint_as_float(max(kb, vb) == 255u ? 0x7fffffffu : kb << 23);
            }
        uint32_t wt[2][LG][2];  // weights as B fragments: keys 8 h + 2 tig (+1), row 8 rg + g
        bool grown = false;
        float alpha[LG][2];
#pragma unroll
        for (int rg = 0; rg < LG; ++rg) {
          const float2 factor = my_factors[4 * rg];
          int2 limit = make_int2(0, 0);
          if (masked) limit = my_limits[4 * rg];
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = 16 * n + 8 * h + g;
                float& v = s[n][rg][2 * h + e];
                const float k = PAIR && second[rg][e] ? ks[n][h][C::SUBS - 1] : ks[n][h][0];
                v *= k * (e ? factor.y : factor.x);
                if (masked && key0 + key > (e ? limit.y : limit.x)) v = -INFINITY;
                mx[e] = fmaxf(mx[e], v);
              }
          float ref[2], sum[2] = {0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
            const float mn = fmaxf(m[rg][e], mx[e]);
            ref[e] = mn == -INFINITY ? 0.f : mn;  // nothing seen yet
            alpha[rg][e] = ex2(m[rg][e] - ref[e]);
            grown |= alpha[rg][e] != 1.f;
            m[rg][e] = mn;
            ref[e] -= kWeightLog2;
          }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float w[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                w[e] = ex2(s[n][rg][2 * h + e] - ref[e]);
                sum[e] += w[e];
              }
              wt[n][rg][h] = transpose8(pack2<__half>(w[0], w[1]));
            }
#pragma unroll
          for (int e = 0; e < 2; ++e) l[rg][e] = l[rg][e] * alpha[rg][e] + sum[e];
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int rg = 0; rg < LG; ++rg)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[c][rg][e] *= alpha[rg][e & 1];
        }

        // ---- O^T += V^T W^T; bytes behind the context (or the stage's only block) read as zero
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          uint32_t vs[C::SUBS][2];  // V scales of keys 16 n + 8 h + 2 tig (+1)
#pragma unroll
          for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              vs[u][h] = scale_pair(*reinterpret_cast<const uint16_t*>(sc + (C::SUBS + u) * kRowsStage + 16 * n + 8 * h +
                                                                       2 * tig));
          uint32_t pick[2] = {0x3120u, 0x3120u};  // (t0 d0, t1 d0, t0 d1, t1 d1) of (t0 d0, t0 d1, t1 d0, t1 d1)
          if (end < kRowsStage) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int t0 = 16 * n + 8 * h + 2 * tig;
              pick[h] = t0 + 1 < end ? 0x3120u : (t0 < end ? 0x4140u : 0x4444u);
            }
          }
#pragma unroll
          for (int c = 0; c < CH; c += 2) {
            uint32_t w[4];  // (keys 0-7, chunk c), (keys 8-15, c), (0-7, c + 1), (8-15, c + 1)
            ldm4t(stage + n * C::BLOCK + C::TILE + tile_at<D>(8 * (mi & 1) + ri, c + (mi >> 1)), w);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x = __byte_perm(w[2 * i], 0, pick[0]), y = __byte_perm(w[2 * i + 1], 0, pick[1]);
              const uint32_t(&v2)[2] = vs[PAIR && c + i >= CH / 2 ? 1 : 0];
              const uint32_t a0 = mul_h2(widen_lo(x), v2[0]), a1 = mul_h2(widen_hi(x), v2[0]),
                             a2 = mul_h2(widen_lo(y), v2[1]), a3 = mul_h2(widen_hi(y), v2[1]);
#pragma unroll
              for (int rg = 0; rg < LG; ++rg) mma16(o[c + i][rg], a0, a1, a2, a3, wt[n][rg][0], wt[n][rg][1]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) rows_arrive(&empty[st]);
      }
    };
    const int live = (d.tokens * p.group + 7) / 8;
    if (RG == 1 || live <= 1)
      stages(std::integral_constant<int, 1>{});
    else if (RG == 2 || live == 2)
      stages(std::integral_constant<int, RG < 2 ? RG : 2>{});
    else
      stages(std::integral_constant<int, RG>{});

    // ---- join the warps: common maximum, then a tree over the accumulators
    float big[RG][2];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[rg][e] += __shfl_xor_sync(0xffffffffu, l[rg][e], x);
        if (g == 0) ml[warp * 8 * RG + 8 * rg + 2 * tig + e] = make_float2(m[rg][e], l[rg][e]);
      }
    rows_sync<W>();
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2* v = ml + 8 * rg + 2 * tig + e;
        big[rg][e] = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) big[rg][e] = fmaxf(big[rg][e], v[w * 8 * RG].x);
        const float ref = big[rg][e] == -INFINITY ? 0.f : big[rg][e];
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += v[w * 8 * RG].y * ex2(v[w * 8 * RG].x - ref);
        const float f = ex2(m[rg][e] - ref);
        l[rg][e] = sum;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          o[c][rg][e] *= f;
          o[c][rg][2 + e] *= f;
        }
      }
    // Halves of the dims go to the neighbour, then quarters to the other pair, so that all four
    // warps add and store: with a tree that ends in one warp, 100 chunks of five tokens over
    // about 300 keys took 78 us instead of 70.
    static_assert(W == 4, "two exchanges");
    constexpr int H = CH / 2, Q4 = CH / 4, N4 = 4 * RG;
    constexpr int STEP = W * H * N4 <= C::MERGES * C::NO ? H : Q4;  // chunks an exchange has room for
    const bool odd = warp & 1, upper = warp & 2;
    float two[H][N4], all4[Q4][N4];  // sums of two warps, of all
#pragma unroll
    for (int c0 = 0; c0 < H; c0 += STEP) {
#pragma unroll
      for (int c = 0; c < STEP; ++c)
#pragma unroll
        for (int e = 0; e < N4; ++e)
          merge[((warp * STEP + c) * N4 + e) * 32 + lane] = odd ? o[c0 + c][e / 4][e % 4] : o[H + c0 + c][e / 4][e % 4];
      rows_sync<W>();
#pragma unroll
      for (int c = 0; c < STEP; ++c)
#pragma unroll
        for (int e = 0; e < N4; ++e)
          two[c0 + c][e] = (odd ? o[H + c0 + c][e / 4][e % 4] : o[c0 + c][e / 4][e % 4]) +
                           merge[(((warp ^ 1) * STEP + c) * N4 + e) * 32 + lane];
      rows_sync<W>();
    }
#pragma unroll
    for (int c = 0; c < Q4; ++c)
#pragma unroll
      for (int e = 0; e < N4; ++e) merge[((warp * Q4 + c) * N4 + e) * 32 + lane] = upper ? two[c][e] : two[Q4 + c][e];
    rows_sync<W>();
#pragma unroll
    for (int c = 0; c < Q4; ++c)
#pragma unroll
      for (int e = 0; e < N4; ++e)
        all4[c][e] = (upper ? two[Q4 + c][e] : two[c][e]) + merge[(((warp ^ 2) * Q4 + c) * N4 + e) * 32 + lane];
    const int chunk0 = (odd ? H : 0) + (upper ? Q4 : 0);
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * rg + 2 * tig + e, tok = r / p.group, head = kvh * p.group + (r - tok * p.group);
        if (tok >= d.tokens) continue;
        const float f = d.part < 0 ? 1.f / l[rg][e] : 1.f;
        const int64_t at = ((int64_t(slice) * p.num_kv_heads + kvh) * 2 + d.part) * (8 * RG) + r;
        T* dst = static_cast<T*>(p.out) + int64_t(d.row0 + tok) * p.o_st + int64_t(head) * p.o_sh + 2 * g;
        // With PAIR a row's dims are its own head's, the first 64 or the second.
        if (!PAIR || second[rg][e] == odd) {
#pragma unroll
          for (int c = 0; c < Q4; ++c) {
            const int chunk = PAIR ? (chunk0 + c) % H : chunk0 + c;
            const float x = all4[c][4 * rg + e] * f, y = all4[c][4 * rg + 2 + e] * f;
            if (d.part < 0)
              *reinterpret_cast<uint32_t*>(dst + 16 * chunk) = pack2<T>(x, y);
            else
              *reinterpret_cast<float2*>(p.part_o + at * DO + 16 * chunk + 2 * g) = make_float2(x, y);
          }
        }
        if (warp == 0 && d.part >= 0 && g == 0) p.part_ml[at] = make_float2(big[rg][e], l[rg][e]);
      }
  }
  if (!ok && lane == 0) set_error(err, PA_KV8_ERR_TIMEOUT);
}

// Joins the partials of tiles that a cut fell into.  CTA (s, kvh, z): the shared tile that
// starts in slice s, if there is one (the attention kernel left word), and some of its rows; a
// lane takes D / 32 elements of a row.  What bounds it is latency (the tile, then (m, l), then
// accumulators) and that most CTAs have nothing to do, so they learn that from one load; when
// each looked its place up on the work line, one token over 517 keys took 11.5 us instead of
// 9.4 and 64 x 4,096 keys 119 instead of 114.  In small tiles, which a long context leaves in
// many parts, the CTA's warps share out the parts of kCombineRows rows (BY_PARTS); in 256-row
// tiles every warp has rows of its own, as many at a time.  Four rows took 3 us more for 100
// tokens over 4,000 keys and for 24 chunks of five over 6,000, one row 3 us more for 48 x 700.
constexpr int kCombineWarps = 8, kCombineRows = 2;

template <typename T, int D, bool BY_PARTS>
__global__ void __launch_bounds__(32 * kCombineWarps)
    kv8_combine_kernel(const Kv8AttnParams p, int rows, int key_step) {
  constexpr int E = D / 32, P = 2, NR = kCombineRows;
  __shared__ float s_acc[BY_PARTS ? kCombineWarps : 1][NR][D];
  __shared__ float2 s_ml[BY_PARTS ? kCombineWarps : 1][NR];
  pdl_wait();
  pdl_release();
  const Kv8Join join = p.joins[blockIdx.x];
  const int live = join.tokens * p.group;  // rows of the tile
  if (live == 0) return;
  const LineCuts cuts(join);
  LineTile t{};
  t.start = join.start;
  t.keys = join.keys;
  const int s = blockIdx.x + 1, kvh = blockIdx.y, last = join.last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int ROWS = BY_PARTS ? NR : kCombineWarps * NR;  // of the CTA at a time
  const int first_part = BY_PARTS ? warp : 0, part_step = BY_PARTS ? kCombineWarps : 1;
  for (int z0 = blockIdx.z * ROWS; z0 < live; z0 += ROWS * gridDim.z) {
    const int r0 = z0 + (BY_PARTS ? 0 : warp * NR);
    // A slice's part of the tile is its slot 1 if it starts the tile, else slot 0; it is empty
    // where both of its cuts move up to the same key.  Lanes look after 32 parts at a time.
    float acc[NR][E], m[NR], sum[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      m[n] = -INFINITY;
      sum[n] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[n][e] = 0.f;
    }
    for (int i0 = s - 1 + first_part; i0 <= last; i0 += 32 * part_step) {
      const int i = i0 + lane * part_step;
      const bool mine = i <= last && line_key(t, cuts.at(i + 1), key_step) > line_key(t, cuts.at(i), key_step);
      const int64_t at = mine ? ((int64_t(i) * p.num_kv_heads + kvh) * 2 + (i == s - 1 ? 1 : 0)) * rows + r0 : -1;
      float2 v[NR];
#pragma unroll
      for (int n = 0; n < NR; ++n)
        v[n] = mine && r0 + n < live ? p.part_ml[at + n] : make_float2(-INFINITY, 0.f);
      float f[NR];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        float mn = v[n].x;
#pragma unroll
        for (int d = 16; d; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
        mn = fmaxf(mn, m[n]);
        const float ref = mn == -INFINITY ? 0.f : mn, old = ex2(m[n] - ref);
        f[n] = ex2(v[n].x - ref);
        m[n] = mn;
        float part = v[n].y * f[n];
#pragma unroll
        for (int d = 16; d; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
        sum[n] = sum[n] * old + part;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[n][e] *= old;
      }
      const int parts = min(32, (last - i0) / part_step + 1);
      for (int k0 = 0; k0 < parts; k0 += P) {
        float o[P][NR][E], fk[P][NR];
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const int64_t ak = __shfl_sync(0xffffffffu, at, (k0 + k) & 31);
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            fk[k][n] = __shfl_sync(0xffffffffu, f[n], (k0 + k) & 31);
#pragma unroll
            for (int e = 0; e < E; ++e) o[k][n][e] = 0.f;
            if (k0 + k < parts && ak >= 0 && r0 + n < live)
              VecLoad<float, E>::run(p.part_o + (ak + n) * D + E * lane, o[k][n]);
          }
        }
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
          for (int n = 0; n < NR; ++n)
            if (k0 + k < parts)
#pragma unroll
              for (int e = 0; e < E; ++e) acc[n][e] += o[k][n][e] * fk[k][n];
      }
    }
    if constexpr (BY_PARTS) {  // join the warps; warp n finishes row n
#pragma unroll
      for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int e = 0; e < E; ++e) s_acc[warp][n][E * lane + e] = acc[n][e];
        if (lane == 0) s_ml[warp][n] = make_float2(m[n], sum[n]);
      }
      __syncthreads();
      if (warp < NR) {
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kCombineWarps; ++w) mm = fmaxf(mm, s_ml[w][warp].x);
        const float ref = mm == -INFINITY ? 0.f : mm;
        sum[0] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[0][e] = 0.f;
#pragma unroll
        for (int w = 0; w < kCombineWarps; ++w) {
          const float2 v = s_ml[w][warp];
          const float f = ex2(v.x - ref);
          sum[0] += v.y * f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[0][e] += s_acc[w][warp][E * lane + e] * f;
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < (BY_PARTS ? 1 : NR); ++n) {
      const int r = BY_PARTS ? r0 + warp : r0 + n, tok = r / p.group, head = kvh * p.group + (r - tok * p.group);
      if (r >= live || (BY_PARTS && warp >= NR)) break;
      T* dst = static_cast<T*>(p.out) + int64_t(join.row0 + tok) * p.o_st + int64_t(head) * p.o_sh + E * lane;
      const float inv = 1.f / sum[n];
#pragma unroll
      for (int e = 0; e < E; e += 2)
        *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(acc[n][e] * inv, acc[n][e + 1] * inv);
    }
  }
}

// ------------------------------------------------------------------ dispatch
template <typename T, int D, int RG, bool PAIR>
static cudaError_t rows_one(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int* err,
                            cudaStream_t stream) {
  using C = RowsCfg<D, RG, PAIR>;
  auto kern = kv8_rows_kernel<T, D, RG, PAIR>;
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
  return launch_pdl(kern, dim3(p.slices * p.num_kv_heads), dim3(C::THREADS), C::SMEM, stream, tk, tv, p, err);
}

template <typename T, int D, bool PAIR>
static cudaError_t rows_by_groups(int row_groups, const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p,
                                  int* err, cudaStream_t s) {
  switch (row_groups) {
    case 1: return rows_one<T, D, 1, PAIR>(tk, tv, p, err, s);
    case 2: return rows_one<T, D, 2, PAIR>(tk, tv, p, err, s);
    case 3: return rows_one<T, D, 3, PAIR>(tk, tv, p, err, s);
    default: return cudaErrorInvalidValue;
  }
}

template <typename T>
static cudaError_t rows_by_shape(int head_dim, bool pair, int row_groups, const CUtensorMap& tk, const CUtensorMap& tv,
                                 const Kv8AttnParams& p, int* err, cudaStream_t s) {
  if (pair) return rows_by_groups<T, 128, true>(row_groups, tk, tv, p, err, s);
  return head_dim == 64 ? rows_by_groups<T, 64, false>(row_groups, tk, tv, p, err, s)
                        : rows_by_groups<T, 128, false>(row_groups, tk, tv, p, err, s);
}

int kv8_rows_slices(int row_groups, int num_kv_heads, int sms) {
  const int n = sms * rows_ctas(row_groups) / num_kv_heads;
  return n < 1 ? 1 : n;
}

cudaError_t launch_kv8_rows(int dtype, int head_dim, bool pair, int row_groups, const CUtensorMap& tk,
                            const CUtensorMap& tv, const Kv8AttnParams& p, int* err, cudaStream_t stream) {
  return dtype == PA_DTYPE_F16 ? rows_by_shape<__half>(head_dim, pair, row_groups, tk, tv, p, err, stream)
                               : rows_by_shape<__nv_bfloat16>(head_dim, pair, row_groups, tk, tv, p, err, stream);
}

template <typename T, int D>
static cudaError_t combine_one(int rows, int key_step, const Kv8AttnParams& p, cudaStream_t stream) {
  const int live = p.tile_tokens * p.group;
  const dim3 block(32 * kCombineWarps);
  constexpr int kPerCta = kCombineWarps * kCombineRows;
  if (rows <= 8 * kKv8RowGroups)
    return launch_pdl(kv8_combine_kernel<T, D, true>,
                      dim3(p.slices - 1, p.num_kv_heads, (live + kCombineRows - 1) / kCombineRows), block, 0, stream, p,
                      rows, key_step);
  return launch_pdl(kv8_combine_kernel<T, D, false>,
                    dim3(p.slices - 1, p.num_kv_heads, (live + kPerCta - 1) / kPerCta), block, 0, stream, p, rows, key_step);
}

cudaError_t launch_kv8_combine(int dtype, int head_dim, int rows, int key_step, const Kv8AttnParams& p,
                               cudaStream_t stream) {
  if (p.slices < 2) return cudaSuccess;
  if (dtype == PA_DTYPE_F16)
    return head_dim == 64 ? combine_one<__half, 64>(rows, key_step, p, stream)
                          : combine_one<__half, 128>(rows, key_step, p, stream);
  return head_dim == 64 ? combine_one<__nv_bfloat16, 64>(rows, key_step, p, stream)
                        : combine_one<__nv_bfloat16, 128>(rows, key_step, p, stream);
}

cudaError_t launch_kv8_rows_combine(int dtype, int head_dim, int row_groups, const Kv8AttnParams& p,
                                    cudaStream_t stream) {
  return launch_kv8_combine(dtype, head_dim, 8 * row_groups, kRowsKeys, p, stream);
}

}  // namespace pa
