// Attention of longer chunks over the 8-bit paged cache on tcgen05: tiles of 256 (token, head)
// rows, two halves of 128 that share every K and V tile, scores and output accumulated in
// tensor memory.
//
// The arithmetic is kv8_rows.cu's: K_j = k_j 2^a_j and V_j = v_j 2^b_j are exactly fp16 numbers
// (the cache's exponents lie in [-14, 7]), so K and V tiles are widened to fp16 in shared
// memory with their scales multiplied in, nothing is rounded, and both products run as
// fp16 MMAs with float32 accumulators; queries come into fp16 by a power of two per row,
// softmax weights are rounded to fp16.  An fp8 MMA would need Q and P split into several
// 8-bit terms to keep their bits; widening costs 1.5 instructions per two elements and is
// done once per 256 rows.
//
// Work: the tiles' keys laid end to end are cut into equal slices (kv8_line.cuh, steps of 64
// keys), one CTA per SM in all, so a chunk of few tiles over a long context is split along
// the context and every CTA does the same number of keys; a tile that a cut falls into
// leaves float32 partials that kv8_combine joins.
//
// Roles (768 threads, registers dealt out by setmaxnreg):
//   warps 0-3, 4-7  softmax of rows 0-127 / 128-255, one thread per row (TMEM lane): brings the
//                   warp's query rows into shared memory, reads scores, keeps maximum and sum,
//                   writes P to TMEM, the epilogue.  Rows are read and written in global memory
//                   by D / 8 lanes each, through the query tile: with a thread per row a piece
//                   cost 4 us more (333 tokens 43 us against 34, 1,000 over 16,384 298 : 294)
//   warps 8-11      K: staged e4m3 -> fp16 in the swizzled layout (3 stages), 16 keys a warp;
//                   12-15: V (2 stages).  Two warps each took 1 us per tile of 64 keys, more
//                   than anything else
//   warps 16, 17    S = Q K^T issue of either half (16 also allocates TMEM)
//   warps 18, 19    O += P V issue of either half
//   warps 20, 21    K / V producers: block table, TMA of e4m3 boxes and the scale bytes into
//                   staging rings of 4 swizzled tiles (K's with V's scale bytes beside, for
//                   the rows that stand for NaN: the softmax learns of them with the scores)
//   warp 22         finds the slice's pieces (a 2-slot ring)
// TMEM columns of a half: two score buffers of 64, O [128, 128 + D).  A row's weights go over
// the first 32 columns of the scores they came from (each thread has read its own by then),
// so S of the next tile is issued a tile ahead and its latency lies behind a softmax: with one
// score buffer and P beside it a tile of keys took 1.6 us, of which the softmax is 0.7.
//
// A piece of at most 128 rows runs as twins: both halves hold the same rows and take every
// other key tile, each with its own maximum, sum and accumulator; at the end the first half's
// threads read the second's accumulator (the same TMEM lanes, other columns) and join them.
// What bounds a half is the chain of one row's softmax (1 us a tile: 64 exponentials among 240
// instructions that wait for one another), not a unit's rate, so two chains do almost twice the
// keys.
//
// The staging rings are what the widening needs: with a tile's loads in registers, one tile
// ahead, 128-row tiles and two CTAs per SM the loads' latency (over 1 us per tile) was
// exposed and 1,000 tokens over 16,384 keys took 546 us; without any loads the same kernel
// took 291, without widening 254.
//
// Measured with the join (32 query heads, 8 KV heads of 128): 1,000 tokens over 16,384 keys 264 us
// in short bursts (985 TFLOP/s, 59 % of the measured bf16 GEMM rate; floor 157) and 284 to 291 call
// after call under the power cap, 13 x 2,047 tokens 612 (the 16-bit path's prefill 501), 30 tokens
// over 100,000 keys 81, a prompt of 333 tokens 26.  40 bytes of a thread's registers are spilled
// (64 dims: 56).  A tile of 64 keys takes 1.1 us, the softmax's
// chain; the tensor pipe is busy 53 % of the time, the exponential unit 50 %, issue slots 58 %.
// What did not help: two threads per row (a meeting of two warps a tile, 1.2 times the
// instructions: 297 us), turns at the exponential unit (277), 16 widening warps (281), the tile's
// maximum taken only where the weights with the old one sum past 2^14 (278).
//
// Every mbarrier wait is bounded; the TMEM allocation is released on every path.
#include <cuda_fp16.h>

#include "kv8.h"
#include "kv8_launch.cuh"
#include "kv8_line.cuh"
#include "kv8_widen.cuh"
#include "pa_common.cuh"
#include "tc_common.cuh"
#include "tc_softmax.cuh"

namespace pa {

constexpr int kTileRows = kKv8TileRows;
constexpr int kHalfRows = 128;
constexpr int kTileKeys = 64;
constexpr int kTileKStages = 3;
constexpr int kTileVStages = 2;
constexpr int kTileRing = 4;     // staged e4m3 tiles, K and V each
constexpr int kTileThreads = 768;
// Registers a thread: at launch and by role.  What the softmax takes, the others have given back.
constexpr int kTileRegs = 80, kSoftmaxRegs = 136, kWidenRegs = 64, kIssueRegs = 32, kLoadRegs = 48;
static_assert(256 * (kSoftmaxRegs + kWidenRegs) + 128 * (kIssueRegs + kLoadRegs) <= kTileThreads * kTileRegs,
              "a share above the launch's would be waited for");
constexpr int kTileQBox = kHalfRows * 128;  // 128 rows x 64 elements, 128-byte swizzle
constexpr int kTileBox = kTileKeys * 128;   // 64 keys x 64 elements
constexpr int kTileConsumers = 22;          // warps that read a piece: 8 softmax, 8 widening, 4 issuers, 2 producers
// Fewest keys a slice gets: below this its partial costs more than the keys it takes over.  A
// prompt of 333 tokens takes 43 us with 128, 63 with 512; one of 60 beside another 26 with 128
// and 36 with 256; calls that fill the GPU do not care.
constexpr int kTileMinKeys = 128;
// The subtracted maximum is raised only past this headroom (log2): P stays below 2^8 times the
// shift and the output accumulator is rarely rescaled.
constexpr float kTileLazy = 8.f;
// Weights and their sum stand times 2^7, which cancels: at most 2^15, and fp16 keeps 11 bits down
// to 2^-21 of the maximum and loses at most 2^-32 of it below (unshifted 2^-25: with 100,000 keys
// that far below a few, 0.3 % of the values).
constexpr float kTileWeightLog2 = 7.f;

struct TilePiece {
  int32_t row0;    // packed index of the tile's first token; -1: no more pieces
  int32_t tokens;  // of the tile
  int32_t pos0;    // position of the first token
  int32_t ctx, seq;
  int32_t j0, j1;  // tiles of 64 keys
  int32_t part;    // -1: the whole tile, else the CTA's partial slot
};

// g counts the CTA's key tiles, n those that a half works on (all of them, or as a twin every
// other).  A parity wait tells only neighbouring phases apart, so whoever waits on a ring also
// holds it back: a half passes the K and V stages of the other's tiles on itself.
struct TileBars {
  uint64_t st_full[2][kTileRing], st_empty[2][kTileRing];  // staging of K, V: landed / read
  uint64_t k_full[kTileKStages], k_free[kTileKStages];     // fp16 tiles, by g; freed by both halves
  uint64_t v_full[kTileVStages], v_free[kTileVStages];
  uint64_t s_full[2][2], s_free[2][2], p_full[2][2];       // score buffers of a half, by n
  uint64_t q_full[2];
  uint64_t x_full, x_free;                                 // the second half's result: there / read
  uint64_t d_full[2], d_empty[2];
  uint32_t tmem_base;
};

constexpr int kTileNanRing = 16;  // tiles whose NaN rows are kept: K runs at most 8 ahead of a softmax

template <int D>
struct TileCfg {
  static constexpr int NH = D / 64;
  static constexpr int Q_BYTES = 2 * NH * kTileQBox;
  static constexpr int KV_BYTES = NH * kTileBox;
  static constexpr int ST_BYTES = kTileKeys * D;
  static constexpr int OFF_K = Q_BYTES;
  static constexpr int OFF_V = OFF_K + kTileKStages * KV_BYTES;
  static constexpr int OFF_ST = OFF_V + kTileVStages * KV_BYTES;          // [K, V][ring]
  static constexpr int OFF_SCALE = OFF_ST + 2 * kTileRing * ST_BYTES;
  static constexpr int OFF_DESC = OFF_SCALE + 3 * kTileRing * kTileKeys;  // [ring][K 64, V 64], [ring][V 64]
  static constexpr int OFF_NAN = OFF_DESC + 2 * int(sizeof(TilePiece));   // [tile][4 x 16 keys]
  static constexpr int OFF_TWIN = OFF_NAN + kTileNanRing * 8;             // (m, l) of the twin's rows
  static constexpr int OFF_BAR = OFF_TWIN + kHalfRows * 8;
  static constexpr int SMEM = OFF_BAR + int(sizeof(TileBars));
  static constexpr uint32_t TMEM_COLS = 512, COL_HALF = 256;
  static constexpr uint32_t COL_O = 2 * kTileKeys;
  static_assert(COL_O + D <= COL_HALF, "TMEM budget");
  static_assert(SMEM <= 227 * 1024 && OFF_DESC % 16 == 0 && OFF_BAR % 8 == 0, "shared memory");
};

// A scale byte as two fp16 copies of 2^(b - 127); 255 is NaN.
__device__ __forceinline__ uint32_t scale_h2(uint32_t b) {
  const uint32_t h = b == 255u ? 0x7e00u : (max(113u, min(134u, b)) - 112u) << 10;
  return h | (h << 16);
}

// A value that is the same in the whole warp, known to the compiler as such.
__device__ __forceinline__ int warp_uniform(int v) { return __reduce_max_sync(0xffffffffu, v); }

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}

// A widening warp's 16 keys of a staged 64-key tile: read into registers, then widened into the
// swizzled tile.  A lane takes a 16-byte chunk of N rows, D / 16 lanes a row.  With 128 dims the
// eight lanes that one access serves at a time hold half of two rows that differ in bits 0 and
// 2: their chunks then lie in different banks both where they are read and where they are
// written, though a row's two 64-column boxes map to the same banks.  (Whole rows in order with
// half of the lanes storing their second chunk first cost eight selects a row: 5 % of all
// instructions.)
template <int D>
struct WidenPart {
  static constexpr int N = D / 32;        // rows of a lane: 16 rows x D / 16 chunks over 32 lanes
  uint4 x[N];
  uint32_t scale;                         // of key `lane`, lanes 0-15
  uint32_t from[2], to[2];                // of the lane's first two rows: chunk read, first chunk written
  int row;                                // the first; the i-th is row_at(i)

  __device__ __forceinline__ int row_at(int i) const {
    return D == 128 ? (row ^ (4 * (i & 1))) + 8 * (i >> 1) : row + 8 * i;
  }
  __device__ __forceinline__ explicit WidenPart(int lane, int row0) {
    const int l2 = (lane >> 2) & 1, l3 = (lane >> 3) & 1, l4 = lane >> 4;
    row = D == 128 ? 5 * l2 + 2 * l4 : lane / 4;
    const int chunk = D == 128 ? (lane & 3) + 4 * l3 : lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      from[i] = tile_at<D>(row0 + row_at(i), chunk);
      to[i] = (chunk >> 2) * kTileBox + sw_off(row0 + row_at(i), 2 * (chunk & 3));
    }
  }
  // Rows i and i + 2 differ in bit 3, which no swizzle looks at.
  __device__ __forceinline__ static uint32_t later(int i, int row_bytes) { return uint32_t(8 * row_bytes * (i >> 1)); }

  // Rows at and past `live` (behind the context) read as zeros.
  __device__ __forceinline__ void read(const uint8_t* staged, const uint8_t* scales, int lane, int live) {
    scale = scales[lane & 15];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const uint4*>(staged + from[i & 1] + later(i, D));
    if (live < 16) {
      if (lane >= live) scale = 0u;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (row_at(i) >= live) x[i] = make_uint4(0, 0, 0, 0);
    }
  }

  // V's rows that stand for NaN are widened to zeros (the softmax puts the NaN in the weight).
  __device__ __forceinline__ void store(uint8_t* tile, bool is_v) const {
    const uint32_t s2 = is_v && scale == 255u ? 0u : scale_h2(scale);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t sc = __shfl_sync(0xffffffffu, s2, row_at(i));
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint8_t* dst = tile + later(i, 128);
      *reinterpret_cast<uint4*>(dst + to[i & 1]) =
          make_uint4(mul_h2(widen_lo(w[0]), sc), mul_h2(widen_hi(w[0]), sc), mul_h2(widen_lo(w[1]), sc),
                     mul_h2(widen_hi(w[1]), sc));
      *reinterpret_cast<uint4*>(dst + (to[i & 1] ^ 16)) =
          make_uint4(mul_h2(widen_lo(w[2]), sc), mul_h2(widen_hi(w[2]), sc), mul_h2(widen_lo(w[3]), sc),
                     mul_h2(widen_hi(w[3]), sc));
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    kv8_tiles_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const Kv8AttnParams p, int* err) {
  using C = TileCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sK = smem + C::OFF_K;
  uint8_t* sV = smem + C::OFF_V;
  TilePiece* desc = reinterpret_cast<TilePiece*>(smem + C::OFF_DESC);
  uint16_t* nan_rows = reinterpret_cast<uint16_t*>(smem + C::OFF_NAN);
  float2* twin_ml = reinterpret_cast<float2*>(smem + C::OFF_TWIN);
  TileBars* bars = reinterpret_cast<TileBars*>(smem + C::OFF_BAR);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slice = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x % p.num_kv_heads;
  // Behind the kernel for few rows: what this reads was complete before that let it start; the
  // wait before every end makes this kernel's completion imply that one's.
  if (p.first) pdl_wait();
  pdl_release();
  LineFinder finder(p, err);
  const int64_t total = finder.total;
  const LineCuts cuts(total, p.slices, kTileMinKeys);
  const bool tells = kvh == 0;  // of the tile that its slice shares with the next ones
  if (total == 0 || slice >= cuts.n) {
    if (tid == 0 && tells) p.joins[slice].tokens = 0;
    pdl_wait();
    return;
  }

  if (warp == 16) {
    tmem_alloc(&bars->tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i)
      for (int s = 0; s < kTileRing; ++s) {
        mbar_init(&bars->st_full[i][s], kTileKeys / 16);
        mbar_init(&bars->st_empty[i][s], 4);
      }
    for (int s = 0; s < kTileKStages; ++s) {
      mbar_init(&bars->k_full[s], 4);
      mbar_init(&bars->k_free[s], 2);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->v_full[s], 4);
      mbar_init(&bars->v_free[s], 2);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bars->s_full[h][s], 1);
        mbar_init(&bars->s_free[h][s], 1);
        mbar_init(&bars->p_full[h][s], 128);
      }
      mbar_init(&bars->q_full[s], 128);
      mbar_init(&bars->d_full[s], 1);
      mbar_init(&bars->d_empty[s], kTileConsumers);
    }
    mbar_init(&bars->x_full, kHalfRows);
    mbar_init(&bars->x_free, kHalfRows);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  // The next piece of the ring, for one consuming warp; false when a wait ran out.
  auto next_piece = [&](int k, TilePiece& d) {
    const bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->d_full[k & 1], (k >> 1) & 1));
    if (ok) {
      d = desc[k & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->d_empty[k & 1]);
    }
    return ok;
  };
  auto is_twin = [&](const TilePiece& d) { return d.tokens * p.group <= kHalfRows; };
  // The second twin of a piece with one key tile: its query rows are not loaded and not waited for.
  auto is_idle = [](bool twin, int h, const TilePiece& d) { return twin && h == 1 && d.j1 - d.j0 < 2; };

  bool ok = true;
  if (warp >= 20) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
    if (warp == 22) {
      // ---------------------------------------------------------- pieces
      const int64_t x1 = cuts.at(slice + 1);
      int64_t x = cuts.at(slice);
      if (lane == 0 && tells) p.joins[slice].tokens = 0;
      for (int k = 0;; ++k) {
        LinePiece at;
        const bool more = line_next_piece(finder, x, x1, kTileKeys, at);
        if (k >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&bars->d_empty[k & 1], ((k >> 1) - 1) & 1));
        if (!ok) break;
        if (lane == 0) {
          TilePiece d{};
          d.row0 = -1;
          if (more) {
            const LineTile& t = at.t;
            const int t0 = t.index * p.tile_tokens;
            d.row0 = t.first + t0;
            d.tokens = min(p.tile_tokens, t.q - t0);
            d.ctx = t.ctx;
            d.pos0 = t.ctx - t.q + t0;
            d.seq = t.seq;
            d.j0 = at.k0 / kTileKeys;
            d.j1 = (at.k1 + kTileKeys - 1) / kTileKeys;
            d.part = at.k0 > 0 ? 0 : (at.k1 < t.keys ? 1 : -1);
          }
          desc[k & 1] = d;
          mbar_arrive(&bars->d_full[k & 1]);
          if (d.part == 1 && tells) p.joins[slice] = line_join(at.t, cuts, slice, p.tile_tokens);
        }
        if (!more) break;
      }
    } else if (warp < 22) {
      // ---------------------------------------------------------- producers: warp 20 K, 21 V
      const int v = warp - 20;
      const CUtensorMap* map = v ? &tv : &tk;
      uint8_t* ring = smem + C::OFF_ST + v * kTileRing * C::ST_BYTES;
      uint8_t* scale_ring = smem + C::OFF_SCALE + (v ? 2 * kTileRing * kTileKeys : 0);
      const int scale_step = v ? kTileKeys : 2 * kTileKeys;
      if (lane == 0) prefetch_tmap(map);
      const int shift = p.block_shift;
      // Each lane looks after one of 32 groups of 16 keys (8 tiles): its slot and scales are
      // read one round ahead; the lane issues its own box.
      auto look_up = [&](const int32_t* row, int group, int ctx, int& slot, uint4 (&sc)[2]) {
        slot = -1;
        if (16 * group < ctx) {
          int id = __ldg(row + (group >> shift));
          if (id < 0 || id >= p.pool_blocks) {
            set_error(err, PA_KV8_ERR_BLOCK);
            id = 0;
          }
          const int off = (group & ((1 << shift) - 1)) * 16;
          slot = (id << (shift + 4)) + off;
          const int64_t at = ((int64_t(id) * p.num_kv_heads + kvh) << (shift + 4)) + off;
          sc[1] = __ldg(reinterpret_cast<const uint4*>(p.v_scale + at));
          if (!v) sc[0] = __ldg(reinterpret_cast<const uint4*>(p.k_scale + at));
        }
      };
      int n = 0;  // tiles issued
      for (int k = 0; ok; ++k) {
        TilePiece d;
        ok = next_piece(k, d);
        if (!ok || d.row0 < 0) break;
        const int32_t* row = p.tables + int64_t(d.seq) * p.table_stride;
        int slot, slot_next = -1;
        uint4 sc[2] = {}, sc_next[2] = {};
        look_up(row, 4 * d.j0 + lane, d.ctx, slot, sc);
        for (int j0 = d.j0; j0 < d.j1 && ok; j0 += 8) {
          if (j0 + 8 < d.j1) look_up(row, 4 * (j0 + 8) + lane, d.ctx, slot_next, sc_next);
          for (int j = j0; j < min(j0 + 8, d.j1); ++j, ++n) {
            const int s = n % kTileRing;
            if (n >= kTileRing)
              ok = __all_sync(0xffffffffu, mbar_wait(&bars->st_empty[v][s], ((n / kTileRing) - 1) & 1));
            if (!ok) break;
            const int part = lane - 4 * (j - j0);
            if (part >= 0 && part < 4) {
              uint64_t* bar = &bars->st_full[v][s];
              if (slot >= 0) {
                uint8_t* dst = scale_ring + s * scale_step + 16 * part;
                if (!v) {
                  *reinterpret_cast<uint4*>(dst) = sc[0];
                  dst += kTileKeys;
                }
                *reinterpret_cast<uint4*>(dst) = sc[1];
                mbar_arrive_expect_tx(bar, 16 * D);  // releases the scales too
                tma_load_3d(ring + s * C::ST_BYTES + part * 16 * D, map, 0, kvh, slot, bar);
              } else {
                mbar_arrive(bar);  // behind the context: the widening warps put zeros
              }
            }
            __syncwarp();
          }
          slot = slot_next;
          sc[0] = sc_next[0];
          sc[1] = sc_next[1];
        }
      }
      if (!ok)  // leave with no copy into this CTA's shared memory in flight
        for (int i = max(0, n - kTileRing); i < n; ++i) mbar_wait(&bars->st_full[v][i % kTileRing], (i / kTileRing) & 1);
    }
  } else if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    // These loops are written for uniform registers: what an MMA needs (its descriptors above
    // all) is the same in the whole warp and known to be, and one elected thread issues.  With
    // a loop of lane 0's alone an S of 8 MMAs was 150 instructions, each waiting for the last.
    const int h = warp_uniform(warp) & 1;
    const bool leader = elect_one();
    const uint32_t tbase = warp_uniform(bars->tmem_base) + h * C::COL_HALF;
    const uint32_t tS = tbase, tO = tbase + C::COL_O;
    if (warp < 18) {
      // ---------------------------------------------------------- S issue of half h
      constexpr uint32_t idS = idesc_f16<__half>(kHalfRows, kTileKeys, false);
      const uint64_t q0 = smem_desc_sw128(smem_u32(smem + h * (C::Q_BYTES / 2)), 16, 1024);
      const uint64_t k0 = smem_desc_sw128(smem_u32(sK), 16, 1024);
      int s = 0, turn = 0, n = 0, queries = 0;  // K stage and its phase
      for (int k = 0; ok; ++k) {
        TilePiece d;
        ok = next_piece(k, d);
        if (!ok || warp_uniform(d.row0) < 0) break;
        const int tiles = warp_uniform(d.j1 - d.j0);
        const bool twin = warp_uniform(d.tokens) * p.group <= kHalfRows;
        if (!(twin && h == 1 && tiles < 2)) ok = __all_sync(0xffffffffu, mbar_wait(&bars->q_full[h], queries++ & 1));
        for (int i = 0; i < tiles && ok; ++i) {
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->k_full[s], turn));
          if (!ok) break;
          if (twin && (i & 1) != h) {
            if (leader) mbar_arrive(&bars->k_free[s]);
          } else {
            if (n >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_free[h][n & 1], ((n >> 1) - 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const uint32_t to = tS + (n & 1) * kTileKeys;
            const uint64_t kd = k0 + uint32_t(s * (C::KV_BYTES >> 4));
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                umma_f16(to, q0 + ((kk >> 2) * (kTileQBox >> 4) + (kk & 3) * 2),
                         kd + ((kk >> 2) * (kTileBox >> 4) + (kk & 3) * 2), idS, kk > 0 ? 1u : 0u);
              umma_commit(&bars->s_full[h][n & 1]);
              umma_commit(&bars->k_free[s]);
            }
            ++n;
          }
          if (++s == kTileKStages) {
            s = 0;
            turn ^= 1;
          }
        }
      }
    } else {
      // ---------------------------------------------------------- P.V issue of half h
      constexpr uint32_t idO = idesc_f16<__half>(kHalfRows, D, true);
      const uint64_t v0 = smem_desc_sw128(smem_u32(sV), kTileBox, 1024);
      int g = 0, n = 0;
      for (int k = 0; ok; ++k) {
        TilePiece d;
        ok = next_piece(k, d);
        if (!ok || warp_uniform(d.row0) < 0) break;
        const int tiles = warp_uniform(d.j1 - d.j0);
        const bool twin = warp_uniform(d.tokens) * p.group <= kHalfRows;
        uint32_t accumulate = 0;
        for (int i = 0; i < tiles && ok; ++i, ++g) {
          const int s = g & 1, b = n & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_full[s], (g >> 1) & 1));
          if (!ok) break;
          if (twin && (i & 1) != h) {
            if (leader) mbar_arrive(&bars->v_free[s]);
            continue;
          }
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->p_full[h][b], (n >> 1) & 1));
          if (!ok) break;
          tc_fence_after();
          const uint32_t from = tS + b * kTileKeys;
          const uint64_t vd = v0 + uint32_t(s * (C::KV_BYTES >> 4));
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < kTileKeys / 16; ++kk)
              umma_f16_ts(tO, from + 8 * kk, vd + kk * (2048 >> 4), idO, kk > 0 ? 1u : accumulate);
            umma_commit(&bars->s_free[h][b]);
            umma_commit(&bars->v_free[s]);
          }
          accumulate = 1;
          ++n;
        }
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ widening: warps 8-11 K, 12-15 V
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenRegs));
    const int v = warp >= 12 ? 1 : 0, row0 = 16 * (warp & 3);
    const int stages = v ? kTileVStages : kTileKStages;
    uint64_t* full = v ? bars->v_full : bars->k_full;
    uint64_t* freed = v ? bars->v_free : bars->k_free;
    const uint8_t* ring = smem + C::OFF_ST + v * kTileRing * C::ST_BYTES;
    const uint8_t* scale_ring = smem + C::OFF_SCALE + (v ? 2 * kTileRing * kTileKeys : 0) + row0;
    const int scale_step = v ? kTileKeys : 2 * kTileKeys;
    uint8_t* out = v ? sV : sK;
    int n = 0, s = 0, round = 0;
    WidenPart<D> part(lane, row0);
    for (int k = 0; ok; ++k) {
      TilePiece d;
      ok = next_piece(k, d);
      if (!ok || d.row0 < 0) break;
      for (int j = d.j0; j < d.j1; ++j, ++n) {
        const int st = n % kTileRing;
        ok = mbar_wait(&bars->st_full[v][st], (n / kTileRing) & 1);
        const int live = d.ctx - j * kTileKeys - row0;
        const uint8_t* sc = scale_ring + st * scale_step;
        part.read(ring + st * C::ST_BYTES, sc, lane, live);
        if (round > 0) ok = ok && mbar_wait(&freed[s], (round - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (!v) {
          const uint32_t nans = __ballot_sync(0xffffffffu, lane < min(16, live) && sc[kTileKeys + lane] == 255);
          if (lane == 0) nan_rows[4 * (n % kTileNanRing) + (warp & 3)] = uint16_t(nans);
        }
        part.store(out + s * C::KV_BYTES, v != 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars->st_empty[v][st]);
          mbar_arrive(&full[s]);
        }
        if (++s == stages) {
          s = 0;
          ++round;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax (one row per thread)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int h = warp >> 2;
    const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tbase = bars->tmem_base + h * C::COL_HALF + lane_base;
    const uint32_t tS = tbase, tO = tbase + C::COL_O;
    uint8_t* sQ = smem + h * (C::Q_BYTES / 2);
    const int lane_row = tid & (kHalfRows - 1);
    // Rows in global memory are read and written by kRowLanes lanes each, kRowsAtOnce at a time.
    constexpr int kRowLanes = D / 8, kRowsAtOnce = 32 / kRowLanes, kRowBatch = 4;
    const int warp_row = lane_row & ~31, row_of = lane / kRowLanes, row_chunk = lane % kRowLanes;
    int g0 = 0, n = 0, twins = 0;  // tiles of the CTA before this piece, tiles of this half, twin pieces
    for (int k = 0; ok; ++k) {
      TilePiece d;
      ok = next_piece(k, d);
      if (!ok || d.row0 < 0) break;
      const bool twin = is_twin(d);
      const int r = twin ? lane_row : tid, t_row = r / p.group, head = kvh * p.group + (r - t_row * p.group);
      const int t_eff = min(t_row, d.tokens - 1);  // spare rows repeat the last token and are not stored
      const int qpos = d.pos0 + t_eff;

      // The query rows as fp16 into the swizzled tile.  The previous piece's last S has retired
      // (its scores were read), so the tile is free.  A warp brings its own 32 rows, kRowLanes
      // lanes on each: a lane that read its own row alone would touch a line a load.
      float qs = 0.f;
      if (!is_idle(twin, h, d)) {
        const T* src = static_cast<const T*>(p.q) + int64_t(d.row0 + t_eff) * p.q_st + int64_t(head) * p.q_sh;
        float up_own = query_power<T>(0.f);
#pragma unroll 1
        for (int i0 = 0; i0 < kRowLanes; i0 += kRowBatch) {
          uint4 w[kRowBatch];
#pragma unroll
          for (int i = 0; i < kRowBatch; ++i) {
            const T* from = reinterpret_cast<const T*>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), (i0 + i) * kRowsAtOnce + row_of));
            w[i] = *reinterpret_cast<const uint4*>(from + 8 * row_chunk);
          }
#pragma unroll
          for (int i = 0; i < kRowBatch; ++i) {
            const int row = (i0 + i) * kRowsAtOnce + row_of;
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            float2 f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = unpack2(u[e], (T*)nullptr);
            float up = up_own;
            if (DType<T>::code == PA_DTYPE_BF16) {
              float big = 0.f;
#pragma unroll
              for (int e = 0; e < 4; ++e) big = fmaxf(big, fmaxf(fabsf(f[e].x), fabsf(f[e].y)));
#pragma unroll
              for (int m = 1; m < kRowLanes; m <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, m));
              up = query_power<T>(big);
              const float mine = __shfl_sync(0xffffffffu, up, (lane % kRowsAtOnce) * kRowLanes);
              if (lane / kRowsAtOnce == i0 + i) up_own = mine;
            }
            // The scores' maximum is taken before the scale, so the scale's sign goes into the row.
            const float mul = p.qscale < 0.f ? -up : up;
            *reinterpret_cast<uint4*>(sQ + (row_chunk >> 3) * kTileQBox + sw_off(warp_row + row, row_chunk & 7)) =
                make_uint4(pack2<__half>(f[0].x * mul, f[0].y * mul), pack2<__half>(f[1].x * mul, f[1].y * mul),
                           pack2<__half>(f[2].x * mul, f[2].y * mul), pack2<__half>(f[3].x * mul, f[3].y * mul));
          }
        }
        qs = fmaxf(fabsf(p.qscale) / up_own, 1e-37f);
        fence_proxy_async_smem();
        mbar_arrive(&bars->q_full[h]);
      }

      // The second half's accumulator is the first's to read until it says so.
      if (h == 1 && twins > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars->x_free, (twins - 1) & 1));
      if (!ok) break;
      float m_run = -INFINITY, l_run = 0.f;
      bool first = true;
      for (int j = d.j0 + (twin ? h : 0); j < d.j1; j += twin ? 2 : 1, ++n) {
        const int pb = n & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[h][pb], (n >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        uint32_t sr[kTileKeys];
        tmem_ld32_at<0>(tS + pb * kTileKeys, sr);
        tmem_ld32_at<32>(tS + pb * kTileKeys + 32, sr);
        tmem_wait_ld();

        const int lim = qpos - j * kTileKeys;  // key column c is visible iff c <= lim
        if (__any_sync(0xffffffffu, lim < kTileKeys - 1)) {
#pragma unroll
          for (int c = 0; c < kTileKeys; ++c) sr[c] = c <= lim ? sr[c] : __float_as_uint(-INFINITY);
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kTileKeys; c += 2)
          mx4[(c >> 1) & 3] = fmax3(mx4[(c >> 1) & 3], __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
        const float mx_s = fmax3(fmaxf(mx4[0], mx4[1]), mx4[2], mx4[3]) * qs;
        const bool grow = mx_s > m_run + kTileLazy;
        const float m_new = grow ? mx_s : m_run;
        const float alpha = grow ? ex2(m_run - m_new) : 1.f;
        // A piece may start past a row's last key: nothing seen, all weights 0.
        const float ref = (m_new == -INFINITY ? 0.f : m_new) - kTileWeightLog2;
        const uint64_t sc2 = f2pack(qs, qs), mn2 = f2pack(-ref, -ref);
        uint64_t rs2[2] = {0ull, 0ull};
        uint32_t pk[kTileKeys / 2];
#pragma unroll
        for (int c = 0; c < kTileKeys; c += 2) {
          float x0, x1;
          f2unpack(fma2(f2pack(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), sc2, mn2), x0, x1);
          const float e0 = ex2(x0), e1 = ex2(x1);
          rs2[(c >> 1) & 1] = add2(rs2[(c >> 1) & 1], f2pack(e0, e1));
          pk[c / 2] = pack2<__half>(e0, e1);
        }
        float r0, r1, r2, r3;
        f2unpack(rs2[0], r0, r1);
        f2unpack(rs2[1], r2, r3);
        l_run = l_run * alpha + ((r0 + r1) + (r2 + r3));
        m_run = m_new;

        // V rows that stand for NaN: the weight of a key that is seen becomes NaN, others stay 0.
        const uint2 nans = *reinterpret_cast<const uint2*>(nan_rows + 4 * ((g0 + j - d.j0) % kTileNanRing));
        if ((nans.x | nans.y) != 0u) {
#pragma unroll
          for (int c = 0; c < kTileKeys; ++c) {
            const bool hit = (((c < 32 ? nans.x : nans.y) >> (c & 31)) & 1u) && c <= lim;
            if (hit) pk[c / 2] |= (c & 1) ? 0x7e000000u : 0x00007e00u;
          }
        }
        tmem_st32(tS + pb * kTileKeys, *reinterpret_cast<const uint32_t(*)[32]>(&pk[0]));
        if (!first && __any_sync(0xffffffffu, grow)) {  // O *= alpha once the previous P.V retired
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_free[h][pb ^ 1], ((n - 1) >> 1) & 1));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + 32 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(tO + 32 * c, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bars->p_full[h][pb]);
        first = false;
      }
      if (!ok) break;
      g0 += d.j1 - d.j0;
      // ---- epilogue, once the half's last P.V of the piece retired (a twin may have had none)
      if (!first) ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_free[h][(n - 1) & 1], ((n - 1) >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      float mine = 1.f, other = 0.f;  // weights of the two halves' accumulators
      if (twin) {
        if (h == 1) {
          ++twins;
          twin_ml[lane_row] = make_float2(m_run, l_run);
          tc_fence_before();
          mbar_arrive(&bars->x_full);
          continue;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->x_full, twins & 1));
        if (!ok) break;
        ++twins;
        tc_fence_after();
        const float2 v = twin_ml[lane_row];
        const float m = fmaxf(m_run, v.x), ref = m == -INFINITY ? 0.f : m;
        mine = ex2(m_run - ref);
        other = ex2(v.x - ref);
        l_run = l_run * mine + v.y * other;
        m_run = m;
      }
      const bool joined = twin && d.j1 - d.j0 > 1;  // else the second half has no accumulator
      auto result = [&](int c, uint32_t (&o)[32]) {
        tmem_ld32(tO + 32 * c, o);
        if (joined) {
          uint32_t v[32];
          tmem_ld32(tO + C::COL_HALF + 32 * c, v);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[e] = __float_as_uint(__uint_as_float(o[e]) * mine + __uint_as_float(v[e]) * other);
        } else {
          tmem_wait_ld();
        }
      };
      // The rows go out through the half's query tile, free by now, each warp's own 32.
      uint8_t* const sO = sQ;
      auto put = [&](int chunk, const uint4& w) {
        *reinterpret_cast<uint4*>(sO + (chunk >> 3) * kTileQBox + sw_off(lane_row, chunk & 7)) = w;
      };
      auto get = [&](int row) {
        return *reinterpret_cast<const uint4*>(sO + (row_chunk >> 3) * kTileQBox + sw_off(warp_row + row, row_chunk & 7));
      };
      const int stored = d.tokens * p.group - (r - lane);  // rows of the warp that exist
      if (d.part < 0) {
        const float inv = 1.f / l_run;
        T* dst = static_cast<T*>(p.out) + int64_t(d.row0 + t_eff) * p.o_st + int64_t(head) * p.o_sh;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          result(c, o);
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint4 w;
            w.x = pack2<T>(__uint_as_float(o[e + 0]) * inv, __uint_as_float(o[e + 1]) * inv);
            w.y = pack2<T>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
            w.z = pack2<T>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
            w.w = pack2<T>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
            put(4 * c + e / 8, w);
          }
        }
        __syncwarp();
#pragma unroll 4
        for (int i = 0; i < kRowLanes; ++i) {
          const int row = i * kRowsAtOnce + row_of;
          T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), row));
          if (row < stored) *reinterpret_cast<uint4*>(to + 8 * row_chunk) = get(row);
        }
        __syncwarp();
      } else {
        // 32-bit values: half a row at a time.
        const int64_t at = ((int64_t(slice) * p.num_kv_heads + kvh) * 2 + d.part) * kTileRows + r;
        float* to = p.part_o + (at - lane) * D + 4 * row_chunk;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            uint32_t o[32];
            result(half * (D / 64) + c, o);
#pragma unroll
            for (int e = 0; e < 32; e += 4) put(8 * c + e / 4, make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]));
          }
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < kRowLanes; ++i) {
            const int row = i * kRowsAtOnce + row_of;
            if (row < stored) *reinterpret_cast<uint4*>(to + row * D + half * (D / 2)) = get(row);
          }
          __syncwarp();
        }
        if (lane < stored) p.part_ml[at] = make_float2(m_run, l_run);
      }
      if (twin) {
        tc_fence_before();
        mbar_arrive(&bars->x_free);
      }
      // The next piece's first P.V overwrites O only after p_full, which these threads arrive
      // on after the loads above completed (tcgen05.wait::ld).
    }
  }
  if (!ok && lane == 0) set_error(err, PA_KV8_ERR_TIMEOUT);

  pdl_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(bars->tmem_base, C::TMEM_COLS);
  }
}

// ------------------------------------------------------------------ dispatch
template <typename T, int D>
static cudaError_t tiles_one(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int* err,
                             cudaStream_t stream) {
  using C = TileCfg<D>;
  auto kern = kv8_tiles_kernel<T, D>;
  int dev = 0;
  cudaGetDevice(&dev);
  static bool configured[64] = {};
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    cudaFuncAttributes built;
    e = cudaFuncGetAttributes(&built, kern);
    if (e != cudaSuccess) return e;
    if (built.numRegs < kTileRegs) return cudaErrorInvalidConfiguration;  // see kTileRegs
    configured[dev] = true;
  }
  return launch_pdl(kern, dim3(p.slices * p.num_kv_heads), dim3(kTileThreads), C::SMEM, stream, tk, tv, p, err);
}

int kv8_tiles_slices(int num_kv_heads, int sms) {
  const int n = sms / num_kv_heads;
  return n < 1 ? 1 : n;
}

template <typename T>
static cudaError_t tiles_by_dim(int head_dim, const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p,
                                int* err, cudaStream_t s) {
  return head_dim == 64 ? tiles_one<T, 64>(tk, tv, p, err, s) : tiles_one<T, 128>(tk, tv, p, err, s);
}

cudaError_t launch_kv8_tiles(int dtype, int head_dim, const CUtensorMap& tk, const CUtensorMap& tv,
                             const Kv8AttnParams& p, int* err, cudaStream_t stream) {
  return dtype == PA_DTYPE_F16 ? tiles_by_dim<__half>(head_dim, tk, tv, p, err, stream)
                               : tiles_by_dim<__nv_bfloat16>(head_dim, tk, tv, p, err, stream);
}

cudaError_t launch_kv8_tiles_combine(int dtype, int head_dim, const Kv8AttnParams& p, cudaStream_t stream) {
  return launch_kv8_combine(dtype, head_dim, kTileRows, kTileKeys, p, stream);
}

}  // namespace pa
