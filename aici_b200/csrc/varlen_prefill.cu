// Variable-length causal prefill attention for sm_100a: tcgen05 MMA with TMEM accumulators,
// operands staged by TMA, online softmax in registers.
//
// Semantics follow mha_varlen_fwd of rllm/tch-cuda/kernels/flash_attn (flash_api.cpp:447-618,
// flash_fwd_kernel.h:590-1136): O = softmax(scale * Q K^T + causal mask) V per packed sequence
// and head, fp32 scores and accumulation, probabilities rounded to bf16 before P V, kv head =
// head / (num_heads / num_heads_k), causal mask aligned to the bottom-right corner
// (softmax.h:159-168), rows that see no column give 0 (flash_fwd_kernel.h:1056).
//
// The kernel comes in three shapes (PrefillCfg below): one query tile per CTA with two CTAs per SM
// for short sequences, two query tiles per CTA for long ones, and the two-tile shape on pairs of
// CTAs whose MMAs span two SMs.  The roles, in the two-tile shape:
// one CTA per SM owns TWO 128-row query tiles that share their key/value tiles: two query heads
// of one kv-head group when the group size is even (same rows, same causal extent), else two
// consecutive row tiles of one head.  Each key/value tile of 128 tokens is loaded once for both.
//   warp 8    : TMA producer (Q0, Q1 once; then K_0, V_0, K_1, V_1, ... through a 4-stage ring of
//               32 KB stages, 128-byte swizzle, no multicast)
//   warp 9    : TMEM owner (all 512 columns: S0, S1, O0, O1) and MMA issuer.  S_t = Q_t K_j^T in SS
//               form, O_t += P_t V_j in TS form (P read from TMEM where it overwrote S_t, V as an
//               MN-major shared-memory operand).  Issue order S0 S1 | PV0 S0' PV1 S1' | ... so that
//               the tensor pipe works on one tile while the other tile's softmax runs.
//   warps 0-3 : softmax of tile 0, warps 4-7: softmax of tile 1.  One query row per thread (= one
//               TMEM lane): tcgen05.ld the scores, mask, exp2 against a running reference maximum
//               (single pass on packed fp32 pairs; the reference moves lazily, judged by the tile's
//               row sum, and a tile whose scores jump too far is redone exactly), bf16 P written
//               back with tcgen05.st; at the end O / sum -> bf16 -> staging in the tile's Q buffer
//               (same swizzled layout) -> TMA stores, or row-by-row stores for a ragged tile.
// (One-tile shape: warps 0-3 softmax, warp 4 producer, warp 5 issuer.)  The grid is ordered
// (head, sequence, row tile), row tile slowest and longest first.
//
// Windowed variant (kWindow; bf16 and f16): a row at position d sees the keys t <= d with t > d - window or
// t < sinks.  A query tile visits the key tiles between its first row's window and its last row's
// diagonal, then those of the sinks; of tiles at an edge only the 32-column chunks that some row sees are
// multiplied (N of the S MMA, K steps of the P V MMAs), so four sinks cost a quarter of a tile.  What bounds
// long calls is what bounds the kernel without a window, the tensor pipe with its operand reads: 3650 clk for
// a step of two tiles where the MMAs alone would take 3136 (in-kernel time stamps, 1.75 GHz under load), of
// which the issuing warp waits 590.  2 x 32768 tokens, 64/8 heads, window 4096: 8.1 to 8.9 ms = 1020 to 928
// TFLOP/s of visible pairs; 4 x 4096, 32/8 heads, window 1024: 312 us = 771, window 128: 141 to 150 us = 247 to 232,
// where a CTA's fixed cost (fill 4300 clk, epilogue 2700) and the diagonal's two passes weigh as much as the MMAs.
// A probability meets the values rounded to the 16-bit type once, as in the kernel without a window: against 64
// bits the output is off by 2.0e-3 of its size, and by the 1.4e-3 of its own rounding where probabilities are exact
// (f16: 2.9e-4 and 2.1e-4).  What the rounding left as a second product, the way of window_decode.cu, would cost a
// second set of P V MMAs: these alone, without the work on the softmax side, take 2 x 32768 from 8.05 to 9.7-10.1
// ms, 8 chunks of 512 over the cache from 120 to 134 us and 4 x 4096, window 1024, from 312 to 354.
// Every barrier wait is bounded; a timeout sets AICI_STATUS_WAIT_TIMEOUT and unwinds.
#include "dependent.cuh"
#include "half_types.cuh"
#include "tcgen05.cuh"
#include "window_chunk.cuh"

namespace aici {

constexpr int kBM = 128;               // query rows per tile
constexpr int kBN = 128;               // keys per tile
constexpr int kHD = 128;               // head size
constexpr int kPanelBytes = 128 * 128; // [128 rows][64 bf16] = one 128B-swizzled panel
constexpr int kTileBytes = 2 * kPanelBytes;
constexpr int kMaxKvStages = 6;        // ring of K/V tiles (K_j and V_j alternate)

// Three shapes of the same kernel.
//   1  one query tile per CTA (short sequences): 256 TMEM columns (S/P [0,128) O [128,256)), a 2-stage
//      K/V ring, 4 softmax warps -- half the shared and tensor memory of shape 2, so TWO CTAs share an
//      SM and one CTA's fill (barriers, TMEM allocation, first loads) and drain (epilogue, stores,
//      exit) run under the other's MMAs.
//   2  two query tiles per CTA that share their K/V tiles (long sequences): all 512 TMEM columns
//      (S0/P0 [0,128) S1/P1 [128,256) O0 [256,384) O1 [384,512)), a 4-stage ring, 8 softmax warps.
//   3  shape 2 on a PAIR of CTAs (a cluster of two on neighbouring SMs) that work on four query heads
//      of one kv head: every MMA is one cta_group::2 instruction over both SMs (M = 256, 128 rows in
//      each CTA's tensor memory) and its B operand is split between them -- each CTA loads and holds
//      only half of every key tile (64 keys) and half of every value tile (64 of the 128 columns).
//      An SS-form S = Q K^T step then reads 6 KB of shared memory per SM instead of 8 KB and a P V
//      step 2 KB instead of 4 KB; shared-memory bandwidth into the tensor core (about 64 B/clk) is
//      what holds shape 2 back.  The leader CTA issues; the other CTA's issuer warp relays "my half
//      has landed" to it; completion comes back to both through multicast commits.
template <int kShape>
struct PrefillCfg {
  static constexpr int kTiles = kShape == 1 ? 1 : 2;
  static constexpr bool kPair = kShape == 3;
  static constexpr int kStages = kShape == 1 ? 2 : (kShape == 2 ? 4 : 6);
  static constexpr int kStageBytes = kPair ? kTileBytes / 2 : kTileBytes;
  static constexpr int kSoftmaxWarps = 4 * kTiles;
  static constexpr int kProducerWarp = 4 * kTiles;
  static constexpr int kMmaWarp = 4 * kTiles + 1;
  static constexpr int kThreads = (4 * kTiles + 2) * 32;
  static constexpr uint32_t kCols = 256u * kTiles;
  static constexpr int kSmemBytes = kTiles * kTileBytes + kStages * kStageBytes + 1024 /*align*/ + 512 /*PrefillSmem*/;
  static constexpr int kCtasPerSm = kTiles == 2 ? 1 : 2;
};
constexpr float kRescaleThreshold = 8.f;  // log2 units: the running reference moves once a score exceeds it by this
// Single-pass tiles: a row sum above the first moves the reference (some score is 2^8 above it, or many are above
// it); at the second or above (or NaN) the tile is redone exactly, for f16 probabilities, whose range ends at
// 65504, at the third.
constexpr float kRescaleSum = 256.f;
constexpr float kDangerSum = 1e30f;
constexpr float kDangerSumF16 = 3e4f;

struct PrefillParams {
  // output [total_q, heads, 128] (strides below) in `world` buffers -- this GPU's and, for the
  // fused head gather, every peer's; this rank's head h is written at head index out_head0 + h
  __nv_bfloat16 *out[8];
  int world, out_head0;
  const int32_t *cu_q;
  const int32_t *cu_k;
  int64_t o_tok_stride, o_head_stride;
  int group;
  int causal;
  int pair_heads;  // 1: the two tiles are heads 2y and 2y+1; 0: two consecutive row tiles of head y
  int tma_store;   // 1: full output tiles leave shared memory as TMA stores (one output buffer only)
  int total_q;     // rows of the packed query / output tensors
  float scale_log2e;
  unsigned int *status;
  // paged variant: keys/values are read from the KV cache through the block table
  const int32_t *block_tables;  // [batch, max_blocks]
  const int32_t *k_lens;        // [batch] tokens of each sequence present in the cache
  int max_blocks;
  int64_t num_blocks;
  // windowed variant: a row at position d sees the keys t <= d with t > d - window or t < sinks
  int window, sinks;
  int longer_than;        // sequences of at most so many tokens are another launch's
  int max_q;              // sequences of more are refused: zero rows and a status
  int batch, grid_heads;  // grid_heads > 0: its grid is (tile, head), heads fastest, and batch_tile finds the tile
};

// One tensor map per output buffer (this GPU's and, for the fused gather, every peer's); the windowed
// variant has one output (1 KB less of kernel arguments for the host to hand over).
struct OutMaps {
  CUtensorMap m[8];
};
struct OutMap {
  CUtensorMap m[1];
};
template <bool kWindow>
struct OutMapsOf {
  using type = OutMaps;
  static const OutMaps &of(const OutMaps &m) { return m; }
};
template <>
struct OutMapsOf<true> {
  using type = OutMap;
  static OutMap of(const OutMaps &m) { return {{m.m[0]}}; }
};

struct PrefillSmem {
  uint64_t q_full[2], kv_full[kMaxKvStages], kv_empty[kMaxKvStages], s_full[2], p_ready[2], o_full[2], staged[2], drain;
  uint64_t q_peer[2], kv_peer[kMaxKvStages];  // CTA pairs: the leader's view of "the other CTA's half has landed"
  uint32_t tmem_base;
  uint32_t aborted;
};

struct TileInfo {
  int h;        // query head
  int m0;       // first query row within the sequence
  int rows;     // valid rows (<= 128); 0 = this tile does not exist
  int n_tiles;  // key/value tiles it visits; 0 = nothing visible
};

// Windowed variant: the keys that some row of a CTA's query tile sees are [0, sinks) and [lo, lim).
// The tiles that hold them are visited from the diagonal downwards, sinks last: the first tile then
// gives (nearly) every row its reference maximum, where an ascending order would start in tiles whose
// leading columns most rows do not see.
struct WindowTiles {
  int lo, lim, sinks;
  int first, n_win;  // first window tile, number of window tiles
  int n_sink;        // tiles of sinks below the first window tile
  __device__ __forceinline__ int tile(int i) const {
    return i < n_win ? first + n_win - 1 - i : n_sink - 1 - (i - n_win);
  }
  // The 32-column chunks [c0, c1) of the i-th visited tile that hold every column some row sees: scores,
  // probabilities and value rows outside them are neither computed nor read.
  __device__ __forceinline__ void chunks(int i, int &c0, int &c1) const {
    const int n0 = tile(i) * kBN;
    const int hi = i < n_win ? lim : min(sinks, lo);
    c1 = (min(hi - n0, kBN) + 31) / 32;
    c0 = i < n_win && sinks <= n0 ? max(lo - n0, 0) / 32 : 0;
  }
};

// Which query tile a CTA of a windowed call takes when the batch is ragged, that is when it may have fewer
// tiles than sequences times the longest one's (the host, which does not know the lengths, counts at most
// total_q / 128 + batch).  The grid has that many tiles in a row, those that do not exist behind all others.
// (In a grid of all sequences times the longest's tiles the empty CTAs wait for an SM's shared memory like
// the others, and real ones behind them: one prompt of 4096 and 63 of 20 tokens, 8/2 heads, window 512: 114
// and 37 us; 4 prompts of 64 to 512, 32 heads, window 128: 15.1 and 13.4 us; 200 of 1 to 400, 8/2 heads: 135
// and 139 us.  Where all sequences are as long as the longest the finding alone would cost 0.4 us a CTA.)
// Sequences and their tiles are counted from the last.  All lanes of a warp take part.  (Clamped sums, as
// long as they do not decrease: no more tiles exist than the grid has places.)
struct BatchTile {
  int b, mb;  // sequence (-1: no tile) and row tile
  int q0, lq, k0, lk;
};
// A running sum of query lengths: rows outside the query tensor are nobody's.
__device__ __forceinline__ int row_sum(const PrefillParams &p, int i) { return min(max(p.cu_q[i], 0), p.total_q); }

template <bool kPaged>
__device__ __forceinline__ BatchTile batch_tile(const PrefillParams &p, int idx, int lane) {
  BatchTile t = {-1, 0, 0, 0, 0, 0};
  if (p.batch <= 32) {
    // a sequence to a lane
    const int i = min(lane, p.batch - 1);
    const int q0 = row_sum(p, i), q1 = row_sum(p, i + 1);
    const int k0 = kPaged ? 0 : p.cu_k[i], k1 = kPaged ? p.k_lens[i] : p.cu_k[i + 1];
    const int n = lane < p.batch && q1 - q0 > p.longer_than ? (q1 - q0 + kBM - 1) / kBM : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    idx = __shfl_sync(0xffffffffu, upto, 31) - 1 - idx;
    if (idx < 0) return t;
    t.b = __popc(__ballot_sync(0xffffffffu, upto <= idx));
    t.mb = idx - __shfl_sync(0xffffffffu, upto - n, t.b);
    t.q0 = __shfl_sync(0xffffffffu, q0, t.b);
    t.lq = __shfl_sync(0xffffffffu, q1 - q0, t.b);
    t.k0 = __shfl_sync(0xffffffffu, k0, t.b);
    t.lk = __shfl_sync(0xffffffffu, k1 - k0, t.b);
    return t;
  }
  // Many sequences: tiles are numbered as if sequence i began at cu[i] / 128 + i, which leaves room for all
  // of its tiles, and the sequence is found by a search with 32 probes a round.
  const int origin = row_sum(p, 0);
  auto start = [&](int i) { return (row_sum(p, i) - origin) / kBM + i; };
  idx = start(p.batch) - 1 - idx;
  if (idx < 0) return t;
  int lo = 0;
  for (int n = p.batch; n > 1;) {
    const int step = (n + 31) / 32, at = lane * step;
    const int skip = (max(__popc(__ballot_sync(0xffffffffu, at < n && start(lo + at) <= idx)), 1) - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  t.mb = idx - start(lo);
  t.q0 = row_sum(p, lo);
  t.lq = row_sum(p, lo + 1) - t.q0;
  if (t.lq <= p.longer_than || t.mb < 0 || t.mb >= (t.lq + kBM - 1) / kBM) return t;
  t.b = lo;
  t.k0 = kPaged ? 0 : p.cu_k[lo];
  t.lk = kPaged ? p.k_lens[lo] : p.cu_k[lo + 1] - t.k0;
  return t;
}

// Bit i: column cb + i is in [lo, hi) or [0, sinks), and below hi.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t visible_bits(int cb, int lo, int hi, int sinks) {
  return bits_below(hi - cb) & (~bits_below(lo - cb) | bits_below(sinks - cb));
}

__device__ __forceinline__ void zero_rows(const PrefillParams &p, int q0, const TileInfo &T, int tid,
                                          int nthreads) {
  for (int i = tid; i < T.rows * (kHD / 8); i += nthreads) {
    const int r = i / (kHD / 8), c = i % (kHD / 8);
    for (int w = 0; w < p.world; ++w)
      *reinterpret_cast<uint4 *>(p.out[w] + (int64_t)(q0 + T.m0 + r) * p.o_tok_stride +
                                 (int64_t)(p.out_head0 + T.h) * p.o_head_stride + c * 8) = make_uint4(0, 0, 0, 0);
  }
}

// kPaged = false: K and V are packed [total_k, Hkv, 128] tensors (tensor maps as for Q).
// kPaged = true : K and V come from the paged cache.  A key tile is 8 blocks of two halves,
//   [16 chunks][8 tokens][8 elements] each (2 KB, no swizzle: exactly the 8-row x 16-byte core
//   matrices the MMA wants, leading offset 128 B between the two chunks of a K step, stride offset
//   2 KB between 8-token groups); a value tile is 8 blocks of [128 d][16 tokens] in the 32-byte swizzle,
//   d reordered in groups of four, one K = 16 MMA per block.  Value columns past the sequence end
//   are zeroed in shared memory before P V (cache slots there may hold anything, NaN included).
//
// kWindow = true: sliding window and sinks (always causal); the CTA's tiles share their rows (one tile, or
// two heads of one kv head).  T: bf16, or f16 in the windowed variant.
template <bool kPaged, int kShape, bool kWindow = false, typename T16 = __nv_bfloat16>
__global__ void __launch_bounds__(PrefillCfg<kShape>::kThreads, PrefillCfg<kShape>::kCtasPerSm)
varlen_prefill_kernel(const __grid_constant__ CUtensorMap tmap_q,
                      const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v,
                      const __grid_constant__ typename OutMapsOf<kWindow>::type tmap_o, const PrefillParams p) {
  using Cfg = PrefillCfg<kShape>;
  constexpr int kTiles = Cfg::kTiles;
  constexpr bool kPair = Cfg::kPair;
  static_assert(!(kPair && kPaged), "the CTA-pair shape reads packed K/V only");
  static_assert(!(kPair && kWindow), "the CTA-pair shape has no window");
  // a probability must stay inside the 16-bit type until the reference has moved
  constexpr float kDanger = Half16<T16>::kDtype == AICI_DTYPE_F16 ? kDangerSumF16 : kDangerSum;
  constexpr int kKvStages = Cfg::kStages;
  constexpr int kStageBytes = Cfg::kStageBytes;
  constexpr int kPrefillThreads = Cfg::kThreads;
  constexpr uint32_t kTmemCols = Cfg::kCols;
  constexpr uint32_t kOCol = 128u * kTiles;  // first column of O0
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // The grid is ordered (head, sequence, row tile) with the row tile as the slowest index: all the
  // longest tiles of the batch start first and the CTAs with one key tile fill the tail.  (Windowed: see
  // BatchTile.)
  // Beside a launch for the short sequences (longer_than > 0) this grid starts while that one runs, which
  // began only when everything before it had ended; CTA 0 leaves after it, so that this grid ends last.
  // CTA 0 also reports running sums that leave the query tensor (windowed: row_sum).
  auto leave = [&]() {
    if (!kWindow || blockIdx.x + blockIdx.y + blockIdx.z != 0) return;
    if (tid == 0 && (p.cu_q[0] < 0 || p.cu_q[p.batch] > p.total_q)) set_status(p.status, AICI_STATUS_BAD_BLOCK);
    if (p.longer_than > 0) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  if (kWindow && p.longer_than == 0) dependent_start();
  int b, q0, lq, k0 = 0, lk = 0, win_mb = 0, win_head = 0;
  if (kWindow && p.grid_heads > 0) {
    const int tile = (int)blockIdx.x / p.grid_heads;
    const BatchTile t = batch_tile<kPaged>(p, tile, lane);
    if (t.b < 0) return leave();
    b = t.b, q0 = t.q0, lq = t.lq, k0 = t.k0, lk = t.lk, win_mb = t.mb;
    win_head = (int)blockIdx.x - tile * p.grid_heads;
  } else {
    b = blockIdx.y;
    win_head = (int)blockIdx.x;
    if (kWindow) q0 = row_sum(p, b), lq = row_sum(p, b + 1) - q0;
    else q0 = p.cu_q[b], lq = p.cu_q[b + 1] - q0;
    if (kPaged) {
      lk = p.k_lens[b];
    } else {
      k0 = p.cu_k[b];
      lk = p.cu_k[b + 1] - k0;
    }
  }
  if (kPaged) {
    if (lk > p.max_blocks * 16) {
      if (tid == 0) set_status(p.status, AICI_STATUS_BAD_BLOCK);
      lk = p.max_blocks * 16;
    }
    if (lk < 0) lk = 0;
  }
  const int n_mblocks = (lq + kBM - 1) / kBM;
  if (kWindow && lq > p.max_q) {
    // Longer than the caller stated: the plain grid has no CTA for some of its tiles, so none is worked on
    // (in the ragged grid neither: what a call gives does not depend on the other sequences' lengths).
    if (tid == 0) set_status(p.status, AICI_STATUS_BAD_BLOCK);
    const int first = p.grid_heads > 0 ? win_mb : (int)blockIdx.z, step = p.grid_heads > 0 ? n_mblocks : (int)gridDim.z;
    for (int mb = first; mb < n_mblocks; mb += step)
      for (int t = 0; t < kTiles; ++t)
        zero_rows(p, q0, TileInfo{kTiles * win_head + t, mb * kBM, min(kBM, lq - mb * kBM), 0}, tid, kPrefillThreads);
    return leave();
  }
  if (kWindow && p.grid_heads == 0) win_mb = n_mblocks - 1 - (int)blockIdx.z;

  // ---- which two tiles does this CTA own? (longest causal tiles are scheduled first) ----------
  TileInfo tiles[2];
  {
    int mb[2], hh[2];
    if (kWindow) {
      mb[0] = win_mb;
      mb[1] = kTiles == 1 ? -1 : win_mb;
      hh[0] = kTiles == 1 ? win_head : 2 * win_head;
      hh[1] = hh[0] + 1;
    } else if (kTiles == 1) {
      mb[0] = n_mblocks - 1 - (int)blockIdx.z;
      mb[1] = -1;  // no second tile
      hh[0] = hh[1] = (int)blockIdx.x;
    } else if (kPair) {
      // clusters of two CTAs along x: CTA x = 2y + r holds heads 4y + 2r and 4y + 2r + 1
      mb[0] = mb[1] = n_mblocks - 1 - (int)blockIdx.z;
      hh[0] = 2 * (int)blockIdx.x;
      hh[1] = hh[0] + 1;
    } else if (p.pair_heads) {
      mb[0] = mb[1] = n_mblocks - 1 - (int)blockIdx.z;
      hh[0] = 2 * (int)blockIdx.x;
      hh[1] = hh[0] + 1;
    } else {
      mb[1] = n_mblocks - 1 - 2 * (int)blockIdx.z;
      mb[0] = mb[1] - 1;
      hh[0] = hh[1] = (int)blockIdx.x;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      TileInfo &T = tiles[t];
      T.h = hh[t];
      T.m0 = mb[t] * kBM;
      T.rows = mb[t] >= 0 && mb[t] < n_mblocks ? min(kBM, lq - T.m0) : 0;
      int lim = lk;
      if (p.causal) lim = min(lk, T.m0 + T.rows + lk - lq);
      T.n_tiles = (T.rows > 0 && lim > 0) ? (lim + kBN - 1) / kBN : 0;
    }
  }
  if (tiles[0].rows == 0 && tiles[1].rows == 0) return leave();
  const int hk = tiles[1].rows > 0 ? tiles[1].h / p.group : tiles[0].h / p.group;
  // tiles that see no key at all are zero rows (flash_fwd_kernel.h:1056)
  if (tiles[0].rows > 0 && tiles[0].n_tiles == 0) zero_rows(p, q0, tiles[0], tid, kPrefillThreads);
  if (tiles[1].rows > 0 && tiles[1].n_tiles == 0) zero_rows(p, q0, tiles[1], tid, kPrefillThreads);
  WindowTiles win = {};
  if (kWindow && (tiles[0].n_tiles > 0 || tiles[1].n_tiles > 0)) {
    const TileInfo &R = tiles[0].n_tiles > 0 ? tiles[0] : tiles[1];
    win.lim = min(lk, R.m0 + R.rows + lk - lq);
    win.sinks = min(p.sinks, win.lim);
    win.lo = max(0, R.m0 + lk - lq - min(p.window, lk) + 1);  // the first row's window begins here
    win.first = win.lo / kBN;
    win.n_win = R.n_tiles - win.first;
    win.n_sink = min((win.sinks + kBN - 1) / kBN, win.first);
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (tiles[t].n_tiles > 0) tiles[t].n_tiles = win.n_sink + win.n_win;
  }
  const int nt0 = tiles[0].n_tiles, nt1 = tiles[1].n_tiles;
  const int nmax = max(nt0, nt1);
  if (nmax == 0) return leave();
  auto tile_of = [&](int j) { return kWindow ? win.tile(j) : j; };  // key tile of the j-th visit
  // end of the keys that count for this CTA, and whether any key of a 16-token block does
  const int k_end = kWindow ? win.lim : lk;
  auto block_counts = [&](int first_token) {
    return first_token < k_end && (!kWindow || first_token + 16 > win.lo || first_token < win.sinks);
  };

  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem;                       // two tiles
  uint8_t *sKV = smem + kTiles * kTileBytes;     // kKvStages stages
  PrefillSmem *sh = reinterpret_cast<PrefillSmem *>(smem + kTiles * kTileBytes + kKvStages * kStageBytes);
  // CTA pairs: rank 0 of the cluster is the leader (issues the MMAs of both CTAs)
  const uint32_t pair_rank = kPair ? cluster_ctarank() : 0u;
  const bool leader = pair_rank == 0u;

  if (tid == 0) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh->q_full[t], 1);
      mbar_init(&sh->s_full[t], 1);
      mbar_init(&sh->p_ready[t], kPair ? 8 : 4);  // pairs: the softmax warps of both CTAs report to the leader
      mbar_init(&sh->q_peer[t], 1);
      mbar_init(&sh->o_full[t], 1);
      mbar_init(&sh->staged[t], 4);
    }
#pragma unroll
    for (int s = 0; s < kKvStages; ++s) {
      mbar_init(&sh->kv_full[s], 1);
      mbar_init(&sh->kv_empty[s], 1);
      mbar_init(&sh->kv_peer[s], 1);
    }
    mbar_init(&sh->drain, 1);
    sh->aborted = 0;
    fence_mbar_init();
  }
  if (warp == Cfg::kMmaWarp) {
    if (kPair) {
      tmem_alloc_pair(&sh->tmem_base, kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&sh->tmem_base, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (kPair) cluster_sync_all();  // the other CTA's barriers exist before anything arrives on them
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = sh->tmem_base;

  if (warp == Cfg::kProducerWarp) {
    // ---------------------------------------------------------------- TMA producer -----------
    if (lane == 0) {
      tma_prefetch_desc(&tmap_q);
      tma_prefetch_desc(&tmap_k);
      tma_prefetch_desc(&tmap_v);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (tiles[t].n_tiles > 0) {
          mbar_expect_tx(&sh->q_full[t], kTileBytes);
          tma_load_3d(sQ + t * kTileBytes, &tmap_q, 0, tiles[t].h, q0 + tiles[t].m0, &sh->q_full[t]);
          tma_load_3d(sQ + t * kTileBytes + kPanelBytes, &tmap_q, 64, tiles[t].h, q0 + tiles[t].m0,
                      &sh->q_full[t]);
        }
      }
    }
    if (kPaged) {
      // All lanes take part: lane l < 8 owns cache block l of the tile (its id is read once per
      // tile, one tile ahead), lanes 0-7 each issue one key copy or one value copy; lane 0 posts the expected byte count.
      const int32_t *bt_row = p.block_tables + (int64_t)b * p.max_blocks;
      auto load_id = [&](int j) {
        int id = 0;
        if (j < nmax && block_counts(tile_of(j) * kBN + (lane & 7) * 16)) {
          id = bt_row[tile_of(j) * 8 + (lane & 7)];
          if (id < 0 || id >= p.num_blocks) {
            set_status(p.status, AICI_STATUS_BAD_BLOCK);
            id = 0;
          }
        }
        return id;
      };
      int id_cur = load_id(0), id_next = 0;
      bool ok = true;
      for (int i = 0; ok && i < 2 * nmax; ++i) {  // i even: K_{i/2}, i odd: V_{i/2}
        const int stage = i % kKvStages;
        const int j = i >> 1;
        if (!(i & 1)) id_next = load_id(j + 1);
        ok = __all_sync(0xffffffffu,
                        mbar_wait_abortable(&sh->kv_empty[stage], (((uint32_t)i / kKvStages) & 1u) ^ 1u, p.status));
        if (!ok) break;
        uint8_t *dst = sKV + stage * kTileBytes;
        const int bi = lane & 7;
        const bool counts = block_counts(tile_of(j) * kBN + bi * 16);  // cache blocks of this tile to load
        const int nb = __popc(__ballot_sync(0xffffffffu, counts) & 0xffu);
        if (lane == 0) mbar_expect_tx(&sh->kv_full[stage], nb * 4096);
        __syncwarp();
        if (i & 1) {
          if (lane < 8 && counts) tma_load_4d(dst + bi * 4096, &tmap_v, 0, 0, hk, id_cur, &sh->kv_full[stage]);
          id_cur = id_next;
        } else {
          if (lane < 8 && counts) tma_load_5d(dst + bi * 4096, &tmap_k, 0, 0, 0, hk, id_cur, &sh->kv_full[stage]);
        }
        __syncwarp();
      }
    } else if (lane == 0) {
      for (int i = 0; i < 2 * nmax; ++i) {  // i even: K_{i/2}, i odd: V_{i/2}
        const int stage = i % kKvStages;
        if (!mbar_wait_abortable(&sh->kv_empty[stage], (((uint32_t)i / kKvStages) & 1u) ^ 1u, p.status)) break;
        uint8_t *dst = sKV + stage * kStageBytes;
        const CUtensorMap *tm = (i & 1) ? &tmap_v : &tmap_k;
        mbar_expect_tx(&sh->kv_full[stage], kStageBytes);
        if (!kPair) {
          tma_load_3d(dst, tm, 0, hk, k0 + tile_of(i >> 1) * kBN, &sh->kv_full[stage]);
          tma_load_3d(dst + kPanelBytes, tm, 64, hk, k0 + tile_of(i >> 1) * kBN, &sh->kv_full[stage]);
        } else if (i & 1) {
          // this CTA's half of the value tile: 64 of the 128 columns, all 128 tokens (one panel)
          tma_load_3d(dst, tm, 64 * (int)pair_rank, hk, k0 + (i >> 1) * kBN, &sh->kv_full[stage]);
        } else {
          // this CTA's half of the key tile: 64 of the 128 tokens (tmap_k's box is 64 rows high),
          // two panels of 64 columns
          const int row = k0 + (i >> 1) * kBN + 64 * (int)pair_rank;
          tma_load_3d(dst, tm, 0, hk, row, &sh->kv_full[stage]);
          tma_load_3d(dst + kPanelBytes / 2, tm, 64, hk, row, &sh->kv_full[stage]);
        }
      }
    }
  } else if (warp == Cfg::kMmaWarp && kPair && !leader) {
    // ---------------------------------------------------------------- relay (pairs, second CTA) --
    // The leader issues the MMAs that read this CTA's shared memory too; it learns from this warp,
    // in consumption order, that this CTA's Q tiles and K/V halves have landed.
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_abortable(bar, parity, p.status));
      return ok;
    };
    for (int t = 0; t < 2 && ok; ++t) {
      if (tiles[t].n_tiles > 0 && wait(&sh->q_full[t], 0)) {
        fence_proxy_async_smem();
        if (lane == 0) mbar_arrive_cluster(&sh->q_peer[t], 0);
      }
    }
    for (int i = 0; ok && i < 2 * nmax; ++i) {
      const int stage = i % kKvStages;
      if (!wait(&sh->kv_full[stage], ((uint32_t)i / kKvStages) & 1u)) break;
      const int j = i >> 1;
      if ((i & 1) && lk - j * kBN < kBN) {
        // value rows behind the end of the sequence are cleared (see the leader's copy of this loop)
        const int valid = lk - j * kBN;
        uint8_t *vt = sKV + stage * kStageBytes;
        for (int idx = valid * 8 + lane; idx < kBN * 8; idx += 32)
          *reinterpret_cast<uint4 *>(vt + (idx >> 3) * 128 + (idx & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(&sh->kv_peer[stage], 0);
    }
  } else if (warp == Cfg::kMmaWarp) {
    // ---------------------------------------------------------------- MMA issuer -------------
    constexpr bool kF16 = Half16<T16>::kDtype == AICI_DTYPE_F16;
    constexpr uint32_t idesc_s = kF16 ? idesc_f16(kBM, kBN, false) : idesc_bf16(kPair ? 2 * kBM : kBM, kBN, false);
    constexpr uint32_t idesc_pv =  // packed V: MN-major; cache V: K-major
        kF16 ? idesc_f16(kBM, kHD, !kPaged) : idesc_bf16(kPair ? 2 * kBM : kBM, kHD, !kPaged);
    constexpr int kKPanel = kPair ? kPanelBytes / 2 : kPanelBytes;  // one 64-column panel of a key (half) tile
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_abortable(bar, parity, p.status));
      return ok;
    };
    // barriers another CTA arrives on: acquire at cluster scope
    auto wait_cluster = [&](uint64_t *bar, uint32_t parity) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_abortable_cluster(bar, parity, p.status));
      return ok;
    };
    auto wait_q = [&](int t) {
      wait(&sh->q_full[t], 0);
      if (kPair) wait_cluster(&sh->q_peer[t], 0);
      return ok;
    };
    auto wait_kv = [&](int i) {
      wait(&sh->kv_full[i % kKvStages], ((uint32_t)i / kKvStages) & 1u);
      if (kPair) wait_cluster(&sh->kv_peer[i % kKvStages], ((uint32_t)i / kKvStages) & 1u);
      return ok;
    };
    auto wait_p = [&](int t, int j) {
      return kPair ? wait_cluster(&sh->p_ready[t], (uint32_t)j & 1u) : wait(&sh->p_ready[t], (uint32_t)j & 1u);
    };
    auto commit = [&](uint64_t *bar) {
      if (kPair) tc_commit_pair(bar, 3);
      else tc_commit(bar);
    };
    // S_t = Q_t K^T.  Q, K: K-major, rows of 128 B, 8-row groups 1024 B apart, two 64-column panels.
    // (windowed: `ch` holds the tile's chunk range, worked out before the waits so that nothing but the
    // instructions themselves lies between a barrier and its MMAs)
    struct Chunks {
      int c0 = 0, c1 = kBN / 32;
      uint32_t idesc_s = 0;
    };
    auto chunks_of = [&](int j) {
      Chunks ch;
      if constexpr (kWindow) {
        if (j < nmax) win.chunks(j, ch.c0, ch.c1);
        ch.idesc_s = (idesc_s & ~(63u << 17)) | ((uint32_t)(4 * (ch.c1 - ch.c0)) << 17);  // N = 32 columns a chunk
      }
      return ch;
    };
    auto issue_s = [&](int t, int i_k, const Chunks &ch) {
      tc_fence_after();
      if (lane == 0) {
        const uint64_t qdesc = smem_desc_sw128(smem_u32(sQ + t * kTileBytes), 16, 1024);
        uint32_t kaddr = smem_u32(sKV + (i_k % kKvStages) * kStageBytes);
        uint32_t s_col = tmem_base + t * 128;
        const uint32_t idesc = kWindow ? ch.idesc_s : idesc_s;
        if constexpr (kWindow) {
          kaddr += ch.c0 * (kPaged ? 8192 : 4096);  // 32 key rows
          s_col += 32 * ch.c0;
        }
        const uint64_t kdesc = kPaged ? smem_desc(kaddr, 128, 2048, 0) : smem_desc_sw128(kaddr, 16, 1024);
#pragma unroll
        for (int ks = 0; ks < kHD / 16; ++ks) {
          const uint64_t adv = (uint64_t)(((ks >> 2) * kPanelBytes + (ks & 3) * 32) >> 4);
          const uint64_t kadv = kPaged ? (uint64_t)((ks * 256) >> 4)
                                       : (uint64_t)(((ks >> 2) * kKPanel + (ks & 3) * 32) >> 4);
          if (kPair) umma_ss_pair(tmem_base + t * 128, qdesc + adv, kdesc + kadv, idesc_s, ks > 0 ? 1u : 0u);
          else umma_ss(s_col, qdesc + adv, kdesc + kadv, idesc, ks > 0 ? 1u : 0u);
        }
        commit(&sh->s_full[t]);
      }
      __syncwarp();
    };
    // O_t += P_t V.  V as B operand: N (= d) contiguous, 64 d per swizzle atom, second atom one
    // panel further (leading offset), 8-token groups 1024 B apart (stride offset).  In a CTA pair
    // each CTA holds one atom (its 64 columns).
    auto issue_pv = [&](int t, int i_v, bool first, bool last, const Chunks &ch) {
      tc_fence_after();
      if (lane == 0) {
        const uint32_t vaddr = smem_u32(sKV + (i_v % kKvStages) * kStageBytes);
        // packed: one MN-major tile, a K step = 16 token rows of 128 B; cache: one block per K step,
        // rows (d) of 32 B with the 32-byte swizzle, 8-row groups 256 B apart
        const uint64_t vdesc = kPaged ? smem_desc(vaddr, 16, 256, 6) : smem_desc_sw128(vaddr, kPanelBytes, 1024);
        const uint32_t vstep = kPaged ? 4096u : 2048u;
        auto step = [&](int ks, bool accumulate) {
          if (kPair)
            umma_ts_pair(tmem_base + kOCol + t * 128, tmem_base + t * 128 + 8 * ks,
                         vdesc + (uint64_t)((ks * vstep) >> 4), idesc_pv, accumulate ? 1u : 0u);
          else
            umma_ts(tmem_base + kOCol + t * 128, tmem_base + t * 128 + 8 * ks, vdesc + (uint64_t)((ks * vstep) >> 4),
                    idesc_pv, accumulate ? 1u : 0u);
        };
        if (!kWindow || ch.c1 - ch.c0 == kBN / 32) {
#pragma unroll
          for (int ks = 0; ks < kBN / 16; ++ks) step(ks, !first || ks > 0);
        } else {
#pragma unroll 1
          for (int ks = 2 * ch.c0; ks < 2 * ch.c1; ++ks) step(ks, !first || ks > 2 * ch.c0);
        }
        if (last) commit(&sh->o_full[t]);
      }
      __syncwarp();
    };
    auto release = [&](int i) {
      if (lane == 0) commit(&sh->kv_empty[i % kKvStages]);
      __syncwarp();
    };

    Chunks ch = chunks_of(0);
    if (nt0 > 0) wait_q(0);
    if (nt1 > 0) wait_q(1);
    if (wait_kv(0)) {
      if (nt0 > 0) issue_s(0, 0, ch);
      if (nt1 > 0) issue_s(1, 0, ch);
      release(0);
    }
    for (int j = 0; ok && j < nmax; ++j) {
      const int i_v = 2 * j + 1, i_kn = 2 * j + 2;
      const Chunks ch_next = chunks_of(j + 1);
      if (!wait_kv(i_v)) break;
      if constexpr (kWindow) {
        // Value rows that no row of this query tile sees -- past its last row's position, or between the
        // sinks and its first row's window -- are cleared: their probabilities are 0, but 0 x NaN is
        // NaN, and blocks without a visible token were not loaded at all.
        const int n0 = tile_of(j) * kBN;
        const int hi = min(kBN, win.lim - n0);
        const int dead0 = min(max(win.sinks - n0, 0), kBN), dead1 = min(max(win.lo - n0, 0), kBN);
        if (hi < kBN || dead0 < dead1) {
          uint8_t *vt = sKV + (i_v % kKvStages) * kStageBytes;
          auto clear = [&](int a, int b) {  // tokens [a, b) of the tile
            if (kPaged) {
              for (int bi = a / 16; bi * 16 < b; ++bi) {
                uint8_t *vb = vt + bi * 4096;
                const int t0 = max(a - bi * 16, 0), t1 = min(b - bi * 16, 16);
                if (t1 - t0 == 16) {
                  for (int idx = lane; idx < 256; idx += 32) reinterpret_cast<uint4 *>(vb)[idx] = make_uint4(0, 0, 0, 0);
                } else {
                  for (int tok = t0; tok < t1; ++tok)
                    for (int d = lane; d < kHD; d += 32) {
                      const int at = d * 32 + (((tok >> 3) ^ ((d >> 2) & 1)) << 4) + (tok & 7) * 2;
                      *reinterpret_cast<uint16_t *>(vb + at) = 0;
                    }
                }
              }
            } else {
              for (int idx = a * 16 + lane; idx < b * 16; idx += 32) {
                const int r = idx / 16, c = idx % 16;
                *reinterpret_cast<uint4 *>(vt + (c >> 3) * kPanelBytes + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
            }
          };
          clear(dead0, max(dead0, dead1));
          clear(hi, kBN);
          fence_proxy_async_smem();
          __syncwarp();
        }
      }
      if (!kWindow && kPaged && lk - j * kBN < kBN) {
        // last tile of the sequence: zero the value columns of tokens >= lk (generic-proxy stores,
        // made visible to the tensor core with a proxy fence)
        const int valid = lk - j * kBN;
        uint8_t *vt = sKV + (i_v % kKvStages) * kStageBytes;
        for (int bi = valid / 16; bi < 8; ++bi) {
          uint8_t *vb = vt + bi * 4096;
          const int first = max(0, valid - bi * 16);
          if (first == 0) {
            for (int idx = lane; idx < 256; idx += 32) reinterpret_cast<uint4 *>(vb)[idx] = make_uint4(0, 0, 0, 0);
          } else {
            for (int d = lane; d < kHD; d += 32)
              for (int tok = first; tok < 16; ++tok)
                *reinterpret_cast<uint16_t *>(vb + d * 32 + ((((tok >> 3) ^ ((d >> 2) & 1))) << 4) + (tok & 7) * 2) = 0;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (!kWindow && !kPaged && lk - j * kBN < kBN) {
        // Packed layout, last tile of the sequence: the rows behind it belong to the next sequence
        // (or were zero-filled past the end of the tensor).  Their probabilities are 0, but 0 x NaN
        // is NaN, so the rows are cleared as the reference's predicated loads clear them
        // (flash_fwd_kernel.h, Clear_OOB_MN).  A token row is 128 B in each panel (two panels; one
        // in a CTA pair, where the other CTA clears its own); the swizzle only permutes bytes
        // inside a row.
        const int valid = lk - j * kBN;
        uint8_t *vt = sKV + (i_v % kKvStages) * kStageBytes;
        constexpr int kPieces = kPair ? 8 : 16;  // 16-byte pieces of a token row held by this CTA
        for (int idx = valid * kPieces + lane; idx < kBN * kPieces; idx += 32) {
          const int r = idx / kPieces, c = idx % kPieces;
          *reinterpret_cast<uint4 *>(vt + (c >> 3) * kPanelBytes + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (j < nt0) {
        if (!wait_p(0, j)) break;
        issue_pv(0, i_v, j == 0, j == nt0 - 1, ch);
      }
      if (j + 1 < nt0) {
        if (!wait_kv(i_kn)) break;
        issue_s(0, i_kn, ch_next);
      }
      if (j < nt1) {
        if (!wait_p(1, j)) break;
        issue_pv(1, i_v, j == 0, j == nt1 - 1, ch);
      }
      release(i_v);
      if (j + 1 < nt1) {
        if (!wait_kv(i_kn)) break;
        issue_s(1, i_kn, ch_next);
      }
      if (j + 1 < nmax) release(i_kn);
      ch = ch_next;
    }
    if (!ok && lane == 0) sh->aborted = 1;
  } else {
    // ---------------------------------------------------------------- softmax / epilogue -----
    const int t = warp >> 2;            // tile of this warpgroup
    const int quad = warp & 3;          // TMEM lane quadrant this warp may access
    const int wtid = tid - t * 128;     // thread index inside the warpgroup
    const TileInfo T = tiles[t];
    uint8_t *sQt = sQ + t * kTileBytes;
    const int row = quad * 32 + lane;
    const int qr = T.m0 + row;
    int lim_row = lk;
    if (p.causal) lim_row = min(lk, qr + 1 + lk - lq);
    // windowed variant: the row sees [lo_row, lim_row) and [0, sinks); sees = it is a row and sees something
    const int lo_row = kWindow ? max(0, qr + 1 + lk - lq - min(p.window, lk)) : 0;
    const bool sees = row < T.rows && lim_row > 0;
    if (kWindow && !sees) lim_row = 0;  // rows of other sequences behind this one's last have no columns
    const uint32_t t_s = tmem_base + t * 128 + ((uint32_t)(quad * 32) << 16);
    const uint32_t t_o = tmem_base + kOCol + t * 128 + ((uint32_t)(quad * 32) << 16);
    const float sc = p.scale_log2e;
    float m_used = -INFINITY, m_next = -INFINITY, l_sum = 0.f;
    bool ok = true, pending = false;

    // Windowed variant of the loop body below: the probabilities of the tile at key n0, visit j.  Whole
    // tiles take the same single pass against the running reference; where a row has none yet, or some
    // chunks hold no column that any row of the CTA sees (the diagonal, the sinks), the maximum comes first and
    // only the 32-column chunks that some row of the warp sees are gone over.
    auto window_tile = [&](int j, int n0, int c0, int c1, bool single_pass, bool full) {
      if (single_pass) {
        uint32_t pk[64];
        uint32_t ra[32], rb[32];
        uint64_t acc = pack_f32x2(0.f, 0.f);
        const float ref = m_used == -INFINITY ? 0.f : m_used;
        const uint64_t sc2 = pack_f32x2(sc, sc), nm2 = pack_f32x2(-ref, -ref);
        tmem_ld32(t_s, ra);
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          tmem_wait_ld();
          uint32_t(&cur)[32] = (c4 & 1) ? rb : ra;
          uint32_t(&nxt)[32] = (c4 & 1) ? ra : rb;
          if (c4 < 3) tmem_ld32(t_s + 32 * (c4 + 1), nxt);
          if (full) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float x0, x1;
              unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(cur[i]), __uint_as_float(cur[i + 1])), sc2, nm2), x0, x1);
              const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
              acc = add_f32x2(acc, pack_f32x2(p0, p1));
              pk[16 * c4 + (i >> 1)] = Half16<T16>::pack(p0, p1);
            }
          } else {
            const uint32_t vis = visible_bits(n0 + 32 * c4, lo_row, lim_row, win.sinks);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float x0, x1;
              unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(cur[i]), __uint_as_float(cur[i + 1])), sc2, nm2), x0, x1);
              const float p0 = fast_exp2((vis >> i) & 1u ? x0 : -INFINITY);
              const float p1 = fast_exp2((vis >> (i + 1)) & 1u ? x1 : -INFINITY);
              acc = add_f32x2(acc, pack_f32x2(p0, p1));
              pk[16 * c4 + (i >> 1)] = Half16<T16>::pack(p0, p1);
            }
          }
        }
        float a0, a1;
        unpack_f32x2(acc, a0, a1);
        const float l_tile = a0 + a1;
        if (!__any_sync(0xffffffffu, !(l_tile < kDanger))) {
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4)
            tmem_st16(t_s + 16 * c4, *reinterpret_cast<uint32_t(*)[16]>(&pk[16 * c4]));
          l_sum += l_tile;
          if (l_tile > kRescaleSum) {
            pending = true;
            m_next = m_used + __log2f(l_tile);
          }
          return;
        }
      }
      uint32_t r[32];
      float mx = -INFINITY;
#pragma unroll 1
      for (int c4 = c0; c4 < c1; ++c4) {
        const uint32_t vis = visible_bits(n0 + 32 * c4, lo_row, lim_row, win.sinks);
        if (!__any_sync(0xffffffffu, vis != 0u)) continue;
        tmem_ld32(t_s + 32 * c4, r);
        tmem_wait_ld();
        if (vis == ~0u) {
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(r[i]));
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if ((vis >> i) & 1u) mx = fmaxf(mx, __uint_as_float(r[i]));
        }
      }
      mx *= sc;  // scale > 0 keeps the order
      if (j == 0) {
        m_used = mx;
      } else {
        const bool need = mx > m_used + kRescaleThreshold;
        if (__any_sync(0xffffffffu, need)) {
          float alpha = 1.f;
          if (need) {
            alpha = fast_exp2(m_used - mx);  // 0 when nothing was visible so far
            m_used = mx;
            l_sum *= alpha;
          }
#pragma unroll 1
          for (int c4 = 0; c4 < 4; ++c4) {
            tmem_ld32(t_o + 32 * c4, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st32(t_o + 32 * c4, r);
          }
          tmem_wait_st();
        }
      }
      const float base = m_used == -INFINITY ? 0.f : m_used;
      const uint64_t sc2 = pack_f32x2(sc, sc), nb2 = pack_f32x2(-base, -base);
      uint64_t acc = pack_f32x2(0.f, 0.f);
#pragma unroll 1
      for (int c4 = c0; c4 < c1; ++c4) {  // ascending: P of a chunk lands on scores already read
        const uint32_t vis = visible_bits(n0 + 32 * c4, lo_row, lim_row, win.sinks);
        uint32_t out[16];
        if (__any_sync(0xffffffffu, vis != 0u)) {
          tmem_ld32(t_s + 32 * c4, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), sc2, nb2), x0, x1);
            const float p0 = fast_exp2((vis >> i) & 1u ? x0 : -INFINITY);
            const float p1 = fast_exp2((vis >> (i + 1)) & 1u ? x1 : -INFINITY);
            acc = add_f32x2(acc, pack_f32x2(p0, p1));
            out[i >> 1] = Half16<T16>::pack(p0, p1);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) out[i] = 0u;
        }
        tmem_st16(t_s + 16 * c4, out);
      }
      float a0, a1;
      unpack_f32x2(acc, a0, a1);
      l_sum += a0 + a1;
    };

    for (int j = 0; j < T.n_tiles; ++j) {
      const int n0 = tile_of(j) * kBN;
      int c0 = 0, c1 = 0;
      bool single_pass = false, full = false;
      if constexpr (kWindow) {  // all that does not depend on the scores, while they are computed
        win.chunks(j, c0, c1);
        single_pass = c1 - c0 == kBN / 32 && !__any_sync(0xffffffffu, sees && m_used == -INFINITY);
        full = n0 + kBN <= lim_row && (n0 >= lo_row || n0 + kBN <= win.sinks);
      }
      ok = mbar_wait_abortable(&sh->s_full[t], (uint32_t)j & 1u, p.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      // A rescale that the previous tile found necessary but left for now: the previous P V has
      // completed (s_full of this tile is committed after it), so O can be touched.
      if (__any_sync(0xffffffffu, pending)) {
        float alpha = 1.f;
        if (pending) {
          alpha = fast_exp2(m_used - m_next);
          m_used = m_next;
          l_sum *= alpha;
          pending = false;
        }
        uint32_t o[32];
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          tmem_ld32(t_o + 32 * c4, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(t_o + 32 * c4, o);
        }
        tmem_wait_st();
      }

      if constexpr (kWindow) {
        window_tile(j, n0, c0, c1, single_pass, full);
      } else {
      const bool full_tile = n0 + kBN <= lim_row;
      // rows that have not seen a single column so far have no reference yet: exact path, except on
      // the first tile, which takes its reference from its own first 32 columns (below)
      bool exact_path = (j > 0) && __any_sync(0xffffffffu, m_used == -INFINITY);
      if (!exact_path) {
        // ---- single pass against the running reference m_used --------------------------------
        // P is computed for the whole row in registers while S is still intact; if some score
        // left the reference so far behind that the row sum nears the end of the fp32 range the tile
        // is redone exactly; if the row sum shows a score 2^8 above the reference (see below), the
        // reference moves after this tile's P V (pending).
        uint32_t pk[64];
        uint32_t ra[32], rb[32];
        float l0 = 0.f, l1 = 0.f;
        uint64_t acc2 = pack_f32x2(0.f, 0.f);
        tmem_ld32(t_s, ra);
        if (j == 0) {
          // First tile: the reference is the largest visible score among the first 32 columns (the
          // visible columns of a row are a prefix, so a row that sees nothing here sees nothing in
          // the tile).  If the rest of the tile lies far above it, the row sum says so as usual.
          tmem_wait_ld();
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i < lim_row) mx = fmaxf(mx, __uint_as_float(ra[i]));
          m_used = mx * sc;  // scale > 0 keeps the order
        }
        const float ref = (m_used == -INFINITY) ? 0.f : m_used;
        const uint64_t sc2 = pack_f32x2(sc, sc), nm2 = pack_f32x2(-ref, -ref);
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          tmem_wait_ld();
          uint32_t(&cur)[32] = (c4 & 1) ? rb : ra;
          uint32_t(&nxt)[32] = (c4 & 1) ? ra : rb;
          if (c4 < 3) tmem_ld32(t_s + 32 * (c4 + 1), nxt);
          if (full_tile) {
            // packed fp32 pairs: one FMA and one add per two scores
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t x = fma_f32x2(pack_f32x2(__uint_as_float(cur[i]), __uint_as_float(cur[i + 1])), sc2, nm2);
              float x0, x1;
              unpack_f32x2(x, x0, x1);
              const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
              acc2 = add_f32x2(acc2, pack_f32x2(p0, p1));
              pk[16 * c4 + (i >> 1)] = Half16<T16>::pack(p0, p1);
            }
          } else {
            const int cb = n0 + 32 * c4;
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t x = fma_f32x2(pack_f32x2(__uint_as_float(cur[i]), __uint_as_float(cur[i + 1])), sc2, nm2);
              float x0, x1;
              unpack_f32x2(x, x0, x1);
              const float p0 = fast_exp2((cb + i < lim_row) ? x0 : -INFINITY);
              const float p1 = fast_exp2((cb + i + 1 < lim_row) ? x1 : -INFINITY);
              acc2 = add_f32x2(acc2, pack_f32x2(p0, p1));
              pk[16 * c4 + (i >> 1)] = Half16<T16>::pack(p0, p1);
            }
          }
        }
        // The tile's row sum tells whether the reference is still good: every score at or below it
        // gives a sum of at most 128, one score 2^8 above it a sum above 256, and a sum that left
        // the fp32 range (or is NaN) means the tile has to be redone against its exact maximum.
        {
          float a0, a1;
          unpack_f32x2(acc2, a0, a1);
          l0 += a0;
          l1 += a1;
        }
        const float l_tile = l0 + l1;
        if (__any_sync(0xffffffffu, !(l_tile < kDanger))) {
          exact_path = true;  // S is untouched: redo the tile with an exact maximum
        } else {
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4)
            tmem_st16(t_s + 16 * c4, *reinterpret_cast<uint32_t(*)[16]>(&pk[16 * c4]));
          l_sum += l_tile;
          if (l_tile > kRescaleSum) {
            // log2 of the sum bounds the largest score from above (by at most 7): a reference a few
            // powers of two above the maximum costs bf16 and fp32 nothing
            pending = true;
            m_next = m_used + __log2f(l_tile);
          }
        }
      }
      if (exact_path) {
        uint32_t r[32];
        // pass 1: row max of the raw scores over visible columns
        float mx = -INFINITY;
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          tmem_ld32(t_s + 32 * c4, r);
          tmem_wait_ld();
          const int cb = n0 + 32 * c4;
          if (cb + 32 <= lim_row) {
#pragma unroll
            for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(r[i]));
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (cb + i < lim_row) mx = fmaxf(mx, __uint_as_float(r[i]));
          }
        }
        mx *= sc;  // scale > 0, so the order is preserved

        // immediate rescale of the running output
        if (j == 0) {
          m_used = mx;
        } else {
          const bool need = mx > m_used + kRescaleThreshold;
          if (__any_sync(0xffffffffu, need)) {
            float alpha = 1.f;
            if (need) {
              alpha = fast_exp2(m_used - mx);  // 0 when nothing was visible so far
              m_used = mx;
              l_sum *= alpha;
            }
#pragma unroll
            for (int c4 = 0; c4 < 4; ++c4) {
              tmem_ld32(t_o + 32 * c4, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
              tmem_st32(t_o + 32 * c4, r);
            }
            tmem_wait_st();
          }
        }
        const float base = (m_used == -INFINITY) ? 0.f : m_used;

        // pass 2: p = exp2(s * scale - base), row sum, bf16 P over the S columns
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          tmem_ld32(t_s + 32 * c4, r);
          tmem_wait_ld();
          const int cb = n0 + 32 * c4;
          uint32_t pk[16];
          if (cb + 32 <= lim_row) {
            const uint64_t sc2 = pack_f32x2(sc, sc), nb2 = pack_f32x2(-base, -base);
            uint64_t acc2 = pack_f32x2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float x0, x1;
              unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), sc2, nb2), x0, x1);
              const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
              acc2 = add_f32x2(acc2, pack_f32x2(p0, p1));
              pk[i >> 1] = Half16<T16>::pack(p0, p1);
            }
            float a0, a1;
            unpack_f32x2(acc2, a0, a1);
            l_sum += a0 + a1;
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float p0 = (cb + i < lim_row) ? fast_exp2(fmaf(__uint_as_float(r[i]), sc, -base)) : 0.f;
              const float p1 = (cb + i + 1 < lim_row) ? fast_exp2(fmaf(__uint_as_float(r[i + 1]), sc, -base)) : 0.f;
              l_sum += p0 + p1;
              pk[i >> 1] = Half16<T16>::pack(p0, p1);
            }
          }
          tmem_st16(t_s + 16 * c4, pk);
        }
      }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (kPair && !leader) mbar_arrive_cluster(&sh->p_ready[t], 0);  // the leader issues this CTA's P V too
        else mbar_arrive(&sh->p_ready[t]);
      }
    }


    if (T.n_tiles == 0) ok = false;
    if (ok) {
      ok = mbar_wait_abortable(&sh->o_full[t], 0, p.status);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok) {
      tc_fence_after();
      const float inv = l_sum > 0.f ? __fdividef(1.f, l_sum) : 0.f;
      // staging tile over the Q buffer in the layout Q arrived in: two panels of [128 rows][64 bf16]
      // with the 128-byte swizzle (16-byte chunk c of a row sits at chunk c ^ (row & 7)), so that a
      // TMA store can take it as it is
      uint8_t *stage = sQt;
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        uint32_t r[32];
        tmem_ld32(t_o + 32 * c4, r);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 v;
          const int f = kPaged ? q : 0;  // cache V: see make_cache_tmap
          v.x = Half16<T16>::pack(__uint_as_float(r[8 * q + (0 ^ f)]) * inv, __uint_as_float(r[8 * q + (1 ^ f)]) * inv);
          v.y = Half16<T16>::pack(__uint_as_float(r[8 * q + (2 ^ f)]) * inv, __uint_as_float(r[8 * q + (3 ^ f)]) * inv);
          v.z = Half16<T16>::pack(__uint_as_float(r[8 * q + (4 ^ f)]) * inv, __uint_as_float(r[8 * q + (5 ^ f)]) * inv);
          v.w = Half16<T16>::pack(__uint_as_float(r[8 * q + (6 ^ f)]) * inv, __uint_as_float(r[8 * q + (7 ^ f)]) * inv);
          const int chunk = 4 * c4 + q;
          *reinterpret_cast<uint4 *>(stage + (chunk >> 3) * kPanelBytes + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) = v;
        }
      }
      // the four warps meet on an mbarrier (bounded wait) rather than a hardware barrier, so a
      // warp that unwound early cannot leave the others waiting forever
      fence_proxy_async_smem();  // a TMA store may read what this thread just wrote
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->staged[t]);
      ok = __all_sync(0xffffffffu, mbar_wait(&sh->staged[t], 0, p.status));
    }
    // A tile whose 128 rows all belong to this sequence, or whose sequence ends exactly where the
    // tensor ends (the copy is clipped there), goes out as two TMA stores; any other tile must not
    // touch rows that are not its own and is written row by row.
    const bool whole = p.tma_store && (T.rows == kBM || q0 + lq == p.total_q);
    if (ok && whole) {
      if (wtid == 0) {
        for (int w = 0; w < p.world; ++w) {  // peers' buffers are plain global addresses to the engine
          tma_store_3d(&tmap_o.m[w], sQt, 0, p.out_head0 + T.h, q0 + T.m0);
          tma_store_3d(&tmap_o.m[w], sQt + kPanelBytes, 64, p.out_head0 + T.h, q0 + T.m0);
        }
        // shared memory must outlive the engine's reads; with peers the writes themselves are
        // awaited too, so that they are done when this grid is and the barrier kernel may signal
        if (p.world > 1) tma_store_commit_and_wait_all(); else tma_store_commit_and_wait_read();
      }
    } else if (ok) {
      const uint8_t *stage = sQt;
      const int64_t obase = (int64_t)(q0 + T.m0) * p.o_tok_stride + (int64_t)(p.out_head0 + T.h) * p.o_head_stride;
#pragma unroll 4
      for (int it = 0; it < 16; ++it) {
        const int rr = it * 8 + (wtid >> 4), chunk = wtid & 15;
        if (rr < T.rows) {
          const uint4 v = *reinterpret_cast<const uint4 *>(stage + (chunk >> 3) * kPanelBytes + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4));
          const int64_t off = obase + (int64_t)rr * p.o_tok_stride + chunk * 8;
          for (int w = 0; w < p.world; ++w) *reinterpret_cast<uint4 *>(p.out[w] + off) = v;
        }
      }
    }
  }

  // ---- teardown ------------------------------------------------------------------------------
  tc_fence_before();
  __syncwarp();
  if (warp == Cfg::kMmaWarp && sh->aborted) {
    // bounded wait for whatever the tensor pipe still owes before the columns are released (only
    // the issuing CTA sets the flag)
    if (lane == 0) tc_commit(&sh->drain);
    __syncwarp();
    mbar_wait(&sh->drain, 0, p.status);
  }
  // pairs: neither CTA may leave (its shared and tensor memory are operands of the other's MMAs)
  // before both are through
  if (kPair) cluster_sync_all();
  else __syncthreads();
  if (warp == Cfg::kMmaWarp) {
    if (kPair) tmem_dealloc_pair(tmem_base, kTmemCols);
    else tmem_dealloc(tmem_base, kTmemCols);
  }
  leave();
}

// ---- host side -------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (fn == nullptr) {
    void *sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) ==
            cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(sym);
  }
  return fn;
}

// Generic tiled map over 16-bit data (declared bf16; f16 tensors use the same maps, since the engine moves
// the elements as they are and fills with zero): dims/box innermost first, strides (bytes) for dims 1..rank-1.
static char *make_tmap_nd(const char *fn, CUtensorMap *map, const void *base, int rank,
                          const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
                          CUtensorMapSwizzle swizzle) {
  EncodeTiledFn enc = encode_fn();
  AICI_CHECK(enc != nullptr, "%s: cuTensorMapEncodeTiled is not available from the driver", fn);
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void *>(base), dims,
                   strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  AICI_CHECK(r == CUDA_SUCCESS, "%s: cuTensorMapEncodeTiled failed with code %d", fn, (int)r);
  return nullptr;
}

// Encoded maps are kept in a small table keyed by everything that went into them (base address,
// extents, strides, kind), guarded by a mutex: a serving loop calls with the same buffers step after
// step, and an encode through the driver costs about as much as the launch itself.  A map depends
// on nothing but its key, so an entry can never be stale; the oldest entry is overwritten when the
// table is full.  Windowed calls (keep = false) encode theirs anew: it is 0.1 to 0.7 us of a host
// call of 16 to 18.
struct TmapKey {
  const void *base;
  int64_t a, b, c, d;
  int kind;
  bool operator==(const TmapKey &o) const {
    return base == o.base && a == o.a && b == o.b && c == o.c && d == o.d && kind == o.kind;
  }
};
constexpr int kTmapCacheSize = 64;
struct TmapCache {
  std::mutex mu;
  TmapKey keys[kTmapCacheSize];
  CUtensorMap maps[kTmapCacheSize];
  int used = 0, next = 0;
  bool find(const TmapKey &k, CUtensorMap *out) {
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < used; ++i)
      if (keys[i] == k) {
        *out = maps[i];
        return true;
      }
    return false;
  }
  void put(const TmapKey &k, const CUtensorMap &m) {
    std::lock_guard<std::mutex> lock(mu);
    const int i = used < kTmapCacheSize ? used++ : (next++ % kTmapCacheSize);
    keys[i] = k;
    maps[i] = m;
  }
};
static TmapCache g_tmap_cache;

// [tokens, heads, 128] bf16 with element strides -> 3-D map, box = 64 (d) x 1 (head) x box_rows (tokens;
// 128, or 64 for the key half-tiles of the CTA-pair shape).
static char *make_tmap(const char *fn, CUtensorMap *map, const void *base, int64_t tokens, int heads,
                       int64_t tok_stride, int64_t head_stride, bool keep, int box_rows = kBM) {
  const TmapKey key = {base, tokens, heads, tok_stride, head_stride, box_rows == kBM ? 0 : 3};
  if (keep && g_tmap_cache.find(key, map)) return nullptr;
  cuuint64_t dims[3] = {(cuuint64_t)kHD, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)tok_stride * 2};
  cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows};
  if (char *e = make_tmap_nd(fn, map, base, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  if (keep) g_tmap_cache.put(key, *map);
  return nullptr;
}

// Paged caches: kind 1 = key cache (5-D), kind 2 = value cache (4-D), one block per box.
// What a copy costs the engine is some 20 clk and its rows of 128 bytes: with 16 key and 8 value copies a tile
// 8 chunks of 512, window 1024, take 121.8 us, with 8 and 8 119.2, and packed keys (4 copies) 110.
static char *make_cache_tmap(const char *fn, CUtensorMap *map, const void *base, bool value,
                             int num_kv_heads, int64_t num_blocks, int64_t kv_head_stride,
                             int64_t kv_block_stride, bool keep) {
  const TmapKey key = {base, num_kv_heads, num_blocks, kv_head_stride, kv_block_stride, value ? 2 : 1};
  if (keep && g_tmap_cache.find(key, map)) return nullptr;
  if (!value) {
    // [blk][h][c = 16][tok = 16][e = 8], a chunk taken as two halves of 8 tokens x 8 elements = 128
    // contiguous bytes (as rows of 16 bytes the engine moves it far slower); the map's order is chunk, then
    // half, so that one copy of a block leaves its halves one behind the other
    cuuint64_t dims[5] = {64, 16, 2, (cuuint64_t)num_kv_heads, (cuuint64_t)num_blocks};
    cuuint64_t str[4] = {256, 128, (cuuint64_t)kv_head_stride * 2, (cuuint64_t)kv_block_stride * 2};
    cuuint32_t box[5] = {64, 16, 2, 1, 1};
    if (char *e = make_tmap_nd(fn, map, base, 5, dims, str, box, CU_TENSOR_MAP_SWIZZLE_NONE)) return e;
  } else {
    // [blk][h][d = 128][tok = 16]: box = one block, four d to a row of 128 bytes (as rows of 32 bytes the engine
    // moves it far slower).  The MMA reads it as rows of 32 bytes with the 32-byte swizzle, address bit 4 ^= bit
    // 7; the 128-byte swizzle of the copy does that and bits 5, 6 ^= bits 8, 9 besides, which only reorders the
    // d in groups of four: column d of the output arrives as column d ^ (d / 8 % 4), and the epilogue knows.
    cuuint64_t dims[4] = {64, 32, (cuuint64_t)num_kv_heads, (cuuint64_t)num_blocks};
    cuuint64_t str[3] = {128, (cuuint64_t)kv_head_stride * 2, (cuuint64_t)kv_block_stride * 2};
    cuuint32_t box[4] = {64, 32, 1, 1};
    if (char *e = make_tmap_nd(fn, map, base, 4, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  }
  if (keep) g_tmap_cache.put(key, *map);
  return nullptr;
}

// Sequences up to this many keys take the one-tile shape (two CTAs per SM), longer ones the
// two-tile shape: with few key tiles per query tile a CTA's fixed cost (fill and drain, about as long
// as three key tiles) is what two resident CTAs hide; with many, sharing each K/V tile between two
// query tiles (half the shared-memory traffic) is worth more.
#ifndef AICI_PREFILL_ONE_TILE_MAX_K
#define AICI_PREFILL_ONE_TILE_MAX_K 2048
#endif

template <bool kPaged, int kShape, bool kWindow = false, typename T16 = __nv_bfloat16>
static char *launch_prefill_shape(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv,
                                  const OutMaps &to, PrefillParams &p, int num_heads, int batch,
                                  int max_seqlen_q, cudaStream_t stream) {
  using Cfg = PrefillCfg<kShape>;
  static OncePerDevice once;
  if (char *e = once.run([]() -> char * {
        AICI_CUDA(cudaFuncSetAttribute(varlen_prefill_kernel<kPaged, kShape, kWindow, T16>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes));
        return nullptr;
      }))
    return e;
  const int mblocks = (max_seqlen_q + kBM - 1) / kBM;
  dim3 grid;
  if (kWindow) {
    const int heads = Cfg::kTiles == 1 ? num_heads : num_heads / 2;
    const int64_t room = (int64_t)p.total_q / kBM + batch, most = (int64_t)batch * mblocks;
    p.pair_heads = Cfg::kTiles == 1 ? 0 : 1;
    p.grid_heads = most > room || p.longer_than > 0 ? heads : 0;
    AICI_CHECK(room * heads < (1ll << 31), "prefill: too many tiles for one call");
    grid = p.grid_heads > 0 ? dim3((unsigned)(room * heads)) : dim3(heads, batch, mblocks);
  } else if (Cfg::kTiles == 1) {
    grid = dim3(num_heads, batch, mblocks);
  } else {
    // two tiles per CTA: two heads of one kv group when the group is even (always so for CTA pairs,
    // whose two CTAs are neighbours in x: four heads of one kv head), else two row tiles
    p.pair_heads = (Cfg::kPair || p.group % 2 == 0) ? 1 : 0;
    grid = dim3(p.pair_heads ? num_heads / 2 : num_heads, batch, p.pair_heads ? mblocks : (mblocks + 1) / 2);
  }
  AICI_CHECK(grid.y <= 65535 && grid.z <= 65535, "prefill: batch and row tiles must fit a grid dimension");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (kWindow) {
    attr[0] = dependent_launch();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  if (Cfg::kPair) {
    // clusters of two CTAs along x: the pair works on four query heads of one kv head
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  cudaError_t le = cudaLaunchKernelEx(&cfg, varlen_prefill_kernel<kPaged, kShape, kWindow, T16>, tq, tk, tv,
                                      OutMapsOf<kWindow>::of(to), p);
  if (le != cudaSuccess) {
    cudaGetLastError();
    int clusters = -1, max_size = -1;
    cudaError_t e1 = cudaSuccess, e2 = cudaSuccess;
    if (Cfg::kPair) {
      e1 = cudaOccupancyMaxActiveClusters(&clusters, varlen_prefill_kernel<kPaged, kShape, kWindow, T16>, &cfg);
      cudaLaunchConfig_t probe = cfg;
      probe.attrs = nullptr;
      probe.numAttrs = 0;
      e2 = cudaOccupancyMaxPotentialClusterSize(&max_size, varlen_prefill_kernel<kPaged, kShape, kWindow, T16>, &probe);
      cudaGetLastError();
    }
    return err("prefill launch (shape %d, grid %u x %u x %u, %d threads, %d bytes of shared memory) failed: %s "
               "[active clusters %d (%s), largest cluster %d (%s)]",
               kShape, grid.x, grid.y, grid.z, Cfg::kThreads, Cfg::kSmemBytes, cudaGetErrorString(le), clusters,
               cudaGetErrorString(e1), max_size, cudaGetErrorString(e2));
  }
  return nullptr;
}

// Windowed variant.  A query tile visits window / 128 + 1 key tiles and the sinks' tiles: by that length
// and not the sequence's a call takes shape 1 or 2; two tiles of a CTA are two heads of one kv head.
// A paged tile is 16 copies where a packed one is 4, and the one-tile shape's two stages hide less of them, so
// sharing tiles between two query tiles pays earlier.  In us one-tile and two-tile, 32/8 heads: paged, 4 x 4096,
// window 640: 283 and 305, 1024: 348 and 366, 1280: 386 and 403, 1536: 421 and 437, 2048: 501 and 492; 8 chunks of
// 512 on 7680 cached: 95.6 and 96.8, 122.8 and 122.2, 142 and 139, 162 and 156, 200 and 190.  Packed, 4 x 4096,
// 2048: 468 and 482, 2560: 525 and 524, 4096: 603 and 578; chunks, 1024: 123 and 124, 2048: 195 and 192, 2560: 230
// and 223, 4096: 334 and 320.
template <bool kPaged, typename T16>
static char *launch_prefill_window(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv,
                                   const OutMaps &to, PrefillParams &p, int num_heads, int batch, int max_seqlen_q,
                                   int max_seqlen_k, cudaStream_t stream) {
  p.pair_heads = 0;
  const int64_t keys = (int64_t)p.window + p.sinks, most = kPaged ? 1280 : 2560;
  if (p.group % 2 != 0 || (keys < max_seqlen_k ? keys : max_seqlen_k) <= most)
    return launch_prefill_shape<kPaged, 1, true, T16>(tq, tk, tv, to, p, num_heads, batch, max_seqlen_q, stream);
  return launch_prefill_shape<kPaged, 2, true, T16>(tq, tk, tv, to, p, num_heads, batch, max_seqlen_q, stream);
}

// Which shape a call takes.  `forced` = 0: by sequence length -- shape 1 up to
// AICI_PREFILL_ONE_TILE_MAX_K keys, shape 2 above; the CTA-pair shape is never chosen by itself (on
// the long-context benchmark it runs at 0.83 of shape 2: what it saves in shared-memory reads it
// loses to the cross-SM hand-over between the softmax warps and the issuing thread).  forced = 1, 2,
// 3: that shape, for tests and comparisons; 3 needs packed K/V and four query heads per kv head in
// one CTA pair (group a multiple of 4).
static char *pick_shape(const char *fn, int forced, bool paged, int num_heads, int group, int max_seqlen_k,
                        int *shape) {
  AICI_CHECK(forced >= 0 && forced <= 3, "%s: shape must be 0 (automatic), 1, 2 or 3", fn);
  AICI_CHECK(forced != 3 || (!paged && group % 4 == 0 && num_heads % 4 == 0),
             "%s: the CTA-pair shape needs packed keys/values and a group size that is a multiple of 4", fn);
  *shape = forced != 0 ? forced : (max_seqlen_k <= AICI_PREFILL_ONE_TILE_MAX_K ? 1 : 2);
  return nullptr;
}

template <bool kPaged>
static char *launch_prefill(int shape, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv,
                            const OutMaps &to, PrefillParams &p, int num_heads, int batch, int max_seqlen_q,
                            cudaStream_t stream) {
  p.pair_heads = 0;
  if (shape == 1)
    return launch_prefill_shape<kPaged, 1>(tq, tk, tv, to, p, num_heads, batch, max_seqlen_q, stream);
  if constexpr (!kPaged) {
    if (shape == 3)
      return launch_prefill_shape<false, 3>(tq, tk, tv, to, p, num_heads, batch, max_seqlen_q, stream);
  }
  return launch_prefill_shape<kPaged, 2>(tq, tk, tv, to, p, num_heads, batch, max_seqlen_q, stream);
}

}  // namespace aici

using namespace aici;

// What the windowed entry points take besides the arguments of the others.
struct WindowArgs {
  int window, sinks;
};

static char *check_window(const char *fn, const WindowArgs &w, int num_heads, int num_kv_heads, int dtype) {
  AICI_CHECK(dtype == AICI_DTYPE_BF16 || dtype == AICI_DTYPE_F16, "%s: only bf16 and f16 are supported (dtype=%d)", fn,
             dtype);
  AICI_CHECK(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
             "%s: num_heads %d not divisible by num_kv_heads %d", fn, num_heads, num_kv_heads);
  AICI_CHECK(w.window >= 1, "%s: window must be at least 1 (got %d)", fn, w.window);
  AICI_CHECK(w.sinks >= 0, "%s: sinks must not be negative (got %d)", fn, w.sinks);
  return nullptr;
}

static char *mha_varlen_fwd_impl(const char *fn, void *const *outs, int world, int out_head0, const void *q,
                                 const void *k, const void *v,
                                     const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k,
                                     int batch, int total_q, int total_k, int num_heads,
                                     int num_heads_k, int head_size, int max_seqlen_q,
                                     int max_seqlen_k, int64_t q_tok_stride, int64_t q_head_stride,
                                     int64_t k_tok_stride, int64_t k_head_stride,
                                     int64_t v_tok_stride, int64_t v_head_stride,
                                     int64_t o_tok_stride, int64_t o_head_stride,
                                     float softmax_scale, int is_causal, int dtype,
                                     aici_stream_t stream, int forced_shape = 0,
                                     const WindowArgs *win = nullptr) {
  void *out = outs[0];
  for (int w = 1; w < world; ++w)
    AICI_CHECK(outs[w] != nullptr && (uintptr_t)outs[w] % 16 == 0,
               "%s: peer output %d must be non-NULL and 16-byte aligned", fn, w);
  if (win != nullptr) {
    if (char *e = check_window(fn, *win, num_heads, num_heads_k, dtype)) return e;
  }
  AICI_CHECK(win != nullptr || dtype == AICI_DTYPE_BF16, "%s: FlashAttention only support bf16 data type (dtype=%d)", fn,
             dtype);
  AICI_CHECK(batch > 0, "%s: batch size must be positive", fn);
  AICI_CHECK(head_size == kHD, "%s: head_size must be 128 (got %d)", fn, head_size);
  AICI_CHECK(num_heads > 0 && num_heads_k > 0 && num_heads % num_heads_k == 0,
             "%s: Number of heads in key/value must divide number of heads in query", fn);
  AICI_CHECK(total_q >= 0 && total_k >= 0 && max_seqlen_q >= 0 && max_seqlen_k >= 0, "%s: negative size", fn);
  AICI_CHECK(softmax_scale > 0.f, "%s: softmax_scale must be positive", fn);
  AICI_CHECK(batch <= 65535 && num_heads <= 65535, "%s: batch and num_heads must fit a grid dimension", fn);
  if (total_q == 0 || max_seqlen_q == 0) return nullptr;
  if (win != nullptr && max_seqlen_q > total_q) max_seqlen_q = total_q;  // any bound will do
  AICI_CHECK(out && q && cu_seqlens_q && cu_seqlens_k, "%s: NULL pointer", fn);
  AICI_CHECK(total_k == 0 || (k && v), "%s: NULL pointer", fn);
  AICI_CHECK(((uintptr_t)out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 == 0,
             "%s: tensors must be 16-byte aligned", fn);
  if (win != nullptr) {  // a stride over a dimension of one is never used and may be whatever a layout left there
    if (total_q == 1) q_tok_stride = kHD;
    if (num_heads == 1) q_head_stride = kHD;
    if (total_k == 1) k_tok_stride = v_tok_stride = kHD;
    if (num_heads_k == 1) k_head_stride = v_head_stride = kHD;
  }
  const int64_t strides[8] = {q_tok_stride, q_head_stride, k_tok_stride, k_head_stride,
                              v_tok_stride, v_head_stride, o_tok_stride, o_head_stride};
  for (int i = 0; i < 8; ++i)
    AICI_CHECK(strides[i] >= kHD && strides[i] % 8 == 0,
               "%s: token and head strides must be multiples of 8 elements and at least head_size", fn);
  // this rank's heads must fit between two token rows of the output buffers
  AICI_CHECK(o_head_stride > o_tok_stride ||
                 (int64_t)(out_head0 + num_heads - 1) * o_head_stride + kHD <= o_tok_stride,
             "%s: heads [%d, %d) do not fit an output row of %lld elements", fn, out_head0,
             out_head0 + num_heads, (long long)o_tok_stride);
  int shape = 0;
  if (char *e = pick_shape(fn, forced_shape, false, num_heads, num_heads / num_heads_k, max_seqlen_k, &shape)) return e;
  if (char *e = check_on_current_device(fn, "q", q)) return e;
  unsigned int *st = status_ptr();
  AICI_CHECK(st != nullptr, "%s: no CUDA device", fn);

  CUtensorMap tq, tk, tv;
  if (char *e = make_tmap(fn, &tq, q, total_q, num_heads, q_tok_stride, q_head_stride, win == nullptr)) return e;
  // an empty key tensor still needs a valid map; no tile of it is ever requested
  const void *kk = total_k > 0 ? k : q;
  const void *vv = total_k > 0 ? v : q;
  const int64_t tk_rows = total_k > 0 ? total_k : 1;
  // the CTA-pair shape loads key tiles in halves of 64 tokens
  if (char *e = make_tmap(fn, &tk, kk, tk_rows, num_heads_k, k_tok_stride, k_head_stride, win == nullptr,
                          shape == 3 ? 64 : kBM))
    return e;
  if (char *e = make_tmap(fn, &tv, vv, tk_rows, num_heads_k, v_tok_stride, v_head_stride, win == nullptr)) return e;

  PrefillParams p;
  for (int i = 0; i < 8; ++i) p.out[i] = static_cast<__nv_bfloat16 *>(i < world ? outs[i] : nullptr);
  p.world = world;
  p.out_head0 = out_head0;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.o_tok_stride = o_tok_stride;
  p.o_head_stride = o_head_stride;
  p.group = num_heads / num_heads_k;
  p.causal = is_causal ? 1 : 0;
  p.scale_log2e = softmax_scale * 1.4426950408889634f;
  p.status = st;
  p.block_tables = nullptr;
  p.k_lens = nullptr;
  p.max_blocks = 0;
  p.num_blocks = 0;
  p.window = win ? win->window : 0;
  p.sinks = win ? win->sinks : 0;
  p.longer_than = 0;
  p.max_q = max_seqlen_q;
  p.batch = batch;
  p.grid_heads = 0;
  // every output buffer gets a tensor map like the query's; this rank's heads start at out_head0
  OutMaps to = {};
  p.total_q = total_q;
  p.tma_store = 1;
  for (int w = 0; w < world; ++w)  // the kernel reads m[w] for w < world only
    if (char *e = make_tmap(fn, &to.m[w], outs[w], total_q, out_head0 + num_heads, o_tok_stride, o_head_stride,
                            win == nullptr))
      return e;
  if (win != nullptr)
    return with_half_type(dtype, [&](auto t) {
      return launch_prefill_window<false, decltype(t)>(tq, tk, tv, to, p, num_heads, batch, max_seqlen_q, max_seqlen_k,
                                                       static_cast<cudaStream_t>(stream));
    });
  return launch_prefill<false>(shape, tq, tk, tv, to, p, num_heads, batch, max_seqlen_q,
                               static_cast<cudaStream_t>(stream));
}

extern "C" char *aici_mha_varlen_fwd(void *out, const void *q, const void *k, const void *v,
                                     const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k,
                                     int batch, int total_q, int total_k, int num_heads,
                                     int num_heads_k, int head_size, int max_seqlen_q,
                                     int max_seqlen_k, int64_t q_tok_stride, int64_t q_head_stride,
                                     int64_t k_tok_stride, int64_t k_head_stride,
                                     int64_t v_tok_stride, int64_t v_head_stride,
                                     int64_t o_tok_stride, int64_t o_head_stride,
                                     float softmax_scale, int is_causal, int dtype,
                                     aici_stream_t stream) {
  void *outs[1] = {out};
  return mha_varlen_fwd_impl("aici_mha_varlen_fwd", outs, 1, 0, q, k, v, cu_seqlens_q, cu_seqlens_k, batch,
                             total_q, total_k, num_heads, num_heads_k, head_size, max_seqlen_q,
                             max_seqlen_k, q_tok_stride, q_head_stride, k_tok_stride, k_head_stride,
                             v_tok_stride, v_head_stride, o_tok_stride, o_head_stride, softmax_scale,
                             is_causal, dtype, stream);
}

// aici_mha_varlen_fwd with the kernel shape chosen by the caller instead of by sequence length (test
// and benchmark hook): 0 = automatic, 1 = one query tile per CTA and two CTAs per SM, 2 = two query
// tiles per CTA, 3 = shape 2 on CTA pairs with two-SM MMAs (tcgen05 cta_group::2).
extern "C" char *aici_mha_varlen_fwd_shape(void *out, const void *q, const void *k, const void *v,
                                           const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k,
                                           int batch, int total_q, int total_k, int num_heads,
                                           int num_heads_k, int head_size, int max_seqlen_q,
                                           int max_seqlen_k, int64_t q_tok_stride, int64_t q_head_stride,
                                           int64_t k_tok_stride, int64_t k_head_stride,
                                           int64_t v_tok_stride, int64_t v_head_stride,
                                           int64_t o_tok_stride, int64_t o_head_stride,
                                           float softmax_scale, int is_causal, int shape, int dtype,
                                           aici_stream_t stream) {
  void *outs[1] = {out};
  return mha_varlen_fwd_impl("aici_mha_varlen_fwd_shape", outs, 1, 0, q, k, v, cu_seqlens_q, cu_seqlens_k,
                             batch, total_q, total_k, num_heads, num_heads_k, head_size, max_seqlen_q,
                             max_seqlen_k, q_tok_stride, q_head_stride, k_tok_stride, k_head_stride,
                             v_tok_stride, v_head_stride, o_tok_stride, o_head_stride, softmax_scale,
                             is_causal, dtype, stream, shape);
}

// Prefill attention whose epilogue is the head-output gather: each finished output tile is stored
// at head index head0 + h of the [total_q, total_heads, 128] buffer of EVERY rank (plain stores to
// peer-mapped memory over NVLink, pushed tile by tile while later tiles are still computing), so
// the gather hides under the attention math; the ranks only need a barrier before reading.
extern "C" char *aici_mha_varlen_fwd_peers(void *const *outs, int world, int head0, const void *q,
                                           const void *k, const void *v, const int32_t *cu_seqlens_q,
                                           const int32_t *cu_seqlens_k, int batch, int total_q,
                                           int total_k, int num_heads, int num_heads_k, int head_size,
                                           int max_seqlen_q, int max_seqlen_k, int64_t q_tok_stride,
                                           int64_t q_head_stride, int64_t k_tok_stride,
                                           int64_t k_head_stride, int64_t v_tok_stride,
                                           int64_t v_head_stride, int64_t o_tok_stride,
                                           int64_t o_head_stride, float softmax_scale, int is_causal,
                                           int dtype, aici_stream_t stream) {
  const char *fn = "aici_mha_varlen_fwd_peers";
  AICI_CHECK(outs != nullptr && world >= 1 && world <= 8, "%s: world must be 1..8", fn);
  AICI_CHECK(head0 >= 0, "%s: negative head offset", fn);
  return mha_varlen_fwd_impl(fn, outs, world, head0, q, k, v, cu_seqlens_q, cu_seqlens_k, batch, total_q,
                             total_k, num_heads, num_heads_k, head_size, max_seqlen_q, max_seqlen_k,
                             q_tok_stride, q_head_stride, k_tok_stride, k_head_stride, v_tok_stride,
                             v_head_stride, o_tok_stride, o_head_stride, softmax_scale, is_causal, dtype,
                             stream);
}

static char *mha_varlen_paged_fwd_impl(const char *fn, void *out, const void *q, const void *key_cache,
                                       const void *value_cache, const int32_t *cu_seqlens_q,
                                       const int32_t *context_lens, const int32_t *block_tables,
                                       int batch, int total_q, int num_heads, int num_kv_heads,
                                       int head_size, int block_size, int max_seqlen_q,
                                       int max_context_len, int max_num_blocks_per_seq,
                                       int64_t num_blocks, int64_t q_tok_stride,
                                       int64_t q_head_stride, int64_t o_tok_stride,
                                       int64_t o_head_stride, int64_t kv_block_stride,
                                       int64_t kv_head_stride, float softmax_scale, int is_causal,
                                       int dtype, aici_stream_t stream, const WindowArgs *win = nullptr) {
  if (win != nullptr) {
    if (char *e = check_window(fn, *win, num_heads, num_kv_heads, dtype)) return e;
  }
  AICI_CHECK(win != nullptr || dtype == AICI_DTYPE_BF16, "%s: only bf16 is supported (dtype=%d)", fn, dtype);
  AICI_CHECK(batch > 0, "%s: batch size must be positive", fn);
  AICI_CHECK(head_size == kHD, "%s: head_size must be 128 (got %d)", fn, head_size);
  AICI_CHECK(block_size == 16, "%s: block_size must be 16 (got %d)", fn, block_size);
  AICI_CHECK(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
             "%s: Number of heads in key/value must divide number of heads in query", fn);
  AICI_CHECK(total_q >= 0 && max_seqlen_q >= 0 && max_context_len >= 0 && max_num_blocks_per_seq >= 0,
             "%s: negative size", fn);
  AICI_CHECK(softmax_scale > 0.f, "%s: softmax_scale must be positive", fn);
  AICI_CHECK(batch <= 65535 && num_heads <= 65535, "%s: batch and num_heads must fit a grid dimension", fn);
  if (total_q == 0 || max_seqlen_q == 0) return nullptr;
  if (win != nullptr && max_seqlen_q > total_q) max_seqlen_q = total_q;  // any bound will do
  AICI_CHECK(out && q && key_cache && value_cache && cu_seqlens_q && context_lens && block_tables,
             "%s: NULL pointer", fn);
  AICI_CHECK(num_blocks > 0, "%s: num_blocks must be positive", fn);
  AICI_CHECK(((uintptr_t)out | (uintptr_t)q | (uintptr_t)key_cache | (uintptr_t)value_cache) % 16 == 0,
             "%s: tensors must be 16-byte aligned", fn);
  if (win != nullptr && total_q == 1) q_tok_stride = kHD;  // never used
  if (win != nullptr && num_heads == 1) q_head_stride = kHD;
  const int64_t strides[4] = {q_tok_stride, q_head_stride, o_tok_stride, o_head_stride};
  for (int i = 0; i < 4; ++i)
    AICI_CHECK(strides[i] >= kHD && strides[i] % 8 == 0,
               "%s: token and head strides must be multiples of 8 elements and at least head_size", fn);
  AICI_CHECK(kv_head_stride == kHD * 16 && kv_block_stride % 8 == 0 &&
                 kv_block_stride >= (int64_t)num_kv_heads * kHD * 16,
             "%s: cache must be [blocks, kv_heads, 128/8, 16, 8] with contiguous head tiles", fn);
  if (char *e = check_on_current_device(fn, "q", q)) return e;
  unsigned int *st = status_ptr();
  AICI_CHECK(st != nullptr, "%s: no CUDA device", fn);

  const bool all_short = win != nullptr && window_chunk_takes(batch, num_heads, num_kv_heads, max_seqlen_q);
  const bool some_short = win != nullptr && !all_short && window_chunk_mixed(batch, total_q, max_seqlen_q);
  if (all_short || some_short) {
    const WindowChunk c = {out, q, key_cache, value_cache, cu_seqlens_q, context_lens, block_tables, batch, total_q,
                           num_heads, num_kv_heads, all_short ? max_seqlen_q : kWindowChunkTokens, max_context_len,
                           max_num_blocks_per_seq, win->window, win->sinks, num_blocks, q_tok_stride, q_head_stride,
                           o_tok_stride, o_head_stride, kv_block_stride, softmax_scale, st, !all_short};
    char *e = launch_window_chunk(c, dtype, static_cast<cudaStream_t>(stream));
    if (e != nullptr || all_short) return e;
  }

  CUtensorMap tq, tk, tv;
  if (char *e = make_tmap(fn, &tq, q, total_q, num_heads, q_tok_stride, q_head_stride, win == nullptr)) return e;
  if (char *e = make_cache_tmap(fn, &tk, key_cache, false, num_kv_heads, num_blocks, kv_head_stride, kv_block_stride,
                               win == nullptr))
    return e;
  if (char *e = make_cache_tmap(fn, &tv, value_cache, true, num_kv_heads, num_blocks, kv_head_stride, kv_block_stride,
                               win == nullptr))
    return e;
  PrefillParams p;
  for (int i = 0; i < 8; ++i) p.out[i] = i == 0 ? static_cast<__nv_bfloat16 *>(out) : nullptr;
  p.world = 1;
  p.out_head0 = 0;
  p.cu_q = cu_seqlens_q;
  p.cu_k = nullptr;
  p.o_tok_stride = o_tok_stride;
  p.o_head_stride = o_head_stride;
  p.group = num_heads / num_kv_heads;
  p.causal = is_causal ? 1 : 0;
  p.scale_log2e = softmax_scale * 1.4426950408889634f;
  p.status = st;
  p.block_tables = block_tables;
  p.k_lens = context_lens;
  p.max_blocks = max_num_blocks_per_seq;
  p.num_blocks = num_blocks;
  p.window = win ? win->window : 0;
  p.sinks = win ? win->sinks : 0;
  p.longer_than = some_short ? kWindowChunkTokens : 0;
  p.max_q = max_seqlen_q;
  p.batch = batch;
  p.grid_heads = 0;
  OutMaps to = {};
  p.total_q = total_q;
  p.tma_store = 1;
  if (char *e = make_tmap(fn, &to.m[0], out, total_q, num_heads, o_tok_stride, o_head_stride, win == nullptr)) return e;
  if (win != nullptr)
    return with_half_type(dtype, [&](auto t) {
      return launch_prefill_window<true, decltype(t)>(tq, tk, tv, to, p, num_heads, batch, max_seqlen_q, max_context_len,
                                                      static_cast<cudaStream_t>(stream));
    });
  int shape = 0;
  if (char *e = pick_shape(fn, 0, true, num_heads, num_heads / num_kv_heads, max_context_len, &shape)) return e;
  return launch_prefill<true>(shape, tq, tk, tv, to, p, num_heads, batch, max_seqlen_q,
                              static_cast<cudaStream_t>(stream));
}

extern "C" char *aici_mha_varlen_paged_fwd(void *out, const void *q, const void *key_cache,
                                           const void *value_cache, const int32_t *cu_seqlens_q,
                                           const int32_t *context_lens, const int32_t *block_tables,
                                           int batch, int total_q, int num_heads, int num_kv_heads,
                                           int head_size, int block_size, int max_seqlen_q,
                                           int max_context_len, int max_num_blocks_per_seq,
                                           int64_t num_blocks, int64_t q_tok_stride,
                                           int64_t q_head_stride, int64_t o_tok_stride,
                                           int64_t o_head_stride, int64_t kv_block_stride,
                                           int64_t kv_head_stride, float softmax_scale, int is_causal,
                                           int dtype, aici_stream_t stream) {
  return mha_varlen_paged_fwd_impl("aici_mha_varlen_paged_fwd", out, q, key_cache, value_cache, cu_seqlens_q,
                                   context_lens, block_tables, batch, total_q, num_heads, num_kv_heads, head_size,
                                   block_size, max_seqlen_q, max_context_len, max_num_blocks_per_seq, num_blocks,
                                   q_tok_stride, q_head_stride, o_tok_stride, o_head_stride, kv_block_stride,
                                   kv_head_stride, softmax_scale, is_causal, dtype, stream);
}

// ---- sliding window and sinks ------------------------------------------------------------------------
extern "C" char *aici_mha_varlen_window_fwd(void *out, const void *q, const void *k, const void *v,
                                            const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k, int batch,
                                            int total_q, int total_k, int num_heads, int num_heads_k, int head_size,
                                            int max_seqlen_q, int max_seqlen_k, int window, int sinks,
                                            int64_t q_tok_stride, int64_t q_head_stride, int64_t k_tok_stride,
                                            int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride,
                                            int64_t o_tok_stride, int64_t o_head_stride, float softmax_scale,
                                            int dtype, aici_stream_t stream) {
  void *outs[1] = {out};
  const WindowArgs win = {window, sinks};
  return mha_varlen_fwd_impl("aici_mha_varlen_window_fwd", outs, 1, 0, q, k, v, cu_seqlens_q, cu_seqlens_k, batch,
                             total_q, total_k, num_heads, num_heads_k, head_size, max_seqlen_q, max_seqlen_k,
                             q_tok_stride, q_head_stride, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride,
                             o_tok_stride, o_head_stride, softmax_scale, 1, dtype, stream, 0, &win);
}

extern "C" char *aici_mha_varlen_paged_window_fwd(void *out, const void *q, const void *key_cache,
                                                  const void *value_cache, const int32_t *cu_seqlens_q,
                                                  const int32_t *context_lens, const int32_t *block_tables, int batch,
                                                  int total_q, int num_heads, int num_kv_heads, int head_size,
                                                  int block_size, int max_seqlen_q, int max_context_len,
                                                  int max_num_blocks_per_seq, int64_t num_blocks, int window,
                                                  int sinks, int64_t q_tok_stride, int64_t q_head_stride,
                                                  int64_t o_tok_stride, int64_t o_head_stride,
                                                  int64_t kv_block_stride, int64_t kv_head_stride,
                                                  float softmax_scale, int dtype, aici_stream_t stream) {
  const WindowArgs win = {window, sinks};
  return mha_varlen_paged_fwd_impl("aici_mha_varlen_paged_window_fwd", out, q, key_cache, value_cache, cu_seqlens_q,
                                   context_lens, block_tables, batch, total_q, num_heads, num_kv_heads, head_size,
                                   block_size, max_seqlen_q, max_context_len, max_num_blocks_per_seq, num_blocks,
                                   q_tok_stride, q_head_stride, o_tok_stride, o_head_stride, kv_block_stride,
                                   kv_head_stride, softmax_scale, 1, dtype, stream, &win);
}
