// Attention of few query rows with a sliding window and sinks over the paged cache: decode (one query
// token per sequence), and short chunks (fast-forwarded tokens, drafts to be verified), whose tokens and
// heads are dealt out to work items of 16 rows; the general prefill kernel takes 128 rows of one head to a
// tile and walks the keys with one CTA.
//
// A query at position d sees the tokens t <= d with t > d - window or t < sinks; the last token of a
// sequence stands at ctx - 1.  Only cache blocks with a visible token are touched: of the block list of a row
// (sequence, kv head) those are the first ones (sinks) and the last ones (window), and "tile i of a
// row" below counts through them:  block(i) = i < n_sink ? i : first + i - n_sink.
//     o = sum_t 2^(c q.k_t - m) v_t / sum_t 2^(c q.k_t - m),   c = scale log2 e,  m = max_t c q.k_t
// in one pass with a running m; results of parts of a row are joined by their m and sums.
//
// What bounds it: every visible key and value is read once (512 bytes per token and kv head), and
// 4 x heads x 128 operations per token go with that, so memory bandwidth decides as soon as the rows fill
// the GPU and latency before.  As in paged_decode.cu a warp is an agent of its own: it streams 4 KB key
// tiles and 4 KB value tiles (16 tokens) into a private ring by bulk copies, multiplies the whole
// query-head group against a tile with mma.sync (heads are the rows of the fragment; 16 rows when a kv
// head has more than 8 query heads) and keeps the softmax state in registers.
//
// A row belongs to one CTA, or, when rows are few, to a cluster of 2, 4 or 8: tile i goes to warp
// i mod warps, the warps join their results through shared memory and the CTAs through distributed
// shared memory.  One launch, no workspace.  With a window rows are much alike, and the CTAs of the
// kv heads of a sequence, started next to each other, read neighbouring 4 KB pieces of the same blocks:
// 1024 rows of 257 tiles took 311 us (6.9 TB/s), against 340 us when all tiles of the batch are cut into
// equal runs for resident warps and a second kernel joins the cut rows (256 rows: 88 against 94 us; 8 rows,
// cluster of 8: 9.8 against 24 us); with probabilities in two parts, as they are now, 314, 87 and 9.8 us.  What
// that other form is better at is a batch with one row far longer than the rest: a CTA alone streams a tile in 0.19
// us, so the last row to start costs at most that times its tiles.
#include "dependent.cuh"
#include "half_types.cuh"
#include "window_chunk.cuh"

namespace aici {

constexpr int kWinHead = 128;
constexpr int kWinBlock = 16;
constexpr int kWinTileBytes = kWinHead * kWinBlock * 2;
constexpr int kWinStageBytes = 2 * kWinTileBytes;  // key tile and value tile
constexpr int kWinWarps = 4;
// 96 KB of ring a CTA, 192 KB an SM with two of them, and as one stage of three is being worked on, 128 KB in flight
constexpr int kWinStages = 3;
constexpr int kWinThreads = kWinWarps * 32;
constexpr int kWinRingBytes = kWinWarps * kWinStages * kWinStageBytes;
constexpr int kWinBarBytes = 128;  // kWinWarps * kWinStages barriers

struct WindowDecodeParams {
  void *out;
  const void *q, *k, *v;
  const int32_t *block_tables, *context_lens;
  int num_seqs, num_heads, num_kv_heads, group, window, sinks, max_blocks, max_context;
  int64_t num_blocks, q_stride, kv_block;
  float scale_log2e;
  unsigned int *status;
  // chunks: first query row of each sequence [num_seqs + 1], head strides and the output's token stride
  const int32_t *cu_q;
  int64_t q_head, o_tok, o_head;
  int items;    // work items of 16 rows to a (sequence, kv head)
  int total_q;  // query rows of the tensor
  int max_tokens;
  int refuse;   // sequences of more than max_tokens tokens: 1 = zero rows and a status, 0 = another launch's
};

// The visible part of a work item: of a (sequence, kv head) in decode; in a chunk, what any of the item's
// tokens sees.
struct WindowRow {
  int ctx, lo, sinks;        // visible: t < ctx && (t >= lo || t < sinks)
  int all_hi, all_lo;        // chunks: t < all_hi is not too late for any token, t >= all_lo not too early
  int first, n_sink, tiles;  // first block of the window, blocks of sinks before it, blocks in all
  __device__ __forceinline__ int block(int i) const { return i < n_sink ? i : first + i - n_sink; }
};

// `tokens`: query tokens of the item, the last of them `back` positions before the sequence's last.
__device__ __forceinline__ WindowRow window_row(const WindowDecodeParams &p, int ctx, int tokens, int back) {
  const int64_t table = (int64_t)p.max_blocks * kWinBlock;
  const int cap = table < p.max_context ? (int)table : p.max_context;
  if (ctx > cap) {
    set_status(p.status, AICI_STATUS_BAD_BLOCK);
    ctx = cap;
  }
  WindowRow r;
  r.ctx = max(ctx, 0) - back;  // below 1: nothing is visible
  r.lo = (int)max((int64_t)r.ctx - (tokens - 1) - p.window, (int64_t)0);
  r.all_hi = r.ctx - (tokens - 1);
  r.all_lo = max(r.ctx - p.window, 0);
  r.sinks = max(min(p.sinks, r.ctx), 0);
  r.first = r.lo / kWinBlock;
  r.n_sink = min((r.sinks + kWinBlock - 1) / kWinBlock, r.first);
  r.tiles = r.ctx > 0 ? r.n_sink + (r.ctx + kWinBlock - 1) / kWinBlock - r.first : 0;
  return r;
}

template <typename T>
__device__ __forceinline__ void mma_half(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_half<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma_half<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Softmax state of the query rows of a kv head against the tiles seen so far, spread over a warp as the
// mma.sync fragments are: lane (g, tig) holds rows g and (kTwo) g + 8, columns 8 n + 2 tig, + 1.  Row = head
// of the group, or in a chunk token * group + head from the item's first row on.
template <typename T, bool kTwo, bool kChunk>
struct GroupState {
  static constexpr int kRows = kTwo ? 2 : 1;
  int hi[kRows], lo[kRows];  // chunks: visible to the row: t < hi && (t >= lo || t < sinks)
  uint32_t qa[8][2 * kRows];
  float o[16][4];  // [n][2..3] stay zero without the second row
  float m[kRows], l[kRows];

  // q0: the sequence's first query row of the tensor, pos0: its position; the item has the rows row0 ..
  // row0 + rows - 1 of the kv head's
  __device__ __forceinline__ void load(const WindowDecodeParams &p, int q0, int pos0, int row0, int rows, int kvh, int g,
                                       int tig) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int i = row0 + g + 8 * r, token = kChunk ? i / p.group : 0, head = i - token * p.group;
      const bool there = g + 8 * r < rows;
      const T *row = static_cast<const T *>(p.q) + (q0 + token) * p.q_stride +
                     (kvh * p.group + head) * (kChunk ? p.q_head : (int64_t)kWinHead) + 2 * tig;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        qa[ks][r] = there ? *reinterpret_cast<const uint32_t *>(row + 16 * ks) : 0u;
        qa[ks][kRows + r] = there ? *reinterpret_cast<const uint32_t *>(row + 16 * ks + 8) : 0u;
      }
      if (kChunk) {
        hi[r] = there ? pos0 + token + 1 : 0;
        lo[r] = (int)max((int64_t)hi[r] - p.window, (int64_t)0);
      }
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  }

  // One staged tile whose first token is t0.
  __device__ __forceinline__ void tile(uint32_t kbase, uint32_t vbase, int t0, const WindowRow &row, float scale,
                                       int lane, int tig) {
    const int mi = lane >> 3, mr = lane & 7;
    // key tile [c = d/8][tok][8]: matrices (c even, tok 0-7), (c odd, tok 0-7), (c even, tok 8-15), (c odd, tok 8-15)
    const uint32_t k_off = ((mi & 1) * kWinBlock + 8 * (mi >> 1) + mr) * 16;
    // value tile [d][tok]: matrices (d 0-7, tok 0-7), (d 0-7, tok 8-15), (d 8-15, tok 0-7), (d 8-15, tok 8-15)
    const uint32_t v_off = (8 * (mi >> 1) + mr) * 32 + (mi & 1) * 16;
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t b00, b01, b10, b11;
      ldmatrix_x4(b00, b01, b10, b11, kbase + ks * (2 * kWinBlock * 16) + k_off);
      const uint32_t a0 = qa[ks][0], a1 = kTwo ? qa[ks][1] : 0u, a2 = qa[ks][kRows], a3 = kTwo ? qa[ks][kRows + 1] : 0u;
      mma_half<T>(s0, a0, a1, a2, a3, b00, b01);
      mma_half<T>(s1, a0, a1, a2, a3, b10, b11);
    }
    // tokens t0 + {2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9}: scores masked by selection, values by clearing
    // (0 x NaN is NaN, and what is not visible may hold anything)
    bool vis[kRows][4];
    uint32_t vm_lo = ~0u, vm_hi = ~0u;
    const bool edge = t0 + kWinBlock > (kChunk ? row.all_hi : row.ctx) ||
                      (t0 < (kChunk ? row.all_lo : row.lo) && t0 + kWinBlock > row.sinks);
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) vis[r][j] = true;
    if (edge) {
      bool any[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + 2 * tig + (j & 1) + 8 * (j >> 1);
        any[j] = t < row.ctx && (t >= row.lo || t < row.sinks);
#pragma unroll
        for (int r = 0; r < kRows; ++r) vis[r][j] = kChunk ? t < hi[r] && (t >= lo[r] || t < row.sinks) : any[j];
      }
      vm_lo = (any[0] ? 0xffffu : 0u) | (any[1] ? 0xffff0000u : 0u);
      vm_hi = (any[2] ? 0xffffu : 0u) | (any[3] ? 0xffff0000u : 0u);
    }
    // A probability goes in as two 16-bit numbers, the rounded value and what the rounding left: the values'
    // product is then as exact as fp32 sums make it, and the output carries one rounding, its own.  (With
    // the rounded value alone the error is half as large again; the second product costs nothing beside
    // the tile's copy.)
    uint32_t pa[2][2], pb[2][2];
    float alpha[kRows];
    bool moved = false;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float x0 = vis[r][0] ? s0[2 * r] * scale : -INFINITY, x1 = vis[r][1] ? s0[2 * r + 1] * scale : -INFINITY;
      const float x2 = vis[r][2] ? s1[2 * r] * scale : -INFINITY, x3 = vis[r][3] ? s1[2 * r + 1] * scale : -INFINITY;
      float mt = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
      const float mn = fmaxf(m[r], mt);
      const float base = mn == -INFINITY ? 0.f : mn;
      alpha[r] = fast_exp2(m[r] - base);  // 0 on the first tile
      moved |= mn != m[r];
      m[r] = mn;
      const float p0 = fast_exp2(x0 - base), p1 = fast_exp2(x1 - base), p2 = fast_exp2(x2 - base), p3 = fast_exp2(x3 - base);
      l[r] = l[r] * alpha[r] + (p0 + p1) + (p2 + p3);
      pa[r][0] = Half16<T>::pack(p0, p1);
      pa[r][1] = Half16<T>::pack(p2, p3);
      const float2 h01 = Half16<T>::unpack(pa[r][0]), h23 = Half16<T>::unpack(pa[r][1]);
      pb[r][0] = Half16<T>::pack(p0 - h01.x, p1 - h01.y);
      pb[r][1] = Half16<T>::pack(p2 - h23.x, p3 - h23.y);
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        o[n][0] *= alpha[0];
        o[n][1] *= alpha[0];
        if (kTwo) {
          o[n][2] *= alpha[kRows - 1];
          o[n][3] *= alpha[kRows - 1];
        }
      }
    }
#pragma unroll
    for (int np = 0; np < 8; ++np) {
      uint32_t v00, v01, v10, v11;
      ldmatrix_x4(v00, v01, v10, v11, vbase + np * (16 * 32) + v_off);
      if (edge) {
        v00 &= vm_lo; v10 &= vm_lo;
        v01 &= vm_hi; v11 &= vm_hi;
      }
      mma_half<T>(o[2 * np], pa[0][0], kTwo ? pa[1][0] : 0u, pa[0][1], kTwo ? pa[1][1] : 0u, v00, v01);
      mma_half<T>(o[2 * np + 1], pa[0][0], kTwo ? pa[1][0] : 0u, pa[0][1], kTwo ? pa[1][1] : 0u, v10, v11);
      mma_half<T>(o[2 * np], pb[0][0], kTwo ? pb[1][0] : 0u, pb[0][1], kTwo ? pb[1][1] : 0u, v00, v01);
      mma_half<T>(o[2 * np + 1], pb[0][0], kTwo ? pb[1][0] : 0u, pb[0][1], kTwo ? pb[1][1] : 0u, v10, v11);
    }
  }

  // Sums over the four lanes of a row.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
  }
};

__device__ __forceinline__ float inverse(float l) { return l > 0.f ? __fdividef(1.f, l) : 0.f; }

// Issues the copies of one tile into stage `count % kWinStages` of a warp's ring (lane 0).
template <typename T>
__device__ __forceinline__ void issue_tile(const WindowDecodeParams &p, uint8_t *ring, uint64_t *full, unsigned count,
                                           int blk, int kvh) {
  const unsigned stage = count % kWinStages;
  uint8_t *dst = ring + stage * kWinStageBytes;
  const int64_t off = blk * p.kv_block + (int64_t)kvh * (kWinHead * kWinBlock);
  fence_proxy_async_smem();  // this warp's earlier reads of the stage come before the refill
  mbar_expect_tx(&full[stage], kWinStageBytes);
  bulk_g2s(dst, static_cast<const T *>(p.k) + off, kWinTileBytes, &full[stage]);
  bulk_g2s(dst + kWinTileBytes, static_cast<const T *>(p.v) + off, kWinTileBytes, &full[stage]);
}

__device__ __forceinline__ int block_id(const WindowDecodeParams &p, int seq, int block) {
  int id = p.block_tables[(int64_t)seq * p.max_blocks + block];
  if (id < 0 || id >= p.num_blocks) {
    set_status(p.status, AICI_STATUS_BAD_BLOCK);
    id = 0;
  }
  return id;
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t local, uint32_t cta) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(cta));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t local, uint32_t cta) {
  uint32_t remote;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(cta));
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote) : "memory");
  return v;
}

template <typename T, bool kTwo, bool kChunk>
__global__ void __launch_bounds__(kWinThreads, 2) window_decode_kernel(const WindowDecodeParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kHeads = kTwo ? 16 : 8;
  // what a warp leaves for its CTA lies in its own ring; what the CTA leaves for the cluster behind the rings
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tig = lane & 3;
  uint8_t *ring = smem + warp * (kWinStages * kWinStageBytes);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kWinRingBytes) + warp * kWinStages;
  float *s_o = reinterpret_cast<float *>(smem + kWinRingBytes + kWinBarBytes);  // [kHeads][128]
  float2 *s_ml = reinterpret_cast<float2 *>(s_o + kHeads * kWinHead);           // [kHeads]
  float2 *s_wml = s_ml + kHeads;                                                // [kWinWarps][kHeads]
  uint32_t rank, ctas;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kWinStages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  dependent_start();

  int item = blockIdx.x / ctas, row0 = 0;
  if (kChunk) {
    row0 = item % p.items * 16;
    item /= p.items;
  }
  const int seq = item / p.num_kv_heads, kvh = item - seq * p.num_kv_heads;
  const int ctx = p.context_lens[seq];
  int q0 = seq, rows = p.group, tokens = 1, back = 0, all_tokens = 1;
  if (kChunk) {
    const int from = p.cu_q[seq], upto = p.cu_q[seq + 1];  // rows outside the query tensor are nobody's
    q0 = min(max(from, 0), p.total_q);
    all_tokens = min(max(upto, q0), p.total_q) - q0;
    if ((from < 0 || upto > p.total_q) && threadIdx.x == 0) set_status(p.status, AICI_STATUS_BAD_BLOCK);
    if (all_tokens > p.max_tokens) {
      if (p.refuse) {
        if (threadIdx.x == 0) set_status(p.status, AICI_STATUS_BAD_BLOCK);
        // its rows are dealt out to the CTAs that it has
        const int width = p.group * (kWinHead / 8), parts = p.items * (int)ctas;
        for (int token = row0 / 16 * (int)ctas + (int)rank; token < all_tokens; token += parts)
          for (int i = threadIdx.x; i < width; i += kWinThreads)
            *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + (q0 + token) * p.o_tok +
                                       (kvh * p.group + i / (kWinHead / 8)) * p.o_head + i % (kWinHead / 8) * 8) =
                make_uint4(0, 0, 0, 0);
      }
      all_tokens = 0;
    }
    rows = (int)max(min((int64_t)all_tokens * p.group - row0, (int64_t)kHeads), (int64_t)0);
    const int last = (row0 + max(rows, 1) - 1) / p.group;  // the item's last token
    tokens = last - row0 / p.group + 1;
    back = max(all_tokens - 1 - last, 0);
  }
  const WindowRow row = window_row(p, ctx, tokens, back);
  const int stride = ctas * kWinWarps, first = rank * kWinWarps + warp;
  // tiles first, first + stride, ...
  const int mine = rows > 0 && row.tiles > first ? (row.tiles - first + stride - 1) / stride : 0;
  GroupState<T, kTwo, kChunk> st;
  st.load(p, q0, row.ctx + back - all_tokens, row0, rows, kvh, g, tig);
  int ids = 0;
  unsigned issued = 0;
  auto produce = [&]() {
    if (issued >= (unsigned)mine) return;
    if (issued % 32 == 0 && issued + lane < (unsigned)mine)
      ids = block_id(p, seq, row.block(first + (int)(issued + lane) * stride));
    const int blk = __shfl_sync(0xffffffffu, ids, issued % 32);
    if (lane == 0) issue_tile<T>(p, ring, full, issued, blk, kvh);
    ++issued;
  };
#pragma unroll
  for (int s = 0; s < kWinStages - 1; ++s) produce();
  bool ok = true;
  unsigned done = 0;
  for (; done < (unsigned)mine; ++done) {
    produce();
    const unsigned stage = done % kWinStages;
    ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], (done / kWinStages) & 1u, p.status));
    if (!ok) break;
    const uint32_t kbase = smem_u32(ring + stage * kWinStageBytes);
    st.tile(kbase, kbase + kWinTileBytes, row.block(first + (int)done * stride) * kWinBlock, row, p.scale_log2e, lane, tig);
    __syncwarp();
  }
  if (!ok)  // give copies already in flight a bounded chance to land
    for (unsigned c = done; c != issued; ++c) mbar_wait(&full[c % kWinStages], (c / kWinStages) & 1u, p.status);
  st.finish();

  // ---- join the warps of the CTA ----------------------------------------------------------------------
  float *w_o = reinterpret_cast<float *>(ring);  // [kHeads][128] of this warp
#pragma unroll
  for (int r = 0; r < GroupState<T, kTwo, kChunk>::kRows; ++r) {
    const int h = g + 8 * r;
    if (h < rows) {
#pragma unroll
      for (int n = 0; n < 16; ++n)
        *reinterpret_cast<float2 *>(w_o + h * kWinHead + 8 * n + 2 * tig) = make_float2(st.o[n][2 * r], st.o[n][2 * r + 1]);
      if (tig == 0) s_wml[warp * kHeads + h] = make_float2(st.m[r], st.l[r]);
    }
  }
  __syncthreads();
  const int items = rows * (kWinHead / 4);  // four elements of a row each
  auto out = [&](int row) {
    if (!kChunk) return static_cast<T *>(p.out) + ((int64_t)seq * p.num_heads + kvh * p.group + row) * kWinHead;
    const int token = (row0 + row) / p.group;
    return static_cast<T *>(p.out) + (q0 + token) * p.o_tok + (kvh * p.group + row0 + row - token * p.group) * p.o_head;
  };
  for (int i = threadIdx.x; i < items; i += kWinThreads) {
    const int h = i >> 5, d = (i & 31) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) m = fmaxf(m, s_wml[w * kHeads + h].x);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) {
      const float2 ml = s_wml[w * kHeads + h];
      const float f = fast_exp2(ml.x - base);
      const float4 v = *reinterpret_cast<const float4 *>(smem + w * (kWinStages * kWinStageBytes) + (h * kWinHead + d) * 4);
      l += f * ml.y;
      a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
    }
    if (ctas == 1) {
      const float inv = inverse(l);
      *reinterpret_cast<uint2 *>(out(h) + d) =
          make_uint2(Half16<T>::pack(a.x * inv, a.y * inv), Half16<T>::pack(a.z * inv, a.w * inv));
    } else {
      *reinterpret_cast<float4 *>(s_o + h * kWinHead + d) = a;
      if ((i & 31) == 0) s_ml[h] = make_float2(m, l);
    }
  }
  if (ctas == 1) return;
  // ---- and the CTAs of the cluster: each takes every ctas-th item ---------------------------------------
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = threadIdx.x * ctas + rank; i < items; i += kWinThreads * ctas) {
    const int h = i >> 5, d = (i & 31) * 4;
    float2 ml[8];
    float4 v[8];
    float m = -INFINITY;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < ctas) {
        ml[c] = ld_cluster2(smem_u32(s_ml + h), c);
        v[c] = ld_cluster4(smem_u32(s_o + h * kWinHead + d), c);
      }
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < ctas) m = fmaxf(m, ml[c].x);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < ctas) {
        const float f = fast_exp2(ml[c].x - base);
        l += f * ml[c].y;
        a.x += f * v[c].x; a.y += f * v[c].y; a.z += f * v[c].z; a.w += f * v[c].w;
      }
    const float inv = inverse(l);
    *reinterpret_cast<uint2 *>(out(h) + d) =
        make_uint2(Half16<T>::pack(a.x * inv, a.y * inv), Half16<T>::pack(a.z * inv, a.w * inv));
  }
  // nobody leaves while its shared memory may still be read
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- host side -----------------------------------------------------------------------------------------
// Most tiles a row can have.
static int64_t most_tiles(int64_t max_context, int64_t window, int64_t sinks, int64_t tokens) {
  const int64_t all = (max_context + kWinBlock - 1) / kWinBlock;
  const int64_t seen = (window + tokens - 1 + kWinBlock - 1) / kWinBlock + 1 + (sinks + kWinBlock - 1) / kWinBlock;
  return seen < all ? seen : all;
}

// CTAs that share a row: as many as keep all rows resident at once, and no more than have tiles to
// work on.  (64 rows of 65 tiles: 14.2, 9.7, 8.2 us with 1, 2, 4 CTAs and 12.6 with 8, two waves; 8 rows of
// 4 tiles: 2.8 us with one CTA, 4.0 with any cluster.)
static int ctas_per_row(int64_t rows, int64_t tiles) {
  int c = 1;
  while (c < 8 && rows * 2 * c <= 2 * sm_count() && tiles > (int64_t)c * kWinWarps) c *= 2;
  return c;
}

template <typename T, bool kTwo, bool kChunk>
static char *launch_window_decode(const WindowDecodeParams &p, int ctas, cudaStream_t stream, bool overlap = true) {
  constexpr int kSmem = kWinRingBytes + kWinBarBytes + (kTwo ? 16 : 8) * (kWinHead * 4 + 8 + kWinWarps * 8);
  static OncePerDevice once;
  if (char *e = once.run([]() -> char * {
        AICI_CUDA(cudaFuncSetAttribute(window_decode_kernel<T, kTwo, kChunk>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        return nullptr;
      }))
    return e;
  cudaLaunchAttribute attr[2];
  attr[0] = dependent_launch();
  attr[0].val.programmaticStreamSerializationAllowed = overlap;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)p.num_seqs * p.num_kv_heads * p.items * ctas));
  cfg.blockDim = dim3(kWinThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  AICI_CUDA(cudaLaunchKernelEx(&cfg, window_decode_kernel<T, kTwo, kChunk>, p));
  return nullptr;
}

char *launch_window_chunk(const WindowChunk &c, int dtype, cudaStream_t stream) {
  WindowDecodeParams p = {};
  p.out = c.out;
  p.q = c.q;
  p.k = c.key_cache;
  p.v = c.value_cache;
  p.block_tables = c.block_tables;
  p.context_lens = c.context_lens;
  p.num_seqs = c.batch;
  p.num_heads = c.num_heads;
  p.num_kv_heads = c.num_kv_heads;
  p.group = c.num_heads / c.num_kv_heads;
  p.window = c.window;
  p.sinks = c.sinks;
  p.max_blocks = c.max_blocks;
  p.max_context = 0x7fffffff;  // as in the general kernel the table's width alone limits a context
  p.num_blocks = c.num_blocks;
  p.q_stride = c.q_tok;
  p.kv_block = c.kv_block;
  p.scale_log2e = c.scale * 1.4426950408889634f;
  p.status = c.status;
  p.cu_q = c.cu_q;
  p.q_head = c.q_head;
  p.o_tok = c.o_tok;
  p.o_head = c.o_head;
  p.items = (int)window_chunk_items(c.max_tokens, p.group);
  p.total_q = c.total_q;
  p.max_tokens = c.max_tokens;
  p.refuse = c.beside ? 0 : 1;
  const int ctas = ctas_per_row((int64_t)c.batch * c.num_kv_heads * p.items,
                                most_tiles(c.max_context, c.window, c.sinks, c.max_tokens));
  return with_half_type(dtype, [&](auto t) -> char * {
    using T = decltype(t);
    return c.max_tokens > 8 / p.group ? launch_window_decode<T, true, true>(p, ctas, stream, !c.beside)
                                      : launch_window_decode<T, false, true>(p, ctas, stream, !c.beside);
  });
}

}  // namespace aici

using namespace aici;

extern "C" char *aici_paged_attention_window(void *out, const void *query, const void *key_cache,
                                             const void *value_cache, int num_kv_heads, float scale,
                                             const int32_t *block_tables, const int32_t *context_lens,
                                             int block_size, int max_context_len, int window, int sinks, int num_seqs,
                                             int num_heads, int head_size, int max_num_blocks_per_seq,
                                             int64_t num_blocks, int64_t q_stride, int64_t kv_block_stride,
                                             int64_t kv_head_stride, int dtype, aici_stream_t stream) {
  const char *fn = "aici_paged_attention_window";
  AICI_CHECK(dtype == AICI_DTYPE_BF16 || dtype == AICI_DTYPE_F16, "%s: only bf16 and f16 are supported (dtype=%d)", fn,
             dtype);
  AICI_CHECK(head_size == kWinHead, "%s: head_size must be 128 (got %d)", fn, head_size);
  AICI_CHECK(block_size == kWinBlock, "%s: block_size must be 16 (got %d)", fn, block_size);
  AICI_CHECK(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
             "%s: num_heads %d not divisible by num_kv_heads %d", fn, num_heads, num_kv_heads);
  const int group = num_heads / num_kv_heads;
  AICI_CHECK(group <= 16, "%s: at most 16 query heads per kv head (got %d)", fn, group);
  AICI_CHECK(window >= 1, "%s: window must be at least 1 (got %d)", fn, window);
  AICI_CHECK(sinks >= 0, "%s: sinks must not be negative (got %d)", fn, sinks);
  AICI_CHECK(scale > 0.f, "%s: scale must be positive", fn);
  AICI_CHECK(num_seqs >= 0 && max_context_len >= 0 && max_num_blocks_per_seq >= 0, "%s: negative size", fn);
  AICI_CHECK((int64_t)num_seqs * num_heads < (1ll << 31), "%s: too many sequences and heads for one call", fn);
  AICI_CHECK(num_blocks > 0, "%s: num_blocks must be positive", fn);
  if (num_seqs <= 1) q_stride = (int64_t)num_heads * head_size;  // never used
  AICI_CHECK(q_stride % 8 == 0 && q_stride >= (int64_t)num_heads * head_size,
             "%s: q_stride must be a multiple of 8 elements and cover one row", fn);
  AICI_CHECK(kv_head_stride == kWinHead * kWinBlock && kv_block_stride % 8 == 0 &&
                 kv_block_stride >= (int64_t)num_kv_heads * kWinHead * kWinBlock,
             "%s: cache must be [blocks, kv_heads, 128/8, 16, 8] with contiguous head tiles", fn);
  if (num_seqs == 0) return nullptr;
  AICI_CHECK(out && query && key_cache && value_cache && block_tables && context_lens, "%s: NULL pointer", fn);
  AICI_CHECK(((uintptr_t)out | (uintptr_t)query | (uintptr_t)key_cache | (uintptr_t)value_cache) % 16 == 0,
             "%s: tensors must be 16-byte aligned", fn);
  if (char *e = check_on_current_device(fn, "query", query)) return e;
  unsigned int *st = status_ptr();
  AICI_CHECK(st != nullptr, "%s: no CUDA device", fn);
  WindowDecodeParams p = {};
  p.out = out;
  p.q = query;
  p.k = key_cache;
  p.v = value_cache;
  p.block_tables = block_tables;
  p.context_lens = context_lens;
  p.num_seqs = num_seqs;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = group;
  p.window = window;
  p.sinks = sinks;
  p.max_blocks = max_num_blocks_per_seq;
  p.max_context = max_context_len;
  p.num_blocks = num_blocks;
  p.q_stride = q_stride;
  p.kv_block = kv_block_stride;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.status = st;
  p.items = 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int ctas = ctas_per_row((int64_t)num_seqs * num_kv_heads, most_tiles(max_context_len, window, sinks, 1));
  return with_half_type(dtype, [&](auto t) -> char * {
    using T = decltype(t);
    return group > 8 ? launch_window_decode<T, true, false>(p, ctas, s) : launch_window_decode<T, false, false>(p, ctas, s);
  });
}
