// Decode attention with a sliding window and sinks over the paged cache (one query token per sequence).
//
// The query of a sequence stands at position ctx - 1 and sees the tokens t < ctx with t >= ctx - window
// or t < sinks.  Only cache blocks with a visible token are touched: of the block list of a row
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
// Two ways of dealing out the work:
//   cluster   few rows: 1 to 8 CTAs of a cluster share a row, tile i going to warp i mod warps, and
//             join their results through distributed shared memory.  One launch, no workspace.
//   spans     many rows: all tiles of the batch laid end to end, every warp of two CTAs per SM takes an
//             equal run, whatever the mix of context lengths; rows cut by a run's border leave fp32
//             partials that a second kernel joins.
#include "half_types.cuh"

namespace aici {

constexpr int kWinHead = 128;
constexpr int kWinBlock = 16;
constexpr int kWinTileBytes = kWinHead * kWinBlock * 2;
constexpr int kWinStageBytes = 2 * kWinTileBytes;  // key tile and value tile
constexpr int kWinWarps = 4;
constexpr int kWinStages = 3;  // 72 KB of ring in flight per SM and CTA pair: enough for the bandwidth-latency product
constexpr int kWinThreads = kWinWarps * 32;
constexpr int kWinSeqs = 1024;     // sequences of one launch (their lengths are summed in shared memory)
constexpr int kWinMinSpan = 4;     // tiles: fewer would make partials a large share of the traffic
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
  // spans
  int *span_cum;  // [num_seqs + 2] tiles before each sequence, then the span
  float *part_m, *part_l, *part_o;
};

// The visible part of a row.
struct WindowRow {
  int ctx, lo, sinks;        // visible: t < ctx && (t >= lo || t < sinks)
  int first, n_sink, tiles;  // first block of the window, blocks of sinks before it, blocks in all
  __device__ __forceinline__ int block(int i) const { return i < n_sink ? i : first + i - n_sink; }
};

__device__ __forceinline__ WindowRow window_row(const WindowDecodeParams &p, int ctx) {
  const int64_t table = (int64_t)p.max_blocks * kWinBlock;
  const int cap = table < p.max_context ? (int)table : p.max_context;
  if (ctx > cap) {
    set_status(p.status, AICI_STATUS_BAD_BLOCK);
    ctx = cap;
  }
  WindowRow r;
  r.ctx = max(ctx, 0);
  r.lo = max(r.ctx - p.window, 0);
  r.sinks = min(p.sinks, r.ctx);
  r.first = r.lo / kWinBlock;
  r.n_sink = min((r.sinks + kWinBlock - 1) / kWinBlock, r.first);
  r.tiles = r.n_sink + (r.ctx + kWinBlock - 1) / kWinBlock - r.first;
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

// Softmax state of a query-head group against the tiles seen so far, spread over a warp as the
// mma.sync fragments are: lane (g, tig) holds rows g and (kTwo) g + 8, columns 8 n + 2 tig, + 1.
template <typename T, bool kTwo>
struct GroupState {
  static constexpr int kRows = kTwo ? 2 : 1;
  uint32_t qa[8][2 * kRows];
  float o[16][4];  // [n][2..3] stay zero without the second row
  float m[kRows], l[kRows];

  __device__ __forceinline__ void load(const WindowDecodeParams &p, int seq, int kvh, int g, int tig) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const T *row = static_cast<const T *>(p.q) + seq * p.q_stride + (int64_t)(kvh * p.group + g + 8 * r) * kWinHead + 2 * tig;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        qa[ks][r] = g + 8 * r < p.group ? *reinterpret_cast<const uint32_t *>(row + 16 * ks) : 0u;
        qa[ks][kRows + r] = g + 8 * r < p.group ? *reinterpret_cast<const uint32_t *>(row + 16 * ks + 8) : 0u;
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
    bool vis[4] = {true, true, true, true};
    uint32_t vm_lo = ~0u, vm_hi = ~0u;
    const bool edge = t0 + kWinBlock > row.ctx || (t0 < row.lo && t0 + kWinBlock > row.sinks);
    if (edge) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + 2 * tig + (j & 1) + 8 * (j >> 1);
        vis[j] = t < row.ctx && (t >= row.lo || t < row.sinks);
      }
      vm_lo = (vis[0] ? 0xffffu : 0u) | (vis[1] ? 0xffff0000u : 0u);
      vm_hi = (vis[2] ? 0xffffu : 0u) | (vis[3] ? 0xffff0000u : 0u);
    }
    uint32_t pa[2][2];
    float alpha[kRows];
    bool moved = false;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float x0 = vis[0] ? s0[2 * r] * scale : -INFINITY, x1 = vis[1] ? s0[2 * r + 1] * scale : -INFINITY;
      const float x2 = vis[2] ? s1[2 * r] * scale : -INFINITY, x3 = vis[3] ? s1[2 * r + 1] * scale : -INFINITY;
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

// ---- cluster ---------------------------------------------------------------------------------------
__device__ __forceinline__ float4 ld_cluster4(uint32_t local, uint32_t cta) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(cta));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t local, uint32_t cta) {
  uint32_t remote;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(cta));
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote) : "memory");
  return v;
}

template <typename T, bool kTwo>
__global__ void __launch_bounds__(kWinThreads, 2) window_decode_cluster_kernel(const WindowDecodeParams p) {
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
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int rowi = blockIdx.x / ctas, seq = rowi / p.num_kv_heads, kvh = rowi - seq * p.num_kv_heads;
  const WindowRow row = window_row(p, p.context_lens[seq]);
  const int stride = ctas * kWinWarps, first = rank * kWinWarps + warp;
  const int mine = row.tiles > first ? (row.tiles - first + stride - 1) / stride : 0;  // tiles first, first + stride, ...
  GroupState<T, kTwo> st;
  st.load(p, seq, kvh, g, tig);
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
  for (int r = 0; r < GroupState<T, kTwo>::kRows; ++r) {
    const int h = g + 8 * r;
    if (h < p.group) {
#pragma unroll
      for (int n = 0; n < 16; ++n)
        *reinterpret_cast<float2 *>(w_o + h * kWinHead + 8 * n + 2 * tig) = make_float2(st.o[n][2 * r], st.o[n][2 * r + 1]);
      if (tig == 0) s_wml[warp * kHeads + h] = make_float2(st.m[r], st.l[r]);
    }
  }
  __syncthreads();
  const int items = p.group * (kWinHead / 4);  // four elements of a head each
  T *out = static_cast<T *>(p.out) + ((int64_t)seq * p.num_heads + kvh * p.group) * kWinHead;
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
      *reinterpret_cast<uint2 *>(out + h * kWinHead + d) = make_uint2(Half16<T>::pack(a.x * inv, a.y * inv), Half16<T>::pack(a.z * inv, a.w * inv));
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
    *reinterpret_cast<uint2 *>(out + h * kWinHead + d) = make_uint2(Half16<T>::pack(a.x * inv, a.y * inv), Half16<T>::pack(a.z * inv, a.w * inv));
  }
  // nobody leaves while its shared memory may still be read
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- spans -----------------------------------------------------------------------------------------
// Some consecutive tiles of one row.  Row (seq, kvh) starts at tile num_kv_heads * cum[seq] + kvh *
// tiles(seq) of the batch; a warp's span is cut into pieces at row ends.  Piece number x / span + row
// index (x = its first tile) is unique, below warps + rows, and consecutive within a row: the joining
// kernel finds a row's partials without a list.
struct WindowPiece {
  WindowRow row;
  int seq, kvh, i0, n;
  bool whole;   // the row has no other piece
  int64_t part; // first head's partial
};

__device__ __forceinline__ bool next_piece(const WindowDecodeParams &p, const int *s_cum, const int *s_ctx, int span,
                                           int &x, int end, int cap, WindowPiece &it) {
  if (x >= end) return false;
  const int e = x / p.num_kv_heads;
  int lo = 0, hi = p.num_seqs;
  while (hi - lo > 1) {  // the last sequence that begins at or before e (empty ones share their successor's start)
    const int mid = (lo + hi) >> 1;
    if (s_cum[mid] <= e) lo = mid;
    else hi = mid;
  }
  it.row = window_row(p, s_ctx[lo]);
  const int rem = x - p.num_kv_heads * s_cum[lo];
  it.seq = lo;
  it.kvh = rem / it.row.tiles;
  it.i0 = rem - it.kvh * it.row.tiles;
  it.n = min(min(it.row.tiles - it.i0, end - x), cap);
  const int begin = x - it.i0;  // the row's first tile
  it.whole = (begin + it.row.tiles - 1) / span == begin / span;
  it.part = (int64_t)(x / span + lo * p.num_kv_heads + it.kvh) * p.group;
  x += it.n;
  return true;
}

template <typename T, bool kTwo>
__global__ void __launch_bounds__(kWinThreads, 2) window_decode_spans_kernel(const WindowDecodeParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tig = lane & 3;
  uint8_t *ring = smem + warp * (kWinStages * kWinStageBytes);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kWinRingBytes) + warp * kWinStages;
  int *s_cum = reinterpret_cast<int *>(smem + kWinRingBytes + kWinBarBytes);
  int *s_ctx = s_cum + p.num_seqs + 1;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kWinStages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // tiles before each sequence: every CTA reads all lengths at once and sums them for itself
  for (int s = threadIdx.x; s < p.num_seqs; s += kWinThreads) {
    const int ctx = p.context_lens[s];
    s_ctx[s] = ctx;
    s_cum[s + 1] = window_row(p, ctx).tiles;
  }
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int s0 = 0; s0 < p.num_seqs; s0 += 32) {
      int incl = s0 + lane < p.num_seqs ? s_cum[s0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (s0 + lane < p.num_seqs) s_cum[s0 + lane + 1] = carry + incl;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_cum[0] = 0;
  }
  __syncthreads();
  const int total = s_cum[p.num_seqs] * p.num_kv_heads;
  const int warps = gridDim.x * kWinWarps;
  const int span = max((total + warps - 1) / warps, kWinMinSpan);
  const int64_t x0 = (int64_t)(blockIdx.x * kWinWarps + warp) * span;
  const int begin = x0 < total ? (int)x0 : total, end = x0 + span < total ? (int)(x0 + span) : total;
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i <= p.num_seqs; i += kWinThreads) p.span_cum[i] = s_cum[i];
    if (threadIdx.x == 0) p.span_cum[p.num_seqs + 1] = span;
  }

  // producer: runs ahead of the consumer across pieces, 32 tiles' block ids at a time
  WindowPiece pp;
  pp.n = 0;
  int px = begin, pt = 0, ids = 0;
  unsigned issued = 0;
  bool p_done = false;
  auto produce = [&]() {
    if (p_done) return;
    if (pt == pp.n) {
      if (!next_piece(p, s_cum, s_ctx, span, px, end, 32, pp)) {
        p_done = true;
        return;
      }
      if (lane < pp.n) ids = block_id(p, pp.seq, pp.row.block(pp.i0 + lane));
      pt = 0;
    }
    const int blk = __shfl_sync(0xffffffffu, ids, pt);
    if (lane == 0) issue_tile<T>(p, ring, full, issued, blk, pp.kvh);
    ++pt;
    ++issued;
  };
#pragma unroll
  for (int s = 0; s < kWinStages - 1; ++s) produce();

  unsigned done = 0;
  int cx = begin;
  bool ok = true;
  WindowPiece it;
  while (ok && next_piece(p, s_cum, s_ctx, span, cx, end, 0x7fffffff, it)) {
    GroupState<T, kTwo> st;
    st.load(p, it.seq, it.kvh, g, tig);
    for (int t = 0; t < it.n; ++t) {
      produce();
      const unsigned stage = done % kWinStages;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], (done / kWinStages) & 1u, p.status));
      if (!ok) break;
      const uint32_t kbase = smem_u32(ring + stage * kWinStageBytes);
      st.tile(kbase, kbase + kWinTileBytes, it.row.block(it.i0 + t) * kWinBlock, it.row, p.scale_log2e, lane, tig);
      __syncwarp();
      ++done;
    }
    if (!ok) break;
    st.finish();
#pragma unroll
    for (int r = 0; r < GroupState<T, kTwo>::kRows; ++r) {
      const int h = g + 8 * r;
      if (h >= p.group) continue;
      const float inv = inverse(st.l[r]);
      if (it.whole) {
        T *dst = static_cast<T *>(p.out) + ((int64_t)it.seq * p.num_heads + it.kvh * p.group + h) * kWinHead + 2 * tig;
#pragma unroll
        for (int n = 0; n < 16; ++n)
          *reinterpret_cast<uint32_t *>(dst + 8 * n) = Half16<T>::pack(st.o[n][2 * r] * inv, st.o[n][2 * r + 1] * inv);
      } else {
        if (tig == 0) {
          p.part_m[it.part + h] = st.m[r];
          p.part_l[it.part + h] = st.l[r];
        }
        float *dst = p.part_o + (it.part + h) * kWinHead + 2 * tig;
#pragma unroll
        for (int n = 0; n < 16; ++n)
          *reinterpret_cast<float2 *>(dst + 8 * n) = make_float2(st.o[n][2 * r], st.o[n][2 * r + 1]);
      }
    }
  }
  if (!ok)
    for (unsigned c = done; c != issued; ++c) mbar_wait(&full[c % kWinStages], (c / kWinStages) & 1u, p.status);
}

// Joins the partials of the rows that spans cut: one warp per (sequence, head), four elements to a lane.
template <typename T>
__global__ void __launch_bounds__(256) window_join_kernel(const WindowDecodeParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, idx = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (idx >= p.num_seqs * p.num_heads) return;
  const int seq = idx / p.num_heads, head = idx - seq * p.num_heads;
  const int kvh = head / p.group, h = head - kvh * p.group;
  const int c0 = p.span_cum[seq], tiles = p.span_cum[seq + 1] - c0, span = p.span_cum[p.num_seqs + 1];
  T *out = static_cast<T *>(p.out) + (int64_t)idx * kWinHead + 4 * lane;
  if (tiles == 0) {  // an empty context: no warp came by this row
    *reinterpret_cast<uint2 *>(out) = make_uint2(0u, 0u);
    return;
  }
  const int g0 = p.num_kv_heads * c0 + kvh * tiles;
  const int n = (g0 + tiles - 1) / span - g0 / span + 1;
  if (n == 1) return;
  const int64_t base = (int64_t)(g0 / span + seq * p.num_kv_heads + kvh) * p.group + h;
  float m = -INFINITY;
  for (int j = lane; j < n; j += 32) m = fmaxf(m, p.part_m[base + (int64_t)j * p.group]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const int64_t at = base + (int64_t)j * p.group;
    const float f = fast_exp2(p.part_m[at] - ref);
    const float4 v = *reinterpret_cast<const float4 *>(p.part_o + at * kWinHead + 4 * lane);
    l += f * p.part_l[at];
    a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
  }
  const float inv = inverse(l);
  *reinterpret_cast<uint2 *>(out) = make_uint2(Half16<T>::pack(a.x * inv, a.y * inv), Half16<T>::pack(a.z * inv, a.w * inv));
}

// ---- host side -----------------------------------------------------------------------------------------
// Most tiles a row can have.
static int64_t most_tiles(int64_t max_context, int64_t window, int64_t sinks) {
  const int64_t all = (max_context + kWinBlock - 1) / kWinBlock;
  const int64_t seen = (window + kWinBlock - 1) / kWinBlock + 1 + (sinks + kWinBlock - 1) / kWinBlock;
  return seen < all ? seen : all;
}

// CTAs that share a row in the cluster form, 0 = spans.
static int cluster_ctas(int num_seqs, int num_kv_heads, int64_t tiles) {
  const int64_t rows = (int64_t)num_seqs * num_kv_heads, places = 2 * sm_count();
  if (rows > places) return 0;
  int c = 1;
  while (c < 8 && rows * 2 * c <= places && tiles > (int64_t)c * kWinWarps) c *= 2;
  return c;
}

// Sequences of one launch of the span form: 32-bit tile numbers, lengths in shared memory.
static int span_seqs(int num_kv_heads, int64_t tiles) {
  const int64_t fit = (1ll << 30) / (num_kv_heads * (tiles + 1));
  return (int)(fit < 1 ? 1 : fit < kWinSeqs ? fit : kWinSeqs);
}

struct WindowWorkspace {
  size_t m_off, l_off, o_off, total;
};

static WindowWorkspace window_workspace(int num_seqs, int num_heads, int num_kv_heads) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  const size_t pieces = (size_t)2 * sm_count() * kWinWarps + (size_t)num_seqs * num_kv_heads;
  const size_t parts = pieces * (num_heads / num_kv_heads);
  WindowWorkspace w;
  w.m_off = up((size_t)(num_seqs + 2) * sizeof(int));
  w.l_off = w.m_off + up(parts * sizeof(float));
  w.o_off = w.l_off + up(parts * sizeof(float));
  w.total = w.o_off + parts * kWinHead * sizeof(float);
  return w;
}

static size_t window_workspace_bytes(int num_seqs, int num_heads, int num_kv_heads, int64_t tiles) {
  if (cluster_ctas(num_seqs, num_kv_heads, tiles) > 0) return 0;
  const int part = span_seqs(num_kv_heads, tiles);
  return window_workspace(num_seqs < part ? num_seqs : part, num_heads, num_kv_heads).total;
}

template <typename T, bool kTwo>
static char *launch_window_decode(WindowDecodeParams p, int64_t tiles, char *workspace, cudaStream_t stream) {
  constexpr int kClusterSmem = kWinRingBytes + kWinBarBytes + (kTwo ? 16 : 8) * (kWinHead * 4 + 8 + kWinWarps * 8);
  constexpr int kSpanSmem = kWinRingBytes + kWinBarBytes + (2 * kWinSeqs + 1) * (int)sizeof(int);
  static OncePerDevice once;
  if (char *e = once.run([]() -> char * {
        AICI_CUDA(cudaFuncSetAttribute(window_decode_cluster_kernel<T, kTwo>, cudaFuncAttributeMaxDynamicSharedMemorySize, kClusterSmem));
        AICI_CUDA(cudaFuncSetAttribute(window_decode_spans_kernel<T, kTwo>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSpanSmem));
        // the same shared-memory split for the joining kernel, so that its CTAs can start on SMs that still
        // run the kernel before it
        AICI_CUDA(cudaFuncSetAttribute(window_join_kernel<T>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                       cudaSharedmemCarveoutMaxShared));
        return nullptr;
      }))
    return e;
  // programmatic dependents: a kernel's prologue overlaps the tail of the one before it, and each waits for
  // it before it touches anything
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(kWinThreads);
  const int ctas = cluster_ctas(p.num_seqs, p.num_kv_heads, tiles);
  if (ctas > 0) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
    cfg.gridDim = dim3(p.num_seqs * p.num_kv_heads * ctas);
    cfg.dynamicSmemBytes = kClusterSmem;
    AICI_CUDA(cudaLaunchKernelEx(&cfg, window_decode_cluster_kernel<T, kTwo>, p));
    return nullptr;
  }
  const int all = p.num_seqs, part = span_seqs(p.num_kv_heads, tiles);
  const WindowWorkspace w = window_workspace(all < part ? all : part, p.num_heads, p.num_kv_heads);
  p.span_cum = reinterpret_cast<int *>(workspace);
  p.part_m = reinterpret_cast<float *>(workspace + w.m_off);
  p.part_l = reinterpret_cast<float *>(workspace + w.l_off);
  p.part_o = reinterpret_cast<float *>(workspace + w.o_off);
  for (int s0 = 0; s0 < all; s0 += part) {  // one after the other on the stream, in the same workspace
    WindowDecodeParams c = p;
    c.num_seqs = all - s0 < part ? all - s0 : part;
    c.out = static_cast<T *>(p.out) + (int64_t)s0 * p.num_heads * kWinHead;
    c.q = static_cast<const T *>(p.q) + s0 * p.q_stride;
    c.block_tables = p.block_tables + (int64_t)s0 * p.max_blocks;
    c.context_lens = p.context_lens + s0;
    const int64_t most = (int64_t)c.num_seqs * c.num_kv_heads * tiles;
    const int64_t need = (most + kWinWarps * kWinMinSpan - 1) / (kWinWarps * kWinMinSpan);
    cfg.gridDim = dim3((unsigned)(need < 1 ? 1 : need < 2 * sm_count() ? need : 2 * sm_count()));
    cfg.blockDim = dim3(kWinThreads);
    cfg.dynamicSmemBytes = kWinRingBytes + kWinBarBytes + (2 * c.num_seqs + 1) * sizeof(int);
    AICI_CUDA(cudaLaunchKernelEx(&cfg, window_decode_spans_kernel<T, kTwo>, c));
    cfg.gridDim = dim3((c.num_seqs * c.num_heads + 7) / 8);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    AICI_CUDA(cudaLaunchKernelEx(&cfg, window_join_kernel<T>, c));
  }
  return nullptr;
}

}  // namespace aici

using namespace aici;

extern "C" size_t aici_paged_attention_window_workspace_bytes(int num_seqs, int num_heads, int num_kv_heads,
                                                              int max_context_len, int window, int sinks) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || max_context_len < 0 || window < 1 || sinks < 0) return 0;
  return window_workspace_bytes(num_seqs, num_heads, num_kv_heads, most_tiles(max_context_len, window, sinks));
}

extern "C" char *aici_paged_attention_window(void *out, const void *query, const void *key_cache,
                                             const void *value_cache, int num_kv_heads, float scale,
                                             const int32_t *block_tables, const int32_t *context_lens,
                                             int block_size, int max_context_len, int window, int sinks, int num_seqs,
                                             int num_heads, int head_size, int max_num_blocks_per_seq,
                                             int64_t num_blocks, int64_t q_stride, int64_t kv_block_stride,
                                             int64_t kv_head_stride, void *workspace, size_t workspace_bytes,
                                             int dtype, aici_stream_t stream) {
  const char *fn = "aici_paged_attention_window";
  AICI_CHECK(dtype == AICI_DTYPE_BF16 || dtype == AICI_DTYPE_F16, "%s: only bf16 and f16 are supported (dtype=%d)", fn, dtype);
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
  const int64_t tiles = most_tiles(max_context_len, window, sinks);
  AICI_CHECK(num_kv_heads * (tiles + 1) <= (1ll << 30), "%s: max_context_len too large", fn);
  const size_t need = window_workspace_bytes(num_seqs, num_heads, num_kv_heads, tiles);
  AICI_CHECK(need == 0 || (workspace != nullptr && workspace_bytes >= need),
             "%s: workspace too small (%zu bytes given, %zu needed)", fn, workspace_bytes, need);
  AICI_CHECK(need == 0 || (uintptr_t)workspace % 256 == 0, "%s: workspace must be 256-byte aligned", fn);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
  return with_half_type(dtype, [&](auto t) -> char * {
    using T = decltype(t);
    return group > 8 ? launch_window_decode<T, true>(p, tiles, ws, s) : launch_window_decode<T, false>(p, tiles, ws, s);
  });
}
