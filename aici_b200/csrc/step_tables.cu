// The index tensors of one serving step built on the GPU from request lengths: running sums, the
// positions and cache slots of the step's tokens, and the block tables grown by the blocks that the
// new tokens begin.  The host-side counterpart is aici_batch_info_build (batch_info.cu), which starts
// from slot lists that a host allocator keeps; here lengths, tables and the free list live in device
// memory, so that a captured step can advance itself.
//
// With cu = running sums of query_lens, token t of request i (cu[i] <= t < cu[i + 1]) has position
// p = context_lens[i] + t - cu[i].  A request holds ceil(context_lens[i] / 16) blocks; a token with
// p % 16 == 0 begins a new one, and the k-th new block of the step, counted in token order, is
// free_blocks[free_count - 1 - k].  slot = block * 16 + p % 16.
//
// The work is a handful of dependent reads and writes of at most a megabyte: latency bounds it, and the
// instructions of the longest thread.  Every CTA reads all the lengths and computes both running sums
// (new tokens, new blocks) for itself in shared memory -- n values, which beats a hand-over between CTAs --
// then the CTAs share out the tokens.  Where an output is an input's own buffer (state that advances in
// place) nothing may be written before every CTA has read the lengths: then the grid is one cluster of up
// to 8 CTAs with its barrier between the two; otherwise it has as many CTAs as have tokens to work on.
#include "common.cuh"

namespace aici {

constexpr int kStepThreads = 512;   // of a CTA at most; half of them for small steps
constexpr int kStepWarps = kStepThreads / 32;
constexpr int kStepBatch = 4;       // lengths a thread loads at once, tokens it works on together
constexpr int kBlockTokens = 16;
constexpr int kMaxStepRequests = 16384;        // 12 bytes of shared memory each
constexpr int kMaxStepTokens = (1 << 30) - 1;
// Running sums saturate here: above every capacity a call can have, and twice it still fits 32 bits.
constexpr unsigned int kSumCap = 1u << 30;

struct StepParams {
  const int32_t *query_lens, *context_lens;
  int32_t *block_tables;
  const int32_t *free_blocks, *free_count;
  int32_t *seqlens_q, *slot_mapping, *logit_idxs, *context_out, *free_count_out;
  int64_t *positions;
  int n, max_blocks, max_tokens, free_capacity;
  int64_t num_blocks, table_stride;
  unsigned int *status;
};

__device__ __forceinline__ unsigned int sat_add(unsigned int a, unsigned int b) { return min(a + b, kSumCap); }

__global__ void __launch_bounds__(kStepThreads) step_tables_kernel(const StepParams p) {
  extern __shared__ __align__(16) int s_mem[];
  // running sums before request i (entry n: the totals), and the context length of request i
  unsigned int *s_tok = reinterpret_cast<unsigned int *>(s_mem);
  unsigned int *s_new = s_tok + p.n + 1;
  int *s_ctx = reinterpret_cast<int *>(s_new + p.n + 1);
  __shared__ unsigned int s_warp_tok[kStepWarps], s_warp_new[kStepWarps];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthreads = blockDim.x;
  const unsigned int rank = blockIdx.x, ctas = gridDim.x;
  if (tid == 0) s_bad = 0;
  __syncthreads();

  // ---- lengths: each thread a run of consecutive requests ------------------------------------------
  const int free_count = *p.free_count;
  const int per = (p.n + nthreads - 1) / nthreads;
  const int i0 = min(tid * per, p.n), i1 = min(i0 + per, p.n);
  const int64_t row_tokens = (int64_t)p.max_blocks * kBlockTokens;
  unsigned int tok = 0, fresh = 0;
  bool bad = free_count < 0 || free_count > p.free_capacity;
  for (int i = i0; i < i1; i += kStepBatch) {
    int q[kStepBatch], c[kStepBatch];
#pragma unroll
    for (int k = 0; k < kStepBatch; ++k) {
      q[k] = i + k < i1 ? p.query_lens[i + k] : 0;
      c[k] = i + k < i1 ? p.context_lens[i + k] : 0;
    }
#pragma unroll
    for (int k = 0; k < kStepBatch; ++k) {
      if (i + k >= i1) break;
      const bool wrong = q[k] < 0 || c[k] < 0 || (int64_t)c[k] + q[k] > row_tokens;
      bad |= wrong;
      s_ctx[i + k] = c[k];
      s_tok[i + k] = tok;  // relative to the thread's run; the runs before it are added below
      s_new[i + k] = fresh;
      if (!wrong) {
        tok = sat_add(tok, (unsigned int)q[k]);
        fresh = sat_add(fresh, (unsigned int)(((int64_t)c[k] + q[k] + kBlockTokens - 1) / kBlockTokens -
                                              ((int64_t)c[k] + kBlockTokens - 1) / kBlockTokens));
      }
    }
  }
  if (bad) s_bad = 1;
  unsigned int tok_incl = tok, new_incl = fresh;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned int a = __shfl_up_sync(0xffffffffu, tok_incl, o);
    const unsigned int b = __shfl_up_sync(0xffffffffu, new_incl, o);
    if (lane >= o) {
      tok_incl = sat_add(tok_incl, a);
      new_incl = sat_add(new_incl, b);
    }
  }
  if (lane == 31) {
    s_warp_tok[warp] = tok_incl;
    s_warp_new[warp] = new_incl;
  }
  __syncthreads();
  // every warp scans the warps' sums for itself
  unsigned int tok_warps = lane < nthreads / 32 ? s_warp_tok[lane] : 0u;
  unsigned int new_warps = lane < nthreads / 32 ? s_warp_new[lane] : 0u;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned int a = __shfl_up_sync(0xffffffffu, tok_warps, o);
    const unsigned int b = __shfl_up_sync(0xffffffffu, new_warps, o);
    if (lane >= o) {
      tok_warps = sat_add(tok_warps, a);
      new_warps = sat_add(new_warps, b);
    }
  }
  const unsigned int tok_total = __shfl_sync(0xffffffffu, tok_warps, 31);
  const unsigned int new_total = __shfl_sync(0xffffffffu, new_warps, 31);
  unsigned int tok_base = __shfl_sync(0xffffffffu, tok_warps, max(warp - 1, 0));
  unsigned int new_base = __shfl_sync(0xffffffffu, new_warps, max(warp - 1, 0));
  if (warp == 0) tok_base = new_base = 0;
  // the runs of the lower lanes of this warp
  const unsigned int tok_prev = __shfl_up_sync(0xffffffffu, tok_incl, 1);
  const unsigned int new_prev = __shfl_up_sync(0xffffffffu, new_incl, 1);
  if (lane > 0) {
    tok_base = sat_add(tok_base, tok_prev);
    new_base = sat_add(new_base, new_prev);
  }
  const bool no_blocks = new_total > (unsigned int)max(free_count, 0);
  const bool refused = s_bad || no_blocks || tok_total > (unsigned int)p.max_tokens;
  for (int i = i0; i < i1; ++i) {
    s_tok[i] = refused ? 0u : sat_add(s_tok[i], tok_base);
    s_new[i] = refused ? 0u : sat_add(s_new[i], new_base);
  }
  if (tid == 0) {
    s_tok[p.n] = refused ? 0u : tok_total;
    s_new[p.n] = refused ? 0u : new_total;
    if (refused && rank == 0) set_status(p.status, s_bad || !no_blocks ? AICI_STATUS_BAD_BLOCK : AICI_STATUS_NO_BLOCKS);
  }
  __syncthreads();
  // in place (the grid is a cluster): every CTA has read the lengths and the count once all have arrived here
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");

  // ---- tokens: four consecutive ones to a thread -----------------------------------------------------
  const int total = (int)s_tok[p.n];
  const int gid = rank * nthreads + tid, threads = ctas * nthreads;
  auto block_of = [&](int req, int ctx, int blk) -> const int32_t * {  // where the id of a request's block is
    const int held = (int)(((unsigned int)ctx + kBlockTokens - 1) / kBlockTokens);
    return blk < held ? p.block_tables + req * p.table_stride + blk
                      : p.free_blocks + (free_count - 1 - (int)(s_new[req] + (unsigned int)(blk - held)));
  };
  auto slot_of = [&](int id, int at) {
    if (id >= 0 && id < p.num_blocks) return id * kBlockTokens + at % kBlockTokens;
    set_status(p.status, AICI_STATUS_BAD_BLOCK);
    return -1;
  };
  // a token that begins a block enters it in the table, a bad id too: what the entry held before may be a block
  // of another request by now
  auto enter = [&](int req, int at, int id) {
    if (at % kBlockTokens == 0) p.block_tables[req * p.table_stride + at / kBlockTokens] = id;
  };
  for (int64_t t64 = (int64_t)kStepBatch * gid; t64 < p.max_tokens; t64 += (int64_t)kStepBatch * threads) {
    const unsigned int t0 = (unsigned int)t64;
    int pos0 = 0, pos1 = 0, pos2 = 0, pos3 = 0, slot0 = -1, slot1 = -1, slot2 = -1, slot3 = -1;
    if (t0 < (unsigned int)total) {
      // the request of the first token: the last i with s_tok[i] <= t0 (requests without tokens share
      // their start with the one behind them, and the last of those is the one that has tokens)
      int lo = 0, hi = p.n;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_tok[mid] <= t0) lo = mid;
        else hi = mid;
      }
      if (t0 + kStepBatch <= s_tok[lo + 1]) {
        // all of one request: at most two blocks
        const int ctx = s_ctx[lo];
        pos0 = ctx + (int)(t0 - s_tok[lo]);
        pos1 = pos0 + 1;
        pos2 = pos0 + 2;
        pos3 = pos0 + 3;
        const int b0 = pos0 / kBlockTokens, b1 = pos3 / kBlockTokens;
        const int id0 = *block_of(lo, ctx, b0), id1 = b1 != b0 ? *block_of(lo, ctx, b1) : id0;
        slot0 = slot_of(id0, pos0);
        slot1 = slot_of(pos1 / kBlockTokens == b0 ? id0 : id1, pos1);
        slot2 = slot_of(pos2 / kBlockTokens == b0 ? id0 : id1, pos2);
        slot3 = slot_of(id1, pos3);
        if (pos0 % kBlockTokens == 0 || b1 != b0) {
          const int begin = b1 * kBlockTokens;  // the block that begins within the four, at its first token
          enter(lo, begin, b1 != b0 ? id1 : id0);
        }
      } else {
        // tokens of several requests: where each one's id is, then all the ids at once
        int req0 = -1, req1 = -1, req2 = -1, req3 = -1;
        auto locate = [&](unsigned int t, int &req, int &pos) -> const int32_t * {
          if (t >= (unsigned int)total) return p.free_count;  // any readable word
          while (t >= s_tok[lo + 1]) ++lo;
          req = lo;
          pos = s_ctx[lo] + (int)(t - s_tok[lo]);
          return block_of(lo, s_ctx[lo], pos / kBlockTokens);
        };
        const int32_t *a0 = locate(t0, req0, pos0), *a1 = locate(t0 + 1, req1, pos1);
        const int32_t *a2 = locate(t0 + 2, req2, pos2), *a3 = locate(t0 + 3, req3, pos3);
        const int id0 = *a0, id1 = *a1, id2 = *a2, id3 = *a3;
        auto settle = [&](int req, int pos, int id, int &slot) {
          if (req < 0) return;
          slot = slot_of(id, pos);
          enter(req, pos, id);
        };
        settle(req0, pos0, id0, slot0);
        settle(req1, pos1, id1, slot1);
        settle(req2, pos2, id2, slot2);
        settle(req3, pos3, id3, slot3);
      }
    }
    if (t64 + kStepBatch <= p.max_tokens) {
      *reinterpret_cast<longlong2 *>(p.positions + t64) = make_longlong2(pos0, pos1);
      *reinterpret_cast<longlong2 *>(p.positions + t64 + 2) = make_longlong2(pos2, pos3);
      *reinterpret_cast<int4 *>(p.slot_mapping + t64) = make_int4(slot0, slot1, slot2, slot3);
    } else {
      const int left = (int)(p.max_tokens - t64);  // 1 to 3
      p.positions[t64] = pos0;
      p.slot_mapping[t64] = slot0;
      if (left > 1) {
        p.positions[t64 + 1] = pos1;
        p.slot_mapping[t64 + 1] = slot1;
      }
      if (left > 2) {
        p.positions[t64 + 2] = pos2;
        p.slot_mapping[t64 + 2] = slot2;
      }
    }
  }

  // ---- requests -------------------------------------------------------------------------------------
  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  for (int i = gid; i <= p.n; i += threads) {
    const unsigned int a = s_tok[i];
    p.seqlens_q[i] = (int)a;
    if (i < p.n) {
      const int q = (int)(s_tok[i + 1] - a);
      p.logit_idxs[i] = q > 0 ? (int)a + q - 1 : -1;
      p.context_out[i] = s_ctx[i] + q;
    }
  }
  if (gid == 0) *p.free_count_out = free_count - (int)s_new[p.n];
}

}  // namespace aici

using namespace aici;

extern "C" char *aici_step_tables(const int32_t *query_lens, const int32_t *context_lens,
                                  int32_t *block_tables, const int32_t *free_blocks,
                                  const int32_t *free_count, int num_requests, int max_blocks_per_seq,
                                  int64_t block_table_stride, int free_capacity, int64_t num_blocks,
                                  int block_size, int max_tokens, int32_t *seqlens_q, int64_t *positions,
                                  int32_t *slot_mapping, int32_t *logit_idxs, int32_t *context_lens_out,
                                  int32_t *free_count_out, aici_stream_t stream) {
  const char *fn = "aici_step_tables";
  AICI_CHECK(block_size == kBlockTokens, "%s: block_size must be 16 (got %d)", fn, block_size);
  AICI_CHECK(num_requests > 0 && num_requests <= kMaxStepRequests, "%s: num_requests must be 1..%d (got %d)", fn,
             kMaxStepRequests, num_requests);
  AICI_CHECK(max_blocks_per_seq > 0 && max_blocks_per_seq <= (1 << 27) - 1 && block_table_stride >= max_blocks_per_seq,
             "%s: bad block table width %d (row stride %lld)", fn, max_blocks_per_seq, (long long)block_table_stride);
  AICI_CHECK(max_tokens >= 0 && max_tokens <= kMaxStepTokens, "%s: bad max_tokens %d", fn, max_tokens);
  AICI_CHECK(free_capacity >= 0, "%s: negative size", fn);
  AICI_CHECK(num_blocks > 0 && num_blocks <= (1 << 27), "%s: num_blocks must be 1..2^27 (slots are 32 bits wide)", fn);
  AICI_CHECK(query_lens && context_lens && block_tables && free_count && seqlens_q && logit_idxs && context_lens_out &&
                 free_count_out,
             "%s: NULL pointer", fn);
  AICI_CHECK((free_blocks || free_capacity == 0) && ((positions && slot_mapping) || max_tokens == 0),
             "%s: NULL pointer", fn);
  AICI_CHECK(((uintptr_t)positions | (uintptr_t)slot_mapping) % 16 == 0,
             "%s: positions and slot_mapping must be 16-byte aligned", fn);
  if (char *e = check_on_current_device(fn, "block_tables", block_tables)) return e;
  unsigned int *st = status_ptr();
  AICI_CHECK(st != nullptr, "%s: no CUDA device", fn);
  static OncePerDevice once;
  if (char *e = once.run([]() -> char * {
        AICI_CUDA(cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (3 * kMaxStepRequests + 2) * (int)sizeof(int)));
        return nullptr;
      }))
    return e;
  StepParams p = {query_lens, context_lens, block_tables, free_blocks, free_count, seqlens_q, slot_mapping,
                  logit_idxs, context_lens_out, free_count_out, positions, num_requests, max_blocks_per_seq,
                  max_tokens, free_capacity, num_blocks, block_table_stride, st};
  auto meets = [](const void *a, int64_t na, const void *b, int64_t nb) {
    return (uintptr_t)a < (uintptr_t)b + 4 * nb && (uintptr_t)b < (uintptr_t)a + 4 * na;
  };
  bool in_place = false;
  const int32_t *outs[4] = {seqlens_q, logit_idxs, context_lens_out, free_count_out};
  const int64_t lens[4] = {num_requests + 1, num_requests, num_requests, 1};
  for (int i = 0; i < 4; ++i)
    in_place = in_place || meets(outs[i], lens[i], query_lens, num_requests) ||
               meets(outs[i], lens[i], context_lens, num_requests) || meets(outs[i], lens[i], free_count, 1);
  const int64_t work = (int64_t)max_tokens + num_requests;
  const int threads = work <= 2 * kStepThreads ? kStepThreads / 2 : kStepThreads;
  const int64_t most = in_place ? 8 : sm_count();
  int ctas = 1;
  while (2 * ctas <= most && work > (int64_t)kStepBatch * threads * ctas) ctas *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = in_place ? ctas : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (3 * (size_t)num_requests + 2) * sizeof(int);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AICI_CUDA(cudaLaunchKernelEx(&cfg, step_tables_kernel, p));
  return nullptr;
}
