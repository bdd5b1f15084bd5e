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
// The work is a handful of dependent reads and writes of at most a megabyte: latency bounds it.  One
// cluster does it in one launch.  Every CTA reads all the lengths and computes both running sums (new
// tokens, new blocks) for itself in shared memory -- n values, which beats a hand-over between CTAs --
// then the CTAs share out the tokens.  The cluster barrier between "all lengths are read" and "the new
// lengths are written" is what lets the outputs be the inputs' own buffers.
#include "common.cuh"

namespace aici {

constexpr int kStepThreads = 512;
constexpr int kStepWarps = kStepThreads / 32;
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
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned int rank, ctas;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  if (tid == 0) s_bad = 0;
  __syncthreads();

  // ---- lengths: each thread a run of consecutive requests ------------------------------------------
  const int free_count = *p.free_count;
  const int per = (p.n + kStepThreads - 1) / kStepThreads;
  const int i0 = min(tid * per, p.n), i1 = min(i0 + per, p.n);
  const int64_t row_tokens = (int64_t)p.max_blocks * kBlockTokens;
  unsigned int tok = 0, fresh = 0;
  bool bad = free_count < 0 || free_count > p.free_capacity;
  for (int i = i0; i < i1; ++i) {
    const int q = p.query_lens[i], c = p.context_lens[i];
    const bool wrong = q < 0 || c < 0 || (int64_t)c + q > row_tokens;
    bad |= wrong;
    s_ctx[i] = c;
    s_tok[i] = tok;  // relative to the thread's run; the runs before it are added below
    s_new[i] = fresh;
    if (!wrong) {
      tok = sat_add(tok, (unsigned int)q);
      fresh = sat_add(fresh, (unsigned int)(((int64_t)c + q + kBlockTokens - 1) / kBlockTokens -
                                            ((int64_t)c + kBlockTokens - 1) / kBlockTokens));
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
  unsigned int tok_base = 0, new_base = 0, tok_total = 0, new_total = 0;
#pragma unroll
  for (int w = 0; w < kStepWarps; ++w) {
    if (w == warp) {
      tok_base = tok_total;
      new_base = new_total;
    }
    tok_total = sat_add(tok_total, s_warp_tok[w]);
    new_total = sat_add(new_total, s_warp_new[w]);
  }
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
  // every CTA has read the lengths and the count once all have arrived here
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");

  // ---- tokens: four consecutive ones to a thread -----------------------------------------------------
  const int total = (int)s_tok[p.n];
  const int gid = rank * kStepThreads + tid, threads = ctas * kStepThreads;
  for (int64_t t0 = 4 * (int64_t)gid; t0 < p.max_tokens; t0 += 4 * (int64_t)threads) {
    int64_t pos[4] = {0, 0, 0, 0};
    int slot[4] = {-1, -1, -1, -1};
    if (t0 < total) {
      // the request of the first token: the last i with s_tok[i] <= t0 (requests without tokens share
      // their start with the one behind them, and the last of those is the one that has tokens)
      int lo = 0, hi = p.n;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_tok[mid] <= (unsigned int)t0) lo = mid;
        else hi = mid;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned int t = (unsigned int)t0 + j;
        if (t < (unsigned int)total) {
          while (t >= s_tok[lo + 1]) ++lo;
          const int c = s_ctx[lo];
          const int at = c + (int)(t - s_tok[lo]);
          const int blk = at / kBlockTokens, held = (c + kBlockTokens - 1) / kBlockTokens;
          int32_t *entry = p.block_tables + lo * p.table_stride + blk;
          int id;
          if (blk < held) {
            id = *entry;
          } else {
            id = p.free_blocks[free_count - 1 - (int)(s_new[lo] + (unsigned int)(blk - held))];
            if (at % kBlockTokens == 0) *entry = id;
          }
          pos[j] = at;
          if (id >= 0 && id < p.num_blocks) slot[j] = id * kBlockTokens + at % kBlockTokens;
          else set_status(p.status, AICI_STATUS_BAD_BLOCK);
        }
      }
    }
    if (t0 + 4 <= p.max_tokens) {
      *reinterpret_cast<longlong2 *>(p.positions + t0) = make_longlong2(pos[0], pos[1]);
      *reinterpret_cast<longlong2 *>(p.positions + t0 + 2) = make_longlong2(pos[2], pos[3]);
      *reinterpret_cast<int4 *>(p.slot_mapping + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
      for (int j = 0; t0 + j < p.max_tokens; ++j) {
        p.positions[t0 + j] = pos[j];
        p.slot_mapping[t0 + j] = slot[j];
      }
    }
  }

  // ---- requests -------------------------------------------------------------------------------------
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
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  while (attr[0].val.clusterDim.x < 8 &&
         (int64_t)max_tokens + num_requests > (int64_t)4 * kStepThreads * attr[0].val.clusterDim.x)
    attr[0].val.clusterDim.x *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(attr[0].val.clusterDim.x);
  cfg.blockDim = dim3(kStepThreads);
  cfg.dynamicSmemBytes = (3 * (size_t)num_requests + 2) * sizeof(int);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AICI_CUDA(cudaLaunchKernelEx(&cfg, step_tables_kernel, p));
  return nullptr;
}
