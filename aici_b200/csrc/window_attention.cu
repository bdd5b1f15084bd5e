// Attention with a sliding window and a few first tokens that stay visible, over the paged cache and
// over packed keys and values.
//
// The query at position p of its sequence sees the tokens t <= p with t > p - window or t < sinks.
//     o = sum_t exp(scale q.k_t - m) v_t / sum_t exp(scale q.k_t - m),   m = max_t scale q.k_t
// One warp per (query row, head) walks the visible tokens with a running maximum and sum; four
// elements of the head to a lane.
#include "half_types.cuh"

namespace aici {

constexpr int kWinHead = 128;
constexpr int kWinBlock = 16;

struct WindowParams {
  void *out;
  const void *q, *k, *v;
  const int32_t *cu_q, *cu_k, *k_lens, *block_tables;  // cu_q NULL: one query per sequence
  int batch, num_heads, group, window, sinks, max_blocks, max_context;
  int64_t num_blocks, q_tok, q_head, o_tok, o_head, k_tok, k_head, v_tok, v_head, kv_block;
  float scale;
  unsigned int *status;
};

template <typename T, bool kPaged>
__global__ void __launch_bounds__(128) window_attention_kernel(const WindowParams p) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y, h = blockIdx.z;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int q0 = p.cu_q ? p.cu_q[b] : b, lq = p.cu_q ? p.cu_q[b + 1] - q0 : 1;
  if (r >= lq) return;
  int k0 = 0, lk;
  if (kPaged) {
    lk = p.k_lens[b];
    const int cap = min((int64_t)p.max_context, (int64_t)p.max_blocks * kWinBlock);
    if (lk > cap) {
      if (lane == 0) set_status(p.status, AICI_STATUS_BAD_BLOCK);
      lk = cap;
    }
  } else {
    k0 = p.cu_k[b];
    lk = p.cu_k[b + 1] - k0;
  }
  const int pos = lk - lq + r, kvh = h / p.group;
  const T *q = static_cast<const T *>(p.q) + (int64_t)(q0 + r) * p.q_tok + h * p.q_head + 4 * lane;
  const uint2 qv = *reinterpret_cast<const uint2 *>(q);
  const float2 qa = Half16<T>::unpack(qv.x), qb = Half16<T>::unpack(qv.y);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t = 0; t <= pos; ++t) {
    if (t >= p.sinks && t + (int64_t)p.window <= pos) {  // to the first token of the window
      t = pos - p.window + 1;
    }
    float kf[4], vf[4];
    if (kPaged) {
      int blk = p.block_tables[(int64_t)b * p.max_blocks + t / kWinBlock];
      if (blk < 0 || blk >= p.num_blocks) {
        if (lane == 0) set_status(p.status, AICI_STATUS_BAD_BLOCK);
        blk = 0;
      }
      const int64_t base = blk * p.kv_block + (int64_t)kvh * kWinHead * kWinBlock;
      const T *kc = static_cast<const T *>(p.k) + base + (lane / 2) * (kWinBlock * 8) + t % kWinBlock * 8 + (lane & 1) * 4;
      const uint2 kv = *reinterpret_cast<const uint2 *>(kc);
      const float2 a = Half16<T>::unpack(kv.x), c = Half16<T>::unpack(kv.y);
      kf[0] = a.x; kf[1] = a.y; kf[2] = c.x; kf[3] = c.y;
      const T *vc = static_cast<const T *>(p.v) + base + 4 * lane * kWinBlock + t % kWinBlock;
#pragma unroll
      for (int i = 0; i < 4; ++i) vf[i] = Half16<T>::to(vc[i * kWinBlock]);
    } else {
      const uint2 kv = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.k) + (int64_t)(k0 + t) * p.k_tok + kvh * p.k_head + 4 * lane);
      const uint2 vv = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.v) + (int64_t)(k0 + t) * p.v_tok + kvh * p.v_head + 4 * lane);
      const float2 a = Half16<T>::unpack(kv.x), c = Half16<T>::unpack(kv.y);
      const float2 d = Half16<T>::unpack(vv.x), e = Half16<T>::unpack(vv.y);
      kf[0] = a.x; kf[1] = a.y; kf[2] = c.x; kf[3] = c.y;
      vf[0] = d.x; vf[1] = d.y; vf[2] = e.x; vf[3] = e.y;
    }
    float s = qa.x * kf[0] + qa.y * kf[1] + qb.x * kf[2] + qb.y * kf[3];
#pragma unroll
    for (int i = 16; i >= 1; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s *= p.scale;
    const float mn = fmaxf(m, s), alpha = __expf(m - mn), e = __expf(s - mn);
    l = l * alpha + e;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * alpha + e * vf[i];
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + (int64_t)(q0 + r) * p.o_tok + h * p.o_head + 4 * lane) =
      make_uint2(Half16<T>::pack(o[0] * inv, o[1] * inv), Half16<T>::pack(o[2] * inv, o[3] * inv));
}

static char *launch_window(const WindowParams &p, bool paged, int max_q, int dtype, cudaStream_t stream) {
  const dim3 grid((max_q + 3) / 4, p.batch, p.num_heads);
  return with_half_type(dtype, [&](auto t) -> char * {
    using T = decltype(t);
    if (paged) window_attention_kernel<T, true><<<grid, 128, 0, stream>>>(p);
    else window_attention_kernel<T, false><<<grid, 128, 0, stream>>>(p);
    AICI_CUDA(cudaGetLastError());
    return nullptr;
  });
}

static char *check_window(const char *fn, int window, int sinks, int num_heads, int num_kv_heads, int head_size,
                          float scale, int dtype) {
  AICI_CHECK(dtype == AICI_DTYPE_BF16 || dtype == AICI_DTYPE_F16, "%s: only bf16 and f16 are supported (dtype=%d)", fn, dtype);
  AICI_CHECK(head_size == kWinHead, "%s: head_size must be 128 (got %d)", fn, head_size);
  AICI_CHECK(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
             "%s: num_heads %d not divisible by num_kv_heads %d", fn, num_heads, num_kv_heads);
  AICI_CHECK(window >= 1, "%s: window must be at least 1 (got %d)", fn, window);
  AICI_CHECK(sinks >= 0, "%s: sinks must not be negative (got %d)", fn, sinks);
  AICI_CHECK(scale > 0.f, "%s: softmax_scale must be positive", fn);
  return nullptr;
}

static char *check_cache(const char *fn, int block_size, int64_t num_blocks, int num_kv_heads, int64_t kv_block_stride,
                         int64_t kv_head_stride) {
  AICI_CHECK(block_size == kWinBlock, "%s: block_size must be 16 (got %d)", fn, block_size);
  AICI_CHECK(num_blocks > 0, "%s: num_blocks must be positive", fn);
  AICI_CHECK(kv_head_stride == kWinHead * kWinBlock && kv_block_stride % 8 == 0 &&
                 kv_block_stride >= (int64_t)num_kv_heads * kWinHead * kWinBlock,
             "%s: cache must be [blocks, kv_heads, 128/8, 16, 8] with contiguous head tiles", fn);
  return nullptr;
}

}  // namespace aici

using namespace aici;

extern "C" size_t aici_paged_attention_window_workspace_bytes(int num_seqs, int num_heads, int num_kv_heads,
                                                              int max_context_len, int window, int sinks) {
  return 256;
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
  if (char *e = check_window(fn, window, sinks, num_heads, num_kv_heads, head_size, scale, dtype)) return e;
  AICI_CHECK(num_heads / num_kv_heads <= 16, "%s: at most 16 query heads per kv head (got %d)", fn, num_heads / num_kv_heads);
  if (char *e = check_cache(fn, block_size, num_blocks, num_kv_heads, kv_block_stride, kv_head_stride)) return e;
  AICI_CHECK(num_seqs >= 0 && max_context_len >= 0 && max_num_blocks_per_seq >= 0, "%s: negative size", fn);
  AICI_CHECK(q_stride % 8 == 0 && q_stride >= (int64_t)num_heads * head_size,
             "%s: q_stride must be a multiple of 8 elements and cover one row", fn);
  if (num_seqs == 0) return nullptr;
  AICI_CHECK(out && query && key_cache && value_cache && block_tables && context_lens, "%s: NULL pointer", fn);
  AICI_CHECK(((uintptr_t)out | (uintptr_t)query | (uintptr_t)key_cache | (uintptr_t)value_cache) % 16 == 0,
             "%s: tensors must be 16-byte aligned", fn);
  if (char *e = check_on_current_device(fn, "query", query)) return e;
  unsigned int *st = status_ptr();
  AICI_CHECK(st != nullptr, "%s: no CUDA device", fn);
  WindowParams p = {};
  p.out = out;
  p.q = query;
  p.k = key_cache;
  p.v = value_cache;
  p.k_lens = context_lens;
  p.block_tables = block_tables;
  p.batch = num_seqs;
  p.num_heads = num_heads;
  p.group = num_heads / num_kv_heads;
  p.window = window;
  p.sinks = sinks;
  p.max_blocks = max_num_blocks_per_seq;
  p.max_context = max_context_len;
  p.num_blocks = num_blocks;
  p.q_tok = q_stride;
  p.q_head = head_size;
  p.o_tok = (int64_t)num_heads * head_size;
  p.o_head = head_size;
  p.kv_block = kv_block_stride;
  p.scale = scale;
  p.status = st;
  return launch_window(p, true, 1, dtype, static_cast<cudaStream_t>(stream));
}
