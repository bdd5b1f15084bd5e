// Rotary positions in the general form: half or interleaved pairs, the whole head or its first
// rot_dim elements, cosine/sine tables in 32 bits (or the tensors' own type) that may be scaled for
// contexts longer than the trained one; alone, or in one pass with the cache write.
//
// For a token at position p and pair j (half: elements j and j + rot_dim / 2; interleaved: 2 j and
// 2 j + 1), with c = table[p][j] and s = table[p][rot_dim / 2 + j]:
//     u = a c - b s,   v = b c + a s
// computed in fp32 and rounded once to the tensors' type (the bf16-only entry point in cache_ops.cu
// follows the reference kernel, which rounds every product).
//
// Everything here is data movement with a handful of operations per 16 bytes.  A unit of work is a
// "chunk": 8 pairs = two 16-byte vectors of a head (half: chunk c of each half; interleaved: 16
// neighbouring elements) with their 8 cosines and 8 sines, so every access is a whole vector whatever
// the layout; it asks for rot_dim to be a multiple of 16.
#include <math.h>

#include "half_types.cuh"

namespace aici {

constexpr int kRotThreads = 256;
constexpr int kRotTok = 16;      // tokens of a cache-writing CTA: one cache block when they are aligned
constexpr int kRotBlock = 16;    // tokens of a cache block
constexpr int kMaxHead = 256;

struct RotaryParams {
  const int64_t *positions;
  void *query, *key;
  const void *value, *table, *slots;
  void *key_cache, *value_cache;
  int num_tokens, num_heads, num_kv_heads, head_size, rot_dim, slot_is_int64;
  int64_t max_position, num_slots, query_stride, key_stride, value_stride;
  unsigned int *status;
};

__device__ __forceinline__ void load8(const float *src, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T *src, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4 *>(src);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Half16<T>::unpack(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Turns one chunk: xv, yv are its two vectors, c and s its cosines and sines.
template <typename T, bool kNeox>
__device__ __forceinline__ void turn(uint4 &xv, uint4 &yv, const float (&c)[8], const float (&s)[8]) {
  uint32_t x[4] = {xv.x, xv.y, xv.z, xv.w}, y[4] = {yv.x, yv.y, yv.z, yv.w};
  if (kNeox) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = Half16<T>::unpack(x[i]), b = Half16<T>::unpack(y[i]);
      x[i] = Half16<T>::pack(a.x * c[2 * i] - b.x * s[2 * i], a.y * c[2 * i + 1] - b.y * s[2 * i + 1]);
      y[i] = Half16<T>::pack(b.x * c[2 * i] + a.x * s[2 * i], b.y * c[2 * i + 1] + a.y * s[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = Half16<T>::unpack(x[i]), b = Half16<T>::unpack(y[i]);
      x[i] = Half16<T>::pack(a.x * c[i] - a.y * s[i], a.y * c[i] + a.x * s[i]);
      y[i] = Half16<T>::pack(b.x * c[4 + i] - b.y * s[4 + i], b.y * c[4 + i] + b.x * s[4 + i]);
    }
  }
  xv = make_uint4(x[0], x[1], x[2], x[3]);
  yv = make_uint4(y[0], y[1], y[2], y[3]);
}

// The heads of one token, turned in place: threads along (head, chunk), chunk fastest, so a warp reads
// whole rows and the cosines and sines come out of the L1.
template <typename T, typename C, bool kNeox>
__device__ __forceinline__ void turn_heads(T *row, int heads, const C *cs, const RotaryParams &p, int tid) {
  const int nc = p.rot_dim / 16;  // chunks of a head
  const int second = kNeox ? p.rot_dim / 2 : 8;
  for (int i = tid; i < heads * nc; i += kRotThreads) {
    const int h = i / nc, c = i - h * nc;
    T *x = row + (int64_t)h * p.head_size + c * (kNeox ? 8 : 16);
    uint4 xv = *reinterpret_cast<const uint4 *>(x), yv = *reinterpret_cast<const uint4 *>(x + second);
    float co[8], si[8];
    load8(cs + c * 8, co);
    load8(cs + p.rot_dim / 2 + c * 8, si);
    turn<T, kNeox>(xv, yv, co, si);
    *reinterpret_cast<uint4 *>(x) = xv;
    *reinterpret_cast<uint4 *>(x + second) = yv;
  }
}

// One CTA to a token: query heads, and the key heads behind them.
template <typename T, typename C, bool kNeox>
__device__ __forceinline__ void rotate_token(const RotaryParams &p, int t, bool with_key) {
  const int64_t pos = p.positions[t];
  if (pos < 0 || pos >= p.max_position) {  // the token stays as it is
    if (threadIdx.x == 0) set_status(p.status, AICI_STATUS_BAD_SLOT);
    return;
  }
  const C *cs = static_cast<const C *>(p.table) + pos * p.rot_dim;
  turn_heads<T, C, kNeox>(static_cast<T *>(p.query) + t * p.query_stride, p.num_heads, cs, p, threadIdx.x);
  if (with_key)
    turn_heads<T, C, kNeox>(static_cast<T *>(p.key) + t * p.key_stride, p.num_kv_heads, cs, p, threadIdx.x);
}

template <typename T, typename C, bool kNeox>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryParams p) {
  rotate_token<T, C, kNeox>(p, blockIdx.x, true);
}

// With the cache write.  The first CTAs take 16 tokens of one kv head each: the key is turned, put
// back and written to the cache, the value goes through shared memory because the cache keeps it
// transposed ([d][token]).  The CTAs behind them turn the query heads, one token each.
template <typename T, typename C, bool kNeox>
__global__ void __launch_bounds__(kRotThreads) rotary_cache_kernel(const RotaryParams p) {
  const int tiles = (p.num_tokens + kRotTok - 1) / kRotTok;
  if (blockIdx.x >= (unsigned)(tiles * p.num_kv_heads)) {
    rotate_token<T, C, kNeox>(p, blockIdx.x - tiles * p.num_kv_heads, false);
    return;
  }
  __shared__ int64_t s_slot[kRotTok], s_pos[kRotTok];
  __shared__ __align__(16) T s_v[kRotTok][kMaxHead + 8];
  const int h = blockIdx.x % p.num_kv_heads, t0 = blockIdx.x / p.num_kv_heads * kRotTok;
  const int tid = threadIdx.x, D = p.head_size;
  const int tokens = min(kRotTok, p.num_tokens - t0);
  if (tid < kRotTok) {
    int64_t slot = -1, pos = -1;
    if (tid < tokens) {
      slot = p.slot_is_int64 ? static_cast<const int64_t *>(p.slots)[t0 + tid]
                             : (int64_t) static_cast<const int32_t *>(p.slots)[t0 + tid];
      if (slot >= p.num_slots) {
        set_status(p.status, AICI_STATUS_BAD_SLOT);
        slot = -1;
      }
      pos = p.positions[t0 + tid];
      if (pos < 0 || pos >= p.max_position) {  // the token stays as it is and is not written
        set_status(p.status, AICI_STATUS_BAD_SLOT);
        pos = -1;
        slot = -1;
      }
    }
    s_slot[tid] = slot;
    s_pos[tid] = pos;
  }
  for (int i = tid; i < tokens * (D / 8); i += kRotThreads) {
    const int tok = i / (D / 8), c = i - tok * (D / 8);
    *reinterpret_cast<uint4 *>(&s_v[tok][c * 8]) = *reinterpret_cast<const uint4 *>(
        static_cast<const T *>(p.value) + (t0 + tok) * p.value_stride + (int64_t)h * D + c * 8);
  }
  __syncthreads();

  // keys: 16 consecutive threads take the 16 tokens of one chunk, so that the cache sees runs of 256
  // bytes.  The chunks behind rot_dim are copied.
  const int nc = p.rot_dim / 16, rest = (D - p.rot_dim) / 8;
  const int tok = tid & (kRotTok - 1);
  if (tok < tokens && s_pos[tok] >= 0) {
    T *k = static_cast<T *>(p.key) + (t0 + tok) * p.key_stride + (int64_t)h * D;
    const C *cs = static_cast<const C *>(p.table) + s_pos[tok] * p.rot_dim;
    const int64_t slot = s_slot[tok];
    T *kc = static_cast<T *>(p.key_cache) +
            (slot >= 0 ? (slot / kRotBlock * p.num_kv_heads + h) * D * kRotBlock + slot % kRotBlock * 8 : 0);
    for (int c = tid / kRotTok; c < nc + rest; c += kRotThreads / kRotTok) {
      if (c < nc) {
        const int e0 = kNeox ? c * 8 : c * 16, e1 = e0 + (kNeox ? p.rot_dim / 2 : 8);
        uint4 xv = *reinterpret_cast<const uint4 *>(k + e0), yv = *reinterpret_cast<const uint4 *>(k + e1);
        float co[8], si[8];
        load8(cs + c * 8, co);
        load8(cs + p.rot_dim / 2 + c * 8, si);
        turn<T, kNeox>(xv, yv, co, si);
        *reinterpret_cast<uint4 *>(k + e0) = xv;
        *reinterpret_cast<uint4 *>(k + e1) = yv;
        if (slot >= 0) {
          *reinterpret_cast<uint4 *>(kc + e0 * kRotBlock) = xv;  // vector e / 8 of the head: 16 tokens x 8 elements each
          *reinterpret_cast<uint4 *>(kc + e1 * kRotBlock) = yv;
        }
      } else if (slot >= 0) {
        const int e = p.rot_dim + (c - nc) * 8;
        *reinterpret_cast<uint4 *>(kc + e * kRotBlock) = *reinterpret_cast<const uint4 *>(k + e);
      }
    }
  }

  // values: 8 tokens whose slots are consecutive and start at a multiple of 8 leave as one vector, any
  // others element by element with consecutive threads on consecutive tokens
  T *vc = static_cast<T *>(p.value_cache);
  bool run[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int64_t s0 = s_slot[8 * g];
    run[g] = s0 >= 0 && s0 % 8 == 0;
#pragma unroll
    for (int j = 1; j < 8; ++j) run[g] = run[g] && s_slot[8 * g + j] == s0 + j;
  }
  for (int i = tid; i < 2 * D; i += kRotThreads) {
    const int g = i >= D, d = g ? i - D : i;
    if (g ? run[1] : run[0]) {
      uint4 val;
      T *e = reinterpret_cast<T *>(&val);
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = s_v[8 * g + j][d];
      const int64_t s0 = s_slot[8 * g];
      *reinterpret_cast<uint4 *>(vc + (s0 / kRotBlock * p.num_kv_heads + h) * D * kRotBlock + d * kRotBlock +
                                 s0 % kRotBlock) = val;
    }
  }
  if (!run[0] || !run[1]) {
    const int64_t slot = s_slot[tok];
    if (slot >= 0 && !(tok < 8 ? run[0] : run[1])) {
      T *dst = vc + (slot / kRotBlock * p.num_kv_heads + h) * D * kRotBlock + slot % kRotBlock;
      for (int d = tid / kRotTok; d < D; d += kRotThreads / kRotTok) dst[d * kRotBlock] = s_v[tok][d];
    }
  }
}

// ---- the table ---------------------------------------------------------------------------------------
struct TableParams {
  double freq[kMaxHead / 2];  // angle per position of each pair
  double by;                  // factor on cosine and sine
  void *out;
  int64_t max_position;
  int rot_dim;
};

__device__ __forceinline__ void put(float *dst, double x) { *dst = (float)x; }
__device__ __forceinline__ void put(__nv_bfloat16 *dst, double x) { *dst = __double2bfloat16(x); }
__device__ __forceinline__ void put(__half *dst, double x) { *dst = __double2half(x); }

template <typename C>
__global__ void __launch_bounds__(kRotThreads) rotary_table_kernel(const __grid_constant__ TableParams p) {
  const int half = p.rot_dim / 2;
  const int64_t i = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  const int64_t pos = i / half;
  const int j = (int)(i - pos * half);
  if (pos >= p.max_position) return;
  double s, c;
  sincos((double)pos * p.freq[j], &s, &c);
  C *row = static_cast<C *>(p.out) + pos * p.rot_dim;
  put(row + j, c * p.by);
  put(row + half + j, s * p.by);
}

// ---- host side -----------------------------------------------------------------------------------------
static char *check_rotary(const char *fn, const RotaryParams &p, int table_dtype, int dtype, bool cache) {
  AICI_CHECK(dtype == AICI_DTYPE_BF16 || dtype == AICI_DTYPE_F16, "%s: only bf16 and f16 are supported (dtype=%d)", fn, dtype);
  AICI_CHECK(table_dtype == AICI_DTYPE_F32 || table_dtype == dtype,
             "%s: cos_sin_cache must be f32 or of the query's type (dtype=%d)", fn, table_dtype);
  AICI_CHECK(p.head_size > 0 && p.head_size % 16 == 0 && p.head_size <= kMaxHead,
             "%s: head_size must be a multiple of 16 up to %d (got %d)", fn, kMaxHead, p.head_size);
  AICI_CHECK(p.rot_dim > 0 && p.rot_dim % 16 == 0 && p.rot_dim <= p.head_size,
             "%s: rot_dim must be a multiple of 16 up to head_size (got %d)", fn, p.rot_dim);
  AICI_CHECK(p.num_tokens >= 0 && p.num_heads > 0 && p.num_kv_heads > 0 && p.max_position > 0, "%s: bad sizes", fn);
  AICI_CHECK(p.query_stride % 8 == 0 && p.key_stride % 8 == 0 &&
                 p.query_stride >= (int64_t)p.num_heads * p.head_size &&
                 p.key_stride >= (int64_t)p.num_kv_heads * p.head_size,
             "%s: token strides must be multiples of 8 elements and cover one row", fn);
  if (p.num_tokens == 0) return nullptr;
  AICI_CHECK(p.positions && p.query && p.key && p.table, "%s: NULL pointer", fn);
  AICI_CHECK(((uintptr_t)p.query | (uintptr_t)p.key | (uintptr_t)p.table) % 16 == 0,
             "%s: tensors must be 16-byte aligned", fn);
  if (cache) {
    AICI_CHECK(p.value && p.key_cache && p.value_cache && p.slots, "%s: NULL pointer", fn);
    AICI_CHECK(((uintptr_t)p.value | (uintptr_t)p.key_cache | (uintptr_t)p.value_cache) % 16 == 0,
               "%s: tensors must be 16-byte aligned", fn);
    AICI_CHECK(p.value_stride % 8 == 0 && p.value_stride >= (int64_t)p.num_kv_heads * p.head_size,
               "%s: token strides must be multiples of 8 elements and cover one row", fn);
    AICI_CHECK(p.num_slots > 0, "%s: num_blocks must be positive", fn);
  }
  const int64_t tiles = (p.num_tokens + kRotTok - 1) / kRotTok;
  AICI_CHECK(tiles * p.num_kv_heads + p.num_tokens < (1ll << 31), "%s: too many tokens and heads for one call", fn);
  return nullptr;
}

template <typename T, typename C, bool kNeox>
static char *launch_rotary(const RotaryParams &p, bool cache, cudaStream_t stream) {
  if (cache) {
    const int tiles = (p.num_tokens + kRotTok - 1) / kRotTok;
    rotary_cache_kernel<T, C, kNeox><<<tiles * p.num_kv_heads + p.num_tokens, kRotThreads, 0, stream>>>(p);
  } else {
    rotary_kernel<T, C, kNeox><<<p.num_tokens, kRotThreads, 0, stream>>>(p);
  }
  AICI_CUDA(cudaGetLastError());
  return nullptr;
}

static char *rotary_impl(const char *fn, RotaryParams p, int is_neox, int table_dtype, int dtype, bool cache,
                         aici_stream_t stream) {
  if (char *e = check_rotary(fn, p, table_dtype, dtype, cache)) return e;
  if (p.num_tokens == 0) return nullptr;
  if (char *e = check_on_current_device(fn, "query", p.query)) return e;
  p.status = status_ptr();
  AICI_CHECK(p.status != nullptr, "%s: no CUDA device", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return with_half_type(dtype, [&](auto t) -> char * {
    using T = decltype(t);
    if (table_dtype == AICI_DTYPE_F32)
      return is_neox ? launch_rotary<T, float, true>(p, cache, s) : launch_rotary<T, float, false>(p, cache, s);
    return is_neox ? launch_rotary<T, T, true>(p, cache, s) : launch_rotary<T, T, false>(p, cache, s);
  });
}

}  // namespace aici

using namespace aici;

extern "C" char *aici_rotary_embedding(const int64_t *positions, void *query, void *key, const void *cos_sin_cache,
                                       int num_tokens, int num_heads, int num_kv_heads, int head_size, int rot_dim,
                                       int is_neox, int64_t max_position, int64_t query_stride, int64_t key_stride,
                                       int table_dtype, int dtype, aici_stream_t stream) {
  RotaryParams p = {};
  p.positions = positions;
  p.query = query;
  p.key = key;
  p.table = cos_sin_cache;
  p.num_tokens = num_tokens;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.head_size = head_size;
  p.rot_dim = rot_dim;
  p.max_position = max_position;
  p.query_stride = query_stride;
  p.key_stride = key_stride;
  return rotary_impl("aici_rotary_embedding", p, is_neox, table_dtype, dtype, false, stream);
}

extern "C" char *aici_rotary_embedding_and_cache(const int64_t *positions, void *query, void *key, const void *value,
                                                 const void *cos_sin_cache, void *key_cache, void *value_cache,
                                                 const void *slot_mapping, int slot_is_int64, int num_tokens,
                                                 int num_heads, int num_kv_heads, int head_size, int rot_dim,
                                                 int is_neox, int64_t max_position, int block_size,
                                                 int64_t num_blocks, int64_t query_stride, int64_t key_stride,
                                                 int64_t value_stride, int table_dtype, int dtype,
                                                 aici_stream_t stream) {
  const char *fn = "aici_rotary_embedding_and_cache";
  AICI_CHECK(block_size == kRotBlock, "%s: block_size must be 16 (got %d)", fn, block_size);
  RotaryParams p = {positions, query, key, value, cos_sin_cache, slot_mapping, key_cache, value_cache,
                    num_tokens, num_heads, num_kv_heads, head_size, rot_dim, slot_is_int64,
                    max_position, num_blocks * kRotBlock, query_stride, key_stride, value_stride, nullptr};
  return rotary_impl(fn, p, is_neox, table_dtype, dtype, true, stream);
}

extern "C" char *aici_rotary_cos_sin_cache(void *out, int64_t max_position, int rot_dim, double base, int scaling,
                                           double factor, int64_t original_context, int dtype,
                                           aici_stream_t stream) {
  const char *fn = "aici_rotary_cos_sin_cache";
  AICI_CHECK(dtype == AICI_DTYPE_F32 || dtype == AICI_DTYPE_BF16 || dtype == AICI_DTYPE_F16, "%s: unsupported dtype %d",
             fn, dtype);
  AICI_CHECK(rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= kMaxHead, "%s: rot_dim must be even and at most %d (got %d)",
             fn, kMaxHead, rot_dim);
  AICI_CHECK(max_position >= 0 && max_position <= (1ll << 31), "%s: max_position must be 0..2^31", fn);
  AICI_CHECK(base > 1.0 && isfinite(base), "%s: base must be above 1", fn);
  AICI_CHECK(scaling >= AICI_ROPE_NONE && scaling <= AICI_ROPE_YARN, "%s: unknown scaling %d", fn, scaling);
  AICI_CHECK(scaling == AICI_ROPE_NONE || (factor >= 1.0 && isfinite(factor)), "%s: factor must be at least 1", fn);
  AICI_CHECK(scaling != AICI_ROPE_YARN || original_context > 0, "%s: original_context must be positive", fn);
  if (max_position == 0) return nullptr;
  AICI_CHECK(out != nullptr, "%s: NULL pointer", fn);
  if (char *e = check_on_current_device(fn, "out", out)) return e;
  TableParams p;
  p.by = 1.0;
  p.out = out;
  p.max_position = max_position;
  p.rot_dim = rot_dim;
  const double two_pi = 6.283185307179586476925286766559;
  if (scaling == AICI_ROPE_NTK) base *= pow(factor, (double)rot_dim / (rot_dim > 2 ? rot_dim - 2 : 1));
  if (scaling == AICI_ROPE_YARN) p.by = 0.1 * log(factor) + 1.0;
  for (int j = 0; j < rot_dim / 2; ++j) {
    double f = pow(base, -2.0 * j / rot_dim);
    if (scaling == AICI_ROPE_LINEAR) f /= factor;
    if (scaling == AICI_ROPE_YARN) {
      // Peng et al., "YaRN" (2023): pairs that turn more than 32 times within the original context
      // keep their frequency, those that turn less than once are stretched by `factor`, the ones
      // between are mixed linearly in the number of turns; cosine and sine carry 0.1 ln(factor) + 1
      const double turns = original_context * f / two_pi;
      const double keep = fmin(fmax((turns - 1.0) / 31.0, 0.0), 1.0);
      f = f * (keep + (1.0 - keep) / factor);
    }
    p.freq[j] = f;
  }
  const int64_t grid = (max_position * (rot_dim / 2) + kRotThreads - 1) / kRotThreads;
  AICI_CHECK(grid < (1ll << 31), "%s: table too large", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == AICI_DTYPE_F32) rotary_table_kernel<float><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
  else if (dtype == AICI_DTYPE_BF16) rotary_table_kernel<__nv_bfloat16><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
  else rotary_table_kernel<__half><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
  AICI_CUDA(cudaGetLastError());
  return nullptr;
}
