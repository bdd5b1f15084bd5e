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
// "chunk": the two 16-byte vectors at elements 8 c and rot_dim / 2 + 8 c of a head, which hold 8 pairs
// in either layout (half: one across the vectors; interleaved: four inside each), with their 8 cosines
// and 8 sines.  So every access is a whole vector and neighbouring threads take neighbouring vectors; it
// asks for rot_dim to be a multiple of 16.
#include <math.h>

#include "half_types.cuh"

namespace aici {

constexpr int kRotThreads = 256;
constexpr int kRotTok = 16;      // tokens of a cache-writing CTA: one cache block when they are aligned
constexpr int kRotBlock = 16;    // tokens of a cache block
constexpr int kMaxHead = 256;

// How the threads of a CTA share out the heads of whole tokens: thread = (token, head slot, chunk),
// chunk fastest, so that a warp reads runs of a row; a thread takes every slots-th head of its token.
struct HeadPlan {
  int slots, tokens;  // head slots, tokens of a CTA at a time
  int ctas;           // CTA i takes the i-th, (i + ctas)-th, ... such run of tokens
};

struct RotaryParams {
  const int64_t *positions;
  void *query, *key;
  const void *value, *table, *slots;
  void *key_cache, *value_cache;
  int num_tokens, num_heads, num_kv_heads, head_size, rot_dim, slot_is_int64;
  int64_t max_position, num_slots, query_stride, key_stride, value_stride;
  unsigned int *status;
  HeadPlan q_plan, k_plan;
  int kv_heads_per_cta;  // cache-writing CTAs: heads of one, one after the other
};

// Four neighbouring table entries.
__device__ __forceinline__ void load4(const float *src, float *x) {
  const float4 a = *reinterpret_cast<const float4 *>(src);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
}
template <typename T>
__device__ __forceinline__ void load4(const T *src, float *x) {
  const uint2 v = *reinterpret_cast<const uint2 *>(src);
  const float2 a = Half16<T>::unpack(v.x), b = Half16<T>::unpack(v.y);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
// Cosines and sines of chunk c from a row of the table: pairs 8 c .. 8 c + 7 (half), or 4 c .. 4 c + 3 and
// those rot_dim / 4 further on (interleaved).
template <typename C, bool kNeox>
__device__ __forceinline__ void load_turn(const C *row, int rot_dim, int c, float (&co)[8], float (&si)[8]) {
  const int a = kNeox ? 8 * c : 4 * c, b = kNeox ? a + 4 : a + rot_dim / 4;
  load4(row + a, co);
  load4(row + b, co + 4);
  load4(row + rot_dim / 2 + a, si);
  load4(row + rot_dim / 2 + b, si + 4);
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

// CTA `cta` of the plan: turns the heads of its tokens in place.  What bounds it is the chain position ->
// table row -> store: the position of a thread's next token is fetched a round ahead, so that in all
// rounds but the first the table row and four heads' vectors travel together.
template <typename T, typename C, bool kNeox>
__device__ __forceinline__ void turn_heads(T *rows, int64_t row_stride, int heads, const HeadPlan &plan, int cta,
                                           const RotaryParams &p) {
  constexpr int kAhead = 4;
  const int nc = p.rot_dim / 16;  // chunks of a head
  const int c = threadIdx.x % nc, rest = threadIdx.x / nc, slot = rest % plan.slots, tok = rest / plan.slots;
  if (tok >= plan.tokens) return;
  const int second = p.rot_dim / 2, stride = plan.ctas * plan.tokens;
  int t = cta * plan.tokens + tok;
  int64_t pos = t < p.num_tokens ? p.positions[t] : 0;
  for (; t < p.num_tokens; t += stride) {
    const int64_t next = t + stride < p.num_tokens ? p.positions[t + stride] : 0;
    if (pos >= 0 && pos < p.max_position) {
      T *x = rows + t * row_stride + c * 8;
      float co[8], si[8];
      for (int h0 = slot; h0 < heads; h0 += kAhead * plan.slots) {
        uint4 xv[kAhead], yv[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int h = h0 + k * plan.slots;
          if (h < heads) {
            xv[k] = *reinterpret_cast<const uint4 *>(x + (int64_t)h * p.head_size);
            yv[k] = *reinterpret_cast<const uint4 *>(x + (int64_t)h * p.head_size + second);
          }
        }
        if (h0 == slot)
          load_turn<C, kNeox>(static_cast<const C *>(p.table) + pos * p.rot_dim, p.rot_dim, c, co, si);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int h = h0 + k * plan.slots;
          if (h < heads) {
            turn<T, kNeox>(xv[k], yv[k], co, si);
            *reinterpret_cast<uint4 *>(x + (int64_t)h * p.head_size) = xv[k];
            *reinterpret_cast<uint4 *>(x + (int64_t)h * p.head_size + second) = yv[k];
          }
        }
      }
    } else {  // the token stays as it is
      set_status(p.status, AICI_STATUS_BAD_SLOT);
    }
    pos = next;
  }
}

template <typename T, typename C, bool kNeox>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryParams p) {
  const int b = blockIdx.x;
  if (b < p.q_plan.ctas)
    turn_heads<T, C, kNeox>(static_cast<T *>(p.query), p.query_stride, p.num_heads, p.q_plan, b, p);
  else
    turn_heads<T, C, kNeox>(static_cast<T *>(p.key), p.key_stride, p.num_kv_heads, p.k_plan, b - p.q_plan.ctas, p);
}

__device__ __forceinline__ void copy_async16(void *dst_smem, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst_smem)), "l"(src) : "memory");
}

// With the cache write.  The first CTAs take 16 tokens and some kv heads each, one head after the other:
// the key is turned, put back and written to the cache, the value goes through shared memory because the
// cache keeps it transposed ([d][token]).  The CTAs behind them turn the query heads.  Where a token goes
// and how far it turns does not change what is read, so a ring of kStages heads is filled by asynchronous
// copies from the start: what bounds this part is bytes in flight (4 KB of keys and of values per head, 72
// KB an SM with three heads ahead and three CTAs; with one head ahead the whole call took 85 us where it
// takes 77, 16384 tokens, 64/8 heads, half of each head rotated).  A thread keeps its token's cosines and
// sines for all its heads.  (A prompt that starts inside a block leaves value by value, 45 against 50 us
// at 8/8 heads; vectors for the half blocks inside a tile, or for those that reach into the next tile with
// the tokens they need fetched twice, were no faster.)
// kUnits: vectors of a key head that a thread handles (2 only for heads of more than 128 elements).
template <typename T, typename C, bool kNeox, int kUnits, int kStages>
__global__ void __launch_bounds__(kRotThreads, kUnits == 1 ? 3 : 2) rotary_cache_kernel(const RotaryParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int tiles = (p.num_tokens + kRotTok - 1) / kRotTok;
  const int groups = (p.num_kv_heads + p.kv_heads_per_cta - 1) / p.kv_heads_per_cta;
  if (blockIdx.x >= (unsigned)(tiles * groups)) {
    turn_heads<T, C, kNeox>(static_cast<T *>(p.query), p.query_stride, p.num_heads, p.q_plan,
                            blockIdx.x - tiles * groups, p);
    return;
  }
  __shared__ int64_t s_slot[kRotTok];
  const int h_begin = blockIdx.x % groups * p.kv_heads_per_cta, h_end = min(h_begin + p.kv_heads_per_cta, p.num_kv_heads);
  const int t0 = blockIdx.x / groups * kRotTok;
  const int tid = threadIdx.x, D = p.head_size, pitch = D + 8;
  const int tokens = min(kRotTok, p.num_tokens - t0);
  // stage of head h: keys [16][D + 8], then values
  auto stage = [&](int h) { return reinterpret_cast<T *>(smem) + (h - h_begin) % kStages * (2 * kRotTok * pitch); };
  auto fetch = [&](int h) {
    if (h < h_end) {
      T *dst = stage(h);
      for (int i = tid; i < tokens * (D / 8); i += kRotThreads) {
        const int tok = i / (D / 8), c = i - tok * (D / 8);
        const int64_t from = (int64_t)h * D + c * 8;
        copy_async16(dst + tok * pitch + c * 8, static_cast<const T *>(p.key) + (t0 + tok) * p.key_stride + from);
        copy_async16(dst + (kRotTok + tok) * pitch + c * 8,
                     static_cast<const T *>(p.value) + (t0 + tok) * p.value_stride + from);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) fetch(h_begin + s);

  const int tok = tid & (kRotTok - 1);
  int64_t slot = -1, pos = -1;
  if (tok < tokens) {
    slot = p.slot_is_int64 ? static_cast<const int64_t *>(p.slots)[t0 + tok]
                           : (int64_t) static_cast<const int32_t *>(p.slots)[t0 + tok];
    pos = p.positions[t0 + tok];
    const bool bad_pos = pos < 0 || pos >= p.max_position;  // the token stays as it is and is not written
    if (bad_pos || slot >= p.num_slots) {
      set_status(p.status, AICI_STATUS_BAD_SLOT);
      slot = -1;
      if (bad_pos) pos = -1;
    }
  }
  if (tid < kRotTok) s_slot[tid] = slot;
  // keys: 16 consecutive threads take the 16 tokens of one unit, so that the cache sees runs of 256
  // bytes.  Units are the chunks, then the vectors behind rot_dim.
  const int nc = p.rot_dim / 16, units = nc + (D - p.rot_dim) / 8;
  float co[kUnits][8], si[kUnits][8];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int u = tid / kRotTok + i * (kRotThreads / kRotTok);
    if (pos >= 0 && u < nc)
      load_turn<C, kNeox>(static_cast<const C *>(p.table) + pos * p.rot_dim, p.rot_dim, u, co[i], si[i]);
  }
  T *key = static_cast<T *>(p.key) + (t0 + tok) * p.key_stride;
  T *kc = static_cast<T *>(p.key_cache) +
          (slot >= 0 ? slot / kRotBlock * p.num_kv_heads * D * kRotBlock + slot % kRotBlock * 8 : 0);
  T *vc = static_cast<T *>(p.value_cache);
  uint32_t runs = 0;

  for (int h = h_begin; h < h_end; ++h) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();  // everybody's copies of this head have landed, and the stage refilled next is read
    fetch(h + kStages - 1);
    const T *s_k = stage(h), *s_v = s_k + kRotTok * pitch;
    if (pos >= 0) {
      T *to = kc + (int64_t)h * D * kRotBlock;  // vector e / 8 of the head: 16 tokens x 8 elements
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = tid / kRotTok + i * (kRotThreads / kRotTok);
        if (u < units) {
          const int e0 = u < nc ? u * 8 : p.rot_dim + (u - nc) * 8, e1 = e0 + p.rot_dim / 2;
          uint4 x = *reinterpret_cast<const uint4 *>(s_k + tok * pitch + e0), y = make_uint4(0, 0, 0, 0);
          if (u < nc) {
            y = *reinterpret_cast<const uint4 *>(s_k + tok * pitch + e1);
            turn<T, kNeox>(x, y, co[i], si[i]);
            *reinterpret_cast<uint4 *>(key + (int64_t)h * D + e0) = x;
            *reinterpret_cast<uint4 *>(key + (int64_t)h * D + e1) = y;
          }
          if (slot >= 0) {
            *reinterpret_cast<uint4 *>(to + e0 * kRotBlock) = x;
            if (u < nc) *reinterpret_cast<uint4 *>(to + e1 * kRotBlock) = y;
          }
        }
      }
    }
    // values: 8 tokens whose slots are consecutive and start at a multiple of 8 leave as one vector, any
    // others element by element with consecutive threads on consecutive tokens
    if (h == h_begin) {
#pragma unroll
      for (int g = 0; g < kRotTok / 8; ++g) {
        const int64_t s0 = s_slot[8 * g];
        bool run = s0 >= 0 && s0 % 8 == 0;
#pragma unroll
        for (int j = 1; j < 8; ++j) run = run && s_slot[8 * g + j] == s0 + j;
        runs |= (run ? 1u : 0u) << g;
      }
    }
    auto value_at = [&](int64_t s) { return vc + (s / kRotBlock * p.num_kv_heads + h) * D * kRotBlock + s % kRotBlock; };
    if (runs != 0u)
      for (int i = tid; i < 2 * D; i += kRotThreads) {  // both halves of a block's row side by side
        const int g = i & 1, d = i >> 1;
        if ((runs >> g) & 1u) {
          uint4 val;
          T *e = reinterpret_cast<T *>(&val);
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = s_v[(8 * g + j) * pitch + d];
          *reinterpret_cast<uint4 *>(value_at(s_slot[8 * g]) + d * kRotBlock) = val;
        }
      }
    if (runs != 3u && slot >= 0 && !((runs >> (tok / 8)) & 1u)) {
      T *dst = value_at(slot);
      for (int d = tid / kRotTok; d < D; d += kRotThreads / kRotTok) dst[d * kRotBlock] = s_v[tok * pitch + d];
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
  int walk;  // positions of a thread
};

__device__ __forceinline__ void put(float *dst, double x) { *dst = (float)x; }
__device__ __forceinline__ void put(__nv_bfloat16 *dst, double x) { *dst = __double2bfloat16(x); }
__device__ __forceinline__ void put(__half *dst, double x) { *dst = __double2half(x); }

// One thread walks p.walk positions of a pair (64, down to 4 where the table is short): sine and cosine of the first
// angle and of one position's turn by the library, the ones between by complex products in 64 bits (each costs a
// relative 2^-52, so 64 of them stay far below the 2^-24 of the result).  Computing every angle on its own costs some 100
// 64-bit operations an entry and takes seven times the store's time.
template <typename C>
__global__ void __launch_bounds__(kRotThreads) rotary_table_kernel(const __grid_constant__ TableParams p) {
  const int half = p.rot_dim / 2;
  const int64_t i = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  const int64_t run = i / half, pos0 = run * p.walk;
  const int j = (int)(i - run * half);
  if (pos0 >= p.max_position) return;
  const int n = (int)min((int64_t)p.walk, p.max_position - pos0);
  double s, c, ds, dc;
  sincos((double)pos0 * p.freq[j], &s, &c);
  sincos(p.freq[j], &ds, &dc);
  c *= p.by;  // the turns keep the length
  s *= p.by;
  C *row = static_cast<C *>(p.out) + pos0 * p.rot_dim + j;
  for (int k = 0; k < n; ++k) {
    put(row, c);
    put(row + half, s);
    const double t = c * dc - s * ds;
    s = s * dc + c * ds;
    c = t;
    row += p.rot_dim;
  }
}

// ---- host side -----------------------------------------------------------------------------------------
static char *check_rotary(const char *fn, const RotaryParams &p, int table_dtype, int dtype, bool cache) {
  AICI_CHECK(dtype == AICI_DTYPE_BF16 || dtype == AICI_DTYPE_F16, "%s: only bf16 and f16 are supported (dtype=%d)", fn,
             dtype);
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
  AICI_CHECK(p.num_tokens < (1 << 29) && (int64_t)(p.num_tokens / 16 + 1) * p.num_kv_heads < (1 << 30),
             "%s: too many tokens and heads for one call", fn);
  return nullptr;
}

// Few tokens: one head to a thread, so that more of the GPU takes part; many: four, which share the
// table row and are in flight together.
static HeadPlan plan_heads(int tokens, int heads, int rot_dim) {
  const int nc = rot_dim / 16, most = kRotThreads / nc;
  const int per = (int64_t)tokens * heads * nc >= (int64_t)4 * 4 * kRotThreads * sm_count() ? 4 : 1;
  HeadPlan plan;
  plan.slots = (heads + per - 1) / per < most ? (heads + per - 1) / per : most;
  plan.tokens = most / plan.slots;
  const int runs = (tokens + plan.tokens - 1) / plan.tokens;
  plan.ctas = per > 1 ? (runs + 3) / 4 : runs;
  return plan;
}

template <typename T, typename C, bool kNeox, int kUnits, int kStages>
static char *launch_rotary_cache(const RotaryParams &p, int grid, cudaStream_t stream) {
  // two tiles of 16 rows a stage; heads of up to 128 elements take four stages, larger ones two
  const size_t smem = (size_t)kStages * 2 * kRotTok * (p.head_size + 8) * sizeof(T);
  rotary_cache_kernel<T, C, kNeox, kUnits, kStages><<<grid, kRotThreads, smem, stream>>>(p);
  AICI_CUDA(cudaGetLastError());
  return nullptr;
}

template <typename T, typename C, bool kNeox>
static char *launch_rotary(RotaryParams p, bool cache, cudaStream_t stream) {
  p.q_plan = plan_heads(p.num_tokens, p.num_heads, p.rot_dim);
  p.k_plan = plan_heads(p.num_tokens, p.num_kv_heads, p.rot_dim);
  if (!cache) {
    rotary_kernel<T, C, kNeox><<<p.q_plan.ctas + p.k_plan.ctas, kRotThreads, 0, stream>>>(p);
  } else {
    const int tiles = (p.num_tokens + kRotTok - 1) / kRotTok;
    p.kv_heads_per_cta = 1;
    while (p.kv_heads_per_cta < 8 && (int64_t)tiles * p.num_kv_heads >= (int64_t)8 * p.kv_heads_per_cta * sm_count())
      p.kv_heads_per_cta *= 2;
    const int grid = tiles * ((p.num_kv_heads + p.kv_heads_per_cta - 1) / p.kv_heads_per_cta) + p.q_plan.ctas;
    const bool one = p.rot_dim / 16 + (p.head_size - p.rot_dim) / 8 <= kRotThreads / kRotTok;
    if (one && p.head_size <= 128) return launch_rotary_cache<T, C, kNeox, 1, 4>(p, grid, stream);
    if (one) return launch_rotary_cache<T, C, kNeox, 1, 2>(p, grid, stream);
    return launch_rotary_cache<T, C, kNeox, 2, 2>(p, grid, stream);
  }
  AICI_CUDA(cudaGetLastError());
  return nullptr;
}

static char *rotary_impl(const char *fn, RotaryParams p, int is_neox, int table_dtype, int dtype, bool cache,
                         aici_stream_t stream) {
  if (p.num_tokens <= 1) {  // the stride of a single token is never used and may be whatever a layout left there
    p.query_stride = (int64_t)p.num_heads * p.head_size;
    p.key_stride = p.value_stride = (int64_t)p.num_kv_heads * p.head_size;
  }
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
                    max_position, num_blocks * kRotBlock, query_stride, key_stride, value_stride, nullptr, {}, {}, 1};
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
  // base^(-2 j / rot_dim) = e^-x with x = 2 j ln(base) / rot_dim, which three roundings leave off by 3 x 2^-53:
  // relative error (3 x + 1) 2^-53, and as e^-x (3 x + 1) < 1.6 an angle is off by less than 1.6 x 2^-53 a position
  // (64 powers, at 2^-53, take the host 1 us longer)
  const double step = 2.0 * log(base) / rot_dim;
  for (int j = 0; j < rot_dim / 2; ++j) {
    double f = exp(-step * j);
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
  // 64 positions to a thread where that leaves eight warps per multiprocessor, fewer for short tables
  p.walk = 64;
  while (p.walk > 4 && max_position * (rot_dim / 2) < (int64_t)p.walk * 256 * sm_count()) p.walk /= 2;
  const int64_t grid = ((max_position + p.walk - 1) / p.walk * (rot_dim / 2) + kRotThreads - 1) / kRotThreads;
  AICI_CHECK(grid < (1ll << 31), "%s: table too large", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == AICI_DTYPE_F32) rotary_table_kernel<float><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
  else if (dtype == AICI_DTYPE_BF16) rotary_table_kernel<__nv_bfloat16><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
  else rotary_table_kernel<__half><<<(unsigned)grid, kRotThreads, 0, s>>>(p);
  AICI_CUDA(cudaGetLastError());
  return nullptr;
}
