// The form of windowed paged prefill for short chunks (window_decode.cu), called by the entry point in
// varlen_prefill.cu, which has checked the arguments.
#pragma once

#include "common.cuh"

namespace aici {

// Work items of 16 rows (tokens x heads of a kv head) to a (sequence, kv head).
inline int64_t window_chunk_items(int64_t max_tokens, int64_t group) { return (max_tokens * group + 15) / 16; }

constexpr int kWindowChunkTokens = 16;

// Whether a call takes this form: chunks of at most 16 tokens, where an item does at least the work of a
// query head (64 sequences at context 8192, window 4096, us here and in the general kernel's 128-row tiles:
// 32 heads over 8, 4 tokens 165 and 805, 16 tokens 492 and 799, 32 tokens 975 and 632; 8 heads over 8, 16
// tokens 166 and 239, 32 tokens 282 and 205), or all items resident at once, two to an SM, since an item's
// keys are then dealt out to a cluster while a tile of the general kernel walks them alone (1 sequence, 32
// heads over 8, window 4096: 4 tokens 14 and 115, 64 tokens 41 and 84, 128 tokens = 256 items 71 and 80,
// 256 tokens = 512 items 140 and 81).
inline bool window_chunk_takes(int64_t batch, int64_t num_heads, int64_t num_kv_heads, int64_t max_tokens) {
  const int64_t items = batch * num_kv_heads * window_chunk_items(max_tokens, num_heads / num_kv_heads);
  return max_tokens <= kWindowChunkTokens ? items < (1ll << 31) /* a grid's width */ : items <= 2 * sm_count();
}

// Whether, in a call that does not, the sequences of at most kWindowChunkTokens tokens get a launch of this
// form beside the general kernel's (a step of single tokens and some chunks).  The host knows no lengths: it
// does so where the mean is below half the longest, or no other sum is possible.  In us, with and without, at
// 32 heads over 8, context 6000, windows 128 and 4096: 63 single tokens and a chunk of 512: 46 and 107, 238 and
// 877; 15 and a chunk: 22 and 40, 96 and 310; 3 and a chunk: 19.6 and 17.4, 90 and 116; 4 chunks of 64 to 512, for
// which there is nothing to gain: 21.1 and 18.3, 92 and 90.
inline bool window_chunk_mixed(int64_t batch, int64_t total_q, int64_t max_tokens) {
  return 2 * total_q < batch * max_tokens || total_q < (kWindowChunkTokens + 1) * (batch - 1) + max_tokens;
}

struct WindowChunk {
  void *out;
  const void *q, *key_cache, *value_cache;
  const int32_t *cu_q, *context_lens, *block_tables;
  int batch, total_q, num_heads, num_kv_heads;
  int max_tokens;  // sequences with more are refused, or (beside) left out
  int max_context, max_blocks, window, sinks;
  int64_t num_blocks, q_tok, q_head, o_tok, o_head, kv_block;
  float scale;
  unsigned int *status;
  bool beside;  // the general kernel's launch follows and starts with it: begin behind all that came before
};

char *launch_window_chunk(const WindowChunk &c, int dtype, cudaStream_t stream);

}  // namespace aici
