// The form of windowed paged prefill for short chunks (window_decode.cu), called by the entry point in
// varlen_prefill.cu, which has checked the arguments.
#pragma once

#include "common.cuh"

namespace aici {

// Work items of 16 rows (tokens x heads of a kv head) to a (sequence, kv head).
inline int64_t window_chunk_items(int64_t max_tokens, int64_t group) { return (max_tokens * group + 15) / 16; }

// Whether a call takes this form: chunks of at most 16 tokens, where an item does at least the work of a
// query head (64 sequences at context 8192, window 4096, us here and in the general kernel's 128-row tiles:
// 32 heads over 8, 4 tokens 166 and 807, 16 tokens 490 and 800, 32 tokens 973 and 630; 8 heads over 8, 16
// tokens 167 and 238, 32 tokens 280 and 217), or all items resident at once, two to an SM, since an item's
// keys are then dealt out to a cluster while a tile of the general kernel walks them alone (1 sequence, 32
// heads over 8, window 4096: 4 tokens 14 and 115, 64 tokens 41 and 85, 128 tokens = 256 items 71 and 81,
// 256 tokens = 512 items 140 and 81).
inline bool window_chunk_takes(int64_t batch, int64_t num_heads, int64_t num_kv_heads, int64_t max_tokens) {
  const int64_t items = batch * num_kv_heads * window_chunk_items(max_tokens, num_heads / num_kv_heads);
  return max_tokens <= 16 ? items < (1ll << 31) /* a grid's width */ : items <= 2 * sm_count();
}

struct WindowChunk {
  void *out;
  const void *q, *key_cache, *value_cache;
  const int32_t *cu_q, *context_lens, *block_tables;
  int batch, total_q, num_heads, num_kv_heads, max_tokens, max_context, max_blocks, window, sinks;
  int64_t num_blocks, q_tok, q_head, o_tok, o_head, kv_block;
  float scale;
  unsigned int *status;
};

char *launch_window_chunk(const WindowChunk &c, int dtype, cudaStream_t stream);

}  // namespace aici
