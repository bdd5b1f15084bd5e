// Calls at the limits of what the windowed operators' C++ host side (include/aici_b200_tch.hpp) is told:
// stated lengths that do not cover the sequences, strides of a single row.  Exit code = number of failures.
#include <cstdio>
#include <cstring>
#include <vector>

#include "aici_b200_tch.hpp"

namespace t = aici::tch;
using t::Kind;
using t::Tensor;

constexpr int H = 2, D = 128, T = 50;
constexpr uint16_t kOne = 0x3f80, kTwo = 0x4000;  // bf16

template <typename E>
static Tensor up(const std::vector<E> &h, std::vector<int64_t> sizes, Kind kind) {
  Tensor d = Tensor::empty(std::move(sizes), kind, 0);
  t::cuda_check("up", cudaMemcpy(d.data, h.data(), h.size() * sizeof(E), cudaMemcpyHostToDevice));
  return d;
}
static std::vector<uint16_t> down(const Tensor &d) {
  std::vector<uint16_t> h((size_t)d.numel());
  t::cuda_check("down", cudaDeviceSynchronize());
  t::cuda_check("down", cudaMemcpy(h.data(), d.data, h.size() * 2, cudaMemcpyDeviceToHost));
  return h;
}

static int fails = 0;
static void expect(bool ok, const char *what) {
  if (!ok) {
    std::printf("[ FAIL ] %s\n", what);
    ++fails;
  }
}
// Rows [a, b) all hold `value`.
static bool rows_are(const std::vector<uint16_t> &o, int a, int b, uint16_t value) {
  for (size_t i = (size_t)a * H * D; i < (size_t)b * H * D; ++i)
    if (o[i] != value) return false;
  return true;
}

// Two sequences of 40 and 10 tokens, queries and keys of ones, values of ones and of twos: every row of a
// sequence is its value.
struct Batch {
  Tensor q, v, kc, vc, cu, ctx, bt;
  Batch() {
    std::vector<uint16_t> ones((size_t)T * H * D, kOne), values(ones);
    for (size_t i = (size_t)40 * H * D; i < values.size(); ++i) values[i] = kTwo;
    q = up(ones, {T, H, D}, Kind::BFloat16);
    v = up(values, {T, H, D}, Kind::BFloat16);
    cu = up(std::vector<int32_t>{0, 40, 50}, {3}, Kind::Int);
    ctx = up(std::vector<int32_t>{40, 10}, {2}, Kind::Int);
    bt = up(std::vector<int32_t>{0, 1, 2, 3, 0, 0}, {2, 3}, Kind::Int);  // blocks 0-2 and 3
    std::vector<uint16_t> keys((size_t)4 * H * D * 16, kOne), cache(keys);
    for (size_t i = (size_t)3 * H * D * 16; i < cache.size(); ++i) cache[i] = kTwo;
    kc = up(keys, {4, H, D / 8, 16, 8}, Kind::BFloat16);
    vc = up(cache, {4, H, D, 16}, Kind::BFloat16);
  }
  std::vector<uint16_t> packed(size_t max_q, size_t max_k) const {
    return down(t::flash_attn_varlen_window(q, q, v, cu, cu, max_q, max_k, 0.01f, 9));
  }
  std::vector<uint16_t> paged(size_t max_q, size_t max_k) const {
    return down(t::flash_attn_varlen_paged_window(q, kc, vc, cu, ctx, bt, max_q, max_k, 0.01f, 9));
  }
};

static void stated_lengths(const Batch &b) {
  for (int form = 0; form < 2; ++form) {
    auto call = [&](size_t max_q, size_t max_k) { return form == 0 ? b.packed(max_q, max_k) : b.paged(max_q, max_k); };
    std::vector<uint16_t> o = call(40, 40);
    expect(rows_are(o, 0, 40, kOne) && rows_are(o, 40, 50, kTwo) && t::last_status() == 0, "lengths as they are");
    for (size_t most : {(size_t)1 << 31, (size_t)1 << 32, ((size_t)1 << 32) + 5}) {
      o = call(most, most);
      expect(rows_are(o, 0, 40, kOne) && rows_are(o, 40, 50, kTwo) && t::last_status() == 0, "lengths beyond 32 bits");
    }
    o = call(12, 40);
    expect(rows_are(o, 0, 40, 0) && rows_are(o, 40, 50, kTwo), "a sequence longer than stated");
    expect(t::last_status() == AICI_STATUS_BAD_BLOCK, "its status");
    o = call(0, 0);
    expect(rows_are(o, 0, 50, 0) && t::last_status() == 0, "a call without tokens");
  }
}

// One query token of one sequence, its first stride left from another layout.
static void single_rows(const Batch &b) {
  std::vector<int32_t> one = {0, 1}, len = {10};
  Tensor cu = up(one, {2}, Kind::Int), ctx = up(len, {1}, Kind::Int), bt = up(std::vector<int32_t>{3}, {1, 1}, Kind::Int);
  for (int64_t stride : {1, 128, 1001}) {
    Tensor q = Tensor::view(b.q.data, {1, H, D}, Kind::BFloat16, 0, {stride, D, 1});
    Tensor v = Tensor::view(b.v.data, {1, H, D}, Kind::BFloat16, 0, {stride, D, 1});
    Tensor o = Tensor::empty({1, H, D}, Kind::BFloat16, 0);
    t::paged_attention_window(o, q, b.kc, b.vc, H, 0.01f, bt, ctx, 16, 10, 4);
    expect(rows_are(down(o), 0, 1, kTwo), "decode of a single row");
    o = t::flash_attn_varlen_paged_window(q, b.kc, b.vc, cu, ctx, bt, 1, 10, 0.01f, 4);
    expect(rows_are(down(o), 0, 1, kTwo), "paged");
    expect(rows_are(down(t::flash_attn_varlen_window(q, q, v, cu, cu, 1, 1, 0.01f, 4)), 0, 1, kOne), "packed");
    Tensor table = t::rotary_cos_sin_cache(4, D, 10000.0, Kind::Float, 0);
    Tensor pos = up(std::vector<int64_t>{0}, {1}, Kind::Int64), slot = up(std::vector<int64_t>{5}, {1}, Kind::Int64);
    const std::vector<uint16_t> twos(H * D, kTwo);
    Tensor q1 = up(twos, {1, H, D}, Kind::BFloat16), k1 = up(twos, {1, H, D}, Kind::BFloat16);
    Tensor kc = Tensor::empty({1, H, D / 8, 16, 8}, Kind::BFloat16, 0), vc = Tensor::empty({1, H, D, 16}, Kind::BFloat16, 0);
    q1.strides[0] = k1.strides[0] = stride;
    t::rotary_embedding(pos, q1, k1, D, table, true);
    t::rotary_embedding_and_cache(pos, q1, k1, v, D, table, true, kc, vc, slot);  // position 0 turns nothing
    expect(rows_are(down(q1), 0, 1, kTwo) && rows_are(down(k1), 0, 1, kTwo), "rotation of a single token");
    std::vector<uint16_t> keys = down(kc), values = down(vc);
    for (int e = 0; e < H * D; ++e)
      expect(keys[e / 8 * 128 + 5 * 8 + e % 8] == kTwo && values[e * 16 + 5] == kOne, "cache write of a single token");
  }
  expect(t::last_status() == 0, "status");
}

int main() {
  t::cuda_check("cudaSetDevice", cudaSetDevice(0));
  try {
    Batch b;
    stated_lengths(b);
    single_rows(b);
  } catch (const std::exception &e) {
    std::printf("[ FAIL ] exception: %s\n", e.what());
    ++fails;
  }
  std::printf("%d failures\n", fails);
  return fails;
}
