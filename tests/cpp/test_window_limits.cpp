// Calls at the limits of what the windowed operators' C++ host side (include/aici_b200_tch.hpp) is told:
// stated lengths that do not cover the sequences.  Exit code = number of failures.
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

int main() {
  t::cuda_check("cudaSetDevice", cudaSetDevice(0));
  try {
    Batch b;
    stated_lengths(b);
  } catch (const std::exception &e) {
    std::printf("[ FAIL ] exception: %s\n", e.what());
    ++fails;
  }
  std::printf("%d failures\n", fails);
  return fails;
}
