// The operators around windowed attention through the C++ host side (include/aici_b200_tch.hpp), in the
// order a serving step calls them: tables, rotary positions with the cache write, attention over the
// cache -- compared with plain loops in double.
//
//   test_window            run on GPU 0, exit code = number of failures
//   test_window --check    refusals that need no GPU
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "aici_b200_tch.hpp"

namespace t = aici::tch;
using t::Kind;
using t::Tensor;

static float from_bf16(uint16_t h) {
  uint32_t u = (uint32_t)h << 16;
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}
static uint16_t to_bf16(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

template <typename T>
static Tensor up(const std::vector<T> &h, std::vector<int64_t> sizes, Kind kind) {
  Tensor d = Tensor::empty(std::move(sizes), kind, 0);
  t::cuda_check("up", cudaMemcpy(d.data, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice));
  return d;
}
template <typename T>
static std::vector<T> down(const Tensor &d) {
  std::vector<T> h((size_t)d.numel());
  t::cuda_check("down", cudaDeviceSynchronize());
  t::cuda_check("down", cudaMemcpy(h.data(), d.data, h.size() * sizeof(T), cudaMemcpyDeviceToHost));
  return h;
}

static int fails = 0;
static void expect(bool ok, const char *what) {
  if (!ok) {
    std::printf("[ FAIL ] %s\n", what);
    ++fails;
  }
}

// One step of two requests, 40 and 3 new tokens, heads 4 / 2, rotated as interleaved pairs over 64 of the 128
// elements, window 9, sinks 2.
static void step() {
  const int H = 4, Hk = 2, D = 128, rot = 64, T = 43, blocks = 12, window = 9, sinks = 2;
  const float scale = 0.088388347f;
  std::vector<int32_t> qlens = {40, 3}, ctx = {0, 0}, tables(2 * 4, -1), free_list = {3, 7, 1, 9, 5}, count = {5};
  Tensor bt = up(tables, {2, 4}, Kind::Int);
  t::StepTables s = t::step_tables(up(qlens, {2}, Kind::Int), up(ctx, {2}, Kind::Int), bt, up(free_list, {5}, Kind::Int),
                                   up(count, {1}, Kind::Int), blocks, T);
  expect(down<int32_t>(s.seqlens_q) == std::vector<int32_t>({0, 40, 43}), "seqlens_q");
  expect(down<int32_t>(s.logit_idxs) == std::vector<int32_t>({39, 42}), "logit_idxs");
  expect(down<int32_t>(s.context_lens) == std::vector<int32_t>({40, 3}), "context_lens");
  expect(down<int32_t>(s.free_count)[0] == 1, "free_count");
  expect(down<int32_t>(bt) == std::vector<int32_t>({5, 9, 1, -1, 7, -1, -1, -1}), "block_tables");
  expect(down<int32_t>(s.slot_mapping)[17] == 9 * 16 + 1, "slot_mapping");

  std::vector<uint16_t> x((size_t)T * (H + 2 * Hk) * D);
  unsigned r = 12345;
  for (auto &v : x) {
    r = r * 1664525u + 1013904223u;
    v = to_bf16(((r >> 8) / 16777216.f - 0.5f) * 4.f);
  }
  Tensor xd = up(x, {T, H + 2 * Hk, D}, Kind::BFloat16);
  const int64_t row = (H + 2 * Hk) * D;
  auto cut = [&](int h0, int n) {
    return Tensor::view(static_cast<uint16_t *>(xd.data) + h0 * D, {T, n, D}, Kind::BFloat16, 0, {row, D, 1});
  };
  Tensor q = cut(0, H), k = cut(H, Hk), v = cut(H + Hk, Hk);
  Tensor cs = t::rotary_cos_sin_cache(64, rot, 10000.0, Kind::Float, 0);
  const std::vector<float> table = down<float>(cs);
  for (int p : {0, 1, 40, 63})
    for (int j : {0, 5, 31})
      expect(std::fabs(table[p * rot + j] - std::cos(p * std::pow(10000.0, -2.0 * j / rot))) < 1e-6, "cosine");
  Tensor kc = Tensor::empty({blocks, Hk, D / 8, 16, 8}, Kind::BFloat16, 0), vc = Tensor::empty({blocks, Hk, D, 16}, Kind::BFloat16, 0);
  t::cuda_check("memset", cudaMemset(kc.data, 0xff, kc.numel() * 2));  // NaN everywhere
  t::cuda_check("memset", cudaMemset(vc.data, 0xff, vc.numel() * 2));
  t::cuda_check("sync", cudaDeviceSynchronize());
  t::rotary_embedding_and_cache(s.positions, q, k, v, D, cs, false, kc, vc, s.slot_mapping);
  const std::vector<uint16_t> y = down<uint16_t>(xd);
  for (int tok : {0, 7, 39, 42}) {
    const int p = tok < 40 ? tok : tok - 40;
    for (int h = 0; h < H + Hk; ++h)
      for (int j : {0, 3, 31}) {
        const size_t at = tok * row + h * D + 2 * j;
        const double a = from_bf16(x[at]), b = from_bf16(x[at + 1]), an = p * std::pow(10000.0, -2.0 * j / rot);
        const double u = a * std::cos(an) - b * std::sin(an);
        // half a step of bf16, and fp32 products and table
        expect(std::fabs(from_bf16(y[at]) - u) <= std::fabs(u) / 256 + 1e-5, "rotated");
        expect(y[tok * row + h * D + rot + j] == x[tok * row + h * D + rot + j], "unrotated part");
      }
  }
  auto check_row = [&](const uint16_t *o, int seq, int pos, int h) {
    const int first = seq == 0 ? 0 : 40, kvh = h / (H / Hk);
    std::vector<double> w;
    std::vector<int> toks;
    double top = -1e300, sum = 0;
    for (int tk = 0; tk <= pos; ++tk)
      if (tk > pos - window || tk < sinks) {
        double d = 0;
        for (int e = 0; e < D; ++e)
          d += (double)from_bf16(y[(first + pos) * row + h * D + e]) * from_bf16(y[(first + tk) * row + (H + kvh) * D + e]);
        toks.push_back(tk);
        w.push_back(d * scale);
        top = std::fmax(top, d * scale);
      }
    for (double &z : w) sum += z = std::exp(z - top);
    for (int e = 0; e < D; ++e) {
      double o64 = 0, mag = 0;
      for (size_t i = 0; i < w.size(); ++i) {
        const double val = from_bf16(y[(first + toks[i]) * row + (H + Hk + kvh) * D + e]);
        o64 += w[i] / sum * val;
        mag += w[i] / sum * std::fabs(val);
      }
      // half a step of bf16 for the output and one for each probability, and fp32 scores
      expect(std::fabs(from_bf16(o[e]) - o64) <= (std::fabs(o64) + mag) / 256 + 1e-4 * mag, "attention");
    }
  };
  Tensor o = t::flash_attn_varlen_paged_window(q, kc, vc, s.seqlens_q, s.context_lens, bt, 40, 40, scale, window, sinks);
  std::vector<uint16_t> oh = down<uint16_t>(o);
  for (int tok = 0; tok < T; ++tok)
    for (int h = 0; h < H; ++h) check_row(&oh[(size_t)(tok * H + h) * D], tok < 40 ? 0 : 1, tok < 40 ? tok : tok - 40, h);
  Tensor o2 = t::flash_attn_varlen_window(q, k, v, s.seqlens_q, s.seqlens_q, 40, 40, scale, window, sinks);
  oh = down<uint16_t>(o2);
  for (int tok = 0; tok < T; ++tok)
    for (int h = 0; h < H; ++h) check_row(&oh[(size_t)(tok * H + h) * D], tok < 40 ? 0 : 1, tok < 40 ? tok : tok - 40, h);
  // the last tokens of both sequences as a decode step
  std::vector<uint16_t> last(2 * H * D);
  for (int i = 0; i < 2; ++i) std::memcpy(&last[i * H * D], &y[(i == 0 ? 39 : 42) * row], H * D * 2);
  Tensor q1 = up(last, {2, H, D}, Kind::BFloat16), o1 = Tensor::empty({2, H, D}, Kind::BFloat16, 0);
  t::paged_attention_window(o1, q1, kc, vc, Hk, scale, bt, s.context_lens, 16, 40, window, sinks);
  oh = down<uint16_t>(o1);
  for (int i = 0; i < 2; ++i)
    for (int h = 0; h < H; ++h) check_row(&oh[(size_t)(i * H + h) * D], i, i == 0 ? 39 : 2, h);
  // rotating alone gives what it gave with the cache write
  Tensor xd2 = up(x, {T, H + 2 * Hk, D}, Kind::BFloat16);
  Tensor q2 = Tensor::view(xd2.data, {T, H, D}, Kind::BFloat16, 0, {row, D, 1});
  Tensor k2 = Tensor::view(static_cast<uint16_t *>(xd2.data) + H * D, {T, Hk, D}, Kind::BFloat16, 0, {row, D, 1});
  t::rotary_embedding(s.positions, q2, k2, D, cs, false);
  expect(down<uint16_t>(xd2) == y, "rotary_embedding");
  expect(t::last_status() == 0, "status");
}

static void refusals() {
  auto says = [](const char *what, auto f) {
    try {
      f();
      expect(false, what);
    } catch (const t::Error &e) {
      expect(std::strstr(e.what(), what) != nullptr, e.what());
    }
  };
  int64_t word[4] = {};
  Tensor host = Tensor::view(word, {1, 1, 128}, Kind::BFloat16, -1), ints = Tensor::view(word, {1}, Kind::Int, -1);
  Tensor kc = Tensor::view(word, {1, 1, 16, 16, 8}, Kind::BFloat16, -1), vc = Tensor::view(word, {1, 1, 128, 16}, Kind::BFloat16, -1);
  Tensor tables = Tensor::view(word, {1, 1}, Kind::Int, -1);
  says("paged_attention_window: tensor must be on a CUDA device",
       [&] { t::paged_attention_window(host, host, kc, vc, 1, 1.f, tables, ints, 16, 1, 1); });
  says("flash_attn_varlen_window: tensor must be on a CUDA device",
       [&] { t::flash_attn_varlen_window(host, host, host, ints, ints, 1, 1, 1.f, 1); });
  says("flash_attn_varlen_paged_window: tensor must be on a CUDA device",
       [&] { t::flash_attn_varlen_paged_window(host, kc, vc, ints, ints, tables, 1, 1, 1.f, 1); });
  says("rotary_embedding: tensor must be on a CUDA device", [&] { t::rotary_embedding(ints, host, host, 128, host, true); });
  says("step_tables: tensor must be on a CUDA device", [&] { t::step_tables(ints, ints, tables, ints, ints, 1, 1); });
}

int main(int argc, char **argv) {
  refusals();
  if (argc > 1 && std::string(argv[1]) == "--check") {
    std::printf("%d failures\n", fails);
    return fails;
  }
  t::cuda_check("cudaSetDevice", cudaSetDevice(0));
  try {
    step();
  } catch (const std::exception &e) {
    std::printf("[ FAIL ] exception: %s\n", e.what());
    ++fails;
  }
  std::printf("%d failures\n", fails);
  return fails;
}
