// Self-check of ragged batches through the paged-KV manager
// (include/molot_amd/paged_kv.hpp) on the GPU: ticks in which sequences bring a prompt, a
// few rows, one or none, over two layers and a third that reads the first one's pages,
// against another manager that takes the same rows by its prefills and decode steps.
// Run by tests/test_cpp_ragged.py.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <stdexcept>
#include <string>
#include <vector>

#include "check_util.hpp"
#include "molot_amd/paged_kv.hpp"

namespace {

using molot::amd::check_hip;
using molot::amd::LayerNorms;
using molot::amd::PagedKVCache;
using molot::amd::Scores;

constexpr int kLayers = 2, kNq = 8, kNkv = 2, kD = 128, kPage = 16, kBlocks = 60;
constexpr float kScale = 0.09f;
// Outputs of order 1 of either path: scores of sum |q k| scale up to 128 * 0.09 to 2^-21 of
// it, a weight by twice that, and the sum to 2^-21 (of V's largest, about 4): 5e-5 each.
constexpr double kTol = 1e-4;

struct Dev {
  float* p = nullptr;
  explicit Dev(const std::vector<float>& x) {
    check_hip(hipMalloc((void**)&p, (x.empty() ? 1 : x.size()) * sizeof(float)), "hipMalloc");
    check_hip(hipMemcpy(p, x.data(), x.size() * sizeof(float), hipMemcpyHostToDevice), "H2D");
  }
  ~Dev() { (void)hipFree(p); }
  Dev(const Dev&) = delete;
  Dev& operator=(const Dev&) = delete;
};
std::vector<float> get(const float* p, size_t n) {
  std::vector<float> x(n);
  check_hip(hipDeviceSynchronize(), "sync");
  check_hip(hipMemcpy(x.data(), p, n * sizeof(float), hipMemcpyDeviceToHost), "D2H");
  return x;
}
std::vector<int32_t> get_ints(const int32_t* p, size_t n) {
  std::vector<int32_t> x(n);
  check_hip(hipDeviceSynchronize(), "sync");
  check_hip(hipMemcpy(x.data(), p, n * sizeof(int32_t), hipMemcpyDeviceToHost), "D2H");
  return x;
}
std::vector<float> normal(Rng& r, size_t n) {
  std::vector<float> x(n);
  r.normal(x);
  return x;
}
double worst(const std::vector<float>& a, const std::vector<float>& b) {
  double w = 0;
  for (size_t i = 0; i < a.size(); ++i) w = std::fmax(w, std::fabs((double)a[i] - b[i]));
  return w;
}
template <typename F>
std::string thrown(F&& f) {
  try {
    f();
  } catch (const std::runtime_error& e) {
    return e.what();
  }
  return "";
}

// One tick of `counts` rows: `a` as a ragged batch, `b` sequence by sequence.
void tick(PagedKVCache& a, PagedKVCache& b, const std::vector<int>& ids, const std::vector<int>& counts,
          const float* freq, const LayerNorms& nm, const Scores& sc, int window, Rng& rng) {
  int T = 0;
  for (int c : counts) T += c;
  std::vector<std::vector<float>> q, k, v, oa;
  for (int l = 0; l < kLayers + 1; ++l) {
    q.push_back(normal(rng, (size_t)T * kNq * kD));
    k.push_back(normal(rng, (size_t)T * kNkv * kD));
    v.push_back(normal(rng, (size_t)T * kNkv * kD));
  }
  std::vector<int> before;
  for (int id : ids) before.push_back(a.length(id));
  a.begin_batch(ids, counts);
  CHECK(a.rows() == T, "rows");
  for (int l = 0; l < kLayers + 1; ++l) {
    Dev dq(q[l]), dk(k[l]), dv(v[l]), d_o(std::vector<float>((size_t)T * kNq * kD, -7.f));
    if (l < kLayers)
      a.step(l, dq.p, dk.p, dv.p, d_o.p, kNq, freq, kScale, window, nm, sc);
    else
      a.step_shared(0, dq.p, d_o.p, kNq, freq, kScale, window, nm, sc);
    oa.push_back(get(d_o.p, (size_t)T * kNq * kD));
  }
  const auto start = get_ints(a.row_start(), ids.size() + 1), pos = get_ints(a.row_pos(), T);
  const auto seqs = get_ints(a.row_seq(), T), slot = get_ints(a.row_slot(), T);
  int r = 0;
  for (size_t i = 0; i < ids.size(); ++i) {
    CHECK(start[i] == r, "row_start");
    for (int m = 0; m < counts[i]; ++m, ++r) {
      const int t = before[i] + m;
      CHECK(seqs[r] == (int)i && pos[r] == t &&
                slot[r] == a.blocks(ids[i])[t / kPage] * kPage + t % kPage,
            "maps of row %d", r);
    }
  }
  a.end_batch();
  r = 0;
  for (size_t i = 0; i < ids.size(); ++i) {
    const int M = counts[i];
    if (M == 0) continue;
    b.begin_prefill(ids[i], M);
    for (int l = 0; l < kLayers + 1; ++l) {
      auto part = [&](const std::vector<float>& x, int heads) {
        return std::vector<float>(x.begin() + (size_t)r * heads * kD,
                                  x.begin() + (size_t)(r + M) * heads * kD);
      };
      Dev dq(part(q[l], kNq)), dk(part(k[l], kNkv)), dv(part(v[l], kNkv)), d_o(part(q[l], kNq));
      const int pos0 = before[i];
      if (l < kLayers)
        b.prefill_scored(l, dq.p, dk.p, dv.p, d_o.p, kNq, pos0, freq, kScale, window, nm, sc);
      else if (sc.softcap == 0.f)
        b.prefill_shared(0, dq.p, d_o.p, kNq, pos0, freq, kScale, window, nm);
      else
        continue;
      const double e = worst(part(oa[l], kNq), get(d_o.p, (size_t)M * kNq * kD));
      CHECK(e < kTol, "layer %d, sequence %d of %d rows after %d: off by %g", l, ids[i], M, pos0, e);
    }
    b.end_prefill();
    CHECK(a.length(ids[i]) == b.length(ids[i]), "length");
    r += M;
  }
}

void run(int kv_dtype, bool rope, float softcap, int window) {
  PagedKVCache a(kLayers, kBlocks, kNkv, kD, kPage, kv_dtype), b(kLayers, kBlocks, kNkv, kD, kPage, kv_dtype);
  Rng rng(17 + kv_dtype);
  std::vector<float> f(kD / 2), w(kD, 1.1f);
  for (int i = 0; i < kD / 2; ++i) f[i] = std::pow(1e4f, -2.f * i / kD);
  Dev freq(f), weights(w);
  LayerNorms nm;
  if (rope) {
    nm.q_norm = nm.k_norm = weights.p;
    nm.eps = 1e-6f;
  }
  Scores sc;
  sc.softcap = softcap;
  std::vector<int> ids;
  for (int i = 0; i < 4; ++i) {
    ids.push_back(a.add_sequence());
    CHECK(b.add_sequence() == ids.back(), "ids");
  }
  const float* fr = rope ? freq.p : nullptr;
  tick(a, b, ids, {150, 1, 33, 16}, fr, nm, sc, window, rng);  // prompts
  tick(a, b, ids, {1, 1, 1, 1}, fr, nm, sc, window, rng);      // one token each
  tick(a, b, {ids[2], ids[0]}, {5, 1}, fr, nm, sc, window, rng);  // some of them, in any order
  a.free_sequence(ids[1]);
  b.free_sequence(ids[1]);
  CHECK(a.add_sequence() == ids[1] && b.add_sequence() == ids[1], "reused id");
  tick(a, b, ids, {1, 70, 0, 3}, fr, nm, sc, window, rng);  // a prompt among tokens, one waits
  CHECK(a.free_blocks() == b.free_blocks(), "blocks");
}

void refusals() {
  PagedKVCache a(1, 4, kNkv, kD, kPage, MOLOT_KV_F32);
  const int i = a.add_sequence(), j = a.add_sequence();
  Dev x(std::vector<float>((size_t)64 * kNq * kD, 0.5f)), y(std::vector<float>((size_t)64 * kNq * kD));
  CHECK(thrown([&] { a.begin_batch({i, i}, {1, 1}); }) == "PagedKVCache: a sequence twice", "twice");
  CHECK(thrown([&] { a.begin_batch({i}, {-1}); }) == "PagedKVCache: a negative count", "negative");
  CHECK(!thrown([&] { a.begin_batch({i, j}, {1}); }).empty(), "sizes");
  CHECK(!thrown([&] { a.begin_batch({i, j}, {0, 0}); }).empty(), "no rows");
  CHECK(!thrown([&] { a.begin_batch({i, 9}, {1, 1}); }).empty(), "no such sequence");
  CHECK(thrown([&] { a.begin_batch({i, j}, {40, 40}); }) == "fwd: KV cache full", "full");
  CHECK(a.length(i) == 0 && a.length(j) == 0, "nothing begun");
  CHECK(!thrown([&] { a.end_batch(); }).empty(), "end without begin");
  CHECK(!thrown([&] { a.step(0, x.p, x.p, x.p, y.p, kNq, nullptr, kScale, 0); }).empty(), "outside");
  a.begin_batch({i}, {2});
  CHECK(!thrown([&] { a.begin_batch({j}, {1}); }).empty(), "in progress");
  CHECK(!thrown([&] { a.begin_decode({j}); }).empty(), "in progress");
  CHECK(!thrown([&] { a.end_decode(); }).empty(), "another step");
  CHECK(!thrown([&] { a.step(0, x.p, nullptr, nullptr, y.p, kNq, nullptr, kScale, 0); }).empty(), "k, v");
  Scores sc;
  sc.key_lo = a.row_start();
  CHECK(!thrown([&] { a.step(0, x.p, x.p, x.p, y.p, kNq, nullptr, kScale, 0, LayerNorms{}, sc); }).empty(),
        "ranges");
  a.step(0, x.p, x.p, x.p, y.p, kNq, nullptr, kScale, 0);
  a.end_batch();
  CHECK(a.length(i) == 2, "length");
  PagedKVCache c(1, 4, kNkv, kD, kPage, MOLOT_KV_F32);
  c.track_weights();
  const int s = c.add_sequence();
  CHECK(!thrown([&] { c.begin_batch({s}, {1}); }).empty(), "a cache held to a budget");
}

}  // namespace

int main() {
  // (rows of fewer bits without a rotation: either path then stores the same ones)
  run(MOLOT_KV_F32, true, 0.f, 0);
  run(MOLOT_KV_F32, true, 30.f, 40);
  run(MOLOT_KV_BF16, false, 0.f, 0);
  run(MOLOT_KV_Q8, false, 0.f, 25);
  refusals();
  if (failures) {
    std::printf("%d FAILURES\n", failures);
    return 1;
  }
  std::printf("ragged batches PASSED\n");
  return 0;
}
