// Self-check of a cache held to a budget through the C++ layer
// (include/molot_amd/attn.hpp, paged_kv.hpp) on the GPU: scored prompts and
// scored decode steps that track their weights, the cache cut whenever it
// reaches its limit, against the same steps on the host in 64 bits.  The host
// keeps each (sequence, KV head)'s rows in slot order with their positions and
// takes the accumulated weights from the device before a cut, so that both
// rank the same numbers.  inv_freq is 0 (positions turn nothing): the rows
// are then the new ones as they came.  Run by tests/test_cpp_budget.py.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <numeric>
#include <stdexcept>
#include <vector>

#include "check_util.hpp"
#include "molot_amd/attn.hpp"
#include "molot_amd/paged_kv.hpp"

namespace {

using molot::amd::check_hip;

constexpr int kNq = 6, kNkv = 2, kG = kNq / kNkv, kD = 64;
constexpr float kScale = 0.125f, kCap = 3.f;
// fp32 sums over at most 128 keys of values of order 1 (2^-24 each, with the
// exponential's and the cap's few roundings): 100 such steps
constexpr double kTol = 100 * 5.97e-8;

template <typename T>
struct Dev {
  T* p = nullptr;
  size_t n;
  explicit Dev(size_t n_) : n(n_) { check_hip(hipMalloc((void**)&p, n * sizeof(T)), "hipMalloc"); }
  ~Dev() { (void)hipFree(p); }
  Dev(const Dev&) = delete;
  Dev& operator=(const Dev&) = delete;
  void put(const std::vector<T>& x) {
    check_hip(hipMemcpy(p, x.data(), x.size() * sizeof(T), hipMemcpyHostToDevice), "H2D");
  }
  std::vector<T> get() const {
    std::vector<T> x(n);
    check_hip(hipMemcpy(x.data(), p, n * sizeof(T), hipMemcpyDeviceToHost), "D2H");
    return x;
  }
};
template <typename T>
T peek(const T* p, int64_t i) {
  T x;
  check_hip(hipMemcpy(&x, p + i, sizeof(T), hipMemcpyDeviceToHost), "D2H");
  return x;
}

// One KV head of a sequence: its slots in order.
struct Head {
  struct Slot {
    std::vector<float> k, v;
    double acc;
    int pos;
  };
  std::vector<Slot> slots;
  // A query of this head's group at pos; its weights, and o.
  std::vector<double> attend(const float* q, int pos, double slope, std::vector<double>& w) const {
    std::vector<double> s(slots.size());
    for (size_t t = 0; t < slots.size(); ++t) {
      double x = 0;
      for (int e = 0; e < kD; ++e) x += (double)q[e] * slots[t].k[e];
      s[t] = kCap * std::tanh(x * kScale / kCap) - slope * std::fabs((double)pos - (double)t);
    }
    const double m = *std::max_element(s.begin(), s.end());
    double l = 0;
    for (double& x : s) l += x = std::exp(x - m);
    std::vector<double> o(kD, 0.0);
    w.resize(s.size());
    for (size_t t = 0; t < s.size(); ++t) {
      w[t] = s[t] / l;
      for (int e = 0; e < kD; ++e) o[e] += w[t] * slots[t].v[e];
    }
    return o;
  }
  void cut(int keep, int recent, int pos) {
    const int n = (int)slots.size();
    if (n <= keep) return;
    std::vector<int> by(n);
    std::iota(by.begin(), by.end(), 0);
    auto first = [&](int t) { return slots[t].pos > pos - recent; };
    std::stable_sort(by.begin(), by.end(), [&](int a, int b) {
      if (first(a) != first(b)) return first(a);
      return !first(a) && slots[a].acc > slots[b].acc;
    });
    std::vector<char> stays(n, 0);
    for (int i = 0; i < keep; ++i) stays[by[i]] = 1;
    int from = keep;
    for (int t = 0; t < keep; ++t) {
      if (stays[t]) continue;
      while (!stays[from]) ++from;
      slots[t] = slots[from++];
    }
    slots.resize(keep);
  }
};

std::vector<float> normal(Rng& r, size_t n) {
  std::vector<float> x(n);
  r.normal(x);
  return x;
}
bool close(double got, double want, double scale) { return std::fabs(got - want) <= kTol * scale; }

// A step's output and weights against the host's, whose weights are then added.
void check_step(std::vector<Head>& heads, const float* q, const float* o, int pos,
                const std::vector<float>& slopes, const char* what) {
  for (int h = 0; h < kNq; ++h) {
    Head& kv = heads[h / kG];
    std::vector<double> w;
    const std::vector<double> want = kv.attend(q + h * kD, pos, slopes[h], w);
    for (int e = 0; e < kD; ++e)
      CHECK(close(o[h * kD + e], want[e], 4.0), "%s: o[%d][%d] = %g, want %g", what, h, e, o[h * kD + e],
            want[e]);
    for (size_t t = 0; t < w.size(); ++t) kv.slots[t].acc += w[t];
  }
}

void append(std::vector<Head>& heads, const float* k, const float* v, int pos) {
  for (int h = 0; h < kNkv; ++h)
    heads[h].slots.push_back({std::vector<float>(k + h * kD, k + (h + 1) * kD),
                              std::vector<float>(v + h * kD, v + (h + 1) * kD), 0.0, pos});
}

// One contiguous cache: a prompt, then steps; cut to kKeep whenever it holds kLimit.
void run_contiguous(const std::vector<float>& slopes) {
  constexpr int kPrompt = 21, kSteps = 90, kLimit = 48, kKeep = 37, kRecent = 9;
  molot::amd::DeviceKV kv(kLimit, kNkv, kD, MOLOT_KV_F32);
  kv.track_weights();
  Dev<float> inv(kD / 2), dsl(kNq);
  inv.put(std::vector<float>(kD / 2, 0.f));
  dsl.put(slopes);
  molot::amd::Scores sc;
  sc.softcap = kCap;
  sc.slopes = dsl.p;
  molot::amd::LayerNorms nm;
  Rng rng(5);
  std::vector<Head> heads(kNkv);
  {
    const auto q = normal(rng, (size_t)kPrompt * kNq * kD), k = normal(rng, (size_t)kPrompt * kNkv * kD),
               v = normal(rng, (size_t)kPrompt * kNkv * kD);
    Dev<float> dq(q.size()), dk(k.size()), dv(v.size()), dof(q.size());
    dq.put(q), dk.put(k), dv.put(v);
    kv.prefill_scored(dq.p, dk.p, dv.p, dof.p, kNq, kPrompt, 0, inv.p, kScale, 0, nm, sc);
    check_hip(hipDeviceSynchronize(), "sync");
    const auto o = dof.get();
    for (int m = 0; m < kPrompt; ++m) {
      append(heads, &k[(size_t)m * kNkv * kD], &v[(size_t)m * kNkv * kD], m);
      std::vector<Head> at = heads;  // (a prompt's weights are not kept)
      check_step(at, &q[(size_t)m * kNq * kD], &o[(size_t)m * kNq * kD], m, slopes, "prompt");
    }
  }
  Dev<float> dq((size_t)kNq * kD), dk((size_t)kNkv * kD), dv((size_t)kNkv * kD), dof((size_t)kNq * kD);
  int pos = kPrompt, cuts = 0;
  for (int step = 0; step < kSteps; ++step, ++pos) {
    const auto q = normal(rng, dq.n), k = normal(rng, dk.n), v = normal(rng, dv.n);
    dq.put(q), dk.put(k), dv.put(v);
    append(heads, k.data(), v.data(), pos);
    kv.decode_scored(dq.p, dk.p, dv.p, dof.p, kNq, pos, inv.p, kScale, 0, nm, sc);
    check_hip(hipDeviceSynchronize(), "sync");
    const int n = kv.n;
    CHECK(n == (int)heads[0].slots.size(), "%d rows, want %zu", n, heads[0].slots.size());
    check_step(heads, q.data(), dof.get().data(), pos, slopes, "decode");
    const bool full = n == kLimit;
    auto compare = [&](bool exact) {
      for (int h = 0; h < kNkv; ++h)
        for (int t = 0; t < kv.n; ++t) {
          Head::Slot& s = heads[h].slots[t];
          const float a = peek(kv.acc, (int64_t)h * kLimit + t);
          CHECK(exact ? a == (float)s.acc : close(a, s.acc, std::fmax(1.0, s.acc)),
                "step %d: acc[%d][%d] = %g, want %g", step, h, t, a, s.acc);
          CHECK(peek(kv.slot_pos, (int64_t)h * kLimit + t) == s.pos, "step %d: slot_pos[%d][%d]", step, h, t);
          s.acc = a;
        }
    };
    if (full || step % 7 == 0) compare(false);
    if (!full) continue;
    kv.evict(kKeep, kRecent, pos);
    for (Head& h : heads) h.cut(kKeep, kRecent, pos);
    ++cuts;
    compare(true);
    std::vector<float> rows((size_t)kKeep * kNkv * kD);
    check_hip(hipMemcpy(rows.data(), kv.v, rows.size() * sizeof(float), hipMemcpyDeviceToHost), "D2H V");
    for (int h = 0; h < kNkv; ++h)
      for (int t = 0; t < kKeep; ++t)
        for (int e = 0; e < kD; ++e)
          CHECK(rows[((size_t)t * kNkv + h) * kD + e] == heads[h].slots[t].v[e], "cut: V[%d][%d][%d]", t, h, e);
  }
  constexpr int kCuts = 1 + (kSteps - (kLimit - kPrompt)) / (kLimit - kKeep);
  CHECK(cuts == kCuts, "%d cuts, want %d", cuts, kCuts);
}

// Three sequences of one pool, prompted at different lengths and decoded as a batch;
// those past the budget are cut every eighth step, and their blocks return.
void run_paged(const std::vector<float>& slopes) {
  constexpr int kSteps = 40, kKeep = 32, kRecent = 11, kLayers = 2;
  const int prompt[3] = {1, 17, 50};
  molot::amd::PagedKVCache kv(kLayers, 24, kNkv, kD, 16, MOLOT_KV_F32);
  kv.track_weights();
  Dev<float> inv(kD / 2), dsl(kNq);
  inv.put(std::vector<float>(kD / 2, 0.f));
  dsl.put(slopes);
  molot::amd::Scores sc;
  sc.softcap = kCap;
  sc.slopes = dsl.p;
  molot::amd::LayerNorms nm;
  Rng rng(6);
  std::vector<int> ids;
  std::vector<std::vector<std::vector<Head>>> heads(3);  // [sequence][layer][head]
  for (int i = 0; i < 3; ++i) {
    ids.push_back(kv.add_sequence());
    heads[i].assign(kLayers, std::vector<Head>(kNkv));
    const int M = prompt[i];
    kv.begin_prefill(ids[i], M);
    for (int l = 0; l < kLayers; ++l) {
      const auto q = normal(rng, (size_t)M * kNq * kD), k = normal(rng, (size_t)M * kNkv * kD),
                 v = normal(rng, (size_t)M * kNkv * kD);
      Dev<float> dq(q.size()), dk(k.size()), dv(v.size()), dof(q.size());
      dq.put(q), dk.put(k), dv.put(v);
      kv.prefill_scored(l, dq.p, dk.p, dv.p, dof.p, kNq, 0, inv.p, kScale, 0, nm, sc);
      check_hip(hipDeviceSynchronize(), "sync");
      const auto o = dof.get();
      for (int m = 0; m < M; ++m) {
        append(heads[i][l], &k[(size_t)m * kNkv * kD], &v[(size_t)m * kNkv * kD], m);
        std::vector<Head> at = heads[i][l];
        check_step(at, &q[(size_t)m * kNq * kD], &o[(size_t)m * kNq * kD], m, slopes, "paged prompt");
      }
    }
    kv.end_prefill();
  }
  Dev<float> dq(3 * (size_t)kNq * kD), dk(3 * (size_t)kNkv * kD), dv(dk.n), dof(dq.n);
  auto slot_at = [&](int i, int h, int t) -> int64_t {
    return ((int64_t)kv.blocks(ids[i])[t / 16] * kNkv + h) * 16 + t % 16;
  };
  auto compare = [&](int step, bool exact) {
    for (int i = 0; i < 3; ++i)
      for (int l = 0; l < kLayers; ++l)
        for (int h = 0; h < kNkv; ++h)
          for (int t = 0; t < kv.length(ids[i]); ++t) {
            Head::Slot& s = heads[i][l][h].slots[t];
            const float a = peek(kv.acc_pages(l), slot_at(i, h, t));
            CHECK(exact ? a == (float)s.acc : close(a, s.acc, std::fmax(1.0, s.acc)),
                  "step %d: acc of %d/%d/%d/%d = %g, want %g", step, i, l, h, t, a, s.acc);
            CHECK(peek(kv.slot_pos_pages(l), slot_at(i, h, t)) == s.pos, "step %d: slot_pos of %d/%d/%d/%d",
                  step, i, l, h, t);
            s.acc = a;
          }
  };
  for (int step = 0; step < kSteps; ++step) {
    kv.begin_decode(ids);
    std::vector<int> pos(3);
    for (int i = 0; i < 3; ++i) pos[i] = prompt[i] + step;
    for (int l = 0; l < kLayers; ++l) {
      const auto q = normal(rng, dq.n), k = normal(rng, dk.n), v = normal(rng, dv.n);
      dq.put(q), dk.put(k), dv.put(v);
      kv.decode_scored(l, dq.p, dk.p, dv.p, dof.p, kNq, inv.p, kScale, 0, nm, sc);
      check_hip(hipDeviceSynchronize(), "sync");
      const auto o = dof.get();
      for (int i = 0; i < 3; ++i) {
        append(heads[i][l], &k[(size_t)i * kNkv * kD], &v[(size_t)i * kNkv * kD], pos[i]);
        check_step(heads[i][l], &q[(size_t)i * kNq * kD], &o[(size_t)i * kNq * kD], pos[i], slopes,
                   "paged decode");
      }
    }
    kv.end_decode();
    for (int i = 0; i < 3; ++i)
      CHECK(kv.position(ids[i]) == pos[i] + 1, "position %d, want %d", kv.position(ids[i]), pos[i] + 1);
    if (step % 8 != 7) continue;
    compare(step, false);
    kv.evict(ids, kKeep, kRecent);
    check_hip(hipDeviceSynchronize(), "sync");
    for (int i = 0; i < 3; ++i)
      for (auto& layer : heads[i])
        for (Head& h : layer) h.cut(kKeep, kRecent, pos[i]);
    compare(step, true);
    for (int i = 0; i < 3; ++i)
      CHECK((int)kv.blocks(ids[i]).size() <= (kv.length(ids[i]) + 15) / 16, "blocks kept past the budget");
  }
  // a sequence's blocks given to a new one: nothing of the old one's counts
  kv.free_sequence(ids[2]);
  const int id = kv.add_sequence();
  ids[2] = id;
  heads[2].assign(kLayers, std::vector<Head>(kNkv));
  kv.begin_prefill(id, 5);
  for (int l = 0; l < kLayers; ++l) {
    const auto q = normal(rng, 5 * (size_t)kNq * kD), k = normal(rng, 5 * (size_t)kNkv * kD),
               v = normal(rng, 5 * (size_t)kNkv * kD);
    Dev<float> pq(q.size()), pk(k.size()), pv(v.size()), po(q.size());
    pq.put(q), pk.put(k), pv.put(v);
    kv.prefill_scored(l, pq.p, pk.p, pv.p, po.p, kNq, 0, inv.p, kScale, 0, nm, sc);
    check_hip(hipDeviceSynchronize(), "sync");
    for (int m = 0; m < 5; ++m)
      append(heads[2][l], &k[(size_t)m * kNkv * kD], &v[(size_t)m * kNkv * kD], m);
  }
  kv.end_prefill();
  compare(kSteps, true);
}

template <typename F>
void refuses(F&& fn, const char* what) {
  bool threw = false;
  try {
    fn();
  } catch (const std::runtime_error&) {
    threw = true;
  }
  CHECK(threw, "%s was not refused", what);
}

void run_refusals() {
  molot::amd::DeviceKV kv(8, kNkv, kD, MOLOT_KV_F32);
  refuses([&] { kv.evict(4, 1, 7); }, "evict without track_weights");
  kv.n = 1;
  refuses([&] { kv.track_weights(); }, "track_weights on a cache in use");
  molot::amd::PagedKVCache pg(1, 4, kNkv, kD, 16, MOLOT_KV_F32);
  const int id = pg.add_sequence();
  refuses([&] { pg.evict({id}, 4, 1); }, "paged evict without track_weights");
  pg.track_weights();
  refuses([&] { pg.evict({id, id}, 4, 1); }, "a sequence twice");
  refuses([&] { pg.evict({id}, -1, 1); }, "a negative budget");
  pg.begin_decode({id});
  refuses([&] { pg.evict({id}, 4, 1); }, "evict in a step");
}

}  // namespace

int main() {
  std::vector<float> slopes(kNq);
  for (int h = 0; h < kNq; ++h) slopes[h] = std::exp2f(-(float)(h + 1));
  run_contiguous(slopes);
  run_paged(slopes);
  run_refusals();
  std::printf(failures ? "%d FAILED\n" : "PASSED\n", failures);
  return failures ? 1 : 0;
}
