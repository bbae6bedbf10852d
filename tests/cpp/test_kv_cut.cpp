// Self-check of the C++ layer over caches that rows were evicted from
// (include/molot_amd/attn.hpp, paged_kv.hpp) on the GPU: prompts, steps and
// shared-KV layers of the next turn, whose positions run ahead of the slots,
// against attention over the rows stored, in 64 bits: row m of a prompt sees
// the rows before it and its own.  Run by tests/test_cpp_cut.py.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <stdexcept>
#include <vector>

#include "check_util.hpp"
#include "molot_amd/attn.hpp"
#include "molot_amd/paged_kv.hpp"

namespace {

using molot::amd::check_hip;

constexpr int kNq = 8, kNkv = 4, kG = kNq / kNkv, kD = 128;
constexpr float kScale = 0.09f;
// An output of values of order 1 (sums over under 700 keys): a score's products to 2^-21
// of their sum of about |q| |k| scale = 128 * 0.09, a weight by twice that, the sum by
// 2^-21 once more: 2 * 11.5 * 2^-21 + 2^-21 = 1.2e-5 of V's largest, about 4.
constexpr double kTol = 5e-5;

struct Dev {
  float* p = nullptr;
  size_t n;
  explicit Dev(size_t n_) : n(n_) { check_hip(hipMalloc((void**)&p, n * sizeof(float)), "hipMalloc"); }
  explicit Dev(const std::vector<float>& x) : Dev(x.size()) {
    check_hip(hipMemcpy(p, x.data(), n * sizeof(float), hipMemcpyHostToDevice), "H2D");
  }
  ~Dev() { (void)hipFree(p); }
  Dev(const Dev&) = delete;
  Dev& operator=(const Dev&) = delete;
};
std::vector<float> get(const void* p, size_t n) {
  std::vector<float> x(n);
  check_hip(hipDeviceSynchronize(), "sync");
  check_hip(hipMemcpy(x.data(), p, n * sizeof(float), hipMemcpyDeviceToHost), "D2H");
  return x;
}
std::vector<float> normal(Rng& r, size_t n) {
  std::vector<float> x(n);
  r.normal(x);
  return x;
}

// Rows q[M][kNq][kD], the last of which sees all of K, V [n][kNkv][kD].
void check_rows(const std::vector<float>& q, const std::vector<float>& K, const std::vector<float>& V,
                const std::vector<float>& o, int M, int n, const char* what) {
  double worst = 0;
  std::vector<double> w;
  for (int m = 0; m < M; ++m)
    for (int h = 0; h < kNq; ++h) {
      const float* qr = &q[((size_t)m * kNq + h) * kD];
      const int hi = n - M + m + 1;
      w.assign(hi, 0.0);
      double top = -1e300, l = 0;
      for (int t = 0; t < hi; ++t) {
        for (int e = 0; e < kD; ++e) w[t] += (double)qr[e] * K[((size_t)t * kNkv + h / kG) * kD + e];
        top = std::max(top, w[t] *= kScale);
      }
      for (double& x : w) l += x = std::exp(x - top);
      for (int e = 0; e < kD; ++e) {
        double x = 0;
        for (int t = 0; t < hi; ++t) x += w[t] * V[((size_t)t * kNkv + h / kG) * kD + e];
        const double err = std::fabs(x / l - o[((size_t)m * kNq + h) * kD + e]);
        worst = std::isnan(err) ? 1e30 : std::max(worst, err);
      }
    }
  CHECK(worst <= kTol, "%s: error %g, bound %g", what, worst, kTol);
  std::printf("%s: error %.2e\n", what, worst);
}

template <typename F>
bool throws(F&& fn) {
  try {
    fn();
  } catch (const std::runtime_error&) {
    return true;
  }
  return false;
}

struct Rows {
  std::vector<float> q, k, v;
  Dev dq, dk, dv, dout;
  Rows(Rng& r, int M)
      : q(normal(r, (size_t)M * kNq * kD)), k(normal(r, (size_t)M * kNkv * kD)),
        v(normal(r, (size_t)M * kNkv * kD)), dq(q), dk(k), dv(v), dout(q.size()) {}
  std::vector<float> out() const { return get(dout.p, dout.n); }
};

// A prompt of 40, cut to 24; then a prompt of M, a layer that shares its rows, steps.
void run_contiguous(int M) {
  molot::amd::DeviceKV kv(40 + M, kNkv, kD, MOLOT_KV_F32);
  kv.track_weights();
  const molot::amd::LayerNorms nm;
  Rng rng(11);
  Rows a(rng, 24), b(rng, 16), c(rng, M), sh(rng, M);
  auto rows = [&](const void* p) { return get(p, (size_t)kv.n * kNkv * kD); };
  kv.prefill(a.dq.p, a.dk.p, a.dv.p, a.dout.p, kNq, 24, 0, nullptr, kScale, 0, nm);
  check_rows(a.q, rows(kv.k), rows(kv.v), a.out(), 24, kv.n, "first prompt");
  kv.evict(20, 6, 23);
  kv.prefill(b.dq.p, b.dk.p, b.dv.p, b.dout.p, kNq, 16, 24, nullptr, kScale, 0, nm);
  check_rows(b.q, rows(kv.k), rows(kv.v), b.out(), 16, kv.n, "a prompt after a small cut");
  kv.evict(24, 10, 39);
  CHECK(kv.n == 24, "%d rows left", kv.n);
  kv.prefill(c.dq.p, c.dk.p, c.dv.p, c.dout.p, kNq, M, 40, nullptr, kScale, 0, nm);
  check_rows(c.q, rows(kv.k), rows(kv.v), c.out(), M, kv.n, "a prompt after a cut");
  kv.prefill_shared(sh.dq.p, sh.dout.p, kNq, M, 40, nullptr, kScale, 0, nm);
  check_rows(sh.q, rows(kv.k), rows(kv.v), sh.out(), M, kv.n, "its shared layer");
  for (int i = 0; i < 2; ++i) {
    Rows s(rng, 1), t(rng, 1);
    kv.decode(s.dq.p, s.dk.p, s.dv.p, s.dout.p, kNq, 40 + M + i, nullptr, kScale, 0, nm);
    check_rows(s.q, rows(kv.k), rows(kv.v), s.out(), 1, kv.n, "a step");
    kv.decode_shared(t.dq.p, t.dout.p, kNq, 40 + M + i, nullptr, kScale, 0, nm);
    check_rows(t.q, rows(kv.k), rows(kv.v), t.out(), 1, kv.n, "its shared layer");
  }
}

void run_paged(int M) {
  constexpr int kPage = 16;
  molot::amd::PagedKVCache kv(1, 64, kNkv, kD, kPage, MOLOT_KV_F32);
  kv.track_weights();
  const molot::amd::LayerNorms nm;
  Rng rng(12);
  const int other = kv.add_sequence(), id = kv.add_sequence();
  auto rows = [&](const void* p, int s, int n) {
    const std::vector<float> pool = get(p, (size_t)64 * kNkv * kPage * kD);
    std::vector<float> x((size_t)n * kNkv * kD);
    for (int t = 0; t < n; ++t)
      for (int h = 0; h < kNkv; ++h)
        std::memcpy(&x[((size_t)t * kNkv + h) * kD],
                    &pool[(((size_t)kv.blocks(s)[t / kPage] * kNkv + h) * kPage + t % kPage) * kD],
                    kD * sizeof(float));
    return x;
  };
  auto prompt = [&](int s, int len, const char* what) {
    Rows r(rng, len), sh(rng, len);
    const int pos0 = kv.position(s), n = kv.length(s) + len;
    kv.begin_prefill(s, len);
    kv.prefill(0, r.dq.p, r.dk.p, r.dv.p, r.dout.p, kNq, pos0, nullptr, kScale, 0, nm);
    check_rows(r.q, rows(kv.k_pages(0), s, n), rows(kv.v_pages(0), s, n), r.out(), len, n, what);
    kv.prefill_shared(0, sh.dq.p, sh.dout.p, kNq, pos0, nullptr, kScale, 0, nm);
    check_rows(sh.q, rows(kv.k_pages(0), s, n), rows(kv.v_pages(0), s, n), sh.out(), len, n,
               "its shared layer");
    kv.end_prefill();
  };
  prompt(other, 9, "another sequence's prompt");
  prompt(id, 40, "first paged prompt");
  kv.evict({id, other}, 24, 10);
  CHECK(kv.length(id) == 24 && kv.position(id) == 40 && kv.position(other) == 9, "lengths after the cut");
  prompt(id, M, "a paged prompt after a cut");
  prompt(other, 7, "a sequence that was not cut");
  Rows s(rng, 2), t(rng, 2);
  kv.begin_decode({id, other});
  kv.decode(0, s.dq.p, s.dk.p, s.dv.p, s.dout.p, kNq, nullptr, kScale, 0, nm);
  kv.decode_shared(0, t.dq.p, t.dout.p, kNq, nullptr, kScale, 0, nm);
  for (int i = 0; i < 2; ++i) {
    const int sid = i ? other : id, n = kv.length(sid) + 1;
    const size_t at = (size_t)i * kNq * kD;
    auto part = [&](const std::vector<float>& x) {
      return std::vector<float>(x.begin() + at, x.begin() + at + kNq * kD);
    };
    const auto K = rows(kv.k_pages(0), sid, n), V = rows(kv.v_pages(0), sid, n);
    check_rows(part(s.q), K, V, part(s.out()), 1, n, "a paged step");
    check_rows(part(t.q), K, V, part(t.out()), 1, n, "its shared layer");
  }
  kv.end_decode();
}

// Windows are of positions, the kernels' of slots: refused over a cut cache, in every
// call, unless they hold every position; as before in one that was not cut.
void run_windows() {
  const molot::amd::LayerNorms nm;
  const molot::amd::Scores sc;
  Rng rng(13);
  Rows r(rng, 40), s(rng, 5);
  molot::amd::DeviceKV kv(64, kNkv, kD, MOLOT_KV_F32);
  kv.track_weights();
  auto all = [&](int window, int pos, bool want, const char* what) {
    const int n = kv.n;
    auto expect = [&](const char* call, auto&& fn) {
      CHECK(throws(fn) == want, "%s: %s, window %d", what, call, window);
      if (want) CHECK(kv.n == n, "%s: %s appended", what, call);
      kv.n = n;  // (each call at the same length)
    };
    expect("decode", [&] { kv.decode(s.dq.p, s.dk.p, s.dv.p, s.dout.p, kNq, pos, nullptr, kScale, window, nm); });
    expect("decode_scored", [&] {
      kv.decode_scored(s.dq.p, s.dk.p, s.dv.p, s.dout.p, kNq, pos, nullptr, kScale, window, nm, sc);
    });
    expect("decode_shared", [&] { kv.decode_shared(s.dq.p, s.dout.p, kNq, pos, nullptr, kScale, window, nm); });
    expect("attend", [&] { kv.attend(s.dq.p, s.dout.p, kNq, kScale, pos, window); });
    expect("prefill", [&] {
      kv.prefill(s.dq.p, s.dk.p, s.dv.p, s.dout.p, kNq, 5, pos - 4, nullptr, kScale, window, nm);
    });
    expect("prefill_scored", [&] {
      kv.prefill_scored(s.dq.p, s.dk.p, s.dv.p, s.dout.p, kNq, 5, pos - 4, nullptr, kScale, window, nm, sc);
    });
    expect("prefill_shared", [&] {
      kv.prefill_shared(s.dq.p, s.dout.p, kNq, 5, pos - 4, nullptr, kScale, window, nm);
    });
  };
  kv.prefill(r.dq.p, r.dk.p, r.dv.p, r.dout.p, kNq, 40, 0, nullptr, kScale, 16, nm);
  all(16, 44, false, "not cut");
  kv.evict(50, 3, 39);
  all(16, 44, false, "a budget above the length");
  kv.evict(20, 3, 39);
  all(44, 44, true, "cut");
  all(16, 44, true, "cut");
  all(45, 44, false, "cut, every position in the window");
  all(0, 44, false, "cut, no window");
  kv.reset();
  kv.prefill(r.dq.p, r.dk.p, r.dv.p, r.dout.p, kNq, 40, 0, nullptr, kScale, 16, nm);
  all(16, 44, false, "reset");
  kv.evict(20, 3, 39);
  all(16, 44, true, "cut again");
  kv.evict(0, 3, 39);
  Rows one(rng, 1);
  CHECK(throws([&] {
          kv.decode(one.dq.p, one.dk.p, one.dv.p, one.dout.p, kNq, 40, nullptr, kScale, 16, nm);
        }), "cut to nothing: the next token");
  kv.n = 0;  // (without reset)
  kv.prefill(r.dq.p, r.dk.p, r.dv.p, r.dout.p, kNq, 40, 0, nullptr, kScale, 16, nm);
  all(16, 44, false, "from position 0 again");

  molot::amd::PagedKVCache pg(1, 32, kNkv, kD, 16, MOLOT_KV_F32);
  pg.track_weights();
  const int whole = pg.add_sequence(), cut = pg.add_sequence();
  auto prompt = [&](int id, Rows& x, int M, int window, bool want, const char* what) {
    const int pos0 = pg.position(id);
    pg.begin_prefill(id, M);
    CHECK(throws([&] {
            pg.prefill(0, x.dq.p, x.dk.p, x.dv.p, x.dout.p, kNq, pos0, nullptr, kScale, window, nm);
          }) == want, "%s: prefill, window %d", what, window);
    CHECK(throws([&] {
            pg.prefill_scored(0, x.dq.p, x.dk.p, x.dv.p, x.dout.p, kNq, pos0, nullptr, kScale, window, nm, sc);
          }) == want, "%s: prefill_scored, window %d", what, window);
    CHECK(throws([&] { pg.prefill_shared(0, x.dq.p, x.dout.p, kNq, pos0, nullptr, kScale, window, nm); }) ==
              want, "%s: prefill_shared, window %d", what, window);
    if (want)  // (the step is ended with its rows)
      pg.prefill(0, x.dq.p, x.dk.p, x.dv.p, x.dout.p, kNq, pos0, nullptr, kScale, 0, nm);
    pg.end_prefill();
  };
  prompt(whole, r, 40, 16, false, "not cut");
  prompt(cut, r, 40, 16, false, "not cut");
  pg.evict({cut}, 20, 3);
  prompt(whole, s, 5, 16, false, "another sequence's cut");
  prompt(cut, s, 5, 16, true, "cut");
  prompt(cut, s, 5, 50, false, "cut, every position in the window");
  Rows t(rng, 2);
  auto step = [&](const std::vector<int>& ids, int window, bool want, const char* what) {
    pg.begin_decode(ids);
    CHECK(throws([&] { pg.decode(0, t.dq.p, t.dk.p, t.dv.p, t.dout.p, kNq, nullptr, kScale, window, nm); }) ==
              want, "%s: decode, window %d", what, window);
    CHECK(throws([&] {
            pg.decode_scored(0, t.dq.p, t.dk.p, t.dv.p, t.dout.p, kNq, nullptr, kScale, window, nm, sc);
          }) == want, "%s: decode_scored, window %d", what, window);
    CHECK(throws([&] { pg.decode_shared(0, t.dq.p, t.dout.p, kNq, nullptr, kScale, window, nm); }) == want,
          "%s: decode_shared, window %d", what, window);
    if (want) pg.decode(0, t.dq.p, t.dk.p, t.dv.p, t.dout.p, kNq, nullptr, kScale, 0, nm);
    pg.end_decode();
  };
  step({whole}, 16, false, "not cut");                 // positions 45; cut's: 50 next
  step({whole, cut}, 16, true, "one of them cut");
  step({cut, whole}, 51, true, "one of them cut");     // its token's position is 51
  step({cut, whole}, 53, false, "cut, every position in the window");
  pg.free_sequence(cut);
  CHECK(pg.add_sequence() == cut, "the id again");
  prompt(cut, r, 40, 16, false, "a new sequence");
  check_hip(hipDeviceSynchronize(), "sync");
}

}  // namespace

int main() {
  try {
    for (int M : {7, 30, 600}) {
      std::printf("[case] prompts of %d\n", M);
      std::fflush(stdout);
      run_contiguous(M);
      run_paged(M);
    }
    run_windows();
  } catch (const std::exception& e) {
    CHECK(false, "%s", e.what());
  }
  std::printf(failures ? "%d FAILED\n" : "PASSED\n", failures);
  return failures ? 1 : 0;
}
