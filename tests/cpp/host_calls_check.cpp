// What the library's host code does around its launches, without a GPU
// (fake_hip.hpp).  One case a run, by name; run by tests/test_host_calls.py.
#include "fake_hip.hpp"

#include <cstdio>
#include <cstring>
#include <set>

#include "check_util.hpp"
#include "molot_amd/attn_hip.h"

namespace {

template <typename T>
T* at(int i) {  // device arrays: 16-byte aligned addresses that nothing reads
  return reinterpret_cast<T*>((1ull << 38) + (uintptr_t)i * (1ull << 30));
}
const hipStream_t kStream = reinterpret_cast<hipStream_t>(0x1000);

int evict(int nkv, int n, int keep, hipStream_t s) {
  return molot_hip_kv_evict(at<void>(0), at<void>(1), at<float>(2), at<int32_t>(3), nkv, n, 128, keep, 100,
                            n - 1, n, MOLOT_KV_F32, s);
}
int scored_step(int nkv, int slot, hipStream_t s) {
  return molot_hip_decode_step_scored(at<float>(0), at<float>(1), at<float>(2), at<void>(3), at<void>(4),
                                      at<float>(5), 4 * nkv, nkv, 128, slot, slot, nullptr, nullptr, 0, 0.f,
                                      at<float>(6), 0.1f, 0, 50.f, nullptr, at<float>(7), at<int32_t>(8),
                                      slot + 1, MOLOT_KV_F32, s);
}
int prompt(int nkv, int M, int slot0, hipStream_t s) {
  return molot_hip_prefill_step(at<float>(0), at<float>(1), at<float>(2), at<void>(3), at<void>(4),
                                at<float>(5), 4 * nkv, nkv, 128, M, slot0, slot0, nullptr, nullptr, 0, 0.f,
                                at<float>(6), 0.1f, 0, MOLOT_KV_F32, s);
}

// Host threads that share a stream: a call's launches hand workspaces on to each other,
// so no other call's come between.
void run_threads() {
  for (int i = 0; i < 2; ++i) {  // (workspaces sized)
    CHECK(evict(8, 40000, 30000, kStream) == 0, "evict");
    CHECK(scored_step(8, 40000, kStream) == 0, "step");
    CHECK(prompt(8, 2000, 3000, kStream) == 0, "prompt");
  }
  fake::reset();
  fake::state().pause_us = 200;
  std::vector<std::thread> threads;
  constexpr int kThreads = 6, kCalls = 12;
  for (int t = 0; t < kThreads; ++t)
    threads.emplace_back([t] {
      for (int i = 0; i < kCalls; ++i) {
        fake::call = 1 + t * kCalls + i;
        const int st = t % 3 == 0   ? evict(1 + t, 20000 + 100 * i, 17000, kStream)
                       : t % 3 == 1 ? scored_step(1 + t, 3000 + 100 * i, kStream)
                                    : prompt(1 + t, 600 + i, 2000, kStream);
        CHECK(st == 0, "thread %d: status %d", t, st);
      }
    });
  for (auto& t : threads) t.join();
  std::set<int> done;
  int last = 0, several = 0, count = 0;
  for (const fake::Launch& l : fake::state().launches) {
    if (l.call != last) {
      CHECK(done.insert(l.call).second, "call %d: %s after another call's launch", l.call, l.kernel.c_str());
      count = 0;
    }
    several += ++count == 2;
    last = l.call;
  }
  CHECK((int)done.size() == kThreads * kCalls, "%zu calls launched", done.size());
  CHECK(several >= kThreads * kCalls, "%d calls of several launches", several);
}

}  // namespace

int main(int argc, char** argv) {
  const struct {
    const char* name;
    void (*run)();
  } cases[] = {{"threads", run_threads}};
  for (const auto& c : cases)
    if (argc == 2 && !std::strcmp(argv[1], c.name)) {
      c.run();
      std::printf(failures ? "%d FAILED\n" : "PASSED\n", failures);
      return failures ? 1 : 0;
    }
  std::printf("no such case\n");
  return 2;
}
