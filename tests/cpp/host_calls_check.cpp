// What the library's host code does around its launches, without a GPU
// (fake_hip.hpp).  One case a run, by name; run by tests/test_host_calls.py.
#include "fake_hip.hpp"

#include <cstdio>
#include <cstring>
#include <set>

#include "check_util.hpp"
#include "molot_amd/attn.hpp"
#include "molot_amd/attn_hip.h"
#include "molot_amd/paged_kv.hpp"

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

// A workspace that is asked for a little more at every call is allocated a few times, and
// what was outgrown, which stays, is less than twice the live buffer.  (least: above the
// other workspace's sizes.)
constexpr size_t kMiB = (size_t)1 << 20;
template <typename F>
void rising(const char* what, int calls, size_t least, int most_allocations, size_t cap, F&& call) {
  fake::reset();
  for (int i = 0; i < calls; ++i) {
    const int st = call(i);
    CHECK(st == 0, "%s, call %d: status %d", what, i, st);
  }
  size_t live = 0, all = 0;
  int count = 0;
  for (size_t bytes : fake::state().mallocs) {
    if (bytes < least) continue;
    ++count;
    live = bytes;
    all += bytes;
  }
  CHECK(count >= 1 && count <= most_allocations, "%s: %d allocations", what, count);
  CHECK(all - live < 2 * live, "%s: %zu MiB outgrown, %zu live", what, (all - live) / kMiB, live / kMiB);
  CHECK(live <= cap, "%s: %zu MiB", what, live / kMiB);
}
hipStream_t stream(int i) { return reinterpret_cast<hipStream_t>((uintptr_t)0x2000 + 16 * i); }

void run_growth() {
  // a long prompt by chunks of 2048 over an fp32 cache: pieces of 1 GiB from 131072 rows on
  rising("scored prompts", 64, 1000 * kMiB, 2, (size_t)8 << 30, [](int i) {
    return molot_hip_attn_prefill_scored(at<float>(0), at<void>(1), at<void>(2), at<float>(3), 32, 8, 2048,
                                         131072 + 2048 * i, 128, 0.1f, 129024 + 2048 * i, 0, 50.f, nullptr,
                                         nullptr, nullptr, MOLOT_KV_F32, stream(0));
  });
  // up to the limit of 8 GiB
  rising("long scored prompts", 40, 1000 * kMiB, 4, (size_t)8 << 30, [](int i) {
    return molot_hip_attn_prefill_scored(at<float>(0), at<void>(1), at<void>(2), at<float>(3), 32, 8, 256,
                                         25000 * (i + 1), 128, 0.1f, 25000 * (i + 1) - 256, 0, 50.f, nullptr,
                                         nullptr, nullptr, MOLOT_KV_F32, stream(1));
  });
  // a batch that keeps its weights, four rows more at a time: 1.1 GiB of scores
  rising("weights", 200, 512 * kMiB, 2, (size_t)8 << 30, [](int i) {
    return molot_hip_attn_decode_paged_scored(at<float>(0), at<void>(1), at<void>(2), at<float>(3),
                                              at<int32_t>(4), at<int32_t>(5), nullptr, 64, 8192, 70000 + 4 * i,
                                              64, 1, 64, 16, 0.1f, 0, 50.f, nullptr, at<float>(6),
                                              MOLOT_KV_BF16, stream(2));
  });
  // plain prompts stay within 1 GiB
  rising("plain prompts", 60, 78 * kMiB, 5, (size_t)1 << 30, [](int i) {
    return molot_hip_attn_prefill_gqa(at<float>(0), at<void>(1), at<void>(2), at<float>(3), 32, 8, 200,
                                      10000 + 2000 * i, 128, 0.1f, 9800 + 2000 * i, 0, MOLOT_KV_F32, stream(3));
  });
  // evictions of a growing cache: lists, keys and counts of every slot
  rising("evictions", 100, kMiB, 6, (size_t)1 << 30,
         [](int i) { return evict(8, 100000 + 5000 * i, 90000, stream(4)); });
  // no memory for twice the size: what the call needs
  const auto prompt_of = [](int N) {
    return molot_hip_attn_prefill_scored(at<float>(0), at<void>(1), at<void>(2), at<float>(3), 32, 8, 2048, N,
                                         128, 0.1f, N - 2048, 0, 50.f, nullptr, nullptr, nullptr, MOLOT_KV_F32,
                                         stream(5));
  };
  CHECK(prompt_of(140000) == 0, "the first prompt");
  fake::reset();
  fake::state().most = 1300 * kMiB;
  CHECK(prompt_of(150000) == 0, "a prompt with little memory left");
  bool pieces = false;
  for (const auto& l : fake::state().launches) pieces |= l.kernel.find("wide_split") != std::string::npos;
  CHECK(pieces && fake::state().refused.size() == 1, "a prompt with little memory left: its pieces");
  CHECK(hipGetLastError() == hipSuccess, "an error was left behind");
  fake::state().most = SIZE_MAX;
}

// A call that finds no memory for its workspace says so, and leaves nothing for the
// next one: its launches are not taken for failed.
void run_no_memory() {
  const auto refused = [](const char* what, auto&& call) {
    fake::reset();
    fake::state().most = kMiB / 4;
    const int st = call(true);
    CHECK(st == (int)hipErrorOutOfMemory, "%s: status %d", what, st);
    for (const auto& l : fake::state().launches)  // (but for the check of the dispatch, once)
      CHECK(l.kernel.find("xcc_probe") != std::string::npos, "%s: %s", what, l.kernel.c_str());
    CHECK(fake::last_error == hipSuccess, "%s: an error was left behind", what);
    const int next = call(false);
    CHECK(next == 0, "%s: the next call's status %d", what, next);
    fake::state().most = SIZE_MAX;
  };
  refused("a step", [](bool large) {
    return molot_hip_decode_step(at<float>(0), at<float>(1), at<float>(2), at<void>(3), at<void>(4),
                                 at<float>(5), 32, 8, 128, large ? 30000 : 20, 20, nullptr, 0.1f, 0,
                                 MOLOT_KV_F32, stream(10));
  });
  refused("an eviction", [](bool large) { return evict(8, large ? 40000 : 100, 90, stream(11)); });
  refused("a step's weights", [](bool large) {
    return large ? scored_step(8, 30000, stream(12))
                 : molot_hip_kv_track(at<float>(0), nullptr, 8, 10, 1, 9, 10, stream(12));
  });
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

// track_weights without the memory for all of it: none of it is kept, the cache runs on
// as one that tracks nothing, and a later call gets it all.
void run_track() {
  const molot::amd::LayerNorms nm;
  for (int given = 0; given < 2; ++given) {
    molot::amd::DeviceKV kv(64, 4, 128, MOLOT_KV_F32);
    const int live = fake::state().live;
    fake::state().left = given;
    CHECK(throws([&] { kv.track_weights(); }), "contiguous: no error");
    fake::state().left = INT32_MAX;
    CHECK(fake::state().live == live && !kv.acc && !kv.slot_pos, "contiguous: kept after %d", given);
    CHECK(!throws([&] {
            kv.prefill(at<float>(0), at<float>(1), at<float>(2), at<float>(3), 8, 8, 0, nullptr, 0.1f, 0, nm);
          }), "contiguous: the next prompt");
    kv.reset();
    kv.track_weights();
    CHECK(kv.acc && kv.slot_pos, "contiguous: not allocated");
  }
  for (int given = 0; given < 4; ++given) {
    molot::amd::PagedKVCache kv(2, 8, 4, 128, 16, MOLOT_KV_F32);
    const int live = fake::state().live;
    fake::state().left = given;
    CHECK(throws([&] { kv.track_weights(); }), "paged: no error");
    fake::state().left = INT32_MAX;
    CHECK(fake::state().live == live, "paged: %d kept after %d", fake::state().live - live, given);
    for (int l = 0; l < 2; ++l) CHECK(!kv.acc_pages(l) && !kv.slot_pos_pages(l), "paged: layer %d kept", l);
    CHECK(throws([&] { kv.evict({kv.add_sequence()}, 4, 1); }), "paged: evicts without books");
    kv.track_weights();
    for (int l = 0; l < 2; ++l) CHECK(kv.acc_pages(l) && kv.slot_pos_pages(l), "paged: layer %d without", l);
    const int id = kv.add_sequence();
    kv.begin_prefill(id, 20);
    for (int l = 0; l < 2; ++l)
      CHECK(!throws([&] {
              kv.prefill(l, at<float>(0), at<float>(1), at<float>(2), at<float>(3), 8, 0, nullptr, 0.1f, 0, nm);
            }), "paged: the next prompt");
    kv.end_prefill();
    CHECK(!throws([&] { kv.evict({id}, 10, 4); }), "paged: evict");
  }
}

// A batch whose larger block table finds no memory: an error, and the next one runs.
void run_table() {
  const molot::amd::LayerNorms nm;
  molot::amd::PagedKVCache kv(1, 64, 4, 128, 16, MOLOT_KV_F32);
  std::vector<int> ids;
  for (int i = 0; i < 8; ++i) ids.push_back(kv.add_sequence());
  auto step = [&](const std::vector<int>& batch) {
    kv.begin_decode(batch);
    kv.decode(0, at<float>(0), at<float>(1), at<float>(2), at<float>(3), 8, nullptr, 0.1f, 0, nm);
    kv.end_decode();
  };
  step({ids[0]});
  fake::state().left = 0;
  CHECK(throws([&] { step(ids); }), "no error");
  fake::state().left = INT32_MAX;
  CHECK(!throws([&] { step({ids[0]}); }), "the small batch again");
  CHECK(!throws([&] { step(ids); }), "the large one");
  CHECK(kv.length(ids[0]) == 3 && kv.length(ids[7]) == 1, "lengths");
}

}  // namespace

int main(int argc, char** argv) {
  const struct {
    const char* name;
    void (*run)();
  } cases[] = {{"threads", run_threads}, {"growth", run_growth}, {"no_memory", run_no_memory}, {"track", run_track}, {"table", run_table}};
  for (const auto& c : cases)
    if (argc == 2 && !std::strcmp(argv[1], c.name)) {
      c.run();
      std::printf(failures ? "%d FAILED\n" : "PASSED\n", failures);
      return failures ? 1 : 0;
    }
  std::printf("no such case\n");
  return 2;
}
