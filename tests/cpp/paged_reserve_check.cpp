// The blocks that PagedKVCache's steps reserve, without a GPU (fake_hip.hpp): a step that
// does not begin leaves the pool and its sequences as they were.  Run by
// tests/test_paged_reserve.py.
#include "fake_hip.hpp"

#include <cstdio>
#include <functional>
#include <string>
#include <vector>

#include "check_util.hpp"
#include "molot_amd/paged_kv.hpp"

namespace {

using molot::amd::PagedKVCache;

std::string thrown(const std::function<void()>& f) {
  try {
    f();
  } catch (const std::runtime_error& e) {
    return e.what();
  }
  return "";
}
const char* const kFull = "fwd: KV cache full";

// f is refused with `why` (empty: with any error), and the blocks stay where they were.
void refused(const char* what, PagedKVCache& kv, const std::vector<int>& ids, const char* why,
             const std::function<void()>& f) {
  const int left = kv.free_blocks();
  std::vector<std::vector<int>> held;
  std::vector<int> lens;
  for (int id : ids) {
    held.push_back(kv.blocks(id));
    lens.push_back(kv.length(id));
  }
  const std::string err = thrown(f);
  CHECK(*why ? err == why : !err.empty(), "%s: '%s'", what, err.c_str());
  CHECK(kv.free_blocks() == left, "%s: %d blocks left of %d", what, kv.free_blocks(), left);
  for (size_t i = 0; i < ids.size(); ++i)
    CHECK(kv.blocks(ids[i]) == held[i] && kv.length(ids[i]) == lens[i], "%s: sequence %d", what, ids[i]);
}

// A batch that does not fit, after sequences that do; then what fits.
void run_batch() {
  PagedKVCache kv(1, 4, 2, 128, 16, MOLOT_KV_F32);
  const int a = kv.add_sequence(), b = kv.add_sequence(), c = kv.add_sequence();
  refused("batch", kv, {a, b, c}, kFull, [&] { kv.begin_batch({a, b, c}, {20, 40, 1}); });
  CHECK(thrown([&] { kv.begin_batch({b, c}, {40, 16}); }).empty(), "a batch that fits");
  kv.end_batch();
  CHECK(kv.free_blocks() == 0 && kv.blocks(a).empty(), "its blocks");
  refused("one row more", kv, {a, b, c}, kFull, [&] { kv.begin_batch({b, c, a}, {8, 0, 1}); });
  CHECK(thrown([&] { kv.begin_batch({b, c}, {8, 0}); }).empty(), "rows of the blocks at hand");
  kv.end_batch();
  CHECK(kv.length(a) == 0 && kv.length(b) == 48 && kv.length(c) == 16, "lengths");
}

// The order in which blocks come off the pool is that without the refused batch.
void run_order() {
  PagedKVCache x(1, 40, 2, 128, 16, MOLOT_KV_F32), y(1, 40, 2, 128, 16, MOLOT_KV_F32);
  std::vector<int> ids;
  for (int i = 0; i < 3; ++i) {
    ids.push_back(x.add_sequence());
    CHECK(y.add_sequence() == ids.back(), "ids");
  }
  refused("batch", x, ids, kFull, [&] { x.begin_batch(ids, {100, 33, 600}); });
  for (PagedKVCache* kv : {&x, &y}) {
    kv->begin_batch(ids, {17, 90, 1});
    kv->end_batch();
  }
  for (int id : ids) CHECK(x.blocks(id) == y.blocks(id), "blocks of sequence %d", id);
}

// Batches that fail past the reservation: too many rows' arrays for the device's memory.
void run_no_memory() {
  PagedKVCache kv(1, 60, 2, 128, 16, MOLOT_KV_F32);
  const int a = kv.add_sequence(), b = kv.add_sequence();
  fake::state().left = 0;
  refused("table", kv, {a, b}, "", [&] { kv.begin_batch({a, b}, {30, 5}); });
  fake::state().left = 1;  // (the table's)
  refused("rows", kv, {a, b}, "", [&] { kv.begin_batch({a, b}, {30, 5}); });
  fake::state().left = 0;
  refused("prompt", kv, {a, b}, "", [&] { kv.begin_prefill(b, 700); });
  fake::state().left = INT32_MAX;
  CHECK(thrown([&] { kv.begin_batch({a, b}, {30, 5}); }).empty(), "with memory");
  kv.end_batch();
  CHECK(kv.free_blocks() == 57, "blocks");
}

void run_decode() {
  PagedKVCache kv(1, 2, 2, 128, 16, MOLOT_KV_F32);
  const int a = kv.add_sequence(), b = kv.add_sequence(), c = kv.add_sequence();
  refused("decode", kv, {a, b, c}, kFull, [&] { kv.begin_decode({a, b, c}); });
  CHECK(thrown([&] { kv.begin_decode({b, c}); }).empty(), "a step that fits");
  kv.end_decode();
  refused("prompt", kv, {a, b, c}, kFull, [&] { kv.begin_prefill(b, 16); });
  refused("no such sequence", kv, {a, b, c}, "", [&] { kv.begin_decode({b, 7}); });
}

}  // namespace

int main(int argc, char** argv) {
  const struct {
    const char* name;
    void (*run)();
  } cases[] = {{"batch", run_batch}, {"order", run_order}, {"no_memory", run_no_memory}, {"decode", run_decode}};
  for (const auto& c : cases)
    if (argc == 2 && c.name == std::string(argv[1])) {
      c.run();
      std::printf(failures ? "%d FAILED\n" : "PASSED\n", failures);
      return failures ? 1 : 0;
    }
  std::printf("no such case\n");
  return 2;
}
