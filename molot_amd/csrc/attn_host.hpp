// Host parts of the library that its sources share: settings, workspaces, the
// plan and the launch of a decode attention (attn_decode.hip).
#ifndef MOLOT_AMD_CSRC_ATTN_HOST_HPP_
#define MOLOT_AMD_CSRC_ATTN_HOST_HPP_

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <mutex>

#include "attn_args.hpp"

namespace molot_host __attribute__((visibility("hidden"))) {

// Process-wide settings (molot_hip_set_*): atomics, so a setter racing with
// launches on other host threads is well defined; a launch reads each once.
extern std::atomic<int> g_merge;      // split-K merge: -1 automatic, 0 combine kernel, 1 in the launch
extern std::atomic<int> g_bf16_mfma;  // bf16 KV (D = 64, 128) on the matrix-core kernel

inline int knob(const std::atomic<int>& k) { return k.load(std::memory_order_relaxed); }

// Dynamic LDS a workgroup may take (the CU's 160 KiB).
constexpr size_t kMaxLds = 160 * 1024;

int num_cus();
inline int pick_gh(int G) {
  if (G % 8 == 0) return 8;
  if (G % 4 == 0) return 4;
  if (G % 2 == 0) return 2;
  return 1;
}

// Held from a call's first use of a workspace to its last launch: its launches hand
// the workspace on to each other, so those of another host thread on the stream may
// not come between (an eviction's lists, read after them, would be something else's).
// Recursive: a prompt's launches include those of its parts.
extern std::recursive_mutex g_launch_mu;
using LaunchLock = std::lock_guard<std::recursive_mutex>;

// Per-(device, stream) workspaces: the split-K partials (with the arrival words
// of the in-launch merge), and the prefill's pieces, which the weights' scores
// share.  MOLOT_ENOWS: a capture that would have to grow one.
int workspace(void* stream, size_t bytes, unsigned long long** ctr, void** out);
int pieces_workspace(void* stream, size_t bytes, void** out);
constexpr size_t kMaxPiecesBytes = (size_t)1 << 30;  // the most that pieces_workspace is asked for,
constexpr size_t kMaxScoredBytes = (size_t)8 << 30;  // and by scored calls, which have no other path
                                                     // for long prompts, and none for the weights

// Chunking and workspace of one launch.
int plan_launch(AttnArgs& a, int d, int span, int gh, int nsubs, int B, int align, int wpc,
                void* stream, bool cyclic = false);
// Launches an attention kernel of a planned problem and, for a split context,
// the merge of its chunks after it on the same stream.
int launch_pair(AttnFn kern, int threads, size_t lds, AttnArgs a, int gh, int d, int nsubs, int B,
                bool paged, bool rope, void* stream);

// The combine kernel merges this launch's chunks instead.
inline void no_merge(AttnArgs& a) {
  a.ctr = nullptr;
  a.xmap = 0;
  a.mrg = 0;
}

// One attention launch over a contiguous or a paged cache, of plain scores or
// of scored ones (AttnArgs::scored): attn_flat.hip, attn_paged.hip and their
// scored counterparts, built side by side.
int run_flat(AttnArgs& a, bool rope, int d, int kv_dtype, int span, int B, void* stream);
int run_paged(AttnArgs& a, bool rope, int d, int kv_dtype, int span, int B, void* stream);
int run_flat_scored(AttnArgs& a, bool rope, int d, int kv_dtype, int span, int B, void* stream);
int run_paged_scored(AttnArgs& a, bool rope, int d, int kv_dtype, int span, int B, void* stream);

// The last M of a contiguous cache's n slots are new, the newest at pos
// (molot_hip_kv_track; kv_evict.hip).
int kv_track(float* acc, int32_t* slot_pos, int nkv, int n, int M, int pos, int acc_cap,
             void* stream);

}  // namespace molot_host

#endif  // MOLOT_AMD_CSRC_ATTN_HOST_HPP_
