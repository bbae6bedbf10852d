// Launches of the decode attention kernels: the instance of a head dim, cache
// type, layout and head group, its plan and its LDS.
#ifndef MOLOT_AMD_CSRC_ATTN_LAUNCH_HPP_
#define MOLOT_AMD_CSRC_ATTN_LAUNCH_HPP_

#include <algorithm>

#include "attn_host.hpp"
#include "attn_kernels.hpp"
#include "molot_amd/attn_hip.h"

namespace {

using namespace molot_host;

// A planned launch of attn_kernel with configuration C.
template <int D, int GH, typename T, bool PAGED, bool ROPE, bool PAD, typename C, bool SC>
int launch_planned(AttnArgs a, int nsubs, int B, void* stream) {
  if (a.mrg && sizeof(float) * (size_t)Lds(D, GH, C::NW, C::RB, a.chunk, a.page_shift, PAGED,
                                           a.mrg).total > kMaxLds)
    no_merge(a);  // the merge's statistics do not fit beside the kernel's LDS
  const Lds L(D, GH, C::NW, C::RB, a.chunk, a.page_shift, PAGED, a.mrg);
  return launch_pair(attn_kernel<D, GH, T, PAGED, ROPE, PAD, C, SC>, C::NT,
                     sizeof(float) * (size_t)L.total, a, GH, D, nsubs, B, PAGED, ROPE, stream);
}

template <int D, int GH, typename T, bool PAGED, bool ROPE, bool PAD, typename C, bool SC>
int launch_cfg(AttnArgs a, int span, int nsubs, int B, void* stream) {
  // Q8 (d = 256): the heads of a token share 128-byte lines (see launch_pair)
  a.chunk_fast = sizeof(T) == 1;
  a.nseq = B;
  // contiguous caches: 32-row groups dealt round robin (the kernel's gmap);
  // prefill rows, like paged batches, tile each row's range in contiguous
  // chunks and merge them in the combine kernel
  const bool perseq = PAGED || (!ROPE && a.pf);
  int st = plan_launch(a, D, span, GH, nsubs, B, perseq ? C::RB : 32, 1, stream, !perseq);
  if (st) return st;
  if (a.pf) no_merge(a);
  if constexpr (sizeof(T) == 1 && C::NW > 8) {
    // Q8 chunks of at most 4 blocks a wave on 8 waves: a 1024-token window
    // of 8q/4kv/d256 (32-row chunks) 14.45 -> 10.9 us per step; 512-row
    // chunks (32k tokens, no window) stay on 16 waves (26.0 against 27.8 us)
    if (a.chunk <= 8 * 4 * C::RB)
      return launch_planned<D, GH, T, PAGED, ROPE, PAD,
                            Cfg<D, GH, T, C::LPR, C::RB, 8, C::NBUF>, SC>(a, nsubs, B, stream);
  }
  return launch_planned<D, GH, T, PAGED, ROPE, PAD, C, SC>(a, nsubs, B, stream);
}

// bf16 or Q8 KV, D = 64 or 128: the matrix-core kernel.  Workgroups per CU
// in the plan (measured): a contiguous cache 1 (c5 kernel 96.0 -> 93.2 us
// against 2; with two per CU the one dispatched second streams at about
// half the rate of the first, and the chunks left to it form the tail);
// paged batches are cut finer, their sequences differing in length: bf16
// 16 (c4 240.2 -> 235.6 us against 8), Q8 8 (c4q8: 141.5 us, 150.1 at 16).
template <int D, int GH, bool PAGED, bool ROPE, bool Q8, bool SC>
int launch_mfma(AttnArgs a, int span, int nsubs, int B, void* stream) {
  constexpr int kWpc = PAGED ? (Q8 ? 8 : 16) : 1;
  a.chunk_fast = Q8;
  a.matrix = 1;
  a.q8 = Q8;
  a.nseq = B;
  // two workgroups fit a CU; the in-launch merge needs a slot's chunks on one XCD
  // (nor for long sequences that fill the chip whatever their chunks: 64
  // sequences of 512 .. 8192 rows, bf16: 215.0 against 216.6 us; nor for
  // batches that fit in one round of single tiles: 7 of 13 .. 192, 64q, bf16:
  // 10.8 against 11.4)
  const int fit = 2 * num_cus();
  const int64_t slots = (int64_t)B * a.nkv * nsubs;
  if (PAGED && !a.pf && !a.ext_ws && knob(g_merge) <= 0 && (slots < fit || span <= kDynMax) &&
      slots * ((span + kTile - 1) / kTile) > fit)
    a.dyn = fit;
  int st = plan_launch(a, D, span, GH, nsubs, B, kTile, kWpc, stream, !PAGED);
  if (st) return st;
  // by default the combine kernel: its four waves per workgroup would fold
  // the chunks in sequential rounds (c5: 111.7 against 99.5 us per step)
  if (knob(g_merge) < 0 && !a.brief) no_merge(a);
  if (a.mrg && sizeof(float) * (size_t)LdsM(D, GH, a.chunk, a.page_shift, PAGED, Q8, a.mrg).total >
                   kMaxLds)
    no_merge(a);
  const LdsM L(D, GH, a.chunk, a.page_shift, PAGED, Q8, a.mrg);
  return launch_pair(attn_mfma_kernel<D, GH, PAGED, ROPE, Q8, SC>, kMfmaThreads,
                     sizeof(float) * (size_t)L.total, a, GH, D, nsubs, B, PAGED, ROPE, stream);
}

template <int D, int GH, typename T, bool PAGED, bool ROPE, bool PAD, bool SC>
int launch_attn(const AttnArgs& a, int span, int nsubs, int B, void* stream) {
  return launch_cfg<D, GH, T, PAGED, ROPE, PAD, typename Tune<D, GH, T>::C, SC>(a, span, nsubs, B,
                                                                           stream);
}

// Query heads per workgroup: up to 8 (d <= 256) or 4 (d = 512, whose
// 8-head workgroup would need 99 KB of LDS for its waves' partial o; 8 q
// heads of a KV head then run as two subgroups reading the rows twice).
constexpr int kMaxGhWide = 4;
template <int D, typename T, bool PAGED, bool ROPE, bool PAD, bool SC>
int dispatch_gh(int gh, const AttnArgs& a, int span, int nsubs, int B, void* st) {
  switch (gh) {
    case 1: return launch_attn<D, 1, T, PAGED, ROPE, PAD, SC>(a, span, nsubs, B, st);
    case 2: return launch_attn<D, 2, T, PAGED, ROPE, PAD, SC>(a, span, nsubs, B, st);
    case 4: return launch_attn<D, 4, T, PAGED, ROPE, PAD, SC>(a, span, nsubs, B, st);
    case 8:
      if constexpr (D <= 256 && !(sizeof(T) == 1 && D <= 128))
        return launch_attn<D, 8, T, PAGED, ROPE, PAD, SC>(a, span, nsubs, B, st);
      break;
  }
  return MOLOT_EINVAL;
}

// The vector-ALU kernels are built for D = 64, 128, 256 and 512; any other
// even head dim d <= 512 runs padded in the next of them (q zero-padded to
// D, K/V rows read at their stored length d).
template <int D, typename T, bool PAGED, bool ROPE, bool SC>
int dispatch_pad(int d, int gh, const AttnArgs& a, int span, int nsubs, int B, void* st) {
  return d == D ? dispatch_gh<D, T, PAGED, ROPE, false, SC>(gh, a, span, nsubs, B, st)
                : dispatch_gh<D, T, PAGED, ROPE, true, SC>(gh, a, span, nsubs, B, st);
}

template <typename T, bool PAGED, bool ROPE, bool SC>
int dispatch_d(int d, int gh, const AttnArgs& a, int span, int nsubs, int B, void* st) {
  if constexpr (sizeof(T) == 1) {  // Q8: 64 and 128 whole take the matrix cores (run_attn)
    if (d < 64) return dispatch_gh<64, T, PAGED, ROPE, true, SC>(gh, a, span, nsubs, B, st);
    if (d < 128) return dispatch_gh<128, T, PAGED, ROPE, true, SC>(gh, a, span, nsubs, B, st);
  } else {
    if (d <= 64) return dispatch_pad<64, T, PAGED, ROPE, SC>(d, gh, a, span, nsubs, B, st);
    if (d <= 128) return dispatch_pad<128, T, PAGED, ROPE, SC>(d, gh, a, span, nsubs, B, st);
  }
  if (d <= 256) return dispatch_pad<256, T, PAGED, ROPE, SC>(d, gh, a, span, nsubs, B, st);
  return dispatch_pad<512, T, PAGED, ROPE, SC>(d, gh, a, span, nsubs, B, st);
}

template <bool PAGED, bool ROPE, bool SC>
int dispatch_attn(int d, int kv_dtype, int gh, const AttnArgs& a, int span, int nsubs, int B,
                  void* st) {
  if (kv_dtype == MOLOT_KV_F32) return dispatch_d<float, PAGED, ROPE, SC>(d, gh, a, span, nsubs, B, st);
  if (kv_dtype == MOLOT_KV_Q8)  // 64 and 128 take the matrix cores (run_attn)
    return dispatch_d<q8_t, PAGED, ROPE, SC>(d, gh, a, span, nsubs, B, st);
  return dispatch_d<bf16_t, PAGED, ROPE, SC>(d, gh, a, span, nsubs, B, st);
}

template <int D, bool PAGED, bool ROPE, bool Q8, bool SC>
int dispatch_mfma(int gh, const AttnArgs& a, int span, int nsubs, int B, void* st) {
  switch (gh) {
    case 1: return launch_mfma<D, 1, PAGED, ROPE, Q8, SC>(a, span, nsubs, B, st);
    case 2: return launch_mfma<D, 2, PAGED, ROPE, Q8, SC>(a, span, nsubs, B, st);
    case 4: return launch_mfma<D, 4, PAGED, ROPE, Q8, SC>(a, span, nsubs, B, st);
    case 8: return launch_mfma<D, 8, PAGED, ROPE, Q8, SC>(a, span, nsubs, B, st);
    case 16: return launch_mfma<D, 16, PAGED, ROPE, Q8, SC>(a, span, nsubs, B, st);
  }
  return MOLOT_EINVAL;
}

template <bool PAGED, bool ROPE, bool SC>
int run_attn(AttnArgs& a, int d, int kv_dtype, int span, int B, void* stream) {
  a.dh = d;
  const int G = a.nq / a.nkv;
  const bool q8 = kv_dtype == MOLOT_KV_Q8;
  // (prefill rows have ranges of their own in a contiguous cache, which the
  // matrix-core kernel does not take: the vector-ALU kernel)
  if (!a.pf && (q8 || (kv_dtype == MOLOT_KV_BF16 && g_bf16_mfma)) && (d == 64 || d == 128)) {
    // up to 16 q heads of a group share each K/V tile on the MFMA columns;
    // Q8 caches of D = 64, 128 run here, D = 256 and 512 on the vector-ALU
    // kernel
    const int gh = G % 16 == 0 ? 16 : pick_gh(G);
    const int nsubs = G / gh;
    if (q8)
      return d == 64 ? dispatch_mfma<64, PAGED, ROPE, true, SC>(gh, a, span, nsubs, B, stream)
                     : dispatch_mfma<128, PAGED, ROPE, true, SC>(gh, a, span, nsubs, B, stream);
    return d == 64 ? dispatch_mfma<64, PAGED, ROPE, false, SC>(gh, a, span, nsubs, B, stream)
                   : dispatch_mfma<128, PAGED, ROPE, false, SC>(gh, a, span, nsubs, B, stream);
  }
  // Q8 rows padded to D <= 128 hold 16 q elements a lane per head: at most
  // 4 heads a workgroup there too
  const int gh = d > 256 || (q8 && d < 128) ? std::min(pick_gh(G), kMaxGhWide) : pick_gh(G);
  const int nsubs = G / gh;
  return dispatch_attn<PAGED, ROPE, SC>(d, kv_dtype, gh, a, span, nsubs, B, stream);
}

}  // namespace

#endif  // MOLOT_AMD_CSRC_ATTN_LAUNCH_HPP_
