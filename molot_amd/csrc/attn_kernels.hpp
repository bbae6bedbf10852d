// The decode attention kernels (attn_kernel, attn_mfma_kernel) and the parts
// of them that the merge and prefill kernels share.
#ifndef MOLOT_AMD_CSRC_ATTN_KERNELS_HPP_
#define MOLOT_AMD_CSRC_ATTN_KERNELS_HPP_

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "attn_args.hpp"
#include "device_util.hpp"
#include "paged_plan.hpp"
#include "score_mod.hpp"

namespace {

// Sum over the workgroup (at most 16 waves); every thread gets the total.
__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = group_sum<64>(v);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
  for (int k = 0; k < (int)((blockDim.x + 63) >> 6); ++k) t += sh[k];
  __syncthreads();
  return t;
}

// Maximum over the workgroup (at most 16 waves); every thread gets it.
__device__ __forceinline__ float block_max(float v, float* sh) {
  v = group_max<64>(v);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = sh[0];
  for (int k = 1; k < (int)((blockDim.x + 63) >> 6); ++k) t = fmaxf(t, sh[k]);
  __syncthreads();
  return t;
}
// ---------------------------------------------------------------------------
// Fused decode attention.
//
// SC: a scored launch (AttnArgs::scored): the scores of the launch's rows go through
// the cap and the bias before the softmax, and where the caller keeps weights they
// are also stored, with each chunk's (max, sum), for attn_weights_kernel.  us a step,
// unscored | nothing to score, a cap, slopes, both | weights, weights and a cap:
//   32q/8kv/d128 fp32, 16385 rows   25.9 | 26.2, 26.3, 27.0, 27.2 | 26.5, 26.6
//   bf16, 16001                     18.9 | 19.3, 19.5, 19.6, 19.7 | 20.0, 20.2
//   Q8, 16001                       15.9 | 17.1, 17.5, 17.1, 17.6 | 17.5, 18.1
//   64q/8kv/d128 bf16, 131072       100 | 98, 98, 98, 98 | 126, 126
//   8q/4kv/d256 fp32, window 1024   8.7 | 9.0, 9.1, 9.7, 9.8 | 8.9, 8.9
//   13 paged sequences of 1 to 2999 rows, Q8: 19.3 | 20.3, 20.5 | 23.0, 23.5
// So a scored step is bounded by what bounds the plain one; the weights by their second
// launch (0.3 to 3 us) and, in a long cache, by the stores of the scores between the loads.
//
// Grid (nkv * subgroups, sequences, chunks).  Workgroup (h/sub, b, c) owns
// chunk c of the context rows of KV head h and the GH query heads
// hq0 .. hq0+GH-1 of that head's group: a paged cache's rows [tb, tb + cnt),
// a contiguous cache's 32-row groups c, c + nchunks, c + 2*nchunks, ... of the
// range.  The workgroups sharing (b, h/sub) form a "slot".
//   1. prologue: the first block(s) of K/V rows of every wave, then q of the
//      GH heads into LDS; with ROPE, q is rotated there, and the workgroup
//      holding the chunk that contains the new token rotates k_new and
//      rounds k/v to the cache type in LDS.  Every wave issues the same
//      loads on every path and the barriers order LDS only, so nothing waits
//      for the K/V blocks in flight before it has to;
//   2. every wave streams blocks of RB rows (NBUF blocks in flight); blocks
//      past the first NBUF per wave are claimed from a workgroup counter in
//      LDS, so waves that are served faster take more.  Scores of the GH
//      heads per K row (LPR lanes per row, DPP sums); online softmax per
//      wave (running max, rescale of the accumulators); probabilities through
//      a per-wave LDS slice to the PV lanes (LPR2 lanes per V row, 16 bytes
//      each);
//   3. the new token (ROPE, last chunk): folded in by wave 0 from LDS, and
//      stored into the cache slot n-1 by subgroup 0 as the kernel's last
//      step (no workgroup reads that slot in this launch);
//   4. the waves' (max, sum, o) are merged through LDS; every thread derives
//      its own outputs' chunk partial.  A single-chunk problem writes
//      o / sum (and the rotated q) directly;
//   5. otherwise the chunk partial (o, max, sum) goes to the workspace, and
//      combine_kernel, launched next on the same stream, merges the chunks
//      of every slot with log-sum-exp weights and writes O (and, with ROPE,
//      the rotated q, which chunk 0 leaves in the workspace: q is rotated in
//      place, so it is written back only after every workgroup has read it).

// Work mapping of one kernel instance.
//   LPR   lanes cooperating on one K row in the score loop (DPP sums across them)
//   RB    rows per wave block
//   NW    waves per workgroup
//   NBUF  blocks in flight per wave: 1 (load, then score) or 2 (one block is
//         scored while the next one's loads are outstanding)
template <int D, int GH, typename T, int LPR_, int RB_, int NW_, int NBUF_ = 1>
struct Cfg {
  static constexpr int NBUF = NBUF_;
  static_assert(NBUF == 1 || NBUF == 2, "one or two blocks in flight");
  static constexpr int VW = KVT<T>::VW;
  static constexpr int LPR = LPR_;
  static constexpr int NV = D / (LPR * VW);  // 16-byte vectors per lane per K row
  static constexpr int EPL = NV * VW;        // q elements per lane
  static constexpr int RPS = 64 / LPR;       // K rows per wave step
  // PV: a V row is LPR2 <= 64 lanes of NV2 16-byte vectors each (NV2 = 2
  // for fp32 rows of 512 elements); lane cs holds row elements
  // (v2*LPR2 + cs)*VW .. +VW-1, so each v2 reads LPR2*16 contiguous bytes
  static constexpr int NV2 = (D / VW + 63) / 64;
  static constexpr int LPR2 = D / (VW * NV2);  // lanes per V row
  static constexpr int AW = VW * NV2;          // o accumulators per head and lane
  static constexpr int RPI = 64 / LPR2;        // V rows per wave step
  static constexpr int RB = RB_;
  static constexpr int KS = RB / RPS;  // K steps per block
  static constexpr int VS = RB / RPI;  // V steps per block
  static constexpr int NW = NW_;
  static constexpr int NT = NW * 64;
  static constexpr int P = GH * D;
  // chunk partial: PP output pairs per thread (P > NT), Q threads per copy
  static constexpr int PP = (P + NT - 1) / NT;
  static constexpr int Q = P < NT ? P : NT;
  static_assert(NV >= 1 && D % (LPR * VW) == 0 && LPR <= 64, "bad score mapping");
  static_assert(LPR2 * VW * NV2 == D && LPR2 <= 64 && 64 % LPR2 == 0, "bad PV mapping");
  static_assert(RB % RPS == 0 && RB % RPI == 0, "bad block");
  static_assert(P % 64 == 0 || P <= NT, "pairs per phase");
};

// Default mapping: q registers (GH x D/LPR) kept at <= 32 where the 16-byte
// vector allows it; one block in flight per wave; 8-row blocks at two waves
// per SIMD where D <= 128 and the register estimate allows, else the block size with the
// most waves per SIMD; one workgroup per CU (NW = 4 x waves per SIMD, at
// most 16).
template <int D, int GH, typename T>
struct Tune {
  static constexpr int VW = KVT<T>::VW;
  static constexpr int lpr() {
    int l = D / VW < 8 ? D / VW : 8;  // Q8 at D = 64: 4 lanes of 16 codes a row
    while (GH * D / l > 32 && l < D / VW && l < 64) l *= 2;
    return l;
  }
  static constexpr int LPR = lpr();
  static constexpr int NV = D / (LPR * VW);
  static constexpr int NV2 = (D / VW + 63) / 64;
  static constexpr int RPS = 64 / LPR, RPI = 64 / (D / (VW * NV2));
  static constexpr int loads(int rb) { return (rb / RPS) * NV + (rb / RPI) * NV2; }
  static constexpr int regs(int rb) {  // one block of data + its addresses
    return GH * NV * VW + GH * VW * NV2 + 6 * loads(rb) + (rb / RPS) * GH + 3 * GH + 40;
  }
  static constexpr int wps(int rb) {
    const int r = (regs(rb) + 7) / 8 * 8;
    const int w = 512 / r;
    return w > 4 ? 4 : w;
  }
  static constexpr bool ok(int rb) {
    return rb % RPS == 0 && rb % RPI == 0 && loads(rb) <= 16 && wps(rb) >= 2;
  }
  // 8-row blocks and two waves per SIMD where the registers allow (D <= 128):
  // the same bytes in flight per CU as 4-row blocks at four waves per SIMD,
  // with half the waves to merge at the chunk's end (measured, 32q/8kv/d128
  // fp32: step 28.8 -> 27.3 us at n = 16385, 14.0 -> 13.3 us at n = 4097;
  // at d = 256, 8q/4kv with a 1024 window, 12 waves of 4-row blocks stay
  // faster: 9.3 against 9.6 us).
  // d = 512: the largest block whose loads fit at two waves per SIMD (fp32
  // 4 rows = 16 KB of K and V a wave, bf16 8 rows), else at one.
  static constexpr bool fits(int rb, int w) {
    return rb % RPS == 0 && rb % RPI == 0 && loads(rb) <= 16 && wps(rb) >= w;
  }
  static constexpr int rb() {
    if (D <= 128 && ok(8)) return 8;
    if (D > 256) {
      for (int w : {2, 1})
        for (int r : {16, 8, 4, 2, 1})
          if (fits(r, w)) return r;
    }
    int best = 0;
    for (int r : {16, 4})
      if (ok(r) && (best == 0 || wps(r) > wps(best))) best = r;
    if (best) return best;
    return RPS > RPI ? RPS : RPI;
  }
  static constexpr int RB = rb();
  static constexpr int nw() {
    const int w = RB == 8 ? 2 : (wps(RB) >= 1 ? wps(RB) : 1);
    int nw = 4 * w;
    // wave-merge buffer <= 32 KiB (64 KiB at d = 512, one workgroup a CU:
    // two waves per SIMD instead of one: 8q/2kv/d512 Q8 step
    // 32.7 -> 29.8 us, fp32 61.5 -> 60.9 us)
    while (nw > 4 && nw * GH * D > (D > 256 ? 16384 : 8192)) nw -= 4;
    return nw;
  }
  static constexpr int NW = nw();
  // d = 512 (fp32 and bf16) and d = 128 fp32: two blocks of half the rows
  // in flight, so a wave's next loads go out before it scores the current
  // block (same box, interleaved: 8q/2kv/d512 step fp32 60.9 -> 60.2 us,
  // bf16 36.4 -> 34.4 us; 32q/8kv/d128 fp32 at n = 4097 12.11 -> 11.99 us,
  // at n = 16385 25.88 against 25.85 us; two 8-row blocks 13.04 and 26.31).
  // Q8 keeps one block (2.6x slower with two of half the rows), and d = 256
  // gains nothing (8q/4kv window 1024: 9.28 against 9.28 us).
  static constexpr bool H2 = (D > 256 || (D == 128 && sizeof(T) == 4)) && sizeof(T) != 1 &&
                             RB >= 2 && (RB / 2) % RPS == 0 && (RB / 2) % RPI == 0;
  using C = Cfg<D, GH, T, LPR, H2 ? RB / 2 : RB, NW, H2 ? 2 : 1>;
};

// Dynamic LDS layout shared by host (size) and device (offsets), in floats.
struct Lds {
  int qs, cs, sn, knew, vnew, nw, pw, wm, wl, red, blk, misc, mrg, qw, psum, total;
  __host__ __device__ Lds(int D, int GH, int NW, int RB, int chunk, int page_shift, bool paged,
                          int merge) {
    const bool wide = D / 4 > 64;  // a q row spans more than one wave (d = 512)
    int o = 0;
    qs = o; o += GH * D;
    qw = o; o += wide ? D : 0;       // q norm weights
    // q rows' sums of squares, per 64 quads (padded: later regions are read
    // as 16-byte vectors)
    psum = o; o += wide ? (GH * (D / 256) + 3) / 4 * 4 : 0;
    cs = o; o += D / 2;
    sn = o; o += D / 2;
    knew = o; o += D;
    vnew = o; o += D;
    nw = o; o += D;                  // k norm weights
    pw = o; o += NW * RB * GH;
    wm = o; o += NW * GH;
    wl = o; o += NW * GH;
    red = o; o += NW * GH * D;       // per-wave o
    blk = o; o += paged ? ((chunk >> page_shift) + 2) : 0;
    misc = o; o += 8;                // block claim counter, merge flag
    mrg = o; o += merge;             // in-launch merge: chunk statistics
    total = o;
  }
};


// RMS norms of the step's fresh vectors (forward.h:554, 562-563):
// y = (x * 1/sqrt(mean(x^2) + eps)) * w (rmsnorm, include/molot/norm.h:9-28).
//
// q, in registers before it is staged: thread i of the prologue holds the
// float4 i of the GH q rows, so each row is D/4 aligned lanes of a wave and
// its sum of squares a group sum, with no LDS round trip and no barrier.
template <int D, int QPT>
__device__ __forceinline__ void q_norm_regs(const AttnArgs& a, f32x4 (&qv)[QPT],
                                            const f32x4 (&qw)[QPT], int dh) {
  static_assert(D / 4 <= 64 && 64 % (D / 4) == 0, "a q row within one wave");
#pragma unroll
  for (int u = 0; u < QPT; ++u) {
    float ss = qv[u][0] * qv[u][0];
    ss = fmaf(qv[u][1], qv[u][1], ss);
    ss = fmaf(qv[u][2], qv[u][2], ss);
    ss = fmaf(qv[u][3], qv[u][3], ss);
    const float inv = 1.0f / sqrtf(group_sum<D / 4>(ss) / (float)dh + a.eps);
#pragma unroll
    for (int e = 0; e < 4; ++e) qv[u][e] = qv[u][e] * inv * qw[u][e];
  }
}

// k and v of the new token, in the workgroup that appends it: the waves'
// partial sums of squares go to LDS before the prologue's barrier (k: one
// element per thread; v: all nkv*D values of v_new, see v_norm_load), and
// the threads that rotate k and round v after that barrier scale them:
// k by 1/sqrt(mean(k^2) + eps) and its weights (staged in LDS), v by the RMS
// of all of v_new without weights (rmsnorm_plain, norm.h:82-96).
__device__ __forceinline__ void k_norm_share(int w, int lane, float ss, float* ksum) {
  ss = group_sum<64>(ss);
  if (lane == 0) ksum[w] = ss;
}

struct NewNorms {
  float kinv, vinv;
  __device__ __forceinline__ void apply(const AttnArgs& a, const float* kw, int j, int half,
                                        float& k0, float& k1, float& v0, float& v1) const {
    if (a.k_norm) {
      k0 = k0 * kinv * kw[j];
      k1 = k1 * kinv * kw[j + half];
    }
    if (a.v_norm) {
      v0 *= vinv;
      v1 *= vinv;
    }
  }
};

template <int D, int NW>
__device__ __forceinline__ NewNorms new_norms(const AttnArgs& a, const float* ksum,
                                              const float* vsum, int dh) {
  NewNorms r{1.f, 1.f};
  if (a.k_norm) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) ss += ksum[k];
    r.kinv = 1.0f / sqrtf(ss / (float)dh + a.eps);
  }
  if (a.v_norm) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) ss += vsum[k];
    r.vinv = 1.0f / sqrtf(ss / (float)(a.nkv * dh) + a.eps);
  }
  return r;
}

// The joint v norm needs all nkv*D values of the sequence's v_new.  Their
// loads are issued in the prologue before any K/V row (loads retire in
// order, so the sum below does not wait for the stream's first block), up
// to kVnPT per thread; the rest, if any, are summed by a plain loop.
constexpr int kVnPT = 8;

template <int D, int NT>
__device__ __forceinline__ void v_norm_load(const AttnArgs& a, int b, int tid, float (&vq)[kVnPT],
                                            int dh) {
  const float* vx = a.v_new + (int64_t)b * a.nkv * dh;
  const int nv = a.nkv * dh;
#pragma unroll
  for (int u = 0; u < kVnPT; ++u) vq[u] = tid + u * NT < nv ? vx[tid + u * NT] : 0.f;
}

// The wave's sum of squares of its threads' shares into vsum[w].
template <int D, int NT>
__device__ __forceinline__ void v_norm_share(const AttnArgs& a, int b, int tid, int w, int lane,
                                             const float (&vq)[kVnPT], float* vsum, int dh) {
  float ss = 0.f;
#pragma unroll
  for (int u = 0; u < kVnPT; ++u) ss = fmaf(vq[u], vq[u], ss);
  const float* vx = a.v_new + (int64_t)b * a.nkv * dh;
  for (int j = tid + kVnPT * NT; j < a.nkv * dh; j += NT) ss = fmaf(vx[j], vx[j], ss);
  ss = group_sum<64>(ss);
  if (lane == 0) vsum[w] = ss;
}

// The workgroup's chunk partial from its waves' partials in LDS: running
// max wm[w*GH + g], sum wl[w*GH + g] and unnormalised o red[w*RS + g*D + d]
// of wave w (waves without rows hold max -inf).  A single-chunk problem
// writes O = o / l (and, with ROPE, the rotated q from qs) directly;
// otherwise (o, max, sum) goes to the workspace for combine_kernel.
// ---------------------------------------------------------------------------
// In-launch merge of the split-K chunk partials.
//
// Workgroup i runs on XCD i % 8 (the dispatch order of MI355X in its
// single-partition mode, checked once per device by xcd_map_ok() before the
// library relies on it), and the launch places every chunk of a slot on the
// same XCD.  The slot's partials therefore meet in one L2, the coherence
// point of that XCD's CUs, and the hand-off needs no cache writeback:
//   - each workgroup stores its partial (plain stores, which write through
//     the CU's L1 into the L2), waits until the L2 has acknowledged them
//     (a workgroup-scope release fence, s_waitcnt vmcnt(0), in every thread,
//     then a barrier) and adds one arrival to the slot's 64-bit arrival word
//     (a device-scope atomic, coherent across the XCDs);
//   - the arrival adds 1 + x*2^13 + x^2*2^29 for its XCD x = XCC_ID: the
//     word counts the arrivals (bits 0-12), and sums x (bits 13-28) and x^2
//     (bits 29-63).  The workgroup whose add completes the count arrived
//     last: every other chunk's stores were acknowledged before its arrival.
//     It resets the word to 0 for the next launch.  All nch chunks ran on
//     its own XCD m exactly when the sums are nch*m and nch*m^2 (the
//     variance of the XCDs is then 0), checked from the atomic's own
//     return value, so a violated dispatch assumption can never be read
//     from a stale record: the output is then NaN, never a stale merge;
//   - it reads the partials back with loads that miss the L1 (cache policy
//     sc0), so they come from the L2, merges them with log-sum-exp weights
//     as combine_kernel does and writes O and, with ROPE, the rotated q
//     (every workgroup of the slot has read q by the time it arrives).
// No workgroup waits for another: nothing spins, and a launch's arrivals
// are exactly its slots' chunk counts, so the words are back at zero when
// it ends (they are zeroed when the workspace is allocated).
constexpr int kArriveCountBits = 13;  // arrivals of a slot: at most kMergeMaxChunks
constexpr int kArriveSumBits = 16;    // sum of XCC_ID over the arrivals (<= 7 * 4096)
__device__ __forceinline__ unsigned long long arrive_word(int x) {
  const unsigned long long ux = (unsigned long long)x;
  return 1ull | (ux << kArriveCountBits) | ((ux * ux) << (kArriveCountBits + kArriveSumBits));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t l2_rsrc(const float* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, 0x7FFFFFFF, 0x00020000);
}
// The scores of KV head h of sequence b (AttnArgs::scores), none of a step that keeps none.
// Stores past the end are dropped, so the kernels' loops store at every tile, a lane without
// a score at offset -1: with a store under a branch the wait for the next tile's rows, which
// counts what was issued after them, would wait for the stores as well.  us a step, 64q/8kv/
// d128 bf16, 131072 keys: 137 with the branch, 130 without; 16384: 21.9, 20.4 (a step that
// keeps no scores pays 0.2).
template <typename A>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t score_rsrc(const A& a, int b, int h) {
  const int64_t rows = a.sc_rows * (a.nq / a.nkv);
  return __builtin_amdgcn_make_buffer_rsrc(a.scores + ((int64_t)b * a.nkv + h) * rows, 0,
                                           a.scores ? (int)(4 * rows) : 0, 0x00020000);
}
// Loads at a byte offset of a resource, missing the L1 (cache policy sc0).
__device__ __forceinline__ f32x4 ld_l2x4(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 1));
}

__device__ __forceinline__ float2 ld_l2x2(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 1));
}

// XCD (accelerator complex) of the calling wave: hardware register XCC_ID.
__device__ __forceinline__ int xcc_id() {
  return (int)(__builtin_amdgcn_s_getreg((20) | (0 << 6) | (3 << 11)) & 15);
}

// Output element pr of a head group's GH x D tile (head g = pr / D, element
// j = pr % D) in the caller's [..][dh] rows: its index from qrow0's row, or
// -1 for the padding (j >= dh) of a padded launch.
__device__ __forceinline__ int64_t out_index(int64_t qrow0, int pr, int D, int dh) {
  const int g = pr / D, j = pr - g * D;
  return j < dh ? (qrow0 + g) * dh + j : -1;
}

// Stores float4 quad q (elements 4q .. 4q+3 of the GH x D tile) of a head
// group's output; dh is even, so a quad is whole or half inside a row.
__device__ __forceinline__ void store_quad(float* o, int64_t qrow0, int q, f32x4 v, int D, int dh) {
  const int64_t i0 = out_index(qrow0, 4 * q, D, dh);
  if (i0 < 0) return;
  if (dh == D || 4 * q % D + 4 <= dh) {
    if ((i0 & 3) == 0) {
      *reinterpret_cast<f32x4*>(o + i0) = v;
    } else {  // dh % 4 == 2: an 8-byte aligned row start
      *reinterpret_cast<float2*>(o + i0) = float2{v[0], v[1]};
      *reinterpret_cast<float2*>(o + i0 + 2) = float2{v[2], v[3]};
    }
  } else {
    *reinterpret_cast<float2*>(o + i0) = float2{v[0], v[1]};
  }
}

constexpr int kMergeMaxChunks = 4096;  // chunks of a slot merged in the launch
static_assert(kMergeMaxChunks < (1 << kArriveCountBits) &&
                  7 * kMergeMaxChunks < (1 << kArriveSumBits) &&
                  49ull * kMergeMaxChunks < (1ull << (64 - kArriveCountBits - kArriveSumBits)),
              "arrival word fields");
constexpr int kMergeAutoSpan = 8192;   // rows from which the default merges in the launch
constexpr int kMergeMaxPhases = 64;    // threads per float4 quad of the output (NT / quads)
constexpr int kMergeRound = 8;         // chunks per thread whose loads are in flight together

// LDS floats of the in-launch merge's phase statistics (Lds::mrg, LdsM::mrg).
__host__ __device__ constexpr int merge_lds_floats(int gh) { return 2 * kMergeMaxPhases * gh; }

// The merge of the workgroup that completes a slot.  Thread t owns float4
// quad q = t % QV of the slot's output (head g = 4q / D) in phase
// ph = t / QV; it folds chunks ph, ph + PH, ph + 2*PH, ... with a running
// log-sum-exp, kMergeRound chunks' loads in flight at a time and only the
// chunks that exist loaded.  The PH phases of a quad then merge once
// through LDS: their (max, sum) per head at mst, their o at mred.  Wave 0
// alone reads the chunks' XCD records (lane c: chunks c, c + 64, ...): with
// a record load per chunk in every thread the merge took 0.4 us longer
// (32q/8kv/d128 fp32, n = 16385).
// RED: floats of LDS at mred (the phase sums: PH*P floats).
template <int D, int GH, int NW, int NT, bool ROPE, int RED, int QSTR = D>
__device__ __forceinline__ void arrive_and_merge(const AttnArgs& a, int64_t slot, int nch,
                                                 int64_t qrow0, const float* qs, float* mst,
                                                 float* mred, int* flag, int tid, int lane,
                                                 int dh) {
  constexpr int P = GH * D;
  // this thread's partial stores are acknowledged by the L2 (vmcnt(0):
  // outside threadgroup-split mode the workgroup-scope release fence alone
  // need not wait for them)
  wait_vmcnt<0>();
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  lds_barrier();
  if (tid == 0) {
    const int x = xcc_id();
    const unsigned long long tot = atomicAdd(a.ctr + slot, arrive_word(x)) + arrive_word(x);
    const bool last = (int)(tot & ((1ull << kArriveCountBits) - 1)) == nch;
    if (last) atomicExch(a.ctr + slot, 0ull);  // ready for the next launch
    const unsigned long long n64 = (unsigned long long)nch, x64 = (unsigned long long)x;
    const bool one_xcd = ((tot >> kArriveCountBits) & ((1ull << kArriveSumBits) - 1)) == n64 * x64 &&
                         (tot >> (kArriveCountBits + kArriveSumBits)) == n64 * x64 * x64;
    flag[0] = last;
    flag[1] = last && !one_xcd;  // a chunk of the slot ran on another XCD
  }
  lds_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  if (!flag[0]) return;  // uniform over the workgroup

  constexpr int QV = P / 4;                     // float4 quads of the slot's output
  // phases per quad: as many as the threads allow and the phase sums' LDS holds
  constexpr int PH0 = NT >= QV ? NT / QV : 1;
  constexpr int PH = PH0 * P <= RED ? PH0 : (RED / P > 1 ? RED / P : 1);
  constexpr int NQ = NT >= QV ? 1 : (QV + NT - 1) / NT;  // quads per thread
  static_assert(P % 4 == 0 && D % 4 == 0, "float4 quads");
  static_assert(PH <= kMergeMaxPhases, "phase statistics fit their LDS");
  const int ph = NT >= QV ? tid / QV : 0;
  const bool act = ph < PH;  // threads past PH * QV idle (NT not a multiple of QV)
  const __amdgpu_buffer_rsrc_t ro = l2_rsrc(a.part_o + slot * a.nchunks * P);
  const __amdgpu_buffer_rsrc_t rm = l2_rsrc(a.part_ml + slot * a.nchunks * (GH * 2));
  int qd[NQ], g[NQ];
  float m[NQ], l[NQ];
  f32x4 o[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    qd[i] = NT >= QV ? tid % QV : min(tid + i * NT, QV - 1);
    g[i] = 4 * qd[i] / D;
    m[i] = -INFINITY;
    l[i] = 0.f;
    o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int c0 = act ? ph : nch; c0 < nch; c0 += PH * kMergeRound) {
    float2 st[NQ][kMergeRound];
    f32x4 ov[NQ][kMergeRound];
#pragma unroll
    for (int u = 0; u < kMergeRound; ++u) {
      const int cc = c0 + PH * u;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (cc < nch) {
          st[i][u] = ld_l2x2(rm, 8 * (cc * GH + g[i]));
          ov[i][u] = ld_l2x4(ro, 16 * (cc * QV + qd[i]));
        } else {
          st[i][u] = float2{-INFINITY, 0.f};
          ov[i][u] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      float mn = m[i];
#pragma unroll
      for (int u = 0; u < kMergeRound; ++u) mn = fmaxf(mn, st[i][u].x);
      const float al = softmax_exp(m[i] - mn);  // m = -inf on the first round: 0
      l[i] *= al;
      o[i] *= al;
#pragma unroll
      for (int u = 0; u < kMergeRound; ++u) {
        const float wc = softmax_exp(st[i][u].x - mn);  // absent chunks: e^-inf = 0
        l[i] = fmaf(wc, st[i][u].y, l[i]);
        o[i] += wc * ov[i][u];
      }
      m[i] = mn;
    }
  }
  // The hand-off above holds only if every chunk of the slot ran on this
  // XCD (one L2): otherwise the output is NaN, never a silently stale merge.
  const float bad = flag[1] ? __builtin_nanf("") : 0.f;
  if constexpr (PH > 1) {
    // a phase's (max, sum) is the same for every quad of a head: the
    // thread holding the head's first quad publishes it
    if (act) {
      reinterpret_cast<f32x4*>(mred)[ph * QV + qd[0]] = o[0];
      if ((4 * qd[0]) % D == 0) {
        mst[(ph * GH + g[0]) * 2] = m[0];
        mst[(ph * GH + g[0]) * 2 + 1] = l[0];
      }
    }
    lds_barrier();
    if (tid < QV) {
      float M = -INFINITY;
#pragma unroll
      for (int q2 = 0; q2 < PH; ++q2) M = fmaxf(M, mst[(q2 * GH + g[0]) * 2]);
      float Ls = 0.f;
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q2 = 0; q2 < PH; ++q2) {
        const float wq = softmax_exp(mst[(q2 * GH + g[0]) * 2] - M);  // phases with no chunk: 0
        Ls = fmaf(wq, mst[(q2 * GH + g[0]) * 2 + 1], Ls);
        acc += wq * reinterpret_cast<const f32x4*>(mred)[q2 * QV + tid];
      }
      store_quad(a.o, qrow0, tid, acc / Ls + bad, D, dh);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int q4 = NT >= QV ? tid : tid + i * NT;
      if (act && q4 < QV) store_quad(a.o, qrow0, q4, o[i] / l[i] + bad, D, dh);
    }
  }
  if constexpr (ROPE) {
    if (a.q_out)
      for (int i = tid; i < P; i += NT) {
        const int64_t oi = out_index(qrow0, i, D, dh);
        if (oi >= 0) a.q_out[oi] = qs[(i / D) * QSTR + i % D];
      }
  }
}

// SC: the waves' maxima at wm are in base-2 units, and (with scores) the chunk's
// (max, sum) goes to stats in them too.
template <int D, int GH, int NW, int NT, bool ROPE, int RED, bool XSW = false, int QSTR = D,
          bool SC = false>
__device__ __forceinline__ void finish_chunk(const AttnArgs& a, const float* wm, const float* wl,
                                             const float* red, int RS, const float* qs, int tid,
                                             int lane, bool split, int64_t slot, int c,
                                             int64_t qrow0, int nch, float* mst, float* mred,
                                             int* flag, int dh) {
  constexpr int P = GH * D;
  // Every thread derives the chunk partial of its own output pairs from the
  // wave partials (wave weights e^(m_w - M); waves without rows weigh
  // e^-inf = 0).  Pairs: tid % Q + i*Q, i < PP; phase ph = tid / P.
  constexpr int PP = (P + NT - 1) / NT, Q = P < NT ? P : NT;
  const int ph = PP == 1 ? tid / P : 0;
  int pr_[PP], g_[PP];
  bool pv_[PP];
  float po[PP], pm[PP], pl[PP];
  // The 64 pairs of a wave lie in one head (D is a multiple of 64), so the
  // wave weights are wave-uniform: lane ww < NW computes wave ww's weight,
  // DPP/shuffle reductions give the chunk max and sum, and the weights reach
  // every lane through readlane.
  static_assert(D % 64 == 0 && NW <= 64, "wave-uniform head per 64 pairs");
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    pr_[i] = tid % Q + i * Q;
    pv_[i] = pr_[i] < P;
    g_[i] = pv_[i] ? pr_[i] / D : 0;
    const int g = __builtin_amdgcn_readfirstlane(g_[i]);
    const float mw_l = lane < NW ? wm[lane * GH + g] : -INFINITY;
    const float m = group_max<NW <= 16 ? 16 : 64>(mw_l);  // lanes >= NW hold -inf
    // waves without rows weigh 0 (also when no wave of the chunk has one)
    const float d_l = mw_l - m;
    const float e_l =
        lane < NW && mw_l != -INFINITY ? (SC ? exp2_hw(d_l) : softmax_exp(d_l)) : 0.f;
    const float l = group_sum<NW <= 16 ? 16 : 64>(lane < NW ? e_l * wl[lane * GH + g] : 0.f);
    float o = 0.f;
    // XSW: head g's element j at g*D + (j ^ 4*(g % 8)) (the matrix-core
    // kernel's conflict-free layout)
    const int ri =
        !pv_[i] ? 0 : XSW ? g_[i] * D + ((pr_[i] - g_[i] * D) ^ (4 * (g_[i] & 7))) : pr_[i];
#pragma unroll
    for (int ww = 0; ww < NW; ++ww)
      o = fmaf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(e_l), ww)),
               red[ww * RS + ri], o);
    po[i] = o;
    pm[i] = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(m)));
    pl[i] = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(l)));
  }
  const bool lead = ph == 0;  // phase 0 threads own the chunk partial's outputs
  if constexpr (SC) {
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      if (a.scores && lead && pv_[i] && pr_[i] - g_[i] * D == 0) {
        float* st = a.stats + ((slot * a.nchunks + c) * GH + g_[i]) * 2;
        st[0] = pm[i];
        st[1] = pl[i];
      }
      pm[i] *= kLn2;
    }
  }
  if (!split) {
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const int64_t oi = lead && pv_[i] ? out_index(qrow0, pr_[i], D, dh) : -1;
      if (oi >= 0) a.o[oi] = po[i] / pl[i];
    }
    if constexpr (ROPE) {
      if (a.q_out)
        for (int i = tid; i < P; i += NT) {
          const int64_t oi = out_index(qrow0, i, D, dh);
          if (oi >= 0) a.q_out[oi] = qs[(i / D) * QSTR + i % D];
        }
    }
    return;
  }

  // ---- 5. the chunk partial for the combine kernel ----
  // Plain stores: the combine kernel runs after this one on the same stream,
  // so the kernel boundary orders them; no flag, counter or cleared memory
  // is needed between the two launches.
  float* po_s = a.part_o + (slot * a.nchunks + c) * P;
  float* pml_s = a.part_ml + (slot * a.nchunks + c) * (GH * 2);
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    if (!(lead && pv_[i])) continue;
    po_s[pr_[i]] = po[i];
    if (pr_[i] - g_[i] * D == 0) {
      pml_s[2 * g_[i]] = pm[i];
      pml_s[2 * g_[i] + 1] = pl[i];
    }
  }
  if (a.ctr) {  // in-launch merge: the workgroup completing the slot merges it
    arrive_and_merge<D, GH, NW, NT, ROPE, RED, QSTR>(a, slot, nch, qrow0, qs, mst, mred, flag, tid,
                                               lane, dh);
    return;
  }
  if constexpr (ROPE) {  // the rotated q leaves through the combine kernel
    if (c == 0 && a.q_out)
      for (int i = tid; i < P; i += NT) a.qrot[slot * P + i] = qs[(i / D) * QSTR + i % D];
  }
}

// A sequence of a batch whose window leaves no cache row attended, in a
// launch that appends nothing (a layer reading another layer's KV,
// forward.h:578-585): its q rows are still normed and rotated in place, as
// forward.h:554-558 does before every attention call, and its o is 0
// (attn.h:162 with no rows).  The whole workgroup takes this path; nothing
// else is in flight, so plain workgroup barriers are free here.  Same
// arithmetic as rope_append_kernel: (x * 1/sqrt(mean(x^2) + eps)) * w, then
// the NEOX rotation by the fp32 angle pos * inv_freq[j] (sine and cosine in
// double, rounded).
template <int NT>
__device__ void empty_range_q(const AttnArgs& a, int64_t qrow0, int gh, int dh, int pos,
                              float* sh) {
  const int tid = threadIdx.x, half = dh / 2;
  const bool rot = a.inv_freq != nullptr;
  for (int g = 0; g < gh; ++g) {
    const float* x = a.q + (qrow0 + g) * dh;
    float* y = a.q_out + (qrow0 + g) * dh;
    float inv = 1.f;
    if (a.q_norm) {  // uniform
      float ss = 0.f;
      for (int j = tid; j < dh; j += NT) ss = fmaf(x[j], x[j], ss);
      inv = 1.0f / sqrtf(block_sum(ss, sh) / (float)dh + a.eps);
    }
    for (int j = tid; j < half; j += NT) {
      float x0 = x[j], x1 = x[j + half];
      if (a.q_norm) {
        x0 = x0 * inv * a.q_norm[j];
        x1 = x1 * inv * a.q_norm[j + half];
      }
      if (rot) {
        const float ang = (float)pos * a.inv_freq[j];
        double sd, cd;
        sincos((double)ang, &sd, &cd);
        const float c = (float)cd, sn = (float)sd;
        y[j] = x0 * c - x1 * sn;
        y[j + half] = x0 * sn + x1 * c;
      } else {
        y[j] = x0;
        y[j + half] = x1;
      }
    }
  }
}

// SC: scored launches (AttnArgs::scored).
template <int D, int GH, typename T, bool PAGED, bool ROPE, bool PAD, typename C, bool SC>
__global__ __launch_bounds__(C::NT) void attn_kernel(AttnArgs a) {
  using V16 = typename KVT<T>::vec;
  constexpr int VW = C::VW, LPR = C::LPR, NV = C::NV, EPL = C::EPL, RPS = C::RPS;
  constexpr int LPR2 = C::LPR2, RPI = C::RPI, RB = C::RB, KS = C::KS, VS = C::VS;
  constexpr int NV2 = C::NV2, AW = C::AW;
  constexpr int NW = C::NW, NT = C::NT, P = C::P;

  extern __shared__ float smem[];
  const Lds L(D, GH, NW, RB, a.chunk, a.page_shift, PAGED, a.mrg);
  float* qs = smem + L.qs;
  float* knew = smem + L.knew;
  float* vnew = smem + L.vnew;
  int* misc = reinterpret_cast<int*>(smem + L.misc);

  // PAD: heads of DH < D elements, run as D with q zero-padded (load_pad)
  const int DH = PAD ? a.dh : D;
  // Q8 (D = 256; the matrix-core kernel takes 64 and 128): 16 codes per
  // 16-byte load, an fp32 scale per K and V row, applied to the row's score
  // and to its probability in PV
  constexpr bool Q8 = sizeof(T) == 1;
  const int G = a.nq / a.nkv;
  const int nsub = G / GH;
  // chunk slot z (chunk c = nch - 1 - z, below), (KV head, subgroup) index
  // hs and sequence b of this workgroup; X (KV head, subgroup) pairs per
  // sequence
  const int X = a.nkv * nsub;
  int z = blockIdx.z, hs = blockIdx.x, b = blockIdx.y;
  if (a.xmap) {  // slot id % 8 runs on XCD id % 8 (launch_pair); padding ids exit
    const int s8 = (int)(blockIdx.x & 7);
    if (s8 >= a.slots) return;
    z = (int)(blockIdx.x >> 3);
    hs = s8 % X;
    b = s8 / X;
  } else if (a.chunk_fast) {  // Q8: a chunk's heads on one XCD, as attn_mfma_kernel
    const int k = (int)(blockIdx.x >> 3);
    const int pi = (k / X) * 8 + (int)(blockIdx.x & 7);  // padded ids (z >= nchunks) exit below
    z = pi / a.nseq;
    b = pi - z * a.nseq;
    hs = k % X;
  }
  const int sub = hs % nsub;
  const int h = hs / nsub;
  const int hq0 = h * G + sub * GH;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);  // wave-uniform

  int n = a.n, t0 = a.t0, pos = a.pos;
  // per-sequence ranges in contiguous chunks: a paged batch, or prefill rows
  bool perseq = PAGED;
  if constexpr (!ROPE) perseq = PAGED || a.pf;  // uniform
  if (perseq) {
    if (!ROPE && a.pf) {
      pos = a.pos + b;
      n = min(pos + 1, a.n);
      if constexpr (SC) {
        if (a.key_hi) n = max(0, min(a.key_hi[b], a.n));
      }
    } else {
      n = a.seq_lens[b];
      pos = a.pos_arr ? a.pos_arr[b] : n - 1;
    }
    t0 = (a.window > 0 && pos - a.window + 1 > 0) ? pos - a.window + 1 : 0;
    if constexpr (SC && !ROPE) {
      if (a.pf && a.key_lo) t0 = max(t0, a.key_lo[b]);
    }
    if (t0 > n) t0 = n;
  }
  // Chunks tile the cache rows [t0, cend); a fused step's new token (slot
  // n-1) is not read from the cache but folded into the last chunk.
  const bool fold = ROPE && a.fold;  // this launch appends and folds in the new token
  const int cend = fold ? n - 1 : n;
  int nch = a.nchunks;
  if (perseq) {
    const int span = cend - t0;
    nch = span > 0 ? (span + a.chunk - 1) / a.chunk : (fold ? 1 : 0);
    if (nch > a.nchunks) nch = a.nchunks;
  }
  if (z >= nch) {  // whole workgroup: chunk past this sequence's end (never arrives)
    if (z == 0) {  // empty attended range: o = 0 (include/molot/attn.h:162 with no rows)
      for (int i = tid; i < GH * DH; i += NT) a.o[((int64_t)b * a.nq + hq0) * DH + i] = 0.f;
      if (ROPE && !fold && a.q_out)  // nothing appended: q still leaves normed and rotated
        empty_range_q<NT>(a, (int64_t)b * a.nq + hq0, GH, DH, pos, smem);
    }
    return;
  }
  // Chunks in reverse: the last one, which holds the new token (and with it
  // the append, the fold and any norms of k and v), is dispatched first.
  const int c = nch - 1 - z;
  const int tb = t0 + c * a.chunk;
  const int cntg = max(0, min(a.chunk, cend - tb));  // rows read from the cache
  const bool is_new = fold && c == nch - 1;          // this chunk folds in the new token
  const bool split = nch > 1;
  const int64_t slot = (int64_t)b * X + hs;

  const T* __restrict__ Kb = reinterpret_cast<const T*>(a.k);
  const T* __restrict__ Vb = reinterpret_cast<const T*>(a.v);
  const int64_t hoff = (int64_t)h * a.head_stride;
  const int64_t qrow0 = (int64_t)b * a.nq + hq0;

  // ---- 1. prologue ----
  if constexpr (PAGED) {
    int32_t* sblk_w = reinterpret_cast<int32_t*>(smem + L.blk);
    // the chunk's pages (at least the one holding row tb, which exists:
    // tb <= n-1, so the clamped loads of an empty chunk stay in bounds)
    const int p0 = tb >> a.page_shift;
    const int p1 = max(p0, (tb + cntg - 1) >> a.page_shift);
    for (int i = tid; i <= p1 - p0; i += NT)
      sblk_w[i] = a.block_table[(int64_t)b * a.max_blocks + p0 + i];
    lds_barrier();
  }
  const int32_t* sblk = reinterpret_cast<const int32_t*>(smem + L.blk);
  auto row_ptr = [&](const T* base, int t) -> const T* {
    if constexpr (PAGED) {
      const int pg = (t >> a.page_shift) - (tb >> a.page_shift);
      return base + (int64_t)sblk[pg] * a.block_stride + hoff +
             (int64_t)(t & ((1 << a.page_shift) - 1)) * a.tok_stride;
    } else {
      return base + (int64_t)t * a.tok_stride + hoff;
    }
  };
  // Q8: the fp32 scale of row t of head h
  auto sc_ptr = [&](const T* base, int t) -> const float* {
    const char* p = reinterpret_cast<const char*>(base) + a.sc_off + h * a.sc_head;
    if constexpr (PAGED) {
      const int pg = (t >> a.page_shift) - (tb >> a.page_shift);
      return reinterpret_cast<const float*>(p + (int64_t)sblk[pg] * a.block_stride) +
             (t & ((1 << a.page_shift) - 1));
    } else {
      return reinterpret_cast<const float*>(p + (int64_t)t * a.tok_stride);
    }
  };
  const int s = lane % LPR;    // scores: lane within a K row group
  const int rr = lane / LPR;   // scores: row of the group within a K step
  const int cs = lane % LPR2;  // PV: columns cs*VW .. cs*VW+VW-1
  const int rs = lane / LPR2;  // PV: row within a V step
  V16 kA[KS][NV], vA[VS][NV2], kB[KS][NV], vB[VS][NV2];
  float ksA[KS], vsA[VS], ksB[KS], vsB[VS];  // Q8 row scales (unused otherwise)
  // Every wave issues the same sequence of global loads on every path: the
  // compiler counts outstanding loads per path and, where paths merge with
  // different counts, waits for all of them.  Rows past the end (a partial
  // block, or a block past the last) load the last row instead (the first
  // of an empty range): no branch around the loads, no extra HBM traffic
  // (lines of a row already read), and a probability of e^-inf = 0 where
  // they are scored at all.
  // Row mapping.  Paged: the chunk's rows [tb, tb + cntg), in order.  A
  // contiguous cache: the chunk's local row lr lies in its (lr/32)-th 32-row
  // group, the range's group c + (lr/32)*nch (groups dealt round robin, so
  // the launch's workgroups read neighbouring rows at any moment; blocks of
  // RB rows never straddle a group).
  static_assert(32 % RB == 0, "blocks within 32-row groups");
  const int rlim = perseq ? cntg : cend - t0;  // rows of the chunk / of the whole range
  const int rfirst = perseq ? tb : t0;
  const int rmax = max(rlim - 1, 0);
  auto gmap = [&](int lr) -> int {  // local row -> row from rfirst
    return perseq ? lr : (c + (lr >> 5) * nch) * 32 + (lr & 31);
  };
  // Local rows of this chunk: its valid rows come first, so every block
  // below nblk starts with a valid row (a block of no valid rows would meet
  // m_run = -inf with a -inf score: e^(-inf - -inf) is NaN).  The chunk
  // holding the range's last group counts only that group's valid rows.
  int nrows = cntg;
  if (!perseq) {
    const int groups = (rlim + 31) / 32;
    nrows = 0;
    if (c < groups) {
      const int last = (groups - 1 - c) / nch;  // local index of the chunk's last group
      nrows = 32 * last + min(32, rlim - 32 * (c + last * nch));
    }
  }
  auto load_block = [&](V16 (&kr)[KS][NV], V16 (&vr)[VS][NV2], float (&ksr)[KS], float (&vsr)[VS],
                        int rbase) {
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int t = rfirst + min(gmap(rbase + k * RPS + rr), rmax);
      const T* p = row_ptr(Kb, t);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if constexpr (PAD)
          kr[k][v] = load_pad(p, (v * LPR + s) * VW, DH);
        else
          kr[k][v] = load16(p + (v * LPR + s) * VW);
      }
      if constexpr (Q8) ksr[k] = *sc_ptr(Kb, t);
    }
#pragma unroll
    for (int k = 0; k < VS; ++k) {
      const int t = rfirst + min(gmap(rbase + k * RPI + rs), rmax);
      const T* p = row_ptr(Vb, t);
#pragma unroll
      for (int v2 = 0; v2 < NV2; ++v2) {
        if constexpr (PAD)
          vr[k][v2] = load_pad(p, (v2 * LPR2 + cs) * VW, DH);
        else
          vr[k][v2] = load16(p + (v2 * LPR2 + cs) * VW);
      }
      if constexpr (Q8) vsr[k] = *sc_ptr(Vb, t);
    }
  };
  const int nblk = (nrows + RB - 1) / RB;
  // First row of a wave's block.  SC: the claimed ones from the chunk's newest on, since a
  // bias by distance raises the scores towards them: the running max then settles with
  // the first instead of moving, and every sum with it, a block at a time.  (The blocks
  // before the claims stay in order: their loads wait for no count.)  us a step, 29
  // paged sequences of 49 to 1946 rows, slopes: 32q/8kv/d128 fp32 63.5 -> 60.0, 8q/4kv/d256
  // Q8 41.0 -> 37.4; 16385 fp32 rows 27.3 -> 27.0.
  auto block_row = [&](int blk) -> int {
    constexpr int kFixed = C::NBUF * NW;
    return (SC && blk >= kFixed ? kFixed + nblk - 1 - blk : blk) * RB;
  };
  // The prologue's own global loads go first: loads retire in order, so
  // waiting for them does not also wait for the K/V blocks issued next.
  constexpr int QV = GH * D / 4;  // float4s of q of the group
  constexpr int QPT = (QV + NT - 1) / NT;
  // the fresh k and v rows: KPT elements a thread (two at d = 512 on 4 waves)
  constexpr int KPT = (D + NT - 1) / NT;
  static_assert(D / 2 <= NT, "one thread per rotation pair in the prologue");
  // a q row wider than a wave (d = 512): its norm sums through LDS (psum)
  constexpr bool QWIDE = D / 4 > 64;
  f32x4 qv[QPT];
  // A padded launch reads the q rows (and the q norm weights) at their
  // stored length DH, in two-element pieces, each selected to 0 past DH:
  // q's zero padding to D.
  auto row_quad = [&](const float* base, int i, int64_t stride) -> f32x4 {
    if constexpr (!PAD) {
      return reinterpret_cast<const f32x4*>(base)[i];
    } else {
      const int g = i / (D / 4), j = 4 * (i - g * (D / 4));
      const float* r = base + g * stride;
      const float2 lo = *reinterpret_cast<const float2*>(r + (j < DH ? j : 0));
      const float2 hi = *reinterpret_cast<const float2*>(r + (j + 2 < DH ? j + 2 : 0));
      return f32x4{j < DH ? lo.x : 0.f, j < DH ? lo.y : 0.f, j + 2 < DH ? hi.x : 0.f,
                   j + 2 < DH ? hi.y : 0.f};
    }
  };
#pragma unroll
  for (int u = 0; u < QPT; ++u) qv[u] = row_quad(a.q + qrow0 * DH, min(tid + u * NT, QV - 1), DH);
  float invf = 0.f, knv[KPT], vnv[KPT], kwv[KPT];
#pragma unroll
  for (int u = 0; u < KPT; ++u) knv[u] = vnv[u] = kwv[u] = 0.f;
  f32x4 qwt[QPT];  // q norm weights of this thread's q elements
  if constexpr (ROPE) {
    // every path issues these loads: a layer without RoPE (inv_freq NULL)
    // or without an append reads q in their place (nq >= nkv rows), unused
    const float* ivp = a.inv_freq ? a.inv_freq : a.q;
    const float* knp = fold ? a.k_new : a.q;
    const float* vnp = fold ? a.v_new : a.q;
    invf = ivp[min(tid, DH / 2 - 1)];
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const int j = tid + u * NT;
      knv[u] = knp[((int64_t)b * a.nkv + h) * DH + min(j, DH - 1)];
      vnv[u] = vnp[((int64_t)b * a.nkv + h) * DH + min(j, DH - 1)];
      if (j >= DH) knv[u] = vnv[u] = 0.f;  // the padding of the new k and v rows
    }
    if (a.q_norm) {
#pragma unroll
      for (int u = 0; u < QPT; ++u)
        qwt[u] = row_quad(a.q_norm, min(tid + u * NT, QV - 1) % (D / 4), 0);
    }
    if (is_new && a.k_norm) {
#pragma unroll
      for (int u = 0; u < KPT; ++u) kwv[u] = a.k_norm[min(tid + u * NT, DH - 1)];
    }
  }
  float vq[kVnPT];
  const bool vn = ROPE && is_new && a.v_norm;  // uniform over the workgroup
  if (vn) v_norm_load<D, NT>(a, b, tid, vq, DH);
  // each wave's first NBUF blocks: w (and w + NW); the rest are claimed
  int bA = w, bB = w + NW;
  load_block(kA, vA, ksA, vsA, block_row(bA));
  if constexpr (C::NBUF == 2) load_block(kB, vB, ksB, vsB, block_row(bB));
  if (tid == 0) {
    misc[0] = C::NBUF * NW;  // next block to claim
  }
  if constexpr (ROPE) {
    if (a.q_norm) {
      if constexpr (!QWIDE) {
        q_norm_regs<D, QPT>(a, qv, qwt, DH);
      } else {
        // 64 consecutive quads (one wave's share of a u) lie in one row:
        // their sum of squares to psum[row][part]; the weights to qw.  The
        // rotation pass below applies the norm.
#pragma unroll
        for (int u = 0; u < QPT; ++u) {
          const int i = tid + u * NT;
          if (i < QV) {  // uniform over the wave: QV is a multiple of 64
            float ss = qv[u][0] * qv[u][0];
            ss = fmaf(qv[u][1], qv[u][1], ss);
            ss = fmaf(qv[u][2], qv[u][2], ss);
            ss = fmaf(qv[u][3], qv[u][3], ss);
            ss = group_sum<64>(ss);
            if (lane == 0) smem[L.psum + i / 64] = ss;
            if (i < D / 4) reinterpret_cast<f32x4*>(smem + L.qw)[i] = qwt[u];
          }
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < QPT; ++u) {
    const int i = tid + u * NT;
    if (i < QV) reinterpret_cast<f32x4*>(qs)[i] = qv[u];
  }
  if constexpr (ROPE) {
    float* csn = smem + L.cs;
    float* sn = smem + L.sn;
    const bool rot = a.inv_freq != nullptr;  // uniform: no RoPE on a NoPE layer
    if (rot && tid < DH / 2) {
      const float ang = (float)pos * invf;
      double sd, cd;
      sincos((double)ang, &sd, &cd);
      csn[tid] = (float)cd;
      sn[tid] = (float)sd;
    }
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const int j = tid + u * NT;
      if (j < D) {
        if (is_new) {
          knew[j] = knv[u];
          vnew[j] = vnv[u];
        }
        smem[L.nw + j] = kwv[u];
      }
    }
    if (vn) v_norm_share<D, NT>(a, b, tid, w, lane, vq, smem + L.wl, DH);
    if (is_new && a.k_norm) {
      float ss = 0.f;
#pragma unroll
      for (int u = 0; u < KPT; ++u) ss = fmaf(knv[u], knv[u], ss);  // 0 past D
      k_norm_share(w, lane, ss, smem + L.wm);
    }
    lds_barrier();
    // NEOX pairs (j, j + DH/2) of the stored head (attn.h:17-28); a q row
    // wider than a wave takes its norm here: (x * inv) * w, as q_norm_regs
    const int half = DH / 2;
    const bool qwn = QWIDE && a.q_norm;
    for (int i = tid; (rot || qwn) && i < GH * half; i += NT) {
      const int g = i / half, j = i - g * half;
      float x0 = qs[g * D + j], x1 = qs[g * D + j + half];
      if (qwn) {
        float ss = 0.f;
#pragma unroll
        for (int pt = 0; pt < D / 256; ++pt) ss += smem[L.psum + g * (D / 256) + pt];
        const float inv = 1.0f / sqrtf(ss / (float)DH + a.eps);
        x0 = x0 * inv * smem[L.qw + j];
        x1 = x1 * inv * smem[L.qw + j + half];
      }
      qs[g * D + j] = rot ? x0 * csn[j] - x1 * sn[j] : x0;
      qs[g * D + j + half] = rot ? x0 * sn[j] + x1 * csn[j] : x1;
    }
    if (is_new) {
      // the appended row as the cache will hold it: normed (as configured),
      // rotated k, k and v rounded to the cache type (stored into the cache
      // after the stream)
      const NewNorms nn = new_norms<D, NW>(a, smem + L.wm, smem + L.wl, DH);
      for (int j = tid; j < half; j += NT) {
        float k0 = knew[j], k1 = knew[j + half];
        float v0 = vnew[j], v1 = vnew[j + half];
        nn.apply(a, smem + L.nw, j, half, k0, k1, v0, v1);
        float r0 = rot ? k0 * csn[j] - k1 * sn[j] : k0;
        float r1 = rot ? k0 * sn[j] + k1 * csn[j] : k1;
        if constexpr (sizeof(T) == 2) {
          r0 = __uint_as_float((uint32_t)f32_to_bf16(r0) << 16);
          r1 = __uint_as_float((uint32_t)f32_to_bf16(r1) << 16);
          v0 = __uint_as_float((uint32_t)f32_to_bf16(v0) << 16);
          v1 = __uint_as_float((uint32_t)f32_to_bf16(v1) << 16);
        }
        knew[j] = r0;
        knew[j + half] = r1;
        vnew[j] = v0;
        vnew[j + half] = v1;
      }
    }
  }
  lds_barrier();

  // q registers: lane s of a K row group holds elements (v*LPR + s)*VW + e
  float qr[GH][EPL];
  // Base-2 scores: the dot products are scaled by scale*log2(e) as a whole
  // (one rounding per score, as the natural-units scale), not through a
  // pre-scaled q, whose per-element rounding perturbs q itself: with q
  // channels 1000x the rest that was 1.7e-5 normwise off float64, outside
  // the 1e-5 bar the score-scaled form meets.
  const float qsc = a.scale * kLog2e;
#pragma unroll
  for (int g = 0; g < GH; ++g)
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e4 = 0; e4 < VW; e4 += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(qs + g * D + (v * LPR + s) * VW + e4);
        qr[g][v * VW + e4 + 0] = x[0];
        qr[g][v * VW + e4 + 1] = x[1];
        qr[g][v * VW + e4 + 2] = x[2];
        qr[g][v * VW + e4 + 3] = x[3];
      }

  // SC: the cap and the heads' slopes in base-2 units, and this (sequence, KV
  // head)'s scores (row t at (t - t0) * G)
  static_assert(!SC || (LPR >= GH && LPR % GH == 0), "a lane of a row for every head");
  [[maybe_unused]] float slope = 0.f, cap2 = 0.f, rcap = 0.f;  // of head s % GH
  [[maybe_unused]] float m_own = -INFINITY;                    // and its running max
  [[maybe_unused]] __amdgpu_buffer_rsrc_t swr;
  if constexpr (SC) {
    if (a.slopes) slope = a.slopes[hq0 + s % GH] * kLog2e;
    cap2 = a.softcap * kLog2e;
    rcap = a.softcap > 0.f ? 1.f / cap2 : 0.f;
    swr = score_rsrc(a, b, h);
  }

  // ---- 2. streaming blocks with a per-wave online softmax ----
  float* pw = smem + L.pw + w * RB * GH;
  float m_run[GH], l_run[GH], acc[GH][AW];
#pragma unroll
  for (int g = 0; g < GH; ++g) {
    m_run[g] = -INFINITY;
    l_run[g] = 0.f;
#pragma unroll
    for (int e = 0; e < AW; ++e) acc[g][e] = 0.f;
  }
  int next_fixed = w + C::NBUF * NW;  // fixed order: wave w takes blocks w, w+NW, w+2NW, ...
  auto claim = [&]() -> int {
    if (!a.dynamic) {
      const int v = next_fixed;
      next_fixed += NW;
      return v;
    }
    int v = 0;
    if (lane == 0) v = atomicAdd(&misc[0], 1);
    return __builtin_amdgcn_readfirstlane(v);
  };
  auto consume = [&](const V16 (&kr)[KS][NV], const V16 (&vr)[VS][NV2], const float (&ksr)[KS],
                     const float (&vsr)[VS], int rbase) {
    // scores of this lane group's rows
    float sc[KS][GH];
    float bmax[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) bmax[g] = -INFINITY;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      float d[GH];
#pragma unroll
      for (int g = 0; g < GH; ++g) d[g] = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float x[VW];
        KVT<T>::unpack(kr[k][v], x);
#pragma unroll
        for (int e = 0; e < VW; ++e)
#pragma unroll
          for (int g = 0; g < GH; ++g) d[g] = fmaf(qr[g][v * VW + e], x[e], d[g]);
      }
      const bool valid = rbase + k * RPS + rr < nrows;
#pragma unroll
      for (int g = 0; g < GH; ++g) {
        const float t = group_sum<LPR>(d[g]) * (Q8 ? qsc * ksr[k] : qsc);
        if constexpr (SC) {
          sc[k][g] = t;
        } else {
          sc[k][g] = valid ? t : -INFINITY;
          bmax[g] = fmaxf(bmax[g], sc[k][g]);
        }
      }
    }
    if constexpr (SC) {
      // Every lane of a row holds the row's GH sums; from here on lane s takes head
      // s % GH alone: one cap, bias, comparison and exponential a row instead of GH
      // (32q/8kv/d128 fp32, 16385 rows, cap and slopes: 30.0 -> 27.2 us, the plain step 25.9).
      const int g0 = s % GH;
      float x[KS];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        x[k] = sc[k][0];
#pragma unroll
        for (int g = 1; g < GH; ++g) x[k] = g0 == g ? sc[k][g] : x[k];
      }
      if (a.softcap > 0.f) cap_scores<KS>(x, cap2, rcap);
      // rows of a block follow each other in the cache (blocks lie within 32-row groups)
      const int t_lane = rfirst + gmap(rbase) + rr;
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const float y = fmaf(-slope, fabsf((float)(pos - t_lane - k * RPS)), x[k]);
        x[k] = rbase + k * RPS + rr < nrows ? y : -INFINITY;
        top = fmaxf(top, x[k]);
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int at = t_lane + k * RPS - t0;
        const bool mine = s < GH && rbase + k * RPS + rr < nrows;
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[k]), swr,
                                              mine ? 4 * (at * G + sub * GH + s) : -1, 0, 0);
      }
      if (__builtin_amdgcn_ballot_w64(top > m_own + kLazyMax) != 0) {  // wave-uniform
        auto top_off = [&](auto OFFC) {
          constexpr int off = decltype(OFFC)::value;
          if constexpr (off >= LPR) top = max_xor<off>(top);
        };
        top_off(std::integral_constant<int, 1>{});
        top_off(std::integral_constant<int, 2>{});
        top_off(std::integral_constant<int, 4>{});
        top_off(std::integral_constant<int, 8>{});
        top_off(std::integral_constant<int, 16>{});
        top_off(std::integral_constant<int, 32>{});
        const float mn = fmaxf(m_own, top);
        const float alpha = exp2_hw(m_own - mn);  // m_own = -inf -> 0
        m_own = mn;
#pragma unroll
        for (int g = 0; g < GH; ++g) {
          const float al = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(alpha), g));
          l_run[g] *= al;
#pragma unroll
          for (int e = 0; e < AW; ++e) acc[g][e] *= al;
        }
      }
      if (s < GH) {
#pragma unroll
        for (int k = 0; k < KS; ++k) pw[(k * RPS + rr) * GH + s] = exp2_hw(x[k] - m_own);
      }
    } else {
    // The running max moves only when a score passes it by more than
    // kLazyMax (p <= 2^8 otherwise; o and l always share the max they were
    // formed with): most blocks skip the block max across the wave's row
    // groups and the rescale.
    bool grow = false;
#pragma unroll
    for (int g = 0; g < GH; ++g) grow |= bmax[g] > m_run[g] + kLazyMax;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {  // wave-uniform
#pragma unroll
      for (int g = 0; g < GH; ++g) {
        auto bmax_off = [&](auto OFFC) {
          constexpr int off = decltype(OFFC)::value;
          if constexpr (off >= LPR) bmax[g] = max_xor<off>(bmax[g]);
        };
        bmax_off(std::integral_constant<int, 1>{});
        bmax_off(std::integral_constant<int, 2>{});
        bmax_off(std::integral_constant<int, 4>{});
        bmax_off(std::integral_constant<int, 8>{});
        bmax_off(std::integral_constant<int, 16>{});
        bmax_off(std::integral_constant<int, 32>{});
        const float mn = fmaxf(m_run[g], bmax[g]);
        const float alpha = exp2_hw(m_run[g] - mn);  // m_run = -inf -> 0
        m_run[g] = mn;
        l_run[g] *= alpha;
#pragma unroll
        for (int e = 0; e < AW; ++e) acc[g][e] *= alpha;
      }
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if (s == 0) {
#pragma unroll
        for (int g = 0; g < GH; ++g) pw[(k * RPS + rr) * GH + g] = exp2_hw(sc[k][g] - m_run[g]);
      }
    }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < VS; ++k) {
      float x[AW];
#pragma unroll
      for (int v2 = 0; v2 < NV2; ++v2) KVT<T>::unpack(vr[k][v2], x + v2 * VW);
      float p[GH];
#pragma unroll
      for (int g = 0; g < GH; ++g) p[g] = pw[(k * RPI + rs) * GH + g];
#pragma unroll
      for (int g = 0; g < GH; ++g) {
        l_run[g] += p[g];
        const float pv = Q8 ? p[g] * vsr[k] : p[g];  // Q8: codes times the V row's scale
#pragma unroll
        for (int e = 0; e < AW; ++e) acc[g][e] = fmaf(pv, x[e], acc[g][e]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  };
  // Two buffers, A and B, alternate: a block's successor is claimed before
  // the block is consumed and loaded right after, so one block is always in
  // flight while the other is scored.  On the path that continues, every
  // load is unconditional (the exits drain the other buffer), so the
  // compiler waits only for the buffer about to be consumed.  Claims are
  // monotone: once a claim is past the end, every later one is too.
  // The explicit waits state what the compiler cannot always derive at the
  // rotated loop's header: the older buffer is complete while the younger
  // buffer's LB loads stay in flight.
  constexpr int LB = KS * NV + VS;  // loads per block
  if constexpr (C::NBUF == 1) {
    // one block in flight: score it, claim and load the next
    while (bA < nblk) {
      const int nx = claim();
      consume(kA, vA, ksA, vsA, block_row(bA));
      bA = nx;
      if (bA < nblk) load_block(kA, vA, ksA, vsA, block_row(bA));
    }
  } else if (bA < nblk) {
    if (bB >= nblk) {
      consume(kA, vA, ksA, vsA, block_row(bA));
    } else {
      for (;;) {
        int nx = claim();
        wait_vmcnt<LB>();
        consume(kA, vA, ksA, vsA, block_row(bA));
        if (nx >= nblk) {
          consume(kB, vB, ksB, vsB, block_row(bB));
          break;
        }
        bA = nx;
        load_block(kA, vA, ksA, vsA, block_row(bA));
        nx = claim();
        wait_vmcnt<LB>();
        consume(kB, vB, ksB, vsB, block_row(bB));
        if (nx >= nblk) {
          consume(kA, vA, ksA, vsA, block_row(bA));
          break;
        }
        bB = nx;
        load_block(kB, vB, ksB, vsB, block_row(bB));
      }
    }
  }

  if constexpr (SC) {
#pragma unroll
    for (int g = 0; g < GH; ++g)
      m_run[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(m_own), g));
  }

  // ---- 3. the new token, folded in by wave 0 from LDS (its append to the
  // cache comes last, below) ----
  // Q8: wave 0 quantizes the k and v rows as the cache will hold them (the
  // reference quantizer, quant.h:34-50: s = absmax / 127, codes round(x/s))
  // and leaves code * s in LDS for the fold
  [[maybe_unused]] int kcode[Q8 ? D / 64 : 1], vcode[Q8 ? D / 64 : 1];
  [[maybe_unused]] float kscale = 0.f, vscale = 0.f;
  if constexpr (Q8) {
    if (is_new && w == 0) {
      constexpr int EPL = D / 64;
      float kx[EPL], vx[EPL];
      float ka = 0.f, va = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        kx[e] = knew[lane + 64 * e];
        vx[e] = vnew[lane + 64 * e];
        ka = fmaxf(ka, fabsf(kx[e]));
        va = fmaxf(va, fabsf(vx[e]));
      }
      kscale = q8_scale(group_max<64>(ka));
      vscale = q8_scale(group_max<64>(va));
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        kcode[e] = q8_code(kx[e], kscale);
        vcode[e] = q8_code(vx[e], vscale);
        knew[lane + 64 * e] = (float)kcode[e] * kscale;
        vnew[lane + 64 * e] = (float)vcode[e] * vscale;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the fold reads other lanes' rows
    }
  }
  if (is_new && w == 0) {
    // LDS reads first, unconditional and vector-wide: the lanes of PV row 0
    // add the row's values, the others add 0 (a select per element, not a
    // branch around each read)
    const float one = rs == 0 ? 1.f : 0.f;
    float vx[AW];
#pragma unroll
    for (int v2 = 0; v2 < NV2; ++v2)
#pragma unroll
      for (int e4 = 0; e4 < VW; e4 += 4) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(vnew + (v2 * LPR2 + cs) * VW + e4);
#pragma unroll
        for (int e = 0; e < 4; ++e) vx[v2 * VW + e4 + e] = t[e] * one;
      }
    float part[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      part[g] = 0.f;
#pragma unroll
      for (int j = lane; j < D; j += 64) part[g] = fmaf(qs[g * D + j], knew[j], part[g]);
    }
    if constexpr (SC) {  // (every lane: its part is then the whole score)
#pragma unroll
      for (int g = 0; g < GH; ++g) part[g] = wave_reduce<false>(part[g]) * qsc;
      if (a.softcap > 0.f) cap_scores<GH>(part, cap2, rcap);
      const float dist = fabsf((float)(pos - (n - 1)));
#pragma unroll
      for (int g = 0; g < GH; ++g) {
        const float sl = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(slope), g));
        part[g] = fmaf(-sl, dist, part[g]);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(part[g]), swr,
                                              lane == 0 ? 4 * ((n - 1 - t0) * G + sub * GH + g) : -1, 0, 0);
      }
    }
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      const float snew = SC ? part[g] : wave_reduce<false>(part[g]) * qsc;
      const float mn = fmaxf(m_run[g], snew);
      const float alpha = exp2_hw(m_run[g] - mn);
      const float p = exp2_hw(snew - mn);
      m_run[g] = mn;
      l_run[g] = l_run[g] * alpha + p * one;
#pragma unroll
      for (int e = 0; e < AW; ++e) acc[g][e] = acc[g][e] * alpha + p * vx[e];
    }
  }

  // ---- 4. merge the waves ----
  // lanes LPR2 apart hold the same columns of other rows: sum them, in
  // ascending offsets
  auto merge_off = [&](auto OFFC) {
    constexpr int off = decltype(OFFC)::value;
    if constexpr (off >= LPR2) {
#pragma unroll
      for (int g = 0; g < GH; ++g) {
        l_run[g] = sum_xor<off>(l_run[g]);
#pragma unroll
        for (int e = 0; e < AW; ++e) acc[g][e] = sum_xor<off>(acc[g][e]);
      }
    }
  };
  merge_off(std::integral_constant<int, 1>{});
  merge_off(std::integral_constant<int, 2>{});
  merge_off(std::integral_constant<int, 4>{});
  merge_off(std::integral_constant<int, 8>{});
  merge_off(std::integral_constant<int, 16>{});
  merge_off(std::integral_constant<int, 32>{});
  float* wm = smem + L.wm;
  float* wl = smem + L.wl;
  float* red = smem + L.red;
  if (lane == 0) {
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      wm[w * GH + g] = SC ? m_run[g] : m_run[g] * kLn2;  // natural units for the merges
      wl[w * GH + g] = l_run[g];
    }
  }
  if (rs == 0) {
#pragma unroll
    for (int g = 0; g < GH; ++g)
#pragma unroll
      for (int v2 = 0; v2 < NV2; ++v2)
#pragma unroll
        for (int e = 0; e < VW; ++e)
          red[(w * GH + g) * D + (v2 * LPR2 + cs) * VW + e] = acc[g][v2 * VW + e];
  }
  lds_barrier();
  finish_chunk<D, GH, NW, NT, ROPE, NW * P, false, D, SC>(a, wm, wl, red, P, qs, tid, lane, split, slot, c,
                                             qrow0, nch,
                                    smem + L.mrg, red, misc + 1, DH);

  // ---- 6. the append (subgroup 0; no workgroup reads that slot in this
  // launch).  Last, because nothing may wait for these stores: vmcnt counts
  // stores too, and a wait placed after them for an older load would hold
  // the fold and the merge until the stores complete. ----
  if (is_new && sub == 0 && (Q8 ? w == 0 : tid < DH)) {  // (d = 512: tid, tid + NT)
    const int slot_row = n - 1;
    int64_t off, soff;  // element (Q8: byte) offset of the row; Q8: of its scale
    if constexpr (PAGED) {
      const int64_t blk = a.block_table[(int64_t)b * a.max_blocks + (slot_row >> a.page_shift)];
      const int sl = slot_row & ((1 << a.page_shift) - 1);
      off = blk * a.block_stride + hoff + (int64_t)sl * a.tok_stride;
      soff = blk * a.block_stride + a.sc_off + h * a.sc_head + 4 * sl;
    } else {
      off = (int64_t)slot_row * a.tok_stride + hoff;
      soff = (int64_t)slot_row * a.tok_stride + a.sc_off + h * a.sc_head;
    }
    if constexpr (Q8) {
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        if (lane + 64 * e >= DH) continue;  // a padded row ends at DH codes
        reinterpret_cast<int8_t*>(a.k)[off + lane + 64 * e] = (int8_t)kcode[e];
        reinterpret_cast<int8_t*>(a.v)[off + lane + 64 * e] = (int8_t)vcode[e];
      }
      if (lane == 0) {
        *reinterpret_cast<float*>(reinterpret_cast<char*>(a.k) + soff) = kscale;
        *reinterpret_cast<float*>(reinterpret_cast<char*>(a.v) + soff) = vscale;
      }
    } else if constexpr (sizeof(T) == 2) {  // exact bf16 values: the rounding returns their bits
      for (int j = tid; j < DH; j += NT) {
        reinterpret_cast<uint16_t*>(a.k)[off + j] = f32_to_bf16(knew[j]);
        reinterpret_cast<uint16_t*>(a.v)[off + j] = f32_to_bf16(vnew[j]);
      }
    } else {
      for (int j = tid; j < DH; j += NT) {
        reinterpret_cast<float*>(a.k)[off + j] = knew[j];
        reinterpret_cast<float*>(a.v)[off + j] = vnew[j];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// bf16 KV on the matrix cores.
//
// A wave takes tiles of 32 cache rows of the workgroup's KV head (claimed
// like the blocks of attn_kernel) and keeps the GH <= 16 query heads of the
// group on the 16 columns of v_mfma_f32_16x16x32_bf16:
//   scores  S^T (32 rows x 16 heads) = K (32 x D) . Q^T (D x 16), two 16-row
//           halves, D/32 k-steps each.  K goes from HBM straight into the A
//           operand: lane l holds row l%16 and elements 8*(l/16)..+7 of a
//           32-wide k-step, one 16-byte load.  q (fp32) enters as three bf16
//           pieces hi + mid + lo, which together hold its 24-bit significand,
//           so the scores are the fp32 products of q with the bf16 K summed
//           in fp32.
//   softmax the accumulator of a half holds, in lane l, head l%16 and rows
//           4*(l/16)+r: a lane owns one head and 8 rows of the tile, and the
//           online max / rescale run in place (max across the 4 lanes of a
//           head by two shuffles).
//   PV      O^T (D x 16) += V^T (D x 32) . P^T (32 x 16) per 16-row block of
//           O^T.  The k index of this product runs over the tile's rows in
//           the order tau(g, e) = 16*(e/4) + 4g + e%4 (g = l/16): exactly the
//           8 probabilities lane l already holds, so P is the B operand as it
//           stands (again as bf16 hi + mid + lo).  V is staged in LDS
//           (row-major, 16-byte units XOR-swizzled by row: vt_off) and read
//           back with ds_read_b64_tr_b16: lane l reads 8 bytes of row l/4
//           (+16) at column 16*dt + 4*(l%4), and the transpose hands lane i of
//           each 16-lane group element i%4 of lane 4e+i/4's read as slot e,
//           i.e. V[tau(g, e)][16*dt + i]: the A operand.
// Prologue, new token and chunk output are those of attn_kernel.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Chunks of a paged batch on the matrix-core kernel, from the sequences'
// lengths (paged_plan.hpp).

// A sequence's rows and query position, and the cache rows it attends.
struct SeqLen {
  int n = 0, pos = -1;
};
__device__ __forceinline__ SeqLen seq_len(const int32_t* seq_lens, const int32_t* pos_arr, int b,
                                          int nseq) {
  SeqLen s;
  if (b < nseq) {
    s.n = seq_lens[b];
    s.pos = pos_arr ? pos_arr[b] : s.n - 1;
  }
  return s;
}
// (limit: the host's bound of the rows.  A longer sequence would take pairs
// and partials that the launch does not have.)
__device__ __forceinline__ int seq_span(SeqLen s, int window, bool fold, int limit) {
  int t0 = (window > 0 && s.pos - window + 1 > 0) ? s.pos - window + 1 : 0;
  if (t0 > s.n) t0 = s.n;
  return min(max((fold ? s.n - 1 : s.n) - t0, 0), limit);
}
// The launch's chunk (wave-uniform; every lane of the wave takes part).
// first: sequence (lane)'s, loaded by the caller.
__device__ __forceinline__ int paged_chunk(const int32_t* seq_lens, const int32_t* pos_arr,
                                           SeqLen first, int nseq, int window, bool fold,
                                           int limit, int heads, int target, bool q8) {
  const int lane = threadIdx.x & 63;
  int rows = lane < nseq ? seq_span(first, window, fold, limit) : 0;
  for (int b = lane + 64; b < nseq; b += 64)
    rows += seq_span(seq_len(seq_lens, pos_arr, b, nseq), window, fold, limit);
  rows = __builtin_amdgcn_readlane(wave_scan(rows), 63);
  return dyn_chunk(rows, nseq, heads, target, q8);
}

constexpr int kMfmaWaves = 4;                  // waves per workgroup
constexpr int kMfmaThreads = kMfmaWaves * 64;
constexpr int kTile = 32;                      // cache rows per wave step

template <int D>
constexpr int kMfmaQStride = D + 4;

// LDS of attn_mfma_kernel, in floats.  vt: per wave, 32 staged V rows of D
// bf16 (16*D floats), which after the stream hold the wave's partial o;
// sc (Q8): per wave, the K then the V row scales of its current tile.
struct LdsM {
  int qs, cs, sn, knew, vnew, nw, wm, wl, sc, vt, blk, misc, mrg, total;
  __host__ __device__ LdsM(int D, int GH, int chunk, int page_shift, bool paged, bool q8,
                           int merge) {
    int o = 0;
    qs = o; o += GH * (D + 4);  // rows kMfmaQStride<D> = D + 4 floats apart
    cs = o; o += D / 2;
    sn = o; o += D / 2;
    knew = o; o += D;
    vnew = o; o += D;
    nw = o; o += D;  // k norm weights
    wm = o; o += kMfmaWaves * GH;
    wl = o; o += kMfmaWaves * GH;
    o = (o + 3) & ~3;
    sc = o; o += q8 ? kMfmaWaves * 2 * kTile : 0;
    o = (o + 63) & ~63;  // 256-byte aligned: the swizzle's bank pattern
    vt = o; o += kMfmaWaves * kTile * D / 2;
    blk = o; o += paged ? ((chunk >> page_shift) + 2) : 0;
    misc = o; o += 8;  // tile claim counter, merge flag
    mrg = o; o += merge;  // in-launch merge: chunk statistics
    total = o;
  }
};

// Byte offset of 16-byte unit ch (elements 8ch .. 8ch+7) of staged V row r:
// unit ch of the row is stored at unit ch ^ f(r).  Measured on MI355X
// (SQ_LDS_BANK_CONFLICT of each access pattern alone), a 16-byte LDS store
// serves 8 lanes a cycle and conflicts unless their addresses fall in
// distinct 16-byte slots mod 128 bytes, and ds_read_b64_tr_b16 serves 32
// lanes a cycle, distinct 8-byte slots mod 256 bytes.  The stores put rows
// r0 .. r0+7 of one unit ch in 8 lanes: distinct when the low 3 bits of f
// run over 8 values; a transposed read takes units 2dt and 2dt+1 of 8 rows:
// 16 distinct units of a 256-byte span when f >> 1 runs over 8 values.
// D = 128 or 256 (16 or 32 units a row): f(r) = 2(r%8) + (r/4)%2 meets
// both; D = 64 (8 units, 2 rows per 256 bytes): f(r) = r%8.  The
// 32-byte-segment swizzle this replaces conflicted 2-way on every store.
template <int D>
__device__ __forceinline__ int vt_f(int r) {
  return D != 64 ? (((r & 7) << 1) | ((r >> 2) & 1)) : (r & 7);
}
template <int D>
__device__ __forceinline__ int vt_off(int r, int ch) {
  return r * (2 * D) + 16 * (ch ^ vt_f<D>(r));
}

// Byte offset of 16-byte unit ch of a staged K row (the prefill's A operand
// of the scores, read by 16-byte loads of 16 keys at one unit): unit ch of
// key r at ch ^ (r % 16) (D = 64: r % 8).  Measured, a 16-byte LDS read
// serves 16 lanes a cycle, conflict-free on 16 distinct units mod 256 bytes.
template <int D>
__device__ __forceinline__ int kt_f(int r) {
  return D == 64 ? (r & 7) : (r & 15);
}
template <int D>
__device__ __forceinline__ int kt_off(int r, int ch) {
  return r * (2 * D) + 16 * (ch ^ kt_f<D>(r));
}

// x = hi + mid + lo in bf16 (round to nearest even at each step); the three
// pieces carry the full fp32 significand.
__device__ __forceinline__ void split3(float x, __bf16& hi, __bf16& mid, __bf16& lo) {
  hi = (__bf16)x;
  float r = x - (float)hi;
  mid = (__bf16)r;
  r -= (float)mid;
  lo = (__bf16)r;
}

__device__ __forceinline__ f32x4 mfma_bf16(bf16x8_t a, bf16x8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma_f16(f16x8_t a, f16x8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 16 int8 codes -> 16 bf16 (exact: |code| <= 127), bytes 0-7 into lo, 8-15
// into hi, each in memory order.  One v_cvt_pk_bf16_f32 per pair (its
// rounding is the identity on these values).
__device__ __forceinline__ void i8x16_to_bf16(const u32x4& x, u32x4& lo, u32x4& hi) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = x[i];
    const float f0 = (float)(int8_t)(w & 0xFF), f1 = (float)(int8_t)((w >> 8) & 0xFF);
    const float f2 = (float)(int8_t)((w >> 16) & 0xFF), f3 = (float)((int32_t)w >> 24);
    u32x4& dst = i < 2 ? lo : hi;
    dst[2 * (i & 1)] = bf16_pair_exact(f0, f1);
    dst[2 * (i & 1) + 1] = bf16_pair_exact(f2, f3);
  }
}

// Matrix-core decode over a bf16 (Q8 = false) or Q8 (Q8 = true) cache.
//
// Q8: each lane reads 16 codes per 16-byte load, covering two k-steps: load
// j of lane group g holds row bytes 64j + 16g .. +15, so k-step kk, element
// e is head-dim index 64*(kk/2) + 16g + 8*(kk%2) + e, and q^T takes the same
// order.  Codes widen to bf16 exactly; a score is (codes . q) * s_k * scale,
// and the PV operand is p * s_v in the same three bf16 pieces as bf16's p
// (the row sum l takes p itself).  Lane (row l%16) loads its A-row's two
// scales; they pass through a per-wave LDS slot to the accumulator lanes of
// rows 16u + 4*(l/16) + r.  The new token's k (rotated) and v rows are
// quantized in the workgroup like the cache rows and folded in as code * s.
// SC: scored launches (AttnArgs::scored).
template <int D, int GH, bool PAGED, bool ROPE, bool Q8, bool SC>
__global__ __launch_bounds__(kMfmaThreads, 2) void attn_mfma_kernel(AttnArgs a) {
  static_assert(D == 64 || D == 128, "MFMA tiles cover D = 64 or 128");
  static_assert(GH >= 1 && GH <= 16, "the group's q heads on the 16 MFMA columns");
  constexpr int NW = kMfmaWaves, NT = kMfmaThreads;
  constexpr int KK = D / 32;  // k-steps of the score product
  constexpr int DT = D / 16;  // 16-row blocks of O^T
  constexpr int RS = kTile * D / 2;  // floats of a wave's LDS region
  constexpr int KL = Q8 ? D / 64 : KK;  // 16-byte loads per row and lane (K or V)
  using E = typename std::conditional<Q8, int8_t, bf16_t>::type;

  constexpr int DH = D;  // never padded
  constexpr int QSTR = kMfmaQStride<D>;  // floats between q rows in LDS
  extern __shared__ float smem[];
  const LdsM L(D, GH, a.chunk, a.page_shift, PAGED, Q8, a.mrg);
  float* qs = smem + L.qs;
  float* knew = smem + L.knew;
  float* vnew = smem + L.vnew;
  int* misc = reinterpret_cast<int*>(smem + L.misc);

  // chunk slot z (chunk c = nch - 1 - z, below), (KV head, subgroup) index
  // hs and sequence b of this workgroup
  const int G = a.nq / a.nkv;
  const int nsub = G / GH;
  int z, hs, b;
  int chunk = a.chunk;
  int sn = 0, spos = 0;  // dyn: the sequence's length and position
  if (PAGED && a.dyn) {
    // flat over the (sequence, chunk) pairs (at least one a sequence), the
    // sequences in order; Q8: all heads of a pair on one XCD, as below
    const int HS = a.nkv * nsub;
    const bool fold = ROPE && a.fold;
    SeqLen sl = seq_len(a.seq_lens, a.pos_arr, (int)(threadIdx.x & 63), a.nseq);
    chunk = paged_chunk(a.seq_lens, a.pos_arr, sl, a.nseq, a.window, fold,
                        a.dyn_span, HS, a.dyn, Q8);
    const int id = (int)blockIdx.x;
    int pi;
    if (Q8) {
      const int k = id >> 3;
      pi = (k / HS) * 8 + (id & 7);
      hs = k % HS;
    } else {
      pi = id / HS;
      hs = id % HS;
    }
    b = -1;
    z = 0;
    for (int b0 = 0; b0 < a.nseq; b0 += 64) {
      const int bl = b0 + (int)(threadIdx.x & 63);
      if (b0) sl = seq_len(a.seq_lens, a.pos_arr, bl, a.nseq);
      const int cnt =
          bl < a.nseq ? max(1, dyn_chunks(seq_span(sl, a.window, fold, a.dyn_span), chunk)) : 0;
      const int upto = wave_scan(cnt);
      const uint64_t past = __builtin_amdgcn_ballot_w64(upto > pi);
      if (past) {  // the first lane whose pairs reach past pi
        const int l = __builtin_ctzll(past);
        b = b0 + l;
        z = pi - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(cnt, l));
        sn = __builtin_amdgcn_readlane(sl.n, l);
        spos = __builtin_amdgcn_readlane(sl.pos, l);
        break;
      }
      pi -= __builtin_amdgcn_readlane(upto, 63);
    }
    if (b < 0) return;  // past the last pair
  } else if (a.chunk_fast) {  // workgroup id runs on XCD id % 8 (launch_pair)
    const int HS = a.nkv * nsub;
    const int k = (int)(blockIdx.x >> 3);
    // (sequence, chunk) pair pi = (k / HS) * 8 + id % 8, chunk slot slowest;
    // padded ids (z >= nchunks) exit below
    const int pi = (k / HS) * 8 + (int)(blockIdx.x & 7);
    z = pi / a.nseq;
    b = pi - z * a.nseq;
    hs = k % HS;
  } else if (a.xmap) {  // slot id % 8 runs on XCD id % 8 (launch_pair); padding ids exit
    const int s8 = (int)(blockIdx.x & 7);
    if (s8 >= a.slots) return;
    z = (int)(blockIdx.x >> 3);
    hs = s8 % (a.nkv * nsub);
    b = s8 / (a.nkv * nsub);
  } else {
    z = blockIdx.z;
    hs = blockIdx.x;
    b = blockIdx.y;
  }
  const int sub = hs % nsub;
  const int h = hs / nsub;
  const int hq0 = h * G + sub * GH;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m16 = lane & 15, g4 = lane >> 4;

  int n = a.n, t0 = a.t0, pos = a.pos;
  if constexpr (PAGED) {
    n = a.dyn ? sn : a.seq_lens[b];
    pos = a.dyn ? spos : a.pos_arr ? a.pos_arr[b] : n - 1;
    t0 = (a.window > 0 && pos - a.window + 1 > 0) ? pos - a.window + 1 : 0;
    if (t0 > n) t0 = n;
  }
  const bool fold = ROPE && a.fold;  // this launch appends and folds in the new token
  const int cend = fold ? n - 1 : n;
  int nch = a.nchunks;
  if constexpr (PAGED) {
    const int span = min(cend - t0, a.dyn_span);
    nch = span > 0 ? dyn_chunks(span, chunk) : (fold ? 1 : 0);
    if (nch > a.nchunks) nch = a.nchunks;
  }
  if (z >= nch) {
    if (z == 0) {  // empty attended range: o = 0, and q normed and rotated (empty_range_q)
      for (int i = tid; i < GH * D; i += NT) a.o[((int64_t)b * a.nq + hq0) * D + i] = 0.f;
      if (ROPE && !fold && a.q_out) empty_range_q<NT>(a, (int64_t)b * a.nq + hq0, GH, D, pos, smem);
    }
    return;
  }
  const int c = nch - 1 - z;  // the new token's chunk first, as in attn_kernel
  const int tb = t0 + c * chunk;
  const int cntg = max(0, min(chunk, cend - tb));
  const bool is_new = fold && c == nch - 1;
  const bool split = nch > 1;
  const int64_t slot = (int64_t)b * a.nkv * nsub + hs;

  const E* __restrict__ Kb = reinterpret_cast<const E*>(a.k);
  const E* __restrict__ Vb = reinterpret_cast<const E*>(a.v);
  const int64_t hoff = (int64_t)h * a.head_stride;
  const int64_t qrow0 = (int64_t)b * a.nq + hq0;

  // ---- prologue ----
  if constexpr (PAGED) {
    int32_t* sblk_w = reinterpret_cast<int32_t*>(smem + L.blk);
    const int p0 = tb >> a.page_shift;
    const int p1 = max(p0, (tb + cntg - 1) >> a.page_shift);
    for (int i = tid; i <= p1 - p0; i += NT)
      sblk_w[i] = a.block_table[(int64_t)b * a.max_blocks + p0 + i];
    lds_barrier();
  }
  const int32_t* sblk = reinterpret_cast<const int32_t*>(smem + L.blk);
  auto row_ptr = [&](const E* base, int t) -> const E* {
    if constexpr (PAGED) {
      const int pg = (t >> a.page_shift) - (tb >> a.page_shift);
      return base + (int64_t)sblk[pg] * a.block_stride + hoff +
             (int64_t)(t & ((1 << a.page_shift) - 1)) * a.tok_stride;
    } else {
      return base + (int64_t)t * a.tok_stride + hoff;
    }
  };
  // Q8: the fp32 scale of row t of head h
  auto sc_ptr = [&](const E* base, int t) -> const float* {
    const char* p = reinterpret_cast<const char*>(base) + a.sc_off + h * a.sc_head;
    if constexpr (PAGED) {
      const int pg = (t >> a.page_shift) - (tb >> a.page_shift);
      return reinterpret_cast<const float*>(p + (int64_t)sblk[pg] * a.block_stride) +
             (t & ((1 << a.page_shift) - 1));
    } else {
      return reinterpret_cast<const float*>(p + (int64_t)t * a.tok_stride);
    }
  };
  // Row mapping.  Paged: the chunk's rows [tb, tb + cntg), in order.  A
  // contiguous cache: tile k of chunk c is the range's 32-row tile
  // c + k*nch (cyclic), so at any moment the launch's workgroups read
  // neighbouring tiles (a streaming probe of c5's layout: 5.17 TB/s with
  // each chunk one block of rows, 5.78 TB/s cyclic).  Rows past the end load
  // the last row of the range (the first of an empty one): every wave issues
  // the same loads on every path.
  const int rlim = PAGED ? cntg : cend - t0;  // rows of the chunk / of the whole range
  const int rfirst = PAGED ? tb : t0;
  const int rmax = max(rlim - 1, 0);
  int ntiles;
  if constexpr (PAGED) {
    ntiles = (cntg + kTile - 1) / kTile;
  } else {
    const int gt = (rlim + kTile - 1) / kTile;  // tiles of the range
    ntiles = c < gt ? (gt - 1 - c) / nch + 1 : 0;
  }
  auto tile_row = [&](int tile) -> int {  // first row of a tile, from rfirst
    if (SC && tile >= NW && tile < ntiles) tile = NW + ntiles - 1 - tile;  // as attn_kernel's block_row
    return PAGED ? tile * kTile : (c + tile * nch) * kTile;
  };
  u32x4 kr[2][KL], vr[2][KL];
  float skr[2] = {0.f, 0.f}, svr[2] = {0.f, 0.f};  // Q8: scales of this lane's A-rows
  // Rows load without the streaming hint here (measured: c4 bf16 -8%, c5q8
  // -16% kernel time): Q8 KV heads share lines (the token's scales; in a
  // token-major cache, the head rows too), so a line fetched for one head
  // has to stay in L2 for the next, and the paged rows gain as well.
  auto load_tile = [&](int tile) {
    if constexpr (Q8) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = rfirst + min(tile_row(tile) + 16 * u + m16, rmax);
        skr[u] = *sc_ptr(Kb, t);
        svr[u] = *sc_ptr(Vb, t);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = rfirst + min(tile_row(tile) + 16 * u + m16, rmax);
      const E* pk = row_ptr(Kb, t);
      const E* pv = row_ptr(Vb, t);
      if constexpr (Q8) {
#pragma unroll
        for (int j = 0; j < KL; ++j)
          kr[u][j] = *reinterpret_cast<const u32x4*>(pk + 64 * j + 16 * g4);
#pragma unroll
        for (int j = 0; j < KL; ++j)
          vr[u][j] = *reinterpret_cast<const u32x4*>(pv + 16 * (g4 + 4 * j));
      } else {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          kr[u][kk] = *reinterpret_cast<const u32x4*>(pk + 32 * kk + 8 * g4);
#pragma unroll
        for (int q = 0; q < KK; ++q)
          vr[u][q] = *reinterpret_cast<const u32x4*>(pv + 8 * (g4 + 4 * q));
      }
    }
  };
  constexpr int QV = GH * D / 4;
  constexpr int QPT = (QV + NT - 1) / NT;
  static_assert(D <= NT, "one thread per head-dim element in the prologue");
  f32x4 qv[QPT];
#pragma unroll
  for (int u = 0; u < QPT; ++u)
    qv[u] = reinterpret_cast<const f32x4*>(a.q + qrow0 * D)[min(tid + u * NT, QV - 1)];
  float invf = 0.f, knv = 0.f, vnv = 0.f, kwv = 0.f;
  f32x4 qwt[QPT];  // q norm weights of this thread's q elements
  if constexpr (ROPE) {
    // every path issues these loads: a layer without RoPE (inv_freq NULL)
    // or without an append reads q in their place (nq >= nkv rows), unused
    const float* ivp = a.inv_freq ? a.inv_freq : a.q;
    const float* knp = fold ? a.k_new : a.q;
    const float* vnp = fold ? a.v_new : a.q;
    invf = ivp[min(tid, D / 2 - 1)];
    knv = knp[((int64_t)b * a.nkv + h) * D + min(tid, D - 1)];
    vnv = vnp[((int64_t)b * a.nkv + h) * D + min(tid, D - 1)];
    if (a.q_norm) {
#pragma unroll
      for (int u = 0; u < QPT; ++u)
        qwt[u] = reinterpret_cast<const f32x4*>(a.q_norm)[min(tid + u * NT, QV - 1) % (D / 4)];
    }
    if (is_new && a.k_norm) kwv = a.k_norm[min(tid, D - 1)];
  }
  float vq[kVnPT];
  const bool vn = ROPE && is_new && a.v_norm;  // uniform over the workgroup
  if (vn) v_norm_load<D, NT>(a, b, tid, vq, DH);
  int tile = w;  // each wave's first tile; the rest are claimed
  load_tile(tile);
  if (tid == 0) misc[0] = NW;
  if constexpr (ROPE) {
    if (a.q_norm) q_norm_regs<D, QPT>(a, qv, qwt, DH);
  }
#pragma unroll
  for (int u = 0; u < QPT; ++u) {
    const int i = tid + u * NT;
    if (i < QV) *reinterpret_cast<f32x4*>(qs + (i / (D / 4)) * QSTR + 4 * (i % (D / 4))) = qv[u];
  }
  if constexpr (ROPE) {
    float* csn = smem + L.cs;
    float* sn = smem + L.sn;
    const bool rot = a.inv_freq != nullptr;  // uniform: no RoPE on a NoPE layer
    if (rot && tid < D / 2) {
      const float ang = (float)pos * invf;
      double sd, cd;
      sincos((double)ang, &sd, &cd);
      csn[tid] = (float)cd;
      sn[tid] = (float)sd;
    }
    if (is_new && tid < D) {
      knew[tid] = knv;
      vnew[tid] = vnv;
    }
    if (vn) v_norm_share<D, NT>(a, b, tid, w, lane, vq, smem + L.wl, DH);
    if (tid < D) smem[L.nw + tid] = kwv;
    if (is_new && a.k_norm) k_norm_share(w, lane, tid < D ? knv * knv : 0.f, smem + L.wm);
    lds_barrier();
    for (int i = tid; rot && i < GH * (D / 2); i += NT) {
      const int g = i / (D / 2), j = i - g * (D / 2);
      const float x0 = qs[g * QSTR + j], x1 = qs[g * QSTR + j + D / 2];
      qs[g * QSTR + j] = x0 * csn[j] - x1 * sn[j];
      qs[g * QSTR + j + D / 2] = x0 * sn[j] + x1 * csn[j];
    }
    if (is_new) {
      const NewNorms nn = new_norms<D, NW>(a, smem + L.wm, smem + L.wl, DH);
      for (int j = tid; j < D / 2; j += NT) {
        float k0 = knew[j], k1 = knew[j + D / 2];
        float v0 = vnew[j], v1 = vnew[j + D / 2];
        nn.apply(a, smem + L.nw, j, D / 2, k0, k1, v0, v1);
        const float r0 = rot ? k0 * csn[j] - k1 * sn[j] : k0;
        const float r1 = rot ? k0 * sn[j] + k1 * csn[j] : k1;
        if constexpr (Q8) {  // quantized after the stream (whole rows)
          knew[j] = r0;
          knew[j + D / 2] = r1;
          vnew[j] = v0;
          vnew[j + D / 2] = v1;
        } else {
          knew[j] = __uint_as_float((uint32_t)f32_to_bf16(r0) << 16);
          knew[j + D / 2] = __uint_as_float((uint32_t)f32_to_bf16(r1) << 16);
          vnew[j] = __uint_as_float((uint32_t)f32_to_bf16(v0) << 16);
          vnew[j + D / 2] = __uint_as_float((uint32_t)f32_to_bf16(v1) << 16);
        }
      }
    }
  }
  lds_barrier();

  int next_fixed = w + NW;
  auto claim = [&]() -> int {
    if (!a.dynamic) {
      const int v = next_fixed;
      next_fixed += NW;
      return v;
    }
    int v = 0;
    if (lane == 0) v = atomicAdd(&misc[0], 1);
    return __builtin_amdgcn_readfirstlane(v);
  };

  // q^T as the B operand: lane l holds head l%16 (zero past GH), elements
  // 32*kk + 8*(l/16) + e (Q8: 64*(kk/2) + 16*(l/16) + 8*(kk%2) + e), scaled
  // by scale*log2(e), in three bf16 pieces.  16-byte reads of rows QSTR =
  // D + 4 floats apart: the 8 lanes of a read (heads r .. r+7) fall in 8
  // distinct 16-byte slots (rows of D floats: one slot, 8-way conflicts).
  const float qsc = a.scale * kLog2e;
  bf16x8_t qh[KK], qm[KK], ql[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
#pragma unroll
    for (int e4 = 0; e4 < 8; e4 += 4) {
      const int di = Q8 ? 64 * (kk >> 1) + 16 * g4 + 8 * (kk & 1) + e4 : 32 * kk + 8 * g4 + e4;
      const f32x4 x4 = m16 < GH ? *reinterpret_cast<const f32x4*>(qs + m16 * QSTR + di)
                                : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        __bf16 hi, mid, lo;
        split3(x4[e] * qsc, hi, mid, lo);
        qh[kk][e4 + e] = hi;
        qm[kk][e4 + e] = mid;
        ql[kk][e4 + e] = lo;
      }
    }

  // SC, as attn_kernel; the lane's head is m16
  [[maybe_unused]] float slope = 0.f, cap2 = 0.f, rcap = 0.f;
  [[maybe_unused]] __amdgpu_buffer_rsrc_t swr;
  [[maybe_unused]] const int swo = 4 * (sub * GH + m16);
  if constexpr (SC) {
    if (a.slopes && m16 < GH) slope = a.slopes[hq0 + m16] * kLog2e;
    cap2 = a.softcap * kLog2e;
    rcap = a.softcap > 0.f ? 1.f / cap2 : 0.f;
    swr = score_rsrc(a, b, h);
  }

  // ---- stream ----
  char* vt = reinterpret_cast<char*>(smem + L.vt + w * RS);
  f32x4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  float* scw = smem + L.sc + w * (2 * kTile);  // Q8: this wave's scale slots
  while (tile < ntiles) {
    // V rows into this wave's LDS region (lane: row 16u + l%16, 16-byte
    // units l/16 + 4q), swizzled by vt_off
    f32x4 sk4[2], sv4[2];  // Q8: scales of accumulator rows 16u + 4*(l/16) + r
    if constexpr (Q8) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          // load j holds row bytes 16*(l/16 + 4j): 32-byte bf16 segment l/16 + 4j
          const int r = 16 * u + m16, s = g4 + 4 * j;
          u32x4 lo, hi;
          i8x16_to_bf16(vr[u][j], lo, hi);
          *reinterpret_cast<u32x4*>(vt + vt_off<D>(r, 2 * s)) = lo;
          *reinterpret_cast<u32x4*>(vt + vt_off<D>(r, 2 * s + 1)) = hi;
        }
      if (g4 == 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          scw[16 * u + m16] = skr[u];
          scw[kTile + 16 * u + m16] = svr[u];
        }
      }
      // the slots are this wave's own: LDS keeps its order, and the fence
      // keeps the compiler from moving the reads above the writes
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        sk4[u] = *reinterpret_cast<const f32x4*>(scw + 16 * u + 4 * g4);
        sv4[u] = *reinterpret_cast<const f32x4*>(scw + kTile + 16 * u + 4 * g4);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < KK; ++q) {
          const int r = 16 * u + m16, ch = g4 + 4 * q;
          *reinterpret_cast<u32x4*>(vt + vt_off<D>(r, ch)) = vr[u][q];
        }
    }
    // scores of the two 16-row halves
    f32x4 sacc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sacc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (Q8) {
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          u32x4 lo, hi;
          i8x16_to_bf16(kr[u][j], lo, hi);
          const bf16x8_t k0 = __builtin_bit_cast(bf16x8_t, lo);
          const bf16x8_t k1 = __builtin_bit_cast(bf16x8_t, hi);
          sacc[u] = mfma_bf16(k0, ql[2 * j], sacc[u]);
          sacc[u] = mfma_bf16(k0, qm[2 * j], sacc[u]);
          sacc[u] = mfma_bf16(k0, qh[2 * j], sacc[u]);
          sacc[u] = mfma_bf16(k1, ql[2 * j + 1], sacc[u]);
          sacc[u] = mfma_bf16(k1, qm[2 * j + 1], sacc[u]);
          sacc[u] = mfma_bf16(k1, qh[2 * j + 1], sacc[u]);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const bf16x8_t kv = __builtin_bit_cast(bf16x8_t, kr[u][kk]);
          sacc[u] = mfma_bf16(kv, ql[kk], sacc[u]);
          sacc[u] = mfma_bf16(kv, qm[kk], sacc[u]);
          sacc[u] = mfma_bf16(kv, qh[kk], sacc[u]);
        }
      }
    }
    // the next tile's loads go out while this one is finished
    const int nx = claim();
    if (nx < ntiles) load_tile(nx);
    // online softmax (base 2) on the accumulators: lane = head l%16, rows
    // 16u + 4*(l/16) + r
    float sv[2][4];
    float tmax = -INFINITY;
    if constexpr (SC) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = Q8 ? sacc[i / 4][i % 4] * sk4[i / 4][i % 4] : sacc[i / 4][i % 4];
      if (a.softcap > 0.f) cap_scores<8>(x, cap2, rcap);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = tile_row(tile) + 16 * (i / 4) + 4 * g4 + i % 4;
        const int t = rfirst + row;
        const float y = fmaf(-slope, fabsf((float)(pos - t)), x[i]);
        sv[i / 4][i % 4] = row < rlim ? y : -INFINITY;
        tmax = fmaxf(tmax, sv[i / 4][i % 4]);
      }
      // rows 16u + 4*g4 .. +3 of a head side by side (chunks start at multiples of 4)
      bool part = false;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = tile_row(tile) + 16 * u + 4 * g4, at = rfirst - t0 + row;
        part = part || (row < rlim && row + 4 > rlim);
        __builtin_amdgcn_raw_buffer_store_b128(
            __builtin_bit_cast(u32x4, f32x4{sv[u][0], sv[u][1], sv[u][2], sv[u][3]}), swr,
            m16 < GH && row + 4 <= rlim ? 4 * (at * G + swo) : -1, 0, 0);
      }
      if (__builtin_amdgcn_ballot_w64(part) != 0) {  // the rows' end, once: another wave may own the next
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int u = i / 4, row = tile_row(tile) + 16 * u + 4 * g4, at = rfirst - t0 + row;
          __builtin_amdgcn_raw_buffer_store_b32(
              __float_as_uint(sv[u][i % 4]), swr,
              m16 < GH && row + 4 > rlim && row + i % 4 < rlim ? 4 * (at * G + swo + i % 4) : -1, 0, 0);
        }
      }
    } else
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = tile_row(tile) + 16 * u + 4 * g4 + r;
        sv[u][r] = row < rlim ? (Q8 ? sacc[u][r] * sk4[u][r] : sacc[u][r]) : -INFINITY;
        tmax = fmaxf(tmax, sv[u][r]);
      }
    tmax = max_xor32(max_xor16(tmax));
    // finite: a claimed tile has a row; the first tile always moves the max
    if (__builtin_amdgcn_ballot_w64(tmax > m_run + kLazyMax) != 0) {
      const float mn = fmaxf(m_run, tmax);
      const float alpha = exp2_hw(m_run - mn);
      m_run = mn;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    }
    bf16x8_t ph, pm, pl;
    float ps = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = exp2_hw(sv[u][r] - m_run);
        ps += p;
        __bf16 hi, mid, lo;
        split3(Q8 ? p * sv4[u][r] : p, hi, mid, lo);
        ph[4 * u + r] = hi;
        pm[4 * u + r] = mid;
        pl[4 * u + r] = lo;
      }
    l_run += ps;
    __builtin_amdgcn_wave_barrier();
    // PV: V^T of the 16-row block dt by two transposed reads
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      i16x4_t t2[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = (lane >> 2) + 16 * u;
        t2[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4_t*)(
                vt + vt_off<D>(r, 2 * dt + ((lane & 3) >> 1)) + 8 * (lane & 1)));
      }
      const bf16x8_t av = __builtin_bit_cast(
          bf16x8_t, __builtin_shufflevector(t2[0], t2[1], 0, 1, 2, 3, 4, 5, 6, 7));
      o[dt] = mfma_bf16(av, pl, o[dt]);
      o[dt] = mfma_bf16(av, pm, o[dt]);
      o[dt] = mfma_bf16(av, ph, o[dt]);
    }
    __builtin_amdgcn_wave_barrier();
    tile = nx;
  }

  // ---- the new token: folded in by wave 0 (appended by subgroup 0 at the
  // very end, like attn_kernel's append: nothing may wait for those stores) ----
  [[maybe_unused]] int kcode[D / 64], vcode[D / 64];  // Q8: the row's codes
  [[maybe_unused]] float kscale = 0.f, vscale = 0.f;  // Q8: and scales
  if constexpr (Q8) {
    if (is_new && w == 0) {
      // quantize the k and v rows as the cache holds them; LDS gets code * s
      constexpr int EPL = D / 64;
      float kx[EPL], vx[EPL];
      float ka = 0.f, va = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        kx[e] = knew[lane + 64 * e];
        vx[e] = vnew[lane + 64 * e];
        ka = fmaxf(ka, fabsf(kx[e]));
        va = fmaxf(va, fabsf(vx[e]));
      }
      kscale = q8_scale(group_max<64>(ka));
      vscale = q8_scale(group_max<64>(va));
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        kcode[e] = q8_code(kx[e], kscale);
        vcode[e] = q8_code(vx[e], vscale);
        knew[lane + 64 * e] = (float)kcode[e] * kscale;
        vnew[lane + 64 * e] = (float)vcode[e] * vscale;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the fold reads other lanes' rows
    }
  }
  if (is_new && w == 0) {
    float part = 0.f;
    if (m16 < GH) {
#pragma unroll 8
      for (int d = g4 * (D / 4); d < (g4 + 1) * (D / 4); ++d)
        part = fmaf(qs[m16 * QSTR + d], knew[d], part);
    }
    part = sum_xor32(sum_xor16(part));
    float snew = part * qsc;  // base 2, as the streamed scores
    if constexpr (SC) {
      float x[1] = {snew};
      if (a.softcap > 0.f) cap_scores<1>(x, cap2, rcap);
      snew = fmaf(-slope, fabsf((float)(pos - (n - 1))), x[0]);
      const int at = n - 1 - t0;
      __builtin_amdgcn_raw_buffer_store_b32(
          __float_as_uint(snew), swr,
          g4 == 0 && m16 < GH ? 4 * ((at & ~3) * G + swo + (at & 3)) : -1, 0, 0);
    }
    const float mn = fmaxf(m_run, snew);
    const float alpha = exp2_hw(m_run - mn);
    const float p = exp2_hw(snew - mn);
    m_run = mn;
    l_run = l_run * alpha + (g4 == 0 ? p : 0.f);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[dt][r] = o[dt][r] * alpha + p * vnew[16 * dt + 4 * g4 + r];
  }

  // ---- the wave's partial into its own LDS region, then the chunk ----
  l_run = sum_xor32(sum_xor16(l_run));
  float* wm = smem + L.wm;
  float* wl = smem + L.wl;
  float* red = smem + L.vt;
  if (m16 < GH) {
    if (g4 == 0) {
      wm[w * GH + m16] = SC ? m_run : m_run * kLn2;  // natural units for the merge
      wl[w * GH + m16] = l_run;
    }
    // head m16's row with its float index XOR 4*(m16 % 8): the 8 lanes of a
    // store then hit distinct 16-byte slots (rows of D floats alone: 8-way)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<f32x4*>(red + w * RS + m16 * D + ((16 * dt + 4 * g4) ^ (4 * (m16 & 7)))) =
          o[dt];
  }
  lds_barrier();
  finish_chunk<D, GH, NW, NT, ROPE, NW * RS, true, QSTR, SC>(a, wm, wl, red, RS, qs, tid, lane, split, slot, c,
                                              qrow0, nch,
                                    smem + L.mrg, red, misc + 1, DH);

  // ---- the append, last ----
  const bool store_new = is_new && sub == 0 && (Q8 ? w == 0 : tid < D);
  if (store_new) {
    const int slot_row = n - 1;
    int64_t off, soff;  // element (Q8: byte) offset of the row; Q8: of its scale
    if constexpr (PAGED) {
      const int64_t blk = a.block_table[(int64_t)b * a.max_blocks + (slot_row >> a.page_shift)];
      const int sl = slot_row & ((1 << a.page_shift) - 1);
      off = blk * a.block_stride + hoff + (int64_t)sl * a.tok_stride;
      soff = blk * a.block_stride + a.sc_off + h * a.sc_head + 4 * sl;
    } else {
      off = (int64_t)slot_row * a.tok_stride + hoff;
      soff = (int64_t)slot_row * a.tok_stride + a.sc_off + h * a.sc_head;
    }
    if constexpr (!Q8) {
      reinterpret_cast<uint16_t*>(a.k)[off + tid] = f32_to_bf16(knew[tid]);
      reinterpret_cast<uint16_t*>(a.v)[off + tid] = f32_to_bf16(vnew[tid]);
    } else {
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        reinterpret_cast<int8_t*>(a.k)[off + lane + 64 * e] = (int8_t)kcode[e];
        reinterpret_cast<int8_t*>(a.v)[off + lane + 64 * e] = (int8_t)vcode[e];
      }
      if (lane == 0) {
        *reinterpret_cast<float*>(reinterpret_cast<char*>(a.k) + soff) = kscale;
        *reinterpret_cast<float*>(reinterpret_cast<char*>(a.v) + soff) = vscale;
      }
    }
  }
}

}  // namespace

#endif  // MOLOT_AMD_CSRC_ATTN_KERNELS_HPP_
