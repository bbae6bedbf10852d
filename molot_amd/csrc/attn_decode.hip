// MI355X (gfx950) fused RoPE + GQA decode attention.
//
// This file: the C ABI, the host's plans and the kernels around the attention:
//   rope_append_kernel   RoPE of q (in place) and of the new k, append of the
//                        rotated k and v into the cache slot
//                        (include/molot/forward.h:556-575);
//   combine_kernel       log-sum-exp merge of a split context's chunk partials
//                        (combine_wave_kernel: of few chunks; combine_rows_kernel:
//                        of a prefill's key splits);
//   attn_weights_kernel  the softmax weights of a scored launch, summed a KV head
//                        (combine_weights_kernel: beside the merge);
//   prefill_mfma16_kernel, pf_split_kernel.
// The decode attention's kernels are in attn_kernels.hpp, its instances in
// attn_flat.hip, attn_paged.hip and, scored, attn_flat_scored.hip and
// attn_paged_scored.hip; the prefill's others in prefill_narrow.hip and
// prefill_wide.hip; a cache's eviction in kv_evict.hip.
//
// All shapes are validated on the host before any launch.
#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <mutex>
#include <type_traits>
#include <utility>
#include <vector>

#include "attn_args.hpp"
#include "attn_host.hpp"
#include "attn_kernels.hpp"
#include "device_util.hpp"
#include "molot_amd/attn_hip.h"
#include "paged_plan.hpp"
#include "prefill.hpp"
#include "prefill_wide.hpp"
#include "ws_growth.hpp"

namespace {

// ---------------------------------------------------------------------------
// RoPE + append.
struct RopeArgs {
  float* q;            // [B][nq][d], rotated in place (may be null)
  const float* k_new;  // [B][nkv][d]
  const float* v_new;  // [B][nkv][d]
  void* K;
  void* V;
  const float* inv_freq;  // [d/2]
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* pos_arr;
  const float* q_norm;  // [d] q RMS-norm weights (NULL: no q norm)
  const float* k_norm;  // [d] k RMS-norm weights (NULL: no k norm)
  int64_t tok_stride, head_stride, block_stride;
  int nq, nkv, d, slot, pos, max_blocks, page, kv_dtype, append;
  int v_norm;           // RMS-norm v over all nkv*d values, no weights
  float eps;
  int tokens;           // grid row b = token b of a prefill: slot + b at pos + b
  int64_t sc_off, sc_head;  // Q8 scales, as AttnArgs::sc_off / sc_head
  // prefill over an fp32 or Q8 cache: the appended rows also leave their
  // pieces (as pf_split_kernel writes them) at row slot - pc_T0 of
  // [K, V][nkv][3][pc_R][d], when that row lies in [0, pc_R) (NULL: none)
  uint16_t* pieces;
  int pc_T0, pc_R;
  // pieces per value in the layout of prefill_wide.hpp (0: the three-slot
  // layout of pf_split_kernel)
  int pc_np;
  int own;  // with pc_np: mark the rows that PfArgs::own launches form again
};

// One workgroup per (head of q or k, sequence); one thread per rotation pair.
// Angle is the fp32 product pos*inv_freq[i] (include/molot/attn.h:22); its
// sine and cosine are evaluated in double and rounded, i.e. a full-range,
// correctly rounded (barring double rounding) fp32 sin/cos.  With the
// layer's norms (forward.h:554, 562-563) a head is RMS-normed before its
// rotation: (x * 1/sqrt(mean(x^2) + eps)) * w (include/molot/norm.h:9-28),
// and v by the RMS of all nkv*d values of the sequence's v (norm.h:82-96).
__global__ void rope_append_kernel(RopeArgs a) {
  __shared__ float sh[16];
  const int hh = blockIdx.x;
  const int b = blockIdx.y;
  const int half = a.d >> 1;
  const int i = threadIdx.x;
  const bool act = i < half;  // the reductions need every thread
  const int ic = act ? i : 0;
  int pos = a.pos;
  int slot = a.slot;
  if (a.seq_lens) {
    slot = a.seq_lens[b] - 1;
    pos = a.pos_arr ? a.pos_arr[b] : slot;
  } else if (a.tokens) {
    slot += b;
    pos += b;
  }
  const bool rot = a.inv_freq != nullptr;  // a NoPE layer (inv_freq NULL) is not rotated
  float c = 1.f, s = 0.f;
  if (rot) {
    const float ang = (float)pos * a.inv_freq[ic];
    double sd, cd;
    sincos((double)ang, &sd, &cd);
    c = (float)cd;
    s = (float)sd;
  }
  auto rms_inv = [&](float ss, int n) { return 1.0f / sqrtf(ss / (float)n + a.eps); };
  if (hh < a.nq) {
    if (!a.q) return;
    float* x = a.q + ((int64_t)b * a.nq + hh) * a.d;
    float x0 = act ? x[i] : 0.f, x1 = act ? x[i + half] : 0.f;
    if (a.q_norm) {
      const float inv = rms_inv(block_sum(x0 * x0 + x1 * x1, sh), a.d);
      x0 = x0 * inv * a.q_norm[ic];
      x1 = x1 * inv * a.q_norm[ic + half];
    }
    if (act) {
      x[i] = rot ? x0 * c - x1 * s : x0;
      x[i + half] = rot ? x0 * s + x1 * c : x1;
    }
    return;
  }
  if (!a.append) return;
  const int kh = hh - a.nq;
  const float* kx = a.k_new + ((int64_t)b * a.nkv + kh) * a.d;
  const float* vx = a.v_new + ((int64_t)b * a.nkv + kh) * a.d;
  float k0 = act ? kx[i] : 0.f, k1 = act ? kx[i + half] : 0.f;
  float v0 = act ? vx[i] : 0.f, v1 = act ? vx[i + half] : 0.f;
  if (a.k_norm) {
    const float inv = rms_inv(block_sum(k0 * k0 + k1 * k1, sh), a.d);
    k0 = k0 * inv * a.k_norm[ic];
    k1 = k1 * inv * a.k_norm[ic + half];
  }
  if (a.v_norm) {
    const float* vall = a.v_new + (int64_t)b * a.nkv * a.d;
    float part = 0.f;
    for (int j = i; j < a.nkv * a.d; j += blockDim.x) part = fmaf(vall[j], vall[j], part);
    const float inv = rms_inv(block_sum(part, sh), a.nkv * a.d);
    v0 *= inv;
    v1 *= inv;
  }
  const float r0 = rot ? k0 * c - k1 * s : k0;  // 0 on the threads past the pairs
  const float r1 = rot ? k0 * s + k1 * c : k1;
  float ks = 0.f, vs = 0.f;
  if (a.kv_dtype == MOLOT_KV_Q8) {  // uniform: every thread takes the maxima
    ks = q8_scale(block_max(fmaxf(fabsf(r0), fabsf(r1)), sh));
    vs = q8_scale(block_max(fmaxf(fabsf(v0), fabsf(v1)), sh));
  }
  if (!act) return;
  // element (Q8: byte) offset of the row, and (Q8) of its scale
  int64_t off, soff;
  if (a.block_table) {
    const int64_t blk = a.block_table[(int64_t)b * a.max_blocks + slot / a.page];
    off = blk * a.block_stride + (int64_t)kh * a.head_stride + (int64_t)(slot % a.page) * a.tok_stride;
    soff = blk * a.block_stride + a.sc_off + kh * a.sc_head + 4 * (int64_t)(slot % a.page);
  } else {
    off = (int64_t)slot * a.tok_stride + (int64_t)kh * a.head_stride;
    soff = (int64_t)slot * a.tok_stride + a.sc_off + kh * a.sc_head;
  }
  if (a.kv_dtype == MOLOT_KV_Q8) {
    int8_t* kd = (int8_t*)a.K + off;
    int8_t* vd = (int8_t*)a.V + off;
    kd[i] = (int8_t)q8_code(r0, ks);
    kd[i + half] = (int8_t)q8_code(r1, ks);
    vd[i] = (int8_t)q8_code(v0, vs);
    vd[i + half] = (int8_t)q8_code(v1, vs);
    if (i == 0) {
      *(float*)((char*)a.K + soff) = ks;
      *(float*)((char*)a.V + soff) = vs;
    }
  } else if (a.kv_dtype == MOLOT_KV_F32) {
    float* kd = (float*)a.K + off;
    float* vd = (float*)a.V + off;
    kd[i] = r0;
    kd[i + half] = r1;
    vd[i] = v0;
    vd[i + half] = v1;
  } else {
    uint16_t* kd = (uint16_t*)a.K + off;
    uint16_t* vd = (uint16_t*)a.V + off;
    kd[i] = f32_to_bf16(r0);
    kd[i + half] = f32_to_bf16(r1);
    vd[i] = f32_to_bf16(v0);
    vd[i + half] = f32_to_bf16(v1);
  }
}

// The prefill's RoPE/append (and the q prologue): one workgroup of 4 waves
// per token instead of one per (head, token).  The token's sine and cosine
// are taken once (in double, as rope_append_kernel) into LDS; wave w takes
// heads w, w + 4, ..., lane l the pairs l, l + 64, ... of a head, so a head's
// norm sum and Q8 maximum stay in its wave.  Sums run as rope_append_kernel's
// (per 64 pairs, added in order), so rows of d <= 128 come out bit-identical.
// 2048 tokens of 32q/8kv/d128: 81920 single-wave workgroups became 2048.
constexpr int kRopeTokThreads = 256;
constexpr int kRopeMaxPairs = 1024;  // d <= 2048
// KMAX: pair groups of 64 a head holds at most (d <= 128 KMAX); P32: the
// rows' pieces in the layout of prefill_wide.hpp, pc_np of them, else in the
// three slots of pf_split_kernel.
template <int KMAX, bool P32>
__global__ __launch_bounds__(kRopeTokThreads) void rope_append_tok_kernel(RopeArgs a) {
  __shared__ float cs_s[kRopeMaxPairs], sn_s[kRopeMaxPairs];
  __shared__ float sh[16];
  const int b = blockIdx.x;
  const int half = a.d >> 1;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int pos = a.pos + b, slot = a.slot + b;
  const bool rot = a.inv_freq != nullptr;
  for (int i = tid; rot && i < half; i += kRopeTokThreads) {
    const float ang = (float)pos * a.inv_freq[i];
    double sd, cd;
    sincos((double)ang, &sd, &cd);
    cs_s[i] = (float)cd;
    sn_s[i] = (float)sd;
  }
  auto rms_inv = [&](float ss, int n) { return 1.0f / sqrtf(ss / (float)n + a.eps); };
  // the v norm: one RMS over the token's nkv*d values (wave 0, stride 64)
  if (a.append && a.v_norm && w == 0) {
    const float* vall = a.v_new + (int64_t)b * a.nkv * a.d;
    float part = 0.f;
    for (int j = lane; j < a.nkv * a.d; j += 64) part = fmaf(vall[j], vall[j], part);
    part = group_sum<64>(part);
    if (lane == 0) sh[0] = rms_inv(part, a.nkv * a.d);
  }
  __syncthreads();
  const float vinv = a.append && a.v_norm ? sh[0] : 1.f;
  const int nk = (half + 63) / 64;  // pair groups of 64 per head
  // Each wave walks its heads with the next head's rows loaded before the
  // current head's stores go out (heads own disjoint rows), so a wave waits
  // for one load latency in all rather than one per head.
  auto load_q = [&](int hh, float* y0, float* y1) {
    const float* x = a.q + ((int64_t)b * a.nq + hh) * a.d;
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      if (k >= nk) break;
      const int j = lane + 64 * k;
      y0[k] = j < half ? x[j] : 0.f;
      y1[k] = j < half ? x[j + half] : 0.f;
    }
  };
  if (a.q) {
    float x0[KMAX], x1[KMAX], n0[KMAX] = {}, n1[KMAX] = {};
    if (w < a.nq) load_q(w, n0, n1);
    for (int hh = w; hh < a.nq; hh += kRopeTokThreads / 64) {
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        x0[k] = n0[k];
        x1[k] = n1[k];
      }
      if (hh + kRopeTokThreads / 64 < a.nq) load_q(hh + kRopeTokThreads / 64, n0, n1);
      float* x = a.q + ((int64_t)b * a.nq + hh) * a.d;
      float ss = 0.f;
      if (a.q_norm) {
#pragma unroll
        for (int k = 0; k < KMAX; ++k) {
          if (k >= nk) break;
          ss += group_sum<64>(x0[k] * x0[k] + x1[k] * x1[k]);
        }
      }
      const float inv = a.q_norm ? rms_inv(ss, a.d) : 1.f;
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        if (k >= nk) break;
        const int j = lane + 64 * k;
        if (j >= half) continue;
        float y0 = x0[k], y1 = x1[k];
        if (a.q_norm) {
          y0 = y0 * inv * a.q_norm[j];
          y1 = y1 * inv * a.q_norm[j + half];
        }
        x[j] = rot ? y0 * cs_s[j] - y1 * sn_s[j] : y0;
        x[j + half] = rot ? y0 * sn_s[j] + y1 * cs_s[j] : y1;
      }
    }
  }
  if (!a.append) return;
  // KV heads: wave w takes heads kh with (nq + kh) % 4 == w
  auto load_kv = [&](int kh, float* k0, float* k1, float* v0, float* v1) {
    const float* kx = a.k_new + ((int64_t)b * a.nkv + kh) * a.d;
    const float* vx = a.v_new + ((int64_t)b * a.nkv + kh) * a.d;
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      if (k >= nk) break;
      const int j = lane + 64 * k;
      k0[k] = j < half ? kx[j] : 0.f;
      k1[k] = j < half ? kx[j + half] : 0.f;
      v0[k] = j < half ? vx[j] : 0.f;
      v1[k] = j < half ? vx[j + half] : 0.f;
    }
  };
  constexpr int kWaves = kRopeTokThreads / 64;
  const int kh0 = ((w - a.nq) % kWaves + kWaves) % kWaves;
  float nk0[KMAX] = {}, nk1[KMAX] = {}, nv0[KMAX] = {}, nv1[KMAX] = {};
  if (kh0 < a.nkv) load_kv(kh0, nk0, nk1, nv0, nv1);
  for (int kh = kh0; kh < a.nkv; kh += kWaves) {
    float r0[KMAX], r1[KMAX], v0[KMAX], v1[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      r0[k] = nk0[k];
      r1[k] = nk1[k];
      v0[k] = nv0[k] * vinv;
      v1[k] = nv1[k] * vinv;
    }
    if (kh + kWaves < a.nkv) load_kv(kh + kWaves, nk0, nk1, nv0, nv1);
    float ss = 0.f;
    if (a.k_norm) {
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        if (k >= nk) break;
        ss += group_sum<64>(r0[k] * r0[k] + r1[k] * r1[k]);
      }
    }
    const float kinv = a.k_norm ? rms_inv(ss, a.d) : 1.f;
    float kmax = 0.f, vmax = 0.f;
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      if (k >= nk) break;
      const int j = lane + 64 * k;
      const int jc = j < half ? j : 0;
      float k0 = r0[k], k1 = r1[k];
      if (a.k_norm) {
        k0 = k0 * kinv * a.k_norm[jc];
        k1 = k1 * kinv * a.k_norm[jc + half];
      }
      r0[k] = rot ? k0 * cs_s[jc] - k1 * sn_s[jc] : k0;  // 0 past the pairs
      r1[k] = rot ? k0 * sn_s[jc] + k1 * cs_s[jc] : k1;
      kmax = fmaxf(kmax, fmaxf(fabsf(r0[k]), fabsf(r1[k])));
      vmax = fmaxf(vmax, fmaxf(fabsf(v0[k]), fabsf(v1[k])));
    }
    float ks = 0.f, vs = 0.f;
    if (a.kv_dtype == MOLOT_KV_Q8) {
      ks = q8_scale(group_max<64>(kmax));
      vs = q8_scale(group_max<64>(vmax));
    }
    int64_t off, soff;
    if (a.block_table) {
      const int64_t blk = a.block_table[slot / a.page];
      off = blk * a.block_stride + (int64_t)kh * a.head_stride + (int64_t)(slot % a.page) * a.tok_stride;
      soff = blk * a.block_stride + a.sc_off + kh * a.sc_head + 4 * (int64_t)(slot % a.page);
    } else {
      off = (int64_t)slot * a.tok_stride + (int64_t)kh * a.head_stride;
      soff = (int64_t)slot * a.tok_stride + a.sc_off + kh * a.sc_head;
    }
    #pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      if (k >= nk) break;
      const int j = lane + 64 * k;
      if (j >= half) continue;
      if (a.kv_dtype == MOLOT_KV_Q8) {
        int8_t* kd = (int8_t*)a.K + off;
        int8_t* vd = (int8_t*)a.V + off;
        kd[j] = (int8_t)q8_code(r0[k], ks);
        kd[j + half] = (int8_t)q8_code(r1[k], ks);
        vd[j] = (int8_t)q8_code(v0[k], vs);
        vd[j + half] = (int8_t)q8_code(v1[k], vs);
      } else if (a.kv_dtype == MOLOT_KV_F32) {
        float* kd = (float*)a.K + off;
        float* vd = (float*)a.V + off;
        kd[j] = r0[k];
        kd[j + half] = r1[k];
        vd[j] = v0[k];
        vd[j + half] = v1[k];
      } else {
        uint16_t* kd = (uint16_t*)a.K + off;
        uint16_t* vd = (uint16_t*)a.V + off;
        kd[j] = f32_to_bf16(r0[k]);
        kd[j + half] = f32_to_bf16(r1[k]);
        vd[j] = f32_to_bf16(v0[k]);
        vd[j + half] = f32_to_bf16(v1[k]);
      }
    }
    if (a.kv_dtype == MOLOT_KV_Q8 && lane == 0) {
      *(float*)((char*)a.K + soff) = ks;
      *(float*)((char*)a.V + soff) = vs;
    }
    // the row's pieces for the prefill (of the cached values: fp32 as
    // stored, Q8 as code * scale), the bits pf_split_kernel writes: K and
    // V as two fp16 pieces of the row scaled by a power of two (split2h,
    // the row's unit at float pr of the head's third piece)
    const int pr = slot - a.pc_T0;
    if (a.pieces && (P32 || a.kv_dtype != MOLOT_KV_BF16) && pr >= 0 && pr < a.pc_R) {
      const int np = P32 ? a.pc_np : 0;
      const int64_t Rp = np ? wide_padded_rows(a.pc_R) : a.pc_R;
      const int64_t pstride = Rp * a.d;  // one piece of one head
      const int64_t hstride = np ? wide_head_elems(a.d, np, Rp) : 3 * pstride;
      // the value a piece holds: as cached (three-slot layout: Q8 code *
      // scale; else its code, the scale goes into the unit)
      auto cached = [&](float x, float sc) {
        if (a.kv_dtype == MOLOT_KV_Q8) return np ? (float)q8_code(x, sc) : (float)q8_code(x, sc) * sc;
        if (P32 && a.kv_dtype == MOLOT_KV_BF16)
          return __uint_as_float((uint32_t)f32_to_bf16(x) << 16);
        return x;
      };
      float kpm = 0.f, vpm = 0.f;  // the rows' largest |k| and |v| as cached
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        if (k >= nk) break;
        if (lane + 64 * k < half) {
          kpm = fmaxf(kpm, fmaxf(fabsf(cached(r0[k], ks)), fabsf(cached(r1[k], ks))));
          vpm = fmaxf(vpm, fmaxf(fabsf(cached(v0[k], vs)), fabsf(cached(v1[k], vs))));
        }
      }
      kpm = group_max<64>(kpm);
      const int kshift = f16_row_shift(kpm);
      vpm = group_max<64>(vpm);
      const bool q8u = np && a.kv_dtype == MOLOT_KV_Q8;
      const float ksc = q8u ? ks : 1.f, vsc = q8u ? vs : 1.f;
      float mk = 0.f, mv = 0.f;  // wide_split_kernel's marks
      if (P32 && a.own) {
#pragma unroll
        for (int k = 0; k < KMAX; ++k) {
          if (k >= nk) break;
          if (lane + 64 * k < half) {
            mk = fmaf(cached(r0[k], ks) * ksc, 0.f, fmaf(cached(r1[k], ks) * ksc, 0.f, mk));
            mv = fmaf(cached(v0[k], vs) * vsc, 0.f, fmaf(cached(v1[k], vs) * vsc, 0.f, mv));
          }
        }
        mk = own_mark(kpm * ksc, group_sum<64>(mk), 0);
        mv = own_mark(vpm * vsc, group_sum<64>(mv), 1);
      }
      const int vshift = f16_vrow_shift(vpm);
      uint16_t* ok = a.pieces + (int64_t)kh * hstride + (int64_t)pr * a.d;
      uint16_t* ov = ok + (int64_t)a.nkv * hstride;
      if (lane == 0) {  // the units of a head's rows side by side after its pieces
        const int64_t uo = (np ? np : 2) * pstride - (int64_t)pr * a.d;
        reinterpret_cast<float*>(ok + uo)[pr] = f16_row_unit(kshift) * ksc + mk;
        reinterpret_cast<float*>(ov + uo)[pr] = f16_vrow_unit(vpm, vshift) * vsc + mv;
      }
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        if (k >= nk) break;
        const int j = lane + 64 * k;
        if (j >= half) continue;
        uint32_t pk[2], pv[2];
        split2h(cached(r0[k], ks), cached(r1[k], ks), kshift, pk[0], pk[1]);
        split2h(cached(v0[k], vs), cached(v1[k], vs), vshift, pv[0], pv[1]);
#pragma unroll
        for (int pc = 0; pc < 2; ++pc) {
          if (pc == 1 && np == 1) break;
          ok[pc * pstride + j] = (uint16_t)(pk[pc] & 0xFFFF);
          ok[pc * pstride + j + half] = (uint16_t)(pk[pc] >> 16);
          ov[pc * pstride + j] = (uint16_t)(pv[pc] & 0xFFFF);
          ov[pc * pstride + j + half] = (uint16_t)(pv[pc] >> 16);
        }
      }
    }
  }
  // the rows of zeros after the pieces, dealt to the tokens' workgroups
  if constexpr (P32) {
    const int64_t Rp = wide_padded_rows(a.pc_R), hs = wide_head_elems(a.d, a.pc_np, Rp);
    const int upr = a.d / 8;  // 16-byte units a row
    const int n = 2 * a.nkv * a.pc_np * upr;
    for (int64_t r = a.pc_R + b; r < Rp; r += gridDim.x) {
      for (int i = tid; i < n; i += kRopeTokThreads) {
        const int j = i % upr, p = i / upr % a.pc_np, hd = i / upr / a.pc_np;
        *reinterpret_cast<u32x4*>(a.pieces + hd * hs + (p * Rp + r) * a.d + 8 * j) =
            u32x4{0u, 0u, 0u, 0u};
        if (j == 0 && p == 0)
          reinterpret_cast<float*>(a.pieces + hd * hs + a.pc_np * Rp * a.d)[r] = 0.f;
      }
    }
  }
}

// rope_append_tok_kernel for M tokens of head dim d (<= 2048), in the
// narrowest instance: each pair group past d/2 costs registers and issue
// slots (1999 tokens of 8q/2kv/d512: 63 us in the 16-group instance, 29 in
// the 4-group one).
int launch_rope_tok(const RopeArgs& r, int M, void* stream) {
  const int half = r.d / 2;
  auto k = half <= 64 ? (r.pieces && r.pc_np ? rope_append_tok_kernel<1, true>
                                             : rope_append_tok_kernel<1, false>)
           : half <= 128 ? rope_append_tok_kernel<2, false>
           : half <= 256 ? rope_append_tok_kernel<4, false>
                         : rope_append_tok_kernel<kRopeMaxPairs / 64, false>;
  hipLaunchKernelGGL(k, dim3(M), dim3(kRopeTokThreads), 0, (hipStream_t)stream, r);
  return (int)hipGetLastError();
}

// ---------------------------------------------------------------------------
// Causal prefill attention (include/molot/gemm.h:409-446) on the matrix cores.
//
// The query rows of one KV head are r = m*G + g: token m (position pos0 + m)
// and q head h*G + g of the group.  A workgroup of 4 waves owns 64
// consecutive rows, wave w the 16 rows w*16.. on the 16 columns of the
// matrix instructions.  It streams the keys its rows attend, 32 per tile,
// through LDS, with the next tile's global loads in flight while the
// current one is used; each row is masked to its own causal end
// min(pos+1, N) and window start.  Query blocks run from the last (most
// keys) to the first, heads fastest across the grid.
// The reference's exps are libm expf summed in double with the weights
// normalised before PV; here the hardware base-2 exp of scores pre-scaled by
// log2(e), fp32 running sums with a lazy max rescale, and one division at
// the end (fp32 rounding differences).

// Cache offset (elements of T; Q8: bytes) of row t of KV head h, and for Q8
// the byte offset of its scale (soff).  Token-major: [N][nkv*D] (Q8 rows of
// nkv*D codes, then nkv scales padded to 16 bytes); paged: blocks of
// [nkv][page][D] (Q8: [nkv][page][D] codes, then [nkv][page] scales).
template <int D, typename T, bool PAGED>
__device__ __forceinline__ int64_t pf_row_off(const PfArgs& a, int h, int t, int64_t& soff) {
  constexpr bool Q8 = std::is_same<T, q8_t>::value;
  const int pg = 1 << a.page_shift;
  const int64_t R = (int64_t)a.nkv * D + ((4 * a.nkv + 15) & ~15);
  const int64_t BB = (int64_t)a.nkv * pg * (D + 4);
  if constexpr (PAGED) {
    const int64_t blk = a.block_table[t >> a.page_shift];
    const int sl = t & (pg - 1);
    if constexpr (Q8) {
      soff = blk * BB + (int64_t)a.nkv * pg * D + 4 * ((int64_t)h * pg + sl);
      return blk * BB + ((int64_t)h * pg + sl) * D;
    }
    return ((blk * a.nkv + h) * pg + sl) * (int64_t)a.dh;
  } else {
    if constexpr (Q8) {
      soff = (int64_t)t * R + (int64_t)a.nkv * D + 4 * h;
      return (int64_t)t * R + (int64_t)h * D;
    }
    return ((int64_t)t * a.nkv + h) * (int64_t)a.dh;
  }
}

// K and V of the keys [T0, T0 + R) as pieces (the values the prefill kernel
// would split per tile: fp32 rows, or Q8 code * s), into [K, V][nkv][3][R][D]
// (16-bit elements): K and V rows as two fp16 pieces of the row scaled by a
// power of two (split2h), the rows' units (floats) side by side at the start
// of the third.  Thread: one 8-element unit of one row, a row's D/8 units in
// consecutive lanes; grid (units / 256, nkv, 2).
template <int D, typename T, bool PAGED>
__global__ __launch_bounds__(256) void pf_split_kernel(PfArgs a, uint16_t* out) {
  constexpr bool Q8 = std::is_same<T, q8_t>::value;
  static_assert(sizeof(T) != 2, "bf16 caches are exact in one piece");
  constexpr int UPR = D / 8;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= (int64_t)a.Rsplit * UPR) return;
  const int h = blockIdx.y, kv = blockIdx.z;
  const int r = (int)(u / UPR), j = (int)(u - (int64_t)r * UPR);
  int64_t soff = 0;
  const int64_t off = pf_row_off<D, T, PAGED>(a, h, a.T0 + r, soff) + 8 * j;
  const void* base = kv ? a.v : a.k;
  float x[8];
  if (8 * j >= a.dh) {  // the padding of a head dim below D (a multiple of 8): zero pieces
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
  } else if constexpr (Q8) {
    const uint2 c = *reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(base) + off);
    const float s = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(base) + soff);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = (float)(int8_t)(((e < 4 ? c.x : c.y) >> (8 * (e & 3))) & 0xFF) * s;
  } else {
    const f32x4 x0 = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(base) + off);
    const f32x4 x1 = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(base) + off + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = x0[e];
      x[4 + e] = x1[e];
    }
  }
  auto row = [&](int p) { return out + ((((int64_t)kv * a.nkv + h) * 3 + p) * a.R + r) * D; };
  // two fp16 pieces of the row scaled by a power of two (split2h), the
  // row's unit (a float) at float r of the head's third piece
  uint32_t pc[2][4];
  float xm = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) xm = fmaxf(xm, fabsf(x[e]));
  xm = group_max<D / 8>(xm);  // the row's UPR lanes
  const int shift = kv ? f16_vrow_shift(xm) : f16_row_shift(xm);
#pragma unroll
  for (int e = 0; e < 8; e += 2) split2h(x[e], x[e + 1], shift, pc[0][e / 2], pc[1][e / 2]);
  if (j == 0)  // the units of a head's rows side by side in its third piece: row r's at float r
    reinterpret_cast<float*>(out + (((int64_t)kv * a.nkv + h) * 3 + 2) * a.R * D)[r] =
        kv ? f16_vrow_unit(xm, shift) : f16_row_unit(shift);
#pragma unroll
  for (int p = 0; p < 2; ++p)
    *reinterpret_cast<u32x4*>(row(p) + 8 * j) = u32x4{pc[p][0], pc[p][1], pc[p][2], pc[p][3]};
}

// Waves per prefill workgroup (16 query rows each): 8, so that 128 rows
// share each staged key tile and its split into pieces (32q/8kv/d128 fp32,
// 2048-token prompt: 285 -> 237 us).  fp32 pieces at d = 256 too (two
// waves a SIMD in 256 registers; 2048-token Gemma-style prompt: 127 ->
// 104 us, its grid then split over the keys).  A launch whose 8-wave grid
// would leave CUs idle and cannot be split takes 4 waves (512-token prompt
// after 16384 cached tokens: 1452 us on 8 waves, 1414 on 4).
constexpr int kPfWaves = 8;

// The kernel: every fp32 product is taken as 16-bit pieces on the dense
// matrix cores (16x the fp32 matrix rate).  Over fp32 and Q8 values both
// products take two fp16 pieces of each operand (split2h: hi = fp16(y),
// lo = fp16(y - hi) of y scaled by a power of two below 2^14) and three
// products (lo*hi, hi*lo, hi*hi) on v_mfma_f32_16x16x32_f16, the dropped
// lo*lo within 2^-22 of the term.  Scores: q and K rows scaled by their own
// powers of two, the score then times the two rows' units.  PV: V rows
// scaled the same way; each key's V unit folds into its p, and each query
// row's y = p * u_key stays below 2^14 through a running power of two that
// o carries (3 products a term instead of six bf16 ones: 2048-token prompt
// 194 -> 176 us with the scores' pieces, 173 -> 162 us with PV's).  A bf16
// cache needs one K/V piece (its values are exact) and q and P as three
// bf16 pieces (split3): three bf16 products each.  Tiles of 32 keys are
// staged into LDS as pieces:
//   K [KP][32 keys][D] 16-bit, 16-byte units XOR-swizzled by key (kt_off),
//     read as the A operand of S^T = K . Q^T: lane l key 16u + l%16,
//     elements 32s + 8(l/16) .. +7, Q^T in the same element order in
//     registers; fp32 and Q8 values: pieces 0 and 1 fp16 hi and lo, the
//     third slot the tile's 32 row units side by side (floats, f16_row_unit);
//   V [KP][32 keys][D] 16-bit, 16-byte units XOR-swizzled by key (vt_off),
//     read as V^T by ds_read_b64_tr_b16 as in attn_mfma_kernel: the A
//     operand of O^T += V^T . P^T, with P in the registers the score
//     accumulator left it in (key 16u + 4(l/16) + r of lane l, slot 4u + r);
//     fp32 and Q8 values as K (f16_vrow_unit).
// A tile's loads put keys 0..7 of one 16-byte column in lanes 0..7 and the
// next column in lanes 8..15 (128 contiguous bytes of each of 8 rows per 64
// lanes), so every LDS store of a piece is conflict-free too.
// D = 256 stages 100 KB (fp32 pieces) and runs one workgroup per CU.
template <int D, typename T, bool PAGED, int PW, bool PRE = false>
__global__ __launch_bounds__(64 * PW, PW == 4 && D < 256 ? 2 : 1)
void prefill_mfma16_kernel(PfArgs a) {
  static_assert(D == 64 || D == 128 || D == 256, "16-bit-piece prefill: D = 64, 128, 256");
  static_assert(PW == 4 || PW == 8, "4 or 8 waves");
  static_assert(!PRE || (sizeof(T) == 4 && !PAGED), "PRE: one instance per D and PW (pieces)");
  constexpr int NT = 64 * PW, QB = NT / 4;
  constexpr int KT = 32, KH = 2;
  constexpr int KP = sizeof(T) == 2 ? 1 : 3;  // staged pieces of K and V
  constexpr int KRB = 2 * D;                  // bytes of a staged K row
  constexpr int VRB = 2 * D;                  // bytes of a staged V row
  constexpr int QS = D / 32;                  // 32-element steps of the scores
  constexpr int DT = D / 16;
  constexpr int VW = KVT<T>::VW;              // elements per 16-byte load
  constexpr int CH = KT * D / VW;             // 16-byte chunks per tile (K or V)
  constexpr int CPT = (CH + NT - 1) / NT;
  constexpr bool Q8 = std::is_same<T, q8_t>::value;
  static_assert(CH % NT == 0 || CH < NT, "whole chunks per thread");
  static_assert((D / VW) % 4 == 0 && CH % 64 == 0 && 16 % VW == 0, "chunk mapping");
  // 8 waves (one workgroup a CU): two tile buffers where they fit, one
  // barrier a tile (a buffer is rewritten only after every wave has passed
  // the barrier that follows its last use); 4 waves: one buffer, so that two
  // workgroups share a CU's LDS
  constexpr int NBUF = PW == 8 && 2 * KP * KT * (KRB + VRB) <= 160 * 1024 ? 2 : 1;
  // KKV (pieces from the workspace, one buffer of each): a second K buffer
  // where it fits beside them, so that the next tile's K copies run under
  // the whole tile and its V copies under the next tile's scores
  constexpr bool KKV = PRE && NBUF == 1 && KP * KT * (2 * KRB + VRB) * (PW == 4 && D < 256 ? 2 : 1) <=
                                              160 * 1024;
  __shared__ __attribute__((aligned(16))) char kp_buf[KKV ? 2 : NBUF][KP * KT * KRB];
  __shared__ __attribute__((aligned(16))) char vp_buf[NBUF][KP * KT * VRB];

  const int G = a.nq / a.nkv;
  const int h = blockIdx.x % a.nkv;  // heads fastest: every XCD gets every head's share
  const int rest = (int)(blockIdx.x / a.nkv);
  const int sp = rest % a.nsplit;               // key split
  const int qb = a.nqb - 1 - rest / a.nsplit;  // latest rows (most keys) first
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g4 = lane >> 4;
  const int rows = a.M * G;
  const int r0 = qb * QB;
  const int rl = min(r0 + QB, rows) - 1;
  auto t0_of = [&](int m) {
    const int pos = a.pos0 + m;
    int t0 = (a.window > 0 && pos - a.window + 1 > 0) ? pos - a.window + 1 : 0;
    return t0 > a.N ? a.N : t0;
  };
  auto nn_of = [&](int m) { return a.pos0 + m + 1 < a.N ? a.pos0 + m + 1 : a.N; };
  const int kt_lo = t0_of(r0 / G);
  const int kt_hi = nn_of(rl / G);
  const int ntile_all = kt_hi > kt_lo ? (kt_hi - kt_lo + KT - 1) / KT : 0;
  // this split's tiles [tb0, tb0 + ntile) of the block's range
  const int tb0 = (int)((int64_t)sp * ntile_all / a.nsplit);
  const int ntile = (int)((int64_t)(sp + 1) * ntile_all / a.nsplit) - tb0;
  const int kt_s = kt_lo + tb0 * KT;  // this split's first key
  const int row = r0 + 16 * w + c16;
  const bool rv = row < rows;
  const int m = rv ? row / G : 0;
  const int g = rv ? row - m * G : 0;
  const int rt0 = rv ? t0_of(m) : 0, rnn = rv ? nn_of(m) : 0;
  const int64_t qoff = ((int64_t)m * a.nq + h * G + g) * a.dh;  // q and O rows of dh elements

  // Q^T pieces (B operand): lane l row c16, elements 32s + 8*g4 + e, scaled
  // by scale*log2(e) (base-2 scores).  Against a bf16 cache (KP = 1, exact
  // K) three bf16 pieces; against fp32 and Q8 values (KP = 3) two fp16
  // pieces of the row scaled by a power of two (split2h; the row's 4 lanes
  // share its largest |q|), as K: three products per score term instead of
  // six bf16 ones, and the scores take the q and K row units back.
  const float qsc = a.scale * kLog2e;
  [[maybe_unused]] bf16x8_t qh[QS], qm[QS], ql[QS];
  [[maybe_unused]] f16x8_t fqh[QS], fql[QS];
  [[maybe_unused]] float qunit = 1.f;
  float qx[QS][8];
#pragma unroll
  for (int s = 0; s < QS; ++s) {
    const float* qp = a.q + qoff + 32 * s + 8 * g4;
    const bool qin = rv && 32 * s + 8 * g4 < a.dh;  // zero padding past dh (a multiple of 8)
    const f32x4 x0 = qin ? *reinterpret_cast<const f32x4*>(qp) : f32x4{0.f, 0.f, 0.f, 0.f};
    const f32x4 x1 = qin ? *reinterpret_cast<const f32x4*>(qp + 4) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      qx[s][e] = x0[e] * qsc;
      qx[s][4 + e] = x1[e] * qsc;
    }
  }
  if constexpr (KP == 3) {
    float qm8 = 0.f;
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) qm8 = fmaxf(qm8, fabsf(qx[s][e]));
    const int qshift = f16_row_shift(max_xor32(max_xor16(qm8)));
    qunit = f16_row_unit(qshift);
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      uint32_t h4[4], l4[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) split2h(qx[s][e], qx[s][e + 1], qshift, h4[e / 2], l4[e / 2]);
      fqh[s] = __builtin_bit_cast(f16x8_t, u32x4{h4[0], h4[1], h4[2], h4[3]});
      fql[s] = __builtin_bit_cast(f16x8_t, u32x4{l4[0], l4[1], l4[2], l4[3]});
    }
  } else {
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      uint32_t h4[4], m4[4], l4[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) split3x2(qx[s][e], qx[s][e + 1], h4[e / 2], m4[e / 2], l4[e / 2]);
      qh[s] = __builtin_bit_cast(bf16x8_t, u32x4{h4[0], h4[1], h4[2], h4[3]});
      qm[s] = __builtin_bit_cast(bf16x8_t, u32x4{m4[0], m4[1], m4[2], m4[3]});
      ql[s] = __builtin_bit_cast(bf16x8_t, u32x4{l4[0], l4[1], l4[2], l4[3]});
    }
  }

  // tile loads: chunk c (16 bytes of the cache type) is key c%8 of its
  // key octet, column (c/8) % (D/VW) of the row, octet c / (8*D/VW).  KP = 3
  // (K split by rows, below): row-major, key c / (D/VW), column c % (D/VW),
  // so a row's D/VW chunks sit in consecutive lanes of one wave.
  constexpr int NCR = D / VW;  // chunks per row
  static_assert(KP != 3 || (NCR <= 64 && 64 % NCR == 0 && NT % NCR == 0), "rows within waves");
  auto chunk_of = [&](int c, int& key, int& e) {
    if constexpr (KP == 3) {
      key = c / NCR;
      e = VW * (c % NCR);
    } else {
      key = (c & 7) + 8 * (c / (8 * NCR));
      e = VW * ((c >> 3) % NCR);
    }
  };
  const T* Kb = reinterpret_cast<const T*>(a.k);
  const T* Vb = reinterpret_cast<const T*>(a.v);
  auto row_off = [&](int t, int64_t& soff) -> int64_t {
    return pf_row_off<D, T, PAGED>(a, h, t, soff);
  };
  // PRE: the tile's pieces straight from the split workspace into LDS, with
  // global_load_lds_dwordx4: lane l of a wave's load lands at the 16 bytes
  // base + 16*l of a 1 KB block (checked on the GPU), so lane l loads the
  // unit the swizzled layout keeps there (unit ch of key r at ch ^ f(r):
  // slot j holds unit j ^ f(r)).  No registers and no arithmetic per element.
  // The source is a wave-uniform row base (the tile's first key) plus a
  // 32-bit lane offset (key within the tile, clamped to the range's last
  // key, and its unit), so the loads take a scalar base and the per-tile
  // address arithmetic stays off the vector ALU.  The two pieces, then the
  // tile's 32 row units (128 bytes, dma4) to the start of the third piece
  // slot
  // (all 64 lanes: lanes 32..63 repeat the last key's unit into the unused
  // bytes 128..255 of the slot, so no lane is masked off)
  auto dunits = [&](int tk, char* buf, int kv) {
    const char* units = reinterpret_cast<const char*>(
        a.pieces + (((int64_t)kv * a.nkv + h) * 3 + 2) * a.R * D) + 4 * (int64_t)(tk - a.T0);
    const uint32_t lo = (uint32_t)(4 * min(min(lane, KT - 1), kt_hi - 1 - tk));
    dma4(units, lo, (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)(
                        buf + 2 * KT * (2 * D)));
  };
  auto dload = [&](int tk, char* kbuf, char* vbuf) {
    constexpr int UPR = D / 8;             // 16-byte units per row
    constexpr int KPB = 64 / UPR;          // keys per 1 KB block
    constexpr int BPP = KT / KPB;          // blocks per piece
    constexpr int NBL = 2 * 2 * BPP;       // blocks per tile (K, V; 2 pieces)
    const int r_in = lane / UPR, jpos = lane % UPR;
    const int lastr = kt_hi - 1 - tk;      // the range's last key, from the tile's first
    if (w < 2) dunits(tk, w ? vbuf : kbuf, w);
#pragma unroll
    for (int bi0 = 0; bi0 < NBL; bi0 += PW) {
      const int bi = bi0 + w;  // wave-uniform
      if (NBL % PW != 0 && bi >= NBL) break;
      const int kv = bi / (2 * BPP), rem = bi - kv * 2 * BPP;
      const int pc = rem / BPP, kb = rem - pc * BPP;
      const int r = kb * KPB + r_in;
      const int ch = jpos ^ (kv ? vt_f<D>(r) : kt_f<D>(r));
      const char* rows = reinterpret_cast<const char*>(
          a.pieces + ((((int64_t)kv * a.nkv + h) * 3 + pc) * a.R + (tk - a.T0)) * D);
      const uint32_t lo = (uint32_t)(min(r, lastr) * (2 * D) + 16 * ch);
      char* dst = (kv ? vbuf : kbuf) + pc * KT * (2 * D) + kb * 1024;
      dma16(rows, lo, (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst);
    }
  };
  // K (kv = 0) or V (kv = 1) of a tile alone: NL copies a wave (every wave
  // copies the units, the same bytes to the same place, so that the waves
  // count alike)
  constexpr int NL = 2 * (KT / (64 / (D / 8))) / PW + 1;
  auto dload1 = [&](int tk, char* buf, int kv) {
    constexpr int UPR = D / 8, KPB = 64 / UPR, BPP = KT / KPB;
    static_assert(!KKV || (2 * BPP) % PW == 0, "the same copies in every wave");
    const int r_in = lane / UPR, jpos = lane % UPR;
    const int lastr = kt_hi - 1 - tk;
    dunits(tk, buf, kv);
#pragma unroll
    for (int bi0 = 0; bi0 < 2 * BPP; bi0 += PW) {
      const int bi = bi0 + w;  // wave-uniform
      const int pc = bi / BPP, kb = bi - pc * BPP;
      const int r = kb * KPB + r_in;
      const int ch = jpos ^ (kv ? vt_f<D>(r) : kt_f<D>(r));
      const char* rows = reinterpret_cast<const char*>(
          a.pieces + ((((int64_t)kv * a.nkv + h) * 3 + pc) * a.R + (tk - a.T0)) * D);
      const uint32_t lo = (uint32_t)(min(r, lastr) * (2 * D) + 16 * ch);
      char* dst = buf + pc * KT * (2 * D) + kb * 1024;
      dma16(rows, lo, (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst);
    }
  };
  typename KVT<T>::vec kreg[CPT], vreg[CPT];
  [[maybe_unused]] float ksc[CPT], vsc[CPT];
  auto load_tile = [&](int tk) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + NT * i;
      if (CH < NT && c >= CH) break;
      int key, e;
      chunk_of(c, key, e);
      const int t = min(tk + key, kt_hi - 1);  // rows past the range: the last one (masked)
      int64_t soff = 0;
      const int64_t off = row_off(t, soff) + e;
      if constexpr (Q8) {
        ksc[i] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(a.k) + soff);
        vsc[i] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(a.v) + soff);
      }
      if (e < a.dh) {  // a padded launch: columns past the stored head dim read as 0
        kreg[i] = load16(Kb + off);
        vreg[i] = load16(Vb + off);
      } else {
        kreg[i] = typename KVT<T>::vec{};
        vreg[i] = typename KVT<T>::vec{};
      }
    }
  };
  // the chunk's values as KP pieces (K of fp32 and Q8 values: two fp16 of
  // the row scaled by a power of two, its unit in the third), 4 elements
  // (8 bytes) at a time
  auto store_tile = [&](char* kp_s, char* vp_s) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + NT * i;
      if (CH < NT && c >= CH) break;
      int key, e;
      chunk_of(c, key, e);
      float kx[VW], vx[VW];
      KVT<T>::unpack(kreg[i], kx);
      KVT<T>::unpack(vreg[i], vx);
      if constexpr (Q8) {  // code * s, the dequantized value
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          kx[j] *= ksc[i];
          vx[j] *= vsc[i];
        }
      }
      [[maybe_unused]] int kshift = 0, vshift = 0;
      if constexpr (KP == 3) {  // the K and V rows' scales: largest |x| over the row's NCR lanes
        float km = 0.f, vm = 0.f;
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          km = fmaxf(km, fabsf(kx[j]));
          vm = fmaxf(vm, fabsf(vx[j]));
        }
        kshift = f16_row_shift(group_max<NCR>(km));
        vm = group_max<NCR>(vm);
        vshift = f16_vrow_shift(vm);
        if (e == 0) {  // the tile's row units side by side in the third slot
          reinterpret_cast<float*>(kp_s + 2 * KT * KRB)[key] = f16_row_unit(kshift);
          reinterpret_cast<float*>(vp_s + 2 * KT * VRB)[key] = f16_vrow_unit(vm, vshift);
        }
      }
#pragma unroll
      for (int j4 = 0; j4 < VW; j4 += 4) {
        const int ej = e + j4;
        uint32_t kpc[KP][2], vpc[KP][2];  // 4 elements of each piece
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          if constexpr (KP == 3) {
            split2h(kx[j4 + j], kx[j4 + j + 1], kshift, kpc[0][j / 2], kpc[1][j / 2]);
            split2h(vx[j4 + j], vx[j4 + j + 1], vshift, vpc[0][j / 2], vpc[1][j / 2]);
          } else {  // exact bf16 values
            kpc[0][j / 2] = bf16_pair(kx[j4 + j], kx[j4 + j + 1]);
            vpc[0][j / 2] = bf16_pair(vx[j4 + j], vx[j4 + j + 1]);
          }
        }
        const int kofs = kt_off<D>(key, ej >> 3) + 8 * ((ej >> 2) & 1);
        const int vofs = vt_off<D>(key, ej >> 3) + 8 * ((ej >> 2) & 1);
#pragma unroll
        for (int p = 0; p < (KP == 3 ? 2 : 1); ++p) {  // the third piece holds the row's unit only
          *reinterpret_cast<u32x2*>(kp_s + p * KT * KRB + kofs) = u32x2{kpc[p][0], kpc[p][1]};
          *reinterpret_cast<u32x2*>(vp_s + p * KT * VRB + vofs) = u32x2{vpc[p][0], vpc[p][1]};
        }
      }
    }
  };

  f32x4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;

  // scores of the two 16-key halves of the tile at kp_s, smallest piece
  // products first; even and odd 32-element steps into separate
  // accumulators (four independent MFMA chains, added at the end)
  // piece products in the order they enter an accumulator, smallest first:
  // (K or V piece, q or P piece: 0 hi, 1 mid, 2 lo)
  constexpr int NPR = KP == 3 ? 6 : 3;
  // 32-element steps whose operands are read together, and 16-row V blocks
  // (d = 256: fewer, to stay in 256 registers)
  constexpr int SJ = D == 256 ? 1 : 2;
  constexpr int NDT = D == 256 ? 2 : (DT >= 4 ? 4 : DT);
  constexpr int PRK[6] = {KP == 3 ? 1 : 0, KP == 3 ? 2 : 0, 0, 1, 0, 0};
  constexpr int PRQ[6] = {KP == 3 ? 1 : 2, KP == 3 ? 0 : 1, KP == 3 ? 2 : 0, 0, 1, 0};
  // scores of the two 16-key halves of the tile at kp_s.  SJ 32-element
  // steps at a time: their staged K operands (both halves, every piece) are
  // read first, then the piece products go out piece by piece across the
  // accumulators (even and odd steps of each half), so that consecutive
  // matrix instructions are independent; each accumulator takes its
  // products in the same order as one at a time.  The two step parities are
  // added at the end.
  // KP = 3 (fp32 and Q8 values): K and q as two fp16 pieces each, three
  // products per term (lo*hi, hi*lo, hi*hi; the dropped lo*lo is within
  // 2^-22 of the term), then the q and K row units multiply each score.
  constexpr int FPK[3] = {1, 0, 0};
  constexpr int FPQ[3] = {0, 1, 0};
  auto scores = [&](const char* kp_s, f32x4 (&sacc)[KH]) {
    f32x4 sacc2[KH][2];
#pragma unroll
    for (int u = 0; u < KH; ++u) sacc2[u][0] = sacc2[u][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s0 = 0; s0 < QS; s0 += SJ) {
      if constexpr (KP == 3) {
        f16x8_t kk[SJ][KH][2];
#pragma unroll
        for (int j = 0; j < SJ; ++j)
#pragma unroll
          for (int u = 0; u < KH; ++u) {
            const char* kb = kp_s + kt_off<D>(16 * u + c16, 4 * (s0 + j) + g4);
#pragma unroll
            for (int p = 0; p < 2; ++p)
              kk[j][u][p] = *reinterpret_cast<const f16x8_t*>(kb + p * KT * KRB);
          }
#pragma unroll
        for (int t = 0; t < 3; ++t)
#pragma unroll
          for (int j = 0; j < SJ; ++j)
#pragma unroll
            for (int u = 0; u < KH; ++u) {
              f32x4& acc = sacc2[u][(s0 + j) & 1];
              acc = mfma_f16(kk[j][u][FPK[t]], FPQ[t] == 0 ? fqh[s0 + j] : fql[s0 + j], acc);
            }
      } else {
        bf16x8_t kk[SJ][KH][KP];
#pragma unroll
        for (int j = 0; j < SJ; ++j)
#pragma unroll
          for (int u = 0; u < KH; ++u) {
            const char* kb = kp_s + kt_off<D>(16 * u + c16, 4 * (s0 + j) + g4);
#pragma unroll
            for (int p = 0; p < KP; ++p)
              kk[j][u][p] = *reinterpret_cast<const bf16x8_t*>(kb + p * KT * KRB);
          }
#pragma unroll
        for (int t = 0; t < NPR; ++t)
#pragma unroll
          for (int j = 0; j < SJ; ++j)
#pragma unroll
            for (int u = 0; u < KH; ++u) {
              const bf16x8_t& qp = PRQ[t] == 0 ? qh[s0 + j] : PRQ[t] == 1 ? qm[s0 + j] : ql[s0 + j];
              f32x4& acc = sacc2[u][(s0 + j) & 1];
              acc = mfma_bf16(kk[j][u][PRK[t]], qp, acc);
            }
      }
    }
#pragma unroll
    for (int u = 0; u < KH; ++u) sacc[u] = sacc2[u][0] + sacc2[u][1];
    if constexpr (KP == 3) {
      // keys 16u + 4*g4 .. +3's units: floats 16u + 4*g4 .. of the third slot
      // (the q row's unit, the same for the row's every score, is the
      // softmax's: its max and exponent arguments take it)
#pragma unroll
      for (int u = 0; u < KH; ++u) {
        const f32x4 ku = *reinterpret_cast<const f32x4*>(kp_s + 2 * KT * KRB + 4 * (16 * u + 4 * g4));
#pragma unroll
        for (int r = 0; r < 4; ++r) sacc[u][r] *= ku[r];
      }
    }
  };
  // online softmax (base 2) of this lane's row over its 8 keys of the tile
  // at tk.  Lazy rescale, as in the decode kernel: the running max moves
  // only when a score exceeds it by more than kLazyMax (p <= 2^8 otherwise);
  // o and l always share the max they were formed with.  Leaves P^T (the
  // B operand's order: pv[4u + r] is key 16u + 4*g4 + r), the factor alpha
  // that o and l take before P is added (1 unless the max moved) and the
  // tile's row sum.
  // FULL (a std::integral_constant): every key of the tile is in every
  // row's range, so no key is masked and every probability is an exp.
  auto softmax = [&](auto FULL, const f32x4 (&sacc)[KH], int tk, float (&pv)[4 * KH],
                     float& alpha, bool& grow, int& gsh, float& ps) {
    constexpr bool full = decltype(FULL)::value;
    float sv[KH][4];
    float tmax = -INFINITY;
#pragma unroll
    for (int u = 0; u < KH; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = tk + 16 * u + 4 * g4 + r;
        sv[u][r] = (full || (t >= rt0 && t < rnn)) ? sacc[u][r] : -INFINITY;
        tmax = fmaxf(tmax, sv[u][r]);
      }
    // the scores over fp32 and Q8 values still lack the q row's unit qunit
    // (a power of two): tmax takes it, and each exponent argument as one fma,
    // s * qunit - m, rounded once as the difference of the scaled score was
    tmax = max_xor32(max_xor16(tmax)) * qunit;
    grow = tmax > m_run + kLazyMax;  // false while the row has no key (-inf)
    const float mn = grow ? fmaxf(m_run, tmax) : m_run;
    alpha = m_run == -INFINITY ? 1.f : exp2_hw(m_run - mn);  // exp2(0) = 1 exactly
    // floor(log2(1 / alpha)) (> 8, at most 1000) when a finite max moved
    gsh = (grow && m_run != -INFINITY) ? (int)fminf(floorf(mn - m_run), 1000.f) : 0;
    m_run = mn;
    ps = 0.f;
#pragma unroll
    for (int u = 0; u < KH; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        pv[4 * u + r] =
            (!full && sv[u][r] == -INFINITY) ? 0.f : exp2_hw(fmaf(sv[u][r], qunit, -m_run));
        ps += pv[4 * u + r];
      }
  };
  // V^T of the 16-row blocks dt0 .. dt0 + NDT - 1 (A operands of PV), piece
  // p of the staged tile at vp_s: two transposed reads per block
  auto read_vt = [&](const char* vp_s, int dt0, int p, auto& av) {
#pragma unroll
    for (int j = 0; j < NDT; ++j) {
      i16x4_t t2[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = (lane >> 2) + 16 * u;
        t2[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4_t*)(
                vp_s + p * KT * VRB + vt_off<D>(r, 2 * (dt0 + j) + ((lane & 3) >> 1)) +
                8 * (lane & 1)));
      }
      av[j][p] = __builtin_bit_cast(typename std::remove_reference<decltype(av[j][p])>::type,
                                    __builtin_shufflevector(t2[0], t2[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  // fp32 and Q8 values (KP = 3): PV takes y = p * u_key * 2^wsh as two fp16
  // pieces, u_key the key's V row unit (V's pieces are the row over u_key),
  // so that o = 2^wsh * sum p v.  wsh (per query row: this lane's column of
  // O^T) keeps y below 2^14: it follows the largest p * u_key of the row's
  // keys so far, and when the running max moves (o and l scaled by alpha)
  // it may grow by floor(log2(1 / alpha)), so that the unit follows o down.
  // Each term is then held to 2^-22 of itself, or to 2^-25 of the
  // row's unit 2^(14 - wsh) (2^-37 of its largest p * |v| term) below.
  constexpr int kNoShift = 1 << 20;  // no key yet (o = 0)
  [[maybe_unused]] int wsh = kNoShift;
  // o += P V over the tile at vp_s.  bf16 caches (exact V): P as three bf16
  // pieces, V^T of NDT 16-row blocks at a time, their operands first, then
  // the piece products piece by piece across the NDT accumulators (each in
  // the same order as one block at a time).  fp32 and Q8 values: y and V as
  // two fp16 pieces each, three products per term (lo*hi, hi*lo, hi*hi; the
  // dropped lo*lo is within 2^-22 of the term), as the scores.  gsh: the
  // softmax's floor(log2(1 / alpha)) when the running max moved, else 0.
  auto pv_acc = [&](const char* vp_s, const float (&pv)[4 * KH], int gsh) {
    if constexpr (KP == 3) {
      float z[4 * KH];  // p * u_key, u_key from the tile's units in the third slot
      float zt = 0.f;
#pragma unroll
      for (int u = 0; u < KH; ++u) {
        const f32x4 uk = *reinterpret_cast<const f32x4*>(vp_s + 2 * KT * VRB + 4 * (16 * u + 4 * g4));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          z[4 * u + r] = pv[4 * u + r] * uk[r];
          zt = fmaxf(zt, z[4 * u + r]);
        }
      }
      zt = max_xor32(max_xor16(zt));  // the row's 32 keys (its column's 4 lanes)
      const int ns = min(min(wsh + gsh, kNoShift), zt > 0.f ? f16_row_shift(zt) : kNoShift);
      if (__builtin_amdgcn_ballot_w64(ns != wsh) != 0) {  // o into the new unit (exact)
        const int dsh = ns - wsh;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[dt][i] = ldexpf(o[dt][i], dsh);
      }
      wsh = ns;
      uint32_t h4[4], l4[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) split2h(z[e], z[e + 1], ns, h4[e / 2], l4[e / 2]);
      const f16x8_t yh = __builtin_bit_cast(f16x8_t, u32x4{h4[0], h4[1], h4[2], h4[3]});
      const f16x8_t yl = __builtin_bit_cast(f16x8_t, u32x4{l4[0], l4[1], l4[2], l4[3]});
#pragma unroll
      for (int dt0 = 0; dt0 < DT; dt0 += NDT) {
        f16x8_t av[NDT][2];
        read_vt(vp_s, dt0, 0, av);
        read_vt(vp_s, dt0, 1, av);
#pragma unroll
        for (int t = 0; t < 3; ++t)
#pragma unroll
          for (int j = 0; j < NDT; ++j)
            o[dt0 + j] = mfma_f16(av[j][FPK[t]], FPQ[t] == 0 ? yh : yl, o[dt0 + j]);
      }
    } else {
      uint32_t ph4[4], pm4[4], pl4[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) split3x2(pv[e], pv[e + 1], ph4[e / 2], pm4[e / 2], pl4[e / 2]);
      const bf16x8_t ph = __builtin_bit_cast(bf16x8_t, u32x4{ph4[0], ph4[1], ph4[2], ph4[3]});
      const bf16x8_t pm = __builtin_bit_cast(bf16x8_t, u32x4{pm4[0], pm4[1], pm4[2], pm4[3]});
      const bf16x8_t pl = __builtin_bit_cast(bf16x8_t, u32x4{pl4[0], pl4[1], pl4[2], pl4[3]});
#pragma unroll
      for (int dt0 = 0; dt0 < DT; dt0 += NDT) {
        bf16x8_t av[NDT][KP];
#pragma unroll
        for (int p = 0; p < KP; ++p) read_vt(vp_s, dt0, p, av);
#pragma unroll
        for (int t = 0; t < NPR; ++t)
#pragma unroll
          for (int j = 0; j < NDT; ++j) {
            const bf16x8_t& pp = PRQ[t] == 0 ? ph : PRQ[t] == 1 ? pm : pl;
            o[dt0 + j] = mfma_bf16(av[j][PRK[t]], pp, o[dt0 + j]);
          }
      }
    }
  };
  // o and l take alpha, then l the tile's sum (two roundings, as the
  // running sums of the decode kernels)
  auto rescale = [&](float alpha, bool grow, float ps) {
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    }
    {
#pragma clang fp contract(off)
      l_run = l_run * alpha + ps;
    }
  };

  if constexpr (KKV) {
    // Iteration it: the scores read K(it) while K(it+1) is copied into the
    // other K buffer (last read by the scores of it-1, before the barrier
    // that ended it-1); PV reads V(it), copied at the end of it-1 under the
    // scores and softmax of it; V(it+1) is copied once every wave is past
    // PV(it).  Each wave counts its own copies: NL for K or V of a tile.
    if (ntile > 0) {
      dload(kt_s, kp_buf[0], vp_buf[0]);
      wait_vmcnt<0>();
      __syncthreads();
    }
    for (int it = 0; it < ntile; ++it) {
      const int tk = kt_s + it * KT;
      const bool more = it + 1 < ntile;
      if (more) dload1(tk + KT, kp_buf[(it + 1) & 1], 0);
      f32x4 sacc[KH];
      scores(kp_buf[it & 1], sacc);
      float pv[4 * KH];
      float alpha, ps;
      bool grow;
      int gsh;
      if (__builtin_amdgcn_ballot_w64(!(rv && tk >= rt0 && tk + KT <= rnn)) == 0)
        softmax(std::true_type{}, sacc, tk, pv, alpha, grow, gsh, ps);
      else
        softmax(std::false_type{}, sacc, tk, pv, alpha, grow, gsh, ps);
      rescale(alpha, grow, ps);
      // V(it) is in LDS (K(it+1), copied after it, may still be in flight)
      if (more)
        wait_vmcnt<NL>();
      else
        wait_vmcnt<0>();
      lds_barrier();
      pv_acc(vp_buf[0], pv, gsh);
      if (more) {
        lds_barrier();  // every wave is past PV(it)
        dload1(tk + KT, vp_buf[0], 1);
        wait_vmcnt<NL>();  // K(it+1) is in LDS (V(it+1) may still be in flight)
        lds_barrier();
      }
    }
  } else {
    if constexpr (PRE) {
      if (ntile > 0) dload(kt_s, kp_buf[0], vp_buf[0]);
      wait_vmcnt<0>();  // this wave's direct loads are in LDS
      __syncthreads();
    } else {
      if (ntile > 0) load_tile(kt_s);
    }
    for (int it = 0; it < ntile; ++it) {
      const int tk = kt_s + it * KT;
      const int bf = NBUF == 2 ? (it & 1) : 0;
      const char* kp_s = kp_buf[bf];
      const char* vp_s = vp_buf[bf];
      if constexpr (PRE) {
        // the other buffer was last read in the previous tile, which every
        // wave finished before the barrier that ended it
        if constexpr (NBUF == 2)
          if (it + 1 < ntile) dload(tk + KT, kp_buf[bf ^ 1], vp_buf[bf ^ 1]);
      } else {
        store_tile(kp_buf[bf], vp_buf[bf]);
        __syncthreads();
        if (it + 1 < ntile) load_tile(tk + KT);  // in flight while this tile is used
      }
      f32x4 sacc[KH];
      scores(kp_s, sacc);
      float pv[4 * KH];
      float alpha, ps;
      bool grow;
      int gsh;
      // interior tile: every row of the wave attends all of its keys
      if (__builtin_amdgcn_ballot_w64(!(rv && tk >= rt0 && tk + KT <= rnn)) == 0)
        softmax(std::true_type{}, sacc, tk, pv, alpha, grow, gsh, ps);
      else
        softmax(std::false_type{}, sacc, tk, pv, alpha, grow, gsh, ps);
      rescale(alpha, grow, ps);
      pv_acc(vp_s, pv, gsh);
      if constexpr (PRE) {
        if constexpr (NBUF == 1) {
          __syncthreads();  // every wave is done with the buffer
          if (it + 1 < ntile) dload(tk + KT, kp_buf[0], vp_buf[0]);
        }
        wait_vmcnt<0>();  // this wave's direct loads of the next tile are in LDS
        __syncthreads();
      } else {
        if constexpr (NBUF == 1) __syncthreads();  // the tile's LDS is rewritten next
      }
    }
  }
  l_run = sum_xor32(sum_xor16(l_run));
  if constexpr (KP == 3) {  // o back from 2^wsh * sum p v (a power of two; no key: o = 0)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dt][i] = ldexpf(o[dt][i], -wsh);
  }
  if (rv && a.nsplit > 1) {  // the split's partial: unnormalised o, max in natural units, sum
    const int64_t ps = ((int64_t)m * a.nq + h * G + g) * a.nsplit + sp;
    float* po = a.part_o + ps * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(po + 16 * dt + 4 * g4) = o[dt];
    if (g4 == 0) {
      a.part_ml[2 * ps] = m_run == -INFINITY ? -INFINITY : m_run * kLn2;
      a.part_ml[2 * ps + 1] = l_run;
    }
  } else if (rv) {
    const float inv = l_run > 0.f ? 1.f / l_run : 0.f;  // no key: O = 0 (gemm.h:438)
    float* orow = a.o + qoff;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      if (16 * dt + 4 * g4 < a.dh) *reinterpret_cast<f32x4*>(orow + 16 * dt + 4 * g4) = o[dt] * inv;
  }
}

// Log-sum-exp combine of the chunk partials of split-K launches.  Grid
// (slots, P/pairs), the slot fastest: workgroup id % 8 is the XCD, so where
// the attention launch ran a slot's chunks on XCD slot % 8 (its slot index
// fastest over a multiple of 8 slots) the combine reads their partials from
// that XCD's L2 (32q/8kv/d128 fp32 at n = 4097: step 12.8 -> 12.1 us).  A
// workgroup takes `pairs` output pairs of one head of a
// slot (pairs divides D) with 256/pairs threads per pair, thread phase ph
// folding chunks ph, ph + phases, ...  The chunk weights e^(m_c - M) and the
// sum L are computed once per workgroup into LDS; the first round of o
// loads is issued before that, so a whole combine costs about one memory
// round trip when phases * kCombRound covers the chunks (comb_pairs picks
// the pairs so: 64 pairs of 4 phases up to 32 chunks, 16 pairs of 16 phases
// from 65).  Slots whose sequence has a single chunk were written by the
// attention kernel itself.
struct CombArgs {
  const float* part_o;
  const float* part_ml;
  const float* qrot;
  float* o;
  float* q_out;
  const int32_t* seq_lens;
  const int32_t* pos_arr;
  int nq, nkv, gh, nsub, d, nchunks, chunk, window, rope;
  int paged;  // 2: of Q8 rows
  int fold;  // the attention launch folded in a new token (its chunks tile n - 1 rows)
  int dh;    // head dim as stored (d: the partials' padded head dim)
  // prefill rows (AttnArgs::pf): row b at pos0 + b of a cache of n rows; dyn: n
  // is AttnArgs::dyn_span and pos0 dyn_likely (shared fields, so that the
  // arguments stay within two 64-byte lines: the first loads wait for each, 0.14
  // us a step of 13 sequences)
  int pf, pos0, n;
  int pairs;        // combine_kernel: output pairs per workgroup (16, 32 or 64)
  int dyn, nseq;    // AttnArgs::dyn: the chunk from the sequences' lengths
};
static_assert(sizeof(CombArgs) <= 128, "two lines");

// Chunks of sequence b of a per-sequence launch (a paged batch, or prefill
// rows), as the attention kernel derives them.
__device__ __forceinline__ int comb_chunks(const CombArgs& a, int b) {
  int n, pos;
  int lo = 0;
  if (a.pf) {
    pos = a.pos0 + b;
    n = pos + 1 < a.n ? pos + 1 : a.n;
    // prefill rows with key ranges: seq_lens is key_lo, pos_arr key_hi
    if (a.pos_arr) n = max(0, min(a.pos_arr[b], a.n));
    if (a.seq_lens) lo = a.seq_lens[b];
  } else {
    n = a.seq_lens[b];
    pos = a.pos_arr ? a.pos_arr[b] : n - 1;
  }
  int t0 = (a.window > 0 && pos - a.window + 1 > 0) ? pos - a.window + 1 : 0;
  t0 = max(t0, lo);
  if (t0 > n) t0 = n;
  int span = (a.fold ? n - 1 : n) - t0;
  int chunk = a.chunk;
  if (a.dyn) {
    span = min(span, a.n);
    const SeqLen first = seq_len(a.seq_lens, a.pos_arr, (int)(threadIdx.x & 63), a.nseq);
    chunk = paged_chunk(a.seq_lens, a.pos_arr, first, a.nseq, a.window, a.fold, a.n,
                        a.nkv * a.nsub, a.dyn, a.paged == 2);
  }
  const int nch = span > 0 ? (span + chunk - 1) / chunk : (a.fold ? 1 : 0);
  return nch > a.nchunks ? a.nchunks : nch;
}

constexpr int kCombThreads = 256;
constexpr int kCombPairs = 64;                          // most pairs per workgroup
constexpr int kCombRound = 8;                           // o loads in flight per thread

// Pairs per combine workgroup for nch chunks: the fewest phases (threads per
// pair) whose one round of kCombRound loads each covers the chunks, at most
// 16 (8q/2kv/d512, 128 chunks per KV head: 6.2 us on 64 pairs of 4 phases).
__host__ __device__ constexpr int comb_pairs(int nch) {
  int ph = 4;
  while (ph < 16 && ph * kCombRound < nch) ph *= 2;
  return kCombThreads / ph;
}
constexpr int kMaxChunks = 4096;

// LDS of one combine workgroup, in floats: the chunk weights and sums of
// the launch's chunk count, the phases' partial sums and L.
__host__ __device__ constexpr int comb_lds_floats(int nchunks) { return 2 * nchunks + kCombThreads + 4; }

// Outputs yb * pairs .. of slot `slot`; csm: comb_lds_floats floats.
__device__ __forceinline__ void combine_slot(const CombArgs& a, int slot, int yb, float* csm) {
  float* wts = csm;                  // [nchunks] m_c, then the chunk weight e^(m_c - M)
  float* lsv = csm + a.nchunks;      // [nchunks] l_c
  float* pacc = lsv + a.nchunks;     // [kCombThreads]
  float& s_l = pacc[kCombThreads];   // L = sum_c e^(m_c - M) l_c
  const int P = a.gh * a.d;
  const int pairs = a.pairs, phases = kCombThreads / pairs;
  const int pb = yb * pairs;
  const int t = threadIdx.x;
  const int rows = a.nkv * a.nsub;  // slots per sequence
  const int b = slot / rows, y = slot - b * rows;
  const int pl = t % pairs, ph = t / pairs;
  const int pair = pb + pl;  // < P: P is a multiple of 64
  const int g = pb / a.d;    // one head per workgroup
  const float* po = a.part_o + (int64_t)slot * a.nchunks * P + pair;
  const float* pml = a.part_ml + (int64_t)slot * a.nchunks * a.gh * 2 + 2 * g;
  // The first round of o loads and wave 0's first statistics go out before
  // this sequence's chunk count is known (paged: it needs seq_lens, another
  // round trip): they stay within the launch's nchunks slots of the
  // workspace, and only chunks below the count are used.
  // dyn: within the likely chunks, since a bound for any lengths is far more than
  // most batches of several rounds have (Q8 16q/2kv/d128, 63 sequences of 1000 .. 9000 rows at 768
  // rows a chunk: step 58.1 -> 46.4 us)
  const int spec = a.dyn ? a.pos0 : a.nchunks;
  float ov[kCombRound];
#pragma unroll
  for (int u = 0; u < kCombRound; ++u)
    ov[u] = po[(int64_t)min(ph + phases * u, spec - 1) * P];
  float m1 = -INFINITY, l1 = 0.f;
  if (t < 64) {
    const int c1 = min(t, a.nchunks - 1);
    m1 = pml[(int64_t)c1 * a.gh * 2];
    l1 = pml[(int64_t)c1 * a.gh * 2 + 1];
  }
  // this sequence's chunk count, as the attention kernel derives it
  const int nch = a.paged || a.pf ? comb_chunks(a, b) : a.nchunks;
  if (nch <= 1) return;  // uniform over the workgroup
  if (t < 64) {  // wave 0: chunk weights and L of head g
    float mloc = -INFINITY;
    for (int cc = t; cc < nch; cc += 64) {
      const float m = cc == t ? m1 : pml[(int64_t)cc * a.gh * 2];
      wts[cc] = m;
      lsv[cc] = cc == t ? l1 : pml[(int64_t)cc * a.gh * 2 + 1];
      mloc = fmaxf(mloc, m);
    }
    const float M = wave_reduce<true>(mloc);
    float lloc = 0.f;
    for (int cc = t; cc < nch; cc += 64) {  // the lane's own LDS entries
      // a prefill row no split attended: M = -inf, weights 0, O = 0 below
      const float wgt = M == -INFINITY ? 0.f : softmax_exp(wts[cc] - M);
      wts[cc] = wgt;
      lloc = fmaf(wgt, lsv[cc], lloc);
    }
    const float Ls = wave_reduce<false>(lloc);
    if (t == 0) s_l = Ls;
  }
  __syncthreads();
  float acc = 0.f;
#pragma unroll
  for (int u = 0; u < kCombRound; ++u) {
    const int cc = ph + phases * u;
    if (cc < nch) acc = fmaf(wts[cc], cc < spec ? ov[u] : po[(int64_t)cc * P], acc);
  }
  for (int c0 = ph + phases * kCombRound; c0 < nch; c0 += phases * kCombRound) {
#pragma unroll
    for (int u = 0; u < kCombRound; ++u)
      ov[u] = po[(int64_t)min(c0 + phases * u, nch - 1) * P];
#pragma unroll
    for (int u = 0; u < kCombRound; ++u) {
      const int cc = c0 + phases * u;
      if (cc < nch) acc = fmaf(wts[cc], ov[u], acc);
    }
  }
  pacc[t] = acc;
  __syncthreads();
  if (ph == 0) {
    float o = acc;
    for (int q2 = 1; q2 < phases; ++q2) o += pacc[q2 * pairs + pl];
    const int G = a.nq / a.nkv;
    const int h = y / a.nsub, sub = y - h * a.nsub;
    const int64_t oi = out_index((int64_t)b * a.nq + h * G + sub * a.gh, pair, a.d, a.dh);
    if (oi >= 0) {
      a.o[oi] = s_l > 0.f ? o / s_l : 0.f;
      if (a.rope && a.q_out) a.q_out[oi] = a.qrot[(int64_t)slot * P + pair];
    }
  }
}

__global__ __launch_bounds__(kCombThreads) void combine_kernel(CombArgs a) {
  extern __shared__ float csm[];
  combine_slot(a, blockIdx.x, blockIdx.y, csm);
}

// The merge for a few chunks per slot (R >= nchunks, R <= 64), one wave per
// 64 output pairs of one head, with no LDS and no barrier: lane c holds chunk c's (m, l), DPP
// reductions give the max M and L = sum_c e^(m_c - M) l_c, and every lane
// sums its pair over the chunks with the weights broadcast by readlane.
// All R >= nchunks o loads and the statistics go out at once, before this
// sequence's chunk count is known (paged: it needs seq_lens): they stay
// within the launch's nchunks slots of the workspace, and only chunks below
// the count are used.  Grid (slots, P/threads), the slot fastest, as
// combine_kernel's.
constexpr int kCombWaveThreads = 256;
template <int R>
__device__ __forceinline__ void combine_wave_slot(const CombArgs& a, int slot, int pair) {
  const int P = a.gh * a.d;
  const int lane = threadIdx.x & 63;
  const int g = __builtin_amdgcn_readfirstlane(pair / a.d);  // d % 64 == 0: one head per wave
  const int rows = a.nkv * a.nsub;  // slots per sequence
  const int b = slot / rows, y = slot - b * rows;
  const float* po = a.part_o + (int64_t)slot * a.nchunks * P + pair;
  const float* pml = a.part_ml + (int64_t)slot * a.nchunks * a.gh * 2 + 2 * g;
  float ov[R];
#pragma unroll
  for (int u = 0; u < R; ++u) ov[u] = po[(int64_t)min(u, a.nchunks - 1) * P];
  const int cl = min(lane, a.nchunks - 1);
  const float mc = pml[(int64_t)cl * a.gh * 2], lc = pml[(int64_t)cl * a.gh * 2 + 1];
  // this sequence's chunk count, as the attention kernel derives it
  const int nch = a.paged || a.pf ? comb_chunks(a, b) : a.nchunks;
  if (nch <= 1) return;  // uniform over the workgroup
  const bool live = lane < nch;
  const float M = wave_reduce<true>(live ? mc : -INFINITY);
  // a slot whose chunks all saw no key (max -inf) gets O = 0, as in combine_kernel
  const float wc = live && M != -INFINITY ? softmax_exp(mc - M) : 0.f;
  const float L = wave_reduce<false>(live ? wc * lc : 0.f);
  float acc = 0.f;
#pragma unroll
  for (int u = 0; u < R; ++u)
    if (u < nch) acc = fmaf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(wc), u)), ov[u], acc);
  const int G = a.nq / a.nkv;
  const int h = y / a.nsub, sub = y - h * a.nsub;
  const int64_t oi = out_index((int64_t)b * a.nq + h * G + sub * a.gh, pair, a.d, a.dh);
  if (oi >= 0) {
    a.o[oi] = L > 0.f ? acc / L : 0.f;
    if (a.rope && a.q_out) a.q_out[oi] = a.qrot[(int64_t)slot * P + pair];
  }
}

template <int R>
__global__ __launch_bounds__(kCombWaveThreads) void combine_wave_kernel(CombArgs a) {
  // (the pair is below P: blockDim divides P)
  combine_wave_slot<R>(a, blockIdx.x, blockIdx.y * blockDim.x + threadIdx.x);
}

// The prefill's key-split merge: slot s = (token, q head) of one head, P = D
// partial outputs over R >= nchunks splits.  A wave takes 64V consecutive
// outputs of one slot (V = 4 at D % 256 == 0, 2 at D % 128 == 0, else 1), so
// a 2048-token prompt of 8 q heads at d = 256 runs 16384 waves instead of
// 65536; the arithmetic and its order are combine_wave_kernel's (lane c
// holds split c's (m, l), DPP reductions give M and L, the weights reach
// every lane by readlane), so the outputs are the same bits.  Four waves a
// workgroup, consecutive units (slot, 64V-span); units past the last exit.
template <int V>
__device__ __forceinline__ void load_v(const float* p, float* x) {
  if constexpr (V == 4) {
    const f32x4 t = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = t[e];
  } else if constexpr (V == 2) {
    const f32x2 t = *reinterpret_cast<const f32x2*>(p);
    x[0] = t[0];
    x[1] = t[1];
  } else {
    x[0] = *p;
  }
}
// SOME: rows may have fewer splits than the launch, or be done (prefill_tile.hpp,
// block_splits): the statistics first, then the partials that count.
template <int R, int V, bool SOME = false>
__global__ __launch_bounds__(kCombWaveThreads) void combine_rows_kernel(CombArgs a, int64_t units) {
  const int D = a.d;
  const int spans = D / (64 * V);
  const int64_t unit = (int64_t)blockIdx.x * (kCombWaveThreads / 64) + (threadIdx.x >> 6);
  if (unit >= units) return;  // wave-uniform
  const int lane = threadIdx.x & 63;
  const int64_t slot = unit / spans;
  const int pair = (int)(unit - slot * spans) * 64 * V + V * lane;
  const float* po = a.part_o + slot * a.nchunks * D + pair;
  const float* pml = a.part_ml + slot * a.nchunks * 2;
  float ov[R][V];
  if constexpr (!SOME) {
#pragma unroll
    for (int u = 0; u < R; ++u) load_v<V>(po + (int64_t)min(u, a.nchunks - 1) * D, ov[u]);
  }
  const int cl = min(lane, a.nchunks - 1);
  const f32x2 ml = *reinterpret_cast<const f32x2*>(pml + 2 * cl);
  int nch = a.nchunks;
  if constexpr (SOME) {
    if (__int_as_float(__builtin_amdgcn_readlane(__float_as_int(ml[1]), 0)) < 0.f) return;
    // (splits without a key, the ones past a block's among them, weigh nothing and come
    // last but for a row's own: those before them have finite partials)
    nch = 64 - __builtin_clzll(__builtin_amdgcn_ballot_w64(lane < nch && ml[1] != 0.f) | 1ull);
#pragma unroll
    for (int u = 0; u < R; ++u) load_v<V>(po + (int64_t)min(u, nch - 1) * D, ov[u]);
  }
  const bool live = lane < nch;
  const float M = wave_reduce<true>(live ? ml[0] : -INFINITY);
  const float wc = live && M != -INFINITY ? softmax_exp(ml[0] - M) : 0.f;
  const float L = wave_reduce<false>(live ? wc * ml[1] : 0.f);
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
#pragma unroll
  for (int u = 0; u < R; ++u)
    if (u < nch) {
      const float wu = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wc), u));
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(wu, ov[u][e], acc[e]);
    }
  float o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = L > 0.f ? acc[e] / L : 0.f;
  if (a.dh == D) {
    float* dst = a.o + slot * D + pair;
    if constexpr (V == 4) {
      *reinterpret_cast<f32x4*>(dst) = f32x4{o[0], o[1], o[2], o[3]};
    } else if constexpr (V == 2) {
      *reinterpret_cast<f32x2*>(dst) = f32x2{o[0], o[1]};
    } else {
      *dst = o[0];
    }
  } else {  // a padded launch: the stored head dim's outputs only
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (pair + e < a.dh) a.o[slot * a.dh + pair + e] = o[e];
  }
}

// The softmax weights of a scored launch, summed over the query heads of each KV
// head and added to acc: w = 2^(s - M) / L, M and L the merge of a head's chunk
// statistics.  Thread: one row, its heads' scores side by side; grid (rows, KV
// heads, sequences).  The sum runs over the heads in order, by one thread.
struct WeightArgs {
  CombArgs c;
  const float* scores;
  const float* stats;
  float* acc;
  int32_t* slot_pos;
  const int32_t* block_table;
  int64_t sc_rows;
  int n, t0, pos, max_blocks, page_shift, acc_cap, fresh;
  int sc_span;  // AttnArgs::sc_span
  int blocked;  // the scores in the matrix-core kernel's order
};
constexpr int kWeightThreads = 256;
constexpr int kWeightAhead = 8;  // heads whose scores a thread has in flight through the merge

// Rows kWeightThreads * rb .. of (sequence b, KV head h).  A short chain of loads (the
// statistics, the scores, the page's number and the sum that it leads to) bounds a block,
// so they go out together; us a step with weights, one after the other against
// together (32q/8kv/d128): 16384 bf16 rows 20.4 -> 20.0, 301 fp32 rows 10.6 -> 10.2; 131072
// rows of 64q/8kv 130 -> 126.  (Scores read a unit of 4 rows a lane, and turned in LDS, are
// whole lines a load, and 1 us slower: a block's next waits were not hidden.)
// wsm: 2 * G floats.
__device__ __forceinline__ void weigh_rows(const WeightArgs& w, int rb, int h, int b, float* wsm) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int G = w.c.nq / w.c.nkv, gh = w.c.gh;
  const bool paged = w.c.paged != 0;
  int n = w.n, t0 = w.t0, pos = w.pos, nch = w.c.nchunks;
  if (paged) {
    n = w.c.seq_lens[b];
    pos = w.c.pos_arr ? w.c.pos_arr[b] : n - 1;
    t0 = (w.c.window > 0 && pos - w.c.window + 1 > 0) ? pos - w.c.window + 1 : 0;
    if (t0 > n) t0 = n;
    nch = comb_chunks(w.c, b);
  }
  const int span = min(n - t0, w.sc_span);
  const int row0 = rb * kWeightThreads;
  auto index = [&](int t) -> int64_t {
    if (!paged) return (int64_t)h * w.acc_cap + t;
    const int64_t blk = w.block_table[(int64_t)b * w.max_blocks + (t >> w.page_shift)];
    return ((blk * w.c.nkv + h) << w.page_shift) + (t & ((1 << w.page_shift) - 1));
  };
  // a fresh row outside the range (before its window, whose start is n at most, or past
  // the bound of the lengths)
  if (w.fresh && n > 0 && (n - 1 < t0 || n - 1 >= t0 + span) && rb == 0 && tid == 0) {
    const int64_t i = index(n - 1);
    w.acc[i] = 0.f;
    if (w.slot_pos) w.slot_pos[i] = pos;
  }
  if (row0 >= span) return;
  const int slot0 = b * w.c.nkv * w.c.nsub + h * w.c.nsub;
  const int row = row0 + tid, t = t0 + row;
  const bool in = row < span, set = w.fresh && t == n - 1;
  const float* s = w.scores + ((int64_t)b * w.c.nkv + h) * w.sc_rows * G;
  const bool quads = !w.blocked && (G & 3) == 0;
  const float* x = s + (w.blocked ? (int64_t)(row & ~3) * G + (row & 3) : (int64_t)row * G);
  const int step = w.blocked ? 4 : 1;
  float ahead[kWeightAhead];
#pragma unroll
  for (int g = 0; g < kWeightAhead; g += 4) {
    if (quads) {
      const f32x4 y = in && g < G ? *reinterpret_cast<const f32x4*>(x + g) : f32x4{};
#pragma unroll
      for (int e = 0; e < 4; ++e) ahead[g + e] = y[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) ahead[g + e] = in && g + e < G ? x[step * (g + e)] : 0.f;
    }
  }
  const int64_t i = in ? index(t) : 0;
  const float old = in && !set ? w.acc[i] : 0.f;
  float *mx = wsm, *inv = wsm + G;
  for (int g = tid >> 6; g < G; g += kWeightThreads / 64) {  // a wave a head
    const float* st = w.stats + ((int64_t)(slot0 + g / gh) * w.c.nchunks * gh + g % gh) * 2;
    auto ml = [&](int c) { return *reinterpret_cast<const f32x2*>(st + (int64_t)c * gh * 2); };
    const f32x2 first = lane < nch ? ml(lane) : f32x2{-INFINITY, 0.f};
    float m = first[0], l = 0.f;
    for (int c = lane + 64; c < nch; c += 64) m = fmaxf(m, ml(c)[0]);
    m = group_max<64>(m);
    for (int c = lane; c < nch; c += 64) {
      const f32x2 x = c == lane ? first : ml(c);
      l += x[0] == -INFINITY ? 0.f : x[1] * exp2_hw(x[0] - m);
    }
    l = group_sum<64>(l);
    if (lane == 0) {
      mx[g] = m;
      inv[g] = 1.f / l;
    }
  }
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int g = 0; g < kWeightAhead; ++g)
    if (g < G) sum = fmaf(exp2_hw(ahead[g] - mx[g]), inv[g], sum);
  if (in) {
#pragma unroll 4
    for (int g = kWeightAhead; g < G; ++g) sum = fmaf(exp2_hw(x[step * g] - mx[g]), inv[g], sum);
  }
  if (!in) return;
  w.acc[i] = set ? sum : old + sum;
  if (set && w.slot_pos) w.slot_pos[i] = pos;
}
__global__ __launch_bounds__(kWeightThreads) void attn_weights_kernel(WeightArgs w) {
  extern __shared__ float wsm[];
  weigh_rows(w, blockIdx.x, blockIdx.y, blockIdx.z, wsm);
}

// The merge of a split launch and its weights, side by side in one launch (neither
// needs the other): workgroups below ncomb merge as combine_wave_kernel<R> or, R = 0,
// combine_kernel, the others weigh.  us a pass, two launches against one: 16001 bf16
// rows of 32q/8kv/d128 25.1 against 22.6; 13 paged sequences, Q8, 27.2 against 22.9 (now
// 20.0 and 23.4).
template <int R>
__global__ __launch_bounds__(kCombThreads) void combine_weights_kernel(WeightArgs w, int ncomb,
                                                                       int slots) {
  static_assert(kCombThreads == kWeightThreads && kCombThreads == kCombWaveThreads, "one block size");
  extern __shared__ float csm[];
  const int id = blockIdx.x;
  if (id < ncomb) {  // the slot fastest
    const int slot = id % slots, yb = id / slots;
    if constexpr (R > 0) {
      const int pair = yb * kCombThreads + threadIdx.x;
      if (pair < w.c.gh * w.c.d) combine_wave_slot<R>(w.c, slot, pair);  // (whole waves: 64 | P)
    } else {
      combine_slot(w.c, slot, yb, csm);
    }
    return;
  }
  const int i = id - ncomb, h = i % w.c.nkv;
  const int nb = (int)((w.sc_rows + kWeightThreads - 1) / kWeightThreads);
  const int rb = i / w.c.nkv % nb, b = i / w.c.nkv / nb;
  weigh_rows(w, rb, h, b, csm);
}

__global__ void vexp_kernel(const float* x, float* y, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) y[i] = softmax_exp(x[i]);
}

// The probabilities' exponential as the kernels take it: the natural-units
// argument scaled to base 2 (one fp32 rounding), then v_exp_f32.
__global__ void prob_exp_kernel(const float* x, float* y, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) y[i] = exp2_hw(x[i] * kLog2e);
}

__global__ void zero_kernel(float* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) p[i] = 0.f;
}

// ---------------------------------------------------------------------------
// Host side.

constexpr int kMaxChunk = 2048;
constexpr int kMaxSlots = 1 << 16;  // combine grid y: (sequence, head group) pairs per launch

// Process-wide settings (molot_hip_set_*): atomics, so a setter racing with
// launches on other host threads is well defined; a launch reads each once.
std::atomic<int> g_split_chunk{0};  // tokens per chunk, 0 = automatic
std::atomic<int> g_wgs_per_cu{0};   // workgroups per CU, 0 = the plan's own
std::atomic<int> g_dynamic{1};      // block order: 1 = claimed by waves as they free up, 0 = fixed

}  // namespace
namespace molot_host {
std::atomic<int> g_bf16_mfma{1};
std::atomic<int> g_merge{-1};
std::recursive_mutex g_launch_mu;
}  // namespace molot_host
namespace {
using namespace molot_host;

// Launch profiling (off by default): while on, every attention launch
// outside graph capture goes through hipExtLaunchKernelGGL with a start and
// a stop event per kernel, which HIP stamps from the dispatch itself (the
// kernel's execution, without the gap before it).  molot_hip_profile_end()
// waits for the events and returns the summed durations.
// (g_launch_mu guards the records.)
struct ProfRec {
  hipEvent_t a0, a1, c0, c1;  // attention kernel, combine kernel
  bool combine;
};
bool g_prof_on = false;
int g_prof_cap = 0;
std::vector<ProfRec> g_prof;

bool prof_active(void* stream) {
  if (!g_prof_on) return false;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing((hipStream_t)stream, &cap) != hipSuccess) return false;
  return cap == hipStreamCaptureStatusNone && (int)g_prof.size() < g_prof_cap;
}

hipEvent_t prof_event() {
  hipEvent_t e = nullptr;
  if (hipEventCreate(&e) != hipSuccess) return nullptr;
  return e;
}

void prof_destroy(ProfRec& r) {
  for (hipEvent_t e : {r.a0, r.a1, r.c0, r.c1})
    if (e) (void)hipEventDestroy(e);
}

struct WsKey {
  int dev;
  void* stream;
  bool operator<(const WsKey& o) const {
    return dev != o.dev ? dev < o.dev : stream < o.stream;
  }
};
// Per-(device, stream) workspace of the split-K partials, grown on demand.
// Layout: [u64 ctr[kMaxSlots] | partials].  The arrival words of the
// in-launch merge are zeroed once, when the buffer is allocated (a fill
// kernel on the stream, ordered before any launch that uses them), and
// every launch leaves them at zero.  The partials are filled and read
// within a step (by the attention kernel, or by it and the combine kernel
// next on the same stream), so they need no clearing and hold nothing
// between steps.  An outgrown buffer is retired, never freed: a graph
// captured earlier on the stream still points at it.
constexpr size_t kCtrBytes = sizeof(unsigned long long) * (size_t)kMaxSlots;
struct WsBuf {
  void* ptr = nullptr;
  size_t bytes = 0;  // partials
};
std::mutex g_ws_mu;
std::map<WsKey, WsBuf> g_ws;
std::vector<void*> g_retired;

__global__ void zero_kernel(float* p, int64_t n);
bool xcd_map_ok(int dev);

// Allocates `want` bytes, or where there is no memory for them the `bytes` that the call
// needs; *got is the size.  A failure is the call's status, and not left for the next
// launch's hipGetLastError.
hipError_t grow(void** p, size_t bytes, size_t want, size_t* got) {
  *got = want;
  hipError_t e = hipMalloc(p, want);
  if (e != hipSuccess) (void)hipGetLastError();
  if (e == hipErrorOutOfMemory && want > bytes) {
    *got = bytes;
    e = hipMalloc(p, bytes);
    if (e != hipSuccess) (void)hipGetLastError();
  }
  return e;
}

}  // namespace
int molot_host::workspace(void* stream, size_t bytes, unsigned long long** ctr, void** out) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return (int)e;
  std::lock_guard<std::mutex> lk(g_ws_mu);
  WsBuf& w = g_ws[WsKey{dev, stream}];
  if (!w.ptr || w.bytes < bytes) {
    // a graph being captured cannot allocate: the caller sizes the
    // workspace with one launch of the shape before capturing
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    e = hipStreamIsCapturing((hipStream_t)stream, &cap);
    if (e != hipSuccess) return (int)e;
    if (cap != hipStreamCaptureStatusNone) return MOLOT_ENOWS;
    (void)xcd_map_ok(dev);  // the one-time dispatch check, outside any capture
    const size_t want = std::max(grown_bytes(bytes, w.bytes, SIZE_MAX), (size_t)1 << 20);
    size_t got = 0;
    void* p = nullptr;
    e = grow(&p, kCtrBytes + bytes, kCtrBytes + want, &got);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(zero_kernel, dim3((unsigned)(kCtrBytes / 4 / 256)), dim3(256), 0,
                       (hipStream_t)stream, reinterpret_cast<float*>(p), (int64_t)(kCtrBytes / 4));
    e = hipGetLastError();
    if (e != hipSuccess) {
      (void)hipFree(p);
      return (int)e;
    }
    if (w.ptr) g_retired.push_back(w.ptr);
    w.ptr = p;
    w.bytes = got - kCtrBytes;
  }
  *ctr = reinterpret_cast<unsigned long long*>(w.ptr);
  *out = reinterpret_cast<char*>(w.ptr) + kCtrBytes;
  return 0;
}
namespace {

// Per-(device, stream) workspace of the prefill's pre-split K/V pieces and of
// the weights' scores, grown as grown_bytes says.  Under stream capture it
// cannot grow: the caller then splits per tile instead.
std::map<WsKey, WsBuf> g_pieces_ws;

}  // namespace
int molot_host::pieces_workspace(void* stream, size_t bytes, void** out) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return (int)e;
  std::lock_guard<std::mutex> lk(g_ws_mu);
  WsBuf& w = g_pieces_ws[WsKey{dev, stream}];
  if (!w.ptr || w.bytes < bytes) {
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    e = hipStreamIsCapturing((hipStream_t)stream, &cap);
    if (e != hipSuccess) return (int)e;
    if (cap != hipStreamCaptureStatusNone) return MOLOT_ENOWS;
    const size_t want =
        grown_bytes(bytes, w.bytes, bytes <= kMaxPiecesBytes ? kMaxPiecesBytes : kMaxScoredBytes);
    size_t got = 0;
    void* p = nullptr;
    e = grow(&p, bytes, want, &got);
    if (e != hipSuccess) return (int)e;
    if (w.ptr) g_retired.push_back(w.ptr);
    w.ptr = p;
    w.bytes = got;
  }
  *out = w.ptr;
  return 0;
}
namespace {

// Dispatch check for the in-launch merge, once per device: a probe launch
// records the XCD (hardware register XCC_ID) of every workgroup of a 4096-
// workgroup grid, and the merge is used only if workgroup i always ran on
// the same XCD as workgroup i % 8 (MI355X's round-robin dispatch in its
// single-partition mode; with one XCD per device the check holds
// trivially).  Read-only after the first call for a device.
__device__ int g_xcc_probe[4096];
__global__ void xcc_probe_kernel() {
  if (threadIdx.x == 0)
    g_xcc_probe[blockIdx.x] = xcc_id();
}
std::mutex g_xcd_mu;
std::map<int, bool> g_xcd_ok;

bool xcd_map_ok(int dev) {
  std::lock_guard<std::mutex> lk(g_xcd_mu);
  auto it = g_xcd_ok.find(dev);
  if (it != g_xcd_ok.end()) return it->second;
  bool ok = false;
  std::vector<int> xcc(4096, -1);
  hipStream_t st = nullptr;
  if (hipStreamCreateWithFlags(&st, hipStreamNonBlocking) == hipSuccess) {
    hipLaunchKernelGGL(xcc_probe_kernel, dim3(4096), dim3(64), 0, st);
    if (hipGetLastError() == hipSuccess &&
        hipMemcpyFromSymbolAsync(xcc.data(), HIP_SYMBOL(g_xcc_probe), sizeof(int) * 4096, 0,
                                 hipMemcpyDeviceToHost, st) == hipSuccess &&
        hipStreamSynchronize(st) == hipSuccess) {
      ok = true;
      for (int i = 0; i < 4096; ++i) ok = ok && xcc[i] >= 0 && xcc[i] == xcc[i % 8];
    }
    (void)hipStreamDestroy(st);
  }
  g_xcd_ok[dev] = ok;
  return ok;
}

bool xcd_ok_cached(int dev) {
  std::lock_guard<std::mutex> lk(g_xcd_mu);
  auto it = g_xcd_ok.find(dev);
  return it != g_xcd_ok.end() && it->second;
}

// Scratch of the no-allocation entry point (molot_hip_decode_step_noalloc):
// the split-K partials of one launch, in device memory that exists from
// module load to process end on every device the library runs on.  Host
// code never passes `scratch` itself (on the host it is only a stand-in
// for the symbol): noalloc_scratch() resolves the device's address once per
// device with hipGetSymbolAddress and hands out that pointer.  Every call
// on a device shares its array; the partials are written and read within
// one step, so nothing needs clearing between calls, and calls that
// overlap on one device race on it.
constexpr size_t kScratchBytes = (size_t)4 << 20;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];
std::mutex g_scratch_mu;
std::map<int, void*> g_scratch_ptr;

int noalloc_scratch(void** out) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return (int)e;
  std::lock_guard<std::mutex> lk(g_scratch_mu);
  auto it = g_scratch_ptr.find(dev);
  if (it == g_scratch_ptr.end()) {
    void* ptr = nullptr;
    e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));  // this device is current
    if (e != hipSuccess) return (int)e;
    if (!ptr) return (int)hipErrorInvalidSymbol;
    it = g_scratch_ptr.emplace(dev, ptr).first;
  }
  *out = it->second;
  return 0;
}

int g_num_cus = 0;
}  // namespace
int molot_host::num_cus() {
  if (g_num_cus) return g_num_cus;
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess &&
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess &&
      cus > 0)
    g_num_cus = cus;
  else
    cus = 256;
  return cus;
}
namespace {

// Tokens per chunk: enough chunks that the launch holds `wpc` workgroups
// per CU (one by default: a workgroup fills its CU), rounded up to a
// multiple of `align` rows (a forced size too: the matrix-core kernel deals
// 32-row tiles to the chunks, and every chunk must get one).
int plan_chunk(int span, int rows_of_wgs, int align, int wpc, int split, int wpcu) {
  int chunk = split;
  if (chunk <= 0) {
    const long target = (long)(wpcu > 0 ? wpcu : wpc) * num_cus();
    long nch = (target + rows_of_wgs - 1) / rows_of_wgs;
    if (nch < 1) nch = 1;
    chunk = (int)((span + nch - 1) / nch);
  }
  chunk = (chunk + align - 1) / align * align;
  if (chunk > kMaxChunk) chunk = kMaxChunk;
  if (chunk < 8) chunk = 8;
  return chunk;
}

// Chunking + workspace of one launch.  `span` bounds every sequence's row
// range tiled by chunks (cache rows only when the kernel folds in the new
// token); B * nkv * subgroups slots share each chunk index.  `cyclic`: the
// kernel deals `align`-row tiles to the chunks round robin (the matrix-core
// kernel on a contiguous cache), so only the chunk count matters: the
// workgroup target's, at most one chunk per tile (a.chunk is then nominal).
//
// A split context is merged in the launch itself (arrive_and_merge) when the
// device dispatches workgroup i to XCD i % 8 and every chunk of a slot can
// run on one XCD: with the grid's slot index fastest that holds when the
// slot count is a multiple of 8; fewer than 8 slots take a 1-D grid that
// puts slot s on XCD s (xmap).  Other slot counts, token-major Q8 launches
// (whose grid groups the heads of a chunk on one XCD instead) and slots of
// more than kMergeMaxChunks chunks use combine_kernel.
// Short contexts of one sequence: an eager step of two dependent launches
// costs more than it computes, so up to kOneChunkSpan rows one workgroup a slot
// takes the context, and up to kBriefSpan at most 16 chunks a slot (the
// matrix-core kernel past 512 rows: 128, a tile a wave) are merged in the
// launch, on 4 XCDs or more.  The vector-ALU kernel only to kBriefWork rows *
// outputs a slot (its merge folds more the longer), and not over Q8, whose
// heads share an XCD a chunk.  us an eager step at 60 / 300 / 900 / 2040 rows,
// the combine kernel against these: 32q/8kv/d128 fp32 8.2, 9.1, 9.5, 10.4
// against 6.8, 8.0, 8.9, (11.0); bf16 9.6, 10.3, 10.8, 10.9 against 7.3, 9.2,
// 9.2, 9.9; Q8 10.3, 11.2, 11.5, 11.8 against 7.8, 9.8, 9.8, 10.3; 64q/8kv/d128
// fp32 9.8, 10.6, 11.0, 13.2 against 9.5, 9.8, (12.1), (15.4); 8q/4kv/d256 fp32
// 7.9, 8.7, 9.5 against 6.4, 8.2, 9.5.
constexpr int kOneChunkSpan = 64, kBriefSpan = 2048;
constexpr long kBriefWork = 1 << 19;
// How a launch's chunks are merged (g_merge).  A launch that keeps weights has a second
// one for them in any case, which merges beside it (combine_weights_kernel): left to the
// library it does, us a step with weights, merged in the launch against beside the
// weights: fp32 32q/8kv/d128 301 rows 10.3 / 7.7, 16385 29.7 / 26.4; 8q/4kv/d256, window
// 1024, 12.0 / 8.7.
int merge_mode(const AttnArgs& a) {
  const int m = knob(g_merge);
  return m < 0 && a.acc ? 0 : m;
}
// Rows of scores kept of a sequence of at most `span` cache rows: those, the appended
// one, and up to a unit of 4 of the matrix-core kernel's order.
int64_t score_rows(int span) { return ((int64_t)std::max(span, 0) + 4) & ~3ll; }
}  // namespace
int molot_host::plan_launch(AttnArgs& a, int d, int span, int gh, int nsubs, int B, int align, int wpc,
                void* stream, bool cyclic) {
  const int rows = a.nkv * nsubs * B;
  const int split = knob(g_split_chunk), wpcu = knob(g_wgs_per_cu);
  DynPlan p{};
  a.dyn_span = 0x7FFFFFFF;
  if (cyclic) {
    const long tiles = span > 0 ? ((long)span + align - 1) / align : 1;
    long nch;
    if (split > 0) {
      const long ch = ((long)split + align - 1) / align * align;
      nch = span > 0 ? (span + ch - 1) / ch : 1;
    } else {
      const long target = (long)(wpcu > 0 ? wpcu : wpc) * num_cus();
      nch = (target + rows - 1) / rows;
      if (wpcu <= 0 && d <= 256 && span <= kOneChunkSpan) {
        nch = 1;
      } else if (wpcu <= 0 && d <= 256 && span <= kBriefSpan && merge_mode(a) < 0 &&
                 (rows % 8 == 0 || (rows >= 4 && rows < 8)) &&
                 (a.matrix || (!a.chunk_fast && (long)span * gh * d <= kBriefWork))) {
        a.brief = 1;
        if (a.matrix) a.chunk_fast = 0;  // a slot's chunks on one XCD instead
        nch = std::min(nch, a.matrix && span > 512 ? (span + 127L) / 128 : 16L);
      }
    }
    nch = std::max(1L, std::min({nch, tiles, (long)kMaxChunks}));
    a.nchunks = (int)nch;
    a.chunk = (int)((tiles + nch - 1) / nch * align);
  } else if (a.dyn && split <= 0 && wpcu <= 0 && span > 0 &&
             (int64_t)B * span * a.nkv * nsubs < ((int64_t)1 << 30) &&
             (p = dyn_plan(span, B, a.nkv * nsubs, a.dyn, a.q8)).nchunks <= kMaxChunks) {
    a.chunk = kDynMax;
    a.nchunks = p.nchunks;
    a.dyn_span = span;
    a.dyn_pairs = p.pairs;
    a.dyn_likely = p.likely;
    a.dyn_min = p.min_chunk;
  } else {
    a.dyn = 0;
    a.chunk = plan_chunk(span > 0 ? span : 1, rows, align, wpc, split, wpcu);
    a.nchunks = span > 0 ? (span + a.chunk - 1) / a.chunk : 1;
    // bound the chunk count (grid x, and the combine's per-pair loop)
    while (a.nchunks > kMaxChunks && a.chunk < kMaxChunk) {
      a.chunk *= 2;
      a.nchunks = (span + a.chunk - 1) / a.chunk;
    }
    if (a.nchunks > kMaxChunks) return MOLOT_ENOTSUP;
  }
  a.part_o = nullptr;
  a.part_ml = nullptr;
  a.qrot = nullptr;
  a.ctr = nullptr;
  a.xmap = 0;
  a.slots = rows;
  a.mrg = 0;
  const size_t stats = a.acc ? (size_t)rows * a.nchunks * gh * 2 : 0;
  if (a.nchunks == 1 && !stats) return 0;  // single chunk: written directly, no combine
  if (a.nchunks > 1 && (long)rows > kMaxSlots) return MOLOT_ENOTSUP;  // (nothing to merge: any number)
  if (stats) {  // the scores of every attended row, for the weights
    if (B > 65535 || a.nq / a.nkv > 4096) return MOLOT_ENOTSUP;  // attn_weights_kernel's grid, its LDS
    a.sc_rows = score_rows(span);
    // (a paged span counts it; a sequence's rows past the span may have no scores)
    a.sc_span = a.block_table ? std::max(span, 0) : (int)a.sc_rows;
    const size_t bytes = sizeof(float) * (size_t)B * a.nq * a.sc_rows;
    // (a KV head's own by 31-bit offsets: score_rsrc)
    if (bytes > kMaxScoredBytes || 4 * a.sc_rows * (a.nq / a.nkv) > 0x7FFFFF00) return MOLOT_ENOTSUP;
    void* sc = nullptr;
    const int st = pieces_workspace(stream, bytes, &sc);
    if (st) return st;
    a.scores = reinterpret_cast<float*>(sc);
  }
  const size_t P = (size_t)gh * d;
  const bool parts = a.nchunks > 1;
  const size_t po = parts ? (size_t)rows * a.nchunks * P : 0;
  const size_t pml = parts ? (size_t)rows * a.nchunks * gh * 2 : 0;
  const size_t qr = parts ? (size_t)rows * P : 0;
  void* ws = nullptr;
  unsigned long long* ctr = nullptr;
  const size_t need = sizeof(float) * (po + pml + qr + stats);
  if (a.ext_ws) {
    // a caller-provided workspace (molot_hip_decode_step_noalloc): no
    // allocation, and the combine kernel merges (no counters to keep)
    if ((int64_t)need > a.ext_ws_bytes) return MOLOT_E2BIG;
    a.part_o = reinterpret_cast<float*>(a.ext_ws);
    a.part_ml = a.part_o + po;
    a.qrot = a.part_ml + pml;
    return 0;
  }
  const int st = workspace(stream, need, &ctr, &ws);
  if (st) return st;
  if (stats) a.stats = reinterpret_cast<float*>(ws) + po + pml + qr;
  if (!parts) return 0;
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = a.part_o + po;
  a.qrot = a.part_ml + pml;
  int dev = 0;
  // automatic: in the launch when the slots fill the 8 XCDs evenly on a
  // contiguous cache and the context is long (measured, 32q/8kv/d128 fp32:
  // step 27.3 -> 26.4 us at n = 16385; at n = 4097 the combine kernel is
  // 0.1 us faster; fewer slots would leave XCDs idle under the 1-D map, and
  // batches of short paged sequences merge few chunks cheaply in the
  // combine kernel: c4 234.8 against 239.3 us).  The matrix-core kernel
  // keeps the combine kernel (launch_mfma).
  const int mk = merge_mode(a);
  const bool want =
      mk > 0 || (mk < 0 && (a.brief || (rows % 8 == 0 && !a.block_table && span >= kMergeAutoSpan)));
  const bool merge = want && !a.chunk_fast && (rows % 8 == 0 || rows < 8) &&
                     a.nchunks <= kMergeMaxChunks && hipGetDevice(&dev) == hipSuccess &&
                     xcd_ok_cached(dev);
  if (merge) {
    a.ctr = ctr;
    a.xmap = rows % 8 != 0;
    a.mrg = merge_lds_floats(gh);
  }
  return 0;
}
namespace {

// geometry of this thread's last attention launch (molot_hip_last_plan)
thread_local int t_last_nchunks = 0;
thread_local int t_last_chunk = 0;

CombArgs comb_args(const AttnArgs& a, int gh, int d, int nsubs, bool paged, bool rope) {
  CombArgs cb{};
  cb.part_o = a.part_o;
  cb.part_ml = a.part_ml;
  cb.qrot = a.qrot;
  cb.o = a.o;
  cb.q_out = a.q_out;
  cb.seq_lens = a.seq_lens;
  cb.pos_arr = a.pos_arr;
  cb.nq = a.nq;
  cb.nkv = a.nkv;
  cb.gh = gh;
  cb.nsub = nsubs;
  cb.d = d;
  cb.dh = a.dh;
  cb.nchunks = a.nchunks;
  cb.chunk = a.chunk;
  cb.window = a.window;
  cb.rope = rope ? 1 : 0;
  cb.paged = !paged ? 0 : a.q8 ? 2 : 1;
  cb.fold = rope && a.fold ? 1 : 0;
  cb.pf = rope ? 0 : a.pf;
  if (cb.pf) {  // the rows' key ranges (comb_chunks), in fields it has no other use for
    cb.seq_lens = a.key_lo;
    cb.pos_arr = a.key_hi;
  }
  cb.pos0 = a.dyn ? a.dyn_likely : a.pos;
  cb.n = a.dyn ? a.dyn_span : a.n;
  cb.dyn = a.dyn;
  cb.nseq = a.nseq;
  return cb;
}

// The weights of a launch that left its scores (AttnArgs::acc).
WeightArgs weight_args(const CombArgs& cb, const AttnArgs& a) {
  WeightArgs w{};
  w.c = cb;
  w.scores = a.scores;
  w.stats = a.stats;
  w.acc = a.acc;
  w.slot_pos = a.slot_pos;
  w.block_table = a.block_table;
  w.sc_rows = a.sc_rows;
  w.sc_span = a.sc_span;
  w.n = a.n;
  w.t0 = a.t0;
  w.pos = a.pos;
  w.max_blocks = a.max_blocks;
  w.page_shift = a.page_shift;
  w.acc_cap = a.acc_cap;
  w.fresh = a.fresh;
  w.blocked = a.matrix;
  return w;
}

int launch_weights(const CombArgs& cb, const AttnArgs& a, int B, void* stream) {
  const WeightArgs w = weight_args(cb, a);
  const dim3 grid((unsigned)((a.sc_rows + kWeightThreads - 1) / kWeightThreads), a.nkv, B);
  hipLaunchKernelGGL(attn_weights_kernel, grid, dim3(kWeightThreads),
                     2 * sizeof(float) * (size_t)(a.nq / a.nkv), (hipStream_t)stream, w);
  return (int)hipGetLastError();
}

// Launches an attention kernel of a planned problem and, for a split
// context, combine_kernel after it on the same stream.
}  // namespace
int molot_host::launch_pair(AttnFn kern, int threads, size_t lds, AttnArgs a, int gh, int d, int nsubs,
                int B, bool paged, bool rope, void* stream) {
  if (lds > kMaxLds) return (int)hipErrorInvalidConfiguration;
  if ((gh * d) % kCombPairs || d % kCombPairs) return MOLOT_ENOTSUP;  // combine tiling
  t_last_nchunks = a.nchunks;
  t_last_chunk = a.dyn ? a.dyn_min : a.chunk;
  a.dynamic = knob(g_dynamic);
  LaunchLock lock(g_launch_mu);
  const bool prof = !a.ext_ws && prof_active(stream);
  const bool combine = a.nchunks > 1 && !a.ctr;  // a second launch merges the chunks
  ProfRec pr{nullptr, nullptr, nullptr, nullptr, combine};
  // Workgroup i runs on XCD i % 8 (its L2 and its share of the CUs), and
  // workgroups are dispatched in linear order.  With the (KV head, subgroup)
  // index fastest, every XCD gets the same heads' share of every chunk and
  // sequence (equal work however the chunks of a batch differ in length),
  // and the chunk index slowest makes the XCDs stream the same rows at the
  // same time.  chunk_fast (Q8 caches) groups by chunk instead: the KV heads
  // of one token share 128-byte lines (token-major: head rows of d bytes at
  // t*R + h*d, the token's scales after them; paged: the page's scales
  // after its codes, 64 bytes a head), so all heads of a (sequence, chunk)
  // pair go to one XCD, whose L2 then fetches each shared line once.  A 1-D
  // grid of 8 * ceil(pairs / 8) * heads workgroups: id runs pair
  // (id / 8 / heads) * 8 + id % 8 (chunk slot pair / B of sequence pair % B)
  // and head (id / 8) % heads, so each pair is on one XCD whatever the
  // counts, its heads are dispatched together, and the padding ids exit at
  // once.
  // xmap (in-launch merge, fewer than 8 slots): a 1-D grid of 8 * nchunks
  // workgroups, id running chunk slot id / 8 of slot id % 8, so each slot's
  // chunks share an XCD; ids of absent slots exit at once.
  const int64_t dheads = (int64_t)a.nkv * nsubs;
  const dim3 grid = a.dyn ? dim3((unsigned)((a.chunk_fast ? (a.dyn_pairs + 7) / 8 * 8 : a.dyn_pairs) *
                                            dheads), 1, 1)
                    : a.chunk_fast
                        ? dim3((unsigned)(((int64_t)B * a.nchunks + 7) / 8 * 8 * a.nkv * nsubs), 1, 1)
                        : a.xmap ? dim3((unsigned)(8 * a.nchunks), 1, 1)
                                 : dim3(a.nkv * nsubs, B, a.nchunks);
  if (prof) {
    pr.a0 = prof_event();
    pr.a1 = prof_event();
    hipExtLaunchKernelGGL(kern, grid, dim3(threads), lds, (hipStream_t)stream, pr.a0, pr.a1, 0,
                          a);
  } else {
    hipLaunchKernelGGL(kern, grid, dim3(threads), lds, (hipStream_t)stream, a);
  }
  int st = (int)hipGetLastError();
  if (st || !combine) {
    if (prof) g_prof.push_back(pr);
    return st || !a.acc ? st : launch_weights(comb_args(a, gh, d, nsubs, paged, rope), a, B, stream);
  }
  CombArgs cb = comb_args(a, gh, d, nsubs, paged, rope);
  // At most 8 chunks (batches of sequences: many slots, few chunks): one
  // wave per 64 pairs (combine_wave_kernel<R>, R = 4 or 8 o loads per lane).
  // More chunks: combine_kernel, whose 4 phases per pair keep the loads per
  // lane at 8 a round (the wave kernel issued 32-64 per lane and was 0.4 us
  // slower at 32 and 64 chunks).
  const int P = gh * d;
  const int wthreads = P % 256 == 0 ? 256 : (P % 128 == 0 ? 128 : 64);
  const int slots = a.nkv * nsubs * B;
  using CombFn = void (*)(CombArgs);
  const bool wave = a.nchunks <= 8;
  const CombFn ck = a.nchunks <= 4 ? combine_wave_kernel<4>
                    : wave         ? combine_wave_kernel<8>
                                   : combine_kernel;
  cb.pairs = comb_pairs(a.dyn ? a.dyn_likely : a.nchunks);
  const dim3 cgrid = wave ? dim3(slots, P / wthreads) : dim3(slots, P / cb.pairs);
  const dim3 cblock = wave ? dim3(wthreads) : dim3(kCombThreads);
  const size_t clds = wave ? 0 : sizeof(float) * (size_t)comb_lds_floats(a.nchunks);  // <= 33 KB
  const int64_t ncomb = (int64_t)slots * (wave ? (P + kCombThreads - 1) / kCombThreads : P / cb.pairs);
  const int64_t nweigh = a.acc ? (a.sc_rows + kWeightThreads - 1) / kWeightThreads * a.nkv * B : 0;
  if (a.acc && !prof && ncomb + nweigh <= 0x7FFFFFFF) {
    using FinFn = void (*)(WeightArgs, int, int);
    const FinFn fk = a.nchunks <= 4 ? combine_weights_kernel<4>
                     : wave         ? combine_weights_kernel<8>
                                    : combine_weights_kernel<0>;
    const size_t wlds = std::max(clds, 2 * sizeof(float) * (size_t)(a.nq / a.nkv));
    hipLaunchKernelGGL(fk, dim3((unsigned)(ncomb + nweigh)), dim3(kCombThreads), wlds,
                       (hipStream_t)stream, weight_args(cb, a), (int)ncomb, slots);
    return (int)hipGetLastError();
  }
  if (prof) {
    pr.c0 = prof_event();
    pr.c1 = prof_event();
    hipExtLaunchKernelGGL(ck, cgrid, cblock, clds, (hipStream_t)stream, pr.c0, pr.c1, 0, cb);
    g_prof.push_back(pr);
  } else {
    hipLaunchKernelGGL(ck, cgrid, cblock, clds, (hipStream_t)stream, cb);
  }
  st = (int)hipGetLastError();
  return st || !a.acc ? st : launch_weights(cb, a, B, stream);
}
namespace {

// Head dims the prefill's matrix-core kernel is built for; decode on fp32
// and bf16 caches takes any even d up to 512, Q8 caches q8_d: any multiple
// of 4 (a token's fp32 scales follow its nkv*d codes, 4-byte aligned).
bool supported_d(int d) { return d == 64 || d == 128 || d == 256; }
bool decode_d(int d) { return d >= 2 && d <= 512 && d % 2 == 0; }
bool q8_d(int d) { return d >= 4 && d <= 512 && d % 4 == 0; }

bool valid_kv(int kv_dtype) {
  return kv_dtype == MOLOT_KV_F32 || kv_dtype == MOLOT_KV_BF16 || kv_dtype == MOLOT_KV_Q8;
}

// bytes of one K/V element (Q8: one code)
int kv_esz(int kv_dtype) { return kv_dtype == MOLOT_KV_F32 ? 4 : kv_dtype == MOLOT_KV_BF16 ? 2 : 1; }

// Q8 byte layouts: a token-major row (codes, then the nkv scales padded to
// 16 bytes) and a paged block (codes [nkv][page][d], then scales [nkv][page])
int64_t q8_row_bytes(int nkv, int d) { return (int64_t)nkv * d + ((4 * (int64_t)nkv + 15) & ~15); }
int64_t q8_block_bytes(int nkv, int d, int page) { return (int64_t)nkv * page * (d + 4); }

int check_common(int nq, int nkv, int d, int kv_dtype) {
  if (nq <= 0 || nkv <= 0 || nq % nkv != 0) return MOLOT_EINVAL;
  if (!valid_kv(kv_dtype)) return MOLOT_EINVAL;
  if (!decode_d(d)) return MOLOT_ENOTSUP;
  if (kv_dtype == MOLOT_KV_Q8 && !q8_d(d)) return MOLOT_ENOTSUP;  // Q8: 64, 128, 256, 512
  return 0;
}

// The strides and scale offsets of the token-major cache [cap][nkv*d]
// (Q8: its byte layout) in a or r.
template <typename A>
void token_major(A& a, int nkv, int d, int kv_dtype) {
  const bool q8 = kv_dtype == MOLOT_KV_Q8;
  a.tok_stride = q8 ? q8_row_bytes(nkv, d) : (int64_t)nkv * d;
  a.head_stride = d;
  a.sc_off = (int64_t)nkv * d;
  a.sc_head = 4;
}

// The same for pages [block][nkv][page][d].
template <typename A>
void paged_layout(A& a, int nkv, int d, int page, int kv_dtype) {
  a.tok_stride = d;
  a.head_stride = (int64_t)page * d;
  a.block_stride =
      kv_dtype == MOLOT_KV_Q8 ? q8_block_bytes(nkv, d, page) : (int64_t)nkv * page * d;
  a.sc_off = (int64_t)nkv * page * d;
  a.sc_head = 4LL * page;
}

// Q8 pages: 16-byte aligned blocks need nkv*page scales to fill 16 bytes
bool q8_pages_ok(int nkv, int page, int kv_dtype) {
  return kv_dtype != MOLOT_KV_Q8 || ((int64_t)nkv * page) % 4 == 0;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

int zero_out(float* O, int64_t count, hipStream_t st) {
  if (count <= 0) return 0;
  const int64_t blocks = (count + 255) / 256;
  hipLaunchKernelGGL(zero_kernel, dim3((unsigned)blocks), dim3(256), 0, st, O, count);
  return (int)hipGetLastError();
}

template <bool PAGED, bool ROPE>
int run_attn(AttnArgs& a, int d, int kv_dtype, int span, int B, void* stream) {
  LaunchLock lock(g_launch_mu);
  if (PAGED && a.acc) {  // the weights' scores within their workspace: sequences by parts
    const int64_t most = (int64_t)kMaxScoredBytes / (4 * a.nq * score_rows(span));
    if (most >= 1 && B > most) {
      for (int b0 = 0; b0 < B; b0 += (int)most) {
        AttnArgs p = a;
        const int64_t qf = (int64_t)b0 * a.nq * d, kf = (int64_t)b0 * a.nkv * d;
        p.q += qf;
        p.o += qf;
        if (ROPE) {
          p.q_out += qf;
          p.k_new += kf;
          p.v_new += kf;
        }
        p.block_table += (int64_t)b0 * a.max_blocks;
        p.seq_lens += b0;
        if (p.pos_arr) p.pos_arr += b0;
        const int st = run_attn<PAGED, ROPE>(p, d, kv_dtype, span, std::min((int)most, B - b0), stream);
        if (st) return st;
      }
      return 0;
    }
  }
  if (a.scored)
    return PAGED ? run_paged_scored(a, ROPE, d, kv_dtype, span, B, stream)
                 : run_flat_scored(a, ROPE, d, kv_dtype, span, B, stream);
  return PAGED ? run_paged(a, ROPE, d, kv_dtype, span, B, stream)
               : run_flat(a, ROPE, d, kv_dtype, span, B, stream);
}

// The layer's norms of the fresh q, k and v (forward.h:554, 562-563).
struct Norms {
  const float* q = nullptr;  // per-head q weights [d], NULL: none
  const float* k = nullptr;  // per-head k weights [d], NULL: none
  int v = 0;                 // v over all nkv*d values, no weights
  float eps = 0.f;
};

bool norms_ok(const Norms& nm) { return nm.eps >= 0.f && nm.eps < INFINITY; }

// How a scored entry forms its scores, and where its weights go.
struct Scoring {
  int on = 0;
  float softcap = 0.f;
  const float* slopes = nullptr;
  float* acc = nullptr;
  int32_t* slot_pos = nullptr;
  int acc_cap = 0;
  const int32_t* key_lo = nullptr;
  const int32_t* key_hi = nullptr;
};

// softcap within the range whose reciprocal and products stay normal floats
bool scoring_ok(const Scoring& sc) {
  if (!(sc.softcap == 0.f || (sc.softcap >= 1e-30f && sc.softcap <= 1e30f))) return false;
  return sc.acc || !sc.slot_pos;
}

void set_scoring(AttnArgs& a, const Scoring& sc, int fresh) {
  a.scored = sc.on;
  a.softcap = sc.softcap;
  a.slopes = sc.slopes;
  a.acc = sc.acc;
  a.slot_pos = sc.slot_pos;
  a.acc_cap = sc.acc_cap;
  a.fresh = fresh;
  a.key_lo = sc.key_lo;
  a.key_hi = sc.key_hi;
}

std::atomic<int> g_presplit{1};  // molot_hip_set_prefill_presplit

template <int D, typename T, bool PAGED>
PfFn pf_kernel_w(int pw) {
  if (pw == 8) return prefill_mfma16_kernel<D, T, PAGED, 8>;
  return prefill_mfma16_kernel<D, T, PAGED, 4>;
}

template <typename T, bool PAGED>
PfFn pf_kernel_d(int d, int pw) {
  if (d == 64) return pf_kernel_w<64, T, PAGED>(pw);
  if (d == 128) return pf_kernel_w<128, T, PAGED>(pw);
  if constexpr (!std::is_same<T, q8_t>::value) return pf_kernel_w<256, T, PAGED>(pw);
  return nullptr;  // Q8 prefill: d = 64, 128
}

// prefill_mfma16_kernel over pre-split pieces (any cache type but bf16).
PfFn pf_kernel_pre(int d, int pw) {
  if (d == 64) return pw == 8 ? prefill_mfma16_kernel<64, float, false, 8, true>
                              : prefill_mfma16_kernel<64, float, false, 4, true>;
  if (d == 128) return pw == 8 ? prefill_mfma16_kernel<128, float, false, 8, true>
                               : prefill_mfma16_kernel<128, float, false, 4, true>;
  return pw == 8 ? prefill_mfma16_kernel<256, float, false, 8, true>
                 : prefill_mfma16_kernel<256, float, false, 4, true>;
}

// The split of cached rows for it.
SplitFn pf_split(int d, int kv_dtype, bool paged) {
  if (kv_dtype == MOLOT_KV_Q8 && d == 64)
    return paged ? pf_split_kernel<64, q8_t, true> : pf_split_kernel<64, q8_t, false>;
  if (kv_dtype == MOLOT_KV_Q8 && d == 128)
    return paged ? pf_split_kernel<128, q8_t, true> : pf_split_kernel<128, q8_t, false>;
  if (kv_dtype == MOLOT_KV_Q8)
    return paged ? pf_split_kernel<256, q8_t, true> : pf_split_kernel<256, q8_t, false>;
  if (d == 64) return paged ? pf_split_kernel<64, float, true> : pf_split_kernel<64, float, false>;
  if (d == 128) return paged ? pf_split_kernel<128, float, true> : pf_split_kernel<128, float, false>;
  return paged ? pf_split_kernel<256, float, true> : pf_split_kernel<256, float, false>;
}

// The prefill kernel of a head dim (64, 128, 256), cache type, layout and
// wave count (pw: 4, or 8 where the instance has it).
PfFn pf_kernel(int d, int kv_dtype, bool paged, int pw) {
  if (kv_dtype == MOLOT_KV_Q8)
    return paged ? pf_kernel_d<q8_t, true>(d, pw) : pf_kernel_d<q8_t, false>(d, pw);
  if (kv_dtype == MOLOT_KV_F32)
    return paged ? pf_kernel_d<float, true>(d, pw) : pf_kernel_d<float, false>(d, pw);
  return paged ? pf_kernel_d<bf16_t, true>(d, pw) : pf_kernel_d<bf16_t, false>(d, pw);
}

}  // namespace

// ===========================================================================
// C ABI
extern "C" {

const char* molot_hip_strerror(int status) {
  switch (status) {
    case MOLOT_OK: return "ok";
    case MOLOT_EINVAL: return "molot_amd: invalid argument";
    case MOLOT_ENOTSUP:
      return "molot_amd: unsupported shape (an even head dim up to 512; Q8 caches a multiple "
             "of 4 up to 512)";
    case MOLOT_ENOSPC: return "molot_amd: KV cache full";
    case MOLOT_ENOWS:
      return "molot_amd: workspace not sized for this shape on a capturing stream (launch the "
             "shape once before capturing)";
    case MOLOT_E2BIG:
      return "molot_amd: the split-K partials of this shape exceed the 4 MiB scratch of "
             "molot_hip_decode_step_noalloc";
  }
  if (status > 0) return hipGetErrorString((hipError_t)status);
  return "molot_amd: unknown status";
}

const char* molot_hip_version(void) { return "molot_amd 0.2"; }

int molot_hip_q8_row_bytes(int nkv, int d) {
  return nkv > 0 && d > 0 ? (int)q8_row_bytes(nkv, d) : 0;
}

int64_t molot_hip_q8_block_bytes(int nkv, int d, int page) {
  return nkv > 0 && d > 0 && page > 0 ? q8_block_bytes(nkv, d, page) : 0;
}

void molot_rope_inv_freq(float base, int d, float* out) {
  for (int i = 0; i < d / 2; ++i) out[i] = 1.0f / powf(base, (2.0f * (float)i) / (float)d);
}

void molot_hip_set_split_chunk(int tokens) { g_split_chunk = tokens > 0 ? tokens : 0; }

int molot_hip_last_plan(int* nchunks, int* chunk) {
  if (!nchunks || !chunk || t_last_nchunks <= 0) return MOLOT_EINVAL;
  *nchunks = t_last_nchunks;
  *chunk = t_last_chunk;
  return 0;
}

void molot_hip_set_block_order(int dynamic) { g_dynamic = dynamic ? 1 : 0; }

void molot_hip_set_bf16_path(int mfma) { g_bf16_mfma = mfma ? 1 : 0; }

int molot_hip_profile_begin(int max_launches) {
  if (max_launches <= 0) return MOLOT_EINVAL;
  LaunchLock lock(g_launch_mu);
  for (ProfRec& r : g_prof) prof_destroy(r);
  g_prof.clear();
  g_prof.reserve(max_launches);
  g_prof_cap = max_launches;
  g_prof_on = true;
  return 0;
}

int molot_hip_profile_end(float* attn_ms, float* combine_ms, int* launches, int* combines) {
  if (!attn_ms || !combine_ms || !launches || !combines) return MOLOT_EINVAL;
  LaunchLock lock(g_launch_mu);
  g_prof_on = false;
  double ta = 0.0, tc = 0.0;
  int n = 0, nc = 0, st = 0;
  for (ProfRec& r : g_prof) {
    if (!r.a0 || !r.a1 || (r.combine && (!r.c0 || !r.c1))) {
      st = (int)hipErrorInvalidValue;
      continue;
    }
    hipError_t e = hipEventSynchronize(r.combine ? r.c1 : r.a1);
    float ms = 0.f;
    if (e == hipSuccess) e = hipEventElapsedTime(&ms, r.a0, r.a1);
    if (e != hipSuccess) {
      st = (int)e;
      continue;
    }
    ta += ms;
    ++n;
    if (r.combine) {
      e = hipEventElapsedTime(&ms, r.c0, r.c1);
      if (e != hipSuccess) {
        st = (int)e;
        continue;
      }
      tc += ms;
      ++nc;
    }
  }
  for (ProfRec& r : g_prof) prof_destroy(r);
  g_prof.clear();
  *attn_ms = (float)ta;
  *combine_ms = (float)tc;
  *launches = n;
  *combines = nc;
  return st;
}

void molot_hip_set_tuning(int wgs_per_cu) { g_wgs_per_cu = wgs_per_cu > 0 ? wgs_per_cu : 0; }

void molot_hip_set_merge(int in_launch) { g_merge = in_launch < 0 ? -1 : (in_launch ? 1 : 0); }

void molot_hip_set_prefill_presplit(int on) { g_presplit = on ? 1 : 0; }

int molot_hip_rope_apply(float* x, int nheads, int d, int pos, const float* inv_freq,
                         void* stream) {
  if (!x || !inv_freq || nheads < 0 || d <= 0 || (d & 1) || d > 2048) return MOLOT_EINVAL;
  if (nheads == 0) return 0;
  RopeArgs a{};
  a.q = x;
  a.inv_freq = inv_freq;
  a.nq = nheads;
  a.d = d;
  a.pos = pos;
  hipLaunchKernelGGL(rope_append_kernel, dim3(nheads, 1), dim3(((d / 2) + 63) / 64 * 64), 0,
                     (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

static int rope_append_impl(float* q, const float* k_new, const float* v_new, void* K, void* V,
                            int nq, int nkv, int d, int slot, int pos, const float* inv_freq,
                            int kv_dtype, const Norms& nm, void* stream) {
  if (nq < 0 || nkv <= 0 || d <= 0 || (d & 1) || d > 2048 || slot < 0) return MOLOT_EINVAL;
  if (!norms_ok(nm)) return MOLOT_EINVAL;
  if ((nq > 0 && !q) || !k_new || !v_new || !K || !V) return MOLOT_EINVAL;
  if (!valid_kv(kv_dtype)) return MOLOT_EINVAL;
  // rows only the attention kernels can read back (their Q8 head dims)
  if (kv_dtype == MOLOT_KV_Q8 && check_common(nkv, nkv, d, kv_dtype)) return MOLOT_ENOTSUP;
  RopeArgs a{};
  a.q = q;
  a.k_new = k_new;
  a.v_new = v_new;
  a.K = K;
  a.V = V;
  a.inv_freq = inv_freq;
  token_major(a, nkv, d, kv_dtype);
  a.nq = nq;
  a.nkv = nkv;
  a.d = d;
  a.slot = slot;
  a.pos = pos;
  a.kv_dtype = kv_dtype;
  a.append = 1;
  a.q_norm = nm.q;
  a.k_norm = nm.k;
  a.v_norm = nm.v;
  a.eps = nm.eps;
  hipLaunchKernelGGL(rope_append_kernel, dim3(nq + nkv, 1), dim3(((d / 2) + 63) / 64 * 64), 0,
                     (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int molot_hip_rope_append(float* q, const float* k_new, const float* v_new, void* K, void* V,
                          int nq, int nkv, int d, int slot, int pos, const float* inv_freq,
                          int kv_dtype, void* stream) {
  return rope_append_impl(q, k_new, v_new, K, V, nq, nkv, d, slot, pos, inv_freq, kv_dtype,
                          Norms{}, stream);
}

static int attn_decode_impl(const float* Q, const void* K, const void* V, float* O, int nq, int nkv,
                            int n, int d, int64_t tok_stride, int64_t head_stride, float scale,
                            int pos_cur, int window, int kv_dtype, const Scoring& sc,
                            void* stream) {
  int st = check_common(nq, nkv, d, kv_dtype);
  if (st) return st;
  if (!Q || !O || n < 0) return MOLOT_EINVAL;
  if (!scoring_ok(sc) || (sc.acc && sc.acc_cap < n)) return MOLOT_EINVAL;
  if (kv_dtype == MOLOT_KV_Q8 && (tok_stride != q8_row_bytes(nkv, d) || head_stride != d))
    return MOLOT_EINVAL;  // Q8: the token-major byte layout only
  int t0 = (window > 0 && pos_cur - window + 1 > 0) ? pos_cur - window + 1 : 0;
  if (t0 > n) t0 = n;
  const int n_att = n - t0;
  if (n_att <= 0) return zero_out(O, (int64_t)nq * d, (hipStream_t)stream);  // o = 0
  if (!K || !V) return MOLOT_EINVAL;
  const int esz = kv_esz(kv_dtype);
  // Rows the kernels can load: at the kernels' head dims (64, 128, 256,
  // 512) 16-byte vectors, so 16-byte aligned row starts; at a padded head
  // dim two-element pieces, so even strides.  A Q8 cache has the fixed
  // layout checked above, whose padded head dims load 4-code pieces.
  const bool padded = d != 64 && d != 128 && d != 256 && d != 512;
  const bool rows_ok = kv_dtype == MOLOT_KV_Q8 ||
                       (padded ? tok_stride % 2 == 0 && head_stride % 2 == 0
                               : (tok_stride * esz) % 16 == 0 && (head_stride * esz) % 16 == 0);
  if (!aligned16(K) || !aligned16(V) || !aligned16(Q) || !aligned16(O) || !rows_ok)
    return MOLOT_EINVAL;
  AttnArgs a{};
  a.q = Q;
  a.k = const_cast<void*>(K);
  a.v = const_cast<void*>(V);
  a.o = O;
  a.tok_stride = tok_stride;
  a.head_stride = head_stride;
  a.sc_off = (int64_t)nkv * d;  // Q8 scales after the row's codes
  a.sc_head = 4;
  a.nq = nq;
  a.nkv = nkv;
  a.n = n;
  a.t0 = t0;
  a.pos = pos_cur;
  a.window = window;
  a.scale = scale;
  set_scoring(a, sc, 0);
  return run_attn<false, false>(a, d, kv_dtype, n_att, 1, stream);
}

int molot_hip_attn_decode_strided(const float* Q, const void* K, const void* V, float* O, int nq,
                                  int nkv, int n, int d, int64_t tok_stride, int64_t head_stride,
                                  float scale, int pos_cur, int window, int kv_dtype,
                                  void* stream) {
  return attn_decode_impl(Q, K, V, O, nq, nkv, n, d, tok_stride, head_stride, scale, pos_cur,
                          window, kv_dtype, Scoring{}, stream);
}

int molot_hip_attn_decode_scored(const float* Q, const void* K, const void* V, float* O, int nq,
                                 int nkv, int n, int d, float scale, int pos_cur, int window,
                                 float softcap, const float* slopes, float* acc, int acc_cap,
                                 int kv_dtype, void* stream) {
  Scoring sc;
  sc.on = 1;
  sc.softcap = softcap;
  sc.slopes = slopes;
  sc.acc = acc;
  sc.acc_cap = acc_cap;
  const int64_t row = kv_dtype == MOLOT_KV_Q8 ? q8_row_bytes(nkv, d) : (int64_t)nkv * d;
  return attn_decode_impl(Q, K, V, O, nq, nkv, n, d, row, d, scale, pos_cur, window, kv_dtype, sc,
                          stream);
}

int molot_hip_attn_decode_gqa_cache(const float* Q, const void* K, const void* V, float* O,
                                    int nq, int nkv, int n, int qhd, float scale, int pos_cur,
                                    int window, int kv_dtype, void* stream) {
  const int64_t row = kv_dtype == MOLOT_KV_Q8 ? q8_row_bytes(nkv, qhd) : (int64_t)nkv * qhd;
  return molot_hip_attn_decode_strided(Q, K, V, O, nq, nkv, n, qhd, row, qhd, scale, pos_cur,
                                       window, kv_dtype, stream);
}

int molot_hip_attn_decode_gqa(const float* Q, const void* K, const void* V, float* O, int nq,
                              int nkv, int n, int d, float scale, int kv_dtype, void* stream) {
  return molot_hip_attn_decode_strided(Q, K, V, O, nq, nkv, n, d, d, (int64_t)n * d, scale, n, 0,
                                       kv_dtype, stream);
}

int molot_hip_attn_decode_gqa_win(const float* Q, const void* K, const void* V, float* O, int nq,
                                  int nkv, int n, int d, float scale, int pos_cur, int window,
                                  int kv_dtype, void* stream) {
  return molot_hip_attn_decode_strided(Q, K, V, O, nq, nkv, n, d, d, (int64_t)n * d, scale,
                                       pos_cur, window, kv_dtype, stream);
}

int molot_hip_attn_decode_head_win(const float* Q, const void* K, const void* V, float* out,
                                   int n, int d, float scale, int pos_cur, int window,
                                   int kv_dtype, void* stream) {
  return molot_hip_attn_decode_strided(Q, K, V, out, 1, 1, n, d, d, (int64_t)n * d, scale,
                                       pos_cur, window, kv_dtype, stream);
}

static int decode_step_impl(float* q, const float* k_new, const float* v_new, void* K, void* V,
                            float* O, int nq, int nkv, int d, int slot, int pos,
                            const float* inv_freq, float scale, int window, int kv_dtype,
                            const Norms& nm, const Scoring& sc, void* stream,
                            void* ext_ws = nullptr, int64_t ext_ws_bytes = 0) {
  int st = check_common(nq, nkv, d, kv_dtype);
  if (st) return st;
  if (!norms_ok(nm)) return MOLOT_EINVAL;
  if (!q || !k_new || !v_new || !K || !V || !O || slot < 0) return MOLOT_EINVAL;
  if (!scoring_ok(sc) || (sc.acc && sc.acc_cap <= slot)) return MOLOT_EINVAL;
  if (!aligned16(K) || !aligned16(V) || !aligned16(q) || !aligned16(O)) return MOLOT_EINVAL;
  const int n = slot + 1;
  int t0 = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
  if (t0 > n) t0 = n;
  if (t0 > n - 1) {
    // the new token itself is outside the window: append, rotate q, o = 0
    st = rope_append_impl(q, k_new, v_new, K, V, nq, nkv, d, slot, pos, inv_freq, kv_dtype, nm,
                          stream);
    if (st) return st;
    if (sc.acc) {
      st = kv_track(sc.acc, sc.slot_pos, nkv, n, 1, pos, sc.acc_cap, stream);
      if (st) return st;
    }
    return zero_out(O, (int64_t)nq * d, (hipStream_t)stream);
  }
  AttnArgs a{};
  a.q_norm = nm.q;
  a.k_norm = nm.k;
  a.v_norm = nm.v;
  a.eps = nm.eps;
  a.q = q;
  a.q_out = q;
  a.k_new = k_new;
  a.v_new = v_new;
  a.k = K;
  a.v = V;
  a.inv_freq = inv_freq;
  a.o = O;
  token_major(a, nkv, d, kv_dtype);
  a.nq = nq;
  a.nkv = nkv;
  a.n = n;
  a.t0 = t0;
  a.pos = pos;
  a.window = window;
  a.scale = scale;
  a.fold = 1;
  a.ext_ws = ext_ws;
  a.ext_ws_bytes = ext_ws_bytes;
  set_scoring(a, sc, 1);
  return run_attn<false, true>(a, d, kv_dtype, n - 1 - t0, 1, stream);  // cache rows
}

int molot_hip_decode_step(float* q, const float* k_new, const float* v_new, void* K, void* V,
                          float* O, int nq, int nkv, int d, int slot, int pos,
                          const float* inv_freq, float scale, int window, int kv_dtype,
                          void* stream) {
  return decode_step_impl(q, k_new, v_new, K, V, O, nq, nkv, d, slot, pos, inv_freq, scale,
                          window, kv_dtype, Norms{}, Scoring{}, stream);
}

int molot_hip_decode_step_noalloc(float* q, const float* k_new, const float* v_new, void* K,
                                  void* V, float* O, int nq, int nkv, int d, int slot, int pos,
                                  const float* inv_freq, float scale, int window, int kv_dtype,
                                  void* stream) {
  void* ws = nullptr;
  const int st = noalloc_scratch(&ws);
  if (st) return st;
  return decode_step_impl(q, k_new, v_new, K, V, O, nq, nkv, d, slot, pos, inv_freq, scale,
                          window, kv_dtype, Norms{}, Scoring{}, stream, ws, (int64_t)kScratchBytes);
}

int molot_hip_decode_step_norm(float* q, const float* k_new, const float* v_new, void* K,
                               void* V, float* O, int nq, int nkv, int d, int slot, int pos,
                               const float* q_norm, const float* k_norm, int v_norm, float eps,
                               const float* inv_freq, float scale, int window, int kv_dtype,
                               void* stream) {
  Norms nm;
  nm.q = q_norm;
  nm.k = k_norm;
  nm.v = v_norm ? 1 : 0;
  nm.eps = eps;
  return decode_step_impl(q, k_new, v_new, K, V, O, nq, nkv, d, slot, pos, inv_freq, scale,
                          window, kv_dtype, nm, Scoring{}, stream);
}

int molot_hip_decode_step_scored(float* q, const float* k_new, const float* v_new, void* K,
                                 void* V, float* O, int nq, int nkv, int d, int slot, int pos,
                                 const float* q_norm, const float* k_norm, int v_norm, float eps,
                                 const float* inv_freq, float scale, int window, float softcap,
                                 const float* slopes, float* acc, int32_t* slot_pos, int acc_cap,
                                 int kv_dtype, void* stream) {
  Norms nm;
  nm.q = q_norm;
  nm.k = k_norm;
  nm.v = v_norm ? 1 : 0;
  nm.eps = eps;
  Scoring sc;
  sc.on = 1;
  sc.softcap = softcap;
  sc.slopes = slopes;
  sc.acc = acc;
  sc.slot_pos = slot_pos;
  sc.acc_cap = acc_cap;
  return decode_step_impl(q, k_new, v_new, K, V, O, nq, nkv, d, slot, pos, inv_freq, scale,
                          window, kv_dtype, nm, sc, stream);
}

static int paged_args(AttnArgs& a, const float* Q, void* K, void* V, float* O,
                      const int32_t* block_table, const int32_t* seq_lens, const int32_t* pos,
                      int B, int max_blocks, int max_seq_len, int nq, int nkv, int d, int page,
                      float scale, int window, int kv_dtype, int* span) {
  int st = check_common(nq, nkv, d, kv_dtype);
  if (st) return st;
  if (!Q || !K || !V || !O || !block_table || !seq_lens || B < 0 || max_blocks <= 0 ||
      max_seq_len < 0 || page <= 0 || (page & (page - 1)))
    return MOLOT_EINVAL;
  if ((int64_t)max_seq_len > (int64_t)max_blocks * page) return MOLOT_EINVAL;
  if (!aligned16(K) || !aligned16(V) || !aligned16(Q) || !aligned16(O)) return MOLOT_EINVAL;
  // head rows of the built dims are whole 16-byte vectors; other even dims
  // run padded, reading two-element pieces (4- or 8-byte aligned)
  if (!q8_pages_ok(nkv, page, kv_dtype)) return MOLOT_EINVAL;
  int shift = 0;
  while ((1 << shift) < page) ++shift;
  a.q = Q;
  a.k = K;
  a.v = V;
  a.o = O;
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.pos_arr = pos;
  paged_layout(a, nkv, d, page, kv_dtype);
  a.nq = nq;
  a.nkv = nkv;
  a.max_blocks = max_blocks;
  a.page_shift = shift;
  a.window = window;
  a.scale = scale;
  // widest attended range of any sequence: with pos[] given, pos may lag the
  // cache end, so only max_seq_len bounds it
  *span = (!pos && window > 0 && window < max_seq_len) ? window : max_seq_len;
  return 0;
}

int molot_hip_attn_decode_paged(const float* Q, const void* K, const void* V, float* O,
                                const int32_t* block_table, const int32_t* seq_lens,
                                const int32_t* pos, int B, int max_blocks, int max_seq_len,
                                int nq, int nkv, int d, int page, float scale, int window,
                                int kv_dtype, void* stream) {
  AttnArgs a{};
  int span = 0;
  int st = paged_args(a, Q, const_cast<void*>(K), const_cast<void*>(V), O, block_table, seq_lens,
                      pos, B, max_blocks, max_seq_len, nq, nkv, d, page, scale, window, kv_dtype,
                      &span);
  if (st) return st;
  if (B == 0) return 0;
  return run_attn<true, false>(a, d, kv_dtype, span, B, stream);
}

int molot_hip_attn_decode_paged_scored(const float* Q, const void* K, const void* V, float* O,
                                       const int32_t* block_table, const int32_t* seq_lens,
                                       const int32_t* pos, int B, int max_blocks, int max_seq_len,
                                       int nq, int nkv, int d, int page, float scale, int window,
                                       float softcap, const float* slopes, float* acc,
                                       int kv_dtype, void* stream) {
  Scoring sc;
  sc.on = 1;
  sc.softcap = softcap;
  sc.slopes = slopes;
  sc.acc = acc;
  if (!scoring_ok(sc)) return MOLOT_EINVAL;
  AttnArgs a{};
  int span = 0;
  int st = paged_args(a, Q, const_cast<void*>(K), const_cast<void*>(V), O, block_table, seq_lens,
                      pos, B, max_blocks, max_seq_len, nq, nkv, d, page, scale, window, kv_dtype,
                      &span);
  if (st) return st;
  if (B == 0) return 0;
  set_scoring(a, sc, 0);
  return run_attn<true, false>(a, d, kv_dtype, span, B, stream);
}

static int rope_append_paged_impl(float* q, const float* k_new, const float* v_new, void* K,
                                  void* V, const int32_t* block_table, const int32_t* seq_lens,
                                  const int32_t* pos, int B, int max_blocks, int nq, int nkv,
                                  int d, int page, const float* inv_freq, int kv_dtype,
                                  const Norms& nm, void* stream);

static int decode_step_paged_impl(float* q, const float* k_new, const float* v_new, void* K,
                                  void* V, float* O, const int32_t* block_table,
                                  const int32_t* seq_lens, const int32_t* pos, int B,
                                  int max_blocks, int max_seq_len, int nq, int nkv, int d,
                                  int page, const float* inv_freq, float scale, int window,
                                  int kv_dtype, const Norms& nm, const Scoring& sc, void* stream) {
  if (!norms_ok(nm) || !scoring_ok(sc)) return MOLOT_EINVAL;
  AttnArgs a{};
  int span = 0;
  int st = paged_args(a, q, K, V, O, block_table, seq_lens, pos, B, max_blocks, max_seq_len, nq,
                      nkv, d, page, scale, window, kv_dtype, &span);
  if (st) return st;
  if (!k_new || !v_new) return MOLOT_EINVAL;
  if (B == 0) return 0;
  set_scoring(a, sc, 1);
  if (pos && (window > 0 || !sc.on)) {
    // a position behind the cache end can leave the new slot outside the
    // window; the split path only folds in rows it attends, so take the
    // unfused kernels there (append, then attention over the cache; a scored
    // step without a window attends every slot whatever the positions)
    st = rope_append_paged_impl(q, k_new, v_new, K, V, block_table, seq_lens, pos, B,
                                max_blocks, nq, nkv, d, page, inv_freq, kv_dtype, nm, stream);
    if (st) return st;
    return run_attn<true, false>(a, d, kv_dtype, span, B, stream);
  }
  a.q_norm = nm.q;
  a.k_norm = nm.k;
  a.v_norm = nm.v;
  a.eps = nm.eps;
  a.q_out = q;
  a.k_new = k_new;
  a.v_new = v_new;
  a.inv_freq = inv_freq;
  a.fold = 1;
  return run_attn<true, true>(a, d, kv_dtype, span, B, stream);  // span >= cache rows
}

int molot_hip_decode_step_paged(float* q, const float* k_new, const float* v_new, void* K,
                                void* V, float* O, const int32_t* block_table,
                                const int32_t* seq_lens, const int32_t* pos, int B,
                                int max_blocks, int max_seq_len, int nq, int nkv, int d, int page,
                                const float* inv_freq, float scale, int window, int kv_dtype,
                                void* stream) {
  return decode_step_paged_impl(q, k_new, v_new, K, V, O, block_table, seq_lens, pos, B,
                                max_blocks, max_seq_len, nq, nkv, d, page, inv_freq, scale,
                                window, kv_dtype, Norms{}, Scoring{}, stream);
}

int molot_hip_decode_step_paged_norm(float* q, const float* k_new, const float* v_new, void* K,
                                     void* V, float* O, const int32_t* block_table,
                                     const int32_t* seq_lens, const int32_t* pos, int B,
                                     int max_blocks, int max_seq_len, int nq, int nkv, int d,
                                     int page, const float* q_norm, const float* k_norm,
                                     int v_norm, float eps, const float* inv_freq, float scale,
                                     int window, int kv_dtype, void* stream) {
  Norms nm;
  nm.q = q_norm;
  nm.k = k_norm;
  nm.v = v_norm ? 1 : 0;
  nm.eps = eps;
  return decode_step_paged_impl(q, k_new, v_new, K, V, O, block_table, seq_lens, pos, B,
                                max_blocks, max_seq_len, nq, nkv, d, page, inv_freq, scale,
                                window, kv_dtype, nm, Scoring{}, stream);
}

int molot_hip_decode_step_paged_scored(
    float* q, const float* k_new, const float* v_new, void* K, void* V, float* O,
    const int32_t* block_table, const int32_t* seq_lens, const int32_t* pos, int B, int max_blocks,
    int max_seq_len, int nq, int nkv, int d, int page, const float* q_norm, const float* k_norm,
    int v_norm, float eps, const float* inv_freq, float scale, int window, float softcap,
    const float* slopes, float* acc, int32_t* slot_pos, int kv_dtype, void* stream) {
  Norms nm;
  nm.q = q_norm;
  nm.k = k_norm;
  nm.v = v_norm ? 1 : 0;
  nm.eps = eps;
  Scoring sc;
  sc.on = 1;
  sc.softcap = softcap;
  sc.slopes = slopes;
  sc.acc = acc;
  sc.slot_pos = slot_pos;
  return decode_step_paged_impl(q, k_new, v_new, K, V, O, block_table, seq_lens, pos, B,
                                max_blocks, max_seq_len, nq, nkv, d, page, inv_freq, scale,
                                window, kv_dtype, nm, sc, stream);
}

int molot_hip_rope_append_paged(float* q, const float* k_new, const float* v_new, void* K,
                                void* V, const int32_t* block_table, const int32_t* seq_lens,
                                const int32_t* pos, int B, int max_blocks, int nq, int nkv, int d,
                                int page, const float* inv_freq, int kv_dtype, void* stream) {
  return rope_append_paged_impl(q, k_new, v_new, K, V, block_table, seq_lens, pos, B, max_blocks,
                                nq, nkv, d, page, inv_freq, kv_dtype, Norms{}, stream);
}

static int rope_append_paged_impl(float* q, const float* k_new, const float* v_new, void* K,
                                  void* V, const int32_t* block_table, const int32_t* seq_lens,
                                  const int32_t* pos, int B, int max_blocks, int nq, int nkv,
                                  int d, int page, const float* inv_freq, int kv_dtype,
                                  const Norms& nm, void* stream) {
  if (!norms_ok(nm)) return MOLOT_EINVAL;
  if (nq < 0 || nkv <= 0 || d <= 0 || (d & 1) || d > 2048 || B < 0 || max_blocks <= 0 ||
      page <= 0)
    return MOLOT_EINVAL;
  if ((nq > 0 && !q) || !k_new || !v_new || !K || !V || !block_table || !seq_lens)
    return MOLOT_EINVAL;
  if (!valid_kv(kv_dtype)) return MOLOT_EINVAL;
  // the page layout every paged attention entry accepts
  if ((page & (page - 1)) || !q8_pages_ok(nkv, page, kv_dtype)) return MOLOT_EINVAL;
  if (kv_dtype == MOLOT_KV_Q8 && check_common(nkv, nkv, d, kv_dtype)) return MOLOT_ENOTSUP;
  if (B == 0) return 0;
  RopeArgs a{};
  a.q = q;
  a.k_new = k_new;
  a.v_new = v_new;
  a.K = K;
  a.V = V;
  a.inv_freq = inv_freq;
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.pos_arr = pos;
  paged_layout(a, nkv, d, page, kv_dtype);
  a.nq = nq;
  a.nkv = nkv;
  a.d = d;
  a.max_blocks = max_blocks;
  a.page = page;
  a.kv_dtype = kv_dtype;
  a.append = 1;
  a.q_norm = nm.q;
  a.k_norm = nm.k;
  a.v_norm = nm.v;
  a.eps = nm.eps;
  hipLaunchKernelGGL(rope_append_kernel, dim3(nq + nkv, B), dim3(((d / 2) + 63) / 64 * 64), 0,
                     (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

// A workspace that the device has no memory for is one that is unavailable:
// the path without it runs instead.
static int without_memory(int st) { return st == (int)hipErrorOutOfMemory ? MOLOT_ENOWS : st; }

// The attended keys of a prefill: [T0, N) with T0 the window start of its
// first query (pos0), split into 16-bit pieces once per launch for fp32 and
// Q8 caches when the pieces fit (kMaxPiecesBytes), there is memory for them and
// the workspace need not grow under capture.  Returns the pieces buffer (NULL: the attention kernel
// splits each staged tile itself) and sets T0 and R.
// only: the launch has no per-tile kernel (a Q8 cache at d = 256): the
// pieces are made whatever the presplit switch says (within the same cap;
// past it, or under a capture that would grow them, such a prefill runs as
// prefill rows).
static int prefill_pieces(int nkv, int N, int d, int pos0, int window, int kv_dtype, void* stream,
                          int presplit, void** ws, int* T0, int64_t* R, bool only = false) {
  *ws = nullptr;
  *T0 = window > 0 && pos0 - window + 1 > 0 ? std::min(pos0 - window + 1, N) : 0;
  *R = (int64_t)N - *T0;
  if (!only && (kv_dtype == MOLOT_KV_BF16 || !presplit)) return 0;
  const size_t need = (size_t)2 * nkv * 3 * *R * d * sizeof(uint16_t);
  void* p = nullptr;
  const int st =
      *R > 0 && need <= kMaxPiecesBytes ? without_memory(pieces_workspace(stream, need, &p))
                                        : MOLOT_ENOWS;
  if (st && st != MOLOT_ENOWS) return st;
  if (!st) *ws = p;
  return 0;
}

// The last position or slot of a prompt: pos0 + m + 1 is an int in the kernels.
constexpr int kMaxPos = 0x7FFFFFFF;

// The widest range of keys that a query row may attend.
static int prefill_span(int N, int window, const Scoring& sc) {
  return window > 0 && window < N && !sc.key_hi ? window : N;
}

// The prefill at a head dim the matrix-core prefill does not tile (an even d
// that is not a multiple of 8; a padded Q8 cache), and above 256 where the
// prompt is too small for prefill_on_pieces or its workspace cannot be had:
// the vector-ALU decode kernel with each query row as a sequence of its own
// (AttnArgs::pf) over the one cache, contiguous or through the prompt's
// block-table row.  Each query row streams its attended rows; neighbouring
// rows of a prompt read the same keys, which the L2 and the Infinity Cache
// serve after the first.
static int prefill_rows(const float* Qm, const void* K, const void* V, float* Om, int nq,
                        int nkv, int M, int N, int d, float scale, int pos0, int window,
                        int kv_dtype, const int32_t* block_row, int page, const Scoring& sc,
                        void* stream) {
  if ((int64_t)M > 65535) return MOLOT_ENOTSUP;  // grid rows: one per query
  AttnArgs a{};
  a.q = Qm;
  a.k = const_cast<void*>(K);
  a.v = const_cast<void*>(V);
  a.o = Om;
  if (block_row) {
    if (page <= 0 || (page & (page - 1)) || !q8_pages_ok(nkv, page, kv_dtype)) return MOLOT_EINVAL;
    paged_layout(a, nkv, d, page, kv_dtype);
    a.block_table = block_row;
    a.max_blocks = 0;  // every row reads the one block-table row
    while ((1 << a.page_shift) < page) ++a.page_shift;
  } else {
    token_major(a, nkv, d, kv_dtype);
  }
  a.nq = nq;
  a.nkv = nkv;
  a.n = N;
  a.pos = pos0;
  a.window = window;
  a.scale = scale;
  a.pf = 1;
  set_scoring(a, sc, 0);
  const int span = prefill_span(N, window, sc);
  // rows m0 .. m0 + rows - 1
  auto launch = [&](int m0, int rows) {
    AttnArgs b = a;
    b.q += (int64_t)m0 * nq * d;
    b.o += (int64_t)m0 * nq * d;
    b.pos += m0;
    if (b.key_lo) b.key_lo += m0;
    if (b.key_hi) b.key_hi += m0;
    return block_row ? run_attn<true, false>(b, d, kv_dtype, span, rows, stream)
                     : run_attn<false, false>(b, d, kv_dtype, span, rows, stream);
  };
  const int st = launch(0, M);
  // more (row, head group) slots than the merge of their chunks takes: by parts
  const int64_t groups = (int64_t)nkv * (nq / nkv / std::min(pick_gh(nq / nkv), 4));  // (or fewer)
  const int part = (int)std::max<int64_t>(1, kMaxSlots / groups);
  if (st != MOLOT_ENOTSUP || M <= part) return st;
  for (int m0 = 0; m0 < M; m0 += part) {
    const int sp = launch(m0, std::min(part, M - m0));
    if (sp) return sp;
  }
  return 0;
}

// Launches a prefill attention kernel of `wgs` workgroups and, where its key
// tiles are split, the merge of the splits' partials after it.
static int launch_prefill(PfFn pk, int64_t wgs, int threads, const PfArgs& a, int D,
                          void* stream) {
  const dim3 grid((unsigned)wgs);
  const int nsplit = a.nsplit;
  int st = 0;
  CombArgs cb{};  // split-K: (token, q head) rows as slots of one head each
  cb.part_o = a.part_o;
  cb.part_ml = a.part_ml;
  cb.o = a.o;
  cb.nq = a.nq;
  cb.nkv = a.nq;
  cb.gh = 1;
  cb.nsub = 1;
  cb.d = D;
  cb.dh = a.dh;
  cb.nchunks = nsplit;
  cb.chunk = 1;
  cb.pairs = comb_pairs(nsplit);
  // at most 8 splits: the row merge, one wave per 64V outputs of a slot
  // (2048 tokens x 8 q heads at d = 256 over 2 splits: 9.2 us, against 22.2
  // with a wave per 64 outputs and 82 us on combine_kernel's 4 workgroups a
  // slot); more splits: combine_kernel
  const bool cwave = nsplit <= 8;
  const int cv = D % 256 == 0 ? 4 : (D % 128 == 0 ? 2 : 1);
  const int64_t cunits = (int64_t)a.M * a.nq * (D / (64 * cv));
  using RowsFn = void (*)(CombArgs, int64_t);
  const RowsFn rk = a.some ? (nsplit <= 4 ? (cv == 4 ? combine_rows_kernel<4, 4, true>
                                           : cv == 2 ? combine_rows_kernel<4, 2, true>
                                                     : combine_rows_kernel<4, 1, true>)
                                        : (cv == 4 ? combine_rows_kernel<8, 4, true>
                                           : cv == 2 ? combine_rows_kernel<8, 2, true>
                                                     : combine_rows_kernel<8, 1, true>))
                  : nsplit <= 4 ? (cv == 4 ? combine_rows_kernel<4, 4>
                                  : cv == 2 ? combine_rows_kernel<4, 2> : combine_rows_kernel<4, 1>)
                                : (cv == 4 ? combine_rows_kernel<8, 4>
                                  : cv == 2 ? combine_rows_kernel<8, 2> : combine_rows_kernel<8, 1>);
  const dim3 cgrid = cwave ? dim3((unsigned)((cunits + 3) / 4))
                           : dim3((unsigned)((int64_t)a.M * a.nq), (unsigned)(D / cb.pairs));
  const dim3 cblock = cwave ? dim3((unsigned)kCombWaveThreads) : dim3(kCombThreads);
  const size_t clds = cwave ? 0 : sizeof(float) * (size_t)comb_lds_floats(nsplit);
  LaunchLock lock(g_launch_mu);
  if (prof_active(stream)) {
    ProfRec pr{prof_event(), prof_event(), nullptr, nullptr, nsplit > 1};
    hipExtLaunchKernelGGL(pk, grid, dim3(threads), 0, (hipStream_t)stream, pr.a0, pr.a1, 0, a);
    st = (int)hipGetLastError();
    if (!st && nsplit > 1) {
      pr.c0 = prof_event();
      pr.c1 = prof_event();
      if (cwave)
        hipExtLaunchKernelGGL(rk, cgrid, cblock, 0, (hipStream_t)stream, pr.c0, pr.c1, 0, cb,
                              cunits);
      else
        hipExtLaunchKernelGGL(combine_kernel, cgrid, cblock, clds, (hipStream_t)stream, pr.c0,
                              pr.c1, 0, cb);
      st = (int)hipGetLastError();
    }
    g_prof.push_back(pr);
    return st;
  }
  hipLaunchKernelGGL(pk, grid, dim3(threads), 0, (hipStream_t)stream, a);
  st = (int)hipGetLastError();
  if (st || nsplit == 1) return st;
  if (cwave)
    hipLaunchKernelGGL(rk, cgrid, cblock, 0, (hipStream_t)stream, cb, cunits);
  else
    hipLaunchKernelGGL(combine_kernel, cgrid, cblock, clds, (hipStream_t)stream, cb);
  return (int)hipGetLastError();
}

// Key splits of a launch of nqb * nkv query blocks of qb rows on the 32-row
// kernels (one workgroup a CU): the count with the least estimated time.  A
// split's cost is its tiles' plus its start and end; the launch's the longest
// split's, or the CUs' share of all of them with half of the shortest for the
// uneven last round; and more than one split pays the merge of their
// partials.
static int pieces_splits(int64_t nqb, int nkv, int M, int N, int G, int qb, int D, bool f32,
                         int pos0, int window, int nq) {
  auto tiles_of = [&](int64_t b) {  // query block b's tiles (32 keys)
    const int64_t m0 = b * qb / G, m1 = std::min<int64_t>(((b + 1) * qb - 1) / G, M - 1);
    const int64_t lo = window > 0 ? std::max<int64_t>(0, pos0 + m0 - window + 1) : 0;
    const int64_t hi = std::min<int64_t>(pos0 + m1 + 1, N);
    return hi > lo ? (double)((hi - lo + kWideTile - 1) / kWideTile) : 0.0;
  };
  const double first = tiles_of(0), last = tiles_of(nqb - 1), mid = tiles_of(nqb / 2);
  const double longest = std::max({first, mid, last}), shortest = std::min({first, mid, last});
  const double total = (first + 4 * mid + last) / 6 * (double)(nqb * nkv);
  // measured, us: a tile (D = 128 two in 2.3 over fp32, 1.75 over one piece;
  // D = 512 3.2) and a split's start and end
  const double kTileUs = (D <= 128 ? 1.15 * D / 128 : 3.2 * D / 512) * (f32 ? 1.0 : 0.75);
  const double kStart = 6.0 / kTileUs;
  const int cus = num_cus();
  double best = 0;
  int ns_best = 1;
  for (int ns = 1; ns <= 64 && ns <= std::max(1.0, longest / 4); ++ns) {
    const double wgs = (double)(nqb * nkv) * ns;
    double est = longest / ns + kStart;
    if (wgs > cus)
      est = std::max(est, (total + wgs * kStart) / cus + 0.5 * (shortest / ns + kStart));
    est *= kTileUs;
    if (ns > 1) est += 4.0 + 8.0 * M * nq * (double)D * ns / 4e6;
    if (ns == 1 || est < best) {
      best = est;
      ns_best = ns;
    }
  }
  return ns_best;
}

// Head dims whose smaller prompts run as prefill rows: those the 16-row
// matrix-core prefill does not tile, and Q8 caches at padded ones (it reads
// whole 16-code chunks of the built dims only).
static bool prefill_by_rows(int d, int kv_dtype) {
  return d > 256 || d % 8 != 0 || (!supported_d(d) && kv_dtype == MOLOT_KV_Q8);
}

// Whether a small prompt's launch (head dims up to 128) takes its keys' pieces
// from one split of them, and not of every staged tile in every query block.
// The split is a launch of its own: it pays where the tiles of one workgroup
// follow each other (4 to 7 of them, fp32 at D = 128; from 8 on the keys are
// split over workgroups), and with 7.5e8 (query head, key, element) products
// of three row blocks of 128 or more over 512 keys or more (not Q8 at D = 128, nor
// where each query head has its own KV head: the split itself then takes as
// much).  Both sides, us a call of the attention alone over fp32 / Q8, per tile
// against pieces, (rows, cached) of 32q/8kv/d128: (40, 150) 20.6 / 17.3 against
// 17.0 / 17.0; (150, 0) 17.7 / 15.1 against 15.1 / 15.1; (77, 0) 12.4 / 10.8
// against 12.2 / 12.3; (77, 150) 19.5 / 19.0 against 20.5 / 20.3; (16, 5000) 35 /
// 33 against 42 / 39; (16, 16000) 89 / 80 against 107 / 97; (150, 1500) 51.5 /
// 48.0 against 49.4 / 50.2; 64q (77, 1500) 56.3 / 52.8 against 49.9 / 51.7; 64q
// (300, 40) 35.6 / 35.3 against 37.2 / 37.3; 32q/8kv/d64 (40, 150) 13.2 / 13.8
// against 13.1 / 13.1; (300, 1500) 46.2 / 50.4 against 43.0 / 43.0;
// 16q/16kv/d128 (500, 500) 37.7 / 35.7 against 35.7 / 36.9 (the step 42.7 / 43.1
// against 45.0 / 46.1).
static bool prefill_split_pays(int M, int N, int nq, int nkv, int D, int kv_dtype, int window) {
  const int64_t span = window > 0 && window < N ? window : N;
  const int64_t tiles = (span + 31) / 32;
  if (kv_dtype == MOLOT_KV_F32 && D == 128 && tiles >= 4 && tiles < 8) return true;
  return (kv_dtype == MOLOT_KV_F32 || D == 64) && nq >= 2 * nkv &&
         (int64_t)M * (nq / nkv) > 256 && span >= 512 &&
         (int64_t)M * nq * span * D >= 750000000;
}

// The head dim a prefill of head dim d is padded to.
static int prefill_D(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : d <= 256 ? 256 : 512; }

// Whether a prefill runs on the 32-row kernels over fp16 pieces
// (prefill_on_pieces): those stage and start more, so they take prompts with
// enough work.  Not at 129 to 256: prefill_wide_kernel built for D = 256 took
// 103 / 117 / 118 us a step (2048 tokens, 8q/4kv/d256, window 1024; fp32 / bf16
// / Q8) against 102 / 90 / 105 on prefill_mfma16_kernel.
// Above 256 the other path is prefill_rows, which streams the keys once a row
// and four query heads; below 8 such passes it is the faster one however long
// the cache.  Both sides, 8q/2kv/d512, us a step over fp32 / bf16 / Q8 caches:
// (rows, cached) = (64, 500) prefill rows 40 / 40 / 37, matrix cores 44 / 38 /
// 38; (8, 4000) 43 / 38 / 37 against 47 / 38 / 41; (24, 4000) 123 / 117 / 96
// against 53 / 44 / 46; (8, 16384) 118 / 94 / 77 against 92 / 64 / 61; (2, 65536),
// the attention, 162 / 92 / 70 against 350 / 177 / 199; (4, 32768) 164 / 96 / 69
// against 177 / 94 / 86.
// Up to 128 it is prefill_mfma16_kernel.  32q/8kv/d128, fp32 / bf16 / Q8:
// (77, 4000) 80 / 64 / 78 against 75 / 64 / 65; (200, 2000) 76 / - / 77
// against 70 / - / 62; (512, 0) 39 / 35 / 40 against 38 / 36 / 37; (200, 500)
// 44 / 35 / 45 against 48 / 45 / 46; (512, 16384) 497 / 414 / 485 against 438
// / 301 / 298.
// At D = 128 that kernel keeps the prompts whose row blocks its key splits (up
// to 16) multiply to the CUs evenly, while there are too few of them to pay for
// the split of the cached rows: the attention, (rows a KV head, cached), other
// against 32 rows, 16q/16kv (128, 16384) fp32 107 against 175, bf16 66 against
// 101, Q8 89 against 92; 32q/8kv (256, 16384) 104 / 69 / 86 against 113 / 73 /
// 72; (512, 4000) 55 / 38 / 51 against 55 / 42 / 42; (512, 16384) 170 / 111 / 152
// against 156 / 102 / 102; (1024, 1500) 47 / 33 / 43 against 44 / 36 / 37.
// (molot_hip_set_prefill_presplit(0) keeps every prompt off them, and so out
// of their workspace.)
static bool prefill_takes_pieces(int d, int M, int N, int nq, int nkv, int kv_dtype, int window,
                                 int presplit) {
  constexpr int64_t kWideWork = 400000, kPairFlops = 1200000000;
  const int64_t span = window > 0 && window < N ? window : N;
  const int64_t pairs = (int64_t)M * nq * span;
  const int G = nq / nkv;
  if (!presplit || M > 65535 || (d > 128 && d <= 256)) return false;
  if (d > 256) return pairs >= kWideWork && (int64_t)M * ((G + 3) / 4) >= 8;
  if (pairs * prefill_D(d) < kPairFlops) return false;
  const int64_t nqb = ((int64_t)M * G + 127) / 128, wgs = nqb * nkv;
  const int cus = num_cus();
  if (prefill_D(d) == 128 && !prefill_by_rows(d, kv_dtype) && 16 * wgs >= cus && cus % wgs == 0) {
    if (nqb <= (kv_dtype == MOLOT_KV_Q8 ? 1 : 2)) return false;
    if (kv_dtype == MOLOT_KV_BF16 && (nqb - 3) * span * nkv < 75000) return false;
  }
  return true;
}

// The same of a scored prefill, whose other path is prefill_rows at every head dim: below
// 64 query rows a KV head that streams the keys a few times, the pieces are two launches
// before the attention.  Causal with a cap, (tokens, cached), us on rows / on pieces; where
// the two meet:
//   16q/4kv/d64    fp32 (300, 0) 18.8 / 20.8, (32, 4000) 38.9 / 26.6; bf16 (16, 4000) 18.6 /
//                  20.8, (300, 0) 22.9 / 19.0; Q8 (32, 0) 10.8 / 12.1, (128, 0) 19.4 / 14.1
//   32q/8kv/d128   fp32 (32, 500) 17.8 / 26.2, (200, 0) 34.7 / 23.2; bf16 (128, 0) 16.7 /
//                  19.2, (200, 0) 28.9 / 21.4; Q8 (16, 300) 16.5 / 21.7, (77, 0) 29.2 / 17.2
//   8q/4kv/d256    fp32 (300, 0) 33.6 / 39.7, (32, 4000) 71.3 / 46.2; bf16 36.3 / 42.0, 45.7 /
//                  38.2; Q8 (77, 500) 32.5 / 37.1, (300, 0) 49.6 / 41.9
//   8q/2kv/d512    fp32 (200, 0) 32.1 / 35.8, (77, 500) 54.6 / 41.2; bf16 (128, 0) 17.0 / 26.1,
//                  (200, 0) 32.8 / 31.3; Q8 17.5 / 26.4, 33.7 / 31.1
//   few rows       (2, 65536): rows by 1.4 to 4 times; (4, 16384): d128 fp32 61 / 86, bf16 50 /
//                  56, Q8 76 / 59
static bool prefill_scored_pieces(int d, int M, int N, int nq, int nkv, int window, int kv_dtype,
                                  const Scoring& sc, int presplit) {
  static constexpr int kPairs[3][4] = {  // thousands of (query row, key), by cache and padded head dim
      {1800, 800, 900, 340}, {1200, 800, 900, 300}, {150, 180, 500, 300}};
  const int64_t span = prefill_span(N, window, sc);
  const int D = prefill_D(d), cache = kv_dtype == MOLOT_KV_F32 ? 0 : kv_dtype == MOLOT_KV_BF16 ? 1 : 2;
  return presplit && M <= 65535 && (int64_t)M * (nq / nkv) >= 64 &&
         (int64_t)M * nq * span >= 1000ll * kPairs[cache][D == 64 ? 0 : D == 128 ? 1 : D == 256 ? 2 : 3];
}

// Their workspace for the attended keys [T0, N).
static int pieces32_workspace(int nkv, int N, int d, int pos0, int window, int kv_dtype, bool scored,
                              void* stream, void** ws, int* T0, int* R) {
  *T0 = window > 0 && pos0 - window + 1 > 0 ? std::min(pos0 - window + 1, N) : 0;
  *R = N - *T0;
  const size_t need = wide_bytes(nkv, prefill_D(d), wide_pieces(kv_dtype == MOLOT_KV_F32), *R);
  if (need > (scored ? kMaxScoredBytes : kMaxPiecesBytes)) return MOLOT_ENOWS;
  return without_memory(pieces_workspace(stream, need, ws));
}

// The prefill on the 32-row kernels (prefill_narrow.hip, prefill_wide.hip):
// the attended keys' pieces first (split_rows of them; the appending step
// wrote the others), then the attention over them.  MOLOT_ENOWS: a capture
// that would have to grow the workspace, no memory for it, or keys past its
// cap (the caller takes the other path).
static int prefill_on_pieces(const float* Qm, const void* K, const void* V, float* Om, int nq,
                             int nkv, int M, int N, int d, float scale, int pos0, int window,
                             int kv_dtype, const int32_t* block_row, int page, const Scoring& sc,
                             void* stream, int split_rows) {
  const int D = prefill_D(d), qb = wide_rows(D);
  PfArgs a{};
  a.q = Qm;
  a.k = K;
  a.v = V;
  a.o = Om;
  a.nq = nq;
  a.nkv = nkv;
  a.M = M;
  a.N = N;
  a.dh = d;
  a.pos0 = pos0;
  a.window = window;
  a.scale = scale;
  a.own = sc.on || prefill_by_rows(d, kv_dtype);
  a.softcap = sc.softcap;
  a.slopes = sc.slopes;
  a.key_lo = sc.key_lo;
  a.key_hi = sc.key_hi;
  a.kv_dtype = kv_dtype;
  if (block_row) {
    if (page <= 0 || (page & (page - 1)) || !q8_pages_ok(nkv, page, kv_dtype))
      return MOLOT_EINVAL;
    a.block_table = block_row;
    while ((1 << a.page_shift) < page) ++a.page_shift;
  }
  void* pieces = nullptr;
  int st = pieces32_workspace(nkv, N, d, pos0, window, kv_dtype, sc.on, stream, &pieces, &a.T0, &a.R);
  if (st) return st;
  if (a.R == 0) return zero_out(Om, (int64_t)M * nq * d, (hipStream_t)stream);  // no key attended
  a.pieces = reinterpret_cast<const uint16_t*>(pieces);
  const int G = nq / nkv;
  const int64_t nqb = ((int64_t)M * G + qb - 1) / qb;
  a.nqb = (int)nqb;
  a.nsplit = pieces_splits(nqb, nkv, M, N, G, qb, D, kv_dtype == MOLOT_KV_F32, pos0, window, nq);
  if (a.nsplit > 1) {
    unsigned long long* ctr = nullptr;
    void* ws = nullptr;
    st = without_memory(
        workspace(stream, sizeof(float) * (size_t)M * nq * a.nsplit * (D + 2), &ctr, &ws));
    if (st && st != MOLOT_ENOWS) return st;
    if (st) {
      a.nsplit = 1;  // under capture, or without memory, the workspace cannot grow
    } else {
      a.part_o = reinterpret_cast<float*>(ws);
      a.part_ml = a.part_o + (size_t)M * nq * a.nsplit * D;
    }
  }
  if (nqb * nkv * a.nsplit > (int64_t)0x7FFFFFFF) return MOLOT_ENOTSUP;
  a.some = sc.on && a.nsplit > 1 && a.nsplit <= 8;  // (more splits: combine_kernel, which reads all)
  a.Rsplit = split_rows < 0 ? a.R : std::min(split_rows, a.R);
  if (a.Rsplit > 0) {
    const int64_t units = (a.Rsplit == a.R ? wide_padded_rows(a.R) : a.Rsplit) * (D / 8);
    hipLaunchKernelGGL(prefill_wide_split(D, kv_dtype, block_row != nullptr),
                       dim3((unsigned)((units + 255) / 256), nkv, 2), dim3(256), 0,
                       (hipStream_t)stream, a, reinterpret_cast<uint16_t*>(pieces));
    st = (int)hipGetLastError();
    if (st) return st;
  }
  return launch_prefill(D <= 128 ? prefill_narrow_fn(D, kv_dtype, a.own, sc.on)
                                 : prefill_wide_fn(D, kv_dtype, sc.on),
                        nqb * nkv * a.nsplit, 64 * kWideWaves, a, D, stream);
}

// presplit: the setting, read once a call (an appending step's RoPE/append
// has written pieces in the layout that it selects).
// split_rows: rows of [T0, N) the split kernel still has to split (the
// appending step wrote the pieces of the others; -1: all of them)
static int attn_prefill_impl(const float* Qm, const void* K, const void* V, float* Om, int nq,
                             int nkv, int M, int N, int d, float scale, int pos0, int window,
                             int kv_dtype, const int32_t* block_row, int page, const Scoring& sc,
                             void* stream, int presplit, int split_rows = -1) {
  int st = check_common(nq, nkv, d, kv_dtype);
  if (st) return st;
  if (!scoring_ok(sc)) return MOLOT_EINVAL;
  // The prefill kernels are built for D = 64, 128, 256.  Any other head dim
  // that is a multiple of 8 below 256 (fp32 or bf16) runs padded to the next
  // D: the split kernel and the per-tile loads read each row at its stored
  // length d and fill the columns past it with 0, q is read and O written
  // at d.  A Q8 cache at d = 256 runs only through the pieces (the kernel
  // that splits staged Q8 tiles itself is built for 64 and 128).  Head dims
  // above 256 and even ones that are not multiples of 8 run as prefill rows
  // (prefill_rows).  Prompts with enough work, at any head dim, take the
  // 32-row kernels instead (prefill_on_pieces).
  const bool padded = !supported_d(d);
  const bool rows_path = prefill_by_rows(d, kv_dtype);
  const bool pieces_only = kv_dtype == MOLOT_KV_Q8 && d == 256;
  const int D = padded ? (d <= 64 ? 64 : d <= 128 ? 128 : 256) : d;
  if (M < 0 || N < 0 || pos0 < 0 || pos0 > kMaxPos - M || (M > 0 && (!Qm || !Om)))
    return MOLOT_EINVAL;
  if (M == 0) return 0;
  LaunchLock lock(g_launch_mu);
  if (N == 0) return zero_out(Om, (int64_t)M * nq * d, (hipStream_t)stream);
  if (!K || !V || !aligned16(K) || !aligned16(V) || !aligned16(Qm) || !aligned16(Om))
    return MOLOT_EINVAL;
  if (sc.on && M > 65535) {  // (the launches' grids) by parts
    constexpr int kPart = 32768;
    for (int m0 = 0; m0 < M; m0 += kPart) {
      Scoring part = sc;
      if (sc.key_lo) part.key_lo += m0;
      if (sc.key_hi) part.key_hi += m0;
      const int Mp = std::min(kPart, M - m0);
      const int Np = sc.key_hi ? N : (int)std::min<int64_t>(N, (int64_t)pos0 + m0 + Mp);
      const int64_t at = (int64_t)m0 * nq * d;
      st = attn_prefill_impl(Qm + at, K, V, Om + at, nq, nkv, Mp, Np, d, scale, pos0 + m0, window,
                             kv_dtype, block_row, page, part, stream, presplit, -1);
      if (st) return st;
    }
    return 0;
  }
  if (sc.on ? prefill_scored_pieces(d, M, N, nq, nkv, window, kv_dtype, sc, presplit)
            : prefill_takes_pieces(d, M, N, nq, nkv, kv_dtype, window, presplit)) {
    st = prefill_on_pieces(Qm, K, V, Om, nq, nkv, M, N, d, scale, pos0, window, kv_dtype, block_row,
                           page, sc, stream, split_rows);
    if (st != MOLOT_ENOWS) return st;
    split_rows = -1;
  }
  if (rows_path || sc.on)
    return prefill_rows(Qm, K, V, Om, nq, nkv, M, N, d, scale, pos0, window, kv_dtype, block_row,
                        page, sc, stream);
  const int64_t rows = (int64_t)M * (nq / nkv);
  auto nqb_of = [&](int w) { return (rows + 16 * w - 1) / (16 * w); };
  int pw = kPfWaves;
  int64_t nqb = nqb_of(pw);
  // A grid of fewer workgroups than CUs (few query rows over a long cache,
  // e.g. a prompt chunk after a long context) splits each query block's key
  // tiles over nsplit workgroups, at least 4 tiles each, and combine_kernel
  // merges their partials (slots: one query row of one head).
  int nsplit = 1;
  float* part = nullptr;
  if (nqb * nkv < num_cus() && (int64_t)M * nq <= 65535) {
    const int last = pos0 + M - 1;  // the query attending the most keys
    const int t0l = window > 0 && last - window + 1 > 0 ? std::min(last - window + 1, N) : 0;
    const int64_t tiles = (std::min(last + 1, N) - t0l + 31) / 32;
    const int64_t want = (num_cus() + nqb * nkv - 1) / (nqb * nkv);
    nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({16, want, tiles / 4}));
    if (nsplit > 1) {
      unsigned long long* ctr = nullptr;
      void* ws = nullptr;
      st = workspace(stream, sizeof(float) * (size_t)M * nq * nsplit * (D + 2), &ctr, &ws);
      if (st && st != MOLOT_ENOWS) return st;
      if (st) nsplit = 1;  // under capture the workspace cannot grow
      else part = reinterpret_cast<float*>(ws);
      st = 0;
    }
  }
  if (nsplit == 1 && pw == 8 && nqb * nkv < num_cus()) {
    pw = 4;  // no split: twice the workgroups on 4 waves
    nqb = nqb_of(4);
  }
  if (nqb * nkv * nsplit > (int64_t)0x7FFFFFFF) return MOLOT_ENOTSUP;
  PfArgs a{};
  a.q = Qm;
  a.k = K;
  a.v = V;
  a.o = Om;
  a.nq = nq;
  a.nkv = nkv;
  a.M = M;
  a.N = N;
  a.pos0 = pos0;
  a.window = window;
  a.nqb = (int)nqb;
  a.scale = scale;
  a.block_table = block_row;
  a.nsplit = nsplit;
  a.part_o = part;
  a.part_ml = part ? part + (size_t)M * nq * nsplit * D : nullptr;
  a.dh = d;
  if (block_row) {
    if (page <= 0 || (page & (page - 1)) || !q8_pages_ok(nkv, page, kv_dtype))
      return MOLOT_EINVAL;
    while ((1 << a.page_shift) < page) ++a.page_shift;
  }
  PfFn pk = pieces_only ? nullptr : pf_kernel(D, kv_dtype, block_row != nullptr, pw);
  if (!pk && !pieces_only) return MOLOT_ENOTSUP;
  // fp32 and Q8 caches: the attended keys as 16-bit pieces, which the
  // attention kernel copies into LDS, where a fresh prompt's step wrote them
  // (split_rows = 0), and at d = 256, split here.  Not under stream capture
  // when the workspace would have to grow, nor past kMaxPiecesBytes, nor at
  // d <= 128 where prefill_split_pays says no: the kernel then splits each
  // staged tile itself.
  if (D == 256 || split_rows == 0 || prefill_split_pays(M, N, nq, nkv, D, kv_dtype, window)) {
    void* ws = nullptr;
    int T0 = 0;
    int64_t R = 0;
    st = prefill_pieces(nkv, N, D, pos0, window, kv_dtype, stream, presplit, &ws, &T0, &R, pieces_only);
    if (st) return st;
    if (!ws && pieces_only) {
      if (R == 0) return zero_out(Om, (int64_t)M * nq * d, (hipStream_t)stream);  // no key attended
      // a capture that would have to grow them, or past the cap: the vector-
      // ALU kernel reads the Q8 rows itself
      return prefill_rows(Qm, K, V, Om, nq, nkv, M, N, d, scale, pos0, window, kv_dtype,
                          block_row, page, sc, stream);
    }
    if (ws) {
      a.pieces = reinterpret_cast<const uint16_t*>(ws);
      a.T0 = T0;
      a.R = (int)R;
      a.Rsplit = split_rows < 0 ? (int)R : (int)std::min<int64_t>(split_rows, R);
      if (a.Rsplit > 0) {
        const int64_t units = (int64_t)a.Rsplit * (D / 8);
        hipLaunchKernelGGL(pf_split(D, kv_dtype, block_row != nullptr),
                           dim3((unsigned)((units + 255) / 256), nkv, 2), dim3(256), 0,
                           (hipStream_t)stream, a, reinterpret_cast<uint16_t*>(ws));
        st = (int)hipGetLastError();
        if (st) return st;
      }
      pk = pf_kernel_pre(D, pw);
    }
  }
  const int pf_threads = 64 * pw;
  return launch_prefill(pk, nqb * nkv * nsplit, pf_threads, a, D, stream);
}

int molot_hip_attn_prefill_gqa(const float* Qm, const void* K, const void* V, float* Om, int nq,
                               int nkv, int M, int N, int d, float scale, int pos0, int window,
                               int kv_dtype, void* stream) {
  return attn_prefill_impl(Qm, K, V, Om, nq, nkv, M, N, d, scale, pos0, window, kv_dtype,
                           nullptr, 0, Scoring{}, stream,
                           g_presplit.load(std::memory_order_relaxed));
}

// A scored prefill's arguments.
static Scoring prefill_scoring(float softcap, const float* slopes, const int32_t* key_lo,
                               const int32_t* key_hi) {
  Scoring sc;
  sc.on = 1;
  sc.softcap = softcap;
  sc.slopes = slopes;
  sc.key_lo = key_lo;
  sc.key_hi = key_hi;
  return sc;
}

int molot_hip_attn_prefill_scored(const float* Qm, const void* K, const void* V, float* Om, int nq,
                                  int nkv, int M, int N, int d, float scale, int pos0, int window,
                                  float softcap, const float* slopes, const int32_t* key_lo,
                                  const int32_t* key_hi, int kv_dtype, void* stream) {
  return attn_prefill_impl(Qm, K, V, Om, nq, nkv, M, N, d, scale, pos0, window, kv_dtype,
                           nullptr, 0, prefill_scoring(softcap, slopes, key_lo, key_hi), stream,
                           g_presplit.load(std::memory_order_relaxed));
}

static int prefill_step_impl(float* q, const float* k_new, const float* v_new, void* K, void* V,
                             float* O, int nq, int nkv, int d, int M, int slot0, int pos0,
                             const float* q_norm, const float* k_norm, int v_norm, float eps,
                             const float* inv_freq, float scale, int window, int kv_dtype,
                             const int32_t* block_row, int page, int max_blocks,
                             const Scoring& sc, void* stream) {
  int st = check_common(nq, nkv, d, kv_dtype);
  if (st) return st;
  if (!scoring_ok(sc)) return MOLOT_EINVAL;
  // the prefill kernels' head dims, a multiple of 8 below 256 run padded, or
  // prefill rows (d > 256, not a multiple of 8, or a padded Q8 cache; see
  // attn_prefill_impl)
  const bool pieces_only = kv_dtype == MOLOT_KV_Q8 && d == 256;  // no per-tile kernel
  Norms nm;
  nm.q = q_norm;
  nm.k = k_norm;
  nm.v = v_norm ? 1 : 0;
  nm.eps = eps;
  if (!norms_ok(nm) || M < 0 || slot0 < 0 || pos0 < 0 || slot0 > kMaxPos - M || pos0 > kMaxPos - M)
    return MOLOT_EINVAL;
  if (M == 0) return 0;
  if (!q || !k_new || !v_new || !K || !V || !O) return MOLOT_EINVAL;
  if ((int64_t)M > 65535) return MOLOT_ENOTSUP;  // one grid row per token
  if (block_row && ((int64_t)slot0 + M > (int64_t)max_blocks * page || page <= 0 ||
                    (page & (page - 1)) || !q8_pages_ok(nkv, page, kv_dtype)))
    return MOLOT_EINVAL;
  LaunchLock lock(g_launch_mu);
  RopeArgs r{};
  r.q = q;
  r.k_new = k_new;
  r.v_new = v_new;
  r.K = K;
  r.V = V;
  r.inv_freq = inv_freq;
  if (block_row) {  // every token of the one sequence through its block-table row
    r.block_table = block_row;
    r.max_blocks = 0;
    r.page = page;
    paged_layout(r, nkv, d, page, kv_dtype);
  } else {
    token_major(r, nkv, d, kv_dtype);
  }
  r.nq = nq;
  r.nkv = nkv;
  r.d = d;
  r.slot = slot0;
  r.pos = pos0;
  r.kv_dtype = kv_dtype;
  r.append = 1;
  r.tokens = 1;
  r.q_norm = nm.q;
  r.k_norm = nm.k;
  r.v_norm = nm.v;
  r.eps = nm.eps;
  // the appended rows leave their pieces as they are stored; the split
  // kernel then covers only the cached rows before them, and a fresh prompt
  // needs no split launch (eager steps of 2048-token prompts: 32q/8kv/d128
  // fp32 252 -> 249 us, 8q/4kv/d256 window 1024 164.7 -> 161.6 us)
  void* pws = nullptr;
  int T0 = 0;
  int split_rows = -1;
  const int presplit = g_presplit.load(std::memory_order_relaxed);
  // (a row never sees the rows appended after it: where rows were evicted from the cache
  // the positions run ahead of the slots, and the attention goes by the slots)
  const int apos = std::min(pos0, slot0);
  if (sc.on ? prefill_scored_pieces(d, M, slot0 + M, nq, nkv, window, kv_dtype, sc, presplit)
            : prefill_takes_pieces(d, M, slot0 + M, nq, nkv, kv_dtype, window, presplit)) {
    // at d = 512 the split of all rows is as fast (8q/2kv, 1999 tokens: 29 + 7
    // us against 49 for a RoPE/append that leaves the pieces), and a scored step's of Q8
    // rows, whose marks cost the append as much (2048 tokens with a cap, split of all /
    // left by the append: 32q/8kv/d128 fp32 150.5 / 147.5, bf16 122.6 / 120.3, Q8 123.0 /
    // 124.1; 16q/4kv/d64 86.2 / 84.7, 76.2 / 75.5, 77.4 / 77.1)
    if ((d == 64 || d == 128) && !(sc.on && kv_dtype == MOLOT_KV_Q8)) {
      int R = 0;
      st = pieces32_workspace(nkv, slot0 + M, d, apos, window, kv_dtype, sc.on, stream, &pws, &T0,
                              &R);
      if (st && st != MOLOT_ENOWS) return st;
      if (!st) {
        r.pc_R = R;
        r.pc_np = wide_pieces(kv_dtype == MOLOT_KV_F32);
        r.own = sc.on;
      }
    }
  } else if (supported_d(d) && !sc.on) {
    int64_t R = 0;
    st = prefill_pieces(nkv, slot0 + M, d, apos, window, kv_dtype, stream, presplit, &pws, &T0, &R,
                        pieces_only);
    if (st) return st;
    r.pc_R = (int)R;
    // cached rows attended: split per tile where that is faster
    if (d <= 128 && slot0 > T0 && !prefill_split_pays(M, slot0 + M, nq, nkv, d, kv_dtype, window))
      pws = nullptr;
  }
  if (pws) {
    r.pieces = reinterpret_cast<uint16_t*>(pws);
    r.pc_T0 = T0;
    split_rows = std::max(0, slot0 - T0);
  }
  st = launch_rope_tok(r, M, stream);
  if (st) return st;
  return attn_prefill_impl(q, K, V, O, nq, nkv, M, slot0 + M, d, scale, apos, window, kv_dtype,
                           block_row, page, sc, stream, presplit, split_rows);
}

int molot_hip_prefill_step(float* q, const float* k_new, const float* v_new, void* K, void* V,
                           float* O, int nq, int nkv, int d, int M, int slot0, int pos0,
                           const float* q_norm, const float* k_norm, int v_norm, float eps,
                           const float* inv_freq, float scale, int window, int kv_dtype,
                           void* stream) {
  return prefill_step_impl(q, k_new, v_new, K, V, O, nq, nkv, d, M, slot0, pos0, q_norm, k_norm,
                           v_norm, eps, inv_freq, scale, window, kv_dtype, nullptr, 0, 0,
                           Scoring{}, stream);
}

int molot_hip_prefill_step_scored(float* q, const float* k_new, const float* v_new, void* K,
                                  void* V, float* O, int nq, int nkv, int d, int M, int slot0,
                                  int pos0, const float* q_norm, const float* k_norm, int v_norm,
                                  float eps, const float* inv_freq, float scale, int window,
                                  float softcap, const float* slopes, const int32_t* key_lo,
                                  const int32_t* key_hi, int kv_dtype, void* stream) {
  return prefill_step_impl(q, k_new, v_new, K, V, O, nq, nkv, d, M, slot0, pos0, q_norm, k_norm,
                           v_norm, eps, inv_freq, scale, window, kv_dtype, nullptr, 0, 0,
                           prefill_scoring(softcap, slopes, key_lo, key_hi), stream);
}

int molot_hip_prefill_step_paged(float* q, const float* k_new, const float* v_new, void* K,
                                 void* V, float* O, const int32_t* block_row, int max_blocks,
                                 int page, int nq, int nkv, int d, int M, int slot0, int pos0,
                                 const float* q_norm, const float* k_norm, int v_norm, float eps,
                                 const float* inv_freq, float scale, int window, int kv_dtype,
                                 void* stream) {
  if (!block_row || max_blocks <= 0) return MOLOT_EINVAL;
  return prefill_step_impl(q, k_new, v_new, K, V, O, nq, nkv, d, M, slot0, pos0, q_norm, k_norm,
                           v_norm, eps, inv_freq, scale, window, kv_dtype, block_row, page,
                           max_blocks, Scoring{}, stream);
}

int molot_hip_prefill_step_paged_scored(
    float* q, const float* k_new, const float* v_new, void* K, void* V, float* O,
    const int32_t* block_row, int max_blocks, int page, int nq, int nkv, int d, int M, int slot0,
    int pos0, const float* q_norm, const float* k_norm, int v_norm, float eps,
    const float* inv_freq, float scale, int window, float softcap, const float* slopes,
    const int32_t* key_lo, const int32_t* key_hi, int kv_dtype, void* stream) {
  if (!block_row || max_blocks <= 0) return MOLOT_EINVAL;
  return prefill_step_impl(q, k_new, v_new, K, V, O, nq, nkv, d, M, slot0, pos0, q_norm, k_norm,
                           v_norm, eps, inv_freq, scale, window, kv_dtype, block_row, page,
                           max_blocks, prefill_scoring(softcap, slopes, key_lo, key_hi), stream);
}

// Norm and RoPE of M rows of queries [M][nq][d] at positions pos0 + m, in
// place, no append (the RoPE/append kernel with its KV part off).
static int q_prologue(float* q, int nq, int d, int M, int pos0, const float* q_norm, float eps,
                      const float* inv_freq, void* stream) {
  if (nq < 0 || M < 0 || d <= 0 || (d & 1) || d > 2048 || pos0 < 0 || pos0 > kMaxPos - M)
    return MOLOT_EINVAL;
  if (!(eps >= 0.f && eps < INFINITY)) return MOLOT_EINVAL;
  if (nq == 0 || M == 0) return 0;
  if (!q) return MOLOT_EINVAL;
  if ((int64_t)M > 65535) return MOLOT_ENOTSUP;  // one grid row per token
  if (!q_norm && !inv_freq) return 0;            // nothing to apply
  RopeArgs r{};
  r.q = q;
  r.inv_freq = inv_freq;
  r.nq = nq;
  r.nkv = 1;
  r.d = d;
  r.pos = pos0;
  r.tokens = 1;
  r.q_norm = q_norm;
  r.eps = eps;
  return launch_rope_tok(r, M, stream);
}

int molot_hip_prefill_q(float* q, int nq, int d, int M, int pos0, const float* q_norm, float eps,
                        const float* inv_freq, void* stream) {
  return q_prologue(q, nq, d, M, pos0, q_norm, eps, inv_freq, stream);
}

int molot_hip_decode_step_shared(float* q, const void* K, const void* V, float* O, int nq,
                                 int nkv, int d, int n, int pos, const float* q_norm, float eps,
                                 const float* inv_freq, float scale, int window, int kv_dtype,
                                 void* stream) {
  int st = check_common(nq, nkv, d, kv_dtype);
  if (st) return st;
  if (!q || !K || !V || !O || n <= 0 || pos < 0) return MOLOT_EINVAL;  // n = 0: forward.h:580
  if (!(eps >= 0.f && eps < INFINITY)) return MOLOT_EINVAL;
  if (!aligned16(K) || !aligned16(V) || !aligned16(q) || !aligned16(O)) return MOLOT_EINVAL;
  int t0 = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
  if (t0 >= n) {  // nothing attended: q still gets its norm and RoPE, o = 0
    st = q_prologue(q, nq, d, 1, pos, q_norm, eps, inv_freq, stream);
    if (st) return st;
    return zero_out(O, (int64_t)nq * d, (hipStream_t)stream);
  }
  AttnArgs a{};
  a.q = q;
  a.q_out = q;
  a.k = const_cast<void*>(K);
  a.v = const_cast<void*>(V);
  a.inv_freq = inv_freq;
  a.o = O;
  token_major(a, nkv, d, kv_dtype);
  a.nq = nq;
  a.nkv = nkv;
  a.n = n;
  a.t0 = t0;
  a.pos = pos;
  a.window = window;
  a.scale = scale;
  a.q_norm = q_norm;
  a.eps = eps;
  a.fold = 0;  // all n slots are the source layer's; nothing appended
  return run_attn<false, true>(a, d, kv_dtype, n - t0, 1, stream);
}

int molot_hip_decode_step_paged_shared(float* q, const void* K, const void* V, float* O,
                                       const int32_t* block_table, const int32_t* seq_lens,
                                       const int32_t* pos, int B, int max_blocks, int max_seq_len,
                                       int nq, int nkv, int d, int page, const float* q_norm,
                                       float eps, const float* inv_freq, float scale, int window,
                                       int kv_dtype, void* stream) {
  if (!(eps >= 0.f && eps < INFINITY)) return MOLOT_EINVAL;
  AttnArgs a{};
  int span = 0;
  int st = paged_args(a, q, const_cast<void*>(K), const_cast<void*>(V), O, block_table, seq_lens,
                      pos, B, max_blocks, max_seq_len, nq, nkv, d, page, scale, window, kv_dtype,
                      &span);
  if (st) return st;
  if (B == 0) return 0;
  a.q_out = q;
  a.inv_freq = inv_freq;
  a.q_norm = q_norm;
  a.eps = eps;
  a.fold = 0;
  return run_attn<true, true>(a, d, kv_dtype, span, B, stream);
}

int molot_hip_attn_prefill_paged(const float* Qm, const void* K, const void* V, float* Om,
                                 const int32_t* block_row, int max_blocks, int page, int nq,
                                 int nkv, int M, int N, int d, float scale, int pos0, int window,
                                 int kv_dtype, void* stream) {
  if (!block_row || max_blocks <= 0 || N < 0 || (int64_t)N > (int64_t)max_blocks * page)
    return MOLOT_EINVAL;
  return attn_prefill_impl(Qm, K, V, Om, nq, nkv, M, N, d, scale, pos0, window, kv_dtype,
                           block_row, page, Scoring{}, stream,
                           g_presplit.load(std::memory_order_relaxed));
}

int molot_hip_attn_prefill_paged_scored(const float* Qm, const void* K, const void* V, float* Om,
                                        const int32_t* block_row, int max_blocks, int page, int nq,
                                        int nkv, int M, int N, int d, float scale, int pos0,
                                        int window, float softcap, const float* slopes,
                                        const int32_t* key_lo, const int32_t* key_hi,
                                        int kv_dtype, void* stream) {
  if (!block_row || max_blocks <= 0 || N < 0 || (int64_t)N > (int64_t)max_blocks * page)
    return MOLOT_EINVAL;
  return attn_prefill_impl(Qm, K, V, Om, nq, nkv, M, N, d, scale, pos0, window, kv_dtype,
                           block_row, page, prefill_scoring(softcap, slopes, key_lo, key_hi),
                           stream, g_presplit.load(std::memory_order_relaxed));
}

int molot_hip_vexp(const float* x, float* y, int64_t n, void* stream) {
  if (n < 0 || (n > 0 && (!x || !y))) return MOLOT_EINVAL;
  if (n == 0) return 0;
  const int64_t blocks = (n + 255) / 256;
  hipLaunchKernelGGL(vexp_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, x,
                     y, n);
  return (int)hipGetLastError();
}

int molot_hip_prob_exp(const float* x, float* y, int64_t n, void* stream) {
  if (n < 0 || (n > 0 && (!x || !y))) return MOLOT_EINVAL;
  if (n == 0) return 0;
  const int64_t blocks = (n + 255) / 256;
  hipLaunchKernelGGL(prob_exp_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                     x, y, n);
  return (int)hipGetLastError();
}

}  // extern "C"
