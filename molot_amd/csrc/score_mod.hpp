// Attention scores past the dot product: a cap by tanh and a bias by distance.
#ifndef MOLOT_AMD_CSRC_SCORE_MOD_HPP_
#define MOLOT_AMD_CSRC_SCORE_MOD_HPP_

#include <hip/hip_runtime.h>

#include "device_util.hpp"

namespace {

// Scores s in base-2 units (times log2 e) to c * tanh(s / c), c = cap * log2 e.
//
// With x = s / c, c * tanh(x) = s + s * x^2 * P(x^2): near 0 the result keeps s's
// own bits, where cap * tanh(s / cap) would lose some to a division and two more
// roundings.  P is of degree 4, fitted for this bound (least squares, reweighted
// until the relative errors were even) on |x| < 0.625: within 8.8e-9 of tanh,
// relatively (fp32's half step is 6.0e-8).  Past it c * (1 - 2 / (1 + e^(2|x|))), whose subtraction
// loses at most a bit there.  It is formed only where a lane of the wave has such
// a score: the scores of capped layers are mostly some tenths of the cap.  An
// infinity ends at +-c, a NaN stays one.
constexpr float kCapSmall = 0.625f;
__device__ __forceinline__ float cap_near(float s, float rcap) {
  const float x = s * rcap, y = x * x;
  float p = fmaf(-0.00570497056f, y, 0.0206390712f);
  p = fmaf(p, y, -0.0537397079f);
  p = fmaf(p, y, 0.133314416f);
  p = fmaf(p, y, -0.333332807f);
  return fmaf(s * y, p, s);
}
// (near: cap_near(s).  A NaN takes the series, and stays one; an infinity's reciprocal is 0.)
__device__ __forceinline__ float cap_any(float s, float near, float cap2, float rcap) {
  const float x = fabsf(s * rcap);
  const float e = exp2_hw(x * (2.f * kLog2e));
  const float far = copysignf(fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + e), cap2), s);
  return x >= kCapSmall ? far : near;
}
// again(i): s[i] as it came, formed a second time: a copy of the scores kept for the far
// ones would cost the near ones, in place, a move each.
template <int N, typename AGAIN>
__device__ __forceinline__ void cap_scores(float (&s)[N], float cap2, float rcap, AGAIN&& again) {
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) big = fmaxf(big, fabsf(s[i]));
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = cap_near(s[i], rcap);
  if (__builtin_amdgcn_ballot_w64(big * rcap >= kCapSmall) != 0) {  // wave-uniform
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = cap_any(again(i), s[i], cap2, rcap);
  }
}
template <int N>
__device__ __forceinline__ void cap_scores(float (&s)[N], float cap2, float rcap) {
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) big = fmaxf(big, fabsf(s[i]));
  if (__builtin_amdgcn_ballot_w64(big * rcap >= kCapSmall) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = cap_near(s[i], rcap);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = cap_any(s[i], cap_near(s[i], rcap), cap2, rcap);
}

}  // namespace

#endif  // MOLOT_AMD_CSRC_SCORE_MOD_HPP_
