// The prefill attention launch shared by its kernel sources.
#ifndef MOLOT_AMD_CSRC_PREFILL_HPP_
#define MOLOT_AMD_CSRC_PREFILL_HPP_

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

struct PfArgs {
  const float* q;  // [M][nq][D]
  const void* k;   // token-major cache [N][nkv*D], or pages [block][nkv][page][D]
  const void* v;
  float* o;        // [M][nq][D]
  const int32_t* block_table;  // paged: the sequence's row of block ids
  int nq, nkv, M, N, pos0, window, nqb;  // nqb: blocks of 16 * (waves) query rows per KV head
  int dh;  // head dim as stored (< D: the launch runs padded to D, through the pieces)
  int page_shift;
  float scale;
  // 32-row kernels: a query row's output depends on the keys it attends alone
  // (own_mark, below); the cache type then says how to read them
  int own, kv_dtype;
  // the attended keys [T0, T0 + R) of every KV head split into 16-bit pieces
  // once for the launch (pf_split_kernel): [K, V][nkv][3 pieces][R][D]; NULL:
  // the kernel splits each staged tile itself
  const uint16_t* pieces;
  int T0, R;
  int Rsplit;  // pf_split_kernel splits rows [T0, T0 + Rsplit); the appending step wrote the rest
  // split-K over the key tiles (nsplit > 1): split s of a query block takes
  // its share of the tiles and writes unnormalised o and (max, sum) per query
  // row, slot m*nq + head, to part_o [slot][nsplit][D] and part_ml
  // [slot][nsplit][2]; combine_kernel merges them into O
  int nsplit;
  float* part_o;
  float* part_ml;
  // Scored launches of the 32-row kernels (their SC instances): the scores and the
  // rows' key ranges as AttnArgs has them
  float softcap;
  const float* slopes;
  const int32_t* key_lo;
  const int32_t* key_hi;
  int some;  // a block of few tiles takes fewer than nsplit splits (block_splits)
};

using PfFn = void (*)(PfArgs);
using SplitFn = void (*)(PfArgs, uint16_t*);

namespace {

// Rows that the pieces cannot hold for every query row alike.  A product over a
// tile takes each of its keys for all its query rows, a masked one times zero:
// a non-finite V row reaches rows that do not attend it, and a K row's infinity
// leaves no score of its sign.  Where each query row used to read its own keys
// alone (head dims above 256 and those that are not multiples of 8, Q8 at any
// padded one: PfArgs::own) the split marks such rows, and those out of the
// units' range, by a NaN unit, and a workgroup that met one forms its rows'
// results again from the cache (own_rows, prefill_tile.hpp).
constexpr float kOwnMaxK = 3.0e23f;   // 2^78: past it a raw score times its unit may overflow
constexpr float kOwnMinV = 7.9e-31f;  // 2^-100: below it a V row's unit keeps fewer bits
__device__ __forceinline__ float own_mark(float xmax, float nonfinite, int kv) {
  const bool out = kv ? xmax > 0.f && xmax < kOwnMinV : xmax > kOwnMaxK;
  return out ? NAN : nonfinite;  // 0, or NaN
}

}  // namespace

#endif  // MOLOT_AMD_CSRC_PREFILL_HPP_
