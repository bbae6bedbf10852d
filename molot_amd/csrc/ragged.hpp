// Ragged batches: what the kernels of ragged.hip and ragged_tile.hip share.
//
// A batch packs the new rows of B sequences, row_start[b] .. row_start[b + 1] - 1
// those of sequence b, which end its kv_lens[b] rows in the paged cache.  The query
// rows of one KV head and sequence are r = m*G + g: new row m, q head g of the
// group.  A tile is some consecutive rows r of one sequence, a unit a tile's part
// of its keys: what one workgroup computes for one KV head.
#ifndef MOLOT_AMD_CSRC_RAGGED_HPP_
#define MOLOT_AMD_CSRC_RAGGED_HPP_

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "device_util.hpp"
#include "molot_amd/attn_hip.h"
#include "prefill_tile.hpp"

// A launch's units, in the workspace, for the attention and the merge after it.
struct RaggedHead {
  int nunits, nparts, pad[2];
};
// The new rows of a sequence: first packed row, rows, and the slot of the first.
struct RaggedSeq {
  int start, rows, slot0;
};
struct RaggedUnit {
  int seq, r0;   // sequence, first row r of the tile
  int lo, hi;    // keys [lo, hi)
  int part;      // of a split tile: the unit's place in the partials (-1: whole)
  int split, nsplit;
  int wide;      // a wide tile
  RaggedSeq s;
  int rows;      // of the tile
};
static_assert(sizeof(RaggedUnit) == 48, "16-byte loads");

struct RaggedArgs {
  const float* q;  // [T][nq][d]
  const char* k;   // pages [num_blocks][nkv][page][d] (Q8: and scales)
  const char* v;
  float* o;        // [T][nq][d]
  const int32_t* block_table;  // [B][max_blocks]
  const int32_t* kv_lens;      // [B], the new rows counted
  const int32_t* row_start;    // [B + 1]
  int T, B, max_blocks, num_blocks;
  int cap;  // slots of a sequence at most
  int nq, nkv, G, d, page_shift, window, kv_dtype;
  float scale, softcap;
  const float* slopes;
  RaggedHead* head;
  RaggedUnit* units;
  int32_t* tiles;   // [B + 1][2]: wide and narrow tiles of the sequences before
  int32_t* part_unit;  // the unit of every part
  float* part_o;    // [part][nkv][slot_rows][D] unnormalised o
  float* part_ml;   // [part][nkv][slot_rows][2] (max in base 2, sum)
  int slot_rows;    // rows of a partial's slot
  // Tiles: of ql rows r, and for the last `few` of a sequence narrow ones (ragged_slim).
  // Units: up to `target` of them (a KV head) beyond one a tile, of at least min_keys keys;
  // a key costs a wide tile `weight` times a narrow one's.
  int qs, ql, few, target, min_keys, weight;
  int max_units, max_parts;
};

// The matrix-core kernel of a head dim (a multiple of 8 up to 256) and cache type, and
// the threads of its workgroups.
using RaggedFn = void (*)(RaggedArgs);
struct RaggedTile {
  RaggedFn fn;
  int threads, wide, narrow;  // (rows of its tiles)
};
RaggedTile ragged_tile(int d, int kv_dtype, bool scored) __attribute__((visibility("hidden")));

namespace {

// The new rows of sequence b as the kernels take them, whatever the arrays hold.
__device__ __forceinline__ RaggedSeq ragged_seq(const RaggedArgs& a, int b) {
  const int s0 = max(0, min(a.row_start[b], a.T));
  const int s1 = max(s0, min(a.row_start[b + 1], a.T));
  const int n = max(0, min(a.kv_lens[b], a.max_blocks << a.page_shift));
  return {s0, s1 - s0, n - (s1 - s0)};
}
// Rows of the narrow tiles that a sequence of R rows r ends in: 16, or where more are left
// the most that one takes (two tiles would read and convert every key twice).
constexpr int kSlimRows = 16;
__device__ __forceinline__ int ragged_slim(const RaggedArgs& a, int R) {
  return R % a.ql > kSlimRows ? a.qs : kSlimRows;
}
// The keys [lo, hi) of the query row at `slot` (< 0: none).
__device__ __forceinline__ int ragged_lo(const RaggedArgs& a, int slot) {
  return a.window > 0 && slot - a.window + 1 > 0 ? min(slot - a.window + 1, a.cap) : 0;
}
__device__ __forceinline__ int ragged_hi(const RaggedArgs& a, int slot) {
  return max(0, min(slot + 1, a.cap));
}
// The block of slot t of sequence b; ids out of the pool read its first block.
__device__ __forceinline__ int ragged_block(const RaggedArgs& a, int b, int t) {
  const int id = a.block_table[(int64_t)b * a.max_blocks + (t >> a.page_shift)];
  return (unsigned)id < (unsigned)a.num_blocks ? id : 0;
}
// Elements (Q8: bytes) of row t of KV head h from the pool's start, and a Q8 row's scale.
template <typename T>
__device__ __forceinline__ int64_t ragged_row_of(const RaggedArgs& a, int blk, int h, int t,
                                                 int64_t& scale) {
  const int page = 1 << a.page_shift, sl = t & (page - 1);
  if constexpr (!std::is_same<T, q8_t>::value)
    return (((int64_t)blk * a.nkv + h) * page + sl) * a.d;
  const int64_t rows = (int64_t)a.nkv * page, b0 = (int64_t)blk * rows * (a.d + 4);
  scale = b0 + rows * a.d + 4 * ((int64_t)h * page + sl);
  return b0 + ((int64_t)h * page + sl) * a.d;
}

// The scores past the product of query row r (head h*G + g) at its slot.
__device__ __forceinline__ RowScore ragged_score(const RaggedArgs& a, int head, int slot) {
  return row_score_of(a, a.slopes ? a.slopes[head] * kLog2e : 0.f, slot);
}

// Query row r of a unit by one wave, over the row's own keys alone: lanes over the head
// dim (elements lane + 64*i), NK keys in flight.  To O, or to the unit's partials.
// The rows of ragged_valu_kernel, and of the matrix-core kernel those over cached rows
// that its pieces cannot hold (infinities, NaN): a row that they do not belong to is
// not reached by them.
template <int EPL, typename T>
__device__ __forceinline__ void ragged_own_row(const RaggedArgs& a, const RaggedUnit& u, int h, int r) {
  constexpr int D = 64 * EPL, NK = 4;
  constexpr bool Q8 = std::is_same<T, q8_t>::value;
  const int lane = threadIdx.x & 63;
  const RaggedSeq& s = u.s;
  if (r >= s.rows * a.G) return;
  const int m = r / a.G, g = r - m * a.G, slot = s.slot0 + m, head = h * a.G + g;
  const int lo = max(ragged_lo(a, slot), u.lo), hi = min(ragged_hi(a, slot), u.hi);
  // (lanes past d read the row's last element, so that no load waits for a branch)
  auto elem = [&](const char* base, int64_t off, int e) {
    const int64_t i = off + min(e, a.d - 1);
    float x;
    if constexpr (Q8) x = (float)reinterpret_cast<const int8_t*>(base)[i];
    else if constexpr (std::is_same<T, bf16_t>::value)
      x = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(base)[i] << 16);
    else x = reinterpret_cast<const float*>(base)[i];
    return e < a.d ? x : 0.f;
  };
  const RowScore score = ragged_score(a, head, slot);
  const int64_t at = ((int64_t)(s.start + m) * a.nq + head) * a.d;
  float q[EPL], o[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    q[i] = lane + 64 * i < a.d ? a.q[at + lane + 64 * i] : 0.f;
    o[i] = 0.f;
  }
  const float qsc = a.scale * kLog2e;
  float mx = -INFINITY, l = 0.f;
  for (int t0 = lo; t0 < hi; t0 += NK) {
    float x[NK], k[NK][EPL], v[NK][EPL], ks[NK], vs[NK];
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int t = min(t0 + j, hi - 1);
      int64_t sc = 0;
      const int64_t off = ragged_row_of<T>(a, ragged_block(a, u.seq, t), h, t, sc);
      ks[j] = Q8 ? *reinterpret_cast<const float*>(a.k + sc) : 1.f;
      vs[j] = Q8 ? *reinterpret_cast<const float*>(a.v + sc) : 1.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        k[j][i] = elem(a.k, off, lane + 64 * i);
        v[j][i] = elem(a.v, off, lane + 64 * i);
      }
    }
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) dot = fmaf(q[i], k[j][i], dot);
      x[j] = wave_reduce<false>(dot) * (ks[j] * qsc);
    }
    float raw[NK];
#pragma unroll
    for (int j = 0; j < NK; ++j) raw[j] = x[j];
    score.apply<NK>(x, [&](int j) { return t0 + j; }, [&](int j) { return raw[j]; });
    float mn = mx;
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      if (t0 + j >= hi) x[j] = -INFINITY;
      mn = fmaxf(mn, x[j]);
    }
    if (mn > mx) {
      const float f = exp2_hw(mx - mn);
      l *= f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) o[i] *= f;
      mx = mn;
    }
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      if (t0 + j >= hi) break;
      const float p = x[j] == -INFINITY ? 0.f : exp2_hw(x[j] - mx);
      l += p;
#pragma unroll
      for (int i = 0; i < EPL; ++i) o[i] = fmaf(p, Q8 ? v[j][i] * vs[j] : v[j][i], o[i]);
    }
  }
  if (u.part >= 0) {
    const int64_t ps = ((int64_t)u.part * a.nkv + h) * a.slot_rows + (r - u.r0);
#pragma unroll
    for (int i = 0; i < EPL; ++i) a.part_o[ps * D + lane + 64 * i] = o[i];
    if (lane == 0) {  // (a NaN sum stays one through the merge)
      a.part_ml[2 * ps] = mx > -INFINITY || l == 0.f ? mx : 0.f;
      a.part_ml[2 * ps + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no key: O = 0
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (lane + 64 * i < a.d) a.o[at + lane + 64 * i] = o[i] * inv;
}

}  // namespace

#endif  // MOLOT_AMD_CSRC_RAGGED_HPP_
