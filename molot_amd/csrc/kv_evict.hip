// Eviction from a KV cache by accumulated attention weight.
//
// Per KV head, `keep` of n slots stay: first the slots whose position is among the
// `recent` newest (slot_pos > pos - recent), then those of the highest acc, ties
// to the lowest slot.  The slots that stay and lie past keep move, in order, into
// the ones before it that do not, in order: a cache cut by a few rows moves only
// those, in place, and no row is read and written by the same launch (sources lie
// at or past keep, destinations before it).  Attention does not ask for an order
// of the rows: a row's position is in its rotated key.
//
// Two launches: evict_select_kernel finds each head's moves, evict_move_kernel
// makes them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "attn_host.hpp"
#include "device_util.hpp"
#include "molot_amd/attn_hip.h"

namespace {

using namespace molot_host;

// The slots of a cache: rows, acc and slot_pos.
struct SlotArgs {
  char* k;
  char* v;
  float* acc;
  int32_t* slot_pos;
  const int32_t* block_table;  // NULL: contiguous
  const int32_t* seq_lens;
  const int32_t* pos_arr;
  int nkv, n, pos, acc_cap, max_blocks, page_shift;
  int limit;                   // rows of a sequence at most
  // Bytes: a token's, a head's and a block's stride, a head row's length; Q8: of
  // its scale's place and of the stride between heads' scales (AttnArgs::sc_off)
  int64_t tok, head, block, row;
  int64_t sc_off, sc_head, sc_tok;
  int q8;
};

__device__ __forceinline__ int rows_of(const SlotArgs& a, int b) {
  return a.block_table ? max(0, min(a.seq_lens[b], a.limit)) : a.n;
}
__device__ __forceinline__ int newest_of(const SlotArgs& a, int b, int n) {
  return !a.block_table ? a.pos : a.pos_arr ? a.pos_arr[b] : n - 1;
}
// Index of slot t of KV head h in acc and slot_pos.
__device__ __forceinline__ int64_t slot_index(const SlotArgs& a, int b, int h, int t) {
  if (!a.block_table) return (int64_t)h * a.acc_cap + t;
  const int64_t blk = a.block_table[(int64_t)b * a.max_blocks + (t >> a.page_shift)];
  return ((blk * a.nkv + h) << a.page_shift) + (t & ((1 << a.page_shift) - 1));
}

// The last M rows of each sequence are new: acc 0, positions up to the newest's.
__global__ __launch_bounds__(256) void kv_track_kernel(SlotArgs a, int M) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int n = rows_of(a, b);
  const int t = n - 1 - (int)(blockIdx.x * 256 + threadIdx.x);
  if (t < 0 || t < n - M) return;
  const int64_t i = slot_index(a, b, h, t);
  a.acc[i] = 0.f;
  if (a.slot_pos) a.slot_pos[i] = newest_of(a, b, n) - (n - 1 - t);
}

// acc as an unsigned number of the same order (-0 as 0); a NaN is above every
// number, and a recent slot above that.
__device__ __forceinline__ uint32_t slot_key(float acc, bool recent) {
  if (recent) return 0xFFFFFFFFu;
  if (acc != acc) return 0xFFFFFFFEu;
  const uint32_t u = __float_as_uint(acc + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

// Sum over the workgroup's waves of 1 to 3 wave-uniform counts (c[i] of every
// wave), in every lane.  buf: kSelWaves ints a count; the caller alternates two of
// them from call to call, so that one barrier is enough.
template <int N>
__device__ __forceinline__ void count_all(int (&c)[N], int* buf) {
  static_assert(N >= 1 && N <= 3, "16 lanes a count");
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[i * kSelWaves + w] = c[i];
  }
  lds_barrier();
  int x = lane < N * kSelWaves ? buf[lane] : 0;
#pragma unroll
  for (int off = 1; off < 16; off *= 2) x += __shfl_xor(x, off);
#pragma unroll
  for (int i = 0; i < N; ++i) c[i] = __builtin_amdgcn_readlane(x, 16 * i);
}
// The sum of one count over the waves before this one, and over all.
__device__ __forceinline__ void count_before(int c, int* buf, int& before, int& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (lane == 0) buf[w] = c;
  lds_barrier();
  const int x = lane < kSelWaves ? buf[lane] : 0;
  int y = lane < w ? x : 0, z = x;
#pragma unroll
  for (int off = 1; off < 16; off *= 2) {
    y += __shfl_xor(y, off);
    z += __shfl_xor(z, off);
  }
  before = __builtin_amdgcn_readlane(y, 0);
  all = __builtin_amdgcn_readlane(z, 0);
}

// Keys of a thread: K of them, wave w's i-th of slot first + (w * K + i) * 64 + lane,
// so that the waves, their steps and the lanes run in slot order; absent ones are 0,
// below every key of a slot (those are of numbers >= -NaN's image, at least 1).
template <int K>
struct Keys {
  uint32_t k[K];
  __device__ __forceinline__ static int slot(int i) {
    return ((int)(threadIdx.x >> 6) * K + i) * 64 + (int)(threadIdx.x & 63);
  }
  // How many are at least t, in this wave.
  __device__ __forceinline__ int at_least(uint32_t t) const {
    int c = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) c += __popcll(__builtin_amdgcn_ballot_w64(k[i] >= t));
    return c;
  }
};

// The `want`-th largest of the workgroup's keys, two bits a step from bit 31 (top:
// the bits above `from` are known): the largest T that at least want keys reach.
// Each step counts three candidates, whatever the keys are; a radix pass's counters
// would meet most lanes of a wave in a few bins (weights of a few exponents).
template <int K>
__device__ __forceinline__ uint32_t kth_largest(const Keys<K>& keys, uint32_t top, int from,
                                                int want, int* buf) {
  uint32_t T = top;
  for (int s = from; s >= 0; s -= 2) {
    const uint32_t one = 1u << s;
    int c[3] = {keys.at_least(T + one), keys.at_least(T + 2 * one), keys.at_least(T + 3 * one)};
    count_all<3>(c, buf + ((s >> 1) & 1) * 3 * kSelWaves);
    T += c[2] >= want ? 3 * one : c[1] >= want ? 2 * one : c[0] >= want ? one : 0u;
  }
  return T;
}

// A row move: the units of a row of K and V that this thread takes.  U: bytes of a
// unit (16 where rows are whole units, else 4).
template <int U>
struct Unit;
template <>
struct Unit<16> {
  using type = u32x4;
};
template <>
struct Unit<4> {
  using type = uint32_t;
};

__device__ __forceinline__ int64_t row_offset(const SlotArgs& a, int b, int h, int t, int64_t& sc) {
  if (!a.block_table) {
    sc = (int64_t)t * a.tok + a.sc_off + h * a.sc_head;
    return (int64_t)t * a.tok + h * a.head;
  }
  const int64_t blk = a.block_table[(int64_t)b * a.max_blocks + (t >> a.page_shift)];
  const int sl = t & ((1 << a.page_shift) - 1);
  sc = blk * a.block + a.sc_off + h * a.sc_head + sl * a.sc_tok;
  return blk * a.block + h * a.head + sl * a.tok;
}

// Moves [first, count) of the lists, step `threads` (this thread's number tid of
// them): K and V rows, their scales, acc and slot_pos.  Flat over (move, unit), R
// units a thread in flight.
template <int U, int R>
__device__ __forceinline__ void move_rows(const SlotArgs& a, int b, int h, const int32_t* dst,
                                          const int32_t* src, int count, int tid, int threads) {
  using T = typename Unit<U>::type;
  const int upr = (int)(a.row / U);
  const int total = count * upr;  // (a launch's lists are bounded: launch_evict)
  for (int u0 = tid; u0 < total; u0 += R * threads) {
    T kx[R], vx[R];
    int64_t to[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int u = u0 + r * threads;
      if (u >= total) break;
      const int i = u / upr, j = u - i * upr;
      int64_t sto, sat;
      const int64_t at = row_offset(a, b, h, src[i], sat) + (int64_t)j * U;
      to[r] = row_offset(a, b, h, dst[i], sto) + (int64_t)j * U;
      kx[r] = *reinterpret_cast<const T*>(a.k + at);
      vx[r] = *reinterpret_cast<const T*>(a.v + at);
      if (j == 0) {
        if (a.q8) {
          *reinterpret_cast<float*>(a.k + sto) = *reinterpret_cast<const float*>(a.k + sat);
          *reinterpret_cast<float*>(a.v + sto) = *reinterpret_cast<const float*>(a.v + sat);
        }
        const int64_t ito = slot_index(a, b, h, dst[i]), iat = slot_index(a, b, h, src[i]);
        a.acc[ito] = a.acc[iat];
        a.slot_pos[ito] = a.slot_pos[iat];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (u0 + r * threads >= total) break;
      *reinterpret_cast<T*>(a.k + to[r]) = kx[r];
      *reinterpret_cast<T*>(a.v + to[r]) = vx[r];
    }
  }
}

// The moves among a workgroup's slots, whose first is `first`: of the slots with key
// > T or, the first `ties` of them in slot order from number eq0 on, == T, those at
// or past keep (lo false), or of the others those before it (lo), to list[at ..].
// Returns how many.  buf: 2 * kSelWaves ints.
template <int K>
__device__ __forceinline__ int list_slots(const Keys<K>& keys, int first, int n, int keep, uint32_t T,
                                          int ties, int eq0, bool want_holes, bool want_moves,
                                          int32_t* holes, int32_t* moves, int hole0, int move0,
                                          int most, int* buf, int& nmoves) {
  const int lane = threadIdx.x & 63;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  int eqs = 0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const bool in = first + Keys<K>::slot(i) < n;
    eqs += __popcll(__builtin_amdgcn_ballot_w64(in && keys.k[i] == T));
  }
  int eq_at, all;
  count_before(eqs, buf, eq_at, all);
  eq_at += eq0;
  uint64_t hm[K], mm[K];  // a step's holes and moves, a bit a lane
  int ch = 0, cm = 0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int t = first + Keys<K>::slot(i);
    const bool in = t < n;
    const bool eq = in && keys.k[i] == T;
    const uint64_t be = __builtin_amdgcn_ballot_w64(eq);
    const bool stays = in && (keys.k[i] > T || (eq && eq_at + __popcll(be & below) < ties));
    eq_at += __popcll(be);
    hm[i] = __builtin_amdgcn_ballot_w64(in && t < keep && !stays);
    mm[i] = __builtin_amdgcn_ballot_w64(t >= keep && stays);
    ch += __popcll(hm[i]);
    cm += __popcll(mm[i]);
  }
  int h_at, m_at, nh;
  count_before(ch, buf + kSelWaves, h_at, nh);
  lds_barrier();
  count_before(cm, buf, m_at, nmoves);
  h_at += hole0;
  m_at += move0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int t = first + Keys<K>::slot(i);
    // (as many moves as holes; the bound holds whatever another stream does to acc)
    const int hi = h_at + __popcll(hm[i] & below), mi = m_at + __popcll(mm[i] & below);
    if (want_holes && (hm[i] >> lane & 1) && hi < most) holes[hi] = t;
    if (want_moves && (mm[i] >> lane & 1) && mi < most) moves[mi] = t;
    h_at += __popcll(hm[i]);
    m_at += __popcll(mm[i]);
  }
  return nh;
}

// Sequences of at most 1024 K rows: a workgroup a (KV head, sequence) holds the
// keys in registers.  FUSE: it makes the moves too (lists in LDS, most <=
// kFuseMoves); else the lists go to evict_move_kernel.
constexpr int kFuseMoves = 2048;
constexpr int64_t kFuseBytes = 32 * 1024;  // of K (and of V) a head

template <int K, bool FUSE>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(SlotArgs a, int keep, int recent,
                                                                   int most, int32_t* counts,
                                                                   int32_t* lists, int unit16) {
  const int h = blockIdx.x, b = blockIdx.y;
  const int n = rows_of(a, b);
  const int64_t pair = (int64_t)b * a.nkv + h;
  if (n <= keep) {
    if (!FUSE && threadIdx.x == 0) counts[pair] = 0;
    return;
  }
  const int oldest = newest_of(a, b, n) - recent;  // recent: past it
  Keys<K> keys;
  float x[K];
  int32_t p[K];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int64_t j = slot_index(a, b, h, min(Keys<K>::slot(i), n - 1));
    x[i] = a.acc[j];
    p[i] = a.slot_pos[j];
  }
#pragma unroll
  for (int i = 0; i < K; ++i) keys.k[i] = Keys<K>::slot(i) < n ? slot_key(x[i], p[i] > oldest) : 0u;
  __shared__ int buf[6 * kSelWaves];
  __shared__ int32_t own[FUSE ? 2 * kFuseMoves : 1];
  const uint32_t T = kth_largest<K>(keys, 0u, 30, keep, buf);
  int more[1] = {keys.at_least(T + 1u)};  // (T + 1 of the largest key, all recent: 0, none past it)
  if (T == 0xFFFFFFFFu) more[0] = 0;
  lds_barrier();
  count_all<1>(more, buf);
  lds_barrier();
  int32_t* dst = FUSE ? own : lists + pair * 2 * most;
  int32_t* src = dst + (FUSE ? kFuseMoves : most);
  int nm;
  const int nh = list_slots<K>(keys, 0, n, keep, T, keep - more[0], 0, true, true, dst, src, 0, 0, most,
                               buf, nm);
  const int moves = min(min(nm, nh), most);
  if constexpr (FUSE) {
    __syncthreads();
    if (unit16)
      move_rows<16, 2>(a, b, h, dst, src, moves, threadIdx.x, kSelThreads);
    else
      move_rows<4, 2>(a, b, h, dst, src, moves, threadIdx.x, kSelThreads);
  } else if (threadIdx.x == 0) {
    counts[pair] = moves;
  }
}

// The listed moves; grid (workgroups a pair, KV heads, sequences).
template <int U>
__global__ __launch_bounds__(256) void evict_move_kernel(SlotArgs a, int most, const int32_t* counts,
                                                         const int32_t* lists) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t pair = (int64_t)b * a.nkv + h;
  const int32_t* dst = lists + pair * 2 * most;
  move_rows<U, 4>(a, b, h, dst, dst + most, counts[pair], blockIdx.x * 256 + threadIdx.x,
                  gridDim.x * 256);
}

// ---------------------------------------------------------------------------
// Longer sequences: chunks of kChunk slots, a workgroup each, on either side of
// keep (so that a chunk has holes or moves, never both): nlo of [0, keep), then
// nhi of [keep, n).
//   evict_keys_kernel   a chunk's keys, and its counts of their top kTopBits bits;
//   evict_pick_kernel   the bin of the keep-th largest key from all chunks' counts
//                       (summed again by every chunk: they are small), then the
//                       chunk's keys above the bin counted, those in it listed;
//   evict_rank_kernel   a workgroup a (KV head, sequence): T among the listed keys,
//                       and where each chunk's equals and list entries start;
//   evict_list_kernel   the chunks' holes and moves.
constexpr int kChunkK = 8, kChunk = kSelThreads * kChunkK;
constexpr int kTopBits = 12, kBins = 1 << kTopBits, kLowBits = 32 - kTopBits;
static_assert(kLowBits % 2 == 0 && kBins == 4 * kSelThreads, "two bits a step; four bins a thread");
constexpr int kRankK = 16;  // listed keys a thread keeps in registers

struct LongArgs {
  SlotArgs s;
  int keep, recent, most, nlo, nhi;
  uint32_t* keys;      // [pair][chunks][kChunk]
  uint32_t* listed;    // [pair][chunks][kChunk]: the keys of the bin
  uint16_t* bins;      // [pair][chunks][kBins]
  int32_t* chunk_at;   // [pair][chunks][4]: keys above the bin, listed; then equals and entries before
  int32_t* rank;       // [pair][4]: bin, still wanted in it, T, equals that stay
  int32_t* counts;     // [pair]
  int32_t* lists;      // [pair][2][most]
};

// First slot and end of chunk c of a sequence of n rows.
__device__ __forceinline__ void chunk_range(const LongArgs& g, int n, int c, int& first, int& end) {
  const bool lo = c < g.nlo;
  first = lo ? c * kChunk : g.keep + (c - g.nlo) * kChunk;
  end = min(first + kChunk, lo ? min(g.keep, n) : n);
}

__global__ __launch_bounds__(kSelThreads) void evict_keys_kernel(LongArgs g) {
  const SlotArgs& a = g.s;
  const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, nc = g.nlo + g.nhi;
  const int n = rows_of(a, b);
  if (n <= g.keep) return;
  int first, end;
  chunk_range(g, n, c, first, end);
  const int64_t pair = (int64_t)b * a.nkv + h;
  __shared__ int hist[kBins];
  for (int i = threadIdx.x; i < kBins; i += kSelThreads) hist[i] = 0;
  const int oldest = newest_of(a, b, n) - g.recent;
  float x[kChunkK];
  int32_t p[kChunkK];
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int64_t j = slot_index(a, b, h, min(first + Keys<kChunkK>::slot(i), n - 1));
    x[i] = a.acc[j];
    p[i] = a.slot_pos[j];
  }
  __syncthreads();
  uint32_t* keys = g.keys + (pair * nc + c) * kChunk;
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int t = Keys<kChunkK>::slot(i);
    if (first + t >= end) continue;
    const uint32_t k = slot_key(x[i], p[i] > oldest);
    keys[t] = k;
    atomicAdd(&hist[k >> kLowBits], 1);
  }
  __syncthreads();
  uint16_t* bins = g.bins + (pair * nc + c) * kBins;
  for (int i = threadIdx.x; i < kBins; i += kSelThreads) bins[i] = (uint16_t)hist[i];
}

__global__ __launch_bounds__(kSelThreads) void evict_pick_kernel(LongArgs g) {
  const SlotArgs& a = g.s;
  const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, nc = g.nlo + g.nhi, tid = threadIdx.x;
  const int n = rows_of(a, b);
  const int64_t pair = (int64_t)b * a.nkv + h;
  if (n <= g.keep) return;
  // bins 4 tid .. 4 tid + 3 over the chunks; then the sums of the bins above
  __shared__ int buf[6 * kSelWaves];
  __shared__ int pick[2];
  const uint32_t* bins = reinterpret_cast<const uint32_t*>(g.bins + pair * nc * kBins) + 2 * tid;
  int cnt[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (int i = 0; i < nc; ++i) {  // (a chunk of no slots has counts of 0)
    const uint32_t x = bins[(int64_t)i * (kBins / 2)], y = bins[(int64_t)i * (kBins / 2) + 1];
    cnt[0] += (int)(x & 0xFFFFu);
    cnt[1] += (int)(x >> 16);
    cnt[2] += (int)(y & 0xFFFFu);
    cnt[3] += (int)(y >> 16);
  }
  const int lane = tid & 63;
  const int mine = cnt[0] + cnt[1] + cnt[2] + cnt[3];
  int up = mine;  // this lane's and the lanes' after it
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int y = __shfl_down(up, off);
    if (lane + off < 64) up += y;
  }
  const int wave = __builtin_amdgcn_readlane(up, 0);
  int before, all;
  count_before(wave, buf, before, all);
  int above = all - before - wave + up - mine;  // keys of the bins above this thread's
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    if (above < g.keep && above + cnt[i] >= g.keep) {  // one bin of all
      pick[0] = 4 * tid + i;
      pick[1] = g.keep - above;
    }
    above += cnt[i];
  }
  __syncthreads();
  const uint32_t bin = (uint32_t)pick[0];
  int first, end;
  chunk_range(g, n, c, first, end);
  const uint32_t* keys = g.keys + (pair * nc + c) * kChunk;
  uint32_t* listed = g.listed + (pair * nc + c) * kChunk;
  uint32_t k[kChunkK];
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int t = Keys<kChunkK>::slot(i);
    k[i] = first + t < end ? keys[t] : 0u;
  }
  int more = 0, in = 0;
  uint64_t m[kChunkK];
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const bool live = first + Keys<kChunkK>::slot(i) < end;
    more += __popcll(__builtin_amdgcn_ballot_w64(live && (k[i] >> kLowBits) > bin));
    m[i] = __builtin_amdgcn_ballot_w64(live && (k[i] >> kLowBits) == bin);
    in += __popcll(m[i]);
  }
  int at, total, m_before, m_all;
  count_before(in, buf + kSelWaves, at, total);
  count_before(more, buf + 2 * kSelWaves, m_before, m_all);
  const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    if (m[i] >> lane & 1) listed[at + __popcll(m[i] & below)] = k[i];
    at += __popcll(m[i]);
  }
  if (tid == 0) {
    int32_t* ca = g.chunk_at + (pair * nc + c) * 4;
    ca[0] = m_all;
    ca[1] = total;
    if (c == 0) {
      g.rank[pair * 4] = (int32_t)bin;
      g.rank[pair * 4 + 1] = pick[1];
    }
  }
}

__global__ __launch_bounds__(kSelThreads) void evict_rank_kernel(LongArgs g) {
  const SlotArgs& a = g.s;
  const int h = blockIdx.x, b = blockIdx.y, nc = g.nlo + g.nhi, tid = threadIdx.x;
  const int lane = tid & 63, w = tid >> 6;
  const int n = rows_of(a, b);
  const int64_t pair = (int64_t)b * a.nkv + h;
  if (n <= g.keep) {
    if (tid == 0) g.counts[pair] = 0;
    return;
  }
  __shared__ int buf[6 * kSelWaves];
  __shared__ uint32_t ends[2];
  extern __shared__ int32_t cn[];  // [nc][3]: listed before the chunk, its keys past T, equals
  int32_t* ca = g.chunk_at + pair * nc * 4;
  const uint32_t* listed = g.listed + pair * nc * kChunk;
  const uint32_t top = (uint32_t)g.rank[pair * 4] << kLowBits;
  const int want = g.rank[pair * 4 + 1];
  if (tid < 2) ends[tid] = tid ? 0u : 0xFFFFFFFFu;
  int total = 0;
  if (w == 0) {  // the chunks' starts in the concatenated list
    for (int c0 = 0; c0 < nc; c0 += 64) {
      int first, end;
      const int c = c0 + lane;
      if (c < nc) chunk_range(g, n, c, first, end);
      const int x = c < nc && first < end ? ca[4 * c + 1] : 0;
      int y = x;
#pragma unroll
      for (int off = 1; off < 64; off *= 2) {
        const int z = __shfl_up(y, off);
        if (lane >= off) y += z;
      }
      if (c < nc) {
        cn[3 * c] = total + y - x;
        cn[3 * c + 1] = cn[3 * c + 2] = 0;
      }
      total += __builtin_amdgcn_readlane(y, 63);
    }
    if (lane == 0) buf[0] = total;
  }
  __syncthreads();
  total = buf[0];
  __syncthreads();
  // key j of the concatenated list: chunk by bisection
  auto key_at = [&](int j) -> uint32_t {
    int lo = 0, hi = nc - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (cn[3 * mid] <= j) lo = mid;
      else hi = mid - 1;
    }
    return listed[(int64_t)lo * kChunk + j - cn[3 * lo]];
  };
  uint32_t T;
  Keys<kRankK> keys;
  const bool fits = total <= kSelThreads * kRankK;
  if (fits) {
#pragma unroll
    for (int i = 0; i < kRankK; ++i) {
      const int j = Keys<kRankK>::slot(i);
      keys.k[i] = j < total ? key_at(j) : 0u;
    }
    T = kth_largest<kRankK>(keys, top, kLowBits - 2, want, buf);
  } else {
    // too many of one bin for the registers: the smallest and the largest first (weights
    // that are all one value end here), then a bit a step over the list
    uint32_t mn = 0xFFFFFFFFu, mx = 0u;
    for (int j = tid; j < total; j += kSelThreads) {
      const uint32_t k = key_at(j);
      mn = min(mn, k);
      mx = max(mx, k);
    }
    atomicMin(&ends[0], mn);
    atomicMax(&ends[1], mx);
    __syncthreads();
    T = top;
    if (ends[0] == ends[1]) {
      T = ends[0];
    } else {
      for (int s = kLowBits - 1; s >= 0; --s) {
        int c[1] = {0};
        for (int j0 = 0; j0 < total; j0 += kSelThreads)
          c[0] += __popcll(__builtin_amdgcn_ballot_w64(j0 + tid < total &&
                                                       key_at(min(j0 + tid, total - 1)) >= T + (1u << s)));
        count_all<1>(c, buf + (s & 1) * kSelWaves);
        if (c[0] >= want) T += 1u << s;
      }
    }
  }
  // every chunk's listed keys past T and equal to it
  __syncthreads();
  for (int c = w; c < nc; c += kSelWaves) {
    int first, end;
    chunk_range(g, n, c, first, end);
    const int cnt = first < end ? ca[4 * c + 1] : 0;
    int gt = 0, eq = 0;
    for (int j0 = 0; j0 < cnt; j0 += 64) {
      const uint32_t k = j0 + lane < cnt ? listed[(int64_t)c * kChunk + j0 + lane] : 0u;
      gt += __popcll(__builtin_amdgcn_ballot_w64(j0 + lane < cnt && k > T));
      eq += __popcll(__builtin_amdgcn_ballot_w64(j0 + lane < cnt && k == T));
    }
    if (lane == 0) {
      cn[3 * c + 1] = gt;
      cn[3 * c + 2] = eq;
    }
  }
  __syncthreads();
  if (w != 0) return;
  // equals that stay, and the starts of the chunks' equals and list entries
  int gt = 0;
  for (int c = lane; c < nc; c += 64) gt += cn[3 * c + 1];
#pragma unroll
  for (int off = 1; off < 64; off *= 2) gt += __shfl_xor(gt, off);
  const int ties = want - gt;
  int eq0 = 0, hole0 = 0, move0 = 0;
  for (int c0 = 0; c0 < nc; c0 += 64) {
    const int c = c0 + lane;
    int first = 0, end = 0;
    if (c < nc) chunk_range(g, n, c, first, end);
    const bool live = c < nc && first < end;
    const int eq = live ? cn[3 * c + 2] : 0;
    int e = eq;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int z = __shfl_up(e, off);
      if (lane >= off) e += z;
    }
    const int eq_at = eq0 + e - eq;
    const int stay = live ? ca[4 * c] + cn[3 * c + 1] + min(max(ties - eq_at, 0), eq) : 0;
    const int hole = live && c < g.nlo ? end - first - stay : 0, move = live && c >= g.nlo ? stay : 0;
    int x = hole, y = move;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int z = __shfl_up(x, off), q = __shfl_up(y, off);
      if (lane >= off) {
        x += z;
        y += q;
      }
    }
    if (c < nc) {
      ca[4 * c + 2] = eq_at;
      ca[4 * c + 3] = c < g.nlo ? hole0 + x - hole : move0 + y - move;
    }
    eq0 += __builtin_amdgcn_readlane(e, 63);
    hole0 += __builtin_amdgcn_readlane(x, 63);
    move0 += __builtin_amdgcn_readlane(y, 63);
  }
  if (lane == 0) {
    g.rank[pair * 4 + 2] = (int32_t)T;
    g.rank[pair * 4 + 3] = ties;
    g.counts[pair] = min(min(hole0, move0), g.most);
  }
}

__global__ __launch_bounds__(kSelThreads) void evict_list_kernel(LongArgs g) {
  const SlotArgs& a = g.s;
  const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, nc = g.nlo + g.nhi;
  const int n = rows_of(a, b);
  if (n <= g.keep) return;
  int first, end;
  chunk_range(g, n, c, first, end);
  if (first >= end) return;
  const int64_t pair = (int64_t)b * a.nkv + h;
  const uint32_t* keys = g.keys + (pair * nc + c) * kChunk;
  Keys<kChunkK> k;
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int t = Keys<kChunkK>::slot(i);
    k.k[i] = first + t < end ? keys[t] : 0u;
  }
  __shared__ int buf[6 * kSelWaves];
  const int32_t* ca = g.chunk_at + (pair * nc + c) * 4;
  int32_t* dst = g.lists + pair * 2 * g.most;
  int nm;
  (void)list_slots<kChunkK>(k, first, end, g.keep, (uint32_t)g.rank[pair * 4 + 2], g.rank[pair * 4 + 3],
                            ca[2], c < g.nlo, c >= g.nlo, dst, dst + g.most, ca[3], ca[3], g.most, buf,
                            nm);
}

int launch_track(const SlotArgs& a, int M, int B, void* stream) {
  if (M == 0 || B == 0) return 0;
  hipLaunchKernelGGL(kv_track_kernel, dim3((unsigned)((M + 255) / 256), a.nkv, B), dim3(256), 0,
                     (hipStream_t)stream, a, M);
  return (int)hipGetLastError();
}

// Longest sequence the one-workgroup selection takes.
constexpr int kSelMax = kSelThreads * 16;

template <bool FUSE>
void launch_select(const SlotArgs& a, int n, int keep, int recent, int most, int32_t* counts,
                   int32_t* lists, int unit16, int B, hipStream_t st) {
  auto go = [&](auto k) {
    hipLaunchKernelGGL((evict_select_kernel<decltype(k)::value, FUSE>), dim3(a.nkv, B),
                       dim3(kSelThreads), 0, st, a, keep, recent, most, counts, lists, unit16);
  };
  const int K = (n + kSelThreads - 1) / kSelThreads;
  if (K <= 1) go(std::integral_constant<int, 1>{});
  else if (K <= 2) go(std::integral_constant<int, 2>{});
  else if (K <= 4) go(std::integral_constant<int, 4>{});
  else if (K <= 6) go(std::integral_constant<int, 6>{});
  else if (K <= 8) go(std::integral_constant<int, 8>{});
  else if (K <= 12) go(std::integral_constant<int, 12>{});
  else go(std::integral_constant<int, 16>{});
}

// n: rows of the longest sequence.
int launch_evict(const SlotArgs& a, int n, int keep, int recent, int B, void* stream) {
  if (n <= keep || keep == 0 || B == 0) return 0;  // nothing moves
  const hipStream_t hs = (hipStream_t)stream;
  const int most = std::min(n - keep, keep);
  // units of 16 bytes where every row, head and token starts on one
  const int unit16 = a.row % 16 == 0 && a.tok % 16 == 0 && a.head % 16 == 0 && a.block % 16 == 0;
  const int upr = (int)(a.row / (unit16 ? 16 : 4));
  if ((int64_t)most * upr > 0x70000000) return MOLOT_ENOTSUP;  // units of a head's moves
  if (n <= kSelMax && most <= kFuseMoves && (int64_t)most * a.row <= kFuseBytes) {
    launch_select<true>(a, n, keep, recent, most, nullptr, nullptr, unit16, B, hs);
    return (int)hipGetLastError();
  }
  const size_t pairs = (size_t)B * a.nkv;
  LongArgs g{};
  g.s = a;
  g.keep = keep;
  g.recent = recent;
  g.most = most;
  g.nlo = (keep + kChunk - 1) / kChunk;
  g.nhi = (n - keep + kChunk - 1) / kChunk;
  const size_t nc = n <= kSelMax ? 0 : (size_t)g.nlo + g.nhi;
  const size_t lds = sizeof(int32_t) * 3 * nc;
  if (lds > 128 * 1024) return MOLOT_ENOTSUP;  // 89 million rows
  // [lists | counts | rank, chunk_at | keys | listed | bins]
  const size_t words = pairs * (2 * (size_t)most + 1 + (nc ? 4 + 4 * nc + 2 * nc * kChunk + nc * (kBins / 2) : 0));
  unsigned long long* ctr = nullptr;
  void* ws = nullptr;
  int st = workspace(stream, sizeof(int32_t) * words, &ctr, &ws);
  if (st) return st;
  g.lists = reinterpret_cast<int32_t*>(ws);
  g.counts = g.lists + pairs * 2 * most;
  if (!nc) {
    launch_select<false>(a, n, keep, recent, most, g.counts, g.lists, unit16, B, hs);
  } else {
    g.rank = g.counts + pairs;
    g.chunk_at = g.rank + 4 * pairs;
    g.keys = reinterpret_cast<uint32_t*>(g.chunk_at + 4 * pairs * nc);
    g.listed = g.keys + pairs * nc * kChunk;
    g.bins = reinterpret_cast<uint16_t*>(g.listed + pairs * nc * kChunk);
    const dim3 chunks((unsigned)nc, a.nkv, B), block(kSelThreads);
    hipLaunchKernelGGL(evict_keys_kernel, chunks, block, 0, hs, g);
    hipLaunchKernelGGL(evict_pick_kernel, chunks, block, 0, hs, g);
    hipLaunchKernelGGL(evict_rank_kernel, dim3(a.nkv, B), block, lds, hs, g);
    hipLaunchKernelGGL(evict_list_kernel, chunks, block, 0, hs, g);
  }
  st = (int)hipGetLastError();
  if (st) return st;
  // a workgroup takes 256 threads * 4 units a round; enough of them to fill the chip
  const int64_t units = (int64_t)most * upr;
  const int64_t wgs = std::max<int64_t>(1, std::min<int64_t>((units + 1023) / 1024, 4096));
  const dim3 grid((unsigned)wgs, a.nkv, B);
  if (unit16)
    hipLaunchKernelGGL(evict_move_kernel<16>, grid, dim3(256), 0, hs, a, most, g.counts, g.lists);
  else
    hipLaunchKernelGGL(evict_move_kernel<4>, grid, dim3(256), 0, hs, a, most, g.counts, g.lists);
  return (int)hipGetLastError();
}

// The layout of a cache (attn_hip.h) in bytes.
int cache_layout(SlotArgs& a, int nkv, int d, int page, int kv_dtype) {
  if (kv_dtype != MOLOT_KV_F32 && kv_dtype != MOLOT_KV_BF16 && kv_dtype != MOLOT_KV_Q8)
    return MOLOT_EINVAL;
  const bool q8 = kv_dtype == MOLOT_KV_Q8;
  if (d < 2 || d > 512 || d % 2 || (q8 && d % 4)) return MOLOT_ENOTSUP;
  const int64_t esz = kv_dtype == MOLOT_KV_F32 ? 4 : q8 ? 1 : 2;
  a.q8 = q8;
  a.row = d * esz;
  if (page) {
    a.tok = a.row;
    a.head = (int64_t)page * a.row;
    a.block = q8 ? molot_hip_q8_block_bytes(nkv, d, page) : (int64_t)nkv * page * a.row;
    a.sc_off = (int64_t)nkv * page * d;
    a.sc_head = 4LL * page;
    a.sc_tok = 4;
  } else {
    a.tok = q8 ? molot_hip_q8_row_bytes(nkv, d) : (int64_t)nkv * a.row;
    a.head = a.row;
    a.sc_off = (int64_t)nkv * d;
    a.sc_head = 4;
  }
  return 0;
}

int flat_slots(SlotArgs& a, float* acc, int32_t* slot_pos, int nkv, int n, int pos, int acc_cap) {
  if (!acc || nkv <= 0 || nkv > 65535 || n < 0 || acc_cap < n) return MOLOT_EINVAL;
  a.acc = acc;
  a.slot_pos = slot_pos;
  a.nkv = nkv;
  a.n = a.limit = n;
  a.pos = pos;
  a.acc_cap = acc_cap;
  return 0;
}

int paged_slots(SlotArgs& a, float* acc, int32_t* slot_pos, const int32_t* block_table,
                const int32_t* seq_lens, const int32_t* pos, int B, int max_blocks,
                int max_seq_len, int nkv, int page) {
  if (!acc || !block_table || !seq_lens || B < 0 || nkv <= 0 || max_blocks <= 0 ||
      max_seq_len < 0 || page <= 0 || (page & (page - 1)) ||
      (int64_t)max_seq_len > (int64_t)max_blocks * page)
    return MOLOT_EINVAL;
  if (B > 65535 || nkv > 65535) return MOLOT_ENOTSUP;  // grid rows
  a.acc = acc;
  a.slot_pos = slot_pos;
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.pos_arr = pos;
  a.nkv = nkv;
  a.max_blocks = max_blocks;
  while ((1 << a.page_shift) < page) ++a.page_shift;
  a.limit = max_seq_len;
  return 0;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace

int molot_host::kv_track(float* acc, int32_t* slot_pos, int nkv, int n, int M, int pos,
                         int acc_cap, void* stream) {
  SlotArgs a{};
  const int st = flat_slots(a, acc, slot_pos, nkv, n, pos, acc_cap);
  if (st) return st;
  if (M < 0 || M > n) return MOLOT_EINVAL;
  return launch_track(a, M, 1, stream);
}

extern "C" {

int molot_hip_kv_track(float* acc, int32_t* slot_pos, int nkv, int n, int M, int pos, int acc_cap,
                       void* stream) {
  return molot_host::kv_track(acc, slot_pos, nkv, n, M, pos, acc_cap, stream);
}

int molot_hip_kv_track_paged(float* acc, int32_t* slot_pos, const int32_t* block_table,
                             const int32_t* seq_lens, const int32_t* pos, int B, int max_blocks,
                             int max_seq_len, int M, int nkv, int page, void* stream) {
  SlotArgs a{};
  const int st = paged_slots(a, acc, slot_pos, block_table, seq_lens, pos, B, max_blocks,
                             max_seq_len, nkv, page);
  if (st) return st;
  if (M < 0) return MOLOT_EINVAL;
  return launch_track(a, std::min(M, max_seq_len), B, stream);
}

int molot_hip_kv_evict(void* K, void* V, float* acc, int32_t* slot_pos, int nkv, int n, int d,
                       int keep, int recent, int pos, int acc_cap, int kv_dtype, void* stream) {
  SlotArgs a{};
  int st = flat_slots(a, acc, slot_pos, nkv, n, pos, acc_cap);
  if (st) return st;
  if (!K || !V || !slot_pos || keep < 0 || recent < 0 || !aligned16(K) || !aligned16(V))
    return MOLOT_EINVAL;
  st = cache_layout(a, nkv, d, 0, kv_dtype);
  if (st) return st;
  a.k = reinterpret_cast<char*>(K);
  a.v = reinterpret_cast<char*>(V);
  return launch_evict(a, n, keep, recent, 1, stream);
}

int molot_hip_kv_evict_paged(void* K, void* V, float* acc, int32_t* slot_pos,
                             const int32_t* block_table, const int32_t* seq_lens,
                             const int32_t* pos, int B, int max_blocks, int max_seq_len, int nkv,
                             int d, int page, int keep, int recent, int kv_dtype, void* stream) {
  SlotArgs a{};
  int st = paged_slots(a, acc, slot_pos, block_table, seq_lens, pos, B, max_blocks, max_seq_len,
                       nkv, page);
  if (st) return st;
  if (!K || !V || !slot_pos || keep < 0 || recent < 0 || !aligned16(K) || !aligned16(V))
    return MOLOT_EINVAL;
  st = cache_layout(a, nkv, d, page, kv_dtype);
  if (st) return st;
  if (a.q8 && ((int64_t)nkv * page) % 4) return MOLOT_EINVAL;  // blocks stay 16-byte aligned
  a.k = reinterpret_cast<char*>(K);
  a.v = reinterpret_cast<char*>(V);
  return launch_evict(a, max_seq_len, keep, recent, B, stream);
}

}  // extern "C"
