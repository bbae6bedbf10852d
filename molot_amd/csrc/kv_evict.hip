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
// Up to 16384 slots evict_select_kernel finds each head's moves and, where they are
// few, makes them; else evict_move_kernel does.  Longer caches find theirs in four
// launches over chunks (evict_keys_kernel and on).
//
// What bounds it (kernel trace).  A short cut is a chain of latencies in one workgroup a
// head (load, count, scan, list, move): 4352 bf16 slots of 8 heads (d = 128) cut to 4096
// in 9.9 us, and kv_track_kernel 2.0, against 0.5 for the bytes; 32 paged sequences of
// 700 to 1399 Q8 rows cut to 1024 in 12.5.  131072 bf16 slots of 8 heads cut by 8192:
// keys 7.8, pick 9.4, rank 3.8, list 5.1 us (a launch each, a chunk of 4096 slots a
// workgroup; pick reads every chunk's counts in each of them, 67 MB, and so grows with the
// square of the chunks) and the moves 13.2, which read and write 67 MB at 5.1 TB/s.
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
// The newest position that is not recent.
__device__ __forceinline__ int64_t oldest_of(const SlotArgs& a, int b, int n, int recent) {
  return (int64_t)newest_of(a, b, n) - recent;
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

// A workgroup's keys in LDS, in slot order: thread t has the `each` slots from t * each
// on (odd: the threads' reads then fall in different banks).  Absent slots' keys are 0,
// below every slot's (at least 1).  So a thread counts its own slots in vector
// registers and one scan gives every thread its place; with a wave on 64 neighbouring
// slots the ballots and their counts were bound by the scalar unit, which 16 waves
// share (4352 slots: 7000 cycles for the lists, 22500 for a selection by ballots).
struct Keys {
  uint32_t* k;
  int each;
  template <typename F>
  __device__ __forceinline__ void own(F&& fn) const {  // fn(slot, key) of this thread's slots
    const int t0 = (int)threadIdx.x * each;
#pragma unroll 4
    for (int i = 0; i < each; ++i) fn(t0 + i, k[t0 + i]);
  }
};
__host__ __device__ constexpr int key_each(int n) { return (n + kSelThreads - 1) / kSelThreads | 1; }

// x summed over aligned groups of 16 lanes (DPP within a row; no LDS round trip).
__device__ __forceinline__ int row_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false);   // quad_perm [1,0,3,2]
  x += __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false);   // quad_perm [2,3,0,1]
  x += __builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, false);  // row_half_mirror
  x += __builtin_amdgcn_update_dpp(0, x, 0x140, 0xF, 0xF, false);  // row_mirror
  return x;
}
// Lanes below this one in a ballot.
__device__ __forceinline__ int lanes_below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// The sums over the waves before this one, and over all, of a wave-uniform count.
// buf: kSelWaves ints, free again after the next barrier.
__device__ __forceinline__ void count_before(int c, int* buf, int& before, int& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (lane == 0) buf[w] = c;
  lds_barrier();
  const int x = lane < kSelWaves ? buf[lane] : 0;
  before = __builtin_amdgcn_readlane(row_sum(lane < w ? x : 0), 0);
  all = __builtin_amdgcn_readlane(row_sum(x), 0);
}
// The sums over the threads before this one, and over all, of a count each.
__device__ __forceinline__ int place_of(int c, int* buf, int& all) {
  const int upto = wave_scan(c);
  int before;
  count_before(__builtin_amdgcn_readlane(upto, 63), buf, before, all);
  return before + upto - c;
}

// The keep-th largest key T, the keys past it and those equal to it.
struct Cut {
  uint32_t T;
  int above, equal;
};
constexpr int kFew = 256;
struct alignas(16) SelectLds {
  int hist[4096];
  uint32_t few[kFew];
  int buf[4 * kSelWaves];
  uint32_t ends[2];
  int nfew;
  int pick[2];
  Cut cut;
};

// The `want`-th largest of the workgroup's keys, which share the bits above shift + 12
// (top): 12 bits by counters in LDS, then, of the keys in that bin, the one that
// enough others are above where they are few, at once where they are all one value,
// else a bit a step.
__device__ __forceinline__ Cut kth_largest(const Keys& keys, uint32_t top, int shift, int want,
                                           SelectLds& L) {
  const int tid = threadIdx.x, lane = tid & 63;
  reinterpret_cast<u32x4*>(L.hist)[tid] = u32x4{0u, 0u, 0u, 0u};
  if (tid < 2) L.ends[tid] = tid ? 0u : 0xFFFFFFFFu;
  if (tid == 2) L.nfew = 0;
  lds_barrier();
  const int total_keys = keys.each * kSelThreads;
#pragma unroll 4
  for (int t = tid; t < total_keys; t += kSelThreads) {  // (neighbours' keys differ more than a
    const uint32_t k = keys.k[t];                        // thread's order would: fewer clashes)
    if (k) atomicAdd(&L.hist[(k >> shift) & 4095u], 1);
  }
  lds_barrier();
  {
    const u32x4 c = reinterpret_cast<const u32x4*>(L.hist)[tid];  // bins 4 tid ..
    const int mine = (int)(c[0] + c[1] + c[2] + c[3]);
    int all;
    const int place = place_of(mine, L.buf, all);
    int above = all - place - mine;  // keys of the bins above this thread's
    if (above < want && above + mine >= want) {  // one thread
      int i = 3;
      for (; i > 0; --i) {
        if (above + (int)c[i] >= want) break;
        above += (int)c[i];
      }
      L.pick[0] = 4 * tid + i;
      L.pick[1] = above;
    }
  }
  lds_barrier();
  const uint32_t bin = (uint32_t)L.pick[0];
  const int above = L.pick[1], left = want - above, total = L.hist[bin];
  auto in_bin = [&](uint32_t k) { return k != 0u && ((k >> shift) & 4095u) == bin; };
  if (total <= kFew) {  // (uniform)
#pragma unroll 4
    for (int t = tid; t < total_keys; t += kSelThreads) {
      const uint32_t k = keys.k[t];
      if (in_bin(k)) L.few[atomicAdd(&L.nfew, 1)] = k;  // (in any order)
    }
    if (tid < kFew && tid >= total) L.few[tid] = 0u;
    lds_barrier();
    // four threads a key, a quarter of the others each
    const uint32_t mine = L.few[tid >> 2];
    int gt = 0, eq = 0;
#pragma unroll 4
    for (int i = tid & 3; i < total; i += 4) {
      const uint32_t k = L.few[i];
      gt += k > mine;
      eq += k == mine;
    }
    int both = gt | eq << 16;
    both += __builtin_amdgcn_update_dpp(0, both, 0xB1, 0xF, 0xF, false);  // quad_perm [1,0,3,2]
    both += __builtin_amdgcn_update_dpp(0, both, 0x4E, 0xF, 0xF, false);  // quad_perm [2,3,0,1]
    gt = both & 0xFFFF;
    eq = both >> 16;
    if ((tid >> 2) < total && gt < left && gt + eq >= left)  // one value: equal keys write the same
      L.cut = Cut{mine, above + gt, eq};
    lds_barrier();
    return L.cut;
  }
  uint32_t mn = 0xFFFFFFFFu, mx = 0u;
  keys.own([&](int, uint32_t k) {
    mn = min(mn, in_bin(k) ? k : 0xFFFFFFFFu);
    mx = max(mx, in_bin(k) ? k : 0u);
  });
#pragma unroll 1
  for (int off = 1; off < 64; off *= 2) {
    mn = min(mn, (uint32_t)__shfl_xor((int)mn, off));
    mx = max(mx, (uint32_t)__shfl_xor((int)mx, off));
  }
  if (lane == 0) {
    atomicMin(&L.ends[0], mn);
    atomicMax(&L.ends[1], mx);
  }
  lds_barrier();
  if (L.ends[0] == L.ends[1]) return Cut{L.ends[0], above, total};
  auto reach = [&](uint32_t t, int* buf) {
    int c = 0, all;
    keys.own([&](int, uint32_t k) { c += in_bin(k) && k >= t; });
    (void)place_of(c, buf, all);
    return all;
  };
  uint32_t T = top | bin << shift;
  int turn = 0;
#pragma unroll 1
  for (uint32_t one = 1u << (shift - 1); one; one >>= 1) {
    if (reach(T + one, L.buf + turn) >= left) T += one;
    turn ^= kSelWaves;  // (two buffers by turns: one barrier a step)
  }
  const int more = T == 0xFFFFFFFFu ? 0 : reach(T + 1u, L.buf + turn);
  const int from = reach(T, L.buf + 2 * kSelWaves);
  return Cut{T, above + more, from - more};
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

// The listed moves 0 .. count - 1, by `threads` threads of which this is number tid:
// K and V rows flat over (move, unit), R units a thread in flight; acc, slot_pos and a
// Q8 row's scales a thread a move, loaded before the rows' first units.
template <int U, int R>
__device__ __forceinline__ void move_rows(const SlotArgs& a, int b, int h, const int32_t* dst,
                                          const int32_t* src, int count, int tid, int threads) {
  using T = typename Unit<U>::type;
  struct Slot {
    float acc, ks, vs;
    int32_t pos;
  };
  auto load = [&](int i) {
    Slot x{};
    const int64_t at = slot_index(a, b, h, src[i]);
    x.acc = a.acc[at];
    x.pos = a.slot_pos[at];
    if (a.q8) {
      int64_t sc;
      (void)row_offset(a, b, h, src[i], sc);
      x.ks = *reinterpret_cast<const float*>(a.k + sc);
      x.vs = *reinterpret_cast<const float*>(a.v + sc);
    }
    return x;
  };
  auto store = [&](int i, const Slot& x) {
    const int64_t to = slot_index(a, b, h, dst[i]);
    a.acc[to] = x.acc;
    a.slot_pos[to] = x.pos;
    if (a.q8) {
      int64_t sc;
      (void)row_offset(a, b, h, dst[i], sc);
      *reinterpret_cast<float*>(a.k + sc) = x.ks;
      *reinterpret_cast<float*>(a.v + sc) = x.vs;
    }
  };
  Slot first{};
  if (tid < count) first = load(tid);
  const int upr = (int)(a.row / U);
  const int total = count * upr;  // (bounded by launch_evict)
#pragma unroll 1
  for (int u0 = tid; u0 < total; u0 += R * threads) {
    T kx[R], vx[R];
    int64_t to[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int u = min(u0 + r * threads, total - 1);  // (past the end: loaded, not stored)
      const int i = u / upr, j = u - i * upr;
      int64_t sc;
      const int64_t at = row_offset(a, b, h, src[i], sc) + (int64_t)j * U;
      to[r] = row_offset(a, b, h, dst[i], sc) + (int64_t)j * U;
      kx[r] = *reinterpret_cast<const T*>(a.k + at);
      vx[r] = *reinterpret_cast<const T*>(a.v + at);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (u0 + r * threads >= total) break;
      *reinterpret_cast<T*>(a.k + to[r]) = kx[r];
      *reinterpret_cast<T*>(a.v + to[r]) = vx[r];
    }
  }
  if (tid < count) store(tid, first);
#pragma unroll 1
  for (int i = tid + threads; i < count; i += threads) store(i, load(i));
}

// The holes and moves among a workgroup's slots first .. end - 1: a slot stays whose
// key is past T, or is T and among the first `ties` such from number eq0 on (`equal`
// of them in all); holes are the others before keep, moves the stayers at or past it.
// They go, in order, to holes[hole0 ..] and moves[move0 ..] (NULL: not wanted); their
// numbers come back in nholes, nmoves.
__device__ __forceinline__ void list_slots(const Keys& keys, int first, int end, int keep, uint32_t T,
                                           int ties, int equal, int eq0, int32_t* holes,
                                           int32_t* moves, int hole0, int move0, int most,
                                           SelectLds& L, int& nholes, int& nmoves) {
  const bool split = ties < equal;  // (uniform) some equals stay, some go
  int eq_at = 0;                    // this thread's first equal is number eq_at
  if (split) {
    int c = 0, all;
    keys.own([&](int, uint32_t k) { c += k == T; });
    eq_at = eq0 + place_of(c, L.buf, all);
  }
  // this thread's slots before keep, and then those past it: keys from k0 on, first
  // slot t0
  const uint32_t* k0 = keys.k + (int)threadIdx.x * keys.each;
  const int t0 = first + (int)threadIdx.x * keys.each;
  const int low = min(keys.each, max(0, min(keep, end) - t0));
  const int upto = min(keys.each, max(0, end - t0));
  int c = 0, all;  // holes, moves << 16 (at most 17408 slots)
  if (!split) {
#pragma unroll 4
    for (int i = 0; i < low; ++i) c += k0[i] < T;
    if (low < upto) {
      int m = 0;
#pragma unroll 4
      for (int i = low; i < upto; ++i) m += k0[i] >= T;
      c += m << 16;
    }
  } else {
    int eq = eq_at;
    for (int i = 0; i < upto; ++i) {
      const uint32_t k = k0[i];
      const bool st = k > T || (k == T && eq++ < ties);
      if (st == (i >= low)) c += i < low ? 1 : 1 << 16;
    }
  }
  const int place = place_of(c, L.buf + kSelWaves, all);
  nholes = all & 0xFFFF;
  nmoves = all >> 16;
  if (c == 0) return;
  int h_at = hole0 + (place & 0xFFFF), m_at = move0 + (place >> 16), eq = eq_at;
  for (int i = 0; i < upto; ++i) {
    const uint32_t k = k0[i];
    const bool st = split ? k > T || (k == T && eq++ < ties) : k >= T;
    if (st != (i >= low)) continue;
    // (as many moves as holes; the bound holds whatever another stream does to acc)
    if (i < low) {
      if (holes && h_at < most) holes[h_at] = t0 + i;
      ++h_at;
    } else {
      if (moves && m_at < most) moves[m_at] = t0 + i;
      ++m_at;
    }
  }
}

// Sequences of at most kSelMax rows: a workgroup a (KV head, sequence), its keys in
// LDS.  FUSE: it makes the moves too (lists in LDS, most <= kFuseMoves); else the
// lists go to evict_move_kernel.
constexpr int kSelMax = 16384;
constexpr int kFuseMoves = 2048;
constexpr int64_t kFuseBytes = 64 * 1024;  // of K (and of V) a head

template <bool FUSE>
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
  extern __shared__ uint32_t key_lds[];  // [key_each(longest) * kSelThreads]
  __shared__ SelectLds L;
  __shared__ int32_t own[FUSE ? 2 * kFuseMoves : 1];
  const int64_t oldest = oldest_of(a, b, n, recent);  // recent: past it
  const Keys keys{key_lds, key_each(n)};
  for (int t0 = threadIdx.x; t0 < keys.each * kSelThreads; t0 += 8 * kSelThreads) {
    float x[8];
    int32_t p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t j = slot_index(a, b, h, min(t0 + i * kSelThreads, n - 1));
      x[i] = a.acc[j];
      p[i] = a.slot_pos[j];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = t0 + i * kSelThreads;
      if (t < keys.each * kSelThreads) key_lds[t] = t < n ? slot_key(x[i], p[i] > oldest) : 0u;
    }
  }
  const Cut cut = kth_largest(keys, 0u, 20, keep, L);
  lds_barrier();
  int32_t* dst = FUSE ? own : lists + pair * 2 * most;
  int32_t* src = dst + (FUSE ? kFuseMoves : most);
  int nh, nm;
  list_slots(keys, 0, n, keep, cut.T, keep - cut.above, cut.equal, 0, dst, src, 0, 0, most, L, nh, nm);
  const int moves = min(min(nm, nh), most);
  if constexpr (FUSE) {
    __syncthreads();
    if (unit16)
      move_rows<16, 4>(a, b, h, dst, src, moves, threadIdx.x, kSelThreads);
    else
      move_rows<4, 4>(a, b, h, dst, src, moves, threadIdx.x, kSelThreads);
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
// Longer sequences: chunks of 4096 or 8192 slots (CK a thread), a workgroup each, on either side of
// keep (so that a chunk has holes or moves, never both): nlo of [0, keep), then
// nhi of [keep, n).
//   evict_keys_kernel   a chunk's keys, and its counts of their top kTopBits bits;
//   evict_pick_kernel   the bin of the keep-th largest key from all chunks' counts
//                       (summed again by every chunk: they are small), then the
//                       chunk's keys above the bin counted, those in it listed;
//   evict_rank_kernel   a workgroup a (KV head, sequence): T among the listed keys,
//                       and where each chunk's equals and list entries start;
//   evict_list_kernel   the chunks' holes and moves.
constexpr int kTopBits = 12, kBins = 1 << kTopBits, kLowBits = 32 - kTopBits;
static_assert(kBins == 4 * kSelThreads, "four bins a thread");

constexpr int kAt = 6;
struct LongArgs {
  SlotArgs s;
  int keep, recent, most, nlo, nhi, chunk;
  uint32_t* keys;      // [pair][chunks][chunk]
  uint32_t* listed;    // [pair][chunks][chunk]: the keys of the bin
  uint16_t* bins;      // [pair][chunks][kBins]
  int32_t* chunk_at;   // [pair][chunks][kAt]: keys above the bin, listed; then equals and entries
                       // before; the smallest and largest listed
  int32_t* rank;       // [pair][4]: bin, still wanted in it (then the equals of T), T, equals that stay
  int32_t* counts;     // [pair]
  int32_t* lists;      // [pair][2][most]
};

// First slot and end of chunk c of a sequence of n rows.
__device__ __forceinline__ void chunk_range(const LongArgs& g, int n, int c, int& first, int& end) {
  const bool lo = c < g.nlo;
  first = lo ? c * g.chunk : g.keep + (c - g.nlo) * g.chunk;
  end = min(first + g.chunk, lo ? min(g.keep, n) : n);
}

template <int CK>
__global__ __launch_bounds__(kSelThreads) void evict_keys_kernel(LongArgs g) {
  constexpr int kChunkK = CK, kChunk = kSelThreads * CK;
  const SlotArgs& a = g.s;
  const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, nc = g.nlo + g.nhi, tid = threadIdx.x;
  const int n = rows_of(a, b);
  if (n <= g.keep) return;
  int first, end;
  chunk_range(g, n, c, first, end);
  const int64_t pair = (int64_t)b * a.nkv + h;
  __shared__ __attribute__((aligned(16))) int hist[kBins];
  reinterpret_cast<u32x4*>(hist)[tid] = u32x4{0u, 0u, 0u, 0u};
  const int64_t oldest = oldest_of(a, b, n, g.recent);
  float x[kChunkK];
  int32_t p[kChunkK];
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int64_t j = slot_index(a, b, h, min(first + kSelThreads * i + tid, n - 1));
    x[i] = a.acc[j];
    p[i] = a.slot_pos[j];
  }
  __syncthreads();
  uint32_t* keys = g.keys + (pair * nc + c) * kChunk;
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int t = kSelThreads * i + tid;
    if (first + t >= end) continue;
    const uint32_t k = slot_key(x[i], p[i] > oldest);
    keys[t] = k;
    atomicAdd(&hist[k >> kLowBits], 1);
  }
  __syncthreads();
  const u32x4 v = reinterpret_cast<const u32x4*>(hist)[tid];  // (a chunk's counts fit 16 bits)
  reinterpret_cast<u32x2*>(g.bins + (pair * nc + c) * kBins)[tid] =
      u32x2{v[0] | v[1] << 16, v[2] | v[3] << 16};
}

template <int CK>
__global__ __launch_bounds__(kSelThreads) void evict_pick_kernel(LongArgs g) {
  constexpr int kChunkK = CK, kChunk = kSelThreads * CK;
  const SlotArgs& a = g.s;
  const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, nc = g.nlo + g.nhi, tid = threadIdx.x;
  const int n = rows_of(a, b);
  const int64_t pair = (int64_t)b * a.nkv + h;
  if (n <= g.keep) return;
  int first, end;
  chunk_range(g, n, c, first, end);
  const uint32_t* keys = g.keys + (pair * nc + c) * kChunk;
  uint32_t k[kChunkK];
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int t = kSelThreads * i + tid;
    k[i] = keys[first + t < end ? t : 0];
  }
  // bins 4 tid .. 4 tid + 3 over the chunks; then the sums of the bins above
  __shared__ int buf[kSelWaves];
  __shared__ int pick[2];
  __shared__ int found[2];      // the chunk's keys above the bin, and in it
  __shared__ uint32_t ends[2];  // the smallest and largest in it
  if (tid < 2) {
    found[tid] = 0;
    ends[tid] = tid ? 0u : 0xFFFFFFFFu;
  }
  const u32x2* bins = reinterpret_cast<const u32x2*>(g.bins + pair * nc * kBins) + tid;
  int cnt[4] = {0, 0, 0, 0};
#pragma unroll 1
  for (int i0 = 0; i0 < nc; i0 += 8) {  // (a chunk of no slots has counts of 0)
    u32x2 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = bins[(int64_t)min(i0 + i, nc - 1) * (kBins / 4)];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i >= nc) continue;
      cnt[0] += (int)(x[i][0] & 0xFFFFu);
      cnt[1] += (int)(x[i][0] >> 16);
      cnt[2] += (int)(x[i][1] & 0xFFFFu);
      cnt[3] += (int)(x[i][1] >> 16);
    }
  }
  const int lane = tid & 63;
  const int upto = wave_scan(cnt[0] + cnt[1] + cnt[2] + cnt[3]);  // the lanes' up to this one
  int before, all;
  count_before(__builtin_amdgcn_readlane(upto, 63), buf, before, all);
  int above = all - before - upto;  // keys of the bins above this thread's
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
  uint32_t* listed = g.listed + (pair * nc + c) * kChunk;
  uint32_t mn = 0xFFFFFFFFu, mx = 0u;
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const bool live = first + kSelThreads * i + tid < end;
    const uint64_t more = __builtin_amdgcn_ballot_w64(live && (k[i] >> kLowBits) > bin);
    const bool in = live && (k[i] >> kLowBits) == bin;
    const uint64_t m = __builtin_amdgcn_ballot_w64(in);
    int at = 0;
    if (lane == 0) {
      if (more) atomicAdd(&found[0], __popcll(more));
      if (m) at = atomicAdd(&found[1], __popcll(m));
    }
    at = __builtin_amdgcn_readfirstlane(at);
    if (in) {
      listed[at + lanes_below(m)] = k[i];  // (in any order within the chunk)
      mn = min(mn, k[i]);
      mx = max(mx, k[i]);
    }
  }
  // a wave whose keys are one value adds them at once
  const uint64_t some = __builtin_amdgcn_ballot_w64(mx != 0u);
  if (some) {
    const uint32_t v = __builtin_amdgcn_readlane(mx, __builtin_ctzll(some));
    const bool same = __builtin_amdgcn_ballot_w64(mx != 0u && (mn != v || mx != v)) == 0;
    if (same ? lane == 0 : mx != 0u) {
      atomicMin(&ends[0], same ? v : mn);
      atomicMax(&ends[1], same ? v : mx);
    }
  }
  __syncthreads();
  if (tid == 0) {
    int32_t* ca = g.chunk_at + (pair * nc + c) * kAt;
    ca[0] = found[0];
    ca[1] = found[1];
    ca[4] = (int32_t)ends[0];
    ca[5] = (int32_t)ends[1];
    if (c == 0) {
      g.rank[pair * 4] = (int32_t)bin;
      g.rank[pair * 4 + 1] = pick[1];
    }
  }
}

// Listed keys that the rank kernel holds in LDS at once.
constexpr int kRankMax = 17 * kSelThreads;  // (key_each: odd)

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
  __shared__ SelectLds L;
  extern __shared__ uint32_t rank_lds[];  // [kRankMax] keys, then cn
  int32_t* cn = reinterpret_cast<int32_t*>(rank_lds + kRankMax);  // [nc][3]: listed before the
                                                                  // chunk, its keys past T, equals
  int32_t* ca = g.chunk_at + pair * nc * kAt;
  const uint32_t* listed = g.listed + pair * nc * g.chunk;
  const uint32_t top = (uint32_t)g.rank[pair * 4] << kLowBits;
  const int want = g.rank[pair * 4 + 1];
  // (a chunk past the sequence's end has written no counts)
  auto live = [&](int c) {
    int first, end;
    chunk_range(g, n, c, first, end);
    return first < end;
  };
  if (tid < 2) L.ends[tid] = tid ? 0u : 0xFFFFFFFFu;
  __syncthreads();
  if (w == 0) {  // the chunks' starts in the concatenated list
    int total = 0;
#pragma unroll 1
    for (int c0 = 0; c0 < nc; c0 += 64) {
      const int c = c0 + lane;
      const int x = c < nc && live(c) ? ca[kAt * c + 1] : 0;
      if (x) {
        atomicMin(&L.ends[0], (uint32_t)ca[kAt * c + 4]);
        atomicMax(&L.ends[1], (uint32_t)ca[kAt * c + 5]);
      }
      const int y = wave_scan(x);
      if (c < nc) {
        cn[3 * c] = total + y - x;
        cn[3 * c + 1] = cn[3 * c + 2] = 0;
      }
      total += __builtin_amdgcn_readlane(y, 63);
    }
    if (lane == 0) L.nfew = total;
  }
  __syncthreads();
  const int total = L.nfew;
  auto count_of = [&](int c) { return (c + 1 < nc ? cn[3 * c + 3] : total) - cn[3 * c]; };
  // a wave a chunk, its listed keys 256 at a time: fn(first place in the list, chunk, keys)
  auto each_chunk = [&](auto&& fn) {
#pragma unroll 1
    for (int c = w; c < nc; c += kSelWaves) {
      const int cnt = count_of(c);
      const uint32_t* from = listed + (int64_t)c * g.chunk;
#pragma unroll 1
      for (int j0 = 0; j0 < cnt; j0 += 256) {
        uint32_t k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = from[min(j0 + 64 * i + lane, cnt - 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + 64 * i < cnt) fn(c, j0 + 64 * i + lane, j0 + 64 * i + lane < cnt, k[i]);
      }
    }
  };
  Cut cut;
  const uint32_t smallest = L.ends[0];
  const bool one_value = smallest == L.ends[1];
  __syncthreads();
  if (one_value) {  // (weights that are all 0, say)
    cut.T = smallest;
    for (int c = tid; c < nc; c += kSelThreads) cn[3 * c + 2] = count_of(c);
  } else if (total <= kRankMax) {
    const Keys keys{rank_lds, key_each(total)};
    for (int j = total + tid; j < keys.each * kSelThreads; j += kSelThreads) rank_lds[j] = 0u;
    for (int j0 = tid; j0 < total; j0 += 8 * kSelThreads) {
      uint32_t k[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = min(j0 + i * kSelThreads, total - 1);
        int lo = 0, hi = nc - 1;  // its chunk
        while (lo < hi) {
          const int mid = (lo + hi + 1) / 2;
          if (cn[3 * mid] <= j) lo = mid;
          else hi = mid - 1;
        }
        k[i] = listed[(int64_t)lo * g.chunk + j - cn[3 * lo]];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + i * kSelThreads < total) rank_lds[j0 + i * kSelThreads] = k[i];
    }
    __syncthreads();
    cut = kth_largest(keys, top, kLowBits - 12, want, L);
    // every chunk's listed keys past T and equal to it: a wave a chunk
    for (int c = w; c < nc; c += kSelWaves) {
      const int cnt = count_of(c), at = cn[3 * c];
      int both = 0;
      for (int j = lane; j < cnt; j += 64) {
        const uint32_t k = rank_lds[at + j];
        both += k > cut.T ? 1 : k == cut.T ? 1 << 16 : 0;
      }
      both = __builtin_amdgcn_readlane(wave_scan(both), 63);  // (a chunk's counts fit 16 bits)
      if (lane == 0) {
        cn[3 * c + 1] = both & 0xFFFF;
        cn[3 * c + 2] = both >> 16;
      }
    }
  } else {
    // too many of one bin for LDS: a bit a step over the lists
    cut.T = top;
    int turn = 0;
#pragma unroll 1
    for (uint32_t one = 1u << (kLowBits - 1); one; one >>= 1) {
      int c = 0;
      each_chunk([&](int, int, bool in, uint32_t k) {
        c += __popcll(__builtin_amdgcn_ballot_w64(in && k >= cut.T + one));
      });
      int before, all;
      count_before(c, L.buf + turn, before, all);
      if (all >= want) cut.T += one;
      turn ^= kSelWaves;
    }
    each_chunk([&](int c, int, bool in, uint32_t k) {
      const int gt = __popcll(__builtin_amdgcn_ballot_w64(in && k > cut.T));
      const int eq = __popcll(__builtin_amdgcn_ballot_w64(in && k == cut.T));
      if (lane == 0) {
        cn[3 * c + 1] += gt;
        cn[3 * c + 2] += eq;
      }
    });
  }
  __syncthreads();
  if (w != 0) return;
  // equals that stay, and the starts of the chunks' equals and list entries
  int gt = 0;
  for (int c = lane; c < nc; c += 64) gt += cn[3 * c + 1];
  gt = __builtin_amdgcn_readlane(wave_scan(gt), 63);
  const int ties = want - gt;
  int eq0 = 0, hole0 = 0, move0 = 0;
#pragma unroll 1
  for (int c0 = 0; c0 < nc; c0 += 64) {
    const int c = c0 + lane;
    int first = 0, end = 0;
    if (c < nc) chunk_range(g, n, c, first, end);
    const bool some = c < nc && first < end;
    const int eq = some ? cn[3 * c + 2] : 0;
    const int e = wave_scan(eq);
    const int eq_at = eq0 + e - eq;
    const int stay = some ? ca[kAt * c] + cn[3 * c + 1] + min(max(ties - eq_at, 0), eq) : 0;
    const int hole = some && c < g.nlo ? end - first - stay : 0, move = some && c >= g.nlo ? stay : 0;
    const int x = wave_scan(hole), y = wave_scan(move);
    if (c < nc) {
      ca[kAt * c + 2] = eq_at;
      ca[kAt * c + 3] = c < g.nlo ? hole0 + x - hole : move0 + y - move;
    }
    eq0 += __builtin_amdgcn_readlane(e, 63);
    hole0 += __builtin_amdgcn_readlane(x, 63);
    move0 += __builtin_amdgcn_readlane(y, 63);
  }
  if (lane == 0) {
    g.rank[pair * 4 + 1] = eq0;  // (the equals in all)
    g.rank[pair * 4 + 2] = (int32_t)cut.T;
    g.rank[pair * 4 + 3] = ties;
    g.counts[pair] = min(min(hole0, move0), g.most);
  }
}

template <int CK>
__global__ __launch_bounds__(kSelThreads) void evict_list_kernel(LongArgs g) {
  constexpr int kChunkK = CK, kChunk = kSelThreads * CK;
  const SlotArgs& a = g.s;
  const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, nc = g.nlo + g.nhi, tid = threadIdx.x;
  const int n = rows_of(a, b);
  if (n <= g.keep) return;
  int first, end;
  chunk_range(g, n, c, first, end);
  if (first >= end) return;
  const int64_t pair = (int64_t)b * a.nkv + h;
  const uint32_t* from = g.keys + (pair * nc + c) * kChunk;
  __shared__ uint32_t k[key_each(kChunk) * kSelThreads];
  __shared__ SelectLds L;
  uint32_t x[kChunkK];
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int t = kSelThreads * i + tid;
    x[i] = from[first + t < end ? t : 0];
  }
#pragma unroll
  for (int i = 0; i < kChunkK; ++i) {
    const int t = kSelThreads * i + tid;
    k[t] = first + t < end ? x[i] : 0u;
  }
  k[kChunk + tid] = 0u;
  const int32_t* ca = g.chunk_at + (pair * nc + c) * kAt;
  const int32_t* rk = g.rank + pair * 4;
  const int eq0 = ca[2], at = ca[3], equal = rk[1], ties = rk[3];
  const uint32_t T = (uint32_t)rk[2];
  int32_t* dst = g.lists + pair * 2 * g.most;
  const bool lo = c < g.nlo;
  __syncthreads();
  int nh, nm;
  list_slots(Keys{k, key_each(kChunk)}, first, end, g.keep, T, ties, equal, eq0, lo ? dst : nullptr,
             lo ? nullptr : dst + g.most, at, at, g.most, L, nh, nm);
}

int launch_track(const SlotArgs& a, int M, int B, void* stream) {
  if (M == 0 || B == 0) return 0;
  hipLaunchKernelGGL(kv_track_kernel, dim3((unsigned)((M + 255) / 256), a.nkv, B), dim3(256), 0,
                     (hipStream_t)stream, a, M);
  return (int)hipGetLastError();
}

// n: rows of the longest sequence.
int launch_evict(const SlotArgs& a, int n, int keep, int recent, int B, void* stream) {
  if (n <= keep || keep == 0 || B == 0) return 0;  // nothing moves
  LaunchLock lock(g_launch_mu);
  const hipStream_t hs = (hipStream_t)stream;
  const int most = std::min(n - keep, keep);
  // units of 16 bytes where every row, head and token starts on one
  const size_t key_bytes = sizeof(uint32_t) * kSelThreads * (size_t)key_each(std::min(n, kSelMax));
  const int unit16 = a.row % 16 == 0 && a.tok % 16 == 0 && a.head % 16 == 0 && a.block % 16 == 0;
  const int upr = (int)(a.row / (unit16 ? 16 : 4));
  if ((int64_t)most * upr > 0x70000000) return MOLOT_ENOTSUP;  // units of a head's moves
  if (n <= kSelMax && most <= kFuseMoves && (int64_t)most * a.row <= kFuseBytes) {
    hipLaunchKernelGGL(evict_select_kernel<true>, dim3(a.nkv, B), dim3(kSelThreads), key_bytes, hs, a,
                       keep, recent, most, nullptr, nullptr, unit16);
    return (int)hipGetLastError();
  }
  const size_t pairs = (size_t)B * a.nkv;
  LongArgs g{};
  g.s = a;
  g.keep = keep;
  g.recent = recent;
  g.most = most;
  // Chunks of 4096 slots where their workgroups fit the CUs in one round, up to 80 a head
  // (each sums all the chunks' counts); else of 8192.  us a pass of tracking and cutting
  // 8192 of the bf16 slots (d = 128; the caches' turn about), for 4096 / 8192: 8 heads, 20000
  // slots 28.0 / 33.4, 65536 30.2 / 34.7, 114688 33.5 / 37.2, 131072 (256 chunks) 33.4 / 36.7;
  // cut by 5000 (264 chunks) 37.8 / 33.8; 147456 41.0 / 38.5, 200000 45.5 / 40.6.  4 heads,
  // 200000 34.7 / 36.4, 270000 (272) 46.8 / 37.7.  32 heads, 28000 34.3 / 38.3, 36000 (288) 39.3 /
  // 39.3.  One head, 65536 26.6 / 31.0, 262144 32.8 / 34.4, 327680 (80) 35.6 / 35.4, 393216 37.6 /
  // 36.4, 1048576 59.4 / 47.5.
  auto cut = [&](int chunk) {
    g.chunk = chunk;
    g.nlo = (keep + chunk - 1) / chunk;
    g.nhi = (n - keep + chunk - 1) / chunk;
  };
  cut(4 * kSelThreads);
  if (g.nlo + g.nhi > 80 || (int64_t)(g.nlo + g.nhi) * (int64_t)pairs > num_cus())
    cut(8 * kSelThreads);
  const size_t nc = n <= kSelMax ? 0 : (size_t)g.nlo + g.nhi;
  const size_t lds = sizeof(int32_t) * (kRankMax + 3 * nc);
  if (lds + sizeof(SelectLds) > kMaxLds) return MOLOT_ENOTSUP;  // past 40 million rows
  // [bins | lists | counts | rank, chunk_at | keys | listed]
  const size_t words = pairs * (2 * (size_t)most + 1 + (nc ? 4 + kAt * nc + 2 * nc * g.chunk + nc * (kBins / 2) : 0));
  unsigned long long* ctr = nullptr;
  void* ws = nullptr;
  int st = workspace(stream, sizeof(int32_t) * words, &ctr, &ws);
  if (st) return st;
  g.bins = reinterpret_cast<uint16_t*>(ws);
  g.lists = reinterpret_cast<int32_t*>(ws) + pairs * nc * (kBins / 2);
  g.counts = g.lists + pairs * 2 * most;
  if (!nc) {
    hipLaunchKernelGGL(evict_select_kernel<false>, dim3(a.nkv, B), dim3(kSelThreads), key_bytes, hs, a,
                       keep, recent, most, g.counts, g.lists, unit16);
  } else {
    g.rank = g.counts + pairs;
    g.chunk_at = g.rank + 4 * pairs;
    g.keys = reinterpret_cast<uint32_t*>(g.chunk_at + kAt * pairs * nc);
    g.listed = g.keys + pairs * nc * g.chunk;
    const dim3 chunks((unsigned)nc, a.nkv, B), block(kSelThreads);
    const bool half = g.chunk == 4 * kSelThreads;
    hipLaunchKernelGGL(half ? evict_keys_kernel<4> : evict_keys_kernel<8>, chunks, block, 0, hs, g);
    hipLaunchKernelGGL(half ? evict_pick_kernel<4> : evict_pick_kernel<8>, chunks, block, 0, hs, g);
    hipLaunchKernelGGL(evict_rank_kernel, dim3(a.nkv, B), block, lds, hs, g);
    hipLaunchKernelGGL(half ? evict_list_kernel<4> : evict_list_kernel<8>, chunks, block, 0, hs, g);
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
