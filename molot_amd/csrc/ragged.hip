// Ragged batches: packed rows of sequences of different lengths over a paged cache.
//
//   ragged_plan_kernel    block tables, lengths and slot maps from the requests' lengths
//   ragged_rows_kernel    the rows' maps of larger batches
//   ragged_append_kernel  norms, RoPE and append of the packed rows by their slots
//   ragged_units_kernel   the attention's units of work from the lengths
//   ragged_valu_kernel    attention of any head dim and cache type, on the vector ALU
//   ragged_merge_kernel   the merge of split tiles
// No reference counterpart: the reference runs one sequence a Runner
// (include/molot/forward.h:48-51).
#include "ragged.hpp"

#include <algorithm>
#include <cmath>

#include "attn_host.hpp"
#include "prefill_tile.hpp"

namespace {

using namespace molot_host;

// ---------------------------------------------------------------------------
// Plan.
//
// With len_b rows cached (0 of a finished sequence) and count_b new ones, sequence b
// takes ceil((len_b + count_b) / page) - ceil(len_b / page) blocks.  The free list is
// a stack: finished sequences push their blocks (b, then the block's index, ascending),
// then the new blocks are popped in the same order, so a block's place in the stack is
// a prefix sum and every row finds its block by itself.  What bounds it: one workgroup's chain
// of loads, scans and the rows' search (6 us of 64 sequences; 19 of 4099, and 5.5 for their 64k
// rows in a launch of their own).  Nothing is committed before the whole batch is known to
// fit, in blocks of the pool: a plan that fails writes its status, lengths as they were, and
// rows of no sequence.
struct PlanArgs {
  const int32_t* counts;
  const int32_t* done;
  const int32_t* pos;
  const int32_t* seq_lens;
  int32_t* kv_lens;
  int32_t* block_table;
  int32_t* free_blocks;
  const int32_t* free_count;
  int32_t* free_left;
  int32_t* row_start;
  int32_t* row_seq;
  int32_t* row_pos;
  int32_t* row_slot;
  int32_t* status;
  int32_t* taken;  // workspace: [B + 1] new blocks of the sequences before; the stack's top
  int B, max_blocks, page_shift, num_blocks, max_rows;
};

constexpr int kPlanThreads = 1024;
// Sequences whose prefix sums fit in LDS: a row's search then takes log2(B) LDS reads.
constexpr int kPlanSeqs = 4096;
constexpr int kPlanMost = 1 << 20;  // rows, blocks a sequence: sums of 1024 stay below 2^31

// Exclusive prefix over the workgroup of x, and the total.
template <int NT>
__device__ __forceinline__ int block_scan(int x, int* sh, int& total) {
  constexpr int NW = NT / 64;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int inc = wave_scan(x);
  __syncthreads();  // the last scan's sums are read
  if (lane == 63) sh[w] = inc;
  __syncthreads();
  const int other = wave_scan(lane < NW ? sh[lane] : 0);
  total = __builtin_amdgcn_readlane(other, NW - 1);
  const int before = w ? __builtin_amdgcn_readlane(other, w - 1) : 0;
  return before + inc - x;
}

// A sequence's part in the plan: its rows cached (0 once it is finished), new rows, new
// blocks and blocks given back; st: what is wrong with it.
struct PlanSeq {
  int len, count, take, give, st;
};
__device__ __forceinline__ PlanSeq plan_seq(const PlanArgs& a, int b) {
  const bool in = b < a.B;
  const int i = in ? b : 0;  // (B > 0)
  const int len = a.seq_lens[i], count = in ? a.counts[i] : 0;
  const bool done = a.done && a.done[i] != 0;
  const int64_t cap = (int64_t)a.max_blocks << a.page_shift;
  const int64_t from = done || !in ? 0 : len;
  const int r = (1 << a.page_shift) - 1;
  auto blocks = [&](int64_t n) { return (int)((n + r) >> a.page_shift); };
  PlanSeq s{};
  if (in && (len < 0 || count < 0 || len > cap || from + count > cap)) {
    s.st = MOLOT_EINVAL;
  } else if (count > a.max_rows) {
    s.st = MOLOT_E2BIG;
  } else {
    s.len = (int)from;
    s.count = count;
    if (a.free_blocks) {
      s.take = blocks(from + count) - blocks(from);
      s.give = in && done ? blocks(len) : 0;
    }
  }
  return s;
}

// Row r of the batch, of sequence b whose rows start at `start`: its maps, and the
// table's entry where the row opens a block that the plan takes.
__device__ __forceinline__ void plan_row(const PlanArgs& a, int r, int b, int start, int len,
                                         int taken, int top) {
  const int slot = len + r - start, j = slot >> a.page_shift, mask = (1 << a.page_shift) - 1;
  const int have = (len + mask) >> a.page_shift;
  int32_t* entry = a.block_table + (int64_t)b * a.max_blocks + j;
  int id;
  if (!a.free_blocks || j < have) {
    id = *entry;
  } else {
    id = a.free_blocks[top - 1 - (taken + j - have)];
    if ((slot & mask) == 0) *entry = id;
  }
  a.row_seq[r] = b;
  a.row_pos[r] = a.pos ? a.pos[b] + (r - start) : slot;
  a.row_slot[r] = (unsigned)id < (unsigned)a.num_blocks ? (id << a.page_shift) + (slot & mask) : -1;
}
__device__ __forceinline__ void plan_no_row(const PlanArgs& a, int r) {
  a.row_seq[r] = -1;
  a.row_pos[r] = 0;
  a.row_slot[r] = -1;
}
// The sequence of row r: the last with start(b) <= r (those without rows, which start
// where the next does, are passed over).
template <typename START>
__device__ __forceinline__ int plan_find(int B, int r, START&& start) {
  int lo = 0, hi = B;  // start(lo) <= r < start(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start(mid) <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Rounds of sequences at once, the fewest that even passes of at most kPlanBatch rounds take
// (plan_rounds): 1500, 4096, 4099, 5121, 8192 and 65536 sequences of one row take 10.1, 14.4,
// 15.0, 17.9, 20.3 and 105 us so, one round at a time 10.0, 15.3, 16.3, 18.3, 21.7 and 113;
// 6 or 8 rounds at once no less (5121 17.8, 8192 21.0, 65536 107).
constexpr int kPlanBatch = 5;
int plan_rounds(int B) {
  const int rounds = std::max(1, (B + kPlanThreads - 1) / kPlanThreads);
  const int passes = (rounds + kPlanBatch - 1) / kPlanBatch;
  return (rounds + passes - 1) / passes;
}
// Sequences b0 + tid, b0 + kPlanThreads + tid, ...: their loads in flight together.
template <int N>
__device__ __forceinline__ void plan_batch(const PlanArgs& a, int b0, PlanSeq (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = plan_seq(a, b0 + kPlanThreads * i + (int)threadIdx.x);
}

// One workgroup.  `rows`: it writes the rows' maps too, else ragged_rows_kernel does.
template <int N>
__global__ __launch_bounds__(kPlanThreads) void ragged_plan_kernel(PlanArgs a, int rows) {
  __shared__ int sh[kPlanThreads / 64], s_st;
  __shared__ unsigned long long s_sum[3];
  __shared__ int s_start[kPlanSeqs + 1], s_taken[kPlanSeqs];
  const int tid = threadIdx.x;
  const bool pool = a.free_blocks != nullptr;
  const int count0 = pool ? *a.free_count : 0;
  auto none = [&](int id) { return (unsigned)id >= (unsigned)a.num_blocks; };
  // the list's top, on its way beside the sequences
  const bool listed = pool && tid < count0 && count0 <= a.num_blocks;
  const int id0 = listed ? a.free_blocks[count0 - 1 - tid] : 0;
  if (tid < 3) s_sum[tid] = 0;
  if (tid == 0) s_st = 0;
  // totals, and whether the batch fits
  unsigned long long nrows = 0, take = 0, give = 0;  // (lane 63's are the wave's)
  int st = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads * N) {
    PlanSeq s[N];
    plan_batch(a, b0, s);
    int x = 0, y = 0, z = 0;  // (each at most N * kPlanMost: a wave's sum stays below 2^31)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      st = min(st, s[i].st);
      x += s[i].count;
      y += s[i].take;
      z += s[i].give;
    }
    nrows += wave_scan(x);
    take += wave_scan(y);
    give += wave_scan(z);
  }
  __syncthreads();
  if (st) atomicMin(&s_st, st);  // of several, the same one whatever the order
  if ((tid & 63) == 63) {
    atomicAdd(&s_sum[0], nrows);
    atomicAdd(&s_sum[1], take);
    atomicAdd(&s_sum[2], give);
  }
  __syncthreads();
  nrows = s_sum[0], take = s_sum[1], give = s_sum[2];
  st = s_st;
  if (st == 0 && nrows > (unsigned long long)a.max_rows) st = MOLOT_E2BIG;
  if (pool && st == 0) {
    if (count0 < 0 || give > (unsigned long long)a.num_blocks || count0 > a.num_blocks - (int)give)
      st = MOLOT_EINVAL;
    else if (take > (unsigned long long)count0 + give)
      st = MOLOT_ENOSPC;
  }
  const int top = count0 + (int)(st ? 0 : give);
  // finished sequences' blocks above the stack's top (unused places if the plan fails)
  // (a sequence's blocks by a wave: their number is uneven, and a lane each would wait for
  // the longest), and whether they and the new blocks are blocks of the pool
  if (st == 0 && (give > 0 || take > 0)) {
    const int old = take > give ? (int)(take - give) : 0;  // new blocks off the list as it was
    bool bad = tid < old && none(id0);
    for (int i = tid + kPlanThreads; i < old; i += kPlanThreads) bad |= none(a.free_blocks[count0 - 1 - i]);
    int base = count0;
    for (int b0 = 0; give > 0 && b0 < a.B; b0 += kPlanThreads) {
      const PlanSeq s = plan_seq(a, b0 + tid);
      int all;
      const int at = base + block_scan<kPlanThreads>(s.give, sh, all);
      base += all;
      for (uint64_t left = __builtin_amdgcn_ballot_w64(s.give > 0); left; left &= left - 1) {
        const int l = __builtin_ctzll(left);
        const int n = __builtin_amdgcn_readlane(s.give, l), to = __builtin_amdgcn_readlane(at, l);
        const int32_t* from = a.block_table + (int64_t)(b0 + (tid & ~63) + l) * a.max_blocks;
        for (int j = tid & 63; j < n; j += 64) {
          const int id = from[j];
          bad |= none(id);
          a.free_blocks[to + j] = id;
        }
      }
    }
    __threadfence_block();
    if (__syncthreads_or(bad)) st = MOLOT_EINVAL;
  }
  // the batch as it will be
  int row0 = 0, taken0 = 0;
  for (int b1 = 0; b1 < a.B; b1 += kPlanThreads * N) {
    PlanSeq all[N];
    plan_batch(a, b1, all);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int b = b1 + kPlanThreads * i + tid;
      if (b1 + kPlanThreads * i >= a.B) break;  // (the whole workgroup)
      PlanSeq s = all[i];
      if (st) s = PlanSeq{b < a.B ? a.seq_lens[b] : 0, 0, 0, 0, 0};
      int nr, nt;
      const int rs = row0 + block_scan<kPlanThreads>(s.count, sh, nr);
      const int tk = taken0 + block_scan<kPlanThreads>(s.take, sh, nt);
      row0 += nr;
      taken0 += nt;
      if (b < a.B) {
        a.row_start[b] = rs;
        a.kv_lens[b] = s.len + s.count;
        if (!rows) a.taken[b] = tk;
        if (rows && b < kPlanSeqs) {
          s_start[b] = rs;
          s_taken[b] = tk;
        }
      }
    }
  }
  if (tid == 0) {
    a.row_start[a.B] = row0;
    if (rows) s_start[a.B] = row0;
    else a.taken[a.B] = top;
    if (pool) *a.free_left = st ? count0 : top - taken0;
    *a.status = st;
  }
  if (!rows) return;
  __threadfence_block();
  __syncthreads();
  for (int r = tid; r < a.max_rows; r += kPlanThreads) {
    if (r >= row0) {
      plan_no_row(a, r);
      continue;
    }
    const int b = plan_find(a.B, r, [&](int i) { return s_start[i]; });
    plan_row(a, r, b, s_start[b], a.kv_lens[b] - (s_start[b + 1] - s_start[b]), s_taken[b], top);
  }
}

__global__ __launch_bounds__(256) void ragged_rows_kernel(PlanArgs a) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= a.max_rows) return;
  if (r >= a.row_start[a.B]) {
    plan_no_row(a, r);
    return;
  }
  const int b = plan_find(a.B, r, [&](int i) { return a.row_start[i]; });
  const int start = a.row_start[b];
  plan_row(a, r, b, start, a.kv_lens[b] - (a.row_start[b + 1] - start), a.taken[b], a.taken[a.B]);
}

// ---------------------------------------------------------------------------
// Units.
//
// The host knows neither the lengths nor the counts, only bounds (rows T, sequences B),
// so one workgroup forms the attention's work list from them: the tiles of every
// sequence, the keys each attends, and from their costs (a wide tile's key counts `weight`
// narrow ones) the share of a workgroup that the chip holds at once.  Tiles that cost more are
// split; so at most `target` units, one such workgroup each, come on top of one a tile.  The
// list goes by cost, the largest first: the workgroups that start last are short.  One
// workgroup's chain of loads and scans, 6 to 9 us of 3 to 64 sequences; in a step it runs beside
// the append.
constexpr int kUnitBuckets = 64;

// Tiles of a sequence of R rows r: wide ones as long as more than `few` rows are left, then
// narrow ones.
__device__ __forceinline__ int wide_tiles(const RaggedArgs& a, int R) {
  return R / a.ql + (R % a.ql > a.few ? 1 : 0);
}
__device__ __forceinline__ int slim_tiles(const RaggedArgs& a, int R) {
  const int rows = ragged_slim(a, R);
  return R % a.ql > a.few ? 0 : (R % a.ql + rows - 1) / rows;
}
// A tile's keys: [lo, hi), kt of 32.
struct UnitTile {
  int seq, r0, lo, hi, wide, rows, kt;
  RaggedSeq s;
};
template <typename BEFORE>
__device__ __forceinline__ UnitTile unit_tile(const RaggedArgs& a, int t, int nwide, BEFORE&& before) {
  const int kind = t >= nwide, i = kind ? t - nwide : t;
  const int b = plan_find(a.B, i, [&](int s) { return before(s, kind); });
  const RaggedSeq s = ragged_seq(a, b);
  const int R = s.rows * a.G, rows = kind ? ragged_slim(a, R) : a.ql;
  const int r0 = (kind ? R / a.ql * a.ql : 0) + (i - before(b, kind)) * rows;
  const int r1 = min(r0 + rows, R) - 1;
  const int lo = ragged_lo(a, s.slot0 + r0 / a.G);
  const int hi = max(lo, ragged_hi(a, s.slot0 + r1 / a.G));
  return {b, r0, lo, hi, !kind, rows, (hi - lo + 31) >> 5, s};
}

// NT threads of one workgroup.
template <int NT>
__device__ __forceinline__ void make_units(const RaggedArgs& a) {
  __shared__ int sh[NT / 64], s_bucket[kUnitBuckets], s_none;
  __shared__ unsigned long long s_cost;
  __shared__ int s_tiles[2 * (kPlanSeqs + 1)];
  const int tid = threadIdx.x;
  const bool in_lds = a.B <= kPlanSeqs;
  if (tid == 0) s_cost = s_none = 0;
  if (tid < kUnitBuckets) s_bucket[tid] = 0;
  int nwide = 0, nslim = 0;
  bool none = false;
  for (int b0 = 0; b0 < a.B; b0 += NT) {
    const int b = b0 + tid;
    const int R = b < a.B ? ragged_seq(a, b).rows * a.G : 0;
    none |= b < a.B && a.row_start[b + 1] < a.row_start[b];
    int t0, t1;
    const int w = nwide + block_scan<NT>(wide_tiles(a, R), sh, t0);
    const int s = nslim + block_scan<NT>(slim_tiles(a, R), sh, t1);
    nwide += t0;
    nslim += t1;
    if (b < a.B) {
      int* at = in_lds ? s_tiles + 2 * b : a.tiles + 2 * b;
      at[0] = w;
      at[1] = s;
    }
  }
  if (none) s_none = 1;  // (past the scans' barriers)
  __threadfence_block();
  __syncthreads();
  // Starts that ascend are those of at most T rows, which the lists' bounds stand on.
  if (s_none) {
    if (tid == 0) a.head->nunits = a.head->nparts = 0;
    return;
  }
  const int ntiles = nwide + nslim;
  auto before = [&](int b, int kind) { return in_lds ? s_tiles[2 * b + kind] : a.tiles[2 * b + kind]; };
  // (a batch of at most NT tiles keeps them; a larger one finds each again)
  const bool once = ntiles <= NT;
  UnitTile mine{};
  unsigned long long cost = 0;
  for (int t = tid; t < ntiles; t += NT) {
    const UnitTile u = unit_tile(a, t, nwide, before);
    if (once) mine = u;
    cost += (unsigned)u.kt * (unsigned)(u.wide ? a.weight : 1);
  }
  atomicAdd(&s_cost, cost);
  __syncthreads();
  // the keys (of 32) a unit takes at most: whole intervals of its kind
  auto up = [](unsigned long long x, int n) { return (int)((min(x, 1ull << 26) + n - 1) / n * n); };
  const unsigned long long share = (s_cost + a.target - 1) / a.target;
  const int most_wide = up(max((share + a.weight - 1) / a.weight, (unsigned long long)a.min_keys >> 5), 2);
  const int most_slim = up(max(share, (unsigned long long)a.min_keys >> 5), 8);
  const float top = (float)max(most_wide * a.weight, most_slim);
  // how a tile is split: n units of `size`
  auto split = [&](const UnitTile& u, int& size) {
    const int most = u.wide ? most_wide : most_slim;
    if (u.kt <= most) {
      size = u.kt;
      return 1;
    }
    const int n = (u.kt + most - 1) / most;
    size = up((u.kt + n - 1) / n, u.wide ? 2 : 8);
    return (u.kt + size - 1) / size;
  };
  auto bucket = [&](const UnitTile& u, int size) {
    const float c = (float)(size * (u.wide ? a.weight : 1));
    return max(0, kUnitBuckets - 1 - (int)(c / top * (kUnitBuckets - 1)));
  };
  for (int t = tid; t < ntiles; t += NT) {
    const UnitTile u = once ? mine : unit_tile(a, t, nwide, before);
    int size;
    const int n = split(u, size);
    atomicAdd(&s_bucket[bucket(u, size)], n);
  }
  __syncthreads();
  if (tid < 64) {
    const int n = s_bucket[tid], all = wave_scan(n);
    s_bucket[tid] = all - n;
    if (tid == 63) a.head->nunits = min(all, a.max_units);
  }
  __syncthreads();
  int nparts = 0;
  for (int t0 = 0; t0 < ntiles; t0 += NT) {
    const int t = t0 + tid;
    UnitTile u{};
    int n = 0, size = 1;
    if (t < ntiles) {
      u = once ? mine : unit_tile(a, t, nwide, before);
      n = split(u, size);
    }
    int parts;
    const int pt = nparts + block_scan<NT>(n > 1 ? n : 0, sh, parts);
    nparts += parts;
    // (the order within a bucket is any: a unit's results do not depend on its place)
    const int at = n ? atomicAdd(&s_bucket[bucket(u, size)], n) : 0;
    for (int i = 0; i < n; ++i) {
      if (at + i >= a.max_units || (n > 1 && pt + i >= a.max_parts)) break;  // (never: the bounds hold)
      const int lo = u.lo + size * i * 32, hi = i + 1 < n ? lo + size * 32 : u.hi;
      a.units[at + i] = RaggedUnit{u.seq, u.r0, lo, hi, n > 1 ? pt + i : -1, i, n, u.wide, u.s, u.rows};
      if (n > 1) a.part_unit[pt + i] = at + i;
    }
  }
  if (tid == 0) a.head->nparts = min(nparts, a.max_parts);
}

__global__ __launch_bounds__(kPlanThreads) void ragged_units_kernel(RaggedArgs a) {
  make_units<kPlanThreads>(a);
}

// ---------------------------------------------------------------------------
// Norms, RoPE and append of the packed rows (what bounds it: the stream, 103 MB of 2279 rows of
// 32q/8kv/d128 bf16 in 24 us, 4.3 TB/s; 40 rows, 3.6 us: a wave's chain of loads, angles and
// sums): row r's heads normed and rotated at
// row_pos[r], k and v stored at row_slot[r] (< 0: the row is left as it is).  A
// wave takes some heads of a row, lane l the pairs l, l + 64, ...; angles, sums and
// roundings are those of rope_append_tok_kernel.
struct AppendArgs {
  float* q;
  const float* k_new;  // NULL: q alone
  const float* v_new;
  char* K;
  char* V;
  const int32_t* row_pos;
  const int32_t* row_slot;
  const float* q_norm;
  const float* k_norm;
  const float* inv_freq;
  int nq, nkv, d, page_shift, v_norm, kv_dtype;
  int each;  // heads a wave
  int64_t slots;  // of the pool
  float eps;
};
constexpr int kAppendThreads = 256, kAppendWaves = kAppendThreads / 64;
// Heads a wave at most, past the rows that fill the chip: each shares the wave's angles, and
// fewer waves are in flight.  At most 2, 4, 6, 10 and 16 (us, normed rows): 4000 of 32q/8kv/d128
// bf16 41, 37, 36, 35, 38, 8192 of them fp32 92, 87, 90, 94, 97; 8192 of 8q/8kv/d64 bf16 35, 31,
// 33, 34, 39; of 8q/4kv/d256 47, 41, 42, 44, 47; 4000 of 64q/8kv/d128 69, 62, 56, 57, 54.
constexpr int kAppendHeads = 6;

// UNITS: a step's; one more workgroup forms the attention's units meanwhile.
template <int KMAX, bool UNITS>
__global__ __launch_bounds__(kAppendThreads) void ragged_append_kernel(AppendArgs a, RaggedArgs u) {
  if (UNITS && blockIdx.x == 0) {
    if (blockIdx.y == 0) make_units<kAppendThreads>(u);
    return;
  }
  const int r = UNITS ? (int)blockIdx.x - 1 : (int)blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int half = a.d >> 1;
  const int64_t at = a.row_slot[r];
  if (at < 0 || at >= a.slots) return;  // (the whole workgroup)
  const int pos = a.row_pos[r];
  const bool rot = a.inv_freq != nullptr;
  const int heads = a.nq + (a.k_new ? a.nkv : 0);
  const int h0 = (blockIdx.y * kAppendWaves + w) * a.each, h1 = min(h0 + a.each, heads);
  if (h0 >= h1) return;
  // a head's x (q's or k's) and v, the next one's in flight while one is used
  float n0[KMAX], n1[KMAX], nv0[KMAX], nv1[KMAX];
  auto load = [&](int hh) {
    const bool isq = hh < a.nq;
    const float* x = isq ? a.q + ((int64_t)r * a.nq + hh) * a.d
                         : a.k_new + ((int64_t)r * a.nkv + (hh - a.nq)) * a.d;
    const float* vx = a.v_new + ((int64_t)r * a.nkv + (hh - a.nq)) * a.d;  // (not read for q)
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      const int j = lane + 64 * k;
      const bool in = j < half;
      n0[k] = in ? x[j] : 0.f;
      n1[k] = in ? x[j + half] : 0.f;
      nv0[k] = in && !isq ? vx[j] : 0.f;
      nv1[k] = in && !isq ? vx[j + half] : 0.f;
    }
  };
  load(h0);
  // a lane's pairs are the same in every head: its angles in registers
  float cs[KMAX], sn[KMAX];
#pragma unroll
  for (int k = 0; k < KMAX; ++k) {
    cs[k] = 1.f;
    sn[k] = 0.f;
    if (rot && 64 * k < half) {
      const float ang = (float)pos * a.inv_freq[min(lane + 64 * k, half - 1)];
      double sd, cd;
      sincos((double)ang, &sd, &cd);
      cs[k] = (float)cd;
      sn[k] = (float)sd;
    }
  }
  auto rms_inv = [&](float ss, int n) { return 1.0f / sqrtf(ss / (float)n + a.eps); };
  for (int hh = h0; hh < h1; ++hh) {
    const bool isq = hh < a.nq;
    const int kh = hh - a.nq;
    const float* weight = isq ? a.q_norm : a.k_norm;
    float x0[KMAX], x1[KMAX], v0[KMAX], v1[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      x0[k] = n0[k];
      x1[k] = n1[k];
      v0[k] = nv0[k];
      v1[k] = nv1[k];
    }
    if (hh + 1 < h1) load(hh + 1);
    if (weight) {
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < KMAX; ++k)
        if (64 * k < half) ss += group_sum<64>(x0[k] * x0[k] + x1[k] * x1[k]);
      const float inv = rms_inv(ss, a.d);
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        const int j = min(lane + 64 * k, half - 1);
        x0[k] = x0[k] * inv * weight[j];
        x1[k] = x1[k] * inv * weight[j + half];
      }
    }
    float r0[KMAX], r1[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      r0[k] = rot ? x0[k] * cs[k] - x1[k] * sn[k] : x0[k];
      r1[k] = rot ? x0[k] * sn[k] + x1[k] * cs[k] : x1[k];
    }
    if (isq) {
      float* y = a.q + ((int64_t)r * a.nq + hh) * a.d;
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        const int j = lane + 64 * k;
        if (j < half) {
          y[j] = r0[k];
          y[j + half] = r1[k];
        }
      }
      continue;
    }
    if (a.v_norm) {  // one RMS over the row's nkv*d values
      const float* vall = a.v_new + (int64_t)r * a.nkv * a.d;
      float part = 0.f;
      for (int j = lane; j < a.nkv * a.d; j += 64) part = fmaf(vall[j], vall[j], part);
      const float inv = rms_inv(group_sum<64>(part), a.nkv * a.d);
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        v0[k] *= inv;
        v1[k] *= inv;
      }
    }
    const int page = 1 << a.page_shift, sl = (int)(at & (page - 1));
    const int64_t blk = at >> a.page_shift, rows = (int64_t)a.nkv * page;
    const int64_t in_block = ((int64_t)kh * page + sl) * a.d;
    if (a.kv_dtype == MOLOT_KV_Q8) {
      float kmax = 0.f, vmax = 0.f;
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        if (lane + 64 * k >= half) continue;
        kmax = fmaxf(kmax, fmaxf(fabsf(r0[k]), fabsf(r1[k])));
        vmax = fmaxf(vmax, fmaxf(fabsf(v0[k]), fabsf(v1[k])));
      }
      const float ks = q8_scale(group_max<64>(kmax)), vs = q8_scale(group_max<64>(vmax));
      const int64_t b0 = blk * rows * (a.d + 4), so = b0 + rows * a.d + 4 * ((int64_t)kh * page + sl);
      int8_t* kd = reinterpret_cast<int8_t*>(a.K) + b0 + in_block;
      int8_t* vd = reinterpret_cast<int8_t*>(a.V) + b0 + in_block;
#pragma unroll
      for (int k = 0; k < KMAX; ++k) {
        const int j = lane + 64 * k;
        if (j >= half) continue;
        kd[j] = (int8_t)q8_code(r0[k], ks);
        kd[j + half] = (int8_t)q8_code(r1[k], ks);
        vd[j] = (int8_t)q8_code(v0[k], vs);
        vd[j + half] = (int8_t)q8_code(v1[k], vs);
      }
      if (lane == 0) {
        *reinterpret_cast<float*>(a.K + so) = ks;
        *reinterpret_cast<float*>(a.V + so) = vs;
      }
      continue;
    }
    const int64_t off = blk * rows * a.d + in_block;
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
      const int j = lane + 64 * k;
      if (j >= half) continue;
      if (a.kv_dtype == MOLOT_KV_F32) {
        float* kd = reinterpret_cast<float*>(a.K) + off;
        float* vd = reinterpret_cast<float*>(a.V) + off;
        kd[j] = r0[k];
        kd[j + half] = r1[k];
        vd[j] = v0[k];
        vd[j + half] = v1[k];
      } else {
        uint16_t* kd = reinterpret_cast<uint16_t*>(a.K) + off;
        uint16_t* vd = reinterpret_cast<uint16_t*>(a.V) + off;
        kd[j] = f32_to_bf16(r0[k]);
        kd[j + half] = f32_to_bf16(r1[k]);
        vd[j] = f32_to_bf16(v0[k]);
        vd[j + half] = f32_to_bf16(v1[k]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Attention of any head dim and cache type: a unit's rows a wave each (ragged_own_row).
// What bounds it: the latency of a key's rows and of the wave's sum, four keys at a time;
// the units' splits (64 keys on, eight workgroups a CU) fill the chip.  16 sequences of one row
// after 2000, 8q/2kv/d512: bf16 75 us (1.75 TB/s), Q8 90; 200 fresh fp32 rows 52.
constexpr int kValuWaves = 4;
template <int EPL, typename T>
__global__ __launch_bounds__(64 * kValuWaves) void ragged_valu_kernel(RaggedArgs a) {
  const int u = blockIdx.x / a.nkv, h = blockIdx.x - u * a.nkv;
  if (u >= a.head->nunits) return;
  const RaggedUnit t = a.units[u];
  ragged_own_row<EPL, T>(a, t, h, t.r0 + (int)(threadIdx.x >> 6));
}

// ---------------------------------------------------------------------------
// The merge of a split tile's n units: o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
// Latency (unit, statistics, rows): 4 to 6 us of narrow tiles, 10 to 14 where wide ones are split.
// The workgroups of the tile's parts share its rows: up to kMergeFew units a wave takes a
// row by itself, past them a workgroup's waves share a row's units.
constexpr int kMergeThreads = 256, kMergeWaves = kMergeThreads / 64, kMergeFew = 16;
template <int EPL>
__global__ __launch_bounds__(kMergeThreads) void ragged_merge_kernel(RaggedArgs a) {
  constexpr int D = 64 * EPL;
  __shared__ float s_o[kMergeWaves][D], s_l[kMergeWaves], s_m[kMergeWaves];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int p = blockIdx.x / a.nkv, h = blockIdx.x - p * a.nkv;
  if (p >= a.head->nparts) return;
  const RaggedUnit t = a.units[a.part_unit[p]];
  const RaggedSeq& s = t.s;
  const int n = t.nsplit, p0 = p - t.split;
  const int rows = min(t.rows, s.rows * a.G - t.r0);
  const bool shared = n > kMergeFew;  // uniform
  const int first = t.split * gridDim.y + blockIdx.y, groups = n * gridDim.y;
  for (int i = shared ? first : first * kMergeWaves + w; i < rows;
       i += shared ? groups : groups * kMergeWaves) {
    const int64_t slot = ((int64_t)p0 * a.nkv + h) * a.slot_rows + i;
    const int64_t step = (int64_t)a.nkv * a.slot_rows;  // to the next unit's
    float M = -INFINITY, L = 0.f, o[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = 0.f;
    for (int c = shared ? w : 0; c < n; c += shared ? 4 * kMergeWaves : 4) {
      float m[4], l[4], x[4][EPL];
      const int by = shared ? kMergeWaves : 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t at = slot + min(c + j * by, n - 1) * step;
        m[j] = c + j * by < n ? a.part_ml[2 * at] : -INFINITY;
        l[j] = a.part_ml[2 * at + 1];
#pragma unroll
        for (int e = 0; e < EPL; ++e) x[j][e] = a.part_o[at * D + lane + 64 * e];
      }
      const float mn = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), M);
      if (mn == -INFINITY) continue;  // no key so far (wave-uniform)
      const float f = exp2_hw(M - mn);
      L *= f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (m[j] == -INFINITY) continue;
        const float g = exp2_hw(m[j] - mn);
        L = fmaf(l[j], g, L);
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[e] = fmaf(x[j][e], g, o[e]);
      }
      M = mn;
    }
    if (shared) {  // the same i in every wave
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EPL; ++e) s_o[w][lane + 64 * e] = o[e];
      if (lane == 0) {
        s_l[w] = L;
        s_m[w] = M;
      }
      __syncthreads();
      if (w) continue;
#pragma unroll
      for (int j = 1; j < kMergeWaves; ++j) {
        const float mj = s_m[j], mn = fmaxf(M, mj);
        if (mj == -INFINITY) continue;
        const float f = exp2_hw(M - mn), g = exp2_hw(mj - mn);
        L = L * f + s_l[j] * g;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[e] = o[e] * f + s_o[j][lane + 64 * e] * g;
        M = mn;
      }
    }
    const int m = (t.r0 + i) / a.G, g = t.r0 + i - m * a.G;
    float* out = a.o + (((int64_t)s.start + m) * a.nq + h * a.G + g) * a.d;
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < EPL; ++e)
      if (lane + 64 * e < a.d) out[lane + 64 * e] = o[e] * inv;
  }
}

// ---------------------------------------------------------------------------
// Host.

// Keys of a sequence: the kernels count them in an int, up to 511 past the last (the next
// tile's blocks of the last wave, and what a tile or a split is rounded up to).
constexpr int kMostKeys = 0x7FFFFFFF - 1024;

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

int shift_of(int page) {
  int s = 0;
  while ((1 << s) < page) ++s;
  return s;
}

// What the entries over packed rows share (d: any that the cache type takes).
int check_ragged(int nq, int nkv, int d, int page, int num_blocks, int kv_dtype) {
  if (nq <= 0 || nkv <= 0 || nq % nkv) return MOLOT_EINVAL;
  if (kv_dtype != MOLOT_KV_F32 && kv_dtype != MOLOT_KV_BF16 && kv_dtype != MOLOT_KV_Q8)
    return MOLOT_EINVAL;
  if (d < 2 || d > 512 || d % 2 || (kv_dtype == MOLOT_KV_Q8 && d % 4)) return MOLOT_ENOTSUP;
  if (page <= 0 || (page & (page - 1)) || num_blocks <= 0 ||
      (int64_t)num_blocks * page > 0x7FFFFFFF)
    return MOLOT_EINVAL;
  if (kv_dtype == MOLOT_KV_Q8 && ((int64_t)nkv * page) % 4) return MOLOT_EINVAL;  // 16-byte blocks
  if (nkv > 4096 || nq > 65536) return MOLOT_ENOTSUP;  // the grids, and rows r in 31 bits
  return 0;
}

// units: a step's attention, whose units the launch forms too (NULL: none).
int launch_append(AppendArgs a, int T, const RaggedArgs* units, void* stream) {
  const int heads = a.nq + (a.k_new ? a.nkv : 0);
  // heads a wave: enough waves for the chip, and then more for each angle
  a.each = (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)T * heads / 8192, kAppendHeads));
  const int y = (heads + kAppendWaves * a.each - 1) / (kAppendWaves * a.each);
  const int half = a.d / 2;
  auto k = half <= 64    ? units ? ragged_append_kernel<1, true> : ragged_append_kernel<1, false>
           : half <= 128 ? units ? ragged_append_kernel<2, true> : ragged_append_kernel<2, false>
           : units       ? ragged_append_kernel<4, true> : ragged_append_kernel<4, false>;
  hipLaunchKernelGGL(k, dim3(T + (units ? 1 : 0), y), dim3(kAppendThreads), 0, (hipStream_t)stream, a,
                     units ? *units : RaggedArgs{});
  return (int)hipGetLastError();
}

// The attention's workspace, in one piece.
struct Layout {
  size_t units, tiles, part_unit, part_ml, part_o, all;
  Layout(const RaggedArgs& a, int D) {
    size_t at = sizeof(RaggedHead);
    auto take = [&](size_t bytes) {
      const size_t was = at;
      at += (bytes + 255) / 256 * 256;
      return was;
    };
    at = (at + 255) / 256 * 256;
    units = take(sizeof(RaggedUnit) * (size_t)a.max_units);
    tiles = take(sizeof(int32_t) * 2 * ((size_t)a.B + 1));
    part_unit = take(sizeof(int32_t) * (size_t)a.max_parts);
    const size_t slots = (size_t)a.max_parts * a.nkv * a.slot_rows;
    part_ml = take(sizeof(float) * 2 * slots);
    part_o = take(sizeof(float) * D * slots);
    all = at;
  }
};

// A wide tile's key against a narrow one's.  Alone the two take 3 to 1 (us a key and CU at
// 32q/8kv/d128 bf16, fp32 and Q8: 0.097, 0.117 and 0.085 for 512 rows after 16384, 0.032,
// 0.051 and 0.025 for 64 sequences of one row); mixed, where wide units run beside narrow ones
// that wait for memory, wide ones that are cut shorter still end sooner: 512 rows beside 63
// decoding sequences (bf16) 137 us at 3, 130 at 6, 127 at 8 and 10.
constexpr int kWideWeight = 8;

template <typename T>
RaggedFn valu_of(int D) {
  return D == 64    ? ragged_valu_kernel<1, T>
         : D == 128 ? ragged_valu_kernel<2, T>
         : D == 256 ? ragged_valu_kernel<4, T> : ragged_valu_kernel<8, T>;
}

// append, T rows: a step's, before the attention.
int launch_attention(RaggedArgs a, const AppendArgs* append, void* stream) {
  LaunchLock lock(g_launch_mu);
  const int cus = num_cus();
  const int D = a.d <= 64 ? 64 : a.d <= 128 ? 128 : a.d <= 256 ? 256 : 512;
  RaggedFn attend = a.kv_dtype == MOLOT_KV_F32    ? valu_of<float>(D)
                    : a.kv_dtype == MOLOT_KV_BF16 ? valu_of<bf16_t>(D)
                                                  : valu_of<q8_t>(D);
  RaggedFn merge = D == 64 ? ragged_merge_kernel<1>
                   : D == 128 ? ragged_merge_kernel<2>
                   : D == 256 ? ragged_merge_kernel<4> : ragged_merge_kernel<8>;
  int threads = 64 * kValuWaves;
  a.qs = a.ql = a.slot_rows = kValuWaves;
  a.few = 0;  // every tile a wide one
  a.min_keys = 64;
  a.weight = 1;
  int per_cu = 8;
  // (the matrix-core kernel's offsets are of 31 bits within a block, and of 35 in a pool)
  const int64_t block = ((int64_t)a.nkv << a.page_shift) *
                        (a.kv_dtype == MOLOT_KV_Q8 ? a.d + 4 : a.d * (a.kv_dtype == MOLOT_KV_BF16 ? 2 : 4));
  if (a.d <= 256 && a.d % 8 == 0 && block <= 0x7FFFFFFF && a.num_blocks * block <= (8ll << 32)) {
    const RaggedTile t = ragged_tile(a.d, a.kv_dtype, a.softcap > 0.f || a.slopes);
    attend = t.fn;
    threads = t.threads;
    a.qs = t.narrow;
    a.ql = t.wide;
    // Two narrow tiles at most.  16 sequences of 64 rows r after 2000, in narrow tiles and in a
    // wide one: bf16 67 and 74 us, Q8 59 and 70 (two tiles of 32); fp32 123 and 98, d = 256 bf16
    // (40 rows r) 102 and 54 (three or four of 16).
    a.few = 2 * t.narrow;
    a.min_keys = 512;  // (512 to 1024 the same; 256 leaves a wave one tile)
    a.weight = kWideWeight;
    // (a tile holds no more rows than the batch)
    a.slot_rows = (int64_t)a.T * a.G <= kSlimRows ? kSlimRows : (int64_t)a.T * a.G <= a.few ? a.qs : a.ql;
    per_cu = 1;  // (a workgroup takes a CU: 2 units 157 us where one takes 139, 32 drafts on Q8)
  }
  a.target = (per_cu * cus + a.nkv - 1) / a.nkv;
  // Bounds: a sequence of R rows r has at most R / ql wide tiles and one more, or narrow
  // ones for up to `few` rows; its splits add at most its share of target, and a split tile
  // has at most twice that (ragged_units_kernel).
  const int64_t R = (int64_t)a.T * a.G;
  const int64_t seqs = std::min(a.T, a.B);
  const int64_t tiles = R / a.ql + seqs * std::max(1, (a.few + a.qs - 1) / a.qs);
  if (R > 0x3FFFFFFF || (tiles + a.target) * a.nkv * threads > 0xFFFFFFFF) return MOLOT_ENOTSUP;
  a.max_units = (int)(tiles + a.target);
  a.max_parts = a.cap > a.min_keys ? 2 * a.target : 0;  // (else no tile is split)
  const Layout l(a, D);
  void* ws = nullptr;
  unsigned long long* ctr = nullptr;
  const int st = workspace(stream, l.all, &ctr, &ws);
  if (st) return st;
  char* w = reinterpret_cast<char*>(ws);
  a.head = reinterpret_cast<RaggedHead*>(w);
  a.units = reinterpret_cast<RaggedUnit*>(w + l.units);
  a.tiles = reinterpret_cast<int32_t*>(w + l.tiles);
  a.part_unit = reinterpret_cast<int32_t*>(w + l.part_unit);
  a.part_ml = reinterpret_cast<float*>(w + l.part_ml);
  a.part_o = reinterpret_cast<float*>(w + l.part_o);
  if (append) {
    const int sa = launch_append(*append, a.T, &a, stream);
    if (sa) return sa;
  } else {
    hipLaunchKernelGGL(ragged_units_kernel, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
  }
  hipLaunchKernelGGL(attend, dim3((unsigned)(a.max_units * a.nkv)), dim3(threads), 0,
                     (hipStream_t)stream, a);
  if (a.max_parts)
    hipLaunchKernelGGL(merge, dim3((unsigned)(a.max_parts * a.nkv), std::min(a.slot_rows / kMergeWaves, 8)),
                       dim3(kMergeThreads), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int attention_args(RaggedArgs& a, const float* Q, const void* K, const void* V, float* O,
                   const int32_t* block_table, const int32_t* kv_lens, const int32_t* row_start,
                   int T, int B, int max_blocks, int num_blocks, int max_len, int nq, int nkv, int d,
                   int page, float scale, int window, float softcap, const float* slopes,
                   int kv_dtype) {
  const int st = check_ragged(nq, nkv, d, page, num_blocks, kv_dtype);
  if (st) return st;
  if (T < 0 || B < 0 || max_blocks <= 0 || max_len < 0 ||
      (int64_t)max_blocks * page > 0x7FFFFFFF || max_len > (int64_t)max_blocks * page)
    return MOLOT_EINVAL;
  if (T > 0 && B > 0 &&  // (an empty batch's arrays may be NULL)
      (!Q || !K || !V || !O || !block_table || !kv_lens || !row_start || Q == O))
    return MOLOT_EINVAL;
  if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !aligned16(O)) return MOLOT_EINVAL;
  if (T > kPlanMost || B > kPlanMost || max_len > kMostKeys) return MOLOT_ENOTSUP;
  if (!(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f))) return MOLOT_EINVAL;
  a.q = Q;
  a.k = reinterpret_cast<const char*>(K);
  a.v = reinterpret_cast<const char*>(V);
  a.o = O;
  a.block_table = block_table;
  a.kv_lens = kv_lens;
  a.row_start = row_start;
  a.T = T;
  a.B = B;
  a.max_blocks = max_blocks;
  a.num_blocks = num_blocks;
  a.cap = max_len;
  a.nq = nq;
  a.nkv = nkv;
  a.G = nq / nkv;
  a.d = d;
  a.page_shift = shift_of(page);
  a.window = window;
  a.kv_dtype = kv_dtype;
  a.scale = scale;
  a.softcap = softcap;
  a.slopes = slopes;
  return 0;
}

int append_args(AppendArgs& a, float* q, const float* k_new, const float* v_new, void* K, void* V,
                const int32_t* row_pos, const int32_t* row_slot, int T, int num_blocks, int nq,
                int nkv, int d, int page, const float* q_norm, const float* k_norm, int v_norm,
                float eps, const float* inv_freq, int kv_dtype) {
  const int st = check_ragged(nq, nkv, d, page, num_blocks, kv_dtype);
  if (st) return st;
  if (!(eps >= 0.f && eps < INFINITY) || T < 0) return MOLOT_EINVAL;
  if (T > 0 && (!q || !row_pos || !row_slot || !k_new != !v_new || (k_new && (!K || !V))))
    return MOLOT_EINVAL;
  if (T > kPlanMost) return MOLOT_ENOTSUP;
  a.q = q;
  a.k_new = k_new;
  a.v_new = v_new;
  a.K = reinterpret_cast<char*>(K);
  a.V = reinterpret_cast<char*>(V);
  a.row_pos = row_pos;
  a.row_slot = row_slot;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.inv_freq = inv_freq;
  a.nq = nq;
  a.nkv = nkv;
  a.d = d;
  a.page_shift = shift_of(page);
  a.v_norm = v_norm;
  a.kv_dtype = kv_dtype;
  a.slots = (int64_t)num_blocks * page;
  a.eps = eps;
  return 0;
}

}  // namespace

extern "C" {

int molot_hip_ragged_plan(const int32_t* counts, const int32_t* done, const int32_t* pos,
                          const int32_t* seq_lens, int32_t* kv_lens, int32_t* block_table,
                          int32_t* free_blocks, const int32_t* free_count, int32_t* free_left,
                          int B, int max_blocks, int page, int num_blocks, int max_rows,
                          int32_t* row_start, int32_t* row_seq, int32_t* row_pos,
                          int32_t* row_slot, int32_t* status, void* stream) {
  if (!row_start || !status || B < 0 || max_blocks <= 0 || page <= 0 || (page & (page - 1)) ||
      num_blocks <= 0 || max_rows < 0 || (int64_t)num_blocks * page > 0x7FFFFFFF ||
      (int64_t)max_blocks * page > 0x7FFFFFFF)
    return MOLOT_EINVAL;
  if (B > 0 && (!counts || !seq_lens || !kv_lens || !block_table)) return MOLOT_EINVAL;
  if (max_rows > 0 && (!row_seq || !row_pos || !row_slot)) return MOLOT_EINVAL;
  if (free_blocks ? !free_count || !free_left : done != nullptr) return MOLOT_EINVAL;
  if (B > kPlanMost || max_rows > kPlanMost || max_blocks > kPlanMost) return MOLOT_ENOTSUP;
  PlanArgs a{counts,  done,     pos,     seq_lens, kv_lens, block_table, free_blocks, free_count,
             free_left, row_start, row_seq, row_pos, row_slot, status,   nullptr,
             B,       max_blocks, shift_of(page), num_blocks, max_rows};
  // The rows' maps of small batches in the same launch, their search in LDS.
  const bool rows = max_rows <= 4 * kPlanThreads && B <= kPlanSeqs;
  LaunchLock lock(g_launch_mu);
  if (!rows) {
    void* ws = nullptr;
    unsigned long long* ctr = nullptr;
    const int st = workspace(stream, sizeof(int32_t) * ((size_t)B + 1), &ctr, &ws);
    if (st) return st;
    a.taken = reinterpret_cast<int32_t*>(ws);
  }
  const int n = plan_rounds(B);
  auto plan = n == 1   ? ragged_plan_kernel<1>
              : n == 2 ? ragged_plan_kernel<2>
              : n == 3 ? ragged_plan_kernel<3>
              : n == 4 ? ragged_plan_kernel<4> : ragged_plan_kernel<kPlanBatch>;
  hipLaunchKernelGGL(plan, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, a, rows ? 1 : 0);
  if (!rows && max_rows > 0)
    hipLaunchKernelGGL(ragged_rows_kernel, dim3((max_rows + 255) / 256), dim3(256), 0,
                       (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int molot_hip_rope_append_ragged(float* q, const float* k_new, const float* v_new, void* K, void* V,
                                 const int32_t* row_pos, const int32_t* row_slot, int T,
                                 int num_blocks, int nq, int nkv, int d, int page,
                                 const float* q_norm, const float* k_norm, int v_norm, float eps,
                                 const float* inv_freq, int kv_dtype, void* stream) {
  AppendArgs a{};
  const int st = append_args(a, q, k_new, v_new, K, V, row_pos, row_slot, T, num_blocks, nq, nkv, d,
                             page, q_norm, k_norm, v_norm, eps, inv_freq, kv_dtype);
  if (st || T == 0) return st;
  return launch_append(a, T, nullptr, stream);
}

int molot_hip_attn_ragged(const float* Q, const void* K, const void* V, float* O,
                          const int32_t* block_table, const int32_t* kv_lens,
                          const int32_t* row_start, int T, int B, int max_blocks, int num_blocks,
                          int max_len, int nq, int nkv, int d, int page, float scale, int window,
                          float softcap, const float* slopes, int kv_dtype, void* stream) {
  RaggedArgs a{};
  const int st = attention_args(a, Q, K, V, O, block_table, kv_lens, row_start, T, B, max_blocks,
                                num_blocks, max_len, nq, nkv, d, page, scale, window, softcap,
                                slopes, kv_dtype);
  if (st || T == 0 || B == 0) return st;
  return launch_attention(a, nullptr, stream);
}

int molot_hip_step_ragged(float* q, const float* k_new, const float* v_new, void* K, void* V,
                          float* O, const int32_t* block_table, const int32_t* kv_lens,
                          const int32_t* row_start, const int32_t* row_pos, const int32_t* row_slot,
                          int T, int B, int max_blocks, int num_blocks, int max_len, int nq, int nkv,
                          int d, int page, const float* q_norm, const float* k_norm, int v_norm,
                          float eps, const float* inv_freq, float scale, int window, float softcap,
                          const float* slopes, int kv_dtype, void* stream) {
  RaggedArgs a{};
  int st = attention_args(a, q, K, V, O, block_table, kv_lens, row_start, T, B, max_blocks,
                          num_blocks, max_len, nq, nkv, d, page, scale, window, softcap, slopes,
                          kv_dtype);
  if (st) return st;
  AppendArgs r{};
  st = append_args(r, q, k_new, v_new, K, V, row_pos, row_slot, T, num_blocks, nq, nkv, d, page,
                   q_norm, k_norm, v_norm, eps, inv_freq, kv_dtype);
  if (st || T == 0 || B == 0) return st;
  return launch_attention(a, &r, stream);
}

}  // extern "C"
