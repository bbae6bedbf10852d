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

// One workgroup a (KV head, sequence).  Four passes over the keys, 8 bits each from
// the top, find the keep-th largest key T and how many of its equals stay; then a
// pass in slot order lists the moves.
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(SlotArgs a, int keep, int recent,
                                                                   int most, int32_t* counts,
                                                                   int32_t* lists) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int n = rows_of(a, b);
  const int64_t pair = (int64_t)b * a.nkv + h;
  if (n <= keep) {
    if (tid == 0) counts[pair] = 0;
    return;
  }
  const int oldest = newest_of(a, b, n) - recent;  // recent: past it
  auto key_at = [&](int t) {
    const int64_t i = slot_index(a, b, h, t);
    return slot_key(a.acc[i], a.slot_pos[i] > oldest);
  };
  __shared__ int hist[256];
  __shared__ int pick[2];
  __shared__ int wsum[3][kSelWaves];
  uint32_t prefix = 0;
  int want = keep;  // of the keys that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t = tid; t < n; t += kSelThreads) {
      const uint32_t k = key_at(t);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255, left = want;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      pick[0] = d;
      pick[1] = left;
    }
    __syncthreads();
    prefix |= (uint32_t)pick[0] << shift;
    want = pick[1];
    __syncthreads();
  }
  // in slot order: equals of T so far, holes and moves so far
  int eq0 = 0, hole0 = 0, move0 = 0;
  int32_t* dst = lists + pair * 2 * most;
  int32_t* src = dst + most;
  for (int t0 = 0; t0 < n; t0 += kSelThreads) {
    const int t = t0 + tid;
    const bool in = t < n;
    const uint32_t k = in ? key_at(t) : 0u;
    const bool eq = in && k == prefix;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    const uint64_t beq = __builtin_amdgcn_ballot_w64(eq);
    if (lane == 0) wsum[0][w] = __popcll(beq);
    __syncthreads();
    int eq_at = eq0 + __popcll(beq & below);
    int eq_all = 0;
    for (int i = 0; i < kSelWaves; ++i) {
      if (i < w) eq_at += wsum[0][i];
      eq_all += wsum[0][i];
    }
    const bool stays = in && (k > prefix || (eq && eq_at < want));
    const bool hole = in && t < keep && !stays, move = t >= keep && stays;
    const uint64_t bh = __builtin_amdgcn_ballot_w64(hole), bm = __builtin_amdgcn_ballot_w64(move);
    if (lane == 0) {
      wsum[1][w] = __popcll(bh);
      wsum[2][w] = __popcll(bm);
    }
    __syncthreads();
    int ha = hole0 + __popcll(bh & below), ma = move0 + __popcll(bm & below);
    for (int i = 0; i < kSelWaves; ++i) {
      if (i < w) {
        ha += wsum[1][i];
        ma += wsum[2][i];
      }
      hole0 += wsum[1][i];
      move0 += wsum[2][i];
    }
    // (as many moves as holes; the bound holds whatever another stream does to acc)
    if (hole && ha < most) dst[ha] = t;
    if (move && ma < most) src[ma] = t;
    eq0 += eq_all;
    __syncthreads();
  }
  if (tid == 0) counts[pair] = min(min(move0, hole0), most);
}

// A wave a move: the K and V rows, their scales, acc and slot_pos.
__global__ __launch_bounds__(256) void evict_move_kernel(SlotArgs a, int most, const int32_t* counts,
                                                         const int32_t* lists) {
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63;
  const int64_t pair = (int64_t)b * a.nkv + h;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= counts[pair]) return;
  const int32_t* dst = lists + pair * 2 * most;
  const int to = dst[i], at = dst[most + i];
  auto row_of = [&](int t, int64_t& sc) -> int64_t {
    if (!a.block_table) {
      sc = (int64_t)t * a.tok + a.sc_off + h * a.sc_head;
      return (int64_t)t * a.tok + h * a.head;
    }
    const int64_t blk = a.block_table[(int64_t)b * a.max_blocks + (t >> a.page_shift)];
    const int sl = t & ((1 << a.page_shift) - 1);
    sc = blk * a.block + a.sc_off + h * a.sc_head + sl * a.sc_tok;
    return blk * a.block + h * a.head + sl * a.tok;
  };
  int64_t sto, sat;
  const int64_t rto = row_of(to, sto), rat = row_of(at, sat);
  for (int64_t e = 4 * lane; e < a.row; e += 256) {
    *reinterpret_cast<uint32_t*>(a.k + rto + e) = *reinterpret_cast<const uint32_t*>(a.k + rat + e);
    *reinterpret_cast<uint32_t*>(a.v + rto + e) = *reinterpret_cast<const uint32_t*>(a.v + rat + e);
  }
  if (lane == 0) {
    if (a.q8) {
      *reinterpret_cast<float*>(a.k + sto) = *reinterpret_cast<const float*>(a.k + sat);
      *reinterpret_cast<float*>(a.v + sto) = *reinterpret_cast<const float*>(a.v + sat);
    }
    const int64_t ito = slot_index(a, b, h, to), iat = slot_index(a, b, h, at);
    a.acc[ito] = a.acc[iat];
    a.slot_pos[ito] = a.slot_pos[iat];
  }
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
  const int most = std::min(n - keep, keep);
  const size_t pairs = (size_t)B * a.nkv;
  unsigned long long* ctr = nullptr;
  void* ws = nullptr;
  const int st = workspace(stream, sizeof(int32_t) * pairs * (1 + 2 * (size_t)most), &ctr, &ws);
  if (st) return st;
  int32_t* counts = reinterpret_cast<int32_t*>(ws);
  int32_t* lists = counts + pairs;
  hipLaunchKernelGGL(evict_select_kernel, dim3(a.nkv, B), dim3(kSelThreads), 0, (hipStream_t)stream,
                     a, keep, recent, most, counts, lists);
  const int e = (int)hipGetLastError();
  if (e) return e;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)((most + 3) / 4), a.nkv, B), dim3(256), 0,
                     (hipStream_t)stream, a, most, counts, lists);
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
