// Attention of ragged batches on the matrix cores, head dims up to 256 that are
// multiples of 8.
//
// A workgroup takes one unit (ragged.hpp) of one KV head: S^T = K . Q^T with a query row a
// column of the matrix instructions, the softmax in registers (a lane holds one row and
// some keys of a tile of 32, the lanes around it the others), and O^T += V^T . P^T with P
// where the score accumulator left it (V^T by transposed LDS reads in the same key order).
// q and p are two fp16 pieces, K and V row-scaled pieces (two of an fp32 row, one of a
// bf16 or Q8 row): the products of prefill_narrow.hip.  There the pieces come from a launch
// of their own over one sequence's keys; here the keys of a batch are many
// sequences', most of them read by few rows, so every workgroup makes the pieces of its
// own tiles on their way from the pages to LDS.
//
// Wide tiles (prompts): 256 rows, 32 a wave (at d = 256, where those would take 256
// registers for q and o, 128 rows, 16 a wave).  The workgroup stages an interval of one or two
// tiles of 32 keys together, double buffered.  Waves w and w + 4 share a SIMD: the first half
// of the waves stages the next interval after its products, the second before them, so that
// one's conversions meet the other's products; the interval after next is in flight meanwhile.
// What bounds them: the chain of an interval (staging, products, barrier).  2048 fresh rows at
// 32q/8kv/d128 bf16, fp32 and Q8, on several cards: 147 to 162, 184 to 198 and 143 to 156 us with
// units and merge (bf16 212 to 234 TFLOP/s of the layer's 34 GFLOP, 37 to 40 % of the matrix cores'
// rate over two products a term); 512 after 16384: 327 to 377, 468 to 480 and 313 to 337 us (bf16 370
// to 427 TFLOP/s, 64 to 74 %).
// Narrow tiles (one row, drafts): 16 rows or 32, every wave a key group by itself with its own
// LDS, so no wave waits for another: a tile's K, then its V, take the same place, and the next
// tile's are in flight.  What bounds them: the stream where there is enough of it (64 sequences
// of one row after 100 to 3880, bf16, fp32 and Q8: 113, 195 and 74 us, the bytes at 4.6, 5.3 and
// 3.6 TB/s), else a wave's chain a tile.
// The key groups' (m, l, o) are merged through LDS at the end.
#include "ragged.hpp"

#include <type_traits>

#include "prefill_wide.hpp"

namespace {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// q's pieces in LDS (a member that points there: else its reads would be flat ones)
typedef const __attribute__((address_space(3))) f16x8_t* lds_q_t;

// Maximum over aligned groups of N lanes (8, 16 or 32), as group_max.
template <int CTRL>
__device__ __forceinline__ unsigned dpp_u(unsigned x) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}
template <int N>
__device__ __forceinline__ unsigned group_umax(unsigned v) {
  v = max(v, dpp_u<0xB1>(v));
  v = max(v, dpp_u<0x4E>(v));
  v = max(v, dpp_u<0x141>(v));
  if constexpr (N >= 16) v = max(v, dpp_u<0x140>(v));
  if constexpr (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  return v;
}

// Eight elements of a cached row as loaded.
template <typename T>
struct Raw;
template <>
struct Raw<float> {
  f32x4 x[2];
};
template <>
struct Raw<bf16_t> {
  u32x4 x;
};
template <>
struct Raw<q8_t> {
  u32x2 x;
};

// The pieces of eight elements, and what the unit of their row (x = piece * unit) follows
// from: the bits of its largest |x|, of Q8 rows whether it has a code but zero.  LPR lanes
// hold the row.
template <int NP>
struct Pieces {
  u32x4 p[NP];
  unsigned top;
};
template <int LPR>
__device__ __forceinline__ Pieces<2> make_pieces(const Raw<float>& r, int kv) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max(m, __float_as_uint(r.x[i][e]) & 0x7FFFFFFFu);
  m = group_umax<LPR>(m);
  const float top = __uint_as_float(m);
  const int shift = kv ? f16_vrow_shift(top) : f16_row_shift(top);
  const float sc = ldexpf(1.f, shift);
  Pieces<2> out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t hi, lo;
    mix_split(r.x[i >> 1][2 * (i & 1)], r.x[i >> 1][2 * (i & 1) + 1], sc, hi, lo);
    out.p[0][i] = hi;
    out.p[1][i] = lo;
  }
  out.top = m;
  return out;
}
// A NaN unit marks a row that the pieces cannot hold (own_mark).
__device__ __forceinline__ float unit_of(float, unsigned m, int kv) {
  const float top = __uint_as_float(m);
  const int shift = kv ? f16_vrow_shift(top) : f16_row_shift(top);
  return (kv ? f16_vrow_unit(top, shift) : f16_row_unit(shift)) +
         own_mark(top, m >= 0x7F800000u ? NAN : 0.f, kv);
}
// bf16 to fp16 by its bits: with the row's largest exponent field e, off = max(e - 30, 0)
// is taken from every exponent (fp16's 1 .. 30 then hold 30 binades, each value with
// all its 8 bits; smaller ones, 2^-29 of the largest, go to 0 or near it) and the
// mantissa moves up by 3: 2.5 instructions a pair where a conversion through fp32 takes 7.
template <int LPR>
__device__ __forceinline__ Pieces<1> make_pieces(const Raw<bf16_t>& r, int kv) {
  uint32_t t[4];  // (scalars: a bit cast of a vector's element would take the first)
  u16x2 m2 = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = r.x[i] & 0x7FFF7FFFu;
    m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(u16x2, t[i]));
  }
  const unsigned m = group_umax<LPR>(max((unsigned)m2[0], (unsigned)m2[1]));
  const int e = (int)(m >> 7);
  const unsigned off = (unsigned)max(e - 30, 0);
  const unsigned short sub = (unsigned short)(off << 7);
  const u16x2 sub2 = {sub, sub};
  Pieces<1> out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u16x2 y = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, t[i]), sub2);
    y = y << (unsigned short)3;
    out.p[0][i] = (r.x[i] & 0x80008000u) | __builtin_bit_cast(uint32_t, y);
  }
  out.top = m;
  return out;
}
__device__ __forceinline__ float unit_of(bf16_t, unsigned m, int kv) {
  const int e = (int)(m >> 7);
  const float unit = kv && m == 0 ? 0.f : __uint_as_float((unsigned)(max(e - 30, 0) + 15) << 23);  // 2^(off - 112)
  return unit + own_mark(__uint_as_float(m << 16), e == 255 ? NAN : 0.f, kv);
}
// Codes are exact in fp16: 0x6400 + (code ^ 0x80) is 1152 + code.
template <int LPR>
__device__ __forceinline__ Pieces<1> make_pieces(const Raw<q8_t>& r, int kv) {
  Pieces<1> out;
  const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = r.x[i >> 1] ^ 0x80808080u;
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, x, i & 1 ? 0x04030402u : 0x04010400u);
    out.p[0][i] = __builtin_bit_cast(uint32_t, (f16x2)(__builtin_bit_cast(f16x2, b) - bias));
  }
  out.top = 1;
  if (kv) out.top = group_umax<LPR>(min(r.x[0] | r.x[1], 1u));
  return out;
}
// (a row of zeros weighs nothing whatever its scale)
__device__ __forceinline__ float q8_unit(float scale, unsigned any, int kv) {
  const float unit = any ? scale : 0.f;
  const bool out_of = !(unit >= 0.f) || unit > kOwnMaxK * 0.0078125f || (kv && unit > 0.f && unit < kOwnMinV);
  return unit + (out_of ? NAN : 0.f);
}

// SC: scores past the product (a cap, slopes).
template <int D, typename T, bool SC>
struct Tile {
  static constexpr int NW = 8, NT = 64 * NW;
  static constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  static constexpr int KT = 32;
  static constexpr int WR = D <= 128 ? 32 : 16;  // wide tiles: rows a wave,
  static constexpr int QL = NW * WR;             // and of the tile;
  static constexpr int IT = D <= 128 ? 2 : 1;    // tiles of keys an interval
  static constexpr int RB = 2 * D;               // bytes of a staged row of one piece
  static constexpr int PB = KT * RB;             // of a tile's piece
  static constexpr int TB = NP * PB;             // of a tile
  static constexpr int NWN = TB <= 16384 ? NW : NW / 2;  // narrow tiles: waves whose tiles fit
  static constexpr int LPR = D / 8;              // lanes of a row
  static constexpr int CW = IT * KT * LPR / NT;   // chunks of 8 elements a thread, wide
  static constexpr int CN = KT * LPR / 64;        // and a lane, narrow
  static constexpr int max2(int x, int y) { return x > y ? x : y; }
  // Narrow tiles: rows at most (32 drafts of 20 rows and 500 to 9000 keys, 16 and 32 rows a
  // tile: Q8 144 and 128 us, bf16 183 and 164, but fp32, whose reads bound it, 289 and 298).
  static constexpr int SR = D <= 128 && sizeof(T) < 4 ? 32 : 16;
  static constexpr int kMerge = NWN / 2 * SR * D * 4;
  static constexpr int kData = max2(max2(4 * IT * TB, NWN * TB), kMerge);
  static constexpr int kUnits = max2(NWN * 2, 4 * IT) * KT * 4;  // narrow: [wave][K, V][32]
  static constexpr int kQ = kData + max2(kUnits, NW / 2 * 64 * 8);
  // Narrow tiles of more than 16 rows or d > 128: q's pieces lie in LDS, the same for every
  // wave (in registers, 64 of them, beside the rows in flight and o they spill: 195 registers
  // of the fp32 kernels at d = 256).
  static constexpr bool QLDS = D > 128;
  static constexpr int LDS = kQ + SR * D * 4;
  static_assert(LDS <= 160 * 1024, "fits a CU");

  using elem_t = T;
  using raw_t = Raw<T>;

  // Where rows lie, in bytes: block blk at blk * block, row sl of KV head h of it at
  // head + sl * row, and a Q8 row's scale at scales + 4 * sl.  (The host takes the blocks
  // that fit 31 bits.)
  struct Pages {
    unsigned block, head, row, scales;
    int mask;
  };
  __device__ static __forceinline__ Pages pages(const RaggedArgs& a, int h) {
    constexpr bool Q8 = std::is_same<T, q8_t>::value;
    const unsigned page = 1u << a.page_shift, rows = a.nkv * page;
    Pages p;
    p.row = a.d * (unsigned)sizeof(T);
    p.block = rows * (p.row + (Q8 ? 4 : 0));
    p.head = h * page * p.row;
    p.scales = rows * a.d + 4 * h * page;
    p.mask = (int)page - 1;
    return p;
  }
  // Where row t of block blk starts in a pool, and its Q8 scale.
  __device__ static __forceinline__ uint64_t row_at(const Pages& p, int blk, int t) {
    return (uint64_t)(unsigned)blk * p.block + (p.head + (unsigned)(t & p.mask) * p.row);
  }
  __device__ static __forceinline__ float scale_at(const Pages& p, const char* pool, int blk, int t) {
    return *reinterpret_cast<const float*>(pool + (uint64_t)(unsigned)blk * p.block +
                                           (p.scales + 4 * (unsigned)(t & p.mask)));
  }
  // Eight elements.  once: no other workgroup reads the row soon.
  __device__ static __forceinline__ void load(const char* x, bool once, raw_t& r) {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f32x4* v = reinterpret_cast<const f32x4*>(x) + i;
        r.x[i] = once ? __builtin_nontemporal_load(v) : *v;
      }
    } else if constexpr (std::is_same<T, bf16_t>::value) {
      const u32x4* v = reinterpret_cast<const u32x4*>(x);
      r.x = once ? __builtin_nontemporal_load(v) : *v;
    } else {
      r.x = *reinterpret_cast<const u32x2*>(x);
    }
  }
  // N chunks of a thread into LDS: chunk i is unit j of row r + STEP*i of the tile (rows
  // past it: of the next), r < KT, STEP a power of two past r or a multiple of KT.  tops:
  // Pieces::top.
  template <int N, int STEP>
  __device__ static __forceinline__ void pieces(const raw_t (&raw)[N], int kv, int r, int j, char* tile,
                                                unsigned (&tops)[N]) {
    const int base = r * RB + 16 * (j ^ (kv ? wv_f<D>(r) : wk_f<D>(r)));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Pieces<NP> x = make_pieces<LPR>(raw[i], kv);
      tops[i] = x.top;
      // (the swizzle of row r + STEP*i is r's and STEP*i's by exclusive or)
      constexpr int M = KT - 1;
      const int up = STEP * i & M;
      char* to = tile + STEP * i / KT * TB + ((base ^ (16 * (kv ? wv_f<D>(up) : wk_f<D>(up)))) + up * RB);
#pragma unroll
      for (int p = 0; p < NP; ++p) *reinterpret_cast<u32x4*>(to + p * PB) = x.p[p];
    }
  }
};

// What the rows of a wave share whatever their number: the row of this lane.
template <int D, typename T, bool SC>
struct RowsBase {
  using C = Tile<D, T, SC>;
  float qunit, fac, mark;
  RowState rs;
  RowScore score;
  int lo, hi;  // the row's keys of this unit
  int room;

  // q's pieces, N steps: step k the elements STEP*k + 8*part .. +7 of row r, as an operand.
  // gmax: the maximum over the row's lanes.
  template <int N, int STEP, typename GMAX>
  __device__ __forceinline__ void init(const RaggedArgs& a, const RaggedUnit& u, const RaggedSeq& sq, int h,
                                       int r, int part, GMAX&& gmax, f16x8_t (&qh)[N], f16x8_t (&ql)[N]) {
    const bool rv = r < sq.rows * a.G;
    const int m = rv ? r / a.G : 0, g = rv ? r - m * a.G : 0, slot = sq.slot0 + m;
    // (a row past the last: any keys, not stored)
    lo = rv ? max(ragged_lo(a, slot), u.lo) : 0;
    hi = rv ? min(ragged_hi(a, slot), u.hi) : 0x7FFFFFFF;
    const float* qr = a.q + (((int64_t)sq.start + m) * a.nq + h * a.G + g) * a.d;
    const float qsc = a.scale * kLog2e;
    // (read twice, the largest first: all of the row at once would take 8 * N registers)
    auto eight = [&](int k, float (&x)[8]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e0 = STEP * k + 8 * part + 4 * i;
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        if (rv && e0 < a.d) y = *reinterpret_cast<const f32x4*>(qr + e0);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e] * qsc;
      }
    };
    float qm = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float x[8];
      eight(k, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) qm = fmaxf(qm, fabsf(x[e]));
    }
    int again = 0;  // (the pointer itself, kept from the compiler so, would make flat loads)
    asm volatile("" : "+v"(again));
    qr += again;
    const int shift = f16_row_shift(gmax(qm));
    qunit = f16_row_unit(shift);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float x[8];
      eight(k, x);
      uint32_t h4[4], l4[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) split2h(x[e], x[e + 1], shift, h4[e / 2], l4[e / 2]);
      qh[k] = __builtin_bit_cast(f16x8_t, u32x4{h4[0], h4[1], h4[2], h4[3]});
      ql[k] = __builtin_bit_cast(f16x8_t, u32x4{l4[0], l4[1], l4[2], l4[3]});
    }
    if constexpr (SC) score = ragged_score(a, h * a.G + g, slot);
    fac = 1.f;
    mark = 0.f;
    room = wide_room(u.hi - u.lo);
  }
  // The same into LDS, for every wave of the workgroup (each writes the same): [step][piece]
  // [lane], at this lane.
  template <int N, int STEP, typename GMAX>
  __device__ __forceinline__ lds_q_t init_lds(const RaggedArgs& a, const RaggedUnit& u,
                                             const RaggedSeq& sq, int h, int r, int lane, int part,
                                             GMAX&& gmax, char* lds) {
    f16x8_t hi[N], lo[N];
    init<N, STEP>(a, u, sq, h, r, part, gmax, hi, lo);
    f16x8_t* const to = reinterpret_cast<f16x8_t*>(lds) + lane;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      to[128 * q] = hi[q];
      to[128 * q + 64] = lo[q];
    }
    return (lds_q_t)to;
  }
  // The tile's probabilities of this lane's N keys, slot(e) their slots.
  template <int N, typename SLOT, typename GMAX>
  __device__ __forceinline__ void tile(float (&x)[N], const float (&ku)[N], const float (&vu)[N], int tk,
                                       SLOT&& slot, GMAX&& gmax, uint32_t (&yh)[N / 2],
                                       uint32_t (&yl)[N / 2]) {
    const bool full = __builtin_amdgcn_ballot_w64(tk < lo || tk + C::KT > hi) == 0;
    auto dead = [&](int e) {
      const int t = slot(e);
      return t < lo || t >= hi;
    };
    if constexpr (SC)
      fac = softmax_tile<N>(x, ku, vu, qunit, rs, full, gmax, dead, yh, yl,
                            [&](float (&z)[N], auto&& again) { score.template apply<N>(z, slot, again); },
                            room);
    else
      fac = softmax_tile<N>(x, ku, vu, qunit, rs, full, gmax, dead, yh, yl);
  }
};

// 32 rows of a wave over its tiles (v_mfma_f32_32x32x16_f16).
template <int D, typename T, bool SC, bool QLDS>
struct Rows32 : RowsBase<D, T, SC> {
  using B = RowsBase<D, T, SC>;
  using C = typename B::C;
  using B::fac, B::mark;
  static constexpr int NR = 32, NV = D / 8;  // rows; vectors of 4 outputs a lane
  static constexpr int QS = D / 16, DB = D / 32, NP = C::NP, RB = C::RB, PB = C::PB;
  f16x8_t qh[QLDS ? 1 : QS], ql[QLDS ? 1 : QS];
  lds_q_t qs;  // QLDS: [step][piece][lane], at this lane
  f32x16 o[DB], s;
  uint32_t yh[8], yl[8];

  __device__ static __forceinline__ float gmax(float v) { return max_xor32(v); }
  __device__ static __forceinline__ float gsum(float v) { return sum_xor32(v); }
  __device__ __forceinline__ void init(const RaggedArgs& a, const RaggedUnit& u, const RaggedSeq& sq, int h,
                                       int r, int lane, char* lds = nullptr) {
    if constexpr (QLDS) qs = B::template init_lds<QS, 16>(a, u, sq, h, r, lane, lane >> 5, gmax, lds);
    else B::template init<QS, 16>(a, u, sq, h, r, lane >> 5, gmax, qh, ql);
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.f;
  }
  // Output vector v of this lane, and where its four elements lie in the row.
  __device__ __forceinline__ f32x4 get(int v) const {
    const auto& x = o[v >> 2];
    const int i = 4 * (v & 3);
    return f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
  }
  __device__ __forceinline__ void put(int v, f32x4 y) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[v >> 2][4 * (v & 3) + e] = y[e];
  }
  __device__ static __forceinline__ int place(int v, int lane) {
    return 32 * (v >> 2) + 8 * (v & 3) + 4 * (lane >> 5);
  }

  // S^T of a tile: keys 8*(i/4) + 4*hh + i%4.  Of each step the products with a low piece
  // first: they are small beside the others, whose sum alone then rounds at its size.
  __device__ __forceinline__ void scores(const char* tile, int lane) {
    const int c32 = lane & 31, hh = lane >> 5;
    const char* kr = tile + c32 * RB;
    const int kx = 16 * (hh ^ wk_f<D>(c32));
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    f16x8_t k[2][2][NP], x[2][2][2];
    auto read_k = [&](int k0) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
          x[(k0 >> 1) & 1][j][p] = QLDS ? qs[128 * (k0 + j) + 64 * p] : (p ? ql : qh)[QLDS ? 0 : k0 + j];
#pragma unroll
        for (int p = 0; p < NP; ++p)
          k[(k0 >> 1) & 1][j][p] =
              *reinterpret_cast<const f16x8_t*>(kr + p * PB + (kx ^ (32 * (k0 + j))));
      }
    };
    read_k(0);
#pragma unroll
    for (int k0 = 0; k0 < QS; k0 += 2) {
      if (k0 + 2 < QS) read_k(k0 + 2);
      __builtin_amdgcn_sched_barrier(0);
      const auto& c = k[(k0 >> 1) & 1];
      const auto& y = x[(k0 >> 1) & 1];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (NP == 2) s = mfma32_f16(c[j][1], y[j][0], s);
        s = mfma32_f16(c[j][0], y[j][1], s);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) s = mfma32_f16(c[j][0], y[j][0], s);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  __device__ __forceinline__ void softmax(const float* ku_, const float* vu_, int tk, int lane) {
    const int hh = lane >> 5;
    float x[16], ku[16], vu[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(ku_ + 4 * hh + 8 * i);
      const f32x4 z = *reinterpret_cast<const f32x4*>(vu_ + 4 * hh + 8 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[4 * i + e] = s[4 * i + e];
        ku[4 * i + e] = y[e];
        vu[4 * i + e] = z[e];
      }
    }
    mark = fmaf(ku_[lane & 31] + vu_[lane & 31], 0.f, mark);
    B::template tile<16>(x, ku, vu, tk, [&](int e) { return tk + 8 * (e >> 2) + 4 * hh + (e & 3); }, gmax, yh,
                         yl);
  }

  // O^T += V^T . P^T.  A transposed read's 16-lane group (2*hh + x) takes keys 16j + 8u +
  // 4hh .. +3 of the block's 16 columns 16x ..: slots 4u + i of the A operand, P's order.
  __device__ __forceinline__ void pv(char* tile, int lane) {
    const int hh = lane >> 5;
    if (__builtin_amdgcn_ballot_w64(fac != 1.f) != 0) {
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= fac;
    }
    const int l16 = lane & 15, rr = 4 * hh + (l16 >> 2);
    char* vr = tile + rr * RB + 32 * ((lane >> 4) & 1) + 16 * ((l16 & 3) >> 1) + 8 * (l16 & 1);
    const int vx = 16 * wv_f<D>(rr);
    f16x8_t av[2][2][NP];
    auto read_v = [&](int q) {  // step q: key half j, output blocks b0 and b0 + 1
      const int j = q / (DB / 2), b0 = 2 * (q % (DB / 2));
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          i16x4_t t2[2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
            t2[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4_t*)(vr + p * PB + (16 * j + 8 * u) * RB +
                                                             ((64 * (b0 + b)) ^ vx)));
          av[q & 1][b][p] =
              __builtin_bit_cast(f16x8_t, __builtin_shufflevector(t2[0], t2[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    read_v(0);
#pragma unroll
    for (int q = 0; q < DB; ++q) {
      if (q + 1 < DB) read_v(q + 1);
      __builtin_amdgcn_sched_barrier(0);
      const int j = q / (DB / 2), b0 = 2 * (q % (DB / 2));
      const f16x8_t ph =
          __builtin_bit_cast(f16x8_t, u32x4{yh[4 * j], yh[4 * j + 1], yh[4 * j + 2], yh[4 * j + 3]});
      const f16x8_t pl =
          __builtin_bit_cast(f16x8_t, u32x4{yl[4 * j], yl[4 * j + 1], yl[4 * j + 2], yl[4 * j + 3]});
      auto& vc = av[q & 1];
      if constexpr (NP == 2) {
#pragma unroll
        for (int b = 0; b < 2; ++b) o[b0 + b] = mfma32_f16(vc[b][1], ph, o[b0 + b]);
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) o[b0 + b] = mfma32_f16(vc[b][0], pl, o[b0 + b]);
#pragma unroll
      for (int b = 0; b < 2; ++b) o[b0 + b] = mfma32_f16(vc[b][0], ph, o[b0 + b]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

__device__ __forceinline__ f32x4 mfma16_f16(f16x8_t a, f16x8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 16 rows of a wave (v_mfma_f32_16x16x32_f16): half the registers.  A lane holds the keys
// 16*b + 4*(lane / 16) + i of row lane % 16, e = 4*b + i.
template <int D, typename T, bool SC, bool QLDS>
struct Rows16 : RowsBase<D, T, SC> {
  using B = RowsBase<D, T, SC>;
  using C = typename B::C;
  using B::fac, B::mark;
  static constexpr int NR = 16, NV = D / 16;
  static constexpr int QS = D / 32, NP = C::NP, RB = C::RB, PB = C::PB;
  f16x8_t qh[QLDS ? 1 : QS], ql[QLDS ? 1 : QS];
  lds_q_t qs;  // QLDS: [step][piece][lane], at this lane
  f32x4 o[NV], s[2];
  uint32_t yh[4], yl[4];

  __device__ static __forceinline__ float gmax(float v) { return max_xor32(max_xor16(v)); }
  __device__ static __forceinline__ float gsum(float v) { return sum_xor32(sum_xor16(v)); }
  __device__ __forceinline__ void init(const RaggedArgs& a, const RaggedUnit& u, const RaggedSeq& sq, int h,
                                       int r, int lane, char* lds = nullptr) {
    if constexpr (QLDS) qs = B::template init_lds<QS, 32>(a, u, sq, h, r, lane, lane >> 4, gmax, lds);
    else B::template init<QS, 32>(a, u, sq, h, r, lane >> 4, gmax, qh, ql);
#pragma unroll
    for (int v = 0; v < NV; ++v) o[v] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ f32x4 get(int v) const { return o[v]; }
  __device__ __forceinline__ void put(int v, f32x4 y) { o[v] = y; }
  __device__ static __forceinline__ int place(int v, int lane) { return 16 * v + 4 * (lane >> 4); }

  __device__ __forceinline__ void scores(const char* tile, int lane) {
    const int r = lane & 15;  // (rows r and 16 + r have one swizzle)
    const char* kr = tile + r * RB;
    const int kx = 16 * ((lane >> 4) ^ wk_f<D>(r));
    f32x4 low[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) s[b] = low[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    f16x8_t k[2][2][NP], x[2][2];
    auto read_k = [&](int q) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
        x[q & 1][p] = QLDS ? qs[128 * q + 64 * p] : (p ? ql : qh)[QLDS ? 0 : q];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int p = 0; p < NP; ++p)
          k[q & 1][b][p] = *reinterpret_cast<const f16x8_t*>(kr + 16 * b * RB + p * PB + (kx ^ (64 * q)));
    };
    read_k(0);
#pragma unroll
    for (int q = 0; q < QS; ++q) {
      if (q + 1 < QS) read_k(q + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] = mfma16_f16(k[q & 1][b][0], x[q & 1][0], s[b]);
#pragma unroll
      for (int b = 0; b < 2; ++b) low[b] = mfma16_f16(k[q & 1][b][0], x[q & 1][1], low[b]);
      if constexpr (NP == 2) {
#pragma unroll
        for (int b = 0; b < 2; ++b) low[b] = mfma16_f16(k[q & 1][b][1], x[q & 1][0], low[b]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[b][i] += low[b][i];
  }

  __device__ __forceinline__ void softmax(const float* ku_, const float* vu_, int tk, int lane) {
    const int g = lane >> 4;
    float x[8], ku[8], vu[8];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(ku_ + 16 * b + 4 * g);
      const f32x4 z = *reinterpret_cast<const f32x4*>(vu_ + 16 * b + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[4 * b + i] = s[b][i];
        ku[4 * b + i] = y[i];
        vu[4 * b + i] = z[i];
      }
    }
    mark = fmaf(ku_[lane & 31] + vu_[lane & 31], 0.f, mark);
    B::template tile<8>(x, ku, vu, tk, [&](int e) { return tk + 16 * (e >> 2) + 4 * g + (e & 3); }, gmax, yh, yl);
  }

  // A transposed read's 16-lane group g takes keys 16b + 4g .. +3 of 16 columns: P's order.
  __device__ __forceinline__ void pv(char* tile, int lane) {
    if (__builtin_amdgcn_ballot_w64(fac != 1.f) != 0) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[v][i] *= fac;
    }
    const int l16 = lane & 15, rr = 4 * (lane >> 4) + (l16 >> 2);
    char* vr = tile + rr * RB + 8 * (l16 & 1);
    const int vx = 16 * (((l16 & 3) >> 1) ^ wv_f<D>(rr));  // (rows rr and 16 + rr alike)
    const f16x8_t ph = __builtin_bit_cast(f16x8_t, u32x4{yh[0], yh[1], yh[2], yh[3]});
    const f16x8_t pl = __builtin_bit_cast(f16x8_t, u32x4{yl[0], yl[1], yl[2], yl[3]});
    f16x8_t av[2][2][NP];
    auto read_v = [&](int v0) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          i16x4_t t2[2];
#pragma unroll
          for (int b = 0; b < 2; ++b)
            t2[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4_t*)(vr + p * PB + 16 * b * RB +
                                                             (vx ^ (32 * (v0 + j)))));
          av[(v0 >> 1) & 1][j][p] =
              __builtin_bit_cast(f16x8_t, __builtin_shufflevector(t2[0], t2[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    read_v(0);
#pragma unroll
    for (int v0 = 0; v0 < NV; v0 += 2) {
      if (v0 + 2 < NV) read_v(v0 + 2);
      __builtin_amdgcn_sched_barrier(0);
      auto& vc = av[(v0 >> 1) & 1];
      if constexpr (NP == 2) {
#pragma unroll
        for (int j = 0; j < 2; ++j) o[v0 + j] = mfma16_f16(vc[j][1], ph, o[v0 + j]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) o[v0 + j] = mfma16_f16(vc[j][0], pl, o[v0 + j]);
#pragma unroll
      for (int j = 0; j < 2; ++j) o[v0 + j] = mfma16_f16(vc[j][0], ph, o[v0 + j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// The end of a unit: x the rows of this wave, group rg of RG of key group kg of KG.
template <int RG, int KG, typename X>
__device__ __forceinline__ void finish(const RaggedArgs& a, const RaggedUnit& u, const RaggedSeq& sq, int h,
                                       X& x, int rg, int kg, char* lds) {
  using C = typename X::C;
  constexpr int D = X::NV * 4 * (64 / X::NR);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int r = u.r0 + X::NR * rg + (lane & (X::NR - 1));
  // a row that the pieces cannot hold: the unit's rows again, each over its own keys
  if (__syncthreads_or(x.mark != 0.f)) {
    for (int i = w; i < RG * X::NR; i += C::NW) ragged_own_row<D / 64, typename C::elem_t>(a, u, h, u.r0 + i);
    return;
  }
  // the key groups' merge, halves at a time: o in units of 2^m
  float l = X::gsum(x.rs.l), m = x.rs.m;
#pragma unroll
  for (int v = 0; v < X::NV; ++v) {
    f32x4 y = x.get(v);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = ldexpf(y[e], -x.rs.wsh);
    x.put(v, y);
  }
#pragma unroll
  for (int half = KG / 2; half > 0; half /= 2) {
    const int at = (kg & (half - 1)) * RG + rg;
    f32x4* mo = reinterpret_cast<f32x4*>(lds) + at * X::NV * 64 + lane;
    f32x2* ml = reinterpret_cast<f32x2*>(lds + C::kData) + at * 64 + lane;
    if (kg >= half && kg < 2 * half) {
#pragma unroll
      for (int v = 0; v < X::NV; ++v) mo[v * 64] = x.get(v);
      *ml = f32x2{m, l};
    }
    __syncthreads();
    if (kg < half) {
      const f32x2 st = *ml;
      const float M = fmaxf(m, st[0]), f0 = exp2_hw(m - M), f1 = exp2_hw(st[0] - M);
      m = M;
      l = l * f0 + st[1] * f1;
#pragma unroll
      for (int v = 0; v < X::NV; ++v) {
        const f32x4 z = mo[v * 64];
        f32x4 y = x.get(v);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = y[e] * f0 + z[e] * f1;
        x.put(v, y);
      }
    }
    if (half > 1) __syncthreads();
  }
  if (kg > 0 || r >= sq.rows * a.G) return;
  const bool part = u.part >= 0;
  const int64_t ps = ((int64_t)u.part * a.nkv + h) * a.slot_rows + (r - u.r0);
  const int mm = r / a.G, g = r - mm * a.G;
  float* out = part ? a.part_o + ps * D : a.o + (((int64_t)sq.start + mm) * a.nq + h * a.G + g) * a.d;
  const int dh = part ? D : a.d;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no key: O = 0
#pragma unroll
  for (int v = 0; v < X::NV; ++v) {
    const int e0 = X::place(v, lane);
    f32x4 y = x.get(v);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = part ? y[e] : div_by(y[e], l, inv);
    if (e0 < dh) *reinterpret_cast<f32x4*>(out + e0) = y;
  }
  if (part && lane < X::NR)
    *reinterpret_cast<f32x2*>(a.part_ml + 2 * ps) = f32x2{l == 0.f ? -INFINITY : m, l};
}

template <int D, typename T, bool SC>
__global__ __launch_bounds__((Tile<D, T, SC>::NT)) void ragged_tile_kernel(RaggedArgs a) {
  using C = Tile<D, T, SC>;
  constexpr int KT = C::KT, LPR = C::LPR;
  __shared__ __attribute__((aligned(16))) char lds[C::LDS];
  float* const units = reinterpret_cast<float*>(lds + C::kData);

  const int ui = blockIdx.x / a.nkv, h = blockIdx.x - ui * a.nkv;
  if (ui >= a.head->nunits) return;
  const RaggedUnit u = a.units[ui];
  const RaggedSeq& sq = u.s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ntile = (u.hi - u.lo + KT - 1) / KT;
  const int last = u.hi - 1;  // rows past it read it again (masked)
  const int32_t* table = a.block_table + (int64_t)u.seq * a.max_blocks;
  // The table's entry for row t; whether it is a block of the pool is asked where it is
  // used, an interval later (here it would wait for every load in flight).
  auto block_of = [&](int t) { return table[min(t, last) >> a.page_shift]; };
  auto valid = [&](int id) { return (unsigned)id < (unsigned)a.num_blocks ? id : 0; };
  const typename C::Pages pg = C::pages(a, h);

  if (u.wide) {
    using X = typename std::conditional<C::WR == 32, Rows32<D, T, SC, false>,
                                        Rows16<D, T, SC, false>>::type;
    const bool rows = u.r0 + X::NR * w < sq.rows * a.G;  // else this wave only stages
    constexpr int KI = C::IT * KT;                       // keys an interval
    const int nint = (ntile + C::IT - 1) / C::IT;
    auto tile_buf = [&](int kv, int bf, int g) { return lds + ((kv * 2 + bf) * C::IT + g) * C::TB; };
    auto unit_buf = [&](int kv, int bf, int g) { return units + ((kv * 2 + bf) * C::IT + g) * KT; };
    constexpr bool Q8 = std::is_same<T, q8_t>::value;
    typename C::raw_t kr[C::CW], vr[C::CW];
    float ks[C::CW], vs[C::CW];  // (Q8)
    int blk[C::CW];
    // chunk i of this thread: unit j of row rr + STEP*i of the interval's tiles in a row
    constexpr int STEP = C::NT / LPR;
    static_assert(STEP % KT == 0 || C::IT == 1, "chunks of a thread: of tiles, or of one tile");
    const int rr = tid / LPR, j = tid % LPR;
    // (lanes past d take the row's first: they meet zeros of q, or columns that are not stored)
    const unsigned at = 8 * j < a.d ? 8 * j * (unsigned)sizeof(T) : 0;
    auto key = [&](int it, int i) { return u.lo + KI * it + rr + STEP * i; };
    auto blocks = [&](int it) {
#pragma unroll
      for (int i = 0; i < C::CW; ++i) blk[i] = block_of(key(it, i));
    };
    // the rows of interval it, and the blocks of the one after it (its rows' clamp: any it)
    auto fetch = [&](int it) {
#pragma unroll
      for (int i = 0; i < C::CW; ++i) {
        const int t = min(key(it, i), last), b = valid(blk[i]);
        const uint64_t row = C::row_at(pg, b, t) + at;
        C::load(a.k + row, false, kr[i]);
        C::load(a.v + row, false, vr[i]);
        if constexpr (Q8) {
          ks[i] = C::scale_at(pg, a.k, b, t);
          vs[i] = C::scale_at(pg, a.v, b, t);
        }
      }
      blocks(it + 1);
    };
    // (an interval's tiles lie one after the other, and their units)
    auto stage = [&](int it) {
      unsigned ku[C::CW], vu[C::CW];
      const int r0 = rr % KT, g0 = rr / KT;
      C::template pieces<C::CW, STEP>(kr, 0, r0, j, tile_buf(0, it & 1, g0), ku);
      C::template pieces<C::CW, STEP>(vr, 1, r0, j, tile_buf(1, it & 1, g0), vu);
      if (j == 0) {
#pragma unroll
        for (int i = 0; i < C::CW; ++i) {
          float k, v;
          if constexpr (Q8) {
            k = q8_unit(ks[i], 1, 0);
            v = q8_unit(vs[i], vu[i], 1);
          } else {
            k = unit_of(T{}, ku[i], 0);
            v = unit_of(T{}, vu[i], 1);
          }
          unit_buf(0, it & 1, 0)[rr + STEP * i] = k;
          unit_buf(1, it & 1, 0)[rr + STEP * i] = v;
        }
      }
    };
    if (nint > 0) {
      blocks(0);
      fetch(0);
    }
    X x;  // (the first rows on their way)
    x.init(a, u, sq, h, u.r0 + X::NR * w + (lane & (X::NR - 1)), lane);
    if (nint > 0) {
      stage(0);
      fetch(1);
    }
    __syncthreads();
    const bool first = w < C::NW / 2;
    for (int it = 0; it < nint; ++it) {
      const int bf = it & 1;
      const bool more = it + 1 < nint;
      if (!first && more) {
        stage(it + 1);
        fetch(it + 2);
      }
      if (rows) {
#pragma unroll
        for (int g = 0; g < C::IT; ++g) {
          x.scores(tile_buf(0, bf, g), lane);
          x.softmax(unit_buf(0, bf, g), unit_buf(1, bf, g), u.lo + KI * it + KT * g, lane);
          x.pv(tile_buf(1, bf, g), lane);
        }
      }
      if (first && more) {
        stage(it + 1);
        fetch(it + 2);
      }
      lds_barrier();
    }
    finish<C::NW, 1>(a, u, sq, h, x, w, 0, lds);
    return;
  }

  auto narrow = [&](auto& x) {
    using X = typename std::remove_reference<decltype(x)>::type;
    const int r = u.r0 + (lane & (X::NR - 1));
    if (w >= C::NWN) {
      x.init(a, u, sq, h, r, lane, lds + C::kQ);
    } else {
      char* const buf = lds + w * C::TB;
      float* const ub = units + w * 2 * KT;
      // K and V each have their registers where those are few enough
      constexpr bool BOTH = C::CN * (int)sizeof(typename C::raw_t) <= 128;
      constexpr bool Q8 = std::is_same<T, q8_t>::value;
      // (an fp32 tile of d = 256 takes 128: its halves one after the other)
      constexpr int HALVES = C::CN * (int)sizeof(typename C::raw_t) > 256 ? 2 : 1, CH = C::CN / HALVES;
      typename C::raw_t raw[BOTH ? 2 : 1][CH];
      float scale[2];          // (Q8: of key lane % 32)
      constexpr int RPI = 64 / LPR;  // rows of a load
      const int r_in = lane / LPR, j = lane % LPR, key = lane & 31;
      const unsigned at = 8 * j < a.d ? 8 * j * (unsigned)sizeof(T) : 0;
      const char *kp = a.k + at, *vp = a.v + at;
      // A lane forms the place of one key, in units of 8 bytes, and the key's lanes take it
      // from there.
      auto ids = [&](int t) { return block_of(u.lo + t * KT + key); };
      auto slot_of = [&](int t) { return min(u.lo + t * KT + key, last); };
      auto place = [&](int t, int id) { return (unsigned)(C::row_at(pg, valid(id), slot_of(t)) >> 3); };
      auto fetch = [&](int kv, int t, int id, unsigned off, int half = 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
          C::load((kv ? vp : kp) + ((uint64_t)(unsigned)__shfl((int)off, r_in + RPI * (half * CH + i)) << 3),
                  true, raw[BOTH ? kv : 0][i]);
        if constexpr (Q8) scale[kv] = C::scale_at(pg, kv ? a.v : a.k, valid(id), slot_of(t));
      };
      auto stage = [&](int kv, unsigned off) {
        float* const to = ub + kv * KT;
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          unsigned top[CH];
          const int r = r_in + RPI * CH * half;
          if (half) fetch(kv, 0, 0, off, half);
          C::template pieces<CH, RPI>(raw[BOTH ? kv : 0], kv, r, j, buf, top);
          if (j == 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i) to[r + RPI * i] = __uint_as_float(top[i]);
          }
        }
        asm volatile("" ::: "memory");  // the wave's own LDS: in order
        const unsigned mine = __float_as_uint(to[key]);
        float unit;
        if constexpr (Q8) unit = q8_unit(scale[kv], mine, kv);
        else unit = unit_of(T{}, mine, kv);
        to[key] = unit;  // (both lanes of a key the same)
        asm volatile("" ::: "memory");
      };
      int id = 0, idn = 0;
      unsigned off = 0;
      if (w < ntile) {
        id = ids(w);
        off = place(w, id);
        fetch(0, w, id, off);
        if (BOTH) fetch(1, w, id, off);
        idn = ids(w + C::NWN);
      }
      x.init(a, u, sq, h, r, lane, lds + C::kQ);  // (the first rows on their way)
      for (int t = w; t < ntile; t += C::NWN) {
        const bool more = t + C::NWN < ntile;
        stage(0, off);
        const unsigned off1 = off;
        if (!BOTH) fetch(1, t, id, off);
        if (more) {
          id = idn;
          off = place(t + C::NWN, id);
          idn = ids(t + 2 * C::NWN);
          if (BOTH) fetch(0, t + C::NWN, id, off);
        }
        x.scores(buf, lane);
        asm volatile("" ::: "memory");
        stage(1, off1);
        if (more) fetch(BOTH ? 1 : 0, t + C::NWN, id, off);
        x.softmax(ub, ub + KT, u.lo + t * KT, lane);
        x.pv(buf, lane);
        asm volatile("" ::: "memory");
      }
    }
    finish<1, C::NWN>(a, u, sq, h, x, 0, w, lds);
  };
  if constexpr (C::SR == 32) {
    if (u.rows == 32) {
      Rows32<D, T, SC, true> x;
      narrow(x);
      return;
    }
  }
  Rows16<D, T, SC, C::QLDS> x;
  narrow(x);
}

template <int D, bool SC>
RaggedTile tile_of(int kv_dtype) {
  using C = Tile<D, float, SC>;  // (the wide rows are every type's)
  return {kv_dtype == MOLOT_KV_F32    ? ragged_tile_kernel<D, float, SC>
          : kv_dtype == MOLOT_KV_BF16 ? ragged_tile_kernel<D, bf16_t, SC>
                                      : ragged_tile_kernel<D, q8_t, SC>,
          C::NT, C::QL, kv_dtype == MOLOT_KV_F32 ? C::SR : Tile<D, bf16_t, SC>::SR};
}

}  // namespace

RaggedTile ragged_tile(int d, int kv_dtype, bool scored) {
  if (d <= 64) return scored ? tile_of<64, true>(kv_dtype) : tile_of<64, false>(kv_dtype);
  if (d <= 128) return scored ? tile_of<128, true>(kv_dtype) : tile_of<128, false>(kv_dtype);
  return scored ? tile_of<256, true>(kv_dtype) : tile_of<256, false>(kv_dtype);
}
