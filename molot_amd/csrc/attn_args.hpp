// The decode attention launch shared by its kernel and host sources.
#ifndef MOLOT_AMD_CSRC_ATTN_ARGS_HPP_
#define MOLOT_AMD_CSRC_ATTN_ARGS_HPP_

#include <cstdint>

struct AttnArgs {
  const float* q;        // [B][nq][D]; un-rotated when the kernel applies RoPE
  float* q_out;          // [B][nq][D] rotated q (ROPE); written after every read of q
  const float* k_new;    // [B][nkv][D] fp32 (ROPE)
  const float* v_new;    // [B][nkv][D] fp32 (ROPE)
  void* k;               // KV cache
  void* v;
  const float* inv_freq; // [D/2] (ROPE)
  float* o;              // [B][nq][D]
  float* part_o;         // [slots][nchunks][GH*D] chunk partial o (split-K)
  float* part_ml;        // [slots][nchunks][GH][2] chunk partial (max, sum)
  float* qrot;           // [slots][GH*D] rotated q for the combine kernel (ROPE)
  void* ext_ws;          // host side only: caller-provided workspace (NULL: the library's)
  int64_t ext_ws_bytes;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* pos_arr;
  int64_t tok_stride, head_stride, block_stride;
  int nq, nkv, n, t0, pos, chunk, nchunks, max_blocks, page_shift, window;
  int dh;                // head dim as stored (< D: the kernel runs padded to its D)
  int dynamic;           // 1: waves claim blocks from a workgroup counter; 0: fixed order
  int chunk_fast;        // 1-D grid, the KV heads of a chunk on one XCD (Q8; see launch_pair)
  // Prefill rows (attention-only launches): "sequence" b is query row b of a
  // prompt, at position pos + b, attending [t0_b, min(pos + b + 1, n)) of the
  // one cache (contiguous, or the prompt's block-table row: max_blocks = 0),
  // t0_b from the window (include/molot/gemm.h:409-446).
  int pf;
  int nseq;              // chunk_fast, dyn: sequences of the launch
  // Paged matrix-core launches: the rows a chunk takes follow the sequences'
  // lengths (paged_chunk), so that about dyn workgroups have work (0: chunk
  // as given).  chunk then bounds it from above (the LDS layout), nchunks the
  // chunks of a sequence of at most dyn_span rows (dyn = 0: no limit), and the
  // grid is flat over the (sequence, chunk) pairs.
  int dyn, dyn_span;
  int dyn_min;           // host side: the least chunk (and dyn_pairs, below)
  int matrix, brief;     // host side: the matrix-core kernel; a short context (kBriefSpan)
  // In-launch merge (see arrive_and_merge): every chunk of a slot runs on one
  // XCD, and the workgroup that completes a slot merges its chunk partials.
  int fold;              // ROPE: 1 = the step appends the new token (folded into the last
                         // chunk, slot n-1); 0 = q prologue only (a layer reading another
                         // layer's KV: all n slots come from the cache)
  unsigned long long* ctr;  // [slots] arrival words (arrive_and_merge), zero between launches
                            // (NULL: combine kernel)
  int xmap;              // 1-D grid of 8 * nchunks: slot id % 8 on XCD id % 8 (fewer than 8 slots)
  int slots;             // slots of the launch (xmap)
  int mrg;               // floats of LDS for the merge's chunk statistics (0: no in-launch merge)
  float scale;
  // the layer's norms of the fresh vectors (ROPE only; NULL / 0: none)
  const float* q_norm;   // [D] weights of the per-head q RMS norm
  const float* k_norm;   // [D] weights of the per-head k RMS norm
  int v_norm;            // RMS-norm v over all nkv*D values, no weights
  float eps;
  // Q8 caches: byte offset of head 0's fp32 row scales from the token's row
  // (token-major) or the block (paged), and the byte stride between heads'
  // scales; a paged block's scales step 4 bytes per slot
  int64_t sc_off, sc_head;
  int q8;                // host side: a matrix-core launch on Q8 rows
  int dyn_likely;        // host side: DynPlan::likely
  int dyn_pairs;         // host side: (sequence, chunk) pairs the grid holds
  // Scored launches (the SC instances).  softcap > 0: a score s becomes softcap *
  // tanh(s / softcap); slopes (device [nq], NULL: none): then s -= slope_h * |pos - t|
  // at slot t; key_lo, key_hi (prefill rows; device [M], NULL: none): the first
  // key of a row's range where that lies past its window's, and its end in
  // place of pos + 1.
  int scored;            // host side: the SC instances
  float softcap;
  const float* slopes;
  const int32_t* key_lo;
  const int32_t* key_hi;
  // The weights (acc): the launch leaves its scores, in base-2 units, at
  // scores[(sequence, KV head)][sc_rows rows from t0][nq / nkv heads] (the
  // matrix-core kernel: [sc_rows / 4][heads][4 rows]) and each
  // chunk's (max in base 2, sum) at stats[slot][nchunks][GH] for
  // attn_weights_kernel, which adds the softmax weights to acc (layout of the
  // C ABI) (NULL: no weights).  fresh: slot n - 1 was appended by this call: its
  // acc is set, not added to, and with slot_pos so is its position.
  float* scores;
  float* stats;
  float* acc;            // host side, as the rest
  int32_t* slot_pos;
  int64_t sc_rows;
  int acc_cap, fresh;
  int sc_span;           // rows from t0 that the launch forms scores of, whatever the lengths
};
using AttnFn = void (*)(AttnArgs);

#endif  // MOLOT_AMD_CSRC_ATTN_ARGS_HPP_
