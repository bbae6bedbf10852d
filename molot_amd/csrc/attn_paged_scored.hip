// Decode attention over a paged cache, scored: the kernels' instances.
#include "attn_launch.hpp"

int molot_host::run_paged_scored(AttnArgs& a, bool rope, int d, int kv_dtype, int span, int B,
                                 void* stream) {
  return rope ? run_attn<true, true, true>(a, d, kv_dtype, span, B, stream)
              : run_attn<true, false, true>(a, d, kv_dtype, span, B, stream);
}
