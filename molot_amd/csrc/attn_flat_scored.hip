// Decode attention over a contiguous cache, scored: the kernels' instances.
#include "attn_launch.hpp"

int molot_host::run_flat_scored(AttnArgs& a, bool rope, int d, int kv_dtype, int span, int B,
                                void* stream) {
  return rope ? run_attn<false, true, true>(a, d, kv_dtype, span, B, stream)
              : run_attn<false, false, true>(a, d, kv_dtype, span, B, stream);
}
