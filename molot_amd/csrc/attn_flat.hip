// Decode attention over a contiguous cache: the kernels' instances.
#include "attn_launch.hpp"

int molot_host::run_flat(AttnArgs& a, bool rope, int d, int kv_dtype, int span, int B,
                         void* stream) {
  return rope ? run_attn<false, true, false>(a, d, kv_dtype, span, B, stream)
              : run_attn<false, false, false>(a, d, kv_dtype, span, B, stream);
}
