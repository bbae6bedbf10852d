// Decode attention over a paged cache: the kernels' instances.
#include "attn_launch.hpp"

int molot_host::run_paged(AttnArgs& a, bool rope, int d, int kv_dtype, int span, int B,
                          void* stream) {
  return rope ? run_attn<true, true, false>(a, d, kv_dtype, span, B, stream)
              : run_attn<true, false, false>(a, d, kv_dtype, span, B, stream);
}
