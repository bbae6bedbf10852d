// How the library's workspaces grow.  Plain C++.
#ifndef MOLOT_AMD_CSRC_WS_GROWTH_HPP_
#define MOLOT_AMD_CSRC_WS_GROWTH_HPP_

#include <algorithm>
#include <cstddef>

// Bytes to allocate for a call that needs `bytes` where a buffer of `have` (0: none) is too
// small: twice the old size, but no more than `most` where the call needs no more.  An
// outgrown buffer stays allocated (a captured graph may point at it), so buffers of
// just the size asked for would pile up as a cache grows row by row.  Doubled, all the
// outgrown ones are less than the live one; the last, at `most`, may follow one of
// nearly its size, and then they are less than twice it.
constexpr size_t grown_bytes(size_t bytes, size_t have, size_t most) {
  return std::max(bytes, std::min(2 * have, most));
}

#endif  // MOLOT_AMD_CSRC_WS_GROWTH_HPP_
