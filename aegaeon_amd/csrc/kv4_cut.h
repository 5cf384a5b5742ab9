// How the attention of several query tokens over the 4-bit cache cuts its keys:
// arithmetic alone, without device code.
#pragma once

#include <cstdint>

namespace aegkv {

// The ranges into which n_kt key steps are cut at a span of at most `span` each (one
// without any step; INT32_MAX: uncut).
constexpr int ranges_of(int n_kt, int span) {
  const uint32_t r = ((uint32_t)n_kt + (uint32_t)span - 1) / (uint32_t)span;  // < 2^32
  return r > 1 ? (int)r : 1;
}

}  // namespace aegkv
