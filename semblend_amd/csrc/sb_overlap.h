// Whether the rows of an output share elements: two threads would write them in no order. Compiled for the host as
// well, so that a CPU test can compare it with all pairs of rows.
#pragma once

#include <cstdint>

namespace sb {
namespace {

// Whether rows of `dim` elements at t * token + h * head (strides in elements), t < tokens, h < heads,
// share elements: some difference of two places is below dim.
inline bool rows_overlap(int64_t tokens, int64_t heads, int64_t dim, int64_t token, int64_t head) {
  token = token < 0 ? -token : token, head = head < 0 ? -head : head;
  if ((tokens > 1 && token < dim) || (heads > 1 && head < dim)) return true;
  if (tokens <= 1 || heads <= 1) return false;
  // (the usual orders: heads within a token, or tokens within a head)
  if (token >= (heads - 1) * head + dim || head >= (tokens - 1) * token + dim) return false;
  for (int64_t h = 1; h < heads; ++h) {  // both strides are dim at least: the nearest tokens on either side
    const int64_t t = h * head / token, rest = h * head - t * token;
    if (t >= tokens) break;
    if (rest < dim || (t + 1 < tokens && token - rest < dim)) return true;
  }
  return false;
}

}  // namespace
}  // namespace sb
