// sb::rows_overlap (semblend_amd/csrc/sb_overlap.h) against all pairs of rows, for every small size and stride.
#include <cstdio>
#include <cstdlib>

#include "../semblend_amd/csrc/sb_overlap.h"

int main() {
  long bad = 0, shared = 0, total = 0;
  for (int tokens = 1; tokens <= 5; ++tokens)
    for (int heads = 1; heads <= 5; ++heads)
      for (int dim = 1; dim <= 4; ++dim)
        for (int token = -24; token <= 24; ++token)
          for (int head = -24; head <= 24; ++head) {
            bool want = false;
            for (int a = 0; a < tokens * heads; ++a)
              for (int b = 0; b < a; ++b)
                want |= std::abs((a / heads - b / heads) * token + (a % heads - b % heads) * head) < dim;
            ++total, shared += want;
            bad += want != sb::rows_overlap(tokens, heads, dim, token, head);
          }
  std::printf("%ld cases, %ld shared, %ld wrong\n", total, shared, bad);
  return bad != 0;
}
