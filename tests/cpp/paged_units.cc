// Lines "kv_heads rows keys" from stdin: whether a sequence is refused, sequences of a launch, and the most units that such a
// launch numbers by any kernel that it may be given.
#include "mi355_kernels/paged_units.h"

#include <algorithm>
#include <cstdio>

int main() {
  long long kv, rows, keys;
  while (std::scanf("%lld %lld %lld", &kv, &rows, &keys) == 3) {
    using namespace mi355::paged;
    long long const at_once = sequences_at_once(kv, rows, keys);
    long long most = 0;
    // what a launch counts (paged_attention.h): units of a sequence x heads, heads in blocks of 16 rows at least; a window may
    // begin 31 keys into its first tile, which the units begin with
    long long const blocks = (rows + 15) / 16, heads = at_once * kv * blocks;
    for (int waves : {1, 4, 8}) {
      if (waves > 1 || one_wavefront(heads, rows, keys)) {
        long long const unit = 32LL * waves;
        most = std::max(most, heads * std::max(1LL, (keys + unit - 1) / unit));
      }
    }
    std::printf("%d %lld %lld\n", too_many_units(kv, rows, keys) ? 1 : 0, at_once, most);
  }
  return 0;
}
