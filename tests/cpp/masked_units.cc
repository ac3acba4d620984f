// Lines "kv_heads group new_tokens keys window sinks" from stdin: sequences of a launch of attention of few rows within a window, and the most units that it
// numbers by any kernel that it may be given.
#include "mi355_kernels/paged_units.h"

#include <algorithm>
#include <cstdio>

int main() {
  long long kv, group, tokens, keys, window, sinks;
  while (std::scanf("%lld %lld %lld %lld %lld %lld", &kv, &group, &tokens, &keys, &window, &sinks) == 6) {
    using namespace mi355::paged;
    long long const rows = tokens * group, seen = keys_seen(keys, window, sinks, tokens), at_once = masked_at_once(kv, rows, seen), heads = at_once * kv;
    long long most = 0;
    for (int waves : {1, 4, 8}) {
      if (waves > 1 || one_wavefront(heads, rows, seen)) {
        long long const unit = 32LL * waves;
        most = std::max(most, heads * std::max(1LL, (seen + unit - 1) / unit));
      }
    }
    std::printf("%lld %lld\n", at_once, most);
  }
  return 0;
}
