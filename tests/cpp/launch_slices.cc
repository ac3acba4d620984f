// Lines "total most" from stdin: launches, and what they cover; -1 where a part does not follow the one before.
#include "slices.h"

#include <cstdio>

int main() {
  long long total, most;
  while (std::scanf("%lld %lld", &total, &most) == 2) {
    long long next = 0, launches = 0;
    int const rc = mi355::in_slices(total, most, [&](long long at, long long count) {
      launches++;
      if (at != next || count < 1 || count > most || launches > 1 << 20) {
        return -1;
      }
      next += count;
      return 0;
    });
    std::printf("%d %lld %lld\n", rc, launches, next);
  }
  return 0;
}
