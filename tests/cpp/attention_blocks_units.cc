// Lines "tokens group kv_heads sequences ragged" from stdin: whether such a call is counted, and the workgroups of its largest launch.
#include "mi355_kernels/attention_blocks_units.h"

#include <algorithm>
#include <cstdio>

int main() {
  long long tokens, group, kv, sequences;
  int ragged;
  while (std::scanf("%lld %lld %lld %lld %d", &tokens, &group, &kv, &sequences, &ragged) == 5) {
    using namespace mi355::blocks;
    bool const counted = fit(tokens, group, kv, sequences, ragged != 0);
    long long units = 0;
    if (counted && sequences > 0) {
      long long const rows = tokens / sequences * group;
      units = ragged != 0 ? blocks_of(tokens, group, sequences) * kv : std::min(sequences, sequences_at_once(rows, kv)) * row_blocks(rows) * kv;
    }
    std::printf("%d %lld\n", counted ? 1 : 0, units);
  }
}
