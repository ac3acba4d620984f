// What attention of blocks of rows counts in 32 bits, for the host: the rows of a key-value head (new tokens times the query
// heads that share it), and the workgroups of a launch, whose threads the runtime counts in 32 bits.
#pragma once

namespace mi355 {
namespace blocks {

constexpr int kRows = 128;                          // of a block
constexpr long long kWorkgroups = (1LL << 24) - 1;  // of 256 threads

// Blocks of a ragged batch: sequence i's begin at blocks_of(its first token, group, i), and fit before the next one's.
inline long long blocks_of(long long tokens, long long group, long long sequences) { return tokens * group / kRows + sequences; }
// Blocks of a sequence with `rows` rows for each key-value head, and sequences of a launch.
inline long long row_blocks(long long rows) { return (rows + kRows - 1) / kRows; }
inline long long sequences_at_once(long long rows, long long kv_heads) { return rows < 1 ? kWorkgroups : kWorkgroups / (row_blocks(rows) * kv_heads); }

// Whether a call can be counted: `tokens` rows of queries, in equal numbers of `sequences` or ragged.
inline bool fit(long long tokens, long long group, long long kv_heads, long long sequences, bool ragged) {
  if (sequences < 1 || tokens * group > 1 << 30) {
    return sequences < 1;
  }
  return ragged ? blocks_of(tokens, group, sequences) <= kWorkgroups / kv_heads : sequences_at_once(tokens / sequences * group, kv_heads) >= 1;
}

}  // namespace blocks
}  // namespace mi355
