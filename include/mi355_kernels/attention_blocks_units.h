// What attention of blocks of rows counts in 32 bits, for the host: the rows of a key-value head (new tokens times the query
// heads that share it) and the blocks of a launch, of one block more for every sequence at most.
#pragma once

namespace mi355 {
namespace blocks {

constexpr int kRows = 128;  // of a block

inline long long blocks_of(long long tokens, long long group, long long sequences) { return tokens * group / kRows + sequences; }
inline bool fit(long long tokens, long long group, long long kv_heads, long long sequences) {
  return tokens * group <= 1 << 30 && tokens * group * kv_heads <= 1LL << 40 && blocks_of(tokens, group, sequences) <= (1LL << 30) / kv_heads;
}

}  // namespace blocks
}  // namespace mi355
