// What paged attention counts in 32 bits, for the host: its kernels number the units of work of a launch, 32 keys for every
// wavefront of a workgroup, with an int.  Callers have bounded kv_heads * rows by 2^29 and keys by 2^30.
#pragma once

#include <climits>

namespace mi355 {
namespace paged {

constexpr int kTile = 32;  // keys of a wavefront at a time

// Thousands of heads over tables of a few keys may go to workgroups of one wavefront, all others to four or eight.
constexpr long long kManyHeads = 2048, kShortTable = 512;
inline bool one_wavefront(long long heads, long long rows, long long keys) { return heads >= kManyHeads && keys <= kShortTable && rows <= 16; }
// the smallest unit of a kernel that a call may be given, over tables that name `keys` keys
inline int smallest_unit(long long rows, long long keys) { return one_wavefront(LLONG_MAX, rows, keys) ? kTile : 4 * kTile; }

// Units of a sequence with `rows` rows for each of its key-value heads, at most: a head has blocks of 16 rows or more, and
// keys that begin within a tile.
inline long long units_of_sequence(long long kv_heads, long long rows, long long keys) {
  return kv_heads * (rows / 16 + 1) * (keys / smallest_unit(rows, keys) + 2);
}
// Whether a sequence alone has too many.  (A quarter of what an int counts, in units of 128 keys; 3.4 times as many of 32,
// where there are those, still fit.)
inline bool too_many_units(long long kv_heads, long long rows, long long keys) {
  return kv_heads * (rows / 16 + 1) * (keys / (4 * kTile) + 2) > INT_MAX / 4;
}
// Sequences of a launch.
inline long long sequences_at_once(long long kv_heads, long long rows, long long keys) {
  long long const fit = INT_MAX / 2 / units_of_sequence(kv_heads, rows, keys);
  return fit < 1 ? 1 : fit;
}

// With a window, and the first `sinks` tokens: the keys that new_tokens rows in a row see together, at most, and the sequences of a launch.  Which kernel has the call
// goes by these keys and not by the table's, and so does the size of its units.
inline long long keys_seen(long long keys, long long window, long long sinks, long long new_tokens) {
  long long const seen = window != 0 ? window + new_tokens - 1 + sinks : keys;
  return seen < keys ? seen : keys;
}
inline long long masked_at_once(long long kv_heads, long long rows, long long seen) { return sequences_at_once(kv_heads, rows, seen); }

}  // namespace paged
}  // namespace mi355
