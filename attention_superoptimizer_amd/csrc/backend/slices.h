// A count that goes in several launches.
#pragma once

namespace mi355 {

// launch(at, count) for parts of `most` (at least 1) that make up `total`, until one does not give 0: what it gives.
// (64 bits: the place behind the last part may not fit an int.)
template <class Launch>
int in_slices(long long total, long long most, Launch launch) {
  for (long long at = 0; at < total; at += most) {
    if (int rc = launch(at, total - at < most ? total - at : most)) {
      return rc;
    }
  }
  return 0;
}

}  // namespace mi355
