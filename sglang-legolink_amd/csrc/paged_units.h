// Arithmetic that the paged attention kernels share with their host side.
#ifndef PAGED_UNITS_H
#define PAGED_UNITS_H

namespace {

// Key tiles of a chunk in a call that does not split (64 keys each: as many as an
// int counts).
constexpr int kOneChunk = 33554431;

// How many parts of `part` (at least 1) hold `total` (at least 0); one for none.
// (Unsigned: the sum of two ints may pass 2^31 - 1, where a call's one chunk holds
// any length.)
constexpr int parts_of(int total, int part) {
  const unsigned parts = (static_cast<unsigned>(total) + static_cast<unsigned>(part) - 1u) / static_cast<unsigned>(part);
  return parts == 0u ? 1 : static_cast<int>(parts);
}

}  // namespace

#endif  // PAGED_UNITS_H
