// Segments of a piece's keys: as many as have their pages' numbers in LDS at once
// (chunk_share.hip, chunk_attention.hip).  A piece may end within 2^17 keys of 2^31, so that
// a position and a segment may pass 31 bits: what is left of the piece is counted
// instead, which only falls.
#pragma once

#include <cstdint>

namespace svdmlp {

// Keys of a segment, in whole tiles of `tile`: they lie in at most `ids` pages wherever
// they begin, and are at most 2^24 tiles.  (ids > tile <= 64)
constexpr int segment_keys(int ids, int page, int tile) {
  const int64_t tiles = (int64_t)(ids - 1) * page / tile;
  return (int)(tiles < (int64_t)1 << 24 ? tiles : (int64_t)1 << 24) * tile;
}

struct Segments {
  int left, most;  // keys not taken yet, keys of a segment

  constexpr Segments(int keys, int most_) : left(keys), most(most_) {}
  constexpr bool more() const { return left > 0; }
  constexpr int keys() const { return left < most ? left : most; }
  constexpr void next() { left -= most; }  // (left is over 0 and most at most 2^30)
};

}  // namespace svdmlp
