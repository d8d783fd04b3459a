// Segments of a piece's keys: as many as have their pages' numbers in LDS at once
// (chunk_share.hip, chunk_attention.hip).
#pragma once

#include <algorithm>
#include <cstdint>

namespace svdmlp {

constexpr int64_t kChunkTokensMost = 0x7ffe0000;  // tokens of a sequence that attention over chunks takes
constexpr int64_t kSegmentMost = 1 << 16;         // keys of a segment
// Behind the last key there is room for a segment and for the last tiles' ends.
static_assert(kChunkTokensMost + kSegmentMost + 4096 <= 0x7fffffff, "positions fit 31 bits");

// Keys of a segment, in whole tiles of `tile`: they lie in at most `ids` pages wherever
// they begin.  (64 >= tile, ids > tile)
constexpr int segment_keys(int ids, int page, int tile) {
  return (int)std::min((int64_t)(ids - 1) * page / tile, kSegmentMost / tile) * tile;
}

}  // namespace svdmlp
