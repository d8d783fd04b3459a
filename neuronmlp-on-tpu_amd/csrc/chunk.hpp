// What the kernels of attention over chunks share (chunk_attention.hip,
// chunk_share.hip, chunk_wave.hip): which block does what, and where its sums go.
#pragma once

#include <math.h>

#include <algorithm>

#include "attn.hpp"
#include "decoder.hpp"

namespace svdmlp {

namespace {  // as the kernels that take them

// Inclusive prefix sums and maxima over the wave, in the vector unit (rows of 16
// lanes by shifts, then the last lane of a row and of half the wave to the others).
template <class F>
__device__ __forceinline__ int scan(int v, int none, F f) {
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false));
  return f(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false));
}
__device__ __forceinline__ int sums_upto(int v) {
  return scan(v, 0, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int most_upto(int v) {
  return scan(v, 0, [](int a, int b) { return max(a, b); });
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int i) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, i) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32);
}

// A tile, and unit u of its `units`.
struct Place {
  int hk, b, tile, start, n, len, u, units;
};

// The bounds of the first 64 sequences, which a block keeps in LDS for its later
// pieces: read again while other blocks load keys, they took 4 us.
struct Kept {
  int start[64], n[64], len[64], ends[64];
};

// The work of a class (all of a wave's lanes together).  Units fit 31 bits: the host
// chooses their size so.
template <bool MANY>
class Line {
 public:
  // first: the block's first one, whose bounds are read and kept; all of its threads are here.
  __device__ __forceinline__ Line(const ChunkParams& p, const ChunkClass& k, int lane, SVDMLP_ATTN_LDS Kept* kept, bool first)
      : p_(p), k_(k), lane_(lane) {
    int tiles = 0;
    Carry c = {};
    for (int b0 = 0; b0 < p_.B; b0 += 64) {
      Some s;
      if (b0 == 0 && !first) {
        s = tiles_of({kept->start[lane], kept->n[lane], kept->len[lane], 0, __builtin_amdgcn_readfirstlane(kept->ends[lane])});
        c.ends = s.ends;
      } else {
        s = some(b0, c);
      }
      if (b0 == 0 && first) {
        if (threadIdx.x < 64) kept->start[lane] = s.start, kept->n[lane] = s.n, kept->len[lane] = s.len, kept->ends[lane] = s.ends;
        __syncthreads();
      }
      if (b0 == 0) first_ = s;
      tiles += sum(s.tiles);
    }
    slope_ = k_.slope;
    if (p_.B <= 64 && (int64_t)tiles * p_.Hk <= k_.blocks && alone(tiles)) return;
    // Tiles that are blocks of their own: whole rounds of them, all but the last.
    const int rounds = MANY ? (int)((int64_t)tiles * p_.Hk / k_.blocks) - 1 : 0;
    from_ = max(rounds, 0) * (int64_t)k_.blocks / p_.Hk;
    whole = from_ * p_.Hk;
    int units = 0;
    c = {};
    for (int b0 = 0; b0 < p_.B; b0 += 64) {
      Some s = first_;
      if (b0) s = some(b0, c);
      else c.ends = s.ends;
      order(s, b0, c);
      if (b0 == 0) first_ = s;
      units += sum(s.mine);
    }
    total = units * p_.Hk;
    part = max((total + k_.blocks - 1) / k_.blocks, k_.least);
  }
  // Few tiles: where each can be cut into equal pieces, one a block, that are hardly
  // longer than equal parts of the line, no block takes the time of two pieces'
  // starts and ends.  A tile's units are then those pieces.  Tiles of one sequence that
  // are cut alike also read the same keys at the same time, from L2, which is worth
  // half a part in bf16 (160 rows over 120000 keys, 8 heads of 128: 401 us by the
  // line, 233 alike); fp32 is bound by its products (701 tokens of three sequences,
  // 16 heads of 64: 65 us by the line, 68 alike).
  __device__ __forceinline__ bool alone(int tiles) {
    const int most = first_.a + slope_ * max(first_.tiles - 1, 0), n = tiles * p_.Hk;
    const int line = sum(upto(first_.a, first_.tiles, first_.tiles)) * p_.Hk;
    const int even = max((line + k_.blocks - 1) / k_.blocks, k_.least);
    const int slack = k_.alike && tiles > __builtin_popcountll(__ballot(first_.tiles > 0)) ? max(even / 2, k_.start) : k_.start;
    int best = 0;
    for (int i = 0; i < 8 && !best; ++i) {
      const int length = max((int)((float)line / (float)(k_.blocks - n * i / 8)) + 1, k_.least);
      if (length > even + slack) break;
      if (sum(first_.tiles * ((most + length - 1) / length)) * p_.Hk <= k_.blocks) best = length;
    }
    if (!best) return false;
    first_.a = (most + best - 1) / best;
    slope_ = 0;
    from_ = whole = 0;
    Carry c = {};
    order(first_, 0, c);
    total = sum(first_.mine) * p_.Hk;
    part = 1;
    return true;
  }
  // Tile `id` of those that are blocks of their own.
  __device__ __forceinline__ void tile(int id, Place& w) const {
    const int q = id / p_.Hk;
    w.hk = id - q * p_.Hk;
    w.u = 0;
    Carry c = {};
    for (int b0 = 0; b0 < p_.B; b0 += 64) {
      const Some s = batch(b0, c);
      const uint64_t hit = __ballot(q >= s.before && q < s.before + s.tiles);
      if (hit) return take(s, b0, __builtin_ctzll(hit), q, w);
    }
  }
  // The place `at` of the line; false: it ends before.
  __device__ __forceinline__ bool find(int at, Place& w) const {
    if (at >= total) return false;
    Carry c = {};
    for (int b0 = 0; b0 < p_.B; b0 += 64) {
      const Some s = batch(b0, c);
      const int begin = s.units_before * p_.Hk;
      const uint64_t hit = __ballot(at >= begin && at < begin + s.mine * p_.Hk);
      if (hit) {
        const int i = __builtin_ctzll(hit);
        const int before = __builtin_amdgcn_readlane(s.before, i), tiles = __builtin_amdgcn_readlane(s.tiles, i);
        const int a = __builtin_amdgcn_readlane(s.a, i), z0 = max(from_ - before, 0), base = upto(a, tiles, z0);
        int rest = at - __builtin_amdgcn_readlane(begin, i);
        // MANY: tile by tile, each for all heads; else head by head, each with all its
        // tiles, whose keys then stay in an XCD's L2.
        const int each = MANY ? p_.Hk : 1;
        if constexpr (!MANY) {
          const int mine = __builtin_amdgcn_readlane(s.mine, i);
          w.hk = rest / mine;
          rest -= w.hk * mine;
        }
        int lo = z0, hi = tiles - 1;  // the last tile (in order) that begins at or before `rest`
        while (lo < hi) {
          const int mid = (lo + hi + 1) / 2;
          if ((upto(a, tiles, mid) - base) * each <= rest) lo = mid;
          else hi = mid - 1;
        }
        take(s, b0, i, before + lo, w);
        w.u = rest - (upto(a, tiles, lo) - base) * each;
        if constexpr (MANY) {
          w.hk = w.u / w.units;
          w.u -= w.hk * w.units;
        }
        return true;
      }
    }
    return false;
  }
  // A cut that falls `u` units into a tile lies at the tile's start or end instead
  // where that is near.
  __device__ __forceinline__ int cut(int u, int units) const { return u < part / 8 ? 0 : units - u < part / 8 ? units : u; }

  int whole;        // tiles that are blocks of their own
  int total, part;  // units of the line, and of a block

 private:
  struct Some {  // 64 sequences, one a lane
    int start, n, len, tiles, ends;
    int a;                           // tile i (of rows i k.rows ..) has a + k.slope i units
    int before, units_before, mine;  // in order: tiles before its own, units of the line before its own, its own
  };
  struct Carry {
    int ends, tiles, units;
  };
  __device__ __forceinline__ static int sum(int v) { return __builtin_amdgcn_readlane(sums_upto(v), 63); }
  // Units of the first m tiles of a sequence, the last rows' first.
  __device__ __forceinline__ int upto(int a, int tiles, int m) const {
    const uint32_t n = m;  // (where the slope is 0 the other factor may be anything)
    return (int)(n * a + (uint32_t)slope_ * (n * (uint32_t)(tiles - 1) - n * (n - 1) / 2));
  }
  // Bounds that leave the rows or run backwards are cut, so that no row is of two
  // sequences; lengths beyond the table too.  c.ends: rows up to there are taken.
  __device__ __forceinline__ Some some(int b0, Carry& c) const {
    Some s = {};
    const int b = b0 + lane_;
    int from = 0, to = 0;
    if (b < p_.B) {
      from = min(max(p_.cu[b], 0), p_.T);
      to = min(max(p_.cu[b + 1], 0), p_.T);
      s.len = (int)min((int64_t)max(p_.lengths[b], 0), (int64_t)p_.width * p_.page);
    }
    const int upto = max(most_upto(to), c.ends);
    const int before = __builtin_amdgcn_update_dpp(0, upto, 0x138, 0xf, 0xf, false);  // the lane before's
    s.start = max(from, lane_ == 0 ? c.ends : before);
    s.n = max(to - s.start, 0);
    c.ends = s.ends = __builtin_amdgcn_readlane(upto, 63);
    return tiles_of(s);
  }
  __device__ __forceinline__ Some tiles_of(Some s) const {
    const int rows = s.n * (p_.Hq / p_.Hk);
    s.tiles = rows >= k_.from && rows <= k_.upto ? (rows + k_.rows - 1) >> k_.rows_log : 0;
    s.a = (max(s.len - s.n, 0) >> k_.unit_log) + k_.slope + k_.start;
    return s;
  }
  // The order of tiles: by index, or (MANY) by the sequences' lengths, the longest first,
  // among 64.
  __device__ __forceinline__ void order(Some& s, int b0, Carry& c) const {
    if constexpr (MANY) {
      s.before = c.tiles + sum_before(s, s.tiles);
    } else {
      s.before = c.tiles + sums_upto(s.tiles) - s.tiles;
    }
    const int z0 = min(max(from_ - s.before, 0), s.tiles);
    s.mine = upto(s.a, s.tiles, s.tiles) - upto(s.a, s.tiles, z0);
    if constexpr (MANY) {
      s.units_before = c.units + sum_before(s, s.mine);
    } else {
      s.units_before = c.units + sums_upto(s.mine) - s.mine;
    }
    c.tiles += sum(s.tiles);
    c.units += sum(s.mine);
  }
  // The sum of v over the sequences longer than a lane's (of the same length, of a
  // lower number), of those that have tiles.
  __device__ __forceinline__ int sum_before(const Some& s, int v) const {
    int total = 0;
    for (uint64_t left = __ballot(s.tiles > 0); left; left &= left - 1) {
      const int j = __builtin_ctzll(left), len = __builtin_amdgcn_readlane(s.len, j), x = __builtin_amdgcn_readlane(v, j);
      total += len > s.len || (len == s.len && j < lane_) ? x : 0;
    }
    return total;
  }
  __device__ __forceinline__ Some batch(int b0, Carry& c) const {
    if (b0 == 0) {
      if (p_.B > 64) c = {first_.ends, sum(first_.tiles), sum(first_.mine)};
      return first_;
    }
    Some s = some(b0, c);
    order(s, b0, c);
    return s;
  }
  __device__ __forceinline__ void take(const Some& s, int b0, int i, int q, Place& w) const {
    w.b = b0 + i;
    w.start = __builtin_amdgcn_readlane(s.start, i);
    w.n = __builtin_amdgcn_readlane(s.n, i);
    w.len = __builtin_amdgcn_readlane(s.len, i);
    w.tile = __builtin_amdgcn_readlane(s.tiles, i) - 1 - (q - __builtin_amdgcn_readlane(s.before, i));
    w.units = __builtin_amdgcn_readlane(s.a, i) + slope_ * w.tile;
  }

  const ChunkParams& p_;
  const ChunkClass& k_;
  const int lane_;
  Some first_;
  int from_, slope_;  // from_: tiles (in order, without their heads) before those of the line
};

// What chunk_join_kernel reads of a tile that begins in a block and goes on in others:
// its pieces (0: there is none) and where its rows go.
struct JoinNote {
  int pieces, row0, rows, start, hk, pad[3];
};
__device__ __forceinline__ JoinNote* note_of(const ChunkParams& p, const ChunkClass& k, int block) {
  return reinterpret_cast<JoinNote*>(p.part + k.notes_at) + block;
}

// What a block does of a tile: units from .. upto of it, keys kbeg .. kend.
struct Piece {
  int from, upto, kbeg, kend;
  bool whole;
};
// The keys of a tile, up to its last row's own, shared out over its units by steps
// (of k.step keys, which a block takes at once).
__device__ __forceinline__ int keys_upto(const ChunkClass& k, const Place& w, int keys, int u) {
  if (u == w.units) return keys;
  const int steps = (keys + k.step - 1) / k.step;
  return min(min((int)((float)u * ((float)steps / (float)w.units)), steps) * k.step, keys);
}
__device__ __forceinline__ void keys_of(const ChunkParams& p, const ChunkClass& k, const Place& w, Piece& piece) {
  const int last = min(w.n - 1, (w.tile * k.rows + k.rows - 1) / (p.Hq / p.Hk));
  const int keys = max(w.len - w.n + last + 1, 0);
  piece.whole = piece.from == 0 && piece.upto == w.units;
  piece.kbeg = piece.from ? keys_upto(k, w, keys, piece.from) : 0;
  piece.kend = keys_upto(k, w, keys, piece.upto);
}
// A block's way along the line: where it is (-1 before its first piece), where its
// part ends, and which part that is.
struct Walk {
  int at = -1, end = 0, block = 0;
};
// The block's next piece.  (The line is computed again for each: kept, it takes
// registers that the products need.)
template <bool MANY>
__device__ __forceinline__ bool next_piece(const ChunkParams& p, const ChunkClass& k, int lane, SVDMLP_ATTN_LDS Kept* kept, Walk& walk, Place& w, Piece& piece) {
  const bool first_piece = walk.at < 0;
  if (!first_piece && walk.at >= walk.end) return false;
  const Line<MANY> line(p, k, lane, kept, first_piece);
  if (MANY && (int)blockIdx.x < line.whole) {
    walk.at = walk.end;
    line.tile(blockIdx.x, w);
    piece.from = 0, piece.upto = w.units;
    keys_of(p, k, w, piece);
    return true;
  }
  if (first_piece) {
    // Parts that lie side by side go to one XCD.
    walk.block = blockIdx.x - line.whole;
    if (walk.block >= k.blocks) return false;
    if constexpr (!MANY) walk.block = xcd_remap(walk.block, k.blocks);
    const int64_t begin = (int64_t)walk.block * line.part;
    walk.end = (int)min((int64_t)line.total, begin + line.part);
    walk.at = (int)min(begin, (int64_t)line.total);
    if (threadIdx.x == 0 && k.blocks > 1) note_of(p, k, walk.block)->pieces = 0;
  }
  const int block = walk.block, end = walk.end;
  int& at = walk.at;
  bool first = first_piece;
  while (at < end && line.find(at, w)) {
    const int tile_at = at - w.u;
    piece.from = first ? line.cut(w.u, w.units) : 0;
    first = false;
    piece.upto = tile_at + w.units > end ? line.cut(end - tile_at, w.units) : w.units;
    at = tile_at + w.units;
    if (piece.from >= piece.upto) continue;  // its neighbour takes it
    keys_of(p, k, w, piece);
    if (piece.from == 0 && piece.upto < w.units && threadIdx.x == 0) {
      // The last block with a piece of it.
      int last = (tile_at + w.units - 1) / line.part;
      if (last > block + 1 && line.cut((int)((int64_t)last * line.part - tile_at), w.units) == w.units) --last;
      *note_of(p, k, block) = {last - block + 1, w.tile * k.rows, w.n * (p.Hq / p.Hk), w.start, w.hk, {}};
    }
    return true;
  }
  return false;
}

// A block's sums of its first and of its last piece, where those are no whole
// tiles: [D / 4][rows][4] floats, then [rows][2], the maximum and the sum of the
// weights.
__device__ __forceinline__ float* sums_of(const ChunkParams& p, const ChunkClass& k, int block, bool starts) {
  return p.part + k.part_at + ((int64_t)block * 2 + (starts ? 1 : 0)) * k.rows * (p.D + 2);
}

// x / page, of x below 2^31, where a page holds several tokens; and of any page.
__device__ __forceinline__ int page_of_many(const ChunkParams& p, int x) { return (int)(__umulhi((uint32_t)x, p.page_mul) >> p.page_shift); }
__device__ __forceinline__ int page_of(const ChunkParams& p, int x) { return p.page == 1 ? x : page_of_many(p, x); }

// The kernel's arguments (the first one), read again: what only a tile's end needs
// takes no registers before.
__device__ __forceinline__ const ChunkParams& args_again() {
  typedef const ChunkParams __attribute__((address_space(4))) * Args;
  Args a = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *(const ChunkParams*)a;
}

}  // namespace

}  // namespace svdmlp
