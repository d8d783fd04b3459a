// Rows of a paged cache moved within it, in every layer's caches by one launch:
//   copy_pages    the first rows of a page to another page (forks, compaction)
//   keep_drafts   the accepted ones of a sequence's drafts to behind its context
// Both only move bytes: bound by HBM, each read and written once, and by a
// launch where they are few.  500 pages of 16 tokens, 8 heads of 128, in the 64
// caches of 32 layers: 424 us, 5.0 TB/s; 8 partly filled ones 6.1 us.  Drafts of 16
// sequences (8 each, 32 layers) 5.8 us, of 128 sequences (64 each) 25, 4.3 TB/s.
#include <algorithm>

#include "common.hpp"
#include "decoder.hpp"

namespace svdmlp {

namespace {

template <int UNIT>
struct UnitOf;
template <>
struct UnitOf<16> {
  typedef u32x4 type;
};
template <>
struct UnitOf<4> {
  typedef uint32_t type;
};
template <>
struct UnitOf<2> {
  typedef uint16_t type;
};

constexpr int kPer = 4;  // units a thread of copy_pages has on its way

// Units of UNIT bytes; FLAT: a page's rows lie one behind the other.  A block
// takes 256 kPer units of one page of one cache.
template <int UNIT, bool FLAT>
__global__ __launch_bounds__(256) void page_copy_kernel(PageCopyParams p) {
  using U = typename UnitOf<UNIT>::type;
  int64_t id = blockIdx.x;
  const int part = (int)(id % p.parts);
  id /= p.parts;
  const int cache = (int)(id % p.c.n);
  const int64_t i = p.first + id / p.c.n;
  const int64_t src = p.src[i], dst = p.dst[i];
  if (src < 0 || dst < 0 || src >= p.c.pages || dst >= p.c.pages || src == dst) return;
  const int units = p.row_units * (p.rows ? min(max(p.rows[i], 0), p.c.page) : p.c.page);  // (under 2^30: checked by the caller)
  char* const base = static_cast<char*>(p.c.base[cache]);
  const U* const from = reinterpret_cast<const U*>(base + src * p.c.p_s * p.c.es);
  U* const to = reinterpret_cast<U*>(base + dst * p.c.p_s * p.c.es);
  auto place = [&](int u) -> int64_t {
    if constexpr (FLAT) return u;
    const int row = u / p.row_units, rest = u - row * p.row_units;
    const int head = rest / p.head_units, piece = rest - head * p.head_units;
    return (row * p.c.t_s + head * p.c.h_s) * p.c.es / UNIT + piece;
  };
  const int u0 = part * 256 * kPer + threadIdx.x;
  U v[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k)
    if (u0 + 256 * k < units) v[k] = from[place(u0 + 256 * k)];
#pragma unroll
  for (int k = 0; k < kPer; ++k)
    if (u0 + 256 * k < units) to[place(u0 + 256 * k)] = v[k];
}

// A thread takes one unit of a row of one cache, and moves it for every accepted
// draft in order.  Those are increasing numbers, so row i comes from a row that is
// not before it, and no row is written before it has been read.
constexpr int kRows = 8;  // on their way at once

template <int UNIT>
__global__ __launch_bounds__(256) void draft_keep_kernel(DraftKeepParams p) {
  using U = typename UnitOf<UNIT>::type;
  __shared__ int64_t from[kDraftsMost], to[kDraftsMost];
  __shared__ int count;
  const int64_t id = blockIdx.x;
  const int part = (int)(id % p.parts), b = (int)(id / p.parts);
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const int64_t room = (int64_t)p.width * p.c.page;
    const int len = (int)min((int64_t)max(p.lengths[b], 0), room), context = len - p.drafts;
    const int at = lane < p.m ? p.path[(int64_t)b * p.m + lane] : -1;
    int before = __shfl_up(at, 1);
    if (lane == 0) before = -1;
    const bool good = context >= 0 && lane < p.m && at > before && at < p.drafts;
    const uint64_t bad = ~__ballot(good);
    const int kept = bad ? __builtin_ctzll(bad) : 64;
    auto place = [&](int x) -> int64_t {  // of token x, in elements; -1: in no page of the cache
      const int pg = p.table[(int64_t)b * p.table_b + x / p.c.page];
      return pg >= 0 && pg < p.c.pages ? pg * p.c.p_s + (x % p.c.page) * p.c.t_s : -1;
    };
    if (lane < kept) {
      from[lane] = place(context + at);
      to[lane] = place(context + lane);
    }
    if (lane == 0) {
      count = kept;
      if (part == 0) p.new_lengths[b] = context >= 0 ? context + kept : len;
    }
  }
  __syncthreads();
  const int64_t u = (int64_t)part * 256 + threadIdx.x;
  if (u >= (int64_t)p.c.n * p.row_units) return;
  const int cache = (int)(u / p.row_units), rest = (int)(u - (int64_t)cache * p.row_units);
  const int head = rest / p.head_units, piece = rest - head * p.head_units;
  char* const base = static_cast<char*>(p.c.base[cache]) + (int64_t)head * p.c.h_s * p.c.es + (int64_t)piece * UNIT;
  for (int i0 = 0; i0 < count; i0 += kRows) {
    U v[kRows];
    bool move[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int i = min(i0 + k, count - 1);
      move[k] = i0 + k < count && from[i] >= 0 && to[i] >= 0 && from[i] != to[i];
      if (move[k]) v[k] = *reinterpret_cast<const U*>(base + from[i] * p.c.es);
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k)
      if (move[k]) *reinterpret_cast<U*>(base + to[min(i0 + k, count - 1)] * p.c.es) = v[k];
  }
}

// Bytes of a unit: 16 where every address is whole pieces, else an element.
int unit_of(const CacheSet& c, bool vec) { return vec ? 16 : c.es; }

template <int UNIT>
hipError_t copy(PageCopyParams p, int64_t m, hipStream_t st) {
  const CacheSet& c = p.c;
  p.head_units = c.D * c.es / UNIT, p.row_units = c.Hk * p.head_units;
  const bool flat = (c.Hk == 1 || c.h_s == c.D) && (c.page == 1 || c.t_s == (int64_t)c.Hk * c.D);
  const int64_t parts = ((int64_t)p.row_units * c.page + 256 * kPer - 1) / (256 * kPer);
  if (!fits_launch(parts * c.n, 256)) return hipErrorInvalidValue;
  p.parts = (int)parts;
  const int64_t most = (((int64_t)1 << 32) - 1) / 256 / (parts * c.n);  // pages a launch
  for (p.first = 0; p.first < m; p.first += most) {
    const int64_t blocks = std::min(most, m - p.first) * parts * c.n;
    if (flat) hipLaunchKernelGGL((page_copy_kernel<UNIT, true>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((page_copy_kernel<UNIT, false>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int UNIT>
hipError_t keep(DraftKeepParams p, hipStream_t st) {
  p.head_units = p.c.D * p.c.es / UNIT, p.row_units = p.c.Hk * p.head_units;
  const int64_t parts = ((int64_t)p.c.n * p.row_units + 255) / 256;
  if (!fits_launch(parts * p.B, 256)) return hipErrorInvalidValue;
  p.parts = (int)parts;
  hipLaunchKernelGGL((draft_keep_kernel<UNIT>), dim3((unsigned)(parts * p.B)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_copy_pages(const PageCopyParams& p, int64_t m, bool vec, hipStream_t st) {
  if (m <= 0) return hipSuccess;
  const int unit = unit_of(p.c, vec);
  return unit == 16 ? copy<16>(p, m, st) : unit == 4 ? copy<4>(p, m, st) : copy<2>(p, m, st);
}

hipError_t launch_keep_drafts(const DraftKeepParams& p, bool vec, hipStream_t st) {
  if (p.B <= 0) return hipSuccess;
  const int unit = unit_of(p.c, vec);
  return unit == 16 ? keep<16>(p, st) : unit == 4 ? keep<4>(p, st) : keep<2>(p, st);
}

}  // namespace svdmlp
