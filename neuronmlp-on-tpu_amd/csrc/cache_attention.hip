// Attention of the n new tokens of each sequence onto a paged cache that holds
// the sequence's context and them: token i sees every key of the context, and
// of the new ones those that its row of the tree names (no tree: the ones up to
// itself).  n = 1 is the decode step.
//
// Bound by the cache's bytes, read once for all heads of a group and all new
// tokens (up to 128 rows).  Up to 32 rows nothing is shared between waves: each
// takes tiles of 32 keys of its block's chunk through LDS of its own (direct
// loads), with no barrier in the loop.  Where there is work for every wave of the
// card, a block is one wave, and eight of them share a CU, one's start and end
// hidden behind the others' loads; where there is not, a block's four waves share
// a chunk, and their sums meet in LDS.  Up to 64 rows a wave takes both 32s of
// its tile.  Over 64, four waves load each tile together and take 32 rows each:
// a quarter of the loads, three tiles ahead of the one computed.
// A long context is cut into chunks, one a block; the last block of a (sequence,
// head, row tile) to arrive joins the chunks' partial sums, in the chunks' order
// (the same bits every time), or, over 64 rows, a kernel of its own.
// Heads of 128 in bf16, 8 of keys: one sequence of 4097 tokens 14.3 us (latency:
// a chunk of 256 keys, then the join); 64 sequences of up to 4096 120.8 us
// (4.3 TB/s of a copy's 5.2); 16 tokens' trees of 8 sequences of up to 16384, 128
// rows a head, 95.3 us (3.4 TB/s, the pace of 32-row tiles).
#include <algorithm>

#include "wave_attention.hpp"

namespace svdmlp {

namespace {

template <bool BF16, int DP, int QG, int NW, bool SHARE = false>
hipError_t run(const CacheParams& p, hipStream_t st) {
  // One tile in LDS a wave where its sums fit it: twice as many waves a CU, whose
  // loads and products overlap (64 sequences 127 -> 121 us; one sequence, whose
  // 264 blocks then run in one round, 18 -> 14).
  constexpr int RB = DP * (BF16 ? 2 : 4);
  using C = CacheCfg<BF16, DP, QG, NW, false, SHARE ? 65536 / (64 * RB) : QG == 1 && RB >= 256 ? 1 : 2, SHARE>;
  const int64_t rtiles = ((int64_t)p.n * (p.Hq / p.Hk) + C::ROWS - 1) / C::ROWS;
  const int64_t blocks = rtiles * p.Hk * p.chunks;
  const int64_t joins = ((int64_t)p.B * p.n * p.Hq + 3) / 4;
  const bool joined = SHARE && p.splits > 1;  // by a kernel of its own
  if (!fits_launch(blocks, 64 * NW) || (joined && !fits_launch(joins, 256))) return hipErrorInvalidValue;
  CacheParams q = p;
  q.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (p.page == 1 << s && p.page >= C::RPI) q.page_shift = s;
  hipLaunchKernelGGL((cache_kernel<C>), dim3((unsigned)blocks), dim3(64 * NW), 0, st, q);
  if (joined) hipLaunchKernelGGL((cache_join_kernel<BF16>), dim3((unsigned)joins), dim3(256), 0, st, p, (int)rtiles);
  return hipGetLastError();
}

// Rows a block, as far as their sums fit: 64 a wave where there are more than 32,
// and four waves of 32 that share a tile where there are more than 64 (8 sequences
// of up to 16384 tokens, 40, 64, 72 and 128 rows: 77.7, 87.6, 119.5 and 124.6 us
// by 64 a wave, 83.4, 86.1, 85.9 and 100.7 shared; of up to 8000 in fp32, 40, 64
// and 72 rows: 41.7, 48.8, 67.4 and 52.8, 54.7, 54.9).
int block_rows(int n, int Hq, int Hk, int D, bool bf16) {
  const int64_t rows = (int64_t)n * (Hq / Hk);
  return rows <= 32 || D > (bf16 ? 128 : 64) ? 32 : rows <= 64 ? 64 : 128;
}

}  // namespace

CachePlan plan_cache_attention(int B, int n, int Hq, int Hk, int D, bool bf16, int page, int64_t capacity, int cus) {
  CachePlan plan;
  const int64_t rows = (int64_t)n * (Hq / Hk), rt = block_rows(n, Hq, Hk, D, bf16);
  plan.rtiles = (int)((rows + rt - 1) / rt);
  const int64_t base = (int64_t)B * Hk * plan.rtiles;
  const int row = D * (bf16 ? 2 : 4), waves = row <= 256 ? 4 : row <= 512 ? 2 : 1;  // of a block that shares a chunk
  // One wave a block, of chunks of 256 keys, where those give every SIMD one.
  // Else, and where a wave has 64 rows (whose partial sums, written and read,
  // would be half of such a chunk's keys and values), blocks that share a
  // chunk, of chunks that give every CU one; or three, of different lengths, if
  // the chunks stay long.  Blocks that share their tiles: two a CU, which is what
  // fits (trees of 16 over up to 16384 tokens, one, two, three, four a CU: 131,
  // 95, 115, 109 us).
  constexpr int64_t kSolo = 256;
  plan.waves = rt == 32 && base * ((capacity + kSolo - 1) / kSolo) >= 4 * (int64_t)cus ? 1 : waves;
  int64_t c = kSolo;
  if (plan.waves > 1 || waves == 1) c = std::max(capacity * base / cus / 3, std::min<int64_t>(1024, capacity * base / cus));
  // Over four waves a SIMD, chunks of at least as many keys as keep all row tiles'
  // partial sums to a quarter of the keys and values (512 rows of heads of 256, 96
  // sequences of up to 21800 tokens: 2.89 GB of them and 3.21 ms by chunks of 384
  // keys, 0.56 GB and 2.10 ms by 2048; 128 rows, 32 of 16384: 454 and 344 us).
  else c = std::max(c, std::min(rows * (bf16 ? 4 : 2), capacity * base / (16 * cus)));
  // Of few sequences, whose lengths may be any part of the table's width, from
  // the lengths (shared_chunk), 512 at least; many even out by themselves (heads
  // of 128, 8 of keys, 16 new tokens; 4 sequences of up to 32768 tokens 75 us from
  // the lengths, 101 from the width; 8 of 16384 102 and 103, of 8192 48 and 58; 16
  // of 8192 135 and 116; 64 of 4000 242 and 198; 8 of 8192, 64 new tokens, 119 and 172).
  const bool choose = rt == 128 && B <= 64 && (B <= 8 || base * 4 <= cus);
  if (rt == 128) c = choose ? 512 : std::max<int64_t>(512, capacity * base / (2 * cus));
  c = std::max<int64_t>(c, (capacity + kSplitsMost - 1) / kSplitsMost);
  // (a single wave of rows of 1 KB: a tile, whose products take 7 us)
  const int64_t step = waves == 1 ? 32 : 128;
  c = std::max(step, (c + step - 1) / step * step);
  c = std::min(c, (int64_t)kPagesMost * page / 128 * 128);
  plan.chunk = (int)std::min<int64_t>(c, 0x7fffff80);
  plan.splits = (int)((capacity + plan.chunk - 1) / plan.chunk);
  plan.shared = rt == 128;
  plan.slots = 2 * cus;
  plan.chunk_most = plan.chunk;
  plan.chunks = B * plan.splits;
  if (choose && plan.splits > 1) {
    plan.chunk_most = (int)std::min((int64_t)kPagesMost * page, (int64_t)0x7fffff80);
    // at most total / chunk + B
    const int64_t most = std::max(plan.slots / ((int64_t)Hk * plan.rtiles), (B * capacity + plan.chunk_most - 1) / plan.chunk_most);
    plan.chunks = (int)std::min(B + most, (int64_t)plan.chunks);
  }
  return plan;
}

hipError_t launch_cache_attention(const CacheParams& p, bool bf16, const CachePlan& plan, hipStream_t st) {
  if (p.B <= 0 || p.n <= 0) return hipSuccess;
  const bool two = block_rows(p.n, p.Hq, p.Hk, p.D, bf16) == 64, one = plan.waves == 1;
  if (plan.shared) {
    if (!bf16) return run<false, 64, 1, 4, true>(p, st);
    return p.D <= 64 ? run<true, 64, 1, 4, true>(p, st) : run<true, 128, 1, 4, true>(p, st);
  }
  if (bf16) {
    if (p.D <= 64) return two ? run<true, 64, 2, 4>(p, st) : (one ? run<true, 64, 1, 1>(p, st) : run<true, 64, 1, 4>(p, st));
    if (p.D <= 128) return two ? run<true, 128, 2, 4>(p, st) : (one ? run<true, 128, 1, 1>(p, st) : run<true, 128, 1, 4>(p, st));
    return one ? run<true, 256, 1, 1>(p, st) : run<true, 256, 1, 2>(p, st);
  }
  if (p.D <= 64) return two ? run<false, 64, 2, 4>(p, st) : (one ? run<false, 64, 1, 1>(p, st) : run<false, 64, 1, 4>(p, st));
  if (p.D <= 128) return one ? run<false, 128, 1, 1>(p, st) : run<false, 128, 1, 2>(p, st);
  return run<false, 256, 1, 1>(p, st);
}

}  // namespace svdmlp
