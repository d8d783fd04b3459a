// Attention of packed chunks of new tokens onto a paged cache that holds each
// sequence's context and them: new token i of sequence b's n is token
// lengths[b] - n + i of it and sees the keys up to itself.  A sequence may have
// one new token (it generates) or thousands (a chunk of its prompt), all in one
// call.
//
// A row is a new token and one of the heads that share a key/value head.  Three
// kernels share a call's sequences by their rows a key/value head, which only the
// device knows: chunk_wave_kernel takes tiles of 32 rows (chunk_wave.hip), those of
// sequences that generate; chunk_share_kernel of 128 (chunk_share.hip);
// chunk_pipe_kernel of 256 (bf16, heads up to 128).
//
// The work of a class of sequences is a line: for every row tile and key/value head
// as many units as the tile has keys, about.  It is cut into equal parts, one a
// block, whatever the lengths are: a block takes the end of a tile, some whole
// ones, the start of another.  chunk_join_kernel adds the sums of the tiles that
// lie in several parts, of which there are fewer than blocks, always in their
// order.  Where tiles of 128 or 256 rows are many, the first ones are blocks of
// their own, the longest first, and only the last one or two a CU are such a line:
// blocks that start together on tiles of one head read the same keys at the same
// time, from one XCD's L2.
//
// What bounds them: tiles of 32 rows the cache's bytes (96 sequences of 4000 tokens
// that generate, heads of 128: 300 us, 5.2 TB/s, a copy's rate) and, in fp32, the
// matrix unit (73% busy); tiles of 256 rows the matrix unit and the softmax beside
// it in the one wave a SIMD (8192 tokens of four sequences onto 16384, 64 heads of
// 128: 1.64 ms, 1.08 PFLOP/s of a product's 1.25; 512 onto 32768: 265 us, 1.03).  A
// server's step, 63 sequences of up to 4096 that generate and a chunk of 449, 187 us:
// 117 for the generating ones (4.5 TB/s), 53 for the chunk (five pieces of a tile, 15
// of the 53 for their starts and ends), some 20 to add them (34 MB of sums of pieces
// at 2.5 TB/s, whatever the registers, and so waves, of the join).  Few tokens: latency, a chain of
// loads (bounds, pages, keys), the join a launch of its own: 37 tokens 16 us.
//
// bf16: the weights are rounded to bf16 for the second product and summed after it
// (attn.hpp: why), so that results are off by 0.0020-0.0024 rms of the definition in 64 bits, of
// which their own rounding is 0.0017; a second part of each weight would halve the rate of that
// product.  fp32: 3e-7.
#include "chunk.hpp"
#include "pipe_attention.hpp"

namespace svdmlp {

namespace {

// ---------------------------------------------------------------------------
// 256 rows a tile
// ---------------------------------------------------------------------------

constexpr int kIds = 4096;  // pages whose numbers lie in LDS

// FULL: heads that fill their place.  Keys and values are laid out alike, and a
// page holds whole loads (C::RPL rows).
template <class C, bool FULL>
__global__ __launch_bounds__(256, 1) void chunk_pipe_kernel(ChunkParams p, ChunkClass k) {
  constexpr int RB = C::RB, QG = C::QG, KB = C::KB, DB = C::DB;
  __shared__ __attribute__((aligned(1024))) char lds[C::NS * C::STAGE];
  __shared__ int ids[kIds];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const attn_lds base = (attn_lds)lds;
  if constexpr (!FULL)  // zeros where a head is shorter than its place (never loaded)
    for (int i = threadIdx.x; i < C::NS * C::STAGE / 16; i += 256) *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(base + 16 * i) = u32x4{0u, 0u, 0u, 0u};

  __shared__ Kept kept;
  for (Walk walk;;) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // what follows from it is not kept over the pieces
    const int col = lane & 31, half = lane >> 5;
    Place w;
    Piece part;
    if (!next_piece<true>(p, k, lane, (SVDMLP_ATTN_LDS Kept*)&kept, walk, w, part)) return;
    const int G = p.Hq / p.Hk, npieces = p.D / 8, row0 = w.tile * C::BM, rows = w.n * G, context = w.len - w.n;
    const int all = part.kend - part.kbeg;  // keys of this piece, its first number 0 from here on
    const int token0 = context - part.kbeg;  // the first new token's key
    const int whole = max(min(token0 + row0 / G + 1, all), 0) / KB;  // tiles that every row sees

    const char* const kb = static_cast<const char*>(p.kc) + (int64_t)w.hk * p.k_h * 2;
    const char* const vb = static_cast<const char*>(p.vc) + (int64_t)w.hk * p.v_h * 2;
    const int* const table = p.table + (int64_t)w.b * p.table_b;
    const uint32_t cache_pages = (uint32_t)min(p.pages, (int64_t)0x7fffffff);
    auto valid = [&](int pg) { return (uint32_t)pg < cache_pages; };
    // This wave's loads of a tile: rows wave * LOADS * RPL .. of its keys and values.
    const int lrow = wave * C::LOADS * C::RPL + lane / C::PIECES, lc = lane % C::PIECES;
    uint32_t koff[C::LOADS], voff;  // a lane's place in a load: its row of RPL, its piece
    const int vc = lc ^ v_swz<RB, true>(lrow);
#pragma unroll
    for (int j = 0; j < C::LOADS; ++j) koff[j] = (uint32_t)(lane / C::PIECES * (int)p.k_t * 2 + 16 * (lc ^ k_swz<RB>(lrow + j * C::RPL)));
    voff = (uint32_t)(lane / C::PIECES * (int)p.k_t * 2 + 16 * vc);
    // (page strides and pages are below 2^32 bytes)
    const uint32_t page_step = (uint32_t)(p.k_p * 2), row_step = (uint32_t)(p.k_t * 2);
    u32x4 qf[QG][C::STEPS];
    PipeWave<C> pw(qf, lane, p.c);
    int tok[QG];  // a row's token
#pragma unroll
    for (int g = 0; g < QG; ++g) tok[g] = min(row0 + (wave * QG + g) * 32 + col, rows - 1) / G;  // rows behind the last repeat it, and are not stored

    // Segments of as many keys as have their pages' numbers in LDS.
    const int most = segment_keys(kIds, p.page, KB) / KB;  // tiles of a segment
    for (int t0 = 0; t0 * KB < all; t0 += most) {
      const int kbeg = part.kbeg + t0 * KB, nkeys = (int)min((int64_t)(all - t0 * KB), (int64_t)most * KB), tiles = (nkeys + KB - 1) / KB;
      const int first = token0 - t0 * KB;
      __syncthreads();  // (with what the last segment left in LDS)
      // The pages' numbers, and whether all are pages of the cache.  One that is not
      // holds no keys: page 0 is read for it, and masked.
      const int pg0 = page_of_many(p, kbeg), pages = page_of_many(p, kbeg + nkeys - 1) - pg0 + 1;
      bool lost = false;
      for (int i0 = threadIdx.x; i0 < pages; i0 += 256 * 8) {
        int v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = table[pg0 + min(i0 + 256 * j, pages - 1)];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          lost |= !valid(v[j]);
          if (i0 + 256 * j < pages) ids[i0 + 256 * j] = valid(v[j]) ? v[j] : 0;
        }
      }
      // Zeros in the last stage's values, which the first step multiplies by zero weights.
      for (int i = threadIdx.x; i < C::UNIT / 16; i += 256)
        *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(base + (C::NS - 1) * C::STAGE + C::TILE + C::UNIT + 16 * i) = u32x4{0u, 0u, 0u, 0u};
      const bool holes = __syncthreads_or(lost);
      // (The queries again for every segment: kept, they would be moved for every product.)
#pragma unroll
      for (int g = 0; g < QG; ++g) {
        const int r = min(row0 + (wave * QG + g) * 32 + col, rows - 1);
        const char* qp = static_cast<const char*>(p.q) + ((int64_t)(w.start + tok[g]) * p.q_t + (int64_t)(w.hk * G + r - tok[g] * G) * p.q_h) * 2;
#pragma unroll
        for (int s = 0; s < C::STEPS; ++s) {
          const int c = 2 * s + half;
          qf[g][s] = FULL || c < npieces ? *reinterpret_cast<const u32x4*>(qp + 16 * c) : u32x4{0u, 0u, 0u, 0u};
        }
      }
      const int full = holes ? 0 : min(max(whole - t0, 0), nkeys / KB);

      // Lane j's place of load j of a tile of keys, in bytes (behind the last key: rows
      // of its load's page).  Kept for the tile behind the last one asked for.
      const int mine = (wave * C::LOADS + lane % C::LOADS) * C::RPL, end = (nkeys - 1) / C::RPL * C::RPL;
      int key, pg, id;
      auto look = [&](int t) {
        key = kbeg + min(t * KB + mine, end);
        pg = page_of_many(p, key);
        id = ids[pg - pg0];
      };
      auto place = [&]() -> int64_t { return (int64_t)((uint64_t)(uint32_t)id * page_step + (uint32_t)(key - pg * p.page) * row_step); };
      auto places = [&](int t) {
        look(t);
        return place();
      };
      auto issue_keys = [&](int t, int64_t where) {
        const uint32_t to = (uint32_t)(uintptr_t)(base + (t % C::NS) * C::STAGE) + wave * C::LOADS * 1024;
#pragma unroll
        for (int j = 0; j < C::LOADS; ++j) {
          const int64_t a = lane_of(where, j);
          if (FULL || (lc ^ k_swz<RB>(lrow + j * C::RPL)) < npieces) load_lds16(kb + a, koff[j], to + j * 1024);
        }
      };
      auto issue_values = [&](int t, int64_t where) {
        const uint32_t to = (uint32_t)(uintptr_t)(base + (t % C::NS) * C::STAGE) + C::TILE + wave * C::LOADS * 1024;
#pragma unroll
        for (int j = 0; j < C::LOADS; ++j) {
          const int64_t a = lane_of(where, j);
          if (FULL || vc < npieces) load_lds16(vb + a, voff, to + j * 1024);
        }
      };
      const int64_t at0 = places(0), at1 = places(1);
      int64_t ahead = places(2), next = places(3);  // of the last tile of keys asked for, and of the one behind it
      issue_keys(0, at0);
      if (tiles > 1) issue_keys(1, at1);
      issue_values(0, at0);
      if (tiles > 2) issue_keys(2, ahead);
      if (tiles > 1) issue_values(1, at1);
      // Before tile t: the keys of tile t + 1 and the values of tile t are there for
      // every wave (they were asked for two tiles ago; what was asked for one tile
      // ago may still be on its way), and every wave is done with the keys of tile
      // t - 1 and the values of tile t - 2, whose places are filled again.
      auto arrive = [&](int t) {
        if (t + 2 < tiles) wait_loads<2 * C::LOADS>();
        else wait_loads<0>();
        asm volatile("s_barrier" ::: "memory");
        if (t + 3 < tiles) issue_keys(t + 3, next);
        if (t + 2 < tiles) issue_values(t + 2, ahead);
        ahead = next;
      };
      // The places of tile t + 4's keys, looked up beside tile t's products.
      int t = 0;
      auto beside = [&](int n) {
        if (n == 1) look(t + 4);
        if (n == 9) next = place();
      };

      // The queries in accumulation registers, from which products take them (the
      // compiler would move each there and back: 75 moves a step, a fifth of its time).
#pragma unroll
      for (int g = 0; g < QG; ++g)
#pragma unroll
        for (int s = 0; s < C::STEPS; ++s) asm volatile("" : "+a"(qf[g][s]));
      if (full > 0) pw.whole_tiles(base, full, t, t0 > 0, arrive, beside);
      for (; t < tiles; ++t) {
        arrive(t);
        next = places(t + 4);
        const attn_lds cur = base + (t % C::NS) * C::STAGE;
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
          const int k0 = t * KB + 32 * u;
          const int seen = min(first + (row0 + (wave + 1) * QG * 32 - 1) / G, nkeys - 1);  // the wave's last key
          if (k0 > seen) break;
          f32x16 s[QG];
          u32x4 pb[QG][2];
          float scale[QG];
          const attn_lds vt = cur + C::TILE + u * C::UNIT;
          uint32_t there = 0xffffffffu;
          if (holes) there = (uint32_t)__ballot(k0 + col < nkeys && valid(table[page_of_many(p, kbeg + min(k0 + col, nkeys - 1))]));
          there >>= 4 * half;
          pw.scores(cur + u * C::UNIT, vt, s);
#pragma unroll
          for (int g = 0; g < QG; ++g) {
            const int last = min(first + tok[g], nkeys - 1) - k0 - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int x = 8 * (i >> 2) + (i & 3);
              s[g][i] = x <= last && (there >> x & 1u) ? s[g][i] : -INFINITY;
            }
          }
          if (pw.reference(s, scale)) pw.rescale(scale);
          pw.weights(s, pb);
          pw.values(vt, pb, true);
        }
      }
    }

    const ChunkParams& e = args_again();
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      pw.l[g] += __shfl_xor(pw.l[g], 32);
      const float inv = part.whole ? inverse_sum(pw.l[g]) : 1.f;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) pw.o[g][d][i] *= inv;
    }
    // Infinities and NaN among the values of the plain loop were taken as
    // zeros, for the rows that do not see them; the rows that do get them here.
    // (Where a page is lost all tiles of its segment are in the plain loop; those
    // of others add to what they hold already.)
    if (__any(pw.bad != 0)) {
      for (int key = 0; key < all; ++key) {
        const int at = page_of_many(e, part.kbeg + key), pg = table[at];
        if (!valid(pg)) continue;
        const uint16_t* const vp = reinterpret_cast<const uint16_t*>(vb + ((int64_t)pg * e.v_p + (int64_t)(part.kbeg + key - at * e.page) * e.v_t) * 2);
        bool any = false;
        for (int x = lane; x < e.D; x += 64) any |= not_finite<false>((uint32_t)vp[x] << 16) != 0;
        if (!__any(any)) continue;
        uint32_t see[QG];
#pragma unroll
        for (int g = 0; g < QG; ++g) see[g] = key <= token0 + tok[g] ? 0xffffffffu : 0u;
        int D = e.D;
        asm volatile("" : "+s"(D));  // its comparisons stay in the loop: hoisted, they spill
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int x = 32 * d + 8 * (i >> 2) + 4 * half + (i & 3);
            const uint32_t v = x >= D ? 0u : (uint32_t)vp[x] << 16, mask = not_finite<false>(v);
#pragma unroll
            for (int g = 0; g < QG; ++g) pw.o[g][d][i] += __uint_as_float(v & mask & see[g]);
          }
      }
    }
    float* const sums = part.whole ? nullptr : sums_of(e, k, walk.block, part.from == 0);
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      const int rr = (wave * QG + g) * 32 + col, r = row0 + rr;
      if (r < rows) {
        const int64_t op = (int64_t)(w.start + tok[g]) * e.o_t + (int64_t)(w.hk * G + (r - tok[g] * G)) * e.o_h;
        if (sums && half == 0) reinterpret_cast<f32x2*>(sums + C::BM * e.D)[rr] = f32x2{pw.m[g], pw.l[g]};
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int x = 32 * d + 8 * b + 4 * half;
            if (!FULL && x >= e.D) continue;
            const f32x4 v = {pw.o[g][d][4 * b], pw.o[g][d][4 * b + 1], pw.o[g][d][4 * b + 2], pw.o[g][d][4 * b + 3]};
            if (sums) reinterpret_cast<f32x4*>(sums)[(x >> 2) * C::BM + rr] = v;
            else store4<true>(e.out, op + x, v);
          }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Tiles in several parts
// ---------------------------------------------------------------------------

// Joins the sums of the tile that begins in a block and goes on in those behind it.
// A block takes 32 rows of it, a thread every eighth 16 bytes (four elements) of one.
template <bool BF16>
__device__ __forceinline__ void join(const ChunkParams& p, const ChunkClass& k, int id) {
  const int G = p.Hq / p.Hk, block = id >> (k.rows_log - 5), group = id - (block << (k.rows_log - 5));
  const JoinNote w = *note_of(p, k, block);
  const int pieces = w.pieces;
  if (pieces == 0) return;
  const int rr = group * 32 + (threadIdx.x & 31), r = w.row0 + rr;
  if (r >= w.rows) return;
  const int64_t ml_at = (int64_t)k.rows * p.D + 2 * rr;
  // The block's second sums, then the others' first ones.
  auto sums = [&](int j) { return sums_of(p, k, block + min(j, pieces - 1), j == 0); };
  const int t = r / G;
  const int64_t out = (int64_t)(w.start + t) * p.o_t + (int64_t)(w.hk * G + r - t * G) * p.o_h;
  constexpr int kCols = 4, kPieces = 4;  // on their way at once
  for (int c0 = threadIdx.x / 32; 4 * c0 < p.D; c0 += 8 * kCols) {
    f32x4 o[kCols] = {};
    float m = -INFINITY, l = 0.f;
    for (int j0 = 0; j0 < pieces; j0 += kPieces) {
      f32x2 v[kPieces];
      f32x4 x[kPieces][kCols];
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const float* const from = sums(j0 + j);
        v[j] = *reinterpret_cast<const f32x2*>(from + ml_at);
#pragma unroll
        for (int q = 0; q < kCols; ++q) x[j][q] = reinterpret_cast<const f32x4*>(from)[min(c0 + 8 * q, p.D / 4 - 1) * k.rows + rr];
      }
      float most = m;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) most = fmaxf(most, v[j].x);
      const float a = m == most ? 1.f : exp2f(m - most);
      m = most;
      l *= a;
#pragma unroll
      for (int q = 0; q < kCols; ++q) o[q] *= a;
      // (a piece without a score over -infinity: its sums are zeros, or not finite and stay so)
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        if (j0 + j < pieces) {
          const float b = v[j].x == -INFINITY ? 1.f : exp2f(v[j].x - m);
          l += v[j].y * b;
#pragma unroll
          for (int q = 0; q < kCols; ++q) o[q] += x[j][q] * b;
        }
    }
    const float inv = inverse_sum(l);
#pragma unroll
    for (int q = 0; q < kCols; ++q)
      if (4 * (c0 + 8 * q) < p.D) store4<BF16>(p.out, out + 4 * (c0 + 8 * q), o[q] * inv);
  }
}
template <bool BF16>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkParams p, ChunkPlan plan) {
  const int id = blockIdx.x, some = id - plan.many.joins, few = some - plan.some.joins;
  if (some < 0) join<BF16>(p, plan.many, id);
  else if (few < 0) join<BF16>(p, plan.some, some);
  else join<BF16>(p, plan.few, few);
}

template <int DP>
void run_pipe(const ChunkParams& p, const ChunkClass& k, hipStream_t st) {
  const dim3 grid((unsigned)k.grid);
  if (p.D < DP) hipLaunchKernelGGL((chunk_pipe_kernel<PipeCfg<DP>, false>), grid, dim3(256), 0, st, p, k);
  else hipLaunchKernelGGL((chunk_pipe_kernel<PipeCfg<DP>, true>), grid, dim3(256), 0, st, p, k);
}

// Waves of a block of 32-row tiles: as many as have stages in half of a CU's LDS.
int wave_block(int64_t D, bool bf16) { return D * (bf16 ? 2 : 4) <= 256 ? 4 : 2; }

}  // namespace

ChunkPlan plan_chunk_attention(int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D, bool bf16, bool alike, int64_t page, int64_t capacity, int64_t cus) {
  ChunkPlan plan = {};
  const int64_t rows = T * (Hq / Hk);  // at most, a key/value head
  auto fill = [&](ChunkClass& k, int64_t from, int64_t upto, int tile_log, int step, int64_t blocks, int64_t least, int64_t start) {
    const int64_t tile = (int64_t)1 << tile_log, G = Hq / Hk;
    k.from = (int)std::min<int64_t>(from, 0x7fffffff), k.upto = (int)std::min<int64_t>(upto, 0x7fffffff);
    k.rows = (int)tile, k.rows_log = tile_log, k.step = step, k.alike = bf16;
    if (upto < from) return;
    // Sequences of the class, and their tiles: at most one short tile each.
    const int64_t n = std::min(B, rows / from);
    int64_t tiles = rows / tile + n;
    if (upto < rows) tiles = std::min(tiles, n * ((upto + tile - 1) / tile));
    // Units that the line has at most: a tile's context, its own tokens and those of
    // the tiles before it.
    int log = 0;
    auto units = [&] {
      const double of = (double)(capacity >> log) + (double)(start >> log) + 2 + (double)((tile / G) >> log) * (double)tiles;
      return of * (double)tiles * (double)Hk;
    };
    while (units() >= (double)(1 << 30) && log < 31) ++log;
    k.unit_log = log, k.slope = (int)((tile / G) >> log), k.start = (int)(start >> log) + 1;
    k.fits = units() < (double)(1 << 30) && tiles * Hk < (int64_t)1 << 23;
    k.least = (int)std::max<int64_t>(least >> log, 1);
    k.blocks = (int)std::max<int64_t>(std::min<int64_t>(blocks, (int64_t)std::min(units() / (double)k.least, 1e9) + 1), 1);
    // (blocks without work cost their share too: the tiles that have blocks of their own
    // are whole rounds, one less than all)
    k.grid = k.blocks + (tile_log > 5 ? (int)std::max<int64_t>(std::min<int64_t>(tiles * Hk, 1 << 23) / k.blocks - 1, 0) * k.blocks : 0);
    if (k.blocks == 1) return;
    k.joins = (k.blocks - 1) * (int)(tile / 32);  // (no tile begins in the last block and goes on)
    k.notes_at = plan.floats;
    k.part_at = plan.floats + (int64_t)k.blocks * (sizeof(JoinNote) / 4);
    plan.floats = k.part_at + (int64_t)k.blocks * 2 * tile * (D + 2);
  };
  const int wave = 32 * wave_block(D, bf16);
  const bool pipe = bf16 && D <= 128 && alike && page % (D <= 64 ? PipeCfg<64>::RPL : PipeCfg<128>::RPL) == 0;
  // The largest sequences of each class, in rows a key/value head (of 3000 keys each,
  // 32 over 8 heads of 128 unless said; us by tiles of 32, 128 and 256 rows).  Tiles
  // of 32 rows read the keys again for each, from L2 as long as a head's tiles run
  // together, which they do while all fit the card: 16 bf16 sequences of 64 rows 63,
  // 82, 92; 64 of 48 rows and 2000 keys 201, 160, 215; of 256 rows and 1000 keys 313,
  // 190, 182.  One sequence gains most from them: 120 rows of 4000 keys 27, 35, 37,
  // 512 rows 35, 47, 38.  fp32 is bound by its products: 8 of 128 rows 135, 168; 48
  // of 128 rows 835, 873, of 512 rows 3403, 2964.  Heads of 256 in bf16, 16 over 2:
  // 8 sequences of 64 rows 36, 43; 64 of 128 rows 194, 164; in fp32, where a CU
  // holds a single wave that shares nothing, one sequence of 8 rows 221, 115.
  // A class takes some 5 us where it has nothing to do: small calls have one, and most
  // two, where most sequences must be of few rows.
  const bool full = B * Hk > cus && rows > 32 * B;
  int64_t few = bf16 ? (D <= 128 && full ? 32 : 64) : D <= 128 ? rows : 0, some = !pipe ? rows : full ? 128 : few;
  if (bf16 && rows <= 256) few = rows;
  else if (bf16 && B == 1) few = 0, some = pipe ? 0 : rows;  // (whose rows are the call's)
  few = std::min(few, rows), some = std::max(few, std::min(some, rows));
  // Blocks that a CU holds at once, the keys a block takes at least, and those that a
  // tile's start and end take as long as.  Half as many blocks again, or twice as
  // many, that start as others end, lose to their starts: 64 sequences that generate
  // 149, 164, 159 us; 701 fp32 tokens 66, 83, 81 (3200: 421, 454, 395).  Starts of 128 or
  // 400 keys are within 2% of 256, but for fp32 (701 tokens 66, 71 by 128).
  fill(plan.many, some + 1, rows, 8, 64, cus, 512, 384);
  fill(plan.some, few + 1, some, 7, 32, cus * (D <= 128 ? 2 : 1), 256, 256);
  fill(plan.few, 1, few, 5, wave, cus * (!bf16 ? 2 : D <= 64 ? 3 : D <= 128 ? 2 : 1), 512, 256);
  return plan;
}

hipError_t launch_chunk_attention(const ChunkParams& p, bool bf16, const ChunkPlan& plan, hipStream_t st) {
  if (p.T <= 0 || p.B <= 0) return hipSuccess;
  for (const ChunkClass* k : {&plan.many, &plan.some, &plan.few})
    if (k->blocks && !k->fits) return hipErrorInvalidValue;
  if (plan.many.blocks) p.D <= 64 ? run_pipe<64>(p, plan.many, st) : run_pipe<128>(p, plan.many, st);
  if (plan.some.blocks) launch_chunk_shared(p, plan.some, bf16, st);
  if (plan.few.blocks) launch_chunk_waves(p, plan.few, bf16, st);
  if (const int joins = plan.many.joins + plan.some.joins + plan.few.joins) {
    if (bf16) hipLaunchKernelGGL((chunk_join_kernel<true>), dim3((unsigned)joins), dim3(256), 0, st, p, plan);
    else hipLaunchKernelGGL((chunk_join_kernel<false>), dim3((unsigned)joins), dim3(256), 0, st, p, plan);
  }
  return hipGetLastError();
}

}  // namespace svdmlp
