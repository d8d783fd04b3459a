// Attention of packed chunks of new tokens onto a paged cache that holds each
// sequence's context and them: new token i of sequence b's n is token
// lengths[b] - n + i of it and sees the keys up to itself.  A sequence may have
// one new token (it generates) or thousands (a chunk of its prompt), all in one
// call.
//
// A row is a new token and one of the heads that share a key/value head.  Two
// kernels share a call's sequences by their rows a key/value head, which only the
// device knows: chunk_pipe_kernel takes 256 rows a block (bf16, heads up to 128,
// sequences of over kFewRows rows), chunk_wave_kernel 32.  Each cuts long
// contexts into chunks of keys, by the lengths, so that about p.slots blocks have
// as much to do; chunk_join_kernel adds what the chunks of a row tile found.
#include <math.h>

#include <algorithm>

#include "decoder.hpp"
#include "pipe_attention.hpp"

namespace svdmlp {

namespace {

constexpr int kSplitsMost = 64;  // chunks of a sequence

// What a block does: rows row0 .. of sequence b, keys kbeg .. kend of it.
struct Work {
  int b, hk, tile, start, n, len, split, chunks;
  int64_t part;  // of the sums of tiles in several chunks
};

struct Sequence {
  int start, n, len, tiles;
};
// Sequence b's rows of q, its tokens in the cache, and its row tiles of the class
// (0: of the other class, or no rows).  Bounds that leave the rows or run
// backwards, and lengths beyond the table, are cut.
__device__ __forceinline__ Sequence sequence_of(const ChunkParams& p, const ChunkClass& k, int b) {
  Sequence s = {0, 0, 0, 0};
  if (b >= p.B) return s;
  s.start = min(max(p.cu[b], 0), p.T);
  s.n = min(max(p.cu[b + 1], s.start), p.T) - s.start;
  s.len = (int)min((int64_t)max(p.lengths[b], 0), (int64_t)p.width * p.page);
  const int rows = s.n * (p.Hq / p.Hk);
  s.tiles = rows >= k.from && rows <= k.upto ? (rows + k.rows - 1) / k.rows : 0;
  return s;
}

__device__ __forceinline__ int64_t lanes_sum(int64_t v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ int64_t lanes_upto(int64_t v, int lane) {  // inclusive prefix sums
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t w = __shfl_up(v, o);
    if (lane >= o) v += w;
  }
  return v;
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int i) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, i) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32);
}

// Keys a chunk: as many chunks as there are slots, over all tiles of the class, at
// least k.least keys each and at most kSplitsMost of a sequence.
__device__ __forceinline__ int chunk_keys(const ChunkParams& p, const ChunkClass& k, const Sequence& first, int lane) {
  int64_t keys = 0;
  int longest = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const Sequence s = b0 ? sequence_of(p, k, b0 + lane) : first;
    keys += (int64_t)s.tiles * s.len;
    if (s.tiles) longest = max(longest, s.len);
  }
  keys = lanes_sum(keys);
  for (int o = 32; o > 0; o >>= 1) longest = max(longest, __shfl_xor(longest, o));
  const int64_t want = max((keys * p.Hk + k.slots - 1) / k.slots, (int64_t)(longest + kSplitsMost - 1) / kSplitsMost);
  const int64_t c = (max(want, (int64_t)k.least) + 63) / 64 * 64;
  return __builtin_amdgcn_readfirstlane((int)min(c, (int64_t)0x7fffffc0));
}
__device__ __forceinline__ int chunks_of(int len, int chunk) { return max(1, (int)(((int64_t)len + chunk - 1) / chunk)); }

// Item `id` of the class: of all (chunk, tile) pairs with JOIN false, of the tiles
// in several chunks with JOIN true, times key/value heads.  False: there is none.
template <bool JOIN>
__device__ __forceinline__ bool find_work(const ChunkParams& p, const ChunkClass& k, int64_t id, int lane, Work& w) {
  w.hk = (int)(id % p.Hk);
  id /= p.Hk;
  const Sequence first = sequence_of(p, k, lane);
  const int chunk = chunk_keys(p, k, first, lane);
  int64_t before = 0, parts = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const Sequence s = b0 ? sequence_of(p, k, b0 + lane) : first;
    const int chunks = chunks_of(s.len, chunk);
    const int64_t sums = chunks > 1 ? (int64_t)s.tiles * chunks : 0;
    const int64_t mine = JOIN ? (chunks > 1 ? s.tiles : 0) : (int64_t)s.tiles * chunks;
    const int64_t upto = lanes_upto(mine, lane), sums_upto = lanes_upto(sums, lane);
    const uint64_t hit = __ballot(id < before + upto);
    if (hit) {
      const int i = __builtin_ctzll(hit);
      const int rest = (int)(id - before - lane_of(upto - mine, i));
      w.b = b0 + i;
      w.chunks = __builtin_amdgcn_readlane(chunks, i);
      w.tile = JOIN ? rest : rest / w.chunks;
      w.split = JOIN ? 0 : rest - w.tile * w.chunks;
      w.start = __builtin_amdgcn_readlane(s.start, i);
      w.n = __builtin_amdgcn_readlane(s.n, i);
      w.len = __builtin_amdgcn_readlane(s.len, i);
      w.part = ((parts + lane_of(sums_upto - sums, i) + (int64_t)w.tile * w.chunks) * p.Hk + w.hk * w.chunks) + w.split;
      return true;
    }
    before += lane_of(upto, 63);
    parts += lane_of(sums_upto, 63);
  }
  return false;
}

// A tile's keys: those up to its last row's own token; a chunk takes the same part
// of them, in whole tiles of keys.
struct Keys {
  int all, per;
};
__device__ __forceinline__ Keys keys_of(const Work& w, int row0, int tile_rows, int G) {
  const int last = min(w.n - 1, (row0 + tile_rows - 1) / G);
  const int all = max(w.len - w.n + last + 1, 0);
  return {all, ((all + w.chunks - 1) / w.chunks + 63) / 64 * 64};
}

// The sums of a chunk, of `rows` rows: [D / 4][rows][4] floats, then [rows][2], the
// maximum and the sum of the weights.
__device__ __forceinline__ float* sums_of(const ChunkParams& p, const ChunkClass& k, int64_t part) {
  return p.part + k.part_at + part * k.rows * (p.D + 2);
}

// x / page, of x below 2^31.
__device__ __forceinline__ int page_of(const ChunkParams& p, int x) {
  return p.page == 1 ? x : (int)(__umulhi((uint32_t)x, p.page_mul) >> p.page_shift);
}

// ---------------------------------------------------------------------------
// 32 rows a block
// ---------------------------------------------------------------------------

template <bool BF16_, int DP_, int NW_>
struct WaveCfg {
  static constexpr bool BF16 = BF16_;
  static constexpr int DP = DP_, NW = NW_, ES = BF16 ? 2 : 4, RB = DP * ES, PIECES = RB / 16, STEPS = RB / 32, DB = DP / 32;
  static constexpr int TILE = 32 * RB, STAGE = 2 * TILE;  // keys, values
  static constexpr int RPL = 64 / PIECES, LOADS = 32 / RPL;
  static constexpr bool QREG = DP < 256;  // the queries in registers, else in LDS
  static constexpr int ROWS = 32;
  static_assert(STAGE >= ROWS * DP * 4, "a wave's sums fit its stage");
};

__device__ const u32x4 kNoKey = {0u, 0u, 0u, 0u};  // what lanes without a key load

// A block's waves share its rows: each takes every NW-th tile of 32 keys through
// LDS of its own, and their sums meet in LDS at the end.
template <class C>
__global__ __launch_bounds__(64 * C::NW, 1) void chunk_wave_kernel(ChunkParams p, ChunkClass k) {
  constexpr bool BF16 = C::BF16, QREG = C::QREG;
  constexpr int ES = C::ES, RB = C::RB, DB = C::DB, NW = C::NW;
  __shared__ __attribute__((aligned(1024))) char lds[NW * C::STAGE];
  __shared__ __attribute__((aligned(16))) char qlds[QREG ? 16 : C::STEPS * 1024];
  __shared__ float stats[NW][32][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int G = p.Hq / p.Hk;
  Work w;
  if (!find_work<false>(p, k, blockIdx.x, lane, w)) return;
  const int row0 = w.tile * 32, rows = w.n * G, context = w.len - w.n;
  const Keys keys = keys_of(w, row0, 32, G);
  const int kbeg = w.split * keys.per, kend = min(keys.all, kbeg + keys.per);
  if ((w.split > 0 && kbeg >= keys.all) || (w.chunks > 1 && w.part >= k.parts)) return;
  const int shared = context + row0 / G + 1;  // keys that every row sees

  u32x4 qf[QREG ? C::STEPS : 1];
  const int npieces = p.D * ES / 16;
  const int r = min(row0 + col, rows - 1);  // rows behind the last repeat it, and are not stored
  const int tok = r / G, last = context + tok;  // the row's last key
  {
    const char* const qp = static_cast<const char*>(p.q) + ((int64_t)(w.start + tok) * p.q_t + (int64_t)(w.hk * G + r - tok * G) * p.q_h) * ES;
    if constexpr (QREG)
#pragma unroll
      for (int s = 0; s < C::STEPS; ++s) {
        const int c = 2 * s + half;
        qf[s] = c < npieces ? *reinterpret_cast<const u32x4*>(qp + 16 * c) : u32x4{0u, 0u, 0u, 0u};
      }
    else
      for (int s = wave; s < C::STEPS; s += NW) {
        const int c = 2 * s + half;
        *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>((attn_lds)qlds + (s * 64 + lane) * 16) =
            c < npieces ? *reinterpret_cast<const u32x4*>(qp + 16 * c) : u32x4{0u, 0u, 0u, 0u};
      }
  }
  f32x16 o[DB];
  RowState st = {-INFINITY, 0.f};
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  const attn_lds mine = (attn_lds)lds + wave * C::STAGE;
  if (p.D < C::DP)  // pieces behind the head's end: never loaded, zeros
    for (int i = lane; i < C::STAGE / 16; i += 64) *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(mine + 16 * i) = u32x4{0u, 0u, 0u, 0u};

  const char* const kb = static_cast<const char*>(p.kc) + (int64_t)w.hk * p.k_h * ES;
  const char* const vb = static_cast<const char*>(p.vc) + (int64_t)w.hk * p.v_h * ES;
  const int* const table = p.table + (int64_t)w.b * p.table_b;
  const TileLane<RB, BF16> at(lane);
  const int lrow = lane / C::PIECES, lc = lane % C::PIECES;
  const int kpiece0 = lc ^ k_swz<RB>(lrow), vpiece0 = lc ^ v_swz<RB, BF16>(lrow);
  const uint32_t krow = (uint32_t)(lrow * (int)p.k_t * ES), vrow = (uint32_t)(lrow * (int)p.v_t * ES);
  uint32_t bad = 0;

  // The page and place of one key: lane i's of key ku + its part of the tile.  With
  // whole loads in a page (alike) lane j looks up load j, else lane i key i.
  const bool alike = p.alike && p.page % C::RPL == 0;
  auto key_of = [&](int ku) { return alike ? min(ku + lane % C::LOADS * C::RPL, (kend - 1) / C::RPL * C::RPL) : min(ku + col, kend - 1); };
  auto page_at = [&](int ku) -> int { return ku < kend ? table[page_of(p, key_of(ku))] : 0; };

  // One tile: S = K Q^T, the weights, O += V^T P^T.  Pieces are read from LDS
  // kAhead products before they are needed, the first of V behind the weights.
  // masked: not every row sees every key of it; infinities and NaN among its values
  // are taken as zeros, for those that do not, and the others get them at the end.
  auto unit = [&](auto masked_, int ku, uint32_t seen) {
    constexpr bool masked = decltype(masked_)::value;
    const attn_lds lk = mine, lv = mine + C::TILE;
    constexpr int kAhead = RB < 1024 ? 4 : 2, VF = BF16 ? 2 * DB : 16 * DB;  // VF: pieces of V
    u32x4 kf[kAhead], vf[kAhead], qa[kAhead];
    auto read_query = [&](int t) { return *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>((attn_lds)qlds + (t * 64 + lane) * 16); };
    auto read_value = [&](int f) {
      if constexpr (BF16) vf[f % kAhead] = at.values(lv, f / DB, f % DB);
      else vf[f % kAhead].x = at.value(lv, f / DB, f % DB);
    };
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      kf[t] = at.key(lk, t);
      if constexpr (!QREG) qa[t] = read_query(t);
    }
    f32x16 s = {};
#pragma unroll
    for (int t = 0; t < C::STEPS; ++t) {
      __builtin_amdgcn_sched_barrier(0);
      s = attn_mfma<BF16>(kf[t % kAhead], QREG ? qf[QREG ? t : 0] : qa[t % kAhead], s);
      if (t + kAhead < C::STEPS) {
        kf[t % kAhead] = at.key(lk, t + kAhead);
        if constexpr (!QREG) qa[t % kAhead] = read_query(t + kAhead);
      } else read_value(t + kAhead - C::STEPS);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (masked) {
      const int n = last - ku + 1;
      const uint32_t see = (seen & (n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u)) >> (4 * half);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = see >> (8 * (i >> 2) + (i & 3)) & 1u ? s[i] : -INFINITY;
    }
    float mx = lane_max(s) * p.c;
    if (__any(mx > st.m + kSlack)) {
      const float m = fmaxf(st.m, fmaxf(mx, __shfl_xor(mx, 32)));
      const float a = m == -INFINITY ? 1.f : exp2f(st.m - m);
      st.m = m;
      st.l *= a;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= a;
    }
    const float m = st.m == -INFINITY ? 0.f : st.m;
    u32x4 pb[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, -m));
    if constexpr (BF16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        pb[i / 4][i % 4] = pack_bf16x2(s[2 * i], s[2 * i + 1]);
        st.l = add_pair(pb[i / 4][i % 4], st.l);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) st.l += s[i];
    }
#pragma unroll
    for (int f = 0; f < VF; ++f) {
      __builtin_amdgcn_sched_barrier(0);
      u32x4 v = vf[f % kAhead];
      if constexpr (masked)
#pragma unroll
        for (int e = 0; e < (BF16 ? 4 : 1); ++e) v[e] = scrub<BF16>(v[e], bad);
      if constexpr (BF16) o[f % DB] = attn_mfma<true>(v, pb[f / DB], o[f % DB]);
      else o[f % DB] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v.x), s[f / DB], o[f % DB], 0, 0, 0);
      if (f + kAhead < VF) read_value(f + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  // The tile's loads, whose page `pg` is known; `pg` is then the next tile's.
  // Returns which of its keys are there.  A page outside the cache holds none:
  // page 0 (whole loads) or zeros are loaded for it, and masked.
  constexpr int STEP = 32 * NW;
  int ku = kbeg + 32 * wave;
  int pg = page_at(ku);
  auto load = [&](int ku, int& pg) -> uint32_t {
    const bool there = pg >= 0 && pg < p.pages;
    const int key = key_of(ku), in = key - page_of(p, key) * p.page;
    uint32_t seen = ku + 32 <= kend ? 0xffffffffu : (1u << (kend - ku)) - 1u;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage's last reads are done
    const uint32_t base = (uint32_t)(uintptr_t)mine;
    int kpiece = kpiece0, vpiece = vpiece0;
    // where registers are short, the loads' offsets are computed each time
    if constexpr (RB >= 256) asm volatile("" : "+v"(kpiece), "+v"(vpiece));
    if (alike) {
      const int64_t off = ((int64_t)(there ? pg : 0) * p.k_p + (int64_t)in * p.k_t) * ES;
      const uint32_t lost = (uint32_t)__ballot(!there) & (uint32_t)((1ull << C::LOADS) - 1);
      if (lost)
#pragma unroll 1
        for (int j = 0; j < C::LOADS; ++j)
          if (lost >> j & 1u) seen &= ~((uint32_t)((1ull << C::RPL) - 1) << (j * C::RPL));
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) {
        const int ck = kpiece ^ k_swz<RB>(j * C::RPL), cv = vpiece ^ v_swz<RB, BF16>(j * C::RPL);
        const int64_t a = lane_of(off, j);
        if (ck < npieces) load_lds16(kb + a, krow + 16 * ck, base + j * 1024);
        if (cv < npieces) load_lds16(vb + a, vrow + 16 * cv, base + C::TILE + j * 1024);
      }
    } else {
      seen &= ~(uint32_t)__ballot(!there);  // (both halves alike)
#pragma unroll 1
      for (int j = 0; j < C::LOADS; ++j) {
        const int row = j * C::RPL + lrow, pgr = __shfl(pg, row), inr = __shfl(in, row);
        const int ck = lc ^ k_swz<RB>(row), cv = lc ^ v_swz<RB, BF16>(row);
        const bool is = seen >> row & 1u;
        const char* const kp = is ? kb + ((int64_t)pgr * p.k_p + (int64_t)inr * p.k_t) * ES + 16 * ck : reinterpret_cast<const char*>(&kNoKey);
        const char* const vp = is ? vb + ((int64_t)pgr * p.v_p + (int64_t)inr * p.v_t) * ES + 16 * cv : reinterpret_cast<const char*>(&kNoKey);
        if (ck < npieces) load_lds16(kp, base + j * 1024);
        if (cv < npieces) load_lds16(vp, base + C::TILE + j * 1024);
      }
    }
    pg = page_at(ku + STEP);
    wait_loads<0>();
    return seen;
  };
  __syncthreads();
  // Whole tiles that every row sees, up to the first that is not; then the others,
  // masked.  (Two loops: a branch in one kept the registers of both.)
  if constexpr (RB < 1024)  // (else two copies of a tile's code do not fit the registers)
    for (; ku + 31 < min(shared, kend); ku += STEP) {
      const int held = pg;
      if (load(ku, pg) != 0xffffffffu) {
        pg = held;  // loaded again below
        break;
      }
      unit(std::false_type{}, ku, 0xffffffffu);
    }
  const int masked_from = ku;
  for (; ku < kend; ku += STEP) {
    const uint32_t seen = load(ku, pg);
    unit(std::true_type{}, ku, seen);
  }

  // Each wave's sums, scaled to the block's maximum, in its own LDS; then all
  // threads add the waves' in order.  Row r's 16-byte pieces are spread by r.
  constexpr int OP = C::DP / 4, OM = OP < 32 ? OP - 1 : 31;
  const float l = st.l + __shfl_xor(st.l, 32);
  if (half == 0) {
    stats[wave][col][0] = st.m;
    stats[wave][col][1] = l;
  }
  __syncthreads();
  {
    float m = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) m = fmaxf(m, stats[x][col][0]);
    const float a = st.m == -INFINITY ? 1.f : exp2f(st.m - m);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int piece = 8 * d + 2 * q + half;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[d][4 * q + e] * a;
        *reinterpret_cast<SVDMLP_ATTN_LDS f32x4*>(mine + (col * OP + (piece ^ (col & OM))) * 16) = v;
      }
  }
  if (__any(bad != 0)) {
    for (int kt = masked_from; kt < kend; kt += STEP) {
      for (int key = kt; key < min(kt + 32, kend); ++key) {
        const int pg = table[page_of(p, key)];
        if (pg < 0 || pg >= p.pages) continue;
        const char* const vp = vb + ((int64_t)pg * p.v_p + (int64_t)(key - page_of(p, key) * p.page) * p.v_t) * ES;
        auto value = [&](int e) -> uint32_t {
          return BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(vp)[e] << 16 : reinterpret_cast<const uint32_t*>(vp)[e];
        };
        bool any = false;
        for (int e = lane; e < p.D; e += 64) any |= not_finite<false>(value(e)) != 0;
        if (!__any(any)) continue;
        for (int e = 0; e < p.D; ++e) {
          const uint32_t x = value(e);
          if (not_finite<false>(x) && half == 0 && key <= last)
            *(SVDMLP_ATTN_LDS float*)(mine + (col * OP + ((e >> 2) ^ (col & OM))) * 16 + 4 * (e & 3)) += __uint_as_float(x);
        }
      }
    }
  }
  __syncthreads();
  float* const sums = w.chunks > 1 ? sums_of(p, k, w.part) : nullptr;
  for (int i = threadIdx.x; i < 32 * OP; i += 64 * NW) {
    // (sums go out row by row, results piece by piece of a row)
    const int rr = w.chunks > 1 ? i % 32 : i / OP, piece = w.chunks > 1 ? i / 32 : i % OP, row = row0 + rr;
    if (row >= rows || 4 * piece >= p.D) continue;
    float m = -INFINITY, sum = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NW; ++x) m = fmaxf(m, stats[x][rr][0]);
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float mw = stats[x][rr][0];
      sum += mw == -INFINITY ? stats[x][rr][1] : stats[x][rr][1] * exp2f(mw - m);
      v += *reinterpret_cast<SVDMLP_ATTN_LDS f32x4*>((attn_lds)lds + x * C::STAGE + (rr * OP + (piece ^ (rr & OM))) * 16);
    }
    if (w.chunks > 1) {
      reinterpret_cast<f32x4*>(sums)[piece * 32 + rr] = v;
      if (piece == 0) reinterpret_cast<f32x2*>(sums + 32 * p.D)[rr] = f32x2{m, sum};
    } else {
      v *= inverse_sum(sum);
      const int t = row / G;
      store4<BF16>(p.out, (int64_t)(w.start + t) * p.o_t + (int64_t)(w.hk * G + row - t * G) * p.o_h + 4 * piece, v);
    }
  }
}

// ---------------------------------------------------------------------------
// 256 rows a block
// ---------------------------------------------------------------------------

constexpr int kIds = 2048;  // pages whose numbers lie in LDS, two halves of them

template <class C>
__global__ __launch_bounds__(256, 1) void chunk_pipe_kernel(ChunkParams p, ChunkClass k) {
  constexpr int RB = C::RB, QG = C::QG, KB = C::KB, DB = C::DB;
  __shared__ __attribute__((aligned(1024))) char lds[C::NS * C::STAGE];
  __shared__ int ids[kIds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int G = p.Hq / p.Hk;
  Work w;
  if (!find_work<false>(p, k, blockIdx.x, lane, w)) return;
  const int row0 = w.tile * C::BM, rows = w.n * G, context = w.len - w.n;
  const Keys all = keys_of(w, row0, C::BM, G);
  const int kbeg = w.split * all.per;
  if ((w.split > 0 && kbeg >= all.all) || (w.chunks > 1 && w.part >= k.parts)) return;
  const int nkeys = min(all.all, kbeg + all.per) - kbeg;  // of this chunk, its first number 0 from here on
  const int first = context - kbeg;                       // the first new token's key
  const int tiles = (nkeys + KB - 1) / KB;
  const int npieces = p.D / 8;

  // The chunk's pages: the numbers of the first ones in LDS, and whether all are
  // pages of the cache.
  const int* const table = p.table + (int64_t)w.b * p.table_b;
  const int pg0 = page_of(p, kbeg), pages = nkeys > 0 ? page_of(p, kbeg + nkeys - 1) - pg0 + 1 : 0;
  auto valid = [&](int pg) { return pg >= 0 && pg < p.pages; };
  bool lost = false;
  for (int i0 = threadIdx.x; i0 < pages; i0 += 256 * 8) {
    int v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = table[pg0 + min(i0 + 256 * j, pages - 1)];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lost |= !valid(v[j]);
      if (i0 + 256 * j < min(pages, kIds)) ids[i0 + 256 * j] = v[j];
    }
  }
  const attn_lds base = (attn_lds)lds;
  // Zeros where a head is shorter than its place (never loaded), and in the
  // last stage's values, which the first step multiplies by zero weights.
  if (p.D < C::DP) {
    for (int i = threadIdx.x; i < C::NS * C::STAGE / 16; i += 256) *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(base + 16 * i) = u32x4{0u, 0u, 0u, 0u};
  } else {
    for (int i = threadIdx.x; i < C::UNIT / 16; i += 256)
      *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(base + (C::NS - 1) * C::STAGE + C::TILE + C::UNIT + 16 * i) = u32x4{0u, 0u, 0u, 0u};
  }
  const bool holes = __syncthreads_or(lost);
  const int full = holes ? 0 : max(min(first + row0 / G + 1, nkeys), 0) / KB;  // whole tiles that every row sees

  const char* const kb = static_cast<const char*>(p.kc) + (int64_t)w.hk * p.k_h * 2;
  const char* const vb = static_cast<const char*>(p.vc) + (int64_t)w.hk * p.v_h * 2;
  // This wave's loads of a tile: rows wave * LOADS * RPL .. of its keys and values.
  const int lrow = wave * C::LOADS * C::RPL + lane / C::PIECES, lc = lane % C::PIECES;
  const bool alike = p.alike && p.page % C::RPL == 0;  // whole loads in a page, both caches laid out alike
  uint32_t koff[C::LOADS], voff;  // a lane's place in a load: its row of RPL, its piece
  bool kin[C::LOADS];
  const int vc = lc ^ v_swz<RB, true>(lrow);
#pragma unroll
  for (int j = 0; j < C::LOADS; ++j) {
    const int c = lc ^ k_swz<RB>(lrow + j * C::RPL);
    koff[j] = (uint32_t)(lane / C::PIECES * (int)p.k_t * 2 + 16 * c);
    kin[j] = c < npieces;
  }
  voff = (uint32_t)(lane / C::PIECES * (int)p.v_t * 2 + 16 * vc);
  const bool vin = vc < npieces;
  int loaded = kIds;  // pages whose numbers have been put into LDS
  // The place of key `x` of the chunk, in elements; its page's number is in LDS.
  // (A page outside the cache holds no keys: page 0 is read for it, and masked.)
  auto place = [&](int x, int64_t p_s, int64_t t_s) -> int64_t {
    const int key = kbeg + min(x, nkeys - 1), pg = page_of(p, key), id = ids[(pg - pg0) & (kIds - 1)];
    return (int64_t)(valid(id) ? id : 0) * p_s + (int64_t)(key - pg * p.page) * t_s;
  };
  int64_t ahead = 0;  // alike: lane j's place of load j of the last tile of keys asked for
  auto issue_keys = [&](int t) {
    if (t >= tiles) return;
    const uint32_t to = (uint32_t)(uintptr_t)(base + (t % C::NS) * C::STAGE) + wave * C::LOADS * 1024;
    if (alike) {
      // (keys behind the last: rows of its load's page)
      const int x = t * KB + (wave * C::LOADS + lane % C::LOADS) * C::RPL;
      ahead = place(min(x, (nkeys - 1) / C::RPL * C::RPL), p.k_p, p.k_t) * 2;
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) {
        const int64_t a = lane_of(ahead, j);
        if (kin[j]) load_lds16(kb + a, koff[j], to + j * 1024);
      }
    } else {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) {
        const int row = lrow + j * C::RPL;
        if (kin[j]) load_lds16(kb + place(t * KB + row, p.k_p, p.k_t) * 2 + 16 * (lc ^ k_swz<RB>(row)), to + j * 1024);
      }
    }
  };
  auto issue_values = [&](int t, int64_t where) {
    if (t >= tiles) return;
    const uint32_t to = (uint32_t)(uintptr_t)(base + (t % C::NS) * C::STAGE) + C::TILE + wave * C::LOADS * 1024;
    if (alike) {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) {
        const int64_t a = lane_of(where, j);
        if (vin) load_lds16(vb + a, voff, to + j * 1024);
      }
    } else {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j)
        if (vin) load_lds16(vb + place(t * KB + lrow + j * C::RPL, p.v_p, p.v_t) * 2 + 16 * vc, to + j * 1024);
    }
  };
  u32x4 qf[QG][C::STEPS];
  int tok[QG];
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const int r = min(row0 + (wave * QG + g) * 32 + col, rows - 1);  // rows behind the last repeat it, and are not stored
    tok[g] = r / G;
    const char* qp = static_cast<const char*>(p.q) + ((int64_t)(w.start + tok[g]) * p.q_t + (int64_t)(w.hk * G + r - tok[g] * G) * p.q_h) * 2;
#pragma unroll
    for (int s = 0; s < C::STEPS; ++s) {
      const int c = 2 * s + half;
      qf[g][s] = c < npieces ? *reinterpret_cast<const u32x4*>(qp + 16 * c) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  issue_keys(0);
  const int64_t ahead0 = ahead;
  issue_keys(1);
  issue_values(0, ahead0);
  const int64_t ahead1 = ahead;
  issue_keys(2);
  issue_values(1, ahead1);
  PipeWave<C> pw(qf, lane, p.c);
  // Before tile t: the keys of tile t + 1 and the values of tile t are there for
  // every wave (they were asked for two tiles ago; what was asked for one tile
  // ago may still be on its way), and every wave is done with the keys of tile
  // t - 1 and the values of tile t - 2, whose places are filled again.
  auto arrive = [&](int t) {
    if (t + 2 < tiles) wait_loads<2 * C::LOADS>();
    else wait_loads<0>();
    asm volatile("s_barrier" ::: "memory");
    if (loaded < pages) {
      // No wave asks for a page before tile t + 2's any more: once those are in the
      // second half of the numbers, the first half's place takes the next ones.
      const int now = page_of(p, kbeg + min((t + 2) * KB, nkeys - 1)) - pg0;
      if (now >= loaded - kIds / 2) {
        for (int i = threadIdx.x; i < kIds / 2; i += 256)
          if (loaded + i < pages) ids[(loaded + i) & (kIds - 1)] = table[pg0 + loaded + i];
        loaded += kIds / 2;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    }
    const int64_t here = ahead;
    issue_keys(t + 3);
    issue_values(t + 2, here);
  };

  int t = 0;
  if (full > 0) pw.whole_tiles(base, full, t, arrive);
  for (; t < tiles; ++t) {
    arrive(t);
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
      if (holes) {
        const int pg = kbeg + k0 + col < kbeg + nkeys ? table[page_of(p, kbeg + k0 + col)] : -1;
        there = (uint32_t)__ballot(valid(pg));
      }
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

  const bool joined = w.chunks > 1;
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    pw.l[g] += __shfl_xor(pw.l[g], 32);
    const float inv = joined ? 1.f : inverse_sum(pw.l[g]);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) pw.o[g][d][i] *= inv;
  }
  // Infinities and NaN among the values of the plain loop were taken as
  // zeros, for the rows that do not see them; the rows that do get them here.
  if (__any(pw.bad != 0)) {
    for (int key = full * KB; key < nkeys; ++key) {
      const int at = page_of(p, kbeg + key), pg = table[at];
      if (!valid(pg)) continue;
      const uint16_t* const vp = reinterpret_cast<const uint16_t*>(vb + ((int64_t)pg * p.v_p + (int64_t)(kbeg + key - at * p.page) * p.v_t) * 2);
      uint32_t see[QG];
#pragma unroll
      for (int g = 0; g < QG; ++g) see[g] = key <= first + tok[g] ? 0xffffffffu : 0u;
      int D = p.D;
      asm volatile("" : "+s"(D));  // its comparisons stay in the loop: hoisted, they spill
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int e = 32 * d + 8 * (i >> 2) + 4 * half + (i & 3);
          const uint32_t x = e >= D ? 0u : (uint32_t)vp[e] << 16, mask = not_finite<false>(x);
#pragma unroll
          for (int g = 0; g < QG; ++g) pw.o[g][d][i] += __uint_as_float(x & mask & see[g]);
        }
    }
  }
  float* const sums = joined ? sums_of(p, k, w.part) : nullptr;
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const int rr = (wave * QG + g) * 32 + col, r = row0 + rr;
    if (r >= rows) continue;
    const int64_t op = (int64_t)(w.start + tok[g]) * p.o_t + (int64_t)(w.hk * G + (r - tok[g] * G)) * p.o_h;
    if (joined && half == 0) reinterpret_cast<f32x2*>(sums + C::BM * p.D)[rr] = f32x2{pw.m[g], pw.l[g]};
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int e = 32 * d + 8 * b + 4 * half;
        if (e >= p.D) continue;
        const f32x4 v = {pw.o[g][d][4 * b], pw.o[g][d][4 * b + 1], pw.o[g][d][4 * b + 2], pw.o[g][d][4 * b + 3]};
        if (joined) reinterpret_cast<f32x4*>(sums)[(e >> 2) * C::BM + rr] = v;
        else store4<true>(p.out, op + e, v);
      }
  }
}

// ---------------------------------------------------------------------------
// The chunks' sums
// ---------------------------------------------------------------------------

// Joins the chunks of every tile that was cut: a thread takes 16 bytes of a row's
// sums (four elements), a block 256 of them, and goes on with the block `gridDim`
// further.
template <bool BF16>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkParams p, ChunkClass many, ChunkClass few) {
  const int lane = threadIdx.x & 63, G = p.Hq / p.Hk;
  auto join = [&](const ChunkClass& k) {
    const int per = 256 / k.rows, units = (p.D / 4 + per - 1) / per;  // units of a tile
    for (int64_t id = blockIdx.x;; id += gridDim.x) {
      Work w;
      if (!find_work<true>(p, k, id / units, lane, w)) return;
      const int unit = (int)(id % units), rr = threadIdx.x % k.rows, piece = unit * per + threadIdx.x / k.rows;
      const int row0 = w.tile * k.rows, r = row0 + rr;
      const Keys keys = keys_of(w, row0, k.rows, G);
      const int used = max(1, keys.per ? (keys.all + keys.per - 1) / keys.per : 1);
      if (r < w.n * G && 4 * piece < p.D && w.part + used <= k.parts) {
        const int64_t step = (int64_t)k.rows * (p.D + 2);  // floats of a chunk's sums
        const float* const sums = sums_of(p, k, w.part);
        const f32x4* const from = reinterpret_cast<const f32x4*>(sums) + piece * k.rows + rr;
        const f32x2* const ml = reinterpret_cast<const f32x2*>(sums + k.rows * p.D) + rr;
        float m = -INFINITY, l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < used; s0 += 8) {
          f32x2 v[8];
          f32x4 x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int64_t s = min(s0 + j, used - 1) * step;
            v[j] = *reinterpret_cast<const f32x2*>(reinterpret_cast<const float*>(ml) + s);
            x[j] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(from) + s);
          }
          float most = m;
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, v[j].x);
          const float a = m == most ? 1.f : exp2f(m - most);
          l *= a;
          o *= a;
          m = most;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            // (a chunk without a score over -infinity: its sums are zeros, or not finite and stay so)
            const float b = s0 + j >= used ? 0.f : v[j].x == -INFINITY ? 1.f : exp2f(v[j].x - m);
            if (s0 + j < used) {
              l += v[j].y * b;
              o += x[j] * b;
            }
          }
        }
        o *= inverse_sum(l);
        const int t = r / G;
        store4<BF16>(p.out, (int64_t)(w.start + t) * p.o_t + (int64_t)(w.hk * G + r - t * G) * p.o_h + 4 * piece, o);
      }
    }
  };
  if (many.parts) join(many);
  if (few.parts) join(few);
}

template <bool BF16, int DP, int NW>
void run_wave(const ChunkParams& p, const ChunkClass& k, hipStream_t st) {
  hipLaunchKernelGGL((chunk_wave_kernel<WaveCfg<BF16, DP, NW>>), dim3((unsigned)k.blocks), dim3(64 * NW), 0, st, p, k);
}

}  // namespace

ChunkPlan plan_chunk_attention(int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D, bool bf16, int64_t capacity, int64_t cus) {
  ChunkPlan plan = {};
  const int64_t rows = T * (Hq / Hk);  // at most, a key/value head
  const bool pipe = bf16 && D <= 128;
  auto fill = [&](ChunkClass& k, int64_t from, int64_t upto, int tile, int64_t slots, int least) {
    k.from = (int)std::min<int64_t>(from, 0x7fffffff), k.upto = (int)std::min<int64_t>(upto, 0x7fffffff);
    k.rows = tile, k.least = least;
    if (rows < from) return;
    // Sequences of the class, and their tiles: at most one short tile each.
    const int64_t n = std::min(B, rows / from);
    int64_t tiles = rows / tile + n;
    if (upto < rows) tiles = std::min(tiles, n * ((upto + tile - 1) / tile));
    const int64_t chunks = std::min<int64_t>((capacity + least - 1) / least, kSplitsMost);  // of a tile
    k.slots = (int)std::max<int64_t>(slots, 1);
    k.blocks = std::min(tiles * Hk * chunks, tiles * Hk + slots);
    // Tiles in several chunks have at most twice as many as there are slots.
    if (chunks > 1) k.parts = std::min(tiles * Hk * chunks, 2 * slots);
    k.part_at = plan.floats;
    plan.floats += k.parts * tile * (D + 2);
  };
  if (pipe) {
    fill(plan.many, kFewRows + 1, rows, 256, cus, 512);
    fill(plan.few, 1, kFewRows, 32, 4 * cus, 256);
  } else {
    fill(plan.few, 1, rows, 32, 4 * cus, 256);
  }
  return plan;
}

hipError_t launch_chunk_attention(const ChunkParams& p, bool bf16, const ChunkPlan& plan, int cus, hipStream_t st) {
  if (p.T <= 0 || p.B <= 0) return hipSuccess;
  if (!fits_launch(plan.many.blocks, 256) || !fits_launch(plan.few.blocks, 256)) return hipErrorInvalidValue;
  if (plan.many.blocks) {
    if (p.D <= 64) hipLaunchKernelGGL((chunk_pipe_kernel<PipeCfg<64>>), dim3((unsigned)plan.many.blocks), dim3(256), 0, st, p, plan.many);
    else hipLaunchKernelGGL((chunk_pipe_kernel<PipeCfg<128>>), dim3((unsigned)plan.many.blocks), dim3(256), 0, st, p, plan.many);
  }
  if (plan.few.blocks) {
    if (bf16) p.D <= 64 ? run_wave<true, 64, 4>(p, plan.few, st) : p.D <= 128 ? run_wave<true, 128, 4>(p, plan.few, st) : run_wave<true, 256, 2>(p, plan.few, st);
    else p.D <= 64 ? run_wave<false, 64, 4>(p, plan.few, st) : p.D <= 128 ? run_wave<false, 128, 2>(p, plan.few, st) : run_wave<false, 256, 1>(p, plan.few, st);
  }
  if (plan.many.parts || plan.few.parts) {
    const dim3 grid((unsigned)(4 * cus));
    if (bf16) hipLaunchKernelGGL((chunk_join_kernel<true>), grid, dim3(256), 0, st, p, plan.many, plan.few);
    else hipLaunchKernelGGL((chunk_join_kernel<false>), grid, dim3(256), 0, st, p, plan.many, plan.few);
  }
  return hipGetLastError();
}

}  // namespace svdmlp
