// Attention of up to 32 rows a wave (64 with QG = 2): the kernel of
// cache_attention.hip (new tokens onto a paged cache) and, with CacheCfg::PROMPT,
// of prompts of few rows (prompt_attention.hip).  Without CacheCfg::SHARE each
// wave takes every NW-th tile of 32 keys through LDS of its own, with no barrier
// in the loop; a block's waves share its rows, and their sums meet in LDS at the
// end.  With it every wave takes every tile, for rows of its own; each loads a
// part of it, and a barrier a tile keeps them together.
#pragma once

#include <math.h>

#include <type_traits>

#include "attn.hpp"
#include "decoder.hpp"

namespace svdmlp {

constexpr int kSplitsMost = 64;   // chunks of a sequence
constexpr int kJoin = 16;         // chunks' sums in flight when they are joined
constexpr int kPagesMost = 1024;  // whole pages of a chunk: their numbers lie in LDS

template <bool BF16_, int DP_, int QG_, int NW_, bool PROMPT_ = false, int STAGES_ = 2, bool SHARE_ = false>
struct CacheCfg {
  static constexpr bool PROMPT = PROMPT_;  // packed prompts in place of a paged cache
  static constexpr bool BF16 = BF16_;
  static constexpr int DP = DP_, QG = QG_;
  static constexpr int ES = BF16 ? 2 : 4;
  static constexpr int RB = DP * ES;
  static constexpr int PIECES = RB / 16;
  static constexpr int STEPS = RB / 32;
  static constexpr int NW = NW_;  // waves a block
  static constexpr int STAGES = STAGES_;  // tiles in LDS a wave: 1 where another block of the CU hides its loads
  static constexpr int TILE = 32 * RB;
  static constexpr int STAGE = 2 * TILE;  // keys, values
  static constexpr bool SHARE = SHARE_;  // every wave takes every tile, for 32 rows of its own; all load them
  static constexpr int WROWS = 32 * QG, ROWS = SHARE ? NW * WROWS : WROWS;  // rows of a wave, of a block
  static constexpr int RPI = 64 / PIECES;        // rows a load
  static constexpr int LOADS = 32 / RPI;         // loads a tile, of keys and of values
  static constexpr int MINE = SHARE ? LOADS / NW : LOADS;  // of them a wave's
  static constexpr bool QREG = DP < 256;  // Q in registers
  static_assert(QREG || (QG == 1 && !SHARE), "Q in LDS: one copy for the block");
  static constexpr int LDS = (SHARE ? 1 : NW) * STAGES * STAGE;
  static_assert(LDS / NW >= WROWS * DP * 4, "a wave's sums fit its part of LDS");
  static_assert(!SHARE || (LOADS % NW == 0 && STAGES > 2), "shared tiles");
};

// 16 bytes of zeros that lanes without a key load.
static __device__ const u32x4 kZeroPiece = {0u, 0u, 0u, 0u};

// Lane j's v, the same for all lanes (j a constant).
__device__ __forceinline__ int64_t lane64(int64_t v, int j) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, j) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), j) << 32);
}

// Partial sums cross blocks, and so XCDs with an L2 each, by device-scope (sc1)
// accesses past the L2, without any cache maintenance: fences that write back
// and drop the L2 for every block made a call of 4096 blocks 325 us instead of
// 137.  Offsets are in bytes from a sequence's part.
constexpr int kDevice = 16;  // the sc1 bit of a buffer access
__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_of(const CacheParams& p, int b, int floats) {
  const int64_t rows = (int64_t)p.n * p.Hq * p.splits;
  float* const base = p.part + (floats == 2 ? (int64_t)p.B * rows * p.D : 0) + (int64_t)b * rows * floats;
  return __builtin_amdgcn_make_buffer_rsrc(base, 0, (int)(rows * floats * 4), 0x00020000);
}

__device__ __forceinline__ int held(const CacheParams& p, int b) {
  const int64_t cap = (int64_t)p.width * p.page;
  return (int)min((int64_t)max(p.lengths[b], 0), cap);
}

// Keys of a chunk of blocks that share their tiles: as many chunks as blocks run
// at once, over all sequences, heads and row tiles.  (From the table's width
// instead, sequences of unequal lengths left half the card idle.)
__device__ __forceinline__ int shared_chunk(const CacheParams& p, int rtiles, int lane) {
  if (p.chunk == p.chunk_most) return p.chunk;
  int64_t total = lane < p.B ? held(p, lane) : 0;  // (up to 64 sequences)
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
  const int64_t want = ((total * p.Hk * rtiles + p.slots - 1) / p.slots + 127) / 128 * 128;
  return __builtin_amdgcn_readfirstlane((int)min(max(want, (int64_t)p.chunk), (int64_t)p.chunk_most));
}
__device__ __forceinline__ int chunks_of(int len, int chunk) {  // the first always answers
  return max(1, (int)(((int64_t)len + chunk - 1) / chunk));
}

// Which of the 32 keys from `draft` keys after the context on a token sees,
// whose row of the tree is `row`: all of the context.
__device__ __forceinline__ uint32_t seen32(uint64_t row, int draft) {
  if (draft >= 64) return 0;
  if (draft >= 0) return (uint32_t)(row >> draft);
  if (draft <= -32) return 0xffffffffu;
  return (uint32_t)(row << -draft) | ((1u << -draft) - 1u);
}

// Which of the 32 keys from ku on a token sees that sees keys up to `last`.
__device__ __forceinline__ uint32_t upto32(int last, int ku) {
  const int n = last - ku + 1;
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
}

template <class C>
__global__ __launch_bounds__(64 * C::NW, 1) void cache_kernel(CacheParams p) {
  constexpr bool BF16 = C::BF16;
  constexpr bool PROMPT = C::PROMPT, SHARE = C::SHARE;
  constexpr int ES = C::ES, RB = C::RB, QG = C::QG, DB = C::DP / 32, NW = C::NW;
  __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
  __shared__ __attribute__((aligned(16))) char qlds[C::QREG ? 16 : C::STEPS * 1024];
  __shared__ float stats[NW][C::WROWS][2];
  __shared__ int ids[PROMPT ? 1 : kPagesMost + 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int G = p.Hq / p.Hk;
  // The block's rows (r0 .. of `rows`, sequence rows start ..), keys kbeg ..
  // kend, of which those before `context` are seen by every row.
  int rows, rtiles = 1, rt = 0, hk, b = 0, split = 0, used = 1, r0, start = 0, kbeg = 0, kend, context, pg0 = 0, chunk = 0, at_chunk = 0;
  if constexpr (PROMPT) {
    RowTile where;
    if (!find_rows(p.cu, p.T, p.B, p.Hk, G, C::ROWS, lane, where)) return;
    hk = where.hk, start = where.start, r0 = where.row0, rows = where.len * G;
    kend = p.causal ? min(where.len, (r0 + C::ROWS - 1) / G + 1) : where.len;
    context = p.causal ? r0 / G + 1 : where.len;
  } else {
    rows = p.n * G;
    rtiles = (rows + C::ROWS - 1) / C::ROWS;
    int id = blockIdx.x;
    hk = id % p.Hk;
    id /= p.Hk;
    rt = id % rtiles;
    id /= rtiles;
    chunk = p.chunk;
    if (SHARE && p.chunk < p.chunk_most) {
      // Chunk `id` of all sequences' in order.
      chunk = shared_chunk(p, rtiles, lane);
      const int n = lane < p.B ? chunks_of(held(p, lane), chunk) : 0;
      int upto = n;
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
      }
      const uint64_t hit = __ballot(id < upto);
      if (!hit) return;
      b = __builtin_ctzll(hit), split = id - __builtin_amdgcn_readlane(upto - n, b);
    } else {
      b = id % p.B, split = id / p.B;
    }
    at_chunk = SHARE && p.chunk == p.chunk_most ? b * p.splits + split : id;
    const int len = held(p, b);
    r0 = rt * C::ROWS;
    used = chunks_of(len, chunk);
    if (split >= used) return;
    kbeg = split * chunk, kend = kbeg + min(len - kbeg, chunk);  // (kbeg + chunk may pass 2^31)
    context = len - p.n;
    // The chunk's pages.
    pg0 = kbeg / p.page;
    const int npages = min(p.width - pg0, (int)min((int64_t)chunk + p.page - 1, (int64_t)kPagesMost * p.page) / p.page + 1);
    for (int i = threadIdx.x; i < npages; i += 64 * NW) ids[i] = p.table[(int64_t)b * p.table_b + pg0 + i];
  }

  const int w0 = r0 + (SHARE ? wave * C::WROWS : 0);  // the wave's first row
  // Heads of over 128 elements leave no registers for Q: its pieces lie in LDS, in
  // the order of the products.
  constexpr bool QREG = C::QREG;
  u32x4 qf[QG][QREG ? C::STEPS : 1];
  int qi[QG];  // which of the sequence's (new) tokens
  const int npieces = p.D * ES / 16;
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const int r = min(w0 + 32 * g + col, rows - 1);  // rows behind the last repeat it, and are not stored
    qi[g] = r / G;
    const char* const qptr = static_cast<const char*>(p.q) + ((int64_t)b * p.q_b + (int64_t)(start + qi[g]) * p.q_t + (int64_t)(hk * G + r - qi[g] * G) * p.q_h) * ES;
    if constexpr (QREG)
#pragma unroll
      for (int s = 0; s < C::STEPS; ++s) {
        const int c = 2 * s + half;
        qf[g][s] = c < npieces ? *reinterpret_cast<const u32x4*>(qptr + 16 * c) : u32x4{0u, 0u, 0u, 0u};
      }
    else
      for (int s = wave; s < C::STEPS; s += NW) {
        const int c = 2 * s + half;
        *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>((attn_lds)qlds + (s * 64 + lane) * 16) =
            c < npieces ? *reinterpret_cast<const u32x4*>(qptr + 16 * c) : u32x4{0u, 0u, 0u, 0u};
      }
  }
  // Each row's 64 bits of the tree, where the chunk reaches the new tokens: a
  // lane reads one byte of a token's row, and a ballot gathers them.
  uint64_t row_sees[QG];
#pragma unroll
  for (int g = 0; g < QG; ++g) row_sees[g] = (2ull << qi[g]) - 1;  // a chain (token 63: all)
  if (!PROMPT && p.tree && kend > context) {
    const uint8_t* const tree = p.tree + (int64_t)b * p.tree_b;
    const int first = min(w0, rows - 1) / G, last = min(w0 + C::WROWS - 1, rows - 1) / G;
    for (int t = first; t <= last; ++t) {
      const uint64_t bits = __ballot(tree[(int64_t)t * p.tree_q + min(lane, p.n - 1)] != 0);
#pragma unroll
      for (int g = 0; g < QG; ++g) row_sees[g] = qi[g] == t ? bits : row_sees[g];
    }
  }
  f32x16 o[QG][DB];
  RowState st[QG];
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    st[g] = {-INFINITY, 0.f};
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[g][d][i] = 0.f;
  }
  // The loop's loads are counted (wait_loads): none of the above may be among them.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  const attn_lds mine = (attn_lds)lds + wave * (C::LDS / NW);
  const char* const kb = static_cast<const char*>(p.kc) + ((int64_t)start * p.k_t + (int64_t)hk * p.k_h) * ES;
  const char* const vb = static_cast<const char*>(p.vc) + ((int64_t)start * p.v_t + (int64_t)hk * p.v_h) * ES;
  // Key `key - context` of the tokens that not all see: whether row group g's lane does.
  auto sees = [&](int g, int key) -> bool {
    if constexpr (PROMPT) return !p.causal || key <= qi[g];
    else return seen32(row_sees[g], key - context) & 1u;
  };
  const TileLane<RB, BF16> at(lane);
  const float per_page = PROMPT ? 1.f : 1.0f / (float)p.page;
  // A prompt's key is a page of one row.
  const int64_t k_p = PROMPT ? p.k_t : p.k_p, v_p = PROMPT ? p.v_t : p.v_p;
  uint32_t bad = 0;

  // The row (page, place in it) of key ku + row; -1: of none.
  auto place = [&](int ku, int row, int* in) -> int {
    if constexpr (PROMPT) {
      *in = 0;
      return ku + row < kend ? ku + row : -1;
    }
    const int first = ku / p.page, x = ku - first * p.page + row;
    // x < page + 32: one division of small numbers, exact in 32 bits
    const int q = p.page >= 32 ? (x >= p.page) : (int)(((float)x + 0.5f) * per_page);
    *in = x - q * p.page;
    const int i = first + q - pg0;
    const int pg = ku + row < kend ? ids[i] : -1;
    return pg >= 0 && pg < p.pages ? pg : -1;
  };
  // A lane's part of a load's addresses: row lane / PIECES of its RPI rows,
  // piece lane % PIECES, both swizzled; load j adds a constant (the swizzles
  // pick bits of the row, so that they combine by exclusive or).
  const int lrow = lane / C::PIECES, lc = lane % C::PIECES;
  const int kpiece0 = lc ^ k_swz<RB>(lrow), vpiece0 = lc ^ v_swz<RB, BF16>(lrow);
  const uint32_t krow = (uint32_t)(lrow * (int)p.k_t * ES), vrow = (uint32_t)(lrow * (int)p.v_t * ES);
  const bool alike = p.page_shift >= 0 && p.k_p == p.v_p && p.k_t == p.v_t;
  // Loads of the tile at key ku; true: all 32 keys are there.
  const int j0 = SHARE ? wave * C::MINE : 0;  // the first load of this wave
  auto issue = [&](int ku, attn_lds stage) -> bool {
    const uint32_t base = (uint32_t)(uintptr_t)stage;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage's last reads are done
    int kpiece = kpiece0, vpiece = vpiece0;
    // where registers are short, the loads' offsets are computed each time
    if constexpr (QG == 2 || RB >= 512) asm volatile("" : "+v"(kpiece), "+v"(vpiece));
    if constexpr (PROMPT) {
      if (ku + 32 <= kend) {
        const char* const kt = kb + (int64_t)ku * p.k_t * ES;
        const char* const vt = vb + (int64_t)ku * p.v_t * ES;
#pragma unroll
        for (int i = 0; i < C::MINE; ++i) {
          const int j = j0 + i, ck = kpiece ^ k_swz<RB>(j * C::RPI), cv = vpiece ^ v_swz<RB, BF16>(j * C::RPI);
          if (ck < npieces) load_lds16(kt + (int64_t)j * C::RPI * p.k_t * ES, krow + 16 * ck, base + j * 1024);
          if (cv < npieces) load_lds16(vt + (int64_t)j * C::RPI * p.v_t * ES, vrow + 16 * cv, base + C::TILE + j * 1024);
        }
        return true;
      }
    }
    if (!PROMPT && alike && ku + 32 <= kend) {
      // Pages of a power of two that hold whole loads, both caches laid out
      // alike: lane j finds load j's page, and the place of its rows goes to
      // all lanes through scalar registers.
      const int key = ku + lane % C::LOADS * C::RPI, pg = ids[(key >> p.page_shift) - pg0], in = key & (p.page - 1);
      if (__all(pg >= 0 && pg < p.pages)) {
        const int64_t off = ((int64_t)pg * p.k_p + (int64_t)in * p.k_t) * ES;
        if (p.D == C::DP) {
#pragma unroll
          for (int i = 0; i < C::MINE; ++i) {
            const int j = j0 + i;
            const int64_t at = lane64(off, j);
            load_lds16(kb + at, krow + 16 * (kpiece ^ k_swz<RB>(j * C::RPI)), base + j * 1024);
            load_lds16(vb + at, vrow + 16 * (vpiece ^ v_swz<RB, BF16>(j * C::RPI)), base + C::TILE + j * 1024);
          }
        } else {
#pragma unroll
          for (int i = 0; i < C::MINE; ++i) {
            const int j = j0 + i;
            const int ck = kpiece ^ k_swz<RB>(j * C::RPI), cv = vpiece ^ v_swz<RB, BF16>(j * C::RPI);
            const int64_t at = lane64(off, j);
            if (ck < npieces) load_lds16(kb + at, krow + 16 * ck, base + j * 1024);
            if (cv < npieces) load_lds16(vb + at, vrow + 16 * cv, base + C::TILE + j * 1024);
          }
        }
        return true;
      }
    }
#pragma unroll 2
    for (int i = 0; i < C::MINE; ++i) {
      const int j = j0 + i, row = j * C::RPI + lrow;
      int in;
      const int pg = place(ku, row, &in);
      const int ck = lc ^ k_swz<RB>(row), cv = lc ^ v_swz<RB, BF16>(row);
      const char* kp = kb + ((int64_t)pg * k_p + (int64_t)in * p.k_t) * ES + 16 * ck;
      const char* vp = vb + ((int64_t)pg * v_p + (int64_t)in * p.v_t) * ES + 16 * cv;
      kp = pg >= 0 ? kp : reinterpret_cast<const char*>(&kZeroPiece);
      vp = pg >= 0 ? vp : reinterpret_cast<const char*>(&kZeroPiece);
      if (ck < npieces) load_lds16(kp, base + j * 1024);
      if (cv < npieces) load_lds16(vp, base + C::TILE + j * 1024);
    }
    return false;
  };
  if (p.D < C::DP) {  // pieces behind the head's end: never loaded, zeros
    for (int i = lane; i < C::LDS / NW / 16; i += 64) *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(mine + 16 * i) = u32x4{0u, 0u, 0u, 0u};
    if constexpr (SHARE) __syncthreads();
  }

  // One tile: S = K Q^T, the weights, O += V^T P^T.  Pieces are read from LDS
  // kAhead products before they are needed, the first of V behind the weights
  // (a read takes as long as two products, and one wave a SIMD hides nothing).
  constexpr int kAhead = RB < 1024 ? 4 : 2, VF = BF16 ? 2 * DB : 16 * DB;  // VF: pieces of V
  static_assert(C::STEPS >= kAhead && VF >= kAhead, "pieces");
  auto unit = [&](auto masked_, attn_lds stage, int ku, uint32_t there) {
    constexpr bool masked = decltype(masked_)::value;
    const attn_lds lk = stage, lv = stage + C::TILE;
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
    f32x16 s[QG];
#pragma unroll
    for (int g = 0; g < QG; ++g) s[g] = f32x16{};
#pragma unroll
    for (int t = 0; t < C::STEPS; ++t) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < QG; ++g) {
        s[g] = attn_mfma<BF16>(kf[t % kAhead], QREG ? qf[g][QREG ? t : 0] : qa[t % kAhead], s[g]);
      }
      if (t + kAhead < C::STEPS) {
        kf[t % kAhead] = at.key(lk, t + kAhead);
        if constexpr (!QREG) qa[t % kAhead] = read_query(t + kAhead);
      } else read_value(t + kAhead - C::STEPS);
    }
    __builtin_amdgcn_sched_barrier(0);
    u32x4 pb[QG][2];
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      if constexpr (masked) {
        uint32_t see = there;
        if constexpr (PROMPT) see &= p.causal ? upto32(qi[g], ku) : 0xffffffffu;
        else see &= seen32(row_sees[g], ku - context);
        see >>= 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[g][i] = see >> (8 * (i >> 2) + (i & 3)) & 1u ? s[g][i] : -INFINITY;
      }
      float mx = fmaxf(s[g][0], s[g][1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2) mx = fmaxf(fmaxf(mx, s[g][i]), s[g][i + 1]);
      mx *= p.c;
      if (__any(mx > st[g].m + kSlack)) {
        const float m = fmaxf(st[g].m, fmaxf(mx, __shfl_xor(mx, 32)));
        const float a = m == -INFINITY ? 1.f : exp2f(st[g].m - m);
        st[g].m = m;
        st[g].l *= a;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[g][d][i] *= a;
      }
      const float m = st[g].m == -INFINITY ? 0.f : st[g].m;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[g][i] = __builtin_amdgcn_exp2f(fmaf(s[g][i], p.c, -m));
      if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pb[g][i / 4][i % 4] = pack_bf16x2(s[g][2 * i], s[g][2 * i + 1]);
          st[g].l = add_pair(pb[g][i / 4][i % 4], st[g].l);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) st[g].l += s[g][i];
      }
    }
#pragma unroll
    for (int f = 0; f < VF; ++f) {
      __builtin_amdgcn_sched_barrier(0);
      u32x4 v = vf[f % kAhead];
      if constexpr (masked) {
#pragma unroll
        for (int w = 0; w < (BF16 ? 4 : 1); ++w) v[w] = scrub<BF16>(v[w], bad);
      }
#pragma unroll
      for (int g = 0; g < QG; ++g) {
        if constexpr (BF16) o[g][f % DB] = attn_mfma<true>(v, pb[g][f / DB], o[g][f % DB]);
        else o[g][f % DB] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v.x), s[g][f / DB], o[g][f % DB], 0, 0, 0);
      }
      if (f + kAhead < VF) read_value(f + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  // Whole tiles that every row sees, up to the first that is not; then the
  // others, masked.  Two loops: in one, the sums of 64 rows were copied between
  // the files of registers for each tile (380 moves).
  constexpr int STEP = SHARE ? 32 : 32 * NW;  // from a tile of the wave to its next
  int ku = kbeg + (SHARE ? 0 : 32 * wave);
  bool whole = false;
  attn_lds cur = mine, nxt = mine + (C::STAGES - 1) * C::STAGE;
  int issued = 0;       // SHARE: tiles whose loads are on their way or done,
  uint32_t wholes = 0;  // and which of the last 32 are whole
  auto issue_next = [&] {
    const int at = kbeg + 32 * issued;
    if (at >= kend) return;
    const uint32_t bit = 1u << (issued & 31);
    wholes = issue(at, (attn_lds)lds + issued % C::STAGES * C::STAGE) ? wholes | bit : wholes & ~bit;
    ++issued;
  };
  if constexpr (SHARE) {
    for (int i = 0; i < C::STAGES - 1; ++i) issue_next();
    whole = wholes & 1;
  } else if (C::STAGES > 1 && ku < kend) {
    whole = issue(ku, cur);
  }
  // Loads of tiles ahead; returns with the one at ku there, as `cur`.  The value: whether the next is whole.
  auto advance = [&]() -> bool {
    bool next_whole = false;
    if constexpr (SHARE) {
      const int t = (ku - kbeg) / 32;
      if (issued - t == C::STAGES - 1) wait_loads<(C::STAGES - 2) * 2 * C::MINE>();
      else wait_loads<0>();
      // Every wave's part of tile t is there, and every wave is done with tile t - 1, whose place is filled again.
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      issue_next();
      cur = (attn_lds)lds + t % C::STAGES * C::STAGE;
      next_whole = wholes >> ((t + 1) & 31) & 1;
    } else if constexpr (C::STAGES == 1) {
      next_whole = issue(ku, cur);
      wait_loads<0>();
    } else if (ku + STEP < kend) {
      next_whole = issue(ku + STEP, nxt);
      wait_loads<(2 * C::LOADS < 63 ? 2 * C::LOADS : 63)>();
    } else {
      wait_loads<0>();
    }
    return next_whole;
  };
  auto swap = [&] {
    const attn_lds t = cur;
    cur = nxt;
    nxt = t;
  };
  if constexpr (RB < 1024)  // (else two copies of a tile's code do not fit the registers)
    for (; ku + 31 < context && ku + 31 < kend; ku += STEP) {
      if (C::STAGES > 1 && !whole) break;
      const bool next_whole = advance();
      if (C::STAGES == 1 && !next_whole) break;  // loaded again below
      unit(std::false_type{}, cur, ku, 0xffffffffu);
      whole = next_whole;
      if constexpr (!SHARE) swap();
    }
  const int masked_from = ku;
  for (; ku < kend; ku += STEP) {
    advance();
    int in;
    unit(std::true_type{}, cur, ku, (uint32_t)__ballot(place(ku, col, &in) >= 0));
    if constexpr (!SHARE) swap();
  }

  // Each wave's sums, scaled to the block's maximum, in its own LDS; then all
  // threads add the waves' in order.  Row r's 16-byte pieces are spread by r.
  constexpr int OP = C::DP / 4;  // pieces of a row of sums
  constexpr int OM = OP < 32 ? OP - 1 : 31;
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const float l = st[g].l + __shfl_xor(st[g].l, 32);
    if (half == 0) {
      stats[wave][32 * g + col][0] = st[g].m;
      stats[wave][32 * g + col][1] = l;
    }
  }
  __syncthreads();
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    float m = SHARE ? st[g].m : -INFINITY;
    if constexpr (!SHARE)
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, stats[w][32 * g + col][0]);
    const float a = st[g].m == -INFINITY ? 1.f : exp2f(st[g].m - m);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int piece = 8 * d + 2 * q + half;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[g][d][4 * q + e] * a;
        *reinterpret_cast<SVDMLP_ATTN_LDS f32x4*>(mine + ((32 * g + col) * OP + (piece ^ (col & OM))) * 16) = v;
      }
  }
  // Infinities and NaN among the values of the masked tiles were taken as
  // zeros, for the rows that do not see them; the rows that do get them here.
  if (__any(bad != 0)) {
    for (int kt = masked_from; kt < kend; kt += STEP)
      for (int key = kt; key < min(kt + 32, kend); ++key) {
        int in;
        const int pg = place(key, 0, &in);
        if (pg < 0) continue;
        const char* const vp = vb + ((int64_t)pg * v_p + (int64_t)in * p.v_t) * ES;
        auto value = [&](int e) -> uint32_t {
          return BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(vp)[e] << 16 : reinterpret_cast<const uint32_t*>(vp)[e];
        };
        bool any = false;
        for (int e = lane; e < p.D; e += 64) any |= not_finite<false>(value(e));
        if (!__any(any)) continue;
        for (int e = 0; e < p.D; ++e) {
          const uint32_t w = value(e);
          if (not_finite<false>(w) && half == 0)
#pragma unroll
            for (int g = 0; g < QG; ++g)
              if (sees(g, key)) {
                SVDMLP_ATTN_LDS float* const sum =
                    (SVDMLP_ATTN_LDS float*)(mine + ((32 * g + col) * OP + ((e >> 2) ^ (col & OM))) * 16) + (e & 3);
                *sum += __uint_as_float(w);
              }
        }
      }
  }
  __syncthreads();
  const __amdgpu_buffer_rsrc_t sums = part_of(p, b, PROMPT ? 0 : p.D), ml = part_of(p, b, PROMPT ? 0 : 2);
  for (int i = threadIdx.x; i < C::ROWS * OP; i += 64 * NW) {
    const int rr = i / OP, piece = i % OP, r = r0 + rr;
    if (r >= rows || 4 * piece >= p.D) continue;
    float m = -INFINITY, l = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    const int wr = rr % C::WROWS;  // the row in its wave, or in each
    const attn_lds at = (attn_lds)lds + (wr * OP + (piece ^ (wr & OM))) * 16;
    if constexpr (SHARE) {
      const int w = rr / C::WROWS;
      m = stats[w][wr][0], l = stats[w][wr][1];
      v = *reinterpret_cast<SVDMLP_ATTN_LDS f32x4*>(at + w * (C::LDS / NW));
    } else {
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, stats[w][wr][0]);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = stats[w][wr][0];
        l += mw == -INFINITY ? stats[w][wr][1] : stats[w][wr][1] * exp2f(mw - m);
        v += *reinterpret_cast<SVDMLP_ATTN_LDS f32x4*>(at + w * (C::LDS / NW));
      }
    }
    const int t = r / G, h = hk * G + r - t * G;
    if (PROMPT || used == 1) {
      v *= inverse_sum(l);
      store4<BF16>(p.out, (int64_t)b * p.o_b + (int64_t)(start + t) * p.o_t + (int64_t)h * p.o_h + 4 * piece, v);
    } else if (SHARE) {
      const int64_t row = ((int64_t)at_chunk * p.n + t) * p.Hq + h;
      *reinterpret_cast<f32x4*>(p.part + row * p.D + 4 * piece) = v;
      if (piece == 0) *reinterpret_cast<f32x2*>(p.part + (int64_t)p.chunks * p.n * p.Hq * p.D + 2 * row) = f32x2{m, l};
    } else {
      const int row = (t * p.Hq + h) * p.splits + split;
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), sums, (row * p.D + 4 * piece) * 4, 0, kDevice);
      if (piece == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, ml, row * 8, 0, kDevice);
    }
  }
  if (PROMPT || SHARE || used == 1) return;

  // The last block to get here joins the chunks.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's sums are out
  __syncthreads();
  int* const counter = p.counters + ((int64_t)b * p.Hk + hk) * rtiles + rt;
  int last = 0;
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == used - 1;
    if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // as the next call finds it
    stats[0][0][0] = last ? 1.f : 0.f;
  }
  __syncthreads();
  if (stats[0][0][0] == 0.f) return;
  SVDMLP_ATTN_LDS float* const weight = (SVDMLP_ATTN_LDS float*)(attn_lds)lds;  // [row][kSplitsMost]
  const int nrows = min(C::ROWS, rows - r0);
  auto part_row = [&](int rr) -> int {
    const int r = r0 + rr, t = r / G;
    return (t * p.Hq + hk * G + r - t * G) * p.splits;
  };
  // An item: 16 bytes of a row's sums.  Few items are shared by `parts` threads
  // each, a thread taking every parts-th chunk, kJoin in flight.
  constexpr int NT = 64 * NW;
  const int dp = p.D / 4, items = nrows * dp;
  int parts = 1;
  while (2 * parts * items <= NT && parts < 8) parts *= 2;
  const int lanes = NT / parts, part = threadIdx.x / lanes;
  u32x4 x[kJoin];
  auto fetch = [&](int item, int k0) {  // behind the last chunk zeros
    const int rr = item / dp, at0 = (part_row(rr) * p.D + 4 * (item - rr * dp)) * 4;
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      const int s = part + parts * (k0 + k);
      x[k] = __builtin_amdgcn_raw_buffer_load_b128(sums, s < used ? (uint32_t)(at0 + s * p.D * 4) : 0x80000000u, 0, kDevice);
    }
  };
  int item = threadIdx.x % lanes;
  if (item < items) fetch(item, 0);
  // Meanwhile the chunks' weights: a wave takes a row, its lanes the chunks'
  // maxima and sums.
  for (int rr = wave; rr < nrows; rr += NW) {
    f32x2 v = {-INFINITY, 0.f};
    if (lane < used) v = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(ml, (part_row(rr) + lane) * 8, 0, kDevice));
    float m = v.x;
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float a = v.x == -INFINITY ? 1.f : exp2f(v.x - m);
    float l = v.y * a;
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    weight[rr * kSplitsMost + lane] = lane < used ? a * inverse_sum(l) : 0.f;
  }
  __syncthreads();
  auto gather = [&](int item, bool fetched) -> f32x4 {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; part + parts * k0 < used; k0 += kJoin) {
      if (!fetched || k0 > 0) fetch(item, k0);
#pragma unroll
      for (int k = 0; k < kJoin; ++k)
        v += __builtin_bit_cast(f32x4, x[k]) * weight[item / dp * kSplitsMost + min(part + parts * (k0 + k), kSplitsMost - 1)];
    }
    return v;
  };
  auto write = [&](int item, f32x4 v) {
    const int rr = item / dp, r = r0 + rr, t = r / G, h = hk * G + r - t * G;
    store4<BF16>(p.out, (int64_t)b * p.o_b + (int64_t)t * p.o_t + (int64_t)h * p.o_h + 4 * (item - rr * dp), v);
  };
  if (parts > 1) {  // one item a thread
    SVDMLP_ATTN_LDS f32x4* const others = (SVDMLP_ATTN_LDS f32x4*)((attn_lds)lds + C::ROWS * kSplitsMost * 4);
    static_assert(C::ROWS * kSplitsMost * 4 + NT * 16 <= C::LDS || PROMPT, "weights and the parts' sums fit the stages");
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (item < items) v = gather(item, true);
    others[threadIdx.x] = v;
    __syncthreads();
    if (part > 0 || item >= items) return;
    for (int q = 1; q < parts; ++q) v += others[threadIdx.x + q * lanes];
    write(item, v);
    return;
  }
  bool fetched = true;
  for (; item < items; item += NT) {
    write(item, gather(item, fetched));
    fetched = false;
  }
}

// The chunks' sums of blocks that share their tiles, joined: a wave a row, a lane
// two elements.  (Joined by the last block, 128 rows of 8 chunks took 37 us.)
template <bool BF16>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheParams p, int rtiles) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  const int heads = p.n * p.Hq, b = (int)(row / heads), th = (int)(row - (int64_t)b * heads);
  if (b >= p.B) return;
  const int chunk = shared_chunk(p, rtiles, lane), used = chunks_of(held(p, b), chunk);
  if (used == 1) return;
  int first = b * p.splits;
  if (p.chunk < p.chunk_most) {
    first = lane < b ? chunks_of(held(p, lane), chunk) : 0;
    for (int o = 32; o > 0; o >>= 1) first += __shfl_xor(first, o);
  }
  const int64_t at = (int64_t)__builtin_amdgcn_readfirstlane(first) * heads + th;
  const float* const ml = p.part + (int64_t)p.chunks * heads * p.D + 2 * at;
  f32x2 v = {-INFINITY, 0.f};
  if (lane < used) v = *reinterpret_cast<const f32x2*>(ml + (int64_t)lane * heads * 2);
  float m = v.x;
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float a = v.x == -INFINITY ? 1.f : exp2f(v.x - m);
  float l = v.y * a;
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  const float weight = lane < used ? a * inverse_sum(l) : 0.f;
  if (2 * lane >= p.D) return;
  const float* const sums = p.part + at * p.D + 2 * lane;
  f32x2 o = {0.f, 0.f};
  for (int s0 = 0; s0 < used; s0 += 8) {
    f32x2 x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = *reinterpret_cast<const f32x2*>(sums + (int64_t)min(s0 + k, used - 1) * heads * p.D);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s0 + k < used) o += x[k] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), s0 + k));
  }
  const int t = th / p.Hq, h = th - t * p.Hq;
  const int64_t to = (int64_t)b * p.o_b + (int64_t)t * p.o_t + (int64_t)h * p.o_h + 2 * lane;
  if constexpr (BF16) *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + to) = pack_bf16x2(o.x, o.y);
  else *reinterpret_cast<f32x2*>(static_cast<float*>(p.out) + to) = o;
}

}  // namespace svdmlp
