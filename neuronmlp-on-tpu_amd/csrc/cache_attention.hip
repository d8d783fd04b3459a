// Attention of the n new tokens of each sequence onto a paged cache that holds
// the sequence's context and them: token i sees every key of the context, and
// of the new ones those that its row of the tree names (no tree: the ones up to
// itself).  n = 1 is the decode step.
//
// Bound by the cache's bytes, read once for all heads of a group and all new
// tokens (up to 32 * QG rows).  Nothing is shared between waves: each of a
// block's waves takes every NW-th tile of 32 keys of the block's chunk through
// LDS of its own (direct loads, the next tile's in flight while one is
// computed), with no barrier in the loop, and their sums meet at the end.
// A long context is cut into chunks, one a block; a second launch joins their
// partial sums in the chunks' order (no atomics: the same bits every time).
#include <math.h>

#include <algorithm>

#include "attn.hpp"
#include "decoder.hpp"

namespace svdmlp {

namespace {

constexpr int kPagesMost = 1024;  // whole pages of a chunk: their numbers lie in LDS

template <bool BF16_, int DP_, int QG_>
struct CacheCfg {
  static constexpr bool BF16 = BF16_;
  static constexpr int DP = DP_, QG = QG_;
  static constexpr int ES = BF16 ? 2 : 4;
  static constexpr int RB = DP * ES;
  static constexpr int PIECES = RB / 16;
  static constexpr int STEPS = RB / 32;
  static constexpr int NW = RB <= 256 ? 4 : RB == 512 ? 2 : 1;  // waves: two stages of two tiles each in 160 KB
  static constexpr int TILE = 32 * RB;
  static constexpr int STAGE = 2 * TILE;  // keys, values
  static constexpr int ROWS = 32 * QG;
  static constexpr int RPI = 64 / PIECES;        // rows a load
  static constexpr int LOADS = 32 / RPI;         // loads a tile, of keys and of values
  static_assert(2 * STAGE >= ROWS * DP * 4, "a wave's sums fit its stages");
};

// 16 bytes of zeros that lanes without a key load.
__device__ const u32x4 kZeroPiece = {0u, 0u, 0u, 0u};

__device__ __forceinline__ int held(const CacheParams& p, int b) {
  const int64_t cap = (int64_t)p.width * p.page;
  return (int)min((int64_t)max(p.lengths[b], 0), cap);
}

// Which of the 32 keys from `draft` keys after the context on a token sees,
// whose row of the tree is `row`: all of the context.
__device__ __forceinline__ uint32_t seen32(uint64_t row, int draft) {
  if (draft >= 64) return 0;
  if (draft >= 0) return (uint32_t)(row >> draft);
  if (draft <= -32) return 0xffffffffu;
  return (uint32_t)(row << -draft) | ((1u << -draft) - 1u);
}

template <class C>
__global__ __launch_bounds__(64 * C::NW, 1) void cache_kernel(CacheParams p) {
  constexpr bool BF16 = C::BF16;
  constexpr int ES = C::ES, RB = C::RB, QG = C::QG, DB = C::DP / 32, NW = C::NW;
  __shared__ __attribute__((aligned(1024))) char lds[NW * 2 * C::STAGE];
  __shared__ float stats[NW][C::ROWS][2];
  __shared__ int ids[kPagesMost + 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int G = p.Hq / p.Hk;
  const int rows = p.n * G;
  const int rtiles = (rows + C::ROWS - 1) / C::ROWS;
  int id = blockIdx.x;
  const int hk = id % p.Hk;
  id /= p.Hk;
  const int rt = id % rtiles;
  id /= rtiles;
  const int b = id % p.B, split = id / p.B;
  const int len = held(p, b);
  const int kbeg = split * p.chunk, kend = min(len, kbeg + p.chunk);
  if (kbeg >= kend && p.splits > 1) return;  // the join knows from the length
  const int context = len - p.n;             // keys that every row sees

  // The chunk's pages, and the queries.
  const int pg0 = kbeg / p.page;
  const int npages = min(p.width - pg0, (int)min((int64_t)p.chunk + p.page - 1, (int64_t)kPagesMost * p.page) / p.page + 1);
  for (int i = threadIdx.x; i < npages; i += 64 * NW) ids[i] = p.table[(int64_t)b * p.table_b + pg0 + i];
  // Heads of over 128 elements leave no registers for Q: its pieces are read
  // again (from the caches) for every tile.
  constexpr bool QREG = C::DP < 256;
  u32x4 qf[QG][QREG ? C::STEPS : 1];
  const char* qptr[QG];
  int qi[QG];  // which of the new tokens
  const int npieces = p.D * ES / 16;
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const int r = min(rt * C::ROWS + 32 * g + col, rows - 1);  // rows behind the last repeat it, and are not stored
    qi[g] = r / G;
    qptr[g] = static_cast<const char*>(p.q) + ((int64_t)b * p.q_b + (int64_t)qi[g] * p.q_t + (int64_t)(hk * G + r - qi[g] * G) * p.q_h) * ES;
    if constexpr (QREG)
#pragma unroll
      for (int s = 0; s < C::STEPS; ++s) {
        const int c = 2 * s + half;
        qf[g][s] = c < npieces ? *reinterpret_cast<const u32x4*>(qptr[g] + 16 * c) : u32x4{0u, 0u, 0u, 0u};
      }
  }
  // Each row's 64 bits of the tree, where the chunk reaches the new tokens: a
  // lane reads one byte of a token's row, and a ballot gathers them.
  uint64_t row_sees[QG];
#pragma unroll
  for (int g = 0; g < QG; ++g) row_sees[g] = (2ull << qi[g]) - 1;  // a chain (token 63: all)
  if (p.tree && kend > context) {
    const uint8_t* const tree = p.tree + (int64_t)b * p.tree_b;
    const int first = rt * C::ROWS / G, last = min(rt * C::ROWS + C::ROWS - 1, rows - 1) / G;
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

  const attn_lds mine = (attn_lds)lds + wave * 2 * C::STAGE;
  const char* const kb = static_cast<const char*>(p.kc) + (int64_t)hk * p.k_h * ES;
  const char* const vb = static_cast<const char*>(p.vc) + (int64_t)hk * p.v_h * ES;
  const TileLane<RB, BF16> at(lane);
  const float per_page = 1.0f / (float)p.page;
  uint32_t bad = 0;

  // The row (page, place in it) of key ku + row; -1: of none.
  auto place = [&](int ku, int row, int* in) -> int {
    const int first = ku / p.page, x = ku - first * p.page + row;
    // x < page + 32: one division of small numbers, exact in 32 bits
    const int q = p.page >= 32 ? (x >= p.page) : (int)(((float)x + 0.5f) * per_page);
    *in = x - q * p.page;
    const int i = first + q - pg0;
    const int pg = ku + row < kend ? ids[i] : -1;
    return pg >= 0 && pg < p.pages ? pg : -1;
  };
  auto issue = [&](int ku, attn_lds stage) {
    const uint32_t base = (uint32_t)(uintptr_t)stage;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage's last reads are done
#pragma unroll
    for (int j = 0; j < C::LOADS; ++j) {
      const int row = j * C::RPI + lane / C::PIECES, c = lane % C::PIECES;
      int in;
      const int pg = place(ku, row, &in);
      const int ck = c ^ k_swz<RB>(row), cv = c ^ v_swz<RB, BF16>(row);
      const char* kp = kb + ((int64_t)pg * p.k_p + (int64_t)in * p.k_t) * ES + 16 * ck;
      const char* vp = vb + ((int64_t)pg * p.v_p + (int64_t)in * p.v_t) * ES + 16 * cv;
      kp = pg >= 0 && ck < npieces ? kp : reinterpret_cast<const char*>(&kZeroPiece);
      vp = pg >= 0 && cv < npieces ? vp : reinterpret_cast<const char*>(&kZeroPiece);
      load_lds16(kp, base + j * 1024);
      load_lds16(vp, base + C::TILE + j * 1024);
    }
  };

  int ku = kbeg + 32 * wave;
  attn_lds cur = mine, nxt = mine + C::STAGE;
  if (ku < kend) issue(ku, cur);
  for (; ku < kend; ku += 32 * NW) {
    if (ku + 32 * NW < kend) {
      issue(ku + 32 * NW, nxt);
      wait_loads<(2 * C::LOADS < 63 ? 2 * C::LOADS : 63)>();
    } else {
      wait_loads<0>();
    }
    const attn_lds lk = cur, lv = cur + C::TILE;
    const bool masked = ku + 31 >= context;
    int in;
    const uint32_t there = (uint32_t)__ballot(place(ku, col, &in) >= 0);  // keys that lie in a page of the cache
    f32x16 s[QG];
#pragma unroll
    for (int g = 0; g < QG; ++g)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[g][i] = 0.f;
#pragma unroll
    for (int t = 0; t < C::STEPS; ++t) {
      const u32x4 kf = at.key(lk, t);
#pragma unroll
      for (int g = 0; g < QG; ++g) {
        if constexpr (!QREG) {
          const int c = 2 * t + half;
          qf[g][0] = c < npieces ? *reinterpret_cast<const u32x4*>(qptr[g] + 16 * c) : u32x4{0u, 0u, 0u, 0u};
        }
        s[g] = attn_mfma<BF16>(kf, qf[g][QREG ? t : 0], s[g]);
      }
    }
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      if (masked || there != 0xffffffffu) {
        const uint32_t see = (there & seen32(row_sees[g], ku - context)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[g][i] = see >> (8 * (i >> 2) + (i & 3)) & 1u ? s[g][i] : -INFINITY;
      }
      float mx = s[g][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[g][i]);
      mx = fmaxf(mx, __shfl_xor(mx, 32)) * p.c;
      if (__any(mx > st[g].m + kSlack)) {
        const float m = fmaxf(st[g].m, mx);
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
      for (int i = 0; i < 16; ++i) {
        s[g][i] = __builtin_amdgcn_exp2f(fmaf(s[g][i], p.c, -m));
        st[g].l += s[g][i];
      }
    }
    if constexpr (BF16) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        u32x4 pb[QG];
#pragma unroll
        for (int g = 0; g < QG; ++g)
#pragma unroll
          for (int w = 0; w < 4; ++w) pb[g][w] = pack_bf16x2(s[g][8 * t + 2 * w], s[g][8 * t + 2 * w + 1]);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          u32x4 vf = at.values(lv, t, d);
          if (masked)
#pragma unroll
            for (int w = 0; w < 4; ++w) vf[w] = scrub<true>(vf[w], bad);
#pragma unroll
          for (int g = 0; g < QG; ++g) o[g][d] = attn_mfma<true>(vf, pb[g], o[g][d]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          uint32_t w = at.value(lv, i, d);
          if (masked) w = scrub<false>(w, bad);
#pragma unroll
          for (int g = 0; g < QG; ++g)
            o[g][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w), s[g][i], o[g][d], 0, 0, 0);
        }
    }
    const attn_lds swap = cur;
    cur = nxt;
    nxt = swap;
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
    float m = -INFINITY;
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
    for (int kt = kbeg + 32 * wave; kt < kend; kt += 32 * NW) {
      if (kt + 31 < context) continue;
      for (int key = kt; key < min(kt + 32, kend); ++key) {
        int in;
        const int pg = place(key, 0, &in);
        if (pg < 0) continue;
        const char* const vp = vb + ((int64_t)pg * p.v_p + (int64_t)in * p.v_t) * ES;
        for (int e = 0; e < p.D; ++e) {
          const uint32_t w = BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(vp)[e] << 16 : reinterpret_cast<const uint32_t*>(vp)[e];
          if (not_finite<false>(w) && half == 0)
#pragma unroll
            for (int g = 0; g < QG; ++g)
              if (seen32(row_sees[g], key - context) & 1u) {
                SVDMLP_ATTN_LDS float* const sum =
                    (SVDMLP_ATTN_LDS float*)(mine + ((32 * g + col) * OP + ((e >> 2) ^ (col & OM))) * 16) + (e & 3);
                *sum += __uint_as_float(w);
              }
        }
      }
    }
  }
  __syncthreads();
  const int64_t total = (int64_t)p.B * p.n * p.Hq;
  for (int i = threadIdx.x; i < C::ROWS * OP; i += 64 * NW) {
    const int rr = i / OP, piece = i % OP, r = rt * C::ROWS + rr;
    if (r >= rows || 4 * piece >= p.D) continue;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, stats[w][rr][0]);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = stats[w][rr][0];
      l += mw == -INFINITY ? stats[w][rr][1] : stats[w][rr][1] * exp2f(mw - m);
      v += *reinterpret_cast<SVDMLP_ATTN_LDS f32x4*>((attn_lds)lds + w * 2 * C::STAGE + (rr * OP + (piece ^ (rr & OM))) * 16);
    }
    const int t = r / G, h = hk * G + r - t * G;
    if (p.splits == 1) {
      v *= inverse_sum(l);
      store4<BF16>(p.out, (int64_t)b * p.o_b + (int64_t)t * p.o_t + (int64_t)h * p.o_h + 4 * piece, v);
    } else {
      const int64_t row = (((int64_t)b * p.n + t) * p.Hq + h) * p.splits + split;
      *reinterpret_cast<f32x4*>(p.part + row * p.D + 4 * piece) = v;
      if (piece == 0) *reinterpret_cast<f32x2*>(p.part + total * p.splits * p.D + 2 * row) = f32x2{m, l};
    }
  }
}

// Joins the chunks' partial sums: `per` groups of LPR lanes share a row, each
// takes every per-th chunk, and the first adds the groups' sums in order.
template <bool BF16, int LPR>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheParams p, int per) {
  constexpr int GROUPS = 256 / LPR;
  __shared__ f32x4 sums[GROUPS][LPR];
  const int group = threadIdx.x / LPR, piece = threadIdx.x % LPR, sub = group % per;
  const int64_t total = (int64_t)p.B * p.n * p.Hq;
  const int64_t row = (int64_t)blockIdx.x * (GROUPS / per) + group / per;
  const bool in = row < total && 4 * piece < p.D;
  const int64_t bt = row / p.Hq;
  const int h = (int)(row - bt * p.Hq), b = (int)(bt / p.n), t = (int)(bt - (int64_t)b * p.n);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  if (in) {
    const int used = min(p.splits, (int)(((int64_t)held(p, b) + p.chunk - 1) / p.chunk));
    const float* const part = p.part + row * p.splits * p.D + 4 * piece;
    const f32x2* const ml = reinterpret_cast<const f32x2*>(p.part + total * p.splits * p.D) + row * p.splits;
    float m = -INFINITY;
    for (int s = 0; s < used; ++s) m = fmaxf(m, ml[s].x);
    for (int s = 0; s < used; ++s) l += ml[s].y * (ml[s].x == -INFINITY ? 1.f : exp2f(ml[s].x - m));
    for (int s = sub; s < used; s += per)
      v += *reinterpret_cast<const f32x4*>(part + (int64_t)s * p.D) * (ml[s].x == -INFINITY ? 1.f : exp2f(ml[s].x - m));
  }
  if (per > 1) {
    sums[group][piece] = v;
    __syncthreads();
    if (sub) return;
    for (int g = 1; g < per; ++g) v += sums[group + g][piece];
  }
  if (in) store4<BF16>(p.out, (int64_t)b * p.o_b + (int64_t)t * p.o_t + (int64_t)h * p.o_h + 4 * piece, v * inverse_sum(l));
}

template <bool BF16, int DP, int QG>
hipError_t run(const CacheParams& p, hipStream_t st) {
  using C = CacheCfg<BF16, DP, QG>;
  const int64_t rtiles = ((int64_t)p.n * (p.Hq / p.Hk) + C::ROWS - 1) / C::ROWS;
  const int64_t blocks = rtiles * p.Hk * p.B * p.splits;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((cache_kernel<C>), dim3((unsigned)blocks), dim3(64 * C::NW), 0, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  constexpr int LPR = DP <= 64 ? 16 : DP <= 128 ? 32 : 64;
  int per = 1;
  while (per < 256 / LPR && per < p.splits) per *= 2;
  const int64_t total = (int64_t)p.B * p.n * p.Hq, rpb = 256 / LPR / per;
  hipLaunchKernelGGL((cache_join_kernel<BF16, LPR>), dim3((unsigned)((total + rpb - 1) / rpb)), dim3(256), 0, st, p, per);
  return hipGetLastError();
}

// 64 rows a wave where there are more than 32 and their sums fit the registers.
int row_groups(int n, int Hq, int Hk, int D, bool bf16) {
  return (int64_t)n * (Hq / Hk) > 32 && D <= (bf16 ? 128 : 64) ? 2 : 1;
}

}  // namespace

void plan_cache_attention(int B, int n, int Hq, int Hk, int D, bool bf16, int page, int64_t capacity, int cus,
                          int* splits, int* chunk) {
  const int64_t rows = (int64_t)n * (Hq / Hk), rt = 32 * row_groups(n, Hq, Hk, D, bf16);
  const int64_t base = (int64_t)B * Hk * ((rows + rt - 1) / rt);
  int64_t want = std::max<int64_t>(1, 16 * cus / base);
  int64_t c = ((capacity + want - 1) / want + 127) / 128 * 128;
  c = std::min(c, std::max<int64_t>(128, (int64_t)kPagesMost * page / 128 * 128));
  *chunk = (int)std::min<int64_t>(c, 0x7fffff80);
  *splits = (int)((capacity + *chunk - 1) / *chunk);
}

hipError_t launch_cache_attention(const CacheParams& p, bool bf16, hipStream_t st) {
  if (p.B <= 0 || p.n <= 0) return hipSuccess;
  const bool two = row_groups(p.n, p.Hq, p.Hk, p.D, bf16) == 2;
  if (bf16) {
    if (p.D <= 64) return two ? run<true, 64, 2>(p, st) : run<true, 64, 1>(p, st);
    if (p.D <= 128) return two ? run<true, 128, 2>(p, st) : run<true, 128, 1>(p, st);
    return run<true, 256, 1>(p, st);
  }
  if (p.D <= 64) return two ? run<false, 64, 2>(p, st) : run<false, 64, 1>(p, st);
  if (p.D <= 128) return run<false, 128, 1>(p, st);
  return run<false, 256, 1>(p, st);
}

}  // namespace svdmlp
