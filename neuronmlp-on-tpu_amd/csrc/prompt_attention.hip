// Attention of packed sequences onto themselves, O = softmax(c Q K^T + mask) V,
// causal or not; query head h reads key/value head h / (Hq / Hk).
//
// A block takes some rows of one key/value head and sequence (row = token * G +
// head of the group: the group's heads share every key and value that the block
// loads) and walks the keys in tiles through LDS, one pass, with the running
// maximum and sum.  Three kernels: prompt_pipe_kernel (bf16, heads up to 128, many
// rows), the one of wave_attention.hpp (few rows, many short sequences, fp32),
// prompt_kernel (heads up to 256).
#include <math.h>

#include <algorithm>

#include "pipe_attention.hpp"
#include "wave_attention.hpp"

namespace svdmlp {

namespace {

// The kernel of heads over 128: four waves of 32 rows share tiles of 32 keys in
// LDS; the registers' loads of the next tile wait while one is computed.  Bound by
// its LDS reads (a piece feeds one product) and registers: 8 heads of 256, 8 of
// keys, 4000 tokens causal 247 us, 265 TFLOP/s (6 us of it for the sum of the
// weights as rounded).
template <bool BF16_>
struct PromptCfg {
  static constexpr bool BF16 = BF16_;
  static constexpr int DP = 256;  // head elements held (D rounded up)
  static constexpr int ES = BF16 ? 2 : 4;
  static constexpr int RB = DP * ES;         // bytes of a key row in LDS
  static constexpr int PIECES = RB / 16;
  static constexpr int STEPS = RB / 32;      // 32-byte steps of the head
  static constexpr int KB = 32;              // keys a tile
  static constexpr int BM = 128;             // rows a block
  static constexpr int TILE = KB * RB;
};

template <class C>
__global__ __launch_bounds__(256, 1) void prompt_kernel(PromptParams p) {
  constexpr bool BF16 = C::BF16;
  constexpr int ES = C::ES, RB = C::RB, KB = C::KB, DB = C::DP / 32;
  __shared__ __attribute__((aligned(1024))) char lds[2 * C::TILE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
  const int G = p.Hq / p.Hk;

  RowTile where;
  if (!find_rows(p.cu, p.T, p.B, p.Hk, G, C::BM, lane, where)) return;
  const int hk = where.hk, start = where.start, len = where.len, row0 = where.row0, rows = len * G;
  const int tok_last = min(len - 1, (row0 + C::BM - 1) / G);
  const int tok_first = row0 / G;
  const int nkeys = p.causal ? tok_last + 1 : len;

  // Q: lane half h holds the 16-byte piece 2 s + h of its row at step s.
  u32x4 qf[C::STEPS];
  const int npieces = p.D * ES / 16;
  const int r = row0 + wave * 32 + col;
  const bool in = r < rows;
  const int tok = in ? r / G : 0;
  const char* const qp = static_cast<const char*>(p.q) + ((int64_t)(start + tok) * p.q_t + (int64_t)(hk * G + (in ? r - tok * G : 0)) * p.q_h) * ES;
#pragma unroll
  for (int s = 0; s < C::STEPS; ++s) {
    const int c = 2 * s + half;
    qf[s] = in && c < npieces ? *reinterpret_cast<const u32x4*>(qp + 16 * c) : u32x4{0u, 0u, 0u, 0u};
  }

  f32x16 o[DB];
  RowState st = {-INFINITY, 0.f};
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  const char* const kbase = static_cast<const char*>(p.k) + ((int64_t)start * p.k_t + (int64_t)hk * p.k_h) * ES;
  const char* const vbase = static_cast<const char*>(p.v) + ((int64_t)start * p.v_t + (int64_t)hk * p.v_h) * ES;
  const attn_lds lk = (attn_lds)lds, lv = lk + C::TILE;
  const TileLane<RB, BF16> at(lane);
  uint32_t bad = 0;

  // The next tile's pieces wait in registers while one is computed.
  constexpr int PER = KB * C::PIECES / 256;
  u32x4 kv[PER], vv[PER];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = threadIdx.x + 256 * j, row = i / C::PIECES, c = i % C::PIECES;
      const bool in = k0 + row < nkeys && c < npieces;
      kv[j] = in ? *reinterpret_cast<const u32x4*>(kbase + (int64_t)(k0 + row) * p.k_t * ES + 16 * c) : u32x4{0u, 0u, 0u, 0u};
      vv[j] = in ? *reinterpret_cast<const u32x4*>(vbase + (int64_t)(k0 + row) * p.v_t * ES + 16 * c) : u32x4{0u, 0u, 0u, 0u};
    }
  };
  fetch(0);
  for (int k0 = 0; k0 < nkeys; k0 += KB) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = threadIdx.x + 256 * j, row = i / C::PIECES, c = i % C::PIECES;
      *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(lk + row * RB + ((c ^ k_swz<RB>(row)) << 4)) = kv[j];
      *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(lv + row * RB + ((c ^ v_swz<RB, BF16>(row)) << 4)) = vv[j];
    }
    __syncthreads();
    if (k0 + KB < nkeys) fetch(k0 + KB);
    const bool masked = p.causal && k0 + KB - 1 > tok_first;  // not every row sees every key
    const bool edge = masked || k0 + KB > nkeys;
    f32x16 s = {};
#pragma unroll
    for (int t = 0; t < C::STEPS; ++t) s = attn_mfma<BF16>(at.key(lk, t), qf[t], s);
    if (edge) {
      const int last = p.causal ? min(tok, nkeys - 1) : nkeys - 1;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = k0 + 8 * (i >> 2) + 4 * half + (i & 3);
        s[i] = key <= last ? s[i] : -INFINITY;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32)) * p.c;
    if (__any(mx > st.m + kSlack)) {
      const float m = fmaxf(st.m, mx);
      const float a = m == -INFINITY ? 1.f : exp2f(st.m - m);
      st.m = m;
      st.l *= a;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= a;
    }
    const float m = st.m == -INFINITY ? 0.f : st.m;
    float pf[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      pf[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, -m));
      if constexpr (!BF16) st.l += pf[i];
    }
    if constexpr (BF16) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {  // 16 keys each
        u32x4 pb;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          pb[w] = pack_bf16x2(pf[8 * t + 2 * w], pf[8 * t + 2 * w + 1]);
          st.l = add_pair(pb[w], st.l);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          u32x4 vf = at.values(lv, t, d);
          if (masked)
#pragma unroll
            for (int w = 0; w < 4; ++w) vf[w] = scrub<true>(vf[w], bad);
          o[d] = attn_mfma<true>(vf, pb, o[d]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          uint32_t w = at.value(lv, i, d);
          if (masked) w = scrub<false>(w, bad);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w), pf[i], o[d], 0, 0, 0);
        }
    }
  }

  const float inv = inverse_sum(st.l + __shfl_xor(st.l, 32));
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] *= inv;
  // Infinities and NaN among the values of the masked tiles were taken as
  // zeros, for the rows that do not see them; the rows that do get them here.
  if (__any(bad != 0)) {
    for (int key = (tok_first + 1) / KB * KB; key < nkeys; ++key) {
      const char* const vp = vbase + (int64_t)key * p.v_t * ES;
      const uint32_t see = key <= tok ? 0xffffffffu : 0u;
      int D = p.D;
      asm volatile("" : "+s"(D));  // its comparisons stay in the loop: hoisted, they spill
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int e = 32 * d + 8 * (i >> 2) + 4 * half + (i & 3);
          const uint32_t w = e >= D ? 0u : BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(vp)[e] << 16 : reinterpret_cast<const uint32_t*>(vp)[e];
          o[d][i] += __uint_as_float(w & not_finite<false>(w) & see);
        }
    }
  }
  if (!in) return;
  const int64_t op = (int64_t)(start + tok) * p.o_t + (int64_t)(hk * G + (r - tok * G)) * p.o_h;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int e = 32 * d + 8 * b + 4 * half;
      if (e < p.D) store4<BF16>(p.out, op + e, f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]});
    }
}

// The bf16 kernel for many rows (the walk: pipe_attention.hpp).
// Bound by the matrix unit: 16384 tokens of 32 heads of 128, causal, 1.90 ms,
// 1.16 PFLOP/s (a library product of 8192^3: 1.24); 17 packed prompts of 8191
// tokens 95 us, where the diagonal's tiles and the blocks' starts weigh most.
template <class C>
__global__ __launch_bounds__(256, 1) void prompt_pipe_kernel(PromptParams p) {
  constexpr int RB = C::RB, QG = C::QG, KB = C::KB, DB = C::DP / 32;
  __shared__ __attribute__((aligned(1024))) char lds[C::NS * C::STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int G = p.Hq / p.Hk;
  RowTile rt;
  if (!find_rows(p.cu, p.T, p.B, p.Hk, G, C::BM, lane, rt)) return;
  const int row0 = rt.row0, rows = rt.len * G;
  const int tok_last = min(rt.len - 1, (row0 + C::BM - 1) / G), tok_first = row0 / G;
  const int nkeys = p.causal ? tok_last + 1 : rt.len;
  const int shared = p.causal ? tok_first + 1 : rt.len;  // keys that every row sees
  const int tiles = (nkeys + KB - 1) / KB, full = shared / KB;
  const int npieces = p.D / 8;

  const attn_lds base = (attn_lds)lds;
  const char* const kb = static_cast<const char*>(p.k) + ((int64_t)rt.start * p.k_t + (int64_t)rt.hk * p.k_h) * 2;
  const char* const vb = static_cast<const char*>(p.v) + ((int64_t)rt.start * p.v_t + (int64_t)rt.hk * p.v_h) * 2;
  // This wave's loads of a tile: rows wave * LOADS * RPL .. of keys (of tile tk)
  // and of values (of tile tv).  In whole tiles a lane's offsets are the same
  // every time; in the last one rows behind the last key repeat it (masked).
  uint32_t koff[C::LOADS], voff;
  const int lrow = wave * C::LOADS * C::RPL + lane / C::PIECES, lc = lane % C::PIECES;
  bool kin[C::LOADS];
  const int vc = lc ^ v_swz<RB, true>(lrow);
#pragma unroll
  for (int j = 0; j < C::LOADS; ++j) {
    const int row = lrow + j * C::RPL, c = lc ^ k_swz<RB>(row);
    koff[j] = (uint32_t)(row * (int)p.k_t * 2 + 16 * c);
    kin[j] = c < npieces;
  }
  voff = (uint32_t)(lrow * (int)p.v_t * 2 + 16 * vc);
  const bool vin = vc < npieces;
  auto issue_keys = [&](int t) {
    if (t >= tiles) return;
    const uint32_t at = (uint32_t)(uintptr_t)(base + (t % C::NS) * C::STAGE) + wave * C::LOADS * 1024;
    const char* const kt = kb + (int64_t)t * KB * p.k_t * 2;
    if ((t + 1) * KB <= nkeys) {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j)
        if (kin[j]) load_lds16(kt, koff[j], at + j * 1024);
    } else {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) {
        const int row = lrow + j * C::RPL, r = min(row, nkeys - 1 - t * KB);
        if (kin[j]) load_lds16(kt, (uint32_t)(r * (int)p.k_t * 2 + 16 * (lc ^ k_swz<RB>(row))), at + j * 1024);
      }
    }
  };
  auto issue_values = [&](int t) {
    if (t >= tiles) return;
    const uint32_t at = (uint32_t)(uintptr_t)(base + (t % C::NS) * C::STAGE) + C::TILE + wave * C::LOADS * 1024;
    const char* const vt = vb + (int64_t)t * KB * p.v_t * 2;
    if ((t + 1) * KB <= nkeys) {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j)
        if (vin) load_lds16(vt + (int64_t)j * C::RPL * p.v_t * 2, voff, at + j * 1024);
    } else {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) {
        const int r = min(lrow + j * C::RPL, nkeys - 1 - t * KB);
        if (vin) load_lds16(vt, (uint32_t)(r * (int)p.v_t * 2 + 16 * vc), at + j * 1024);
      }
    }
  };
  // Zeros where a head is shorter than its place (never loaded), and in the
  // last stage's values, which the first step multiplies by zero weights.
  if (p.D < C::DP) {
    for (int i = threadIdx.x; i < C::NS * C::STAGE / 16; i += 256) *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(base + 16 * i) = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  } else {
    for (int i = threadIdx.x; i < C::UNIT / 16; i += 256)
      *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(base + (C::NS - 1) * C::STAGE + C::TILE + C::UNIT + 16 * i) = u32x4{0u, 0u, 0u, 0u};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before the first barrier
  }
  issue_keys(0);
  issue_keys(1);
  issue_values(0);
  issue_keys(2);
  issue_values(1);

  u32x4 qf[QG][C::STEPS];
  int tok[QG];
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const int r = min(row0 + (wave * QG + g) * 32 + col, rows - 1);  // rows behind the last repeat it, and are not stored
    tok[g] = r / G;
    const char* qp = static_cast<const char*>(p.q) + ((int64_t)(rt.start + tok[g]) * p.q_t + (int64_t)(rt.hk * G + r - tok[g] * G) * p.q_h) * 2;
#pragma unroll
    for (int s = 0; s < C::STEPS; ++s) {
      const int c = 2 * s + half;
      qf[g][s] = c < npieces ? *reinterpret_cast<const u32x4*>(qp + 16 * c) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  PipeWave<C> w(qf, lane, p.c);
  // Before tile t: the keys of tile t + 1 and the values of tile t are there for
  // every wave (they were asked for two tiles ago; what was asked for one tile
  // ago may still be on its way), and every wave is done with the keys of tile
  // t - 1 and the values of tile t - 2, whose places are filled again.
  auto arrive = [&](int t) {
    if (t + 2 < tiles) wait_loads<2 * C::LOADS>();
    else wait_loads<0>();
    asm volatile("s_barrier" ::: "memory");
    issue_keys(t + 3);
    issue_values(t + 2);
  };

  int t = 0;
  if (full > 0) w.whole_tiles(base, full, t, false, arrive, [](int) {});
  for (; t < tiles; ++t) {
    arrive(t);
    const attn_lds cur = base + (t % C::NS) * C::STAGE;
#pragma unroll 1
    for (int u = 0; u < 2; ++u) {
      const int k0 = t * KB + 32 * u;
      const int seen = p.causal ? min((row0 + (wave + 1) * QG * 32 - 1) / G, nkeys - 1) : nkeys - 1;  // the wave's last key
      if (k0 > seen) break;
      f32x16 s[QG];
      u32x4 pb[QG][2];
      float scale[QG];
      const attn_lds vt = cur + C::TILE + u * C::UNIT;
      w.scores(cur + u * C::UNIT, vt, s);
#pragma unroll
      for (int g = 0; g < QG; ++g) {
        const int last = (p.causal ? tok[g] : nkeys - 1) - k0 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[g][i] = 8 * (i >> 2) + (i & 3) <= last ? s[g][i] : -INFINITY;
      }
      if (w.reference(s, scale)) w.rescale(scale);
      w.weights(s, pb);
      w.values(vt, pb, true);
    }
  }

#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const float inv = inverse_sum(w.l[g] + __shfl_xor(w.l[g], 32));
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) w.o[g][d][i] *= inv;
  }
  // Infinities and NaN among the values of the plain loop were taken as
  // zeros, for the rows that do not see them; the rows that do get them here.
  if (__any(w.bad != 0)) {
    for (int key = full * KB; key < nkeys; ++key) {
      const uint16_t* const vp = reinterpret_cast<const uint16_t*>(vb + (int64_t)key * p.v_t * 2);
      uint32_t see[QG];
#pragma unroll
      for (int g = 0; g < QG; ++g) see[g] = !p.causal || key <= tok[g] ? 0xffffffffu : 0u;
      int D = p.D;
      asm volatile("" : "+s"(D));  // its comparisons stay in the loop: hoisted, they spill
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int e = 32 * d + 8 * (i >> 2) + 4 * half + (i & 3);
          const uint32_t x = e >= D ? 0u : (uint32_t)vp[e] << 16, mask = not_finite<false>(x);
#pragma unroll
          for (int g = 0; g < QG; ++g) w.o[g][d][i] += __uint_as_float(x & mask & see[g]);
        }
    }
  }
#pragma unroll
  for (int g = 0; g < QG; ++g) {
    const int r = row0 + (wave * QG + g) * 32 + col;
    if (r >= rows) continue;
    const int64_t op = (int64_t)(rt.start + tok[g]) * p.o_t + (int64_t)(rt.hk * G + (r - tok[g] * G)) * p.o_h;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int e = 32 * d + 8 * b + 4 * half;
        if (e < p.D) store4<true>(p.out, op + e, f32x4{w.o[g][d][4 * b], w.o[g][d][4 * b + 1], w.o[g][d][4 * b + 2], w.o[g][d][4 * b + 3]});
      }
  }
}

template <bool BF16>
hipError_t run(const PromptParams& p, hipStream_t st) {
  using C = PromptCfg<BF16>;
  // A sequence's last tile may be short: at most one more tile a sequence.
  const int64_t tiles = (int64_t)p.T * (p.Hq / p.Hk) / C::BM + p.B;
  if (!fits_launch(tiles * p.Hk, 256)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((prompt_kernel<C>), dim3((unsigned)(tiles * p.Hk)), dim3(256), 0, st, p);
  return hipGetLastError();
}

template <int DP>
hipError_t run_pipe(const PromptParams& p, hipStream_t st) {
  using C = PipeCfg<DP>;
  const int64_t tiles = (int64_t)p.T * (p.Hq / p.Hk) / C::BM + p.B;
  if (!fits_launch(tiles * p.Hk, 256)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((prompt_pipe_kernel<C>), dim3((unsigned)(tiles * p.Hk)), dim3(256), 0, st, p);
  return hipGetLastError();
}

// Without SHARE one tile in LDS a wave, so that two blocks share a CU and hide each other's
// loads, starts and ends: with two tiles and one block a CU 512 tokens of 32
// heads took 18 us instead of 13; 64-row blocks of two tiles 18 too.
template <bool BF16, int DP, int NW, bool SHARE = false>
hipError_t run_wave(const PromptParams& p, hipStream_t st) {
  using C = CacheCfg<BF16, DP, 1, NW, true, SHARE ? 512 / DP : 1, SHARE>;
  CacheParams w = {};
  w.q = p.q, w.kc = p.k, w.vc = p.v, w.out = p.out, w.cu = p.cu;
  w.q_t = p.q_t, w.q_h = p.q_h, w.k_t = p.k_t, w.k_h = p.k_h, w.v_t = p.v_t, w.v_h = p.v_h, w.o_t = p.o_t, w.o_h = p.o_h;
  w.T = p.T, w.B = p.B, w.Hq = p.Hq, w.Hk = p.Hk, w.D = p.D, w.causal = p.causal, w.splits = 1, w.c = p.c;
  const int64_t tiles = (int64_t)p.T * (p.Hq / p.Hk) / C::ROWS + p.B;
  if (!fits_launch(tiles * p.Hk, 64 * NW)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((cache_kernel<C>), dim3((unsigned)(tiles * p.Hk)), dim3(64 * NW), 0, st, w);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_prompt_attention(const PromptParams& p, bool bf16, int cus, hipStream_t st) {
  if (p.T <= 0) return hipSuccess;
  const int64_t rows = (int64_t)p.T * p.Hq;
  // Many rows of bf16: 256-row blocks; else 32-row ones whose waves share the
  // keys.  32 heads of 128, 1000 / 1300 / 2048 tokens: 34 / 42 / 61 us in the
  // former, 32 / 44 / 77 in the latter (17 packed prompts of 8191 tokens 97 /
  // 190); 16 heads of 64, 2048 / 4096 / 8192 tokens: 45 / 81 / 185, 24 / 66 / 238.
  if (bf16 && p.D <= 64) return rows >= (int64_t)cus * 384 ? run_pipe<64>(p, st) : run_wave<true, 64, 4>(p, st);
  if (bf16 && p.D <= 128) {
    // Short sequences: 128-row blocks, two a CU, which hide each other's starts
    // and ends (8192 tokens in sequences of 64 / 128 / 256 / 512: 53 / 58 / 69 / 87
    // us, by the 256-row blocks 68 / 65 / 76 / 83).
    if (rows < (int64_t)cus * 144) return run_wave<true, 128, 4>(p, st);
    return (int64_t)p.T * (p.Hq / p.Hk) < (int64_t)1536 * p.B ? run_wave<true, 128, 4, true>(p, st) : run_pipe<128>(p, st);
  }
  if (!bf16 && p.D <= 64) return run_wave<false, 64, 4>(p, st);
  if (!bf16 && p.D <= 128) return run_wave<false, 128, 2>(p, st);
  return bf16 ? run<true>(p, st) : run<false>(p, st);
}

}  // namespace svdmlp
