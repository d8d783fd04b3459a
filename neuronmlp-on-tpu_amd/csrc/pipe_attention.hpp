// The walk over keys of the bf16 kernels for many rows (prompt_attention.hip,
// chunk_attention.hip): 4 waves of 64 rows, and keys in tiles of 64 through LDS
// that all of them share.
//
// Over the keys that every row of the block sees it is pipelined in units of 32
// keys.  A step does three things that do not wait for each other,
//     S(u + 1) = K(u + 1) Q^T        matrix unit
//     P(u) = exp2(c S(u) - m)        vector unit
//     O += V(u - 1)^T P(u - 1)^T     matrix unit
// so that with one wave a SIMD neither unit waits for the other.  Its order is
// laid down in the source: a slot is one MFMA (32 cycles) and what fits beside
// it, one or two weights and an LDS read of a piece needed some slots later.
// 64 rows a wave halve the LDS reads a product (one piece of K or V feeds two
// MFMAs).  Tiles of 64 keys come straight to LDS, the keys three and the
// values two tiles ahead, in four stages each; the loop is unrolled over the
// stages, whose offsets are then constants.  Keys that only some rows see and the
// last, short tile follow in a plain loop.
#pragma once

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "attn.hpp"

namespace svdmlp {

namespace {  // as the kernels that take them

template <int DP_>
struct PipeCfg {
  static constexpr int DP = DP_, QG = 2, RB = DP * 2, PIECES = RB / 16, STEPS = RB / 32, KB = 64, BM = 256, NS = 4;
  static constexpr int TILE = KB * RB, STAGE = 2 * TILE, UNIT = 32 * RB, DB = DP / 32;
  static constexpr int LOADS = TILE / 4096;  // 1 KB loads a wave and tile, of keys and of values
  static constexpr int RPL = 64 / PIECES;    // rows a load
  static constexpr int FRAGS = STEPS + 2 * DB, SLOTS = QG * FRAGS;  // LDS pieces and MFMAs a step
  static constexpr int AHEAD = 4;                                   // pieces read before they are needed
  static constexpr int PER = 16 * QG / SLOTS;                       // weights a slot
  static_assert(FRAGS % AHEAD == 0 && PER * SLOTS == 16 * QG, "slots");
};

// What a wave holds of its 64 rows, and its part of the walk.
template <class C>
struct PipeWave {
  static constexpr int QG = C::QG, KB = C::KB, DB = C::DB;
  const u32x4 (&qf)[QG][C::STEPS];  // queries: lane half h holds the 16-byte piece 2 s + h of its row at step s
  f32x16 o[QG][DB];
  float m[QG], l[QG];
  u32x4 piece[C::AHEAD];
  const TileLane<C::RB, true> at;
  const float c;
  uint32_t bad = 0;  // bits where a masked tile's values had infinities or NaN

  __device__ __forceinline__ PipeWave(const u32x4 (&q)[QG][C::STEPS], int lane, float c_) : qf(q), at(lane), c(c_) {
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[g][d][i] = 0.f;
    }
  }

  // S = K Q^T of the 32 keys at kt; the first pieces of V at vt are read behind
  // it (an LDS read takes as long as two products, and one wave a SIMD hides none).
  __device__ __forceinline__ void scores(attn_lds kt, attn_lds vt, f32x16 (&s)[QG]) {
#pragma unroll
    for (int t = 0; t < C::AHEAD; ++t) piece[t] = at.key(kt, t);
#pragma unroll
    for (int t = 0; t < C::STEPS; ++t) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < QG; ++g) {
        if (t == 0) s[g] = f32x16{};
        s[g] = attn_mfma<true>(piece[t % C::AHEAD], qf[g][t], s[g]);
      }
      const int n = t + C::AHEAD;
      piece[t % C::AHEAD] = n < C::STEPS ? at.key(kt, n) : at.values(vt, (n - C::STEPS) / DB, (n - C::STEPS) % DB);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // O += V^T P^T of the 32 keys at vt, whose first pieces are read.
  __device__ __forceinline__ void values(attn_lds vt, const u32x4 (&pb)[QG][2], bool masked) {
#pragma unroll
    for (int f = 0; f < 2 * DB; ++f) {
      __builtin_amdgcn_sched_barrier(0);
      u32x4 vf = piece[f % C::AHEAD];
      if (masked)
#pragma unroll
        for (int w = 0; w < 4; ++w) vf[w] = scrub<true>(vf[w], bad);
#pragma unroll
      for (int g = 0; g < QG; ++g) o[g][f % DB] = attn_mfma<true>(vf, pb[g][f / DB], o[g][f % DB]);
      if (f + C::AHEAD < 2 * DB) piece[f % C::AHEAD] = at.values(vt, (f + C::AHEAD) / DB, (f + C::AHEAD) % DB);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // Where a score passes the reference by over kSlack: the new reference, and
  // what sums so far are to be multiplied by.
  __device__ __forceinline__ bool reference(const f32x16 (&s)[QG], float (&scale)[QG]) {
    float mx[QG];
    bool over = false;
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      mx[g] = most_of(s[g]) * c;
      over |= mx[g] > m[g] + kSlack;
    }
    if (!__any(over)) return false;
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      const float n = fmaxf(m[g], fmaxf(mx[g], __shfl_xor(mx[g], 32)));
      scale[g] = n == -INFINITY ? 1.f : exp2f(m[g] - n);
      m[g] = n;
      l[g] *= scale[g];
    }
    return true;
  }
  __device__ __forceinline__ void weights(const f32x16 (&s)[QG], u32x4 (&pb)[QG][2]) {
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      const float ref = m[g] == -INFINITY ? 0.f : m[g];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float a = __builtin_amdgcn_exp2f(fmaf(s[g][8 * t + 2 * w], c, -ref));
          const float b = __builtin_amdgcn_exp2f(fmaf(s[g][8 * t + 2 * w + 1], c, -ref));
          pb[g][t][w] = pack_bf16x2(a, b);
          l[g] = add_pair(pb[g][t][w], l[g]);
        }
    }
  }
  __device__ __forceinline__ void rescale(const float (&scale)[QG]) {
#pragma unroll
    for (int g = 0; g < QG; ++g)
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[g][d][i] *= scale[g];
  }

  // Tiles 0 to full - 1 (at least one), of keys that every row sees; arrive(t)
  // returns when tile t can be read, and beside(n) is what a slot n of its first
  // step may do with what the matrix unit leaves it.  again: rows have sums already.  Before the first step the values of the
  // last stage's second unit are multiplied by zero weights: they have to be
  // finite.
  template <class Arrive, class Beside>
  __device__ __forceinline__ void whole_tiles(attn_lds base, int full, int& t, bool again, Arrive arrive, Beside beside) {
    f32x16 s0[QG], s1[QG];
    u32x4 p0[QG][2], p1[QG][2], frag[C::AHEAD];
    float scale[QG], over[QG];  // over: the score beyond which the reference moves
    bool moved = false;
#pragma unroll
    for (int g = 0; g < QG; ++g) p1[g][0] = p1[g][1] = u32x4{0u, 0u, 0u, 0u};
    // Places in the stages whose offsets do not fit an instruction (64 KB).
    constexpr int NEAR = std::min(C::NS, 65536 / C::STAGE);
    TileLane<C::RB, true> at2 = at;
    if constexpr (NEAR < C::NS) {
#pragma unroll
      for (int i = 0; i < TileLane<C::RB, true>::KN; ++i) {
        at2.k[i] += NEAR * C::STAGE;
        asm volatile("" : "+v"(at2.k[i]));
      }
#pragma unroll
      for (int i = 0; i < TileLane<C::RB, true>::VN; ++i) {
        at2.v[i] += NEAR * C::STAGE;
        asm volatile("" : "+v"(at2.v[i]));
      }
    }
    // Piece f of the step at unit U of the tile in stage S: K of the unit after
    // it, then V of the unit before it.
    auto read = [&](auto S_, auto U_, int f) {
      constexpr int S = decltype(S_)::value, U = decltype(U_)::value;
      if (f < C::STEPS) {
        constexpr int st = U ? (S + 1) % C::NS : S;
        frag[f % C::AHEAD] = (st < NEAR ? at : at2).key(base + st % NEAR * C::STAGE + (U ? 0 : C::UNIT), f);
      } else {
        constexpr int st = U ? S : (S + C::NS - 1) % C::NS;
        frag[f % C::AHEAD] = (st < NEAR ? at : at2).values(base + st % NEAR * C::STAGE + C::TILE + (U ? 0 : C::UNIT),
                                                          (f - C::STEPS) / DB, (f - C::STEPS) % DB);
      }
    };
    auto step = [&](auto S_, auto U_, f32x16 (&sc)[QG], f32x16 (&sn)[QG], u32x4 (&pc)[QG][2], const u32x4 (&pp)[QG][2]) {
      constexpr int S = decltype(S_)::value, U = decltype(U_)::value;
      constexpr int MPS = C::SLOTS >= 32 ? 2 : 4;  // maxima a slot, in the last 8 or 4
      float hold = 0.f, mx[QG] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < C::SLOTS; ++n) {
        const int f = n / QG, g = n % QG;
        __builtin_amdgcn_sched_barrier(0);
        if (f < C::STEPS) {
          if (f == 0) sn[g] = f32x16{};
          sn[g] = attn_mfma<true>(frag[f % C::AHEAD], qf[g][f], sn[g]);
        } else {
          const int v = f - C::STEPS;
          o[g][v % DB] = attn_mfma<true>(frag[f % C::AHEAD], pp[g][v / DB], o[g][v % DB]);
        }
        if (g == QG - 1) {  // the piece's last product: its registers take the one AHEAD of it
          if (f + C::AHEAD < C::FRAGS) read(S_, U_, f + C::AHEAD);
          else read(std::integral_constant<int, U ? (S + 1) % C::NS : S>{}, std::integral_constant<int, 1 - U>{}, f + C::AHEAD - C::FRAGS);
        }
        // The maximum of the new scores, once they are complete.
        if (n >= C::SLOTS - 16 * QG / 2 / MPS) {
#pragma unroll
          for (int q = 0; q < MPS; ++q) {
            const int i = (n - (C::SLOTS - 16 * QG / 2 / MPS)) * MPS + q, wg = i / 8, wi = 2 * (i % 8);
            mx[wg] = fmaxf(fmaxf(mx[wg], sn[wg][wi]), sn[wg][wi + 1]);
          }
        }
        // Weights PER n ..; the empty asm keeps them in their slot.
#pragma unroll
        for (int q = 0; q < C::PER; ++q) {
          const int i = n * C::PER + q, wg = i / 16, wi = i % 16;
          const float e = __builtin_amdgcn_exp2f(fmaf(sc[wg][wi], c, -m[wg]));
          if (i % 2 == 0) {
            hold = e;
            asm volatile("" : "+v"(hold));
          } else {
            uint32_t both = pack_bf16x2(hold, e);
            l[wg] = add_pair(both, l[wg]);
            asm volatile("" : "+v"(both), "+v"(l[wg]));
            pc[wg][wi / 8][wi % 8 / 2] = both;
          }
        }
        if constexpr (U == 0) beside(n);
      }
      __builtin_amdgcn_sched_barrier(0);
      bool any = moved;
#pragma unroll
      for (int g = 0; g < QG; ++g) any |= mx[g] > over[g];
      if (__any(any)) {  // rare: a reference moves, or has moved
        if (moved) rescale(scale);
        // behind the last unit here come keys that not every row sees, or none
        moved = (U == 0 || t + 1 < full) && reference(sn, scale);
#pragma unroll
        for (int g = 0; g < QG; ++g) over[g] = (m[g] + kSlack) / c;
      }
    };
    arrive(0);
    scores(base, base, s0);
    if (reference(s0, scale) && again) rescale(scale);  // (else nothing has been summed yet)
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      if (m[g] == -INFINITY) m[g] = -1e30f;  // no finite score yet: a finite reference that any will move
      over[g] = (m[g] + kSlack) / c;
    }
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
#pragma unroll
    for (int f = 0; f < C::AHEAD; ++f) read(I0{}, I0{}, f);
#define SVDMLP_PIPE_TILE(S)                 \
  step(S{}, I0{}, s0, s1, p0, p1);          \
  step(S{}, I1{}, s1, s0, p1, p0);          \
  if (++t == full) break;                   \
  arrive(t);
    for (;;) {
      SVDMLP_PIPE_TILE(I0)
      SVDMLP_PIPE_TILE(I1)
      SVDMLP_PIPE_TILE(I2)
      SVDMLP_PIPE_TILE(I3)
    }
#undef SVDMLP_PIPE_TILE
    const attn_lds last = base + ((t - 1) % C::NS) * C::STAGE + C::TILE + C::UNIT;
#pragma unroll
    for (int f = 0; f < C::AHEAD; ++f) piece[f] = at.values(last, f / DB, f % DB);
    values(last, p1, false);
  }
};

}  // namespace

}  // namespace svdmlp
