// RMS norms of the heads of queries and keys with the rotary positions behind
// them, in one pass:
//     y = w x / sqrt(mean(x^2) + eps)            over a head's D values, in 32 bits
//     (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)
// for the pairs of the first `rot` values; y is rounded once, after the turn.
// With a cache the keys and the values go straight to their rows of it.  Angles
// as in rope.hip.
//
// Bound by HBM: every value is read and written once; apart, the norm and the
// turn would read and write them twice.  L lanes hold a head between its sum of
// squares and its turn, a 16-byte piece and its partner each, so that the sum is
// a few exchanges of lanes and pairs never leave their lane.  A block takes a
// token, four where those are many.
#include <algorithm>
#include <type_traits>

#include "decoder.hpp"
#include "rope.hpp"

namespace svdmlp {

namespace {

template <int E>
__device__ __forceinline__ void scaled(float* x, float by, const float* w) {
  if constexpr (E == 1) {
    x[0] *= by * w[0];
  } else {
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      const f32x4 g = reinterpret_cast<const f32x4*>(w)[q];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * q + e] *= by * g[e];
    }
  }
}

// VEC: D, rot, every stride and every base in whole 16-byte pieces (half layout:
// rot / 2 too); a unit of a head is then a piece of its first half with its
// partner (half layout) or a piece (interleaved, and behind rot), else a pair or,
// behind rot, a value.  BATCH heads of a group of lanes are on their way at once.
template <bool BF16, bool VEC, int L, int TOK, int BATCH>
__global__ __launch_bounds__(256) void head_norm_turn_kernel(NormRopeParams p) {
  constexpr int ES = BF16 ? 2 : 4, E = VEC ? 16 / ES : 1, GROUPS = 256 / L;
  using Raw = std::conditional_t<VEC, u32x4, float>;
  extern __shared__ float cs[];  // [TOK][rot / 2] cosines, then as many sines
  const RopeParams& r = p.r;
  const int half = r.rot / 2;
  const int64_t t0 = (int64_t)blockIdx.x * TOK;
  const int tokens = (int)min((int64_t)TOK, r.T - t0);
  float* const sn = cs + TOK * half;
  const bool append = r.slots != nullptr, inside = VEC && r.interleaved;  // inside: both of a pair in one piece
  const int turned = inside ? r.rot / E : half / E, units = turned + (r.D - r.rot) / E;
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  // The places of unit u's values in the head.
  auto first = [&](int u) { return u >= turned ? r.rot + (u - turned) * E : !VEC && r.interleaved ? 2 * u : u * E; };
  auto second = [&](int u) { return !VEC && r.interleaved ? 2 * u + 1 : half + u * E; };
  auto paired = [&](int u) { return u < turned && !inside; };
  auto raw = [&](const char* src, int at) -> Raw {
    if constexpr (VEC) return *reinterpret_cast<const u32x4*>(src + at * ES);
    else return ld1<BF16>(src, at);
  };
  auto values = [&](Raw v, float* x) {
    if constexpr (VEC) unpack<BF16>(v, x);
    else x[0] = v;
  };
  auto give = [&](char* dst, int at, const float* x) {
    if constexpr (VEC) *reinterpret_cast<u32x4*>(dst + at * ES) = pack<BF16>(x);
    else st1<BF16>(dst, at, x[0]);
  };
  // Unit u of a head: normalised, turned and stored.
  auto finish = [&](int tt, char* dst, int u, Raw va, Raw vb, float rstd, const float* w) {
    const int a = first(u), b = second(u);
    float x[E], y[E];
    values(va, x);
    scaled<E>(x, rstd, w + a);
    if (paired(u)) {
      values(vb, y);
      scaled<E>(y, rstd, w + b);
      const float *c = cs + tt * half + u * E, *s = sn + tt * half + u * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = x[e], g = y[e];
        x[e] = f * c[e] - g * s[e];
        y[e] = g * c[e] + f * s[e];
      }
      give(dst, b, y);
    } else if (VEC && u < turned) {
      const float *c = cs + tt * half + u * (E / 2), *s = sn + tt * half + u * (E / 2);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const float f = x[2 * e], g = x[2 * e + 1];
        x[2 * e] = f * c[e] - g * s[e];
        x[2 * e + 1] = g * c[e] + f * s[e];
      }
    }
    give(dst, a, x);
  };
  // Heads of q or of k of the block's tokens, BATCH a group of lanes: their first
  // units are loaded, then (before the first of them) the angles are awaited.
  bool waited = false;
  auto pass = [&](auto is_q, int heads) {
    constexpr bool Q = decltype(is_q)::value;
    for (int i0 = group; i0 < tokens * heads || !waited; i0 += GROUPS * BATCH) {
      Raw va[BATCH], vb[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int i = min(i0 + GROUPS * j, tokens * heads - 1), tt = TOK == 1 ? 0 : i / heads, h = i - tt * heads;
        const char* const src = Q ? static_cast<const char*>(r.q) + ((t0 + tt) * r.q_t + h * r.q_h) * ES
                                  : static_cast<const char*>(r.k) + ((t0 + tt) * r.k_t + h * r.k_h) * ES;
        va[j] = vb[j] = Raw{};
        if (lane < units) {
          va[j] = raw(src, first(lane));
          if (paired(lane)) vb[j] = raw(src, second(lane));
        }
      }
      if (!waited) {
        for (int i = threadIdx.x; i < tokens * half; i += 256) turn(r.pos[t0 + i / half], r.inv_freq[i % half], r.scale, &cs[i], &sn[i]);
        __syncthreads();
        waited = true;
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int i = i0 + GROUPS * j;
        if (i >= tokens * heads) break;
        const int tt = TOK == 1 ? 0 : i / heads, h = i - tt * heads;
        const int64_t t = t0 + tt;
        const char* const src = Q ? static_cast<const char*>(r.q) + (t * r.q_t + h * r.q_h) * ES : static_cast<const char*>(r.k) + (t * r.k_t + h * r.k_h) * ES;
        float ss = 0.f, x[E];
        auto add = [&](Raw v) {
          values(v, x);
#pragma unroll
          for (int e = 0; e < E; ++e) ss += x[e] * x[e];
        };
        add(va[j]);  // (zeros where there is no unit or partner)
        add(vb[j]);
        for (int u = lane + L; u < units; u += L) {
          add(raw(src, first(u)));
          if (paired(u)) add(raw(src, second(u)));
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        const float rstd = 1.0f / sqrtf(ss / (float)r.D + p.eps);
        char* dst;
        if constexpr (Q) {
          dst = static_cast<char*>(r.qo) + (t * r.qo_t + h * r.qo_h) * ES;
        } else if (append) {
          const int64_t slot = r.slots[t];
          if (slot < 0 || slot >= r.pages * r.page) continue;  // no row of the cache
          const int64_t pg = slot / r.page;
          dst = static_cast<char*>(r.ko) + (pg * r.ko_p + (slot - pg * r.page) * r.ko_t + h * r.ko_h) * ES;
        } else {
          dst = static_cast<char*>(r.ko) + (t * r.ko_t + h * r.ko_h) * ES;
        }
        const float* const w = Q ? p.q_w + (int64_t)h * p.qw_h : p.k_w + (int64_t)h * p.kw_h;
        if (lane < units) finish(tt, dst, lane, va[j], vb[j], rstd, w);
        // (an output may be its input: a unit's values are read before they are written, by the same lane)
        for (int u = lane + L; u < units; u += L) finish(tt, dst, u, raw(src, first(u)), paired(u) ? raw(src, second(u)) : Raw{}, rstd, w);
      }
    }
  };
  pass(std::true_type{}, r.Hq);
  pass(std::false_type{}, r.Hk);
  if (!append) return;
  // Values: copied.
  const int pieces = r.D / E, all = tokens * r.Hk * pieces;
  for (int i = threadIdx.x; i < all; i += 256) {
    const int head = i / pieces, tt = head / r.Hk, h = head - tt * r.Hk, at = (i - head * pieces) * E;
    const int64_t t = t0 + tt, slot = r.slots[t];
    if (slot < 0 || slot >= r.pages * r.page) continue;
    const int64_t pg = slot / r.page;
    const char* const src = static_cast<const char*>(r.v) + (t * r.v_t + h * r.v_h) * ES;
    char* const dst = static_cast<char*>(r.vo) + (pg * r.vo_p + (slot - pg * r.page) * r.vo_t + h * r.vo_h) * ES;
    if constexpr (VEC) *reinterpret_cast<u32x4*>(dst + at * ES) = *reinterpret_cast<const u32x4*>(src + at * ES);
    else if constexpr (BF16) reinterpret_cast<uint16_t*>(dst)[at] = reinterpret_cast<const uint16_t*>(src)[at];
    else reinterpret_cast<uint32_t*>(dst)[at] = reinterpret_cast<const uint32_t*>(src)[at];
  }
}

template <bool BF16, bool VEC, int L>
hipError_t run(const NormRopeParams& p, hipStream_t st) {
  const RopeParams& r = p.r;
  // (one token a block while those are few, as rope.hip)
  if (r.T < 4096) {
    hipLaunchKernelGGL((head_norm_turn_kernel<BF16, VEC, L, 1, 1>), dim3((unsigned)r.T), dim3(256), r.rot * 4, st, p);
    return hipGetLastError();
  }
  constexpr int64_t kTokens = 1 << 24;  // a launch
  static_assert(kTokens / 4 * 256 < (int64_t)1 << 32, "threads of a launch");
  constexpr int ES = BF16 ? 2 : 4;
  for (int64_t t = 0; t < r.T; t += kTokens) {
    NormRopeParams n = p;
    RopeParams& c = n.r;
    c.T = std::min(kTokens, r.T - t);
    c.q = static_cast<const char*>(r.q) + t * r.q_t * ES, c.k = static_cast<const char*>(r.k) + t * r.k_t * ES;
    c.qo = static_cast<char*>(r.qo) + t * r.qo_t * ES, c.pos = r.pos + t;
    if (r.slots) c.v = static_cast<const char*>(r.v) + t * r.v_t * ES, c.slots = r.slots + t;
    else c.ko = static_cast<char*>(r.ko) + t * r.ko_t * ES;
    hipLaunchKernelGGL((head_norm_turn_kernel<BF16, VEC, L, 4, 4>), dim3((unsigned)((c.T + 3) / 4)), dim3(256), 4 * r.rot * 4, st, n);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <bool BF16>
hipError_t pick(const NormRopeParams& p, bool vec, hipStream_t st) {
  if (!vec) return run<BF16, false, 64>(p, st);
  // As many lanes as a head has units: heads of 128 in bf16, turned whole, 8.
  constexpr int E = BF16 ? 8 : 4;
  const int units = (p.r.interleaved ? p.r.rot : p.r.rot / 2) / E + (p.r.D - p.r.rot) / E;
  if (units <= 8) return run<BF16, true, 8>(p, st);
  if (units <= 16) return run<BF16, true, 16>(p, st);
  if (units <= 32) return run<BF16, true, 32>(p, st);
  return run<BF16, true, 64>(p, st);
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeParams& p, bool bf16, bool vec, hipStream_t st) {
  if (p.r.T <= 0) return hipSuccess;
  return bf16 ? pick<true>(p, vec, st) : pick<false>(p, vec, st);
}

}  // namespace svdmlp
