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
// token: more of them a block, or heads on their way ahead of others, cost
// registers and so waves (6007 tokens of 32 + 8 heads of 128 in bf16 24 us, 5.1
// TB/s, a copy's rate; by four tokens a block 28, two 26).  Seven waves a SIMD: 72
// registers, without the bound 96 and 25 us, by eight (24 bytes spilled) 32.  16 tokens into
// a cache: 5.2 us, latency.
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
// behind rot, a value.
template <bool BF16, bool VEC, int L>
__global__ __launch_bounds__(256, 7) void head_norm_turn_kernel(NormRopeParams p) {
  constexpr int ES = BF16 ? 2 : 4, E = VEC ? 16 / ES : 1, GROUPS = 256 / L;
  using Raw = std::conditional_t<VEC, u32x4, float>;
  extern __shared__ float cs[];  // rot / 2 cosines, then as many sines
  const RopeParams& r = p.r;
  const int half = r.rot / 2;
  const int64_t t = blockIdx.x;
  float* const sn = cs + half;
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
  auto finish = [&](char* dst, int u, Raw va, Raw vb, float rstd, const float* w) {
    const int a = first(u), b = second(u);
    float x[E], y[E];
    values(va, x);
    scaled<E>(x, rstd, w + a);
    if (paired(u)) {
      values(vb, y);
      scaled<E>(y, rstd, w + b);
      const float *c = cs + u * E, *s = sn + u * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = x[e], g = y[e];
        x[e] = f * c[e] - g * s[e];
        y[e] = g * c[e] + f * s[e];
      }
      give(dst, b, y);
    } else if (VEC && u < turned) {
      const float *c = cs + u * (E / 2), *s = sn + u * (E / 2);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const float f = x[2 * e], g = x[2 * e + 1];
        x[2 * e] = f * c[e] - g * s[e];
        x[2 * e + 1] = g * c[e] + f * s[e];
      }
    }
    give(dst, a, x);
  };
  const int64_t slot = append ? r.slots[t] : 0;
  const bool stored = slot >= 0 && (!append || slot < r.pages * r.page);  // (else no row of the cache)
  const int64_t pg = append && stored ? slot / r.page : 0, row = slot - pg * r.page;
  // Heads of q or of k, one a group of lanes; the first of them is loaded before
  // the angles are computed.
  bool waited = false;
  auto pass = [&](auto is_q, int heads) {
    constexpr bool Q = decltype(is_q)::value;
    for (int h = group; h < heads || !waited; h += GROUPS) {
      const char* const src = Q ? static_cast<const char*>(r.q) + (t * r.q_t + min(h, heads - 1) * r.q_h) * ES
                                : static_cast<const char*>(r.k) + (t * r.k_t + h * r.k_h) * ES;
      Raw va{}, vb{};
      if (lane < units) {
        va = raw(src, first(lane));
        if (paired(lane)) vb = raw(src, second(lane));
      }
      if (!waited) {
        for (int i = threadIdx.x; i < half; i += 256) turn(r.pos[t], r.inv_freq[i], r.scale, &cs[i], &sn[i]);
        __syncthreads();
        waited = true;
        if (h >= heads) break;
      }
      float ss = 0.f, x[E];
      auto add = [&](Raw v) {
        values(v, x);
#pragma unroll
        for (int e = 0; e < E; ++e) ss += x[e] * x[e];
      };
      add(va);  // (zeros where there is no unit or partner)
      add(vb);
      for (int u = lane + L; u < units; u += L) {
        add(raw(src, first(u)));
        if (paired(u)) add(raw(src, second(u)));
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
      const float rstd = 1.0f / sqrtf(ss / (float)r.D + p.eps);
      if (!Q && !stored) continue;
      char* const dst = Q ? static_cast<char*>(r.qo) + (t * r.qo_t + h * r.qo_h) * ES
                          : static_cast<char*>(r.ko) + (append ? pg * r.ko_p + row * r.ko_t + h * r.ko_h : t * r.ko_t + h * r.ko_h) * ES;
      const float* const w = Q ? p.q_w + (int64_t)h * p.qw_h : p.k_w + (int64_t)h * p.kw_h;
      if (lane < units) finish(dst, lane, va, vb, rstd, w);
      // (an output may be its input: a unit's values are read before they are written, by the same lane)
      for (int u = lane + L; u < units; u += L) finish(dst, u, raw(src, first(u)), paired(u) ? raw(src, second(u)) : Raw{}, rstd, w);
    }
  };
  pass(std::true_type{}, r.Hq);
  pass(std::false_type{}, r.Hk);
  if (!append || !stored) return;
  // Values: copied.
  const int pieces = r.D / E;
  for (int i = threadIdx.x; i < r.Hk * pieces; i += 256) {
    const int h = i / pieces, at = (i - h * pieces) * E;
    const char* const src = static_cast<const char*>(r.v) + (t * r.v_t + h * r.v_h) * ES;
    char* const dst = static_cast<char*>(r.vo) + (pg * r.vo_p + row * r.vo_t + h * r.vo_h) * ES;
    if constexpr (VEC) *reinterpret_cast<u32x4*>(dst + at * ES) = *reinterpret_cast<const u32x4*>(src + at * ES);
    else if constexpr (BF16) reinterpret_cast<uint16_t*>(dst)[at] = reinterpret_cast<const uint16_t*>(src)[at];
    else reinterpret_cast<uint32_t*>(dst)[at] = reinterpret_cast<const uint32_t*>(src)[at];
  }
}

template <bool BF16, bool VEC, int L>
hipError_t run(const NormRopeParams& p, hipStream_t st) {
  constexpr int64_t kTokens = 1 << 23;  // a launch
  static_assert(kTokens * 256 < (int64_t)1 << 32, "threads of a launch");
  constexpr int ES = BF16 ? 2 : 4;
  const RopeParams& r = p.r;
  for (int64_t t = 0; t < r.T; t += kTokens) {
    NormRopeParams n = p;
    RopeParams& c = n.r;
    c.T = std::min(kTokens, r.T - t);
    c.q = static_cast<const char*>(r.q) + t * r.q_t * ES, c.k = static_cast<const char*>(r.k) + t * r.k_t * ES;
    c.qo = static_cast<char*>(r.qo) + t * r.qo_t * ES, c.pos = r.pos + t;
    if (r.slots) c.v = static_cast<const char*>(r.v) + t * r.v_t * ES, c.slots = r.slots + t;
    else c.ko = static_cast<char*>(r.ko) + t * r.ko_t * ES;
    hipLaunchKernelGGL((head_norm_turn_kernel<BF16, VEC, L>), dim3((unsigned)c.T), dim3(256), r.rot * 4, st, n);
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
