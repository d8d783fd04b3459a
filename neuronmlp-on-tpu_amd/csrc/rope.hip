// Rotary positions: each pair (a, b) of a head's first `rot` values is turned
// by the angle pos * inv_freq[p],
//     (a, b) -> (a cos - b sin, b cos + a sin),
// p the pair's number; a pair is (p, p + rot/2) (half layout) or (2p, 2p + 1)
// (interleaved).  The rest of the head is copied.  With a cache, the turned
// keys and the values go straight to their rows of it.
//
// The angle is a product in 64 bits: in 32 its error at position 100000 is
// already 0.004.  It is reduced to a quarter turn in 64 bits, and only the rest
// (at most pi/4, so exact to 5e-8) goes on in 32.  The cosines of a token are
// computed once for all its heads, through LDS.
//
// Bound by HBM: every value is read and written once.  A block takes a few
// tokens, its threads their 16-byte pieces.  6007 tokens of 32 + 8 heads of 128
// in bf16: 23.5 us, 5.2 TB/s, a copy's rate; 16 into a cache: 4.4 us, latency.
#include <algorithm>

#include "decoder.hpp"
#include "rope.hpp"

namespace svdmlp {

namespace {

// TOK tokens a block.  VEC: D, rot, every stride and every base in whole
// 16-byte pieces (half layout: rot / 2 too).
template <bool BF16, bool VEC, int TOK>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
  constexpr int ES = BF16 ? 2 : 4, E = 16 / ES;
  extern __shared__ float cs[];  // [TOK][rot / 2] cosines, then as many sines
  const int half = p.rot / 2;
  const int64_t t0 = (int64_t)blockIdx.x * TOK;
  float* const sn = cs + TOK * half;
  for (int i = threadIdx.x; i < TOK * half; i += 256) {
    const int64_t t = t0 + i / half;
    if (t < p.T) turn(p.pos[t], p.inv_freq[i % half], p.scale, &cs[i], &sn[i]);
  }
  __syncthreads();
  const bool append = p.slots != nullptr;
  const int heads = p.Hq + p.Hk * (append ? 2 : 1);
  // units of a head: VEC half layout, piece j of the first half with its
  // partner, then the pieces behind rot; VEC interleaved, the pieces; else
  // single values behind rot and pairs before.
  const int turned = VEC ? (p.interleaved ? p.rot / E : half / E) : half;
  const int units = turned + (VEC ? (p.D - p.rot) / E : p.D - p.rot);
  const int total = heads * units;
  // i / d as a product with d's reciprocal, exact below 2^16 (a head's units
  // and a block's are that few for all but giant calls)
  const bool small = TOK * total < 65536;
  const uint32_t mtotal = small ? 0xffffffffu / (uint32_t)total + 1 : 0, munits = small ? 0xffffffffu / (uint32_t)units + 1 : 0;
  auto quotient = [&](int i, int d, uint32_t m) -> int { return d == 1 ? i : small ? (int)__umulhi((uint32_t)i, m) : i / d; };
  for (int i = threadIdx.x; i < TOK * total; i += 256) {
    const int tt = TOK == 1 ? 0 : quotient(i, total, mtotal), rest = i - tt * total;
    const int64_t t = t0 + tt;
    if (t >= p.T) break;
    const int hh = quotient(rest, units, munits), u = rest - hh * units;
    const char* src;
    char* dst;
    bool plain = false;
    if (hh < p.Hq) {
      src = static_cast<const char*>(p.q) + (t * p.q_t + hh * p.q_h) * ES;
      dst = static_cast<char*>(p.qo) + (t * p.qo_t + hh * p.qo_h) * ES;
    } else {
      const bool val = hh >= p.Hq + p.Hk;
      const int h = hh - p.Hq - (val ? p.Hk : 0);
      plain = val;
      src = val ? static_cast<const char*>(p.v) + (t * p.v_t + h * p.v_h) * ES
                : static_cast<const char*>(p.k) + (t * p.k_t + h * p.k_h) * ES;
      if (append) {
        const int64_t slot = p.slots[t];
        if (slot < 0 || slot >= p.pages * p.page) continue;  // no row of the cache
        const int64_t pg = slot / p.page, row = slot - pg * p.page;
        dst = val ? static_cast<char*>(p.vo) + (pg * p.vo_p + row * p.vo_t + h * p.vo_h) * ES
                  : static_cast<char*>(p.ko) + (pg * p.ko_p + row * p.ko_t + h * p.ko_h) * ES;
      } else {
        dst = static_cast<char*>(p.ko) + (t * p.ko_t + h * p.ko_h) * ES;
      }
    }
    if constexpr (VEC) {
      const u32x4* s4 = reinterpret_cast<const u32x4*>(src);
      u32x4* d4 = reinterpret_cast<u32x4*>(dst);
      if (u >= turned) {  // behind the turned part
        const int j = p.rot / E + (u - turned);
        d4[j] = s4[j];
      } else if (!p.interleaved) {
        const u32x4 va = s4[u], vb = s4[u + half / E];
        if (plain) {
          d4[u] = va;
          d4[u + half / E] = vb;
          continue;
        }
        float a[E], b[E], x[E], y[E];
        unpack<BF16>(va, a);
        unpack<BF16>(vb, b);
        const float *c = cs + tt * half + u * E, *s = sn + tt * half + u * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[e] = a[e] * c[e] - b[e] * s[e];
          y[e] = b[e] * c[e] + a[e] * s[e];
        }
        d4[u] = pack<BF16>(x);
        d4[u + half / E] = pack<BF16>(y);
      } else {
        const u32x4 va = s4[u];
        if (plain) {
          d4[u] = va;
          continue;
        }
        float a[E], x[E];
        unpack<BF16>(va, a);
        const float *c = cs + tt * half + u * (E / 2), *s = sn + tt * half + u * (E / 2);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          x[2 * e] = a[2 * e] * c[e] - a[2 * e + 1] * s[e];
          x[2 * e + 1] = a[2 * e + 1] * c[e] + a[2 * e] * s[e];
        }
        d4[u] = pack<BF16>(x);
      }
    } else {
      if (u >= turned) {
        const int j = p.rot + (u - turned);
        st1<BF16>(dst, j, ld1<BF16>(src, j));
      } else {
        const int ia = p.interleaved ? 2 * u : u, ib = p.interleaved ? 2 * u + 1 : u + half;
        const float a = ld1<BF16>(src, ia), b = ld1<BF16>(src, ib);
        const float c = plain ? 1.f : cs[tt * half + u], s = plain ? 0.f : sn[tt * half + u];
        st1<BF16>(dst, ia, plain ? a : a * c - b * s);
        st1<BF16>(dst, ib, plain ? b : b * c + a * s);
      }
    }
  }
}

}  // namespace

hipError_t launch_rope(const RopeParams& p, bool bf16, bool vec, hipStream_t st) {
  if (p.T <= 0) return hipSuccess;
  auto go = [&](auto b, auto v) {
    constexpr bool B = decltype(b)::value, V = decltype(v)::value;
    // One token a block while those are few, else four: their cosines keep all
    // 256 threads busy at 128 turned values (2501 fp32 tokens of 32 heads of 64:
    // 9.9 us by one, 14.6 by four).
    if (p.T < 4096) {
      hipLaunchKernelGGL((rope_kernel<B, V, 1>), dim3((unsigned)p.T), dim3(256), p.rot * 4, st, p);
      return hipGetLastError();
    }
    constexpr int64_t kTokens = 1 << 24;  // a launch
    static_assert(kTokens / 4 * 256 < (int64_t)1 << 32, "threads of a launch");
    constexpr int ES = B ? 2 : 4;
    for (int64_t t = 0; t < p.T; t += kTokens) {
      RopeParams c = p;
      c.T = std::min(kTokens, p.T - t);
      c.q = static_cast<const char*>(p.q) + t * p.q_t * ES, c.k = static_cast<const char*>(p.k) + t * p.k_t * ES;
      c.qo = static_cast<char*>(p.qo) + t * p.qo_t * ES, c.pos = p.pos + t;
      if (p.slots) c.v = static_cast<const char*>(p.v) + t * p.v_t * ES, c.slots = p.slots + t;
      else c.ko = static_cast<char*>(p.ko) + t * p.ko_t * ES;
      hipLaunchKernelGGL((rope_kernel<B, V, 4>), dim3((unsigned)((c.T + 3) / 4)), dim3(256), 4 * p.rot * 4, st, c);
      if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  using T = std::true_type;
  using F = std::false_type;
  if (bf16) return vec ? go(T{}, T{}) : go(T{}, F{});
  return vec ? go(F{}, T{}) : go(F{}, F{});
}

}  // namespace svdmlp
