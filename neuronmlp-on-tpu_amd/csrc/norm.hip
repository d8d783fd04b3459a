// The sum after a block of a decoder layer and the norm before the next one:
//     b' = post * b / sqrt(mean(b^2) + eps)     (where the block's output is normalised)
//     r  = x + scale * gate * b'
//     n  = weight * r / sqrt(mean(r^2) + eps)
// Sums and r in 32 bits; n is of r before its rounding.  The framework's
// RMSNorm in front of the MLP block (block.hip) takes the same mean.
//
// Bound by HBM: x, b (and a gate of rows) are read once and r, n written once.
// One block a row holds it in registers between the two sums.  4096 rows of 8192
// in bf16, normalised branch and gate: 60.5 us, 4.4 TB/s (a copy: 5.2); 8 rows of
// 4096: 3.6 us, latency.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "decoder.hpp"

namespace svdmlp {

namespace {

template <int NT>
__device__ __forceinline__ float block_sum(float v, float* part) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) t += part[i];
  return t;
}

// E values a piece, PER pieces a thread.
template <bool BF16, int E>
__device__ __forceinline__ void load(const void* p, int64_t piece, float* f) {
  if constexpr (E == 1) {
    f[0] = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p)[piece]) : static_cast<const float*>(p)[piece];
  } else {
    const u32x4 v = static_cast<const u32x4*>(p)[piece];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (BF16) {
        f[2 * w] = __uint_as_float(v[w] << 16);
        f[2 * w + 1] = __uint_as_float(v[w] & 0xffff0000u);
      } else {
        f[w] = __uint_as_float(v[w]);
      }
    }
  }
}
template <bool BF16, int E>
__device__ __forceinline__ void store(void* p, int64_t piece, const float* f) {
  if constexpr (E == 1) {
    if constexpr (BF16) static_cast<uint16_t*>(p)[piece] = (uint16_t)f32_to_bf16_bits(f[0]);
    else static_cast<float*>(p)[piece] = f[0];
  } else {
    u32x4 v;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (BF16) v[w] = pack_bf16x2(f[2 * w], f[2 * w + 1]);
      else v[w] = __float_as_uint(f[w]);
    }
    static_cast<u32x4*>(p)[piece] = v;
  }
}
template <int E>
__device__ __forceinline__ void gains(const float* w, int64_t piece, float* f) {
  if constexpr (E == 1) {
    f[0] = w[piece];
  } else {
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      const f32x4 g = reinterpret_cast<const f32x4*>(w)[piece * (E / 4) + q];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * q + e] = g[e];
    }
  }
}

template <bool BF16, int E, int NT, int PER>
__global__ __launch_bounds__(NT) void residual_norm_kernel(ResidualNormParams p) {
  constexpr int ES = BF16 ? 2 : 4;
  __shared__ float part[2][16];
  const int64_t row = blockIdx.x;
  const int pieces = p.d / E;
  const char* x = static_cast<const char*>(p.x) + row * p.x_t * ES;
  const char* b = static_cast<const char*>(p.branch) + row * p.b_t * ES;
  const char* g = static_cast<const char*>(p.gate) + row * p.g_t * ES;
  float xr[PER][E], br[PER][E];
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int i = threadIdx.x + NT * q;
    if (i < pieces) {
      load<BF16, E>(x, i, xr[q]);
      if (p.branch) load<BF16, E>(b, i, br[q]);
    }
  }
  if (p.branch) {
    float rstd = p.scale;
    if (p.post) {
      float ss = 0.f;
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (threadIdx.x + NT * q < pieces)
#pragma unroll
          for (int e = 0; e < E; ++e) ss += br[q][e] * br[q][e];
      rstd = 1.0f / sqrtf(block_sum<NT>(ss, part[0]) / (float)p.d + p.eps) * p.scale;
    }
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int i = threadIdx.x + NT * q;
      if (i >= pieces) continue;
      float w[E];
      if (p.post) {
        gains<E>(p.post, i, w);
#pragma unroll
        for (int e = 0; e < E; ++e) br[q][e] *= w[e];
      }
      if (p.gate) {
        load<BF16, E>(g, i, w);
#pragma unroll
        for (int e = 0; e < E; ++e) br[q][e] *= w[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) xr[q][e] += rstd * br[q][e];
    }
  }
  if (p.r) {
    char* r = static_cast<char*>(p.r) + row * p.r_t * ES;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int i = threadIdx.x + NT * q;
      if (i < pieces) store<BF16, E>(r, i, xr[q]);
    }
  }
  if (!p.n) return;
  float ss = 0.f;
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (threadIdx.x + NT * q < pieces)
#pragma unroll
      for (int e = 0; e < E; ++e) ss += xr[q][e] * xr[q][e];
  const float rstd = 1.0f / sqrtf(block_sum<NT>(ss, part[1]) / (float)p.d + p.eps);
  char* n = static_cast<char*>(p.n) + row * p.n_t * ES;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int i = threadIdx.x + NT * q;
    if (i >= pieces) continue;
    float w[E], o[E];
    gains<E>(p.weight, i, w);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = w[e] * (xr[q][e] * rstd);
    store<BF16, E>(n, i, o);
  }
}

template <bool BF16, int E, int NT, int PER>
hipError_t run(const ResidualNormParams& p, hipStream_t st) {
  constexpr int64_t kRows = 1 << 21;  // a launch
  static_assert(kRows * NT < (int64_t)1 << 32, "threads of a launch");
  auto from = [](auto* t, int64_t elements) {
    using V = std::conditional_t<std::is_const_v<std::remove_pointer_t<decltype(t)>>, const char, char>;
    return t ? static_cast<V*>(t) + elements * (BF16 ? 2 : 4) : nullptr;
  };
  for (int64_t row = 0; row < p.T; row += kRows) {
    ResidualNormParams q = p;
    q.T = std::min(kRows, p.T - row);
    q.x = from(p.x, row * p.x_t), q.branch = from(p.branch, row * p.b_t), q.gate = from(p.gate, row * p.g_t);
    q.r = from(p.r, row * p.r_t), q.n = from(p.n, row * p.n_t);
    hipLaunchKernelGGL((residual_norm_kernel<BF16, E, NT, PER>), dim3((unsigned)q.T), dim3(NT), 0, st, q);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_residual_norm(const ResidualNormParams& p, bool bf16, bool vec, hipStream_t st) {
  if (p.T <= 0) return hipSuccess;
  // The fewest pieces a thread that 256 threads hold, more threads above.
  const int pieces = vec ? p.d / (bf16 ? 8 : 4) : p.d;
  if (!vec) {
    if (pieces <= 4096) return bf16 ? run<true, 1, 512, 8>(p, st) : run<false, 1, 512, 8>(p, st);
    return bf16 ? run<true, 1, 1024, 32>(p, st) : run<false, 1, 1024, 32>(p, st);
  }
  if (bf16) {
    if (pieces <= 256) return run<true, 8, 256, 1>(p, st);
    if (pieces <= 512) return run<true, 8, 256, 2>(p, st);
    if (pieces <= 1024) return run<true, 8, 256, 4>(p, st);
    return run<true, 8, 1024, 4>(p, st);
  }
  if (pieces <= 256) return run<false, 4, 256, 1>(p, st);
  if (pieces <= 1024) return run<false, 4, 256, 4>(p, st);
  if (pieces <= 4096) return run<false, 4, 1024, 4>(p, st);
  return run<false, 4, 1024, 8>(p, st);
}

}  // namespace svdmlp
