// What the attention kernels share (prompt_attention.hip, cache_attention.hip).
//
// A wave works on 32 rows (a row: one query token and one of the heads that
// share a key/value head) and 32 keys at a time, with 32 x 32 MFMA blocks:
//     S^T = K Q^T        rows of the result: keys, columns: query rows
//     O^T = V^T P^T      rows: head elements, columns: query rows
// so a lane holds one query row throughout (lane % 32; the halves of the wave
// share it, with 16 of the 32 keys each): the softmax statistics are the lane's
// own, one exchange between the halves apart, and the weights P leave the first
// product in the registers that the second one takes.  D of a 32 x 32 block:
// lane = 32 h + col, register i = 4 b + r is row 8 b + 4 h + r.  The second
// product's sum over keys may take them in any order, so key 8 b + 4 h + r is
// given the place that its weight already has.
//
// Statistics are in 32 bits, in the log2 domain: p = exp2(c s - m), c the scale
// times log2(e), off by at most 3 2^-24 of itself (both factors' rounding and
// the product's), beside the D roundings of the score's own sum.
// bf16: the weights are rounded to bf16 for the second product, whose operands
// are of that type (two parts a weight, for 16 bits, would make it half as many
// products again in all).  Each is off by at most 2^-8 of itself, so a result by
// 2^-8 of the weighted mean of |v - out|; with random keys and values results
// are off by 0.0020 to 0.0023 rms, by 0.0016 to 0.0017 from their own rounding
// alone.  The sum is of the rounded weights: values that all keys share come out
// as they are.
#pragma once

#include "common.hpp"

namespace svdmlp {

typedef float f32x16 __attribute__((ext_vector_type(16)));

#define SVDMLP_ATTN_LDS __attribute__((address_space(3)))
typedef SVDMLP_ATTN_LDS char* attn_lds;

typedef __bf16 attn_bf16x4 __attribute__((ext_vector_type(4)));

// Four rows of one column of a bf16 matrix in LDS: in each group of 16 lanes,
// lane i's address points at 4 elements of row i / 4, columns 4 (i % 4) ..,
// and it receives column i.
__device__ __forceinline__ u32x2 attn_read_tr(attn_lds p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((SVDMLP_ATTN_LDS attn_bf16x4*)(p)));
}

// One 32-byte step of the head (16 bf16 or 8 fp32 values): lane half h holds
// the step's 16-byte piece h of both operands.
template <bool BF16>
__device__ __forceinline__ f32x16 attn_mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
    return c;
  }
}

// Where the 16-byte piece c of a key row lies in its row of the LDS tile.
// RB: bytes of a row (128, 256, 512 or 1024).  K rows are read 16 bytes a
// lane, 16 lanes (256 bytes, all banks) a pass, of 16 different rows and one
// piece: the rows' pieces are spread over the 16 places.
template <int RB>
__device__ __forceinline__ int k_swz(int row) {
  return RB == 128 ? (row >> 1) & 7 : row & 15;
}
// V rows, bf16: a transposing read takes 64 bytes of 4 consecutive rows a
// pass; fp32: 128 bytes of two rows 4 apart.
template <int RB, bool BF16>
__device__ __forceinline__ int v_swz(int row) {
  if constexpr (BF16) return RB == 128 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
  else return ((row >> 2) & 1) << 3;
}

// A lane's places in a tile, relative to it: the swizzle moves pieces within
// 256 bytes (or the shorter row), so that a few offsets a lane, and constants,
// reach every piece.
template <int RB, bool BF16>
struct TileLane {
  static constexpr int KN = RB >= 256 ? 8 : RB / 32;
  static constexpr int VN = BF16 ? (RB >= 256 ? 4 : 2) : 2;
  int k[KN];  // the 16-byte piece of step t of key row lane % 32: k[t % KN] + 256 (t / KN)
  int v[VN];  // bf16: block d of rows 4 half .. + 3 (transposing): v[d % VN] + 64 VN (d / VN); fp32: of row 4 half

  __device__ __forceinline__ explicit TileLane(int lane) {
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int t = 0; t < KN; ++t) k[t] = col * RB + (((2 * t + half) ^ k_swz<RB>(col)) << 4);
#pragma unroll
    for (int d = 0; d < VN; ++d) {
      if constexpr (BF16) {
        const int l16 = lane & 15, row = 4 * half + (l16 >> 2);
        v[d] = row * RB + ((64 * d + 32 * ((lane >> 4) & 1) + 8 * (l16 & 3)) ^ (v_swz<RB, true>(row) << 4));
      } else {
        v[d] = 4 * half * RB + ((128 * d + 4 * col) ^ (v_swz<RB, false>(4 * half) << 4));
      }
    }
  }
  __device__ __forceinline__ u32x4 key(attn_lds tile, int t) const {
    return *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(tile + k[t % KN] + 256 * (t / KN));
  }
  // 16 keys from row 16 t on of 32 head elements from 32 d on, in the order of
  // the weights: rows 4 half .. + 3, then those + 8.
  __device__ __forceinline__ u32x4 values(attn_lds tile, int t, int d) const {
    attn_lds p = tile + v[d % VN] + 64 * VN * (d / VN) + 16 * t * RB;
    const u32x2 a = attn_read_tr(p), b = attn_read_tr(p + 8 * RB);
    return u32x4{a.x, a.y, b.x, b.y};
  }
  // fp32: element 32 d + lane % 32 of row 8 (i / 4) + 4 half + i % 4
  __device__ __forceinline__ uint32_t value(attn_lds tile, int i, int d) const {
    return *reinterpret_cast<SVDMLP_ATTN_LDS uint32_t*>(tile + v[d % VN] + 128 * VN * (d / VN) + (8 * (i >> 2) + (i & 3)) * RB);
  }
};

__device__ __forceinline__ float most_of(const f32x16& s) {
  float m = fmaxf(s[0], s[1]);
#pragma unroll
  for (int i = 2; i < 16; i += 2) m = fmaxf(fmaxf(m, s[i]), s[i + 1]);
  return m;
}

// All ones where a value (one fp32 or two bf16 a word) is an infinity or NaN;
// in integer arithmetic, since comparisons keep a scalar register pair each.
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (BF16) return ((((w >> 7) & 0x00ff00ffu) + 0x00010001u) >> 8 & 0x00010001u) * 0xffffu;
  else return 0u - ((((w >> 23) & 0xffu) + 1u) >> 8);
}

// Replaces infinities and NaN by zero; bad gets bits where there was one.
template <bool BF16>
__device__ __forceinline__ uint32_t scrub(uint32_t w, uint32_t& bad) {
  const uint32_t mask = not_finite<BF16>(w);
  bad |= mask;
  return w & ~mask;
}

// The softmax state of one query row (one lane of each half): m is the
// reference of the exponents (log2 domain), l the lane's half of the sum.
struct RowState {
  float m, l;
};

// The reference only has to be near the maximum: it is moved (and what was
// summed scaled) when a score exceeds it by more than this many powers of two,
// so that weights stay below 2^8 and sums far from overflow.
constexpr float kSlack = 8.0f;

// The rows of a block: sequence rows start .. start + len of the tensors, of
// key/value head hk, its rows row0 ...
struct RowTile {
  int start, len, hk, row0;
};

// The block's sequence and row tile; false: none.  Tiles of BM rows are numbered
// sequence by sequence, a sequence's last rows (the most keys of a causal call)
// first.  The grid covers the most tiles that B sequences of T rows can have.
__device__ __forceinline__ bool find_rows(const int* cu, int T, int B, int Hk, int G, int BM, int lane, RowTile& rt) {
  rt.hk = blockIdx.x % Hk;
  int tile = blockIdx.x / Hk;
  rt.start = 0;
  rt.len = T;
  if (cu) {
    rt.len = -1;
    for (int b0 = 0; b0 < B; b0 += 64) {
      const int b = b0 + lane;
      int s = 0, n = 0;
      if (b < B) {
        s = min(max(cu[b], 0), T);
        n = min(max(cu[b + 1], s), T) - s;
      }
      const int tiles = (int)(((int64_t)n * G + BM - 1) / BM);
      int before = tiles;  // inclusive prefix sum
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(before, o);
        if (lane >= o) before += v;
      }
      const uint64_t hit = __ballot(tile < before);
      if (hit) {
        const int i = __builtin_ctzll(hit);
        tile -= __builtin_amdgcn_readlane(before - tiles, i);
        rt.start = __builtin_amdgcn_readlane(s, i);
        rt.len = __builtin_amdgcn_readlane(n, i);
        break;
      }
      tile -= __builtin_amdgcn_readlane(before, 63);
    }
    if (rt.len < 0) return false;
  }
  const int tiles = (rt.len * G + BM - 1) / BM;
  if (tile >= tiles) return false;
  rt.row0 = (tiles - 1 - tile) * BM;
  return true;
}

// 16 bytes a lane from global memory straight to LDS, lane i's to base + 16 i.
// The compiler does not know of the load: wait_loads before the tile is read.
__device__ __forceinline__ void load_lds16(const void* p, uint32_t base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"((uint32_t)__builtin_amdgcn_readfirstlane((int)base)), "v"(p)
               : "memory");
}
// The same from a base that all lanes share and an offset of each.
__device__ __forceinline__ void load_lds16(const void* p, uint32_t offset, uint32_t base) {
  const uint64_t a = (uint64_t)p;
  const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"((uint32_t)__builtin_amdgcn_readfirstlane((int)base)), "v"(offset), "s"(u)
               : "memory");
}
// 4 bytes a lane, lane i's to base + 4 i.
__device__ __forceinline__ void load_lds4(const void* p, uint32_t base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :
               : "s"((uint32_t)__builtin_amdgcn_readfirstlane((int)base)), "v"(p)
               : "memory");
}
// Until at most N of the wave's loads are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N <= 63, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

typedef __bf16 bf16x2_dot __attribute__((ext_vector_type(2)));

// acc + both bf16 values of w.
__device__ __forceinline__ float add_pair(uint32_t w, float acc) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_dot, w), __builtin_bit_cast(bf16x2_dot, 0x3f803f80u), acc, false);
}

// 1 / l; a row without keys gives zeros, NaN stays.
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }

template <bool BF16>
__device__ __forceinline__ void store4(void* p, int64_t i, f32x4 v) {
  if constexpr (BF16)
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p) + i) = u32x2{pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w)};
  else
    *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = v;
}

}  // namespace svdmlp
