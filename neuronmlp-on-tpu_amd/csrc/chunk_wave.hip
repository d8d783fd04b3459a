// Attention over chunks, of tiles of 32 rows (chunk_attention.hip): sequences that
// generate, short chunks, and fp32 heads up to 128.
#include "chunk.hpp"

namespace svdmlp {

namespace {

// How a cache is read: whole loads in a page and keys and values laid out alike
// (kWhole: heads that fill their place too), or key by key.
enum CacheKind { kAny, kAlike, kWhole };

template <bool BF16_, int DP_, int NW_, CacheKind KIND_>
struct WaveCfg {
  static constexpr bool ALIKE = KIND_ != kAny, FULL = KIND_ == kWhole;
  static constexpr bool BF16 = BF16_;
  static constexpr int DP = DP_, NW = NW_, ES = BF16 ? 2 : 4, RB = DP * ES, PIECES = RB / 16, STEPS = RB / 32, DB = DP / 32;
  static constexpr int TILE = 32 * RB, STAGE = 2 * TILE;  // keys, values
  static constexpr int RPL = 64 / PIECES, LOADS = 32 / RPL;
  static constexpr bool QREG = DP < 256;  // the queries in registers, else in LDS
  static_assert(STAGE >= 32 * DP * 4, "a wave's sums fit its stage");
};

__device__ const u32x4 kNoKey = {0u, 0u, 0u, 0u};  // what lanes without a key load

// A block's waves share its rows: each takes every NW-th tile of 32 keys through
// LDS of its own, and their sums meet in LDS at the end.  A wave's next keys are on
// their way while it multiplies the values, its next values while it multiplies
// the keys, and the numbers of its pages a tile before.  Two blocks a CU (three of
// bf16 heads up to 64), so that one's start and end lie behind the other's
// products.  Two waves a block, twice as many blocks: bf16 heads of 128, 37 tokens
// 17.1 -> 20.4 us, 64 sequences that generate 149 -> 158; fp32 heads of 64, 701 tokens 66
// -> 71, 3200 tokens 452 -> 396.
template <class C>
__global__ __launch_bounds__(64 * C::NW, 1) void chunk_wave_kernel(ChunkParams p, ChunkClass k) {
  constexpr bool BF16 = C::BF16, QREG = C::QREG;
  constexpr int ES = C::ES, RB = C::RB, DB = C::DB, NW = C::NW, STEP = 32 * NW;
  __shared__ __attribute__((aligned(1024))) char lds[NW * C::STAGE];
  __shared__ __attribute__((aligned(16))) char qlds[QREG ? 16 : C::STEPS * 1024];
  __shared__ float stats[NW][32][2];
  __shared__ int ids[NW][2][64];  // the pages of a wave's next two tiles: a lane's key's
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = p.Hq / p.Hk, npieces = p.D * ES / 16;
  const attn_lds mine = (attn_lds)lds + wave * C::STAGE;

  __shared__ Kept kept;
  for (Walk walk;;) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // what follows from it is not kept over the pieces
    const int col = lane & 31, half = lane >> 5;
    Place w;
    Piece piece;
    if (!next_piece<false>(p, k, lane, (SVDMLP_ATTN_LDS Kept*)&kept, walk, w, piece)) return;
    const TileLane<RB, BF16> at(lane);
    const int lrow = lane / C::PIECES, lc = lane % C::PIECES;
    const int kpiece0 = lc ^ k_swz<RB>(lrow), vpiece0 = lc ^ v_swz<RB, BF16>(lrow);
    const uint32_t krow = (uint32_t)(lrow * (int)p.k_t * ES), vrow = (uint32_t)(lrow * (int)p.v_t * ES);
    const int row0 = w.tile * 32, rows = w.n * G, context = w.len - w.n, kend = piece.kend;
    const int shared = context + row0 / G + 1;  // keys that every row sees
    __syncthreads();                            // (with what the last piece left in LDS)

    u32x4 qf[QREG ? C::STEPS : 1];
    const int r = min(row0 + col, rows - 1);      // rows behind the last repeat it, and are not stored
    const int tok = r / G, last = context + tok;  // the row's last key
    {
      const char* const qp = static_cast<const char*>(p.q) + ((int64_t)(w.start + tok) * p.q_t + (int64_t)(w.hk * G + r - tok * G) * p.q_h) * ES;
      if constexpr (QREG)
#pragma unroll
        for (int s = 0; s < C::STEPS; ++s) {
          const int c = 2 * s + half;
          qf[s] = C::FULL || c < npieces ? *reinterpret_cast<const u32x4*>(qp + 16 * c) : u32x4{0u, 0u, 0u, 0u};
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
    if constexpr (!C::FULL)  // pieces behind the head's end: never loaded, zeros
      for (int i = lane; i < C::STAGE / 16; i += 64) *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(mine + 16 * i) = u32x4{0u, 0u, 0u, 0u};

    const char* const kb = static_cast<const char*>(p.kc) + (int64_t)w.hk * p.k_h * ES;
    const char* const vb = static_cast<const char*>(p.vc) + (int64_t)w.hk * p.v_h * ES;
    const int* const table = p.table + (int64_t)w.b * p.table_b;
    uint32_t bad = 0;

    // The key that a lane looks up of the tile at ku, one that is there: alike, lane j
    // load j's, else lane i key i.
    auto page_number = [&](int key) { return C::ALIKE ? page_of_many(p, key) : page_of(p, key); };
    auto key_of = [&](int ku) {
      return C::ALIKE ? min(ku + lane % C::LOADS * C::RPL, (kend - 1) / C::RPL * C::RPL) : min(ku + col, kend - 1);
    };
    auto ask_pages = [&](int ku, int slot) {
      load_lds4(table + page_number(key_of(min(ku, kend - 1))), (uint32_t)(uintptr_t)(attn_lds)&ids[wave][slot][0]);
    };
    const uint32_t pages = (uint32_t)min(p.pages, (int64_t)0x7fffffff);
    auto valid = [&](int id) { return (uint32_t)id < pages; };
    // Which keys of a tile are there: a page outside the cache holds none (page 0,
    // for whole loads, or zeros are loaded for it, and masked).
    auto keys_there = [&](int ku, int id) -> uint32_t {
      uint32_t seen = ku + 32 <= kend ? 0xffffffffu : (1u << (kend - ku)) - 1u;
      const uint32_t lost = (uint32_t)__ballot(!valid(id));
      if constexpr (!C::ALIKE) return seen & ~lost;
      if (lost & (uint32_t)((1ull << C::LOADS) - 1))
#pragma unroll 1
        for (int j = 0; j < C::LOADS; ++j)
          if (lost >> j & 1u) seen &= ~((uint32_t)((1ull << C::RPL) - 1) << (j * C::RPL));
      return seen;
    };
    // The loads of a tile's keys or values (row, its rows' part of the address; swz:
    // where load j's pieces lie), LOADS of them in any case.
    auto ask = [&](const char* base, int64_t p_s, int64_t t_s, uint32_t row, int piece0, auto swz, attn_lds to, int ku, int id) {
      const uint32_t lds_at = (uint32_t)(uintptr_t)to;
      // where registers are short, the loads' offsets are computed each time
      if constexpr (RB >= 256) asm volatile("" : "+v"(piece0));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last reads there are done
      if constexpr (C::ALIKE) {
        const int key = key_of(ku);
        // (page strides and pages are below 2^32 bytes)
        const int64_t off = (int64_t)((uint64_t)(uint32_t)(valid(id) ? id : 0) * (uint32_t)(p_s * ES) + (uint32_t)(key - page_number(key) * p.page) * (uint32_t)(t_s * ES));
#pragma unroll
        for (int j = 0; j < C::LOADS; ++j) {
          const int c = piece0 ^ swz(j * C::RPL);
          const int64_t a = lane_of(off, j);
          if (C::FULL || c < npieces) load_lds16(base + a, row + 16 * c, lds_at + j * 1024);
        }
      } else {
#pragma unroll 1
        for (int j = 0; j < C::LOADS; ++j) {
          const int x = j * C::RPL + lrow, page = __shfl(id, x), key = min(ku + x, kend - 1), c = lc ^ swz(x);
          const char* const src = valid(page) ? base + ((int64_t)page * p_s + (int64_t)(key - page_of(p, key) * p.page) * t_s) * ES + 16 * c
                                              : reinterpret_cast<const char*>(&kNoKey);
          if (c < npieces) load_lds16(src, lds_at + j * 1024);
        }
      }
    };
    auto ask_keys = [&](int ku, int id) { ask(kb, p.k_p, p.k_t, krow, kpiece0, [](int x) { return k_swz<RB>(x); }, mine, ku, id); };
    auto ask_values = [&](int ku, int id) { ask(vb, p.v_p, p.v_t, vrow, vpiece0, [](int x) { return v_swz<RB, BF16>(x); }, mine + C::TILE, ku, id); };

    int ku = piece.kbeg + 32 * wave, slot = 0;
    uint32_t seen = 0;
    // The loop's loads are counted (wait_loads): none of the above may be among them.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (ku < kend) {
      ask_pages(ku, 0);
      ask_pages(ku + STEP, 1);
      wait_loads<0>();
      const int id = ids[wave][0][lane];
      seen = keys_there(ku, id);
      ask_keys(ku, id);
      ask_values(ku, id);
    }
    if constexpr (!QREG) __syncthreads();

    // One tile: S = K Q^T, the weights, O += V^T P^T.  Pieces are read from LDS
    // kAhead products before they are needed.  masked: not every row sees every key
    // of it; infinities and NaN among its values are taken as zeros, for those that
    // do not, and the others get them at the end.
    auto unit = [&](auto masked_) {
      constexpr bool masked = decltype(masked_)::value;
      constexpr int kAhead = 4, VF = BF16 ? 2 * DB : 16 * DB;  // VF: pieces of V
      u32x4 kf[kAhead], vf[kAhead], qa[kAhead];
      auto read_query = [&](int t) { return *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>((attn_lds)qlds + (t * 64 + lane) * 16); };
      auto read_value = [&](int f) {
        if constexpr (BF16) vf[f % kAhead] = at.values(mine + C::TILE, f / DB, f % DB);
        else vf[f % kAhead].x = at.value(mine + C::TILE, f / DB, f % DB);
      };
      const int next = ku + STEP;
      const bool more = next < kend;
      wait_loads<C::LOADS>();  // all but the values: the keys are there, and the next pages
#pragma unroll
      for (int t = 0; t < kAhead; ++t) {
        kf[t] = at.key(mine, t);
        if constexpr (!QREG) qa[t] = read_query(t);
      }
      f32x16 s = {};
#pragma unroll
      for (int t = 0; t < C::STEPS; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        s = attn_mfma<BF16>(kf[t % kAhead], QREG ? qf[QREG ? t : 0] : qa[t % kAhead], s);
        if (t + kAhead < C::STEPS) {
          kf[t % kAhead] = at.key(mine, t + kAhead);
          if constexpr (!QREG) qa[t % kAhead] = read_query(t + kAhead);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      int id = 0;
      if (more) {
        slot ^= 1;
        id = ids[wave][slot][lane];
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(id)::"memory");  // before its place is filled again
        ask_pages(next + STEP, slot ^ 1);
        ask_keys(next, id);
        wait_loads<C::LOADS + 1>();  // the values are there
      } else {
        wait_loads<0>();
      }
#pragma unroll
      for (int f = 0; f < kAhead; ++f) read_value(f);
      if constexpr (masked) {
        const int n = last - ku + 1;
        const uint32_t see = (seen & (n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = see >> (8 * (i >> 2) + (i & 3)) & 1u ? s[i] : -INFINITY;
      }
      float mx = most_of(s) * p.c;
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
      ku = next;
      if (more) {
        ask_values(next, id);
        seen = keys_there(next, id);
      }
    };
    // Whole tiles that every row sees, up to the first that is not; then the others,
    // masked.  (Two loops: a branch in one kept the registers of both.)
    while (ku + 31 < min(shared, kend) && seen == 0xffffffffu) unit(std::false_type{});
    const int masked_from = ku;
    while (ku < kend) unit(std::true_type{});

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
          const int c = 8 * d + 2 * q + half;
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = o[d][4 * q + e] * a;
          *reinterpret_cast<SVDMLP_ATTN_LDS f32x4*>(mine + (col * OP + (c ^ (col & OM))) * 16) = v;
        }
    }
    if (__any(bad != 0)) {
      for (int kt = masked_from; kt < kend; kt += STEP)
        for (int key = kt; key < min(kt + 32, kend); ++key) {
          const int id = table[page_of(p, key)];
          if (!valid(id)) continue;
          const char* const vp = vb + ((int64_t)id * p.v_p + (int64_t)(key - page_of(p, key) * p.page) * p.v_t) * ES;
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
    __syncthreads();
    const ChunkParams& e = args_again();
    float* const sums = piece.whole ? nullptr : sums_of(e, k, walk.block, piece.from == 0);
    for (int i = threadIdx.x; i < 32 * OP; i += 64 * NW) {
      // (sums go out row by row, results piece by piece of a row)
      const int rr = piece.whole ? i / OP : i % 32, c = piece.whole ? i % OP : i / 32, row = row0 + rr;
      if (row >= rows || 4 * c >= e.D) continue;
      float m = -INFINITY, sum = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NW; ++x) m = fmaxf(m, stats[x][rr][0]);
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        const float mw = stats[x][rr][0];
        sum += mw == -INFINITY ? stats[x][rr][1] : stats[x][rr][1] * exp2f(mw - m);
        v += *reinterpret_cast<SVDMLP_ATTN_LDS f32x4*>((attn_lds)lds + x * C::STAGE + (rr * OP + (c ^ (rr & OM))) * 16);
      }
      if (piece.whole) {
        v *= inverse_sum(sum);
        const int t = row / G;
        store4<BF16>(e.out, (int64_t)(w.start + t) * e.o_t + (int64_t)(w.hk * G + row - t * G) * e.o_h + 4 * c, v);
      } else {
        reinterpret_cast<f32x4*>(sums)[c * 32 + rr] = v;
        if (c == 0) reinterpret_cast<f32x2*>(sums + 32 * e.D)[rr] = f32x2{m, sum};
      }
    }
  }
}

template <bool BF16, int DP, int NW>
void run(const ChunkParams& p, const ChunkClass& k, hipStream_t st) {
  const dim3 grid((unsigned)k.grid), block(64 * NW);
  const bool alike = p.alike && p.page % WaveCfg<BF16, DP, NW, kAlike>::RPL == 0 && p.page > 1;
  if (!alike) hipLaunchKernelGGL((chunk_wave_kernel<WaveCfg<BF16, DP, NW, kAny>>), grid, block, 0, st, p, k);
  else if (p.D < DP) hipLaunchKernelGGL((chunk_wave_kernel<WaveCfg<BF16, DP, NW, kAlike>>), grid, block, 0, st, p, k);
  else hipLaunchKernelGGL((chunk_wave_kernel<WaveCfg<BF16, DP, NW, kWhole>>), grid, block, 0, st, p, k);
}

}  // namespace

void launch_chunk_waves(const ChunkParams& p, const ChunkClass& k, bool bf16, hipStream_t st) {
  if (bf16) p.D <= 64 ? run<true, 64, 4>(p, k, st) : p.D <= 128 ? run<true, 128, 4>(p, k, st) : run<true, 256, 2>(p, k, st);
  else p.D <= 64 ? run<false, 64, 4>(p, k, st) : run<false, 128, 2>(p, k, st);  // (heads of over 128: chunk_share_kernel)
}

}  // namespace svdmlp
