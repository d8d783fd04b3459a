// Attention over chunks, of tiles of 128 rows (chunk_attention.hip): bf16 sequences of
// some tens of rows, and of many where chunk_pipe_kernel does not go (heads over
// 128, pages that its loads do not fit); all of fp32 heads over 128.
//
// Four waves of 32 rows share tiles of 32 keys in LDS; each loads a part of a tile,
// STAGES - 1 tiles ahead, and a barrier a tile keeps them together.  Against tiles
// of 32 rows the keys and values are read a quarter as often, and a start and an
// end are shared by four times the rows; heads of over 128 fit their queries into
// registers, with one wave a SIMD.
// Bound there by LDS, which 32 rows a wave read as long as they multiply, and the
// softmax behind it (the matrix unit is busy 28% of the time): 4000 tokens of 8
// heads of 256 165 us, 396 TFLOP/s; 1000 tokens each of 8 sequences of 8000, 583.
// fp32 heads of 256: 61% busy, 78 TFLOP/s.  64 sequences of 12 tokens, 2000 keys, heads of
// 128: 160 us, 3.3 TB/s.
#include "chunk.hpp"

namespace svdmlp {

namespace {

template <bool BF16_, int DP_, int STAGES_>
struct ShareCfg {
  static constexpr bool BF16 = BF16_;
  static constexpr int DP = DP_, ES = BF16 ? 2 : 4, RB = DP * ES, PIECES = RB / 16, STEPS = RB / 32, DB = DP / 32;
  static constexpr int NW = 4, ROWS = 32 * NW, KB = 32, TILE = KB * RB, STAGE = 2 * TILE, STAGES = STAGES_;
  static constexpr int RPL = 64 / PIECES, LOADS = KB / RPL, MINE = LOADS / NW;  // rows a load, loads of keys a tile, a wave's
  static_assert(MINE * NW == LOADS && STAGES >= 2, "every wave loads");
};

constexpr int kShareIds = 2048;  // pages whose numbers lie in LDS

template <class C>
__global__ __launch_bounds__(256, 1) void chunk_share_kernel(ChunkParams p, ChunkClass k) {
  constexpr bool BF16 = C::BF16;
  constexpr int ES = C::ES, RB = C::RB, DB = C::DB, KB = C::KB;
  __shared__ __attribute__((aligned(1024))) char lds[C::STAGES * C::STAGE];
  __shared__ int ids[kShareIds];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const attn_lds base = (attn_lds)lds;
  if (p.D < C::DP)  // pieces behind the head's end: never loaded, zeros
    for (int i = threadIdx.x; i < C::STAGES * C::STAGE / 16; i += 256) *reinterpret_cast<SVDMLP_ATTN_LDS u32x4*>(base + 16 * i) = u32x4{0u, 0u, 0u, 0u};

  __shared__ Kept kept;
  for (Walk walk;;) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // what follows from it is not kept over the pieces
    const int col = lane & 31, half = lane >> 5;
    Place w;
    Piece piece;
    if (!next_piece<true>(p, k, lane, (SVDMLP_ATTN_LDS Kept*)&kept, walk, w, piece)) return;
    const int G = p.Hq / p.Hk, npieces = p.D * ES / 16, row0 = w.tile * C::ROWS, rows = w.n * G, context = w.len - w.n;
    const int shared = context + row0 / G + 1;     // keys that every row sees
    const int rr = wave * 32 + col, r = min(row0 + rr, rows - 1);  // rows behind the last repeat it, and are not stored
    const int tok = r / G, last = context + tok;   // the row's last key
    const char* const kb = static_cast<const char*>(p.kc) + (int64_t)w.hk * p.k_h * ES;
    const char* const vb = static_cast<const char*>(p.vc) + (int64_t)w.hk * p.v_h * ES;
    const int* const table = p.table + (int64_t)w.b * p.table_b;
    const uint32_t cache_pages = (uint32_t)min(p.pages, (int64_t)0x7fffffff);
    auto valid = [&](int pg) { return (uint32_t)pg < cache_pages; };
    // Where registers are short, a lane's places in the tiles are computed for every tile.
    auto here = [&] {
      int x = lane;
      if constexpr (RB >= 1024) asm volatile("" : "+v"(x));
      return x;
    };

    u32x4 qf[C::STEPS];
    f32x16 o[DB];
    RowState st = {-INFINITY, 0.f};
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    uint32_t bad = 0;

    // Segments of as many keys as have their pages' numbers in LDS.
    const int most = segment_keys(kShareIds, p.page, KB);
    for (int kbeg = piece.kbeg; kbeg < piece.kend; kbeg += most) {
      const int kend = (int)min((int64_t)piece.kend, (int64_t)kbeg + most), tiles = (kend - kbeg + KB - 1) / KB;
      __syncthreads();  // (with what the last segment left in LDS)
      // The pages' numbers, and whether all are pages of the cache.  One that is not
      // holds no keys: page 0 is read for it, and masked.
      const int pg0 = page_of(p, kbeg), pages = page_of(p, kend - 1) - pg0 + 1;
      bool lost = false;
      for (int i0 = threadIdx.x; i0 < pages; i0 += 256 * 4) {
        int v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = table[pg0 + min(i0 + 256 * j, pages - 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lost |= !valid(v[j]);
          if (i0 + 256 * j < pages) ids[i0 + 256 * j] = valid(v[j]) ? v[j] : 0;
        }
      }
      const bool holes = __syncthreads_or(lost);
      const char* const qp = static_cast<const char*>(p.q) + ((int64_t)(w.start + tok) * p.q_t + (int64_t)(w.hk * G + r - tok * G) * p.q_h) * ES;
#pragma unroll
      for (int s = 0; s < C::STEPS; ++s) {
        const int c = 2 * s + half;
        qf[s] = c < npieces ? *reinterpret_cast<const u32x4*>(qp + 16 * c) : u32x4{0u, 0u, 0u, 0u};
      }
      // This wave's loads of tile t: MINE of keys and as many of values in any case.
      auto issue = [&](int t) {
        const uint32_t to = (uint32_t)(uintptr_t)(base + t % C::STAGES * C::STAGE) + wave * C::MINE * 1024;
        const int x = here(), lrow = wave * C::MINE * C::RPL + x / C::PIECES, lc = x % C::PIECES;
#pragma unroll
        for (int j = 0; j < C::MINE; ++j) {
          const int row = lrow + j * C::RPL, key = min(kbeg + t * KB + row, kend - 1), pg = page_of(p, key);
          const int64_t id = ids[pg - pg0], in = key - pg * p.page;
          const int ck = lc ^ k_swz<RB>(row), cv = lc ^ v_swz<RB, BF16>(row);
          if (ck < npieces) load_lds16(kb + (id * p.k_p + in * p.k_t) * ES + 16 * ck, to + j * 1024);
          if (cv < npieces) load_lds16(vb + (id * p.v_p + in * p.v_t) * ES + 16 * cv, to + C::TILE + j * 1024);
        }
      };
      // The loop's loads are counted (wait_loads): none of the above may be among them.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      for (int t = 0; t < C::STAGES - 1 && t < tiles; ++t) issue(t);

      // One tile: S = K Q^T, the weights, O += V^T P^T.  Pieces are read from LDS
      // kAhead products before they are needed, the first of V behind the weights.
      auto unit = [&](auto masked_, int t) {
        constexpr bool masked = decltype(masked_)::value;
        // Every wave's part of tile t is there, and every wave is done with tile t - 1,
        // whose place is filled again.
        if (t + C::STAGES - 2 < tiles) wait_loads<(C::STAGES - 2) * 2 * C::MINE>();
        else wait_loads<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + C::STAGES - 1 < tiles) issue(t + C::STAGES - 1);
        const attn_lds lk = base + t % C::STAGES * C::STAGE, lv = lk + C::TILE;
        const TileLane<RB, BF16> at(here());
        const int ku = kbeg + t * KB;
        constexpr int kAhead = RB < 1024 ? 4 : 2, VF = BF16 ? 2 * DB : 16 * DB;  // VF: pieces of V
        u32x4 kf[kAhead], vf[kAhead];
        auto read_value = [&](int f) {
          if constexpr (BF16) vf[f % kAhead] = at.values(lv, f / DB, f % DB);
          else vf[f % kAhead].x = at.value(lv, f / DB, f % DB);
        };
#pragma unroll
        for (int s = 0; s < kAhead; ++s) kf[s] = at.key(lk, s);
        f32x16 s = {};
#pragma unroll
        for (int x = 0; x < C::STEPS; ++x) {
          __builtin_amdgcn_sched_barrier(0);
          s = attn_mfma<BF16>(kf[x % kAhead], qf[x], s);
          if (x + kAhead < C::STEPS) kf[x % kAhead] = at.key(lk, x + kAhead);
          else read_value(x + kAhead - C::STEPS);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (masked) {
          const int n = min(last, kend - 1) - ku + 1;
          uint32_t see = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
          if (holes) see &= (uint32_t)__ballot(valid(table[page_of(p, min(ku + col, kend - 1))]));
          see >>= 4 * half;
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
      };
      // Whole tiles that every row of the block sees; then the others, masked.
      int t = 0;
      if constexpr (RB < 1024) {  // (else two copies of a tile's code do not fit the registers)
        const int whole = holes ? 0 : max(min(shared, kend) - kbeg, 0) / KB;
        for (; t < whole; ++t) unit(std::false_type{}, t);
      }
      for (; t < tiles; ++t) unit(std::true_type{}, t);
    }

    const ChunkParams& e = args_again();
    const float l = st.l + __shfl_xor(st.l, 32), inv = piece.whole ? inverse_sum(l) : 1.f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] *= inv;
    // Infinities and NaN among the values of masked tiles were taken as zeros, for
    // the rows that do not see them; the rows that do get them here.  (Those of
    // other tiles add to what they hold already.)
    if (__any(bad != 0)) {
      for (int key = piece.kbeg; key < piece.kend; ++key) {
        const int pg = page_of(e, key), id = table[pg];
        if (!valid(id)) continue;
        const char* const vp = vb + ((int64_t)id * e.v_p + (int64_t)(key - pg * e.page) * e.v_t) * ES;
        auto value = [&](int x) -> uint32_t {
          return BF16 ? (uint32_t)reinterpret_cast<const uint16_t*>(vp)[x] << 16 : reinterpret_cast<const uint32_t*>(vp)[x];
        };
        bool any = false;
        for (int x = lane; x < e.D; x += 64) any |= not_finite<false>(value(x)) != 0;
        if (!__any(any)) continue;
        const uint32_t see = key <= last ? 0xffffffffu : 0u;
        int D = e.D;
        asm volatile("" : "+s"(D));  // its comparisons stay in the loop: hoisted, they spill
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int x = 32 * d + 8 * (i >> 2) + 4 * half + (i & 3);
            const uint32_t v = x >= D ? 0u : value(x);
            o[d][i] += __uint_as_float(v & not_finite<false>(v) & see);
          }
      }
    }
    if (row0 + rr < rows) {
      float* const sums = piece.whole ? nullptr : sums_of(e, k, walk.block, piece.from == 0);
      const int64_t out = (int64_t)(w.start + tok) * e.o_t + (int64_t)(w.hk * G + (r - tok * G)) * e.o_h;
      if (sums && half == 0) reinterpret_cast<f32x2*>(sums + C::ROWS * e.D)[rr] = f32x2{st.m, l};
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int x = 32 * d + 8 * b + 4 * half;
          if (x >= e.D) continue;
          const f32x4 v = {o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
          if (sums) reinterpret_cast<f32x4*>(sums)[(x >> 2) * C::ROWS + rr] = v;
          else store4<BF16>(e.out, out + x, v);
        }
    }
  }
}

template <bool BF16, int DP, int STAGES>
void run(const ChunkParams& p, const ChunkClass& k, hipStream_t st) {
  hipLaunchKernelGGL((chunk_share_kernel<ShareCfg<BF16, DP, STAGES>>), dim3((unsigned)k.grid), dim3(256), 0, st, p, k);
}

}  // namespace

// Stages for two blocks a CU (plan_chunk_attention takes two of heads up to 128), or
// for one where a wave takes over half of a SIMD's registers.
void launch_chunk_shared(const ChunkParams& p, const ChunkClass& k, bool bf16, hipStream_t st) {
  if (bf16) p.D <= 64 ? run<true, 64, 4>(p, k, st) : p.D <= 128 ? run<true, 128, 4>(p, k, st) : run<true, 256, 4>(p, k, st);
  else run<false, 256, 2>(p, k, st);  // (shorter heads: chunk_wave_kernel)
}

}  // namespace svdmlp
