// Parameters and launchers of the operators around the MLP block of a decoder
// layer: rotary positions (rope.hip), attention over packed prompts
// (prompt_attention.hip), attention over a paged cache (cache_attention.hip),
// and the residual sum with the norms on both sides of a block (norm.hip).
// Strides are in elements; the last dimension of every tensor is contiguous.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace svdmlp {

// Whether one launch can have so many blocks: HIP cuts a grid of 2^32 threads or
// more to its low 32 bits, without an error.
inline bool fits_launch(int64_t blocks, int threads) { return blocks * threads < (int64_t)1 << 32; }

struct RopeParams {
  const void* q;  // (T, Hq, D)
  const void* k;  // (T, Hk, D)
  const void* v;  // (T, Hk, D), append only
  const int64_t* pos;      // (T)
  const double* inv_freq;  // (rot / 2)
  void* qo;  // (T, Hq, D)
  void* ko;  // (T, Hk, D), or the key cache (pages, page, Hk, D)
  void* vo;  // the value cache, append only
  const int64_t* slots;  // (T): page * page_size + row; null: ko is (T, Hk, D)
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;
  int64_t qo_t, qo_h;
  int64_t ko_p, ko_t, ko_h, vo_p, vo_t, vo_h;  // page, token and head strides of the outputs (page: append only)
  int64_t T, pages;
  int page, Hq, Hk, D, rot;
  float scale;  // on cos and sin
  int interleaved;
};
hipError_t launch_rope(const RopeParams& p, bool bf16, bool vec, hipStream_t st);

struct ResidualNormParams {
  const void* x;       // (T, d) the residual stream
  const void* branch;  // (T, d) the block's output, or null
  const float* post;   // (d) gains of the norm of the branch, or null
  const void* gate;    // (T, d) or (d) (g_t = 0), or null
  const float* weight; // (d) gains of the norm of r, or null
  void* r;             // (T, d), or null
  void* n;             // (T, d), or null
  int64_t x_t, b_t, g_t, r_t, n_t;
  int64_t T;
  int d;
  float scale, eps;
};
constexpr int kResidualNormMaxD = 32768;
hipError_t launch_residual_norm(const ResidualNormParams& p, bool bf16, bool vec, hipStream_t st);

struct PromptParams {
  const void *q, *k, *v;  // (T, Hq, D), (T, Hk, D) twice
  void* out;              // (T, Hq, D)
  const int* cu;          // (B + 1) first row of each sequence and the end of the last; null: one sequence of T rows
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h;
  int T, B, Hq, Hk, D;
  float c;  // softmax scale * log2(e)
  int causal;
};
hipError_t launch_prompt_attention(const PromptParams& p, bool bf16, int cus, hipStream_t st);

struct CacheParams {
  const void* q;          // (B, n, Hq, D)
  const void *kc, *vc;    // (pages, page, Hk, D)
  const int* table;       // (B, width) pages of each sequence in order
  const int* lengths;     // (B) tokens held, the n new ones among them
  const uint8_t* tree;    // (B, n, n) or (n, n) (tree_b = 0) bytes, or null: a chain
  void* out;              // (B, n, Hq, D)
  float* part;            // split partials, or null with splits == 1
  int* counters;          // one a (sequence, key/value head, row tile), zero before and after; null with splits == 1
  int64_t q_b, q_t, q_h, k_p, k_t, k_h, v_p, v_t, v_h, o_b, o_t, o_h, table_b, tree_b, tree_q;
  int64_t pages;
  int page, width, B, n, Hq, Hk, D;
  int page_shift;     // log2 of a page that is a power of two and holds whole loads, else -1 (set by the launcher)
  const int* cu;      // prompts only (wave_attention.hpp): their bounds, rows and mask; n, table, lengths unused
  int T, causal;
  int splits, chunk;  // keys are cut into chunks of `chunk` (a multiple of the key tile), one a block
  int chunk_most, chunks;  // shared tiles: the kernel's choice lies in chunk .. chunk_most; chunks in all, at most
  int slots;               // and the blocks that run at once
  float c;
};
// How a call is cut: `splits` chunks of `chunk` keys cover the table's
// `capacity`, a block of `waves` waves each; rtiles row tiles a sequence and head.
constexpr int64_t kTokenStrideMost = 1 << 23;  // a 64-row tile's byte offsets fit 31 bits, in both types
constexpr int64_t kCachePagesMost = 65536;  // pages of a sequence: 64 chunks of 1024
// Blocks of 128 rows (plan.shared) choose their chunk on the device, from the
// lengths: `chunk` to chunk_most keys (equal: no choice), `chunks` of them in all.
struct CachePlan {
  int splits, chunk, waves, rtiles, chunk_most, chunks, slots;
  bool shared;
};
CachePlan plan_cache_attention(int B, int n, int Hq, int Hk, int D, bool bf16, int page, int64_t capacity, int cus);
// Floats of the partial sums: D sums, the maximum and the sum of weights of
// every (token, head) of every chunk.
inline int64_t cache_part_floats(const CachePlan& plan, int n, int Hq, int D) {
  return plan.splits > 1 ? (int64_t)plan.chunks * n * Hq * (D + 2) : 0;
}
// Counters: one a (sequence, key/value head, row tile) whose last block joins the chunks.
inline int64_t cache_counters(const CachePlan& plan, int B, int Hk) {
  return plan.splits > 1 && !plan.shared ? (int64_t)B * Hk * plan.rtiles : 0;
}
hipError_t launch_cache_attention(const CacheParams& p, bool bf16, const CachePlan& plan, hipStream_t st);

}  // namespace svdmlp
