// Parameters and launchers of the operators around the MLP block of a decoder
// layer: rotary positions (rope.hip) and head norms before them (norm_rope.hip),
// attention over packed prompts (prompt_attention.hip), attention over a paged
// cache (cache_attention.hip), the residual sum with the norms on both sides of a
// block (norm.hip), and moves within a cache (cache_pages.hip).
// Strides are in elements; the last dimension of every tensor is contiguous.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "segments.hpp"

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

struct NormRopeParams {
  RopeParams r;
  const float *q_w, *k_w;  // gains: (D) or, with a stride, (heads, D)
  int64_t qw_h, kw_h;
  float eps;
};
hipError_t launch_norm_rope(const NormRopeParams& p, bool bf16, bool vec, hipStream_t st);

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

// Sequences whose rows (new tokens x heads of a group) number from .. upto take
// tiles of `rows` rows; their work is a line of units of 2^unit_log keys, of which a
// block takes at least `least`.
struct ChunkClass {
  int from, upto, rows, rows_log;
  int unit_log, slope, start, least;  // slope: a tile has so many units more than the one before it; start: as many as a tile's start and end take
  int step;                    // keys that a block takes at once
  int alike;                   // whether tiles of a sequence gain from being cut alike (Line::alone)
  int blocks, grid;            // parts of the line, blocks of the launch; 0: no sequence can be of the class
  int joins;                   // blocks that join the sums of tiles in several parts
  int fits;                    // whether units and tiles fit the kernels' numbers
  int64_t notes_at, part_at;   // from which float of the workspace on: a note a block, two tiles' sums a block
};
struct ChunkParams {
  const void* q;        // (T, Hq, D), sequence b's new tokens in rows cu[b] .. cu[b + 1]
  const void *kc, *vc;  // (pages, page, Hk, D)
  const int* table;     // (B, width)
  const int* lengths;   // (B) tokens held, the new ones last among them
  const int* cu;        // (B + 1)
  void* out;            // (T, Hq, D)
  float* part;
  int64_t q_t, q_h, k_p, k_t, k_h, v_p, v_t, v_h, o_t, o_h, table_b, pages;
  int page, width, T, B, Hq, Hk, D;
  uint32_t page_mul;  // x / page = umulhi(x, page_mul) >> page_shift, for x < 2^31 and a page of over one token
  int page_shift;
  int alike;  // keys and values have the same page and token strides, and those and a page are below 2^32 bytes
  float c;    // softmax scale * log2(e)
};
struct ChunkPlan {
  ChunkClass many, some, few;  // tiles of 256, 128 and 32 rows
  int64_t floats;              // of the workspace
};
// alike: ChunkParams::alike; a workspace for calls of either kind takes the larger plan.
ChunkPlan plan_chunk_attention(int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D, bool bf16, bool alike, int64_t page, int64_t capacity, int64_t cus);
void launch_chunk_waves(const ChunkParams& p, const ChunkClass& k, bool bf16, hipStream_t st);
void launch_chunk_shared(const ChunkParams& p, const ChunkClass& k, bool bf16, hipStream_t st);
hipError_t launch_chunk_attention(const ChunkParams& p, bool bf16, const ChunkPlan& plan, hipStream_t st);

// The caches (pages, page, Hk, D) of a model's layers, all laid out alike: as many
// as a launch's arguments hold.
constexpr int kCachesMost = 128;
struct CacheSet {
  void* base[kCachesMost];
  int64_t pages, p_s, t_s, h_s;  // strides in elements
  int n, es, page, Hk, D;        // es: bytes of an element
};
struct PageCopyParams {
  CacheSet c;
  const int *src, *dst, *rows;  // pages, and how many of a page's rows, or null: all
  int64_t first;                // of the launch's pages
  int row_units, head_units, parts;  // set by the launcher
};
hipError_t launch_copy_pages(const PageCopyParams& p, int64_t m, bool vec, hipStream_t st);

constexpr int kDraftsMost = 64;
struct DraftKeepParams {
  CacheSet c;
  const int* table;    // (B, width)
  const int* lengths;  // (B), the drafts last among the tokens
  const int* path;     // (B, m)
  int* new_lengths;    // (B)
  int64_t table_b;
  int width, B, m, drafts;
  int row_units, head_units, parts;  // set by the launcher
};
hipError_t launch_keep_drafts(const DraftKeepParams& p, bool vec, hipStream_t st);

}  // namespace svdmlp
