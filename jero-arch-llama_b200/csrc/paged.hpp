// Paged batch operators: the checked arguments of the C entry points as the
// kernels take them, and the launchers.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "jal.h"

namespace jal {

constexpr int kPagedSMs = 148;          // B200: what the splits of a call are sized for
constexpr int kPagedMaxHeadDim = 256;   // head_dim: multiples of 8 up to this
constexpr int kPagedMaxSplits = 64;     // most pieces the keys of one row are cut into

// The cache as the kernels read it: element (page, head, slot, d) of a pool at
// page * page_stride + head * head_stride + slot * slot_stride + d.
struct PagedView {
  const void *k, *v;
  const int32_t *table;
  int64_t page_stride, head_stride, slot_stride;
  int32_t n_pages, page_size, page_shift;  // page_shift: log2 of page_size, or -1
  int32_t max_pages, hkv, hd, dtype;
  int32_t cap;  // max_pages * page_size: positions a table row has
};

// The arguments of the C entry points, checked, with their defaults filled in.
jal_paged_kv checked_kv(const jal_paged_kv *in);
PagedView view_of(const jal_paged_kv &kv);

struct AttnParams {
  PagedView kv;
  const void *q;
  void *out;
  const int32_t *q_start, *kv_len;
  const int32_t *group_start, *prefix_len;  // shared prefixes, or null
  int64_t q_stride, out_stride;             // elements between rows
  int32_t n_seqs, n_rows, max_q, n_groups;
  int32_t G, hq, act;                       // query heads per KV head, query heads, dtype of q / out
  int32_t window, n_sink;
  int32_t splits, prefix_splits;            // pieces of a sequence's own keys; of a shared prefix's (0: read by each)
  int32_t tiles, prefix_tiles;              // row tiles of a sequence; of a group
  float scale_log2;                         // softmax scale * log2(e)
  float *part_o;                            // [slot][n_rows][hq][hd], unnormalised
  float2 *part_ml;                          // [slot][n_rows][hq]: what the weights refer to (base 2), their sum
};

// How one call is cut; the workspace size follows from it.
struct AttnPlan {
  int rows;                    // query rows of a tile (a sequence's own keys)
  int prefix_rows;             // query rows of a tile (shared prefixes; 0 = none)
  int tiles, prefix_tiles, splits, prefix_splits;
  bool direct;                 // one piece per row: written straight to out
  size_t bytes;                // workspace
};
AttnPlan plan_attention(const jal_paged_kv &kv, const jal_ragged_batch &b, const jal_prefix_groups *g, size_t n_heads_q,
                        int act, size_t window, size_t n_sink);
void launch_paged_attention(AttnParams p, const AttnPlan &plan, cudaStream_t s);
// Into how many pieces the keys of `blocks` blocks' rows go, and the kernel that
// joins the pieces' results (launched behind the one that makes them).
int attention_pieces(int64_t blocks, int64_t keys, int resident, int64_t start_keys, bool joined);
void launch_attention_join(const AttnParams &p, int prefix_rows, cudaStream_t s);

struct AppendParams {
  PagedView kv;
  void *kw, *vw;  // the pools, writable
  const void *q, *k, *v;
  void *q_out;
  const float *inv_freq;
  const int32_t *q_start, *kv_len;
  int64_t q_stride, q_out_stride, kv_stride;
  int32_t n_seqs, n_rows, hq, act, rotary, neox;
};
void launch_rope_kv_append(const AppendParams &p, cudaStream_t s);

struct BeamParams {
  const void *logits;
  const float *cum;
  float *scores;
  int32_t *parents, *tokens;
  int64_t row_stride;
  int32_t n_seqs, n_beams, vocab, k, dtype, chunks;
  void *ws;
};
// Pieces a row of logits is cut into, and the workspace bytes of a selection.
int beam_chunks(size_t n_rows, size_t vocab);
size_t beam_workspace(size_t n_seqs, size_t n_beams, size_t vocab, size_t k);
// Whether the joining block of one sequence can take that many lists.
bool beam_fits(size_t n_beams, size_t vocab, size_t k);
void launch_beam_select(const BeamParams &p, cudaStream_t s);

struct ReorderParams {
  PagedView kv;
  void *kw, *vw;
  const int32_t *kv_len, *parents, *fresh;
  int32_t *new_table, *new_len;
  int64_t layer_stride;
  int32_t n_seqs, n_beams, n_layers;
};
void launch_beam_reorder(const ReorderParams &p, cudaStream_t s);

}  // namespace jal
