// Operators over a paged cache of 8- or 4-bit codes, and the verification of
// drafted tokens: the checked arguments as the kernels take them, and the launchers.
#pragma once

#include "common.hpp"
#include "paged.hpp"

namespace jal {

// A head's row below the first of these is stored as zeros, one that reaches the
// second (or holds a NaN) as NaN: its scale and the scale's inverse stay normal.
constexpr float kQuantLeast = 0x1p-100f, kQuantMost = 0x1p100f;

// Scales: f32 at page * s_page + head * s_head + slot.  The codes' places are a
// PagedView whose strides are bytes.
struct QuantScales {
  const float *k, *v;
  int64_t s_page, s_head;
};

// Launches a kernel that may start while the launch before it still runs: every block
// waits (pdl_wait()) before it looks at what that can have written, so what is saved is the
// way of the launch itself (about 1.5 us of a short call).
template <class F, class... A>
void launch_beside(F kernel, int64_t blocks, int threads, int smem, cudaStream_t s, const A &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  JAL_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
}

struct QuantAppendParams {
  AppendParams a;
  float *ks, *vs;
  int64_t s_page, s_head;
};
void launch_quant_kv_append(const QuantAppendParams &p, int bits, cudaStream_t s);

struct QuantAttnParams {
  AttnParams a;
  QuantScales sc;
};
struct QuantAttnPlan {
  int rows;  // query rows of a tile
  int tiles, splits;
  bool direct;
  size_t bytes;
};
QuantAttnPlan plan_quant_attention(const jal_quant_kv &kv, const jal_ragged_batch &b, size_t n_heads_q, int act,
                                   size_t window, size_t n_sink);
void launch_quant_attention(const QuantAttnParams &p, int bits, const QuantAttnPlan &plan, cudaStream_t s);

struct QuantReadParams {
  PagedView from, into;
  QuantScales sc;
  void *kw, *vw;
  const int32_t *first, *kv_len;
  int32_t n_seqs;
  int64_t max_len;
};
void launch_quant_kv_read(const QuantReadParams &p, int bits, cudaStream_t s);

struct VerifySums {
  double zx, zy, px, qx;  // sums of p and q over a part of the vocabulary; of p and q where p > q
};
struct VerifyParams {
  const void *logits, *draft;  // draft: null where drafts have no probabilities
  int64_t stride, draft_stride;
  const int32_t *q_start, *kv_len, *tokens;
  const float *uniform, *temperature, *draft_temperature;
  int32_t *out_tokens, *n_accepted, *new_len;
  VerifySums *parts;  // [n_seqs][parts of the vocabulary]
  float2 *part;       // [2][n_rows][chunks]: target's, then draft's
  int32_t *arrived;   // [n_seqs]: blocks that have left their sums
  int32_t n_seqs, n_rows, vocab, chunks, dtype;
};
// Pieces a row of logits is cut into.
int verify_chunks(size_t n_rows, size_t vocab);
// Bytes of the workspace; its places into p, where that is given.
size_t verify_workspace(size_t n_seqs, size_t n_rows, size_t vocab, VerifyParams *p, void *ws);
void launch_verify_drafts(const VerifyParams &p, cudaStream_t s);

}  // namespace jal
