// C entry points of the paged batch operators: arguments are checked here, on
// the host, before anything is enqueued.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "common.hpp"
#include "jal.h"
#include "paged.hpp"

using namespace jal;

namespace {

constexpr uint64_t kMaxPositions = 0x7fffffffull - 65536;  // tiles run past the last position by less than 65536
constexpr uint64_t kMaxInt = 0x7fffffffull;

bool float_type(int t) { return t == JAL_F32 || t == JAL_F16 || t == JAL_BF16; }
size_t type_bytes(int t) { return t == JAL_F32 ? 4 : 2; }

// `p` is memory of the current device: a tensor of another device, or of the
// host, would fault in the kernel.
void on_device(const void *p, const char *what, int device) {
  cudaPointerAttributes a = {};
  JAL_CUDA(cudaPointerGetAttributes(&a, p));
  if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
    fail(JAL_ERR_INVALID_ARGUMENT, "%s is not device memory", what);
  if (a.type == cudaMemoryTypeDevice && a.device != device)
    fail(JAL_ERR_INVALID_ARGUMENT, "%s is on device %d, the current device is %d", what, a.device, device);
}
int current_device() {
  int d = 0;
  JAL_CUDA(cudaGetDevice(&d));
  return d;
}
void aligned16(const void *p, const char *what) {
  if ((uintptr_t)p % 16) fail(JAL_ERR_TENSOR_BOUNDS, "%s is not 16-byte aligned", what);
}
// Arrays that kernels read and write as 4-byte values: an address between two of
// them would fault.
void aligned4(const void *p, const char *what) {
  if ((uintptr_t)p % 4) fail(JAL_ERR_TENSOR_BOUNDS, "%s is not 4-byte aligned", what);
}

// A cache view with its defaults filled in.
jal_paged_kv checked_kv(const jal_paged_kv *in) {
  NEED(in);
  jal_paged_kv kv = *in;
  NEED(kv.k);
  NEED(kv.v);
  NEED(kv.page_table);
  if (!float_type(kv.dtype)) fail(JAL_ERR_CAPABILITY_MISMATCH, "paged cache of type %d", kv.dtype);
  if (kv.head_dim == 0 || kv.head_dim % 8 || kv.head_dim > (uint64_t)kPagedMaxHeadDim)
    fail(JAL_ERR_CAPABILITY_MISMATCH, "head_dim %llu: multiples of 8 up to %d", (unsigned long long)kv.head_dim,
         kPagedMaxHeadDim);
  if (kv.n_heads_kv == 0 || kv.n_heads_kv > 65535 || kv.page_size == 0 || kv.n_pages == 0 || kv.max_pages == 0)
    fail(JAL_ERR_TENSOR_BOUNDS, "paged cache without heads, pages or slots");
  if (kv.n_pages > kMaxInt || kv.page_size > kMaxPositions || kv.max_pages > kMaxPositions / kv.page_size ||
      kv.n_seqs > kMaxInt)
    fail(JAL_ERR_TENSOR_BOUNDS, "paged cache: more than 2^31 pages, positions or sequences");
  if (!kv.page_stride && !kv.head_stride && !kv.slot_stride) {
    kv.slot_stride = kv.head_dim;
    kv.head_stride = kv.page_size * kv.slot_stride;
    kv.page_stride = kv.n_heads_kv * kv.head_stride;
  }
  if (kv.page_stride % 8 || kv.head_stride % 8 || kv.slot_stride % 8)
    fail(JAL_ERR_TENSOR_BOUNDS, "paged cache strides have to be multiples of 8");
  if (kv.page_size > 1 && kv.slot_stride < kv.head_dim)
    fail(JAL_ERR_TENSOR_BOUNDS, "slot stride %llu, head_dim %llu", (unsigned long long)kv.slot_stride,
         (unsigned long long)kv.head_dim);
  const uint64_t most = 1ull << 40;
  if (kv.page_stride > most || kv.head_stride > most || kv.slot_stride > most)
    fail(JAL_ERR_TENSOR_BOUNDS, "paged cache stride above 2^40");
  aligned16(kv.k, "k pool");
  aligned16(kv.v, "v pool");
  aligned4(kv.page_table, "page_table");
  return kv;
}

PagedView view_of(const jal_paged_kv &kv) {
  PagedView v = {};
  v.k = kv.k;
  v.v = kv.v;
  v.table = kv.page_table;
  v.page_stride = (int64_t)kv.page_stride;
  v.head_stride = (int64_t)kv.head_stride;
  v.slot_stride = (int64_t)kv.slot_stride;
  v.n_pages = (int32_t)kv.n_pages;
  v.page_size = (int32_t)kv.page_size;
  v.page_shift = -1;
  if ((kv.page_size & (kv.page_size - 1)) == 0)
    for (v.page_shift = 0; (1ull << v.page_shift) < kv.page_size;) v.page_shift++;
  v.max_pages = (int32_t)kv.max_pages;
  v.hkv = (int32_t)kv.n_heads_kv;
  v.hd = (int32_t)kv.head_dim;
  v.dtype = kv.dtype;
  v.cap = (int32_t)(kv.max_pages * kv.page_size);
  return v;
}

jal_ragged_batch checked_batch(const jal_ragged_batch *in, const jal_paged_kv &kv) {
  NEED(in);
  jal_ragged_batch b = *in;
  NEED(b.q_start);
  NEED(b.kv_len);
  aligned4(b.q_start, "q_start");
  aligned4(b.kv_len, "kv_len");
  if (b.n_seqs > kv.n_seqs)
    fail(JAL_ERR_TENSOR_BOUNDS, "batch of %llu sequences over a table of %llu", (unsigned long long)b.n_seqs,
         (unsigned long long)kv.n_seqs);
  if (b.n_rows > kMaxPositions) fail(JAL_ERR_TENSOR_BOUNDS, "batch of 2^31 rows or more");
  if (b.max_q_len > b.n_rows) b.max_q_len = b.n_rows;
  b.max_kv_len = std::min<uint64_t>(std::max<uint64_t>(b.max_kv_len, 1), kv.max_pages * kv.page_size);
  return b;
}

void check_act(int dtype, const jal_paged_kv &kv) {
  if (!float_type(dtype) || (dtype != kv.dtype && dtype != JAL_F32))
    fail(JAL_ERR_CAPABILITY_MISMATCH, "rows of type %d over a cache of type %d (the cache's type or f32)", dtype,
         kv.dtype);
}

int64_t row_stride(size_t stride, size_t width, const char *what) {
  if (stride == 0) stride = width;
  if (stride < width || stride % 8 || stride > (1ull << 40))
    fail(JAL_ERR_TENSOR_BOUNDS, "%s stride %zu: a multiple of 8, at least %zu", what, stride, width);
  return (int64_t)stride;
}

void check_heads(size_t hq, const jal_paged_kv &kv, const jal_ragged_batch &b) {
  if (hq == 0 || hq % kv.n_heads_kv || hq > 65535)
    fail(JAL_ERR_CAPABILITY_MISMATCH, "%zu query heads over %llu KV heads", hq, (unsigned long long)kv.n_heads_kv);
  if (b.n_rows * (hq / kv.n_heads_kv) > kMaxPositions)  // (row, head of the group) pairs are counted in 32 bits
    fail(JAL_ERR_TENSOR_BOUNDS, "batch of 2^31 rows times heads of a group or more");
}

jal_prefix_groups checked_groups(const jal_prefix_groups *in, const jal_paged_kv &kv, const jal_ragged_batch &b) {
  NEED(in);
  jal_prefix_groups g = *in;
  if (g.n_groups) {
    NEED(g.group_start);
    NEED(g.prefix_len);
    aligned4(g.group_start, "group_start");
    aligned4(g.prefix_len, "prefix_len");
  }
  if (g.n_groups > kMaxInt) fail(JAL_ERR_TENSOR_BOUNDS, "more than 2^31 groups");
  g.max_group = std::min<uint64_t>(g.max_group, b.n_seqs);
  g.max_prefix_len = std::min<uint64_t>(g.max_prefix_len, kv.max_pages * kv.page_size);
  if (g.n_groups == 0 || g.max_prefix_len == 0 || g.max_group == 0) g.n_groups = 0;
  return g;
}

void check_grid(const AttnPlan &a, const jal_paged_kv &kv, const jal_ragged_batch &b, const jal_prefix_groups *g,
                size_t hq) {
  const double blocks = (double)kv.n_heads_kv * ((double)a.tiles * a.splits * (double)b.n_seqs +
                                                 (g ? (double)a.prefix_tiles * a.prefix_splits * (double)g->n_groups : 0));
  if (blocks > 2e9 || (!a.direct && std::min((double)b.n_rows, (double)b.n_seqs * (double)b.max_q_len) * (double)hq > 2e9))
    fail(JAL_ERR_CAPABILITY_MISMATCH, "batch too large for one launch");
}

void attention(const jal_paged_kv *kv_in, const jal_ragged_batch *batch, const jal_prefix_groups *groups, int dtype,
               const void *q, size_t hq, size_t q_stride, float scale, size_t window, size_t n_sink, void *out,
               size_t out_stride, void *ws, size_t ws_len, void *stream) {
  const jal_paged_kv kv = checked_kv(kv_in);
  const jal_ragged_batch b = checked_batch(batch, kv);
  jal_prefix_groups g = {};
  if (groups) g = checked_groups(groups, kv, b);
  check_act(dtype, kv);
  check_heads(hq, kv, b);
  NEED(q);
  NEED(out);
  const float scale_log2 = scale * 1.4426950408889634f;  // softmax by powers of two
  if (!std::isfinite(scale_log2)) fail(JAL_ERR_INVALID_ARGUMENT, "attention scale is not finite or too large");
  AttnParams p = {};
  p.kv = view_of(kv);
  p.q_stride = row_stride(q_stride, hq * kv.head_dim, "q");
  p.out_stride = row_stride(out_stride, hq * kv.head_dim, "out");
  aligned16(q, "q");
  aligned16(out, "out");
  if (q == out && p.q_stride != p.out_stride && b.n_rows > 1)
    fail(JAL_ERR_TENSOR_BOUNDS, "out is q with another stride");
  if (b.n_seqs == 0 || b.n_rows == 0 || b.max_q_len == 0) return;
  window = std::min<size_t>(window, kMaxInt);
  n_sink = std::min<size_t>(n_sink, kMaxInt);
  const AttnPlan plan = plan_attention(kv, b, g.n_groups ? &g : nullptr, hq, dtype, window, n_sink);
  check_grid(plan, kv, b, g.n_groups ? &g : nullptr, hq);
  if (plan.bytes) {
    NEED(ws);
    aligned16(ws, "workspace");
    if (ws_len < plan.bytes)
      fail(JAL_ERR_TENSOR_BOUNDS, "workspace of %zu bytes, %zu needed", ws_len, plan.bytes);
  }
  const int dev = current_device();
  on_device(q, "q", dev);
  on_device(out, "out", dev);
  on_device(kv.k, "k pool", dev);
  on_device(kv.v, "v pool", dev);
  on_device(kv.page_table, "page_table", dev);
  on_device(b.q_start, "q_start", dev);
  on_device(b.kv_len, "kv_len", dev);
  if (plan.bytes) on_device(ws, "workspace", dev);
  if (g.n_groups) {
    on_device(g.group_start, "group_start", dev);
    on_device(g.prefix_len, "prefix_len", dev);
  }
  p.q = q;
  p.out = out;
  p.q_start = b.q_start;
  p.kv_len = b.kv_len;
  p.group_start = g.n_groups ? g.group_start : nullptr;
  p.prefix_len = g.n_groups ? g.prefix_len : nullptr;
  p.n_seqs = (int32_t)b.n_seqs;
  p.n_rows = (int32_t)b.n_rows;
  p.max_q = (int32_t)b.max_q_len;
  p.n_groups = (int32_t)g.n_groups;
  p.hq = (int32_t)hq;
  p.G = (int32_t)(hq / kv.n_heads_kv);
  p.act = dtype;
  p.window = (int32_t)window;
  p.n_sink = (int32_t)n_sink;
  p.splits = plan.splits;
  p.prefix_splits = plan.prefix_splits;
  p.tiles = plan.tiles;
  p.prefix_tiles = plan.prefix_tiles;
  p.scale_log2 = scale_log2;
  p.part_o = (float *)ws;
  if (plan.bytes)
    p.part_ml = (float2 *)(p.part_o + (size_t)(plan.splits + plan.prefix_splits) * b.n_rows * hq * kv.head_dim);
  launch_paged_attention(p, plan, (cudaStream_t)stream);
}

}  // namespace

extern "C" {

int jal_op_rope_kv_append(const jal_paged_kv *kv_in, const jal_ragged_batch *batch, int dtype, const void *k,
                          const void *v, size_t kv_stride, const float *inv_freq, size_t rotary_dim, int neox,
                          const void *q, void *q_out, size_t n_heads_q, size_t q_stride, size_t q_out_stride,
                          void *stream) {
  return guard([&] {
    const jal_paged_kv kv = checked_kv(kv_in);
    const jal_ragged_batch b = checked_batch(batch, kv);
    check_act(dtype, kv);
    NEED(k);
    NEED(v);
    if (rotary_dim % 2 || rotary_dim > kv.head_dim)
      fail(JAL_ERR_CAPABILITY_MISMATCH, "rotary_dim %zu of head_dim %llu", rotary_dim, (unsigned long long)kv.head_dim);
    if (rotary_dim) {
      NEED(inv_freq);
      aligned4(inv_freq, "inv_freq");
    }
    AppendParams p = {};
    p.kv = view_of(kv);
    p.kv_stride = row_stride(kv_stride, kv.n_heads_kv * kv.head_dim, "k / v");
    aligned16(k, "k");
    aligned16(v, "v");
    if (q) {
      NEED(q_out);
      if (n_heads_q == 0 || n_heads_q > 65535) fail(JAL_ERR_CAPABILITY_MISMATCH, "%zu query heads", n_heads_q);
      p.q_stride = row_stride(q_stride, n_heads_q * kv.head_dim, "q");
      p.q_out_stride = row_stride(q_out_stride, n_heads_q * kv.head_dim, "q_out");
      aligned16(q, "q");
      aligned16(q_out, "q_out");
      if (q == q_out && p.q_stride != p.q_out_stride)
        fail(JAL_ERR_TENSOR_BOUNDS, "q_out is q with another stride");
    }
    if (b.n_seqs == 0 || b.n_rows == 0) return;
    const int dev = current_device();
    on_device(k, "k", dev);
    on_device(v, "v", dev);
    on_device(kv.k, "k pool", dev);
    on_device(kv.v, "v pool", dev);
    on_device(kv.page_table, "page_table", dev);
    on_device(b.q_start, "q_start", dev);
    on_device(b.kv_len, "kv_len", dev);
    if (rotary_dim) on_device(inv_freq, "inv_freq", dev);
    if (q) {
      on_device(q, "q", dev);
      on_device(q_out, "q_out", dev);
    }
    p.kw = kv.k;
    p.vw = kv.v;
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_out = q_out;
    p.inv_freq = inv_freq;
    p.q_start = b.q_start;
    p.kv_len = b.kv_len;
    p.n_seqs = (int32_t)b.n_seqs;
    p.n_rows = (int32_t)b.n_rows;
    p.hq = (int32_t)n_heads_q;
    p.act = dtype;
    p.rotary = (int32_t)rotary_dim;
    p.neox = neox;
    launch_rope_kv_append(p, (cudaStream_t)stream);
  });
}

int jal_op_paged_attention(const jal_paged_kv *kv, const jal_ragged_batch *batch, int dtype, const void *q,
                           size_t n_heads_q, size_t q_stride, float scale, size_t sliding_window, size_t n_sink,
                           void *out, size_t out_stride, void *workspace, size_t workspace_len, void *stream) {
  return guard([&] {
    attention(kv, batch, nullptr, dtype, q, n_heads_q, q_stride, scale, sliding_window, n_sink, out, out_stride,
              workspace, workspace_len, stream);
  });
}

int jal_op_shared_prefix_attention(const jal_paged_kv *kv, const jal_ragged_batch *batch,
                                   const jal_prefix_groups *groups, int dtype, const void *q, size_t n_heads_q,
                                   size_t q_stride, float scale, void *out, size_t out_stride, void *workspace,
                                   size_t workspace_len, void *stream) {
  return guard([&] {
    NEED(groups);
    attention(kv, batch, groups, dtype, q, n_heads_q, q_stride, scale, 0, 0, out, out_stride, workspace, workspace_len,
              stream);
  });
}

static size_t attention_bytes(const jal_paged_kv *kv_in, const jal_ragged_batch *batch, const jal_prefix_groups *groups,
                              int dtype, size_t hq, size_t window, size_t n_sink) {
  const jal_paged_kv kv = checked_kv(kv_in);
  const jal_ragged_batch b = checked_batch(batch, kv);
  jal_prefix_groups g = {};
  if (groups) g = checked_groups(groups, kv, b);
  check_act(dtype, kv);
  check_heads(hq, kv, b);
  if (b.n_seqs == 0 || b.n_rows == 0 || b.max_q_len == 0) return 0;
  return plan_attention(kv, b, g.n_groups ? &g : nullptr, hq, dtype, std::min<size_t>(window, kMaxInt),
                        std::min<size_t>(n_sink, kMaxInt))
      .bytes;
}

int jal_op_paged_attention_workspace(const jal_paged_kv *kv, const jal_ragged_batch *batch, int dtype,
                                     size_t n_heads_q, size_t sliding_window, size_t n_sink, size_t *bytes) {
  return guard([&] {
    NEED(bytes);
    *bytes = attention_bytes(kv, batch, nullptr, dtype, n_heads_q, sliding_window, n_sink);
  });
}

int jal_op_shared_prefix_attention_workspace(const jal_paged_kv *kv, const jal_ragged_batch *batch,
                                             const jal_prefix_groups *groups, int dtype, size_t n_heads_q,
                                             size_t *bytes) {
  return guard([&] {
    NEED(bytes);
    NEED(groups);
    *bytes = attention_bytes(kv, batch, groups, dtype, n_heads_q, 0, 0);
  });
}

static void check_beams(size_t n_seqs, size_t n_beams, size_t vocab, size_t k) {
  if (n_beams == 0 || vocab == 0 || vocab > kMaxInt / 2)
    fail(JAL_ERR_TENSOR_BOUNDS, "%zu beams over a vocabulary of %zu", n_beams, vocab);
  if (k == 0 || k > 64 || k > n_beams * vocab)
    fail(JAL_ERR_CAPABILITY_MISMATCH, "%zu of %zu x %zu continuations (1 to 64)", k, n_beams, vocab);
  if (n_beams > 65535 || n_seqs > 65535 || n_seqs * n_beams > 65535)
    fail(JAL_ERR_CAPABILITY_MISMATCH, "%zu x %zu beams (65535 at most)", n_seqs, n_beams);
  if (!beam_fits(n_beams, vocab, k))
    fail(JAL_ERR_CAPABILITY_MISMATCH, "%zu beams, %zu best of a vocabulary of %zu: too many candidates", n_beams, k,
         vocab);
}

int jal_op_beam_select(const void *logits, int dtype, size_t row_stride_in, const float *cum, size_t n_seqs,
                       size_t n_beams, size_t vocab, size_t k, float *scores, int32_t *parents, int32_t *tokens,
                       void *workspace, size_t workspace_len, void *stream) {
  return guard([&] {
    NEED(logits);
    NEED(cum);
    NEED(scores);
    NEED(parents);
    NEED(tokens);
    aligned4(cum, "cum");
    aligned4(scores, "scores");
    aligned4(parents, "parents");
    aligned4(tokens, "tokens");
    if (!float_type(dtype)) fail(JAL_ERR_CAPABILITY_MISMATCH, "logits of type %d", dtype);
    check_beams(n_seqs, n_beams, vocab, k);
    const size_t stride = row_stride_in ? row_stride_in : vocab;
    if (stride < vocab || stride > (1ull << 40))
      fail(JAL_ERR_TENSOR_BOUNDS, "logits stride %zu, vocabulary %zu", stride, vocab);
    if ((uintptr_t)logits % type_bytes(dtype)) fail(JAL_ERR_TENSOR_BOUNDS, "logits are not aligned to their type");
    if (n_seqs == 0) return;
    const size_t need = beam_workspace(n_seqs, n_beams, vocab, k);
    NEED(workspace);
    aligned16(workspace, "workspace");
    if (workspace_len < need) fail(JAL_ERR_TENSOR_BOUNDS, "workspace of %zu bytes, %zu needed", workspace_len, need);
    if (scores == cum && k != n_beams && n_seqs > 1)
      fail(JAL_ERR_TENSOR_BOUNDS, "scores are cum, with %zu best of %zu beams", k, n_beams);
    const int dev = current_device();
    on_device(logits, "logits", dev);
    on_device(cum, "cum", dev);
    on_device(scores, "scores", dev);
    on_device(parents, "parents", dev);
    on_device(tokens, "tokens", dev);
    on_device(workspace, "workspace", dev);
    BeamParams p = {};
    p.logits = logits;
    p.cum = cum;
    p.scores = scores;
    p.parents = parents;
    p.tokens = tokens;
    p.row_stride = (int64_t)stride;
    p.n_seqs = (int32_t)n_seqs;
    p.n_beams = (int32_t)n_beams;
    p.vocab = (int32_t)vocab;
    p.k = (int32_t)k;
    p.dtype = dtype;
    p.chunks = beam_chunks(n_seqs * n_beams, vocab);
    p.ws = workspace;
    launch_beam_select(p, (cudaStream_t)stream);
  });
}

int jal_op_beam_select_workspace(size_t n_seqs, size_t n_beams, size_t vocab, size_t k, size_t *bytes) {
  return guard([&] {
    NEED(bytes);
    check_beams(n_seqs, n_beams, vocab, k);
    *bytes = beam_workspace(n_seqs, n_beams, vocab, k);
  });
}

int jal_op_beam_reorder(const jal_paged_kv *kv_in, size_t n_layers, size_t layer_stride, const int32_t *kv_len,
                        const int32_t *parents, const int32_t *fresh_pages, size_t n_seqs, size_t n_beams,
                        int32_t *new_table, int32_t *new_len, void *stream) {
  return guard([&] {
    const jal_paged_kv kv = checked_kv(kv_in);
    NEED(kv_len);
    NEED(parents);
    NEED(fresh_pages);
    NEED(new_table);
    NEED(new_len);
    aligned4(kv_len, "kv_len");
    aligned4(parents, "parents");
    aligned4(fresh_pages, "fresh_pages");
    aligned4(new_table, "new_table");
    aligned4(new_len, "new_len");
    if (n_beams == 0 || n_layers == 0 || n_layers > 65535)
      fail(JAL_ERR_TENSOR_BOUNDS, "%zu beams in %zu layers", n_beams, n_layers);
    if (n_beams > kMaxInt || n_seqs > kMaxInt || n_seqs * n_beams > kv.n_seqs)
      fail(JAL_ERR_TENSOR_BOUNDS, "%zu x %zu beams over a table of %llu", n_seqs, n_beams,
           (unsigned long long)kv.n_seqs);
    if (layer_stride == 0) layer_stride = kv.n_pages * kv.page_stride;
    if (layer_stride % 8 || layer_stride > (1ull << 48))
      fail(JAL_ERR_TENSOR_BOUNDS, "layer stride %zu: a multiple of 8", layer_stride);
    if (new_table == kv.page_table || new_len == kv_len)
      fail(JAL_ERR_TENSOR_BOUNDS, "the new table and lengths cannot be the old ones");
    if (n_seqs == 0) return;
    const int dev = current_device();
    on_device(kv.k, "k pool", dev);
    on_device(kv.v, "v pool", dev);
    on_device(kv.page_table, "page_table", dev);
    on_device(kv_len, "kv_len", dev);
    on_device(parents, "parents", dev);
    on_device(fresh_pages, "fresh_pages", dev);
    on_device(new_table, "new_table", dev);
    on_device(new_len, "new_len", dev);
    ReorderParams p = {};
    p.kv = view_of(kv);
    p.kw = kv.k;
    p.vw = kv.v;
    p.kv_len = kv_len;
    p.parents = parents;
    p.fresh = fresh_pages;
    p.new_table = new_table;
    p.new_len = new_len;
    p.layer_stride = (int64_t)layer_stride;
    p.n_seqs = (int32_t)n_seqs;
    p.n_beams = (int32_t)n_beams;
    p.n_layers = (int32_t)n_layers;
    launch_beam_reorder(p, (cudaStream_t)stream);
  });
}

}  // extern "C"
