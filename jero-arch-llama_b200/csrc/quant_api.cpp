// C entry points of the quantised paged cache and of draft verification:
// arguments are checked here, on the host, before anything is enqueued.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "jal.h"
#include "paged_args.hpp"
#include "quant_kv.hpp"

using namespace jal;

namespace {

// A cache view with its defaults filled in.
jal_quant_kv checked_quant(const jal_quant_kv *in) {
  NEED(in);
  jal_quant_kv kv = *in;
  NEED(kv.k);
  NEED(kv.v);
  NEED(kv.k_scale);
  NEED(kv.v_scale);
  NEED(kv.page_table);
  if (kv.bits != 8 && kv.bits != 4) fail(JAL_ERR_CAPABILITY_MISMATCH, "cache of %d-bit codes (8 or 4)", kv.bits);
  const uint64_t unit = 128 / (uint64_t)kv.bits;  // codes in 16 bytes
  if (kv.head_dim == 0 || kv.head_dim % unit || kv.head_dim > (uint64_t)kPagedMaxHeadDim)
    fail(JAL_ERR_CAPABILITY_MISMATCH, "head_dim %llu with %d-bit codes: multiples of %llu up to %d",
         (unsigned long long)kv.head_dim, kv.bits, (unsigned long long)unit, kPagedMaxHeadDim);
  if (kv.n_heads_kv == 0 || kv.n_heads_kv > 65535 || kv.page_size == 0 || kv.n_pages == 0 || kv.max_pages == 0)
    fail(JAL_ERR_TENSOR_BOUNDS, "paged cache without heads, pages or slots");
  if (kv.n_pages > kMaxInt || kv.page_size > kMaxPositions || kv.max_pages > kMaxPositions / kv.page_size ||
      kv.n_seqs > kMaxInt)
    fail(JAL_ERR_TENSOR_BOUNDS, "paged cache: more than 2^31 pages, positions or sequences");
  const uint64_t row = kv.head_dim * (uint64_t)kv.bits / 8;
  if (!kv.page_stride && !kv.head_stride && !kv.slot_stride) {
    kv.slot_stride = row;
    kv.head_stride = kv.page_size * kv.slot_stride;
    kv.page_stride = kv.n_heads_kv * kv.head_stride;
  }
  if (!kv.scale_page_stride && !kv.scale_head_stride) {
    kv.scale_head_stride = kv.page_size;
    kv.scale_page_stride = kv.n_heads_kv * kv.page_size;
  }
  if (kv.page_stride % 16 || kv.head_stride % 16 || kv.slot_stride % 16)
    fail(JAL_ERR_TENSOR_BOUNDS, "strides of codes have to be multiples of 16 bytes");
  if (kv.page_size > 1 && kv.slot_stride < row)
    fail(JAL_ERR_TENSOR_BOUNDS, "slot stride %llu, a row has %llu bytes", (unsigned long long)kv.slot_stride,
         (unsigned long long)row);
  const uint64_t most = 1ull << 40;
  if (kv.page_stride > most || kv.head_stride > most || kv.slot_stride > most || kv.scale_page_stride > most ||
      kv.scale_head_stride > most)
    fail(JAL_ERR_TENSOR_BOUNDS, "paged cache stride above 2^40");
  aligned16(kv.k, "k codes");
  aligned16(kv.v, "v codes");
  aligned4(kv.k_scale, "k_scale");
  aligned4(kv.v_scale, "v_scale");
  aligned4(kv.page_table, "page_table");
  return kv;
}

// The places of the codes: strides in bytes.
PagedView codes_of(const jal_quant_kv &kv) {
  jal_paged_kv p = {};
  p.k = kv.k;
  p.v = kv.v;
  p.page_table = kv.page_table;
  p.n_pages = kv.n_pages;
  p.page_size = kv.page_size;
  p.n_heads_kv = kv.n_heads_kv;
  p.head_dim = kv.head_dim;
  p.n_seqs = kv.n_seqs;
  p.max_pages = kv.max_pages;
  p.page_stride = kv.page_stride;
  p.head_stride = kv.head_stride;
  p.slot_stride = kv.slot_stride;
  return view_of(p);
}
QuantScales scales_of(const jal_quant_kv &kv) {
  return {kv.k_scale, kv.v_scale, (int64_t)kv.scale_page_stride, (int64_t)kv.scale_head_stride};
}
void cache_on_device(const jal_quant_kv &kv, int dev) {
  on_device(kv.k, "k codes", dev);
  on_device(kv.v, "v codes", dev);
  on_device(kv.k_scale, "k_scale", dev);
  on_device(kv.v_scale, "v_scale", dev);
  on_device(kv.page_table, "page_table", dev);
}

void check_rows(int dtype) {
  if (!float_type(dtype)) fail(JAL_ERR_CAPABILITY_MISMATCH, "rows of type %d", dtype);
}
void check_heads(size_t hq, const jal_quant_kv &kv, const jal_ragged_batch &b) {
  if (hq == 0 || hq % kv.n_heads_kv || hq > 65535)
    fail(JAL_ERR_CAPABILITY_MISMATCH, "%zu query heads over %llu KV heads", hq, (unsigned long long)kv.n_heads_kv);
  if (b.n_rows * (hq / kv.n_heads_kv) > kMaxPositions)  // (row, head of the group) pairs are counted in 32 bits
    fail(JAL_ERR_TENSOR_BOUNDS, "batch of 2^31 rows times heads of a group or more");
}

}  // namespace

extern "C" {

int jal_op_quant_kv_append(const jal_quant_kv *kv_in, const jal_ragged_batch *batch, int dtype, const void *k,
                           const void *v, size_t kv_stride, const float *inv_freq, size_t rotary_dim, int neox,
                           const void *q, void *q_out, size_t n_heads_q, size_t q_stride, size_t q_out_stride,
                           void *stream) {
  return guard([&] {
    const jal_quant_kv kv = checked_quant(kv_in);
    const jal_ragged_batch b = checked_batch(batch, kv.n_seqs, kv.max_pages * kv.page_size);
    check_rows(dtype);
    NEED(k);
    NEED(v);
    if (rotary_dim % 2 || rotary_dim > kv.head_dim)
      fail(JAL_ERR_CAPABILITY_MISMATCH, "rotary_dim %zu of head_dim %llu", rotary_dim, (unsigned long long)kv.head_dim);
    if (rotary_dim) {
      NEED(inv_freq);
      aligned4(inv_freq, "inv_freq");
    }
    QuantAppendParams p = {};
    AppendParams &a = p.a;
    a.kv = codes_of(kv);
    a.kv_stride = row_stride(kv_stride, kv.n_heads_kv * kv.head_dim, "k / v");
    aligned16(k, "k");
    aligned16(v, "v");
    if (q) {
      NEED(q_out);
      if (n_heads_q == 0 || n_heads_q > 65535) fail(JAL_ERR_CAPABILITY_MISMATCH, "%zu query heads", n_heads_q);
      a.q_stride = row_stride(q_stride, n_heads_q * kv.head_dim, "q");
      a.q_out_stride = row_stride(q_out_stride, n_heads_q * kv.head_dim, "q_out");
      aligned16(q, "q");
      aligned16(q_out, "q_out");
      if (q == q_out && a.q_stride != a.q_out_stride && b.n_rows > 1)
        fail(JAL_ERR_TENSOR_BOUNDS, "q_out is q with another stride");
    }
    if (b.n_seqs == 0 || b.n_rows == 0) return;
    const int dev = current_device();
    cache_on_device(kv, dev);
    on_device(k, "k", dev);
    on_device(v, "v", dev);
    on_device(b.q_start, "q_start", dev);
    on_device(b.kv_len, "kv_len", dev);
    if (rotary_dim) on_device(inv_freq, "inv_freq", dev);
    if (q) {
      on_device(q, "q", dev);
      on_device(q_out, "q_out", dev);
    }
    a.kw = kv.k;
    a.vw = kv.v;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.inv_freq = inv_freq;
    a.q_start = b.q_start;
    a.kv_len = b.kv_len;
    a.n_seqs = (int32_t)b.n_seqs;
    a.n_rows = (int32_t)b.n_rows;
    a.hq = (int32_t)n_heads_q;
    a.act = dtype;
    a.rotary = (int32_t)rotary_dim;
    a.neox = neox;
    p.ks = kv.k_scale;
    p.vs = kv.v_scale;
    p.s_page = (int64_t)kv.scale_page_stride;
    p.s_head = (int64_t)kv.scale_head_stride;
    launch_quant_kv_append(p, kv.bits, (cudaStream_t)stream);
  });
}

int jal_op_quant_kv_attention(const jal_quant_kv *kv_in, const jal_ragged_batch *batch, int dtype, const void *q,
                              size_t hq, size_t q_stride, float scale, size_t window, size_t n_sink, void *out,
                              size_t out_stride, void *ws, size_t ws_len, void *stream) {
  return guard([&] {
    const jal_quant_kv kv = checked_quant(kv_in);
    const jal_ragged_batch b = checked_batch(batch, kv.n_seqs, kv.max_pages * kv.page_size);
    check_rows(dtype);
    check_heads(hq, kv, b);
    NEED(q);
    NEED(out);
    const float scale_log2 = scale * 1.4426950408889634f;  // softmax by powers of two
    if (!std::isfinite(scale_log2)) fail(JAL_ERR_INVALID_ARGUMENT, "attention scale is not finite or too large");
    QuantAttnParams p = {};
    AttnParams &a = p.a;
    a.kv = codes_of(kv);
    a.q_stride = row_stride(q_stride, hq * kv.head_dim, "q");
    a.out_stride = row_stride(out_stride, hq * kv.head_dim, "out");
    aligned16(q, "q");
    aligned16(out, "out");
    if (q == out && a.q_stride != a.out_stride && b.n_rows > 1)
      fail(JAL_ERR_TENSOR_BOUNDS, "out is q with another stride");
    if (b.n_seqs == 0 || b.n_rows == 0 || b.max_q_len == 0) return;
    window = std::min<size_t>(window, kMaxInt);
    n_sink = std::min<size_t>(n_sink, kMaxInt);
    const QuantAttnPlan plan = plan_quant_attention(kv, b, hq, dtype, window, n_sink);
    const double rows = std::min((double)b.n_rows, (double)b.n_seqs * (double)b.max_q_len);
    if ((double)kv.n_heads_kv * plan.tiles * plan.splits * (double)b.n_seqs > 2e9 ||
        (!plan.direct && rows * (double)hq > 2e9))
      fail(JAL_ERR_CAPABILITY_MISMATCH, "batch too large for one launch");
    if (plan.bytes) {
      NEED(ws);
      aligned16(ws, "workspace");
      if (ws_len < plan.bytes)
        fail(JAL_ERR_TENSOR_BOUNDS, "workspace of %zu bytes, %zu needed", ws_len, plan.bytes);
    }
    const int dev = current_device();
    cache_on_device(kv, dev);
    on_device(q, "q", dev);
    on_device(out, "out", dev);
    on_device(b.q_start, "q_start", dev);
    on_device(b.kv_len, "kv_len", dev);
    if (plan.bytes) on_device(ws, "workspace", dev);
    a.q = q;
    a.out = out;
    a.q_start = b.q_start;
    a.kv_len = b.kv_len;
    a.n_seqs = (int32_t)b.n_seqs;
    a.n_rows = (int32_t)b.n_rows;
    a.max_q = (int32_t)b.max_q_len;
    a.hq = (int32_t)hq;
    a.G = (int32_t)(hq / kv.n_heads_kv);
    a.act = dtype;
    a.window = (int32_t)window;
    a.n_sink = (int32_t)n_sink;
    a.splits = plan.splits;
    a.tiles = plan.tiles;
    a.scale_log2 = scale_log2;
    a.part_o = (float *)ws;
    if (plan.bytes) a.part_ml = (float2 *)(a.part_o + (size_t)plan.splits * b.n_rows * hq * kv.head_dim);
    p.sc = scales_of(kv);
    launch_quant_attention(p, kv.bits, plan, (cudaStream_t)stream);
  });
}

int jal_op_quant_kv_attention_workspace(const jal_quant_kv *kv_in, const jal_ragged_batch *batch, int dtype, size_t hq,
                                        size_t window, size_t n_sink, size_t *bytes) {
  return guard([&] {
    NEED(bytes);
    const jal_quant_kv kv = checked_quant(kv_in);
    const jal_ragged_batch b = checked_batch(batch, kv.n_seqs, kv.max_pages * kv.page_size);
    check_rows(dtype);
    check_heads(hq, kv, b);
    *bytes = 0;
    if (b.n_seqs == 0 || b.n_rows == 0 || b.max_q_len == 0) return;
    *bytes = plan_quant_attention(kv, b, hq, dtype, std::min<size_t>(window, kMaxInt), std::min<size_t>(n_sink, kMaxInt))
                 .bytes;
  });
}

int jal_op_quant_kv_read(const jal_quant_kv *kv_in, const int32_t *first, const int32_t *kv_len, size_t n_seqs,
                         size_t max_len, const jal_paged_kv *into_in, void *stream) {
  return guard([&] {
    const jal_quant_kv kv = checked_quant(kv_in);
    const jal_paged_kv into = checked_kv(into_in);
    NEED(kv_len);
    aligned4(kv_len, "kv_len");
    aligned4(first, "first");
    if (into.n_heads_kv != kv.n_heads_kv || into.head_dim != kv.head_dim)
      fail(JAL_ERR_TENSOR_BOUNDS, "%llu heads of %llu read into %llu heads of %llu", (unsigned long long)kv.n_heads_kv,
           (unsigned long long)kv.head_dim, (unsigned long long)into.n_heads_kv, (unsigned long long)into.head_dim);
    if (n_seqs > kv.n_seqs || n_seqs > into.n_seqs)
      fail(JAL_ERR_TENSOR_BOUNDS, "%zu sequences over tables of %llu and %llu", n_seqs, (unsigned long long)kv.n_seqs,
           (unsigned long long)into.n_seqs);
    max_len = std::min<size_t>(max_len, std::min(kv.max_pages * kv.page_size, into.max_pages * into.page_size));
    if (n_seqs == 0 || max_len == 0) return;
    const int dev = current_device();
    cache_on_device(kv, dev);
    on_device(into.k, "into's k pool", dev);
    on_device(into.v, "into's v pool", dev);
    on_device(into.page_table, "into's page_table", dev);
    on_device(kv_len, "kv_len", dev);
    if (first) on_device(first, "first", dev);
    QuantReadParams p = {};
    p.from = codes_of(kv);
    p.into = view_of(into);
    p.sc = scales_of(kv);
    p.kw = into.k;
    p.vw = into.v;
    p.first = first;
    p.kv_len = kv_len;
    p.n_seqs = (int32_t)n_seqs;
    p.max_len = (int64_t)max_len;
    launch_quant_kv_read(p, kv.bits, (cudaStream_t)stream);
  });
}

static size_t verify_bytes(const jal_ragged_batch &b, size_t vocab) {
  if (vocab == 0 || vocab >= (1ull << 30)) fail(JAL_ERR_TENSOR_BOUNDS, "vocabulary of %zu", vocab);
  if (b.n_seqs > (kMaxInt >> 4)) fail(JAL_ERR_TENSOR_BOUNDS, "%llu sequences", (unsigned long long)b.n_seqs);
  const size_t chunks = b.n_rows ? (size_t)verify_chunks(b.n_rows, vocab) : 1;
  if (2 * b.n_rows * chunks > kMaxInt)
    fail(JAL_ERR_CAPABILITY_MISMATCH, "batch of %llu rows too large for one launch", (unsigned long long)b.n_rows);
  return verify_workspace(b.n_seqs, b.n_rows, vocab, nullptr, nullptr);
}

int jal_op_verify_drafts(const jal_ragged_batch *batch, const void *logits, int dtype, size_t stride,
                         const void *draft_logits, size_t draft_stride, size_t vocab, const int32_t *tokens,
                         const float *uniform, const float *temperature, const float *draft_temperature,
                         int32_t *out_tokens, int32_t *n_accepted, int32_t *new_len, void *ws, size_t ws_len,
                         void *stream) {
  return guard([&] {
    const jal_ragged_batch b = checked_batch(batch, kMaxInt, kMaxPositions);
    NEED(logits);
    NEED(tokens);
    NEED(uniform);
    NEED(out_tokens);
    NEED(n_accepted);
    if (!float_type(dtype)) fail(JAL_ERR_CAPABILITY_MISMATCH, "logits of type %d", dtype);
    const size_t need = verify_bytes(b, vocab);
    if (!stride) stride = vocab;
    if (!draft_stride) draft_stride = vocab;
    if (stride < vocab || stride > (1ull << 40) || draft_stride < vocab || draft_stride > (1ull << 40))
      fail(JAL_ERR_TENSOR_BOUNDS, "logits strides %zu and %zu, vocabulary %zu", stride, draft_stride, vocab);
    if ((uintptr_t)logits % type_bytes(dtype) || (uintptr_t)draft_logits % type_bytes(dtype))
      fail(JAL_ERR_TENSOR_BOUNDS, "logits are not aligned to their type");
    aligned4(tokens, "tokens");
    aligned4(uniform, "uniform");
    aligned4(temperature, "temperature");
    aligned4(draft_temperature, "draft_temperature");
    aligned4(out_tokens, "out_tokens");
    aligned4(n_accepted, "n_accepted");
    aligned4(new_len, "new_len");
    // (Blocks of a sequence read tokens while another writes.)
    const uintptr_t in = (uintptr_t)tokens, to = (uintptr_t)out_tokens, bytes = b.n_rows * sizeof(int32_t);
    if (to == in || (to < in + bytes && in < to + bytes)) fail(JAL_ERR_TENSOR_BOUNDS, "out_tokens overlaps tokens");
    if (b.n_seqs == 0) return;
    if (need) {
      NEED(ws);
      aligned16(ws, "workspace");
      if (ws_len < need) fail(JAL_ERR_TENSOR_BOUNDS, "workspace of %zu bytes, %zu needed", ws_len, need);
    }
    const int dev = current_device();
    on_device(b.q_start, "q_start", dev);
    on_device(b.kv_len, "kv_len", dev);
    on_device(logits, "logits", dev);
    on_device(tokens, "tokens", dev);
    on_device(uniform, "uniform", dev);
    on_device(out_tokens, "out_tokens", dev);
    on_device(n_accepted, "n_accepted", dev);
    if (draft_logits) on_device(draft_logits, "draft_logits", dev);
    if (temperature) on_device(temperature, "temperature", dev);
    if (draft_temperature) on_device(draft_temperature, "draft_temperature", dev);
    if (new_len) on_device(new_len, "new_len", dev);
    if (need) on_device(ws, "workspace", dev);
    VerifyParams p = {};
    p.logits = logits;
    p.draft = draft_logits;
    p.stride = (int64_t)stride;
    p.draft_stride = (int64_t)draft_stride;
    p.q_start = b.q_start;
    p.kv_len = b.kv_len;
    p.tokens = tokens;
    p.uniform = uniform;
    p.temperature = temperature;
    p.draft_temperature = draft_temperature ? draft_temperature : temperature;
    p.out_tokens = out_tokens;
    p.n_accepted = n_accepted;
    p.new_len = new_len;
    verify_workspace(b.n_seqs, b.n_rows, vocab, &p, ws);
    p.n_seqs = (int32_t)b.n_seqs;
    p.n_rows = (int32_t)b.n_rows;
    p.vocab = (int32_t)vocab;
    p.chunks = b.n_rows ? verify_chunks(b.n_rows, vocab) : 1;
    p.dtype = dtype;
    launch_verify_drafts(p, (cudaStream_t)stream);
  });
}

int jal_op_verify_drafts_workspace(const jal_ragged_batch *batch, size_t vocab, size_t *bytes) {
  return guard([&] {
    NEED(bytes);
    *bytes = verify_bytes(checked_batch(batch, kMaxInt, kMaxPositions), vocab);
  });
}

}  // extern "C"
