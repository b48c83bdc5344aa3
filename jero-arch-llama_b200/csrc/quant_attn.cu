// Attention of a ragged batch over a paged cache of 8- or 4-bit codes: the plan of a
// call and its launches.
#include <algorithm>

#include "common.hpp"
#include "quant_attn_mma.cuh"
#include "quant_attn_tc.cuh"

namespace jal {

namespace {

using namespace paged;

// Tiles of eight rows of a block, by registers.
constexpr int most_tiles(int hd, int ns) { return hd > 128 || (hd > 64 && ns > 1) ? 2 : 3; }

template <int BITS, int NS, int HD, int R8>
void run_mma(const QuantAttnParams &p, const QuantAttnPlan &plan, cudaStream_t s) {
  const int64_t blocks = (int64_t)p.a.kv.hkv * p.a.splits * p.a.tiles * p.a.n_seqs;
  constexpr int smem = QuantShape<BITS, NS, HD, R8>::smem;
  static_assert(smem <= 232448 - 2048, "shared memory of a block");
  JAL_CUDA(cudaFuncSetAttribute(k_quant_attn_mma<BITS, NS, HD, R8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  launch_beside(k_quant_attn_mma<BITS, NS, HD, R8>, blocks, kMmaThreads, smem, s, p, plan.direct);
}
template <int BITS, int NS, int HD>
void run_tc(const QuantAttnParams &p, const QuantAttnPlan &plan, cudaStream_t s) {
  const int64_t blocks = (int64_t)p.a.kv.hkv * p.a.splits * p.a.tiles * p.a.n_seqs;
  constexpr int smem = QuantTcShape<BITS, NS, HD>::smem;
  JAL_CUDA(cudaFuncSetAttribute(k_quant_attn_tc<BITS, NS, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  launch_beside(k_quant_attn_tc<BITS, NS, HD>, blocks, kTcThreads, smem, s, p, plan.direct);
}
template <int BITS, int NS, int HD>
void run_rows(const QuantAttnParams &p, const QuantAttnPlan &plan, cudaStream_t s) {
  if constexpr (HD <= 128) {
    if (plan.rows == kTcRows) return run_tc<BITS, NS, HD>(p, plan, s);
  }
  if (plan.rows == 8) return run_mma<BITS, NS, HD, 1>(p, plan, s);
  if constexpr (most_tiles(HD, NS) >= 3) {
    if (plan.rows == 24) return run_mma<BITS, NS, HD, 3>(p, plan, s);
  }
  run_mma<BITS, NS, HD, 2>(p, plan, s);
}
template <int BITS, int NS>
void run_hd(const QuantAttnParams &p, const QuantAttnPlan &plan, cudaStream_t s) {
  if (p.a.kv.hd <= 64) run_rows<BITS, NS, 64>(p, plan, s);
  else if (p.a.kv.hd <= 128) run_rows<BITS, NS, 128>(p, plan, s);
  else run_rows<BITS, NS, 256>(p, plan, s);
}
template <int BITS>
void run_type(const QuantAttnParams &p, const QuantAttnPlan &plan, cudaStream_t s) {
  if (p.a.act == JAL_F32) run_hd<BITS, 2>(p, plan, s);
  else run_hd<BITS, 1>(p, plan, s);
}

constexpr int64_t kBlockKeys = 256;
// More (row, head of the group) pairs that share keys than these go to the tcgen05 kernel, up to
// here the integer one is as fast or faster (32 heads, 8 KV heads of 128, 8 bits; 64 and 68
// pairs, integer | tcgen05: 48 sequences of 2048 keys 154 | 161 us, f32 rows 187 | 191; one of
// 16384 keys 45 | 39, f32 rows 55 | 47, and there 32 pairs 37 | 39 and 36 | 46).
constexpr int64_t kTcLeast = 64;

}  // namespace

QuantAttnPlan plan_quant_attention(const jal_quant_kv &kv, const jal_ragged_batch &b, size_t hq, int act, size_t window,
                                   size_t n_sink) {
  QuantAttnPlan a = {};
  const int64_t G = (int64_t)(hq / kv.n_heads_kv), hkv = (int64_t)kv.n_heads_kv, pairs = (int64_t)b.max_q_len * G;
  const int ns = act == JAL_F32 ? 2 : 1;
  a.rows = kv.head_dim <= 128 && pairs > kTcLeast
               ? kTcRows
               : 8 * (int)std::min<int64_t>(most_tiles((int)kv.head_dim, ns), (pairs + 7) / 8);
  a.tiles = (int)((pairs + a.rows - 1) / a.rows);
  int64_t keys = (int64_t)b.max_kv_len;
  if (window) keys = std::min<int64_t>(keys, (int64_t)(window + n_sink + b.max_q_len));
  const int64_t blocks = a.tiles * hkv * (int64_t)b.n_seqs;
  if (a.rows == kTcRows) {  // a block fills an SM: cut only as far as that gives idle ones work
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kPagedMaxSplits, keys / (2 * kTcKeys)));
    a.splits = (int)std::min(most, std::max<int64_t>(1, kPagedSMs / std::max<int64_t>(1, blocks)));
  } else {
    a.splits = attention_pieces(blocks, keys, quant_blocks(kv.bits, (int)kv.head_dim, a.rows / 8, ns), kBlockKeys, false);
  }
  a.direct = a.splits == 1;
  if (!a.direct)
    a.bytes = (size_t)a.splits * b.n_rows * hq * (kv.head_dim * sizeof(float) + sizeof(float2)) + 256;
  return a;
}

void launch_quant_attention(const QuantAttnParams &p, int bits, const QuantAttnPlan &plan, cudaStream_t s) {
  if (bits == 8) run_type<8>(p, plan, s);
  else run_type<4>(p, plan, s);
  if (!plan.direct) launch_attention_join(p.a, 0, s);
}

}  // namespace jal
