// Attention of a ragged batch over a paged cache: the plan of a call, the f32
// kernel, and the joining of the pieces that the keys were cut into.
#include <algorithm>

#include "common.hpp"
#include "paged_attn_mma.cuh"
#include "paged_attn_tc.cuh"
#include "paged_dev.cuh"

namespace jal {

namespace {

using namespace paged;

// ---- the f32 kernel ---------------------------------------------------------
// f32 caches: one pass over the tile's keys with the running maximum and sum of
// each row, everything in f32 on the CUDA cores.  K and V tiles of kF32Keys keys
// go round two stages of shared memory, each warp copying its quarter of a tile's
// rows with cp.async one tile ahead; 128 threads work on them as 8 row groups x 16
// key (or dim) groups.  Few rows are bound by shared memory, which a thread reads
// three times (16 bytes of q, twice 16 of K) for eight multiply-adds, not by the
// cache: 48 rows of up to 4100 keys take 540 to 590 us, 2.8 TB/s (843 us without the
// copies ahead).
constexpr int kF32Threads = 128;
constexpr int kF32Keys = 32;

template <int HD, int RT>
struct F32Smem {
  float q[RT][HD + 4];
  float k[2][kF32Keys][HD + 4];
  float v[2][kF32Keys][HD];
  float s[RT][kF32Keys + 4];
  RowSpan span[RT];
  uint32_t present[2][kF32Threads / 32];
};

template <int HD, int RT>
__global__ void __launch_bounds__(kF32Threads) k_paged_attn_f32(const __grid_constant__ AttnParams p, const int part,
                                                                const bool direct) {
  extern __shared__ __align__(16) char smem_raw[];
  auto &sm = *(F32Smem<HD, RT> *)smem_raw;
  pdl_trigger();
  Tile t;
  if (!block_tile(p, part, RT, kF32Keys, t)) return;
  constexpr int R = RT / 8, KC = kF32Keys / 16, DC = HD / 16, kMine = kF32Keys / 4;
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16, warp = tid / 32, lane = tid % 32;
  const int hd = p.kv.hd;
  // This warp's rows of the tile at u: looked up by its first lanes one tile ahead.
  auto locate = [&](int u) -> Slot {
    const int k = u + warp * kMine + lane;
    return lane < kMine && k < t.u1 ? slot_of(p.kv, t, t.key(k)) : Slot{-1, 0};
  };
  auto copy = [&](const Slot &where, int stage) {
    const int64_t at = slot_offset(p.kv, where, t.head);
    const uint32_t bits = __ballot_sync(0xffffffffu, at >= 0);
    if (lane == 0) sm.present[stage][warp] = bits & ((1u << kMine) - 1);
#pragma unroll
    for (int i = 0; i < kMine * (HD / 4) / 32; i++) {
      const int r = (i * 32 + lane) / (HD / 4), d = (i * 32 + lane) % (HD / 4) * 4;
      const int64_t o = __shfl_sync(0xffffffffu, at, r);
      const bool there = o >= 0 && d < hd;
      const int64_t e = there ? o + d : 0;
      copy16(smem_u32(&sm.k[stage][warp * kMine + r][d]), (const float *)p.kv.k + e, there);
      copy16(smem_u32(&sm.v[stage][warp * kMine + r][d]), (const float *)p.kv.v + e, there);
    }
    copies_done();
  };
  Slot next = locate(t.u0);
  copy(next, 0);
  next = locate(t.u0 + kF32Keys);
  for (int i = tid; i < RT * (HD / 4); i += kF32Threads) {
    const int j = i / (HD / 4), d = i % (HD / 4) * 4;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (j < t.rows && d < hd) x = *(const float4 *)((const float *)p.q + q_offset(p, t, j) + d);
    *(float4 *)&sm.q[j][d] =
        make_float4(x.x * p.scale_log2, x.y * p.scale_log2, x.z * p.scale_log2, x.w * p.scale_log2);
  }
  for (int j = tid; j < RT; j += kF32Threads)  // (rows that do not exist see everything)
    sm.span[j] = j < t.rows ? row_span(p, t, row_mask(p, t, j)) : RowSpan{0x7fffffff, 0, 0};
  float o[R][DC], m[R], l[R];
#pragma unroll
  for (int i = 0; i < R; i++) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < DC; c++) o[i][c] = 0.0f;
  }
  float bad = 0.0f;
  int stage = 0;
  for (int u = t.u0; u < t.u1; u += kF32Keys, stage ^= 1) {
    copies_wait<0>();
    __syncthreads();  // the tile is there, and the other stage has been read
    const Slot at = next;
    next = locate(u + 2 * kF32Keys);
    copy(at, stage ^ 1);
    uint32_t bits = 0;
#pragma unroll
    for (int w = 0; w < kF32Threads / 32; w++) bits |= sm.present[stage][w] << (w * kMine);
    bool whole = bits == 0xffffffffu;
#pragma unroll
    for (int i = 0; i < R; i++) whole = whole && sm.span[ty + 8 * i].all(u, kF32Keys);
    const bool masked = __any_sync(0xffffffffu, !whole);
    float s[R][KC];
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
      for (int c = 0; c < KC; c++) s[i][c] = 0.0f;
#pragma unroll 8
    for (int d = 0; d < HD; d += 4) {
      float4 a[R], b[KC];
#pragma unroll
      for (int i = 0; i < R; i++) a[i] = *(const float4 *)&sm.q[ty + 8 * i][d];
#pragma unroll
      for (int c = 0; c < KC; c++) b[c] = *(const float4 *)&sm.k[stage][tx + 16 * c][d];
#pragma unroll
      for (int i = 0; i < R; i++)
#pragma unroll
        for (int c = 0; c < KC; c++) {
          s[i][c] = fmaf(a[i].x, b[c].x, s[i][c]);
          s[i][c] = fmaf(a[i].y, b[c].y, s[i][c]);
          s[i][c] = fmaf(a[i].z, b[c].z, s[i][c]);
          s[i][c] = fmaf(a[i].w, b[c].w, s[i][c]);
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
      const uint32_t see = masked ? bits & sm.span[ty + 8 * i].bits(u) : 0xffffffffu;
      float top = m[i];
#pragma unroll
      for (int c = 0; c < KC; c++) {
        if (!((see >> (tx + 16 * c)) & 1)) s[i][c] = -INFINITY;
        top = fmaxf(top, s[i][c]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float safe = top == -INFINITY ? 0.0f : top;
      const float corr = exp2f(m[i] - safe);
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < KC; c++) {
        const float e = exp2f(s[i][c] - safe);
        sum += e;
        sm.s[ty + 8 * i][tx + 16 * c] = e;
      }
      l[i] = l[i] * corr + sum;
      m[i] = top;
#pragma unroll
      for (int c = 0; c < DC; c++) o[i][c] *= corr;
    }
    if (masked) {  // values that some rows must not meet: x * 0 is NaN where x is not finite
      for (int r = 0; r < kF32Keys; r++)
#pragma unroll
        for (int c = 0; c < DC; c++) bad = fmaf(sm.v[stage][r][tx + 16 * c], 0.0f, bad);
    }
    __syncwarp();  // a row group's weights are written and read by one warp
#pragma unroll 4
    for (int r = 0; r < kF32Keys; r += 4) {
      float4 w[R];
#pragma unroll
      for (int i = 0; i < R; i++) w[i] = *(const float4 *)&sm.s[ty + 8 * i][r];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float v[DC];
#pragma unroll
        for (int c = 0; c < DC; c += 4) *(float4 *)&v[c] = *(const float4 *)&sm.v[stage][r + e][tx * 4 + (c / 4) * 64];
#pragma unroll
        for (int i = 0; i < R; i++) {
          const float we = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
#pragma unroll
          for (int c = 0; c < DC; c++) o[i][c] = fmaf(we, v[c], o[i][c]);
        }
      }
    }
    __syncwarp();
  }
  copies_wait<0>();
  if (__syncthreads_or(bad != bad)) {
    for (int j = warp; j < t.rows; j += kF32Threads / 32) attend_row_alone(p, t, j, direct);
    return;
  }
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int j = ty + 8 * i;
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    if (j >= t.rows) continue;
    const int64_t oo = out_offset(p, t, j), pi = part_index(p, t, j);
    const float inv = !direct ? 1.0f : l[i] == 0.0f ? 0.0f : 1.0f / l[i];
    float *const dst = direct ? (float *)p.out + oo : p.part_o + pi * hd;
    if (!direct && tx == 0) p.part_ml[pi] = make_float2(m[i], l[i]);
#pragma unroll
    for (int c = 0; c < DC; c += 4) {
      const int d = tx * 4 + (c / 4) * 64;
      if (d < hd)
        *(float4 *)(dst + d) = make_float4(o[i][c] * inv, o[i][c + 1] * inv, o[i][c + 2] * inv, o[i][c + 3] * inv);
    }
  }
}

// ---- joining the pieces -----------------------------------------------------
// One block for each (token row, query head): the pieces' sums rescaled to the
// largest of their maxima and added, each warp every fourth piece with eight
// pieces' loads under way, the warps in order at the end.  A piece without a
// visible key has sum 0 and is not read.  The blocks go by the rows of the buffers,
// with a search for the sequence, or by the sequences' first max_q rows where that is
// fewer: one long prompt among single rows makes the second count large, buffers for
// larger batches the first.  (Two kernels: in one, registers for both halve the blocks
// of an SM, and eight groups behind prefixes take 121 us instead of 114.)  Whose row
// it is, is looked up before the wait for the pieces: the batch was there before the
// launch that makes them.
constexpr int kJoinWarps = 4, kJoinThreads = kJoinWarps * 32;
static_assert(2 * kPagedMaxSplits <= kJoinThreads, "a thread looks at one piece's maximum and sum");

template <bool BY_ROW>
__global__ void __launch_bounds__(kJoinThreads) k_paged_attn_join(const __grid_constant__ AttnParams p, const int prefix_rows) {
  __shared__ float weight[kJoinThreads];
  __shared__ float red[kJoinWarps];
  __shared__ float4 part[kJoinWarps][kPagedMaxHeadDim / 4];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, head = blockIdx.x % p.hq, tok = blockIdx.x / p.hq;
  const int s = BY_ROW ? warp_seq_of_row(p.q_start, p.n_seqs, tok) : tok / p.max_q;
  int g_first = 0, g_last = 0, g_row = 0, beg, end;
  if (p.prefix_splits) {
    const int g = seq_of_row(p.group_start, 0, p.n_groups, s);
    g_first = __ldg(p.group_start + g);
    g_last = __ldg(p.group_start + g + 1);
    g_row = __ldg(p.q_start + min(max(g_first, 0), p.n_seqs));
  }
  seq_rows(p.q_start, p.n_rows, s, beg, end);
  pdl_wait();
  const int row = BY_ROW ? tok : beg + (tok - s * p.max_q);
  if (row < beg || row >= end || row - beg >= p.max_q) return;
  int first = p.prefix_splits;  // a sequence outside every group has its own keys alone
  if (g_first <= s && s < g_last) {
    first = 0;
    const int rows = row - min(max(g_row, 0), p.n_rows) + 1;
    if ((int64_t)rows * p.G > (int64_t)p.prefix_tiles * prefix_rows) return;  // past max_group: not computed
  }
  const int n = p.prefix_splits + p.splits, hd = p.kv.hd;
  const int64_t stride = (int64_t)p.n_rows * p.hq, at = (int64_t)row * p.hq + head;
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (tid >= first && tid < n) ml = p.part_ml[tid * stride + at];
  float top = warp_max(ml.x);
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWarps; w++) top = fmaxf(top, red[w]);
  const float w = ml.y == 0.0f ? 0.0f : exp2f(ml.x - (top == -INFINITY ? 0.0f : top));
  weight[tid] = w;
  if (ml.y == 0.0f) weight[tid] = -1.0f;  // (not a weight of 0: what a piece far below the others holds may be NaN)
  float total = warp_sum(w * ml.y);
  __syncthreads();
  if (lane == 0) red[warp] = total;
  __syncthreads();
  total = 0.0f;
#pragma unroll
  for (int k = 0; k < kJoinWarps; k++) total += red[k];
  const int chunks = hd / 4;  // float4 pieces of a row: two a lane at most
  float4 o[2] = {};
  for (int k = warp; k < n; k += kJoinWarps * 8) {
    float4 v[8][2];
    float c[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int piece = k + e * kJoinWarps;
      c[e] = piece < n ? weight[piece] : -1.0f;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        v[e][h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c[e] != -1.0f && lane + 32 * h < chunks)
          v[e][h] = *((const float4 *)(p.part_o + (piece * stride + at) * hd) + lane + 32 * h);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        o[h].x = fmaf(c[e], v[e][h].x, o[h].x);
        o[h].y = fmaf(c[e], v[e][h].y, o[h].y);
        o[h].z = fmaf(c[e], v[e][h].z, o[h].z);
        o[h].w = fmaf(c[e], v[e][h].w, o[h].w);
      }
  }
  part[warp][lane] = o[0];
  part[warp][lane + 32] = o[1];
  __syncthreads();
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t oo = (int64_t)row * p.out_stride + (int64_t)head * hd;
  for (int d = tid; d < hd; d += kJoinThreads) {
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kJoinWarps; k++) sum += ((const float *)part[k])[d];
    store_from_f32(p.out, oo + d, p.act, sum * inv);
  }
}

int64_t blocks_of(const AttnParams &p, int part) {
  const int64_t prefix = (int64_t)p.prefix_splits * p.prefix_tiles * p.n_groups;
  const int64_t own = (int64_t)p.splits * p.tiles * p.n_seqs;
  return p.kv.hkv * ((part == kOwn ? 0 : prefix) + (part == kPrefix ? 0 : own));
}
// `beside`: may start while the launch before it still runs (it waits for that
// one's end itself).
template <class F, class... A>
void launch(F kernel, int64_t blocks, int threads, int smem, bool beside, cudaStream_t s, const A &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = beside ? 1 : 0;
  JAL_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
}
template <class F>
bool run_kernel(F kernel, const AttnParams &p, int part, bool direct, int threads, int smem, cudaStream_t s,
                bool beside = false) {
  const int64_t blocks = blocks_of(p, part);
  if (!blocks) return false;
  JAL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  launch(kernel, blocks, threads, smem, beside, s, p, part, direct);
  return true;
}

template <int HD>
void run_f32(const AttnParams &p, const AttnPlan &plan, cudaStream_t s) {
  if (plan.rows == 8)
    run_kernel(k_paged_attn_f32<HD, 8>, p, kBoth, plan.direct, kF32Threads, (int)sizeof(F32Smem<HD, 8>), s);
  else
    run_kernel(k_paged_attn_f32<HD, 32>, p, kBoth, plan.direct, kF32Threads, (int)sizeof(F32Smem<HD, 32>), s);
}
template <class T, int NS, int HD>
void run_16bit(const AttnParams &p, const AttnPlan &plan, cudaStream_t s) {
  // Prefixes on tcgen05 and a sequence's own keys on mma.sync: two launches that
  // do not depend on each other.  (The second starts beside the first's last blocks:
  // one of the first's fills the shared memory of an SM.)
  const int tc = plan.rows == kTcRows ? plan.prefix_rows != kMmaRows ? kBoth : kOwn : kPrefix;
  bool first = false;
  if constexpr (HD <= 128 && NS <= 2) {
    if (plan.rows == kTcRows || plan.prefix_rows == kTcRows)
      first = run_kernel(k_paged_attn_tc<T, NS, HD>, p, tc, plan.direct, kTcThreads, TcShape<NS, HD>::smem, s);
  }
  if (plan.rows == kMmaRows || plan.prefix_rows == kMmaRows) {
    const int part = plan.rows != kMmaRows ? kPrefix : plan.prefix_rows == kTcRows ? kOwn : kBoth;
    run_kernel(k_paged_attn_mma<T, NS, HD>, p, part, plan.direct, kMmaThreads, MmaShape<NS, HD>::smem, s,
               first);
  }
}
template <class T, int NS>
void run_16bit_hd(const AttnParams &p, const AttnPlan &plan, cudaStream_t s) {
  if (p.kv.hd <= 64) run_16bit<T, NS, 64>(p, plan, s);
  else if (p.kv.hd <= 128) run_16bit<T, NS, 128>(p, plan, s);
  else run_16bit<T, NS, 256>(p, plan, s);
}

// Into how many pieces the keys of `blocks` blocks' rows go: the least of a
// rough count of the time in keys.  The SM with the most blocks takes longest; it
// holds `resident` at once, two of them read as fast as its share of the memory
// allows, and each round of blocks has a start and an end worth kBlockKeys.  The
// pieces have to be joined, by a second kernel that a call with shared prefixes
// needs anyway.  Measured: 131071 keys of 8 KV heads in 37 pieces 94 us, in 40 or 55
// 101 us; 48 rows of up to 4100 keys of 8 KV heads in one piece 132 us, in three
// 142 us; 128 rows of about 1100 keys of 4 KV heads in two pieces 119 us (with their
// prefixes), in three 132 us.  An f32 cache's keys take longer, so a start is worth
// fewer of them: the 48 rows 627 us with 256, 588 us with 48; 64 sequences behind a
// prefix 461 and 451; 131071 keys, eight groups and short calls the same with both.
constexpr int64_t kApartKeys = 320;
// Rows that share their keys from which on the tcgen05 kernel takes them.  Measured
// with 2048 keys of 8 KV heads in us, mma.sync / tcgen05, for 32, 64 and 96 rows: one
// sequence of f16 rows 15 / 17, 17 / 17, 21 / 19, of f32 rows 15 / 23, 19 / 23, 23 / 25;
// 48 sequences of f16 rows 103 / 101, 183 / 102, 265 / 103, of f32 rows 134 / 171,
// 246 / 173, 359 / 175.  So it is late for 33 to 64 rows of many sequences.
constexpr int64_t kTcLeast = 64;
// Blocks of the tcgen05 kernel fill an SM each and write 256 rows of partial
// results, so its keys are cut only as far as that gives idle SMs work.
int tc_pieces(int64_t blocks, int64_t keys) {
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kPagedMaxSplits, keys / (2 * kTcKeys)));
  return (int)std::min(most, std::max<int64_t>(1, kPagedSMs / std::max<int64_t>(1, blocks)));
}
constexpr int64_t kBlockKeys = 256, kF32BlockKeys = 48, kJoinKeys = 256, kPieceKeys = 4, kLeastKeys = 64;
}  // namespace

int attention_pieces(int64_t blocks, int64_t keys, int resident, int64_t start_keys, bool joined) {
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kPagedMaxSplits, keys / kLeastKeys));
  int64_t best = 1, least = INT64_MAX;
  for (int64_t s = 1; s <= most; s++) {
    const int64_t n = (blocks * s + kPagedSMs - 1) / kPagedSMs, k = (keys + s - 1) / s;
    const int64_t time = std::max(k, n * k / 2) + start_keys * ((n + resident - 1) / resident);
    const int64_t cost = time + (s > 1 ? (joined ? 0 : kJoinKeys) + kPieceKeys * s : 0);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return (int)best;
}

AttnPlan plan_attention(const jal_paged_kv &kv, const jal_ragged_batch &b, const jal_prefix_groups *g, size_t hq,
                        int act, size_t window, size_t n_sink) {
  AttnPlan a = {};
  const int64_t G = (int64_t)(hq / kv.n_heads_kv), hkv = (int64_t)kv.n_heads_kv;
  const int64_t pairs = (int64_t)b.max_q_len * G;
  // (A group has no more rows than the batch: one long prompt among single rows.)
  const int64_t group_rows = g ? std::min<int64_t>((int64_t)g->max_group * (int64_t)b.max_q_len, (int64_t)b.n_rows) : 0;
  const int64_t group_pairs = group_rows * G;
  // Which kernel: f32 caches on the CUDA cores; 16-bit ones on mma.sync in
  // tiles of 16 rows, or on tcgen05 in tiles of 256 where enough rows share
  // their keys (three bf16 parts of f32 rows, and head dims above 128, do not
  // fit its shared memory).
  const bool tc = kv.dtype != JAL_F32 && kv.head_dim <= 128 && !(act == JAL_F32 && kv.dtype == JAL_BF16);
  auto rows_for = [&](int64_t n) {
    if (kv.dtype == JAL_F32) return std::max(pairs, group_pairs) <= 8 ? 8 : 32;
    return tc && n > kTcLeast ? kTcRows : kMmaRows;
  };
  auto pieces_for = [&](int rows, int64_t blocks, int64_t keys) {
    return rows == kTcRows ? tc_pieces(blocks, keys)
                           : attention_pieces(blocks, keys, mma_blocks((int)kv.head_dim),
                                              kv.dtype == JAL_F32 ? kF32BlockKeys : kBlockKeys, g != nullptr);
  };
  a.rows = rows_for(pairs);
  a.tiles = (int)((pairs + a.rows - 1) / a.rows);
  int64_t keys = (int64_t)b.max_kv_len;
  if (window) keys = std::min<int64_t>(keys, (int64_t)(window + n_sink + b.max_q_len));
  // A few short sequences: each reads its prefix for itself, in one launch and
  // without joining (4 sequences of 160 keys of 2 KV heads: 8.7 us instead of 12.2, of
  // 310: 10.3 instead of 12.1; of 560 the joined form is the faster one).
  const bool apart = a.tiles * hkv * (int64_t)b.n_seqs <= 2 * kPagedSMs && keys <= kApartKeys && a.rows != kTcRows;
  if (g && g->n_groups && g->max_prefix_len && !apart) {
    a.prefix_rows = rows_for(group_pairs);
    a.prefix_tiles = (int)((group_pairs + a.prefix_rows - 1) / a.prefix_rows);
    a.prefix_splits = pieces_for(a.prefix_rows, a.prefix_tiles * hkv * (int64_t)g->n_groups, (int64_t)g->max_prefix_len);
    keys = std::max<int64_t>(1, keys - (int64_t)g->max_prefix_len);
  }
  a.splits = g && g->n_groups && apart ? 1 : pieces_for(a.rows, a.tiles * hkv * (int64_t)b.n_seqs, keys);
  a.direct = a.splits + a.prefix_splits == 1;
  if (!a.direct)
    a.bytes = (size_t)(a.splits + a.prefix_splits) * b.n_rows * hq * (kv.head_dim * sizeof(float) + sizeof(float2)) + 256;
  return a;
}

void launch_paged_attention(AttnParams p, const AttnPlan &plan, cudaStream_t s) {
  if (p.kv.dtype == JAL_F32) {
    if (p.kv.hd <= 64) run_f32<64>(p, plan, s);
    else if (p.kv.hd <= 128) run_f32<128>(p, plan, s);
    else run_f32<256>(p, plan, s);
  } else if (p.act == JAL_F16) {
    run_16bit_hd<__half, 1>(p, plan, s);
  } else if (p.act == JAL_BF16) {
    run_16bit_hd<__nv_bfloat16, 1>(p, plan, s);
  } else if (p.kv.dtype == JAL_F16) {
    run_16bit_hd<__half, 2>(p, plan, s);
  } else {
    run_16bit_hd<__nv_bfloat16, 3>(p, plan, s);
  }
  if (!plan.direct) launch_attention_join(p, plan.prefix_rows, s);
}

void launch_attention_join(const AttnParams &p, int prefix_rows, cudaStream_t s) {
  const int64_t by_seq = (int64_t)p.n_seqs * p.max_q;
  launch(p.n_rows <= by_seq ? k_paged_attn_join<true> : k_paged_attn_join<false>,
         std::min<int64_t>(p.n_rows, by_seq) * p.hq, kJoinThreads, 0, true, s, p, prefix_rows);
}

}  // namespace jal
