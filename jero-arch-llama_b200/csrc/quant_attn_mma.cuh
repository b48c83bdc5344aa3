// Attention of few query rows over a paged cache of 8- or 4-bit codes on the
// warp-level matrix instructions (mma.sync m16n8k16).  Included by quant_attn.cu.
//
//   out = sum_t softmax(scale * dk[t] * (q . ck[t])) * dv[t] * cv[t]
//
// with codes c and scales d.  Codes are whole numbers of at most 8 bits, which f16
// holds exactly, so the products run over codes, and the scales multiply scores and
// weights in f32: nothing of the cache is rounded.  q is carried as NS f16 parts of
// the row times a power of two (one part for 16-bit rows, which is exact for f16 and for
// bf16 down to 2^-27 of the row's largest; two, 22 bits, for f32 rows), and so are
// the weights times dv.
//
// A block takes MT tiles of 16 query rows of one KV head (the query heads of a
// group, and neighbouring tokens); its four warps take 16 keys each in turn, and
// each is on its own until the end: it copies its keys' codes and scales with cp.async
// into its own ring, and has its own running maxima, sums and output.
//
// A product's terms may be summed in any order, so the fragments of K take the dims
// in the order in which a lane finds them in 16 bytes of a row, and q is laid out
// to match; the columns of V's fragments are the dims that a lane has of one
// row, and the result is put in order at the end.  A code becomes f16 by
// being placed in the low mantissa bits of 1024 (its sum with 1024, exactly), from
// which 1024 and the code's offset are subtracted.
#pragma once

#include "paged_attn_mma.cuh"
#include "quant_kv.hpp"

namespace jal {
namespace paged {

// f16 weights times dv refer to kQuantHeadroom less than the running maximum and to
// the power of two below the largest |dv| so far: they stay below 2^15, and each
// is off by 2^-25 beside its relative error.
constexpr int kQuantHeadroom = 13;

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  uint32_t v;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
  return v;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t v;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(a), "r"(b), "r"(c));
  return v;
}
constexpr uint32_t kH2_1024 = 0x64006400u, kH2_1032 = 0x64086408u, kH2_1152 = 0x64806480u, kH2_16th = 0x2C002C00u,
                   kH2_m72 = 0xD480D480u;

// Codes of one 32-bit word of a row as pairs of f16: 8 bits, 4 codes: (0, 1), (2, 3);
// 4 bits, 8 codes: (0, 4), (1, 5), (2, 6), (3, 7).
template <int BITS>
__device__ __forceinline__ void row_pairs(uint32_t w, uint32_t *pair) {
  if constexpr (BITS == 8) {
    w ^= 0x80808080u;
    pair[0] = h2_sub(__byte_perm(w, kH2_1024, 0x5150), kH2_1152);
    pair[1] = h2_sub(__byte_perm(w, kH2_1024, 0x5352), kH2_1152);
  } else {
    const uint32_t u = w >> 8;
    pair[0] = h2_sub((w & 0x000F000Fu) | kH2_1024, kH2_1032);
    pair[1] = h2_fma((w & 0x00F000F0u) | kH2_1024, kH2_16th, kH2_m72);
    pair[2] = h2_sub((u & 0x000F000Fu) | kH2_1024, kH2_1032);
    pair[3] = h2_fma((u & 0x00F000F0u) | kH2_1024, kH2_16th, kH2_m72);
  }
}
// The same dim of two rows as a pair, for the 4 or 8 codes of a word of each.
template <int BITS>
__device__ __forceinline__ void column_pairs(uint32_t a, uint32_t b, uint32_t *pair) {
  uint32_t lo = __byte_perm(a, b, 0x5410), hi = __byte_perm(a, b, 0x7632);
  if constexpr (BITS == 8) {
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    pair[0] = h2_sub(__byte_perm(lo, kH2_1024, 0x5250), kH2_1152);
    pair[1] = h2_sub(__byte_perm(lo, kH2_1024, 0x5351), kH2_1152);
    pair[2] = h2_sub(__byte_perm(hi, kH2_1024, 0x5250), kH2_1152);
    pair[3] = h2_sub(__byte_perm(hi, kH2_1024, 0x5351), kH2_1152);
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t w = i ? hi : lo, u = w >> 8;
      pair[4 * i] = h2_sub((w & 0x000F000Fu) | kH2_1024, kH2_1032);
      pair[4 * i + 1] = h2_fma((w & 0x00F000F0u) | kH2_1024, kH2_16th, kH2_m72);
      pair[4 * i + 2] = h2_sub((u & 0x000F000Fu) | kH2_1024, kH2_1032);
      pair[4 * i + 3] = h2_fma((u & 0x00F000F0u) | kH2_1024, kH2_16th, kH2_m72);
    }
  }
}

__device__ __forceinline__ void copy4(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t *w) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

// Blocks on an SM, by registers.
constexpr int quant_blocks(int hd, int mt) { return hd > 128 || mt > 1 ? 2 : 3; }

template <int BITS, int NS, int HD, int MT>
struct QuantShape {
  static constexpr int blocks = quant_blocks(HD, MT);
  static constexpr int rows = 16 * MT;
  static constexpr int row_bytes = HD * BITS / 8;
  static constexpr int chunks = row_bytes / 16;           // 16-byte pieces of a row
  static constexpr int half = kMmaKeys * row_bytes;       // bytes of a stage's K (or V)
  static constexpr int stage = 2 * half + 2 * kMmaKeys * 4;
  static constexpr int stages = row_bytes <= 64 ? 6 : row_bytes == 128 ? 4 : 3;
  static constexpr int ring = kMmaWarps * stages * stage;
  static constexpr int q_part = HD / 16 * 512;            // one part of 16 rows, as fragments
  static constexpr int q_bytes = NS * MT * q_part;
  static constexpr int out_row = HD + HD / 4;             // floats of a row where warps' results are joined
  static constexpr int merge = kMmaWarps * rows * out_row * 4;
  static constexpr int smem = q_bytes + (ring > merge ? ring : merge);
  // Where 16-byte piece c of key r lies: conflict-free for the lanes' reads of K (a
  // quarter warp: two neighbouring keys, four pieces) and of V (keys two apart).
  static __device__ __forceinline__ uint32_t k_at(int r, int c) {
    return r * row_bytes + ((chunks >= 8 ? c ^ ((r & 1) << 2) : c) * 16);
  }
  static __device__ __forceinline__ uint32_t v_at(int r, int c) {
    const int pos = (r >> 1) | ((r & 1) << 3);
    const int x = chunks == 16 ? (pos & 1) | ((pos & 2) << 1) : chunks == 8 ? (pos & 3) << 1 : chunks == 4 ? pos & 2 : 0;
    return pos * row_bytes + ((c ^ x) * 16);
  }
};

template <int BITS, int NS, int HD, int MT>
__global__ void __launch_bounds__(kMmaThreads, QuantShape<BITS, NS, HD, MT>::blocks)
    k_quant_attn_mma(const __grid_constant__ QuantAttnParams qp, const bool direct) {
  using S = QuantShape<BITS, NS, HD, MT>;
  const AttnParams &p = qp.a;
  extern __shared__ __align__(128) char smem_raw[];
  __shared__ RowMask masks[S::rows];
  __shared__ float q_scale[S::rows];
  __shared__ float2 row_ml[kMmaWarps][S::rows];
  __shared__ uint32_t present[kMmaWarps][S::stages];
  pdl_trigger();
  Tile t;
  if (!block_tile(p, kOwn, S::rows, kMmaWarps * kMmaKeys, t)) {
    pdl_wait();
    return;
  }
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, hd = p.kv.hd;
  const int n8 = lane / 4, j4 = lane % 4;  // this lane's key (or column), and quarter
  const uint32_t sq = smem_u32(smem_raw), ring = sq + S::q_bytes + warp * (S::stages * S::stage);

  // This warp's keys: chunks of 16 of [u0, u1), every fourth.  Lanes i and i + 16
  // look up where key i of a chunk lies, one chunk ahead of its copies.
  const int n_chunks = (t.u1 - t.u0 + kMmaKeys - 1) / kMmaKeys;
  auto locate = [&](int c) -> Slot {
    const int u = t.u0 + c * kMmaKeys + lane % kMmaKeys;
    return c < n_chunks && u < t.u1 ? slot_of(p.kv, t, t.key(u)) : Slot{-1, 0};
  };
  auto copy = [&](const Slot &where, int stage) {
    const int64_t at = slot_offset(p.kv, where, t.head);
    const uint32_t dst = ring + stage * S::stage;
    const uint32_t bits = __ballot_sync(0xffffffffu, at >= 0) & 0xffffu;
    if (lane == 0) present[warp][stage] = bits;
    {  // lane i: K's scale of key i; lane i + 16: V's
      const int64_t e = at >= 0 ? (int64_t)where.page * qp.sc.s_page + t.head * qp.sc.s_head + where.slot : 0;
      copy4(dst + 2 * S::half + lane * 4, (lane < kMmaKeys ? qp.sc.k : qp.sc.v) + e, at >= 0);
    }
#pragma unroll
    for (int i = 0; i < S::chunks / 2; i++) {
      const int r = (i * 32 + lane) / S::chunks, c = (i * 32 + lane) % S::chunks;
      const int64_t o = __shfl_sync(0xffffffffu, at, r);
      const bool there = o >= 0 && c * (128 / BITS) < hd;
      const int64_t e = there ? o + c * 16 : 0;
      copy16(dst + S::k_at(r, c), (const char *)p.kv.k + e, there);
      copy16(dst + S::half + S::v_at(r, c), (const char *)p.kv.v + e, there);
    }
    copies_done();
  };
  Slot next = locate(warp);
#pragma unroll
  for (int i = 0; i < S::stages - 1; i++) {
    const Slot at = next;
    next = locate(warp + (i + 1) * kMmaWarps);
    copy(at, i);
  }
  // Query rows into shared memory as fragments: a row times 2^e, so that its
  // largest element lies in [2^13, 2^14), in NS f16 parts.  Eight threads a row.
#pragma unroll 1
  for (int m = 0; m < MT; m++) {
    const int r = tid / 8, j = m * 16 + r, sub = tid % 8;
    const bool real = j < t.rows;
    const int64_t qo = real ? q_offset(p, t, j) : 0;
    constexpr int N = HD / 8;  // dims of a thread: fragments ks = sub, sub + 8, .. whole (16 dims each) or halves
    float v[N];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
      // Thread `sub` has the dims sub * 2 + (i / 2) * 16 + i % 2.
      const int d = sub * 2 + (i / 2) * 16 + i % 2;
      v[i] = real && d < hd ? load_as_f32(p.q, qo + d, p.act) : 0.0f;
      if (fabsf(v[i]) < INFINITY) top = fmaxf(top, fabsf(v[i]));
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = top > 0.0f ? 13 - ilogbf(top) : 0;
    // in two steps: 2^e itself may lie outside f32's range
    const float a = exp2f((float)(e / 2)), b = exp2f((float)(e - e / 2));
    if (sub == 0) {
      masks[j] = real ? row_mask(p, t, j) : RowMask{0, 0};
      q_scale[j] = p.scale_log2 * ((1.0f / a) / b);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int d = sub * 2 + (i / 2) * 16 + i % 2;
      // Where the lanes find dim d in a row of K: quarter jj, word w of it, code c of
      // the word; the word's pairs are halves of the fragments ks.
      constexpr int codes = 32 / BITS, lane_bytes = S::chunks >= 4 ? 16 : 8, per_lane = lane_bytes * 8 / BITS;
      const int piece = d / (4 * per_lane), jj = d / per_lane % 4, w = d % per_lane / codes, c = d % codes;
      const int pr = BITS == 8 ? c / 2 : c % 4, h = BITS == 8 ? c % 2 : c / 4;
      const int ks = piece * (per_lane / 4) + w * (codes / 4) + pr / 2, reg = (pr % 2) * 2 + (r >= 8 ? 1 : 0);
      float x = v[i] * a * b;
#pragma unroll
      for (int s = 0; s < NS; s++) {
        const __half part = __float2half_rn(x);
        x -= __half2float(part);
        *(__half *)(smem_raw + (s * MT + m) * S::q_part + ks * 512 + ((r % 8) * 4 + jj) * 16 + reg * 4 + h * 2) = part;
      }
    }
  }
  __syncthreads();

  // Rows 16 m + lane / 4 and that + 8 are this lane's.
  // Rows that do not exist see everything: they have no say in what is masked.
  const RowSpan every = {0x7fffffff, 0, 0};
  RowSpan span[MT][2];
  float f[MT][2];
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int r = m * 16 + h * 8 + n8;
      span[m][h] = r < t.rows ? row_span(p, t, masks[r]) : every;
      f[m][h] = q_scale[r];
    }
  float o[MT][HD / 8][4];
  float top[MT][2], ref[MT][2], l[MT][2];  // running maxima, what the weights refer to, their sums
#pragma unroll
  for (int m = 0; m < MT; m++) {
#pragma unroll
    for (int i = 0; i < HD / 8; i++) o[m][i][0] = o[m][i][1] = o[m][i][2] = o[m][i][3] = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      top[m][h] = ref[m][h] = -INFINITY;
      l[m][h] = 0.0f;
    }
  }
  int unit = 1;  // V's scales are taken over 2^(unit - 127)

  int stage = 0;
#pragma unroll 1
  for (int c = warp; c < n_chunks; c += kMmaWarps) {
    {  // the copies of the chunk stages - 1 ahead
      const Slot at = next;
      const int ahead = c + (S::stages - 1) * kMmaWarps;
      next = locate(ahead + kMmaWarps);
      int ns = stage + S::stages - 1;
      if (ns >= S::stages) ns -= S::stages;
      copy(at, ns);
    }
    copies_wait<S::stages - 1>();
    __syncwarp();
    const uint32_t kb = ring + stage * S::stage, vb = kb + S::half, sb = vb + S::half;
    const uint32_t bits = present[warp][stage];
    float s[MT][2][4] = {};
    {
      constexpr int lane_bytes = S::chunks >= 4 ? 16 : 8, words = lane_bytes / 4, codes = 32 / BITS;
      constexpr int pieces = S::row_bytes / (4 * lane_bytes);
#pragma unroll
      for (int pc = 0; pc < pieces; pc++) {
        uint32_t w[2][words];
#pragma unroll
        for (int n = 0; n < 2; n++) {
          if constexpr (lane_bytes == 16) lds<16>(kb + S::k_at(n * 8 + n8, pc * 4 + j4), w[n]);
          else lds<8>(kb + S::k_at(n * 8 + n8, 0) + j4 * 8, w[n]);
        }
#pragma unroll
        for (int x = 0; x < words; x++) {
          uint32_t b[2][codes / 2];
          row_pairs<BITS>(w[0][x], b[0]);
          row_pairs<BITS>(w[1][x], b[1]);
#pragma unroll
          for (int k = 0; k < codes / 4; k++) {
            const int ks = (pc * words + x) * (codes / 4) + k;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
              for (int i = 0; i < NS; i++) {
                uint32_t a[4];
                lds<16>(sq + (i * MT + m) * S::q_part + ks * 512 + lane * 16, a);
                mma16816<__half>(s[m][0], a, b[0][2 * k], b[0][2 * k + 1]);
                mma16816<__half>(s[m][1], a, b[1][2 * k], b[1][2 * k + 1]);
              }
          }
        }
      }
    }
    // Scales of this lane's keys: 2 j4, 2 j4 + 1 and those + 8.
    uint32_t dkw[2][2], dvw[2][2];
    lds<8>(sb + j4 * 8, dkw[0]);
    lds<8>(sb + 32 + j4 * 8, dkw[1]);
    lds<8>(sb + 64 + j4 * 8, dvw[0]);
    lds<8>(sb + 96 + j4 * 8, dvw[1]);
    const int u = t.u0 + c * kMmaKeys;
    bool whole = bits == 0xffffu;
#pragma unroll
    for (int m = 0; m < MT; m++) whole = whole && span[m][0].all(u, kMmaKeys) && span[m][1].all(u, kMmaKeys);
    const bool masked = __any_sync(0xffffffffu, !whole);
    uint32_t see[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int h = 0; h < 2; h++) see[m][h] = masked ? bits & span[m][h].bits(u) : 0xffffffffu;
    // A larger scale of V than any before: the output is taken over its power of two.
    {
      uint32_t most = 0;
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t x = dvw[n][e] & 0x7fffffffu;
          most = max(most, x < 0x7f800000u ? x : 0u);
        }
      const int e = min((int)(__reduce_max_sync(0xffffffffu, most) >> 23), 253);
      if (e > unit) {
        const float less = exp2f((float)(unit - e));
        unit = e;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < HD / 8; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) o[m][i][q] *= less;
      }
    }
    const float over = __uint_as_float((uint32_t)(254 - unit) << 23);  // 2^(127 - unit)
    uint32_t w[MT][NS][4];
#pragma unroll
    for (int m = 0; m < MT; m++) {
      bool raise = false;
      float now[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float &x = s[m][n][2 * h + e];
            x = x * f[m][h] * __uint_as_float(dkw[n][e]);
            if (masked && !((see[m][h] >> (n * 8 + j4 * 2 + e)) & 1)) x = -INFINITY;
          }
        float x = fmaxf(fmaxf(s[m][0][2 * h], s[m][0][2 * h + 1]), fmaxf(s[m][1][2 * h], s[m][1][2 * h + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        now[h] = fmaxf(top[m][h], fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2)));
        raise = raise || now[h] != top[m][h];
      }
      if (__any_sync(0xffffffffu, raise)) {
        float less[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float r = reference_of<kQuantHeadroom>(now[h]);
          less[h] = now[h] == top[m][h] ? 1.0f : exp2_fast(ref[m][h] - r);
          top[m][h] = now[h];
          ref[m][h] = r;
          l[m][h] *= less[h];
        }
#pragma unroll
        for (int i = 0; i < HD / 8; i++)
#pragma unroll
          for (int q = 0; q < 4; q++) o[m][i][q] *= less[q / 2];
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float r = ref[m][h] == -INFINITY ? 0.0f : ref[m][h];
#pragma unroll
        for (int n = 0; n < 2; n++) {
          float x[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            x[e] = exp2_fast(s[m][n][2 * h + e] - r);
            l[m][h] += x[e];
            x[e] *= __uint_as_float(dvw[n][e]) * over;
            // (What a row does not see has no effect on it, whatever its scale is.)
            if (masked && !((see[m][h] >> (n * 8 + j4 * 2 + e)) & 1)) x[e] = 0.0f;
          }
          uint32_t part[NS];
          split2<__half, NS>(x[0], x[1], part);
#pragma unroll
          for (int i = 0; i < NS; i++) w[m][i][2 * n + h] = part[i];
        }
      }
    }
    {
      // V: this lane's dims are n8 * (HD / 8) .., its keys 2 j4, 2 j4 + 1 and those + 8.
      constexpr int lane_bytes = S::row_bytes / 8, step = lane_bytes < 16 ? lane_bytes : 16, codes = 32 / BITS;
#pragma unroll
      for (int pc = 0; pc < lane_bytes / step; pc++) {
        uint32_t x[4][step / 4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int key = j4 * 2 + k % 2 + (k / 2) * 8, byte = n8 * lane_bytes + pc * 16;
          lds<step>(vb + S::v_at(key, byte / 16) + byte % 16, x[k]);
        }
#pragma unroll
        for (int y = 0; y < step / 4; y++) {
          uint32_t b0[codes], b1[codes];
          column_pairs<BITS>(x[0][y], x[1][y], b0);
          column_pairs<BITS>(x[2][y], x[3][y], b1);
#pragma unroll
          for (int k = 0; k < codes; k++)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
              for (int i = 0; i < NS; i++)
                mma16816<__half>(o[m][(pc * (step / 4) + y) * codes + k], w[m][i], b0[k], b1[k]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
    if (++stage == S::stages) stage = 0;
  }
  copies_wait<0>();
  __syncthreads();  // no warp reads its ring any more
  pdl_wait();
  // The four warps' results, joined through shared memory: element (i, n) of a row, dim
  // n * (HD / 8) + i, at i * 8 + n + i / 4 * 8.
  float *const merge = (float *)(smem_raw + S::q_bytes);
  const float back = exp2f((float)(unit - 127));
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float x = l[m][h];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      const int r = m * 16 + h * 8 + n8;
      if (j4 == 0) row_ml[warp][r] = make_float2(ref[m][h], x);
      float *const a = merge + (warp * S::rows + r) * S::out_row + j4 * 2;
#pragma unroll
      for (int i = 0; i < HD / 8; i++)
        *(float2 *)(a + i * 8 + i / 4 * 8) = make_float2(o[m][i][2 * h] * back, o[m][i][2 * h + 1] * back);
    }
  __syncthreads();
  for (int i = tid; i < t.rows * (HD / 4); i += kMmaThreads) {
    const int j = i / (HD / 4), d = (i % (HD / 4)) * 4;
    if (d >= hd) continue;
    float most = -INFINITY, sum_l = 0.0f;
#pragma unroll
    for (int w = 0; w < kMmaWarps; w++) most = fmaxf(most, row_ml[w][j].x);
    const float safe = most == -INFINITY ? 0.0f : most;
    float sum[4] = {};
    const int n = d / (HD / 8), i0 = d % (HD / 8);
#pragma unroll
    for (int w = 0; w < kMmaWarps; w++) {
      const float2 ml = row_ml[w][j];
      if (ml.y == 0.0f) continue;
      const float a = exp2f(ml.x - safe);
      sum_l = fmaf(a, ml.y, sum_l);
      const float *const v = merge + (w * S::rows + j) * S::out_row + i0 * 8 + n + i0 / 4 * 8;
#pragma unroll
      for (int q = 0; q < 4; q++) sum[q] = fmaf(a, v[q * 8], sum[q]);
    }
    if (direct) {
      const float inv = sum_l == 0.0f ? 0.0f : 1.0f / sum_l;
      const int64_t oo = out_offset(p, t, j) + d;
      if (p.act == JAL_F32)
        *(float4 *)((float *)p.out + oo) = make_float4(sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv);
      else if (p.act == JAL_F16)
        *(uint2 *)((__half *)p.out + oo) = make_uint2(pack2<__half>(sum[0] * inv, sum[1] * inv), pack2<__half>(sum[2] * inv, sum[3] * inv));
      else
        *(uint2 *)((__nv_bfloat16 *)p.out + oo) =
            make_uint2(pack2<__nv_bfloat16>(sum[0] * inv, sum[1] * inv), pack2<__nv_bfloat16>(sum[2] * inv, sum[3] * inv));
    } else {
      const int64_t pi = part_index(p, t, j);
      if (d == 0) p.part_ml[pi] = make_float2(most, sum_l);
      *(float4 *)(p.part_o + pi * hd + d) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    }
  }
}

}  // namespace paged
}  // namespace jal
