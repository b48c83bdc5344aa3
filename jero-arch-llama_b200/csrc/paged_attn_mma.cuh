// Attention of few query rows over a 16-bit paged cache on the warp-level
// matrix instructions (mma.sync m16n8k16).  Included by paged_attn.cu.
//
// A block takes 16 query rows of one KV head (the query heads of a group, and
// neighbouring tokens) and its four warps take 16 keys each in turn.  A warp
// is on its own until the end: it copies its keys with cp.async into its own
// ring of shared memory stages, has its own running maximum, sum and output,
// and never waits for another warp; the four results are joined at the end.
// Few rows against many keys is bound by reading the cache (48 rows of up to 4100
// keys of 8 KV heads: 130 us, 6.1 TB/s; 131071 keys: 92 us, 5.8 TB/s), so what counts is
// bytes in flight: the stages of 4 warps x 3 blocks on an SM, 192 KB.
//
// f32 rows are not rounded to the cache's type: q is split into the sum of NS
// 16-bit parts (two f16 parts of q scaled by a power of two per row, 22 bits;
// three bf16 parts, 24 bits), the weights likewise, and the products of the
// parts are added in f32.  With 16-bit rows (NS = 1) q is exact and the
// weights are rounded once, to 2^-11 or 2^-8 of themselves, less than what
// the rounding of the result costs.
//
// f16 has no bits below 2^-24 and few below 2^-14, so f16 weights refer to
// kHeadroom less than the running maximum (base 2): the largest are near the
// top of the type, and a key's weight is off by 2^-25 of a unit, 2^-40 of
// the largest weight, beside its relative error.  One position far above
// 10^5 others then leaves them their share: 20 nats below the maximum a weight
// still has its 11 bits, 12 nats below it both parts' 22.  The sum and the
// output carry the same power of two, which their quotient does not have.
#pragma once

#include <type_traits>

#include "paged_dev.cuh"

namespace jal {
namespace paged {

constexpr int kMmaRows = 16, kMmaWarps = 4, kMmaKeys = 16;
constexpr int kMmaThreads = kMmaWarps * 32;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes into shared memory; zeros where `there` is false (src is then only
// an address that is not read).
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The remainder of x after its first part in T, NS times: x = sum of parts.
// Three bf16 parts are cut off, not rounded: 8 bits each are all 24, and the
// largest f32 values do not become infinite.
template <class T, int NS>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&part)[NS]) {
  if constexpr (NS == 3) {
#pragma unroll
    for (int i = 0; i < NS; i++) {
      const uint32_t x = __float_as_uint(a) & 0xFFFF0000u, y = __float_as_uint(b) & 0xFFFF0000u;
      part[i] = (x >> 16) | y;
      a -= __uint_as_float(x);
      b -= __uint_as_float(y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NS; i++) {
      part[i] = pack2<T>(a, b);
      const float2 f = unpack2<T>(part[i]);
      a -= f.x;
      b -= f.y;
    }
  }
}

// What weights refer to where the running maximum is `top`: SHIFT less, so that
// the largest weight is 2^SHIFT (of maxima so large that the difference is not
// exact to a quarter, the maximum itself).
template <int SHIFT>
__device__ __forceinline__ float reference_of(float top) {
  return SHIFT && fabsf(top) < 8388608.0f ? top - (float)SHIFT : top;
}
template <class T>
constexpr int kHeadroom = std::is_same<T, __half>::value ? 15 : 0;  // bf16 has the exponents of f32

// Blocks on an SM.  Three, with two stages a warp, read a 131071-key row in 94 us
// where two with three stages took 99 us: one block's start and end go on beside
// the others' copies.  (The registers of head dim 256 allow two.)
constexpr int mma_blocks(int hd) { return hd > 128 ? 2 : 3; }

template <int NS, int HD>
struct MmaShape {
  static constexpr int blocks = mma_blocks(HD);
  static constexpr int stages = HD == 64 ? 4 : 2;
  static constexpr int chunks = HD / 8;              // 16-byte pieces of a row
  static constexpr int half = kMmaKeys * HD * 2;     // bytes of a stage's K (or V)
  static constexpr int ring = kMmaWarps * stages * 2 * half;
  static constexpr int q_bytes = NS * kMmaRows * HD * 2;
  static constexpr int merge = kMmaWarps * kMmaRows * HD * 4;
  static constexpr int smem = q_bytes + (ring > merge ? ring : merge);
};

template <class T, int NS, int HD>
__global__ void __launch_bounds__(kMmaThreads, MmaShape<NS, HD>::blocks) k_paged_attn_mma(const __grid_constant__ AttnParams p, const int part, const bool direct) {
  using S = MmaShape<NS, HD>;
  extern __shared__ __align__(128) char smem_raw[];
  __shared__ RowMask masks[kMmaRows];
  __shared__ float q_scale[kMmaRows];
  __shared__ float2 row_ml[kMmaWarps][kMmaRows];
  __shared__ uint32_t present[kMmaWarps][S::stages];
  pdl_trigger();
  Tile t;
  if (!block_tile(p, part, kMmaRows, kMmaWarps * kMmaKeys, t)) {
    pdl_wait();
    return;
  }
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, hd = p.kv.hd;
  const uint32_t sq = smem_u32(smem_raw), ring = sq + S::q_bytes + warp * (S::stages * 2 * S::half);
  char *const q_sm = smem_raw;

  // This warp's keys: chunks of 16 of [u0, u1), every fourth.  Lanes 0..15
  // look up where a chunk's keys lie one chunk ahead of its copies.
  const int n_chunks = (t.u1 - t.u0 + kMmaKeys - 1) / kMmaKeys;
  auto locate = [&](int c) -> Slot {
    const int u = t.u0 + c * kMmaKeys + lane;
    return lane < kMmaKeys && c < n_chunks && u < t.u1 ? slot_of(p.kv, t, t.key(u)) : Slot{-1, 0};
  };
  auto copy = [&](const Slot &where, int stage) {
    const int64_t at = slot_offset(p.kv, where, t.head);
    const uint32_t dst = ring + stage * 2 * S::half;
    const uint32_t bits = __ballot_sync(0xffffffffu, at >= 0) & 0xffffu;
    if (lane == 0) present[warp][stage] = bits;
    // Eight lanes copy 128 bytes of a row; a lane has the rows lane / 8 + 4 i.
    const int c8 = lane % 8, r8 = lane / 8;
#pragma unroll
    for (int i = 0; i < kMmaKeys / 4; i++) {
      const int64_t o = __shfl_sync(0xffffffffu, at, r8 + 4 * i);
      const int r = r8 + 4 * i;
      const uint32_t d = dst + r * (HD * 2) + ((c8 ^ (r & 7)) * 16);
      const int64_t e = o >= 0 ? o + c8 * 8 : 0;
#pragma unroll
      for (int h = 0; h < HD / 64; h++) {
        const bool there = o >= 0 && h * 64 + c8 * 8 < hd;
        copy16(d + h * 128, (const T *)p.kv.k + (there ? e + h * 64 : 0), there);
        copy16(d + S::half + h * 128, (const T *)p.kv.v + (there ? e + h * 64 : 0), there);
      }
    }
    copies_done();
  };
  Slot next;
  // Query rows into shared memory, in their NS parts, in the swizzle of the
  // key rows.  f16 parts: the row times 2^e, so that the largest element lies
  // in [2^13, 2^14) and the second part keeps its bits.
  {
    const int j = tid / 8;  // 8 threads a row
    constexpr int N = HD / 16;
    const bool real = j < t.rows;
    const int64_t qo = real ? q_offset(p, t, j) : 0;
    float v[2 * N], factor = 1.0f;
    float top = 0.0f;
    uint32_t raw[NS == 1 ? N : 1];  // (asked for before the copies, looked at behind them)
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int d = (tid % 8) * 2 + i * 16;
      if constexpr (NS == 1) {
        raw[i] = real && d < hd ? *(const uint32_t *)((const T *)p.q + qo + d) : 0u;
      } else {
        const float2 f = real && d < hd ? *(const float2 *)((const float *)p.q + qo + d) : make_float2(0.0f, 0.0f);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
    next = locate(warp);
#pragma unroll
    for (int i = 0; i < S::stages - 1; i++) {
      const Slot at = next;
      next = locate(warp + (i + 1) * kMmaWarps);
      copy(at, i);
    }

    if (NS == 2) {
#pragma unroll
      for (int i = 0; i < 2 * N; i++)
        if (fabsf(v[i]) < INFINITY) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int e = top > 0.0f ? 13 - ilogbf(top) : 0;
      // in two steps: 2^e itself may lie outside f32's range
      const float a = exp2f((float)(e / 2)), b = exp2f((float)(e - e / 2));
#pragma unroll
      for (int i = 0; i < 2 * N; i++) v[i] = v[i] * a * b;
      factor = (1.0f / a) / b;
    }
    if (tid % 8 == 0) {
      masks[j] = real ? row_mask(p, t, j) : RowMask{0, 0};
      q_scale[j] = p.scale_log2 * factor;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      uint32_t part[NS];
      if constexpr (NS == 1) part[0] = raw[i];
      else split2<T, NS>(v[2 * i], v[2 * i + 1], part);
      const int ch = 2 * i + (tid % 8) / 4;
#pragma unroll
      for (int s = 0; s < NS; s++)
        *(uint32_t *)(q_sm + (s * kMmaRows + j) * (HD * 2) + ((ch ^ (j & 7)) * 16) + (tid % 4) * 4) = part[s];
    }
  }
  __syncthreads();

  // Rows lane/4 and lane/4 + 8 are this lane's.
  const int r0 = lane / 4;
  // Rows that do not exist see everything: they have no say in what is masked.
  const RowSpan every = {0x7fffffff, 0, 0};
  const RowSpan m0 = r0 < t.rows ? row_span(p, t, masks[r0]) : every;
  const RowSpan m1 = r0 + 8 < t.rows ? row_span(p, t, masks[r0 + 8]) : every;
  const float f0 = q_scale[r0], f1 = q_scale[r0 + 8];
  const RowMask mine = masks[lane < t.rows ? lane : 0];  // (a tile has a row)
  // Are there keys of the tile that some row does not see?  Rows that see the same see all
  // of it, but for a shared prefix, which goes on behind rows inside it.
  const bool mixed = __any_sync(0xffffffffu, mine.lim != masks[0].lim || mine.wlo != masks[0].wlo || mine.lim < t.hi);
  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  // Running maxima, what the weights refer to, and their sums.
  float top0 = -INFINITY, top1 = -INFINITY, ref0 = -INFINITY, ref1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  uint32_t bad = 0;

  int stage = 0;
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
    const uint32_t kb = ring + stage * 2 * S::half, vb = kb + S::half;
    const uint32_t bits = present[warp][stage];
    float s[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < HD / 16; ks++) {
      // K: matrices (keys 0-7, k 0-7), (keys 0-7, k 8-15), (keys 8-15, ..)
      uint32_t b[4];
      const int kr = (lane & 7) + ((lane >> 4) & 1) * 8, kc = 2 * ks + ((lane >> 3) & 1);
      ldsm4(b, kb + kr * (HD * 2) + ((kc ^ (kr & 7)) * 16));
      const int qr = lane & 15, qc = 2 * ks + (lane >> 4);
#pragma unroll
      for (int i = 0; i < NS; i++) {
        uint32_t a[4];
        ldsm4(a, sq + (i * kMmaRows + qr) * (HD * 2) + ((qc ^ (qr & 7)) * 16));
        mma16816<T>(s[0], a, b[0], b[1]);
        mma16816<T>(s[1], a, b[2], b[3]);
      }
    }
    const int u = t.u0 + c * kMmaKeys;
    const bool masked = __any_sync(0xffffffffu, bits != 0xffffu || !m0.all(u, kMmaKeys) || !m1.all(u, kMmaKeys));
    const uint32_t see0 = bits & m0.bits(u), see1 = bits & m1.bits(u);
#pragma unroll
    for (int n = 0; n < 2; n++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        s[n][e] *= f0;
        s[n][2 + e] *= f1;
        if (masked) {
          const int i = n * 8 + (lane & 3) * 2 + e;
          if (!((see0 >> i) & 1)) s[n][e] = -INFINITY;
          if (!((see1 >> i) & 1)) s[n][2 + e] = -INFINITY;
        }
      }
    }
    if (masked && mixed) {  // a value that some row must not meet
#pragma unroll
      for (int i = 0; i < kMmaKeys * S::chunks / 32; i++) {
        uint4 w;
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                     : "r"(vb + (i * 32 + lane) * 16));
        watch8<T>(bad, w);
      }
    }
    float n0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
    float n1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
    n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 1));
    n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 1));
    n0 = fmaxf(top0, fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 2)));
    n1 = fmaxf(top1, fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 2)));
    if (__any_sync(0xffffffffu, n0 != top0 || n1 != top1)) {
      const float r0 = reference_of<kHeadroom<T>>(n0), r1 = reference_of<kHeadroom<T>>(n1);
      const float c0 = n0 == top0 ? 1.0f : exp2_fast(ref0 - r0), c1 = n1 == top1 ? 1.0f : exp2_fast(ref1 - r1);
      top0 = n0;
      top1 = n1;
      ref0 = r0;
      ref1 = r1;
      l0 *= c0;
      l1 *= c1;
#pragma unroll
      for (int i = 0; i < HD / 8; i++) {
        o[i][0] *= c0;
        o[i][1] *= c0;
        o[i][2] *= c1;
        o[i][3] *= c1;
      }
    }
    const float b0 = ref0 == -INFINITY ? 0.0f : ref0, b1 = ref1 == -INFINITY ? 0.0f : ref1;
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        s[n][e] = exp2_fast(s[n][e] - b0);
        s[n][2 + e] = exp2_fast(s[n][2 + e] - b1);
        l0 += s[n][e];
        l1 += s[n][2 + e];
      }
    uint32_t w[NS][4];
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        uint32_t part[NS];
        split2<T, NS>(s[n][2 * h], s[n][2 * h + 1], part);
#pragma unroll
        for (int i = 0; i < NS; i++) w[i][2 * n + h] = part[i];
      }
#pragma unroll
    for (int d = 0; d < HD / 16; d++) {
      // V transposed: matrices (keys 0-7, dims 0-7), (keys 8-15, dims 0-7), (.., dims 8-15)
      uint32_t b[4];
      const int vr = lane & 15, vc = 2 * d + (lane >> 4);
      ldsm4t(b, vb + vr * (HD * 2) + ((vc ^ (vr & 7)) * 16));
#pragma unroll
      for (int i = 0; i < NS; i++) {
        mma16816<T>(o[2 * d], w[i], b[0], b[1]);
        mma16816<T>(o[2 * d + 1], w[i], b[2], b[3]);
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
    if (++stage == S::stages) stage = 0;
  }
  copies_wait<0>();
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  if (__syncthreads_or(watched_bad<T>(bad))) {  // (also: no warp reads its ring any more)
    for (int j = warp; j < t.rows; j += kMmaWarps) attend_row_alone(p, t, j, direct);
    pdl_wait();
    return;
  }

  // A launch beside another one ends after it, so that what waits for this
  // launch has waited for both.
  pdl_wait();
  // The four warps' results, joined through shared memory.
  float *const merge = (float *)(smem_raw + S::q_bytes);
  if ((lane & 3) == 0) {
    row_ml[warp][r0] = make_float2(ref0, l0);
    row_ml[warp][r0 + 8] = make_float2(ref1, l1);
  }
#pragma unroll
  for (int i = 0; i < HD / 8; i++) {
    float *a = merge + (warp * kMmaRows + r0) * HD + i * 8 + (lane & 3) * 2;
    *(float2 *)a = make_float2(o[i][0], o[i][1]);
    *(float2 *)(a + 8 * HD) = make_float2(o[i][2], o[i][3]);
  }
  __syncthreads();
  for (int i = tid; i < t.rows * (HD / 4); i += kMmaThreads) {
    const int j = i / (HD / 4), d = (i % (HD / 4)) * 4;
    if (d >= hd) continue;
    float top = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kMmaWarps; w++) top = fmaxf(top, row_ml[w][j].x);
    const float safe = top == -INFINITY ? 0.0f : top;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kMmaWarps; w++) {
      const float2 ml = row_ml[w][j];
      const float a = ml.y == 0.0f ? 0.0f : exp2f(ml.x - safe);
      const float4 v = *(const float4 *)(merge + (w * kMmaRows + j) * HD + d);
      l = fmaf(a, ml.y, l);
      sum.x = fmaf(a, v.x, sum.x);
      sum.y = fmaf(a, v.y, sum.y);
      sum.z = fmaf(a, v.z, sum.z);
      sum.w = fmaf(a, v.w, sum.w);
    }
    if (direct) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t oo = out_offset(p, t, j) + d;
      if (p.act == JAL_F32)
        *(float4 *)((float *)p.out + oo) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
      else
        *(uint2 *)((T *)p.out + oo) = make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
    } else {
      const int64_t pi = part_index(p, t, j);
      if (d == 0) p.part_ml[pi] = make_float2(top, l);
      *(float4 *)(p.part_o + pi * hd + d) = sum;
    }
  }
}

}  // namespace paged
}  // namespace jal
