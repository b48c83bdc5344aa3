// Attention of few query rows over a paged cache of 8- or 4-bit codes on the
// warp-level integer matrix instructions (mma.sync m16n8k32).  Included by
// quant_attn.cu.
//
//   out = sum_t softmax(scale * dk[t] * (q . ck[t])) * dv[t] * cv[t]
//
// with codes c and scales d.  Codes enter the products as they are stored: a warp that
// widened them to f16 first spent three quarters of its instructions on that (one
// row a sequence of 28 heads, 4 KV heads of 128, over 64 caches of up to 8192 4-bit
// positions: 138 us; so: 73 us).  q, and the weights times dv, are whole numbers over a power of two (q:
// over the row's largest), in balanced digits of 8 bits, v = sum_i 256^i digit_i with
// digit_i in [-128, 127]: two digits for 16-bit rows, four for f32.  The products
// of the digits are exact, and are put together in f32.
//
// A 16-row tile of the instruction holds eight query rows: rows i and i + 8 are the
// upper and lower digit of row i, so one thread has both.  The weights of 32 keys
// are numbers over a 32512th of the largest of them (four digits: 2^-29 of the power of two
// below it), so their share is kept however far below the row's maximum they lie, and their
// products are added to the f32 output for each 32 keys.  An accumulator starts at 1.5 * 2^23 as f32 bits: read
// as f32, it is that plus the sum, exactly.
//
// Errors: q is off by 2^-16 of the row's largest element (16-bit rows; f32: 2^-24 of
// itself and 2^-31 of that), a weight times V's scale by 2^-16 (2^-30) of the largest of its
// 32 keys', or by 2^-126 where that is more.  (Over the power of two below the largest, one or
// two bits fewer, the 64 caches above were a fifth further from the formula, in the same time.)
//
// A block takes R8 tiles of eight query rows of one KV head (the query heads of a
// group, and neighbouring tokens); its four warps take 32 keys each in turn, and
// each is on its own until the end: it copies its keys' codes and scales with cp.async
// into its own ring, and has its own running maxima, sums and output.
//
// What bounds it is instructions: with eight rows a warp issues two products and
// a dozen others on scores and weights for each key and row pair that it has, so an
// SM works where its loads could wait.  Read once, codes and scales would take 33 us of
// the 73 above; 48 sequences of 4 to 6 rows of 32 heads (8 KV heads of 128, up to 12288
// 8-bit positions) take 228 us, 99 for their bytes; one sequence of 131071 positions 52,
// 42 for its bytes.  With all row tiles of a KV head in one block, codes are read
// once for all heads of the group and all drafted tokens.
#pragma once

#include "paged_attn_mma.cuh"
#include "paged_attn_tc.cuh"
#include "quant_kv.hpp"

namespace jal {
namespace paged {

constexpr int kQuantKeys = 32;
constexpr uint32_t kIntZero = 0x4B400000u;  // 1.5 * 2^23 as f32: an integer sum of 0
constexpr float kIntZeroF = 12582912.0f;

// d = c + products of signed bytes with signed (BITS = 8) or unsigned (4) ones.
template <int BITS>
__device__ __forceinline__ void imma(uint32_t (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const uint32_t (&c)[4]) {
  if constexpr (BITS == 8)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
// Two 16 x 16 tiles of bytes, transposed: lane 4 g + j gets of each tile the rows
// 4 j .. 4 j + 3 of column g, and of column g + 8.  Lane i gives row i's address.
__device__ __forceinline__ void ldsm_bytes(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void copy4(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t *w) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}

// 1 / x by the special-function unit: relative error 2^-23.
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The digits of four whole numbers v, byte i of word d the digit d of number i.  NS = 1:
// v + 128 in the low 16 bits of each x; NS = 2: v.
template <int NS>
__device__ __forceinline__ void digits(const uint32_t (&x)[4], uint32_t (&word)[2 * NS]) {
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; i++) y[i] = NS == 1 ? x[i] : x[i] + 0x00808080u;
  const uint32_t a = __byte_perm(y[0], y[1], 0x5140), b = __byte_perm(y[2], y[3], 0x5140);  // bytes 0 and 1 of both
  word[0] = __byte_perm(a, b, 0x5410) ^ 0x80808080u;
  word[1] = __byte_perm(a, b, 0x7632);
  if constexpr (NS == 2) {
    word[1] ^= 0x80808080u;
    const uint32_t c = __byte_perm(y[0], y[1], 0x7362), d = __byte_perm(y[2], y[3], 0x7362);
    word[2] = __byte_perm(c, d, 0x5410) ^ 0x80808080u;
    word[3] = __byte_perm(c, d, 0x7632);
  }
}

// Blocks on an SM, by registers and shared memory.  (Eight 16-bit rows over 4-bit codes:
// four blocks with three stages 73 us where three with four take 75; over 8-bit codes
// 131071 keys 56 and 52.)
constexpr int quant_blocks(int bits, int hd, int r8, int ns) {
  return hd > 128 ? 1 : r8 * ns > 2 ? 2 : bits == 4 && hd > 64 && r8 * ns == 1 ? 4 : 3;
}

template <int BITS, int NS, int HD, int R8>
struct QuantShape {
  static constexpr int blocks = quant_blocks(BITS, HD, R8, NS);
  static constexpr int rows = 8 * R8;
  static constexpr int row_bytes = HD * BITS / 8;
  static constexpr int chunks = row_bytes / 16;            // 16-byte pieces of a row
  static constexpr int half = kQuantKeys * row_bytes;      // bytes of a stage's K (or V)
  static constexpr int stage = 2 * half + 2 * kQuantKeys * 4;
  static constexpr int stages = row_bytes <= 32 ? 6 : row_bytes == 64 ? (blocks == 4 ? 3 : 4) : 2;
  static constexpr int ring = kMmaWarps * stages * stage;
  static constexpr int ksteps = HD / 32;
  static constexpr int q_bytes = NS * R8 * ksteps * 512;   // fragments
  static constexpr int out_row = HD + 4;                   // floats of a row where warps' results are joined
  static constexpr int merge = kMmaWarps * rows * out_row * 4;
  static constexpr int smem = q_bytes + (ring > merge ? ring : merge);
  // Where 16-byte piece c of K's row r and V's row r lies, without conflicts between
  // the lanes that read together: of K two neighbouring rows, four pieces; of V the same
  // piece of eight rows.
  static __device__ __forceinline__ uint32_t k_at(int r, int c) {
    return r * row_bytes + ((chunks >= 8 ? c ^ ((r & 1) << 2) : c) * 16);
  }
  static __device__ __forceinline__ uint32_t v_at(int r, int c) {
    const int x = chunks >= 8 ? r & 7 : chunks == 4 ? (r >> 1) & 3 : (r >> 2) & 1;
    return r * row_bytes + ((c ^ x) * 16);
  }
  // V's row for key i: a lane of the scores has keys 2 j, 2 j + 1 of every eight, and of
  // the weights the rows 4 j .. 4 j + 3 of every sixteen.
  static __device__ __forceinline__ int v_row(int i) { return (i & 16) | ((i & 6) << 1) | ((i & 8) >> 2) | (i & 1); }
};

template <int BITS, int NS, int HD, int R8>
__global__ void __launch_bounds__(kMmaThreads, QuantShape<BITS, NS, HD, R8>::blocks)
    k_quant_attn_mma(const __grid_constant__ QuantAttnParams qp, const bool direct) {
  using S = QuantShape<BITS, NS, HD, R8>;
  const AttnParams &p = qp.a;
  extern __shared__ __align__(128) char smem_raw[];
  __shared__ RowMask masks[S::rows];
  __shared__ float q_scale[S::rows];
  __shared__ float2 row_ml[kMmaWarps][S::rows];
  __shared__ uint32_t present[kMmaWarps][S::stages];
  pdl_wait();
  pdl_trigger();
  Tile t;
  if (!block_tile(p, kOwn, S::rows, kMmaWarps * kQuantKeys, t)) return;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, hd = p.kv.hd;
  const int g = lane / 4, j4 = lane % 4;  // this lane's row (or column), and quarter
  const uint32_t sq = smem_u32(smem_raw), ring = sq + S::q_bytes + warp * (S::stages * S::stage);

  // This warp's keys: chunks of 32 of [u0, u1), every fourth.  A lane looks up where
  // its key of a chunk lies, one chunk ahead of the copies.
  const int n_chunks = (t.u1 - t.u0 + kQuantKeys - 1) / kQuantKeys;
  auto locate = [&](int c) -> Slot {
    const int u = t.u0 + c * kQuantKeys + lane;
    return c < n_chunks && u < t.u1 ? slot_of(p.kv, t, t.key(u)) : Slot{-1, 0};
  };
  auto copy = [&](const Slot &where, int stage) {
    const int64_t at = slot_offset(p.kv, where, t.head);
    const uint32_t dst = ring + stage * S::stage;
    const uint32_t bits = __ballot_sync(0xffffffffu, at >= 0);
    if (lane == 0) present[warp][stage] = bits;
    const int64_t e = at >= 0 ? (int64_t)where.page * qp.sc.s_page + t.head * qp.sc.s_head + where.slot : 0;
    copy4(dst + 2 * S::half + lane * 4, qp.sc.k + e, at >= 0);
    copy4(dst + 2 * S::half + kQuantKeys * 4 + lane * 4, qp.sc.v + e, at >= 0);
    // (Rows that lie one behind the other, as within a page, need not be passed round.)
    const int64_t first = __shfl_sync(0xffffffffu, at, 0);
    if (__all_sync(0xffffffffu, at >= 0 && at == first + lane * S::row_bytes) && hd == HD) {
      const char *const ks = (const char *)p.kv.k + first + lane * 16, *const vs = (const char *)p.kv.v + first + lane * 16;
#pragma unroll
      for (int i = 0; i < S::chunks; i++) {
        const int r = (i * 32 + lane) / S::chunks, c = lane % S::chunks;
        copy16(dst + S::k_at(r, c), ks + i * 512, true);
        copy16(dst + S::half + S::v_at(S::v_row(r), c), vs + i * 512, true);
      }
    } else {
#pragma unroll
      for (int i = 0; i < S::chunks; i++) {
        const int r = (i * 32 + lane) / S::chunks, c = lane % S::chunks;
        const int64_t o = __shfl_sync(0xffffffffu, at, r);
        const bool there = o >= 0 && c * (128 / BITS) < hd;
        const int64_t x = there ? o + c * 16 : 0;
        copy16(dst + S::k_at(r, c), (const char *)p.kv.k + x, there);
        copy16(dst + S::half + S::v_at(S::v_row(r), c), (const char *)p.kv.v + x, there);
      }
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
  // Query rows into shared memory as fragments of digits.  Sixteen threads a row; a
  // thread has the four dims that make one word of a fragment.
  {
    const int r = tid / 16, sub = tid % 16;
#pragma unroll
    for (int m = 0; m < R8; m++) {
      const int j = m * 8 + r;
      const bool real = j < t.rows;
      const int64_t qo = real ? q_offset(p, t, j) : 0;
      constexpr int W = HD / 64;  // words of a thread
      float v[W][4];
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < W; w++) {
        // Word `sub + 16 w` of the row: fragment ks, quarter jj, half h; its dims as a lane
        // finds them in 16 (or 8) bytes of a row of K.
        const int at = sub + 16 * w, ks = at / 8, jj = at / 2 % 4, h = at % 2;
        constexpr int per = (S::chunks >= 4 ? 128 : 64) / BITS;  // codes that a lane reads at once
        const int piece = ks / (per / 8), x = ks % (per / 8);
        const int base = (piece * 4 + jj) * per + x * 8;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int d = BITS == 8 ? base + h * 4 + i : base + 2 * i + h;
          v[w][i] = real && d < hd ? load_as_f32(p.q, qo + d, p.act) : 0.0f;
          top = max(top, __float_as_uint(v[w][i]) & 0x7fffffffu);  // (a NaN's bits are above infinity's)
        }
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      // (The lower two of four digits count as a fraction: whole / most stays in f32's range.)
      constexpr float whole = 127.0f * 256.0f;
      const float most = __uint_as_float(top);
      const bool some = most >= kQuantLeast && most < INFINITY;
      const float over = some ? whole / most : 0.0f;
      if (sub == 0) {
        masks[j] = real ? row_mask(p, t, j) : RowMask{0, 0};
        // (A row with a NaN or an infinity has NaN scores.)
        q_scale[j] = some ? p.scale_log2 * (most / whole) : most < INFINITY ? 0.0f : NAN;
      }
#pragma unroll
      for (int w = 0; w < W; w++) {
        const int at = sub + 16 * w, ks = at / 8, jj = at / 2 % 4, h = at % 2;
        uint32_t x[4], word[2 * NS];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = some ? (uint32_t)__float2int_rn(v[w][i] * over * (NS == 1 ? 1.0f : 65536.0f)) : 0u;
        if (NS == 1)
#pragma unroll
          for (int i = 0; i < 4; i++) x[i] += 128u;
        digits<NS>(x, word);
#pragma unroll
        for (int s = 0; s < NS; s++) {  // fragment s: the digits 2 (NS - 1 - s) + 1 and below it
          char *const f = smem_raw + ((s * R8 + m) * S::ksteps + ks) * 512 + (r * 4 + jj) * 16 + h * 8;
          *(uint32_t *)f = word[2 * (NS - 1 - s) + 1];
          *(uint32_t *)(f + 4) = word[2 * (NS - 1 - s)];
        }
      }
    }
  }
  __syncthreads();

  // Rows that do not exist see everything: they have no say in what is masked.
  const RowSpan every = {0x7fffffff, 0, 0};
  RowSpan span[R8];
  float f[R8];
  float top[R8], l[R8];  // running maxima, which the weights refer to, and their sums
  pair_t o[R8][HD / 8];
  // Where an accumulator of scores starts: 4-bit codes are stored with 8 added.
  uint32_t start[R8][NS][4];
#pragma unroll
  for (int m = 0; m < R8; m++) {
    const int r = m * 8 + g;
    span[m] = r < t.rows ? row_span(p, t, masks[r]) : every;
    f[m] = q_scale[r];
    top[m] = -INFINITY;
    l[m] = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 8; i++) o[m][i] = 0;
#pragma unroll
    for (int s = 0; s < NS; s++) {
      uint32_t c[4] = {kIntZero, kIntZero, kIntZero, kIntZero};
      if (BITS == 4) {
#pragma unroll
        for (int ks = 0; ks < S::ksteps; ks++) {
          uint32_t a[4];
          lds<16>(sq + ((s * R8 + m) * S::ksteps + ks) * 512 + lane * 16, a);
          imma<8>(c, a, 0xF8F8F8F8u, 0xF8F8F8F8u, c);
        }
      }
      start[m][s][0] = start[m][s][1] = c[0];
      start[m][s][2] = start[m][s][3] = c[2];
    }
  }
  uint32_t zero[4] = {kIntZero, kIntZero, kIntZero, kIntZero};
  const pair_t minus = pair(-kIntZeroF, -kIntZeroF), digit = pair(256.0f, 256.0f);
  // What accumulators of the digits hold, in f32; of four digits, over 2^16.
  auto whole_pair = [&](const uint32_t (&c)[NS][4]) -> pair_t {
    const pair_t hi = add2(pair_bits(c[0][0], c[0][1]), minus), lo = add2(pair_bits(c[0][2], c[0][3]), minus);
    pair_t v = fma2(hi, digit, lo);
    if constexpr (NS == 2) {
      const pair_t hi1 = add2(pair_bits(c[1][0], c[1][1]), minus), lo1 = add2(pair_bits(c[1][2], c[1][3]), minus);
      v = fma2(fma2(hi1, digit, lo1), pair(0x1p-16f, 0x1p-16f), v);
    }
    return v;
  };

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
    // Scores: the lane has keys 8 n + 2 j4 and the next one.
    pair_t s[R8][4];
    {
      constexpr int lane_bytes = S::chunks >= 4 ? 16 : 8, words = lane_bytes / 4, pieces = S::row_bytes / (4 * lane_bytes);
      constexpr int steps = words * 4 / BITS;  // of a piece
      uint32_t acc[4][R8][NS][4];
#pragma unroll
      for (int pc = 0; pc < pieces; pc++) {
        uint32_t w[4][words];
#pragma unroll
        for (int n = 0; n < 4; n++) {
          if constexpr (lane_bytes == 16) lds<16>(kb + S::k_at(n * 8 + g, pc * 4 + j4), w[n]);
          else lds<8>(kb + S::k_at(n * 8 + g, 0) + j4 * 8, w[n]);
        }
#pragma unroll
        for (int x = 0; x < steps; x++) {
          const int ks = pc * steps + x;
#pragma unroll
          for (int m = 0; m < R8; m++)
#pragma unroll
            for (int q = 0; q < NS; q++) {
              uint32_t a[4];
              lds<16>(sq + ((q * R8 + m) * S::ksteps + ks) * 512 + lane * 16, a);
#pragma unroll
              for (int n = 0; n < 4; n++) {
                const uint32_t b0 = BITS == 8 ? w[n][(2 * x) % words] : w[n][x % words] & 0x0F0F0F0Fu;
                const uint32_t b1 = BITS == 8 ? w[n][(2 * x + 1) % words] : (w[n][x % words] >> 4) & 0x0F0F0F0Fu;
                imma<BITS>(acc[n][m][q], a, b0, b1, ks ? acc[n][m][q] : start[m][q]);
              }
            }
        }
      }
#pragma unroll
      for (int n = 0; n < 4; n++)
#pragma unroll
        for (int m = 0; m < R8; m++) s[m][n] = whole_pair(acc[n][m]);
    }
    const int u = t.u0 + c * kQuantKeys;
    bool all = bits == 0xffffffffu;
#pragma unroll
    for (int m = 0; m < R8; m++) all = all && span[m].all(u, kQuantKeys);
    const bool masked = __any_sync(0xffffffffu, !all);
    uint32_t dk[4][2], dv[4][2];  // scales of this lane's keys
#pragma unroll
    for (int n = 0; n < 4; n++) {
      lds<8>(sb + n * 32 + j4 * 8, dk[n]);
      lds<8>(sb + kQuantKeys * 4 + n * 32 + j4 * 8, dv[n]);
    }
    uint32_t wa[R8][NS][4];
    float unit[R8];  // what the whole numbers of the weights count
#pragma unroll
    for (int m = 0; m < R8; m++) {
      float y[8];
#pragma unroll
      for (int n = 0; n < 4; n++)
        unpair(mul2(s[m][n], mul2(pair_bits(dk[n][0], dk[n][1]), pair(f[m], f[m]))), y[2 * n], y[2 * n + 1]);
      if (masked) {
        const uint32_t see = (bits & span[m].bits(u)) >> (2 * j4);
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (!((see >> (i / 2 * 8 + i % 2)) & 1)) y[i] = -INFINITY;
      }
      float most = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(top[m], fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2)));
      if (__any_sync(0xffffffffu, most != top[m])) {
        const float less = most == top[m] ? 1.0f : exp2_fast(top[m] - most);
        top[m] = most;
        l[m] *= less;
#pragma unroll
        for (int i = 0; i < HD / 8; i++) o[m][i] = mul2(o[m][i], pair(less, less));
      }
      const float ref = top[m] == -INFINITY ? 0.0f : top[m];
      uint32_t big = 0;
#pragma unroll
      for (int n = 0; n < 4; n++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float &x = y[2 * n + e];
          const bool seen = !masked || x != -INFINITY;  // (what a row does not see has no effect on it)
          x = exp2_fast(x - ref);
          l[m] += x;
          x = seen ? x * __uint_as_float(dv[n][e]) : 0.0f;
          big = max(big, __float_as_uint(x) & 0x7fffffffu);
        }
      }
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // The weights as whole numbers over `unit`: the largest one's 32512th; four digits: 2^-29 of the
      // power of two below it; over 2^-126, where that is more.
      float over;
      if constexpr (NS == 1) {
        const float most = __uint_as_float(max(big, 0x08000000u));  // (2^-111)
        over = 32512.0f * rcp_fast(most);
        unit[m] = big >= 0x7F800000u ? NAN : most * (1.0f / 32512.0f);
      } else {
        const int e = (int)(big >> 23), shift = min(29, e - 1);
        const bool some = e > 0;  // (smaller than 2^-126, all: they count as 0)
        over = some ? __uint_as_float((uint32_t)(254 + shift - e) << 23) : 0.0f;
        unit[m] = e == 255 ? NAN : some ? __uint_as_float((uint32_t)(e - shift + 16) << 23) : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        uint32_t x[4], word[2 * NS];
#pragma unroll
        for (int i = 0; i < 4; i++)
          x[i] = NS == 1 ? __float_as_uint(fmaf(y[4 * h + i], over, kIntZeroF + 128.0f)) : (uint32_t)__float2int_rn(y[4 * h + i] * over);
        digits<NS>(x, word);
#pragma unroll
        for (int q = 0; q < NS; q++) {
          wa[m][q][2 * h] = word[2 * (NS - 1 - q) + 1];
          wa[m][q][2 * h + 1] = word[2 * (NS - 1 - q)];
        }
      }
    }
    // The output: the lane's columns are 2 j4, 2 j4 + 1 of every eight.
    uint32_t first[R8][NS][4];
#pragma unroll
    for (int m = 0; m < R8; m++)
#pragma unroll
      for (int q = 0; q < NS; q++) {
        if constexpr (BITS == 4) imma<8>(first[m][q], wa[m][q], 0xF8F8F8F8u, 0xF8F8F8F8u, zero);
      }
#pragma unroll
    for (int ch = 0; ch < S::chunks; ch++) {
      uint32_t b[4];
      ldsm_bytes(b, vb + S::v_at(lane, ch));
#pragma unroll
      for (int x = 0; x < 2 * 8 / BITS; x++) {
        // 8 bits: columns 0 .. 7, 8 .. 15.  4 bits: the low, then the high halves of each.
        const int h = BITS == 8 ? x : x / 2;
        const uint32_t b0 = BITS == 8 ? b[h] : (b[h] >> (x % 2 * 4)) & 0x0F0F0F0Fu;
        const uint32_t b1 = BITS == 8 ? b[h + 2] : (b[h + 2] >> (x % 2 * 4)) & 0x0F0F0F0Fu;
#pragma unroll
        for (int m = 0; m < R8; m++) {
          uint32_t acc[NS][4];
#pragma unroll
          for (int q = 0; q < NS; q++) imma<BITS>(acc[q], wa[m][q], b0, b1, BITS == 4 ? first[m][q] : zero);
          pair_t &out = o[m][ch * (2 * 8 / BITS) + x];
          out = fma2(whole_pair(acc), pair(unit[m], unit[m]), out);
        }
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
    if (++stage == S::stages) stage = 0;
  }
  copies_wait<0>();
  __syncthreads();  // no warp reads its ring any more
  // The four warps' results, joined through shared memory.
  float *const merge = (float *)(smem_raw + S::q_bytes);
#pragma unroll
  for (int m = 0; m < R8; m++) {
    float x = l[m];
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    const int r = m * 8 + g;
    if (j4 == 0) row_ml[warp][r] = make_float2(top[m], x);
    float *const a = merge + (warp * S::rows + r) * S::out_row;
    if constexpr (BITS == 8) {
#pragma unroll
      for (int i = 0; i < HD / 8; i++) *(pair_t *)(a + i * 8 + j4 * 2) = o[m][i];
    } else {
#pragma unroll
      for (int i = 0; i < HD / 8; i += 2) {  // low and high halves: dims 4 j4, + 2 and + 1, + 3 of every sixteen
        float x0, x1, x2, x3;
        unpair(o[m][i], x0, x2);
        unpair(o[m][i + 1], x1, x3);
        *(float4 *)(a + i * 8 + j4 * 4) = make_float4(x0, x1, x2, x3);
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < t.rows * (HD / 4); i += kMmaThreads) {
    const int j = i / (HD / 4), d = (i % (HD / 4)) * 4;
    if (d >= hd) continue;
    float most = -INFINITY, sum_l = 0.0f;
#pragma unroll
    for (int w = 0; w < kMmaWarps; w++) most = fmaxf(most, row_ml[w][j].x);
    const float safe = most == -INFINITY ? 0.0f : most;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kMmaWarps; w++) {
      const float2 ml = row_ml[w][j];
      if (ml.y == 0.0f) continue;
      const float a = exp2f(ml.x - safe);
      const float4 v = *(const float4 *)(merge + (w * S::rows + j) * S::out_row + d);
      sum_l = fmaf(a, ml.y, sum_l);
      sum.x = fmaf(a, v.x, sum.x);
      sum.y = fmaf(a, v.y, sum.y);
      sum.z = fmaf(a, v.z, sum.z);
      sum.w = fmaf(a, v.w, sum.w);
    }
    if (direct) {
      const float inv = sum_l == 0.0f ? 0.0f : 1.0f / sum_l;
      const int64_t oo = out_offset(p, t, j) + d;
      if (p.act == JAL_F32)
        *(float4 *)((float *)p.out + oo) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
      else if (p.act == JAL_F16)
        *(uint2 *)((__half *)p.out + oo) = make_uint2(pack2<__half>(sum.x * inv, sum.y * inv), pack2<__half>(sum.z * inv, sum.w * inv));
      else
        *(uint2 *)((__nv_bfloat16 *)p.out + oo) =
            make_uint2(pack2<__nv_bfloat16>(sum.x * inv, sum.y * inv), pack2<__nv_bfloat16>(sum.z * inv, sum.w * inv));
    } else {
      const int64_t pi = part_index(p, t, j);
      if (d == 0) p.part_ml[pi] = make_float2(most, sum_l);
      *(float4 *)(p.part_o + pi * hd + d) = sum;
    }
  }
}

}  // namespace paged
}  // namespace jal
