// New keys and values of a ragged batch into a paged cache of 8- or 4-bit codes,
// with the position rotation applied on the way, and positions read back from it.
#include <algorithm>

#include "common.hpp"
#include "paged_attn_tc.cuh"
#include "paged_dev.cuh"
#include "quant_kv.hpp"

namespace jal {

namespace {

using namespace paged;

// cos and sin of pos * inv_freq in 64 bits: the angle less the nearest multiple of
// pi / 2 (in two parts), their power series there (the first terms left out are (pi /
// 4)^16 / 16! = 1e-15 and (pi / 4)^15 / 15! = 2e-14), and the quarter turns.  Codes go by
// values next to a border, so what is quantised is the rotated value to the last bit of
// f32.
__device__ __forceinline__ double2 turn64(int64_t pos, float inv_freq) {
  const double a = (double)pos * (double)inv_freq, n = rint(a * 0.6366197723675814);
  const double r = fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, a)), z = r * r;
  double c = -1.0 / 87178291200.0, s = 1.0 / 6227020800.0;
  c = fma(c, z, 1.0 / 479001600.0);
  s = fma(s, z, -1.0 / 39916800.0);
  c = fma(c, z, -1.0 / 3628800.0);
  s = fma(s, z, 1.0 / 362880.0);
  c = fma(c, z, 1.0 / 40320.0);
  s = fma(s, z, -1.0 / 5040.0);
  c = fma(c, z, -1.0 / 720.0);
  s = fma(s, z, 1.0 / 120.0);
  c = fma(c, z, 1.0 / 24.0);
  s = fma(s, z, -1.0 / 6.0);
  c = fma(c, z, -0.5);
  s = fma(s * z, r, r);
  c = fma(c, z, 1.0);
  const int quarter = (int)(long long)n & 3;
  double2 cs = quarter & 1 ? make_double2(-s, c) : make_double2(c, s);
  if (quarter & 2) cs = make_double2(-cs.x, -cs.y);
  return cs;
}

template <int BITS>
struct Codes;
template <>
struct Codes<8> {
  static constexpr float most = 127.0f;
};
template <>
struct Codes<4> {
  static constexpr float most = 7.0f;
};

// Eight codes, x * per rounded to the nearest integer (ties to even), stored at dim
// d of a row: 1.5 * 2^23 added and looked at bit by bit.
template <int BITS>
__device__ __forceinline__ void store_codes8(uint8_t *row, int d, const float (&x)[8], float per) {
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; e++) c[e] = __float_as_uint(__fadd_rn(__fmul_rn(x[e], per), BITS == 8 ? 12582912.0f : 12582920.0f));
  if constexpr (BITS == 8) {
    uint2 w;
    w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    w.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
    *(uint2 *)(row + d) = w;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) w |= (c[e] & 15u) << (4 * e);
    *(uint32_t *)(row + d / 2) = w;
  }
}

// Eight elements as they are in memory.
template <class T>
struct Raw8 {
  uint4 w;
  __device__ __forceinline__ void load(const T *p) { w = *(const uint4 *)p; }
  __device__ __forceinline__ void widen(float (&v)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = unpack2<T>(u[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Raw8<float> {
  float v[8];
  __device__ __forceinline__ void load(const float *p) { load8(p, v); }
  __device__ __forceinline__ void widen(float (&o)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = v[i];
  }
};

// The pairs of eight dims at d and the eight half a rotation further on, turned: t[i]
// is pair i's cosine and sine.  (k in 64 bits; q, which is rounded to its own type, in f32.)
template <class T1, class T2>
__device__ __forceinline__ void turn8(float (&a)[8], float (&b)[8], const T2 (&t)[8], int neox) {
  if (neox) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const T1 x = a[e], y = b[e];
      a[e] = (float)(x * t[e].x - y * t[e].y);
      b[e] = (float)(x * t[e].y + y * t[e].x);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const T1 x = a[e], y = a[e + 1], z = b[e], w = b[e + 1];
      const T2 f = t[e / 2], g = t[4 + e / 2];
      a[e] = (float)(x * f.x - y * f.y);
      a[e + 1] = (float)(x * f.y + y * f.x);
      b[e] = (float)(z * g.x - w * g.y);
      b[e + 1] = (float)(z * g.y + w * g.x);
    }
  }
}

constexpr int kWarps = 4;

// A warp takes part of a token row's heads, `lanes` neighbouring lanes a head.
// PAIRS (rotary_dim a multiple of 16, or 0): a lane has eight dims and, in the rotated
// part, the eight rotary_dim / 2 further on, so both of a pair's elements are in
// one lane whichever way they are paired.  Otherwise a lane has eight dims and reads
// its partners' elements.  Every lane has read what it needs before any lane of
// the head writes, so q_out may be q.
// Queries come first, then keys and values, with a lane's turns in registers: as one
// loop over all heads each head read them from shared memory again (78 us where it then was
// 70, and is 67: 7 prompts of up to 2048 tokens of 32 and 8 heads of 128, bf16, 4 bits, with
// the new positions read back; memory alone 43).  What is left is instructions: the 64-bit
// rotation of K, the widening and packing of 16-bit rows.  Five blocks an SM: four, six and
// seven were slower.
template <int BITS, class TA, bool PAIRS>
__global__ void __launch_bounds__(kWarps * 32, 5) k_quant_kv_append(const __grid_constant__ QuantAppendParams qp,
                                                                    const int parts, const int lanes) {
  const AppendParams &p = qp.a;
  constexpr int kItems = !PAIRS ? 1 : sizeof(TA) == 4 ? 2 : 4;  // heads of a lane on their way at a time
  constexpr int kKvItems = kItems > 2 ? 2 : 1;
  __shared__ double2 turns[kWarps][kPagedMaxHeadDim / 2];
  pdl_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t unit = (int64_t)blockIdx.x * kWarps + warp;
  const int row = (int)(unit / parts), part = (int)(unit - (int64_t)row * parts);
  if (row >= p.n_rows) return;
  const int first = __ldg(p.q_start), last = __ldg(p.q_start + p.n_seqs);
  const int s = warp_seq_of_row(p.q_start, p.n_seqs, row);
  if (row < first || row >= last) return;
  int beg, end;
  seq_rows(p.q_start, p.n_rows, s, beg, end);
  const int64_t pos64 = (int64_t)__ldg(p.kv_len + s) - (end - row);
  if (pos64 < 0) return;
  const int hd = p.kv.hd, half = p.rotary / 2;
  // (Past the table, and without a page, there is no place for the row's k and v; its
  // queries are turned all the same.)
  int64_t at = -1, s_at = 0;
  if (pos64 < p.kv.cap) {
    const Slot sl = slot_of(p.kv, p.kv.table + (int64_t)s * p.kv.max_pages, (int)pos64);
    at = slot_offset(p.kv, sl, 0);
    s_at = (int64_t)sl.page * qp.s_page + sl.slot;
  }
  const int nq = p.q ? p.hq : 0, heads = nq + 2 * p.kv.hkv;
  const int per = (heads + parts - 1) / parts, stop = min(heads, (part + 1) * per), step = 32 / lanes;
  const int c = lane % lanes, mine = lane / lanes;
  // The eight dims of this lane, and where their partners are.
  const bool rotated = PAIRS ? c < half / 8 : false;
  const int d = PAIRS ? (rotated ? c * 8 : p.rotary + (c - half / 8) * 8) : c * 8;
  const bool inside = d < hd;
  double2 *const cs = turns[warp];
  for (int i = lane; i < half; i += 32) cs[i] = turn64(pos64, __ldg(p.inv_freq + i));
  __syncwarp();
  // This lane's pair i: d + i (split halves); d / 2 + i and (d + half) / 2 + i - 4 (neighbours).
  auto pair_of = [&](int i) { return p.neox ? d + i : i < 4 ? d / 2 + i : (d + half) / 2 + i - 4; };
  // Without PAIRS: element i of a head's row with its partner, wherever that is.
  auto turn1 = [&](const TA *src, int i) -> float {
    const bool low = p.neox ? i < half : i % 2 == 0;
    const int other = p.neox ? (low ? i + half : i - half) : i ^ 1;
    const double2 t = cs[p.neox ? (low ? i : i - half) : i / 2];
    const double y = load_as_f32(src, other, p.act), x = load_as_f32(src, i, p.act);
    return (float)(low ? x * t.x - y * t.y : y * t.y + x * t.x);
  };
  int base = part * per;
  const int q_stop = min(stop, nq);
  if (base < q_stop) {
    const TA *const src = (const TA *)p.q + row * p.q_stride + d;
    TA *const dst = (TA *)p.q_out + row * p.q_out_stride + d;
    float2 t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      t[i] = make_float2(1.0f, 0.0f);
      if (rotated) {
        const double2 x = cs[pair_of(i)];
        t[i] = make_float2((float)x.x, (float)x.y);
      }
    }
    for (; base < q_stop; base += step * kItems) {
      Raw8<TA> ra[kItems], rb[kItems];
#pragma unroll
      for (int k = 0; k < kItems; k++) {
        const int head = base + k * step + mine;
        if (head >= q_stop || !inside) continue;
        ra[k].load(src + head * hd);
        if (rotated) rb[k].load(src + head * hd + half);
      }
#pragma unroll
      for (int k = 0; k < kItems; k++) {
        const int head = base + k * step + mine;
        const bool there = head < q_stop && inside;
        float a[8], b[8];
        if (there) {
          ra[k].widen(a);
          if constexpr (PAIRS) {
            if (rotated) {
              rb[k].widen(b);
              turn8<float>(a, b, t, p.neox);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
              if (d + e < p.rotary) a[e] = turn1(src - d + head * hd, d + e);
          }
        }
        if (!PAIRS) __syncwarp();
        if (there) {
          store8(dst + head * hd, a);
          if (rotated) store8(dst + head * hd + half, b);
        }
      }
    }
    base = q_stop;
  }
  for (; base < stop; base += step * kKvItems) {
    Raw8<TA> ra[kKvItems], rb[kKvItems];
#pragma unroll
    for (int k = 0; k < kKvItems; k++) {
      const int i = base + k * step + mine - nq;
      if (i >= stop - nq || !inside) continue;
      const bool is_k = i < p.kv.hkv;
      const TA *const src = (const TA *)(is_k ? p.k : p.v) + row * p.kv_stride + (is_k ? i : i - p.kv.hkv) * hd + d;
      ra[k].load(src);
      if (rotated) rb[k].load(src + half);
    }
#pragma unroll
    for (int k = 0; k < kKvItems; k++) {
      const int i = base + k * step + mine - nq;
      const bool there = i < stop - nq && inside, is_k = i < p.kv.hkv;
      const int h = is_k ? i : i - p.kv.hkv;
      float a[8] = {}, b[8] = {};
      if (there) {
        ra[k].widen(a);
        if (rotated) rb[k].widen(b);
        if (is_k) {
          if constexpr (PAIRS) {
            if (rotated) {
              double2 t[8];
#pragma unroll
              for (int e = 0; e < 8; e++) t[e] = cs[pair_of(e)];
              turn8<double>(a, b, t, p.neox);
            }
          } else {
            const TA *const src = (const TA *)p.k + row * p.kv_stride + h * hd;
#pragma unroll
            for (int e = 0; e < 8; e++)
              if (d + e < p.rotary) a[e] = turn1(src, d + e);
          }
        }
      }
      // The largest magnitude of the head, by its bits: a NaN's are above infinity's.
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; e++)
        top = max(top, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
      for (int o = lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (!there || at < 0) continue;
      const float m = __uint_as_float(top);
      const bool none = m < kQuantLeast, bad = !(m < kQuantMost);
      const float per_unit = none || bad ? 0.0f : __fdiv_rn(Codes<BITS>::most, m);
      if (bad) {  // (0 x infinity would be NaN: the codes of such a row are 0)
#pragma unroll
        for (int e = 0; e < 8; e++) a[e] = b[e] = 0.0f;
      }
      uint8_t *const dst = (uint8_t *)(is_k ? p.kw : p.vw) + at + h * p.kv.head_stride;
      store_codes8<BITS>(dst, d, a, per_unit);
      if (rotated) store_codes8<BITS>(dst, d + half, b, per_unit);
      if (c == 0)
        (is_k ? qp.ks : qp.vs)[s_at + h * qp.s_head] = bad ? NAN : none ? 0.0f : __fdiv_rn(m, Codes<BITS>::most);
    }
  }
}

template <int BITS, class TA>
void run_append(const QuantAppendParams &p, cudaStream_t s) {
  const bool pairs = p.a.rotary % 16 == 0;
  const int items = pairs ? p.a.rotary / 16 + (p.a.kv.hd - p.a.rotary) / 8 : p.a.kv.hd / 8;
  int lanes = 1;
  while (lanes < items) lanes *= 2;
  // Warps enough to fill the SMs, each with a round of heads at least.
  const int heads = (p.a.q ? p.a.hq : 0) + 2 * p.a.kv.hkv, most = std::max(1, heads / (32 / lanes));
  const int64_t rows = p.a.n_rows;
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(most, 32 * kPagedSMs / rows));
  launch_beside(pairs ? k_quant_kv_append<BITS, TA, true> : k_quant_kv_append<BITS, TA, false>,
                (rows * parts + kWarps - 1) / kWarps, kWarps * 32, 0, s, p, parts, lanes);
}
template <int BITS>
void run_append(const QuantAppendParams &p, cudaStream_t s) {
  if (p.a.act == JAL_F32) run_append<BITS, float>(p, s);
  else if (p.a.act == JAL_F16) run_append<BITS, __half>(p, s);
  else run_append<BITS, __nv_bfloat16>(p, s);
}

// ---- reading back -----------------------------------------------------------
// A block takes kReadSlots positions of one sequence and KV head: its first threads
// look up where they lie and their scales, then a thread has eight dims of a position at
// a time, K and V.  Bound by memory, then by instructions on its way there: 16 sequences of
// up to 4096 4-bit positions of 8 heads of 128 into bf16 take 48 us, 5.6 TB/s (widened one
// by one 54; blocks of 256 threads 49.5, since a block's chain of lengths, table and scales
// comes before its first code; 32 or 128 positions a block are the same).
constexpr int kReadThreads = 128, kReadSlots = 64;

// Eight codes as they are in memory.
template <int BITS>
struct RawCodes8 {
  uint32_t w[BITS / 4];
  __device__ __forceinline__ void load(const uint8_t *row, int d) {
    if constexpr (BITS == 8) {
      const uint2 x = __ldg((const uint2 *)(row + d));
      w[0] = x.x;
      w[1] = x.y;
    } else {
      w[0] = __ldg((const uint32_t *)(row + d / 2));
    }
  }
  // A code in the mantissa of 2^23 (4 bits: where it lies in its half word, as 16^i codes),
  // from which that and the code's offset are taken off; then times the scale.
  __device__ __forceinline__ void widen(float scale, float (&v)[8]) const {
    const pair_t by = pair(scale, scale);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      pair_t x;
      if constexpr (BITS == 8) {
        const uint32_t u = w[e / 4] ^ 0x80808080u;
        x = pair_bits(__byte_perm(u, 0x4B000000u, 0x7440 + e % 4), __byte_perm(u, 0x4B000000u, 0x7441 + e % 4));
        x = add2(x, pair(-8388736.0f, -8388736.0f));
      } else {
        const uint32_t u = e < 4 ? w[0] : w[0] >> 16, low = 15u << (4 * (e % 4)), high = low << 4;
        const float a = e % 4 ? 1.0f / 256.0f : 1.0f, b = a / 16.0f;
        x = pair_bits((u & low) | 0x4B000000u, (u & high) | 0x4B000000u);
        x = fma2(x, pair(a, b), pair(-8388608.0f * a - 8.0f, -8388608.0f * b - 8.0f));
      }
      unpair(mul2(x, by), v[e], v[e + 1]);
    }
  }
};

template <int BITS, class TO>
__global__ void __launch_bounds__(kReadThreads) k_quant_kv_read(const __grid_constant__ QuantReadParams p, const int tiles,
                                                                   const uint32_t over_n8) {
  __shared__ int64_t from_at[kReadSlots], into_at[kReadSlots];
  __shared__ float k_scale[kReadSlots], v_scale[kReadSlots];
  pdl_wait();
  const int tile = blockIdx.x % tiles, rest = blockIdx.x / tiles, head = rest % p.from.hkv, s = rest / p.from.hkv;
  const int beg = p.first ? max(__ldg(p.first + s), 0) : 0;
  const int64_t most = min((int64_t)beg + p.max_len, (int64_t)min(p.from.cap, p.into.cap));
  const int end = (int)min((int64_t)__ldg(p.kv_len + s), most);
  const int64_t t64 = (int64_t)beg + (int64_t)tile * kReadSlots;
  if (t64 >= end) return;
  const int t0 = (int)t64, n = min(kReadSlots, end - t0);
  if (threadIdx.x < n) {
    const int i = threadIdx.x;
    const Slot a = slot_of(p.from, p.from.table + (int64_t)s * p.from.max_pages, t0 + i),
               b = slot_of(p.into, p.into.table + (int64_t)s * p.into.max_pages, t0 + i);
    const int64_t at = slot_offset(p.from, a, head);
    from_at[i] = at;
    into_at[i] = at < 0 ? -1 : slot_offset(p.into, b, head);  // -1: left out
    if (at >= 0) {
      const int64_t s_at = (int64_t)a.page * p.sc.s_page + head * p.sc.s_head + a.slot;
      k_scale[i] = __ldg(p.sc.k + s_at);
      v_scale[i] = __ldg(p.sc.v + s_at);
    }
  }
  __syncthreads();
  // (over_n8 = 2^32 / n8 and a little: quotients of numbers below 2^16 are exact.)
  const int n8 = p.from.hd / 8, total = n * n8;
  // (A lane's pieces of a round, asked for together.)
  constexpr int kRound = 4;
  for (int i0 = threadIdx.x; i0 < total; i0 += kReadThreads * kRound) {
    RawCodes8<BITS> k[kRound], v[kRound];
#pragma unroll
    for (int r = 0; r < kRound; r++) {
      const int i = i0 + r * kReadThreads, t = (int)__umulhi((uint32_t)i, over_n8), d = (i - t * n8) * 8;
      if (i >= total || into_at[t] < 0) continue;
      k[r].load((const uint8_t *)p.from.k + from_at[t], d);
      v[r].load((const uint8_t *)p.from.v + from_at[t], d);
    }
#pragma unroll
    for (int r = 0; r < kRound; r++) {
      const int i = i0 + r * kReadThreads, t = (int)__umulhi((uint32_t)i, over_n8), d = (i - t * n8) * 8;
      if (i >= total || into_at[t] < 0) continue;
      float x[8];
      k[r].widen(k_scale[t], x);
      store8((TO *)p.kw + into_at[t] + d, x);
      v[r].widen(v_scale[t], x);
      store8((TO *)p.vw + into_at[t] + d, x);
    }
  }
}

template <int BITS>
void run_read(const QuantReadParams &p, cudaStream_t s) {
  const int64_t tiles = (p.max_len + kReadSlots - 1) / kReadSlots, blocks = tiles * p.from.hkv * p.n_seqs;
  if (blocks > 2000000000) fail(JAL_ERR_CAPABILITY_MISMATCH, "too many positions for one launch");
  const uint32_t over_n8 = 0xFFFFFFFFu / (uint32_t)(p.from.hd / 8) + 1;
  if (p.into.dtype == JAL_F32) launch_beside(k_quant_kv_read<BITS, float>, blocks, kReadThreads, 0, s, p, (int)tiles, over_n8);
  else if (p.into.dtype == JAL_F16) launch_beside(k_quant_kv_read<BITS, __half>, blocks, kReadThreads, 0, s, p, (int)tiles, over_n8);
  else launch_beside(k_quant_kv_read<BITS, __nv_bfloat16>, blocks, kReadThreads, 0, s, p, (int)tiles, over_n8);
}

}  // namespace

void launch_quant_kv_append(const QuantAppendParams &p, int bits, cudaStream_t s) {
  if (bits == 8) run_append<8>(p, s);
  else run_append<4>(p, s);
}
void launch_quant_kv_read(const QuantReadParams &p, int bits, cudaStream_t s) {
  if (bits == 8) run_read<8>(p, s);
  else run_read<4>(p, s);
}

}  // namespace jal
