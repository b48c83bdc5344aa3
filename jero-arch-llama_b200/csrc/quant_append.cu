// New keys and values of a ragged batch into a paged cache of 8- or 4-bit codes,
// with the position rotation applied on the way, and positions read back from it.
#include <algorithm>

#include "common.hpp"
#include "paged_dev.cuh"
#include "quant_kv.hpp"

namespace jal {

namespace {

using namespace paged;

// cos and sin of pos * inv_freq in 64 bits, the angle reduced to [-pi, pi] by
// 2 pi in two parts.  Codes go by values next to a border, so what is quantised is
// the rotated value to the last bit of f32.
__device__ __forceinline__ double2 turn64(int64_t pos, float inv_freq) {
  const double a = (double)pos * (double)inv_freq, n = rint(a * 0.15915494309189535);
  const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, a));
  double2 cs;
  sincos(r, &cs.y, &cs.x);
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

constexpr int kWarps = 4;

// A warp takes part of a token row's heads, `lanes` neighbouring lanes a head.
// PAIRS (rotary_dim a multiple of 16, or 0): a lane has eight dims and, in the rotated
// part, the eight rotary_dim / 2 further on, so both of a pair's elements are in
// one lane whichever way they are paired.  Otherwise a lane has eight dims and reads
// its partners' elements.  Every lane has read what it needs before any lane of
// the head writes, so q_out may be q.
template <int BITS, class TA, bool PAIRS>
__global__ void __launch_bounds__(kWarps * 32) k_quant_kv_append(const __grid_constant__ QuantAppendParams qp,
                                                                 const int parts, const int lanes) {
  const AppendParams &p = qp.a;
  __shared__ double2 turns[kWarps][kPagedMaxHeadDim / 2];
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
  double2 *const cs = turns[warp];
  for (int i = lane; i < half; i += 32) cs[i] = turn64(pos64, __ldg(p.inv_freq + i));
  __syncwarp();
  const int nq = p.q ? p.hq : 0, heads = nq + 2 * p.kv.hkv;
  const int per = (heads + parts - 1) / parts, stop = min(heads, (part + 1) * per);
  const int c = lane % lanes;
  // The eight dims of this lane, and where their partners are.
  const bool rotated = PAIRS ? c < half / 8 : false;
  const int d = PAIRS ? (rotated ? c * 8 : p.rotary + (c - half / 8) * 8) : c * 8;
  for (int base = part * per; base < stop; base += 32 / lanes) {
    const int head = base + lane / lanes;
    const bool mine = head < stop && d < hd;
    const bool is_q = head < nq, is_k = !is_q && head < nq + p.kv.hkv;
    const int h = is_q ? head : head - nq - (is_k ? 0 : p.kv.hkv);
    const TA *const src = (const TA *)(is_q ? p.q : is_k ? p.k : p.v) + row * (is_q ? p.q_stride : p.kv_stride) + h * hd;
    float a[8] = {}, b[8] = {};
    if (mine) {
      load8(src + d, a);
      if (rotated) load8(src + d + half, b);
      if constexpr (PAIRS) {
        if (rotated && (is_q || is_k)) {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            if (p.neox) {
              const double2 t = cs[d + e];
              const double x = a[e], y = b[e];
              a[e] = (float)(x * t.x - y * t.y);
              b[e] = (float)(x * t.y + y * t.x);
            } else if (e % 2 == 0) {
              const double2 t = cs[(d + e) / 2], u = cs[(d + half + e) / 2];
              const double x = a[e], y = a[e + 1], z = b[e], w = b[e + 1];
              a[e] = (float)(x * t.x - y * t.y);
              a[e + 1] = (float)(x * t.y + y * t.x);
              b[e] = (float)(z * u.x - w * u.y);
              b[e + 1] = (float)(z * u.y + w * u.x);
            }
          }
        }
      } else if (is_q || is_k) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int i = d + e;
          if (i >= p.rotary) continue;
          const bool low = p.neox ? i < half : i % 2 == 0;
          const int other = p.neox ? (low ? i + half : i - half) : i ^ 1;
          const double2 t = cs[p.neox ? (low ? i : i - half) : i / 2];
          const double y = load_as_f32(src, other, p.act), x = load_as_f32(src, i, p.act);
          a[e] = (float)(low ? x * t.x - y * t.y : y * t.y + x * t.x);
        }
      }
    }
    // The largest magnitude of the head, by its bits: a NaN's are above infinity's.
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++)
      top = max(top, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
    for (int o = lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    __syncwarp();
    if (!mine) continue;
    if (is_q) {
      TA *const dst = (TA *)p.q_out + row * p.q_out_stride + h * hd;
      store8(dst + d, a);
      if (rotated) store8(dst + d + half, b);
    } else if (at >= 0) {
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
  const unsigned blocks = (unsigned)((rows * parts + kWarps - 1) / kWarps);
  if (pairs) k_quant_kv_append<BITS, TA, true><<<blocks, kWarps * 32, 0, s>>>(p, parts, lanes);
  else k_quant_kv_append<BITS, TA, false><<<blocks, kWarps * 32, 0, s>>>(p, parts, lanes);
  JAL_CUDA(cudaGetLastError());
}
template <int BITS>
void run_append(const QuantAppendParams &p, cudaStream_t s) {
  if (p.a.act == JAL_F32) run_append<BITS, float>(p, s);
  else if (p.a.act == JAL_F16) run_append<BITS, __half>(p, s);
  else run_append<BITS, __nv_bfloat16>(p, s);
}

// ---- reading back -----------------------------------------------------------
// A block takes kReadSlots positions of one sequence and KV head; a thread has eight
// dims of kReadItems of them, K and V.  Bound by memory.
constexpr int kReadThreads = 256, kReadSlots = 64;

template <int BITS>
__device__ __forceinline__ void widen_codes8(const uint8_t *row, int d, float (&v)[8]) {
  if constexpr (BITS == 8) {
    const uint2 w = *(const uint2 *)(row + d);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e % 4)));
  } else {
    const uint32_t w = *(const uint32_t *)(row + d / 2);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)((int)((w >> (4 * e)) & 15u) - 8);
  }
}

template <int BITS, class TO>
__global__ void __launch_bounds__(kReadThreads) k_quant_kv_read(const __grid_constant__ QuantReadParams p, const int tiles) {
  const int tile = blockIdx.x % tiles, rest = blockIdx.x / tiles, head = rest % p.from.hkv, s = rest / p.from.hkv;
  const int beg = p.first ? max(__ldg(p.first + s), 0) : 0;
  const int64_t most = min((int64_t)beg + p.max_len, (int64_t)min(p.from.cap, p.into.cap));
  const int end = (int)min((int64_t)__ldg(p.kv_len + s), most);
  const int64_t t64 = (int64_t)beg + (int64_t)tile * kReadSlots;
  if (t64 >= end) return;
  const int t0 = (int)t64;
  const int n8 = p.from.hd / 8, total = min(kReadSlots, end - t0) * n8;
  const int32_t *const from = p.from.table + (int64_t)s * p.from.max_pages, *const into = p.into.table + (int64_t)s * p.into.max_pages;
#pragma unroll 4
  for (int i = threadIdx.x; i < total; i += kReadThreads) {
    const int t = t0 + i / n8, d = (i % n8) * 8;
    const Slot a = slot_of(p.from, from, t), b = slot_of(p.into, into, t);
    const int64_t at = slot_offset(p.from, a, head), to = slot_offset(p.into, b, head);
    if (at < 0 || to < 0) continue;
    const int64_t s_at = (int64_t)a.page * p.sc.s_page + head * p.sc.s_head + a.slot;
    const float ks = __ldg(p.sc.k + s_at), vs = __ldg(p.sc.v + s_at);
    float k[8], v[8];
    widen_codes8<BITS>((const uint8_t *)p.from.k + at, d, k);
    widen_codes8<BITS>((const uint8_t *)p.from.v + at, d, v);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      k[e] = __fmul_rn(k[e], ks);
      v[e] = __fmul_rn(v[e], vs);
    }
    store8((TO *)p.kw + to + d, k);
    store8((TO *)p.vw + to + d, v);
  }
}

template <int BITS>
void run_read(const QuantReadParams &p, cudaStream_t s) {
  const int64_t tiles = (p.max_len + kReadSlots - 1) / kReadSlots, blocks = tiles * p.from.hkv * p.n_seqs;
  if (blocks > 2000000000) fail(JAL_ERR_CAPABILITY_MISMATCH, "too many positions for one launch");
  if (p.into.dtype == JAL_F32) k_quant_kv_read<BITS, float><<<(unsigned)blocks, kReadThreads, 0, s>>>(p, (int)tiles);
  else if (p.into.dtype == JAL_F16) k_quant_kv_read<BITS, __half><<<(unsigned)blocks, kReadThreads, 0, s>>>(p, (int)tiles);
  else k_quant_kv_read<BITS, __nv_bfloat16><<<(unsigned)blocks, kReadThreads, 0, s>>>(p, (int)tiles);
  JAL_CUDA(cudaGetLastError());
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
