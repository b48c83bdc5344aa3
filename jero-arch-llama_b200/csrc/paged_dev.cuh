// Device code shared by the kernels over a paged cache: where a key lives,
// which keys a tile of query rows sees, and how its results are written.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "dev_util.cuh"
#include "paged.hpp"

namespace jal {
namespace paged {

__device__ __forceinline__ float load_as_f32(const void *p, int64_t i, int dtype) {
  if (dtype == JAL_F32) return ((const float *)p)[i];
  if (dtype == JAL_F16) return __half2float(((const __half *)p)[i]);
  return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}
__device__ __forceinline__ void store_from_f32(void *p, int64_t i, int dtype, float v) {
  if (dtype == JAL_F32)
    ((float *)p)[i] = v;
  else if (dtype == JAL_F16)
    ((__half *)p)[i] = __float2half_rn(v);
  else
    ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
}

template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*(__half2 *)&w);
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *(uint32_t *)&h;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *(uint32_t *)&h;
}

// Eight consecutive elements as f32 (p 16-byte aligned).
template <class T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
  const uint4 w = *(const uint4 *)p;
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = unpack2<T>(u[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&v)[8]) {
  const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// Adds x * 0 of eight 16-bit elements: NaN in acc once an element was not finite.
template <class T>
__device__ __forceinline__ void watch8(uint32_t &acc, const uint4 &x);
template <>
__device__ __forceinline__ void watch8<__half>(uint32_t &acc, const uint4 &x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; i++) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w[i]), "r"(0u));
}
template <>
__device__ __forceinline__ void watch8<__nv_bfloat16>(uint32_t &acc, const uint4 &x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; i++) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w[i]), "r"(0u));
}
template <class T>
__device__ __forceinline__ bool watched_bad(uint32_t acc) {
  const float2 f = unpack2<T>(acc);
  return f.x != f.x || f.y != f.y;
}
template <class T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  *(uint4 *)p = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float *p, const float (&v)[8]) {
  ((float4 *)p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  ((float4 *)p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// 2^x by the special-function unit: relative error 2^-22, results below 2^-126
// are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Where position t's row of `head` lies.  In two steps, so that the table entry
// can be asked for long before it is needed: `page` is the entry as found.
struct Slot {
  int page, slot;
};
__device__ __forceinline__ Slot slot_of(const PagedView &kv, const int32_t *table_row, int t) {
  const int pi = kv.page_shift >= 0 ? t >> kv.page_shift : t / kv.page_size;
  int page;  // (volatile: the load stays where it is asked for)
  asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(page) : "l"(table_row + pi));
  return {page, kv.page_shift >= 0 ? t & (kv.page_size - 1) : t - pi * kv.page_size};
}
// The element offset, or -1 where the entry is no page of the pool (such a
// key counts as masked and is not read).
__device__ __forceinline__ int64_t slot_offset(const PagedView &kv, const Slot &s, int head) {
  const int64_t at = (int64_t)s.page * kv.page_stride + (int64_t)head * kv.head_stride + (int64_t)s.slot * kv.slot_stride;
  return (unsigned)s.page < (unsigned)kv.n_pages ? at : -1;
}
__device__ __forceinline__ int64_t slot_offset(const PagedView &kv, const int32_t *table_row, int head, int t) {
  return slot_offset(kv, slot_of(kv, table_row, t), head);
}

// Rows [beg, end) of sequence s, kept inside the batch whatever q_start says.
__device__ __forceinline__ void seq_rows(const int32_t *q_start, int n_rows, int s, int &beg, int &end) {
  const int b = __ldg(q_start + s), e = __ldg(q_start + s + 1);
  beg = min(max(b, 0), n_rows);
  end = min(max(e, beg), n_rows);
}
// The sequence in [lo, hi) that holds row r (q_start ascending): the last one
// that starts at or before it.
__device__ __forceinline__ int seq_of_row(const int32_t *q_start, int lo, int hi, int r) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(q_start + mid) <= r) lo = mid; else hi = mid;
  }
  return lo;
}

// The sequence in [0, n) that holds row r, found by the whole warp: 32 starts at
// a time, so two rounds for 1024 sequences instead of ten dependent loads.
__device__ __forceinline__ int warp_seq_of_row(const int32_t *q_start, int n, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;  // q_start[lo] <= r (or lo = 0)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + step * lane;
    const bool before = lane > 0 && at < hi && __ldg(q_start + at) <= r;
    const int k = __popc(__ballot_sync(0xffffffffu, before));
    lo += step * k;
    hi = min(hi, lo + step);
  }
  return lo;
}

// One tile of query rows of one KV head, and the keys it reads.  Tile row j
// is row (first + j) of the (token, head-of-group) pairs counted from token
// row `beg`.  Its keys are the positions [0, ns) and [lo, hi), numbered
// u = 0 .. ns + hi - lo - 1 without a gap, and the tile takes [u0, u1) of
// them; a row of position p sees t <= p with t > p - window or t < n_sink.
struct Tile {
  const int32_t *table;  // the page-table row the keys are read through
  const int32_t *ahead;  // and the one for positions below `shared` (a prefix that a sequence reads for itself)
  int shared;
  int beg, end;          // token rows of the sequence / of the group
  int first, rows;       // first (token, head) pair; pairs of this tile
  int head;              // KV head
  int ns, lo, hi;
  int u0, u1;
  int slot;              // partial slot the results go to
  int limit;             // prefix tiles: keys end here for every row
  int seq_lo, seq_hi;    // sequences whose rows these are
  int64_t shift;         // one sequence: a token row's position is row + shift
  __device__ __forceinline__ int key(int u) const { return u < ns ? u : lo + (u - ns); }
};

__device__ __forceinline__ Slot slot_of(const PagedView &kv, const Tile &t, int key) {
  return slot_of(kv, key < t.shared ? t.ahead : t.table, key);
}

// Position of token row r: -1 before the first position (such a row sees
// nothing), at most the last position of the table.
__device__ __forceinline__ int clamp_position(const AttnParams &p, int64_t pos) {
  return pos < 0 ? -1 : pos >= p.kv.cap ? p.kv.cap - 1 : (int)pos;
}
__device__ __forceinline__ int row_position(const AttnParams &p, const Tile &t, int r) {
  if (t.seq_hi - t.seq_lo == 1) return clamp_position(p, r + t.shift);
  const int s = seq_of_row(p.q_start, t.seq_lo, t.seq_hi, r);
  int b, e;
  seq_rows(p.q_start, p.n_rows, s, b, e);
  return clamp_position(p, (int64_t)__ldg(p.kv_len + s) - (e - r));
}

// Tile `tile` (of `rt` rows) and piece `piece` of block (seq or group) `z`;
// false when there is nothing to do.  Positions at or past the table's end
// see what a row at its end sees.
__device__ __forceinline__ bool make_tile(const AttnParams &p, bool prefix, int z, int head, int tile, int piece,
                                          int rt, int key_align, Tile &t) {
  t.head = head;
  t.seq_lo = z;
  t.seq_hi = z + 1;
  int prefix_len = 0;
  if (prefix) {
    const int a = __ldg(p.group_start + z), b = __ldg(p.group_start + z + 1);
    prefix_len = __ldg(p.prefix_len + z);
    t.seq_lo = min(max(a, 0), p.n_seqs);
    t.seq_hi = min(max(b, t.seq_lo), p.n_seqs);
    if (t.seq_lo == t.seq_hi) return false;
  }
  // (Loads that do not depend on each other, asked for together.)
  int own_first = 0, own_last = 0, own_prefix = 0;
  if (!prefix && p.n_groups) {
    const int g = seq_of_row(p.group_start, 0, p.n_groups, t.seq_lo);
    own_first = __ldg(p.group_start + g);
    own_last = __ldg(p.group_start + g + 1);
    own_prefix = __ldg(p.prefix_len + g);
  }
  const int len = __ldg(p.kv_len + t.seq_lo);
  seq_rows(p.q_start, p.n_rows, t.seq_lo, t.beg, t.end);
  t.shift = (int64_t)len - t.end;
  if (t.seq_hi - t.seq_lo > 1) {
    int e;
    seq_rows(p.q_start, p.n_rows, t.seq_hi - 1, e, t.end);
  }
  int n_tok = t.end - t.beg;
  if (!prefix) n_tok = min(n_tok, p.max_q);
  t.first = tile * rt;
  t.rows = min(rt, n_tok * p.G - t.first);
  if (t.rows <= 0) return false;
  t.table = t.ahead = p.kv.table + (int64_t)t.seq_lo * p.kv.max_pages;
  t.shared = 0;
  const int splits = prefix ? p.prefix_splits : p.splits;
  t.slot = (prefix ? 0 : p.prefix_splits) + piece;
  t.limit = 0x7fffffff;
  if (prefix) {
    t.limit = min(max(prefix_len, 0), p.kv.cap);
    t.ns = t.lo = 0;
    t.hi = t.limit;
  } else {
    const int pf = row_position(p, t, t.beg + t.first / p.G), pl = row_position(p, t, t.beg + (t.first + t.rows - 1) / p.G);
    t.hi = pl + 1;
    t.lo = p.window > 0 ? max(0, pf + 1 - p.window) : 0;
    if (p.n_groups) {  // the keys behind the shared prefix of the sequence's group
      const bool in = own_first <= t.seq_lo && t.seq_lo < own_last;
      const int shared = in ? min(max(own_prefix, 0), p.kv.cap) : 0;
      if (p.prefix_splits) {
        t.lo = shared;
      } else {
        t.shared = shared;
        t.ahead = p.kv.table + (int64_t)min(max(own_first, 0), p.n_seqs - 1) * p.kv.max_pages;
      }
    }
    t.lo = min(t.lo, t.hi);
    t.ns = min(p.n_sink, t.lo);
  }
  const int total = t.ns + (t.hi - t.lo);
  const uint32_t step = (uint32_t)splits * key_align;  // (total + step stays below 2^32)
  const int per = (int)(((uint32_t)total + step - 1) / step) * key_align;
  t.u0 = (int)min((int64_t)total, (int64_t)piece * per);
  t.u1 = (int)min((int64_t)total, (int64_t)t.u0 + per);
  return true;
}

// Which tiles a launch works on.
enum Part { kBoth, kPrefix, kOwn };
// Which tile a block of the flat grid works on: first the shared prefixes'
// (piece fastest, then tile, head, group), then the sequences'.
__device__ __forceinline__ bool block_tile(const AttnParams &p, int part, int rt, int key_align, Tile &t) {
  uint32_t b = blockIdx.x;  // (32-bit divisions: the grid is below 2^31)
  const uint32_t np = part == kOwn ? 0 : (uint32_t)(p.prefix_splits * p.prefix_tiles) * (uint32_t)(p.kv.hkv * p.n_groups);
  const bool prefix = b < np;
  if (!prefix) b -= np;
  const uint32_t splits = prefix ? p.prefix_splits : p.splits, tiles = prefix ? p.prefix_tiles : p.tiles, hkv = p.kv.hkv;
  uint32_t rest = b / splits;
  const int piece = (int)(b - rest * splits);
  b = rest;
  rest = b / tiles;
  const int tile = (int)(tiles - 1 - (b - rest * tiles));  // the last rows see the most keys: first
  const uint32_t z = rest / hkv;
  return make_tile(p, prefix, (int)z, (int)(rest - z * hkv), tile, piece, rt, key_align, t);
}

// What row j of the tile may see: keys t < lim with t >= wlo or t < sink.
struct RowMask {
  int lim, wlo;
  __device__ __forceinline__ bool sees(int t, int n_sink) const { return t < lim && (t >= wlo || t < n_sink); }
};
__device__ __forceinline__ RowMask row_mask(const AttnParams &p, const Tile &t, int j) {
  const int pos = row_position(p, t, t.beg + (t.first + j) / p.G);
  RowMask m;
  m.lim = min(pos + 1, t.limit);
  m.wlo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
  return m;
}
// The same over the key numbers u of the tile: a row sees u < end with u <
// sink or u >= near, whose bounds do not depend on u.
struct RowSpan {
  int end, sink, near;
  // Is all of [u, u + n) seen?
  __device__ __forceinline__ bool all(int u, int n) const { return u + n <= end && (u >= near || u + n <= sink); }
  // Which of the 32 keys from u on are seen.
  __device__ __forceinline__ uint32_t bits(int u) const {
    return below(end - u) & (below(sink - u) | ~below(near - u));
  }
  static __device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
};
__device__ __forceinline__ RowSpan row_span(const AttnParams &p, const Tile &t, const RowMask &m) {
  RowSpan s;
  s.end = m.lim > t.lo ? t.ns + (m.lim - t.lo) : min(m.lim, t.ns);
  s.sink = t.ns + max(0, p.n_sink - t.lo);
  s.near = t.ns + max(0, m.wlo - t.lo);
  return s;
}
__device__ __forceinline__ int64_t q_offset(const AttnParams &p, const Tile &t, int j) {
  const int pair = t.first + j;
  return (int64_t)(t.beg + pair / p.G) * p.q_stride + (int64_t)(t.head * p.G + pair % p.G) * p.kv.hd;
}
__device__ __forceinline__ int64_t out_offset(const AttnParams &p, const Tile &t, int j) {
  const int pair = t.first + j;
  return (int64_t)(t.beg + pair / p.G) * p.out_stride + (int64_t)(t.head * p.G + pair % p.G) * p.kv.hd;
}
// (slot, row, query head) index of the partial results.
__device__ __forceinline__ int64_t part_index(const AttnParams &p, const Tile &t, int j) {
  const int pair = t.first + j;
  return ((int64_t)t.slot * p.n_rows + t.beg + pair / p.G) * p.hq + t.head * p.G + pair % p.G;
}

// Row j by itself, one warp: only keys that the row sees are read, one after
// another.  A product of a zero weight and a NaN or infinite value is NaN, so
// a tile in which such a value stands at a key that some rows see and others
// do not is done again this way; slow, and right for each row.  q and the
// cache are read in their own types, sums are f32.
static __device__ __noinline__ void attend_row_alone(const AttnParams &p, const Tile &t, int j, bool direct) {
  const int lane = threadIdx.x & 31;
  const RowMask mk = row_mask(p, t, j);
  const int64_t qo = q_offset(p, t, j);
  constexpr int N = kPagedMaxHeadDim / 32;
  float q[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int d = lane + 32 * i;
    q[i] = d < p.kv.hd ? load_as_f32(p.q, qo + d, p.act) : 0.0f;
    o[i] = 0.0f;
  }
  for (int u = t.u0; u < t.u1; u++) {
    const int key = t.key(u);
    if (!mk.sees(key, p.n_sink)) continue;
    const int64_t at = slot_offset(p.kv, slot_of(p.kv, t, key), t.head);
    if (at < 0) continue;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int d = lane + 32 * i;
      if (d < p.kv.hd) s = fmaf(q[i], load_as_f32(p.kv.k, at + d, p.kv.dtype), s);
    }
    s = warp_sum(s) * p.scale_log2;
    const float mn = s != s ? s : fmaxf(m, s);  // a NaN score makes the row NaN, as the formula does
    const float c = mn == -INFINITY ? 1.0f : exp2f(m - mn), w = mn == -INFINITY ? 0.0f : exp2f(s - mn);
    l = l * c + w;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int d = lane + 32 * i;
      if (d < p.kv.hd) o[i] = fmaf(w, load_as_f32(p.kv.v, at + d, p.kv.dtype), o[i] * c);
    }
    m = mn;
  }
  const int64_t pi = part_index(p, t, j), oo = out_offset(p, t, j);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (!direct && lane == 0) p.part_ml[pi] = make_float2(m, l);
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int d = lane + 32 * i;
    if (d >= p.kv.hd) continue;
    if (direct)
      store_from_f32(p.out, oo + d, p.act, l == 0.0f ? 0.0f : o[i] * inv);
    else
      p.part_o[pi * p.kv.hd + d] = o[i];
  }
}

}  // namespace paged
}  // namespace jal
