// New keys and values of a ragged batch into the paged cache, with the
// position rotation applied on the way (and to the queries).
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "paged_dev.cuh"

namespace jal {

namespace {

using namespace paged;

constexpr int kAppendThreads = 256;

// cos and sin of pos * inv_freq with the product formed in 64 bits: at
// position 10^5 a product rounded to f32 is off by 4e-3 radians.  The angle is
// reduced to [-pi, pi] in 64 bits and rounded once, to f32.
__device__ __forceinline__ float2 turn(int64_t pos, float inv_freq) {
  const double a = (double)pos * (double)inv_freq;
  const double r = fma(-rint(a * 0.15915494309189535), 6.283185307179586, a);
  float2 cs;
  sincosf((float)r, &cs.y, &cs.x);
  return cs;
}

// One head's row, eight elements at a time: element i and its partner.
template <class TA>
__device__ __forceinline__ void rotated8(const TA *row, int d, int rotary, int neox, const float2 *cs, float (&v)[8]) {
  load8(row + d, v);
  if (d >= rotary) return;
  const int half = rotary / 2;
  if (neox) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int i = d + e;
      if (i >= rotary) continue;
      const bool low = i < half;
      const float2 c = cs[low ? i : i - half];
      const float other = load_as_f32(row, low ? i + half : i - half,
                                      sizeof(TA) == 4 ? JAL_F32 : std::is_same<TA, __half>::value ? JAL_F16 : JAL_BF16);
      v[e] = low ? v[e] * c.x - other * c.y : other * c.y + v[e] * c.x;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if (d + e >= rotary) continue;
      const float2 c = cs[(d + e) / 2];
      const float a = v[e], b = v[e + 1];
      v[e] = a * c.x - b * c.y;
      v[e + 1] = a * c.y + b * c.x;
    }
  }
}

// rotary_dim a multiple of 16 (or 0): a warp takes part of a token row's heads,
// item by item.  An item is eight dims and, in the rotated part, the eight
// rotary_dim / 2 further on, so both of a pair's elements are in one lane
// whichever way they are paired, and q_out may be q.  What bounds it: reading
// the rows and writing the pages once; kItems items of a lane are on their way
// at a time, kept as they are in memory until they are turned.  10833 rows of 48
// heads of 128 bf16 dims: 50 us, 5.3 TB/s (82 us with the items widened as they
// come, which halves the warps an SM holds; 86 us with a block for each row).
constexpr int kWarps = 4;

__device__ __forceinline__ void turn8(float (&a)[8], float (&b)[8], const float2 *cs, int d, int half, int neox) {
#pragma unroll
  for (int e = 0; e < 8; e++) {
    if (neox) {
      const float2 c = cs[d + e];
      const float x = a[e], y = b[e];
      a[e] = x * c.x - y * c.y;
      b[e] = x * c.y + y * c.x;
    } else if (e % 2 == 0) {
      const float2 c = cs[(d + e) / 2], f = cs[(d + half + e) / 2];
      const float x = a[e], y = a[e + 1], z = b[e], w = b[e + 1];
      a[e] = x * c.x - y * c.y;
      a[e + 1] = x * c.y + y * c.x;
      b[e] = z * f.x - w * f.y;
      b[e + 1] = z * f.y + w * f.x;
    }
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

template <class TA, class TK>
__global__ void __launch_bounds__(kWarps * 32, 7) k_rope_kv_append_pairs(const __grid_constant__ AppendParams p, const int parts) {
  constexpr int kItems = sizeof(TA) == 4 ? 2 : 4;
  __shared__ float2 turns[kWarps][kPagedMaxHeadDim / 2];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, unit = blockIdx.x * kWarps + warp;
  const int row = unit / parts, part = unit - row * parts;
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
  const int64_t at = pos64 >= p.kv.cap ? -1 : slot_offset(p.kv, p.kv.table + (int64_t)s * p.kv.max_pages, 0, (int)pos64);
  float2 *const cs = turns[warp];
  for (int i = lane; i < half; i += 32) cs[i] = turn(pos64, __ldg(p.inv_freq + i));
  __syncwarp();
  const int nq = p.q ? p.hq : 0, items = half / 8 + (hd - p.rotary) / 8, total = (nq + 2 * p.kv.hkv) * items;
  const int per = (total + parts - 1) / parts, stop = min(total, (part + 1) * per);
  for (int i = part * per + lane; i < stop; i += 32 * kItems) {
    Raw8<TA> ra[kItems], rb[kItems];
#pragma unroll
    for (int k = 0; k < kItems; k++) {
      const int it = i + 32 * k;
      if (it >= stop) break;
      const int head = it / items, c = it - head * items;
      const bool is_q = head < nq, is_k = !is_q && head < nq + p.kv.hkv;
      const int h = is_q ? head : head - nq - (is_k ? 0 : p.kv.hkv);
      const TA *const src = (const TA *)(is_q ? p.q : is_k ? p.k : p.v) + row * (is_q ? p.q_stride : p.kv_stride) + h * hd;
      if (c < half / 8) {
        ra[k].load(src + c * 8);
        rb[k].load(src + c * 8 + half);
      } else {
        ra[k].load(src + p.rotary + (c - half / 8) * 8);
      }
    }
#pragma unroll
    for (int k = 0; k < kItems; k++) {
      const int it = i + 32 * k;
      if (it >= stop) break;
      const int head = it / items, c = it - head * items;
      const bool is_q = head < nq, is_k = !is_q && head < nq + p.kv.hkv;
      const int h = is_q ? head : head - nq - (is_k ? 0 : p.kv.hkv);
      const bool rotated = c < half / 8;
      const int d = rotated ? c * 8 : p.rotary + (c - half / 8) * 8;
      float a[8], b[8];
      ra[k].widen(a);
      rb[k].widen(b);
      if (rotated && (is_q || is_k)) turn8(a, b, cs, d, half, p.neox);
      if (is_q) {
        TA *const dst = (TA *)p.q_out + row * p.q_out_stride + h * hd;
        store8(dst + d, a);
        if (rotated) store8(dst + d + half, b);
      } else if (at >= 0) {
        TK *const dst = (TK *)(is_k ? p.kw : p.vw) + at + h * p.kv.head_stride;
        store8(dst + d, a);
        if (rotated) store8(dst + d + half, b);
      }
    }
  }
}

// Any rotary_dim: one block per token row.
template <class TA, class TK>
__global__ void __launch_bounds__(kAppendThreads) k_rope_kv_append(const AppendParams p, const int lanes) {
  __shared__ float2 cs[kPagedMaxHeadDim / 2];
  const int row = blockIdx.x, hd = p.kv.hd;
  if (row < p.q_start[0] || row >= p.q_start[p.n_seqs]) return;
  const int s = warp_seq_of_row(p.q_start, p.n_seqs, row);
  int beg, end;
  seq_rows(p.q_start, p.n_rows, s, beg, end);
  const int64_t pos64 = (int64_t)p.kv_len[s] - (end - row);
  if (pos64 < 0) return;
  for (int i = threadIdx.x; i < p.rotary / 2; i += kAppendThreads) cs[i] = turn(pos64, p.inv_freq[i]);
  __syncthreads();
  // A head's row belongs to `lanes` neighbouring lanes, eight elements each.
  // Every lane has read what it needs (its partners' elements too) before any
  // lane writes, so q_out may be q.
  const int nq = p.q ? p.hq : 0, heads = nq + 2 * p.kv.hkv;
  const int32_t *table = p.kv.table + (int64_t)s * p.kv.max_pages;
  const int per_block = kAppendThreads / lanes, d = (threadIdx.x % lanes) * 8;
  for (int base = 0; base < heads; base += per_block) {
    const int head = base + threadIdx.x / lanes;
    const bool mine = head < heads && d < hd;
    const bool is_q = head < nq, is_k = !is_q && head < nq + p.kv.hkv;
    const int h = is_q ? head : head - nq - (is_k ? 0 : p.kv.hkv);
    const TA *src = (const TA *)(is_q ? p.q : is_k ? p.k : p.v) + row * (is_q ? p.q_stride : p.kv_stride) + h * hd;
    float v[8];
    if (mine) {
      if (is_q || is_k) rotated8(src, d, p.rotary, p.neox, cs, v);
      else load8(src + d, v);
    }
    __syncwarp();
    if (!mine) continue;
    if (is_q) {
      store8((TA *)p.q_out + row * p.q_out_stride + h * hd + d, v);
    } else {
      const int64_t at = pos64 >= p.kv.cap ? -1 : slot_offset(p.kv, table, h, (int)pos64);
      if (at >= 0) store8((TK *)(is_k ? p.kw : p.vw) + at + d, v);
    }
  }
}

template <class TA, class TK>
void run(const AppendParams &p, cudaStream_t s) {
  if (p.rotary % 16 == 0) {
    // Warps enough to fill the SMs, each with a round of items at least.
    const int heads = (p.q ? p.hq : 0) + 2 * p.kv.hkv, items = heads * (p.rotary / 16 + (p.kv.hd - p.rotary) / 8);
    const int most = std::max(1, items / (32 * (sizeof(TA) == 4 ? 2 : 4)));
    const int64_t rows = p.n_rows;
    const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(most, 32 * kPagedSMs / rows));
    const unsigned blocks = (unsigned)((rows * parts + kWarps - 1) / kWarps);
    k_rope_kv_append_pairs<TA, TK><<<blocks, kWarps * 32, 0, s>>>(p, parts);
  } else {
    int lanes = 1;
    while (lanes * 8 < p.kv.hd) lanes *= 2;
    k_rope_kv_append<TA, TK><<<(unsigned)p.n_rows, kAppendThreads, 0, s>>>(p, lanes);
  }
  JAL_CUDA(cudaGetLastError());
}

}  // namespace

void launch_rope_kv_append(const AppendParams &p, cudaStream_t s) {
  if (p.act == JAL_F16) run<__half, __half>(p, s);
  else if (p.act == JAL_BF16) run<__nv_bfloat16, __nv_bfloat16>(p, s);
  else if (p.kv.dtype == JAL_F32) run<float, float>(p, s);
  else if (p.kv.dtype == JAL_F16) run<float, __half>(p, s);
  else run<float, __nv_bfloat16>(p, s);
}

}  // namespace jal
