// New keys and values of a ragged batch into the paged cache, with the
// position rotation applied on the way (and to the queries).
#include "common.hpp"
#include "paged_dev.cuh"

namespace jal {

namespace {

using namespace paged;

constexpr int kAppendThreads = 256;

// cos and sin of pos * inv_freq with the product formed in 64 bits: at
// position 10^5 a product rounded to f32 is off by 4e-3 radians.  The angle is
// reduced to [-pi, pi] in 64 bits and rounded once, to f32.
__device__ __forceinline__ float2 turn(int pos, float inv_freq) {
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

// One block per token row.
template <class TA, class TK>
__global__ void __launch_bounds__(kAppendThreads) k_rope_kv_append(const AppendParams p, const int lanes) {
  __shared__ float2 cs[kPagedMaxHeadDim / 2];
  const int row = blockIdx.x, hd = p.kv.hd;
  if (row < p.q_start[0] || row >= p.q_start[p.n_seqs]) return;
  const int s = seq_of_row(p.q_start, 0, p.n_seqs, row);
  int beg, end;
  seq_rows(p.q_start, p.n_rows, s, beg, end);
  const int64_t pos64 = (int64_t)p.kv_len[s] - (end - row);
  if (pos64 < 0 || pos64 >= p.kv.cap) return;
  const int pos = (int)pos64;
  for (int i = threadIdx.x; i < p.rotary / 2; i += kAppendThreads) cs[i] = turn(pos, p.inv_freq[i]);
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
      const int64_t at = slot_offset(p.kv, table, h, pos);
      if (at >= 0) store8((TK *)(is_k ? p.kw : p.vw) + at + d, v);
    }
  }
}

template <class TA, class TK>
void run(const AppendParams &p, cudaStream_t s) {
  int lanes = 1;
  while (lanes * 8 < p.kv.hd) lanes *= 2;
  k_rope_kv_append<TA, TK><<<(unsigned)p.n_rows, kAppendThreads, 0, s>>>(p, lanes);
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
