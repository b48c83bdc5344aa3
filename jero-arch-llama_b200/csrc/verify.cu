// Verification of drafted tokens against the target's probabilities, from given
// random numbers.
//
// Two kernels.  The first reads every row of logits once, in pieces: the largest
// logit m and sum exp((x - m) / T) of each piece (of greedy rows the first of the
// largest).  The second has a cluster of blocks for each sequence: the pieces give
// p(x) and q(x) of every draft, hence the row that emits a token; of that row alone
// the probabilities are formed again, in 64 bits, summed in the order of the
// vocabulary, and searched for the random number.
//
// The sums of the drawn row are in 64 bits because a token is where a number falls
// among up to 2^17 sums: with relative errors of 2^-24 in them, one draw in a hundred
// would be another token.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.hpp"
#include "paged_dev.cuh"
#include "quant_kv.hpp"

namespace jal {

namespace {

using namespace paged;
namespace cg = cooperative_groups;

constexpr int kStatThreads = 256, kDrawThreads = 256, kDrawWarps = kDrawThreads / 32, kCluster = 8;
constexpr float kCold = 1e-5f;  // temperatures up to this: all of the probability on the first largest logit
constexpr float kLog2e = 1.4426950408889634f;

// (An infinite temperature would make 0 x -inf of a logit of -inf.)
__device__ __forceinline__ float temperature_of(const float *t, int s) {
  if (!t) return 1.0f;
  const float x = __ldg(t + s);
  return x > 1e30f ? 1e30f : x;
}
__device__ __forceinline__ bool is_cold(float t) { return !(t > kCold); }

template <class T>
__device__ __forceinline__ float logit(const T *p);
template <>
__device__ __forceinline__ float logit<float>(const float *p) { return __ldg(p); }
template <>
__device__ __forceinline__ float logit<__half>(const __half *p) { return __half2float(__ldg(p)); }
template <>
__device__ __forceinline__ float logit<__nv_bfloat16>(const __nv_bfloat16 *p) { return __bfloat162float(__ldg(p)); }
// (A NaN counts as -inf.)
__device__ __forceinline__ float known(float x) { return x == x ? x : -INFINITY; }

// Elements [lo, hi) of a row by the block's threads, in pieces of 16 bytes where they
// are aligned: f(index, values[N]).
template <class T, class F>
__device__ __forceinline__ void each16(const T *row, int lo, int hi, F &&f) {
  constexpr int N = 16 / sizeof(T);
  const int skip = (int)((16 - ((uintptr_t)(row + lo) & 15)) & 15) / (int)sizeof(T);
  const int a = min(hi, lo + skip), n = (hi - a) / N, b = a + n * N;
  for (int i = lo + threadIdx.x; i < a; i += kStatThreads) {
    float x[N];
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = -INFINITY;
    x[0] = logit(row + i);
    f(i, x);
  }
#pragma unroll 4
  for (int k = threadIdx.x; k < n; k += kStatThreads) {
    const uint4 w = ldg_stream16(row + a + k * N);
    float x[N];
    if constexpr (sizeof(T) == 4) {
      x[0] = __uint_as_float(w.x);
      x[1] = __uint_as_float(w.y);
      x[2] = __uint_as_float(w.z);
      x[3] = __uint_as_float(w.w);
    } else {
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float2 v = unpack2<T>(u[e]);
        x[2 * e] = v.x;
        x[2 * e + 1] = v.y;
      }
    }
    f(a + k * N, x);
  }
  for (int i = b + threadIdx.x; i < hi; i += kStatThreads) {
    float x[N];
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = -INFINITY;
    x[0] = logit(row + i);
    f(i, x);
  }
}

// One piece of one row, target's or draft's: its largest logit with, of warm rows,
// the sum of the exponentials relative to it, of cold ones the first index of it.
template <class T>
__global__ void __launch_bounds__(kStatThreads) k_verify_stats(const __grid_constant__ VerifyParams p) {
  constexpr int N = 16 / sizeof(T);
  __shared__ float red_m[kStatThreads / 32], red_s[kStatThreads / 32];
  __shared__ int red_i[kStatThreads / 32];
  pdl_trigger();
  const int chunk = blockIdx.x % p.chunks, which = blockIdx.x / p.chunks, row = which % p.n_rows;
  const bool draft = which >= p.n_rows;
  const int first = __ldg(p.q_start), last = __ldg(p.q_start + p.n_seqs);
  const int s = warp_seq_of_row(p.q_start, p.n_seqs, row);
  if (row < first || row >= last) return;
  int beg, end;
  seq_rows(p.q_start, p.n_rows, s, beg, end);
  if (row < beg || row >= end || (draft && row == end - 1)) return;
  const float t = temperature_of(draft ? p.draft_temperature : p.temperature, s);
  const int per = ((p.vocab + p.chunks - 1) / p.chunks + 7) / 8 * 8;
  const int lo = (int)min((int64_t)p.vocab, (int64_t)chunk * per), hi = (int)min((int64_t)p.vocab, (int64_t)lo + per);
  const T *const x = (const T *)(draft ? p.draft : p.logits) + row * (draft ? p.draft_stride : p.stride);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float m = -INFINITY, sum = 0.0f;
  int at = 0x7fffffff;
  if (is_cold(t)) {
    each16(x, lo, hi, [&](int i, const float (&v)[N]) {
#pragma unroll
      for (int e = 0; e < N; e++)
        if (v[e] > m || (v[e] == m && i + e < at && m > -INFINITY)) {
          m = v[e];
          at = i + e;
        }
    });
  } else {
    const float c = kLog2e / t;
    each16(x, lo, hi, [&](int, const float (&v)[N]) {
      float most = v[0];
#pragma unroll
      for (int e = 1; e < N; e++) most = fmaxf(most, v[e]);
      if (most > m) {
        sum *= exp2f((m - most) * c);  // (m = -inf: the sum is 0)
        m = most;
      }
      if (m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < N; e++) sum += v[e] == v[e] ? exp2f((v[e] - m) * c) : 0.0f;
      }
    });
    if (m == -INFINITY) sum = 0.0f;
  }
  // Threads, then warps.
  float most = warp_max(m);
  if (is_cold(t)) {
    at = m == most && m > -INFINITY ? at : 0x7fffffff;
    at = __reduce_min_sync(0xffffffffu, at);
  } else {
    sum = m > -INFINITY ? sum * exp2f((m - most) * (kLog2e / t)) : 0.0f;
    sum = warp_sum(sum);
  }
  if (lane == 0) {
    red_m[warp] = most;
    red_s[warp] = sum;
    red_i[warp] = at;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = -INFINITY, total = 0.0f;
    int best = 0x7fffffff;
    for (int w = 0; w < kStatThreads / 32; w++) all = fmaxf(all, red_m[w]);
    for (int w = 0; w < kStatThreads / 32; w++) {
      if (red_m[w] == -INFINITY) continue;
      if (is_cold(t)) {
        if (red_m[w] == all) best = min(best, red_i[w]);
      } else {
        total += red_s[w] * exp2f((red_m[w] - all) * (kLog2e / t));
      }
    }
    p.part[(int64_t)which * p.chunks + chunk] = make_float2(all, is_cold(t) ? __int_as_float(best) : total);
  }
}

// A row's distribution as its pieces give it: the largest logit m, and the sum of
// exp((x - m) / T), or of cold rows the first index of m.  All lanes of a warp.
struct RowStats {
  float m, sum;
  int at;
  __device__ __forceinline__ bool none() const { return !(fabsf(m) < INFINITY); }
};
__device__ __forceinline__ RowStats row_stats(const VerifyParams &p, int which, float t) {
  const int lane = threadIdx.x % 32;
  const float2 *const part = p.part + (int64_t)which * p.chunks;
  float m = -INFINITY;
  for (int i = lane; i < p.chunks; i += 32) m = fmaxf(m, part[i].x);
  RowStats r = {warp_max(m), 0.0f, 0x7fffffff};
  for (int i = lane; i < p.chunks; i += 32) {
    const float2 v = part[i];
    if (v.x == -INFINITY) continue;
    if (is_cold(t)) {
      if (v.x == r.m) r.at = min(r.at, __float_as_int(v.y));
    } else {
      r.sum += v.y * exp2f((v.x - r.m) * (kLog2e / t));
    }
  }
  r.sum = warp_sum(r.sum);
  r.at = __reduce_min_sync(0xffffffffu, r.at);
  return r;
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// exp((x - m) / T) in 64 bits; 0 for -inf and NaN.
struct Weight {
  double m, inv;
  __device__ __forceinline__ double operator()(float x) const {
    return x > -INFINITY ? exp(((double)x - m) * inv) : 0.0;
  }
};

// What the row that emits draws from: exp((x_t - m) / T) / sum, less the draft's.
template <class T>
struct Drawn {
  const T *x, *y;  // target's logits; the draft's, or null
  Weight wx, wy;
  double zx, zy;   // 1 / sums
  int one;         // the token that the draft was sure of, or -1
  __device__ __forceinline__ double p(int t) const { return wx(logit(x + t)) * zx; }
  __device__ __forceinline__ double rest(int t, double px) const {
    if (t == one) return 0.0;
    return y ? fmax(px - wy(logit(y + t)) * zy, 0.0) : px;
  }
};

struct DrawShared {
  double zx, zy;                         // this block's sums of exponentials
  double rest[kDrawWarps], p[kDrawWarps];  // each warp's sums over its part of the vocabulary
  int stop;
  RowStats target, draft;
};

template <class T>
__global__ void __launch_bounds__(kDrawThreads) k_verify_draw(const __grid_constant__ VerifyParams p) {
  __shared__ DrawShared sh;
  constexpr int parts = kCluster * kDrawWarps;  // of the vocabulary, one a warp
  __shared__ double red[2][kDrawWarps], part_rest[parts], part_p[parts];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), s = blockIdx.x / kCluster;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  int beg, end;
  seq_rows(p.q_start, p.n_rows, s, beg, end);
  const float t = temperature_of(p.temperature, s), td = temperature_of(p.draft_temperature, s);
  if (tid == 0) sh.stop = end - 1;
  __syncthreads();
  pdl_wait();
  if (beg == end) {
    if (rank == 0 && tid == 0) {
      p.n_accepted[s] = 0;
      if (p.new_len) p.new_len[s] = p.kv_len[s];
    }
    return;  // (the whole cluster)
  }
  // Every block finds the row that emits: a warp for each draft.
  for (int r = beg + warp; r < end - 1; r += kDrawWarps) {
    if (r > __shfl_sync(0xffffffffu, *(volatile int *)&sh.stop, 0)) break;
    const int x = __ldg(p.tokens + r + 1);
    bool take = false;
    if (x >= 0 && x < p.vocab) {
      const RowStats a = row_stats(p, r, t);
      const float lx = known(logit((const T *)p.logits + r * p.stride + x));
      double px = 0.0, qx = 1.0;
      if (!a.none()) px = is_cold(t) ? (double)(a.at == x) : Weight{a.m, 1.0 / t}(lx) / a.sum;
      if (p.draft) {
        const RowStats b = row_stats(p, p.n_rows + r, td);
        const float ly = known(logit((const T *)p.draft + r * p.draft_stride + x));
        if (!b.none()) qx = is_cold(td) ? (double)(b.at == x) : Weight{b.m, 1.0 / td}(ly) / b.sum;
      }
      take = (double)__ldg(p.uniform + r) * qx < px;
    }
    if (!take && lane == 0) atomicMin(&sh.stop, r);
  }
  __syncthreads();
  const int stop = sh.stop;
  const bool sure = stop == end - 1;  // no draft is refused
  if (warp == 0) {
    const RowStats a = row_stats(p, stop, t);
    if (lane == 0) sh.target = a;
  } else if (warp == 1 && p.draft && !sure) {
    const RowStats b = row_stats(p, p.n_rows + stop, td);
    if (lane == 0) sh.draft = b;
  }
  __syncthreads();
  const RowStats a = sh.target;
  int token = -1;
  bool writes = rank == 0 && warp == 0;  // this warp writes the results
  if (!a.none() && is_cold(t)) {
    token = a.at;
  } else if (!a.none()) {
    Drawn<T> d = {};
    d.x = (const T *)p.logits + stop * p.stride;
    d.wx = Weight{a.m, 1.0 / t};
    d.one = -1;
    if (!sure) {
      const int x = __ldg(p.tokens + stop + 1);
      if (p.draft && !sh.draft.none() && !is_cold(td)) {
        d.y = (const T *)p.draft + stop * p.draft_stride;
        d.wy = Weight{sh.draft.m, 1.0 / td};
      } else {
        d.one = p.draft && !sh.draft.none() ? sh.draft.at : x;
      }
    }
    // This warp's part of the vocabulary, a whole number of 32.
    const int per = (p.vocab + parts * 32 - 1) / (parts * 32) * 32;
    const int mine = rank * kDrawWarps + warp;
    const int lo = (int)min((int64_t)p.vocab, (int64_t)mine * per), hi = (int)min((int64_t)p.vocab, (int64_t)lo + per);
    double zx = 0.0, zy = 0.0;
#pragma unroll 4
    for (int i = lo + lane; i < hi; i += 32) {
      zx += d.wx(logit(d.x + i));
      if (d.y) zy += d.wy(logit(d.y + i));
    }
    zx = warp_sum64(zx);
    zy = warp_sum64(zy);
    if (lane == 0) {
      red[0][warp] = zx;
      red[1][warp] = zy;
    }
    __syncthreads();
    if (tid == 0) {
      sh.zx = sh.zy = 0.0;
      for (int w = 0; w < kDrawWarps; w++) {
        sh.zx += red[0][w];
        sh.zy += red[1][w];
      }
    }
    cluster.sync();
    zx = zy = 0.0;
    for (int k = 0; k < kCluster; k++) {
      const DrawShared *const o = cluster.map_shared_rank(&sh, k);
      zx += o->zx;
      zy += o->zy;
    }
    d.zx = 1.0 / zx;
    d.zy = d.y ? 1.0 / zy : 0.0;
    double rest = 0.0, whole = 0.0;
#pragma unroll 4
    for (int i = lo + lane; i < hi; i += 32) {
      const double px = d.p(i);
      whole += px;
      rest += d.rest(i, px);
    }
    rest = warp_sum64(rest);
    whole = warp_sum64(whole);
    if (lane == 0) {
      sh.rest[warp] = rest;
      sh.p[warp] = whole;
    }
    cluster.sync();
    if (tid < parts) {
      const DrawShared *const o = cluster.map_shared_rank(&sh, tid / kDrawWarps);
      part_rest[tid] = o->rest[tid % kDrawWarps];
      part_p[tid] = o->p[tid % kDrawWarps];
    }
    __syncthreads();
    cluster.sync();  // no block leaves while others read its sums
    // Every warp goes through the parts in order, with the same numbers: the part
    // in which the running sum first exceeds `want`, or the last one with any weight
    // where rounding (or a number that is not below 1) leaves none.
    double total = 0.0;
    for (int k = 0; k < parts; k++) total += part_rest[k];
    const bool from_p = !(total > 0.0);
    const double *const part = from_p ? part_p : part_rest;
    if (from_p) {
      total = 0.0;
      for (int k = 0; k < parts; k++) total += part[k];
    }
    const double want = (double)__ldg(p.uniform + end - 1) * total;
    int chosen = -1;
    bool over = false;
    double run = 0.0, before = 0.0;
    for (int k = 0; k < parts && !over; k++) {
      if (!(part[k] > 0.0)) continue;
      chosen = k;
      before = run;
      run += part[k];
      over = run > want;
    }
    if (mine != max(chosen, 0)) return;
    writes = true;
    int pick = -1, some = -1;
    for (int i0 = lo; i0 < hi && pick < 0; i0 += 32) {
      const int i = i0 + lane;
      double w = 0.0;
      if (i < hi) {
        const double px = d.p(i);
        w = from_p ? px : d.rest(i, px);
      }
      double sum = w;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const double n = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += n;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, w > 0.0 && before + sum > want);
      const uint32_t any = __ballot_sync(0xffffffffu, w > 0.0);
      if (past) pick = i0 + __ffs(past) - 1;
      if (any) some = i0 + 31 - __clz(any);
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    token = pick >= 0 ? pick : some;
  }
  if (!writes) return;
  for (int r = beg + lane; r < end; r += 32) p.out_tokens[r] = r < stop ? __ldg(p.tokens + r + 1) : r == stop ? token : -1;
  if (lane == 0) {
    p.n_accepted[s] = stop - beg;
    if (p.new_len) p.new_len[s] = p.kv_len[s] - (end - 1 - stop);
  }
}

template <class T>
void run(const VerifyParams &p, cudaStream_t s) {
  if (p.n_rows) {
    const int64_t blocks = (int64_t)p.n_rows * p.chunks * (p.draft ? 2 : 1);
    k_verify_stats<T><<<(unsigned)blocks, kStatThreads, 0, s>>>(p);
    JAL_CUDA(cudaGetLastError());
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.n_seqs * kCluster);
  cfg.blockDim = dim3(kDrawThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {kCluster, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.n_rows ? 2 : 1;
  JAL_CUDA(cudaLaunchKernelEx(&cfg, k_verify_draw<T>, p));
}

}  // namespace

int verify_chunks(size_t n_rows, size_t vocab) {
  // Pieces of 4096 logits at least, blocks enough for every SM several times over.
  const size_t most = std::max<size_t>(1, vocab / 4096), want = (size_t)kPagedSMs * 8 / n_rows + 1;
  return (int)std::min<size_t>(64, std::min(most, want));
}

void launch_verify_drafts(const VerifyParams &p, cudaStream_t s) {
  if (p.dtype == JAL_F32) run<float>(p, s);
  else if (p.dtype == JAL_F16) run<__half>(p, s);
  else run<__nv_bfloat16>(p, s);
}

}  // namespace jal
