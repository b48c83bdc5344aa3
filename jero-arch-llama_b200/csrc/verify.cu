// Verification of drafted tokens against the target's probabilities, from given
// random numbers.
//
// Two kernels.  The first reads every row of logits once, in pieces: the largest
// logit m and sum exp((x - m) / T) of each piece (of greedy rows the first of the
// largest).  The second has a few blocks for each sequence: the pieces give p(x) and
// q(x) of every draft, hence the row that emits a token; of that row alone the
// probabilities are formed again, in 64 bits, and summed over parts of the vocabulary;
// the sequence's last block to be done with that finds the part, and in it the token, in
// which the running sum passes the random number.
//
// The sums of the drawn row are in 64 bits because a token is where a number falls
// among up to 2^17 sums: with relative errors of 2^-24 in them, one draw in a hundred
// would be another token.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "paged_attn_tc.cuh"
#include "paged_dev.cuh"
#include "quant_kv.hpp"

namespace jal {

namespace {

using namespace paged;

constexpr int kStatThreads = 256, kDrawThreads = 256, kDrawWarps = kDrawThreads / 32, kDrawBlocks = 32;  // kDrawBlocks: of a sequence, at most
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
// The larger of two words' values (a NaN is passed over), and a word's values.
template <class T>
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t word_max<float>(uint32_t a, uint32_t b) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
template <>
__device__ __forceinline__ uint32_t word_max<__half>(uint32_t a, uint32_t b) {
  uint32_t v;
  asm("max.f16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
  return v;
}
template <>
__device__ __forceinline__ uint32_t word_max<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t v;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
  return v;
}
template <class T>
constexpr uint32_t kLowest = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;

// Elements [lo, hi) of a row by the block's threads, kBatch pieces of 16 bytes at a time
// where they are aligned: f(words, first indexes of the pieces), -inf where there is no
// element.
constexpr int kBatch = 4;
template <class T, class F>
__device__ __forceinline__ void each_batch(const T *row, int lo, int hi, F &&f) {
  constexpr int N = 16 / sizeof(T);
  const int skip = (int)((16 - ((uintptr_t)(row + lo) & 15)) & 15) / (int)sizeof(T);
  const int a = min(hi, lo + skip), n = (hi - a) / N, b = a + n * N;
  auto one = [&](int i) {
    uint32_t w[kBatch * 4];
    int at[kBatch];
#pragma unroll
    for (int e = 0; e < kBatch * 4; e++) w[e] = kLowest<T>;
#pragma unroll
    for (int k = 0; k < kBatch; k++) at[k] = i;
    if constexpr (sizeof(T) == 4) w[0] = __ldg((const uint32_t *)row + i);
    else w[0] = __byte_perm(__ldg((const uint16_t *)row + i), kLowest<T>, 0x5410);
    f(w, at);
  };
  for (int i = lo + threadIdx.x; i < a; i += kStatThreads) one(i);
  for (int k0 = threadIdx.x; k0 < n; k0 += kStatThreads * kBatch) {
    uint32_t w[kBatch * 4];
    int at[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; k++) {
      const int i = k0 + k * kStatThreads;
      at[k] = a + i * N;
      uint4 x = make_uint4(kLowest<T>, kLowest<T>, kLowest<T>, kLowest<T>);
      if (i < n) x = ldg_stream16(row + at[k]);
      w[4 * k] = x.x;
      w[4 * k + 1] = x.y;
      w[4 * k + 2] = x.z;
      w[4 * k + 3] = x.w;
    }
    f(w, at);
  }
  for (int i = b + threadIdx.x; i < hi; i += kStatThreads) one(i);
}
template <class T>
__device__ __forceinline__ float word_top(uint32_t w) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  else {
    const float2 v = unpack2<T>(w);
    return fmaxf(v.x, v.y);
  }
}

// Largest logit and sum of a thread's elements.  Quickly: the exponentials are
// 2^(x c - k), with k the whole number above the largest x c so far, so x c - k is
// rounded once, and the sum is brought to the largest logit at the end.  False where that
// does not do: a NaN (which makes the sum one), or x c that no longer has a fraction.
template <class T>
__device__ __forceinline__ bool sum_up(const T *x, int lo, int hi, float c, float &m, float &sum) {
  float k = -INFINITY;
  m = -INFINITY;
  sum = 0.0f;
  const pair_t c2 = pair(c, c);
  each_batch(x, lo, hi, [&](uint32_t (&w)[kBatch * 4], const int (&)[kBatch]) {
    uint32_t top = word_max<T>(w[0], kLowest<T>);
#pragma unroll
    for (int e = 1; e < kBatch * 4; e++) top = word_max<T>(top, w[e]);
    const float most = word_top<T>(top);
    if (most > m) {
      m = most;
      const float next = ceilf(m * c);
      sum *= exp2_fast(k - next);  // (k = -inf: the sum is 0)
      k = next;
    }
    if (m == -INFINITY) return;
    const pair_t less = pair(-k, -k);
    pair_t part[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < kBatch * 4; e += sizeof(T) / 2) {
      float2 v;
      if constexpr (sizeof(T) == 4) v = make_float2(__uint_as_float(w[e]), __uint_as_float(w[e + 1]));
      else v = unpack2<T>(w[e]);
      float y, z;
      unpair(fma2(pair(v.x, v.y), c2, less), y, z);
      part[e / 2 % 2] = add2(part[e / 2 % 2], pair(exp2_fast(y), exp2_fast(z)));
    }
    float y, z;
    unpair(add2(part[0], part[1]), y, z);
    sum += y + z;
  });
  if (m == -INFINITY || m == INFINITY) return true;
  sum *= exp2f(fmaf(-m, c, k));
  return sum == sum && fabsf(k) < 4194304.0f;
}
// The same for any logits: NaNs passed over, exponents of differences.
template <class T>
__device__ __noinline__ void sum_up_any(const T *x, int lo, int hi, float c, float &m_out, float &sum_out) {
  float m = -INFINITY, sum = 0.0f;
  for (int i = lo + threadIdx.x; i < hi; i += kStatThreads) {
    const float v = fmaxf(logit(x + i), -INFINITY);
    if (v > m) {
      sum *= exp2f((m - v) * c);
      m = v;
    }
    if (v > -INFINITY) sum += exp2f((v - m) * c);
  }
  m_out = m;
  sum_out = sum;
}

// One piece of one row, target's or draft's: its largest logit with, of warm rows,
// the sum of the exponentials relative to it, of cold ones the first index of it.
// One pass: the logits are read once, 84 MB (f32, 32 sequences of up to five rows) in 22
// us and 102 MB (bf16) in 29; memory alone would take 13 and 16, the exponentials (one of
// the special-function units' results for each logit) 5 and 11.
template <class T>
__global__ void __launch_bounds__(kStatThreads) k_verify_stats(const __grid_constant__ VerifyParams p) {
  __shared__ float red_m[kStatThreads / 32], red_s[kStatThreads / 32];
  __shared__ int red_i[kStatThreads / 32];
  pdl_wait();
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
  if (threadIdx.x == 0 && chunk == 0 && row == beg && !draft) p.arrived[s] = 0;
  float m = -INFINITY, sum = 0.0f;
  int at = 0x7fffffff;
  if (is_cold(t)) {
    each_batch(x, lo, hi, [&](uint32_t (&w)[kBatch * 4], const int (&i)[kBatch]) {
#pragma unroll
      for (int k = 0; k < kBatch; k++) {
        uint32_t top = word_max<T>(w[4 * k], kLowest<T>);
#pragma unroll
        for (int e = 1; e < 4; e++) top = word_max<T>(top, w[4 * k + e]);
        const float most = word_top<T>(top);
        if (most < m || most == -INFINITY) continue;
        int first = 0x7fffffff;
#pragma unroll
        for (int e = 3; e >= 0; e--) {
          if constexpr (sizeof(T) == 4) {
            if (__uint_as_float(w[4 * k + e]) == most) first = i[k] + e;
          } else {
            const float2 v = unpack2<T>(w[4 * k + e]);
            if (v.y == most) first = i[k] + 2 * e + 1;
            if (v.x == most) first = i[k] + 2 * e;
          }
        }
        at = most > m ? first : min(at, first);
        m = most;
      }
    });
  } else {
    const float c = kLog2e / t;
    const bool done = sum_up(x, lo, hi, c, m, sum);
    if (__syncthreads_or(!done)) sum_up_any(x, lo, hi, c, m, sum);
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

// 2^y of kTogether numbers y <= 0 side by side (each is a chain of dependent
// operations): to the nearest 32nd in the exponent, whose power comes from a table, and
// the rest, at most 1/64, by its power series; the first term left out is (ln 2 / 64)^5
// / 5! = 1.2e-12 of the result.  0 for y below -1000, and for -inf and NaN.
// All lanes of a warp together: lane i holds the table's entry i.
constexpr int kTogether = 4;
__device__ __forceinline__ void exp2_64(double entry, double (&y)[kTogether]) {
  constexpr double series[5] = {1.0, 6.931471805599453e-01, 2.402265069591007e-01, 5.5504108664821576e-02,
                                9.618129107628477e-03};  // (ln 2)^k / k!
  double p[kTogether];
  int n[kTogether];
  bool some[kTogether];
#pragma unroll
  for (int i = 0; i < kTogether; i++) {
    some[i] = y[i] > -1000.0;
    y[i] = some[i] ? y[i] : 0.0;
    const double t = y[i] + 211106232532992.0;  // 1.5 * 2^47: the low word counts 32nds
    n[i] = __double2loint(t);
    y[i] -= t - 211106232532992.0;
    p[i] = series[4];
  }
#pragma unroll
  for (int k = 3; k >= 0; k--)
#pragma unroll
    for (int i = 0; i < kTogether; i++) p[i] = fma(p[i], y[i], series[k]);
#pragma unroll
  for (int i = 0; i < kTogether; i++) {
    p[i] *= __shfl_sync(0xffffffffu, entry, n[i]);  // (of the lane n % 32)
    y[i] = some[i] ? __hiloint2double(__double2hiint(p[i]) + (n[i] >> 5 << 20), __double2loint(p[i])) : 0.0;
  }
}

// An f32 number in 64 bits by its bits (integer operations, where the conversion would
// take the pipe of the 64-bit ones); zeros and subnormals become numbers of at most
// 2^-126, infinities 2^128, and a NaN is taken for -inf.
__device__ __forceinline__ double wide(float x) {
  const uint32_t u = __float_as_uint(fmaxf(x, -INFINITY));
  return __hiloint2double((int)((u & 0x80000000u) | (((u & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(u << 29));
}
// exp((x - m) / T) in 64 bits, as a power of two.
struct Weight {
  double m, c;
  __device__ __forceinline__ Weight() {}
  __device__ __forceinline__ Weight(float m, float t) : m(m), c(1.4426950408889634 / (double)t) {}
  __device__ __forceinline__ double power(float x) const { return (wide(x) - m) * c; }
  __device__ __forceinline__ double operator()(double entry, float x) const {
    double y[kTogether] = {power(x)};
    exp2_64(entry, y);
    return y[0];
  }
};

// What the row that emits draws from: p, or what of p is above q, each summed apart:
// the token's weight is p / zx - q / zy where that is positive.
template <class T>
struct Drawn {
  const T *x, *y;  // target's logits; the draft's, or null
  Weight wx, wy;
  double border;   // p > q where the exponents of the two differ by more than this
  int one;         // the token that the draft was sure of, or -1
  // Of the tokens at[] below `end`: p and q over their sums' scale, and whether they are
  // drawn from.
  __device__ __forceinline__ void get(double entry, const int (&at)[kTogether], int end, double (&px)[kTogether], double (&qx)[kTogether],
                                      bool (&in)[kTogether]) const {
    float a[kTogether], b[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; i++) {
      a[i] = at[i] < end ? logit(x + at[i]) : -INFINITY;
      b[i] = y && at[i] < end ? logit(y + at[i]) : -INFINITY;
    }
    double gap[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; i++) {
      px[i] = wx.power(a[i]);
      qx[i] = 0.0;
      gap[i] = px[i];
    }
    exp2_64(entry, px);
    if (y) {
#pragma unroll
      for (int i = 0; i < kTogether; i++) {
        qx[i] = wy.power(b[i]);
        gap[i] -= qx[i];
      }
      exp2_64(entry, qx);
    }
#pragma unroll
    for (int i = 0; i < kTogether; i++)
      in[i] = px[i] > 0.0 && (y ? qx[i] == 0.0 || gap[i] > border : at[i] != one);
  }
};

using PartSums = VerifySums;
// (Written by other blocks: past the first-level cache.)
__device__ __forceinline__ PartSums load_sums(const PartSums *p) {
  const double *const d = (const double *)p;
  return {__ldcg(d), __ldcg(d + 1), __ldcg(d + 2), __ldcg(d + 3)};
}
struct Choice {
  double ix, iy;  // 1 / sums
  double want;    // what the running sum has to exceed
  double before;  // the running sum ahead of the part
  int part;
  bool from_p, close;
};
// What of p = px ix is above q = qx iy; 0 where that is within their rounding.  (No product
// is left unrounded, so that it is 0 where the two are the same.)
__device__ __forceinline__ double above(double px, double ix, double qx, double iy) {
  const double p = __dmul_rn(px, ix), w = __dsub_rn(p, __dmul_rn(qx, iy));
  return w > 0x1p-36 * p ? w : 0.0;
}
// Where less than this of p is above q, the two may be nearly the same at nearly all tokens, and
// the border from sums in f32 (2^-20 of p at most is on its wrong side) does not do.
constexpr double kClose = 0x1p-10;
struct DrawShared {
  Choice choice;
  int stop;
  bool last;  // of the sequence's blocks
  RowStats target, draft;
};

// What of p is above q at the tokens [lo, hi), by one warp.
template <class T>
__device__ __noinline__ double sum_above(const T *x, const T *y, float m, float t, float my, float ty, int lo, int hi, double ix,
                                         double iy) {
  const int lane = threadIdx.x % 32;
  const double entry = exp2((double)lane / 32.0);
  Drawn<T> d;
  d.x = x;
  d.y = y;
  d.wx = Weight(m, t);
  d.wy = Weight(my, ty);
  d.border = 0.0;
  d.one = -1;
  double sum = 0.0;
  for (int i0 = lo; i0 < hi; i0 += 32 * kTogether) {
    double px[kTogether], qx[kTogether];
    bool in[kTogether];
    int at[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; i++) at[i] = i0 + 32 * i + lane;
    d.get(entry, at, hi, px, qx, in);
#pragma unroll
    for (int i = 0; i < kTogether; i++) sum += above(px[i], ix, qx[i], iy);
  }
  return warp_sum64(sum);
}

// Bound by instructions: a token of the drawn row costs some 40, a quarter of them
// in 64 bits.  128256 tokens of p and of q for each of 32 sequences take 19 us,
// finding the emitting row 6 before that, finding the token 6 behind it.  The sequence's last block goes on by itself: a cluster of 16 blocks that met for it held the
// SMs longer (64 sequences of 152064: the call 75 us, where it then was 67, and is 62).  A call
// with a sequence whose p and q are nearly the same (kClose) waits for one block's way through
// its row: 32 such sequences of 128256 tokens take 257 us where others take 55.
template <class T>
__global__ void __launch_bounds__(kDrawThreads, 4) k_verify_draw(const __grid_constant__ VerifyParams p, const int blocks) {
  constexpr int most_parts = kDrawBlocks * kDrawWarps;  // of the vocabulary, one a warp
  constexpr int kOfLane = most_parts / 32;           // parts that a lane looks at
  __shared__ DrawShared sh;
  __shared__ double slice[kDrawWarps], weight[most_parts];
  const int parts = blocks * kDrawWarps, s = blockIdx.x / blocks, rank = blockIdx.x - s * blocks;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  // (Read ahead of the wait: the first kernel's blocks have waited for whatever wrote these before
  // they let this one begin.  Without rows there is no first kernel, and they have no say.)
  int beg, end;
  seq_rows(p.q_start, p.n_rows, s, beg, end);
  const float t = temperature_of(p.temperature, s), td = temperature_of(p.draft_temperature, s);
  if (tid == 0) sh.stop = end - 1;
  const double entry = exp2((double)lane / 32.0);
  __syncthreads();
  pdl_wait();
  if (beg == end) {
    if (rank == 0 && tid == 0) {
      p.n_accepted[s] = 0;
      if (p.new_len) p.new_len[s] = p.kv_len[s];
    }
    return;
  }
  // Every block finds the row that emits: a warp for each draft.
  for (int r = beg + warp; r < end - 1; r += kDrawWarps) {
    if (r > __shfl_sync(0xffffffffu, *(volatile int *)&sh.stop, 0)) break;
    const int x = __ldg(p.tokens + r + 1);
    bool take = false;
    if (x >= 0 && x < p.vocab) {
      const RowStats a = row_stats(p, r, t);
      const float lx = logit((const T *)p.logits + r * p.stride + x);
      double px = 0.0, qx = 1.0;
      if (!a.none()) px = is_cold(t) ? (double)(a.at == x) : Weight(a.m, t)(entry, lx) / a.sum;
      if (p.draft) {
        const RowStats b = row_stats(p, p.n_rows + r, td);
        const float ly = logit((const T *)p.draft + r * p.draft_stride + x);
        if (!b.none()) qx = is_cold(td) ? (double)(b.at == x) : Weight(b.m, td)(entry, ly) / b.sum;
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
    Drawn<T> d;
    d.x = (const T *)p.logits + stop * p.stride;
    d.y = nullptr;
    d.wx = Weight(a.m, t);
    d.one = -1;
    if (!sure) {
      const int x = __ldg(p.tokens + stop + 1);
      if (p.draft && !sh.draft.none() && !is_cold(td)) {
        d.y = (const T *)p.draft + stop * p.draft_stride;
        d.wy = Weight(sh.draft.m, td);
        // (From the sums in f32: a token that falls on the wrong side has p and q within
        // 2^-20 of each other, and a weight of next to nothing.  Where that is all there is,
        // the weights are summed again, below.)
        d.border = (double)log2f(a.sum) - (double)log2f(sh.draft.sum);
      } else {
        d.one = p.draft && !sh.draft.none() ? sh.draft.at : x;
      }
    }
    // This warp's part of the vocabulary, a whole number of 32.
    const int per = (p.vocab + parts * 32 - 1) / (parts * 32) * 32;
    const int lo = (int)min((int64_t)p.vocab, (int64_t)(rank * kDrawWarps + warp) * per);
    const int hi = (int)min((int64_t)p.vocab, (int64_t)lo + per);
    PartSums mine = {0.0, 0.0, 0.0, 0.0};
    for (int i0 = lo; i0 < hi; i0 += 32 * kTogether) {
      double px[kTogether], qx[kTogether];
      bool in[kTogether];
      int at[kTogether];
#pragma unroll
      for (int i = 0; i < kTogether; i++) at[i] = i0 + 32 * i + lane;
      d.get(entry, at, hi, px, qx, in);
#pragma unroll
      for (int i = 0; i < kTogether; i++) {
        mine.zx += px[i];
        mine.px += in[i] ? px[i] : 0.0;
        if (d.y) {
          mine.zy += qx[i];
          mine.qx += in[i] ? qx[i] : 0.0;
        }
      }
    }
    mine.zx = warp_sum64(mine.zx);
    mine.px = warp_sum64(mine.px);
    if (d.y) {
      mine.zy = warp_sum64(mine.zy);
      mine.qx = warp_sum64(mine.qx);
    }
    // The sequence's last block to get here goes on with what all have found.
    if (lane == 0) p.parts[(int64_t)s * parts + rank * kDrawWarps + warp] = mine;
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      sh.last = atomicAdd(p.arrived + s, 1) == blocks - 1;
      __threadfence();
    }
    __syncthreads();
    if (!sh.last) return;
    const VerifySums *const all = p.parts + (int64_t)s * parts;
    int some = -1;  // the last token with any weight
    // The first turn takes the parts' weights from what the blocks have summed; the second, where p and q
    // are close (or the first has found no token), from the tokens' own.
    for (int turn = 0; turn < 2; turn++) {
      if (turn) {
        const double ix = sh.choice.ix, iy = sh.choice.iy;
        for (int part = warp; part < parts; part += kDrawWarps) {
          const int p_lo = (int)min((int64_t)p.vocab, (int64_t)part * per), p_hi = (int)min((int64_t)p.vocab, (int64_t)p_lo + per);
          const double sum = sum_above(d.x, d.y, a.m, t, sh.draft.m, td, p_lo, p_hi, ix, iy);
          if (lane == 0) weight[part] = sum;
        }
        __syncthreads();
      }
      // The first warp goes through the parts, kOfLane a lane: the part in which the
      // running sum first exceeds `want`, or the last one with any weight where
      // rounding (or a number that is not below 1) leaves none.
      if (warp == 0) {
        double w[kOfLane], sum = 0.0, ix, iy;
        if (turn == 0) {
          PartSums of[kOfLane];
          double zx = 0.0, zy = 0.0;
#pragma unroll
          for (int k = 0; k < kOfLane; k++) {
            of[k] = PartSums{0.0, 0.0, 0.0, 0.0};
            if (kOfLane * lane + k < parts) of[k] = load_sums(all + kOfLane * lane + k);
            zx += of[k].zx;
            zy += of[k].zy;
          }
          ix = 1.0 / warp_sum64(zx);
          iy = d.y ? 1.0 / warp_sum64(zy) : 0.0;
#pragma unroll
          for (int k = 0; k < kOfLane; k++) sum += w[k] = fmax(of[k].px * ix - of[k].qx * iy, 0.0);
        } else {
          ix = sh.choice.ix;
          iy = sh.choice.iy;
#pragma unroll
          for (int k = 0; k < kOfLane; k++) sum += w[k] = kOfLane * lane + k < parts ? weight[kOfLane * lane + k] : 0.0;
        }
        double total = warp_sum64(sum);
        const bool close = turn == 0 && d.y && total < kClose, from_p = !close && !(total > 0.0);
        if (from_p) {
          sum = 0.0;
#pragma unroll
          for (int k = 0; k < kOfLane; k++) sum += w[k] = kOfLane * lane + k < parts ? __ldcg(&all[kOfLane * lane + k].zx) * ix : 0.0;
          total = warp_sum64(sum);
        }
        const double want = (double)__ldg(p.uniform + end - 1) * total;
        double upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const double n = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += n;
        }
        double run = upto - sum, before = run;  // before: of this lane's first part past `want`, or its last one
        int over = 0x7fffffff, last = -1;
#pragma unroll
        for (int k = 0; k < kOfLane; k++) {
          if (w[k] > 0.0 && over == 0x7fffffff) {
            last = kOfLane * lane + k;
            before = run;
            if (run + w[k] > want) over = last;
          }
          run += w[k];
        }
        int chosen = __reduce_min_sync(0xffffffffu, over);
        if (chosen == 0x7fffffff) chosen = max(__reduce_max_sync(0xffffffffu, last), 0);
        before = __shfl_sync(0xffffffffu, before, chosen / kOfLane);
        if (lane == 0) sh.choice = Choice{ix, iy, want, before, chosen, from_p, close};
      }
      __syncthreads();
      if (sh.choice.close) continue;
      const double ix = sh.choice.ix, iy = sh.choice.iy, want = sh.choice.want;
      double before = sh.choice.before;
      const int chosen = sh.choice.part;
      const bool from_p = sh.choice.from_p;
      // The block goes through the part, kTogether tokens a lane at a time.
      const int c_lo = (int)min((int64_t)p.vocab, (int64_t)chosen * per), c_hi = (int)min((int64_t)p.vocab, (int64_t)c_lo + per);
      for (int base = c_lo; base < c_hi && token < 0; base += kDrawThreads * kTogether) {
        double px[kTogether], qx[kTogether], w[kTogether], sum = 0.0;
        bool in[kTogether];
        int at[kTogether];
        const int first = base + tid * kTogether;
#pragma unroll
        for (int e = 0; e < kTogether; e++) at[e] = first + e;
        d.get(entry, at, c_hi, px, qx, in);
#pragma unroll
        for (int e = 0; e < kTogether; e++) sum += w[e] = from_p ? px[e] * ix : turn || in[e] ? above(px[e], ix, qx[e], iy) : 0.0;
        // Sums up to this lane, of the warps, and up to this warp.
        double upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const double n = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += n;
        }
        __syncthreads();  // (the slices of the round before have been read)
        if (lane == 31) slice[warp] = upto;
        __syncthreads();
        double start = before;
        for (int k = 0; k < warp; k++) start += slice[k];
        for (int k = 0; k < kDrawWarps; k++) before += slice[k];
        start += upto - sum;
        int pick = 0x7fffffff, last = -1;
#pragma unroll
        for (int e = 0; e < kTogether; e++) {
          start += w[e];
          if (w[e] > 0.0) {
            last = first + e;
            if (start > want) pick = min(pick, first + e);
          }
        }
        if (tid == 0) {
          sh.stop = 0x7fffffff;
          sh.target.at = -1;
        }
        __syncthreads();
        pick = __reduce_min_sync(0xffffffffu, pick);
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) {
          if (pick != 0x7fffffff) atomicMin(&sh.stop, pick);
          atomicMax(&sh.target.at, last);
        }
        __syncthreads();
        if (sh.stop != 0x7fffffff) token = sh.stop;
        some = max(some, sh.target.at);
      }
      if (token >= 0 || some >= 0 || !d.y) break;
    }
    if (token < 0) token = some;
    writes = warp == 0;
  }
  if (!writes) return;
  for (int r = beg + lane; r < end; r += 32) p.out_tokens[r] = r < stop ? __ldg(p.tokens + r + 1) : r == stop ? token : -1;
  if (lane == 0) {
    p.n_accepted[s] = stop - beg;
    if (p.new_len) p.new_len[s] = p.kv_len[s] - (end - 1 - stop);
  }
}

// Blocks of a sequence: parts of 128 tokens a warp at least, and all blocks on the SMs
// at once, four on each, where that leaves one for a sequence (32 sequences of 128256
// f32 logits, 18 blocks each: the call takes 50 us; with 16 each 52).
int draw_blocks(size_t n_seqs, size_t vocab) {
  const size_t fit = 4 * kPagedSMs / std::max<size_t>(1, n_seqs), work = (vocab + kDrawWarps * 128 - 1) / (kDrawWarps * 128);
  return (int)std::max<size_t>(1, std::min<size_t>(kDrawBlocks, std::min(fit, work)));
}

template <class T>
void run(const VerifyParams &p, cudaStream_t s) {
  if (p.n_rows) {
    const int64_t blocks = (int64_t)p.n_rows * p.chunks * (p.draft ? 2 : 1);
    launch_beside(k_verify_stats<T>, blocks, kStatThreads, 0, s, p);
  }
  const int blocks = draw_blocks(p.n_seqs, p.vocab);
  launch_beside(k_verify_draw<T>, (int64_t)p.n_seqs * blocks, kDrawThreads, 0, s, p, blocks);
}

}  // namespace

int verify_chunks(size_t n_rows, size_t vocab) {
  // Pieces of 4096 logits at least, blocks enough for every SM several times over.
  const size_t most = std::max<size_t>(1, vocab / 4096), want = (size_t)kPagedSMs * 6 / n_rows + 1;
  return (int)std::min<size_t>(64, std::min(most, want));
}

size_t verify_workspace(size_t n_seqs, size_t n_rows, size_t vocab, VerifyParams *p, void *ws) {
  // Sums of the parts (whole 32 bytes first), the pieces of the rows, the counters.
  const size_t parts = n_seqs * (size_t)draw_blocks(n_seqs, vocab) * kDrawWarps * sizeof(VerifySums);
  const size_t pieces = 2 * n_rows * (n_rows ? (size_t)verify_chunks(n_rows, vocab) : 1) * sizeof(float2);
  if (p) {
    p->parts = (VerifySums *)ws;
    p->part = (float2 *)((char *)ws + parts);
    p->arrived = (int32_t *)((char *)ws + parts + pieces);
  }
  return n_rows ? parts + pieces + n_seqs * sizeof(int32_t) : 0;
}

void launch_verify_drafts(const VerifyParams &p, cudaStream_t s) {
  if (p.dtype == JAL_F32) run<float>(p, s);
  else if (p.dtype == JAL_F16) run<__half>(p, s);
  else run<__nv_bfloat16>(p, s);
}

}  // namespace jal
