// Beam search over a paged cache: the best continuations of each sequence's
// beams over the vocabulary, and the reordering of the beams' page tables.
#include <algorithm>

#include "common.hpp"
#include "paged_dev.cuh"

namespace jal {

namespace {

using namespace paged;

// Selection in two kernels.  Scores of one beam are in the order of its
// logits, so the k best of a row are found on the logits themselves: each
// block takes one chunk of a row, keeps its k best (logit, index) pairs and
// the chunk's maximum and sum of exponentials.  The second kernel joins the
// chunks: log-sum-exp of each row in 64 bits, the candidates' scores
// cum + (x - lse) in 64 bits, and the k best of the sequence.
constexpr int kSelThreads = 256;
constexpr int kSelPer = 32;                       // logits of a chunk per thread
constexpr int kSelChunk = kSelThreads * kSelPer;  // 8192
constexpr int kJoinThreads = 512;
constexpr int kMaxK = 64;

// A key whose unsigned order is (value descending -> larger first, then index
// ascending): NaN counts as -inf, and -0 as +0.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  if (x != x) x = -INFINITY;
  x += 0.0f;
  const uint32_t b = __float_as_uint(x);
  const uint32_t o = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((uint64_t)o << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return ~(uint32_t)key; }

struct ChunkHead {  // what a chunk leaves beside its k keys
  float top, sum;
};

template <class T>
__global__ void __launch_bounds__(kSelThreads) k_beam_chunk(const BeamParams p, uint64_t *keys, ChunkHead *heads) {
  __shared__ uint64_t best[kSelThreads];
  __shared__ uint64_t cand[kMaxK * kSelPer];
  __shared__ float red[2][kSelThreads / 32];
  __shared__ uint64_t floor_key;
  __shared__ int n_cand;
  pdl_trigger();
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const T *x = (const T *)p.logits + row * p.row_stride;
  const int v0 = chunk * kSelChunk;
  const float cum = p.cum[row];
  const bool dead = !(cum > -INFINITY && cum < INFINITY);
  uint64_t mine = 0;  // below every real key
  float v[kSelPer], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSelPer; i++) {
    const int at = v0 + i * kSelThreads + tid;
    v[i] = -INFINITY;
    if (at < p.vocab) {
      v[i] = load_as_f32(x, at, p.dtype);
      if (dead || v[i] != v[i]) v[i] = -INFINITY;
      mine = max(mine, key_of(v[i], at));
    }
    top = fmaxf(top, v[i]);
  }
  top = warp_max(top);
  if (tid % 32 == 0) red[0][tid / 32] = top;
  best[tid] = mine;
  if (tid == 0) { n_cand = 0; floor_key = 0; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; w++) top = fmaxf(top, red[0][w]);
  const float safe = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kSelPer; i++) sum += __expf(v[i] - safe);
  sum = warp_sum(sum);
  if (tid % 32 == 0) red[1][tid / 32] = sum;
  // The k-th largest of the threads' best keys: the k best keys of the chunk
  // are not below it, and only k threads hold such keys, at most kSelPer each.
  int above = 0;
  for (int i = 0; i < kSelThreads; i++) above += best[i] > mine;
  if (above == p.k - 1) floor_key = mine;
  __syncthreads();
  const uint64_t least = max(floor_key, (uint64_t)1);
  if (mine >= least) {
#pragma unroll
    for (int i = 0; i < kSelPer; i++) {
      const int at = v0 + i * kSelThreads + tid;
      if (at >= p.vocab) continue;
      const uint64_t key = key_of(v[i], at);
      if (key >= least) cand[atomicAdd(&n_cand, 1)] = key;
    }
  }
  __syncthreads();
  const int n = n_cand;
  uint64_t *out = keys + ((int64_t)row * p.chunks + chunk) * p.k;
  for (int i = tid; i < n; i += kSelThreads) {
    const uint64_t key = cand[i];
    int rank = 0;
    for (int j = 0; j < n; j++) rank += cand[j] > key;
    if (rank < p.k) out[rank] = key;
  }
  for (int i = tid; i < p.k; i += kSelThreads)
    if (i >= n) out[i] = 0;
  if (tid == 0) {
    float all = 0.0f;
    for (int w = 0; w < kSelThreads / 32; w++) all += red[1][w];
    heads[(int64_t)row * p.chunks + chunk] = {top, all};
  }
}

// (score, flat index): larger score first, then the lower index.
struct Cand {
  double score;
  int64_t at;
};
__device__ __forceinline__ bool ahead(const Cand &a, const Cand &b) {
  return a.score > b.score || (a.score == b.score && a.at < b.at);
}

__global__ void __launch_bounds__(kJoinThreads) k_beam_join(const BeamParams p, const uint64_t *keys,
                                                           const ChunkHead *heads, const int take) {
  extern __shared__ __align__(16) char smem_raw[];
  Cand *cand = (Cand *)smem_raw;               // [k * take]
  Cand *best = cand + (int64_t)p.k * take;     // [kJoinThreads]
  double *lse = (double *)(best + kJoinThreads);  // [n_beams]
  __shared__ int n_cand;
  __shared__ Cand floor_cand;
  pdl_wait();
  const int seq = blockIdx.x, tid = threadIdx.x;
  for (int b = tid / 32; b < p.n_beams; b += kJoinThreads / 32) {
    const ChunkHead *h = heads + ((int64_t)seq * p.n_beams + b) * p.chunks;
    float top = -INFINITY;
    for (int c = tid % 32; c < p.chunks; c += 32) top = fmaxf(top, h[c].top);
    top = warp_max(top);
    double sum = 0.0;
    if (top > -INFINITY && top < INFINITY)
      for (int c = tid % 32; c < p.chunks; c += 32) sum += exp((double)h[c].top - (double)top) * (double)h[c].sum;
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // no finite log-sum-exp (nothing but -inf, or a +inf): the beam is dead
    if (tid % 32 == 0) lse[b] = top > -INFINITY && top < INFINITY ? (double)top + log(sum) : INFINITY;
  }
  if (tid == 0) { n_cand = 0; floor_cand = {-INFINITY, INT64_MAX}; }
  __syncthreads();
  const int per_beam = p.chunks * p.k, total = p.n_beams * per_beam;
  auto get = [&](int i) -> Cand {
    const int b = i / per_beam, j = i % per_beam;
    const double l = lse[b];
    const double cum = p.cum[seq * p.n_beams + b];
    if (l == INFINITY || !(cum > -INFINITY && cum < INFINITY)) {
      // All of a dead beam's scores are -inf: in the order of the index.
      if (j >= min(p.k, p.vocab)) return {-INFINITY, INT64_MAX};
      return {-INFINITY, (int64_t)b * p.vocab + j};
    }
    const uint64_t key = keys[((int64_t)seq * p.n_beams + b) * per_beam + j];
    if (key == 0) return {-INFINITY, INT64_MAX};
    return {cum + ((double)value_of(key) - l), (int64_t)b * p.vocab + index_of(key)};
  };
  Cand mine = {-INFINITY, INT64_MAX};
  for (int i = tid; i < total; i += kJoinThreads) {
    const Cand c = get(i);
    if (ahead(c, mine)) mine = c;
  }
  best[tid] = mine;
  __syncthreads();
  int above = 0;
  for (int i = 0; i < kJoinThreads; i++) above += ahead(best[i], mine);
  if (above == p.k - 1 && mine.at != INT64_MAX) floor_cand = mine;
  __syncthreads();
  const Cand least = floor_cand;
  if (mine.at != INT64_MAX && !ahead(least, mine)) {
    for (int i = tid; i < total; i += kJoinThreads) {
      const Cand c = get(i);
      if (c.at != INT64_MAX && !ahead(least, c)) cand[atomicAdd(&n_cand, 1)] = c;
    }
  }
  __syncthreads();
  const int n = n_cand;
  for (int i = tid; i < n; i += kJoinThreads) {
    const Cand c = cand[i];
    int rank = 0;
    for (int j = 0; j < n; j++) rank += ahead(cand[j], c);
    if (rank < p.k) {
      const int64_t o = (int64_t)seq * p.k + rank;
      p.scores[o] = (float)c.score;
      p.parents[o] = (int32_t)(c.at / p.vocab);
      p.tokens[o] = (int32_t)(c.at % p.vocab);
    }
  }
}

// One block per (beam row, layer): the row's page list from its parent's, and
// this layer's copy of the unfinished page where the row needs its own.
constexpr int kReorderThreads = 256;

__global__ void __launch_bounds__(kReorderThreads) k_beam_reorder(const ReorderParams p, const int elem) {
  const int row = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x;
  const int seq = row / p.n_beams, beam = row % p.n_beams;
  const int32_t *parents = p.parents + (int64_t)seq * p.n_beams;
  const int parent = parents[beam];
  const PagedView &kv = p.kv;
  int32_t *out = p.new_table + (int64_t)row * kv.max_pages;
  if ((unsigned)parent >= (unsigned)p.n_beams) {  // no such beam: an empty row
    if (layer) return;
    for (int j = tid; j < kv.max_pages; j += kReorderThreads) out[j] = -1;
    if (tid == 0) p.new_len[row] = 0;
    return;
  }
  const int source = seq * p.n_beams + parent;
  const int32_t *old = kv.table + (int64_t)source * kv.max_pages;
  const int len = min(max(p.kv_len[source], 0), kv.cap);
  const int full = len / kv.page_size, fill = len - full * kv.page_size;
  bool heir = true;
  for (int j = 0; j < beam; j++) heir &= parents[j] != parent;
  const bool takes = !heir || fill == 0;
  if (layer == 0) {
    for (int j = tid; j < kv.max_pages; j += kReorderThreads)
      out[j] = j < full ? old[j] : j > full ? -1 : takes ? p.fresh[row] : old[j];
    if (tid == 0) p.new_len[row] = len;
  }
  if (!takes || fill == 0) return;
  const int from = old[full], to = p.fresh[row];
  if ((unsigned)from >= (unsigned)kv.n_pages || (unsigned)to >= (unsigned)kv.n_pages) return;
  const int chunks = kv.hd * elem / 16;  // 16-byte pieces of a slot's row
  const int total = kv.hkv * fill * chunks;
  for (int i = tid; i < 2 * total; i += kReorderThreads) {
    const bool is_v = i >= total;
    const int j = is_v ? i - total : i, c = j % chunks, slot = j / chunks % fill, head = j / chunks / fill;
    const int64_t at = layer * p.layer_stride + head * kv.head_stride + slot * kv.slot_stride;
    const char *src = (const char *)(is_v ? kv.v : kv.k) + (at + from * kv.page_stride) * elem + c * 16;
    char *dst = (char *)(is_v ? p.vw : p.kw) + (at + to * kv.page_stride) * elem + c * 16;
    *(uint4 *)dst = *(const uint4 *)src;
  }
}

int join_take(size_t n_beams, size_t chunks, size_t k) {
  return (int)((n_beams * chunks * k + kJoinThreads - 1) / kJoinThreads);
}
size_t join_smem(size_t n_beams, size_t chunks, size_t k) {
  return (k * join_take(n_beams, chunks, k) + kJoinThreads) * sizeof(Cand) + n_beams * sizeof(double);
}

}  // namespace

int beam_chunks(size_t, size_t vocab) { return (int)((vocab + kSelChunk - 1) / kSelChunk); }
bool beam_fits(size_t n_beams, size_t vocab, size_t k, size_t n_rows) {
  return join_smem(n_beams, (size_t)beam_chunks(n_rows, vocab), k) <= 200 * 1024;
}
size_t beam_workspace(size_t n_seqs, size_t n_beams, size_t vocab, size_t k) {
  const size_t chunks = n_seqs * n_beams * (size_t)beam_chunks(n_seqs * n_beams, vocab);
  return chunks * (k * sizeof(uint64_t) + sizeof(ChunkHead));
}

void launch_beam_select(const BeamParams &p, cudaStream_t s) {
  const int64_t rows = (int64_t)p.n_seqs * p.n_beams;
  uint64_t *keys = (uint64_t *)p.ws;
  ChunkHead *heads = (ChunkHead *)(keys + rows * p.chunks * p.k);
  const dim3 grid((unsigned)p.chunks, (unsigned)rows);
  if (p.dtype == JAL_F32) k_beam_chunk<float><<<grid, kSelThreads, 0, s>>>(p, keys, heads);
  else if (p.dtype == JAL_F16) k_beam_chunk<__half><<<grid, kSelThreads, 0, s>>>(p, keys, heads);
  else k_beam_chunk<__nv_bfloat16><<<grid, kSelThreads, 0, s>>>(p, keys, heads);
  JAL_CUDA(cudaGetLastError());
  const size_t smem = join_smem((size_t)p.n_beams, (size_t)p.chunks, (size_t)p.k);
  JAL_CUDA(cudaFuncSetAttribute(k_beam_join, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.n_seqs);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  JAL_CUDA(cudaLaunchKernelEx(&cfg, k_beam_join, p, (const uint64_t *)keys, (const ChunkHead *)heads,
                              join_take((size_t)p.n_beams, (size_t)p.chunks, (size_t)p.k)));
}

void launch_beam_reorder(const ReorderParams &p, cudaStream_t s) {
  const int elem = p.kv.dtype == JAL_F32 ? 4 : 2;
  k_beam_reorder<<<dim3((unsigned)(p.n_seqs * p.n_beams), (unsigned)p.n_layers), kReorderThreads, 0, s>>>(p, elem);
  JAL_CUDA(cudaGetLastError());
}

}  // namespace jal
