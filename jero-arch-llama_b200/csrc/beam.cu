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
// block takes one chunk of a row, keeps its k best (logit, index) pairs in
// order, and the chunk's maximum and sum of exponentials.  The second kernel
// joins them, a warp for each beam: log-sum-exp of the row from the chunks' f32
// sums in 64 bits, the chunks' lists merged from their heads, scores
// cum + ((x - top) - log sum) in 64 bits;
// then one warp merges the beams' lists.  One pass over the logits: 128 rows of
// 128256 f32 logits take 22 us, half the copy rate (45 us with a test and a branch for
// each logit, 176 us with 64-bit keys for each); the join takes 8 us, a chain of short
// steps.
constexpr int kSelThreads = 256, kSelBlocks = 4, kSelPer = 16;
constexpr int kMaxK = 64;
constexpr int kSelList = 1024;  // candidates that are ranked without a second threshold
constexpr int kJoinThreads = 512;
constexpr int kJoinLists = 4;   // chunk lists a lane merges at most: 128 chunks a row
constexpr int kMaxBeams = 256;  // eight lists a lane in the last merge
constexpr size_t kJoinSmem = 96 * 1024;

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

constexpr float kLog2e = 1.44269504f;
struct ChunkHead {  // what a chunk leaves beside its k keys: its largest logit, the sum of 2^((x - top) kLog2e)
  float top, sum;
};

// A block reads its chunk piece by piece, PER logits a thread, 16 bytes at a time
// where the rows are so aligned.  The first piece gives a threshold that k keys
// reach; from then on a thread only looks for a logit above it, which is rare,
// and keeps a running maximum and sum.
template <class T, int PER>
__global__ void __launch_bounds__(kSelThreads, kSelBlocks) k_beam_chunk(const BeamParams p, const int span, const bool wide,
                                                           uint64_t *keys, ChunkHead *heads) {
  constexpr int VEC = 16 / sizeof(T) < PER ? 16 / sizeof(T) : PER, kPiece = kSelThreads * PER;
  constexpr int kList = kMaxK * (PER + 1) > kSelList ? kMaxK * (PER + 1) : kSelList;
  __shared__ uint64_t list[kList];
  __shared__ uint64_t floors[kSelThreads / 32];
  __shared__ float2 sums[kSelThreads / 32];
  __shared__ int n_list;
  pdl_trigger();
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  uint64_t *const out = keys + ((int64_t)row * p.chunks + chunk) * p.k;
  ChunkHead *const head = heads + (int64_t)row * p.chunks + chunk;
  const float cum = p.cum[row];
  if (!(cum > -INFINITY && cum < INFINITY)) {  // a dead beam: nothing of it is looked at
    if (tid == 0) *head = {-INFINITY, 0.0f};
    return;
  }
  const T *const x = (const T *)p.logits + row * p.row_stride;
  const int begin = chunk * span, end = min(begin + span, p.vocab);
  auto place = [&](int piece, int i) { return piece + ((i / VEC) * kSelThreads + tid) * VEC + i % VEC; };
  float v[PER];
  auto load = [&](int piece) {
    if (wide && piece + kPiece <= end) {  // (one branch for all, so that the loads are on their way together)
#pragma unroll
      for (int i = 0; i < PER; i += VEC) {
        if constexpr (VEC == 8) {
          float w[8];
          load8(x + place(piece, i), w);
#pragma unroll
          for (int e = 0; e < 8; e++) v[i + e] = w[e];
        } else {
          const float4 w = *(const float4 *)(x + place(piece, i));
          v[i] = w.x; v[i + 1] = w.y; v[i + 2] = w.z; v[i + 3] = w.w;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const int at = place(piece, i);
        const float w = load_as_f32(x, min(at, end - 1), p.dtype);
        v[i] = at < end ? w : -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = fmaxf(v[i], -INFINITY);  // a NaN counts as -inf
  };
  // The best key of the thread's logits of a piece, the first of the largest;
  // 0, below every key, where it has none.
  auto best_of = [&](int piece, float top) -> uint64_t {
    uint64_t best = 0;
#pragma unroll
    for (int i = PER - 1; i >= 0; i--) {
      const int at = place(piece, i);
      if (at < end && v[i] == top) best = key_of(top, (uint32_t)at);
    }
    return best;
  };
  // The keys of the piece from `least` on into the list, as far as there is
  // room.  Few logits reach `bar`: a mask of them costs less than a test and a
  // branch for each, and the value is read again.
  auto collect = [&](int piece, uint64_t least, float bar, int room) {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) found |= v[i] >= bar ? 1u << i : 0u;
    while (found) {
      const int i = __ffs(found) - 1, at = place(piece, i);
      found &= found - 1;
      if (at >= end) continue;
      const uint64_t key = key_of(load_as_f32(x, at, p.dtype), (uint32_t)at);
      if (key < least) continue;
      const int n = atomicAdd(&n_list, 1);
      if (n < room) list[n] = key;
    }
  };
  // Sums of 2^((v - top) log2 e), with log2 e as it is in f32 throughout: the
  // quotient by the same number at the end makes that an error of 10^-8 of the
  // entropy.  The difference comes before the product: finite logits as low or
  // high as the type has them give 0 or -inf there, where a product of the
  // logit itself would overflow.
  float top = -INFINITY, ref = 0.0f, sum = 0.0f, bar = -INFINITY;  // ref: top, or 0 while there is none
  uint64_t least = 1;
  for (int piece = begin; piece < end; piece += kPiece) {
    load(piece);
    float mine = v[0];
#pragma unroll
    for (int i = 1; i < PER; i++) mine = fmaxf(mine, v[i]);
    if (mine > top) {
      sum *= exp2_fast((top - mine) * kLog2e);
      top = ref = mine;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) sum += exp2_fast((v[i] - ref) * kLog2e);
    if (piece == begin) {
      // At least k groups of threads: the least of the groups' best keys is
      // below k keys at least, so the k best are not below it.
      const int width = p.k <= 8 ? 32 : p.k <= 16 ? 16 : p.k <= 32 ? 8 : 4;
      uint64_t best = best_of(piece, mine);
      for (int o = 1; o < width; o <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
      for (int o = width; o < 32; o <<= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, o));
      if (lane == 0) floors[warp] = best;
      if (tid == 0) n_list = 0;
      __syncthreads();
      least = floors[0];
#pragma unroll
      for (int w = 1; w < kSelThreads / 32; w++) least = min(least, floors[w]);
      least = max(least, (uint64_t)1);
      bar = least == 1 ? -INFINITY : value_of(least);
      if (mine >= bar) collect(piece, least, bar, kSelList);
      if (begin + kPiece < end) {  // the exact threshold of the first piece for the others
        __syncthreads();
        const int n = n_list;
        if (n <= kSelThreads) {
          if (tid < n) {
            const uint64_t key = list[tid];
            int rank = 0;
            for (int j = 0; j < n; j++) rank += list[j] > key;
            if (rank == p.k - 1) floors[0] = key;
          }
          __syncthreads();
          if (n >= p.k) least = floors[0];
          bar = least == 1 ? -INFINITY : value_of(least);
        }
      }
    } else if (mine >= bar) {
      collect(piece, least, bar, kSelList);
    }
  }
  {
    const float all = warp_max(top);
    const float part = warp_sum(top == -INFINITY ? 0.0f : sum * exp2_fast((top - all) * kLog2e));
    if (lane == 0) sums[warp] = make_float2(all, part);
  }
  __syncthreads();
  int n = n_list;
  if (n > kSelList) {
    // Rows in order, or with many equal logits.  Piece by piece once more: the
    // k-th largest of the threads' best keys is a threshold that k threads
    // reach, with PER keys each at most; those and the k best so far are ranked.
    n = 0;
    for (int piece = begin; piece < end; piece += kPiece) {
      __syncthreads();
      const uint64_t kept = tid < min(n, p.k) ? out[tid] : 0;
      load(piece);
      float mine = v[0];
#pragma unroll
      for (int i = 1; i < PER; i++) mine = fmaxf(mine, v[i]);
      const uint64_t best = best_of(piece, mine);
      list[tid] = best;
      if (tid == 0) {
        n_list = 0;
        floors[0] = 1;
      }
      __syncthreads();
      int above = 0;
      for (int i = 0; i < kSelThreads; i++) above += list[i] > best;
      if (above == p.k - 1 && best) floors[0] = best;
      __syncthreads();
      least = floors[0];
      if (best >= least) collect(piece, least, -INFINITY, kList);
      if (kept) list[atomicAdd(&n_list, 1)] = kept;
      __syncthreads();
      n = n_list;
      for (int i = tid; i < n; i += kSelThreads) {
        const uint64_t key = list[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += list[j] > key;
        if (rank < p.k) out[rank] = key;
      }
      __threadfence_block();
    }
  } else {
    for (int i = tid; i < n; i += kSelThreads) {
      const uint64_t key = list[i];
      int rank = 0;
      for (int j = 0; j < n; j++) rank += list[j] > key;
      if (rank < p.k) out[rank] = key;
    }
  }
  for (int i = tid + n; i < p.k; i += kSelThreads) out[i] = 0;
  if (tid == 0) {
    float all = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kSelThreads / 32; w++) all = fmaxf(all, sums[w].x);
#pragma unroll
    for (int w = 0; w < kSelThreads / 32; w++)
      total += sums[w].x == -INFINITY ? 0.0f : sums[w].y * exp2_fast((sums[w].x - all) * kLog2e);
    *head = {all, total};
  }
}

// The largest of the lanes' 64-bit values.
__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return ((uint64_t)hi << 32) | lo;
}
// A key in the order of x.
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double score_of(uint64_t o) {
  return __longlong_as_double((long long)(o >> 63 ? o & 0x7FFFFFFFFFFFFFFFull : ~o));
}

__global__ void __launch_bounds__(kJoinThreads) k_beam_join(const BeamParams p, const uint64_t *keys,
                                                           const ChunkHead *heads, const bool staged) {
  extern __shared__ __align__(16) char smem_raw[];
  uint64_t *const order = (uint64_t *)smem_raw;                // [n_beams][k] scores, in the order of order_of
  int32_t *const token = (int32_t *)(order + p.n_beams * p.k);  // [n_beams][k]
  pdl_wait();
  pdl_trigger();
  const int seq = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int per_beam = p.chunks * p.k, each = min(p.k, p.vocab);
  uint64_t *const stage = (uint64_t *)(smem_raw + (((int64_t)p.n_beams * p.k * 12 + 15) & ~15)) + warp * per_beam;
  for (int b = warp; b < p.n_beams; b += kJoinThreads / 32) {
    const int row = seq * p.n_beams + b;
    const ChunkHead *const h = heads + (int64_t)row * p.chunks;
    const uint64_t *list = keys + (int64_t)row * per_beam;
    if (staged) {
      __syncwarp();
      for (int i = lane; i < per_beam; i += 32) stage[i] = list[i];
      __syncwarp();
      list = stage;
    }
    const double cum = p.cum[row];
    float top = -INFINITY;
    for (int c = lane; c < p.chunks; c += 32) top = fmaxf(top, h[c].top);
    top = warp_max(top);
    // No log-sum-exp: nothing but -inf, or a +inf among them.
    const bool dead = !(cum > -INFINITY && cum < INFINITY && top > -INFINITY && top < INFINITY);
    if (dead) {  // -inf throughout, in the order of the index
      for (int j = lane; j < each; j += 32) {
        order[b * p.k + j] = order_of(-INFINITY);
        token[b * p.k + j] = j;
      }
      continue;
    }
    double sum = 0.0;
    for (int c = lane; c < p.chunks; c += 32)
      if (h[c].top > -INFINITY) sum += exp2(((double)h[c].top - (double)top) * (double)kLog2e) * (double)h[c].sum;
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double lse = log2(sum) / (double)kLog2e;  // of the logits less the largest one
    uint64_t head[kJoinLists];
    int pos[kJoinLists];
#pragma unroll
    for (int i = 0; i < kJoinLists; i++) {
      const int c = lane + 32 * i;
      pos[i] = 0;
      head[i] = c < p.chunks ? list[c * p.k] : 0;
    }
    for (int j = 0; j < each; j++) {
      uint64_t mine = head[0];
#pragma unroll
      for (int i = 1; i < kJoinLists; i++) mine = max(mine, head[i]);
      const uint64_t best = warp_max64(mine);
      if (mine == best) {  // keys are distinct: one lane
#pragma unroll
        for (int i = 0; i < kJoinLists; i++)
          if (head[i] == best) {
            pos[i]++;
            head[i] = pos[i] < p.k ? list[(lane + 32 * i) * p.k + pos[i]] : 0;
          }
        order[b * p.k + j] = order_of(cum + (((double)value_of(best) - (double)top) - lse));
        token[b * p.k + j] = (int32_t)index_of(best);
      }
    }
  }
  __syncthreads();
  if (warp) return;
  // The beams' lists from their heads: the larger score, then the lower beam.
  constexpr int N = kMaxBeams / 32;
  int pos[N];
#pragma unroll
  for (int i = 0; i < N; i++) pos[i] = 0;
  for (int j = 0; j < p.k; j++) {
    uint64_t mine = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int b = lane + 32 * i;
      if (b >= p.n_beams || pos[i] >= each) continue;
      const uint64_t o = order[b * p.k + pos[i]];
      if (o > mine) {
        mine = o;
        at = i;
      }
    }
    const uint64_t best = warp_max64(mine);
    const int beam = (int)__reduce_min_sync(0xffffffffu, mine == best ? (uint32_t)(lane + 32 * at) : 0xffffffffu);
    if (mine == best && beam == lane + 32 * at) {
      int taken = 0;
#pragma unroll
      for (int i = 0; i < N; i++)
        if (i == at) taken = pos[i]++;
      const int64_t o = (int64_t)seq * p.k + j;
      p.scores[o] = (float)score_of(best);
      p.parents[o] = beam;
      p.tokens[o] = token[beam * p.k + taken];
    }
  }
}

// One block per (beam row, layer): the row's page list from its parent's, and
// this layer's copy of the unfinished page where the row needs its own.  Bound by
// reading and writing those pages once: 128 beams in 32 layers read 116 MB of DRAM
// (children of one parent share its page in L2) and write 243 MB in 69 us, 5.2 TB/s.
// (Bulk copies through shared memory took 73 us, eight layers a block 83 us.)
constexpr int kRowThreads = 256;

// One head's filled slots, by a warp; `dense`: they lie one after another.
__device__ __forceinline__ void copy_head(const char *src, char *dst, int fill, int chunks, int64_t slot_bytes,
                                          bool dense) {
  constexpr int kPieces = 4;
  const int total = fill * chunks, lane = threadIdx.x % 32;
  for (int i = lane; i < total; i += 32 * kPieces) {
    uint4 w[kPieces];
    int64_t o[kPieces];
#pragma unroll
    for (int e = 0; e < kPieces; e++) {
      const int k = i + 32 * e;
      o[e] = dense ? (int64_t)k * 16 : (int64_t)(k / chunks) * slot_bytes + (k % chunks) * 16;
      if (k < total) w[e] = *(const uint4 *)(src + o[e]);
    }
#pragma unroll
    for (int e = 0; e < kPieces; e++)
      if (i + 32 * e < total) *(uint4 *)(dst + o[e]) = w[e];
  }
}

__global__ void __launch_bounds__(kRowThreads) k_beam_reorder(const __grid_constant__ ReorderParams p, const int elem) {
  pdl_wait();  // (the parents may come from a selection just before)
  const int row = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x;
  const int seq = row / p.n_beams, beam = row % p.n_beams;
  const int32_t *parents = p.parents + (int64_t)seq * p.n_beams;
  const int parent = parents[beam];
  bool heir = true;
  for (int j = 0; j < beam; j++) heir &= parents[j] != parent;
  if (heir && layer) return;
  const PagedView &kv = p.kv;
  int32_t *out = p.new_table + (int64_t)row * kv.max_pages;
  if ((unsigned)parent >= (unsigned)p.n_beams) {  // no such beam: an empty row
    if (layer) return;
    for (int j = tid; j < kv.max_pages; j += kRowThreads) out[j] = -1;
    if (tid == 0) p.new_len[row] = 0;
    return;
  }
  const int source = seq * p.n_beams + parent, to = p.fresh[row];
  const int32_t *old = kv.table + (int64_t)source * kv.max_pages;
  const int len = min(max(p.kv_len[source], 0), kv.cap);
  const int full = len / kv.page_size, fill = len - full * kv.page_size;
  const int from = fill ? old[full] : -1;  // (a table that is full has no unfinished page)
  // A row that is not the first takes a page of its own; where the unfinished page
  // is missing there is nothing to copy, and its positions stay without one.
  const bool whole = fill == 0, takes = whole || (!heir && (unsigned)from < (unsigned)kv.n_pages);
  if (layer == 0) {
    for (int j = tid; j < kv.max_pages; j += kRowThreads)
      out[j] = j < full ? old[j] : j > full ? -1 : takes ? to : from;
    if (tid == 0) p.new_len[row] = len;
  }
  if (!takes || whole || (unsigned)to >= (unsigned)kv.n_pages) return;
  const int heads = 2 * kv.hkv;
  auto place = [&](int h, int page) {  // byte offset of head h (of K, then of V) in a page of this layer
    return (layer * p.layer_stride + (h >= kv.hkv ? h - kv.hkv : h) * kv.head_stride + page * kv.page_stride) * elem;
  };
  auto pool = [&](int h) { return (char *)(h >= kv.hkv ? p.vw : p.kw); };
  for (int h = tid / 32; h < heads; h += kRowThreads / 32)
    copy_head(pool(h) + place(h, from), pool(h) + place(h, to), fill, kv.hd * elem / 16, kv.slot_stride * elem,
              kv.slot_stride == kv.hd);
}

// How a selection is cut: logits a thread takes at a time, and blocks a row.
// kSelBlocks blocks run on an SM: one round of them where there are rows enough;
// few rows go to more and smaller blocks.
struct SelPlan {
  int per, chunks, span;
};
SelPlan sel_plan(size_t n_rows, size_t vocab) {
  SelPlan a;
  const size_t slots = kSelBlocks * (size_t)kPagedSMs, wide = (vocab + kSelThreads * kSelPer - 1) / (kSelThreads * kSelPer);
  a.per = n_rows * wide < slots / 2 ? 8 : kSelPer;
  const size_t pieces = (vocab + kSelThreads * a.per - 1) / (kSelThreads * a.per);
  const size_t wanted = std::max<size_t>(1, std::min<size_t>(pieces, slots / std::max<size_t>(1, n_rows)));
  const size_t chunks = std::min<size_t>(wanted, 32 * kJoinLists);
  a.span = (int)((((vocab + chunks - 1) / chunks) + 7) / 8 * 8);
  a.chunks = (int)((vocab + a.span - 1) / a.span);
  return a;
}
size_t join_lists(size_t n_beams, size_t k) { return (n_beams * k * 12 + 15) / 16 * 16; }
size_t join_stage(size_t chunks, size_t k) { return kJoinThreads / 32 * chunks * k * sizeof(uint64_t); }

template <class T>
void run_chunks(const BeamParams &p, uint64_t *keys, ChunkHead *heads, cudaStream_t s) {
  const size_t rows = (size_t)p.n_seqs * p.n_beams;
  const bool wide = (uintptr_t)p.logits % 16 == 0 && p.row_stride * sizeof(T) % 16 == 0;
  const dim3 grid((unsigned)p.chunks, (unsigned)rows);
  const SelPlan a = sel_plan(rows, (size_t)p.vocab);
  if (a.per == 8) k_beam_chunk<T, 8><<<grid, kSelThreads, 0, s>>>(p, a.span, wide, keys, heads);
  else k_beam_chunk<T, kSelPer><<<grid, kSelThreads, 0, s>>>(p, a.span, wide, keys, heads);
  JAL_CUDA(cudaGetLastError());
}

}  // namespace

int beam_chunks(size_t n_rows, size_t vocab) { return sel_plan(n_rows, vocab).chunks; }
bool beam_fits(size_t n_beams, size_t vocab, size_t k) {
  return vocab <= (1u << 20) && n_beams <= (size_t)kMaxBeams && join_lists(n_beams, k) <= kJoinSmem;
}
size_t beam_workspace(size_t n_seqs, size_t n_beams, size_t vocab, size_t k) {
  const size_t chunks = n_seqs * n_beams * (size_t)beam_chunks(n_seqs * n_beams, vocab);
  return chunks * (k * sizeof(uint64_t) + sizeof(ChunkHead));
}

void launch_beam_select(const BeamParams &p, cudaStream_t s) {
  const int64_t rows = (int64_t)p.n_seqs * p.n_beams;
  uint64_t *keys = (uint64_t *)p.ws;
  ChunkHead *heads = (ChunkHead *)(keys + rows * p.chunks * p.k);
  if (p.dtype == JAL_F32) run_chunks<float>(p, keys, heads, s);
  else if (p.dtype == JAL_F16) run_chunks<__half>(p, keys, heads, s);
  else run_chunks<__nv_bfloat16>(p, keys, heads, s);
  const size_t lists = join_lists((size_t)p.n_beams, (size_t)p.k), stage = join_stage((size_t)p.chunks, (size_t)p.k);
  const bool staged = lists + stage <= kJoinSmem;
  const size_t smem = lists + (staged ? stage : 0);
  JAL_CUDA(cudaFuncSetAttribute(k_beam_join, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kJoinSmem));
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
  JAL_CUDA(cudaLaunchKernelEx(&cfg, k_beam_join, p, (const uint64_t *)keys, (const ChunkHead *)heads, staged));
}

void launch_beam_reorder(const ReorderParams &p, cudaStream_t s) {
  const int elem = p.kv.dtype == JAL_F32 ? 4 : 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.n_seqs * p.n_beams), (unsigned)p.n_layers);
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  JAL_CUDA(cudaLaunchKernelEx(&cfg, k_beam_reorder, p, elem));
}

}  // namespace jal
