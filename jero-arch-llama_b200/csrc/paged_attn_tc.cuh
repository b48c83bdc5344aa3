// Attention of many query rows over a 16-bit paged cache on the tcgen05 tensor
// cores.  Included by paged_attn.cu.
//
// A block takes 256 query rows of one KV head as two tiles of 128 and runs
// over its keys in tiles of 128: S = Q K^T into tensor memory, softmax weights
// P in registers (two threads a row), P back into tensor memory over S, and
// O += P V with O in tensor memory.  The two row tiles take turns: while the
// tensor cores work on one, a warpgroup forms the weights of the other, so a
// K and a V tile are read once for 256 rows.  Per key tile the tensor cores
// need 4 x 128 x 128 x HD products and the special-function units 2 x 128 x
// 128 exponentials, 2048 cycles each at HD = 128.  What bounds the kernel is how
// these follow one another: a key tile takes about 4400 cycles (scores, weights,
// products, and the waits between the warps that make them; without the exponentials
// it takes 8% less), and a block's start (rows, table, first K tile) and end 10000 and
// 5500 more.  Ragged prompts behind a 1024-position window, 159 GFLOP: 239 to 254 us
// by the box, 0.62 to 0.66 PFLOP/s, with the tensor cores busy for 35% of the time.
// (A quarter or half of the exponentials as polynomials on the multiply-add units: 5 to 20 us slower.  Seven
// loader warps, one softmax warpgroup a row tile, or the query rows asked for before the
// first barrier: no faster.)
//
//   warps 0-15       softmax: four warpgroups, two for each row tile, each with
//                    64 of the tile's 128 keys (warp w reads tensor-memory lanes
//                    32 (w % 4) ..), and the result.  One thread for a row's half:
//                    one warp of a tile on a scheduler cannot hide its own
//                    latencies
//   warps 16-18      K and V rows from their pages into the ring, cp.async
//   warp 19          one thread issues the products
//
// Pages may hold any number of slots, so rows are copied one by one to their
// place in the 128-byte swizzle that the matrix descriptors name: K tiles and
// V tiles are both [HD / 64][128 keys][64 dims], K read as K-major and V as
// MN-major.
//
// The running maximum that the weights refer to is only raised when a row's
// maximum grows by more than 2^kTcSlack, so that O is rescaled rarely.  f32 rows
// (NS = 2, f16 cache) are split like in the mma.sync kernel: two f16 parts of q
// and of the weights.  f16 weights refer to less than the maximum, as there; slack
// and headroom share f16's range.
#pragma once

#include "paged_attn_mma.cuh"
#include "paged_dev.cuh"

namespace jal {
namespace paged {

constexpr int kTcRows = 256, kTcKeys = 128, kTcThreads = 640;
constexpr int kTcSoftmax = 512, kTcLoaders = 3;  // threads; warps
// Growth of a maximum (base 2) that is let stand, and how far below the maximum
// the weights' reference lies.  f16 weights reach 2^15 with them, and each is off by
// 2^-36 of the row's largest weight beside its relative error.  Measured with f16
// rows and scores of a few units, 1024-position window: slack 4 or 8 241 us, 2 260
// us, 1 262 us (O is rescaled in most tiles).
template <class T>
constexpr int kTcSlack = std::is_same<T, __half>::value ? 4 : 8;
template <class T>
constexpr int kTcHeadroom = std::is_same<T, __half>::value ? 11 : 0;

struct TcSync {
  uint64_t q_full, loaded;
  uint64_t kv_full[6], kv_empty[6];
  uint64_t present_full[8];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint32_t tmem;
  int given_up, poison;
  int lim_lo, wlo_lo, wlo_hi;  // of the tile's rows: the least end, the least and largest window start
  // Of a row's halves: the largest score of the key tile, and at the end the sum
  // of the weights.  Before the first tile: what a row's scores are still to be
  // multiplied by (NS = 2, [256]).  Barriers lie between these uses.
  float x[2][2][128];
  float m1[128];  // at the end: what the weights of the second row tile refer to
  alignas(16) uint8_t present[8][16];    // which keys of tile j exist, a bit each, by j % 8
};

template <int NS, int HD>
struct TcShape {
  static constexpr int tile = kTcKeys * HD * 2;            // bytes of a K or V tile
  static constexpr int q_tile = 128 * HD * 2;              // of one part of a row tile
  static constexpr int buffers = HD == 64 ? 6 : NS == 1 ? 5 : 3;
  // The query tiles; at the end 4 KB for each softmax warp.
  static constexpr int q_area = 2 * NS * q_tile > 65536 ? 2 * NS * q_tile : 65536;
  static constexpr int ring = q_area, sync = q_area + buffers * tile, smem = sync + (int)sizeof(TcSync);
};

// ---- pairs of f32 in one instruction
using pair_t = unsigned long long;
__device__ __forceinline__ pair_t pair(float a, float b) {
  pair_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void unpair(pair_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
  pair_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
  pair_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float v;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// ---- tcgen05 ----------------------------------------------------------------
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t lead_bytes, uint32_t stride_bytes) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lead_bytes >> 4) << 16) | ((uint64_t)(stride_bytes >> 4) << 32) |
         (1ull << 46) | (2ull << 61);  // version 1, 128-byte swizzle
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// Arrives on `bar` when every product this thread has issued so far is done.
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#define JAL_R8(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3]), "=r"((r)[i + 4]), \
                     "=r"((r)[i + 5]), "=r"((r)[i + 6]), "=r"((r)[i + 7])
#define JAL_I8(r, i) "r"((r)[i]), "r"((r)[i + 1]), "r"((r)[i + 2]), "r"((r)[i + 3]), "r"((r)[i + 4]), \
                     "r"((r)[i + 5]), "r"((r)[i + 6]), "r"((r)[i + 7])
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];"
      : JAL_R8(r, 0), JAL_R8(r, 8), JAL_R8(r, 16), JAL_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31};" ::JAL_I8(r, 0),
      JAL_I8(r, 8), JAL_I8(r, 16), JAL_I8(r, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::JAL_I8(r, 0),
      JAL_I8(r, 8), "r"(addr)
      : "memory");
}
#undef JAL_R8
#undef JAL_I8


static_assert(TcShape<1, 128>::smem <= 232448 && TcShape<2, 128>::smem <= 232448, "shared memory of a block");

template <class T, int NS, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) k_paged_attn_tc(const __grid_constant__ AttnParams p, const int part, const bool direct) {
  using S = TcShape<NS, HD>;
  extern __shared__ __align__(1024) char smem_tc[];
  TcSync &sy = *(TcSync *)(smem_tc + S::sync);
  pdl_trigger();
  Tile t;
  if (!block_tile(p, part, kTcRows, kTcKeys, t)) return;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, hd = p.kv.hd;
  char *const base_p = smem_tc;
  const uint32_t sq = smem_u32(smem_tc), ring = sq + S::ring;
  const int n_tiles = (t.u1 - t.u0 + kTcKeys - 1) / kTcKeys;
  // At most 128 rows: both row tiles hold them, the first takes the even key
  // tiles and the second the odd ones, and their results are joined.
  const bool twice = t.rows <= 128;

  // Loader: the 16 groups of 8 rows of a tile go round the warps; a lane looks up
  // two of its warp's (up to) 48 rows, one tile ahead, the first before anything else.
  const int w = warp - 16;
  constexpr int kGroups = (16 + kTcLoaders - 1) / kTcLoaders;
  auto group = [&](int k) { return w + k * kTcLoaders; };
  auto locate = [&](int j, int k) -> Slot {
    const int gr = group(k + lane / 8), u = t.u0 + j * kTcKeys + gr * 8 + lane % 8;
    return j < n_tiles && k + lane / 8 < kGroups && gr < 16 && u < t.u1 ? slot_of(p.kv, t, t.key(u)) : Slot{-1, 0};
  };
  Slot next0 = {-1, 0}, next1 = {-1, 0};
  if (warp >= 16 && warp < 16 + kTcLoaders) {
    next0 = locate(0, 0);
    next1 = locate(0, 4);
  }

  if (tid == 0) {
    mbar_init(&sy.q_full, kTcSoftmax);
    mbar_init(&sy.loaded, kTcLoaders * 32);
    for (int i = 0; i < S::buffers; i++) {
      mbar_init(&sy.kv_full[i], kTcLoaders * 32);
      mbar_init(&sy.kv_empty[i], 1);
    }
    for (int i = 0; i < 8; i++) mbar_init(&sy.present_full[i], kTcLoaders);
    for (int i = 0; i < 2; i++) {
      mbar_init(&sy.s_full[i], 1);
      mbar_init(&sy.p_full[i], 256);
      mbar_init(&sy.o_full[i], 1);
    }
    sy.given_up = sy.poison = 0;
    sy.lim_lo = sy.wlo_lo = 0x7fffffff;
    sy.wlo_hi = 0;
    fence_barrier_init();
  }
  if (warp == 19) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sy.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sy.tmem;
  // A wait that gives up (it cannot, unless the code is wrong) sends the
  // block's rows to attend_row_alone instead of hanging the GPU.
  volatile int *given_up = &sy.given_up;
  auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    if (!*given_up && mbar_wait_bounded(bar, parity)) return true;
    *given_up = 1;
    return false;
  };

  // 640 threads of 96 registers: 512 x 104 + 128 x 64.
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp < 16 + kTcLoaders) {
      // ---- the loader
      // Eight lanes copy 128 bytes of a row; a lane has rows lane / 8 and lane / 8
      // + 4 of each group.  Their addresses are passed round once for K and V.
      const int c8 = lane % 8, r8 = lane / 8;
      const uint32_t to0 = r8 * 128 + ((c8 ^ r8) * 16), to1 = (r8 + 4) * 128 + ((c8 ^ (r8 + 4)) * 16);
      // Copies arrive on the buffer's barrier by themselves; the thread that
      // issues the products puts the fence between them and the tensor cores.
      uint32_t bad = 0;
      bool ok = true, ranges = false;
      int b = 0, parity = 1;  // of the buffer's "empty" phase before this use: the first use finds it free
      auto copy = [&](const void *pool_v, const int64_t (&from)[kGroups][2]) {
        ok = __all_sync(0xffffffffu, ok && wait(&sy.kv_empty[b], parity));
        if (!ok) return;
        const char *const pool = (const char *)pool_v + c8 * 16;
        const uint32_t dst = ring + b * S::tile;
#pragma unroll
        for (int k = 0; k < kGroups; k++) {
          if (group(k) >= 16) break;
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const char *const src = pool + from[k][e] * 2;
            const uint32_t to = dst + group(k) * 1024 + (e ? to1 : to0);
#pragma unroll
            for (int h = 0; h < HD / 64; h++) {
              const bool there = from[k][e] >= 0 && h * 64 + c8 * 8 < hd;
              copy16(to + h * (kTcKeys * 128), there ? src + h * 128 : (const char *)pool_v, there);
            }
          }
        }
        copies_done();
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&sy.kv_full[b])) : "memory");
        if (++b == S::buffers) {
          b = 0;
          parity ^= 1;
        }
      };
      // Looks through the V tile in buffer vb for values that some queries must not meet.
      auto scan = [&](int vb) {
        const char *const rows = base_p + S::ring + vb * S::tile;
#pragma unroll
        for (int k = 0; k < kGroups; k++)  // the rows that this warp has copied
#pragma unroll
          for (int h = 0; h < HD / 64 * 2; h++)
            if (group(k) < 16)
              watch8<T>(bad, *(const uint4 *)(rows + (h / 2) * (kTcKeys * 128) + group(k) * 1024 + (h % 2) * 512 + lane * 16));
      };
      int scan_b = -1;
#pragma unroll 1
      for (int j = 0; j < n_tiles; j++) {
        const int64_t at0 = slot_offset(p.kv, next0, t.head), at1 = slot_offset(p.kv, next1, t.head);
        const uint32_t bits0 = __ballot_sync(0xffffffffu, at0 >= 0), bits1 = __ballot_sync(0xffffffffu, at1 >= 0);
        next0 = locate(j + 1, 0);
        next1 = locate(j + 1, 4);
        int64_t from[kGroups][2];
#pragma unroll
        for (int k = 0; k < kGroups; k++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            from[k][e] = __shfl_sync(0xffffffffu, k < 4 ? at0 : at1, (k % 4) * 8 + r8 + 4 * e);
        if (lane < kGroups && group(lane) < 16)  // tile j + 8 comes long after the softmax has read tile j's
          sy.present[j & 7][group(lane)] = (uint8_t)((lane < 4 ? bits0 : bits1) >> (lane % 4 * 8));
        __syncwarp();
        if (lane == 0) mbar_arrive(&sy.present_full[j & 7]);
        copy(p.kv.k, from);
        const int vb = b;
        copy(p.kv.v, from);
        if (!ok) break;
        if (scan_b >= 0) {  // the tile before; its buffer is not filled again before the next round
          copies_wait<2>();
          __syncwarp();
          scan(scan_b);
        }
        if (!ranges) {
          ok = __all_sync(0xffffffffu, wait(&sy.q_full, 0));
          ranges = true;
        }
        const int u = t.u0 + j * kTcKeys, first = t.key(u), last = t.key(min(u + kTcKeys, t.u1) - 1);
        // (Rows of one window's start have no keys between the first positions and it.)
        const bool mixed = (first < sy.wlo_hi && sy.wlo_lo != sy.wlo_hi) || last >= sy.lim_lo;
        scan_b = mixed ? vb : -1;
      }
      copies_wait<0>();
      __syncwarp();
      if (scan_b >= 0) scan(scan_b);
      if (watched_bad<T>(bad)) sy.poison = 1;
      mbar_arrive(&sy.loaded);
    } else {
      // ---- the products: the whole warp runs the loop, so that addresses stay
      // uniform, and one lane issues
      const bool leader = elect_one();
      constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t id = (1u << 4) | (type << 7) | (type << 10) | ((128u >> 4) << 24);
      constexpr uint32_t id_s = id | ((kTcKeys >> 3) << 17), id_o = id | (1u << 16) | ((HD >> 3) << 17);
      const uint64_t q_desc = tc_desc(sq, 16, 1024), k_desc = tc_desc(ring, 16, 1024),
                     v_desc = tc_desc(ring, kTcKeys * 128, 1024);
      auto scores = [&](int i, int kb) {
        if (leader) {
          const uint64_t a = q_desc + (uint32_t)(i * NS * (S::q_tile >> 4)), b = k_desc + (uint32_t)(kb * (S::tile >> 4));
#pragma unroll
          for (int s = 0; s < NS; s++)
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
              const uint32_t off = ((k / 4) * (128 * 128) + (k % 4) * 32) >> 4;
              tc_mma_ss(tmem + i * 128, a + (uint32_t)(s * (S::q_tile >> 4) + off), b + off, id_s, s + k > 0);
            }
          tc_commit(&sy.s_full[i]);
        }
        __syncwarp();
      };
      auto output = [&](int i, int vb, bool first) {
        if (leader) {
          const uint64_t b = v_desc + (uint32_t)(vb * (S::tile >> 4));
#pragma unroll
          for (int s = 0; s < NS; s++)
#pragma unroll
            for (int k = 0; k < kTcKeys / 16; k++)
              tc_mma_ts(tmem + 256 + i * 128, tmem + i * 128 + (k / 4) * 64 + s * 32 + (k % 4) * 8,
                        b + (uint32_t)(k * (2048 >> 4)), id_o, !first || s + k > 0);
        }
        __syncwarp();
      };
      auto release = [&](int b) {
        if (leader) tc_commit(&sy.kv_empty[b]);
        __syncwarp();
      };
      // K tile j is copy 2 j, V tile j copy 2 j + 1; copies go round the buffers.
      auto there = [&](int g) {
        const bool ok = wait(&sy.kv_full[g % S::buffers], (g / S::buffers) & 1);
        fence_proxy_async();  // the rows were written by cp.async, the tensor cores read them by the async proxy
        tc_fence_after();
        return ok;
      };
      bool ok = n_tiles == 0 || wait(&sy.q_full, 0);
      if (twice) {
        for (int j = 0; j < min(n_tiles, 2) && ok; j++) {
          ok = there(2 * j);
          if (!ok) break;
          scores(j, (2 * j) % S::buffers);
          release((2 * j) % S::buffers);
        }
#pragma unroll 1
        for (int j = 0; j < n_tiles && ok; j++) {
          const int i = j & 1, v = 2 * j + 1, k = 2 * j + 4;
          ok = there(v) && wait(&sy.p_full[i], (j >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          output(i, v % S::buffers, j < 2);
          release(v % S::buffers);
          if (j + 2 < n_tiles) {
            ok = there(k);
            if (!ok) break;
            scores(i, k % S::buffers);
            release(k % S::buffers);
          } else {
            if (leader) tc_commit(&sy.o_full[i]);
            __syncwarp();
          }
        }
      } else {
        ok = ok && (n_tiles == 0 || there(0));
        if (ok && n_tiles) {
          scores(0, 0);
          scores(1, 0);
          release(0);
        }
#pragma unroll 1
        for (int j = 0; j < n_tiles && ok; j++) {
          const int v = 2 * j + 1, k = 2 * j + 2;
#pragma unroll
          for (int i = 0; i < 2; i++) {
            ok = ok && (i || there(v)) && wait(&sy.p_full[i], j & 1);
            if (!ok) break;
            tc_fence_after();
            output(i, v % S::buffers, j == 0);
            if (i) release(v % S::buffers);
            if (j + 1 < n_tiles) {
              ok = i || there(k);
              if (!ok) break;
              scores(i, k % S::buffers);
              if (i) release(k % S::buffers);
            } else {
              if (leader) tc_commit(&sy.o_full[i]);
              __syncwarp();
            }
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---- softmax: threads r of the warpgroups 2 i and 2 i + 1 have row r of row tile i
    const int i = warp / 8, half = warp / 4 % 2, r = tid % 128, base = twice ? 0 : i * 128, row = base + r;
    const bool real = row < t.rows;
    const RowMask mk = real ? row_mask(p, t, row) : RowMask{0, 0};
    // Weights are formed with a positive factor: a negative one turns q round,
    // none makes it 0.
    float scale = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
    auto tile_sync = [&]() { asm volatile("bar.sync %0, 256;" ::"r"(1 + i) : "memory"); };
    {  // the query rows into shared memory, 16 rows a warp, neighbouring lanes neighbouring pieces
      const int first = warp % 8 * 16;  // of the row tile
      char *const dst = base_p + i * NS * S::q_tile;
      const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
      const int mine = base + first + lane % 16;
      const int64_t qt = mine < t.rows && p.scale_log2 != 0.0f ? q_offset(p, t, mine) : -1;
      constexpr int CH = HD / 8;
      if constexpr (NS == 1) {
        const int c8 = lane % 8, r8 = lane / 8;
        uint4 w[4][HD / 64];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int64_t o = __shfl_sync(0xffffffffu, qt, r8 + 4 * k);
#pragma unroll
          for (int h = 0; h < HD / 64; h++)
            w[k][h] = o >= 0 && h * 64 + c8 * 8 < hd ? *(const uint4 *)((const T *)p.q + o + h * 64 + c8 * 8)
                                                     : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
          for (int h = 0; h < HD / 64; h++) {
            const int kr = first + r8 + 4 * k;
            const uint4 x = w[k][h];
            *(uint4 *)(dst + h * (128 * 128) + kr * 128 + ((c8 ^ (kr & 7)) * 16)) =
                make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
          }
      } else {
#pragma unroll 2
        for (int k = 0; k < CH / 2; k++) {
          const int kr = (k * 32 + lane) / CH, c = lane % CH;
          const int64_t o = __shfl_sync(0xffffffffu, qt, kr);
          float v[8] = {}, top = 0.0f;
          if (o >= 0 && c * 8 < hd) load8((const float *)p.q + o + c * 8, v);
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (fabsf(v[e]) < INFINITY) top = fmaxf(top, fabsf(v[e]));
#pragma unroll
          for (int x = CH / 2; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          const int e = top > 0.0f ? 13 - ilogbf(top) : 0;
          const float a = (flip ? -1.0f : 1.0f) * exp2f((float)(e / 2)), b = exp2f((float)(e - e / 2));
          uint32_t part2[4][NS];
#pragma unroll
          for (int q = 0; q < 4; q++) split2<T, NS>(v[2 * q] * a * b, v[2 * q + 1] * a * b, part2[q]);
#pragma unroll
          for (int s = 0; s < NS; s++)
            *(uint4 *)(dst + s * S::q_tile + (c / 8) * (128 * 128) + (first + kr) * 128 + (((c % 8) ^ (kr & 7)) * 16)) =
                make_uint4(part2[0][s], part2[1][s], part2[2][s], part2[3][s]);
          if (c == 0) (&sy.x[0][0][0])[i * 128 + first + kr] = (1.0f / fabsf(a)) / b;
        }
        tile_sync();
        scale *= (&sy.x[0][0][0])[i * 128 + r];
      }
      int lo = real ? mk.lim : 0x7fffffff, wl = real ? mk.wlo : 0x7fffffff, wh = real ? mk.wlo : 0;
      lo = __reduce_min_sync(0xffffffffu, lo);
      wl = __reduce_min_sync(0xffffffffu, wl);
      wh = __reduce_max_sync(0xffffffffu, wh);
      if (lane == 0) {
        atomicMin(&sy.lim_lo, lo);
        atomicMin(&sy.wlo_lo, wl);
        atomicMax(&sy.wlo_hi, wh);
      }
      fence_proxy_async();
      mbar_arrive(&sy.q_full);
    }
    const uint32_t quarter = (uint32_t)(warp % 4) << 21;  // lane 32 (warp % 4) of the tensor memory
    const uint32_t ts = tmem + i * 128 + half * 64 + quarter, to = tmem + 256 + i * 128 + quarter;
    const RowSpan span = row_span(p, t, mk);
    float m = -INFINITY, l = 0.0f;  // m: what the weights refer to, scaled to base 2; l: this half's sum
    bool ok = true;
    int turn = 0;  // of this row tile
#pragma unroll 1
    for (int j = twice ? i : 0; j < n_tiles; j += twice ? 2 : 1, turn++) {
      // (A wait that gave up does not leave the loop: the other half waits below.)
      ok = wait(&sy.present_full[j & 7], (j >> 3) & 1) && ok;
      ok = wait(&sy.s_full[i], turn & 1) && ok;
      __syncwarp();
      tc_fence_after();
      float s[2][32];
      tc_ld32(ts, (uint32_t *)s[0]);
      tc_ld32(ts + 32, (uint32_t *)s[1]);
      const int u = t.u0 + j * kTcKeys + half * 64;
      const uint2 here = *(const uint2 *)&sy.present[j & 7][half * 8];
      const bool whole = (here.x & here.y) == 0xffffffffu && span.all(u, 64);
      const bool masked = !__all_sync(0xffffffffu, whole || !real);
      tc_wait_ld();
      if (masked) {
        const uint32_t bits[2] = {here.x & span.bits(u), here.y & span.bits(u + 32)};
#pragma unroll
        for (int e = 0; e < 64; e++)
          if (!((bits[e / 32] >> (e % 32)) & 1)) s[e / 32][e % 32] = -INFINITY;
      }
      float x[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
      for (int e = 4; e < 60; e += 8)
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = max3_nan(x[k], s[(e + 2 * k) / 32][(e + 2 * k) % 32], s[(e + 2 * k + 1) / 32][(e + 2 * k + 1) % 32]);
      const float mine = max3_nan(max3_nan(x[0], x[1], s[1][28]), max3_nan(x[2], x[3], s[1][29]),
                                  max3_nan(s[1][30], s[1][31], s[1][31]));
      sy.x[i][half][r] = mine;
      tile_sync();
      const float top = max3_nan(mine, sy.x[i][half ^ 1][r], mine) * scale;
      // A NaN or an infinite score makes the row NaN, as the formula does.
      if (!(top < INFINITY)) l = NAN;
      // Raise the reference of the rows that need it (the first tile's all).
      // O is at rest: its products up to tile j - 1 were done before S.
      const bool raise = top - m > (float)(kTcSlack<T> + kTcHeadroom<T>);  // (m = -inf: any score)
      if (__any_sync(0xffffffffu, raise)) {
        const float next = raise ? reference_of<kTcHeadroom<T>>(top) : m, c = raise ? exp2_fast(m - next) : 1.0f;
        m = next;
        l *= c;
        if (turn > 0) {  // this half of O's columns
#pragma unroll 1
          for (int d = half * (HD / 2); d < (half + 1) * (HD / 2); d += 32) {
            uint32_t o[32];
            tc_ld32(to + d, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * c);
            tc_st32(to + d, o);
          }
        }
      }
      const float ref = m == -INFINITY ? 0.0f : m;
      // The weights, over this half's own scores: part q of the 64 keys' in the
      // columns 32 q .. of the half.
      pair_t sum[2] = {0, 0};
      const pair_t scale2 = pair(scale, scale), ref2 = pair(-ref, -ref);
#pragma unroll
      for (int c = 0; c < 2; c++) {
        uint32_t w[NS][16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
          float a, b;
          const pair_t x2 = fma2(pair(s[c][2 * e], s[c][2 * e + 1]), scale2, ref2);
          unpair(x2, a, b);
          a = exp2_fast(a);
          b = exp2_fast(b);
          sum[e % 2] = add2(sum[e % 2], pair(a, b));
          uint32_t part2[NS];
          split2<T, NS>(a, b, part2);
#pragma unroll
          for (int q = 0; q < NS; q++) w[q][e] = part2[q];
        }
#pragma unroll
        for (int q = 0; q < NS; q++) tc_st16(ts + q * 32 + c * 16, w[q]);
      }
      {
        float a, b;
        unpair(add2(sum[0], sum[1]), a, b);
        l += a + b;
      }
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&sy.p_full[i]);
    }
    // ---- the result
    // Poison is final once the loader is through.
    const bool has0 = n_tiles > 0, has1 = n_tiles > (twice ? 1 : 0);
    if (twice ? has0 : (i ? has1 : has0)) ok = wait(&sy.o_full[twice ? 0 : i], 0) && ok;
    if (twice && has1) ok = wait(&sy.o_full[1], 0) && ok;
    if (!has0) ok = wait(&sy.q_full, 0) && ok;
    ok = wait(&sy.loaded, 0) && ok;
    __syncwarp();
    tc_fence_after();
    sy.x[i][half][r] = l;
    if (i == 1 && half == 0) sy.m1[r] = m;
    if (twice) asm volatile("bar.sync 3, 512;" ::: "memory");
    else tile_sync();
    if (*given_up || *(volatile int *)&sy.poison) {
      for (int k = warp * 16; k < min(warp * 16 + 16, t.rows); k++) attend_row_alone(p, t, k, direct);
    } else if (!twice || i == 0) {
      // The two halves' sums; twice: the two tiles' results on the larger maximum.
      l += sy.x[i][half ^ 1][r];
      float c0 = 1.0f, c1 = 0.0f;
      if (twice) {
        const float m1 = sy.m1[r], l1 = sy.x[1][0][r] + sy.x[1][1][r], top = fmaxf(m, m1);
        c0 = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        c1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - top);
        l = l * c0 + l1 * c1;
        m = top;
      }
      // 32 dims at a time through the warp's 4 KB of the query tiles' memory
      // (no product reads it any more), so that rows are stored in whole lines.
      const int64_t at = !real ? -1 : direct ? out_offset(p, t, row) : part_index(p, t, row) * hd;
      const float inv = !direct ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
      if (real && !direct && half == 0) p.part_ml[part_index(p, t, row)] = make_float2(m, l);
      const bool wide = !direct || NS == 2;  // f32 rows
      char *const stage = base_p + warp * 4096;
      // 32 dims of this thread's row, times 1 / sum where they are final.
      auto result = [&](int d, float (&o)[32]) {
        if (n_tiles) {
          tc_ld32(to + d, (uint32_t *)o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] = 0.0f;
        }
        if (twice) {
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] *= c0;
          if (has1) {
            float o1[32];
            tc_ld32(to + 128 + d, (uint32_t *)o1);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = fmaf(o1[e], c1, o[e]);
          }
        }
#pragma unroll
        for (int e = 0; e < 32; e++) o[e] *= inv;
      };
      const int first = half * (HD / 2);
      __syncwarp();
      if (wide) {
        float *const out = direct ? (float *)p.out : p.part_o;
#pragma unroll 1
        for (int d = first; d < first + HD / 2 && d < hd; d += 32) {
          float o[32];
          result(d, o);
#pragma unroll
          for (int c = 0; c < 8; c++)
            *(float4 *)(stage + lane * 128 + ((c ^ (lane & 7)) * 16)) =
                make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const int rr = k * 4 + lane / 8, c = lane % 8;
            const int64_t o2 = __shfl_sync(0xffffffffu, at, rr);
            const float4 v = *(const float4 *)(stage + rr * 128 + ((c ^ (rr & 7)) * 16));
            if (o2 >= 0 && d + c * 4 < hd) *(float4 *)(out + o2 + d + c * 4) = v;
          }
          __syncwarp();
        }
      } else {
        constexpr int PC = HD / 16;  // 16-byte pieces of a half row
        auto place = [&](int r, int c) { return stage + r * (HD) + ((HD == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) * 16); };
#pragma unroll
        for (int q = 0; q < HD / 64; q++) {
          float o[32];
          result(first + q * 32, o);
#pragma unroll
          for (int c = 0; c < 4; c++)
            *(uint4 *)place(lane, q * 4 + c) =
                make_uint4(pack2<T>(o[8 * c], o[8 * c + 1]), pack2<T>(o[8 * c + 2], o[8 * c + 3]),
                           pack2<T>(o[8 * c + 4], o[8 * c + 5]), pack2<T>(o[8 * c + 6], o[8 * c + 7]));
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < PC; k++) {
          const int rr = k * (32 / PC) + lane / PC, c = lane % PC;
          const int64_t o2 = __shfl_sync(0xffffffffu, at, rr);
          const uint4 v = *(const uint4 *)place(rr, c);
          if (o2 >= 0 && first + c * 8 < hd) *(uint4 *)((T *)p.out + o2 + first + c * 8) = v;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 19) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace paged
}  // namespace jal
