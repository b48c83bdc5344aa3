// Attention of many query rows over a 16-bit paged cache on the tcgen05 tensor
// cores.  Included by paged_attn.cu.
//
// A block takes 256 query rows of one KV head as two tiles of 128 and runs
// over its keys in tiles of 128: S = Q K^T into tensor memory, softmax weights
// P in registers (one thread a row), P back into tensor memory over S, and
// O += P V with O in tensor memory.  The two row tiles take turns: while the
// tensor cores work on one, a warpgroup forms the weights of the other, so a
// K and a V tile are read once for 256 rows.  Per key tile the tensor cores
// need 4 x 128 x 128 x HD products and the special-function units 2 x 128 x
// 128 exponentials; at HD = 128 the former takes longer, so what bounds the
// kernel is how gaplessly the products are issued.
//
//   warps 0-3, 4-7   softmax of row tile 0, 1 (warp w reads tensor-memory
//                    lanes 32 (w % 4) ..), and the result
//   warps 8-11       K and V rows from their pages into the ring, cp.async
//   warp 12          one thread issues the products
//
// Pages may hold any number of slots, so rows are copied one by one to their
// place in the 128-byte swizzle that the matrix descriptors name: K tiles and
// V tiles are both [HD / 64][128 keys][64 dims], K read as K-major and V as
// MN-major.
//
// The running maximum that the weights refer to is only raised when a row's
// maximum grows by more than 2^8; weights then reach 256 at most, and O is
// rescaled rarely.  f32 rows (NS = 2, f16 cache) are split like in the
// mma.sync kernel: two f16 parts of q and of the weights.
#pragma once

#include "paged_attn_mma.cuh"
#include "paged_dev.cuh"

namespace jal {
namespace paged {

constexpr int kTcRows = 256, kTcKeys = 128, kTcThreads = 512;
constexpr float kTcSlack = 8.0f;  // growth of a maximum (base 2) that is let stand

template <int NS, int HD>
struct TcShape {
  static constexpr int tile = kTcKeys * HD * 2;            // bytes of a K or V tile
  static constexpr int q_tile = 128 * HD * 2;              // of one part of a row tile
  static constexpr int buffers = HD == 64 ? 6 : NS == 1 ? 5 : 3;
  // Groups of copies that may be under way when the loader waits for a free
  // buffer: freeing a V tile takes the next K tile, so buffers - 2 at most.
  static constexpr int pending = buffers == 3 ? 1 : 2;
  static constexpr int smem = 1024 + 2 * NS * q_tile + buffers * tile;
};

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

struct TcSync {
  uint64_t q_full;
  uint64_t kv_full[6], kv_empty[6];
  uint64_t present_full[8];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint32_t tmem;
  int given_up, poison;
  int lim_lo, lim_hi, wlo_lo, wlo_hi;
  uint32_t present[8][4];  // which keys of tile j exist, by j % 8
};

template <class T, int NS, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) k_paged_attn_tc(const AttnParams p, const int part, const bool direct) {
  using S = TcShape<NS, HD>;
  extern __shared__ char smem_raw[];
  __shared__ TcSync sy;
  pdl_trigger();
  Tile t;
  if (!block_tile(p, part, kTcRows, kTcKeys, t)) return;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, hd = p.kv.hd;
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  char *const base_p = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sq = base, ring = base + 2 * NS * S::q_tile;
  const int n_tiles = (t.u1 - t.u0 + kTcKeys - 1) / kTcKeys;

  if (tid == 0) {
    mbar_init(&sy.q_full, 256);
    for (int i = 0; i < S::buffers; i++) {
      mbar_init(&sy.kv_full[i], 128);
      mbar_init(&sy.kv_empty[i], 1);
    }
    for (int i = 0; i < 8; i++) mbar_init(&sy.present_full[i], 4);
    for (int i = 0; i < 2; i++) {
      mbar_init(&sy.s_full[i], 1);
      mbar_init(&sy.p_full[i], 128);
      mbar_init(&sy.o_full[i], 1);
    }
    sy.given_up = sy.poison = 0;
    sy.lim_lo = sy.wlo_lo = 0x7fffffff;
    sy.lim_hi = sy.wlo_hi = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
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
    if (mbar_wait_bounded(bar, parity)) return true;
    *given_up = 1;
    return false;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp < 12) {
      // ---- the loader
      const int w = warp - 8;
      auto locate = [&](int j) -> int64_t {
        const int u = t.u0 + j * kTcKeys + w * 32 + lane;
        return j < n_tiles && u < t.u1 ? slot_offset(p.kv, t.table, t.head, t.key(u)) : -1;
      };
      constexpr int CH = HD / 8, N = 32 * CH / 32;
      bool ok = true, bad = false;
      int arrived = 0;
      // Group g (K tile g / 2 when even, V tile when odd) has landed: rows that
      // some queries must not meet are looked through, then it is handed over.
      auto hand_over = [&](int g) {
        const int b = g % S::buffers;
        if (g & 1) {
          const int u = t.u0 + (g >> 1) * kTcKeys, first = t.key(u), last = t.key(min(u + kTcKeys, t.u1) - 1);
          if (g == 1) ok = ok && wait(&sy.q_full, 0);
          const bool mixed = (first < sy.wlo_hi && sy.wlo_lo != sy.wlo_hi) || (last >= sy.lim_lo && sy.lim_lo != sy.lim_hi);
          if (mixed) {
            const char *rows = base_p + 2 * NS * S::q_tile + b * S::tile + (w * 32) * 128;
#pragma unroll 4
            for (int i = 0; i < HD / 64 * 8; i++) {  // 32 rows x 128 bytes x (HD / 64) of this warp
              const uint4 x = *(const uint4 *)(rows + (i / 8) * (kTcKeys * 128) + ((i % 8) * 32 + lane) * 16);
              const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const float2 f = unpack2<T>(v[e]);
                bad |= !isfinite(f.x) || !isfinite(f.y);
              }
            }
            if (bad) sy.poison = 1;
          }
        }
        fence_proxy_async();
        mbar_arrive(&sy.kv_full[b]);
        arrived = g + 1;
      };
      int64_t next = locate(0);
      for (int j = 0; j < n_tiles && ok; j++) {
        const int64_t at = next;
        const uint32_t bits = __ballot_sync(0xffffffffu, at >= 0);
        next = locate(j + 1);
        if (lane == 0) {  // tile j + 8 comes long after the softmax has read tile j's
          sy.present[j & 7][w] = bits;
          mbar_arrive(&sy.present_full[j & 7]);
        }
#pragma unroll 1
        for (int kv = 0; kv < 2 && ok; kv++) {
          const int g = 2 * j + kv, b = g % S::buffers;
          if (g >= S::buffers) ok = wait(&sy.kv_empty[b], (g / S::buffers - 1) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const T *pool = (const T *)(kv ? p.kv.v : p.kv.k);
          const uint32_t dst = ring + b * S::tile;
#pragma unroll
          for (int i = 0; i < N; i++) {
            const int r = (i * 32 + lane) / CH, c = (i * 32 + lane) % CH, row = w * 32 + r;
            const int64_t o = __shfl_sync(0xffffffffu, at, r);
            const bool there = o >= 0 && c * 8 < hd;
            copy16(dst + (c / 8) * (kTcKeys * 128) + row * 128 + (((c % 8) ^ (row & 7)) * 16),
                   pool + (there ? o + c * 8 : 0), there);
          }
          copies_done();
          if (g >= S::pending) {
            copies_wait<S::pending>();
            hand_over(g - S::pending);
          }
        }
      }
      copies_wait<0>();
      if (ok) {
#pragma unroll 1
        for (int g = arrived; g < 2 * n_tiles; g++) hand_over(g);
      }
    } else if (warp == 12 && lane == 0) {
      // ---- the products
      constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t id = (1u << 4) | (type << 7) | (type << 10) | ((128u >> 4) << 24);
      constexpr uint32_t id_s = id | ((kTcKeys >> 3) << 17), id_o = id | (1u << 16) | ((HD >> 3) << 17);
      auto scores = [&](int i, int j) {
        const uint32_t kb = ring + ((2 * j) % S::buffers) * S::tile;
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
          for (int k = 0; k < HD / 16; k++) {
            const uint32_t off = (k / 4) * (128 * 128) + (k % 4) * 32;
            tc_mma_ss(tmem + i * 128, tc_desc(sq + (i * NS + s) * S::q_tile + off, 16, 1024), tc_desc(kb + off, 16, 1024),
                      id_s, s + k > 0);
          }
        tc_commit(&sy.s_full[i]);
      };
      auto output = [&](int i, int j) {
        const uint32_t vb = ring + ((2 * j + 1) % S::buffers) * S::tile;
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
          for (int k = 0; k < kTcKeys / 16; k++)
            tc_mma_ts(tmem + 256 + i * 128, tmem + i * 128 + s * 64 + k * 8, tc_desc(vb + k * 2048, kTcKeys * 128, 1024), id_o,
                      j > 0 || s + k > 0);
      };
      auto full = [&](int g) { return wait(&sy.kv_full[g % S::buffers], (g / S::buffers) & 1); };
      bool ok = n_tiles == 0 || (wait(&sy.q_full, 0) && full(0));
      if (ok && n_tiles) {
        tc_fence_after();
        scores(0, 0);
        scores(1, 0);
        tc_commit(&sy.kv_empty[0]);
      }
      for (int j = 0; j < n_tiles && ok; j++) {
        for (int i = 0; i < 2 && ok; i++) {
          ok = (i || full(2 * j + 1)) && wait(&sy.p_full[i], j & 1);
          if (!ok) break;
          tc_fence_after();
          output(i, j);
          if (i) tc_commit(&sy.kv_empty[(2 * j + 1) % S::buffers]);
          if (j + 1 < n_tiles) {
            ok = i || full(2 * j + 2);
            if (!ok) break;
            tc_fence_after();
            scores(i, j + 1);
            if (i) tc_commit(&sy.kv_empty[(2 * j + 2) % S::buffers]);
          } else {
            tc_commit(&sy.o_full[i]);
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---- softmax: thread r of warpgroup i has row i * 128 + r
    const int i = warp / 4, r = tid % 128, row = i * 128 + r;
    const bool real = row < t.rows;
    const RowMask mk = real ? row_mask(p, t, row) : RowMask{0, 0};
    // Weights are formed with a positive factor: a negative one turns q round,
    // none makes it 0.
    float scale = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
    {  // its query row into shared memory
      const int64_t qo = real ? q_offset(p, t, row) : 0;
      char *const dst_p = base_p + i * NS * S::q_tile;
      const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
      const bool take = real && p.scale_log2 != 0.0f;
      float a = 1.0f, b = 1.0f;
      if (NS == 2) {
        float top = 0.0f;
        for (int d = 0; real && d < hd; d += 8) {
          float v[8];
          load8((const float *)p.q + qo + d, v);
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (fabsf(v[e]) < INFINITY) top = fmaxf(top, fabsf(v[e]));
        }
        const int e = top > 0.0f ? 13 - ilogbf(top) : 0;
        a = exp2f((float)(e / 2));
        b = exp2f((float)(e - e / 2));
        scale *= (1.0f / a) / b;
        if (flip) a = -a;
      }
#pragma unroll 4
      for (int c = 0; c < HD / 8; c++) {
        uint4 out[NS];
        if (NS == 1) {
          out[0] = make_uint4(0, 0, 0, 0);
          if (take && c * 8 < hd) {
            out[0] = *(const uint4 *)((const T *)p.q + qo + c * 8);
            out[0].x ^= flip;
            out[0].y ^= flip;
            out[0].z ^= flip;
            out[0].w ^= flip;
          }
        } else {
          float v[8] = {};
          if (take && c * 8 < hd) load8((const float *)p.q + qo + c * 8, v);
          uint32_t part2[4][NS];
#pragma unroll
          for (int e = 0; e < 4; e++) split2<T, NS>(v[2 * e] * a * b, v[2 * e + 1] * a * b, part2[e]);
#pragma unroll
          for (int s = 0; s < NS; s++) out[s] = make_uint4(part2[0][s], part2[1][s], part2[2][s], part2[3][s]);
        }
#pragma unroll
        for (int s = 0; s < NS; s++)
          *(uint4 *)(dst_p + s * S::q_tile + (c / 8) * (128 * 128) + r * 128 + (((c % 8) ^ (r & 7)) * 16)) = out[s];
      }
      int lo = real ? mk.lim : 0x7fffffff, hi = real ? mk.lim : 0, wl = real ? mk.wlo : 0x7fffffff, wh = real ? mk.wlo : 0;
      lo = __reduce_min_sync(0xffffffffu, lo);
      hi = __reduce_max_sync(0xffffffffu, hi);
      wl = __reduce_min_sync(0xffffffffu, wl);
      wh = __reduce_max_sync(0xffffffffu, wh);
      if (lane == 0) {
        atomicMin(&sy.lim_lo, lo);
        atomicMax(&sy.lim_hi, hi);
        atomicMin(&sy.wlo_lo, wl);
        atomicMax(&sy.wlo_hi, wh);
      }
      fence_proxy_async();
      mbar_arrive(&sy.q_full);
    }
    const uint32_t quarter = (uint32_t)(warp % 4) << 21;  // lane 32 (warp % 4) of the tensor memory
    const uint32_t ts = tmem + i * 128 + quarter, to = tmem + 256 + i * 128 + quarter;
    float m = -INFINITY, l = 0.0f;  // m: what the weights refer to, scaled to base 2
    bool ok = true;
    for (int j = 0; j < n_tiles; j++) {
      ok = __all_sync(0xffffffffu, wait(&sy.present_full[j & 7], (j >> 3) & 1) && wait(&sy.s_full[i], j & 1));
      if (!ok) break;
      tc_fence_after();
      float s[128];
#pragma unroll
      for (int c = 0; c < 4; c++) tc_ld32(ts + c * 32, (uint32_t *)s + c * 32);
      tc_wait_ld();
      const int u = t.u0 + j * kTcKeys, first = t.key(u), last = t.key(min(u + kTcKeys, t.u1) - 1);
      const uint32_t *here = sy.present[j & 7];
      const bool whole = (here[0] & here[1] & here[2] & here[3]) == 0xffffffffu && first >= mk.wlo && last < mk.lim;
      if (!__all_sync(0xffffffffu, whole || !real)) {
#pragma unroll
        for (int c = 0; c < 128; c++)
          if (!((here[c / 32] >> (c % 32)) & 1) || !mk.sees(t.key(u + c), p.n_sink)) s[c] = -INFINITY;
      }
      float x[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < 128; c += 4) {
        x[0] = fmaxf(x[0], s[c]);
        x[1] = fmaxf(x[1], s[c + 1]);
        x[2] = fmaxf(x[2], s[c + 2]);
        x[3] = fmaxf(x[3], s[c + 3]);
      }
      const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * scale;
      // Raise the reference of the rows that need it (the first tile's all).
      // O is at rest: its products up to tile j - 1 were done before S.
      const bool raise = top > m + kTcSlack || (m == -INFINITY && top > m);
      if (__any_sync(0xffffffffu, raise)) {
        const float c = raise ? exp2_fast(m - top) : 1.0f;
        if (raise) m = top;
        l *= c;
        if (j > 0) {
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            float o[32];
            tc_ld32(to + d, (uint32_t *)o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] *= c;
            tc_st32(to + d, (const uint32_t *)o);
          }
        }
      }
      const float ref = m == -INFINITY ? 0.0f : m;
      float sum[4] = {};
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t w[NS][16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float a = exp2_fast(fmaf(s[c * 32 + 2 * e], scale, -ref)), b = exp2_fast(fmaf(s[c * 32 + 2 * e + 1], scale, -ref));
          sum[e % 4] += a + b;
          uint32_t part2[NS];
          split2<T, NS>(a, b, part2);
#pragma unroll
          for (int q = 0; q < NS; q++) w[q][e] = part2[q];
        }
#pragma unroll
        for (int q = 0; q < NS; q++) tc_st16(ts + q * 64 + c * 16, w[q]);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&sy.p_full[i]);
    }
    // ---- the result
    // Poison is final once the loader has handed over the last V tile.
    const int last_v = 2 * n_tiles - 1;
    if (ok && n_tiles)
      ok = __all_sync(0xffffffffu, wait(&sy.o_full[i], 0) &&
                                       wait(&sy.kv_full[last_v % S::buffers], (last_v / S::buffers) & 1));
    tc_fence_after();
    if (!ok || *given_up || *(volatile int *)&sy.poison) {
      for (int k = warp * 32; k < min(warp * 32 + 32, t.rows); k++) attend_row_alone(p, t, k, direct);
    } else {
      const int64_t oo = real ? out_offset(p, t, row) : 0, pi = real ? part_index(p, t, row) : 0;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (real && !direct) p.part_ml[pi] = make_float2(m, l);
#pragma unroll 1
      for (int d = 0; d < HD; d += 32) {
        float o[32];
        __syncwarp();
        if (n_tiles) {
          tc_ld32(to + d, (uint32_t *)o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (!real || d + e >= hd) continue;
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; k++) v[k] = direct ? o[e + k] * inv : o[e + k];
          if (!direct) store8(p.part_o + pi * hd + d + e, v);
          else if (NS == 2) store8((float *)p.out + oo + d + e, v);
          else store8((T *)p.out + oo + d + e, v);
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace paged
}  // namespace jal
