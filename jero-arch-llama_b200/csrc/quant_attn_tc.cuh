// Attention of many query rows over a paged cache of 8- or 4-bit codes on the tcgen05
// tensor cores.  Included by quant_attn.cu.
//
// The blocks, row tiles, key tiles and tensor-memory layout are those of
// k_paged_attn_tc: 256 query rows of one KV head as two tiles of 128 that take turns,
// key tiles of 128, S = Q K^T and then the weights P in tensor memory, O += P V.
// What differs:
//
//   - K and V tiles hold the codes, widened to f16 on their way into shared memory
//     (whole numbers, exact), and the scales of their keys lie beside them: a score
//     is multiplied by K's, a weight by V's.  Where f16 values of the cache would
//     be rounded to 11 bits twice, nothing but the weights is.
//   - q is carried as f16 parts of the row times a power of two, whatever its type
//     (one part for 16-bit rows; two, 22 bits, for f32).
//   - The weights and their sum refer to the row's maximum alone; weight times dv, which
//     goes to the product with V, over 2^(E - kQuantHeadroom) too, with 2^E the power
//     of two below the largest |dv| that the row has seen.  It stays below 2^15, and each is
//     off by 2^-35 of the row's largest weight times its largest dv beside its relative
//     error.  (One reference for both would lose the sum's earlier part as soon as E grows by
//     more than f32's range, and costs f32 rows bits of the weights' exponents.)
//
// 2048 rows of 32 heads (8 KV heads of 128) behind 6144 cached 8-bit positions take 446
// us (the same over a bf16 cache 258; f32 rows 565).  What is dearer here: three loader warps widen
// 128 x 128 codes a tile (without that, in a private copy, 373), and scales are
// fetched and multiplied with each score and weight (without that too 292).  The 256 blocks are 1.73 rounds of
// 148 SMs; cut into pieces they would have to be joined, 40 us for four.
//
//   warps 0-15       softmax, as there
//   warps 16-18      loaders: codes from their pages, widened, into the ring
//   warp 19          one thread issues the products
#pragma once

#include "quant_attn_mma.cuh"

namespace jal {
namespace paged {

constexpr int kQuantSlack = 4, kQuantHeadroom = 10, kQuantLeastE = -107;  // (an append leaves no smaller scale)

struct QuantTcSync {
  uint64_t q_full;
  uint64_t kv_full[6], kv_empty[6];
  uint64_t present_full[8];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint32_t tmem;
  int given_up;
  // Of a row's halves: the largest score of the key tile, and at the end the sum of the
  // weights.  Before the first tile: the power of two that a row's scores are still to be
  // multiplied by ([256]).  Barriers lie between these uses.
  float x[2][2][128];
  uint8_t e[2][2][128];                // exponents of the largest scale of V that a row's halves see
  bool bad[2][128];                    // rows of q with a NaN or an infinity
  float m1[128], unit1[128];           // at the end, of the second row tile: what its weights refer to, what O counts
  alignas(16) uint8_t present[8][16];  // which keys of tile j exist, a bit each, by j % 8
  alignas(16) float dk[8][128], dv[8][128];  // their scales (K's times the softmax's), 0 where there is
                                             // no key; a V scale that is not finite is a NaN of K's
};

template <int BITS, int NS, int HD>
struct QuantTcShape {
  static constexpr int tile = kTcKeys * HD * 2;  // bytes of a K or V tile
  static constexpr int q_tile = 128 * HD * 2;    // of one part of a row tile
  static constexpr int buffers = HD == 64 ? 6 : NS == 1 ? 4 : 2;
  // The query tiles; at the end 4 KB for each softmax warp.
  static constexpr int q_area = 2 * NS * q_tile > 65536 ? 2 * NS * q_tile : 65536;
  // Codes on their way: of each loader the groups of eight rows that it has of a tile.
  static constexpr int row_bytes = HD * BITS / 8, groups = (16 + kTcLoaders - 1) / kTcLoaders;
  static constexpr int ring = q_area, raw = ring + buffers * tile, sync = raw + kTcLoaders * groups * 8 * row_bytes;
  static constexpr int smem = sync + (int)sizeof(QuantTcSync);
};
static_assert(QuantTcShape<8, 1, 128>::smem <= 232448 && QuantTcShape<8, 2, 128>::smem <= 232448 &&
                  QuantTcShape<8, 2, 64>::smem <= 232448,
              "shared memory of a block");

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  uint32_t v;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
  return v;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t v;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(a), "r"(b), "r"(c));
  return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
// Sixteen codes, in order, as f16: a code is placed in the low mantissa bits of 1024 (its
// sum with 1024, exactly), from which 1024 and the code's offset are subtracted.
template <int BITS>
__device__ __forceinline__ void widen16(const uint32_t *w, uint32_t (&out)[8]) {
  if constexpr (BITS == 8) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t u = w[i] ^ 0x80808080u;
      out[2 * i] = h2_sub(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u);
      out[2 * i + 1] = h2_sub(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u);
    }
  } else {
    // A byte's low half as it is, its high half as 16 times the code.
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t u = __byte_perm(w[i / 4], 0, (uint32_t)(i % 4) * 0x1111u);
      out[i] = h2_fma((u & 0x00F0000Fu) | 0x64006400u, 0x2C003C00u, 0xD480E408u);  // * (1, 1 / 16) - (1032, 72)
    }
  }
}

template <int BITS, int NS, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) k_quant_attn_tc(const __grid_constant__ QuantAttnParams qp, const bool direct) {
  using S = QuantTcShape<BITS, NS, HD>;
  const AttnParams &p = qp.a;
  extern __shared__ __align__(1024) char smem_tc[];
  QuantTcSync &sy = *(QuantTcSync *)(smem_tc + S::sync);
  pdl_wait();
  pdl_trigger();
  Tile t;
  if (!block_tile(p, kOwn, kTcRows, kTcKeys, t)) return;
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
  constexpr int kGroups = S::groups;
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
    sy.given_up = 0;
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
  // A wait that gives up (it cannot, unless the code is wrong) makes the block's rows
  // NaN instead of hanging the GPU.
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
      // Codes come by cp.async, two groups of eight rows at a time, and are widened from there into the ring while the ones behind them are on their way:
      // V's of a tile while K's are widened, then K's of the next tile.  Rows without a
      // key are left as they are: whatever the bytes are, they are codes, and weigh
      // nothing.
      // HD / 16 lanes widen a row, sixteen codes a lane: dims 16 c16 .., two pieces of 16
      // bytes in the swizzle.  (The upper four of eight lanes have their pieces the other
      // way round, so that eight lanes store eight different ones.)
      constexpr int kLanes = HD / 16, kRows = 32 / kLanes;  // lanes of a row; rows of a warp at once
      constexpr int kUnits = kGroups / 2;
      static_assert(kGroups % 2 == 0 && kUnits <= 4, "units of two groups");
      const int c16 = lane % kLanes, r0 = lane / kLanes, flip = c16 / 4;
      char *const raw = smem_tc + S::raw + w * (kGroups * 8 * S::row_bytes);
      const uint32_t raw_s = smem_u32(raw);
      bool ok = true;
      int b = 0, parity = 1;  // of the buffer's "empty" phase before this use: the first use finds it free
      constexpr int kPieces = S::row_bytes / 16, kCopy = 32 / kPieces;  // of a row; rows of a warp's copy
      const int cp = lane % kPieces, cr = lane / kPieces;
      const bool inside = cp * 16 < hd * BITS / 8;
      // Lanes 0 .. 15 (unit 1: 16 .. 31) have the places of a unit's rows.
      auto ask = [&](const void *pool, const int64_t (&from)[2], int unit, bool any) {
#pragma unroll
        for (int i = 0; i < 16 / kCopy; i++) {
          const int r = i * kCopy + cr;
          const int64_t o = __shfl_sync(0xffffffffu, unit < 2 ? from[0] : from[1], unit % 2 * 16 + r);
          if (any && o >= 0 && inside) copy16(raw_s + (unit * 16 + r) * S::row_bytes + cp * 16, (const char *)pool + o + cp * 16, true);
        }
        copies_done();
      };
      auto widen = [&](int unit) {
        copies_wait<kUnits - 1>();
        __syncwarp();
        char *const dst = base_p + S::ring + b * S::tile + c16 / 4 * (kTcKeys * 128);
        constexpr int kSteps = 16 / kRows;
        const int c = c16 % 4 * 2;
        uint32_t x[kSteps][BITS / 2];
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
          const uint32_t at = raw_s + (unit * 16 + i * kRows + r0) * S::row_bytes + c16 * (2 * BITS);
          if constexpr (BITS == 8) {
            lds<8>(at + flip * 8, x[i]);
            lds<8>(at + 8 - flip * 8, x[i] + 2);
          } else {
            x[i][0] = lds4(at + flip * 4);
            x[i][1] = lds4(at + 4 - flip * 4);
          }
        }
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
          const int gr = group(unit * 2 + i * kRows / 8), r = (i * kRows + r0) % 8;
          if (gr >= 16) break;
          uint32_t h[8];
          widen16<BITS>(x[i], h);
          char *const row = dst + gr * 1024 + r * 128;
          *(uint4 *)(row + (((c + flip) ^ r) * 16)) = make_uint4(h[0], h[1], h[2], h[3]);
          *(uint4 *)(row + (((c + 1 - flip) ^ r) * 16)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
        __syncwarp();  // every lane has read the unit before it is filled again
      };
      auto begin = [&]() { return ok = __all_sync(0xffffffffu, ok && wait(&sy.kv_empty[b], parity)); };
      auto end = [&]() {
        mbar_arrive(&sy.kv_full[b]);
        if (++b == S::buffers) {
          b = 0;
          parity ^= 1;
        }
      };
      // Where a tile's rows lie, which of them exist, and their scales.
      int64_t at[2], ahead[2];
      uint32_t bits[2];
      float dk[2], dv[2];
      auto look = [&](int64_t (&to)[2]) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const Slot &sl = e ? next1 : next0;
          to[e] = slot_offset(p.kv, sl, t.head);
          bits[e] = __ballot_sync(0xffffffffu, to[e] >= 0);
          const bool there = to[e] >= 0;
          const int64_t o = there ? (int64_t)sl.page * qp.sc.s_page + t.head * qp.sc.s_head + sl.slot : 0;
          dk[e] = there ? __ldg(qp.sc.k + o) * p.scale_log2 : 0.0f;
          dv[e] = there ? __ldg(qp.sc.v + o) : 0.0f;
          // (Weights of 0 times such a scale would be NaN in rows that do not see it.)
          if (!(fabsf(dv[e]) < INFINITY)) {
            dv[e] = 0.0f;
            dk[e] = NAN;
          }
        }
      };
      if (n_tiles) {
        look(ahead);
        next0 = locate(1, 0);
        next1 = locate(1, 4);
#pragma unroll
        for (int k = 0; k < kUnits; k++) ask(p.kv.k, ahead, k, true);
      }
#pragma unroll 1
      for (int j = 0; j < n_tiles; j++) {
        at[0] = ahead[0];
        at[1] = ahead[1];
        // (Tile j + 8 comes long after the softmax has read tile j's.)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int gr = group(4 * e + lane / 8), key = gr * 8 + lane % 8;
          if (4 * e + lane / 8 < kGroups && gr < 16) {
            sy.dk[j & 7][key] = dk[e];
            sy.dv[j & 7][key] = dv[e];
          }
        }
        if (lane < kGroups && group(lane) < 16)
          sy.present[j & 7][group(lane)] = (uint8_t)((lane < 4 ? bits[0] : bits[1]) >> (lane % 4 * 8));
        __syncwarp();
        if (lane == 0) mbar_arrive(&sy.present_full[j & 7]);
        if (!begin()) break;
#pragma unroll
        for (int k = 0; k < kUnits; k++) {
          widen(k);
          ask(p.kv.v, at, k, true);
        }
        end();
        look(ahead);  // (of the last tile: no row)
        next0 = locate(j + 2, 0);
        next1 = locate(j + 2, 4);
        if (!begin()) break;
#pragma unroll
        for (int k = 0; k < kUnits; k++) {
          widen(k);
          ask(p.kv.k, ahead, k, j + 1 < n_tiles);
        }
        end();
      }
      copies_wait<0>();
    } else {
      // ---- the products: the whole warp runs the loop, so that addresses stay
      // uniform, and one lane issues
      const bool leader = elect_one();
      constexpr uint32_t id = (1u << 4) | ((128u >> 4) << 24);  // f16 x f16 into f32, 128 rows
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
              tc_mma_ts(tmem + 256 + i * 128, tmem + i * 128 + (k / 2) * 32 + s * 16 + (k % 2) * 8,
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
        // (The fence stands here and not behind the stores: there it would wait for the
        // loader's copies that are on their way.)
        fence_proxy_async();
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
    auto tile_sync = [&]() { asm volatile("bar.sync %0, 256;" ::"r"(1 + i) : "memory"); };
    {  // the query rows into shared memory, 16 rows a warp, neighbouring lanes neighbouring pieces
      const int first = warp % 8 * 16;  // of the row tile
      char *const dst = base_p + i * NS * S::q_tile;
      const int mine = base + first + lane % 16;
      const int64_t qt = mine < t.rows ? q_offset(p, t, mine) : -1;
      constexpr int CH = HD / 8;
#pragma unroll 2
      for (int k = 0; k < CH / 2; k++) {
        const int kr = (k * 32 + lane) / CH, c = lane % CH;
        const int64_t o = __shfl_sync(0xffffffffu, qt, kr);
        float v[8] = {};
        if (o >= 0 && c * 8 < hd) {
          if (NS == 2) load8((const float *)p.q + o + c * 8, v);
          else if (p.act == JAL_F16) load8((const __half *)p.q + o + c * 8, v);
          else load8((const __nv_bfloat16 *)p.q + o + c * 8, v);
        }
        uint32_t most = 0;  // (a NaN's bits are above infinity's)
#pragma unroll
        for (int e = 0; e < 8; e++) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
#pragma unroll
        for (int x = CH / 2; x > 0; x >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, x));
        const float top = __uint_as_float(most);
        // A row with a NaN or an infinity goes in as 0, and its result is made NaN at the end: an
        // infinite element's scores may all be -inf, as if the row saw nothing.  One that is next to
        // nothing goes in as 0 too: the inverse of its power of two may lie below f32's range, and
        // the -inf of a masked key times 0 is NaN.
        const bool bad = !(top < INFINITY), some = !bad && top >= kQuantLeast;
        if (!some) {
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] = 0.0f;
        }
        const int e = some ? 13 - ilogbf(top) : 0;
        // in two steps: 2^e itself may lie outside f32's range
        const float a = exp2f((float)(e / 2)), b = exp2f((float)(e - e / 2));
        uint32_t part2[4][NS];
#pragma unroll
        for (int q = 0; q < 4; q++) split2<__half, NS>(v[2 * q] * a * b, v[2 * q + 1] * a * b, part2[q]);
#pragma unroll
        for (int s = 0; s < NS; s++)
          *(uint4 *)(dst + s * S::q_tile + (c / 8) * (128 * 128) + (first + kr) * 128 + (((c % 8) ^ (kr & 7)) * 16)) =
              make_uint4(part2[0][s], part2[1][s], part2[2][s], part2[3][s]);
        if (c == 0) {
          (&sy.x[0][0][0])[i * 128 + first + kr] = (1.0f / a) / b;
          sy.bad[i][first + kr] = bad;
        }
      }
      fence_proxy_async();
      mbar_arrive(&sy.q_full);
    }
    tile_sync();
    const float scale = (&sy.x[0][0][0])[i * 128 + r];  // a power of two: positive
    // (The row tiles' factors overlap the other one's maxima.)
    asm volatile("bar.sync 3, 512;" ::: "memory");
    const uint32_t quarter = (uint32_t)(warp % 4) << 21;  // lane 32 (warp % 4) of the tensor memory
    const uint32_t ts = tmem + i * 128 + half * 64 + quarter, to = tmem + 256 + i * 128 + quarter;
    const RowSpan span = row_span(p, t, mk);
    float m = -INFINITY, l = 0.0f;  // m: what the weights refer to, base 2; l: this half's sum
    int high = kQuantLeastE;        // E: the power of two below V's largest scale that the row has seen
    auto power = [](int e) -> float { return __uint_as_float((uint32_t)(127 + e) << 23); };
    bool ok = true;
    int turn = 0;  // of this row tile
#pragma unroll 1
    for (int j = twice ? i : 0; j < n_tiles; j += twice ? 2 : 1, turn++) {
      // (A wait that gave up does not leave the loop: the other half waits below.)
      ok = wait(&sy.present_full[j & 7], (j >> 3) & 1) && ok;
      ok = wait(&sy.s_full[i], turn & 1) && ok;
      __syncwarp();
      tc_fence_after();
      const int u = t.u0 + j * kTcKeys + half * 64;
      const uint2 here = *(const uint2 *)&sy.present[j & 7][half * 8];
      const bool whole = (here.x & here.y) == 0xffffffffu && span.all(u, 64);
      const bool masked = !__all_sync(0xffffffffu, whole || !real);
      const float *const dk = sy.dk[j & 7] + half * 64, *const dv = sy.dv[j & 7] + half * 64;
      // Scores over the row's factor, masked, back into tensor memory 32 at a time (64 in
      // registers beside their scales are more than a thread has), with their maximum and
      // the largest scale of V (its bits) that the row sees.
      float mine = -INFINITY;
      uint32_t largest = 0;
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float s[32];
        tc_ld32(ts + c * 32, (uint32_t *)s);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 d = *(const float4 *)(dk + c * 32 + e);
          unpair(mul2(pair(s[e], s[e + 1]), pair(d.x, d.y)), s[e], s[e + 1]);
          unpair(mul2(pair(s[e + 2], s[e + 3]), pair(d.z, d.w)), s[e + 2], s[e + 3]);
        }
        if (masked) {
          const uint32_t bits = (c ? here.y : here.x) & span.bits(u + c * 32);
#pragma unroll
          for (int e = 0; e < 32; e++) {
            if ((bits >> e) & 1) largest = max(largest, __float_as_uint(dv[c * 32 + e]) & 0x7fffffffu);
            else s[e] = -INFINITY;
          }
        }
        tc_st32(ts + c * 32, (uint32_t *)s);
        float x[4] = {max3_nan(mine, s[0], s[1]), s[2], s[3], s[4]};
#pragma unroll
        for (int e = 5; e < 29; e += 8)
#pragma unroll
          for (int k = 0; k < 4; k++) x[k] = max3_nan(x[k], s[e + 2 * k], s[e + 2 * k + 1]);
        mine = max3_nan(max3_nan(x[0], x[1], s[29]), max3_nan(x[2], x[3], s[30]), s[31]);
      }
      if (!masked) {
        const uint2 x = *(const uint2 *)(dv + lane * 2);
        largest = __reduce_max_sync(0xffffffffu, max(x.x & 0x7fffffffu, x.y & 0x7fffffffu));
      }
      tc_wait_st();
      sy.x[i][half][r] = mine;
      sy.e[i][half][r] = (uint8_t)(largest >> 23);
      tile_sync();
      const int was = high;
      high = max(high, max((int)(largest >> 23), (int)sy.e[i][half ^ 1][r]) - 127);
      const float top = max3_nan(mine, sy.x[i][half ^ 1][r], mine) * scale;
      // A NaN or an infinite score makes the row NaN, as the formula does.
      if (!(top < INFINITY)) l = NAN;
      // Raise the reference of the rows that need it (the first tile's all).
      // O is at rest: its products up to tile j - 1 were done before S.
      const bool raise = top - m > (float)kQuantSlack || high > was;  // (m = -inf: any score)
      if (__any_sync(0xffffffffu, raise)) {
        const float next = raise ? fmaxf(m, top) : m, less = next == m ? 0.0f : m - next, c = exp2_fast(less + (float)(was - high));
        m = next;
        l *= exp2_fast(less);
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
      // The weights, over this half's own scores: part q of 32 keys in 16 of the columns
      // that held their scores.
      pair_t sum[2] = {0, 0};
      const float lift = power(kQuantHeadroom - high);
      const pair_t scale2 = pair(scale, scale), ref2 = pair(-ref, -ref), lift2 = pair(lift, lift);
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float s[32];
        uint32_t w[NS][16];
        tc_ld32(ts + c * 32, (uint32_t *)s);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 d = *(const float4 *)(dv + c * 32 + 2 * e);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float a, b;
            const pair_t x2 = fma2(pair(s[2 * (e + h)], s[2 * (e + h) + 1]), scale2, ref2);
            unpair(x2, a, b);
            a = exp2_fast(a);
            b = exp2_fast(b);
            sum[h] = add2(sum[h], pair(a, b));
            unpair(mul2(pair(a, b), mul2(h ? pair(d.z, d.w) : pair(d.x, d.y), lift2)), a, b);
            uint32_t part2[NS];
            split2<__half, NS>(a, b, part2);
#pragma unroll
            for (int q = 0; q < NS; q++) w[q][e + h] = part2[q];
          }
        }
#pragma unroll
        for (int q = 0; q < NS; q++) tc_st16(ts + c * 32 + q * 16, w[q]);
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
    const bool has0 = n_tiles > 0, has1 = n_tiles > (twice ? 1 : 0);
    if (twice ? has0 : (i ? has1 : has0)) ok = wait(&sy.o_full[twice ? 0 : i], 0) && ok;
    if (twice && has1) ok = wait(&sy.o_full[1], 0) && ok;
    if (!has0) ok = wait(&sy.q_full, 0) && ok;
    __syncwarp();
    tc_fence_after();
    if (sy.bad[i][r] && l != 0.0f) l = NAN;  // (its scores are 0, so that l counts the keys that it sees)
    sy.x[i][half][r] = l;
    float unit = power(high - kQuantHeadroom);  // what O counts
    if (i == 1 && half == 0) {
      sy.m1[r] = m;
      sy.unit1[r] = unit;
    }
    if (twice) asm volatile("bar.sync 3, 512;" ::: "memory");
    else tile_sync();
    if (!twice || i == 0) {
      // The two halves' sums; twice: the two tiles' results on the larger reference.
      l += sy.x[i][half ^ 1][r];
      float c0 = 1.0f, c1 = 0.0f;
      if (twice) {
        const float m1 = sy.m1[r], l1 = sy.x[1][0][r] + sy.x[1][1][r], top = fmaxf(m, m1);
        c0 = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        c1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - top);
        l = l * c0 + l1 * c1;
        m = top;
        c0 *= unit;
        c1 *= sy.unit1[r];
        unit = 1.0f;
      }
      if (*given_up) l = NAN;
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
        for (int e = 0; e < 32; e++) o[e] = o[e] * inv * unit;
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
        auto pack = [&](float a, float b) { return p.act == JAL_F16 ? pack2<__half>(a, b) : pack2<__nv_bfloat16>(a, b); };
#pragma unroll
        for (int q = 0; q < HD / 64; q++) {
          float o[32];
          result(first + q * 32, o);
#pragma unroll
          for (int c = 0; c < 4; c++)
            *(uint4 *)place(lane, q * 4 + c) = make_uint4(pack(o[8 * c], o[8 * c + 1]), pack(o[8 * c + 2], o[8 * c + 3]),
                                                          pack(o[8 * c + 4], o[8 * c + 5]), pack(o[8 * c + 6], o[8 * c + 7]));
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < PC; k++) {
          const int rr = k * (32 / PC) + lane / PC, c = lane % PC;
          const int64_t o2 = __shfl_sync(0xffffffffu, at, rr);
          const uint4 v = *(const uint4 *)place(rr, c);
          if (o2 >= 0 && first + c * 8 < hd) *(uint4 *)((uint16_t *)p.out + o2 + first + c * 8) = v;
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
