// Linear layer on 8-bit operands: y[t, n] = (sum_k xq[t, k] wq[n, k]) sx[t] sw[n] + b[n], xq and wq in e4m3 with a scale per row (rmsnorm.cu writes both),
// y in fp32, bf16 or fp16.
//
//   k_lin8        tcgen05 kind::f8f6f4, 128 tokens x BN features per tile, accumulators in tensor memory
//   k_lin8_few    up to 8 tokens, where the weights are all there is to read: mma.sync on fragments that go through shared memory as they lie
//
// Bound by the tensor cores where K and N are large (8192 x 4096 x 4096: 95 us, 2.9 PFLOP/s, the tensor pipe 83 % busy; by single CTAs of 128 x 256 105 us:
// a pair reads half of the features' tile each, so a third less goes through shared memory and L2), by the passes over tokens and results where they are small
// (131072 x 64 to 128: 10.8 us, 3.9 TB/s), by the weights for few tokens.
//
// Products of two e4m3 numbers are exact in fp32 and are summed there.  The scales are applied to the sums, so operands stay as they lie in memory.
#include <algorithm>

#include "rows.cuh"
#include "tc_ptx.cuh"
#include "tc_tiles.cuh"

using namespace tc;
using namespace rows;

namespace {

// Set by a bounded wait that gave up (see g_lin_status in linear.cu); launches after it leave at once until it has been reported.
__device__ int g_lin8_status;

struct Lin8Args {
  const uint8_t *x, *w;
  long long ldx, ldw;
  const float *sx, *sw;
  const void* bias; int bias_type;        // or null
  void* y; long long ldy;
  int T, K, N;
  int tiles_m, tiles_n;
  int staged;                             // y through its tensor map
};
struct Lin8Maps { CUtensorMap x, w, y; };

// ------------------------------------------------------------------------------------------------ tokens by the tile
constexpr int L8_EPI = 8;                                 // warps that write results: two to each quarter of the tensor memory
constexpr int L8_THREADS = 32 * (2 + L8_EPI);
constexpr uint32_t L8_OUT = 4096;                         // results on their way out: 32 rows of up to 128 bytes
// BK: bytes of the contraction in a chunk, 128, or 64 where there are no more: a box that is half outside of its matrix takes longer than a full one (131072
// tokens of 64 features to 64: 14.6 us, 12.3).  CTAS: on a multiprocessor.  Two where the contraction is a few chunks: a tile's latencies are most of
// its time then.
// PAIR: two CTAs of a cluster share a tile of 256 tokens; each brings its half of the tokens and of the features, one of them issues the products for both.
template <int BN, int BK, int CTAS, bool PAIR> struct L8 {
  static constexpr int FEATURES = PAIR ? BN / 2 : BN, TOKENS = PAIR ? 256 : 128;      // brought by a CTA; of a tile
  static constexpr uint32_t A = 128 * BK, STAGE = A + FEATURES * BK;
  static constexpr int STAGES = CTAS == 1 ? 192 * 1024 / STAGE : 2, OUTS = CTAS == 2 && BK == 64 ? 2 : 1;      // stages; buffers of a writing warp
  static constexpr uint32_t RING = STAGES * STAGE;
  static constexpr uint32_t SCALES = RING + L8_EPI * OUTS * L8_OUT, BARS = SCALES + L8_EPI * 256;      // per warp: scale and bias of 32 features
  static constexpr uint32_t SMEM = BARS + 16 * STAGES + 64;
  static constexpr int ACC = 2 * BN;                      // tensor memory columns: two tiles
};
static_assert(L8<256, 128, 1, true>::SMEM <= 232448 && L8<256, 128, 1, false>::SMEM <= 232448 && L8<128, 128, 1, false>::SMEM <= 232448 && L8<64, 128, 1, false>::SMEM <= 232448 &&
              2 * (L8<128, 128, 2, false>::SMEM + 1024) <= 233472 && 2 * (L8<128, 64, 2, false>::SMEM + 1024) <= 233472 && 2 * L8<128, 128, 2, false>::ACC <= 512,
              "shared and tensor memory of a multiprocessor");

// Tiles in groups of 16 rows of tiles, column by column inside a group: the CTAs that run at a time share their operands in L2.
__device__ __forceinline__ void tile_at(const Lin8Args& a, int i, int& m, int& n) {
  const int per = 16 * a.tiles_n, group = i / per, rows_here = min(16, a.tiles_m - 16 * group), j = i - group * per;
  n = j / rows_here;
  m = 16 * group + j - n * rows_here;
}

// kind::f8f6f4: D fp32, A and B e4m3, both K-major
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint32_t pack16(float a, float b, __nv_bfloat16) { return pack_bf16(a, b); }
__device__ __forceinline__ uint32_t pack16(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack16(float, float, float) { return 0; }
__device__ __forceinline__ void st_shared16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// ---- a pair of CTAs
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {          // the same place in the pair's first CTA
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void pair_arrive(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void pair_tma_load_2d(uint32_t smem_dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_dst), "l"((uint64_t)map), "r"(cluster_bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t smem_slot, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D: 128 rows in the tensor memory of each CTA; A and B: the same places of both CTAs' shared memory, half of the rows in each
__device__ __forceinline__ void pair_mma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pair_commit(uint32_t bar) {             // on both CTAs' barriers
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// Warp 0 loads, warp 1 multiplies, the others write.  Every wait is bounded; whoever gives up leaves, and so do all that wait for it.
// PAIR: both CTAs load and write, the first one's warp 1 multiplies for both.  Its `full` barriers count the bytes of both, its `acc_empty` the writing warps
// of both; `empty` and `acc_full` are signalled in both.
template <int BN, int BK, int CTAS, bool PAIR, class Y>
__global__ void __launch_bounds__(L8_THREADS, CTAS) k_lin8(const __grid_constant__ Lin8Args a, const __grid_constant__ Lin8Maps maps) {
  using C = L8<BN, BK, CTAS, PAIR>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  const uint32_t full = sbase + C::BARS, empty = full + 8 * C::STAGES, acc_full = empty + 8 * C::STAGES, acc_empty = acc_full + 16, slot = acc_empty + 16;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int chunks = (a.K + BK - 1) / BK, tiles = a.tiles_m * a.tiles_n;
  volatile int& s_abort = *reinterpret_cast<int*>(smem_raw + (slot + 8 - sbase));
  const int rank = PAIR ? (int)cta_rank() : 0, first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
  if (warp == 0 && lane == 0) {
    s_abort = *reinterpret_cast<volatile int*>(&g_lin8_status);
    for (int i = 0; i < C::STAGES; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(acc_full + 8 * i, 1), mbar_init(acc_empty + 8 * i, PAIR ? 2 * L8_EPI : L8_EPI);
    fence_barrier_init();
    fence_proxy_async();
    tma_prefetch_desc(&maps.x);
    tma_prefetch_desc(&maps.w);
  }
  if (warp == 1) {
    if (PAIR) {
      pair_tmem_alloc(slot, C::ACC);
    } else {
      tmem_alloc(slot, C::ACC);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t*>(smem_raw + (slot - sbase));
  wait_for_kernel_before();                              // the operands of a call are often the results of the kernel before
  if (s_abort == 0) {
    if (warp == 0) {
      if (elect_one()) {
        int st = 0, ph = 1;                              // a ring that has not been used yet is empty
        long long fills = 0;
        bool ok = true;
        for (int i = first; i < tiles && ok; i += step) {
          int m, n;
          tile_at(a, i, m, n);
          for (int c = 0; c < chunks && ok; ++c) {
            ok = mbar_wait(empty + 8 * st, ph);
            if (!ok) break;
            const int row = m * C::TOKENS + rank * 128, col = n * BN + rank * C::FEATURES;
            if (PAIR) {
              if (rank == 0) mbar_expect_tx(full + 8 * st, 2 * C::STAGE);
              const uint32_t bar = in_leader(full + 8 * st);
              pair_tma_load_2d(sbase + st * C::STAGE, &maps.x, bar, c * BK, row);
              pair_tma_load_2d(sbase + st * C::STAGE + C::A, &maps.w, bar, c * BK, col);
            } else {
              mbar_expect_tx(full + 8 * st, C::STAGE);
              tma_load_2d(sbase + st * C::STAGE, &maps.x, full + 8 * st, c * BK, row);
              tma_load_2d(sbase + st * C::STAGE + C::A, &maps.w, full + 8 * st, c * BK, col);
            }
            ++fills;
            if (++st == C::STAGES) st = 0, ph ^= 1;
          }
        }
        if (!ok) {                                       // the copies under way end first (a pair's are counted in its first CTA), or this gives up again
          report(&g_lin8_status, ERR_LOAD_WAIT);
          for (long long j = fills > C::STAGES ? fills - C::STAGES : 0; j < fills && rank == 0; ++j)
            mbar_wait(full + 8 * (int)(j % C::STAGES), (int)(j / C::STAGES) & 1);
        }
      }
    } else if (warp == 1) {
      if (rank == 0 && elect_one()) {
        constexpr uint32_t idesc = idesc_e4m3(C::TOKENS, BN);
        constexpr uint32_t layout = BK == 128 ? LAYOUT_SW128 : LAYOUT_SW64;
        const uint64_t a0 = make_smem_desc(sbase, 16, 8 * BK, layout), b0 = make_smem_desc(sbase + C::A, 16, 8 * BK, layout);
        int st = 0, ph = 0, buf = 0, acc_ph = 1;
        bool ok = true;
        for (int i = first; i < tiles && ok; i += step) {
          ok = mbar_wait(acc_empty + 8 * buf, acc_ph);
          tc_fence_after();
          for (int c = 0; c < chunks && ok; ++c) {
            ok = mbar_wait(full + 8 * st, ph);
            if (!ok) break;
            tc_fence_after();
            const int left = a.K - c * BK;
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              if (32 * k < left) {
                const uint64_t ad = desc_advance(a0, st * C::STAGE + 32 * k), bd = desc_advance(b0, st * C::STAGE + 32 * k);
                if (PAIR) pair_mma_e4m3(tmem + buf * BN, ad, bd, idesc, c > 0 || k > 0);
                else mma_e4m3(tmem + buf * BN, ad, bd, idesc, c > 0 || k > 0);
              }
            if (PAIR) pair_commit(empty + 8 * st);
            else mma_commit(empty + 8 * st);
            if (++st == C::STAGES) st = 0, ph ^= 1;
          }
          if (ok) {
            if (PAIR) pair_commit(acc_full + 8 * buf);
            else mma_commit(acc_full + 8 * buf);
          }
          buf ^= 1;
          if (buf == 0) acc_ph ^= 1;
        }
        if (!ok) report(&g_lin8_status, ERR_MMA_WAIT);
      }
    } else {
      const int q = warp & 3, half = (warp - 2) >> 2, me = warp - 2;
      constexpr bool WIDE = sizeof(Y) == 4;
      constexpr int COLS = WIDE || BN == 64 ? 32 : 64, ROW = COLS * (int)sizeof(Y);      // features of a store: rows of 64 or 128 bytes
      const uint32_t out = sbase + C::RING + me * C::OUTS * L8_OUT;
      float2* const sb = reinterpret_cast<float2*>(smem_raw + C::SCALES + me * 256);
      int buf = 0, ph = 0, turn = 0, scaled = -1;
      float sx = 0.f, sw[BN / 64], b[BN / 64];
      // the scales of a tile are read while the one before is written: their way from memory is as long as a small tile's time
      auto row_scale = [&](int i) {
        int m, n;
        if (i >= tiles) return 0.f;
        tile_at(a, i, m, n);
        const int t = m * C::TOKENS + rank * 128 + q * 32 + lane;
        return t < a.T ? a.sx[t] : 0.f;
      };
      auto column_scales = [&](int i) {
        int m, n;
        if (i >= tiles) return;
        tile_at(a, i, m, n);
        if (n == scaled) return;
        scaled = n;
#pragma unroll
        for (int g = 0; g < BN / 64; ++g) {
          const int c = n * BN + half * (BN / 2) + 32 * g + lane;
          sw[g] = c < a.N ? a.sw[c] : 0.f;
          b[g] = c < a.N && a.bias != nullptr ? load_any(a.bias, a.bias_type, c) : 0.f;
        }
      };
      sx = row_scale(first);
      column_scales(first);
      for (int i = first; i < tiles; i += step) {
        int m, n;
        tile_at(a, i, m, n);
        const int c0 = n * BN + half * (BN / 2), row0 = m * C::TOKENS + rank * 128 + q * 32;
        const float next = row_scale(i + step);
        if (!tc::warp_wait(acc_full + 8 * buf, ph, &g_lin8_status, ERR_MMA2_WAIT)) break;
        tc_fence_after();
#pragma unroll
        for (int g0 = 0; g0 < BN / 2; g0 += COLS) {
          const int c = c0 + g0;
          const uint32_t tile = out + turn * L8_OUT;
          if (a.staged) {                                // the bulk store that read this buffer last has done so
            if (lane == 0) {
              if (C::OUTS == 1) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
              else asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            }
            __syncwarp();
          }
#pragma unroll
          for (int g = g0; g < g0 + COLS; g += 32) {
            uint32_t r[32];
            tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + buf * BN + half * (BN / 2) + g, r);
            __syncwarp();
            sb[lane] = make_float2(sw[g / 32], b[g / 32]);
            tmem_ld_wait();
            if (g == BN / 2 - 32) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if (PAIR) pair_arrive(in_leader(acc_empty + 8 * buf));
                else mbar_arrive(acc_empty + 8 * buf);
              }
            }
            __syncwarp();
            float v[32];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float4 f = *reinterpret_cast<const float4*>(sb + e);
              v[e] = fmaf(__uint_as_float(r[e]) * sx, f.x, f.y);
              v[e + 1] = fmaf(__uint_as_float(r[e + 1]) * sx, f.z, f.w);
            }
            // pieces of 16 bytes in the swizzle of the store's map
            const uint32_t row = tile + lane * ROW, turned = ROW == 128 ? lane & 7 : (lane >> 1) & 3;
            if constexpr (WIDE) {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                st_shared16(row + ((k ^ turned) << 4), __float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]),
                            __float_as_uint(v[4 * k + 3]));
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                st_shared16(row + (((k + (g - g0) / 8) ^ turned) << 4), pack16(v[8 * k], v[8 * k + 1], Y()), pack16(v[8 * k + 2], v[8 * k + 3], Y()),
                            pack16(v[8 * k + 4], v[8 * k + 5], Y()), pack16(v[8 * k + 6], v[8 * k + 7], Y()));
            }
          }
          if (a.staged) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0 && c < a.N && row0 < a.T) tma_store_2d(&maps.y, tile, c, row0);
            if (lane == 0) bulk_commit();
          } else {                                       // rows that start anywhere: lanes side by side along each
            __syncwarp();
            const uint8_t* const from = smem_raw + (tile - sbase);
            const int rows_here = min(32, a.T - row0);
            constexpr int PER = 16 / (int)sizeof(Y);     // elements of a piece
#pragma unroll
            for (int g = 0; g < COLS; g += 32) {
              const int e = g + lane;
              Y* const y = static_cast<Y*>(a.y) + (long long)row0 * a.ldy + c + e;
              if (c + e < a.N)
                for (int r = 0; r < rows_here; ++r)
                  y[r * a.ldy] = *reinterpret_cast<const Y*>(from + r * ROW + (((e / PER) ^ (ROW == 128 ? r & 7 : (r >> 1) & 3)) << 4) + e % PER * (int)sizeof(Y));
            }
            __syncwarp();
          }
          if (C::OUTS == 2) turn ^= 1;
        }
        sx = next;
        column_scales(i + step);
        buf ^= 1;
        if (buf == 0) ph ^= 1;
      }
      if (a.staged && lane == 0) bulk_wait_all();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();                              // neither CTA's memory goes while the other may signal in it
  tc_fence_after();
  if (warp == 1) {
    if (PAIR) pair_tmem_dealloc(tmem, C::ACC);
    else tmem_dealloc(tmem, C::ACC);
  }
}

// ------------------------------------------------------------------------------------------------ few tokens
constexpr int FEW_WARPS = 8, FEW_ROWS = 16;
constexpr int FEW_TOKENS = 8, FEW_CHUNK = 2048, FEW_LD = FEW_CHUNK + 64;      // bytes of a row at a time; rows in shared memory: eight lanes read two without conflict
constexpr uint32_t FEW_STAGE = (FEW_ROWS + FEW_TOKENS) * FEW_LD, FEW_SMEM = 2 * FEW_STAGE + 64;
// the last K % 16 bytes of a row
__device__ __forceinline__ uint4 load_tail(bool in, const uint8_t* p, int count) {
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (in && i < count) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void mma_16x8x32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void multiply(uint4 u, uint4 v, uint4 x, float (&d)[4]) {
  mma_16x8x32(d, u.x, v.x, u.y, v.y, x.x, x.y);
  mma_16x8x32(d, u.z, v.z, u.w, v.w, x.z, x.w);
}
// A CTA has 16 features.  Bulk copies bring 2048 bytes of each feature's and each token's row at a time, twice that is under way; the CTA's warps take every
// eighth piece of 64.  Which four bytes of a lane's 16 the product takes for which index of the contraction does not matter as long as tokens and weights
// agree, so a lane's words are used as they come.  Loads to registers instead were ordered one behind another by the compiler (one token, 4096 to 4096
// features, a graph of one call: 10.3 us, so 8.6; in a row of calls 5.5, 3.0 TB/s of weights, where launch and first bytes are most of the time).
template <class Y>
__global__ void __launch_bounds__(32 * FEW_WARPS) k_lin8_few(const __grid_constant__ Lin8Args a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ float part[FEW_WARPS][FEW_ROWS][FEW_TOKENS + 1];
  const uint32_t rows0 = smem_u32(smem_raw), bars = rows0 + 2 * FEW_STAGE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, k0 = (lane & 3) * 16;
  const int n0 = blockIdx.x * FEW_ROWS, whole = a.K & ~15, chunks = (whole + FEW_CHUNK - 1) / FEW_CHUNK;
  const int features = min(FEW_ROWS, a.N - n0);
  // rows that do not exist stay what is there: they meet no row that does
  auto fill = [&](int c) {                               // one warp
    const int st = c & 1, bytes = min(FEW_CHUNK, whole - c * FEW_CHUNK);
    if (lane == 0) mbar_expect_tx(bars + 8 * st, (features + a.T) * (uint32_t)bytes);
    __syncwarp();
    const uint32_t to = rows0 + st * FEW_STAGE;
    if (lane < features) bulk_load(to + lane * FEW_LD, a.w + (long long)(n0 + lane) * a.ldw + c * FEW_CHUNK, bars + 8 * st, bytes);
    if (lane < a.T) bulk_load(to + (FEW_ROWS + lane) * FEW_LD, a.x + (long long)lane * a.ldx + c * FEW_CHUNK, bars + 8 * st, bytes);
  };
  if (threadIdx.x == 0) {
    mbar_init(bars, 1);
    mbar_init(bars + 8, 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  const int lost = *reinterpret_cast<volatile int*>(&g_lin8_status);
  wait_for_kernel_before();
  if (__syncthreads_or(lost)) return;
  if (warp == 0)
    for (int c = 0; c < min(chunks, 2); ++c) fill(c);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < chunks; ++c) {
    const int st = c & 1, bytes = min(FEW_CHUNK, whole - c * FEW_CHUNK);
    if (!__syncthreads_and(mbar_wait(bars + 8 * st, (c >> 1) & 1))) {
      if (threadIdx.x == 0) {
        report(&g_lin8_status, ERR_LOAD_WAIT);
        if (c + 1 < chunks) mbar_wait(bars + 8 * (st ^ 1), ((c + 1) >> 1) & 1);      // the copies under way end first, or this gives up again
      }
      return;
    }
    const uint8_t* const from = smem_raw + st * FEW_STAGE + g * FEW_LD + k0;
#pragma unroll
    for (int d = 0; d < FEW_CHUNK / 64 / FEW_WARPS; ++d) {
      const int k = (warp + d * FEW_WARPS) * 64;
      if (k >= bytes) break;
      const bool in = k + k0 < bytes;
      const uint4 none = make_uint4(0, 0, 0, 0);
      const uint4 u = in ? *reinterpret_cast<const uint4*>(from + k) : none, v = in ? *reinterpret_cast<const uint4*>(from + 8 * FEW_LD + k) : none;
      multiply(u, v, in ? *reinterpret_cast<const uint4*>(from + FEW_ROWS * FEW_LD + k) : none, acc);
    }
    if (c + 2 < chunks) {
      __syncthreads();                                   // all warps are done with this half
      if (warp == 0) fill(c + 2);
    }
  }
  if (whole < a.K && warp == 0) {
    const uint8_t* const w = a.w + (long long)(n0 + g) * a.ldw + whole;
    const uint4 u = load_tail(g < features && k0 == 0, w, a.K - whole), v = load_tail(g + 8 < features && k0 == 0, w + 8 * a.ldw, a.K - whole);
    multiply(u, v, load_tail(g < a.T && k0 == 0, a.x + (long long)g * a.ldx + whole, a.K - whole), acc);
  }
  const int t0 = 2 * (lane & 3);
  part[warp][g][t0] = acc[0], part[warp][g][t0 + 1] = acc[1];
  part[warp][g + 8][t0] = acc[2], part[warp][g + 8][t0 + 1] = acc[3];
  __syncthreads();
  for (int i = threadIdx.x; i < FEW_ROWS * FEW_TOKENS; i += 32 * FEW_WARPS) {
    const int row = i & (FEW_ROWS - 1), t = i / FEW_ROWS, c = blockIdx.x * FEW_ROWS + row;
    if (t >= a.T || c >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < FEW_WARPS; ++k) s += part[k][row][t];
    const float b = a.bias != nullptr ? load_any(a.bias, a.bias_type, c) : 0.f;
    static_cast<Y*>(a.y)[(long long)t * a.ldy + c] = rounded<Y>(fmaf(s * a.sx[t], a.sw[c], b));
  }
}

// ------------------------------------------------------------------------------------------------ host
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                            CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int encoder(Encode* out) {
  static std::atomic<Encode> known{nullptr};
  Encode e = known.load();
  if (e == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    SPION_CUDA_TRY(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
    if (q != cudaDriverEntryPointSuccess || fn == nullptr) return SPION_ERR_CUDA;
    known.store(e = reinterpret_cast<Encode>(fn));
  }
  *out = e;
  return SPION_OK;
}
int map_of(CUtensorMap* m, Encode encode, const void* base, int type, long long cols, long long rows_, long long ld, int box_cols, int box_rows) {
  const int size = type_size(type);
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows_}, strides[1] = {(cuuint64_t)ld * size};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, step[2] = {1, 1};
  const CUtensorMapDataType kind = type == SPION_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == SPION_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : type == SPION_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = encode(m, kind, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            box_cols * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    fprintf(stderr, "spion_b200: cuTensorMapEncodeTiled failed (%d) rows=%lld cols=%lld\n", (int)r, rows_, cols);
    return SPION_ERR_CUDA;
  }
  return SPION_OK;
}

// once per kernel (the static of this instance) and device
template <auto Kernel> int big_shared_memory_of(uint32_t bytes) {
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  SPION_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    SPION_CUDA_TRY(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  return SPION_OK;
}
template <int BN, int BK, int CTAS, bool PAIR, class Y> int launch_tiles(Lin8Args a, cudaStream_t st) {
  using C = L8<BN, BK, CTAS, PAIR>;
  Encode encode;
  int rc = encoder(&encode);
  if (rc != SPION_OK) return rc;
  a.tiles_m = (a.T + C::TOKENS - 1) / C::TOKENS;
  a.tiles_n = (a.N + BN - 1) / BN;
  if ((long long)a.tiles_m * a.tiles_n > 0x7fffffff) return SPION_ERR_SHAPE;
  // (a store ends on a piece of 16 bytes: of a row that ends inside one it would write zeros behind the row)
  a.staged = ((uintptr_t)a.y % 16 == 0) && (a.ldy * (long long)sizeof(Y)) % 16 == 0 && (a.N * (long long)sizeof(Y)) % 16 == 0;
  Lin8Maps maps;
  if ((rc = map_of(&maps.x, encode, a.x, SPION_E4M3, a.K, a.T, a.ldx, BK, 128)) != SPION_OK) return rc;
  if ((rc = map_of(&maps.w, encode, a.w, SPION_E4M3, a.K, a.N, a.ldw, BK, C::FEATURES)) != SPION_OK) return rc;
  if (a.staged) {
    if ((rc = map_of(&maps.y, encode, a.y, type_code<Y>(), a.N, a.T, a.ldy, sizeof(Y) == 4 || BN == 64 ? 32 : 64, 32)) != SPION_OK) return rc;
  } else {
    maps.y = maps.x;                                     // not used
  }
  if ((rc = big_shared_memory_of<k_lin8<BN, BK, CTAS, PAIR, Y>>(C::SMEM)) != SPION_OK) return rc;
  const int tiles = a.tiles_m * a.tiles_n;
  if constexpr (PAIR) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = dim3(L8_THREADS), cfg.dynamicSmemBytes = C::SMEM, cfg.stream = st, cfg.attrs = at;
    // as many pairs as the device holds at a time (multiprocessors are paired inside their groups): the tiles are shared out evenly among those
    static std::atomic<int> pairs[64];
    int dev = 0;
    SPION_CUDA_TRY(cudaGetDevice(&dev));
    int n = dev < 64 ? pairs[dev].load() : 0;
    if (n == 0) {
      cfg.gridDim = dim3(2 * (sm_count() / 2)), cfg.numAttrs = 1;
      SPION_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, k_lin8<BN, BK, CTAS, PAIR, Y>, &cfg));
      if (n <= 0) return SPION_ERR_UNSUPPORTED;
      if (dev < 64) pairs[dev].store(n);
    }
    cfg.gridDim = dim3(2 * std::min(tiles, n)), cfg.numAttrs = 2;
    SPION_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_lin8<BN, BK, CTAS, PAIR, Y>, (const Lin8Args)a, (const Lin8Maps)maps));
    return SPION_OK;
  }
  SPION_CUDA_TRY(launch_after(k_lin8<BN, BK, CTAS, PAIR, Y>, dim3(std::min(tiles, sm_count() * CTAS)), dim3(L8_THREADS), C::SMEM, st, a, maps));
  return SPION_OK;
}
template <class Y> int launch_few(const Lin8Args& a, cudaStream_t st) {
  const int rc = big_shared_memory_of<k_lin8_few<Y>>(FEW_SMEM);
  if (rc != SPION_OK) return rc;
  SPION_CUDA_TRY(launch_after(k_lin8_few<Y>, dim3((a.N + FEW_ROWS - 1) / FEW_ROWS), dim3(32 * FEW_WARPS), FEW_SMEM, st, a));
  return SPION_OK;
}
template <class Y> int launch_any(const Lin8Args& a, cudaStream_t st) {
  // 4096 to 4096 features, few / tiles: 8 tokens 6.1 us / 11.6, 16 tokens (twice the products) 10.4 / 11.6; 512 to 16384, 32 tokens 26 / 6.3: mma.sync is slow on
  // 8-bit operands here, and what it does for more tokens outlasts the weights
  if (a.T <= FEW_TOKENS) return launch_few<Y>(a, st);
  // The largest tile that leaves one to every multiprocessor.  Pairs from more than 512 inner features on, two small CTAs a multiprocessor below; two small / pairs:
  // 65536 x 256 to 256 13.4 us / 16.7, x 384 to 1024 43.1 / 49.1, x 512 to 256 18.6 / 19.8 and to 1024 49.3 / 50.7; 8192 x 640 to 4096 29.9 / 29.6, 32768 x 768 to
  // 1024 35.4 / 30.8, x 1024 to 1024 42.9 / 33.8.  Where there are too few tiles of pairs, one CTA a multiprocessor from more than 256 on, two / one: 20000 x 320 to 64
  // 5.5 / 6.1, 131072 x 512 to 64 17.7 / 17.1, 512 x 320 to 1024 3.9 / 3.7.
  const long long rows_ = (a.T + 127) / 128, sms = sm_count();
  const bool wide = a.N > 64 && rows_ * ((a.N + 127) / 128) >= sms;
  if (a.K <= 64) return wide ? launch_tiles<128, 64, 2, false, Y>(a, st) : launch_tiles<64, 64, 2, false, Y>(a, st);
  if (a.K <= 256) return wide ? launch_tiles<128, 128, 2, false, Y>(a, st) : launch_tiles<64, 128, 2, false, Y>(a, st);
  if (a.N > 128 && rows_ * ((a.N + 255) / 256) >= sms) return a.K <= 512 ? launch_tiles<128, 128, 2, false, Y>(a, st) : launch_tiles<256, 128, 1, true, Y>(a, st);
  return wide ? launch_tiles<128, 128, 1, false, Y>(a, st) : launch_tiles<64, 128, 1, false, Y>(a, st);
}

}  // namespace

int* linear_e4m3_status_word() {
  void* word = nullptr;
  return cudaGetSymbolAddress(&word, g_lin8_status) == cudaSuccess ? static_cast<int*>(word) : nullptr;
}

extern "C" int spion_linear_e4m3(const void* x, long long ldx, const float* x_scale, const void* w, long long ldw, const float* w_scale, const void* bias,
                                 int bias_type, void* y, long long ldy, int y_type, long long T, int K, int N, void* cuda_stream) {
  if (T < 0 || K <= 0 || N <= 0) return SPION_ERR_ARG;
  if (T == 0) return SPION_OK;
  if (x == nullptr || x_scale == nullptr || w == nullptr || w_scale == nullptr || y == nullptr) return SPION_ERR_ARG;
  if (bias != nullptr && bias_type != SPION_F32 && bias_type != SPION_BF16 && bias_type != SPION_F16) return SPION_ERR_ARG;
  if (ldx < K || ldw < K || ldy < N || ((uintptr_t)x | (uintptr_t)w | (uintptr_t)ldx | (uintptr_t)ldw) % 16 != 0) return SPION_ERR_ARG;
  if (T > 0x7fffffff - 256 || K > 0x7fffffff - 256 || N > 0x7fffffff - 256) return SPION_ERR_SHAPE;
  const Lin8Args a = {static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(w), ldx, ldw, x_scale, w_scale, bias, bias_type, y, ldy, (int)T, K, N, 0, 0, 0};
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  if (y_type == SPION_F32) return launch_any<float>(a, st);
  if (y_type == SPION_BF16) return launch_any<__nv_bfloat16>(a, st);
  if (y_type == SPION_F16) return launch_any<__half>(a, st);
  return SPION_ERR_UNSUPPORTED;
}
