// Linear layer on 8-bit operands: y[t, n] = (sum_k xq[t, k] wq[n, k]) sx[t] sw[n] + b[n], xq and wq in e4m3 with a scale per row (rmsnorm.cu writes both),
// y in fp32, bf16 or fp16.
//
//   k_lin8        tcgen05 kind::f8f6f4, 128 tokens x BN features per tile, accumulators in tensor memory
//   k_lin8_few    up to 32 tokens, where the weights are all there is to read: mma.sync on fragments that go from global memory to registers
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
constexpr uint32_t L8_A = 128 * 128;                      // bytes of a chunk of tokens: 128 rows, 128 of the contraction
constexpr uint32_t L8_RING = 192 * 1024;
constexpr uint32_t L8_OUT = 4096;                         // per writing warp: results on their way out
template <int BN> struct L8 {
  static constexpr uint32_t STAGE = L8_A + BN * 128;
  static constexpr int STAGES = L8_RING / STAGE;
  static constexpr uint32_t BARS = L8_RING + L8_EPI * (L8_OUT + 256);      // 256: scale and bias of 32 features
  static constexpr uint32_t SMEM = BARS + 16 * STAGES + 64;
  static constexpr int ACC = 2 * BN;                      // tensor memory columns: two tiles
};
static_assert(L8<256>::SMEM <= 232448 && L8<128>::SMEM <= 232448 && L8<64>::SMEM <= 232448, "shared memory of a CTA");

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

// Warp 0 loads, warp 1 multiplies, the others write.  Every wait is bounded; whoever gives up leaves, and so do all that wait for it.
template <int BN, class Y>
__global__ void __launch_bounds__(L8_THREADS, 1) k_lin8(const __grid_constant__ Lin8Args a, const __grid_constant__ Lin8Maps maps) {
  using C = L8<BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  const uint32_t full = sbase + C::BARS, empty = full + 8 * C::STAGES, acc_full = empty + 8 * C::STAGES, acc_empty = acc_full + 16, slot = acc_empty + 16;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int chunks = (a.K + 127) >> 7, tiles = a.tiles_m * a.tiles_n;
  volatile int& s_abort = *reinterpret_cast<int*>(smem_raw + (slot + 8 - sbase));
  if (warp == 0 && lane == 0) {
    s_abort = *reinterpret_cast<volatile int*>(&g_lin8_status);
    for (int i = 0; i < C::STAGES; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(acc_full + 8 * i, 1), mbar_init(acc_empty + 8 * i, L8_EPI);
    fence_barrier_init();
    fence_proxy_async();
    tma_prefetch_desc(&maps.x);
    tma_prefetch_desc(&maps.w);
  }
  if (warp == 1) {
    tmem_alloc(slot, C::ACC);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t*>(smem_raw + (slot - sbase));
  wait_for_kernel_before();                              // the operands of a call are often the results of the kernel before
  if (s_abort == 0) {
    if (warp == 0) {
      if (elect_one()) {
        int st = 0, ph = 1;                              // a ring that has not been used yet is empty
        bool ok = true;
        for (int i = blockIdx.x; i < tiles && ok; i += gridDim.x) {
          int m, n;
          tile_at(a, i, m, n);
          for (int c = 0; c < chunks && ok; ++c) {
            ok = mbar_wait(empty + 8 * st, ph);
            if (!ok) break;
            mbar_expect_tx(full + 8 * st, C::STAGE);
            tma_load_2d(sbase + st * C::STAGE, &maps.x, full + 8 * st, c * 128, m * 128);
            tma_load_2d(sbase + st * C::STAGE + L8_A, &maps.w, full + 8 * st, c * 128, n * BN);
            if (++st == C::STAGES) st = 0, ph ^= 1;
          }
        }
        if (!ok) report(&g_lin8_status, ERR_LOAD_WAIT);
      }
    } else if (warp == 1) {
      if (elect_one()) {
        constexpr uint32_t idesc = idesc_e4m3(128, BN);
        const uint64_t a0 = make_smem_desc(sbase, 16, 1024, LAYOUT_SW128), b0 = make_smem_desc(sbase + L8_A, 16, 1024, LAYOUT_SW128);
        int st = 0, ph = 0, buf = 0, acc_ph = 1;
        bool ok = true;
        for (int i = blockIdx.x; i < tiles && ok; i += gridDim.x) {
          ok = mbar_wait(acc_empty + 8 * buf, acc_ph);
          tc_fence_after();
          for (int c = 0; c < chunks && ok; ++c) {
            ok = mbar_wait(full + 8 * st, ph);
            if (!ok) break;
            tc_fence_after();
            const int left = a.K - c * 128;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (32 * k < left)
                mma_e4m3(tmem + buf * BN, desc_advance(a0, st * C::STAGE + 32 * k), desc_advance(b0, st * C::STAGE + 32 * k), idesc, c > 0 || k > 0);
            mma_commit(empty + 8 * st);
            if (++st == C::STAGES) st = 0, ph ^= 1;
          }
          if (ok) mma_commit(acc_full + 8 * buf);
          buf ^= 1;
          if (buf == 0) acc_ph ^= 1;
        }
        if (!ok) report(&g_lin8_status, ERR_MMA_WAIT);
      }
    } else {
      const int q = warp & 3, half = (warp - 2) >> 2, me = warp - 2;
      const uint32_t out = sbase + L8_RING + me * L8_OUT;
      float2* const sb = reinterpret_cast<float2*>(smem_raw + L8_RING + L8_EPI * L8_OUT + me * 256);
      int buf = 0, ph = 0, turn = 0;
      for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
        int m, n;
        tile_at(a, i, m, n);
        const int t = m * 128 + q * 32 + lane, c0 = n * BN + half * (BN / 2);
        const float sx = t < a.T ? a.sx[t] : 0.f;
        float sw[BN / 64], b[BN / 64];
#pragma unroll
        for (int g = 0; g < BN / 64; ++g) {
          const int c = c0 + 32 * g + lane;
          sw[g] = c < a.N ? a.sw[c] : 0.f;
          b[g] = c < a.N && a.bias != nullptr ? load_any(a.bias, a.bias_type, c) : 0.f;
        }
        if (!tc::warp_wait(acc_full + 8 * buf, ph, &g_lin8_status, ERR_MMA2_WAIT)) break;
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < BN / 64; ++g) {
          const int c = c0 + 32 * g;
          uint32_t r[32];
          tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + buf * BN + half * (BN / 2) + 32 * g, r);
          sb[lane] = make_float2(sw[g], b[g]);
          tmem_ld_wait();
          if (g == BN / 64 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty + 8 * buf);
          }
          __syncwarp();
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float4 f = *reinterpret_cast<const float4*>(sb + e);
            v[e] = fmaf(__uint_as_float(r[e]) * sx, f.x, f.y);
            v[e + 1] = fmaf(__uint_as_float(r[e + 1]) * sx, f.z, f.w);
          }
          if (c >= a.N) { __syncwarp(); continue; }
          constexpr bool WIDE = sizeof(Y) == 4;
          const uint32_t tile = out + (WIDE ? 0 : (turn & 1) * 2048);
          if (a.staged) {                                // the bulk store that read this buffer last has done so
            if (lane == 0) {
              if (WIDE) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
              else asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            }
            __syncwarp();
          }
          if constexpr (WIDE) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              st_shared16(tile + lane * 128 + ((k ^ (lane & 7)) << 4), __float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]),
                          __float_as_uint(v[4 * k + 2]), __float_as_uint(v[4 * k + 3]));
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              st_shared16(tile + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4), pack16(v[8 * k], v[8 * k + 1], Y()), pack16(v[8 * k + 2], v[8 * k + 3], Y()),
                          pack16(v[8 * k + 4], v[8 * k + 5], Y()), pack16(v[8 * k + 6], v[8 * k + 7], Y()));
          }
          if (a.staged) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&maps.y, tile, c, m * 128 + q * 32);
              bulk_commit();
            }
          } else {                                       // rows that start anywhere: lanes side by side along each
            __syncwarp();
            const uint8_t* const from = smem_raw + (tile - sbase);
            Y* const y = static_cast<Y*>(a.y) + (long long)(m * 128 + q * 32) * a.ldy + c + lane;
            const int rows_here = min(32, a.T - (m * 128 + q * 32));
            if (c + lane < a.N)
              for (int row = 0; row < rows_here; ++row) {
                const uint32_t at = WIDE ? row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4
                                         : row * 64 + (((lane >> 3) ^ ((row >> 1) & 3)) << 4) + (lane & 7) * 2;
                y[row * a.ldy] = *reinterpret_cast<const Y*>(from + at);
              }
            __syncwarp();
          }
          ++turn;
        }
        buf ^= 1;
        if (buf == 0) ph ^= 1;
      }
      if (a.staged && lane == 0) bulk_wait_all();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::ACC);
}

// ------------------------------------------------------------------------------------------------ few tokens
constexpr int FEW_WARPS = 8, FEW_ROWS = 16, FEW_DEPTH = 4;
__device__ __forceinline__ uint4 zero4() { return make_uint4(0, 0, 0, 0); }
// sixteen bytes from place k of a row of K, zeros behind its end
__device__ __forceinline__ uint4 load_row16(const uint8_t* row, int k, int K, bool in) {
  if (!in || k >= K) return zero4();
  if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < K - k; ++i) w[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void mma_16x8x32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A CTA has 16 features, its warps take every eighth piece of 64 of the contraction.  Four lanes read 64 bytes of a row side by side; which four of a lane's 16
// bytes the product takes for which index of the contraction does not matter as long as tokens and weights agree, so a lane's words are used as they come.
template <int NT, class Y>
__global__ void __launch_bounds__(32 * FEW_WARPS) k_lin8_few(const __grid_constant__ Lin8Args a) {
  __shared__ float part[FEW_WARPS][FEW_ROWS][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, k0 = (lane & 3) * 16;
  const int n = blockIdx.x * FEW_ROWS + g;
  const uint8_t* const w0 = a.w + (long long)n * a.ldw;
  const uint8_t* const w1 = w0 + 8 * a.ldw;
  const bool in0 = n < a.N, in1 = n + 8 < a.N;
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  const int pieces = (a.K + 63) >> 6;
  wait_for_kernel_before();
  for (int p0 = warp; p0 < pieces; p0 += FEW_WARPS * FEW_DEPTH) {
    uint4 u[FEW_DEPTH], v[FEW_DEPTH], x[FEW_DEPTH][NT];
#pragma unroll
    for (int d = 0; d < FEW_DEPTH; ++d) {
      const int k = (p0 + d * FEW_WARPS) * 64 + k0;
      u[d] = load_row16(w0, k, a.K, in0);
      v[d] = load_row16(w1, k, a.K, in1);
    }
#pragma unroll
    for (int d = 0; d < FEW_DEPTH; ++d) {
      const int k = (p0 + d * FEW_WARPS) * 64 + k0;
#pragma unroll
      for (int j = 0; j < NT; ++j) x[d][j] = load_row16(a.x + (long long)(8 * j + g) * a.ldx, k, a.K, 8 * j + g < a.T);
    }
#pragma unroll
    for (int d = 0; d < FEW_DEPTH; ++d)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma_16x8x32(acc[j], u[d].x, v[d].x, u[d].y, v[d].y, x[d][j].x, x[d][j].y);
        mma_16x8x32(acc[j], u[d].z, v[d].z, u[d].w, v[d].w, x[d][j].z, x[d][j].w);
      }
  }
  const int t0 = 2 * (lane & 3);
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    part[warp][g][8 * j + t0] = acc[j][0], part[warp][g][8 * j + t0 + 1] = acc[j][1];
    part[warp][g + 8][8 * j + t0] = acc[j][2], part[warp][g + 8][8 * j + t0 + 1] = acc[j][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < FEW_ROWS * 8 * NT; i += 32 * FEW_WARPS) {
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

template <int BN, class Y> int launch_tiles(Lin8Args a, cudaStream_t st) {
  Encode encode;
  int rc = encoder(&encode);
  if (rc != SPION_OK) return rc;
  a.tiles_m = (a.T + 127) / 128;
  a.tiles_n = (a.N + BN - 1) / BN;
  if ((long long)a.tiles_m * a.tiles_n > 0x7fffffff) return SPION_ERR_SHAPE;
  a.staged = ((uintptr_t)a.y % 16 == 0) && (a.ldy * (long long)sizeof(Y)) % 16 == 0;
  Lin8Maps maps;
  if ((rc = map_of(&maps.x, encode, a.x, SPION_E4M3, a.K, a.T, a.ldx, 128, 128)) != SPION_OK) return rc;
  if ((rc = map_of(&maps.w, encode, a.w, SPION_E4M3, a.K, a.N, a.ldw, 128, BN)) != SPION_OK) return rc;
  if (a.staged) {
    if ((rc = map_of(&maps.y, encode, a.y, type_code<Y>(), a.N, a.T, a.ldy, 32, 32)) != SPION_OK) return rc;
  } else {
    maps.y = maps.x;                                     // not used
  }
  static std::atomic<uint64_t> ready{0};                 // devices on which the kernel has its shared memory
  int dev = 0;
  SPION_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    SPION_CUDA_TRY(cudaFuncSetAttribute(k_lin8<BN, Y>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L8<BN>::SMEM));
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  const int tiles = a.tiles_m * a.tiles_n;
  SPION_CUDA_TRY(launch_after(k_lin8<BN, Y>, dim3(std::min(tiles, sm_count())), dim3(L8_THREADS), L8<BN>::SMEM, st, a, maps));
  return SPION_OK;
}
template <class Y> int launch_any(const Lin8Args& a, cudaStream_t st) {
  if (a.T <= 32) {
    const dim3 grid((a.N + FEW_ROWS - 1) / FEW_ROWS), block(32 * FEW_WARPS);
    if (a.T <= 8) SPION_CUDA_TRY(launch_after(k_lin8_few<1, Y>, grid, block, 0, st, a));
    else if (a.T <= 16) SPION_CUDA_TRY(launch_after(k_lin8_few<2, Y>, grid, block, 0, st, a));
    else SPION_CUDA_TRY(launch_after(k_lin8_few<4, Y>, grid, block, 0, st, a));
    return SPION_OK;
  }
  const long long rows_ = (a.T + 127) / 128, sms = sm_count();
  if (a.N > 128 && rows_ * ((a.N + 255) / 256) >= sms) return launch_tiles<256, Y>(a, st);
  if (a.N > 64 && rows_ * ((a.N + 127) / 128) >= sms) return launch_tiles<128, Y>(a, st);
  return launch_tiles<64, Y>(a, st);
}

}  // namespace

// Status word of these kernels on the current device, after the work of a stream (linear.cu reports it with its own)
int linear_e4m3_status(int reset, cudaStream_t st) {
  int v = 0;
  SPION_CUDA_TRY(cudaMemcpyFromSymbolAsync(&v, g_lin8_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
  SPION_CUDA_TRY(cudaStreamSynchronize(st));
  if (v == 0) return SPION_OK;
  if (reset) {
    void* word = nullptr;
    SPION_CUDA_TRY(cudaGetSymbolAddress(&word, g_lin8_status));
    SPION_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(int), st));
    SPION_CUDA_TRY(cudaStreamSynchronize(st));
  }
  fprintf(stderr, "spion_b200: status word of the 8-bit linear layers = 0x%x (a bounded wait gave up)\n", v);
  return SPION_ERR_TIMEOUT;
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
