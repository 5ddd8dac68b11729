// Root-mean-square norm over the last dimension of [M, N] rows, with the residual's addition before it, forward and backward, and the same with
// rows of e4m3 and a scale each as output (what the 8-bit linear layers read).
//
//   s = round(x + r)      rho = (mean_c s_c^2 + eps)^(-1/2)      y_c = s_c w_c rho
//   e4m3: a = max(max_c |y_c|, 2^-100), q_c = e4m3(y_c (448 (1 / a))), scale = a / 448; without a norm (rows to e4m3) y = x
//   backward: n = s rho, c = mean_c(dy_c w_c n_c), dx = rho (dy w - n c) + ds, dw_c = sum over rows of dy_c n_c
//
// Bound by the passes over the token matrices: a row is read once into registers, everything that the row's sums are needed for follows from there.
// Statistics are fp32 sums.  The norm of a 16-bit stream is that of the rounded sum, which is what the next layer and the backward see.  The largest
// |y| is the largest |s w| times rho, rounding included, because rounding keeps the order: sum and maximum take one reduction.
//
// Threads of a row: in the forward 8 lanes up to 256 values, a warp up to 1024, then a CTA of as few threads as hold it in four pieces each; a row that no
// register file holds is read twice.  The backward keeps twice as much: 8 lanes up to 128 values, a warp up to 512, then a CTA with a thread to a piece behind
// a ring (two pieces beyond 8192 values).  us for 33.5 million values, bf16 with a residual / fp32 with bf16 branches, and by the next wider split in brackets:
//   values     forward                             backward
//      128     46.5 (83.4) / 67.4 (83.8)           47.1 (108) / 73.5 (120)
//      256     56.5 (70.8) / 67.0 (68.9)           63.6 (157) / 81.0 (182)
//      512     49.2 (83.7) / 64.3 (64.8)           47.3 (86.2) / 73.6 (106)
//     1024     57.1 (53.4) / 63.8 (65.1)           52.4 (65.6) / 76.8 (79.6)
//     2048     44.8 (54.9) / 64.8 (66.7)           46.3 (67.7) / 78.0 (72.9)
//     4096     44.7 (61.1) / 64.7 (67.9)           46.5 (71.8) / 76.8 (77.9)
//     8192     46.5 (68.2) / 63.8 (72.0)           47.1 (66.7) / 74.3 (84.0)
//    16384     50.6 (62.2) / 65.2 (78.1)           51.5 (138) / 148: two rows of fp32 with their residual's gradient do not fit the ring
// Three forwards of two rows at a time by 8 lanes (16-bit rows up to 64 values) spill 8 to 24 bytes under their bound of four CTAs a multiprocessor.
//
// Pieces of eight elements where every row starts on the boundary of such a piece, single elements otherwise (odd widths).  The number of
// threads of a row is a constant of each kernel, so a piece's place costs no arithmetic.
//
// Measured, of a copy's 6.54 TB/s: 32768 x 2048 bf16 + residual to e4m3 75 us (96 %); both directions: 131072 x 64 fp32 with bf16 branches 39 us (92 %), 8192 x
// 4096 bf16 89 us (92 %), 4096 x 16384 bf16 181 us (90 %); by single elements 4099 x 769 fp32 21 us (37 %), 8192 x 2001 bf16 74 us (55 %): four and two bytes
// an access, and their addresses.  One row of 4096: 2.2 us, a launch.
#include <algorithm>
#include <atomic>

#include "rows.cuh"
#include "tc_ptx.cuh"

using namespace rows;

namespace {

constexpr float SMALL = 0x1p-100f;        // what the scale of a row of zeros follows
constexpr int CTA = 256;                  // threads of a CTA whose warps take rows of their own
constexpr int MAX_PARTS = 1184;           // partial rows of a weight gradient: eight per multiprocessor of 148

// Set by a bounded wait that gave up (the ring of the backward).  The gradients of the rows that its CTA had left are NaN then, and so are all of the launches
// after it until spion_linear_status has reported it.
__device__ int g_rms_status;

struct FwdArgs {
  const void* x; long long ldx;
  const void* r; long long ldr;           // or null
  const void* w; int w_type;              // null: ones
  void* s;                                // [M, N], with r
  void* y; long long ldy;
  float* scale;                           // e4m3: [M]
  float* rho;                             // or null
  long long M; int N; float eps;
  int norm;                               // 0: y = x
};

// (all loads first: a conversion beside its load would wait for it)
template <class W, int VEC, int NV, int TPR> __device__ __forceinline__ void load_weights_of(const W* p, int N, int t, float (&w)[NV * VEC]) {
  Piece<W, VEC> q[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * VEC;
    if (c < N) q[i].load(p + c);
    else q[i].zero();
  }
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) w[i] = q[i / VEC].at(i % VEC);
}
template <int VEC, int NV, int TPR> __device__ __forceinline__ void load_weights(const void* p, int type, int N, int t, float (&w)[NV * VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < NV * VEC; ++i) w[i] = 1.f;
  } else if (type == SPION_F32) {
    load_weights_of<float, VEC, NV, TPR>(static_cast<const float*>(p), N, t, w);
  } else if (type == SPION_BF16) {
    load_weights_of<__nv_bfloat16, VEC, NV, TPR>(static_cast<const __nv_bfloat16*>(p), N, t, w);
  } else {
    load_weights_of<__half, VEC, NV, TPR>(static_cast<const __half*>(p), N, t, w);
  }
}

// e4m3: what y is multiplied with, and the row's scale.  A row with a NaN has the scale NaN, one with an infinity an infinite scale and zeros beside
// NaN: no value of such a row comes back finite.
__device__ __forceinline__ float row_scale(float top, float& scale) {
  const float a = top < SMALL ? SMALL : top;             // (NaN stays)
  scale = a * (1.f / 448.f);
  return 448.f * __frcp_rn(a);
}

// TPR threads to a row: 8 or 32 lanes of a warp, more: a CTA of that many.  Lanes take UR rows at a time, so that enough bytes are in flight.
// NORM false: rows to e4m3 as they are (131072 x 64 bf16: 9.6 us with the sums and products of the norm left in, 8.7 without, a launch among them: 6.5 in a row of calls).
template <bool NORM, class S, class R, class Y, int VEC, int NV, int TPR, int UR>
__global__ void __launch_bounds__(TPR <= 32 ? CTA : TPR, VEC != 8 ? 1 : TPR == 8 && NV <= 2 ? 4 : TPR > 32 && NV == 4 ? 640 / TPR : 1) k_rms_forward(const FwdArgs a) {
  next_may_start();                                                        // a linear layer on 8-bit rows prepares itself beside the last CTAs
  constexpr bool Q = type_code<Y>() == SPION_E4M3;
  constexpr int THREADS = TPR <= 32 ? CTA : TPR, RPC = THREADS / TPR, RPW = TPR <= 32 ? 32 / TPR : 1;      // rows of a CTA and of a warp
  __shared__ float2 part[2][32];
  const int t = TPR <= 32 ? (int)threadIdx.x & (TPR - 1) : (int)threadIdx.x;
  const S* const x = static_cast<const S*>(a.x) + t * VEC;
  const R* const r = static_cast<const R*>(a.r) + t * VEC;
  S* const s = static_cast<S*>(a.s) + t * VEC;
  Y* const y = static_cast<Y*>(a.y) + t * VEC;
  const int left = a.N - t * VEC;                        // piece i of the thread is in the row if i * TPR * VEC < left
  float w[NV * VEC];
  if (NORM) load_weights<VEC, NV, TPR>(a.w, a.w_type, a.N, t, w);
  int buf = 0;
  const float over_n = 1.0f / a.N;
  // `first` is the same for all lanes of a warp: they leave the loop together
  const int sub = TPR <= 32 ? (int)(threadIdx.x & 31) / TPR : 0;
  for (long long first = (long long)blockIdx.x * RPC * UR + (TPR <= 32 ? (threadIdx.x >> 5) * RPW * UR : 0); first < a.M; first += (long long)gridDim.x * RPC * UR) {
    Piece<S, VEC> px[UR][NV];
    float v[UR][NV * VEC];
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const long long row = first + u * RPW + sub;
      const int here = row < a.M ? left : 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i * TPR * VEC < here) px[u][i].load(x + row * a.ldx + i * TPR * VEC);
        else px[u][i].zero();
    }
    if (NORM && a.r != nullptr) {
      Piece<R, VEC> pr[UR][NV];
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        const long long row = first + u * RPW + sub;
        const int here = row < a.M ? left : 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (i * TPR * VEC < here) pr[u][i].load(r + row * a.ldr + i * TPR * VEC);
          else pr[u][i].zero();
      }
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        const long long row = first + u * RPW + sub;
        const int here = row < a.M ? left : 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float sum[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            sum[e] = px[u][i].at(e) + pr[u][i].at(e);
            v[u][i * VEC + e] = as_float(rounded<S>(sum[e]));
          }
          if (i * TPR * VEC < here) Out<S, VEC>::store(s + row * a.N + i * TPR * VEC, sum);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < UR; ++u)
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) v[u][i] = px[u][i / VEC].at(i % VEC);
    }
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const long long row = first + u * RPW + sub;
      const int here = row < a.M ? left : 0;
      float sum = 0.f, top = 0.f, rho = 1.f, f = 1.f;
#pragma unroll
      for (int i = 0; i < NV * VEC; ++i) {
        if (NORM) {
          sum = fmaf(v[u][i], v[u][i], sum);
          v[u][i] *= w[i];
          if (Q) top = max_nan(top, fabsf(v[u][i]));      // (a NaN may be the weight's: the sum does not see it)
        } else {
          top = max_nan(top, fabsf(v[u][i]));
        }
      }
      if (NORM) {
        row_reduce<TPR, Q>(sum, top, part, buf);
        rho = rsqrtf(fmaf(sum, over_n, a.eps));
        top *= rho;
      } else {
        row_max_nan<TPR>(top, part, buf);
      }
      if (Q) {
        float scale;
        f = row_scale(top, scale);
        if (t == 0 && row < a.M) a.scale[row] = scale;
      }
      if (t == 0 && row < a.M && a.rho != nullptr) a.rho[row] = rho;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = !NORM ? v[u][i * VEC + e] * f : Q ? v[u][i * VEC + e] * rho * f : v[u][i * VEC + e] * rho;
        if (i * TPR * VEC < here) Out<Y, VEC>::store(y + row * a.ldy + i * TPR * VEC, o);
      }
    }
  }
}

// Rows that the registers do not hold: a CTA per row, which reads it a second time (from L2, mostly).
template <class S, class R, class Y, int VEC>
__global__ void __launch_bounds__(512) k_rms_forward_wide(const FwdArgs a) {
  constexpr bool Q = type_code<Y>() == SPION_E4M3;
  __shared__ float2 part[2][32];
  const R* const r = static_cast<const R*>(a.r);
  S* const s = static_cast<S*>(a.s);
  int buf = 0;
  for (long long row = blockIdx.x; row < a.M; row += gridDim.x) {
    const S* const x = static_cast<const S*>(a.x) + row * a.ldx;
    Y* const y = static_cast<Y*>(a.y) + row * a.ldy;
    float sum = 0.f, top = 0.f;
#pragma unroll 2
    for (int c = threadIdx.x * VEC; c < a.N; c += blockDim.x * VEC) {
      Piece<S, VEC> px;
      Piece<R, VEC> pr;
      px.load(x + c);
      float v[VEC];
      if (r != nullptr) {
        pr.load(r + row * a.ldr + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = px.at(e) + pr.at(e);
        Out<S, VEC>::store(s + row * a.N + c, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = as_float(rounded<S>(v[e]));
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = px.at(e);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        sum = fmaf(v[e], v[e], sum);
        if (Q) top = max_nan(top, fabsf(v[e] * (a.w == nullptr ? 1.f : load_any(a.w, a.w_type, c + e))));
      }
    }
    float rho = 1.f, f = 1.f;
    if (a.norm) {
      row_reduce<512, Q>(sum, top, part, buf);
      rho = rsqrtf(fmaf(sum, 1.0f / a.N, a.eps));
    } else {
      row_max_nan<512>(top, part, buf);
    }
    if (Q) {
      float scale;
      f = row_scale(top * rho, scale);
      if (threadIdx.x == 0) a.scale[row] = scale;
    }
    if (threadIdx.x == 0 && a.rho != nullptr) a.rho[row] = rho;
    const S* const from = r != nullptr ? s + row * a.N : x;                // this thread's own stores
#pragma unroll 2
    for (int c = threadIdx.x * VEC; c < a.N; c += blockDim.x * VEC) {
      Piece<S, VEC> px;
      px.load(from + c);
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float v = px.at(e) * (a.w == nullptr ? 1.f : load_any(a.w, a.w_type, c + e)) * rho;
        o[e] = Q ? v * f : v;
      }
      Out<Y, VEC>::store(y + c, o);
    }
  }
}

struct BwdArgs {
  const void* s; long long lds;           // the sum (or x, rows lds apart)
  const void* dy;                         // [M, N]
  const void* ds;                         // or null
  const void* w; int w_type;
  const float* rho;
  void* dx;
  void* dr; int dr_type;                  // a second copy of dx in 16 bits, or null
  float* part;                            // [CTAs, N]; null: no weight gradient here
  long long M; int N;
};

// Both gradients of a row from registers.  `carry`: the sums of dy n, column by column.
template <class S, class D, int VEC, int NV, int TPR>
__device__ __forceinline__ void row_backward(const BwdArgs& a, long long row, int here, const Piece<S, VEC> (&ps)[NV], const Piece<D, VEC> (&pd)[NV],
                                             const Piece<S, VEC> (&pk)[NV], float rho, float mean, const float (&w)[NV * VEC], int t) {
  S* const dx = static_cast<S*>(a.dx);
  const float m = mean * rho;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = fmaf(fmaf(-ps[i].at(e), m, pd[i].at(e) * w[i * VEC + e]), rho, pk[i].at(e));
    if (i * TPR * VEC < here) {
      const long long at = row * a.N + (t + i * TPR) * VEC;
      if (dx != nullptr) Out<S, VEC>::store(dx + at, o);
      if (a.dr != nullptr) {
        if (a.dr_type == SPION_BF16) Out<__nv_bfloat16, VEC>::store(static_cast<__nv_bfloat16*>(a.dr) + at, o);
        else Out<__half, VEC>::store(static_cast<__half*>(a.dr) + at, o);
      }
    }
  }
}

// Rows through registers.  The groups of lanes of a CTA leave their sums of a column side by side in shared memory, where they are added in order.
template <class S, class D, int VEC, int NV, int TPR, int UR>
__global__ void __launch_bounds__(TPR <= 32 ? CTA : TPR, TPR <= 32 ? 2 : 512 / TPR) k_rms_backward(const BwdArgs a) {
  next_may_start();                                                        // k_rms_dw
  constexpr int THREADS = TPR <= 32 ? CTA : TPR, RPC = THREADS / TPR, RPW = TPR <= 32 ? 32 / TPR : 1;
  constexpr int WIDTH = TPR * NV * VEC, AT_ONCE = RPC < 8 ? RPC : 8;       // groups of lanes whose sums are in shared memory together
  __shared__ float2 part[2][32];
  __shared__ float sums[RPC > 1 ? AT_ONCE * WIDTH : 1];
  const int t = TPR <= 32 ? (int)threadIdx.x & (TPR - 1) : (int)threadIdx.x, sub = TPR <= 32 ? (int)(threadIdx.x & 31) / TPR : 0;
  const S* const s = static_cast<const S*>(a.s) + t * VEC;
  const D* const dy = static_cast<const D*>(a.dy) + t * VEC;
  const S* const ds = static_cast<const S*>(a.ds) + t * VEC;
  const int left = a.N - t * VEC;
  float w[NV * VEC], acc[NV * VEC];
  load_weights<VEC, NV, TPR>(a.w, a.w_type, a.N, t, w);
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) acc[i] = 0.f;
  int buf = 0;
  const float over_n = 1.0f / a.N;
  for (long long first = (long long)blockIdx.x * RPC * UR + (TPR <= 32 ? (threadIdx.x >> 5) * RPW * UR : 0); first < a.M; first += (long long)gridDim.x * RPC * UR) {
    Piece<S, VEC> ps[UR][NV], pk[UR][NV];
    Piece<D, VEC> pd[UR][NV];
    float rho[UR];
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const long long row = first + u * RPW + sub;
      const int here = row < a.M ? left : 0;
      rho[u] = row < a.M ? a.rho[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i * TPR * VEC < here) ps[u][i].load(s + row * a.lds + i * TPR * VEC), pd[u][i].load(dy + row * a.N + i * TPR * VEC);
        else ps[u][i].zero(), pd[u][i].zero();
        if (a.ds != nullptr && i * TPR * VEC < here) pk[u][i].load(ds + row * a.N + i * TPR * VEC);
        else pk[u][i].zero();
      }
    }
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const long long row = first + u * RPW + sub;
      float sum = 0.f, none = 0.f;
#pragma unroll
      for (int i = 0; i < NV * VEC; ++i) {
        const float d = pd[u][i / VEC].at(i % VEC) * (ps[u][i / VEC].at(i % VEC) * rho[u]);
        acc[i] += d;
        sum = fmaf(d, w[i], sum);
      }
      row_reduce<TPR, false>(sum, none, part, buf);
      row_backward<S, D, VEC, NV, TPR>(a, row, row < a.M ? left : 0, ps[u], pd[u], pk[u], rho[u], sum * over_n, w, t);
    }
  }
  if (a.part == nullptr) return;
  float* const out = a.part + (long long)blockIdx.x * a.N;
  if (RPC == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (i * TPR * VEC < left) out[(t + i * TPR) * VEC + e] = acc[i * VEC + e];
    return;
  }
  constexpr int COLS = (WIDTH + THREADS - 1) / THREADS;
  const int group = threadIdx.x / TPR;
  float total[COLS];
#pragma unroll
  for (int k = 0; k < COLS; ++k) total[k] = 0.f;
  for (int g0 = 0; g0 < RPC; g0 += AT_ONCE) {
    __syncthreads();
    if (group >= g0 && group < g0 + AT_ONCE) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[(group - g0) * WIDTH + (t + i * TPR) * VEC + e] = acc[i * VEC + e];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      const int c = threadIdx.x + k * THREADS;
      if (c < WIDTH)
#pragma unroll
        for (int g = 0; g < AT_ONCE; ++g) total[k] += sums[g * WIDTH + c];
    }
  }
#pragma unroll
  for (int k = 0; k < COLS; ++k) {
    const int c = threadIdx.x + k * THREADS;
    if (c < WIDTH && c < a.N) out[c] = total[k];
  }
}

// Wide rows: a CTA takes its rows one after another out of a ring in shared memory that bulk copies fill several rows ahead, so that the row's sum, which
// everything waits for, does not stop the loads.  The one barrier a row has for its sum also tells that all threads hold their pieces in registers: the
// row's place in the ring is filled anew right after it.
struct Ring { int stages; uint32_t stage, at_dy, at_ds; };                 // bytes
constexpr uint32_t RING_BARS = 128;
template <class S, class D, int NV, int TPR>
__global__ void __launch_bounds__(TPR) k_rms_backward_ring(const BwdArgs a, const Ring ring) {
  next_may_start();                                                        // k_rms_dw
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 part[2][32];
  __shared__ int s_lost;
  const int t = threadIdx.x, left = a.N - t * 8;
  const uint32_t bars = tc::smem_u32(smem), rows0 = bars + RING_BARS;
  const long long step = gridDim.x;
  auto give_up = [&](long long row) {                                      // what this CTA does not form is NaN, from this row on
    float bad[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bad[e] = __int_as_float(0x7fffffff);
    for (int c = t * 8; c < a.N; c += TPR * 8) {
      for (long long r = row; r < a.M; r += step) {
        if (a.dx != nullptr) Out<S, 8>::store(static_cast<S*>(a.dx) + r * a.N + c, bad);
        if (a.dr != nullptr && a.dr_type == SPION_BF16) Out<__nv_bfloat16, 8>::store(static_cast<__nv_bfloat16*>(a.dr) + r * a.N + c, bad);
        if (a.dr != nullptr && a.dr_type != SPION_BF16) Out<__half, 8>::store(static_cast<__half*>(a.dr) + r * a.N + c, bad);
      }
      if (a.part != nullptr) Out<float, 8>::store(a.part + (long long)blockIdx.x * a.N + c, bad);
    }
  };
  auto fill = [&](int st, long long row) {                                 // one thread
    const uint32_t bytes = a.N * (uint32_t)sizeof(S), dbytes = a.N * (uint32_t)sizeof(D), at = rows0 + st * ring.stage, bar = bars + 8 * st;
    tc::mbar_expect_tx(bar, bytes + dbytes + (a.ds != nullptr ? bytes : 0));
    tc::bulk_load(at, static_cast<const S*>(a.s) + row * a.lds, bar, bytes);
    tc::bulk_load(at + ring.at_dy, static_cast<const D*>(a.dy) + row * a.N, bar, dbytes);
    if (a.ds != nullptr) tc::bulk_load(at + ring.at_ds, static_cast<const S*>(a.ds) + row * a.N, bar, bytes);
  };
  if (t == 0) {
    s_lost = *reinterpret_cast<volatile int*>(&g_rms_status) != 0 ? -1 : 0;
    for (int i = 0; i < ring.stages; ++i) tc::mbar_init(bars + 8 * i, 1);
    tc::fence_barrier_init();
    tc::fence_proxy_async();
    for (int i = 0; i < ring.stages && s_lost == 0; ++i)
      if (blockIdx.x + i * step < a.M) fill(i, blockIdx.x + i * step);
  }
  float w[NV * 8], acc[NV * 8];
  load_weights<8, NV, TPR>(a.w, a.w_type, a.N, t, w);
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) acc[i] = 0.f;
  int buf = 0, st = 0, ph = 0;
  const float over_n = 1.0f / a.N;
  float rho = blockIdx.x < a.M ? a.rho[blockIdx.x] : 0.f;
  __syncthreads();
  if (s_lost != 0) return give_up(blockIdx.x);
  __syncthreads();
  for (long long row = blockIdx.x; row < a.M; row += step) {
    const float next = row + step < a.M ? a.rho[row + step] : 0.f;
    if (!tc::mbar_wait(bars + 8 * st, ph)) s_lost = 1;                     // (bounded; the copies of this CTA end by themselves)
    const uint8_t* const at = smem + RING_BARS + st * ring.stage;
    auto piece = [&](int i, Piece<S, 8>& s, Piece<D, 8>& d, Piece<S, 8>& k) {
      const int c = (t + i * TPR) * 8;
      s.zero(), d.zero(), k.zero();
      if (i * TPR * 8 >= left) return;
      s.load_shared(reinterpret_cast<const S*>(at) + c);
      d.load_shared(reinterpret_cast<const D*>(at + ring.at_dy) + c);
      if (a.ds != nullptr) k.load_shared(reinterpret_cast<const S*>(at + ring.at_ds) + c);
    };
    Piece<S, 8> ps[1], pk[1];
    Piece<D, 8> pd[1];
    float sum = 0.f, none = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      piece(i, ps[0], pd[0], pk[0]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = pd[0].at(e) * (ps[0].at(e) * rho);
        acc[i * 8 + e] += d;
        sum = fmaf(d, w[i * 8 + e], sum);
      }
    }
    row_reduce<TPR, false>(sum, none, part, buf);
    if (s_lost) {                                                          // (every thread that set it did so before the barrier)
      if (t == 0) {
        atomicOr(&g_rms_status, 1);
        for (int i = 0; i < ring.stages; ++i)                              // the copies under way end first, or this gives up again
          if (row + (i - st + (i < st ? ring.stages : 0)) * step < a.M) tc::mbar_wait(bars + 8 * i, i < st ? ph ^ 1 : ph);
      }
      return give_up(row);
    }
    const bool more = t == 0 && row + ring.stages * step < a.M;
    if (NV == 1) {                                                         // the thread's piece is in registers
      if (more) fill(st, row + ring.stages * step);
      float w1[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w1[e] = w[e];
      row_backward<S, D, 8, 1, TPR>(a, row, left, ps, pd, pk, rho, sum * over_n, w1, t);
    } else {                                                               // several: read again, and the place is free a barrier later
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        piece(i, ps[0], pd[0], pk[0]);
        float w1[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w1[e] = w[i * 8 + e];
        row_backward<S, D, 8, 1, TPR>(a, row, left - i * TPR * 8, ps, pd, pk, rho, sum * over_n, w1, t + i * TPR);
      }
      __syncthreads();
      if (more) fill(st, row + ring.stages * step);
    }
    rho = next;
    if (++st == ring.stages) st = 0, ph ^= 1;
  }
  if (a.part == nullptr) return;
  float* const out = a.part + (long long)blockIdx.x * a.N;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * TPR * 8 < left) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = acc[i * 8 + e];
      Out<float, 8>::store(out + (t + i * TPR) * 8, o);
    }
}

// Rows that the registers do not hold: dx here, the weight gradient by columns (k_rms_columns).
template <class S, class D, int VEC>
__global__ void __launch_bounds__(512) k_rms_backward_wide(const BwdArgs a) {
  __shared__ float2 part[2][32];
  int buf = 0;
  for (long long row = blockIdx.x; row < a.M; row += gridDim.x) {
    const S* const s = static_cast<const S*>(a.s) + row * a.lds;
    const D* const dy = static_cast<const D*>(a.dy) + row * a.N;
    const S* const ds = a.ds == nullptr ? nullptr : static_cast<const S*>(a.ds) + row * a.N;
    const float rho = a.rho[row];
    float sum = 0.f, none = 0.f;
#pragma unroll 2
    for (int c = threadIdx.x * VEC; c < a.N; c += blockDim.x * VEC) {
      Piece<S, VEC> ps;
      Piece<D, VEC> pd;
      ps.load(s + c), pd.load(dy + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum = fmaf(pd.at(e) * (a.w == nullptr ? 1.f : load_any(a.w, a.w_type, c + e)), ps.at(e) * rho, sum);
    }
    row_reduce<512, false>(sum, none, part, buf);
    const float m = sum / a.N;
#pragma unroll 2
    for (int c = threadIdx.x * VEC; c < a.N; c += blockDim.x * VEC) {
      Piece<S, VEC> ps, pk;
      Piece<D, VEC> pd;
      ps.load(s + c), pd.load(dy + c);
      if (ds != nullptr) pk.load(ds + c);
      else pk.zero();
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float g = pd.at(e) * (a.w == nullptr ? 1.f : load_any(a.w, a.w_type, c + e));
        o[e] = fmaf(g - ps.at(e) * rho * m, rho, pk.at(e));
      }
      if (a.dx != nullptr) Out<S, VEC>::store(static_cast<S*>(a.dx) + row * a.N + c, o);
      if (a.dr != nullptr) {
        if (a.dr_type == SPION_BF16) Out<__nv_bfloat16, VEC>::store(static_cast<__nv_bfloat16*>(a.dr) + row * a.N + c, o);
        else Out<__half, VEC>::store(static_cast<__half*>(a.dr) + row * a.N + c, o);
      }
    }
  }
}
// part[blockIdx.y, c] = sum over the rows blockIdx.y, + gridDim.y, ... of dy_c s_c rho
template <class S, class D>
__global__ void __launch_bounds__(256) k_rms_columns(const BwdArgs a) {
  next_may_start();                                                        // k_rms_dw
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.N) return;
  float acc = 0.f;
  for (long long row = blockIdx.y; row < a.M; row += gridDim.y)
    acc = fmaf(as_float(static_cast<const D*>(a.dy)[row * a.N + c]), as_float(static_cast<const S*>(a.s)[row * a.lds + c]) * a.rho[row], acc);
  a.part[(long long)blockIdx.y * a.N + c] = acc;
}

// dw[c] = sum over the partial rows, in a fixed order: warp w of 32 adds the rows w, w + 32, ..., then the warps' sums in order.
__global__ void __launch_bounds__(1024) k_rms_dw(const float* part, int count, int N, void* dw, int type) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  wait_for_kernel_before();
  if (c < N)
    for (int r = warp; r < count; r += 8 * 32) {                           // eight loads at a time, added one after another
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = r + 32 * k < count ? part[(long long)(r + 32 * k) * N + c] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < N) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += sums[k][lane];
    store_any(dw, type, c, t);
  }
}

// ------------------------------------------------------------------------------------------------ host
// a row starts on a piece's boundary in every matrix that the call has
bool on_boundary(const void* p, long long ld, int type) {
  return p == nullptr || (((uintptr_t)p | (uintptr_t)(ld * type_size(type))) & (uintptr_t)(8 * type_size(type) - 1)) == 0;
}
int grid_of(long long M, int rows_per_cta, int threads) {
  const long long most = (long long)sm_count() * (2048 / threads), need = (M + rows_per_cta - 1) / rows_per_cta;
  return (int)(need < most ? need : most);
}

template <bool NORM, class S, class R, class Y, int VEC, int NV, int TPR, int UR = 1> void launch_forward(const FwdArgs& a, cudaStream_t st) {
  constexpr int THREADS = TPR <= 32 ? CTA : TPR;
  k_rms_forward<NORM, S, R, Y, VEC, NV, TPR, UR><<<grid_of(a.M, THREADS / TPR * UR, THREADS), THREADS, 0, st>>>(a);
}
template <class S, class R, class Y, bool NORM = true>
int forward(const FwdArgs& a, cudaStream_t st) {
  const bool vec = a.N % 8 == 0 && on_boundary(a.x, a.ldx, type_code<S>()) && on_boundary(a.r, a.ldr, type_code<R>()) &&
                   on_boundary(a.s, a.N, type_code<S>()) && on_boundary(a.y, a.ldy, type_code<Y>()) && on_boundary(a.w, a.N, a.w_type);
  // Where there is a multiprocessor to every row, a thread to a piece up to 4096 values.  That / four pieces a thread, us, one row, 148 rows: bf16 with a residual 2048 values
  // 1.97 / 2.18, 2.05 / 2.26, 4096 2.35 / 2.27, 2.45 / 2.40 (to e4m3 2.31 / 2.35, 2.45 / 2.61, fp32 148 rows 2.81 / 3.38), 8192 3.08 / 2.69, 4.55 / 4.51.
  const bool few = a.M <= sm_count();
  if (vec) {
    const int n = a.N / 8;
    if (n <= 8) launch_forward<NORM, S, R, Y, 8, 1, 8, 2>(a, st);
    else if (n <= 16) launch_forward<NORM, S, R, Y, 8, 2, 8>(a, st);
    else if (n <= 32) launch_forward<NORM, S, R, Y, 8, 4, 8>(a, st);
    else if (n <= 64) launch_forward<NORM, S, R, Y, 8, 2, 32>(a, st);
    else if (n <= 128) launch_forward<NORM, S, R, Y, 8, 4, 32>(a, st);
    else if (few && n <= 256) launch_forward<NORM, S, R, Y, 8, 1, 256>(a, st);
    else if (few && n <= 512) launch_forward<NORM, S, R, Y, 8, 1, 512>(a, st);
    else if (n <= 256) launch_forward<NORM, S, R, Y, 8, 4, 64>(a, st);
    else if (n <= 512) launch_forward<NORM, S, R, Y, 8, 4, 128>(a, st);
    else if (n <= 1024) launch_forward<NORM, S, R, Y, 8, 4, 256>(a, st);
    else if (n <= 2048) launch_forward<NORM, S, R, Y, 8, 4, 512>(a, st);
    else k_rms_forward_wide<S, R, Y, 8><<<grid_of(a.M, 1, 512), 512, 0, st>>>(a);
  } else {
    if (a.N <= 128) launch_forward<NORM, S, R, Y, 1, 4, 32, 2>(a, st);
    else if (a.N <= 512) launch_forward<NORM, S, R, Y, 1, 16, 32>(a, st);
    else if (a.N <= 1024) launch_forward<NORM, S, R, Y, 1, 16, 64>(a, st);
    else if (a.N <= 2048) launch_forward<NORM, S, R, Y, 1, 16, 128>(a, st);
    else if (a.N <= 4096) launch_forward<NORM, S, R, Y, 1, 16, 256>(a, st);
    else if (a.N <= 8192) launch_forward<NORM, S, R, Y, 1, 16, 512>(a, st);
    else k_rms_forward_wide<S, R, Y, 1><<<grid_of(a.M, 1, 512), 512, 0, st>>>(a);
  }
  SPION_LAUNCH_CHECK();
  return SPION_OK;
}
template <class S, class R> int forward_out(const FwdArgs& a, int y_type, cudaStream_t st) {
  if (y_type == SPION_E4M3) return forward<S, R, __nv_fp8_e4m3>(a, st);
  if (y_type == type_code<S>()) return forward<S, R, S>(a, st);
  if constexpr (type_code<S>() == SPION_F32) {
    if (y_type == SPION_BF16) return forward<S, R, __nv_bfloat16>(a, st);
    if (y_type == SPION_F16) return forward<S, R, __half>(a, st);
  }
  return SPION_ERR_UNSUPPORTED;
}

// CTAs of a backward: what is resident at a time and no more, because every one of them leaves a partial row
int parts_of(long long M, int rows_per_cta, int per_sm) {
  const long long need = (M + rows_per_cta - 1) / rows_per_cta, most = std::min((long long)sm_count() * per_sm, (long long)MAX_PARTS);
  return (int)(need < most ? need : most);
}
template <class S, class D, int VEC, int NV, int TPR, int UR = 1> int launch_backward(const BwdArgs& a, int per_sm, cudaStream_t st) {
  constexpr int THREADS = TPR <= 32 ? CTA : TPR;
  const int parts = parts_of(a.M, THREADS / TPR * UR, per_sm);
  k_rms_backward<S, D, VEC, NV, TPR, UR><<<parts, THREADS, 0, st>>>(a);
  return parts;
}
// 0: fewer than two rows fit
template <class S, class D, int NV, int TPR> int launch_ring(const BwdArgs& a, int per_sm, cudaStream_t st) {
  Ring r;
  r.at_dy = a.N * (uint32_t)sizeof(S);
  r.at_ds = r.at_dy + a.N * (uint32_t)sizeof(D);
  r.stage = r.at_ds + (a.ds != nullptr ? a.N * (uint32_t)sizeof(S) : 0);
  const uint32_t room = 200u * 1024 / per_sm - RING_BARS;
  r.stages = (int)std::min(room / r.stage, 8u);
  if (r.stages < 2) return 0;
  const uint32_t smem = RING_BARS + r.stages * r.stage;
  static std::atomic<uint64_t> ready{0};                                   // devices on which the kernel has its shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(k_rms_backward_ring<S, D, NV, TPR>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) return 0;
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  const int parts = parts_of(a.M, 1, per_sm);
  k_rms_backward_ring<S, D, NV, TPR><<<parts, TPR, smem, st>>>(a, r);
  return parts;
}

template <class S, class D>
int backward(const BwdArgs& a, void* dw, int dw_type, cudaStream_t st) {
  const bool vec = a.N % 8 == 0 && on_boundary(a.s, a.lds, type_code<S>()) && on_boundary(a.dy, a.N, type_code<D>()) &&
                   on_boundary(a.ds, a.N, type_code<S>()) && on_boundary(a.dx, a.N, type_code<S>()) && on_boundary(a.dr, a.N, a.dr_type) &&
                   on_boundary(a.w, a.N, a.w_type) && on_boundary(a.part, a.N, SPION_F32);
  int parts = 0;
  if (vec) {
    const int n = a.N / 8;
    if (n <= 8) parts = launch_backward<S, D, 8, 1, 8, 2>(a, 2, st);
    else if (n <= 16) parts = launch_backward<S, D, 8, 2, 8>(a, 2, st);
    else if (n <= 64) parts = launch_backward<S, D, 8, 2, 32>(a, 2, st);
    else if (n <= 128) parts = launch_ring<S, D, 1, 128>(a, 4, st);
    else if (n <= 256) parts = launch_ring<S, D, 1, 256>(a, 4, st);
    else if (n <= 512) parts = launch_ring<S, D, 1, 512>(a, 2, st);
    else if (n <= 1024) parts = launch_ring<S, D, 1, 1024>(a, 1, st);
    else if (n <= 2048) parts = launch_ring<S, D, 2, 1024>(a, 1, st);
  } else {
    if (a.N <= 128) parts = launch_backward<S, D, 1, 4, 32, 2>(a, 2, st);
    else if (a.N <= 512) parts = launch_backward<S, D, 1, 16, 32>(a, 2, st);
    else if (a.N <= 1024) parts = launch_backward<S, D, 1, 16, 64>(a, 8, st);
    else if (a.N <= 2048) parts = launch_backward<S, D, 1, 16, 128>(a, 4, st);
    else if (a.N <= 4096) parts = launch_backward<S, D, 1, 16, 256>(a, 2, st);
    else if (a.N <= 8192) parts = launch_backward<S, D, 1, 16, 512>(a, 1, st);
  }
  if (parts == 0) {
    if (vec) k_rms_backward_wide<S, D, 8><<<grid_of(a.M, 1, 512), 512, 0, st>>>(a);
    else k_rms_backward_wide<S, D, 1><<<grid_of(a.M, 1, 512), 512, 0, st>>>(a);
    if (a.part != nullptr) {
      SPION_LAUNCH_CHECK();
      parts = (int)(a.M < 32 ? a.M : 32);
      k_rms_columns<S, D><<<dim3((a.N + 255) / 256, parts), 256, 0, st>>>(a);
    }
  }
  SPION_LAUNCH_CHECK();
  if (a.part == nullptr) return SPION_OK;
  SPION_CUDA_TRY(launch_after(k_rms_dw, dim3((a.N + 31) / 32), dim3(1024), 0, st, (const float*)a.part, parts, a.N, dw, dw_type));
  return SPION_OK;
}

bool stream_type(int t) { return t == SPION_F32 || t == SPION_BF16 || t == SPION_F16; }

}  // namespace

int* rmsnorm_status_word() {
  static StatusWord word;
  return word.on_this_device(g_rms_status);
}

extern "C" {

int spion_rmsnorm_forward(const void* x, long long ldx, int x_type, const void* res, long long ldr, int res_type, const void* w, int w_type,
                          void* sum_out, void* y, long long ldy, int y_type, float* scale, float* rstd, long long M, int N, float eps, int norm,
                          void* cuda_stream) {
  if (M < 0 || N <= 0 || !stream_type(x_type) || (w != nullptr && !stream_type(w_type))) return SPION_ERR_ARG;
  if (M == 0) return SPION_OK;
  if (x == nullptr || y == nullptr || (res != nullptr && sum_out == nullptr) || (y_type == SPION_E4M3) != (scale != nullptr)) return SPION_ERR_ARG;
  if (ldx < 0 || ldy < N || (res != nullptr && ldr < 0)) return SPION_ERR_ARG;
  if (!norm && (y_type != SPION_E4M3 || w != nullptr || res != nullptr)) return SPION_ERR_ARG;
  if (res == nullptr) res_type = x_type;
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  const FwdArgs a = {x, ldx, res, ldr, w, w_type, sum_out, y, ldy, scale, rstd, M, N, eps, norm};
  if (!norm) {
    if (x_type == SPION_F32) return forward<float, float, __nv_fp8_e4m3, false>(a, st);
    if (x_type == SPION_BF16) return forward<__nv_bfloat16, __nv_bfloat16, __nv_fp8_e4m3, false>(a, st);
    return forward<__half, __half, __nv_fp8_e4m3, false>(a, st);
  }
  if (x_type == SPION_F32) {
    if (res_type == SPION_F32) return forward_out<float, float>(a, y_type, st);
    if (res_type == SPION_BF16) return forward_out<float, __nv_bfloat16>(a, y_type, st);
    if (res_type == SPION_F16) return forward_out<float, __half>(a, y_type, st);
    return SPION_ERR_UNSUPPORTED;
  }
  if (res_type != x_type) return SPION_ERR_UNSUPPORTED;
  if (x_type == SPION_BF16) return forward_out<__nv_bfloat16, __nv_bfloat16>(a, y_type, st);
  return forward_out<__half, __half>(a, y_type, st);
}

long long spion_rmsnorm_workspace_floats(long long M, int N) {
  return M <= 0 || N <= 0 ? 0 : (M < MAX_PARTS ? M : MAX_PARTS) * (long long)N;
}

int spion_rmsnorm_backward(const void* s, long long lds, int s_type, const void* dy, int dy_type, const void* ds, const void* w, int w_type,
                           const float* rstd, void* dx, void* dres, int dres_type, void* dw, float* workspace, long long M, int N,
                           void* cuda_stream) {
  if (M < 0 || N <= 0 || !stream_type(s_type) || !stream_type(dy_type) || (w != nullptr && !stream_type(w_type))) return SPION_ERR_ARG;
  if (dres != nullptr && (dres_type == SPION_F32 || !stream_type(dres_type))) return SPION_ERR_ARG;
  if (dw != nullptr && w == nullptr) return SPION_ERR_ARG;
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  if (M == 0) {
    if (dw != nullptr) SPION_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)N * type_size(w_type), st));
    return SPION_OK;
  }
  if (s == nullptr || dy == nullptr || rstd == nullptr || lds < 0 || (dw != nullptr && workspace == nullptr)) return SPION_ERR_ARG;
  const BwdArgs a = {s, lds, dy, ds, w, w_type, rstd, dx, dres, dres_type, dw != nullptr ? workspace : nullptr, M, N};
  if (s_type == SPION_F32) {
    if (dy_type == SPION_F32) return backward<float, float>(a, dw, w_type, st);
    if (dy_type == SPION_BF16) return backward<float, __nv_bfloat16>(a, dw, w_type, st);
    return backward<float, __half>(a, dw, w_type, st);
  }
  if (dy_type != s_type) return SPION_ERR_UNSUPPORTED;
  if (s_type == SPION_BF16) return backward<__nv_bfloat16, __nv_bfloat16>(a, dw, w_type, st);
  return backward<__half, __half>(a, dw, w_type, st);
}

}  // extern "C"
