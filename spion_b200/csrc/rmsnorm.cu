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
// Work split: rows of up to 256 values take 8 lanes (a warp has four rows), up to 1024 a warp, wider ones a CTA; a row that no register file holds is
// read twice.  Pieces of eight elements where every row starts on the boundary of such a piece, single elements otherwise (odd widths).
#include "rows.cuh"

using namespace rows;

namespace {

constexpr float SMALL = 0x1p-100f;        // what the scale of a row of zeros follows
constexpr int CTA = 256;                  // threads of a CTA whose warps take rows of their own
constexpr int MAX_PARTS = 1184;           // partial rows of a weight gradient: eight per multiprocessor of 148

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

template <int VEC, int NV> __device__ __forceinline__ void load_weights(const void* p, int type, int N, int t, int tpr, float (&w)[NV * VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * tpr) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[i * VEC + e] = p == nullptr ? 1.f : c < N ? load_any(p, type, c + e) : 0.f;
  }
}

// e4m3: what y is multiplied with, and the row's scale.  A row with a NaN has the scale NaN (`sum` is NaN then), one with an infinity an infinite
// scale and zeros beside NaN: no value of such a row comes back finite.
__device__ __forceinline__ float row_scale(float top, float sum, float& scale) {
  float a = top < SMALL ? SMALL : top;
  if (sum != sum) a = sum;
  scale = a / 448.f;
  return 448.f * __frcp_rn(a);
}

// SUB lanes to a row, 0: the CTA
template <class S, class R, class Y, int VEC, int NV, int SUB, int THREADS>
__global__ void __launch_bounds__(THREADS) k_rms_forward(const FwdArgs a) {
  constexpr bool Q = type_code<Y>() == SPION_E4M3;
  __shared__ float2 part[2][32];
  const int tpr = SUB ? SUB : (int)blockDim.x, t = SUB ? (int)threadIdx.x & (SUB - 1) : (int)threadIdx.x;
  const int rpc = SUB ? (int)blockDim.x / SUB : 1, sub = SUB ? (int)(threadIdx.x & 31) / SUB : 0;
  const S* const x = static_cast<const S*>(a.x);
  const R* const r = static_cast<const R*>(a.r);
  S* const s = static_cast<S*>(a.s);
  Y* const y = static_cast<Y*>(a.y);
  float w[NV * VEC];
  load_weights<VEC, NV>(a.w, a.w_type, a.N, t, tpr, w);
  int buf = 0;
  const float over_n = 1.0f / a.N;
  // `first` is the same for all lanes of a warp: they leave the loop together
  for (long long first = (long long)blockIdx.x * rpc + (SUB ? (threadIdx.x >> 5) * (32 / (SUB ? SUB : 32)) : 0); first < a.M;
       first += (long long)gridDim.x * rpc) {
    const long long row = first + sub;
    const bool live = row < a.M;
    Piece<S, VEC> px[NV];
    Piece<R, VEC> pr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * tpr) * VEC;
      if (live && c < a.N) px[i].load(x + row * a.ldx + c);
      else px[i].zero();
    }
    float v[NV * VEC];
    if (r != nullptr) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * tpr) * VEC;
        if (live && c < a.N) pr[i].load(r + row * a.ldr + c);
        else pr[i].zero();
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * tpr) * VEC;
        float sum[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          sum[e] = px[i].at(e) + pr[i].at(e);
          v[i * VEC + e] = as_float(rounded<S>(sum[e]));
        }
        if (live && c < a.N) Out<S, VEC>::store(s + row * a.N + c, sum);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV * VEC; ++i) v[i] = px[i / VEC].at(i % VEC);
    }
    float sum = 0.f, top = 0.f;
#pragma unroll
    for (int i = 0; i < NV * VEC; ++i) {
      sum = fmaf(v[i], v[i], sum);
      v[i] *= w[i];
      if (Q) top = fmaxf(top, fabsf(v[i]));
    }
    row_reduce<SUB, Q>(sum, top, part, buf);
    const float rho = a.norm ? rsqrtf(fmaf(sum, over_n, a.eps)) : 1.f;
    float f = rho;
    if (Q) {
      float scale;
      f = row_scale(top * rho, a.norm ? top * rho : sum, scale);
      if (t == 0 && live) a.scale[row] = scale;
    }
    if (t == 0 && live && a.rho != nullptr) a.rho[row] = rho;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * tpr) * VEC;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = Q ? v[i * VEC + e] * rho * f : v[i * VEC + e] * rho;
      if (live && c < a.N) Out<Y, VEC>::store(y + row * a.ldy + c, o);
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
        if (Q) top = fmaxf(top, fabsf(v[e] * (a.w == nullptr ? 1.f : load_any(a.w, a.w_type, c + e))));
      }
    }
    row_reduce<0, Q>(sum, top, part, buf);
    const float rho = a.norm ? rsqrtf(fmaf(sum, 1.0f / a.N, a.eps)) : 1.f;
    float f = 1.f;
    if (Q) {
      float scale;
      f = row_scale(top * rho, a.norm ? top * rho : sum, scale);
      if (threadIdx.x == 0) a.scale[row] = scale;
    }
    if (threadIdx.x == 0 && a.rho != nullptr) a.rho[row] = rho;
    const S* const from = r != nullptr ? s + row * a.N : x;                // this thread's own stores
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

// Warps of a CTA leave their sums of a column side by side in shared memory and add them in order.
template <class S, class D, int VEC, int NV, int SUB, int THREADS>
__global__ void __launch_bounds__(THREADS) k_rms_backward(const BwdArgs a) {
  next_may_start();                                                        // k_rms_dw
  __shared__ float2 part[2][32];
  constexpr int WIDTH = SUB ? SUB * NV * VEC : 1, GROUPS = SUB ? THREADS / SUB : 1;
  constexpr int AT_ONCE = GROUPS < 8 ? GROUPS : 8;                         // groups of lanes whose sums are in shared memory together
  __shared__ float sums[SUB ? AT_ONCE * WIDTH : 1];
  const int tpr = SUB ? SUB : (int)blockDim.x, t = SUB ? (int)threadIdx.x & (SUB - 1) : (int)threadIdx.x;
  const int rpc = SUB ? GROUPS : 1, sub = SUB ? (int)(threadIdx.x & 31) / SUB : 0;
  const S* const s = static_cast<const S*>(a.s);
  const D* const dy = static_cast<const D*>(a.dy);
  const S* const ds = static_cast<const S*>(a.ds);
  S* const dx = static_cast<S*>(a.dx);
  float w[NV * VEC], acc[NV * VEC];
  load_weights<VEC, NV>(a.w, a.w_type, a.N, t, tpr, w);
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) acc[i] = 0.f;
  int buf = 0;
  const float over_n = 1.0f / a.N;
  for (long long first = (long long)blockIdx.x * rpc + (SUB ? (threadIdx.x >> 5) * (32 / (SUB ? SUB : 32)) : 0); first < a.M;
       first += (long long)gridDim.x * rpc) {
    const long long row = first + sub;
    const bool live = row < a.M;
    Piece<S, VEC> ps[NV], pk[NV];
    Piece<D, VEC> pd[NV];
    const float rho = live ? a.rho[row] : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * tpr) * VEC;
      if (live && c < a.N) ps[i].load(s + row * a.lds + c), pd[i].load(dy + row * a.N + c);
      else ps[i].zero(), pd[i].zero();
    }
    if (ds != nullptr) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * tpr) * VEC;
        if (live && c < a.N) pk[i].load(ds + row * a.N + c);
        else pk[i].zero();
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) pk[i].zero();
    }
    float sum = 0.f, none = 0.f;
#pragma unroll
    for (int i = 0; i < NV * VEC; ++i) {
      const float n = ps[i / VEC].at(i % VEC) * rho, d = pd[i / VEC].at(i % VEC);
      acc[i] = fmaf(d, n, acc[i]);
      sum = fmaf(d * w[i], n, sum);
    }
    row_reduce<SUB, false>(sum, none, part, buf);
    const float m = sum * over_n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * tpr) * VEC;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float n = ps[i].at(e) * rho, g = pd[i].at(e) * w[i * VEC + e];
        o[e] = fmaf(g - n * m, rho, pk[i].at(e));
      }
      if (live && c < a.N) {
        if (dx != nullptr) Out<S, VEC>::store(dx + row * a.N + c, o);
        if (a.dr != nullptr) {
          if (a.dr_type == SPION_BF16) Out<__nv_bfloat16, VEC>::store(static_cast<__nv_bfloat16*>(a.dr) + row * a.N + c, o);
          else Out<__half, VEC>::store(static_cast<__half*>(a.dr) + row * a.N + c, o);
        }
      }
    }
  }
  if (a.part == nullptr) return;
  float* const out = a.part + (long long)blockIdx.x * a.N;
  if (SUB == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * tpr) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c < a.N) out[c + e] = acc[i * VEC + e];
    }
    return;
  }
  const int group = threadIdx.x / (SUB ? SUB : 1);
  float total[(WIDTH + THREADS - 1) / THREADS];
#pragma unroll
  for (int k = 0; k < (WIDTH + THREADS - 1) / THREADS; ++k) total[k] = 0.f;
  for (int g0 = 0; g0 < GROUPS; g0 += AT_ONCE) {
    __syncthreads();
    if (group >= g0 && group < g0 + AT_ONCE) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[(group - g0) * WIDTH + (t + i * tpr) * VEC + e] = acc[i * VEC + e];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < (WIDTH + THREADS - 1) / THREADS; ++k) {
      const int c = threadIdx.x + k * THREADS;
      if (c < WIDTH)
#pragma unroll
        for (int g = 0; g < AT_ONCE; ++g) total[k] += sums[g * WIDTH + c];
    }
  }
#pragma unroll
  for (int k = 0; k < (WIDTH + THREADS - 1) / THREADS; ++k) {
    const int c = threadIdx.x + k * THREADS;
    if (c < WIDTH && c < a.N) out[c] = total[k];
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
    for (int c = threadIdx.x * VEC; c < a.N; c += blockDim.x * VEC) {
      Piece<S, VEC> ps;
      Piece<D, VEC> pd;
      ps.load(s + c), pd.load(dy + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum = fmaf(pd.at(e) * (a.w == nullptr ? 1.f : load_any(a.w, a.w_type, c + e)), ps.at(e) * rho, sum);
    }
    row_reduce<0, false>(sum, none, part, buf);
    const float m = sum / a.N;
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
    for (int r = warp; r < count; r += 32) s += part[(long long)r * N + c];
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
int threads_for(int pieces, int per_thread) { return ((pieces + per_thread - 1) / per_thread + 31) / 32 * 32; }

template <class S, class R, class Y>
int forward(const FwdArgs& a, cudaStream_t st) {
  const bool vec = a.N % 8 == 0 && on_boundary(a.x, a.ldx, type_code<S>()) && on_boundary(a.r, a.ldr, type_code<R>()) &&
                   on_boundary(a.s, a.N, type_code<S>()) && on_boundary(a.y, a.ldy, type_code<Y>());
#define SPION_ROWS(VEC, NV, SUB, THREADS, threads) \
  k_rms_forward<S, R, Y, VEC, NV, SUB, THREADS><<<grid_of(a.M, SUB ? (threads) / (SUB ? SUB : 1) : 1, threads), threads, 0, st>>>(a)
  if (vec) {
    const int n = a.N / 8;
    if (n <= 8) SPION_ROWS(8, 1, 8, CTA, CTA);
    else if (n <= 16) SPION_ROWS(8, 2, 8, CTA, CTA);
    else if (n <= 32) SPION_ROWS(8, 4, 8, CTA, CTA);
    else if (n <= 64) SPION_ROWS(8, 2, 32, CTA, CTA);
    else if (n <= 128) SPION_ROWS(8, 4, 32, CTA, CTA);
    else if (a.M <= sm_count() && n <= 1024) SPION_ROWS(8, 1, 0, 1024, threads_for(n, 1));       // few rows: as many threads as pieces
    else if (n <= 2048) SPION_ROWS(8, 4, 0, 512, threads_for(n, 4));
    else k_rms_forward_wide<S, R, Y, 8><<<grid_of(a.M, 1, 512), 512, 0, st>>>(a);
  } else {
    if (a.N <= 128) SPION_ROWS(1, 4, 32, CTA, CTA);
    else if (a.N <= 512) SPION_ROWS(1, 16, 32, CTA, CTA);
    else if (a.N <= 8192) SPION_ROWS(1, 16, 0, 512, threads_for(a.N, 16));
    else k_rms_forward_wide<S, R, Y, 1><<<grid_of(a.M, 1, 512), 512, 0, st>>>(a);
  }
#undef SPION_ROWS
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

template <class S, class D>
int backward(BwdArgs a, void* dw, int dw_type, cudaStream_t st) {
  const bool vec = a.N % 8 == 0 && on_boundary(a.s, a.lds, type_code<S>()) && on_boundary(a.dy, a.N, type_code<D>()) &&
                   on_boundary(a.ds, a.N, type_code<S>()) && on_boundary(a.dx, a.N, type_code<S>()) && on_boundary(a.dr, a.N, a.dr_type);
  int parts = 0;
  // what is resident at a time and no more: every CTA leaves a partial row
#define SPION_ROWS(VEC, NV, SUB, THREADS, threads, per_sm)                                                                      \
  do {                                                                                                                          \
    const int rpc = SUB ? (threads) / (SUB ? SUB : 1) : 1;                                                                      \
    const long long need = (a.M + rpc - 1) / rpc, most = (long long)sm_count() * (per_sm);                                      \
    parts = (int)(need < most ? need : most);                                                                                   \
    if (parts > MAX_PARTS) parts = MAX_PARTS;                                                                                   \
    k_rms_backward<S, D, VEC, NV, SUB, THREADS><<<parts, threads, 0, st>>>(a);                                                  \
  } while (0)
  if (vec) {
    const int n = a.N / 8;
    if (n <= 8) SPION_ROWS(8, 1, 8, CTA, CTA, 6);
    else if (n <= 16) SPION_ROWS(8, 2, 8, CTA, CTA, 3);
    else if (n <= 64) SPION_ROWS(8, 2, 32, CTA, CTA, 3);
    else if (n <= 1024) SPION_ROWS(8, 2, 0, 512, threads_for(n, 2), 1024 / threads_for(n, 2) < 8 ? 1024 / threads_for(n, 2) : 8);
    else if (n <= 2048) SPION_ROWS(8, 2, 0, 1024, threads_for(n, 2), 1);
  } else {
    if (a.N <= 128) SPION_ROWS(1, 4, 32, CTA, CTA, 4);
    else if (a.N <= 512) SPION_ROWS(1, 16, 32, CTA, CTA, 2);
    else if (a.N <= 8192) SPION_ROWS(1, 16, 0, 512, threads_for(a.N, 16), 1024 / threads_for(a.N, 16) < 8 ? 1024 / threads_for(a.N, 16) : 8);
  }
#undef SPION_ROWS
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
  const FwdArgs a = {x, ldx, res, ldr, w, w_type, sum_out, y, ldy, scale, rstd, M, N, eps, norm};
  const cudaStream_t st = (cudaStream_t)cuda_stream;
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
