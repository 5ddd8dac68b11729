// One AdamW step over many tensors in one launch (decoupled weight decay), with first and second moments in 32 or in 8 bits.
//
//   t += 1;  g = clamp(g, -c, c);  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8 bits: blocks of 256 consecutive values of a tensor share a scale for m, in e4m3, and one for v, in e5m2: powers of two that bring the block's
// largest value to [2^7, 2^8) and [2^14, 2^15).  A power of two leaves a value's code where it is when the block's largest value changes a little, so
// only a value's own changes are rounded.  They are rounded up with the probability of the part that is cut off: v moves by a thousandth a step where
// its codes are 12 to 25 % apart, and rounding to nearest would never move it.  The random bits are a hash of (seed, step, tensor, index), 16 for each
// moment: the same bits on every run, nothing to store.  v is never rounded to zero, which would leave m / eps behind.
//
// Bound by the passes over parameters, gradients and moments: 28 bytes a value with 32-bit moments in fp32, 16 with 8-bit ones.  A warp takes a block of
// 256 values at a time, eight to a lane in one access of each array, so the block's maxima stay in registers.  The table of tensors travels as a kernel
// parameter: nothing is uploaded or kept between calls, and a captured step replays with the addresses it was captured with.
#include <math.h>

#include "rows.cuh"

using namespace rows;

namespace {

constexpr int BLOCK = 256, CTA = 256, CHUNK = 8 * BLOCK;       // values of a chunk: a block per warp
constexpr int FEW = 64, MOST = 512;                             // tensors of a launch

struct Tensor {
  void* p;
  const void* g;
  void* copy;                 // or null: p in 16 bits
  long long n, at;            // values, place of the first in the moments (a multiple of 256)
  int chunk, index;           // first chunk of the launch, number of the tensor
};
struct Step {
  void *m, *v;
  float *m_scale, *v_scale;   // 8 bits: one per block
  const float* steps;
  const float* lr_dev;        // or null: lr
  double lr, b1, b2, wd;
  float eps, clip;            // clip < 0: none
  unsigned seed;
  int count, chunks, copy_type;
};
template <int MAX> struct Table {
  Step s;
  Tensor t[MAX];
};

// xor-shift and multiply, twice: the 32-bit mixing function "lowbias32" of C. Wellons
__device__ __forceinline__ unsigned mix(unsigned x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

// x in units of its scale -> code of an 8-bit float with EXP exponent bits: times 2^(bias - 127) an fp32 number has the code's own exponent bits
// (subnormal codes are subnormal fp32 numbers), and the code is what stands above the cut.
template <int EXP> __device__ __forceinline__ unsigned code_of(float x, unsigned noise16) {
  constexpr int MANT = 7 - EXP, CUT = 23 - MANT;
  constexpr float FIT = EXP == 4 ? 0x1p-120f : 0x1p-112f;
  unsigned c = (__float_as_uint(fabsf(x) * FIT) + (noise16 << (CUT - 16))) >> CUT;
  if (!(fabsf(x) <= 3.402823466e38f)) c = x != x || EXP == 4 ? 0x7fu : 0x7cu;
  return c | (__float_as_uint(x) >> 31 << 7);
}
__device__ __forceinline__ float from_e4m3(unsigned c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}
__device__ __forceinline__ float from_e5m2(unsigned c) { return __half2float(__ushort_as_half((unsigned short)(c << 8))); }
// 2^(exponent of a - below); a >= 2^-100
__device__ __forceinline__ float scale_of(float a, int below) { return __uint_as_float(((__float_as_uint(a) >> 23) - below) << 23); }
__device__ __forceinline__ float over_scale(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }      // 1 / a power of two
__device__ __forceinline__ float size_if_finite(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f; }

// The products and sums that the moments' codes depend on are rounded one by one, as written (no contraction).
template <class P, int BITS, int MAX>
__global__ void __launch_bounds__(CTA, 4) k_adamw(const __grid_constant__ Table<MAX> a) {
  next_may_start();                                                      // k_adamw_steps
  __shared__ float s_factor[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int i = 0;
  float known = -1.f, lr_m = 0.f, root_v = 0.f;                          // the step that the factors are for
  const float b1 = (float)a.s.b1, b2 = (float)a.s.b2, c1 = (float)(1.0 - a.s.b1), c2 = (float)(1.0 - a.s.b2);
  const double lr = a.s.lr_dev != nullptr ? (double)*a.s.lr_dev : a.s.lr;
  const float keep = (float)(1.0 - lr * a.s.wd);
  for (int chunk = blockIdx.x; chunk < a.s.chunks; chunk += gridDim.x) {
    int lo = i, hi = a.s.count;                                          // the last tensor that begins at or before the chunk
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.t[mid].chunk <= chunk) lo = mid;
      else hi = mid;
    }
    i = lo;
    const Tensor& t = a.t[i];
    const long long base = (long long)(chunk - t.chunk) * CHUNK + warp * BLOCK;     // of the warp's block in its tensor
    const float step = a.s.steps[t.index] + 1.f;
    P* const p = static_cast<P*>(t.p) + base;
    const P* const g = static_cast<const P*>(t.g) + base;
    const long long left = t.n - base;                                   // may be none
    const bool whole = left >= BLOCK && (((uintptr_t)p | (uintptr_t)g) & (8 * sizeof(P) - 1)) == 0 &&
                       (t.copy == nullptr || ((uintptr_t)t.copy & 15) == 0);
    // whole blocks on a boundary: a lane has values 8 lane .. 8 lane + 7, else values lane, lane + 32, ...
    const int first = whole ? 8 * lane : lane, stride = whole ? 1 : 32;
    const long long at = t.at + base;
    float pv[8], gv[8], m[8], v[8];
    if (whole) {
      Piece<P, 8> pp, pg;
      pp.load(p + first);
      pg.load(g + first);
      if (BITS == 32) {
        Piece<float, 8> pm, pw;
        pm.load(static_cast<const float*>(a.s.m) + at + first);
        pw.load(static_cast<const float*>(a.s.v) + at + first);
#pragma unroll
        for (int e = 0; e < 8; ++e) m[e] = pm.at(e), v[e] = pw.at(e);
      } else {
        const uint2 cm = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.s.m) + at + first);
        const uint2 cv = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.s.v) + at + first);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m[e] = from_e4m3(((e < 4 ? cm.x : cm.y) >> (8 * (e & 3))) & 0xffu);
          v[e] = from_e5m2(((e < 4 ? cv.x : cv.y) >> (8 * (e & 3))) & 0xffu);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) pv[e] = pp.at(e), gv[e] = pg.at(e);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = first + 32 * e;
        const bool in = k < left;
        pv[e] = in ? as_float(p[k]) : 0.f;
        gv[e] = in ? as_float(g[k]) : 0.f;
        if (BITS == 32) {
          m[e] = in ? static_cast<const float*>(a.s.m)[at + k] : 0.f;
          v[e] = in ? static_cast<const float*>(a.s.v)[at + k] : 0.f;
        } else {
          m[e] = in ? from_e4m3(static_cast<const uint8_t*>(a.s.m)[at + k]) : 0.f;
          v[e] = in ? from_e5m2(static_cast<const uint8_t*>(a.s.v)[at + k]) : 0.f;
        }
      }
    }
    float sm = 0.f, sv = 0.f;
    if (BITS == 8 && left > 0) sm = a.s.m_scale[at / BLOCK], sv = a.s.v_scale[at / BLOCK];
    if (step != known) {                                                 // (the same for the whole CTA)
      __syncthreads();
      if (threadIdx.x == 0) s_factor[0] = (float)(lr / (1.0 - pow(a.s.b1, (double)step)));
      if (threadIdx.x == 32) s_factor[1] = (float)(1.0 / sqrt(1.0 - pow(a.s.b2, (double)step)));
      __syncthreads();
      lr_m = s_factor[0], root_v = s_factor[1];
      known = step;
    }
    if (left <= 0) continue;
    float top_m = 0x1p-100f, top_v = 0x1p-100f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (a.s.clip >= 0.f) gv[e] = gv[e] < -a.s.clip ? -a.s.clip : gv[e] > a.s.clip ? a.s.clip : gv[e];      // NaN stays
      if (BITS == 8) m[e] *= sm, v[e] *= sv;
      m[e] = __fadd_rn(__fmul_rn(m[e], b1), __fmul_rn(gv[e], c1));
      v[e] = __fadd_rn(__fmul_rn(v[e], b2), __fmul_rn(__fmul_rn(gv[e], gv[e]), c2));
      pv[e] = pv[e] * keep - lr_m * (m[e] / (sqrtf(v[e]) * root_v + a.s.eps));
      if (BITS == 8) top_m = fmaxf(top_m, size_if_finite(m[e])), top_v = fmaxf(top_v, size_if_finite(v[e]));
    }
    unsigned cm[8], cv[8];
    if (BITS == 8) {
      top_m = lane_max<32>(top_m);
      top_v = lane_max<32>(top_v);
      sm = scale_of(top_m, 7), sv = scale_of(top_v, 14);
      if (lane == 0) a.s.m_scale[at / BLOCK] = sm, a.s.v_scale[at / BLOCK] = sv;
      const float um = over_scale(sm), uv = over_scale(sv);
      const unsigned key = mix(mix(a.s.seed + mix((unsigned)step * 0x9E3779B1u + (unsigned)t.index)) + (unsigned)(base >> 32));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned r = mix((unsigned)(base + first + stride * e) ^ key);
        cm[e] = code_of<4>(m[e] * um, r & 0xffffu);
        cv[e] = code_of<5>(v[e] * uv, r >> 16);
        if (cv[e] == 0 && v[e] > 0.f) cv[e] = 1;
      }
    }
    if (whole) {
      Out<P, 8>::store(p + first, pv);
      if (BITS == 32) {
        Out<float, 8>::store(static_cast<float*>(a.s.m) + at + first, m);
        Out<float, 8>::store(static_cast<float*>(a.s.v) + at + first, v);
      } else {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.s.m) + at + first) =
            make_uint2(cm[0] | cm[1] << 8 | cm[2] << 16 | cm[3] << 24, cm[4] | cm[5] << 8 | cm[6] << 16 | cm[7] << 24);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.s.v) + at + first) =
            make_uint2(cv[0] | cv[1] << 8 | cv[2] << 16 | cv[3] << 24, cv[4] | cv[5] << 8 | cv[6] << 16 | cv[7] << 24);
      }
      if (t.copy != nullptr) {
        if (a.s.copy_type == SPION_BF16) Out<__nv_bfloat16, 8>::store(static_cast<__nv_bfloat16*>(t.copy) + base + first, pv);
        else Out<__half, 8>::store(static_cast<__half*>(t.copy) + base + first, pv);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = first + 32 * e;
        if (k >= left) continue;
        p[k] = rounded<P>(pv[e]);
        if (BITS == 32) {
          static_cast<float*>(a.s.m)[at + k] = m[e];
          static_cast<float*>(a.s.v)[at + k] = v[e];
        } else {
          static_cast<uint8_t*>(a.s.m)[at + k] = (uint8_t)cm[e];
          static_cast<uint8_t*>(a.s.v)[at + k] = (uint8_t)cv[e];
        }
        if (t.copy != nullptr) store_any(t.copy, a.s.copy_type, base + k, pv[e]);
      }
    }
  }
}

// The counts go up when every CTA has read them.
template <int MAX> struct Indices {
  float* steps;
  int count;
  int index[MAX];
};
template <int MAX> __global__ void __launch_bounds__(MAX) k_adamw_steps(const __grid_constant__ Indices<MAX> a) {
  wait_for_kernel_before();
  if ((int)threadIdx.x < a.count) a.steps[a.index[threadIdx.x]] += 1.f;
}

template <class P, int BITS, int MAX>
int launch(const Step& s, const spion_adamw_tensor* ts, int count, float* steps, cudaStream_t st) {
  Table<MAX> a;
  Indices<MAX> ix;
  a.s = s;
  a.s.count = 0;
  ix.steps = steps;
  ix.count = 0;
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    ix.index[ix.count++] = ts[i].index;
    if (ts[i].n == 0) continue;
    a.t[a.s.count++] = Tensor{ts[i].p, ts[i].g, ts[i].copy, ts[i].n, ts[i].at, (int)chunks, ts[i].index};
    chunks += (ts[i].n + CHUNK - 1) / CHUNK;
    if (chunks > 0x7fffffff) return SPION_ERR_SHAPE;
  }
  a.s.chunks = (int)chunks;
  if (chunks > 0) {
    const long long most = (long long)sm_count() * 4;
    k_adamw<P, BITS, MAX><<<(int)(chunks < most ? chunks : most), CTA, 0, st>>>(a);
    SPION_LAUNCH_CHECK();
  }
  SPION_CUDA_TRY(launch_after(k_adamw_steps<MAX>, dim3(1), dim3(MAX), 0, st, ix));
  return SPION_OK;
}
template <class P, int BITS>
int launches(const Step& s, const spion_adamw_tensor* ts, int count, float* steps, cudaStream_t st) {
  for (int i = 0; i < count; i += MOST) {
    const int n = count - i < MOST ? count - i : MOST;
    const int rc = n <= FEW ? launch<P, BITS, FEW>(s, ts + i, n, steps, st) : launch<P, BITS, MOST>(s, ts + i, n, steps, st);
    if (rc != SPION_OK) return rc;
  }
  return SPION_OK;
}

}  // namespace

extern "C" int spion_adamw_step(const spion_adamw_tensor* host_tensors, int count, int type, int state_bits, void* m, void* v, float* m_scale,
                                float* v_scale, float* steps, const float* lr_dev, double lr, double beta1, double beta2, double eps,
                                double weight_decay, double clip_value, unsigned seed, int copy_type, void* cuda_stream) {
  if (count < 0 || (state_bits != 8 && state_bits != 32)) return SPION_ERR_ARG;
  if (count == 0) return SPION_OK;
  if (host_tensors == nullptr || m == nullptr || v == nullptr || steps == nullptr || (state_bits == 8) != (m_scale != nullptr && v_scale != nullptr))
    return SPION_ERR_ARG;
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && weight_decay >= 0) || (lr_dev == nullptr && !(lr >= 0))) return SPION_ERR_ARG;
  if (((uintptr_t)m | (uintptr_t)v) & 31) return SPION_ERR_ARG;
  for (int i = 0; i < count; ++i) {
    const spion_adamw_tensor& t = host_tensors[i];
    if (t.n < 0 || t.at < 0 || t.at % BLOCK || t.index < 0 || (t.n > 0 && (t.p == nullptr || t.g == nullptr))) return SPION_ERR_ARG;
    if (t.copy != nullptr && copy_type != SPION_BF16 && copy_type != SPION_F16) return SPION_ERR_ARG;
  }
  const Step s = {m, v, m_scale, v_scale, steps, lr_dev, lr, beta1, beta2, weight_decay, (float)eps, clip_value >= 0 ? (float)clip_value : -1.f, seed, 0, 0,
                  copy_type};
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  if (type == SPION_F32) return state_bits == 8 ? launches<float, 8>(s, host_tensors, count, steps, st) : launches<float, 32>(s, host_tensors, count, steps, st);
  if (type == SPION_BF16)
    return state_bits == 8 ? launches<__nv_bfloat16, 8>(s, host_tensors, count, steps, st) : launches<__nv_bfloat16, 32>(s, host_tensors, count, steps, st);
  if (type == SPION_F16) return state_bits == 8 ? launches<__half, 8>(s, host_tensors, count, steps, st) : launches<__half, 32>(s, host_tensors, count, steps, st);
  return SPION_ERR_UNSUPPORTED;
}
