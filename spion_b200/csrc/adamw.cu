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
  int index;                  // number of the tensor
};
struct Step {
  void *m, *v;
  float *m_scale, *v_scale;   // 8 bits: one per block
  const float* steps;
  const float* lr_dev;        // or null: lr
  double lr, wd, log_b1, log_b2;
  float b1, b2, c1, c2;       // betas and what is left of one
  float eps, clip;            // clip < 0: none
  unsigned seed;
  int count, chunks, copy_type;
};
template <int MAX> struct Table {
  Step s;
  int chunk[MAX];             // first chunk of each tensor (beside one another: a search touches few lines of the constant memory)
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

// An 8-bit float's code stands in the top byte of a word here.  Times 2^(bias - 127), a value in units of its scale has the code's own exponent bits as an
// fp32 number (subnormal codes are subnormal fp32 numbers): above bit 20 (e4m3) or 21 (e5m2) stands the code, what is added below it is the chance of
// the next one.
constexpr float FIT_E4M3 = 0x1p-120f, FIT_E5M2 = 0x1p-112f;
__device__ __forceinline__ unsigned code_e4m3(float fitted, unsigned r) {
  const unsigned x = __float_as_uint(fitted);                            // sign and size; the size is below 2^27 and stays so
  return ((x + ((r & 0xffffu) << 4)) << 4 & 0x7fffffffu) | (x & 0x80000000u);
}
__device__ __forceinline__ unsigned code_e5m2(float fitted, unsigned r) {
  unsigned x = __float_as_uint(fitted);
  return (x + (r >> 16 << 5)) << 3;
}
// four bytes, each the top one of its word
__device__ __forceinline__ unsigned top_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
__device__ __forceinline__ float2 from_e4m3x2(unsigned two) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
}
__device__ __forceinline__ float2 from_e5m2x2(unsigned word, unsigned select) {      // an e5m2 is the upper byte of an fp16
  const unsigned h = __byte_perm(word, 0, select);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float from_e4m3(unsigned c) { return from_e4m3x2(c).x; }
__device__ __forceinline__ float from_e5m2(unsigned c) { return from_e5m2x2(c, 0x1404).x; }
__device__ __forceinline__ float max_nan(float a, float b) {             // NaN if either is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float lane_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// the update's quotient: two units in the last place are lost beside a parameter that is many times as large
__device__ __forceinline__ float root_of(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 2^(exponent of a - below); a >= 2^-100
__device__ __forceinline__ float scale_of(float a, int below) { return __uint_as_float(((__float_as_uint(a) >> 23) - below) << 23); }
__device__ __forceinline__ float over_scale(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }      // 1 / a power of two
__device__ __forceinline__ float size_if_finite(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f; }

// The products and sums that the moments' codes depend on are rounded one by one, as written (no contraction).
template <class P, int BITS, int MAX>
__global__ void __launch_bounds__(CTA, BITS == 8 ? 3 : 4) k_adamw(const __grid_constant__ Table<MAX> a) {
  next_may_start();                                                      // k_adamw_steps
  __shared__ float s_factor[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int i = 0;
  float known = -1.f, lr_m = 0.f, root_v = 0.f;                          // the step that the factors are for
  const float b1 = a.s.b1, b2 = a.s.b2, c1 = a.s.c1, c2 = a.s.c2;
  const double lr = a.s.lr_dev != nullptr ? (double)*a.s.lr_dev : a.s.lr;
  const float keep = (float)(1.0 - lr * a.s.wd);
  for (int chunk = blockIdx.x; chunk < a.s.chunks; chunk += gridDim.x) {
    int lo = i, hi = a.s.count;                                          // the last tensor that begins at or before the chunk
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.chunk[mid] <= chunk) lo = mid;
      else hi = mid;
    }
    i = lo;
    const Tensor& t = a.t[i];
    const long long base = (long long)(chunk - a.chunk[i]) * CHUNK + warp * BLOCK;     // of the warp's block in its tensor
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
        for (int e = 0; e < 8; e += 2) {
          const unsigned wm = e < 4 ? cm.x : cm.y, wv = e < 4 ? cv.x : cv.y;
          const float2 fm = from_e4m3x2(e & 2 ? wm >> 16 : wm & 0xffffu), fv = from_e5m2x2(wv, e & 2 ? 0x3424 : 0x1404);
          m[e] = fm.x, m[e + 1] = fm.y, v[e] = fv.x, v[e + 1] = fv.y;
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
      if (threadIdx.x == 0) s_factor[0] = (float)(lr / -expm1((double)step * a.s.log_b1));
      if (threadIdx.x == 32) s_factor[1] = (float)(1.0 / sqrt(-expm1((double)step * a.s.log_b2)));
      __syncthreads();
      lr_m = s_factor[0], root_v = s_factor[1];
      known = step;
    }
    if (left <= 0) continue;
    if (a.s.clip >= 0.f)
#pragma unroll
      for (int e = 0; e < 8; ++e) gv[e] = min_nan(max_nan(gv[e], -a.s.clip), a.s.clip);      // NaN stays
    float top_m = 0x1p-100f, top_v = 0x1p-100f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (BITS == 8) m[e] *= sm, v[e] *= sv;
      m[e] = __fadd_rn(__fmul_rn(m[e], b1), __fmul_rn(gv[e], c1));
      v[e] = __fadd_rn(__fmul_rn(v[e], b2), __fmul_rn(__fmul_rn(gv[e], gv[e]), c2));
      pv[e] = pv[e] * keep - lr_m * __fdividef(m[e], root_of(v[e]) * root_v + a.s.eps);
      if (BITS == 8) top_m = max_nan(top_m, fabsf(m[e])), top_v = max_nan(top_v, v[e]);
    }
    uint2 cm, cv;                                                        // codes, one to a byte
    if (BITS == 8) {
      top_m = lane_max_nan(top_m);
      top_v = lane_max_nan(top_v);
      const unsigned key = mix(mix(a.s.seed + mix((unsigned)step * 0x9E3779B1u + (unsigned)t.index)) + (unsigned)(base >> 32));
      unsigned r[8], wm[8], wv[8];                                       // random bits; codes in the top bytes
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = mix((unsigned)(base + first + stride * e) ^ key);
      if (top_m < 0x1p14f && top_v < 0x1p28f) {                          // all finite, and scale and fit are one factor within fp32's range
        sm = scale_of(top_m, 7), sv = scale_of(top_v, 14);
        const float um = over_scale(sm) * FIT_E4M3, uv = over_scale(sv) * FIT_E5M2;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          wm[e] = code_e4m3(m[e] * um, r[e]);
          // never zero beside a first moment that is not
          wv[e] = code_e5m2(v[e] > 0.f ? fmaxf(v[e] * uv, __uint_as_float(1u << 21)) : 0.f, r[e]);
        }
      } else {
        top_m = top_v = 0x1p-100f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top_m = fmaxf(top_m, size_if_finite(m[e])), top_v = fmaxf(top_v, size_if_finite(v[e]));
        sm = scale_of(lane_max<32>(top_m), 7), sv = scale_of(lane_max<32>(top_v), 14);
        const float um = over_scale(sm), uv = over_scale(sv);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          wm[e] = code_e4m3(m[e] * um * FIT_E4M3, r[e]);
          if (size_if_finite(m[e]) != fabsf(m[e])) wm[e] = 0x7fu << 24;  // an infinity is a NaN in e4m3
          wv[e] = code_e5m2(v[e] > 0.f ? fmaxf(v[e] * uv * FIT_E5M2, __uint_as_float(1u << 21)) : 0.f, r[e]);
          if (size_if_finite(v[e]) != v[e]) wv[e] = (v[e] != v[e] ? 0x7fu : 0x7cu) << 24;
        }
      }
      cm = make_uint2(top_bytes(wm[0], wm[1], wm[2], wm[3]), top_bytes(wm[4], wm[5], wm[6], wm[7]));
      cv = make_uint2(top_bytes(wv[0], wv[1], wv[2], wv[3]), top_bytes(wv[4], wv[5], wv[6], wv[7]));
      if (lane == 0) a.s.m_scale[at / BLOCK] = sm, a.s.v_scale[at / BLOCK] = sv;
    }
    if (whole) {
      Out<P, 8>::store(p + first, pv);
      if (BITS == 32) {
        Out<float, 8>::store(static_cast<float*>(a.s.m) + at + first, m);
        Out<float, 8>::store(static_cast<float*>(a.s.v) + at + first, v);
      } else {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.s.m) + at + first) = cm;
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.s.v) + at + first) = cv;
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
          static_cast<uint8_t*>(a.s.m)[at + k] = (uint8_t)((e < 4 ? cm.x : cm.y) >> (8 * (e & 3)));
          static_cast<uint8_t*>(a.s.v)[at + k] = (uint8_t)((e < 4 ? cv.x : cv.y) >> (8 * (e & 3)));
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
    a.chunk[a.s.count] = (int)chunks;
    a.t[a.s.count++] = Tensor{ts[i].p, ts[i].g, ts[i].copy, ts[i].n, ts[i].at, ts[i].index};
    chunks += (ts[i].n + CHUNK - 1) / CHUNK;
    if (chunks > 0x7fffffff) return SPION_ERR_SHAPE;
  }
  a.s.chunks = (int)chunks;
  if (chunks > 0) {
    const long long most = (long long)sm_count() * (BITS == 8 ? 3 : 4);
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
  const Step s = {m, v, m_scale, v_scale, steps, lr_dev, lr, weight_decay, log(beta1), log(beta2), (float)beta1, (float)beta2, (float)(1.0 - beta1),
                  (float)(1.0 - beta2), (float)eps, clip_value >= 0 ? (float)clip_value : -1.f, seed, 0, 0, copy_type};
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  if (type == SPION_F32) return state_bits == 8 ? launches<float, 8>(s, host_tensors, count, steps, st) : launches<float, 32>(s, host_tensors, count, steps, st);
  if (type == SPION_BF16)
    return state_bits == 8 ? launches<__nv_bfloat16, 8>(s, host_tensors, count, steps, st) : launches<__nv_bfloat16, 32>(s, host_tensors, count, steps, st);
  if (type == SPION_F16) return state_bits == 8 ? launches<__half, 8>(s, host_tensors, count, steps, st) : launches<__half, 32>(s, host_tensors, count, steps, st);
  return SPION_ERR_UNSUPPORTED;
}
