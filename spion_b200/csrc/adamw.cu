// One AdamW step over many tensors in one launch, and a small one before it (decoupled weight decay), with first and second moments in 32 or in 8 bits.
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
// Bound by the passes over parameters, gradients and moments: 28 bytes a value with 32-bit moments in fp32 (75 million values 337 us, 6.2 TB/s), 16 with
// 8-bit ones, where the arithmetic of the codes is nearly as long (213 us; in bf16, 10 bytes a value, 205: that arithmetic; with bulk copies to shared memory
// three chunks ahead 213 and 208, one tensor of 75 million 221 instead of 212, so there are none).  A warp takes a block of
// 256 values at a time, eight to a lane in one access of each array, so the block's maxima stay in registers.  The table of tensors travels as a kernel
// parameter: nothing is uploaded or kept between calls, and a captured step replays with the addresses it was captured with.
#include <math.h>

#include <type_traits>

#include "rows.cuh"

using namespace rows;

namespace {

constexpr int BLOCK = 256, CTA = 256, CHUNK = CTA / 32 * BLOCK;  // values that share scales; threads; values that a CTA takes at a time, a block per warp
// Tensors of a launch, by the table that travels with it: up to 64 tensors with that of 64 12.8 us a call on the host, with that of 256 14.1 (the same on the device); one of
// 512, 24 KB, cost 100 tensors 10 us more.
constexpr int FEW = 64, MOST = 256;

struct Tensor {
  void* p;
  const void* g;
  void* copy;                 // or null: p in 16 bits
  long long n, at;            // values, place of the first in the moments (a multiple of 256)
};
struct Step {
  void *m, *v;
  float *m_scale, *v_scale;   // 8 bits: one per block
  const float4* factors;      // of each tensor of the launch, from k_adamw_begin; z < 0: nothing is to be changed
  float b1, b2, c1, c2;       // betas and what is left of one
  float eps, clip;            // clip < 0: none
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
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// The update's quotient: a few units in its last place are lost beside a parameter that is many times as large.  FLUSH: v below fp32's normal numbers, 2^-126,
// counts as zero.  Its corrected root is at most 2^-63 / sqrt(1 - b2) at any step, 2^-24 of an eps of 2^-39 / sqrt(1 - b2) or more (b2 = 0.999: 5.8e-11);
// steps with a smaller eps take the exact forms.
template <bool FLUSH> __device__ __forceinline__ float quotient(float m, float v, float root_v, float eps) {
  if (!FLUSH) return m / (sqrtf(v) * root_v + eps);
  float r, q;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(r * root_v + eps));
  return m * q;
}
// 2^(exponent of a - below); a >= 2^-100
__device__ __forceinline__ float scale_of(float a, int below) { return __uint_as_float(((__float_as_uint(a) >> 23) - below) << 23); }
__device__ __forceinline__ float over_scale(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }      // 1 / a power of two
__device__ __forceinline__ float size_if_finite(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f; }

// What a lane has of a block of 256: eight values as they lie in memory.
template <class P, int BITS> struct Lane {
  Piece<P, 8> p, g;
  typename std::conditional<BITS == 32, Piece<float, 8>, uint2>::type m, v;
  float sm, sv;
};
// The step on eight values.  The products and sums that the moments' codes depend on are rounded one by one, as written (no contraction).
// `place` + `stride` e: the values' places in their tensor.
template <int BITS, bool FLUSH>
__device__ __forceinline__ void update(const Step& s, const float4& f, float (&p)[8], float (&g)[8], float (&m)[8], float (&v)[8], float& sm, float& sv, uint2& cm, uint2& cv,
                                       unsigned place, unsigned stride, unsigned key) {
  if (s.clip >= 0.f)
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = min_nan(max_nan(g[e], -s.clip), s.clip);      // NaN stays
  float top_m = 0x1p-100f, top_v = 0x1p-100f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (BITS == 8) m[e] *= sm, v[e] *= sv;
    m[e] = __fadd_rn(__fmul_rn(m[e], s.b1), __fmul_rn(g[e], s.c1));
    v[e] = __fadd_rn(__fmul_rn(v[e], s.b2), __fmul_rn(__fmul_rn(g[e], g[e]), s.c2));
    p[e] = p[e] * f.x - f.y * quotient<FLUSH>(m[e], v[e], f.z, s.eps);
    if (BITS == 8) top_m = max_nan(top_m, fabsf(m[e])), top_v = max_nan(top_v, v[e]);
  }
  if (BITS == 32) return;
  top_m = lane_max_nan<32>(top_m);
  top_v = lane_max_nan<32>(top_v);
  unsigned wm[8], wv[8];                                                 // codes in the top bytes
  if (top_m < 0x1p14f && top_v < 0x1p28f) {                              // all finite, and scale and fit are one factor within fp32's range
    sm = scale_of(top_m, 7), sv = scale_of(top_v, 14);
    const float um = over_scale(sm) * FIT_E4M3, uv = over_scale(sv) * FIT_E5M2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned r = mix((place + stride * e) ^ key);
      wm[e] = code_e4m3(m[e] * um, r);
      wv[e] = code_e5m2(v[e] > 0.f ? fmaxf(v[e] * uv, __uint_as_float(1u << 21)) : 0.f, r);      // never zero beside a first moment that is not
    }
  } else {
    top_m = top_v = 0x1p-100f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top_m = fmaxf(top_m, size_if_finite(m[e])), top_v = fmaxf(top_v, size_if_finite(v[e]));
    sm = scale_of(lane_max<32>(top_m), 7), sv = scale_of(lane_max<32>(top_v), 14);
    const float um = over_scale(sm), uv = over_scale(sv);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned r = mix((place + stride * e) ^ key);
      wm[e] = code_e4m3(m[e] * um * FIT_E4M3, r);
      if (size_if_finite(m[e]) != fabsf(m[e])) wm[e] = 0x7fu << 24;      // an infinity is a NaN in e4m3
      wv[e] = code_e5m2(v[e] > 0.f ? fmaxf(v[e] * uv * FIT_E5M2, __uint_as_float(1u << 21)) : 0.f, r);
      if (size_if_finite(v[e]) != v[e]) wv[e] = (v[e] != v[e] ? 0x7fu : 0x7cu) << 24;
    }
  }
  cm = make_uint2(top_bytes(wm[0], wm[1], wm[2], wm[3]), top_bytes(wm[4], wm[5], wm[6], wm[7]));
  cv = make_uint2(top_bytes(wv[0], wv[1], wv[2], wv[3]), top_bytes(wv[4], wv[5], wv[6], wv[7]));
}

// A whole block on its boundaries: a lane has values 8 lane .. 8 lane + 7.
template <class P, int BITS, bool FLUSH>
__device__ __forceinline__ void whole_block(const Step& s, const Tensor& t, const Lane<P, BITS>& now, long long base, int lane, const float4& f, unsigned key) {
  const long long k = base + 8 * lane, at = t.at + k;
  float p[8], g[8], m[8], v[8], sm = now.sm, sv = now.sv;
  uint2 cm, cv;
#pragma unroll
  for (int e = 0; e < 8; ++e) p[e] = now.p.at(e), g[e] = now.g.at(e);
  if constexpr (BITS == 32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = now.m.at(e), v[e] = now.v.at(e);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const unsigned x = e < 4 ? now.m.x : now.m.y, y = e < 4 ? now.v.x : now.v.y;
      const float2 fm = from_e4m3x2(e & 2 ? x >> 16 : x & 0xffffu), fv = from_e5m2x2(y, e & 2 ? 0x3424 : 0x1404);
      m[e] = fm.x, m[e + 1] = fm.y, v[e] = fv.x, v[e + 1] = fv.y;
    }
  }
  update<BITS, FLUSH>(s, f, p, g, m, v, sm, sv, cm, cv, (unsigned)k, 1, key);
  Out<P, 8>::store(static_cast<P*>(t.p) + k, p);
  if constexpr (BITS == 32) {
    Out<float, 8>::store(static_cast<float*>(s.m) + at, m);
    Out<float, 8>::store(static_cast<float*>(s.v) + at, v);
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(s.m) + at) = cm;
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(s.v) + at) = cv;
    if (lane == 0) s.m_scale[at / BLOCK] = sm, s.v_scale[at / BLOCK] = sv;
  }
  if (t.copy != nullptr) {
    if (s.copy_type == SPION_BF16) Out<__nv_bfloat16, 8>::store(static_cast<__nv_bfloat16*>(t.copy) + k, p);
    else Out<__half, 8>::store(static_cast<__half*>(t.copy) + k, p);
  }
}
// A tensor's last block, and tensors that lie off the boundaries: a lane has values lane, lane + 32, ...  `begun` waits for the factors.
template <class P, int BITS, bool FLUSH, class F>
__device__ __forceinline__ void edge_block(const Step& s, const Tensor& t, long long base, long long end, int lane, float4& f, unsigned& key, F begun) {
  const int left = (int)min(end - base, (long long)BLOCK);
  const long long at = t.at + base;
  P* const tp = static_cast<P*>(t.p) + base;
  const P* const tg = static_cast<const P*>(t.g) + base;
  float p[8], g[8], m[8], v[8], sm = 0.f, sv = 0.f;
  uint2 cm, cv;
  if (BITS == 8) sm = s.m_scale[at / BLOCK], sv = s.v_scale[at / BLOCK];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int k = lane + 32 * e;
    const bool in = k < left;
    p[e] = in ? as_float(tp[k]) : 0.f;
    g[e] = in ? as_float(tg[k]) : 0.f;
    if (BITS == 32) {
      m[e] = in ? static_cast<const float*>(s.m)[at + k] : 0.f;
      v[e] = in ? static_cast<const float*>(s.v)[at + k] : 0.f;
    } else {
      m[e] = in ? from_e4m3(static_cast<const uint8_t*>(s.m)[at + k]) : 0.f;
      v[e] = in ? from_e5m2(static_cast<const uint8_t*>(s.v)[at + k]) : 0.f;
    }
  }
  begun();
  if (f.z < 0.f) return;
  update<BITS, FLUSH>(s, f, p, g, m, v, sm, sv, cm, cv, (unsigned)(base + lane), 32, key);
  if (BITS == 8 && lane == 0) s.m_scale[at / BLOCK] = sm, s.v_scale[at / BLOCK] = sv;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int k = lane + 32 * e;
    if (k >= left) continue;
    tp[k] = rounded<P>(p[e]);
    if (BITS == 32) {
      static_cast<float*>(s.m)[at + k] = m[e];
      static_cast<float*>(s.v)[at + k] = v[e];
    } else {
      static_cast<uint8_t*>(s.m)[at + k] = (uint8_t)((e < 4 ? cm.x : cm.y) >> (8 * (e & 3)));
      static_cast<uint8_t*>(s.v)[at + k] = (uint8_t)((e < 4 ? cv.x : cv.y) >> (8 * (e & 3)));
    }
    if (t.copy != nullptr) store_any(t.copy, s.copy_type, base + k, p[e]);
  }
}
// the last tensor that begins at or before a chunk, from an earlier one
template <int MAX> __device__ __forceinline__ int tensor_of(const Table<MAX>& a, int chunk, int i) {
  if (i + 1 < a.s.count && a.chunk[i + 1] <= chunk) {
    int hi = a.s.count;
    while (hi - i > 1) {
      const int mid = (i + hi) >> 1;
      if (a.chunk[mid] <= chunk) i = mid;
      else hi = mid;
    }
  }
  return i;
}
template <class P> __device__ __forceinline__ bool on_boundaries(const Tensor& t) {
  return (((uintptr_t)t.p | (uintptr_t)t.g) & (8 * sizeof(P) - 1)) == 0 && ((uintptr_t)t.copy & 15) == 0;
}

constexpr int CTAS = 4;                                                  // resident on a multiprocessor
template <class P, int BITS, bool FLUSH, int MAX>
__global__ void __launch_bounds__(CTA, CTAS) k_adamw(const __grid_constant__ Table<MAX> a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int i = 0;
  for (int chunk = blockIdx.x; chunk < a.s.chunks; chunk += gridDim.x) {
    i = tensor_of(a, chunk, i);
    const Tensor& t = a.t[i];
    const long long base = (long long)(chunk - a.chunk[i]) * CHUNK + warp * BLOCK;     // of the warp's block in its tensor
    if (base >= t.n) continue;
    float4 f;
    unsigned key;
    // k_adamw_begin has been started after everything that this step reads was written: only what it writes itself is waited for, with the block's values
    // on their way
    auto begun = [&] {
      wait_for_kernel_before();
      f = __ldcg(a.s.factors + i);
      key = mix(__float_as_uint(f.w) + (unsigned)(base >> 32));
    };
    if (base + BLOCK > t.n || !on_boundaries<P>(t)) {
      edge_block<P, BITS, FLUSH>(a.s, t, base, t.n, lane, f, key, begun);
      continue;
    }
    const long long k = base + 8 * lane, at = t.at + k;
    Lane<P, BITS> now;
    now.p.load(static_cast<P*>(t.p) + k);
    now.g.load(static_cast<const P*>(t.g) + k);
    if constexpr (BITS == 32) {
      now.m.load(static_cast<const float*>(a.s.m) + at);
      now.v.load(static_cast<const float*>(a.s.v) + at);
    } else {
      now.m = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.s.m) + at);
      now.v = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.s.v) + at);
      now.sm = a.s.m_scale[at / BLOCK];
      now.sv = a.s.v_scale[at / BLOCK];
    }
    begun();
    if (f.z < 0.f) return;
    whole_block<P, BITS, FLUSH>(a.s, t, now, base, lane, f, key);
  }
}

// Counts go up, and what a tensor's values have in common is formed once: {what weight decay leaves, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), random key}.
struct Begin {
  float* steps;
  float4* factors;
  const float* lr_dev;        // or null: lr
  double lr, wd, log_b1, log_b2;
  unsigned seed;
  int count;
  const int *linear, *norm;   // status words of the kernels that form gradients with bounded waits
};
template <int MAX> struct Indices {
  Begin b;
  int index[MAX];
};
template <int MAX> __global__ void __launch_bounds__(MAX) k_adamw_begin(const __grid_constant__ Indices<MAX> a) {
  next_may_start();                                                      // k_adamw
  if ((int)threadIdx.x >= a.b.count) return;
  const int i = a.index[threadIdx.x];
  const int lost = *static_cast<const volatile int*>(a.b.linear) | *static_cast<const volatile int*>(a.b.norm);
  const float step = a.b.steps[i] + 1.f;
  const double lr = a.b.lr_dev != nullptr ? (double)*a.b.lr_dev : a.b.lr;
  float4 f = make_float4((float)(1.0 - lr * a.b.wd), (float)(lr / -expm1((double)step * a.b.log_b1)), (float)(1.0 / sqrt(-expm1((double)step * a.b.log_b2))),
                         __uint_as_float(mix(a.b.seed + mix((unsigned)step * 0x9E3779B1u + (unsigned)i))));
  if (lost != 0) f.z = -1.f;                                             // a wait gave up and has not been reported: the gradients may be what it left
  else a.b.steps[i] = step;
  a.b.factors[threadIdx.x] = f;
}

template <class P, int BITS, bool FLUSH, int MAX>
int launch(const Step& s, const Begin& b, const spion_adamw_tensor* ts, int count, cudaStream_t st) {
  Table<MAX> a;
  Indices<MAX> ix;
  a.s = s;
  a.s.count = 0;
  ix.b = b;
  ix.b.count = 0;
  long long chunks = 0;
  const long long most = (long long)sm_count() * CTAS;
  for (int full = 1; full >= 0; --full)                                  // tensors without values last: they have a count only
    for (int i = 0; i < count; ++i) {
      if ((ts[i].n > 0) != (full == 1)) continue;
      ix.index[ix.b.count++] = ts[i].index;
      if (full == 0) continue;
      a.chunk[a.s.count] = (int)chunks;
      a.t[a.s.count++] = Tensor{ts[i].p, ts[i].g, ts[i].copy, ts[i].n, ts[i].at};
      chunks += (ts[i].n + CHUNK - 1) / CHUNK;
      if (chunks > 0x7fffffff) return SPION_ERR_SHAPE;
    }
  a.s.chunks = (int)chunks;
  k_adamw_begin<MAX><<<1, MAX, 0, st>>>(ix);
  SPION_LAUNCH_CHECK();
  const dim3 grid((unsigned)(chunks < most ? chunks : most));
  if (chunks > 0) SPION_CUDA_TRY(launch_after(k_adamw<P, BITS, FLUSH, MAX>, grid, dim3(CTA), 0, st, a));
  return SPION_OK;
}
template <class P, int BITS>
int launches(const Step& s, const Begin& b, const spion_adamw_tensor* ts, int count, cudaStream_t st) {
  for (int i = 0; i < count; i += MOST) {
    const int n = count - i < MOST ? count - i : MOST;
    const bool flush = s.eps * sqrtf(s.c2) >= 0x1p-39f;
    const int rc = n > FEW ? flush ? launch<P, BITS, true, MOST>(s, b, ts + i, n, st) : launch<P, BITS, false, MOST>(s, b, ts + i, n, st)
                           : flush ? launch<P, BITS, true, FEW>(s, b, ts + i, n, st) : launch<P, BITS, false, FEW>(s, b, ts + i, n, st);
    if (rc != SPION_OK) return rc;
  }
  return SPION_OK;
}

}  // namespace

extern "C" int spion_adamw_step(const spion_adamw_tensor* host_tensors, int count, int type, int state_bits, void* m, void* v, float* m_scale,
                                float* v_scale, float* steps, const float* lr_dev, double lr, double beta1, double beta2, double eps,
                                double weight_decay, double clip_value, unsigned seed, int copy_type, void* workspace, void* cuda_stream) {
  if (count < 0 || (state_bits != 8 && state_bits != 32)) return SPION_ERR_ARG;
  if (count == 0) return SPION_OK;
  if (host_tensors == nullptr || m == nullptr || v == nullptr || steps == nullptr || workspace == nullptr || (state_bits == 8) != (m_scale != nullptr && v_scale != nullptr))
    return SPION_ERR_ARG;
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && weight_decay >= 0) || (lr_dev == nullptr && !(lr >= 0))) return SPION_ERR_ARG;
  if (((uintptr_t)m | (uintptr_t)v) & 31 || (uintptr_t)workspace & 15) return SPION_ERR_ARG;
  for (int i = 0; i < count; ++i) {
    const spion_adamw_tensor& t = host_tensors[i];
    if (t.n < 0 || t.at < 0 || t.at % BLOCK || t.index < 0 || (t.n > 0 && (t.p == nullptr || t.g == nullptr))) return SPION_ERR_ARG;
    if (t.copy != nullptr && copy_type != SPION_BF16 && copy_type != SPION_F16) return SPION_ERR_ARG;
  }
  if (type != SPION_F32 && type != SPION_BF16 && type != SPION_F16) return SPION_ERR_UNSUPPORTED;
  const int *const linear = linear_status_word(), *const norm = rmsnorm_status_word();
  if (linear == nullptr || norm == nullptr) return SPION_ERR_CUDA;
  const Step s = {m, v, m_scale, v_scale, static_cast<const float4*>(workspace), (float)beta1, (float)beta2, (float)(1.0 - beta1), (float)(1.0 - beta2),
                  (float)eps, clip_value >= 0 ? (float)clip_value : -1.f, 0, 0, copy_type};
  const Begin b = {steps, static_cast<float4*>(workspace), lr_dev, lr, weight_decay, log(beta1), log(beta2), seed, 0, linear, norm};
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  if (type == SPION_F32) return state_bits == 8 ? launches<float, 8>(s, b, host_tensors, count, st) : launches<float, 32>(s, b, host_tensors, count, st);
  if (type == SPION_BF16)
    return state_bits == 8 ? launches<__nv_bfloat16, 8>(s, b, host_tensors, count, st) : launches<__nv_bfloat16, 32>(s, b, host_tensors, count, st);
  return state_bits == 8 ? launches<__half, 8>(s, b, host_tensors, count, st) : launches<__half, 32>(s, b, host_tensors, count, st);
}
