// Rows of any width and type for the kernels that treat a row at a time (rmsnorm.cu): pieces of VEC elements per thread, loaded as they lie in
// memory and converted where they are used, so that the loads of all pieces are in flight together.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace rows {

template <class T> __host__ __device__ constexpr int type_code();
template <> __host__ __device__ constexpr int type_code<float>() { return SPION_F32; }
template <> __host__ __device__ constexpr int type_code<__nv_bfloat16>() { return SPION_BF16; }
template <> __host__ __device__ constexpr int type_code<__half>() { return SPION_F16; }
template <> __host__ __device__ constexpr int type_code<__nv_fp8_e4m3>() { return SPION_E4M3; }

static inline int type_size(int type) { return type == SPION_F32 ? 4 : type == SPION_BF16 || type == SPION_F16 ? 2 : 1; }

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half rounded<__half>(float x) { return __float2half_rn(x); }
// nearest e4m3, ties to even; NaN stays NaN, what is beyond 448 becomes 448
template <> __device__ __forceinline__ __nv_fp8_e4m3 rounded<__nv_fp8_e4m3>(float x) {
  __nv_fp8_e4m3 q;
  q.__x = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  return q;
}

// element i of an array of a type that is known at run time only (weights: once per kernel)
__device__ __forceinline__ float load_any(const void* p, int type, long long i) {
  if (type == SPION_F32) return static_cast<const float*>(p)[i];
  if (type == SPION_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int type, long long i, float x) {
  if (type == SPION_F32) static_cast<float*>(p)[i] = x;
  else if (type == SPION_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

// ---- VEC = 8: 32 bytes of fp32, 16 of a 16-bit type, 8 of e4m3, each on a boundary of its size.  VEC = 1: an element.
template <class T, int VEC> struct Piece;
template <class T> struct Piece<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void zero() { v = rounded<T>(0.f); }
  __device__ __forceinline__ float at(int) const { return as_float(v); }
};
template <> struct Piece<float, 8> {
  uint32_t w[8];
  __device__ __forceinline__ void load(const float* p) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
  }
  __device__ __forceinline__ void load_shared(const float* p) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i]); }
};
template <class T> struct Piece16 {
  uint4 q;
  __device__ __forceinline__ void load(const T* p) { q = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void load_shared(const T* p) { load(p); }
  __device__ __forceinline__ void zero() { q = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint32_t word(int i) const { return i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w; }
};
template <> struct Piece<__nv_bfloat16, 8> : Piece16<__nv_bfloat16> {
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? word(i) & 0xffff0000u : word(i) << 16); }
};
template <> struct Piece<__half, 8> : Piece16<__half> {
  __device__ __forceinline__ float at(int i) const { return __half2float(__ushort_as_half((unsigned short)(i & 1 ? word(i) >> 16 : word(i) & 0xffffu))); }
};

template <class T, int VEC> struct Out {
  __device__ static __forceinline__ void store(T* p, const float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = rounded<T>(v[i]);
  }
};
template <> struct Out<float, 8> {
  __device__ static __forceinline__ void store(float* p, const float (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])),
                 "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
                 "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])) : "memory");
  }
};
template <> struct Out<__nv_bfloat16, 8> {
  __device__ static __forceinline__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Out<__half, 8> {
  __device__ static __forceinline__ void store(__half* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Out<__nv_fp8_e4m3, 8> {
  __device__ static __forceinline__ void store(__nv_fp8_e4m3* p, const float (&v)[8]) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | hi << 16;
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
};

// ---- sums and maxima over the TPR threads of a row: lanes (a power of two up to 32), or all warps of the CTA, whose partial results go through shared
// memory.  `buf` alternates between two halves of `part`, so one barrier a row is enough.
template <int LANES> __device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LANES> __device__ __forceinline__ float lane_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// the largest, NaN if one is
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
template <int LANES> __device__ __forceinline__ float lane_max_nan(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int TPR, bool MAX> __device__ __forceinline__ void row_reduce(float& sum, float& top, float2 (*part)[32], int& buf) {
  constexpr int LANES = TPR < 32 ? TPR : 32, WARPS = TPR / 32;
  sum = lane_sum<LANES>(sum);
  if (MAX) top = lane_max_nan<LANES>(top);
  if (TPR <= 32) return;
  if ((threadIdx.x & 31) == 0) part[buf][threadIdx.x >> 5] = make_float2(sum, top);
  __syncthreads();
  const float2 t = (int)(threadIdx.x & 31) < WARPS ? part[buf][threadIdx.x & 31] : make_float2(0.f, 0.f);
  constexpr int UP = WARPS <= 2 ? 2 : WARPS <= 4 ? 4 : WARPS <= 8 ? 8 : WARPS <= 16 ? 16 : 32;
  sum = __shfl_sync(0xffffffffu, lane_sum<UP>(t.x), 0);
  if (MAX) top = __shfl_sync(0xffffffffu, lane_max_nan<UP>(t.y), 0);
  buf ^= 1;
}
template <int TPR> __device__ __forceinline__ void row_max_nan(float& top, float2 (*part)[32], int& buf) {
  top = lane_max_nan<(TPR < 32 ? TPR : 32)>(top);
  if (TPR <= 32) return;
  if ((threadIdx.x & 31) == 0) part[buf][threadIdx.x >> 5].y = top;
  __syncthreads();
  top = lane_max_nan<32>((int)(threadIdx.x & 31) < TPR / 32 ? part[buf][threadIdx.x & 31].y : 0.f);
  buf ^= 1;
}

}  // namespace rows
