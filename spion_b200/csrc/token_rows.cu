// Rows of a token table of any size, and the table's gradient:
//
//   y[t, :] = w[ids[t], :] scale                    dw[v, :] = scale sum_{t: ids[t] = v} g[t, :], in the order of t
//
//   k_lookup                 copies and scales
//   k_digits, k_place        ids with their tokens, sorted by id: a stable radix sort, 9 bits a pass at most
//   k_runs                   whole pieces of PIECE tokens of one id, summed (a padding token's run is thousands long)
//   k_rows                   every row of the table: its tokens' gradients, or the sums of its whole pieces and the tokens beside them
//
// Bound by memory: g is read once, dw written once; ids, orders and partial sums are 1/16 of g or less from 64 features on.  Every sum is a function of
// the tokens' order alone: no atomics on floating-point numbers, the same bits on every run.
#include <algorithm>

#include "rows.cuh"

using namespace rows;

namespace {

constexpr int THREADS = 256, WARPS = 8;
constexpr int PIECE = 64;
constexpr int MAX_BITS = 9, MAX_BINS = 1 << MAX_BITS;

// ------------------------------------------------------------------------------------------------ lookup
// `lanes` threads to a row's chunk of lanes * 8 features: eight side by side each, or one of eight stretches (VEC = 1)
template <int VEC> __device__ __forceinline__ int column(int chunk, int lane, int lanes, int e) {
  return VEC == 8 ? chunk * lanes * 8 + lane * 8 + e : chunk * lanes * 8 + e * lanes + lane;
}
template <class T, int VEC> __device__ __forceinline__ void load8(const T* row, int chunk, int lane, int lanes, long long N, float (&f)[8]) {
  if constexpr (VEC == 8) {
    const long long c = column<8>(chunk, lane, lanes, 0);
    Piece<T, 8> p;
    if (c < N) p.load(row + c);
    else p.zero();
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = p.at(e);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const long long c = column<1>(chunk, lane, lanes, e);
      f[e] = c < N ? as_float(row[c]) : 0.f;
    }
  }
}
template <class T, int VEC> __device__ __forceinline__ void store8(T* row, int chunk, int lane, int lanes, long long N, const float (&f)[8]) {
  if constexpr (VEC == 8) {
    const long long c = column<8>(chunk, lane, lanes, 0);
    if (c < N) Out<T, 8>::store(row + c, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const long long c = column<1>(chunk, lane, lanes, e);
      if (c < N) row[c] = rounded<T>(f[e]);
    }
  }
}

struct Lookup {
  const long long* ids;
  const void* w; long long ldw;
  void* y;
  float scale;
  long long T, V, N;
  int lanes;
};
constexpr int LOOKUP_ROWS = 4;
template <class TW, class TY, int VEC> __global__ void __launch_bounds__(THREADS) k_lookup(const __grid_constant__ Lookup a) {
  next_may_start();
  wait_for_kernel_before();
  const int groups = THREADS / a.lanes, group = threadIdx.x / a.lanes, lane = threadIdx.x - group * a.lanes, chunk = blockIdx.y;
  const long long first = ((long long)blockIdx.x * groups + group) * LOOKUP_ROWS;
  float f[LOOKUP_ROWS][8];
#pragma unroll
  for (int r = 0; r < LOOKUP_ROWS; ++r) {
    const long long t = first + r, id = t < a.T ? a.ids[t] : -1;
    if (id >= 0 && id < a.V) {
      load8<TW, VEC>(static_cast<const TW*>(a.w) + id * a.ldw, chunk, lane, a.lanes, a.N, f[r]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[r][e] = __int_as_float(0x7fffffff);
    }
  }
#pragma unroll
  for (int r = 0; r < LOOKUP_ROWS; ++r) {
    if (first + r >= a.T) break;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[r][e] *= a.scale;
    store8<TY, VEC>(static_cast<TY*>(a.y) + (first + r) * a.N, chunk, lane, a.lanes, a.N, f[r]);
  }
}

// ------------------------------------------------------------------------------------------------ sort
struct Sort {
  const long long* ids;                                    // the first pass: ids, tokens in order
  const uint32_t *key, *token;                             // the others
  uint32_t *key_out, *token_out;
  int* counts;                                             // [CTAs][bins]
  long long T, V, padding;
  int per_cta, per_warp, shift, bins;
};
__device__ __forceinline__ uint32_t key_at(const Sort& a, long long i) {
  if (a.ids == nullptr) return a.key[i];
  const long long id = a.ids[i];
  return id < 0 || id >= a.V || id == a.padding ? (uint32_t)a.V : (uint32_t)id;      // those without a gradient come last
}
__global__ void __launch_bounds__(THREADS) k_digits(const __grid_constant__ Sort a) {
  __shared__ int count[MAX_BINS];
  next_may_start();
  wait_for_kernel_before();
  for (int b = threadIdx.x; b < a.bins; b += THREADS) count[b] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * a.per_cta, end = min(a.T, first + a.per_cta);
  for (long long i = first + threadIdx.x; i < end; i += THREADS) atomicAdd(&count[(key_at(a, i) >> a.shift) & (a.bins - 1)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < a.bins; b += THREADS) a.counts[(long long)blockIdx.x * a.bins + b] = count[b];
}
// Where a CTA's first token of each digit goes is the sum of the counts before it (of the CTAs before it, of smaller digits); a warp takes a stretch of the CTA's
// tokens, 32 at a time, and lanes with the same digit stay in their order.
__global__ void __launch_bounds__(THREADS) k_place(const __grid_constant__ Sort a) {
  __shared__ int at[WARPS][MAX_BINS], digit_first[MAX_BINS], scan[WARPS];
  next_may_start();
  wait_for_kernel_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long cta_first = (long long)blockIdx.x * a.per_cta, cta_end = min(a.T, cta_first + a.per_cta);
  const long long first = min(cta_end, cta_first + (long long)warp * a.per_warp), end = min(cta_end, first + a.per_warp);
  for (int b = lane; b < a.bins; b += 32) at[warp][b] = 0;
  __syncwarp();
  for (long long i = first + lane; i < end; i += 32) atomicAdd(&at[warp][(key_at(a, i) >> a.shift) & (a.bins - 1)], 1);
  __syncthreads();
  // each thread two neighbouring digits
  int before[2] = {0, 0}, all[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = 2 * threadIdx.x + e;
    if (b >= a.bins) continue;
    if (gridDim.x == 1) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) all[e] += at[w][b];
    } else {
#pragma unroll 4
      for (int c = 0; c < (int)gridDim.x; ++c) {
        const int m = a.counts[(long long)c * a.bins + b];
        all[e] += m;
        before[e] += c < (int)blockIdx.x ? m : 0;
      }
    }
  }
  int sum = all[0] + all[1];                               // exclusive sums over the digits
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) scan[warp] = sum;
  __syncthreads();
  int base = sum - all[0] - all[1];
  for (int w = 0; w < warp; ++w) base += scan[w];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = 2 * threadIdx.x + e;
    if (b < a.bins) digit_first[b] = base + before[e];
    base += all[e];
  }
  __syncthreads();
  for (int b = threadIdx.x; b < a.bins; b += THREADS) {
    int next = digit_first[b];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int m = at[w][b];
      at[w][b] = next;
      next += m;
    }
  }
  __syncthreads();
  for (long long i0 = first; i0 < end; i0 += 32) {
    const long long i = i0 + lane;
    const bool in = i < end;
    const uint32_t key = in ? key_at(a, i) : 0, digit = (key >> a.shift) & (a.bins - 1);
    const uint32_t token = in ? (a.ids != nullptr ? (uint32_t)i : a.token[i]) : 0;
    const unsigned same = __match_any_sync(0xffffffffu, in ? digit : 0xffffffffu);
    const int rank = __popc(same & ((1u << lane) - 1));
    int to = 0;
    if (in) to = at[warp][digit] + rank;
    __syncwarp();
    if (in && rank == 0) at[warp][digit] += __popc(same);
    __syncwarp();
    if (in) a.key_out[to] = key, a.token_out[to] = token;
  }
}

// ------------------------------------------------------------------------------------------------ sums
struct Sums {
  const uint32_t *key, *token;                             // sorted
  const void* g; long long ldg;
  float* part;                                             // [pieces][N]
  void* dw;
  float scale;
  long long T, V, N;
  int lanes, rows;                                         // rows of the table a CTA
};
__device__ __forceinline__ void add8(float (&s)[8], const float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] += f[e];
}
// s += the rows of tokens i0 .. i1 - 1 of the sorted order: four loads under way, added one after another
template <class TG, int VEC> __device__ __forceinline__ void add_tokens(const Sums& a, long long i0, long long i1, int chunk, int lane, float (&s)[8]) {
  long long i = i0;
  for (; i + 4 <= i1; i += 4) {
    float f[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) load8<TG, VEC>(static_cast<const TG*>(a.g) + (long long)a.token[i + u] * a.ldg, chunk, lane, a.lanes, a.N, f[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) add8(s, f[u]);
  }
  for (; i < i1; ++i) {
    float f[8];
    load8<TG, VEC>(static_cast<const TG*>(a.g) + (long long)a.token[i] * a.ldg, chunk, lane, a.lanes, a.N, f);
    add8(s, f);
  }
}
template <int VEC> __device__ __forceinline__ void add_parts(const Sums& a, long long j0, long long j1, int chunk, int lane, float (&s)[8]) {
#pragma unroll 4
  for (long long j = j0; j < j1; ++j) {
    float f[8];
    load8<float, VEC>(a.part + j * a.N, chunk, lane, a.lanes, a.N, f);
    add8(s, f);
  }
}
// The groups' sums, added in their order by the first group
__device__ __forceinline__ void join_groups(float (*shared)[8], int groups, int group, int lane, int lanes, float (&s)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) shared[threadIdx.x][e] = s[e];
  __syncthreads();
  if (group == 0)
    for (int k = 1; k < groups; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += shared[k * lanes + lane][e];
  __syncthreads();
}
template <class TG, int VEC> __global__ void __launch_bounds__(THREADS) k_runs(const __grid_constant__ Sums a) {
  __shared__ float shared[THREADS][8];
  next_may_start();
  wait_for_kernel_before();
  const long long first = (long long)blockIdx.x * PIECE;
  const uint32_t key = a.key[first];
  if (key >= a.V || a.key[first + PIECE - 1] != key) return;
  const int groups = THREADS / a.lanes, group = threadIdx.x / a.lanes, lane = threadIdx.x - group * a.lanes, chunk = blockIdx.y;
  const int each = (PIECE + groups - 1) / groups, i0 = min(PIECE, group * each), i1 = min(PIECE, i0 + each);
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  add_tokens<TG, VEC>(a, first + i0, first + i1, chunk, lane, s);
  join_groups(shared, groups, group, lane, a.lanes, s);
  if (group == 0) store8<float, VEC>(a.part + (long long)blockIdx.x * a.N, chunk, lane, a.lanes, a.N, s);
}
// the first place in the order whose key is v or more
__device__ __forceinline__ long long lower_bound(const uint32_t* key, long long T, long long v) {
  long long lo = 0, hi = T;
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (key[mid] < v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}
constexpr int FEW = 32;                                    // tokens that one group adds
template <class TG, class TD, int VEC> __global__ void __launch_bounds__(THREADS) k_rows(const __grid_constant__ Sums a) {
  __shared__ float shared[THREADS][8];
  __shared__ long long start[THREADS + 1];
  next_may_start();
  wait_for_kernel_before();
  const long long v0 = (long long)blockIdx.x * a.rows;
  const int rows_here = (int)min((long long)a.rows, a.V - v0);
  for (int r = threadIdx.x; r <= rows_here; r += THREADS) start[r] = lower_bound(a.key, a.T, v0 + r);
  __syncthreads();
  const int groups = THREADS / a.lanes, group = threadIdx.x / a.lanes, lane = threadIdx.x - group * a.lanes, chunk = blockIdx.y;
  TD* const dw = static_cast<TD*>(a.dw);
  for (int r = group; r < rows_here; r += groups) {
    const long long i0 = start[r], i1 = start[r + 1];
    if (i1 - i0 > FEW) continue;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    add_tokens<TG, VEC>(a, i0, i1, chunk, lane, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] *= a.scale;
    store8<TD, VEC>(dw + (v0 + r) * a.N, chunk, lane, a.lanes, a.N, s);
  }
  for (int r = 0; r < rows_here; ++r) {                    // the others by all groups
    const long long i0 = start[r], i1 = start[r + 1];
    if (i1 - i0 <= FEW) continue;
    const long long p0 = (i0 + PIECE - 1) / PIECE, p1 = max(p0, i1 / PIECE);      // whole pieces
    const long long head = min(i1, p0 * PIECE) - i0, parts = p1 - p0, tail0 = min(i1, p1 * PIECE), all = head + parts + (i1 - tail0);
    const long long each = (all + groups - 1) / groups, m0 = min(all, group * each), m1 = min(all, m0 + each);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (m0 < head) add_tokens<TG, VEC>(a, i0 + m0, i0 + min(m1, head), chunk, lane, s);
    if (m1 > head && m0 < head + parts) add_parts<VEC>(a, p0 + max(m0 - head, 0ll), p0 + min(m1 - head, parts), chunk, lane, s);
    if (m1 > head + parts) add_tokens<TG, VEC>(a, tail0 + max(m0 - head - parts, 0ll), tail0 + (m1 - head - parts), chunk, lane, s);
    join_groups(shared, groups, group, lane, a.lanes, s);
    if (group == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] *= a.scale;
      store8<TD, VEC>(dw + (v0 + r) * a.N, chunk, lane, a.lanes, a.N, s);
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
bool float_type(int t) { return t == SPION_F32 || t == SPION_BF16 || t == SPION_F16; }
bool eights(const void* p, long long ld, long long N, int type) {
  const int piece = type == SPION_F32 ? 32 : 16;
  return N % 8 == 0 && (uintptr_t)p % piece == 0 && ld * type_size(type) % piece == 0;
}
// threads to a row's chunk: the fewest of 4 .. 32 whose eight features each are the row, else 32
int lanes_of(long long N) {
  for (int l = 4; l < 32; l *= 2)
    if (8 * l >= N) return l;
  return 32;
}
struct Sizes {
  long long per_cta, ctas, pieces;
  int passes, bits;
  size_t key[2], token[2], counts, part, all;
};
Sizes sizes_of(long long T, long long V, long long N) {
  Sizes s = {};
  // counts of all CTAs before it are read by every CTA: 128 of them at most
  s.per_cta = std::max(2048ll, ((T + 127) / 128 + 255) / 256 * 256);
  s.ctas = (T + s.per_cta - 1) / s.per_cta;
  int bits = 1;
  while (V >> bits) ++bits;                                // keys 0 .. V
  s.passes = (bits + MAX_BITS - 1) / MAX_BITS;
  s.bits = (bits + s.passes - 1) / s.passes;
  s.pieces = T / PIECE;
  size_t at = 0;
  auto take = [&](long long bytes) {
    const size_t here = at;
    at += (size_t)((bytes + 255) / 256 * 256);
    return here;
  };
  for (int i = 0; i < 2; ++i) s.key[i] = take(4 * T), s.token[i] = take(4 * T);
  s.counts = take(4 * s.ctas * (1ll << s.bits));
  s.part = take(4 * s.pieces * N);
  s.all = at;
  return s;
}
bool sizes_ok(long long T, long long V, long long N) { return T <= 0x7fffffff - 4096 && V <= 0x7fffffff - 4096 && N <= 0x7fffffff / 4; }

template <class TG, int VEC> int launch_sums(const Sums& a, const Sizes& s, int dw_type, cudaStream_t st) {
  const unsigned chunks = (unsigned)((a.N + a.lanes * 8 - 1) / (a.lanes * 8));
  if (s.pieces > 0) SPION_CUDA_TRY(launch_after(k_runs<TG, VEC>, dim3((unsigned)s.pieces, chunks), dim3(THREADS), 0, st, a));
  const dim3 grid((unsigned)((a.V + a.rows - 1) / a.rows), chunks);
  if (dw_type == SPION_F32) SPION_CUDA_TRY(launch_after(k_rows<TG, float, VEC>, grid, dim3(THREADS), 0, st, a));
  else if (dw_type == SPION_BF16) SPION_CUDA_TRY(launch_after(k_rows<TG, __nv_bfloat16, VEC>, grid, dim3(THREADS), 0, st, a));
  else SPION_CUDA_TRY(launch_after(k_rows<TG, __half, VEC>, grid, dim3(THREADS), 0, st, a));
  return SPION_OK;
}
template <class TW, class TY> int launch_lookup(const Lookup& a, bool eight, cudaStream_t st) {
  const int rows_ = THREADS / a.lanes * LOOKUP_ROWS;
  const dim3 grid((unsigned)((a.T + rows_ - 1) / rows_), (unsigned)((a.N + a.lanes * 8 - 1) / (a.lanes * 8)));
  if (eight) SPION_CUDA_TRY(launch_after(k_lookup<TW, TY, 8>, grid, dim3(THREADS), 0, st, a));
  else SPION_CUDA_TRY(launch_after(k_lookup<TW, TY, 1>, grid, dim3(THREADS), 0, st, a));
  return SPION_OK;
}
template <class TW> int launch_lookup(const Lookup& a, int y_type, bool eight, cudaStream_t st) {
  if (y_type == SPION_F32) return launch_lookup<TW, float>(a, eight, st);
  if (y_type == SPION_BF16) return launch_lookup<TW, __nv_bfloat16>(a, eight, st);
  return launch_lookup<TW, __half>(a, eight, st);
}

}  // namespace

extern "C" int spion_token_rows_forward(const long long* ids, const void* w, long long ldw, int w_type, void* y, int y_type, float scale, long long T, long long V,
                                        long long N, void* cuda_stream) {
  if (T < 0 || V < 0 || N <= 0 || !float_type(w_type) || !float_type(y_type) || ldw < N) return SPION_ERR_ARG;
  if (T == 0) return SPION_OK;
  if (ids == nullptr || y == nullptr || (w == nullptr && V > 0)) return SPION_ERR_ARG;
  if (!sizes_ok(T, V, N) || (N + 255) / 256 > 65535) return SPION_ERR_SHAPE;
  const Lookup a = {ids, w, ldw, y, scale, T, V, N, lanes_of(N)};
  const bool eight = eights(w, ldw, N, w_type) && eights(y, N, N, y_type);
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  if (w_type == SPION_F32) return launch_lookup<float>(a, y_type, eight, st);
  if (w_type == SPION_BF16) return launch_lookup<__nv_bfloat16>(a, y_type, eight, st);
  return launch_lookup<__half>(a, y_type, eight, st);
}

extern "C" long long spion_token_rows_workspace_bytes(long long T, long long V, long long N) {
  if (T <= 0 || V <= 0 || N <= 0 || !sizes_ok(T, V, N)) return 0;
  return (long long)sizes_of(T, V, N).all;
}

extern "C" int spion_token_rows_backward(const long long* ids, const void* g, long long ldg, int g_type, void* dw, int dw_type, float scale, long long padding_idx,
                                         long long T, long long V, long long N, void* workspace, void* cuda_stream) {
  if (T < 0 || V < 0 || N <= 0 || !float_type(g_type) || !float_type(dw_type) || ldg < 0) return SPION_ERR_ARG;
  if (V == 0) return SPION_OK;
  if (dw == nullptr || (T > 0 && (ids == nullptr || g == nullptr || workspace == nullptr || (uintptr_t)workspace % 256 != 0))) return SPION_ERR_ARG;
  if (!sizes_ok(T, V, N) || (N + 255) / 256 > 65535) return SPION_ERR_SHAPE;
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  if (T == 0) {
    SPION_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)V * N * type_size(dw_type), st));
    return SPION_OK;
  }
  const Sizes s = sizes_of(T, V, N);
  char* const ws = static_cast<char*>(workspace);
  uint32_t* const key[2] = {(uint32_t*)(ws + s.key[0]), (uint32_t*)(ws + s.key[1])};
  uint32_t* const token[2] = {(uint32_t*)(ws + s.token[0]), (uint32_t*)(ws + s.token[1])};
  for (int pass = 0; pass < s.passes; ++pass) {
    const int in = (pass + 1) & 1, out = pass & 1;
    const Sort a = {pass == 0 ? ids : nullptr, key[in], token[in], key[out], token[out], (int*)(ws + s.counts), T, V, padding_idx, (int)s.per_cta,
                    (int)s.per_cta / WARPS, pass * s.bits, 1 << s.bits};
    if (s.ctas > 1) SPION_CUDA_TRY(launch_after(k_digits, dim3((unsigned)s.ctas), dim3(THREADS), 0, st, a));
    SPION_CUDA_TRY(launch_after(k_place, dim3((unsigned)s.ctas), dim3(THREADS), 0, st, a));
  }
  const int last = (s.passes - 1) & 1, lanes = lanes_of(N);
  const Sums a = {key[last], token[last], g, ldg, (float*)(ws + s.part), dw, scale, T, V, N, lanes, THREADS / lanes * 4};
  const bool eight = eights(g, ldg, N, g_type) && eights(dw, N, N, dw_type);
  if (g_type == SPION_F32) return eight ? launch_sums<float, 8>(a, s, dw_type, st) : launch_sums<float, 1>(a, s, dw_type, st);
  if (g_type == SPION_BF16) return eight ? launch_sums<__nv_bfloat16, 8>(a, s, dw_type, st) : launch_sums<__nv_bfloat16, 1>(a, s, dw_type, st);
  return eight ? launch_sums<__half, 8>(a, s, dw_type, st) : launch_sums<__half, 1>(a, s, dw_type, st);
}
