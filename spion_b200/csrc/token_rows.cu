// Rows of a token table of any size, and the table's gradient:
//
//   y[t, :] = w[ids[t], :] scale                    dw[v, :] = scale sum_{t: ids[t] = v} g[t, :], in the order of t
//
//   k_lookup                 copies and scales
//   k_digits, k_place        ids with their tokens, sorted by id: a stable radix sort, 9 bits a pass at most (k_sort_one: all of it, for few ids)
//   k_sums                   windows of the sorted order, each summed run by run: runs that lie in a window go to dw, the two that may cross its ends to partial sums; zeros for
//                            rows of the table without a token
//   k_join                   the runs that cross windows
//
// Bound by memory: g is read once, dw written once.  Beside them the workspace has 16 bytes a token for two orders and two fp32 rows a window, N / 8 bytes a token in windows of 64 (N / 4, N / 2
// in windows of 32, 16): in windows of 64 an eighth of g for 128 features of 16 bits, a tenth for 64 of fp32, a fifth for 64 of 16 bits.  Sorting moves 30 bytes a token a pass, which the L2 cache keeps.  Windows and not rows of the table
// are what is shared out: tokens are as unequally frequent as words are, and what a window has to load is known before the ids of its runs are looked at (131072 ids of 32000,
// 1024 bf16 features: by rows, each finding its tokens by a search, 105 us; by windows 71, 4.3 TB/s, and 10 to join, 17 with cold caches; the lookup 52, 5.2 TB/s with what the caches keep).  Every sum is a function of the tokens' order alone: no atomics on floating-point
// numbers, the same bits on every run.
#include <algorithm>
#include <type_traits>

#include "rows.cuh"

using namespace rows;

namespace {

constexpr int THREADS = 256;
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

// Sixteen features a thread where table and result have the same 16-bit type and rows on 32 bytes: whole sectors
template <class T> __global__ void __launch_bounds__(THREADS) k_lookup_wide(const __grid_constant__ Lookup a) {
  next_may_start();
  wait_for_kernel_before();
  const int groups = THREADS / a.lanes, group = threadIdx.x / a.lanes, lane = threadIdx.x - group * a.lanes;
  const long long first = ((long long)blockIdx.x * groups + group) * LOOKUP_ROWS, c = ((long long)blockIdx.y * a.lanes + lane) * 16;
  if (c >= a.N) return;
  Piece<float, 8> p[LOOKUP_ROWS];                          // (32 bytes)
#pragma unroll
  for (int r = 0; r < LOOKUP_ROWS; ++r) {
    const long long t = first + r, id = t < a.T ? a.ids[t] : -1;
    if (id >= 0 && id < a.V) {
      p[r].load(reinterpret_cast<const float*>(static_cast<const T*>(a.w) + id * a.ldw + c));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[r].w[e] = 0x7fff7fffu;
    }
  }
#pragma unroll
  for (int r = 0; r < LOOKUP_ROWS; ++r) {
    if (first + r >= a.T) break;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      T v[2];
      *reinterpret_cast<uint32_t*>(v) = p[r].w[e];
      v[0] = rounded<T>(as_float(v[0]) * a.scale), v[1] = rounded<T>(as_float(v[1]) * a.scale);
      f[e] = __uint_as_float(*reinterpret_cast<const uint32_t*>(v));
    }
    Out<float, 8>::store(reinterpret_cast<float*>(static_cast<T*>(a.y) + (first + r) * a.N + c), f);
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
// Exclusive sums over the digits of `count`, one to a thread (`bins` at most as many as threads), on top of `base`
template <int N> __device__ __forceinline__ int scan_digits(int count, int (&shared)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < N; ++w) before += w < warp ? shared[w] : 0;
  return before + sum - count;
}
// 32 keys of a warp, in order: where each goes; `at`: the warp's next place of each digit
__device__ __forceinline__ int place_of(int* at, uint32_t digit, bool in) {
  const unsigned same = __match_any_sync(0xffffffffu, in ? digit : 0xffffffffu);
  const int rank = __popc(same & ((1u << (threadIdx.x & 31)) - 1));
  int to = 0;
  if (in) to = at[digit] + rank;
  __syncwarp();
  if (in && rank == 0) at[digit] += __popc(same);
  __syncwarp();
  return to;
}
// Where a CTA's first token of each digit goes is the sum of the counts before it (of the CTAs before it, of smaller digits); a warp takes a stretch of the CTA's
// tokens, 32 at a time, and lanes with the same digit stay in their order.  Threads take four digits and a share of the CTAs each, sixteen loads under way: one digit and all CTAs
// after another were 20 of 22 us for 64 CTAs.
constexpr int PLACE = 512;
__global__ void __launch_bounds__(PLACE) k_place(const __grid_constant__ Sort a) {
  constexpr int W = PLACE / 32;
  __shared__ int at[W][MAX_BINS], shared[32];
  __shared__ __align__(16) int total[MAX_BINS], first_of[MAX_BINS];
  next_may_start();
  wait_for_kernel_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long cta_first = (long long)blockIdx.x * a.per_cta, cta_end = min(a.T, cta_first + a.per_cta);
  const long long first = min(cta_end, cta_first + (long long)warp * a.per_warp), end = min(cta_end, first + a.per_warp);
  for (int b = lane; b < a.bins; b += 32) at[warp][b] = 0;
  for (int b = threadIdx.x; b < a.bins; b += PLACE) total[b] = first_of[b] = 0;
  __syncthreads();
  for (long long i0 = first; i0 < end; i0 += 128) {
    uint32_t key[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) key[u] = i0 + 32 * u + lane < end ? key_at(a, i0 + 32 * u + lane) : 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + 32 * u + lane < end) atomicAdd(&at[warp][(key[u] >> a.shift) & (a.bins - 1)], 1);
  }
  const int fours = max(1, a.bins / 4), part = threadIdx.x / fours, parts = PLACE / fours, ctas = gridDim.x, each = (ctas + parts - 1) / parts;
  if (part < parts && a.bins >= 4) {
    int all[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0};
    const int4* const counts = reinterpret_cast<const int4*>(a.counts) + (threadIdx.x - part * fours);
#pragma unroll 16
    for (int c = part * each; c < min(ctas, (part + 1) * each); ++c) {
      const int4 m = counts[(long long)c * fours];
      const int in = c < (int)blockIdx.x ? -1 : 0;
      all[0] += m.x, all[1] += m.y, all[2] += m.z, all[3] += m.w;
      before[0] += m.x & in, before[1] += m.y & in, before[2] += m.z & in, before[3] += m.w & in;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int b = 4 * (threadIdx.x - part * fours) + e;
      if (all[e]) atomicAdd(&total[b], all[e]);
      if (before[e]) atomicAdd(&first_of[b], before[e]);
    }
  } else if (a.bins < 4 && threadIdx.x < a.bins) {
    for (int c = 0; c < ctas; ++c) {
      const int m = a.counts[(long long)c * a.bins + threadIdx.x];
      total[threadIdx.x] += m;
      first_of[threadIdx.x] += c < (int)blockIdx.x ? m : 0;
    }
  }
  __syncthreads();
  const int b = threadIdx.x, base = scan_digits<W>(b < a.bins ? total[b] : 0, shared);
  if (b < a.bins) {
    int next = base + first_of[b];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int m = at[w][b];
      at[w][b] = next;
      next += m;
    }
  }
  __syncthreads();
  for (long long i0 = first; i0 < end; i0 += 128) {
    uint32_t key[4], token[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long i = i0 + 32 * u + lane;
      key[u] = i < end ? key_at(a, i) : 0;
      token[u] = i < end ? (a.ids != nullptr ? (uint32_t)i : a.token[i]) : 0;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i0 + 32 * u >= end) break;
      const bool in = i0 + 32 * u + lane < end;
      const int to = place_of(at[warp], (key[u] >> a.shift) & (a.bins - 1), in);
      if (in) a.key_out[to] = key[u], a.token_out[to] = token[u];
    }
  }
}
// All passes by one CTA, keys and tokens in shared memory: one launch instead of four for few ids (4099 of 10007, each kernel alone: 14 us, 25)
constexpr int ONE = 1024, ONE_MAX = 8192;
constexpr uint32_t ONE_SMEM = 4 * ONE_MAX * 4 + 32 * MAX_BINS * 4;
__global__ void __launch_bounds__(ONE) k_sort_one(const __grid_constant__ Sort a, int bits, int passes) {
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ int shared[32];
  int* const at0 = reinterpret_cast<int*>(smem + 4 * ONE_MAX);
  next_may_start();
  wait_for_kernel_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, T = (int)a.T, bins = 1 << bits;
  const int first = min(T, warp * a.per_warp), end = min(T, first + a.per_warp);
  int* const at = at0 + warp * MAX_BINS;
  uint32_t key[8], token[8];
  for (int pass = 0; pass < passes; ++pass) {
    const uint32_t *const kin = smem + (pass & 1) * ONE_MAX, *const tin = kin + 2 * ONE_MAX;
    uint32_t *const kout = smem + ((pass + 1) & 1) * ONE_MAX, *const tout = kout + 2 * ONE_MAX;
    for (int b = lane; b < bins; b += 32) at[b] = 0;
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = first + 32 * u + lane;
      if (i >= end) continue;
      key[u] = pass == 0 ? key_at(a, i) : kin[i];
      token[u] = pass == 0 ? (uint32_t)i : tin[i];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (first + 32 * u + lane < end) atomicAdd(&at[(key[u] >> (pass * bits)) & (bins - 1)], 1);
    __syncthreads();
    const int b = threadIdx.x;
    int count = 0;
    if (b < bins)
      for (int w = 0; w < 32; ++w) count += at0[w * MAX_BINS + b];
    int next = scan_digits<32>(count, shared);
    if (b < bins)
      for (int w = 0; w < 32; ++w) {
        const int m = at0[w * MAX_BINS + b];
        at0[w * MAX_BINS + b] = next;
        next += m;
      }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (first + 32 * u >= end) break;
      const bool in = first + 32 * u + lane < end;
      const int to = place_of(at, (key[u] >> (pass * bits)) & (bins - 1), in);
      if (in) {
        if (pass == passes - 1) a.key_out[to] = key[u], a.token_out[to] = token[u];
        else kout[to] = key[u], tout[to] = token[u];
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ sums
struct Sums {
  const uint32_t *key, *token;                             // sorted
  const void* g; long long ldg;
  float* part;                                             // [windows][2][N]: of the run that a window begins in the middle of; of the one that it ends in the middle of
  void* dw;
  float scale;
  long long T, V, N;
  int lanes, window;                                       // threads to a chunk of a row; tokens of a window
  long long windows;
  unsigned sum_ctas, chunks;                               // CTAs of windows, before those of zeros; chunks of a row
};
template <class T, int VEC> struct Raw8 {                  // eight elements as they lie in memory
  Piece<T, 8> p;
  __device__ __forceinline__ void load(const T* row, int chunk, int lane, int lanes, long long N) {
    const long long c = column<8>(chunk, lane, lanes, 0);
    if (c < N) p.load(row + c);
    else p.zero();
  }
  __device__ __forceinline__ float at(int e) const { return p.at(e); }
};
template <class T> struct Raw8<T, 1> {
  T v[8];
  __device__ __forceinline__ void load(const T* row, int chunk, int lane, int lanes, long long N) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const long long c = column<1>(chunk, lane, lanes, e);
      v[e] = c < N ? row[c] : rounded<T>(0.f);
    }
  }
  __device__ __forceinline__ float at(int e) const { return as_float(v[e]); }
};
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
constexpr int ZERO_ROWS = 64;                              // rows of the table that a CTA looks for tokens of
// Rows of g under way: more of them cost more registers than they hide (131072 x 1024 bf16: four of sixteen features a thread 71 us, eight of eight 88, sixteen of eight, with 154
// registers, 144).
constexpr int DEEP = 4;
// P: pieces of eight features a thread
template <class TG, class TD, int VEC, int P> __global__ void __launch_bounds__(THREADS) k_sums(const __grid_constant__ Sums a) {
  next_may_start();
  wait_for_kernel_before();
  const int groups = THREADS / a.lanes, group = threadIdx.x / a.lanes, lane = threadIdx.x - group * a.lanes;
  TD* const dw = static_cast<TD*>(a.dw);
  // windows first, the chunks of their rows side by side
  const unsigned sums = a.sum_ctas * a.chunks, at = blockIdx.x - (blockIdx.x >= sums ? sums : 0), cta = at / a.chunks;
  const int chunk = (int)(at - cta * a.chunks) * P;
  if (blockIdx.x >= sums) {                                // rows without a token
    __shared__ int start[ZERO_ROWS + 1];
    const long long v0 = (long long)cta * ZERO_ROWS;
    const int rows_here = (int)min((long long)ZERO_ROWS, a.V - v0);
    if ((int)threadIdx.x <= rows_here) start[threadIdx.x] = (int)lower_bound(a.key, a.T, v0 + threadIdx.x);
    __syncthreads();
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int r = group; r < rows_here; r += groups)
      if (start[r] == start[r + 1])
#pragma unroll
        for (int p = 0; p < P; ++p) store8<TD, VEC>(dw + (v0 + r) * a.N, chunk + p, lane, a.lanes, a.N, zero);
    return;
  }
  const long long w = (long long)cta * groups + group;
  if (w >= a.windows) return;
  const int i0 = (int)(w * a.window), i1 = (int)min(a.T, (long long)i0 + a.window);
  const uint32_t none = (uint32_t)a.V;
  uint32_t run = a.key[i0];
  if (run >= none) return;                                 // from here on all are without a gradient
  bool begun = i0 > 0 && a.key[i0 - 1] == run;             // the run began before this window
  const bool goes_on = i1 < a.T && a.key[i1] == a.key[i1 - 1];
  float s[P][8];
  auto clear = [&] {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[p][e] = 0.f;
  };
  auto put = [&](bool crosses) {
    if (run < none) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (begun || crosses) {
          store8<float, VEC>(a.part + (2 * w + !begun) * a.N, chunk + p, lane, a.lanes, a.N, s[p]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) s[p][e] *= a.scale;
          store8<TD, VEC>(dw + (long long)run * a.N, chunk + p, lane, a.lanes, a.N, s[p]);
        }
      }
    }
    begun = false;
  };
  clear();
  // No load waits behind a branch: the last token again where a window ends, rows without a gradient too where one begins; ids and tokens a step ahead.
  uint32_t key[DEEP], token[DEEP];
#pragma unroll
  for (int u = 0; u < DEEP; ++u) key[u] = a.key[min(i0 + u, i1 - 1)], token[u] = a.token[min(i0 + u, i1 - 1)];
  for (int i = i0; i < i1; i += DEEP) {
    Raw8<TG, VEC> g[DEEP][P];
    uint32_t now[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const TG* const row = static_cast<const TG*>(a.g) + (long long)token[u] * a.ldg;
#pragma unroll
      for (int p = 0; p < P; ++p) g[u][p].load(row, chunk + p, lane, a.lanes, a.N);
      now[u] = key[u];
    }
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const int next = min(i + DEEP + u, i1 - 1);
      key[u] = a.key[next], token[u] = a.token[next];
    }
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      if (i + u >= i1) break;
      if (now[u] != run) {
        put(false);
        run = now[u];
        clear();
      }
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[p][e] += g[u][p].at(e);
    }
  }
  put(goes_on);
}
// A group looks at a window: where a run begins in it and goes on, it adds the run's partial sums, or, of many, all groups of the CTA do, a share each.
constexpr int FEW = 16;
template <class TD, int VEC> __global__ void __launch_bounds__(THREADS) k_join(const __grid_constant__ Sums a) {
  __shared__ float shared[THREADS][8];
  __shared__ long long many[THREADS];                      // per group: windows of a long run, or 0
  next_may_start();
  wait_for_kernel_before();
  const int groups = THREADS / a.lanes, group = threadIdx.x / a.lanes, lane = threadIdx.x - group * a.lanes, chunk = blockIdx.y;
  TD* const dw = static_cast<TD*>(a.dw);
  const long long w0 = (long long)blockIdx.x * groups, w = w0 + group;
  auto add = [&](long long from, long long to, float (&s)[8]) {      // the first sums of windows from .. to - 1
#pragma unroll 8
    for (long long j = from; j < to; ++j) {
      float f[8];
      load8<float, VEC>(a.part + 2 * j * a.N, chunk, lane, a.lanes, a.N, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += f[e];
    }
  };
  // windows after w0 + k that the run that begins in window w0 + k and goes on is part of; 0: there is none
  auto run_of = [&](long long w, uint32_t& run) -> long long {
    const long long i0 = w * a.window, i1 = i0 + a.window, far = (w + FEW + 1) * a.window;
    if (w >= a.windows || i1 >= a.T) return 0;
    run = a.key[i1 - 1];                                   // (all of the keys at once)
    const uint32_t next = a.key[i1], before = a.key[max(i0 - 1, 0ll)], far_key = a.key[min(far, a.T - 1)];
    if (run >= a.V || next != run || (i0 > 0 && before == run)) return 0;
    long long lo = 1, hi = a.windows - w;                  // windows of the run: those that begin with its id
    if (far >= a.T || far_key != run) hi = min(hi, (long long)FEW + 1);
    while (lo < hi) {
      const long long mid = (lo + hi) >> 1;
      if (a.key[(w + mid) * a.window] == run) lo = mid + 1;
      else hi = mid;
    }
    return lo - 1;
  };
  uint32_t run = 0;
  const long long more = run_of(w, run);
  if (lane == 0) many[group] = more > FEW ? more : 0;
  if (more > 0 && more <= FEW) {
    float s[8];
    load8<float, VEC>(a.part + (2 * w + 1) * a.N, chunk, lane, a.lanes, a.N, s);
    add(w + 1, w + 1 + more, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] *= a.scale;
    store8<TD, VEC>(dw + (long long)run * a.N, chunk, lane, a.lanes, a.N, s);
  }
  __syncthreads();
  for (int k = 0; k < groups; ++k) {
    const long long all = many[k];
    if (all == 0) continue;
    const long long each = (all + groups - 1) / groups, j0 = min(all, group * each), j1 = min(all, j0 + each);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (group == 0) load8<float, VEC>(a.part + (2 * (w0 + k) + 1) * a.N, chunk, lane, a.lanes, a.N, s);
    add(w0 + k + 1 + j0, w0 + k + 1 + j1, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) shared[threadIdx.x][e] = s[e];
    __syncthreads();
    if (group == 0) {
      for (int o = 1; o < groups; ++o)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += shared[o * a.lanes + lane][e];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] *= a.scale;
      store8<TD, VEC>(dw + (long long)a.key[(w0 + k + 1) * a.window] * a.N, chunk, lane, a.lanes, a.N, s);
    }
    __syncthreads();
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
  long long per_cta, ctas, window, windows;
  int passes, bits;
  bool one;                                                // the sort by one CTA
  size_t key[2], token[2], counts, part, all;
};
Sizes sizes_of(long long T, long long V, long long N) {
  Sizes s = {};
  s.one = T <= ONE_MAX;
  // counts of all CTAs before it are read by every CTA: 128 of them at most
  s.per_cta = s.one ? (T + 1023) / 1024 * 1024 : std::max(1024ll, ((T + 127) / 128 + PLACE - 1) / PLACE * PLACE);
  s.ctas = (T + s.per_cta - 1) / s.per_cta;
  int bits = 1;
  while (V >> bits) ++bits;                                // keys 0 .. V
  s.passes = (bits + MAX_BITS - 1) / MAX_BITS;
  s.bits = (bits + s.passes - 1) / s.passes;
  // Windows of 64 tokens where that leaves 16 warps to every multiprocessor (of 148, whatever the device has: sums and workspaces are a function of the sizes alone), down to 16 where
  // it does not.
  const long long chunks = (N + 255) / 256;
  s.window = 64;
  while (s.window > 16 && (T + s.window - 1) / s.window * chunks < 148 * 16) s.window /= 2;
  s.windows = (T + s.window - 1) / s.window;
  size_t at = 0;
  auto take = [&](long long bytes) {
    const size_t here = at;
    at += (size_t)((bytes + 255) / 256 * 256);
    return here;
  };
  for (int i = 0; i < 2; ++i) s.key[i] = take(4 * T), s.token[i] = take(4 * T);
  s.counts = take(4 * s.ctas * (1ll << s.bits));
  s.part = take(s.windows > 1 ? 8 * s.windows * N : 0);
  s.all = at;
  return s;
}
bool sizes_ok(long long T, long long V, long long N) { return T <= 0x7fffffff - 4096 && V <= 0x7fffffff - 4096 && N <= 0x7fffffff / 4; }

template <class TG, class TD, int VEC> int launch_sums(const Sums& a, cudaStream_t st) {
  constexpr int P = VEC == 8 ? 2 : 1;
  const bool two = P == 2 && a.N > 256;
  Sums b = a;
  if (two) b.chunks = (a.chunks + 1) / 2;
  const long long ctas = ((b.V + ZERO_ROWS - 1) / ZERO_ROWS + b.sum_ctas) * b.chunks;
  if (ctas > 0x7fffffff) return SPION_ERR_SHAPE;
  if (two) SPION_CUDA_TRY(launch_after(k_sums<TG, TD, VEC, P>, dim3((unsigned)ctas), dim3(THREADS), 0, st, b));
  else SPION_CUDA_TRY(launch_after(k_sums<TG, TD, VEC, 1>, dim3((unsigned)ctas), dim3(THREADS), 0, st, b));
  if (a.windows > 1) SPION_CUDA_TRY(launch_after(k_join<TD, VEC>, dim3(a.sum_ctas, a.chunks), dim3(THREADS), 0, st, a));
  return SPION_OK;
}
template <class TG, int VEC> int launch_sums(const Sums& a, int dw_type, cudaStream_t st) {
  if (dw_type == SPION_F32) return launch_sums<TG, float, VEC>(a, st);
  if (dw_type == SPION_BF16) return launch_sums<TG, __nv_bfloat16, VEC>(a, st);
  return launch_sums<TG, __half, VEC>(a, st);
}
template <class TW, class TY> int launch_lookup(const Lookup& a, bool eight, cudaStream_t st) {
  const int rows_ = THREADS / a.lanes * LOOKUP_ROWS;
  const dim3 grid((unsigned)((a.T + rows_ - 1) / rows_), (unsigned)((a.N + a.lanes * 8 - 1) / (a.lanes * 8)));
  if constexpr (std::is_same<TW, TY>::value && sizeof(TW) == 2) {
    if (eight && a.N % 16 == 0 && ((uintptr_t)a.w | (uintptr_t)a.y | (uintptr_t)(a.ldw * 2)) % 32 == 0) {
      Lookup b = a;
      while (b.lanes > 4 && 8 * b.lanes >= a.N) b.lanes /= 2;
      const int rows_16 = THREADS / b.lanes * LOOKUP_ROWS;
      const dim3 grid16((unsigned)((a.T + rows_16 - 1) / rows_16), (unsigned)((a.N + b.lanes * 16 - 1) / (b.lanes * 16)));
      SPION_CUDA_TRY(launch_after(k_lookup_wide<TW>, grid16, dim3(THREADS), 0, st, b));
      return SPION_OK;
    }
  }
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
  const int last = s.one ? 0 : (s.passes - 1) & 1, lanes = lanes_of(N);
  if (s.one) {
    static std::atomic<uint64_t> ready{0};                  // once per device
    int dev = 0;
    SPION_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
      SPION_CUDA_TRY(cudaFuncSetAttribute(k_sort_one, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ONE_SMEM));
      if (dev < 64) ready.fetch_or(1ull << dev);
    }
    const Sort a = {ids, nullptr, nullptr, key[0], token[0], nullptr, T, V, padding_idx, (int)s.per_cta, (int)s.per_cta / 32, 0, 0};
    SPION_CUDA_TRY(launch_after(k_sort_one, dim3(1), dim3(ONE), ONE_SMEM, st, a, s.bits, s.passes));
  } else {
    for (int pass = 0; pass < s.passes; ++pass) {
      const int in = (pass + 1) & 1, out = pass & 1;
      const Sort a = {pass == 0 ? ids : nullptr, key[in], token[in], key[out], token[out], (int*)(ws + s.counts), T, V, padding_idx, (int)s.per_cta,
                      (int)s.per_cta / (PLACE / 32), pass * s.bits, 1 << s.bits};
      SPION_CUDA_TRY(launch_after(k_digits, dim3((unsigned)s.ctas), dim3(THREADS), 0, st, a));
      SPION_CUDA_TRY(launch_after(k_place, dim3((unsigned)s.ctas), dim3(PLACE), 0, st, a));
    }
  }
  const int groups = THREADS / lanes;
  const Sums a = {key[last], token[last], g, ldg, (float*)(ws + s.part), dw, scale, T, V, N, lanes, (int)s.window, s.windows, (unsigned)((s.windows + groups - 1) / groups),
                  (unsigned)((N + lanes * 8 - 1) / (lanes * 8))};
  const bool eight = eights(g, ldg, N, g_type) && eights(dw, N, N, dw_type);
  if (g_type == SPION_F32) return eight ? launch_sums<float, 8>(a, dw_type, st) : launch_sums<float, 1>(a, dw_type, st);
  if (g_type == SPION_BF16) return eight ? launch_sums<__nv_bfloat16, 8>(a, dw_type, st) : launch_sums<__nv_bfloat16, 1>(a, dw_type, st);
  return eight ? launch_sums<__half, 8>(a, dw_type, st) : launch_sums<__half, 1>(a, dw_type, st);
}
