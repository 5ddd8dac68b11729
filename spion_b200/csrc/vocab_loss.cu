// Losses over a vocabulary from the rows before the last layer, without its logits:  z = x W^T + b (T rows of K, V rows of W),
//
//   loss_t = sum_j q_tj (ln q_tj - z_t[i_tj] / tau + lse_t),   lse_t = ln sum_v exp(z_tv / tau)
//
// with one target of weight 1 (cross entropy, tau = 1) or a teacher's k logits, q_t = softmax(logits_t / tau).  Gradients, with g_t what arrives at a row's loss:
//
//   G_tv = g_t / tau (softmax(z_t / tau)_v - sum_{j: i_tj = v} q_tj),   dx = G W,  dW = G^T x,  db = sum_t G_t
//
//   k_flags, k_prepare   which rows count, in order; those rows side by side in the products' type (rows that do not count cost nothing and are never read; where all
//                        count and lie as the products read them, they stay where they are)
//   k_gemm<LOGSUM>       z tile by tile in tensor memory; leaves the largest and the sum of exponentials of a row's columns of the tile, and the targets' z
//   k_finish             lse and loss of each row, and their sum or mean
//   k_gemm<GRAD>         z again, for a piece of the vocabulary; leaves G in 16 bits
//   k_gemm<GRADS>        the two products with it;  k_out joins what was summed apart, and forms db
//   k_few_*              in place of these three, and of the operands' copies, up to sixteen rows of fp32 on the ordinary units
//
// The products are tcgen05 kind::f16, fp32 sums in tensor memory.  A sum there is truncated at every step, by some 2^-23 of it and always towards zero, so few steps go to one
// accumulator where a result has 32 bits (chain_of); what the accumulators hold is added in fp32 registers.  fp32 operands are three bf16 parts each (8 + 8 + 8 bits, exact) and
// six products (few rows: as they are); what is dropped is below 2^-25 of a product.
//
// G is rounded to the type that W has, after it was formed in fp32: the products' other operand has those bits, and their results are rounded to them.  It shows in the results: dx and dW
// of many rows are as far from exact ones by G's rounding as by their own (8192 x 2048 to 32000 against 32 logits, bf16: 2.3e-3 of the norm, 1.7e-3 with G in fp32); two parts of G, which few rows and
// small calls have (see layout_of), would double both products.  In fp16, whose smallest numbers probabilities of a large vocabulary fall below, G holds 2^13 g_t over the largest |g_t|, rounded up to a power of two; the
// factor comes back in fp32.  A probability p of a row whose g is a part r of the largest keeps all its bits while p r >= 2^-26, and is 0 below 2^-38.
// The bias's gradient is summed from G before it is rounded.
#include <algorithm>
#include <type_traits>

#include "rows.cuh"
#include "tc_ptx.cuh"
#include "tc_tiles.cuh"

using namespace tc;
using namespace rows;

namespace {

// Set by a bounded wait that gave up (see g_lin_status in linear.cu); results after it are NaN until it has been reported.
__device__ int g_vocab_status;

constexpr float LN2 = 0.6931471805599453f;
constexpr int MAX_TARGETS = 128;
constexpr int PAD = 256;                                  // rows and vocabulary columns of scratch come in whole tiles

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float not_a_number() { return __int_as_float(0x7fffffff); }

// ------------------------------------------------------------------------------------------------ which rows count
// Kept from the forward for the backward, in the order of the rows that count ("slots"); numbers in units of log2
struct Plan {
  int* head;                // [0]: rows that count; [1]: CTAs of k_finish that are done
  int* slot;                // [T] a row's slot, or -1
  int* row;                 // [Tp] a slot's row
  float* lse;               // [Tp]
  float* less;              // [Tp] of a target of weight 1, if the row has one: its probability less 1.  From its own -ln p, the rounding of whose sum and logarithm
                            // does not grow with the logits: p - 1, with p from a log of the sum as large as they are, would keep that one's rounding alone where the row is sure of it
  int* target;              // [k][Tp]; -1: left out; -2: outside of the vocabulary
  float* q;                 // [k][Tp] (null: one target of weight 1)
};
struct Source {
  const void* p; int type; long long ld;
  int K, Kp, fast;          // 2: rows on 16-byte boundaries, whole pieces of 8; 1: rows of pairs, on boundaries of one; 0: any
};
struct Prep {
  Plan plan;
  const long long* labels;  // [T], or [T, k] where there are teacher logits
  const void* teacher; int teacher_type;                 // [T, k] or null
  long long ignore;
  float inv_tau;
  int T, Tp, V, k;
  int* counts;              // [chunks], or null: each CTA counts for itself
  float* q;                 // [T, k]
  const void* bias; int bias_type;
  float* bias2;             // [Vp + PAD] b log2(e) / tau; -inf behind the vocabulary
  int Vp;
  float c1;                 // log2(e) / tau
  // rows and weights in the products' type
  Source x, w;
  uint16_t *xs, *ws;        // ws: or null, w is read as it lies
  int direct;               // x can be read as it lies, if all rows count
  int few;                  // x and w are read as they lie, whatever counts
  float* loss_rows;         // [T] or null: zeros where a row does not count
  float* zt;                // [k][Tp]
  int chunk;                // rows of a CTA, a multiple of 32; of BLOCK where there are more
  unsigned row_ctas, slices, w_ctas;                     // CTAs of rows: x column slices; then those of w, then those of the bias
};
constexpr int BLOCK = 128, SELF = 4096;                   // rows that a CTA lists at a time; labels (or logits) up to which each CTA counts for itself

// A warp: weights of the targets of eight rows (from t0 on, below `end`).  Bits of those that have one.
template <int WORDS> __device__ __forceinline__ unsigned teacher_weights(const Prep& a, int t0, int end, int lane) {
  float v[8][WORDS];
#pragma unroll
  for (int r = 0; r < 8; ++r)
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const int j = lane + 32 * i;
      const long long at = (long long)(t0 + r) * a.k + j;
      const bool in = t0 + r < end && j < a.k;
      v[r][i] = in && a.labels[at] != -1 ? load_any(a.teacher, a.teacher_type, at) : -INFINITY;
    }
  unsigned found = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) nan |= v[r][i] != v[r][i], top = fmaxf(top, v[r][i]);
    top = lane_max<32>(top);
    if (!(__any_sync(0xffffffffu, nan) || top != -INFINITY)) continue;
    found |= 1u << r;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      v[r][i] = v[r][i] == -INFINITY ? 0.f : expf((v[r][i] - top) * a.inv_tau);
      sum += v[r][i];
    }
    sum = lane_sum<32>(sum);
#pragma unroll
    for (int i = 0; i < WORDS; ++i)
      if (lane + 32 * i < a.k) a.q[(long long)(t0 + r) * a.k + lane + 32 * i] = v[r][i] / sum;
  }
  return found;
}
__device__ __forceinline__ unsigned teacher_weights(const Prep& a, int t0, int end, int lane) {
  return a.k <= 32 ? teacher_weights<1>(a, t0, end, lane) : teacher_weights<MAX_TARGETS / 32>(a, t0, end, lane);
}
__device__ __forceinline__ bool is_entry(const Prep& a, long long at) { return a.labels[at] != -1 && load_any(a.teacher, a.teacher_type, at) != -INFINITY; }
__device__ __forceinline__ void scaled_bias(const Prep& a, int first, int step) {
  for (int v = first; v < a.Vp + PAD; v += step) a.bias2[v] = v >= a.V ? -INFINITY : a.bias != nullptr ? load_any(a.bias, a.bias_type, v) * a.c1 : 0.f;
}
// Rows that count, of each chunk: a warp per chunk, or, with a teacher, a CTA per chunk and eight rows a warp (a warp for all of them, one row after another: 8192 rows of 32
// logits 98 us)
__global__ void __launch_bounds__(256) k_flags(const __grid_constant__ Prep a) {
  __shared__ int part[8];
  next_may_start();
  wait_for_kernel_before();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = (a.T + a.chunk - 1) / a.chunk;
  if (a.teacher == nullptr) {
    const int c = blockIdx.x * 8 + warp;
    if (c >= chunks) return;
    int n = 0;
#pragma unroll 4
    for (int i = 0; i < a.chunk; i += 32) {
      const long long t = (long long)c * a.chunk + i + lane;
      n += __popc(__ballot_sync(0xffffffffu, t < a.T && a.labels[t] != a.ignore));
    }
    if (lane == 0) a.counts[c] = n;
    return;
  }
  int mine = 0;
  const int first = blockIdx.x * a.chunk, end = min(a.T, first + a.chunk);
  for (int t0 = first + 8 * warp; t0 < end; t0 += 64) {
    const unsigned found = teacher_weights(a, t0, end, lane);
    if (lane < 8 && t0 + lane < end) a.plan.slot[t0 + lane] = found >> lane & 1 ? 0 : -1;
    mine += __popc(found);
  }
  if (lane == 0) part[warp] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int w = 0; w < 8; ++w) n += part[w];
    a.counts[blockIdx.x] = n;
  }
}

// ------------------------------------------------------------------------------------------------ rows in the products' type
// Eight elements of a row from column c on, zeros behind its end, as they lie in memory
struct Eight16 {
  uint4 w;
  __device__ __forceinline__ void load(const Source& s, long long row, int c) {
    const __half* const from = static_cast<const __half*>(s.p) + row * s.ld + c;
    if (s.fast == 2) {
      w = c < s.K ? *reinterpret_cast<const uint4*>(from) : make_uint4(0, 0, 0, 0);
      return;
    }
    uint32_t u[4] = {0, 0, 0, 0};
    if (s.fast == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + 2 * i < s.K) u[i] = *reinterpret_cast<const uint32_t*>(from + 2 * i);
      w = make_uint4(u[0], u[1], u[2], u[3]);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < s.K) u[i >> 1] |= (uint32_t) * reinterpret_cast<const uint16_t*>(from + i) << (16 * (i & 1));
    w = make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void store(uint16_t* to, long long) const { *reinterpret_cast<uint4*>(to) = w; }
};
struct Eight32 {
  float f[8];
  __device__ __forceinline__ void load(const Source& s, long long row, int c) {
    const float* const from = static_cast<const float*>(s.p) + row * s.ld + c;
    zero();
    if (s.fast == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + 2 * i < s.K) {
          const float2 v = *reinterpret_cast<const float2*>(from + 2 * i);
          f[2 * i] = v.x, f[2 * i + 1] = v.y;
        }
      return;
    }
    if (s.fast == 2) {
      if (c >= s.K) return;
      const float4 u = reinterpret_cast<const float4*>(from)[0], v = reinterpret_cast<const float4*>(from)[1];
      f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w, f[4] = v.x, f[5] = v.y, f[6] = v.z, f[7] = v.w;
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < s.K) f[i] = from[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
  }
  // three bf16 parts, `plane` elements apart
  __device__ __forceinline__ void store(uint16_t* to, long long plane) const {
    float left[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) left[i] = f[i];
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = pack_bf16(left[2 * i], left[2 * i + 1]);
        left[2 * i] -= bf16_lo(w[i]), left[2 * i + 1] -= bf16_hi(w[i]);
      }
      *reinterpret_cast<uint4*>(to + part * plane) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};
// CTAs of rows: a chunk each, or a slice of its columns.  Its rows that count, to their slots.  FIRST: in the forward, which makes the plan too.
template <class E, bool FIRST> __global__ void __launch_bounds__(256) k_prepare(const __grid_constant__ Prep a) {
  constexpr int PARTS = std::is_same<E, Eight32>::value ? 3 : 1;
  next_may_start();
  wait_for_kernel_before();
  __shared__ int list[BLOCK], part[2][8];
  __shared__ unsigned flags[SELF / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x >= a.row_ctas + a.w_ctas) {
    scaled_bias(a, (blockIdx.x - a.row_ctas - a.w_ctas) * 256 + threadIdx.x, (gridDim.x - a.row_ctas - a.w_ctas) * 256);
    return;
  }
  if (blockIdx.x >= a.row_ctas) {                          // w, padded
    const Source& s = a.w;
    const long long plane = (long long)a.Vp * s.Kp;
    const unsigned pieces = s.Kp / 8;
    for (long long r0 = (blockIdx.x - a.row_ctas) * 8ll + warp; r0 < a.Vp; r0 += a.w_ctas * 8ll)
      for (unsigned c = lane; c < pieces; c += 32) {
        E e;
        if (r0 < a.V) e.load(s, r0, 8 * c);
        else e.zero();
        e.store(a.ws + r0 * s.Kp + 8 * c, plane);
      }
    return;
  }
  const Source& s = a.x;
  const int chunk = blockIdx.x / a.slices, slice = blockIdx.x - chunk * a.slices;
  const long long plane = (long long)a.Tp * s.Kp;
  const int pieces = s.Kp / 8, per = (pieces + a.slices - 1) / a.slices, p0 = slice * per, mine = max(0, min(pieces, p0 + per) - p0);
  auto copy = [&](int first, int here) {                   // the listed rows' columns of this slice, four pieces a thread under way
    const int all = here * mine;
    for (int i0 = threadIdx.x; i0 < all; i0 += 4 * 256) {
      E e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 256 * u, r = i / mine;
        if (i < all) e[u].load(s, list[r], 8 * (p0 + i - r * mine));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 256 * u, r = i / mine;
        if (i < all) e[u].store(a.xs + (long long)(first + r) * s.Kp + 8 * (p0 + i - r * mine), plane);
      }
    }
  };
  const int chunk_end = min(a.T, (chunk + 1) * a.chunk);
  int n;
  if constexpr (FIRST) {
    const int chunks = (a.T + a.chunk - 1) / a.chunk;
    int before = 0, all = 0;
    if (a.counts != nullptr) {
#pragma unroll 4
      for (int c = threadIdx.x; c < chunks; c += 256) {
        const int m = a.counts[c];
        all += m;
        if (c < chunk) before += m;
      }
    } else {
      const int words = (a.T + 31) / 32;
      for (int i = threadIdx.x; i < words; i += 256) flags[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < a.T * a.k; i += 256) {
        const int t = i / a.k;
        if (a.teacher ? is_entry(a, i) : a.labels[i] != a.ignore) atomicOr(&flags[t >> 5], 1u << (t & 31));
      }
      __syncthreads();
      for (int i = threadIdx.x; i < words; i += 256) {
        all += __popc(flags[i]);
        if (i < chunk * (a.chunk / 32)) before += __popc(flags[i]);
      }
      if (slice == 0 && a.teacher != nullptr)
        for (int t0 = chunk * a.chunk + 8 * warp; t0 < chunk_end; t0 += 64) teacher_weights(a, t0, chunk_end, lane);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o), all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) part[0][warp] = before, part[1][warp] = all;
    __syncthreads();
    int first = 0;
    n = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) first += part[0][w], n += part[1][w];
    __syncthreads();
    const bool in_place = a.few || (a.direct && n == a.T);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.plan.head[0] = n, a.plan.head[1] = 0;
    for (int t0 = chunk * a.chunk; t0 < chunk_end; t0 += BLOCK) {
      const int end = min(chunk_end, t0 + BLOCK);
      // a warp for every 32 rows; where its first goes, after another barrier
      const int t = t0 + 32 * warp + lane;
      const bool counts = warp < BLOCK / 32 && t < end && (a.counts == nullptr ? flags[t >> 5] >> (t & 31) & 1 : a.teacher ? a.plan.slot[t] != -1 : a.labels[t] != a.ignore);
      const unsigned who = __ballot_sync(0xffffffffu, counts);
      if (lane == 0) part[0][warp] = __popc(who);
      __syncthreads();
      int place = __popc(who & ((1u << lane) - 1)), here = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        if (w < warp) place += part[0][w];
        here += part[0][w];
      }
      if (counts) list[place] = t;
      if (slice == 0 && warp < BLOCK / 32 && t < end) {
        // (other slices of the chunk may read a slot before or after this: that it is -1 or not stays)
        a.plan.slot[t] = counts ? first + place : -1;
        if (a.loss_rows != nullptr && !counts) a.loss_rows[t] = 0.f;
        if (counts) a.plan.row[first + place] = t;
      }
      __syncthreads();
      if (slice == 0)
        for (int i = threadIdx.x; i < here * a.k; i += 256) {
          const int r = i / a.k, j = i - r * a.k;
          const long long from = (long long)list[r] * a.k + j, to = (long long)j * a.Tp + first + r, v = a.labels[from];
          const float q = a.teacher ? a.q[from] : 1.f;
          a.plan.target[to] = a.teacher && (v == -1 || q == 0.f) ? -1 : v < 0 || v >= a.V ? -2 : (int)v;
          if (a.teacher) a.plan.q[to] = v == -1 ? 0.f : q;
          a.zt[to] = not_a_number();                        // of a target that no tile has
        }
      if (!in_place) copy(first, here);
      first += here;
      __syncthreads();
    }
    if (in_place) return;
  } else {
    n = a.plan.head[0];
    if (a.few || (a.direct && n == a.T)) return;
    for (int first = chunk * a.chunk; first < min(n, (chunk + 1) * a.chunk); first += BLOCK) {
      const int here = min(BLOCK, min(n, (chunk + 1) * a.chunk) - first);
      for (int i = threadIdx.x; i < here; i += 256) list[i] = a.plan.row[first + i];
      __syncthreads();
      copy(first, here);
      __syncthreads();
    }
  }
  // zeros up to the end of the last tile: what it holds is multiplied with zeros
  const int zeros = (n + PAD - 1) / PAD * PAD - n;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < (long long)zeros * pieces; i += a.row_ctas * 256ll)
#pragma unroll
    for (int p = 0; p < PARTS; ++p) *reinterpret_cast<uint4*>(a.xs + p * plane + (long long)n * s.Kp + 8 * i) = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------------------------------------ the four products
enum Mode { LOGSUM, GRAD, GRADS };                        // GRADS: dx and dW, two products in one launch
enum : int { DX, DW };                                    // ... and which of them
constexpr int BK = 64;                                    // elements of the contraction in a chunk: 128 bytes
constexpr uint32_t HALF = 128 * BK * 2;
// What a kernel is made for, beside its product: what it need not do costs registers that the sums want.
enum : int { ONE = 1, THREE = 2, COLUMNS = 4, WIDE = 8, TWO = 16 };  // one target a row (LOGSUM, GRAD); G in three or two parts, sums of G's columns (GRAD); wide tiles (LOGSUM)
// PAIR: two CTAs of a cluster share a tile of 256 x 256; else tiles of 128 x 128, or (WIDE) 128 rows of as many columns as leave one tile to each multiprocessor: few rows, where
// the weights are all there is to read (16 x 2048 to 32000: 250 tiles of 128 43 us alone, 143 of 224 38).  A thread that writes has 64 columns: what it does with them
// is a chain of latencies, and four warps a scheduler hide more of each other's than two with 128 columns each do (8192 x 64 to 64000: k_gemm<LOGSUM> 663 us, so 462; k_gemm<GRAD> 911, 698).
template <int MODE, bool PAIR, int OPT> struct Shape {
  static constexpr bool LARGE = PAIR || (OPT & WIDE);
  static constexpr int BN = LARGE ? 256 : 128, TILE = PAIR ? 256 : 128, W = 64;        // columns (at most) and rows of a tile; columns of a writing thread
  static constexpr int EPI = 4 * BN / W, THREADS = 32 * (2 + EPI), STAGES = OPT & WIDE ? 4 : 6;
  static constexpr uint32_t STAGE = (OPT & WIDE ? 3 : 2) * HALF;                       // of A, and of B
  static constexpr uint32_t BARS = STAGES * STAGE, STAGED = BARS + 16 * STAGES + 128;   // STAGED: 32 x 16 results a writing warp, rows of 17 (DW)
  static constexpr uint32_t SMEM = MODE == GRADS ? STAGED + EPI * 32 * 17 * 4 : STAGED;
};
static_assert(Shape<GRADS, true, 0>::SMEM <= 232448 && Shape<GRADS, false, 0>::SMEM <= 232448 && Shape<LOGSUM, false, WIDE>::SMEM <= 232448, "shared memory of a multiprocessor");

// What the products with G are multiplied with.
struct Coef {
  const float* g;                                         // one number, or null
  const float* unit;                                      // fp16: [0]: the largest |g|, rounded to a power of two; [1]: its reciprocal; else null
  int mean;
  float scale;                                            // 1 / (tau gscale)
  __device__ __forceinline__ float alpha(int n) const {
    if (g == nullptr) return unit ? unit[0] * scale : scale;
    return n > 0 ? (mean ? *g / (float)n : *g) * scale : 0.f;
  }
};
// Parts of dx's contraction.  Alone: the number that leaves the fewest units idle in the last round of tiles, a fiftieth less for each part more (its sums are written and read
// once more), eight at most and eight rounds; 8192 x 2048 from 16384 columns, 256 tiles on 74 pairs: one part 386 us, two 355.  Beside dW's tiles, which fill what is left: the
// share of a unit in all chunks, and half of the longest tile.  G in two parts: up to 32 where there are a few tiles only (71 x 2 to 63111 130 us by eight, 99).
struct Parts {
  int units, chunks;        // of the first piece of the vocabulary: every piece is cut alike
  int other, other_parts;   // tiles of dW beside it, and the parts of their contraction
  int alone;                // parts of a tile that is nearly alone (units for four times as many), or 8
  __device__ int of(int tiles, int n) const {
    if (tiles <= 0 || tiles > 8 * units) return 1;
    const int oc = other ? ((n + BK - 1) / BK + other_parts - 1) / other_parts : 0;
    int best = 1;
    long long least = 0;
    for (int s = 1; (s <= 8 || (s <= alone && 4 * tiles * s <= units)) && (s == 1 || (tiles * s <= 8 * units && 4 * s <= chunks)); ++s) {
      const int c = (chunks + s - 1) / s, rounds = (tiles * s + units - 1) / units;
      const long long longest = c > oc ? c : oc;          // times in chunks of a tile, times twice the units
      const long long time = (other ? 2 * ((long long)tiles * chunks + (long long)other * oc) + longest * units : 2ll * rounds * c * units) * (50 + s);
      if (s == 1 || time < least) best = s, least = time;
    }
    return best;
  }
};
struct Args {
  int on;                                                 // 0: nothing to do (GRADS)
  const int* n;                                           // rows that count
  int products;                                           // 1; 2 of G's two parts; 6 of three parts
  long long plane_a, plane_b;                             // rows of a part in the maps
  int M, N, L;                                            // rows of D (0: n), columns of D, contraction (0: n)
  int row0, most;                                         // first slot and slots of a launch (0: all)
  int bn;                                                 // WIDE: columns of a tile, a multiple of 32
  int col0;                                               // first column of the piece of the vocabulary
  int chain;                                              // (chunk, product) pairs that one accumulator takes, a multiple of `products`
  int splits;                                             // of the contraction (0: by `cut`)
  Parts cut;
  int fp16;                                               // operands are fp16, else bf16
  int direct_rows;                                        // rows of x, where they are read as they lie if all count; else 0
  // LOGSUM, GRAD
  Plan plan; int Tp, k;
  const float* bias2; float c1;
  float2* part; int parts;                                // [slots, parts] largest, sum
  float* zt;                                              // [k][Tp]
  const float* g; Coef coef;                              // per row or null
  uint16_t* G; long long ldg;                             // [planes][Tp][ldg]
  float* colsum;                                          // [Tp / 32][ldg] or null
  float gscale;                                           // 1, or 2^13 in fp16
  // DX, DW
  float* out; long long ldo; int add;                     // fp32 partial sums: [split][rows of whole tiles][ldo]
  void* dw; int dw_type; long long K; int V;              // DW, one split: the result
};
struct Maps { CUtensorMap a, b, x; };                       // x: the rows as they lie, in place of a (LOGSUM, GRAD) or of b (dW)
template <int MODE> struct Call {
  static constexpr int PRODUCTS = MODE == GRADS ? 2 : 1;
  Args a[PRODUCTS];
  Maps maps[PRODUCTS];
};

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
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }
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
__device__ __forceinline__ void pair_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pair_commit(uint32_t bar) {             // on both CTAs' barriers
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// the partial products of the split operands, smallest first: (part of A, part of B); two: of A alone
__device__ __forceinline__ void parts_of(int products, int i, int& a, int& b) {
  a = b = 0;
  if (products <= 2) {
    a = products - 1 - i;
    return;
  }
  a = (0x010210 >> (4 * i)) & 3;                          // 0 1 2 0 1 0
  b = (0x001012 >> (4 * i)) & 3;                          // 2 1 0 1 0 0
}

// What a launch works on, the same in all its warps and (for DX) in the kernel that joins the sums
struct Work { int tiles_m, tiles_n, splits, chunks, per; };
// Parts of dW's contraction: as many as there are units for each tile
__host__ __device__ __forceinline__ int split_by_units(int tiles, int units, int chunks) {
  const int s = units / (tiles > 0 ? tiles : 1), most = chunks / 4;
  return s > most ? (most > 0 ? most : 1) : s > 0 ? s : 1;
}
__device__ __forceinline__ Work work_of(const Args& a, int n, int tile_m, int tile_n) {
  Work w;
  const int rows_ = a.M ? a.M : a.most ? min(a.most, max(0, n - a.row0)) : n;
  w.tiles_m = a.on ? (rows_ + tile_m - 1) / tile_m : 0;
  w.tiles_n = (a.N + tile_n - 1) / tile_n;
  w.chunks = ((a.L ? a.L : n) + BK - 1) / BK;
  w.splits = a.splits ? a.splits : a.cut.of(w.tiles_m * w.tiles_n, n);
  w.per = (w.chunks + w.splits - 1) / w.splits;
  return w;
}
// Tiles in groups of 8 rows of tiles, column by column inside a group: the CTAs that run at a time share their operands in L2 (8192 x 4096 to 128000, forward and
// backward: groups of 4 28.5 ms, 8 and 16 27.3).
constexpr int GROUP = 8;
template <class Wk> __device__ __forceinline__ void item_at(const Wk& w, int i, int& s, int& m, int& n, int& c0, int& c1) {
  const int tiles = w.tiles_m * w.tiles_n;
  s = i / tiles;
  i -= s * tiles;
  const int per = GROUP * w.tiles_n, group = i / per, rows_here = min(GROUP, (int)w.tiles_m - GROUP * group), j = i - group * per;
  n = j / rows_here;
  m = GROUP * group + j - n * rows_here;
  const int chunks = w.chunks, share = w.per;
  c0 = min(s * share, chunks), c1 = min(c0 + share, chunks);
}

__device__ __forceinline__ void st_v8(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
               "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int fp16) {
  if (!fp16) return pack_bf16(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What a writing thread knows of its row before the sums are there: it is read while they are formed
struct Row {
  bool in;                  // the row counts
  int slot, found;          // targets among the thread's columns: how many,
  int width;                // of the thread's columns, those of its tile
  uint32_t two;             // and of the first two the column and the target, a byte each
  float lse, r, less;       // less: ONE, GRAD (others read it where they need it)
};
// f(offset, target) of every target among the columns g .. g + 31 of the thread's
template <int OPT, class F> __device__ __forceinline__ void each_target(const Args& a, const Row& row, int c, int g, F f) {
  constexpr int REMEMBERED = OPT & ONE ? 1 : 2;
#pragma unroll
  for (int i = 0; i < REMEMBERED; ++i) {
    const int off = (int)(row.two >> (16 * i) & 0xff) - g;
    if (row.found > i && (unsigned)off < 32u) f(off, (int)(row.two >> (16 * i + 8) & 0xff));
  }
  if (!(OPT & ONE) && row.found > 2) {                     // seldom: all over again, without those two
    for (int j = (int)(row.two >> 24) + 1; j < a.k; ++j) {
      const int off = a.plan.target[(long long)j * a.Tp + row.slot] - c - g;
      if ((unsigned)off < 32u && g + off < row.width) f(off, j);
    }
  }
}
template <int MODE, int W, int OPT> __device__ __forceinline__ Row row_of(const Args& a, int n, int row, int c, int width) {
  Row r = {};
  if (MODE != LOGSUM && MODE != GRAD) return r;
  r.width = width;
  r.in = row < n;
  r.slot = r.in ? row : 0;
  r.lse = INFINITY;
  if (r.in) {
    const int* const target = a.plan.target + r.slot;
    if (OPT & ONE) {
      const int t = target[0], off = t - c;
      if (off >= 0 && off < width && t >= 0) r.two = off, r.found = 1;
    }
    for (int j0 = 0; !(OPT & ONE) && j0 < a.k; j0 += 16) {  // sixteen loads under way: one after another they are 0.25 us each
      int t[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) t[u] = j0 + u < a.k ? target[(long long)(j0 + u) * a.Tp] : -1;
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const int off = t[u] - c;
        if (off >= 0 && off < width && t[u] >= 0) {
          if (r.found < 2) r.two |= (uint32_t)(off | (j0 + u) << 8) << (16 * r.found);
          ++r.found;
        }
      }
    }
    if (MODE == GRAD) {
      r.lse = a.plan.lse[r.slot];
      if (OPT & ONE) r.less = a.plan.less[r.slot];
      r.r = (a.g ? a.g[a.plan.row[r.slot]] * (a.coef.unit ? a.coef.unit[1] : 1.f) : 1.f) * a.gscale;
    }
  }
  return r;
}

// What a thread does with its sums: row `row` of D, columns col .. col + W - 1
template <int MODE, int W, int OPT, int which> __device__ __forceinline__ void epilogue(const Args& a, int out_row, float (&acc)[W / 32][32], const Row& me, int n, int row, int col, int part, int width, float* stage) {
  const int lane = threadIdx.x & 31;
  if constexpr (MODE == LOGSUM || MODE == GRAD) {
    const int slot = me.slot, c = a.col0 + col;           // of the vocabulary
#pragma unroll
    for (int g = 0; g < W; g += 4) {
      const float4 b = *reinterpret_cast<const float4*>(a.bias2 + c + g);
      acc[g / 32][g % 32] = fmaf(acc[g / 32][g % 32], a.c1, b.x), acc[(g + 1) / 32][(g + 1) % 32] = fmaf(acc[(g + 1) / 32][(g + 1) % 32], a.c1, b.y);
      acc[(g + 2) / 32][(g + 2) % 32] = fmaf(acc[(g + 2) / 32][(g + 2) % 32], a.c1, b.z), acc[(g + 3) / 32][(g + 3) % 32] = fmaf(acc[(g + 3) / 32][(g + 3) % 32], a.c1, b.w);
    }
    if constexpr (MODE == LOGSUM) {
      float top = -INFINITY, sum[4] = {0.f, 0.f, 0.f, 0.f};
      if constexpr ((OPT & WIDE) != 0) {                  // columns of the next tile, or of none
#pragma unroll
        for (int g = 0; g < W; g += 32)
          if (g >= width)
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[g / 32][e] = -INFINITY;
      }
#pragma unroll
      for (int g = 0; g < W; ++g) top = fmaxf(top, acc[g / 32][g % 32]);
#pragma unroll
      for (int g = 0; g < W; g += 32)
        each_target<OPT>(a, me, c, g, [&](int off, int j) {
          float z = 0.f;
#pragma unroll
          for (int e = 0; e < 32; ++e) z = e == off ? acc[(g + e) / 32][(g + e) % 32] : z;
          a.zt[(long long)j * a.Tp + slot] = z;
        });
      const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int g = 0; g < W; ++g) sum[g % 4] += ex2(acc[g / 32][g % 32] - from);
      if (me.in) a.part[(long long)(row - a.row0) * a.parts + part] = make_float2(top, (sum[0] + sum[1]) + (sum[2] + sum[3]));
    } else {
      const float lse = me.lse, r = me.r;
#pragma unroll
      for (int g = 0; g < W; g += 32) {
        float (&v)[32] = acc[g / 32];                      // in place: there is no room for another 32
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = ex2(v[e] - lse) * r;      // zeros of rows that do not count: their lse is inf
        each_target<OPT>(a, me, c, g, [&](int off, int j) {
          if constexpr ((OPT & ONE) != 0) {
            const float less = me.less * r;
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = e == off ? less : v[e];
          } else {
            float q = a.plan.q[(long long)j * a.Tp + slot];
            if (q == 1.f) {                               // in place of p, not beside it (others of the row weigh less than its rounding)
              q = -a.plan.less[slot];
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = e == off ? 0.f : v[e];
            }
            q *= r;
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] -= e == off ? q : 0.f;
          }
        });
        uint16_t* const to = a.G + (long long)row * a.ldg + col + g;
        if constexpr (!(OPT & (THREE | TWO))) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t out[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = pack2(v[16 * h + 2 * e], v[16 * h + 2 * e + 1], a.fp16);
            st_v8(to + 16 * h, out);
          }
        } else {                                          // sixteen columns at a time, part by part
          const long long plane = (long long)a.Tp * a.ldg;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float left[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) left[e] = v[16 * h + e];
#pragma unroll
            for (int p = 0; p < (OPT & THREE ? 3 : 2); ++p) {
              uint32_t out[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                out[e] = pack2(left[2 * e], left[2 * e + 1], OPT & TWO ? a.fp16 : 0);
                if (OPT & TWO && a.fp16) {
                  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&out[e]));
                  left[2 * e] -= f.x, left[2 * e + 1] -= f.y;
                } else {
                  left[2 * e] -= bf16_lo(out[e]), left[2 * e + 1] -= bf16_hi(out[e]);
                }
              }
              st_v8(to + p * plane + 16 * h, out);
            }
          }
        }
        if constexpr ((OPT & COLUMNS) != 0) {             // over the warp's 32 rows: lane l ends with column l
#pragma unroll
          for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < o; ++i) {
              const bool up = lane & o;
              const float give = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
              v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
          a.colsum[(long long)(row >> 5) * a.ldg + col + g + lane] = v[0];
        }
      }
    }
  } else {
    if (MODE == GRADS && which == DW && a.dw != nullptr) {
      const float alpha = a.coef.alpha(n);
      const int v = a.col0 + row;
      if (a.K % 8 == 0) {
        if (v >= a.V) return;
#pragma unroll
        for (int g = 0; g < W; g += 8) {
          if (col + g >= a.K) continue;
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = acc[(g + e) / 32][(g + e) % 32] * alpha;
          const long long at = (long long)v * a.K + col + g;
          if (a.dw_type == SPION_F32) Out<float, 8>::store(static_cast<float*>(a.dw) + at, f);
          else if (a.dw_type == SPION_BF16) Out<__nv_bfloat16, 8>::store(static_cast<__nv_bfloat16*>(a.dw) + at, f);
          else Out<__half, 8>::store(static_cast<__half*>(a.dw) + at, f);
        }
        return;
      }
      // rows that start anywhere: lanes side by side along each (one row a lane: 10007 rows of 770 fp16 126 us, so 31)
#pragma unroll
      for (int g = 0; g < W; g += 16) {
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 16; ++e) stage[17 * lane + e] = acc[(g + e) / 32][(g + e) % 32] * alpha;
        __syncwarp();
        const int c = col + g + (lane & 15), v0 = v - lane;
        if (c < a.K)
#pragma unroll 4
          for (int r = lane >> 4; r < 32; r += 2)
            if (v0 + r < a.V) store_any(a.dw, a.dw_type, (long long)(v0 + r) * a.K + c, stage[17 * r + (lane & 15)]);
      }
      return;
    }
    float* const to = a.out + (long long)out_row * a.ldo + col;
#pragma unroll
    for (int g = 0; g < W; g += 8) {
      if (col + g >= a.ldo) continue;
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = acc[(g + e) / 32][(g + e) % 32];
      if (a.add) {
        Piece<float, 8> was;
        was.load(to + g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += was.at(e);
      }
      Out<float, 8>::store(to + g, f);
    }
  }
}

// Warp 0 loads, warp 1 multiplies, the others take the sums.  Every wait is bounded; whoever gives up reports it and leaves, and so do all that wait for it; the warps
// that write go on with NaN.  PAIR: two CTAs of a cluster share a tile of 256 x 256, each brings 128 rows of either operand and holds 128 rows of the sums; the first one's warp 1
// multiplies for both (see k_lin8 in linear_e4m3.cu, whose scheme this is).  Else tiles of 128 x 128.
// 8192 x 2048 to 32000, bf16: z and its log sums 660 us (1.63 PFLOP/s, the tensor pipe 93 % busy), z and G 705 - 740, dx and dW 1480 (1.45 PFLOP/s, at the power cap).
// Operands whose contraction runs along memory (K-major: x and W in z, G in dx) come as one box of 128 rows x 64; those whose contraction runs across it (MN-major: W in dx, G and x
// in dW) as two boxes of 64 rows x 64.
template <int MODE, bool PAIR, int OPT> __global__ void __launch_bounds__(Shape<MODE, PAIR, OPT>::THREADS, 1) k_gemm(const __grid_constant__ Call<MODE> call) {
  using C = Shape<MODE, PAIR, OPT>;
  constexpr int BN = C::BN, TILE = C::TILE, W = C::W, STAGES = C::STAGES, EPI = C::EPI;
  constexpr uint32_t STAGE = C::STAGE;
  constexpr bool TWO = MODE == GRADS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  const uint32_t full = sbase + C::BARS, empty = full + 8 * STAGES, acc_full = empty + 8 * STAGES, acc_empty = acc_full + 16, slot = acc_empty + 16;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  volatile int& s_abort = *reinterpret_cast<int*>(smem_raw + (slot + 8 - sbase));
  const int rank = PAIR ? (int)cta_rank() : 0, first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
  if (warp == 0 && lane == 0) {
    s_abort = *reinterpret_cast<volatile int*>(&g_vocab_status);
    for (int i = 0; i < STAGES; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(acc_full + 8 * i, 1), mbar_init(acc_empty + 8 * i, PAIR ? 2 * EPI : EPI);
    fence_barrier_init();
    fence_proxy_async();
    for (int i = 0; i < Call<MODE>::PRODUCTS; ++i) {
      tma_prefetch_desc(&call.maps[i].a);
      tma_prefetch_desc(&call.maps[i].b);
      tma_prefetch_desc(&call.maps[i].x);
    }
  }
  if (warp == 1) {
    if (PAIR) {
      pair_tmem_alloc(slot, 2 * BN);
    } else {
      tmem_alloc(slot, 2 * BN);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t*>(smem_raw + (slot - sbase));
  wait_for_kernel_before();
  const int n = *reinterpret_cast<const volatile int*>(call.a[0].n);
  const int bn = OPT & WIDE ? call.a[0].bn : BN;
  const Work w0 = work_of(call.a[0], n, TILE, bn), w1 = TWO ? work_of(call.a[Call<MODE>::PRODUCTS - 1], n, TILE, BN) : Work();
  const bool direct = n == call.a[0].direct_rows;
  const int items0 = w0.splits * w0.tiles_m * w0.tiles_n, items = items0 + (TWO ? w1.splits * w1.tiles_m * w1.tiles_n : 0);
  const bool aborted = s_abort != 0;
  // the writing warps keep it in shared memory: every register beside their sums counts
  volatile Work* const kept = reinterpret_cast<Work*>(smem_raw + (slot + 16 - sbase));
  if (threadIdx.x < (TWO ? 2 : 1)) {
    const Work& w = threadIdx.x ? w1 : w0;
    volatile Work& k = kept[threadIdx.x];
    k.tiles_m = w.tiles_m, k.tiles_n = w.tiles_n, k.splits = w.splits, k.chunks = w.chunks, k.per = w.per;
  }
  __syncthreads();
  if (warp == 0) {
    if (!aborted && elect_one()) {
      int st = 0, ph = 1;                                  // a ring that has not been used yet is empty
      long long fills = 0;
      bool ok = true;
      for (int i = first; i < items && ok; i += step) {
        int s, m, nn, c0, c1;
        const int which = TWO && i >= items0;
        const Args& a = call.a[which];
        const Maps& maps = call.maps[which];
        const bool a_mn = TWO && which == DW, b_mn = TWO;
        const CUtensorMap *const map_a = !TWO && direct ? &maps.x : &maps.a, *const map_b = a_mn && direct ? &maps.x : &maps.b;
        item_at(which ? w1 : w0, i - (which ? items0 : 0), s, m, nn, c0, c1);
        const int ra = m * TILE + rank * 128 + (MODE == LOGSUM ? a.row0 : 0), rb = nn * bn + rank * 128, b0 = a_mn ? 0 : a.col0;
        // of an accumulator's chunks the small products first: what is added is truncated beside the sum so far (two parts of G: chunk by chunk, whose weights the L2 cache still has)
        const int most = a.products > 2 ? a.chain / a.products : 1;
        for (int from = c0; from < c1 && ok; from += most)
          for (int p = 0, c = from; p < a.products && ok;) {
            ok = mbar_wait(empty + 8 * st, ph);
            if (!ok) break;
            int pa, pb;
            parts_of(a.products, p, pa, pb);
            const uint32_t to_a = sbase + st * STAGE, to_b = to_a + HALF;
            uint32_t bar = full + 8 * st;
            if (PAIR) {
              if (rank == 0) mbar_expect_tx(bar, 2 * STAGE);
              bar = in_leader(bar);
            } else {
              mbar_expect_tx(bar, OPT & WIDE ? HALF + bn * BK * 2 : STAGE);
            }
            auto load = [&](uint32_t to, const CUtensorMap* map, int x, int y) {
              if (PAIR) pair_tma_load_2d(to, map, bar, x, y);
              else tma_load_2d(to, map, bar, x, y);
            };
            const int ya = (int)(pa * a.plane_a), yb = (int)(pb * a.plane_b) + b0;
            if (a_mn) {
              load(to_a, map_a, ra, ya + c * BK);
              load(to_a + HALF / 2, map_a, ra + 64, ya + c * BK);
            } else {
              load(to_a, map_a, c * BK, ya + ra);
            }
            if (b_mn) {
              load(to_b, map_b, rb, yb + c * BK);
              load(to_b + HALF / 2, map_b, rb + 64, yb + c * BK);
            } else {
              load(to_b, map_b, c * BK, yb + rb);
            }
            ++fills;
            if (++st == STAGES) st = 0, ph ^= 1;
            if (++c == min(from + most, c1)) c = from, ++p;
          }
      }
      if (!ok) {                                           // the copies under way end first (a pair's are counted in its first CTA), or this gives up again
        report(&g_vocab_status, ERR_LOAD_WAIT);
        for (long long j = fills > STAGES ? fills - STAGES : 0; j < fills && rank == 0; ++j)
          mbar_wait(full + 8 * (int)(j % STAGES), (int)(j / STAGES) & 1);
      }
    }
  } else if (warp == 1) {
    if (!aborted && rank == 0 && elect_one()) {
      const uint32_t kind = call.a[0].fp16 ? 0u : (1u << 7) | (1u << 10);
      const uint32_t shape = (1u << 4) | kind | ((uint32_t)TWO << 16) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
      const uint64_t b0 = make_smem_desc(sbase + HALF, TWO ? HALF / 2 : 16, 1024, LAYOUT_SW128);
      constexpr uint32_t step_b = TWO ? 2048 : 32;
      int st = 0, ph = 0, buf = 0, acc_ph = 1;
      bool ok = true;
      // A_MN at compile time: descriptors that depend on a branch do not stay in uniform registers
      auto multiply = [&](auto a_mn, const Args& a, int all) {
        constexpr bool A_MN = decltype(a_mn)::value;
        constexpr uint32_t step_a = A_MN ? 2048 : 32;
        const uint32_t idesc = shape | ((uint32_t)A_MN << 15);
        const uint64_t a0 = make_smem_desc(sbase, A_MN ? HALF / 2 : 16, 1024, LAYOUT_SW128);
        for (int done = 0; done < all && ok;) {
          ok = mbar_wait(acc_empty + 8 * buf, acc_ph);
          tc_fence_after();
          const int until = min(all, done + a.chain);
          for (bool more = false; done < until && ok; ++done) {
            ok = mbar_wait(full + 8 * st, ph);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              const uint64_t ad = desc_advance(a0, st * STAGE + step_a * k), bd = desc_advance(b0, st * STAGE + step_b * k);
              if (PAIR) pair_mma(tmem + buf * BN, ad, bd, idesc, more);
              else mma_bf16(tmem + buf * BN, ad, bd, idesc, more);
              more = true;
            }
            if (PAIR) pair_commit(empty + 8 * st);
            else mma_commit(empty + 8 * st);
            if (++st == STAGES) st = 0, ph ^= 1;
          }
          if (ok) {
            if (PAIR) pair_commit(acc_full + 8 * buf);
            else mma_commit(acc_full + 8 * buf);
          }
          buf ^= 1;
          if (buf == 0) acc_ph ^= 1;
        }
      };
      for (int i = first; i < items && ok; i += step) {
        int s, m, nn, c0, c1;
        const int which = TWO && i >= items0;
        item_at(which ? w1 : w0, i - (which ? items0 : 0), s, m, nn, c0, c1);
        const int all = (c1 - c0) * call.a[0].products;
        if (TWO && which == DW) multiply(std::integral_constant<bool, TWO>(), call.a[Call<MODE>::PRODUCTS - 1], all);
        else multiply(std::integral_constant<bool, false>(), call.a[0], all);
      }
      if (!ok) report(&g_vocab_status, ERR_MMA_WAIT);
    }
  } else {
    const int q = warp & 3, share = (warp - 2) >> 2;
    int buf = 0, ph = 0;
    bool lost = aborted;
    float acc[W / 32][32];
    for (int i = first;; i += step) {
      int s, m, nn, c0, c1, which = 0, at = i;
      const int before = kept[0].splits * kept[0].tiles_m * kept[0].tiles_n;
      if (i >= before) {
        if (!TWO || i >= before + kept[1].splits * kept[1].tiles_m * kept[1].tiles_n) break;
        which = 1, at = i - before;
      }
      const Args& a = call.a[which];
      item_at(kept[which], at, s, m, nn, c0, c1);
      const int all = (c1 - c0) * a.products;
      const int row = (MODE == LOGSUM ? a.row0 : 0) + m * TILE + rank * 128 + q * 32 + lane, col = nn * bn + share * W, width = OPT & WIDE ? min(W, bn - share * W) : W;
      const Row me = row_of<MODE, W, OPT>(a, n, row, a.col0 + col, width);
      // the first chain's sums as they come, the others' on top, sixteen at a time: more would not fit beside the sums
      auto ready = [&] {
        lost = !tc::warp_wait(acc_full + 8 * buf, ph, &g_vocab_status, ERR_MMA2_WAIT);
        tc_fence_after();
        return !lost;
      };
      auto taken = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) pair_arrive(in_leader(acc_empty + 8 * buf));
          else mbar_arrive(acc_empty + 8 * buf);
        }
        buf ^= 1;
        if (buf == 0) ph ^= 1;
      };
      const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + share * W;
      uint32_t r[W / 32][32];
      if (all > 0 && !lost && ready()) {
#pragma unroll
        for (int g = 0; g < W / 32; ++g) tmem_ld32(from + buf * BN + 32 * g, r[g]);
        tmem_ld_wait();
        taken();
      } else {
#pragma unroll
        for (int g = 0; g < W; ++g) r[g / 32][g % 32] = lost ? 0x7fffffffu : 0u;
      }
#pragma unroll
      for (int g = 0; g < W; ++g) acc[g / 32][g % 32] = __uint_as_float(r[g / 32][g % 32]);
      for (int done = a.chain; done < all && !lost; done += a.chain) {
        if (!ready()) break;
#pragma unroll
        for (int g = 0; g < W; g += 16) {
          uint32_t t[16];
          tmem_ld16(from + buf * BN + g, t);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[(g + e) / 32][(g + e) % 32] += __uint_as_float(t[e]);
        }
        taken();
      }
      if (lost)
#pragma unroll
        for (int g = 0; g < W; ++g) acc[g / 32][g % 32] = not_a_number();
      float* const stage = reinterpret_cast<float*>(smem_raw + C::STAGED) + (warp - 2) * 32 * 17;
      const int out_row = s * kept[which].tiles_m * TILE + row, part = nn * (BN / W) + share;
      if (TWO && which == DW) epilogue<MODE, W, OPT, DW>(call.a[Call<MODE>::PRODUCTS - 1], out_row, acc, me, n, row, col, part, width, stage);
      else epilogue<MODE, W, OPT, DX>(call.a[0], out_row, acc, me, n, row, col, part, width, stage);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();                                // neither CTA's memory goes while the other may signal in it
  tc_fence_after();
  if (warp == 1) {
    if (PAIR) pair_tmem_dealloc(tmem, 2 * BN);
    else tmem_dealloc(tmem, 2 * BN);
  }
}

// ------------------------------------------------------------------------------------------------ losses
struct Finish {
  Plan plan; int Tp, k;
  const float2* part; int parts;
  const float* zt;
  float* loss;              // [T] (reduction 0) or one number
  double* cta_loss;         // [launches][CTAs]
  int reduction;            // 0 none, 1 mean, 2 sum
  int row0, most;           // slots of this launch
  int launch, launches;
};
template <int LANES> __device__ __forceinline__ float row_loss(const Finish& a, int i, int lane, bool lost, float& lse, float& sure) {
  const float2* const p = a.part + (long long)(i - a.row0) * a.parts;
  float top = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int c = lane; c < a.parts; c += LANES) {
    const float2 v = p[c];
    const float m = fmaxf(top, v.x), from = m == -INFINITY ? 0.f : m;
    sum = sum * ex2(top - from) + v.y * ex2(v.x - from);
    top = m;
  }
  const float all = lane_max<LANES>(top), from = all == -INFINITY ? 0.f : all;
  sum = lane_sum<LANES>(sum * ex2(top - from));
  const float rest = log2f(sum);
  lse = from + rest;
  float loss = 0.f;
  sure = -INFINITY;
  for (int j = lane; j < a.k; j += LANES) {
    const long long at = (long long)j * a.Tp + i;
    if (a.plan.target[at] == -1) continue;
    const float q = a.plan.q ? a.plan.q[at] : 1.f, one = (from - a.zt[at]) + rest;       // (lse is rounded, to 2^-24 of itself; this to that of the numbers added up)
    loss += q * ((a.plan.q ? log2f(q) : 0.f) + one);
    if (q == 1.f) sure = one;
  }
  loss = lane_sum<LANES>(loss) * LN2;
  sure = lane_max<LANES>(sure) * LN2;                       // -ln p of a target of weight 1
  return lost ? not_a_number() : loss;
}
// LANES threads per row that counts (4, 8 or 32: the fewest that leave four partial sums or fewer to each, or 32).  A CTA adds its rows' losses, the last one the CTAs', in
// their order and in 64 bits.
template <int LANES> __global__ void __launch_bounds__(256) k_finish(const __grid_constant__ Finish a) {
  next_may_start();
  wait_for_kernel_before();
  __shared__ double sums[256];
  __shared__ int last;
  const int lane = threadIdx.x % LANES, n = *reinterpret_cast<const volatile int*>(a.plan.head);
  const bool lost = *reinterpret_cast<volatile int*>(&g_vocab_status) != 0;
  constexpr int ROWS = 256 / LANES;
  double s = 0.0;
  const int end = min(n, a.row0 + a.most);
  for (int i0 = a.row0 + blockIdx.x * ROWS; i0 < end; i0 += gridDim.x * ROWS) {
    const int i = i0 + threadIdx.x / LANES;
    float lse, sure;
    const float loss = row_loss<LANES>(a, min(i, end - 1), lane, lost, lse, sure);      // (all lanes take part in the sums over lanes)
    if (lane == 0 && i < end) {
      a.plan.lse[i] = loss != loss ? loss : lse;            // a row without a loss has no gradient either: NaN
      a.plan.less[i] = loss != loss ? loss : expm1f(-sure);
      if (a.reduction == 0) a.loss[a.plan.row[i]] = loss;
      s += (double)loss;
    }
  }
  if (a.reduction == 0) return;
  auto add_up = [&] {
    sums[threadIdx.x] = s;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
      if ((int)threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
      __syncthreads();
    }
  };
  add_up();
  if (threadIdx.x == 0) {
    a.cta_loss[a.launch * gridDim.x + blockIdx.x] = sums[0];
    __threadfence();
    last = atomicAdd(a.plan.head + 1, 1) == (int)gridDim.x * a.launches - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  s = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x * a.launches; i += 256) s += *reinterpret_cast<volatile double*>(a.cta_loss + i);
  add_up();
  if (threadIdx.x == 0) *a.loss = a.reduction == 2 ? (float)sums[0] : n > 0 ? (float)(sums[0] / n) : not_a_number();
}

// ------------------------------------------------------------------------------------------------ gradients
// unit[0]: the largest of the rows' |g|, rounded up to a power of two (products by it are exact, and neither it nor its reciprocal leaves the normal numbers); unit[1]: its reciprocal
__global__ void __launch_bounds__(1024) k_unit(const Plan plan, const float* g, float* unit) {
  next_may_start();
  wait_for_kernel_before();
  __shared__ float part[32];
  const int n = *reinterpret_cast<const volatile int*>(plan.head);
  float top = 0.f;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float v = fabsf(g[plan.row[i]]);
    if (v < INFINITY) top = fmaxf(top, v);                  // one that is not finite stays its own row's
  }
  top = lane_max<32>(top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  top = lane_max<32>(part[threadIdx.x]);
  if (threadIdx.x > 0) return;
  const float u = top > 0.f ? exp2f(fminf(fmaxf(ceilf(log2f(top)), -100.f), 126.f)) : 1.f;
  unit[0] = u, unit[1] = 1.f / u;
}
// What leaves: out[r, :] = alpha (sum over the splits of part[split][r, :]), dx by the rows' slots (zeros for rows without one), dw row by row; db[v] = alpha (sum of G's columns).
struct Join {
  const int* slot;                                        // or null: rows as they are
  const float* part; long long ldp;                       // [splits][plane rows][ldp]
  int splits, tile, tiles_n;                              // splits 0: as k_gemm<GRADS> had them
  Parts cut;
  long long plane;                                        // rows of a split (splits given)
  void* out; int type; long long rows, K;
  unsigned ctas;
};
struct Bias { const float* colsum; long long ldg; int columns; void* db; int type; int wide; unsigned ctas; };
struct Leave { const int* head; Coef coef; Join j[2]; Bias b; };

__device__ __forceinline__ void store8(const Join& a, long long r, long long c, const float (&f)[8]) {
  const long long at = r * a.K + c;
  if (a.K % 8 == 0) {
    if (a.type == SPION_F32) Out<float, 8>::store(static_cast<float*>(a.out) + at, f);
    else if (a.type == SPION_BF16) Out<__nv_bfloat16, 8>::store(static_cast<__nv_bfloat16*>(a.out) + at, f);
    else Out<__half, 8>::store(static_cast<__half*>(a.out) + at, f);
  } else if (a.K % 2 == 0) {                               // pairs
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if (c + e >= a.K) break;
      if (a.type == SPION_F32) *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at + e) = make_float2(f[e], f[e + 1]);
      else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at + e) = pack2(f[e], f[e + 1], a.type == SPION_F16);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < a.K) store_any(a.out, a.type, at + e, f[e]);
  }
}
__device__ __forceinline__ void join(const Join& a, unsigned cta, int n, float alpha, float (*shared)[8]) {
  int splits = a.splits;
  long long plane = a.plane;
  if (splits == 0) {
    const int tiles_m = (n + a.tile - 1) / a.tile;
    splits = a.cut.of(tiles_m * a.tiles_n, n);
    plane = (long long)tiles_m * a.tile;
  }
  const int pieces = (int)((a.K + 7) / 8);
  const long long all = a.rows * pieces;
  auto place = [&](long long i, long long& r, int& c) {
    r = all < 0x7fffffff ? (unsigned)i / (unsigned)pieces : i / pieces, c = (int)(i - r * pieces) * 8;
  };
  const long long step = a.ctas * 256ll;
  if (splits <= 8 && all <= step) {                        // a piece a thread: four of its parts under way
    const long long i = cta * 256ll + threadIdx.x;
    if (i >= all) return;
    long long r;
    int c;
    place(i, r, c);
    const long long from = a.slot ? a.slot[r] : r;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (from >= 0)
      for (int s = 0; s < splits; s += 4) {
        Piece<float, 8> p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (s + u < splits) p[u].load(a.part + ((s + u) * plane + from) * a.ldp + c);
          else p[u].zero();
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] += p[u].at(e);
      }
    const float by = from < 0 ? 0.f : alpha;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= by;
    store8(a, r, c, f);
    return;
  }
  if (splits <= 8) {                                       // two pieces a thread under way
    for (long long i0 = cta * 256ll + threadIdx.x; i0 < all; i0 += 2 * step) {
      float f[2][8];
      long long r[2], from[2];
      int c[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const long long i = i0 + u * step;
        place(min(i, all - 1), r[u], c[u]);
        from[u] = i >= all ? -1 : a.slot ? a.slot[r[u]] : r[u];
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[u][e] = 0.f;
      for (int s = 0; s < splits; ++s) {
        Piece<float, 8> p[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (from[u] >= 0) p[u].load(a.part + (s * plane + from[u]) * a.ldp + c[u]);
          else p[u].zero();
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) f[u][e] += p[u].at(e);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (i0 + u * step >= all) break;
        const float by = from[u] < 0 ? 0.f : alpha;        // a row that does not count: zeros, whatever arrives at the loss
#pragma unroll
        for (int e = 0; e < 8; ++e) f[u][e] *= by;
        store8(a, r[u], c[u], f[u]);
      }
    }
    return;
  }
  // of many splits, the eight warps take a share each
  const int lane = threadIdx.x & 31, share = threadIdx.x >> 5, each = (splits + 7) / 8;
  for (long long i0 = cta * 32ll; i0 < all; i0 += a.ctas * 32ll) {
    const long long i = i0 + lane;
    long long r;
    int c;
    place(min(i, all - 1), r, c);
    const long long from = a.slot ? a.slot[r] : r;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (from >= 0)
#pragma unroll 4
      for (int s = share * each; s < min(splits, (share + 1) * each); ++s) {
        Piece<float, 8> p;
        p.load(a.part + (s * plane + from) * a.ldp + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += p.at(e);
      }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) shared[threadIdx.x][e] = f[e];
    __syncthreads();
    if (share > 0 || i >= all) continue;
    for (int o = 1; o < 8; ++o)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += shared[lane + 32 * o][e];
    const float by = from < 0 ? 0.f : alpha;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= by;
    store8(a, r, c, f);
  }
}
__global__ void __launch_bounds__(256, 3) k_out(const __grid_constant__ Leave a) {
  __shared__ float shared[256][8];
  next_may_start();
  wait_for_kernel_before();
  const int n = *reinterpret_cast<const volatile int*>(a.head);
  const float alpha = *reinterpret_cast<volatile int*>(&g_vocab_status) != 0 ? not_a_number() : a.coef.alpha(n);
  // the long chains of sums first: db (32 columns a CTA and eight shares of the blocks of 32 rows; of many blocks 8 columns and 32 shares); dw; dx
  if (blockIdx.x < a.b.ctas) {
    const int wide = a.b.wide, lane = threadIdx.x & (wide - 1), shares = 256 / wide, share = threadIdx.x / wide, c = blockIdx.x * wide + lane;
    float *const flat = &shared[0][0], s = 0.f;
    if (c < a.b.columns)
#pragma unroll 8
      for (int k = share; k < (n + 31) / 32; k += shares) s += a.b.colsum[k * a.b.ldg + c];
    if (wide == 8) {
      s += __shfl_xor_sync(0xffffffffu, s, 8);
      s += __shfl_xor_sync(0xffffffffu, s, 16);
    }
    if ((threadIdx.x & 31) < wide) flat[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x >= wide || c >= a.b.columns) return;
    for (int i = 1; i < 8; ++i) s += flat[32 * i + threadIdx.x];
    store_any(a.b.db, a.b.type, c, s * alpha);
  } else if (blockIdx.x < a.b.ctas + a.j[1].ctas) {
    join(a.j[1], blockIdx.x - a.b.ctas, n, alpha, shared);
  } else {
    join(a.j[0], blockIdx.x - a.b.ctas - a.j[1].ctas, n, alpha, shared);
  }
}

// ------------------------------------------------------------------------------------------------ few rows of fp32
// Up to FEW rows bring so little arithmetic to each weight that the weights' bytes bound the call, and three parts of them in bf16 would be written once and read three times:
// fp32 sums on the ordinary units, w read as it lies, once in the forward and twice in the backward.
// NT rows at most (8 or 16).  In z a warp takes FOUR rows of w with all rows of x, which wait in shared memory in pieces of FEW_K elements: lanes along the contraction, 4 NT sums a
// lane, which one transposing sum over the lanes leaves to lane i (r NT + t).  In dx and dW a thread takes E columns and keeps x and dx of them in registers; G comes row by row.
// Forward and backward, us a call, by tiles / here (2048 to 32000: w read three times and dW written at the measured copy rate take 160): one row 620 / 268, eight 620 / 283, sixteen
// 621 / 410, which shared memory's reads of x bound, so seventeen and more stay with the tiles (32 rows 623); sixteen of 770 to 50021, in single elements, 541 / 468; two of 2656 to
// 427 131 / 86; eight of 16 to 50021 187 / 82.
constexpr int FEW = 16, FOUR = 4, FEW_ROWS = 64;
constexpr long long FEW_WEIGHTS = 1 << 16;                // below, launches take the time (a forward of 16 x 64 to 400: 16 us by tiles, 13 here) and a row alone keeps the loss it has among many
template <int NT> constexpr int FEW_K = NT == 8 ? 1280 : 512;
struct Few {
  Plan plan; int Tp, k;
  const float* x; long long ldx;
  const float* w; long long ldw;
  const float* bias2; float c1;
  int V, K;
  float2* part; int parts;                                // z: [slots, parts] largest, sum
  float* zt;
  const float* g; Coef coef;
  float* G;                                               // [V][NT]
  float* sums; float *dx, *dw;                            // [parts of V][NT][K]; results or null
  void* db; int db_type;
  int columns, groups;                                    // threads along a row of w, and rows side by side
  int per, all_parts;                                     // rows of w of a CTA; parts of dx
  int T;
};
template <int NT, int E, bool BACK> __global__ void __launch_bounds__(256, 2) k_few_z(const __grid_constant__ Few a) {
  constexpr int UNROLL = NT == 8 ? 2 : 1, VALUES = FOUR * NT / 32, TARGETS = MAX_TARGETS + 4;       // (rows of targets on different banks)
  __shared__ __align__(16) float xs[NT * FEW_K<NT>];
  __shared__ __align__(16) int targets[NT * TARGETS];
  __shared__ float2 tops[8][NT];
  next_may_start();
  wait_for_kernel_before();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane % NT;
  const int n = *reinterpret_cast<const volatile int*>(a.plan.head);
  if (n == 0) return;                                     // G is not read either
  const int k4 = (a.k + 3) / 4 * 4;
  for (int i = threadIdx.x; i < NT * k4; i += 256) {
    const int r = i / k4, j = i - r * k4;
    targets[r * TARGETS + j] = r < n && j < a.k ? a.plan.target[(long long)j * a.Tp + r] : -1;
  }
  const bool in = t < n;
  float top = -INFINITY, sum = 0.f, lse = 0.f, by = 0.f;
  if (BACK && in) {
    lse = a.plan.lse[t];
    by = a.g ? a.g[a.plan.row[t]] : 1.f;
  }
  const int pieces = (a.K + FEW_K<NT> - 1) / FEW_K<NT>, piece = ((a.K + pieces - 1) / pieces + 31) / 32 * 32;
  auto bring = [&](int k0, int len) {
    for (int r = warp; r < NT; r += 8) {
      const float* const from = r < n ? a.x + a.plan.row[r] * a.ldx + k0 : nullptr;
#pragma unroll 8
      for (int i = lane; i < len; i += 32) xs[r * piece + i] = from ? from[i] : 0.f;
    }
  };
  if (pieces == 1) bring(0, a.K);
  __syncthreads();
  for (long long v0 = blockIdx.x * 8ll * FOUR; v0 < a.V; v0 += gridDim.x * 8ll * FOUR) {
    float acc[FOUR * NT];
#pragma unroll
    for (int i = 0; i < FOUR * NT; ++i) acc[i] = 0.f;
    const float* from[FOUR];
#pragma unroll
    for (int r = 0; r < FOUR; ++r) from[r] = a.w + min(v0 + warp * FOUR + r, a.V - 1ll) * a.ldw;
    for (int k0 = 0; k0 < a.K; k0 += piece) {
      const int len = min(piece, a.K - k0);
      if (pieces > 1) {
        __syncthreads();
        bring(k0, len);
        __syncthreads();
      }
#pragma unroll UNROLL
      for (int c = lane * E; c < len; c += 32 * E) {
        float w[FOUR][E];
#pragma unroll
        for (int r = 0; r < FOUR; ++r)
          if constexpr (E == 4) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(from[r] + k0 + c));
            w[r][0] = f.x, w[r][1] = f.y, w[r][2] = f.z, w[r][3] = f.w;
          } else {
            w[r][0] = __ldcs(from[r] + k0 + c);
          }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float f[E];
          if constexpr (E == 4) {
            const float4 v = *reinterpret_cast<const float4*>(xs + i * piece + c);
            f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
          } else {
            f[0] = xs[i * piece + c];
          }
#pragma unroll
          for (int r = 0; r < FOUR; ++r)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r * NT + i] = fmaf(w[r][e], f[e], acc[r * NT + i]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < VALUES; ++h) {
      float (&mine)[32] = *reinterpret_cast<float (*)[32]>(acc + 32 * h);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; ++i) {
          const bool up = lane & o;
          const float give = up ? mine[i] : mine[i + o], keep = up ? mine[i + o] : mine[i];
          mine[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      const long long v = v0 + warp * FOUR + (32 * h + lane) / NT;
      if (v >= a.V) continue;
      float z = in ? fmaf(mine[0], a.c1, a.bias2[v]) : 0.f;
      if (BACK) z = in ? ex2(z - lse) * by : 0.f;
      if (in) {
        const int4* const list = reinterpret_cast<const int4*>(targets + t * TARGETS);
        for (int j = 0; j < a.k; j += 4) {
          const int4 four = list[j / 4];
          if (four.x != v && four.y != v && four.z != v && four.w != v) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if ((e == 0 ? four.x : e == 1 ? four.y : e == 2 ? four.z : four.w) != v) continue;
            const long long at = (long long)(j + e) * a.Tp + t;
            if (BACK) {
              const float q = a.plan.q ? a.plan.q[at] : 1.f;
              z = q == 1.f ? a.plan.less[t] * by : z - q * by;
            } else {
              a.zt[at] = z;
            }
          }
        }
      }
      if (BACK) {
        a.G[v * NT + t] = z;
      } else if (in) {
        const float m = fmaxf(top, z), least = m == -INFINITY ? 0.f : m;
        sum = sum * ex2(top - least) + ex2(z - least);
        top = m;
      }
    }
  }
  if (BACK) return;
  auto merge = [&](float m2, float s2) {
    const float m = fmaxf(top, m2), least = m == -INFINITY ? 0.f : m;
    sum = sum * ex2(top - least) + s2 * ex2(m2 - least);
    top = m;
  };
#pragma unroll
  for (int o = 16; o >= NT; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, top, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
    merge(m2, s2);
  }
  if (lane < NT) tops[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp > 0 || lane >= n) return;
  for (int i = 1; i < 8; ++i) merge(tops[i][lane].x, tops[i][lane].y);
  a.part[(long long)lane * a.parts + blockIdx.x] = make_float2(top, sum);
}
template <int NT, int E> __global__ void __launch_bounds__(256, 2) k_few_out(const __grid_constant__ Few a) {
  __shared__ __align__(16) float G[FEW_ROWS * NT], each[256 * NT * E];
  next_may_start();
  wait_for_kernel_before();
  const int n = *reinterpret_cast<const volatile int*>(a.plan.head);
  const float alpha = *reinterpret_cast<volatile int*>(&g_vocab_status) != 0 ? not_a_number() : a.coef.alpha(n);
  const int group = threadIdx.x / a.columns, c = (blockIdx.x * a.columns + threadIdx.x - group * a.columns) * E;
  const bool on = c < a.K, take = on && a.dx != nullptr && n > 0, give = on && a.dw != nullptr;
  float x[NT][E], dx[NT][E];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const float* const from = a.x + (t < n ? a.plan.row[t] : 0) * a.ldx + c;
#pragma unroll
    for (int e = 0; e < E; ++e) x[t][e] = give && t < n ? from[e] : 0.f, dx[t][e] = 0.f;
  }
  const long long begin = (long long)blockIdx.y * a.per, end = min(begin + a.per, (long long)a.V);
  for (long long v0 = begin; v0 < end; v0 += FEW_ROWS) {
    const int here = (int)min((long long)FEW_ROWS, end - v0);
    __syncthreads();
    for (int i = threadIdx.x; i < FEW_ROWS * NT; i += blockDim.x) G[i] = n > 0 && i < here * NT ? a.G[v0 * NT + i] : 0.f;
    __syncthreads();
    if (a.db != nullptr && blockIdx.x == 0)
      for (int i = threadIdx.x; i < here; i += blockDim.x) {
        float s = 0.f;
        for (int t = 0; t < NT; ++t) s += G[i * NT + t];
        store_any(a.db, a.db_type, v0 + i, s * alpha);
      }
    constexpr int U = NT == 8 ? 4 : 8;                    // 8 to 2048 x 32000: eight 292 us for 278; 16: four 446 for 421
    for (int i0 = group; i0 < here; i0 += U * a.groups) {
      float w[U][E];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * a.groups;
        const float* const from = a.w + (v0 + i) * a.ldw + c;
#pragma unroll
        for (int e = 0; e < E; ++e) w[u][e] = 0.f;
        if (!take || i >= here) continue;
        if constexpr (E == 4) {
          const float4 f = __ldcs(reinterpret_cast<const float4*>(from));
          w[u][0] = f.x, w[u][1] = f.y, w[u][2] = f.z, w[u][3] = f.w;
        } else if constexpr (E == 2) {
          const float2 f = __ldcs(reinterpret_cast<const float2*>(from));
          w[u][0] = f.x, w[u][1] = f.y;
        } else {
          w[u][0] = __ldcs(from);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * a.groups;
        if (i >= here) break;
        float f[E];
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = 0.f;
#pragma unroll
        for (int t = 0; t < NT; t += 4) {
          const float4 q = *reinterpret_cast<const float4*>(G + i * NT + t);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            dx[t][e] = fmaf(q.x, w[u][e], dx[t][e]), dx[t + 1][e] = fmaf(q.y, w[u][e], dx[t + 1][e]);
            dx[t + 2][e] = fmaf(q.z, w[u][e], dx[t + 2][e]), dx[t + 3][e] = fmaf(q.w, w[u][e], dx[t + 3][e]);
            f[e] = fmaf(q.x, x[t][e], fmaf(q.y, x[t + 1][e], fmaf(q.z, x[t + 2][e], fmaf(q.w, x[t + 3][e], f[e]))));
          }
        }
        if (!give) continue;
        float* const to = a.dw + (v0 + i) * a.K + c;
        if constexpr (E == 4) __stcs(reinterpret_cast<float4*>(to), make_float4(f[0] * alpha, f[1] * alpha, f[2] * alpha, f[3] * alpha));
        else if constexpr (E == 2) __stcs(reinterpret_cast<float2*>(to), make_float2(f[0] * alpha, f[1] * alpha));
        else __stcs(to, f[0] * alpha);
      }
    }
  }
  if (a.dx == nullptr || n == 0) return;
  // the groups' sums in their order
  const int span = a.columns * E, first = blockIdx.x * span;
  if (group < a.groups)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < E; ++e) each[(group * NT + t) * span + c - first + e] = dx[t][e];
  __syncthreads();
  for (int o = threadIdx.x; o < n * span; o += blockDim.x) {
    float s = 0.f;
    for (int g = 0; g < a.groups; ++g) s += each[g * NT * span + o];
    const int t = o / span, k = first + o - t * span;
    if (k < a.K) a.sums[((long long)blockIdx.y * NT + t) * a.K + k] = s;
  }
}
// dx: 32 columns of a row and eight shares of the parts a CTA
template <int NT> __global__ void __launch_bounds__(256) k_few_join(const __grid_constant__ Few a) {
  __shared__ float shares[8][32];
  next_may_start();
  wait_for_kernel_before();
  const int n = *reinterpret_cast<const volatile int*>(a.plan.head), lane = threadIdx.x & 31, share = threadIdx.x >> 5;
  const float alpha = *reinterpret_cast<volatile int*>(&g_vocab_status) != 0 ? not_a_number() : a.coef.alpha(n);
  const long long c = blockIdx.x * 32ll + lane;
  const int t = blockIdx.y, slot = a.plan.slot[t];
  float s = 0.f;
  if (slot >= 0 && c < a.K)
#pragma unroll 8
    for (int p = share; p < a.all_parts; p += 8) s += a.sums[((long long)p * NT + slot) * a.K + c];
  shares[share][lane] = s;
  __syncthreads();
  if (share > 0 || c >= a.K) return;
  for (int i = 1; i < 8; ++i) s += shares[i][lane];
  a.dx[(long long)t * a.K + c] = slot < 0 ? 0.f : s * alpha;
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
// boxes of 64 columns x box_rows of a matrix of 16-bit elements
int map_of(CUtensorMap* m, const void* base, long long cols, long long rows_, long long ld, int box_rows) {
  Encode encode;
  const int rc = encoder(&encode);
  if (rc != SPION_OK) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows_}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {BK, (cuuint32_t)box_rows}, step[2] = {1, 1};
  auto make = [&] {
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = make();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {                  // a thread that has used the device for nothing yet (a first backward): this makes its context current
    int dev = 0;
    SPION_CUDA_TRY(cudaGetDevice(&dev));
    SPION_CUDA_TRY(cudaSetDevice(dev));
    r = make();
  }
  if (r != CUDA_SUCCESS) {
    fprintf(stderr, "spion_b200: cuTensorMapEncodeTiled failed (%d) rows=%lld cols=%lld\n", (int)r, rows_, cols);
    return SPION_ERR_CUDA;
  }
  return SPION_OK;
}
// CTAs (or pairs) of a kernel that the current device holds at a time
template <int MODE, bool PAIR, int OPT = 0> int units_of(int* units) {
  static std::atomic<int> known[64];
  int dev = 0;
  SPION_CUDA_TRY(cudaGetDevice(&dev));
  int n = dev < 64 ? known[dev].load() : 0;
  if (n == 0) {
    SPION_CUDA_TRY(cudaFuncSetAttribute(k_gemm<MODE, PAIR, OPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<MODE, PAIR, OPT>::SMEM));
    if (PAIR) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = 2, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(2 * (sm_count() / 2)), cfg.blockDim = dim3(Shape<MODE, PAIR, OPT>::THREADS), cfg.dynamicSmemBytes = Shape<MODE, PAIR, OPT>::SMEM, cfg.attrs = at, cfg.numAttrs = 1;
      SPION_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, k_gemm<MODE, PAIR, OPT>, &cfg));
    } else {
      n = sm_count();
    }
    if (n <= 0) return SPION_ERR_UNSUPPORTED;
    if (dev < 64) known[dev].store(n);
  }
  *units = n;
  return SPION_OK;
}
template <int MODE, bool PAIR, int OPT> int launch_gemm(const Call<MODE>& call, long long most_items, cudaStream_t st) {
  int units;
  const int rc = units_of<MODE, PAIR, OPT>(&units);
  if (rc != SPION_OK) return rc;
  // dx splits its contraction by the number of units: it always has all of them
  const int use = MODE == GRADS ? units : (int)std::min<long long>(units, std::max<long long>(most_items, 1));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(PAIR ? 2 * use : use), cfg.blockDim = dim3(Shape<MODE, PAIR, OPT>::THREADS), cfg.dynamicSmemBytes = Shape<MODE, PAIR, OPT>::SMEM, cfg.stream = st, cfg.attrs = at, cfg.numAttrs = PAIR ? 2 : 1;
  SPION_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_gemm<MODE, PAIR, OPT>, call));
  return SPION_OK;
}
template <int MODE, int OPT> int launch_gemm(bool pair, const Call<MODE>& call, long long most_items, cudaStream_t st) {
  return pair ? launch_gemm<MODE, true, OPT>(call, most_items, st) : launch_gemm<MODE, false, OPT>(call, most_items, st);
}
int launch_logsum(bool pair, const Call<LOGSUM>& call, long long most_items, cudaStream_t st) {
  if (call.a[0].bn)
    return call.a[0].k == 1 ? launch_gemm<LOGSUM, false, ONE | WIDE>(call, most_items, st) : launch_gemm<LOGSUM, false, WIDE>(call, most_items, st);
  return call.a[0].k == 1 ? launch_gemm<LOGSUM, ONE>(pair, call, most_items, st) : launch_gemm<LOGSUM, 0>(pair, call, most_items, st);
}
int launch_grad(bool pair, bool two, const Call<GRAD>& call, long long most_items, cudaStream_t st) {
  const Args& a = call.a[0];
  if (two) switch ((a.k == 1 ? ONE : 0) | (a.colsum != nullptr ? COLUMNS : 0)) {
    case 0: return launch_gemm<GRAD, false, TWO>(call, most_items, st);
    case ONE: return launch_gemm<GRAD, false, TWO | ONE>(call, most_items, st);
    case COLUMNS: return launch_gemm<GRAD, false, TWO | COLUMNS>(call, most_items, st);
    default: return launch_gemm<GRAD, false, TWO | ONE | COLUMNS>(call, most_items, st);
  }
  switch ((a.k == 1 ? ONE : 0) | (a.products > 1 ? THREE : 0) | (a.colsum != nullptr ? COLUMNS : 0)) {
    case 0: return launch_gemm<GRAD, 0>(pair, call, most_items, st);
    case 1: return launch_gemm<GRAD, 1>(pair, call, most_items, st);
    case 2: return launch_gemm<GRAD, 2>(pair, call, most_items, st);
    case 3: return launch_gemm<GRAD, 3>(pair, call, most_items, st);
    case 4: return launch_gemm<GRAD, 4>(pair, call, most_items, st);
    case 5: return launch_gemm<GRAD, 5>(pair, call, most_items, st);
    case 6: return launch_gemm<GRAD, 6>(pair, call, most_items, st);
    default: return launch_gemm<GRAD, 7>(pair, call, most_items, st);
  }
}
constexpr long long up(long long x, long long to) { return (x + to - 1) / to * to; }
constexpr long long tiles_of(long long x, long long tile) { return (x + tile - 1) / tile; }
// (chunk, product) pairs, of four steps each, that one accumulator takes; a multiple of the products.  fp32: two chunks, whose ten small products go first: 8 steps of 48 count (one after another,
// 16 pairs, 64 steps: dW of 45754 x 1829 to 29 1.4e-6 of the norm off, so 0.25e-6, and the plain form 0.67e-6; 19652 x 320 to 35829 forward and backward 11.7 ms, with one chunk 12.6, with 16 pairs 11.4).  16 bits: z in small tiles 16
// steps (3012 x 2464 to 2 in fp16, a small loss: 1.7e-6 of it off, so 0.5e-6, at the same time); in tiles of pairs 64, which keep the multiplying warp busy while the others form exponentials (32 steps: 8192 x
// 2048 to 32000 4 % slower, 16 steps 20 %).  dx and dW that are rounded to 16 bits: 256 steps, 2^-15 of the sum at worst, a sixteenth of fp16's half step.
int chain_of(int planes, bool pair, bool rounded) { return planes == 3 ? 12 : rounded ? 64 : pair ? 16 : 4; }

// Sizes and places of a call
struct Layout {
  long long T, Tp, K, Kp, V, Vp, k, ldw, parts;           // parts: partial sums of a row
  int planes, gparts;                                     // parts of the operands; of G
  bool copy_w, direct;                                    // w has to be copied; x can be read as it lies
  int few, few_vector, few_columns, few_groups, few_chunks, few_parts, few_per;      // rows of fp32 that k_few_* take, 8 or 16 (0: none), and their grid
  bool kept;                                              // the operands' copies stay for the backward (in the backward: and serve it)
  int given;                                              // how the forward read its operands, as problems carry it
  bool self;                                              // CTAs count for themselves
  long long rows, launches;                               // slots of a pass over z in the forward, and how many there are
  long long chunk;                                        // rows of a CTA of k_prepare
  int wide;                                               // columns of a wide tile of the forward's z, or 0
  bool pair_z, pair_g;                                    // tiles of pairs of CTAs: in z; in dx and dW
  long long Gp;                                           // columns of a piece of the vocabulary
  int tile_g, dw_splits;
  size_t keep;                                            // bytes of the plan
  size_t xs, w, bias2;                                    // in the plan (kept) or in both workspaces
  size_t part, zt, cta_loss, counts, q, forward;
  size_t g, dxp, dwp, colsum, unit, backward;
};
constexpr long long FEW_ROWS_G = 64, LITTLE_G = 1 << 23, LITTLE_WORK = 1 << 28;       // rows, logits and products whose G has two parts
constexpr long long PIECE_BYTES = 512ll << 20;              // of G: half of it costs 16384 x 1024 to 50021, 2458 rows that count, 1240 us -> 1430, and 8192 x 4096 to 128000 nothing
constexpr long long KEPT_BYTES = 64ll << 20;              // of copies that stay: small beside the device, and making them again costs launches and, for small calls, most of the time
constexpr long long PART_BYTES = 256ll << 20;             // of the partial sums of a pass over z: a sixteenth of 16-bit logits, where there are no more than these
constexpr int FINISH_CTAS = 1024;
// How a forward read its operands: with this alone the backward knows what `keep` holds, wherever its own operands lie (tensors saved for a backward may come back as copies)
enum : int { KNOWN = 1, COPIED_W = 2, DIRECT_X = 4 };

int layout_of(const spion_vocab_problem* p, Layout* l) {
  if (p == nullptr || p->layout < 0 || p->layout > (KNOWN | COPIED_W | DIRECT_X) || (p->layout != 0 && !(p->layout & KNOWN)) || p->T < 0 || p->K <= 0 || p->V <= 0 || p->k <= 0) return SPION_ERR_ARG;
  if (p->type != SPION_F32 && p->type != SPION_BF16 && p->type != SPION_F16) return SPION_ERR_ARG;
  if (p->k > MAX_TARGETS) return SPION_ERR_UNSUPPORTED;
  if (!(p->temperature > 0.f) || !(p->temperature < INFINITY) || p->ldx < 0 || p->ldw < p->K) return SPION_ERR_ARG;
  if (p->reduction < 0 || p->reduction > 2) return SPION_ERR_ARG;
  *l = Layout();
  l->T = p->T, l->K = p->K, l->V = p->V, l->k = p->k;
  l->Tp = up(std::max(p->T, 1ll), PAD), l->Kp = up(p->K, BK), l->Vp = up(p->V, PAD);
  l->planes = p->type == SPION_F32 ? 3 : 1;
  // places are 32-bit numbers in the tensor maps' coordinates and in the lists of rows
  if (p->T > 0x7fffffff / 4 || p->V > 0x7fffffff / 4 || p->K > 0x7fffffff / 4 || l->Tp * l->planes > 0x7fffffff || l->Vp * l->planes > 0x7fffffff) return SPION_ERR_SHAPE;
  l->few = p->type == SPION_F32 && p->T <= FEW && p->V * p->K >= FEW_WEIGHTS ? p->T <= 8 ? 8 : 16 : 0;
  l->copy_w = !l->few && (p->type == SPION_F32 || ((uintptr_t)p->w % 16) != 0 || (p->ldw * 2) % 16 != 0);
  l->direct = p->type != SPION_F32 && ((uintptr_t)p->x % 16) == 0 && (p->ldx * 2) % 16 == 0 && p->ldx >= p->K;
  l->given = p->layout ? p->layout : KNOWN | (l->copy_w ? COPIED_W : 0) | (l->direct ? DIRECT_X : 0);
  const bool copied_w = l->given & COPIED_W, direct_x = l->given & DIRECT_X;
  if (p->type == SPION_F32 && (direct_x || copied_w == (l->few != 0))) return SPION_ERR_ARG;
  l->self = p->T * p->k <= SELF;
  // every CTA reads the counts of all chunks: 4096 of them at most
  l->chunk = p->T <= 16384 ? 32 : std::max<long long>(BLOCK, up((p->T + 4095) / 4096, BLOCK));
  int sms = sm_count();
  if (sms <= 0) return SPION_ERR_CUDA;
  const int pairs = sms / 2;
  // Tiles of pairs where every pair has one, else four times as many small ones.
  auto tiles = [](long long m, long long n) { return m > 128 && n > 128 ? tiles_of(m, 256) * tiles_of(n, 256) : 0; };
  l->pair_z = tiles(l->T, l->V) >= pairs;
  // Wide tiles for few rows, where they keep fifteen of sixteen multiprocessors: as few rounds of them as can be, of one size.  One row of 1024, wide / tiles of 128: to 19200 (120 tiles
  // of 160) 18.1 us / 15.6, 32000 (143 of 224) 20.5 / 21.8, 37888 (148 of 256) 19.8 / 23.3, 50000 (261 of 192) 35.6 / 33.0, 128000 (572 of 224) 62.8 / 71.8; 128 rows: 12.7 / 13.2 to
  // 32000, 50.7 / 50.0 to 128000.
  const long long rounds = tiles_of(l->V, 256ll * sms), columns = up(tiles_of(l->V, sms * rounds), 32);
  l->wide = !l->few && l->T <= 64 && columns > 128 && 16 * tiles_of(l->V, columns) >= 15 * rounds * sms ? (int)columns : 0;
  l->parts = l->wide ? 4 * tiles_of(l->V, l->wide) : l->pair_z ? 4 * tiles_of(l->V, 256) : 2 * tiles_of(l->V, 128);
  l->rows = std::min(l->Tp, std::max<long long>(PAD, PART_BYTES / (8 * l->parts) / PAD * PAD));
  l->launches = tiles_of(l->Tp, l->rows);
  // G beside 16-bit operands: a row's gradient hangs on its target's entry, mostly, whose rounding is then the whole row's, up to twice that of the results; in the mean of many rows both are alike,
  // of few rows it is as it comes (one row of 1304 to 4 in fp16: 3.3e-4 of the norm off, in fp32 products 2.1e-4; 2 rows of 32 to 9704 in bf16 3.7e-3, 2.2e-3).  So few rows, and calls
  // of little work, where launches take the time, have G in two parts.  us forward and backward, one part / two: 16 x 2048 to 32000 195 / 215, 64 x 1024 to 50000 175 / 203, 64 x 2048 to 32000 185 / 205;
  // 2000 x 128 to 1000 89 / 87, 8192 x 32 to 1000 92 / 91, 71 x 2 to 63111 97 / 99; 128 x 4096 to 128000, which keeps one, 1190 / 1390.
  l->gparts = l->planes == 3 ? 3 : !l->pair_z && ((l->T <= FEW_ROWS_G && 2 * l->T <= l->K) || (l->T * l->V <= LITTLE_G && l->T * l->V * l->K <= LITTLE_WORK)) ? 2 : 1;
  l->Gp = std::min(l->Vp, std::max<long long>(PAD, PIECE_BYTES / (2 * l->gparts * l->Tp) / PAD * PAD));
  l->Gp = up(tiles_of(l->Vp, tiles_of(l->Vp, l->Gp)), PAD);               // pieces of one size
  l->pair_g = tiles(l->T, l->K) > 0 && tiles(l->T, l->K) + tiles(l->Gp, l->K) >= pairs;
  l->tile_g = l->pair_g ? 256 : 128;
  // tiles are counted in 32 bits, eight parts of dx's contraction among them
  if (tiles_of(l->T, 128) * tiles_of(l->V, 128) > 0x7fffffff || (8 * tiles_of(l->T, 128) + 2 * tiles_of(l->Gp, 128)) * tiles_of(l->K, 128) > 0x7fffffff) return SPION_ERR_SHAPE;
  l->dw_splits = split_by_units((int)std::min<long long>(tiles_of(l->Gp, l->tile_g) * tiles_of(l->K, l->tile_g), 1 << 20), l->pair_g ? pairs : sms, (int)tiles_of(l->T, BK));
  size_t at = 0;
  auto take = [&](long long bytes) {
    const size_t here = at;
    at += (size_t)up(std::max(bytes, 0ll), 256);
    return here;
  };
  if (l->few) {
    l->parts = std::min<long long>(tiles_of(l->V, 8 * FOUR), 2 * sms);
    l->rows = l->Tp, l->launches = 1;
    l->few_vector = l->K % 4 == 0 && (uintptr_t)p->w % 16 == 0 && p->ldw % 4 == 0;
    const long long along = tiles_of(l->K, l->few_vector ? 32 / l->few : 1);
    l->few_chunks = (int)tiles_of(along, 256);
    l->few_columns = (int)tiles_of(along, l->few_chunks);
    l->few_groups = 256 / l->few_columns;
    l->few_per = (int)up(tiles_of(l->V, std::max<long long>(1, 2 * sms / l->few_chunks)), 16);
    l->few_parts = (int)tiles_of(l->V, l->few_per);
  }
  const long long xs_bytes = l->few ? 0 : 2 * l->planes * l->Tp * l->Kp, ws_bytes = 2 * l->planes * l->Vp * l->Kp;
  l->kept = xs_bytes + (copied_w ? ws_bytes : 0) + 4 * (l->Vp + PAD) <= KEPT_BYTES;
  take(256), take(4 * l->Tp), take(4 * l->Tp), take(4 * l->Tp), take(4 * l->Tp), take(4 * l->k * l->Tp), take(4 * l->k * l->Tp);
  auto operands = [&](bool copy) { l->xs = take(xs_bytes), l->w = take(copy ? ws_bytes : 0), l->bias2 = take(4 * (l->Vp + PAD)); };
  if (l->kept) operands(copied_w);
  l->keep = at;
  // What the forward kept serves where the operands that it read in place can be read in place again (x: if all rows count; a copy of x is kept if not).  Else both are made anew.
  l->kept = l->kept && (copied_w || !l->copy_w) && (!direct_x || l->direct);
  if (l->kept) l->copy_w = copied_w, l->direct = direct_x;
  l->ldw = l->copy_w ? l->Kp : p->ldw;
  at = 0;
  if (!l->kept) operands(l->copy_w);
  const size_t both = at;
  l->part = take(8 * l->rows * l->parts);
  l->zt = take(4 * l->k * l->Tp);
  l->cta_loss = take(8 * FINISH_CTAS * l->launches);
  l->counts = take(4 * tiles_of(l->T, l->chunk));
  l->q = take(4 * l->T * l->k);
  l->forward = at;
  at = both;
  if (l->few) {
    l->g = take(4 * l->few * l->V);
    l->dxp = take(4ll * l->few_parts * l->few * l->K);
    l->backward = at;
    return SPION_OK;
  }
  l->g = take(2 * l->gparts * l->Tp * l->Gp);
  // (as Parts cuts them: one part, or eight rounds of tiles at most, in so many parts)
  const long long tile = l->tile_g, tn = tiles_of(l->K, tile), most_m = 8 * (l->pair_g ? pairs : sms) / tn;
  l->dxp = take(4 * std::max(tiles_of(l->T, tile), std::min(most_m, (l->gparts == 2 ? 32 : 8) * tiles_of(l->T, tile))) * tile * l->Kp);
  l->dwp = take(l->dw_splits > 1 ? 4 * l->dw_splits * up(l->Gp, l->tile_g) * l->Kp : 0);
  l->colsum = take(4 * (l->Tp / 32) * l->Gp);
  l->unit = take(256);
  l->backward = at;
  return SPION_OK;
}
Plan plan_at(const Layout& l, void* keep, bool teacher) {
  char* c = static_cast<char*>(keep);
  Plan p;
  p.head = (int*)c, c += 256;
  const size_t rows_ = (size_t)up(4 * l.Tp, 256), targets = (size_t)up(4 * l.k * l.Tp, 256);
  p.slot = (int*)c, c += rows_;
  p.row = (int*)c, c += rows_;
  p.lse = (float*)c, c += rows_;
  p.less = (float*)c, c += rows_;
  p.target = (int*)c, c += targets;
  p.q = teacher ? (float*)c : nullptr;
  return p;
}
Source source_of(const void* p, int type, long long ld, long long K, long long Kp) {
  const int size = type_size(type);
  auto on = [&](int bytes) { return (uintptr_t)p % bytes == 0 && ld * size % bytes == 0; };
  return {p, type, ld, (int)K, (int)Kp, K % 8 == 0 && on(16) ? 2 : K % 2 == 0 && on(2 * size) ? 1 : 0};
}
Prep prep_of(const spion_vocab_problem* p, const Layout& l, void* keep, char* ws) {
  Prep a = {};
  a.plan = plan_at(l, keep, p->teacher != nullptr);
  a.labels = p->labels, a.teacher = p->teacher, a.teacher_type = p->teacher_type, a.ignore = p->ignore_index;
  a.inv_tau = 1.f / p->temperature;
  a.T = (int)l.T, a.Tp = (int)l.Tp, a.V = (int)l.V, a.k = (int)l.k, a.Vp = (int)l.Vp;
  a.c1 = (float)(1.4426950408889634 / (double)p->temperature);
  char* const operands = l.kept ? static_cast<char*>(keep) : ws;
  a.bias = p->bias, a.bias_type = p->bias_type, a.bias2 = (float*)(operands + l.bias2);
  a.x = source_of(p->x, p->type, p->ldx, l.K, l.Kp), a.w = source_of(p->w, p->type, p->ldw, l.K, l.Kp);
  a.xs = (uint16_t*)(operands + l.xs), a.ws = l.copy_w ? (uint16_t*)(operands + l.w) : nullptr;
  a.direct = l.direct, a.few = l.few;
  const long long chunks = tiles_of(l.T, l.chunk);
  a.chunk = (int)l.chunk;
  // slices of 64 elements of a row at least, where there are too few chunks to fill the device twice
  a.slices = l.few ? 1 : (unsigned)std::max<long long>(1, std::min<long long>(l.Kp / 64, 2 * sm_count() / chunks));
  a.row_ctas = (unsigned)chunks * a.slices;
  a.w_ctas = l.copy_w ? (unsigned)std::min<long long>(tiles_of(l.Vp, 8), 8 * sm_count()) : 0;
  return a;
}
template <bool FIRST> int launch_prepare(const spion_vocab_problem* p, const Prep& a, cudaStream_t st) {
  const dim3 grid(a.row_ctas + a.w_ctas + (unsigned)std::min<long long>(tiles_of(a.Vp, 256), 2 * sm_count()));
  if (p->type == SPION_F32) SPION_CUDA_TRY(launch_after(k_prepare<Eight32, FIRST>, grid, dim3(256), 0, st, a));
  else SPION_CUDA_TRY(launch_after(k_prepare<Eight16, FIRST>, grid, dim3(256), 0, st, a));
  return SPION_OK;
}
// What the two passes over z have in common
int logits_args(const spion_vocab_problem* p, const Layout& l, const Prep& prep, Args* a, Maps* maps) {
  *a = Args();
  a->on = 1;
  a->n = prep.plan.head;
  a->products = l.planes == 1 ? 1 : 6;
  a->plane_a = l.Tp, a->plane_b = l.Vp;
  a->L = (int)l.K;
  a->chain = chain_of(l.planes, l.pair_z, false);
  a->splits = 1;
  a->fp16 = p->type == SPION_F16;
  a->direct_rows = l.direct ? (int)l.T : 0;
  a->plan = prep.plan, a->Tp = (int)l.Tp, a->k = (int)l.k;
  a->bias2 = prep.bias2, a->c1 = prep.c1;
  int rc = map_of(&maps->a, prep.xs, l.Kp, l.planes * l.Tp, l.Kp, 128);
  if (rc == SPION_OK)
    rc = l.copy_w ? map_of(&maps->b, prep.ws, l.Kp, l.planes * l.Vp, l.Kp, 128) : map_of(&maps->b, p->w, l.K, l.V, l.ldw, 128);
  maps->x = maps->a;
  if (rc == SPION_OK && l.direct) rc = map_of(&maps->x, p->x, l.K, l.T, p->ldx, 128);
  return rc;
}

Few few_of(const spion_vocab_problem* p, const Layout& l, const Prep& prep) {
  Few f = {};
  f.plan = prep.plan, f.Tp = (int)l.Tp, f.k = (int)l.k, f.T = (int)l.T;
  f.x = static_cast<const float*>(p->x), f.ldx = p->ldx, f.w = static_cast<const float*>(p->w), f.ldw = p->ldw;
  f.bias2 = prep.bias2, f.c1 = prep.c1, f.V = (int)l.V, f.K = (int)l.K;
  f.parts = (int)l.parts, f.zt = prep.zt;
  f.columns = l.few_columns, f.groups = l.few_groups, f.per = l.few_per, f.all_parts = l.few_parts;
  return f;
}
template <bool BACK> int few_z(const Layout& l, const Few& f, cudaStream_t st) {
  const dim3 grid((unsigned)l.parts);
  if (l.few == 8) SPION_CUDA_TRY(launch_after(l.few_vector ? k_few_z<8, 4, BACK> : k_few_z<8, 1, BACK>, grid, dim3(256), 0, st, f));
  else SPION_CUDA_TRY(launch_after(l.few_vector ? k_few_z<16, 4, BACK> : k_few_z<16, 1, BACK>, grid, dim3(256), 0, st, f));
  return SPION_OK;
}
int few_backward(const Layout& l, const Few& f, cudaStream_t st) {
  const int rc = few_z<true>(l, f, st);
  if (rc != SPION_OK) return rc;
  const dim3 grid(l.few_chunks, l.few_parts), block(l.few_columns * l.few_groups), join((unsigned)tiles_of(l.K, 32), (unsigned)l.T);
  if (l.few == 8) SPION_CUDA_TRY(launch_after(l.few_vector ? k_few_out<8, 4> : k_few_out<8, 1>, grid, block, 0, st, f));
  else SPION_CUDA_TRY(launch_after(l.few_vector ? k_few_out<16, 2> : k_few_out<16, 1>, grid, block, 0, st, f));
  if (f.dx != nullptr) SPION_CUDA_TRY(launch_after(l.few == 8 ? k_few_join<8> : k_few_join<16>, join, dim3(256), 0, st, f));
  return SPION_OK;
}

int check_problem(const spion_vocab_problem* p, const void* keep, const void* workspace) {
  if (p->x == nullptr || p->w == nullptr || p->labels == nullptr || keep == nullptr || workspace == nullptr) return SPION_ERR_ARG;
  if (p->teacher != nullptr && p->teacher_type != SPION_F32 && p->teacher_type != SPION_BF16 && p->teacher_type != SPION_F16) return SPION_ERR_ARG;
  if (p->teacher == nullptr && p->k != 1) return SPION_ERR_ARG;
  if (p->bias != nullptr && p->bias_type != SPION_F32 && p->bias_type != SPION_BF16 && p->bias_type != SPION_F16) return SPION_ERR_ARG;
  if (((uintptr_t)keep | (uintptr_t)workspace) % 256 != 0) return SPION_ERR_ARG;
  return SPION_OK;
}

}  // namespace

int* vocab_status_word() {
  static StatusWord word;
  return word.on_this_device(g_vocab_status);
}

extern "C" int spion_vocab_layout(const spion_vocab_problem* p) {
  Layout l;
  spion_vocab_problem forward;
  if (p != nullptr) forward = *p, forward.layout = 0;
  const int rc = layout_of(p != nullptr ? &forward : nullptr, &l);
  return rc == SPION_OK ? l.given : rc;
}

extern "C" int spion_vocab_sizes(const spion_vocab_problem* p, long long* keep_bytes, long long* forward_bytes, long long* backward_bytes) {
  Layout l;
  const int rc = layout_of(p, &l);
  if (rc != SPION_OK) return rc;
  if (keep_bytes) *keep_bytes = (long long)l.keep;
  if (forward_bytes) *forward_bytes = (long long)l.forward;
  if (backward_bytes) *backward_bytes = (long long)l.backward;
  return SPION_OK;
}

extern "C" int spion_vocab_loss_forward(const spion_vocab_problem* problem, float* loss, void* keep, void* workspace, void* cuda_stream) {
  Layout l;
  spion_vocab_problem own;                                 // with a layout of its own
  if (problem != nullptr) own = *problem, own.layout = 0;
  const spion_vocab_problem* const p = problem != nullptr ? &own : nullptr;
  int rc = layout_of(p, &l);
  if (rc != SPION_OK) return rc;
  if (l.T == 0) return p->reduction == 0 ? SPION_OK : SPION_ERR_ARG;      // nothing to take a mean of
  if ((rc = check_problem(p, keep, workspace)) != SPION_OK) return rc;
  if (loss == nullptr) return SPION_ERR_ARG;
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  char* const ws = static_cast<char*>(workspace);
  Prep prep = prep_of(p, l, keep, ws);
  prep.counts = l.self ? nullptr : (int*)(ws + l.counts), prep.q = (float*)(ws + l.q), prep.zt = (float*)(ws + l.zt);
  prep.loss_rows = p->reduction == 0 ? loss : nullptr;
  if (!l.self) SPION_CUDA_TRY(launch_after(k_flags, dim3((unsigned)tiles_of(tiles_of(l.T, l.chunk), prep.teacher ? 1 : 8)), dim3(256), 0, st, prep));
  if ((rc = launch_prepare<true>(p, prep, st)) != SPION_OK) return rc;
  Call<LOGSUM> call;
  Args& a = call.a[0];
  Few few;
  if (l.few) few = few_of(p, l, prep), few.part = (float2*)(ws + l.part);
  if (!l.few && (rc = logits_args(p, l, prep, &a, &call.maps[0])) != SPION_OK) return rc;
  const int tile = l.pair_z ? 256 : 128;
  if (l.wide) {
    a.bn = l.wide;
    if ((rc = l.copy_w ? map_of(&call.maps[0].b, prep.ws, l.Kp, l.planes * l.Vp, l.Kp, l.wide) : map_of(&call.maps[0].b, p->w, l.K, l.V, l.ldw, l.wide)) != SPION_OK) return rc;
  }
  a.N = (int)l.V, a.part = (float2*)(ws + l.part), a.parts = (int)l.parts, a.zt = prep.zt;
  const int lanes = std::max<int>(a.parts, l.k) <= 16 ? 4 : std::max<int>(a.parts, l.k) <= 32 ? 8 : 32;
  const dim3 grid((unsigned)std::min<long long>(tiles_of(std::min(l.T, l.rows), 256 / lanes), std::min(4 * sm_count(), FINISH_CTAS)));
  for (int pass = 0; pass < l.launches; ++pass) {
    a.row0 = (int)(pass * l.rows), a.most = (int)l.rows;
    if ((rc = l.few ? few_z<false>(l, few, st) : launch_logsum(l.pair_z, call, tiles_of(std::min(l.T, l.rows), tile) * tiles_of(l.V, l.wide ? l.wide : tile), st)) != SPION_OK) return rc;
    const Finish f = {prep.plan, (int)l.Tp, (int)l.k, a.part, a.parts, prep.zt, loss, (double*)(ws + l.cta_loss), p->reduction, a.row0, a.most, pass, (int)l.launches};
    if (lanes == 4) SPION_CUDA_TRY(launch_after(k_finish<4>, grid, dim3(256), 0, st, f));
    else if (lanes == 8) SPION_CUDA_TRY(launch_after(k_finish<8>, grid, dim3(256), 0, st, f));
    else SPION_CUDA_TRY(launch_after(k_finish<32>, grid, dim3(256), 0, st, f));
  }
  return SPION_OK;
}

extern "C" int spion_vocab_loss_backward(const spion_vocab_problem* p, const float* g, const void* keep, void* dx, void* dw, void* db, int db_type, void* workspace,
                                         void* cuda_stream) {
  Layout l;
  int rc = layout_of(p, &l);
  if (rc != SPION_OK) return rc;
  if (l.T == 0) return SPION_ERR_ARG;
  if ((rc = check_problem(p, keep, workspace)) != SPION_OK) return rc;
  if (g == nullptr || (dx == nullptr && dw == nullptr && db == nullptr)) return SPION_ERR_ARG;
  if (db != nullptr && db_type != SPION_F32 && db_type != SPION_BF16 && db_type != SPION_F16) return SPION_ERR_ARG;
  if (((uintptr_t)dx | (uintptr_t)dw) % 32 != 0) return SPION_ERR_ARG;
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  char* const ws = static_cast<char*>(workspace);
  const Prep prep = prep_of(p, l, const_cast<void*>(keep), ws);
  uint16_t* const G = (uint16_t*)(ws + l.g);
  float* const unit = (float*)(ws + l.unit);
  const float gscale = p->type == SPION_F16 ? 8192.f : 1.f;
  const bool by_unit = p->reduction == 0 && p->type == SPION_F16;
  if (by_unit) SPION_CUDA_TRY(launch_after(k_unit, dim3(1), dim3(1024), 0, st, prep.plan, g, unit));
  if (!l.kept && (rc = launch_prepare<false>(p, prep, st)) != SPION_OK) return rc;
  const Coef coef = {p->reduction == 0 ? nullptr : g, by_unit ? unit : nullptr, p->reduction == 1, prep.inv_tau / gscale};
  if (l.few) {
    Few few = few_of(p, l, prep);
    few.g = p->reduction == 0 ? g : nullptr, few.coef = coef;
    few.G = (float*)(ws + l.g), few.sums = (float*)(ws + l.dxp), few.dx = static_cast<float*>(dx), few.dw = static_cast<float*>(dw), few.db = db, few.db_type = db_type;
    return few_backward(l, few, st);
  }
  Call<GRAD> grad;
  Call<GRADS> grads;
  Args& z = grad.a[0];
  Maps &xm = grads.maps[DX], &wm = grads.maps[DW];
  if ((rc = logits_args(p, l, prep, &z, &grad.maps[0])) != SPION_OK) return rc;
  if ((rc = map_of(&xm.a, G, l.Gp, l.gparts * l.Tp, l.Gp, 128)) != SPION_OK) return rc;
  if ((rc = l.copy_w ? map_of(&xm.b, prep.ws, l.Kp, l.planes * l.Vp, l.Kp, 64) : map_of(&xm.b, p->w, l.K, l.V, l.ldw, 64)) != SPION_OK) return rc;
  xm.x = xm.a;
  if ((rc = map_of(&wm.a, G, l.Gp, l.gparts * l.Tp, l.Gp, 64)) != SPION_OK) return rc;
  if ((rc = map_of(&wm.b, prep.xs, l.Kp, l.planes * l.Tp, l.Kp, 64)) != SPION_OK) return rc;
  wm.x = wm.b;
  if (l.direct && (rc = map_of(&wm.x, p->x, l.K, l.T, p->ldx, 64)) != SPION_OK) return rc;
  int dx_units = 0;
  if ((rc = l.pair_g ? units_of<GRADS, true>(&dx_units) : units_of<GRADS, false>(&dx_units)) != SPION_OK) return rc;
  const int tz = l.pair_z ? 256 : 128, tg = l.tile_g;
  z.g = p->reduction == 0 ? g : nullptr, z.G = G, z.ldg = l.Gp, z.gscale = gscale;
  z.coef = coef;
  z.colsum = db != nullptr ? (float*)(ws + l.colsum) : nullptr;
  const int dx_chunks = (int)tiles_of(std::min(l.Gp, l.V), BK);            // every piece's contraction is cut as the first one's: the parts are added piece by piece
  const unsigned most = 8 * sm_count();
  for (long long c = 0; c < l.V; c += l.Gp) {
    const long long columns = std::min(l.Gp, l.V - c), padded = up(columns, PAD);
    z.col0 = (int)c, z.N = (int)padded;
    if ((rc = launch_grad(l.pair_z, l.gparts == 2, grad, tiles_of(l.T, tz) * tiles_of(padded, tz), st)) != SPION_OK) return rc;
    Args b = z;
    b.chain = chain_of(l.planes, l.pair_g, true), b.products = l.gparts == 2 ? 2 : z.products;
    Leave out = {};
    out.head = prep.plan.head, out.coef = z.coef;
    Args &d = grads.a[DX], &e = grads.a[DW];
    d = e = b;
    d.on = dx != nullptr, e.on = dw != nullptr;
    const bool together = dx != nullptr && dw != nullptr;
    d.N = (int)l.K, d.L = (int)columns, d.splits = 0;
    d.cut = {dx_units, dx_chunks, together ? (int)(tiles_of(up(std::min(l.Gp, l.V), PAD), tg) * tiles_of(l.K, tg) * l.dw_splits) : 0, l.dw_splits, l.gparts == 2 ? 32 : 8};
    d.plane_a = l.Tp, d.plane_b = l.Vp;
    d.out = (float*)(ws + l.dxp), d.ldo = l.Kp, d.add = c > 0;
    e.M = (int)padded, e.N = (int)l.K, e.L = 0, e.splits = l.dw_splits;
    e.plane_a = l.Tp, e.plane_b = l.Tp;
    e.out = (float*)(ws + l.dwp), e.ldo = l.Kp, e.add = 0;
    e.dw = l.dw_splits == 1 ? dw : nullptr, e.dw_type = p->type, e.K = l.K, e.V = (int)l.V;
    if ((dx != nullptr || dw != nullptr) && (rc = launch_gemm<GRADS, 0>(l.pair_g, grads, 0, st)) != SPION_OK) return rc;
    if (dx != nullptr && c + l.Gp >= l.V)
      out.j[0] = {prep.plan.slot, d.out, l.Kp, 0, tg, (int)tiles_of(l.K, tg), d.cut, 0, dx, p->type, l.T, l.K,
                  (unsigned)std::min<long long>(tiles_of(l.T * tiles_of(l.K, 8), 256), most)};
    if (dw != nullptr && l.dw_splits > 1)
      out.j[1] = {nullptr, e.out, l.Kp, l.dw_splits, tg, 0, {}, up(padded, tg), static_cast<char*>(dw) + c * l.K * type_size(p->type), p->type, columns, l.K,
                  (unsigned)std::min<long long>(tiles_of(columns * tiles_of(l.K, 8), l.dw_splits >= 8 ? 32 : 256), most)};
    if (db != nullptr) out.b = {z.colsum, l.Gp, (int)columns, static_cast<char*>(db) + c * type_size(db_type), db_type, l.T > 16384 ? 8 : 32,
                                 (unsigned)tiles_of(columns, l.T > 16384 ? 8 : 32)};
    const unsigned ctas = out.j[0].ctas + out.j[1].ctas + out.b.ctas;
    if (ctas > 0) SPION_CUDA_TRY(launch_after(k_out, dim3(ctas), dim3(256), 0, st, out));
  }
  return SPION_OK;
}
