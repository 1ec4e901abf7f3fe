// Softmax cross entropy over the kinds of a table (cgtp_kind_loss_forward, cgtp_kind_loss_backward), without keeping the logits:
//
//   z = scale x W^T  (cap: cap tanh(scale x W^T / cap)),   loss_i = log sum_k exp z_ik - z_i,y(i)
//   dz = g_i (softmax(z)_ik - [k = y(i)]) scale (1 - tanh^2),   dx = dz W,   dW = dz^T x
//
// Rows with a kind are taken together first (the others cost nothing and are not read, whatever they hold): their numbers in
// order, and a copy of them with rows of whole aligned chunks.  The forward forms the logits tile by tile and keeps a running
// maximum and sum for each row; the kinds are cut into `splits` ranges where there are few rows, whose statistics are joined in order.
// The backward forms the logits again, a piece of the kinds at a time (of rows and kinds up to 512 MB): (p - [k = y]) (1 - tanh^2) is rounded
// to the operands' type as the operand of the two products it enters.  g_i multiplies dx afterwards; for dW it multiplies the rows of x,
// divided by the largest |g| (exact where all are equal).  In fp16 the probabilities are scaled by 2^15 into its range.
//
// Bound by the matrix cores: 2 N K C operations forward, 6 N K C backward, where a calculation that kept all logits would do 4.
// 16384 rows, 30011 kinds, 256 bf16 channels: statistics 250-290 us (870-1000 TFLOP/s), logits again and dx 500-580 (870-1000), the
// table's gradient 320 (785), joins and copies of rows 75; 4253 rows with a kind, 50021 kinds, 500 fp16 channels, capped: 255-290 us (730-830).
// Small calls: the launches.  Forward the rows' copy and the statistics, with more than 64 rows their count before, with rows that are no whole aligned
// chunks the table's copy, with more than one range of kinds a join: two to five; backward up to eight.
#include "gff_gemm.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace cgtp {
namespace {

constexpr int kTile = 128, kRowBlocks = 1024, kRowThreads = 256;
// Tiles of the products of both operands from LDS: in fp32 small ones keep more of the GPU busy where there are few (9000 rows, 100 kinds, 128 channels:
// statistics 17 us with tiles of 128, 12 with these, the logits' gradients 18 and 11).  Tables of thousands of kinds, where fp32 runs at 70 to 95 TFLOP/s of
// the library's 153, were not timed with the larger ones, which bring half as many bytes for an operation.
template <typename T> constexpr int kTileOf = sizeof(T) == 4 ? 64 : kTile;
template <typename T> constexpr int kLds = kTileOf<T> * 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T> constexpr float kRaise = __is_same(T, f16_t) ? 32768.f : 1.f;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up_to(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// ---- the rows that have a kind -----------------------------------------------------------------------------------------
template <typename T>
struct RowsOf {
  const T *x;
  const int64_t* kind;
  const float* g;                 // backward, else null
  int64_t n, n_kinds, each;       // each: rows of a workgroup
  int c, ld;
  int *counts, *rows, *target, *count;     // counts: rows with a kind, of each workgroup; count: of all
  unsigned* tops;                 // the largest |g| of each workgroup
  float* row_g;                   // g of the rows with a kind
  const float* lse_of;            // backward: of all rows, and of those with a kind
  float* row_lse;
  T *to, *to_g;                   // the copy, and the copy times g / max |g| (null: not wanted)
  float *loss, *lse;              // forward: zeros for the rows without a kind
  T* grad_x;                      // backward: likewise (null: not wanted)
  int blocks;
};
__device__ __forceinline__ bool has_kind(int64_t k, int64_t n_kinds) { return k >= 0 && k < n_kinds; }

template <typename T>
__device__ __forceinline__ void count_rows(const RowsOf<T>& a, int64_t from, int64_t end, int& count, unsigned& top, int* shared) {
  count = 0;
  top = 0;
  for (int64_t i = from + threadIdx.x; i < end; i += kRowThreads)
    if (has_kind(a.kind[i], a.n_kinds)) {
      ++count;
      if (a.g) top = std::max(top, __float_as_uint(a.g[i]) & 0x7fffffffu);
    }
  for (int o = 32; o; o >>= 1) {
    count += __shfl_xor(count, o);
    top = std::max(top, (unsigned)__shfl_xor((int)top, o));
  }
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { shared[2 * wave] = count; shared[2 * wave + 1] = (int)top; }
  __syncthreads();
  count = 0;
  for (int w = 0; w < kRowThreads / 64; ++w) {
    count += shared[2 * w];
    top = std::max(top, (unsigned)shared[2 * w + 1]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) loss_count_kernel(RowsOf<T> a) {
  __shared__ int shared[2 * kRowThreads / 64];
  const int64_t from = blockIdx.x * a.each;
  int count;
  unsigned top;
  count_rows(a, from, std::min(from + a.each, a.n), count, top, shared);
  if (threadIdx.x == 0) {
    a.counts[blockIdx.x] = count;
    a.tops[blockIdx.x] = top;
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) loss_rows_kernel(RowsOf<T> a) {
  constexpr int CH = 16 / (int)sizeof(T);
  __shared__ int shared[2 * kRowThreads / 64];
  __shared__ int places[kRowThreads];      // place of a row in the copy, -1: none
  const int64_t from = blockIdx.x * a.each, end = std::min(from + a.each, a.n);
  int at = 0;
  unsigned top = 0;
  if (a.blocks > 1) {
    int count = 0;
    for (int i = threadIdx.x; i < a.blocks; i += kRowThreads) {
      if (i < (int)blockIdx.x) count += a.counts[i];
      top = std::max(top, a.tops[i]);
    }
    for (int o = 32; o; o >>= 1) {
      count += __shfl_xor(count, o);
      top = std::max(top, (unsigned)__shfl_xor((int)top, o));
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { shared[2 * wave] = count; shared[2 * wave + 1] = (int)top; }
    __syncthreads();
    for (int w = 0; w < kRowThreads / 64; ++w) {
      at += shared[2 * w];
      top = std::max(top, (unsigned)shared[2 * w + 1]);
    }
  } else {
    int count;
    count_rows(a, from, end, count, top, shared);
  }
  const float most = __uint_as_float(top);
  const int chunks = a.ld / CH;
  for (int64_t r0 = from; r0 < end; r0 += kRowThreads) {
    const int64_t row = r0 + threadIdx.x;
    const int64_t kind = row < end ? a.kind[row] : -1;
    const bool has = has_kind(kind, a.n_kinds);
    const unsigned long long votes = __ballot(has);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    __syncthreads();
    if (lane == 0) shared[wave] = __popcll(votes);
    __syncthreads();
    int place = at;
    for (int w = 0; w < kRowThreads / 64; ++w) {
      if (w < wave) place += shared[w];
      at += shared[w];
    }
    place += __popcll(votes & ((1ull << lane) - 1));
    places[threadIdx.x] = has ? place : -1;
    if (has) {
      a.rows[place] = (int)row;
      a.target[place] = (int)kind;
      if (a.g) {
        a.row_g[place] = a.g[row];
        a.row_lse[place] = a.lse_of[row];
      }
    } else if (row < end && a.loss) {
      a.loss[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
    }
    __syncthreads();
    // chunks of all rows, four of a thread on their way at a time
    const unsigned all = (unsigned)std::min<int64_t>(kRowThreads, end - r0) * (unsigned)chunks;
    for (unsigned i0 = threadIdx.x; i0 < all; i0 += 4 * kRowThreads) {
      u32x4_t v[4];
      int row_at[4], chunk_at[4], to[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned i = i0 + k * kRowThreads;
        row_at[k] = (int)(i / (unsigned)chunks);
        chunk_at[k] = (int)(i - (unsigned)row_at[k] * (unsigned)chunks) * CH;
        to[k] = i < all ? places[row_at[k]] : -2;
        v[k] = u32x4_t{0, 0, 0, 0};
        if (to[k] >= 0 && chunk_at[k] < a.c) v[k] = load_part<u32x4_t, T>(a.x + (r0 + row_at[k]) * a.c + chunk_at[k], a.c - chunk_at[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = chunk_at[k];
        if (to[k] >= 0) {
          *reinterpret_cast<u32x4_t*>(a.to + (int64_t)to[k] * a.ld + c) = v[k];
          if (a.to_g) {
            typedef T vec __attribute__((ext_vector_type(CH)));
            vec e = __builtin_bit_cast(vec, v[k]);
            const float share = most == 0.f ? 0.f : a.g[r0 + row_at[k]] / most;
#pragma unroll
            for (int j = 0; j < CH; ++j) e[j] = (T)((float)e[j] * share);
            *reinterpret_cast<vec*>(a.to_g + (int64_t)to[k] * a.ld + c) = e;
          }
        } else if (to[k] == -1 && a.grad_x && c < a.c) {
          T zero[CH];
#pragma unroll
          for (int e = 0; e < CH; ++e) zero[e] = T(0);
          store_part<T, CH>(a.grad_x + (r0 + row_at[k]) * a.c + c, zero, a.c - c);
        }
      }
    }
  }
  if (threadIdx.x == 0 && (int)blockIdx.x == a.blocks - 1) {
    *a.count = at;
    if (a.g) a.tops[a.blocks] = top;
  }
}

// The table with rows of whole aligned chunks, zeros at their ends.
template <typename T>
__global__ void __launch_bounds__(256) loss_pack_kernel(const T* from, T* to, int64_t n, int c, int ld) {
  constexpr int CH = 16 / (int)sizeof(T);
  const int chunks = ld / CH;
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n * chunks; i += step) {
    const int64_t r = i / chunks;
    const int k = (int)(i - r * chunks) * CH;
    u32x4_t v = {0, 0, 0, 0};
    if (k < c) v = load_part<u32x4_t, T>(from + r * c + k, c - k);
    *reinterpret_cast<u32x4_t*>(to + r * ld + k) = v;
  }
}

// ---- logits -------------------------------------------------------------------------------------------------------------
template <typename T>
struct LogitArgs {
  const T *x, *table;
  const int *count, *target;
  int64_t r0, r_most;             // the rows r0 .. r0 + r_most - 1 of the copy, as far as there are such
  int64_t k0, k_end;              // the kinds of this launch
  int64_t n;                      // rows of the arrays below
  int c, ld, splits, each;        // each: kinds of a split, whole tiles
  float scale, cap;               // scale: to log2 units without a cap, else over the cap; cap: in log2 units, 0: none
  float twice, over, series[4];   // with a cap: -2 log2 e |scale|; 1 / cap; the tangent's series behind its first term, times the cap
  float *loss, *lse_of;           // forward, of all rows
  const int* rows;
  float2* stats;                  // forward, several splits: maximum and sum of each split and row
  float* at;                      // forward: the logit of the row's own kind
  const float* lse;               // backward, of the rows of the copy
  T* dz;                          // backward: (r_most, ld_dz)
  int64_t ld_dz;
  float* planes;                  // dx, see kDx
  int64_t piece;
  int first;
  T* grad_x;                      // kDx with one piece: where one range of kinds leaves dx, times g and scale_dx (null: planes)
  const float* g;
  float scale_dx;
};

// Where |u| is at most this, tanh u is u times five terms of its series in u^2, to 6e-8 of itself; above, (1 - e) / (1 + e) with e =
// exp(-2 |u|), which errs about 1e-7 below it too, where the tangent may be far smaller.
constexpr float kSeries = 0.3f;
template <typename T>
__device__ __forceinline__ float cap_series(float z, float scale, const LogitArgs<T>& a) {
  const float u = z * scale, q = u * u;
  return u * fmaf(q, fmaf(q, fmaf(q, fmaf(q, a.series[3], a.series[2]), a.series[1]), a.series[0]), a.cap);
}
template <typename T>
__device__ __forceinline__ float cap_exponential(float z, const LogitArgs<T>& a) {
  const float e = __builtin_amdgcn_exp2f(fabsf(z) * a.twice);
  return copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e) * a.cap, z);
}
// Logits in log2 units; slope: 1 - tanh^2.
template <typename T>
__device__ __forceinline__ float capped(float z, const LogitArgs<T>& a, float& slope) {
  float t;
  if constexpr (sizeof(T) == 4) {
    t = tanhf(z * a.scale);
    slope = 1.f - t * t;
    return a.cap * t;
  } else {
    const float signed_z = a.scale < 0.f ? -z : z, scale = fabsf(a.scale);
    const float c = fabsf(z) * scale <= kSeries ? cap_series(signed_z, scale, a) : cap_exponential(signed_z, a);
    t = c * a.over;
    slope = 1.f - t * t;
    return c;
  }
}
// Where the gradients' kernels form them again, the scale's sign in the operands: the tangent to some 1e-7 of 1, with the caps that come here (kWalkCap) far
// below what the gradient is rounded to, by fewer registers (with the block's form 16384 rows, 30011 kinds, 256 bf16 channels take 1560 us a step, 1380 so).
__device__ __forceinline__ float cap_for_gradient(float z, float scale, float cap, float& slope) {
  const float r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * scale * (2.f * kLog2e)));
  slope = 4.f * r * (1.f - r);
  return cap - 2.f * cap * r;
}
// A block of a forward's: all by the series, or all by the other.
template <typename T>
__device__ __forceinline__ void cap_block(f32x16_t& z, float scale, const LogitArgs<T>& a) {
  float most = fabsf(z[0]);
#pragma unroll
  for (int e = 1; e < 16; ++e) most = fmaxf(most, fabsf(z[e]));
  if (__any(most * scale > kSeries)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = cap_exponential(z[e], a);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = cap_series(z[e], scale, a);
  }
}

template <typename T>
__device__ __forceinline__ GemmOperand<T> k_rows(const T* p, int64_t row, int64_t ld, int64_t left) {
  return {{p + row * ld, nullptr}, ld, {(int)std::min<int64_t>(left, kTileOf<T>), 0}};
}

template <typename T>
__device__ __forceinline__ void logits_tile(GemmAcc<kTileOf<T>>& acc, char* lds, const LogitArgs<T>& a, int64_t m0, int64_t rows, int64_t k0) {
  constexpr int D = GemmType<T>::kDepth;
  const GemmOperand<T> x = k_rows(a.x, m0, a.ld, rows - m0), w = k_rows(a.table, k0, a.ld, a.k_end - k0);
  gemm_loop<T, kTileOf<T>, true, true, true, false>(acc, lds, (a.ld + D - 1) / D, [&](int64_t t, int64_t& k, int64_t& depth) {
    k = t * D;
    depth = a.ld;
    return x;
  }, [&](int64_t) { return w; });
}

// Maximum and sum of `splits` statistics `each` places apart, eight of them on their way at a time.
__device__ __forceinline__ void join_stats(const float2* p, int64_t each, int splits, float& most, float& sum) {
  most = -INFINITY;
  sum = 0.f;
  for (int s0 = 0; s0 < splits; s0 += 8) {
    float2 v[8];
    float now = most;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = s0 + k < splits ? p[(s0 + k) * each] : float2{-INFINITY, 0.f};
      now = fmaxf(now, v[k].x);
    }
    const float base = now == -INFINITY ? 0.f : now;
    sum *= __builtin_amdgcn_exp2f(most - base);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += v[k].y * __builtin_amdgcn_exp2f(v[k].x - base);
    most = now;
  }
}
// The same by `slices` threads of a workgroup, 256 / slices apart, that have every slices-th statistic each; the first of them has the
// result.  478 rows with statistics of up to 192 ranges each: 17 us with a thread for a row, 5 with sixteen.
__device__ __forceinline__ void join_stats(const float2* p, int64_t each, int splits, int slices, float& most, float& sum) {
  __shared__ float2 shared[256];
  const int per = 256 / slices, slice = threadIdx.x / per;
  join_stats(p + slice * each, each * slices, splits > slice ? (splits - slice + slices - 1) / slices : 0, most, sum);
  if (slices == 1) return;
  shared[threadIdx.x] = {most, sum};
  __syncthreads();
  if (slice == 0) join_stats(shared + threadIdx.x, per, slices, most, sum);
}
// Threads that share a sum of up to `terms` for each of n results: at least eight terms each, and no more than some 64 K threads.
int slices_of(int64_t n, int64_t terms) {
  int slices = 1;
  while (slices < 32 && n * slices < 32 * 1024 && terms >= 16 * slices) slices *= 2;
  return slices;
}
// The loss and the logarithm of the sum (log2 units) of a row from its own kind's logit, a maximum and a sum.
__device__ __forceinline__ void give_loss(float* loss, float* lse, int row, float at, float top, float sum) {
  const float total = (top == -INFINITY ? 0.f : top) + __builtin_amdgcn_logf(sum);
  loss[row] = (total - at) * kLn2;
  if (lse) lse[row] = total;
}
template <typename T>
__device__ __forceinline__ void give_loss(const LogitArgs<T>& a, int64_t row, float at, float top, float sum) {
  give_loss(a.loss, a.lse_of, a.rows[row], at, top, sum);
}

template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 2) loss_stats_kernel(LogitArgs<T> a) {
  __shared__ alignas(16) char lds[kLds<T>];
  const int64_t rows = *a.count, m0 = (int64_t)(blockIdx.x / a.splits) * kTileOf<T>;
  if (m0 >= rows) return;
  const int split = blockIdx.x % a.splits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
  const int64_t first = (int64_t)split * a.each, end = std::min(first + a.each, a.k_end);
  constexpr int B = kTileOf<T> / 64;      // blocks of 32 for a wavefront, each way
  float top[B], sum[B];
  int own[B];
#pragma unroll
  for (int i = 0; i < B; ++i) {
    const int64_t row = m0 + 32 * (B * wm + i) + (lane & 31);
    own[i] = row < rows ? a.target[row] : -1;
    top[i] = -INFINITY;
    sum[i] = 0.f;
  }
  __shared__ float own_places[kTileOf<T>];
  GemmAcc<kTileOf<T>> acc;
  for (int64_t k0 = first; k0 < end; k0 += kTileOf<T>) {
    logits_tile(acc, lds, a, m0, rows, k0);
    __syncthreads();               // the next tile's operands
#pragma unroll
    for (int i = 0; i < B; ++i) {
      float most = top[i];
#pragma unroll
      for (int j = 0; j < B; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int64_t kind = k0 + 32 * (B * wn + j) + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
          float slope, z = acc[i][j][e];
          z = a.cap > 0.f ? capped(z, a, slope) : z * a.scale;
          if (kind == own[i]) {
            if (a.splits > 1) a.at[m0 + 32 * (B * wm + i) + (lane & 31)] = z;
            else own_places[32 * (B * wm + i) + (lane & 31)] = z;
          }
          z = kind < end ? z : -INFINITY;
          acc[i][j][e] = z;
          most = fmaxf(most, z);
        }
      const float base = most == -INFINITY ? 0.f : most;
      float s = sum[i] * __builtin_amdgcn_exp2f(top[i] - base);
#pragma unroll
      for (int j = 0; j < B; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(acc[i][j][e] - base);
      top[i] = most;
      sum[i] = s;
    }
  }
  // the two halves of a wavefront, then the two wavefronts that share rows
  float2* shared = reinterpret_cast<float2*>(lds);      // one for each row of the tile
  auto join = [](float& m, float& s, float m2, float s2) {
    const float most = fmaxf(m, m2), base = most == -INFINITY ? 0.f : most;
    s = s * __builtin_amdgcn_exp2f(m - base) + s2 * __builtin_amdgcn_exp2f(m2 - base);
    m = most;
  };
  __syncthreads();
#pragma unroll
  for (int i = 0; i < B; ++i) {
    join(top[i], sum[i], __shfl_xor(top[i], 32), __shfl_xor(sum[i], 32));
    if (wn == 1 && lane < 32) shared[32 * (B * wm + i) + lane] = {top[i], sum[i]};
  }
  __syncthreads();
  if (wn == 1 || lane >= 32) return;
#pragma unroll
  for (int i = 0; i < B; ++i) {
    const int r = 32 * (B * wm + i) + lane;
    const float2 other = shared[r];
    join(top[i], sum[i], other.x, other.y);
    if (m0 + r >= rows) continue;
    if (a.splits > 1) a.stats[split * a.n + m0 + r] = {top[i], sum[i]};
    else give_loss(a, m0 + r, own_places[r], top[i], sum[i]);
  }
}

// The same from the statistics of several splits.
__global__ void __launch_bounds__(256) loss_join_kernel(const float2* stats, const float* at, const int* rows, const int* count, int64_t n,
                                                        int splits, int slices, float* loss, float* lse) {
  const int per = 256 / slices;
  const int64_t i = (int64_t)blockIdx.x * per + threadIdx.x % per, have = *count;
  float top, sum;
  join_stats(stats + i, n, i < have ? splits : 0, slices, top, sum);
  if (i < have && (int)threadIdx.x < per) give_loss(loss, lse, rows[i], at[i], top, sum);
}

// (p - [k = y]) (1 - tanh^2) of a tile of rows x kinds.
template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 2) loss_dz_kernel(LogitArgs<T> a) {
  __shared__ alignas(16) char lds[kLds<T>];
  const int64_t rows = std::min<int64_t>(*a.count, a.r0 + a.r_most);
  const int tiles_k = (int)((a.k_end - a.k0 + kTileOf<T> - 1) / kTileOf<T>);
  const int64_t m0 = a.r0 + (int64_t)(blockIdx.x / tiles_k) * kTileOf<T>, k0 = a.k0 + (int64_t)(blockIdx.x % tiles_k) * kTileOf<T>;
  if (m0 >= rows) return;
  GemmAcc<kTileOf<T>> acc;
  logits_tile(acc, lds, a, m0, rows, k0);
  gemm_results<kTileOf<T>, false, 1>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, float (&v)[8]) {
    if (m0 + r >= rows) return;
    const float lse = a.lse[m0 + r];
    const int own = a.target[m0 + r];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float slope = 1.f;
      const float z = a.cap > 0.f ? capped(v[e], a, slope) : v[e] * a.scale;
      const float p = __builtin_amdgcn_exp2f(z - lse) - (k0 + c + e == own ? 1.f : 0.f);
      v[e] = k0 + c + e < a.k_end ? p * slope * kRaise<T> : 0.f;
    }
    store_eight(a.dz + (m0 - a.r0 + r) * a.ld_dz + (k0 - a.k0) + c, v, 8);
  });
}

// ---- logits in 16-bit types, up to 512 channels -----------------------------------------------------------------------------
// A wavefront keeps its rows of x in registers, RB blocks of 32 of them over KS steps of 16 channels, and the table's rows go by
// in LDS, 32 kinds (a stage) at a time, for all four wavefronts: read twice as seldom as where both operands come from LDS, and
// the next stage is on its way throughout.  A lane holds one row of x and sixteen neighbouring kinds of a stage: statistics need no
// exchange before the end, and gradients leave as whole chunks.
//
// The gradients' products, up to 256 channels, are of the same kind.  Where x has a gradient one kernel forms dz and adds up dx: a
// lane's sixteen kinds of dz are the next product's operand as they lie, and the stage in LDS, read through the transposing
// loads, the other.  For the table's gradient dz is kept in blocks of 32 rows x 32 kinds in the order in which that product's operand lies in
// a wavefront (turned over in LDS), so that it passes through LDS as it lies while rows of x go by beside it.
//
// In LDS a stage is 32 rows of 2 KS chunks, chunk c of row i at c ^ chunk_mix(i): sixteen lanes that read one chunk of
// neighbouring rows find it in different banks, and so do the transposing loads, of a pair of chunks of four rows.  Row i is that of kind
// 16 (i >> 2 & 1) + 4 (i >> 3) + (i & 3): what the matrix instruction gives a lane is then in order.
constexpr int kStage = 32, kLeastKinds = 128;
enum { kStats, kDz, kDx };

template <int KS, int MODE> struct Walk {
  static constexpr int THREADS = 256, RB = KS <= 16 && MODE != kDx ? 2 : 1, ROWS = THREADS / 2 * RB;
  static constexpr int NC = 2 * KS, PER = kStage * NC / THREADS, BYTES = kStage * NC * 16;
  static constexpr int BUFFERS = 3 * BYTES <= 80 * 1024 ? 3 : 2;
  static constexpr bool BLOCKS = KS <= 16 && MODE != kStats;         // dz in blocks, turned over in 2 KB of LDS a wavefront and block of rows
  static constexpr int LDS = BUFFERS * BYTES + (BLOCKS ? 4 * RB * 2048 : 0);
  static_assert(PER * THREADS == kStage * NC);
  __device__ static __forceinline__ int chunk_mix(int i) {
    return NC % 16 == 0 ? ((i & 7) << 1) | ((i >> 3) & 1) : (((i >> 1) & 3) << 1) | ((i >> 3) & 1);
  }
};
// Four elements of one column for each lane, from four rows that its sixteen lanes' addresses lie in.
__device__ __forceinline__ u32x2_t read_turned(const char* p) {
  typedef short v4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4 lds_v4;
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)p));
}
// Sixteen bytes for each lane from base + at (base the same in all lanes) to LDS, one lane's after the other's.  As assembly, since
// the compiler would wait for all that is on its way to LDS before every transposing load from there: what has to be there is what
// wait_and_meet counts.
struct LdsSource {
  u32x4_t words;
  __device__ __forceinline__ explicit LdsSource(const void* base) {
    const uint64_t p = (uint64_t)base;
    words[0] = __builtin_amdgcn_readfirstlane((unsigned)p);
    words[1] = __builtin_amdgcn_readfirstlane((unsigned)(p >> 32) & 0xffffu);
    words[2] = kOutside;
    words[3] = 0x00027000;
  }
  // to: the place in LDS, the same in all lanes.  The compiler does not see an access to memory here: the wait states between a vector
  // instruction that wrote one of the scalar operands and the access, five, stand in the assembly.
  __device__ __forceinline__ void load(unsigned to, unsigned at) const {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(at), "s"(words) : "memory", "m0");
  }
};
__device__ __forceinline__ unsigned place_in_lds(const char* p) {
  typedef __attribute__((address_space(3))) const char lds_char;
  return (unsigned)(uintptr_t)(lds_char*)p;
}
// The chunks of a stage that a thread brings, THREADS / NC rows apart: row << 16 | bytes from the row's start, where row i of LDS is
// row of(i) of the stage.
template <typename W, typename Of>
__device__ __forceinline__ void stage_places(unsigned (&place)[W::PER], Of&& of) {
#pragma unroll
  for (int p = 0; p < W::PER; ++p) {
    const int q = p * W::THREADS + (int)threadIdx.x, i = q / W::NC;
    place[p] = (unsigned)(of(i) << 16 | (q % W::NC ^ W::chunk_mix(i)) << 4);
  }
}
// Brings a stage whose rows from `left` on are not there: the last one again.
template <typename W>
__device__ __forceinline__ void fetch_stage(const void* base, unsigned row_bytes, int left, const unsigned (&place)[W::PER], unsigned to, int wave) {
  const LdsSource source(base);
  const unsigned last = (unsigned)std::min(left, kStage) - 1;
#pragma unroll
  for (int p = 0; p < W::PER; ++p)
    source.load(to + (p * W::THREADS + wave * 64) * 16, std::min(place[p] >> 16, last) * row_bytes + (place[p] & 0xffffu));
}
// All of a workgroup's wavefronts have read what they asked of LDS, and all but the last COUNT of each one's accesses to memory are done.
template <int COUNT>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(COUNT) : "memory");
}
constexpr int walk_rows(int steps, int mode) { return steps <= 16 && mode != kDx ? 256 : 128; }
constexpr int walk_grid(int) { return 512; }      // eight wavefronts for each compute unit

// How the rows (tiles of them) and the kinds are shared out, by the number of rows with a kind: `splits` ranges of the kinds, so
// that the tiles' ranges fill the grid some whole number of times.  The host asks for the most there can be.
struct Share { int tiles, splits, each; };
constexpr int more_rounds(int mode) { return mode == kDx ? 1 : 3; }        // of the grid than the fewest
__host__ __device__ inline Share share_out(int mode, int64_t rows, int rows_of_tile, int64_t kinds) {
  const int grid = walk_grid(mode);
  Share s;
  s.tiles = (int)((rows + rows_of_tile - 1) / rows_of_tile);
  if (s.tiles < 1) s.tiles = 1;
  const int most = (int)((kinds + kLeastKinds - 1) / kLeastKinds), rounds = (s.tiles + grid - 1) / grid;
  int64_t best = 0;                // cost of a split: rounds of the grid, and a fiftieth of one for each beyond the fewest
  s.splits = 0;
  for (int j = rounds; j <= rounds + more_rounds(mode); ++j) {
    int n = (int)((int64_t)j * grid / s.tiles);
    n = n < most ? n : most;
    const int64_t cost = 50 * ((s.tiles * (int64_t)n + grid - 1) / grid) + j - rounds;
    if (!s.splits || cost * s.splits < best * n) { best = cost; s.splits = n; }
  }
  s.each = (int)((kinds + s.splits - 1) / s.splits + kStage - 1) / kStage * kStage;
  s.splits = (int)((kinds + s.each - 1) / s.each);
  return s;
}
// The most results (a tile's rows for each split) that any number of rows up to `rows` leaves.
inline int64_t most_results(int mode, int64_t rows, int rows_of_tile, int64_t kinds) {
  const int64_t tiles = std::max<int64_t>(1, ceil_div(rows, rows_of_tile));
  return rows_of_tile * std::min(tiles * ceil_div(kinds, kLeastKinds), (ceil_div(tiles, walk_grid(mode)) + more_rounds(mode)) * walk_grid(mode));
}

// kStats: statistics, stats[(tile * splits + split) * ROWS + row].  kDz: the gradients of a piece's logits.  kDx: them too (dz null: not
// wanted) and planes[(tile * splits + split) * ROWS + row][c] of dx, which `first` begins and other pieces add to.
template <typename T, int KS, int MODE, bool CAP>
__global__ void __launch_bounds__(256, 2) loss_walk_kernel(LogitArgs<T> a) {
  typedef Walk<KS, MODE> W;
  constexpr int RB = W::RB, CB = MODE == kDx ? KS / 2 : 1;       // blocks of 32 channels of dx
  constexpr bool DZ = MODE != kStats;
  constexpr int AHEAD_READS = 4;
  typedef T vec8 __attribute__((ext_vector_type(8)));
  __shared__ alignas(16) char lds[W::LDS];
  const int64_t all = *a.count, rows = DZ ? std::min(all, a.r0 + a.r_most) : all;
  if (rows <= a.r0) return;
  // pieces whose dx is added up are all shared out alike
  const Share share = share_out(MODE, rows - a.r0, W::ROWS, MODE == kDx ? a.piece : a.k_end - a.k0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, li = lane & 31;
  const float scale = fabsf(a.scale);
  const unsigned flip = a.scale < 0.f ? 0x80008000u : 0u;
  const unsigned row_bytes = (unsigned)(a.ld * sizeof(T)), lds_at = place_in_lds(lds);
  unsigned place[W::PER];
  stage_places<W>(place, [](int i) { return 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3); });
  // Where a lane reads: chunk c ^ mix of a row is at (place of c = 0) ^ c for the mixed bits of c, plus the others.  q: a row of
  // four for the transposing loads.
  constexpr int MIXED = W::NC % 16 == 0 ? 15 : 7;
  const int q = 4 * half + ((lane & 15) >> 2);
  const int read_rows = (li * W::NC + (half ^ W::chunk_mix(li))) * 16;
  const int read_cols = (q * W::NC + ((((lane & 16) >> 3) + ((lane & 3) >> 1)) ^ W::chunk_mix(q))) * 16 + (lane & 1) * 8;
  const int items = __builtin_amdgcn_readfirstlane(share.tiles * share.splits), splits = __builtin_amdgcn_readfirstlane(share.splits),
            each = __builtin_amdgcn_readfirstlane(share.each);
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    // the same in all lanes, but divided by vector instructions: back to scalar registers
    const int tile = __builtin_amdgcn_readfirstlane(item / splits), split = item - tile * splits;
    const int64_t m0 = a.r0 + (int64_t)tile * W::ROWS + wave * 32 * RB;
    const int64_t first = a.k0 + (int64_t)split * each, end = std::min(first + each, a.k_end);
    const int kinds = (int)std::max<int64_t>(0, end - first), stages = (kinds + kStage - 1) / kStage;
    const int have = (int)std::min<int64_t>(32 * RB, rows - m0) - li;            // rows of the wavefront from this lane's on
    u32x4_t x[RB][KS];
    int own[RB];                   // the row's kind, from this lane's first of a stage on
    float top[RB], sum[RB], lse[RB], own_z[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int64_t row = std::min(m0 + 32 * i + li, rows - 1);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        x[i][s] = *reinterpret_cast<const u32x4_t*>(a.x + row * a.ld + (2 * s + half) * 8);
        x[i][s] ^= flip;
      }
      own[i] = a.target[row] - (int)first - 16 * half;
      if constexpr (DZ) {
        lse[i] = a.lse[row];
        if (32 * i >= have) {      // no row: its dz is zero
          lse[i] = INFINITY;
          own[i] = -(1 << 29);
        }
      } else {
        top[i] = -INFINITY;
        sum[i] = 0.f;
        own_z[i] = 0.f;
      }
    }
    f32x16_t dx[RB][CB];
    if constexpr (MODE == kDx)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) dx[i][j][e] = 0.f;
    // Stages go from memory to LDS without passing through registers, a wavefront's 64 chunks one after the other.  Three buffers:
    // stage t + 2 is on its way while t is worked on (two where three do not fit: t + 1).
    const int left_of_all = (int)(a.k_end - first);
    const char* table = (const char*)(a.table + first * a.ld);
    auto fetch = [&](int t, int buffer) {
      fetch_stage<W>(table + (int64_t)t * kStage * row_bytes, row_bytes, left_of_all - t * kStage, place, lds_at + buffer, wave);
    };
    constexpr int AHEAD = W::BUFFERS - 1;
    wait_and_meet<0>();            // the item before has read its last stage
#pragma unroll
    for (int t = 0; t < AHEAD; ++t)
      if (t < stages) fetch(t, t * W::BYTES);
    // Where dz goes: blocks (kinds / 32, rows / 32), each in two parts of 64 lanes' sixteen bytes, or rows; what is not there, or not wanted,
    // beyond the end of the buffer, where it is dropped.
    unsigned to[RB];
    const int64_t stage_bytes = W::BLOCKS ? a.ld_dz * 64 : 64;
    const char* dz_base = nullptr;
    if constexpr (DZ) {
      dz_base = (const char*)a.dz + (W::BLOCKS ? (first - a.k0) / kStage * stage_bytes + (m0 - a.r0) * 64
                                               : ((m0 - a.r0) * a.ld_dz + (first - a.k0)) * (int64_t)sizeof(T));
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        if constexpr (W::BLOCKS) to[i] = a.dz && m0 + 32 * i < rows ? (unsigned)(i * 2048 + lane * 16) : kOutside;
        else to[i] = a.dz && 32 * i < have ? (unsigned)(((32 * i + li) * a.ld_dz + 16 * half) * (int)sizeof(T)) : kOutside;
      }
    }
    int now_at = 0, next_at = AHEAD * W::BYTES;      // the buffers of stages t and t + AHEAD
    for (int t = 0; t < stages; ++t) {
      // stage t is there (at least the PER loads of the next one have been asked for since), stage t - 1 has been read
      if (AHEAD > 1 && t + 1 < stages) wait_and_meet<W::PER>();
      else wait_and_meet<0>();
      // places for this stage: not kept over the stages, which would take a register for each
      int at_rows = read_rows + now_at, at_cols = read_cols + now_at;
      asm volatile("" : "+v"(at_rows), "+v"(at_cols));
      f32x16_t acc[RB];
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(lds + (at_rows ^ ((2 * s & MIXED) << 4)) + ((2 * s & ~MIXED) << 4));
#pragma unroll
        for (int i = 0; i < RB; ++i) acc[i] = mma_pair<T>(w, x[i][s], acc[i]);
      }
      if constexpr (MODE == kDx) {
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD_READS, 0);
#pragma unroll
        for (int s = 0; s < KS - AHEAD_READS; ++s) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, AHEAD_READS, 0);
      }
      if (t + AHEAD < stages) fetch(t + AHEAD, next_at);        // while the matrix cores are busy
      now_at = now_at == AHEAD * W::BYTES ? 0 : now_at + W::BYTES;
      next_at = next_at == AHEAD * W::BYTES ? 0 : next_at + W::BYTES;
      const int k0 = t * kStage, mine = kinds - k0 - 16 * half;                 // of this lane's sixteen kinds, where not all
      const bool cut = kinds - k0 < kStage;
      if constexpr (DZ) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(dz_base + t * stage_bytes), 0, kOutside, 0x00027000);
        bool some = cut;
#pragma unroll
        for (int i = 0; i < RB; ++i) some = some || __any((unsigned)(own[i] - k0) < 16u);
        vec8 out[RB][2];
        auto gradients = [&](auto odd) {            // odd: a row's own kind is among them, or the kinds end here
#pragma unroll
          for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              f32x2 v;
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float z = acc[i][e + k];
                float slope = 1.f;
                if constexpr (CAP) v[k] = __builtin_amdgcn_exp2f(cap_for_gradient(z, scale, a.cap, slope) - lse[i]);
                else v[k] = __builtin_amdgcn_exp2f(fmaf(z, scale, -lse[i]));
                if (decltype(odd)::value && e + k == own[i] - k0) v[k] -= 1.f;
                if constexpr (CAP) v[k] *= slope;
                if constexpr (kRaise<T> != 1.f) v[k] *= kRaise<T>;
                if (decltype(odd)::value && e + k >= mine) v[k] = 0.f;
              }
              typedef T vec2 __attribute__((ext_vector_type(2)));
              const vec2 r = __builtin_convertvector(v, vec2);
              out[i][e >> 3][e & 7] = r[0];
              out[i][e >> 3][(e & 7) + 1] = r[1];
            }
        };
        if (some) gradients(std::true_type{});
        else gradients(std::false_type{});
        if constexpr (W::BLOCKS) {
          // row li of a block is 64 bytes, chunk c at c ^ (li >> 2 & 3)
#pragma unroll
          for (int i = 0; i < RB; ++i) {
            char* turn = lds + W::BUFFERS * W::BYTES + (wave * RB + i) * 2048;
#pragma unroll
            for (int s = 0; s < 2; ++s)
              *reinterpret_cast<vec8*>(turn + li * 64 + (((2 * half + s) ^ ((li >> 2) & 3)) << 4)) = out[i][s];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              u32x4_t f;
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const int r = 16 * s + 8 * half + 4 * u + ((lane & 15) >> 2), c = ((lane & 16) >> 3) + ((lane & 3) >> 1);
                const u32x2_t v2 = read_turned(turn + r * 64 + ((c ^ ((2 * half + u) & 3)) << 4) + (lane & 1) * 8);
                f[2 * u] = v2[0];
                f[2 * u + 1] = v2[1];
              }
              __builtin_amdgcn_raw_buffer_store_b128(f, rsrc, to[i] + 1024 * s, 0, 0);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s)
              __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, out[i][s]), rsrc, to[i] + 16 * s, 0, 0);
        }
        // dx^T += W^T dz^T: k = 8 s + .. of this half's kinds are rows 16 s + 4 half + 0 .. 3 and 8 more of the stage
        if constexpr (MODE == kDx)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < CB; ++j) {
              u32x4_t f;
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const u32x2_t v2 = read_turned(lds + (at_cols ^ (((4 * j & MIXED) ^ u) << 4)) + ((4 * j & ~MIXED) << 4) +
                                               (16 * s + 8 * u) * W::NC * 16);
                f[2 * u] = v2[0];
                f[2 * u + 1] = v2[1];
              }
#pragma unroll
              for (int i = 0; i < RB; ++i) dx[i][j] = mma_pair<T>(f, __builtin_bit_cast(u32x4_t, out[i][s]), dx[i][j]);
            }
        if constexpr (MODE == kDx) {
          __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD_READS, 1);
#pragma unroll
          for (int s = 0; s < 2 * CB - AHEAD_READS; ++s) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
          }
          __builtin_amdgcn_sched_group_barrier(0x8, AHEAD_READS, 1);
        }
      } else {
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          const int at_own = own[i] - k0;
          const bool has_own = (unsigned)at_own < 16u && at_own < mine;
          if constexpr (CAP) cap_block(acc[i], scale, a);
          const float factor = CAP ? 1.f : scale;
          if (__any(has_own))
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e == at_own && has_own) own_z[i] = acc[i][e] * factor;
          if (cut)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e >= mine) acc[i][e] = -INFINITY;
          float most = acc[i][0];
#pragma unroll
          for (int e = 1; e < 16; ++e) most = fmaxf(most, acc[i][e]);
          most = most == -INFINITY ? most : most * factor;      // a factor of zero
          const float now = fmaxf(top[i], most), base = now == -INFINITY ? 0.f : now;
          float s = sum[i] * __builtin_amdgcn_exp2f(top[i] - base);
          if (cut) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e < mine) s += __builtin_amdgcn_exp2f(fmaf(acc[i][e], factor, -base));
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(fmaf(acc[i][e], factor, -base));
          }
          top[i] = now;
          sum[i] = s;
        }
      }
    }
    if constexpr (!DZ) {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const float other = __shfl_xor(top[i], 32), more = __shfl_xor(sum[i], 32);
        const float now = fmaxf(top[i], other), base = now == -INFINITY ? 0.f : now;
        const float s = sum[i] * __builtin_amdgcn_exp2f(top[i] - base) + more * __builtin_amdgcn_exp2f(other - base);
        const bool in = 32 * i < have, has_own = (unsigned)own[i] < (unsigned)((stages - 1) * kStage + 16) && !(own[i] & 16);
        if (splits > 1) {
          if (half == 0) a.stats[(int64_t)item * W::ROWS + (wave * RB + i) * 32 + li] = {now, s};
          if (in && has_own) a.at[m0 + 32 * i + li] = own_z[i];
        } else {
          const float there = __shfl_xor(own_z[i], 32);
          if (in && half == 0) give_loss(a, m0 + 32 * i + li, has_own ? own_z[i] : there, now, s);
        }
      }
    }
    if constexpr (MODE == kDx) {
      if (a.grad_x && splits == 1) {
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          if (32 * i >= have) continue;
          const int64_t row = m0 + 32 * i + li;
          const float by = a.g[row] * a.scale_dx;
          T* to_row = a.grad_x + (int64_t)a.rows[row] * a.c;
#pragma unroll
          for (int j = 0; j < CB; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int c = 32 * j + 8 * g + 4 * half, left = a.c - c;
              if (left <= 0) continue;
              T v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = (T)(dx[i][j][4 * g + e] * by);
              store_part<T, 4>(to_row + c, v, left);
            }
        }
        continue;
      }
      // as a wavefront holds them: four channels 32 j + 8 g + 4 half + .. of a lane's row, 64 lanes one after the other
      f32x4* to_plane = reinterpret_cast<f32x4*>(a.planes) + ((int64_t)item * 4 + wave) * (RB * CB * 4 * 64) + lane;
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < CB; ++j) {
          f32x4 old[4] = {};
          if (!a.first)
#pragma unroll
            for (int g = 0; g < 4; ++g) old[g] = to_plane[((i * CB + j) * 4 + g) * 64];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
#pragma unroll
            for (int e = 0; e < 4; ++e) old[g][e] += dx[i][j][4 * g + e];
            to_plane[((i * CB + j) * 4 + g) * 64] = old[g];
          }
        }
    }
  }
}

// Planes of the table's gradient: 128 kinds of a piece to a workgroup, by ranges of the rows; x: the rows of xg from the chunk's first
// on, a stage of 32 of them at a time in LDS, and with it the stage's blocks of dz.  A wavefront has 64 kinds and half the channels, so that
// three quarters of an operand are read from LDS for each product, where 32 kinds and all channels take nine eighths.
// planes[(tile * splits + split) * 4 + wavefront], as a wavefront holds them.
template <typename T>
struct TableArgs {
  const T *x, *dz;
  float* planes;
  const int* count;
  int64_t r0, r_most, kinds;      // rows of the chunk (of dz's blocks), kinds of the piece
  int ld, splits;
};
template <typename T, int KS>
__global__ void __launch_bounds__(256, 2) loss_table_kernel(TableArgs<T> a) {
  typedef Walk<KS, kStats> W;
  constexpr int CB = KS / 4, MIXED = W::NC % 16 == 0 ? 15 : 7, TURN = W::NC % 16 == 0 ? 8 : 4, DEEP = 4;
  __shared__ alignas(16) char lds[3 * W::BYTES + 4 * DEEP * 2048];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int rows = (int)std::max<int64_t>(0, std::min<int64_t>(*a.count - a.r0, a.r_most));
  const int all = (rows + kStage - 1) / kStage, each = (all + a.splits - 1) / a.splits, split = blockIdx.x % a.splits;
  const int begin = split * each, stages = std::max(0, std::min(each, all - begin));
  const int64_t block = (int64_t)(blockIdx.x / a.splits) * 4 + wave;            // of 32 kinds, which this wavefront brings
  const unsigned row_bytes = (unsigned)(a.ld * sizeof(T)), lds_at = place_in_lds(lds);
  unsigned place[W::PER];
  stage_places<W>(place, [](int i) { return i; });
  auto fetch = [&](int t, int buffer) {            // rows beyond the last: that one again, against zeros of dz
    const int first = (begin + t) * kStage;
    fetch_stage<W>(a.x + (int64_t)first * a.ld, row_bytes, rows - first, place, lds_at + buffer, wave);
  };
  // blocks beyond the piece's kinds: the last one again, not written
  const int64_t last = (a.kinds + kStage - 1) / kStage - 1;
  const char* dz = (const char*)a.dz + std::min(block, last) * (a.r_most * 64) + (int64_t)begin * 2048;
  const int q = (lane & 15) >> 2, cl = ((lane & 16) >> 3) + ((lane & 3) >> 1);
  // chunks of this half of the channels: 4 (j + CB * part) ^ .., the part's bits among the mixed ones or above them
  const int part = wave & 1, from = 4 * CB * part, pair = wave >> 1;
  const int read = ((8 * half + q) * W::NC + ((cl ^ W::chunk_mix(8 * half + q)))) * 16 + (lane & 1) * 8;
  f32x16_t acc[2][CB];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  // Stages of x are asked for two ahead, blocks of dz, which come from further away, three, into 2 KB a wavefront and stage; in this
  // order throughout, so that where stage t begins PER + 2 accesses younger than its own may be outstanding.
  auto fetch_dz = [&](int t) {
    const LdsSource source(dz + (int64_t)std::min(t, stages - 1) * 2048);
#pragma unroll
    for (int s = 0; s < 2; ++s) source.load(lds_at + 3 * W::BYTES + (t % DEEP * 4 + wave) * 2048 + s * 1024, s * 1024 + lane * 16);
  };
  if (stages > 0) {
    fetch_dz(0);
    fetch_dz(1);
    fetch(0, 0);
    fetch_dz(2);
    if (stages > 1) fetch(1, W::BYTES);
  }
  int now_at = 0, next_at = 2 * W::BYTES;
  for (int t = 0; t < stages; ++t) {
    if (t + 1 < stages) wait_and_meet<W::PER + 2>();
    else wait_and_meet<0>();
    int at = read + now_at;
    asm volatile("" : "+v"(at));
    const char* mine = lds + 3 * W::BYTES + (t % DEEP * 4 + pair * 2) * 2048 + lane * 16;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4_t now[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) now[i] = *reinterpret_cast<const u32x4_t*>(mine + i * 2048 + s * 1024);
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        u32x4_t f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = 4 * j + from;
          const u32x2_t v2 = read_turned(lds + (at ^ (((c & MIXED) ^ (TURN * u)) << 4)) + ((c & ~MIXED) << 4) + (16 * s + 4 * u) * W::NC * 16);
          f[2 * u] = v2[0];
          f[2 * u + 1] = v2[1];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][j] = mma_pair<T>(f, now[i], acc[i][j]);
      }
      if (s == 0) {                // while the matrix cores are busy
        fetch_dz(t + 3);
        if (t + 2 < stages) fetch(t + 2, next_at);
      }
    }
    now_at = now_at == 2 * W::BYTES ? 0 : now_at + W::BYTES;
    next_at = next_at == 2 * W::BYTES ? 0 : next_at + W::BYTES;
  }
  wait_and_meet<0>();              // what was asked for beyond the end
  // planes of 32 kinds and all channels, this half's behind the other's
  f32x4* to_plane = reinterpret_cast<f32x4*>(a.planes) + (((int64_t)blockIdx.x * 4 + pair * 2) * 2 + part) * (CB * 4 * 64) + lane;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
        to_plane[(i * 2 * CB + j) * 4 * 64 + g * 64] = v;
      }
}

// loss and the logarithm of the sum from the shares' statistics.
__global__ void __launch_bounds__(256) loss_walk_join_kernel(const float2* stats, const float* at, const int* rows, const int* count, int rows_of_tile,
                                                             int64_t kinds, int slices, float* loss, float* lse) {
  const int per = 256 / slices;
  const int64_t i = (int64_t)blockIdx.x * per + threadIdx.x % per, n = *count;
  const Share share = share_out(kStats, n, rows_of_tile, kinds);
  if (share.splits == 1) return;   // given already
  float top, sum;
  join_stats(stats + i / rows_of_tile * share.splits * rows_of_tile + i % rows_of_tile, rows_of_tile, i < n ? share.splits : 0, slices, top, sum);
  if (i < n && (int)threadIdx.x < per) give_loss(loss, lse, rows[i], at[i], top, sum);
}

// The kernels above form a capped logit in the backward, and in the forward in a block with large ones, from a tangent that errs some 1e-7 of
// 1: as much of the cap, and that goes into the softmax.  Up to this cap it is 4e-5 of a probability at most, a tenth of what rounding dz to fp16 takes;
// at 1e6 it would be a tenth of the probability.  Above it the tiles of both operands take each tangent to 1e-7 of itself: 16384 rows, 30011 kinds, 256
// bf16 channels 670 us forward and 2140 a step with a cap of 300, 324 and 1270 with one of 256.
constexpr float kWalkCap = 256.f;
// Steps of 16 channels of the kernels above for a width and a cap, 0: not theirs.
int walk_steps(int channels, int size, float cap) {
  if (size == 4 || channels > 512 || cap > kWalkCap) return 0;
  const int steps = (channels + 15) / 16;
  for (int s : {4, 8, 12, 16, 24, 32})
    if (steps <= s) return s;
  return 0;
}
template <int MODE, typename T>
void walk_launch(int steps, const LogitArgs<T>& l, int64_t rows, int64_t kinds, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    const int of_tile = walk_rows(steps, MODE);
    const unsigned grid = (unsigned)std::min<int64_t>(walk_grid(MODE), most_results(MODE, rows, of_tile, kinds) / of_tile);
    const dim3 threads(256);
    auto go = [&](auto ks) {
      constexpr int KS = decltype(ks)::value;
      if constexpr (KS <= 16 || MODE != kDx) {
        if (l.cap > 0.f) hipLaunchKernelGGL((loss_walk_kernel<T, KS, MODE, true>), dim3(grid), threads, 0, s, l);
        else hipLaunchKernelGGL((loss_walk_kernel<T, KS, MODE, false>), dim3(grid), threads, 0, s, l);
      }
    };
    switch (steps) {
      case 4: return go(std::integral_constant<int, 4>{});
      case 8: return go(std::integral_constant<int, 8>{});
      case 12: return go(std::integral_constant<int, 12>{});
      case 16: return go(std::integral_constant<int, 16>{});
      case 24: return go(std::integral_constant<int, 24>{});
      default: return go(std::integral_constant<int, 32>{});
    }
  }
}

// ---- gradients ----------------------------------------------------------------------------------------------------------
// Planes of fp32 results, one for each range of k, added up over the launches of a sum (first: it begins).
template <typename T>
struct ProductArgs {
  const T *dz, *b;                // b: the table from the piece's first kind on, or the rows of x times g from r0 on
  float* planes;
  const int* count;
  int64_t r0, r_most, ld_dz, kinds;      // kinds of the piece
  int c, ld, splits, first;
  // dx of one range of one piece goes where it belongs: row rows[i], times g[i] scale
  T* grad_x;                      // null: planes
  const int* rows;
  const float* g;
  float scale;
};

// planes[s][row][c] += sum over range s of the piece's kinds of dz[row][k] table[k][c]
template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 2) loss_dx_kernel(ProductArgs<T> a) {
  __shared__ alignas(16) char lds[kLds<T>];
  constexpr int D = GemmType<T>::kDepth;
  const int64_t rows = std::min<int64_t>(*a.count - a.r0, a.r_most);
  const int tiles_c = (a.c + kTileOf<T> - 1) / kTileOf<T>, inner = tiles_c * a.splits;
  const int64_t m0 = (int64_t)(blockIdx.x / inner) * kTileOf<T>;
  if (m0 >= rows) return;
  const int split = blockIdx.x % inner / tiles_c, c0 = blockIdx.x % tiles_c * kTileOf<T>;
  const int64_t all = (a.kinds + D - 1) / D, each = (all + a.splits - 1) / a.splits, from = split * each;
  const GemmOperand<T> dz = k_rows(a.dz, m0, a.ld_dz, rows - m0);
  const GemmOperand<T> w = {{a.b + c0, a.b + c0 + kTileOf<T> / 2}, a.ld, {a.ld - c0, a.ld - c0 - kTileOf<T> / 2}};
  GemmAcc<kTileOf<T>> acc;
  gemm_loop<T, kTileOf<T>, true, true, false, false>(acc, lds, std::min(each, all - from), [&](int64_t t, int64_t& k, int64_t& depth) {
    k = (t + from) * D;
    depth = a.kinds;
    return dz;
  }, [&](int64_t) { return w; });
  float* plane = a.planes + split * a.r_most * a.c;
  gemm_results<kTileOf<T>, false, 1>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, float (&v)[8]) {
    const int left = a.c - c0 - c;
    if (m0 + r >= rows || left <= 0) return;
    if (a.grad_x) {
      const float by = a.g[a.r0 + m0 + r] * a.scale;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= by;
      store_eight(a.grad_x + (int64_t)a.rows[a.r0 + m0 + r] * a.c + c0 + c, v, left);
      return;
    }
    float* to = plane + (m0 + r) * a.c + c0 + c;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!a.first && e < left) v[e] += to[e];
    store_eight(to, v, left);
  });
}

// planes[s][kind][c] = sum over range s of the rows of dz[row][kind] xg[row][c]
template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 2) loss_dw_kernel(ProductArgs<T> a) {
  __shared__ alignas(16) char lds[kLds<T>];
  constexpr int D = GemmType<T>::kDepth;
  const int64_t rows = std::max<int64_t>(0, std::min<int64_t>(*a.count - a.r0, a.r_most));
  const int tiles_c = (a.c + kTileOf<T> - 1) / kTileOf<T>, inner = tiles_c * a.splits;
  const int64_t m0 = (int64_t)(blockIdx.x / inner) * kTileOf<T>;
  const int split = blockIdx.x % inner / tiles_c, c0 = blockIdx.x % tiles_c * kTileOf<T>;
  const int64_t all = (rows + D - 1) / D, each = (all + a.splits - 1) / a.splits, from = std::min(split * each, all);
  const int left_k = (int)(a.ld_dz - m0);
  const GemmOperand<T> dz = {{a.dz + m0, a.dz + m0 + kTileOf<T> / 2}, a.ld_dz, {left_k, left_k - kTileOf<T> / 2}};
  const GemmOperand<T> x = {{a.b + c0, a.b + c0 + kTileOf<T> / 2}, a.ld, {a.ld - c0, a.ld - c0 - kTileOf<T> / 2}};
  GemmAcc<kTileOf<T>> acc;
  gemm_loop<T, kTileOf<T>, true, false, false, false>(acc, lds, std::min(each, all - from), [&](int64_t t, int64_t& k, int64_t& depth) {
    k = (t + from) * D;
    depth = rows;
    return dz;
  }, [&](int64_t) { return x; });
  float* plane = a.planes + split * a.kinds * a.c;
  gemm_results<kTileOf<T>, false, 1>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, float (&v)[8]) {
    const int left = a.c - c0 - c;
    if (m0 + r >= a.kinds || left <= 0) return;
    store_eight(plane + (m0 + r) * a.c + c0 + c, v, left);
  });
}

// grad_x[rows[i]] = g_i scale sum of the planes.
template <typename T>
__global__ void __launch_bounds__(256) loss_dx_join_kernel(const float* planes, int splits, const int* rows, const float* g, const int* count,
                                                           int64_t r0, int64_t r_most, int c, float scale, T* grad_x) {
  const int64_t n = std::min<int64_t>(*count - r0, r_most), i = ((int64_t)blockIdx.x * 256 + threadIdx.x);
  const int64_t row = i / c;
  if (row >= n) return;
  float s = 0.f;
#pragma unroll 4
  for (int k = 0; k < splits; ++k) s += planes[k * r_most * c + i];
  grad_x[(int64_t)rows[r0 + row] * c + (i - row * c)] = (T)(s * (g[r0 + row] * scale));
}

// The same from the planes of the kernel that forms dz too; steps: of 16 channels.  `slices` threads of a workgroup share out the planes
// (21 rows, 23215 kinds, 106 channels: 55 us with one thread, 6 with sixteen).
template <typename T>
__global__ void __launch_bounds__(256) loss_walk_dx_kernel(const float* planes, const int* rows, const float* g, const int* count, int64_t r0,
                                                           int64_t r_most, int64_t piece, int rows_of_tile, int steps, int c, float scale,
                                                           int one_piece, int slices, T* grad_x) {
  __shared__ f32x4 shared[256];
  const int64_t n = std::min<int64_t>(*count - r0, r_most);
  if (n <= 0) return;
  const Share share = share_out(kDx, n, rows_of_tile, piece);
  if (one_piece && share.splits == 1) return;      // there already
  // a thread for four channels of a row, in the order of the planes
  const int each = rows_of_tile * 16 * steps / 4, part = each / 4, blocks = steps * 2;       // of a tile, a wavefront; of 8 channels
  const int per = 256 / slices, slice = threadIdx.x / per;
  const int64_t i = (int64_t)blockIdx.x * per + threadIdx.x % per, tile = i / each;
  const int at = (int)(i - tile * each), wave = at / part, of_wave = at % part, lane = of_wave & 63, block = of_wave >> 6;
  const int64_t row = tile * rows_of_tile + (wave * (rows_of_tile / 128) + block / blocks) * 32 + (lane & 31);
  const int ch = block % blocks * 8 + 4 * (lane >> 5), left = c - ch;
  const bool in = tile < share.tiles && row < n && left > 0;
  f32x4 s = {};
  if (in) {
    const f32x4* p = reinterpret_cast<const f32x4*>(planes) + tile * share.splits * each + at;
#pragma unroll 4
    for (int k = slice; k < share.splits; k += slices) s += p[(int64_t)k * each];
  }
  if (slices > 1) {
    shared[threadIdx.x] = s;
    __syncthreads();
    if (slice) return;
    for (int k = 1; k < slices; ++k) s += shared[k * per + threadIdx.x];
  }
  if (!in) return;
  T out[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(s[e] * (g[r0 + row] * scale));
  store_part<T, 4>(grad_x + (int64_t)rows[r0 + row] * c + ch, out, left);
}

// The planes of a piece's kinds, over the chunks of rows: sums += them, or the result in the last chunk.  Four values to a thread; where
// there are many planes of few values, `slices` threads share out the planes and their sums are added in order.  blocks: planes as
// loss_table_kernel leaves them (steps: of 16 channels), else rows of c channels.
template <typename T>
struct TableJoin {
  const float* planes;
  const unsigned* top;
  float* sums;
  T* out;
  int64_t kinds, stride;            // stride: four values, between planes
  int splits, slices, steps, c, first, last, blocks;
  float scale;
};
template <typename T>
__global__ void __launch_bounds__(256) loss_table_join_kernel(TableJoin<T> a) {
  __shared__ f32x4 shared[256];
  const int per = 256 / a.slices, lane = threadIdx.x % per, slice = threadIdx.x / per;
  const int64_t i = (int64_t)blockIdx.x * per + lane;
  int64_t kind, at;                 // at: of the first plane, four values
  int ch;
  if (a.blocks) {
    const int part = 32 * 16 * a.steps / 4;
    const int64_t wave = i / part;
    const int of_wave = (int)(i - wave * part);
    ch = (of_wave >> 6) % (2 * a.steps) * 8 + 4 * ((of_wave & 63) >> 5);
    kind = wave * 32 + (of_wave & 31);
    at = (wave / 4 * a.splits * 4 + wave % 4) * part + of_wave;
  } else {
    const int groups = (a.c + 3) / 4;
    kind = i / groups;
    ch = (int)(i - kind * groups) * 4;
    at = 0;
  }
  const int left = a.c - ch;
  const bool in = kind < a.kinds && left > 0;
  f32x4 s = {};
  if (in) {
    if (a.blocks) {
      const f32x4* p = reinterpret_cast<const f32x4*>(a.planes) + at;
#pragma unroll 4
      for (int k = slice; k < a.splits; k += a.slices) s += p[(int64_t)k * a.stride];
    } else {
      const float* p = a.planes + kind * a.c + ch;
#pragma unroll 4
      for (int k = slice; k < a.splits; k += a.slices)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < left) s[e] += p[(int64_t)k * a.stride + e];
    }
  }
  if (a.slices > 1) {
    shared[threadIdx.x] = s;
    __syncthreads();
    if (slice) return;
    for (int k = 1; k < a.slices; ++k) s += shared[k * per + lane];
  }
  if (!in) return;
  const int64_t to = kind * a.c + ch;
  if (!a.first)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) s[e] += a.sums[to + e];
  if (a.last) {
    T v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)(s[e] * (__uint_as_float(*a.top) * a.scale));
    store_part<T, 4>(a.out + to, v, left);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) a.sums[to + e] = s[e];
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------------
int loss_check(const cgtp_kind_loss_args* a) {
  if (!a) return CGTP_ERR_NULL;
  if (a->dtype != CGTP_F32 && a->dtype != CGTP_BF16 && a->dtype != CGTP_F16) return CGTP_ERR_DTYPE;
  // 2^29 rows are 2^23 workgroups for tiles of 64: a grid has fewer than 2^32 threads
  if (a->n_rows < 0 || a->n_rows > (1 << 29) || a->n_kinds < 1 || a->n_kinds > (1 << 30) || a->channels < 1 || a->channels > 0x7fff)
    return CGTP_ERR_SHAPE;
  // the kernels take scale * log2 e, or scale / cap and cap * log2 e, in 32 bits: below the normal numbers a quotient loses its bits, or is zero
  auto holds = [](float v) { return v == 0.f || (std::fabs(v) >= 0x1p-126f && std::fabs(v) <= 1e38f); };
  if (!holds(a->scale) || !(a->cap <= 0.f || (a->cap >= 1e-37f && a->cap <= 1e38f))) return CGTP_ERR_CONFIG;
  if (a->cap > 0.f && a->scale != 0.f && (a->scale / a->cap == 0.f || !holds(a->scale / a->cap))) return CGTP_ERR_CONFIG;
  if (a->n_rows > 0 && (!a->x || !a->table || !a->kind)) return CGTP_ERR_NULL;
  return CGTP_OK;
}

// What a piece of dz may take.  Each piece adds to the planes of dx and has planes of the table's gradient joined: 16384 rows, 30011 kinds,
// 256 bf16 channels, kernels of a step 1620 us with 128 MB, 1453 with 256, 1365 with 512 and 1317 with the 1 GB of all of it.
constexpr int64_t kDzBytes = 512 << 20;

// What a call's workspace holds, in bytes from its start.
struct Plan {
  int ld, tile, splits, each, blocks, dx_splits, dw_splits, steps;      // steps: of the kernels for 16-bit types, 0: the others
  bool blocks_of_dz, fused;                      // dz in blocks of 32 x 32; dz and dx in one kernel
  int64_t row_each, chunk, piece;          // rows of a workgroup of loss_rows_kernel; rows and kinds of dz
  int64_t counts, tops, rows, target, row_g, at, stats, x, xg, table, dz, dx, dw, sums, all;
};
Plan plan_of(const cgtp_kind_loss_args* a, bool backward) {
  Plan p = {};
  const int64_t size = a->dtype == CGTP_F32 ? 4 : 2, n = a->n_rows, k = a->n_kinds, c = a->channels;
  p.steps = walk_steps(a->channels, (int)size, a->cap);
  p.tile = size == 4 ? kTileOf<float> : kTile;
  p.ld = (int)(p.steps ? 16 * p.steps : up_to(c, 16 / size));
  p.row_each = n <= 64 ? 64 : std::max<int64_t>(16, ceil_div(n, kRowBlocks));      // 64: one workgroup needs no other's count
  p.blocks = (int)std::max<int64_t>(1, ceil_div(n, p.row_each));
  auto take = [&](int64_t bytes) {
    const int64_t at = p.all;
    p.all += up_to(bytes, 256);
    return at;
  };
  p.counts = take(4 * (p.blocks + 1));
  p.tops = take(4 * (p.blocks + 1));
  p.rows = take(4 * n);
  p.target = take(4 * n);
  p.x = take(n * p.ld * size);
  p.table = p.ld == c && aligned16(a->table) ? -1 : take(k * p.ld * size);
  if (!backward) {
    // up to 1024 workgroups of whole tiles, of which two go one after the other rather than be joined: 26 rows, 4216 kinds, 401 fp32
    // channels 42 us with 256 kinds to a workgroup, 12.5 with 64
    const int64_t tiles = ceil_div(n, p.tile), k_tiles = ceil_div(k, p.tile);
    const int64_t splits = k_tiles <= 2 ? 1 : std::max<int64_t>(1, std::min<int64_t>(k_tiles, 1024 / std::max<int64_t>(1, tiles)));
    p.each = (int)(ceil_div(k_tiles, splits) * p.tile);
    p.splits = (int)ceil_div(k, p.each);
    p.at = take(4 * n);
    p.stats = take(8 * (p.steps ? most_results(kStats, n, walk_rows(p.steps, kStats), k) : n * p.splits));
    return p;
  }
  p.row_g = take(4 * n);
  p.at = take(4 * n);                    // lse of the rows of the copy
  p.xg = a->grad_table ? take(n * p.ld * size) : -1;
  // dz: up to kDzBytes, in pieces of about one size; a piece's planes of up to 128 million values
  p.blocks_of_dz = p.steps && p.steps <= 16;
  p.fused = p.blocks_of_dz && a->grad_x;
  // rows at a time: all of them where their dz is one piece, as far as planes of their dx go; else 32768
  const int64_t rows_of_planes = std::max<int64_t>(4096, std::min<int64_t>((1 << 25) / c / kTile * kTile, 131072));
  const int64_t of_one_piece = kDzBytes / size / up_to(k, kTile) / kTile * kTile;
  p.chunk = std::min(up_to(n, kTile), std::min(rows_of_planes, std::max<int64_t>(32768, of_one_piece)));
  const int64_t most = std::max<int64_t>(1024, std::min(kDzBytes / size / p.chunk, (1 << 27) / c) / kTile * kTile);
  p.piece = up_to(ceil_div(k, ceil_div(k, most)), kTile);
  if (p.fused && !a->grad_table) p.piece = up_to(k, kTile);      // no dz
  else p.dz = take(p.chunk * p.piece * size);
  const int64_t tiles_c = ceil_div(c, p.tile), depth = 128 / size;
  // Ranges of k for a product's tiles: two to four workgroups for every compute unit, as many as leave the fewest without one in the last
  // turn, fewer where that is as good within a fiftieth; at least eight stages of k each.  743 rows, 25965 kinds, 240 fp32 channels, dx: 143 us
  // with 48 tiles in eleven ranges, which leave three of 528 workgroups to some units and two to the others, 109 in sixteen.
  auto ranges = [&](int64_t tiles, int64_t k_tiles) {
    int64_t best = 0, rounds = 0;
    for (int64_t j = 2; j <= 4; ++j) {
      const int64_t n = std::max<int64_t>(1, std::min(256 * j / std::max<int64_t>(1, tiles), k_tiles / 8)), now = ceil_div(tiles * n, 256);
      if (!best || 50 * now * best < 49 * rounds * n) { best = n; rounds = now; }
    }
    return (int)best;
  };
  if (p.fused) {
    p.dx = take(most_results(kDx, p.chunk, walk_rows(p.steps, kDx), p.piece) * p.ld * 4);
  } else if (a->grad_x) {
    p.dx_splits = ranges(p.chunk / p.tile * tiles_c, p.piece / depth);
    p.dx = take(p.dx_splits * p.chunk * c * 4);
  }
  if (a->grad_table) {
    if (p.blocks_of_dz) {        // ranges of at least eight stages of rows
      p.dw_splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / (p.piece / kTile), p.chunk / kStage / 8));
      p.dw = take(p.dw_splits * p.piece * p.ld * 4);
    } else {
      p.dw_splits = ranges(p.piece / p.tile * tiles_c, p.chunk / depth);
      p.dw = take(p.dw_splits * p.piece * c * 4);
    }
    if (n > p.chunk) p.sums = take(k * c * 4);
  }
  return p;
}

template <typename T>
RowsOf<T> gather(const cgtp_kind_loss_args* a, const Plan& p, bool backward, hipStream_t s) {
  char* ws = (char*)a->workspace;
  RowsOf<T> r = {};
  r.x = (const T*)a->x;
  r.kind = a->kind;
  r.g = backward ? a->grad_loss : nullptr;
  r.n = a->n_rows;
  r.n_kinds = a->n_kinds;
  r.each = p.row_each;
  r.c = a->channels;
  r.ld = p.ld;
  r.counts = (int*)(ws + p.counts);
  r.count = r.counts + p.blocks;
  r.tops = (unsigned*)(ws + p.tops);
  r.rows = (int*)(ws + p.rows);
  r.target = (int*)(ws + p.target);
  r.to = (T*)(ws + p.x);
  r.blocks = p.blocks;
  if (backward) {
    r.row_g = (float*)(ws + p.row_g);
    r.lse_of = a->lse;
    r.row_lse = (float*)(ws + p.at);
    r.to_g = p.xg < 0 ? nullptr : (T*)(ws + p.xg);
    r.grad_x = (T*)a->grad_x;
  } else {
    r.loss = a->loss;
    r.lse = a->lse;
  }
  if (p.blocks > 1) hipLaunchKernelGGL(loss_count_kernel<T>, dim3(p.blocks), dim3(kRowThreads), 0, s, r);
  hipLaunchKernelGGL(loss_rows_kernel<T>, dim3(p.blocks), dim3(kRowThreads), 0, s, r);
  if (p.table >= 0)
    hipLaunchKernelGGL(loss_pack_kernel<T>, dim3((unsigned)std::min<int64_t>(ceil_div(a->n_kinds * (p.ld * (int64_t)sizeof(T) / 16), 256), 1 << 15)),
                       dim3(256), 0, s, (const T*)a->table, (T*)(ws + p.table), a->n_kinds, a->channels, p.ld);
  return r;
}

template <typename T>
LogitArgs<T> logit_args(const cgtp_kind_loss_args* a, const Plan& p, const RowsOf<T>& r) {
  LogitArgs<T> l = {};
  l.x = r.to;
  l.table = p.table < 0 ? (const T*)a->table : (const T*)((char*)a->workspace + p.table);
  l.count = r.count;
  l.target = r.target;
  l.n = a->n_rows;
  l.c = a->channels;
  l.ld = p.ld;
  l.cap = a->cap > 0 ? a->cap * kLog2e : 0.f;
  l.scale = a->cap > 0 ? a->scale / a->cap : a->scale * kLog2e;
  if (a->cap > 0) {
    l.twice = -2.f * kLog2e * std::fabs(l.scale);
    l.over = 1.f / l.cap;
    const double terms[] = {-1. / 3, 2. / 15, -17. / 315, 62. / 2835};
    for (int i = 0; i < 4; ++i) l.series[i] = (float)(l.cap * terms[i]);
  }
  return l;
}

template <typename T>
int loss_forward(const cgtp_kind_loss_args* a, hipStream_t s) {
  const Plan p = plan_of(a, false);
  char* ws = (char*)a->workspace;
  const RowsOf<T> r = gather<T>(a, p, false, s);
  LogitArgs<T> l = logit_args<T>(a, p, r);
  l.k_end = a->n_kinds;
  l.splits = p.splits;
  l.each = p.each;
  l.loss = a->loss;
  l.lse_of = a->lse;
  l.rows = r.rows;
  l.stats = (float2*)(ws + p.stats);
  l.at = (float*)(ws + p.at);
  if (p.steps) {
    walk_launch<kStats>(p.steps, l, a->n_rows, a->n_kinds, s);
    const int slices = slices_of(a->n_rows, ceil_div(a->n_kinds, kLeastKinds));
    if (a->n_kinds > kLeastKinds)
      hipLaunchKernelGGL(loss_walk_join_kernel, dim3((unsigned)ceil_div(a->n_rows * slices, 256)), dim3(256), 0, s, l.stats, l.at, r.rows, r.count,
                         walk_rows(p.steps, kStats), a->n_kinds, slices, a->loss, a->lse);
    return launch_status();
  }
  hipLaunchKernelGGL(loss_stats_kernel<T>, dim3((unsigned)(ceil_div(a->n_rows, p.tile) * p.splits)), dim3(kGemmThreads), 0, s, l);
  const int slices = slices_of(a->n_rows, p.splits);
  if (p.splits > 1)
    hipLaunchKernelGGL(loss_join_kernel, dim3((unsigned)ceil_div(a->n_rows * slices, 256)), dim3(256), 0, s, l.stats, l.at, r.rows, r.count, a->n_rows,
                       p.splits, slices, a->loss, a->lse);
  return launch_status();
}

template <typename T>
int loss_backward(const cgtp_kind_loss_args* a, hipStream_t s) {
  const Plan p = plan_of(a, true);
  char* ws = (char*)a->workspace;
  const RowsOf<T> r = gather<T>(a, p, true, s);
  LogitArgs<T> l = logit_args<T>(a, p, r);
  l.lse = r.row_lse;
  l.dz = p.fused && !a->grad_table ? nullptr : (T*)(ws + p.dz);
  l.planes = (float*)(ws + p.dx);
  l.piece = p.piece;
  l.ld_dz = p.blocks_of_dz ? p.chunk : p.piece;
  const int64_t c = a->channels, tiles_c = ceil_div(c, p.tile);
  const float scale = a->scale / kRaise<T>;
  ProductArgs<T> d = {};
  d.dz = l.dz;
  d.count = r.count;
  d.ld_dz = p.piece;
  d.c = a->channels;
  d.ld = p.ld;
  d.rows = l.rows = r.rows;
  d.g = l.g = r.row_g;
  d.scale = l.scale_dx = scale;
  const bool one_piece = p.piece >= a->n_kinds;
  if (one_piece) l.grad_x = (T*)a->grad_x;
  if (one_piece && p.dx_splits == 1) d.grad_x = (T*)a->grad_x;
  auto join = [&](bool blocks, int64_t kinds, bool first, bool last, int64_t k0) {
    TableJoin<T> j = {(const float*)(ws + p.dw), r.tops + p.blocks, (float*)(ws + p.sums) + k0 * c, (T*)a->grad_table + k0 * c, kinds,
                      blocks ? 4 * (32 * 16 * p.steps / 4) : kinds * c, p.dw_splits, 1, p.steps, a->channels, first, last, blocks, scale};
    const int64_t threads = blocks ? up_to(kinds, kTile) * p.ld / 4 : kinds * ceil_div(c, 4);
    // 1024 workgroups' worth of threads, at least eight planes each
    while (j.slices < 32 && threads * j.slices < 256 * 1024 && p.dw_splits >= 16 * j.slices) j.slices *= 2;
    hipLaunchKernelGGL(loss_table_join_kernel<T>, dim3((unsigned)ceil_div(threads * j.slices, 256)), dim3(256), 0, s, j);
  };
  for (int64_t r0 = 0; r0 < a->n_rows; r0 += p.chunk) {
    const int64_t row_tiles = ceil_div(std::min(p.chunk, a->n_rows - r0), p.tile);
    const bool last = r0 + p.chunk >= a->n_rows;
    l.r0 = d.r0 = r0;
    l.r_most = d.r_most = p.chunk;
    for (int64_t k0 = 0; k0 < a->n_kinds; k0 += p.piece) {
      l.k0 = k0;
      l.k_end = std::min(a->n_kinds, k0 + p.piece);
      d.kinds = l.k_end - k0;
      const int64_t k_tiles = ceil_div(d.kinds, p.tile);
      l.first = k0 == 0;
      if (p.fused) walk_launch<kDx>(p.steps, l, p.chunk, p.piece, s);
      else if (p.steps) walk_launch<kDz>(p.steps, l, p.chunk, d.kinds, s);
      else hipLaunchKernelGGL(loss_dz_kernel<T>, dim3((unsigned)(row_tiles * k_tiles)), dim3(kGemmThreads), 0, s, l);
      if (a->grad_x && !p.fused) {
        d.b = l.table + k0 * p.ld;
        d.planes = (float*)(ws + p.dx);
        d.splits = p.dx_splits;
        d.first = k0 == 0;
        hipLaunchKernelGGL(loss_dx_kernel<T>, dim3((unsigned)(row_tiles * tiles_c * d.splits)), dim3(kGemmThreads), 0, s, d);
      }
      if (a->grad_table && p.blocks_of_dz) {
        if constexpr (sizeof(T) == 2) {
          const TableArgs<T> w = {r.to_g + r0 * p.ld, l.dz, (float*)(ws + p.dw), r.count, r0, p.chunk, d.kinds, p.ld, p.dw_splits};
          const dim3 grid((unsigned)(k_tiles * w.splits));      // tiles of 128 kinds
          switch (p.steps) {
            case 4: hipLaunchKernelGGL((loss_table_kernel<T, 4>), grid, dim3(256), 0, s, w); break;
            case 8: hipLaunchKernelGGL((loss_table_kernel<T, 8>), grid, dim3(256), 0, s, w); break;
            case 12: hipLaunchKernelGGL((loss_table_kernel<T, 12>), grid, dim3(256), 0, s, w); break;
            default: hipLaunchKernelGGL((loss_table_kernel<T, 16>), grid, dim3(256), 0, s, w);
          }
          join(true, d.kinds, r0 == 0, last, k0);
        }
      } else if (a->grad_table) {
        d.b = r.to_g + r0 * p.ld;
        d.planes = (float*)(ws + p.dw);
        d.splits = p.dw_splits;
        hipLaunchKernelGGL(loss_dw_kernel<T>, dim3((unsigned)(k_tiles * tiles_c * d.splits)), dim3(kGemmThreads), 0, s, d);
        join(false, d.kinds, r0 == 0, last, k0);
      }
    }
    const int64_t rows_now = std::min(p.chunk, a->n_rows - r0);
    if (p.fused) {
      if constexpr (sizeof(T) == 2) {
        if (one_piece && p.piece <= kLeastKinds) continue;      // one range: there already
        const int64_t threads = up_to(rows_now, walk_rows(p.steps, kDx)) * p.ld / 4;
        const int slices = slices_of(threads, ceil_div(p.piece, kLeastKinds));
        hipLaunchKernelGGL(loss_walk_dx_kernel<T>, dim3((unsigned)ceil_div(threads * slices, 256)), dim3(256), 0, s, l.planes, r.rows, r.row_g, r.count,
                           r0, p.chunk, p.piece, walk_rows(p.steps, kDx), p.steps, a->channels, scale, one_piece, slices, (T*)a->grad_x);
      }
    } else if (a->grad_x && !d.grad_x) {
      hipLaunchKernelGGL(loss_dx_join_kernel<T>, dim3((unsigned)ceil_div(rows_now * c, 256)), dim3(256), 0, s, (const float*)(ws + p.dx), p.dx_splits,
                         r.rows, r.row_g, r.count, r0, p.chunk, a->channels, scale, (T*)a->grad_x);
    }
  }
  return launch_status();
}

// A gradient of zeros where there are no rows.
template <typename T>
__global__ void __launch_bounds__(256) loss_zero_kernel(T* out, int64_t n) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) out[i] = T(0);
}
template <typename T>
int zeros(void* out, int64_t n, hipStream_t s) {
  hipLaunchKernelGGL(loss_zero_kernel<T>, dim3((unsigned)std::min<int64_t>(ceil_div(n, 256), 1 << 15)), dim3(256), 0, s, (T*)out, n);
  return launch_status();
}

}  // namespace
}  // namespace cgtp

extern "C" {

int64_t cgtp_kind_loss_workspace_bytes(const cgtp_kind_loss_args* a, int backward) {
  using namespace cgtp;
  return loss_check(a) == CGTP_OK && a->n_rows > 0 ? plan_of(a, backward != 0).all : 0;
}

int cgtp_kind_loss_forward(const cgtp_kind_loss_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = loss_check(a)) return rc;
  if (a->n_rows == 0) return CGTP_OK;
  if (!a->loss) return CGTP_ERR_NULL;
  if (!a->workspace) return CGTP_ERR_WORKSPACE;
  if (!aligned16(a->workspace)) return CGTP_ERR_ALIGN;
  switch (a->dtype) {
    case CGTP_F32: return loss_forward<float>(a, (hipStream_t)stream);
    case CGTP_BF16: return loss_forward<bf16_t>(a, (hipStream_t)stream);
    default: return loss_forward<f16_t>(a, (hipStream_t)stream);
  }
}

int cgtp_kind_loss_backward(const cgtp_kind_loss_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = loss_check(a)) return rc;
  if (!a->grad_x && !a->grad_table) return CGTP_OK;
  hipStream_t s = (hipStream_t)stream;
  if (a->n_rows == 0) {
    if (!a->grad_table) return CGTP_OK;
    const int64_t n = a->n_kinds * a->channels;
    return a->dtype == CGTP_F32 ? zeros<float>(a->grad_table, n, s) : zeros<f16_t>(a->grad_table, n, s);
  }
  if (!a->lse || !a->grad_loss) return CGTP_ERR_NULL;
  if (!a->workspace) return CGTP_ERR_WORKSPACE;
  if (!aligned16(a->workspace)) return CGTP_ERR_ALIGN;
  switch (a->dtype) {
    case CGTP_F32: return loss_backward<float>(a, s);
    case CGTP_BF16: return loss_backward<bf16_t>(a, s);
    default: return loss_backward<f16_t>(a, s);
  }
}

}  // extern "C"
