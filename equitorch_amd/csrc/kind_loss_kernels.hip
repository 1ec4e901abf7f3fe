// Softmax cross entropy over the kinds of a table (cgtp_kind_loss_forward, cgtp_kind_loss_backward), without keeping the logits:
//
//   z = scale x W^T  (cap: cap tanh(scale x W^T / cap)),   loss_i = log sum_k exp z_ik - z_i,y(i)
//   dz = g_i (softmax(z)_ik - [k = y(i)]) scale (1 - tanh^2),   dx = dz W,   dW = dz^T x
//
// Rows with a kind are taken together first (the others cost nothing and are not read, whatever they hold): their numbers in
// order, and a copy of them with rows of whole aligned chunks.  The forward forms the logits tile by tile and keeps a running
// maximum and sum for each row; the kinds are cut into `splits` ranges where there are few rows, whose statistics are joined in order.
// The backward forms the logits again, a piece of the kinds at a time: (p - [k = y]) (1 - tanh^2) is rounded to the operands'
// type as the operand of the two products it enters, small enough to stay in the caches between them.  g_i multiplies dx
// afterwards; for dW it multiplies the rows of x, divided by the largest |g| (exact where all are equal).  In fp16 the
// probabilities are scaled by 2^15 into its range.
#include "gff_gemm.h"

#include <algorithm>
#include <type_traits>

namespace cgtp {
namespace {

constexpr int kTile = 128, kLds = kTile * 256, kRowBlocks = 1024, kRowThreads = 256;
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
      if (a.g) a.row_g[place] = a.g[row];
    } else if (row < end && a.loss) {
      a.loss[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
    }
    __syncthreads();
    const int rows = (int)std::min<int64_t>(kRowThreads, end - r0);
    for (int64_t i = threadIdx.x; i < (int64_t)rows * chunks; i += kRowThreads) {
      const int r = (int)(i / chunks), c = (int)(i % chunks) * CH, to = places[r], left = a.c - c;
      if (to < 0) {
        if (a.grad_x && left > 0) {
          T zero[CH];
#pragma unroll
          for (int e = 0; e < CH; ++e) zero[e] = T(0);
          store_part<T, CH>(a.grad_x + (r0 + r) * a.c + c, zero, left);
        }
        continue;
      }
      u32x4_t v = {0, 0, 0, 0};
      if (left > 0) v = load_part<u32x4_t, T>(a.x + (r0 + r) * a.c + c, left);
      *reinterpret_cast<u32x4_t*>(a.to + (int64_t)to * a.ld + c) = v;
      if (a.to_g) {
        typedef T vec __attribute__((ext_vector_type(CH)));
        vec e = __builtin_bit_cast(vec, v);
        const float share = most == 0.f ? 0.f : a.g[r0 + r] / most;
#pragma unroll
        for (int j = 0; j < CH; ++j) e[j] = (T)((float)e[j] * share);
        *reinterpret_cast<vec*>(a.to_g + (int64_t)to * a.ld + c) = e;
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
  float2* stats;                  // forward: maximum and sum of each split and row
  float* at;                      // forward: the logit of the row's own kind
  const float* lse;               // backward, of the rows of the copy
  T* dz;                          // backward: (r_most, ld_dz)
  int64_t ld_dz;
};

// Logits in log2 units; slope: 1 - tanh^2.
template <typename T>
__device__ __forceinline__ float capped(float z, float scale, float cap, float& slope) {
  const float u = z * scale;
  if constexpr (sizeof(T) == 4) {
    const float t = tanhf(u);
    slope = 1.f - t * t;
    return cap * t;
  } else {
    const float r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * (2.f * kLog2e)));
    slope = 4.f * r * (1.f - r);
    return cap - 2.f * cap * r;
  }
}

template <typename T>
__device__ __forceinline__ GemmOperand<T> k_rows(const T* p, int64_t row, int64_t ld, int64_t left) {
  return {{p + row * ld, nullptr}, ld, {(int)std::min<int64_t>(left, kTile), 0}};
}

template <typename T>
__device__ __forceinline__ void logits_tile(GemmAcc<kTile>& acc, char* lds, const LogitArgs<T>& a, int64_t m0, int64_t rows, int64_t k0) {
  constexpr int D = GemmType<T>::kDepth;
  const GemmOperand<T> x = k_rows(a.x, m0, a.ld, rows - m0), w = k_rows(a.table, k0, a.ld, a.k_end - k0);
  gemm_loop<T, kTile, true, true, true, false>(acc, lds, (a.ld + D - 1) / D, [&](int64_t t, int64_t& k, int64_t& depth) {
    k = t * D;
    depth = a.ld;
    return x;
  }, [&](int64_t) { return w; });
}

template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 2) loss_stats_kernel(LogitArgs<T> a) {
  __shared__ alignas(16) char lds[kLds];
  const int64_t rows = *a.count, m0 = (int64_t)(blockIdx.x / a.splits) * kTile;
  if (m0 >= rows) return;
  const int split = blockIdx.x % a.splits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
  const int64_t first = (int64_t)split * a.each, end = std::min(first + a.each, a.k_end);
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
  int own[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = m0 + 32 * (2 * wm + i) + (lane & 31);
    own[i] = row < rows ? a.target[row] : -1;
  }
  GemmAcc<kTile> acc;
  for (int64_t k0 = first; k0 < end; k0 += kTile) {
    logits_tile(acc, lds, a, m0, rows, k0);
    __syncthreads();               // the next tile's operands
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float most = top[i];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int64_t kind = k0 + 32 * (2 * wn + j) + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
          float slope, z = acc[i][j][e];
          z = a.cap > 0.f ? capped<T>(z, a.scale, a.cap, slope) : z * a.scale;
          if (kind == own[i]) a.at[m0 + 32 * (2 * wm + i) + (lane & 31)] = z;
          z = kind < end ? z : -INFINITY;
          acc[i][j][e] = z;
          most = fmaxf(most, z);
        }
      const float base = most == -INFINITY ? 0.f : most;
      float s = sum[i] * __builtin_amdgcn_exp2f(top[i] - base);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(acc[i][j][e] - base);
      top[i] = most;
      sum[i] = s;
    }
  }
  // the two halves of a wavefront, then the two wavefronts that share rows
  float2* shared = reinterpret_cast<float2*>(lds);
  auto join = [](float& m, float& s, float m2, float s2) {
    const float most = fmaxf(m, m2), base = most == -INFINITY ? 0.f : most;
    s = s * __builtin_amdgcn_exp2f(m - base) + s2 * __builtin_amdgcn_exp2f(m2 - base);
    m = most;
  };
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    join(top[i], sum[i], __shfl_xor(top[i], 32), __shfl_xor(sum[i], 32));
    if (wn == 1 && lane < 32) shared[32 * (2 * wm + i) + lane] = {top[i], sum[i]};
  }
  __syncthreads();
  if (wn == 1 || lane >= 32) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 32 * (2 * wm + i) + lane;
    const float2 other = shared[r];
    join(top[i], sum[i], other.x, other.y);
    if (m0 + r < rows) a.stats[split * a.n + m0 + r] = {top[i], sum[i]};
  }
}

// loss and the logarithm of the sum (log2 units) from the splits' statistics.
__global__ void __launch_bounds__(256) loss_join_kernel(const float2* stats, const float* at, const int* rows, const int* count, int64_t n,
                                                        int splits, float* loss, float* lse) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= *count) return;
  float most = -INFINITY;
  for (int s = 0; s < splits; ++s) most = fmaxf(most, stats[s * n + i].x);
  const float base = most == -INFINITY ? 0.f : most;
  float sum = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float2 v = stats[s * n + i];
    sum += v.y * __builtin_amdgcn_exp2f(v.x - base);
  }
  const float total = base + __builtin_amdgcn_logf(sum);
  loss[rows[i]] = (total - at[i]) * kLn2;
  if (lse) lse[rows[i]] = total;
}

// (p - [k = y]) (1 - tanh^2) of a tile of rows x kinds.
template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 2) loss_dz_kernel(LogitArgs<T> a) {
  __shared__ alignas(16) char lds[kLds];
  const int64_t rows = std::min<int64_t>(*a.count, a.r0 + a.r_most);
  const int tiles_k = (int)((a.k_end - a.k0 + kTile - 1) / kTile);
  const int64_t m0 = a.r0 + (int64_t)(blockIdx.x / tiles_k) * kTile, k0 = a.k0 + (int64_t)(blockIdx.x % tiles_k) * kTile;
  if (m0 >= rows) return;
  GemmAcc<kTile> acc;
  logits_tile(acc, lds, a, m0, rows, k0);
  gemm_results<kTile, false, 1>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, float (&v)[8]) {
    if (m0 + r >= rows) return;
    const float lse = a.lse[m0 + r];
    const int own = a.target[m0 + r];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float slope = 1.f;
      const float z = a.cap > 0.f ? capped<T>(v[e], a.scale, a.cap, slope) : v[e] * a.scale;
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
// In LDS a stage is 32 rows of 2 KS chunks, chunk c of row i at c ^ chunk_mix(i): sixteen lanes that read one chunk of
// neighbouring rows find it in different banks.  Row i is that of kind 16 (i >> 2 & 1) + 4 (i >> 3) + (i & 3): what the matrix
// instruction gives a lane is then in order.
constexpr int kStage = 32, kWalkThreads = 256, kWalkGrid = 512, kLeastKinds = 128;      // the grid: two workgroups for each compute unit

template <int KS> struct Walk {
  static constexpr int RB = KS <= 16 ? 2 : 1, ROWS = 4 * 32 * RB, NC = 2 * KS, PER = kStage * NC / kWalkThreads;
  static constexpr int BYTES = kStage * NC * 16;
  __device__ static __forceinline__ int chunk_mix(int i) { return NC % 16 == 0 ? i & 15 : (i >> 1) & 7; }
};

// How the rows (tiles of them) and the kinds are shared out, by the number of rows with a kind: `splits` ranges of the kinds, so
// that the tiles' ranges fill the grid some whole number of times.  The host asks for the most there can be.
struct Share { int tiles, splits, each; };
__host__ __device__ inline Share share_out(int64_t rows, int rows_of_tile, int64_t kinds) {
  Share s;
  s.tiles = (int)((rows + rows_of_tile - 1) / rows_of_tile);
  if (s.tiles < 1) s.tiles = 1;
  const int most = (int)((kinds + kLeastKinds - 1) / kLeastKinds), rounds = (s.tiles + kWalkGrid - 1) / kWalkGrid;
  int64_t best = 0;                // cost of a split: rounds of the grid, and a fiftieth of one for each beyond the fewest
  s.splits = 0;
  for (int j = rounds; j < rounds + 4; ++j) {
    int n = (int)((int64_t)j * kWalkGrid / s.tiles);
    n = n < most ? n : most;
    const int64_t cost = 50 * ((s.tiles * (int64_t)n + kWalkGrid - 1) / kWalkGrid) + j - rounds;
    if (!s.splits || cost * s.splits < best * n) { best = cost; s.splits = n; }
  }
  s.each = (int)((kinds + s.splits - 1) / s.splits + kStage - 1) / kStage * kStage;
  s.splits = (int)((kinds + s.each - 1) / s.each);
  return s;
}
// The most results (a tile's rows for each split) that any number of rows up to `rows` leaves.
inline int64_t most_results(int64_t rows, int rows_of_tile, int64_t kinds) {
  const int64_t tiles = std::max<int64_t>(1, ceil_div(rows, rows_of_tile));
  return rows_of_tile * std::min(tiles * ceil_div(kinds, kLeastKinds), (ceil_div(tiles, kWalkGrid) + 3) * kWalkGrid);
}

// DZ: the gradients of a piece, else statistics, stats[(tile * splits + split) * ROWS + row].
template <typename T, int KS, bool DZ, bool CAP>
__global__ void __launch_bounds__(kWalkThreads, 2) loss_walk_kernel(LogitArgs<T> a) {
  typedef Walk<KS> W;
  constexpr int RB = W::RB;
  typedef T vec8 __attribute__((ext_vector_type(8)));
  __shared__ alignas(16) char lds[2][W::BYTES];
  const int64_t all = *a.count, rows = DZ ? std::min(all, a.r0 + a.r_most) : all;
  if (rows <= a.r0) return;
  const Share share = share_out(rows - a.r0, W::ROWS, a.k_end - a.k0);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, li = lane & 31;
  const float scale = fabsf(a.scale);
  const unsigned flip = a.scale < 0.f ? 0x80008000u : 0u;
  // where this thread's chunks of a stage come from
  int from_row[W::PER], from_chunk[W::PER];
#pragma unroll
  for (int p = 0; p < W::PER; ++p) {
    const int q = p * kWalkThreads + tid, i = q / W::NC;
    from_row[p] = 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3);
    from_chunk[p] = (q % W::NC ^ W::chunk_mix(i)) * 8;
  }
  const int read = li * W::NC, mixed = W::chunk_mix(li);
  for (int64_t item = blockIdx.x; item < (int64_t)share.tiles * share.splits; item += gridDim.x) {
    const int64_t m0 = a.r0 + item / share.splits * W::ROWS + wave * 32 * RB;
    const int64_t first = a.k0 + item % share.splits * share.each, end = std::min(first + share.each, a.k_end);
    const int stages = (int)((end - first + kStage - 1) / kStage);
    u32x4_t x[RB][KS];
    int own[RB];
    float top[RB], sum[RB], lse[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int64_t row = std::min(m0 + 32 * i + li, rows - 1);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        x[i][s] = *reinterpret_cast<const u32x4_t*>(a.x + row * a.ld + (2 * s + half) * 8);
        x[i][s] ^= flip;
      }
      own[i] = a.target[row];
      if constexpr (DZ) lse[i] = a.lse[row];
      else top[i] = -INFINITY, sum[i] = 0.f;
    }
    u32x4_t next[W::PER];
    auto fetch = [&](int t) {
      const int64_t k = first + (int64_t)t * kStage;
      const T* base = a.table + k * a.ld;
      const int last = (int)std::min<int64_t>(kStage, a.k_end - k) - 1;       // rows beyond the table: the last one again
#pragma unroll
      for (int p = 0; p < W::PER; ++p)
        next[p] = *reinterpret_cast<const u32x4_t*>(base + (int64_t)std::min(from_row[p], last) * a.ld + from_chunk[p]);
    };
    auto store = [&](int t) {
#pragma unroll
      for (int p = 0; p < W::PER; ++p) *reinterpret_cast<u32x4_t*>(lds[t & 1] + (p * kWalkThreads + tid) * 16) = next[p];
    };
    __syncthreads();               // the item before has read its last stage
    fetch(0);
    store(0);
    if (stages > 1) fetch(1);
    for (int t = 0; t < stages; ++t) {
      __syncthreads();             // stage t is there, stage t - 1 has been read
      if (t + 1 < stages) store(t + 1);
      if (t + 2 < stages) fetch(t + 2);
      const char* at = lds[t & 1];
      f32x16_t acc[RB];
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(at + (read + ((2 * s + half) ^ mixed)) * 16);
#pragma unroll
        for (int i = 0; i < RB; ++i) acc[i] = mma_pair<T>(w, x[i][s], acc[i]);
      }
      const int64_t k0 = first + (int64_t)t * kStage;
      const int mine = (int)std::min<int64_t>(end - k0 - 16 * half, 16);      // of this lane's sixteen kinds
      const bool cut = end - k0 < kStage;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const int at_own = (int)std::max<int64_t>(-1, std::min<int64_t>(own[i] - k0 - 16 * half, 16));
        const bool has_own = at_own >= 0 && at_own < mine;
        if constexpr (DZ) {
          float v[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float slope = 1.f, z = acc[i][e];
            if constexpr (CAP) v[e] = __builtin_amdgcn_exp2f(capped<T>(z, scale, a.cap, slope) - lse[i]);
            else v[e] = __builtin_amdgcn_exp2f(fmaf(z, scale, -lse[i]));
            if constexpr (CAP) acc[i][e] = slope;
          }
          if (__any(has_own))
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e == at_own) v[e] -= 1.f;
          vec8 out[2];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if constexpr (CAP) v[e] *= acc[i][e];
            out[e >> 3][e & 7] = (T)(kRaise<T> == 1.f ? v[e] : v[e] * kRaise<T>);
          }
          if (cut)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e >= mine) out[e >> 3][e & 7] = T(0);
          const int64_t row = m0 + 32 * i + li;
          if (row < rows) {
            T* to = a.dz + (row - a.r0) * a.ld_dz + (k0 - a.k0) + 16 * half;
            *reinterpret_cast<vec8*>(to) = out[0];
            *reinterpret_cast<vec8*>(to + 8) = out[1];
          }
        } else {
          if constexpr (CAP)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float slope;
              acc[i][e] = capped<T>(acc[i][e], scale, a.cap, slope);
            }
          const float factor = CAP ? 1.f : scale;
          if (__any(has_own))
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e == at_own && has_own && m0 + 32 * i + li < rows) a.at[m0 + 32 * i + li] = acc[i][e] * factor;
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
        if (half == 0) a.stats[item * W::ROWS + (wave * RB + i) * 32 + li] = {now, s};
      }
    }
  }
}

// loss and the logarithm of the sum from the shares' statistics.
__global__ void __launch_bounds__(256) loss_walk_join_kernel(const float2* stats, const float* at, const int* rows, const int* count, int rows_of_tile,
                                                             int64_t kinds, float* loss, float* lse) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = *count;
  if (i >= n) return;
  const Share share = share_out(n, rows_of_tile, kinds);
  const float2* mine = stats + i / rows_of_tile * share.splits * rows_of_tile + i % rows_of_tile;
  float most = -INFINITY;
  for (int s = 0; s < share.splits; ++s) most = fmaxf(most, mine[(int64_t)s * rows_of_tile].x);
  const float base = most == -INFINITY ? 0.f : most;
  float sum = 0.f;
  for (int s = 0; s < share.splits; ++s) {
    const float2 v = mine[(int64_t)s * rows_of_tile];
    sum += v.y * __builtin_amdgcn_exp2f(v.x - base);
  }
  const float total = base + __builtin_amdgcn_logf(sum);
  loss[rows[i]] = (total - at[i]) * kLn2;
  if (lse) lse[rows[i]] = total;
}

// Steps of 16 channels of the kernels above for a width, 0: not theirs.
int walk_steps(int channels, int size) {
  if (size == 4 || channels > 512) return 0;
  const int steps = (channels + 15) / 16;
  for (int s : {4, 8, 12, 16, 24, 32})
    if (steps <= s) return s;
  return 0;
}
template <bool DZ, typename T>
void walk_launch(int steps, const LogitArgs<T>& l, unsigned grid, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    auto go = [&](auto ks) {
      constexpr int KS = decltype(ks)::value;
      if (l.cap > 0.f) hipLaunchKernelGGL((loss_walk_kernel<T, KS, DZ, true>), dim3(grid), dim3(kWalkThreads), 0, s, l);
      else hipLaunchKernelGGL((loss_walk_kernel<T, KS, DZ, false>), dim3(grid), dim3(kWalkThreads), 0, s, l);
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
};

// planes[s][row][c] += sum over range s of the piece's kinds of dz[row][k] table[k][c]
template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 2) loss_dx_kernel(ProductArgs<T> a) {
  __shared__ alignas(16) char lds[kLds];
  constexpr int D = GemmType<T>::kDepth;
  const int64_t rows = std::min<int64_t>(*a.count - a.r0, a.r_most);
  const int tiles_c = (a.c + kTile - 1) / kTile, inner = tiles_c * a.splits;
  const int64_t m0 = (int64_t)(blockIdx.x / inner) * kTile;
  if (m0 >= rows) return;
  const int split = blockIdx.x % inner / tiles_c, c0 = blockIdx.x % tiles_c * kTile;
  const int64_t all = (a.kinds + D - 1) / D, each = (all + a.splits - 1) / a.splits, from = split * each;
  const GemmOperand<T> dz = k_rows(a.dz, m0, a.ld_dz, rows - m0);
  const GemmOperand<T> w = {{a.b + c0, a.b + c0 + kTile / 2}, a.ld, {a.ld - c0, a.ld - c0 - kTile / 2}};
  GemmAcc<kTile> acc;
  gemm_loop<T, kTile, true, true, false, false>(acc, lds, std::min(each, all - from), [&](int64_t t, int64_t& k, int64_t& depth) {
    k = (t + from) * D;
    depth = a.kinds;
    return dz;
  }, [&](int64_t) { return w; });
  float* plane = a.planes + split * a.r_most * a.c;
  gemm_results<kTile, false, 1>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, float (&v)[8]) {
    const int left = a.c - c0 - c;
    if (m0 + r >= rows || left <= 0) return;
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
  __shared__ alignas(16) char lds[kLds];
  constexpr int D = GemmType<T>::kDepth;
  const int64_t rows = std::max<int64_t>(0, std::min<int64_t>(*a.count - a.r0, a.r_most));
  const int tiles_c = (a.c + kTile - 1) / kTile, inner = tiles_c * a.splits;
  const int64_t m0 = (int64_t)(blockIdx.x / inner) * kTile;
  const int split = blockIdx.x % inner / tiles_c, c0 = blockIdx.x % tiles_c * kTile;
  const int64_t all = (rows + D - 1) / D, each = (all + a.splits - 1) / a.splits, from = std::min(split * each, all);
  const int left_k = (int)(a.ld_dz - m0);
  const GemmOperand<T> dz = {{a.dz + m0, a.dz + m0 + kTile / 2}, a.ld_dz, {left_k, left_k - kTile / 2}};
  const GemmOperand<T> x = {{a.b + c0, a.b + c0 + kTile / 2}, a.ld, {a.ld - c0, a.ld - c0 - kTile / 2}};
  GemmAcc<kTile> acc;
  gemm_loop<T, kTile, true, false, false, false>(acc, lds, std::min(each, all - from), [&](int64_t t, int64_t& k, int64_t& depth) {
    k = (t + from) * D;
    depth = rows;
    return dz;
  }, [&](int64_t) { return x; });
  float* plane = a.planes + split * a.kinds * a.c;
  gemm_results<kTile, false, 1>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, float (&v)[8]) {
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
  for (int k = 0; k < splits; ++k) s += planes[k * r_most * c + i];
  grad_x[(int64_t)rows[r0 + row] * c + (i - row * c)] = (T)(s * (g[r0 + row] * scale));
}

// The planes of a piece's kinds, over the chunks of rows: sums[i] += them, or the result in the last chunk.
template <typename T>
__global__ void __launch_bounds__(256) loss_dw_join_kernel(const float* planes, int splits, int64_t elems, const unsigned* top, float scale,
                                                           int first, int last, float* sums, T* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= elems) return;
  float s = first ? 0.f : sums[i];
  for (int k = 0; k < splits; ++k) s += planes[k * elems + i];
  if (last) out[i] = (T)(s * (__uint_as_float(*top) * scale));
  else sums[i] = s;
}

// lse of the rows of the copy.
__global__ void __launch_bounds__(256) loss_take_kernel(const float* from, const int* rows, const int* count, float* to) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < *count) to[i] = from[rows[i]];
}

// ---- launches -------------------------------------------------------------------------------------------------------------
int loss_check(const cgtp_kind_loss_args* a) {
  if (!a) return CGTP_ERR_NULL;
  if (a->dtype != CGTP_F32 && a->dtype != CGTP_BF16 && a->dtype != CGTP_F16) return CGTP_ERR_DTYPE;
  if (a->n_rows < 0 || a->n_rows > (1 << 30) || a->n_kinds < 1 || a->n_kinds > (1 << 30) || a->channels < 1 || a->channels > 0x7fff)
    return CGTP_ERR_SHAPE;
  if (a->n_rows > 0 && (!a->x || !a->table || !a->kind)) return CGTP_ERR_NULL;
  return CGTP_OK;
}

// What a call's workspace holds, in bytes from its start.
struct Plan {
  int ld, splits, each, blocks, dx_splits, dw_splits, steps, tile_rows;      // steps: of the kernels for 16-bit types, 0: the others
  int64_t row_each, chunk, piece;          // rows of a workgroup of loss_rows_kernel; rows and kinds of dz
  int64_t counts, tops, rows, target, row_g, at, stats, x, xg, table, dz, dx, dw, sums, all;
};
Plan plan_of(const cgtp_kind_loss_args* a, bool backward) {
  Plan p = {};
  const int64_t size = a->dtype == CGTP_F32 ? 4 : 2, n = a->n_rows, k = a->n_kinds, c = a->channels;
  p.steps = walk_steps(a->channels, (int)size);
  p.tile_rows = p.steps && p.steps <= 16 ? 256 : 128;
  p.ld = (int)(p.steps ? 16 * p.steps : up_to(c, 16 / size));
  p.row_each = up_to(std::max<int64_t>(64, ceil_div(n, kRowBlocks)), 64);
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
    // 1024 workgroups where the table has that many tiles for them; a split is whole tiles
    const int64_t tiles = ceil_div(n, kTile), k_tiles = ceil_div(k, kTile);
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(k_tiles, 1024 / std::max<int64_t>(1, tiles)));
    p.each = (int)(ceil_div(k_tiles, splits) * kTile);
    p.splits = (int)ceil_div(k, p.each);
    p.at = take(4 * n);
    p.stats = take(8 * (p.steps ? most_results(n, p.tile_rows, k) : n * p.splits));
    return p;
  }
  p.row_g = take(4 * n);
  p.at = take(4 * n);                    // lse of the rows of the copy
  p.xg = a->grad_table ? take(n * p.ld * size) : -1;
  // dz: up to 64 million values; a piece's planes of up to 128 million
  p.chunk = std::min<int64_t>(up_to(n, kTile), 32768);
  p.piece = std::min<int64_t>(up_to(k, kTile), std::max<int64_t>(1024, std::min((1 << 26) / p.chunk, (1 << 27) / c) / kTile * kTile));
  p.dz = take(p.chunk * p.piece * size);
  const int64_t tiles_c = ceil_div(c, kTile), depth = 128 / size;
  auto ranges = [&](int64_t tiles, int64_t k_tiles) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(512, std::max<int64_t>(1, tiles)), k_tiles / 8));
  };
  if (a->grad_x) {
    p.dx_splits = ranges(p.chunk / kTile * tiles_c, p.piece / depth);
    p.dx = take(p.dx_splits * p.chunk * c * 4);
  }
  if (a->grad_table) {
    p.dw_splits = ranges(p.piece / kTile * tiles_c, p.chunk / depth);
    p.dw = take(p.dw_splits * p.piece * c * 4);
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
  l.stats = (float2*)(ws + p.stats);
  l.at = (float*)(ws + p.at);
  if (p.steps) {
    const unsigned grid = (unsigned)std::min<int64_t>(kWalkGrid, most_results(a->n_rows, p.tile_rows, a->n_kinds) / p.tile_rows);
    walk_launch<false>(p.steps, l, grid, s);
    hipLaunchKernelGGL(loss_walk_join_kernel, dim3((unsigned)ceil_div(a->n_rows, 256)), dim3(256), 0, s, l.stats, l.at, r.rows, r.count,
                       p.tile_rows, a->n_kinds, a->loss, a->lse);
    return launch_status();
  }
  hipLaunchKernelGGL(loss_stats_kernel<T>, dim3((unsigned)(ceil_div(a->n_rows, kTile) * p.splits)), dim3(kGemmThreads), 0, s, l);
  hipLaunchKernelGGL(loss_join_kernel, dim3((unsigned)ceil_div(a->n_rows, 256)), dim3(256), 0, s, l.stats, l.at, r.rows, r.count, a->n_rows,
                     p.splits, a->loss, a->lse);
  return launch_status();
}

template <typename T>
int loss_backward(const cgtp_kind_loss_args* a, hipStream_t s) {
  const Plan p = plan_of(a, true);
  char* ws = (char*)a->workspace;
  const RowsOf<T> r = gather<T>(a, p, true, s);
  LogitArgs<T> l = logit_args<T>(a, p, r);
  float* lse = (float*)(ws + p.at);
  hipLaunchKernelGGL(loss_take_kernel, dim3((unsigned)ceil_div(a->n_rows, 256)), dim3(256), 0, s, a->lse, r.rows, r.count, lse);
  l.lse = lse;
  l.dz = (T*)(ws + p.dz);
  l.ld_dz = p.piece;
  const int64_t c = a->channels, tiles_c = ceil_div(c, kTile);
  const float scale = a->scale / kRaise<T>;
  ProductArgs<T> d = {};
  d.dz = l.dz;
  d.count = r.count;
  d.ld_dz = p.piece;
  d.c = a->channels;
  d.ld = p.ld;
  for (int64_t r0 = 0; r0 < a->n_rows; r0 += p.chunk) {
    const int64_t row_tiles = ceil_div(std::min(p.chunk, a->n_rows - r0), kTile);
    const bool last = r0 + p.chunk >= a->n_rows;
    l.r0 = d.r0 = r0;
    l.r_most = d.r_most = p.chunk;
    for (int64_t k0 = 0; k0 < a->n_kinds; k0 += p.piece) {
      l.k0 = k0;
      l.k_end = std::min(a->n_kinds, k0 + p.piece);
      d.kinds = l.k_end - k0;
      const int64_t k_tiles = ceil_div(d.kinds, kTile);
      if (p.steps) walk_launch<true>(p.steps, l, (unsigned)std::min<int64_t>(kWalkGrid, most_results(p.chunk, p.tile_rows, d.kinds) / p.tile_rows), s);
      else hipLaunchKernelGGL(loss_dz_kernel<T>, dim3((unsigned)(row_tiles * k_tiles)), dim3(kGemmThreads), 0, s, l);
      if (a->grad_x) {
        d.b = l.table + k0 * p.ld;
        d.planes = (float*)(ws + p.dx);
        d.splits = p.dx_splits;
        d.first = k0 == 0;
        hipLaunchKernelGGL(loss_dx_kernel<T>, dim3((unsigned)(row_tiles * tiles_c * d.splits)), dim3(kGemmThreads), 0, s, d);
      }
      if (a->grad_table) {
        d.b = r.to_g + r0 * p.ld;
        d.planes = (float*)(ws + p.dw);
        d.splits = p.dw_splits;
        hipLaunchKernelGGL(loss_dw_kernel<T>, dim3((unsigned)(k_tiles * tiles_c * d.splits)), dim3(kGemmThreads), 0, s, d);
        hipLaunchKernelGGL(loss_dw_join_kernel<T>, dim3((unsigned)ceil_div(d.kinds * c, 256)), dim3(256), 0, s, d.planes, d.splits, d.kinds * c,
                           r.tops + p.blocks, scale, r0 == 0, last, (float*)(ws + p.sums) + k0 * c, (T*)a->grad_table + k0 * c);
      }
    }
    if (a->grad_x)
      hipLaunchKernelGGL(loss_dx_join_kernel<T>, dim3((unsigned)ceil_div(std::min(p.chunk, a->n_rows - r0) * c, 256)), dim3(256), 0, s,
                         (const float*)(ws + p.dx), p.dx_splits, r.rows, r.row_g, r.count, r0, p.chunk, a->channels, scale, (T*)a->grad_x);
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
