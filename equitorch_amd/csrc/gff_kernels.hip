// Gated feed-forward block on invariant channels (cgtp_gff_forward, cgtp_gff_backward):
//
//   g = x Wg,  u = x Wu,  m = act(g) * u,  y = m Wd
//   dm = dy Wd^T,  dg = dm * u * act'(g),  du = dm * act(g),
//   dx = dg Wg^T + du Wu^T,  dWg = x^T dg,  dWu = x^T du,  dWd = m^T dy
//
// x (rows, C_in), Wg, Wu (C_in, H), Wd (H, C_out).  Every product is formed in fp32; m, g, u, dg and du are rounded to the
// operands' type where they are stored, as operands of the next product: the same rounding the inputs have.
//
// 65536 rows of 256 -> 1024 -> 256 channels, bf16, forward and backward: 566 us (the kernels' own figures below are from a trace, one
// after the other, and come to 657).  No pipe is full: the products use a third of the
// matrix cores' cycles at most, LDS a third; with three workgroups on a compute unit a product's short run over k (four tiles
// of 256 channels) and its results alternate.  Two products at a time in one kernel, with 128 rows' operands and results in
// registers, were measured too: 504 us here, but 391 against 362 at 40000 rows, where the last of its few large
// workgroups run alone, and no faster for narrower channels.
#include "gff_gemm.h"

#include <algorithm>
#include <type_traits>

namespace cgtp {
namespace {

constexpr int kActs = 3;       // CGTP_ACT_SILU, CGTP_ACT_GELU, CGTP_ACT_SIGMOID

// act(g) and its derivative.  16-bit types take the hardware's exponential and reciprocal (1e-6
// relative), fp32 the library's.
template <typename T>
__device__ __forceinline__ float gff_sigmoid(float g) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.f + __expf(-g));
  else return 1.f / (1.f + expf(-g));
}
template <typename T, int act>
__device__ __forceinline__ float gff_act(float g) {
  if constexpr (act == CGTP_ACT_GELU) return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
  const float s = gff_sigmoid<T>(g);
  return act == CGTP_ACT_SILU ? g * s : s;
}
template <typename T, int act>
__device__ __forceinline__ float gff_act_grad(float g, float& value) {
  if constexpr (act == CGTP_ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    value = g * cdf;
    return cdf + g * 0.3989422804014327f * expf(-0.5f * g * g);
  }
  const float s = gff_sigmoid<T>(g);
  if constexpr (act == CGTP_ACT_SILU) {
    value = g * s;
    return s + value * (1.f - s);
  }
  value = s;
  return s * (1.f - s);
}

// Workgroups go to the eight XCDs in turn: the tiles of one outer index (which share a panel of an operand) are given to
// one XCD, whose L2 then reads the panel once.
struct TilePlace { int64_t outer; int inner; };
__device__ __forceinline__ TilePlace tile_place(int inner_tiles) {
  const int64_t id = (int64_t)blockIdx.x >> 3;
  return {id / inner_tiles * 8 + (blockIdx.x & 7), (int)(id % inner_tiles)};
}
unsigned tile_grid(int64_t outer, int64_t inner) { return (unsigned)((outer + 7) / 8 * 8 * inner); }

__device__ __forceinline__ int left_of(int64_t n, int64_t from, int most) { return (int)(n - from < most ? n - from : most); }

// LDS of a workgroup: the two operands' tiles, then the results.
template <int TILE> constexpr int kGemmLds = TILE * 256;

template <typename T>
struct UpArgs {
  const T *x, *wg, *wu;
  T *gate, *up, *mid;            // gate and up may be null (inference)
  int64_t n_rows;
  int C, H, ldx, ldw, ldh;       // elements between rows: of x, of the weights, of g, u and m
};

// Eight values of what is kept between the products, whose rows are whole groups of eight.  WHOLE: what lies beyond the row's
// end is read by the next product, against zeros, so it has to be finite.
template <bool WHOLE, typename T>
__device__ __forceinline__ void store_kept(T* to, const float (&v)[8], int left) {
  if (WHOLE && left < 8) {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = e < left ? v[e] : 0.f;
    store_eight(to, w, 8);
  } else {
    store_eight(to, v, WHOLE ? 8 : left);
  }
}

// 65536 rows as above: 162 us, 2.5 TB/s written.
// g, u and m.  A tile is TILE rows x TILE / 2 hidden channels, of Wg and of Wu.
template <typename T, int TILE, bool FAST, int ACT>
__global__ void __launch_bounds__(kGemmThreads, TILE == 128 ? 3 : 4) gff_up_kernel(UpArgs<T> a) {
  __shared__ alignas(16) char lds[kGemmLds<TILE>];
  constexpr int D = GemmType<T>::kDepth, kCols = TILE / 2;
  const TilePlace at = tile_place((a.H + kCols - 1) / kCols);
  const int64_t m0 = at.outer * TILE;
  if (m0 >= a.n_rows) return;
  const int h0 = at.inner * kCols;
  const GemmOperand<T> x = {{a.x + m0 * a.ldx, nullptr}, a.ldx, {left_of(a.n_rows, m0, TILE), 0}};
  const GemmOperand<T> w = {{a.wg + h0, a.wu + h0}, a.ldw, {a.H - h0, a.H - h0}};
  GemmAcc<TILE> acc;
  gemm_loop<T, TILE, FAST, true, false, true>(acc, lds, (a.C + D - 1) / D, [&](int64_t t, int64_t& k0, int64_t& depth) {
    k0 = t * D;
    depth = a.C;
    return x;
  }, [&](int64_t) { return w; });
  gemm_results<TILE, true, 4>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, const float (&g)[8], const float (&u)[8]) {
    const int left = a.H - h0 - c;
    if (r >= x.rows[0] || left <= 0) return;
    const int64_t to = (m0 + r) * a.ldh + h0 + c;
    float m[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = gff_act<T, ACT>(g[e]) * u[e];
    store_kept<FAST>(a.mid + to, m, left);
    if (a.gate) {
      store_kept<FAST>(a.gate + to, g, left);
      store_kept<FAST>(a.up + to, u, left);
    }
  });
}

template <typename T>
struct MidGradArgs {
  const T *gy, *wd, *gate, *up;
  T *g_gate, *g_up;
  int64_t n_rows;
  int H, C, ldg, ldw, ldh;
};

// dg and du from dm = dy Wd^T.  139 us, 4.0 TB/s: bound by memory, the projections read and their gradients written.
template <typename T, int TILE, bool FAST, int ACT>
__global__ void __launch_bounds__(kGemmThreads, TILE == 128 ? 3 : 4) gff_mid_grad_kernel(MidGradArgs<T> a) {
  __shared__ alignas(16) char lds[kGemmLds<TILE>];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place((a.H + TILE - 1) / TILE);
  const int64_t m0 = at.outer * TILE;
  if (m0 >= a.n_rows) return;
  const int h0 = at.inner * TILE;
  const GemmOperand<T> gy = {{a.gy + m0 * a.ldg, nullptr}, a.ldg, {left_of(a.n_rows, m0, TILE), 0}};
  const GemmOperand<T> wd = {{a.wd + (int64_t)h0 * a.ldw, nullptr}, a.ldw, {left_of(a.H, h0, TILE), 0}};
  GemmAcc<TILE> acc;
  gemm_loop<T, TILE, FAST, true, true, false>(acc, lds, (a.C + D - 1) / D, [&](int64_t t, int64_t& k0, int64_t& depth) {
    k0 = t * D;
    depth = a.C;
    return gy;
  }, [&](int64_t) { return wd; });
  // The projections' part is fetched a few places ahead of its use: one wait for memory in place of one for each place.
  constexpr int kAhead = sizeof(T) == 2 ? 4 : 2;
  EightRaw<T> pg[kAhead], pu[kAhead];
  auto fetch = [&](int p, int r, int c) {
    const int left = a.H - h0 - c;
    if (r >= gy.rows[0] || left <= 0) return;
    const int64_t from = (m0 + r) * a.ldh + h0 + c;
    pg[p % kAhead].load(a.gate + from, FAST ? 8 : left);
    pu[p % kAhead].load(a.up + from, FAST ? 8 : left);
  };
  gemm_results<TILE, false, kAhead>(acc, lds, fetch, [&](int p, int r, int c, const float (&dm)[8]) {
    const int left = a.H - h0 - c;
    if (r >= gy.rows[0] || left <= 0) return;
    const int64_t to = (m0 + r) * a.ldh + h0 + c;
    float g[8], u[8];
    pg[p % kAhead].get(g);
    pu[p % kAhead].get(u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float value;
      const float slope = gff_act_grad<T, ACT>(g[e], value);
      g[e] = dm[e] * u[e] * slope;
      u[e] = dm[e] * value;
    }
    store_kept<FAST>(a.g_gate + to, g, left);
    store_kept<FAST>(a.g_up + to, u, left);
  });
}

// How operands and results lie: whole aligned groups of eight elements; operands so, results not; neither (small calls).
enum { kWhole, kPacked, kLoose };

// out = sum over segments of A_s B_s: y = m Wd (one segment), dx = dg Wg^T + du Wu^T (two).  A is contiguous along k.  The
// tiles of k are cut into `splits` ranges where the result has few tiles; a range's result is left in fp32 and the ranges
// are added in order by gff_add_kernel.  y 63 us, dx 116 us (545 and 590 TFLOP/s).
template <typename T>
struct RowsArgs {
  const T *a[2], *b[2];
  T* out;
  float* parts;
  int64_t n_rows, lda, ldb;
  int segments, K, N, splits;      // K: per segment
};
template <typename T, int TILE, int MODE, bool KB>
__global__ void __launch_bounds__(kGemmThreads, TILE == 128 ? 3 : 4) gff_rows_kernel(RowsArgs<T> a) {
  __shared__ alignas(16) char lds[kGemmLds<TILE>];
  constexpr int D = GemmType<T>::kDepth;
  const int tiles_n = (a.N + TILE - 1) / TILE;
  const TilePlace at = tile_place(tiles_n * a.splits);
  const int64_t m0 = at.outer * TILE;
  if (m0 >= a.n_rows) return;
  const int split = at.inner / tiles_n, n0 = at.inner % tiles_n * TILE;
  const int tiles = (a.K + D - 1) / D, all = tiles * a.segments, each = (all + a.splits - 1) / a.splits, first = split * each;
  const int rows = left_of(a.n_rows, m0, TILE), cols = left_of(a.N, n0, TILE);
  GemmAcc<TILE> acc;
  gemm_loop<T, TILE, MODE != kLoose, true, KB, false>(acc, lds, std::min(each, all - first), [&](int64_t t, int64_t& k0, int64_t& depth) {
    t += first;
    k0 = (t < tiles ? t : t - tiles) * D;
    depth = a.K;
    return GemmOperand<T>{{(t < tiles ? a.a[0] : a.a[1]) + m0 * a.lda, nullptr}, a.lda, {rows, 0}};
  }, [&](int64_t t) {
    const T* b = t + first < tiles ? a.b[0] : a.b[1];
    if (KB) return GemmOperand<T>{{b + n0 * a.ldb, nullptr}, a.ldb, {cols, 0}};
    return GemmOperand<T>{{b + n0, b + n0 + TILE / 2}, a.ldb, {cols, cols - TILE / 2}};
  });
  gemm_results<TILE, false, 8>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, const float (&v)[8]) {
    const int left = a.N - n0 - c;
    if (r >= rows || left <= 0) return;
    const int64_t to = (m0 + r) * a.N + n0 + c;
    if (a.splits > 1) store_eight(a.parts + split * a.n_rows * a.N + to, v, MODE == kWhole ? 8 : left);
    else store_eight(a.out + to, v, MODE == kWhole ? 8 : left);
  });
}

// Weight gradients out_j = A_j^T B_j over all rows: both operands contiguous along the tile's rows.  The rows are cut
// into `splits` ranges, as above.  167 us, 620 TFLOP/s, where the library's product takes 272.
template <typename T>
struct WeightJob {
  const T *a, *b;
  T* out;
  int M, N, lda, ldb, first_tile, tiles_n;      // first tile of the job among all jobs' tiles
  int64_t first_part;                 // first element of the job in a range's partial results
};
template <typename T>
struct WeightArgs {
  WeightJob<T> job[3];
  float* parts;
  int64_t n_rows, rows_per_split, part_elems;
  int jobs, tiles, splits;
};
template <typename T, int TILE, int MODE>
__global__ void __launch_bounds__(kGemmThreads, TILE == 128 ? 3 : 4) gff_weight_kernel(WeightArgs<T> w) {
  __shared__ alignas(16) char lds[kGemmLds<TILE>];
  constexpr int D = GemmType<T>::kDepth, kCut = TILE / 2;
  const TilePlace at = tile_place(w.tiles);
  if (at.outer >= w.splits) return;
  const int which = w.jobs > 2 && at.inner >= w.job[2].first_tile ? 2 : w.jobs > 1 && at.inner >= w.job[1].first_tile ? 1 : 0;
  const WeightJob<T> job = w.job[which];
  const int tile = at.inner - job.first_tile;
  const int m0 = tile / job.tiles_n * TILE, n0 = tile % job.tiles_n * TILE;
  const int64_t r0 = at.outer * w.rows_per_split;
  const int64_t end = std::min(w.rows_per_split, w.n_rows - r0);
  const int rows = left_of(job.M, m0, TILE), cols = left_of(job.N, n0, TILE);
  const T *ja = job.a + r0 * job.lda + m0, *jb = job.b + r0 * job.ldb + n0;
  const GemmOperand<T> pa = {{ja, ja + kCut}, job.lda, {rows, rows - kCut}}, pb = {{jb, jb + kCut}, job.ldb, {cols, cols - kCut}};
  GemmAcc<TILE> acc;
  gemm_loop<T, TILE, MODE != kLoose, false, false, false>(acc, lds, (end + D - 1) / D, [&](int64_t t, int64_t& k0, int64_t& depth) {
    k0 = t * D;
    depth = end;
    return pa;
  }, [&](int64_t) { return pb; });
  gemm_results<TILE, false, 8>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, const float (&v)[8]) {
    const int left = job.N - n0 - c;
    if (r >= rows || left <= 0) return;
    const int64_t to = (int64_t)(m0 + r) * job.N + n0 + c;
    if (w.splits > 1) store_eight(w.parts + at.outer * w.part_elems + job.first_part + to, v, MODE == kWhole ? 8 : left);
    else store_eight(job.out + to, v, MODE == kWhole ? 8 : left);
  });
}

// out[i] = sum over the ranges of their partial results, in order.  Up to three outputs, one after the other in a range's part.
template <typename T>
struct AddArgs {
  const float* parts;
  T* out[3];
  int64_t first[3], elems;
  int outs, splits;
};
template <typename T>
__global__ void __launch_bounds__(256) gff_add_kernel(AddArgs<T> a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.elems) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < a.splits; ++k) s += a.parts[k * a.elems + i];
  const int which = a.outs > 2 && i >= a.first[2] ? 2 : a.outs > 1 && i >= a.first[1] ? 1 : 0;
  a.out[which][i - a.first[which]] = (T)s;
}

// Copies of up to five operands whose rows do not start at multiples of eight elements, with rows that do and zeros at their
// ends: read once and written once, while a product reads an operand's tiles many times.
template <typename T>
struct PackArgs {
  const T* from[5];
  T* to[5];
  int64_t groups[5];        // groups: up to and with this operand
  int cols[5];
  int n;
};
template <typename T>
__global__ void __launch_bounds__(256) gff_pack_kernel(PackArgs<T> a) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.groups[a.n - 1]; i += step) {
    int j = 0;
    while (i >= a.groups[j]) ++j;
    const int64_t at = i - (j ? a.groups[j - 1] : 0);
    const unsigned each = (a.cols[j] + 7) / 8;
    const int64_t r = at / each;
    const int c = (int)(at - r * each) * 8;
    EightRaw<T> v;
    v.load(a.from[j] + r * a.cols[j] + c, a.cols[j] - c);
#pragma unroll
    for (int k = 0; k < 8 / EightRaw<T>::N; ++k) *reinterpret_cast<u32x4_t*>(a.to[j] + at * 8 + k * EightRaw<T>::N) = v.v[k];
  }
}

// A handful of rows: the weights are read once for all of them and nothing else counts.  A workgroup takes 32 columns, a
// thread eight of them at every 64th k, in fp32; the 64 sums of a column are added in LDS in a fixed order.
// MATS = 2: x against Wg and Wu, then the activation and the product; MATS = 1: m against Wd.  Bound by latency: one row of
// 256 -> 1024 -> 256 channels, bf16, 4.4 and 7.7 us.
constexpr int kFewRows = 4, kFewCols = 32, kFewSlices = 64;
template <typename T>
struct FewArgs {
  const T *x, *w[2];
  T *gate, *up, *out;
  int n_rows, K, N, ldx, ldo;      // elements between rows of x, of the results
};
template <typename T, int ROWS, int MATS, int ACT>
__global__ void __launch_bounds__(256) gff_few_kernel(FewArgs<T> a) {
  constexpr int kSums = kFewCols * MATS;
  __shared__ float sums[kFewSlices][kSums + 4];
  const int n0 = blockIdx.x * kFewCols, group = threadIdx.x & 3, slice = threadIdx.x >> 2, n = n0 + group * 8, left = a.N - n;
  float acc[ROWS][MATS][8];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][m][e] = 0.f;
  if (left > 0) {
    constexpr int kAhead = ROWS == 1 ? 16 / (MATS * (int)sizeof(T) / 2) : 4;      // loads on their way: 16
    for (int k0 = slice; k0 < a.K; k0 += kFewSlices * kAhead) {
      EightRaw<T> w[kAhead][MATS];
      float x[kAhead][ROWS];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int k = k0 + j * kFewSlices;
        const bool in = k < a.K;
#pragma unroll
        for (int m = 0; m < MATS; ++m) w[j][m].load(a.w[m] + (int64_t)(in ? k : k0) * a.N + n, left);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) x[j][r] = r < a.n_rows && in ? (float)a.x[(int64_t)r * a.ldx + k] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (k0 + j * kFewSlices >= a.K) continue;        // not even 0 times what is read in its place
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          float v[8];
          w[j][m].get(v);
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r][m][e] = fmaf(x[j][r], v[e], acc[r][m][e]);
        }
      }
    }
  }
  // 256 / kSums threads for each sum, then one
  constexpr int kParts = 256 / kSums, kPer = kFewSlices / kParts;
  __shared__ float last[256];
  for (int r = 0; r < ROWS && r < a.n_rows; ++r) {
    __syncthreads();
#pragma unroll
    for (int rr = 0; rr < ROWS; ++rr)
      if (rr == r)
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
          for (int e = 0; e < 8; ++e) sums[slice][m * kFewCols + group * 8 + e] = acc[rr][m][e];
    __syncthreads();
    const int c = threadIdx.x % kSums, part = threadIdx.x / kSums;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) s += sums[part * kPer + k][c];
    last[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < kFewCols && n0 + (int)threadIdx.x < a.N) {
      float t[MATS];
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        t[m] = 0.f;
#pragma unroll
        for (int p = 0; p < kParts; ++p) t[m] += last[p * kSums + m * kFewCols + threadIdx.x];
      }
      const int64_t to = (int64_t)r * a.ldo + n0 + threadIdx.x;
      if constexpr (MATS == 2) {
        a.out[to] = (T)(gff_act<T, ACT>(t[0]) * t[1]);
        if (a.gate) {
          a.gate[to] = (T)t[0];
          a.up[to] = (T)t[1];
        }
      } else {
        a.out[to] = (T)t[0];
      }
    }
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------
int gff_check(const cgtp_gff_args* a) {
  if (!a) return CGTP_ERR_NULL;
  if (a->dtype != CGTP_F32 && a->dtype != CGTP_BF16 && a->dtype != CGTP_F16) return CGTP_ERR_DTYPE;
  if (a->n_rows < 0 || a->n_rows > 0x7fffffff || a->c_in <= 0 || a->c_out <= 0 || a->hidden <= 0) return CGTP_ERR_SHAPE;
  if (a->c_in > 0x7fff || a->c_out > 0x7fff || a->hidden > 0x1ffff) return CGTP_ERR_SHAPE;
  // A grid has fewer than 2^32 threads, 2^24 workgroups.  That many tiles are of 128 rows (those of 64 are for results of fewer than 256
  // tiles of 128), by 64 hidden channels or 128 of x or out, and their rows are rounded up to eight tiles.
  const int64_t cols = std::max({(a->hidden + 63) / 64, (a->c_in + 127) / 128, (a->c_out + 127) / 128});
  if ((a->n_rows + 1023) / 1024 * 8 * cols >= (1 << 24)) return CGTP_ERR_SHAPE;
  if (a->activation < 0 || a->activation >= kActs) return CGTP_ERR_CONFIG;
  if (!a->w_gate || !a->w_up || !a->w_down) return CGTP_ERR_NULL;
  if (a->n_rows > 0 && !a->x) return CGTP_ERR_NULL;
  return CGTP_OK;
}

// What is kept between the products, and the workspace, start at multiples of 16 bytes.
bool kept_aligned(const cgtp_gff_args* a) {
  const void* kept[] = {a->gate, a->up, a->mid, a->grad_gate, a->grad_up, a->workspace};
  for (const void* p : kept)
    if (!aligned16(p)) return false;
  return true;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles of 128 (fewer bytes from memory and LDS for each product) where they give every compute unit a workgroup, else of 64:
// 3001 rows of 128 -> 512 channels, fp32, forward and backward 200 us of kernels with tiles of 128 alone, 89 with these.
bool small_tiles(int64_t tiles_of_128) { return tiles_of_128 < 256; }

int padded(int n) { return (n + 7) & ~7; }

// How a call's operands and results lie.  Rows that are not whole aligned groups are copied first where tiles of 128 are worth
// having: reading such rows takes those tiles more registers than there are.  bf16, forward: 20000 rows of 253 -> 1021
// channels 205 us read in place, 67 copied (256 -> 1024: 62), 3000 of 301 -> 701 59 and 31; below, 500 of 301 -> 701, 20 in
// place, where aligned rows take 17 without the copy's 4.
int mode_of(const cgtp_gff_args* a) {
  const void* ptrs[] = {a->x, a->w_gate, a->w_up, a->w_down, a->out, a->grad_out, a->grad_x, a->grad_w_gate, a->grad_w_up,
                        a->grad_w_down};
  bool whole = a->c_in % 8 == 0 && a->hidden % 8 == 0 && a->c_out % 8 == 0;      // hidden < 2^17: 128 rows of it are below 2^26 bytes
  for (const void* p : ptrs) whole = whole && aligned16(p);
  if (whole) return kWhole;
  return small_tiles(ceil_div(a->n_rows, 128) * ceil_div(a->hidden, 64)) ? kLoose : kPacked;
}

// Ranges that k is cut into for a product of `tiles` results: two workgroups for each compute unit, at least four tiles of k.
int ranges_of(int64_t tiles, int64_t k_tiles) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(tiles < 256 ? 512 / std::max<int64_t>(1, tiles) : 1, k_tiles / 4));
}

struct RowsShape { int tile, splits; };
RowsShape rows_shape(int mode, int64_t n_rows, int N, int64_t k_tiles) {
  RowsShape s;
  s.tile = mode == kLoose || small_tiles(ceil_div(n_rows, 128) * ceil_div(N, 128)) ? 64 : 128;
  s.splits = s.tile == 64 ? ranges_of(ceil_div(n_rows, 64) * ceil_div(N, 64), k_tiles) : 1;
  return s;
}

// The weight gradients' rows: three workgroups for each compute unit, at least eight k tiles each.
struct WeightShape { int tile, splits; int64_t rows_per_split, part_elems; };
WeightShape weight_shape(int mode, const cgtp_gff_args* a) {
  WeightShape s;
  auto tiles = [&](int t) { return ceil_div(a->hidden, t) * (2 * ceil_div(a->c_in, t) + ceil_div(a->c_out, t)); };
  const int depth = a->dtype == CGTP_F32 ? 32 : 64;
  const int64_t most = ceil_div(a->n_rows, 8 * depth);
  s.tile = mode == kLoose || small_tiles(tiles(128) * most) ? 64 : 128;
  s.part_elems = (int64_t)a->hidden * (2 * a->c_in + a->c_out);
  int64_t splits = std::max<int64_t>(1, std::min(std::max<int64_t>(1, 768 / tiles(s.tile)), most));
  if (splits > 8) splits = splits / 8 * 8;           // a range's tiles run on one XCD: as many ranges for each of the eight
  s.rows_per_split = ceil_div(ceil_div(a->n_rows, splits), depth) * depth;
  s.splits = (int)std::max<int64_t>(1, ceil_div(a->n_rows, std::max<int64_t>(1, s.rows_per_split)));
  return s;
}

int64_t k_tiles_of(const cgtp_gff_args* a) { return ceil_div(a->hidden, a->dtype == CGTP_F32 ? 32 : 64); }

// Rows that gff_few_kernel takes.  In 16-bit types the matrix cores' tiles overtake it from the second row on: 4 rows of 500 -> 2000
// channels, bf16, 39 us against 19, fp32 21 against 45; 256 -> 1024 28 against 17, 15 against 19.
bool few_rows(const cgtp_gff_args* a) { return a->n_rows <= (a->dtype == CGTP_F32 ? kFewRows : 1); }

// Bytes of an operand's copy, zero where none is made.
int64_t copy_bytes(const cgtp_gff_args* a, int64_t rows, int cols) { return (rows * padded(cols) * (a->dtype == CGTP_F32 ? 4 : 2) + 15) / 16 * 16; }

// Partial results, then the copies: x, the weights, for a backward the gradient of the output.
struct Workspace { int64_t parts, all; };
Workspace workspace_of(const cgtp_gff_args* a, bool backward) {
  if (!backward && few_rows(a)) return {0, 0};
  const int mode = mode_of(a);
  auto rows = [&](int N, int64_t k_tiles) {
    const RowsShape s = rows_shape(mode, a->n_rows, N, k_tiles);
    return s.splits > 1 ? s.splits * a->n_rows * N * 4 : 0;
  };
  Workspace w = {};
  if (backward) {
    const WeightShape g = weight_shape(mode, a);
    w.parts = std::max(rows(a->c_in, 2 * k_tiles_of(a)), g.splits > 1 ? g.splits * g.part_elems * 4 : 0);
  } else {
    w.parts = rows(a->c_out, k_tiles_of(a));
  }
  w.parts = (w.parts + 15) / 16 * 16;
  w.all = w.parts;
  if (mode == kPacked)
    w.all += copy_bytes(a, a->n_rows, a->c_in) + 2 * copy_bytes(a, a->c_in, a->hidden) + copy_bytes(a, a->hidden, a->c_out) +
             (backward ? copy_bytes(a, a->n_rows, a->c_out) : 0);
  return w;
}

// The operands as the kernels read them.
template <typename T>
struct Operands {
  const T *x, *wg, *wu, *wd, *gy;
  int mode, ldx, ldw, ldd, ldh;      // elements between rows: x, Wg and Wu, Wd and dy, what is kept between the products
};
template <typename T>
Operands<T> operands_of(const cgtp_gff_args* a, bool backward, hipStream_t s) {
  Operands<T> o = {(const T*)a->x, (const T*)a->w_gate, (const T*)a->w_up, (const T*)a->w_down, (const T*)a->grad_out, mode_of(a),
                   a->c_in, a->hidden, a->c_out, padded(a->hidden)};
  if (o.mode != kPacked) return o;
  char* at = (char*)a->workspace + workspace_of(a, backward).parts;
  PackArgs<T> p = {};
  auto copy = [&](const T*& from, int64_t rows, int cols) {
    p.from[p.n] = from;
    p.to[p.n] = (T*)at;
    p.cols[p.n] = cols;
    p.groups[p.n] = (p.n ? p.groups[p.n - 1] : 0) + rows * (padded(cols) / 8);
    ++p.n;
    from = (const T*)at;
    at += copy_bytes(a, rows, cols);
  };
  copy(o.x, a->n_rows, a->c_in);
  copy(o.wg, a->c_in, a->hidden);
  copy(o.wu, a->c_in, a->hidden);
  copy(o.wd, a->hidden, a->c_out);
  if (backward) copy(o.gy, a->n_rows, a->c_out);
  o.ldx = padded(a->c_in);
  o.ldw = padded(a->hidden);
  o.ldd = padded(a->c_out);
  hipLaunchKernelGGL(gff_pack_kernel<T>, dim3((unsigned)std::min<int64_t>(ceil_div(p.groups[p.n - 1], 256), 1 << 16)), dim3(256), 0, s, p);
  return o;
}

// The kernel of an activation: a branch on it for each element costs more than the activation.
template <typename Kernel, typename Of>
Kernel for_act(int act, Of&& of) {
  if (act == CGTP_ACT_SILU) return of(std::integral_constant<int, CGTP_ACT_SILU>{});
  if (act == CGTP_ACT_GELU) return of(std::integral_constant<int, CGTP_ACT_GELU>{});
  return of(std::integral_constant<int, CGTP_ACT_SIGMOID>{});
}
template <typename Kernel, typename Of>
Kernel for_tile(int tile, int mode, Of&& of) {
  typedef std::integral_constant<int, 64> small;
  typedef std::integral_constant<int, 128> large;
  typedef std::integral_constant<int, kWhole> whole;
  typedef std::integral_constant<int, kPacked> packed;
  if (mode == kLoose) return of(small{}, std::integral_constant<int, kLoose>{});
  if (mode == kPacked) return tile == 64 ? of(small{}, packed{}) : of(large{}, packed{});
  return tile == 64 ? of(small{}, whole{}) : of(large{}, whole{});
}

template <typename T>
void add_launch(const AddArgs<T>& a, hipStream_t s) {
  hipLaunchKernelGGL(gff_add_kernel<T>, dim3((unsigned)ceil_div(a.elems, 256)), dim3(256), 0, s, a);
}

template <typename T, bool KB>
void rows_launch(RowsArgs<T> d, int mode, void* workspace, hipStream_t s) {
  const RowsShape shape = rows_shape(mode, d.n_rows, d.N, d.segments * ceil_div(d.K, GemmType<T>::kDepth));
  d.splits = shape.splits;
  d.parts = (float*)workspace;
  auto kern = for_tile<void (*)(RowsArgs<T>)>(shape.tile, mode, [](auto tile, auto m) {
    return gff_rows_kernel<T, decltype(tile)::value, decltype(m)::value, KB>;
  });
  const int64_t mt = ceil_div(d.n_rows, shape.tile), nt = ceil_div(d.N, shape.tile);
  hipLaunchKernelGGL(kern, dim3(tile_grid(mt, nt * d.splits)), dim3(kGemmThreads), 0, s, d);
  if (d.splits > 1) add_launch(AddArgs<T>{d.parts, {d.out, nullptr, nullptr}, {0, 0, 0}, d.n_rows * d.N, 1, d.splits}, s);
}

template <typename T, int ROWS>
void few_launch(const cgtp_gff_args* a, hipStream_t s) {
  const FewArgs<T> u = {(const T*)a->x, {(const T*)a->w_gate, (const T*)a->w_up}, (T*)a->gate, (T*)a->up, (T*)a->mid,
                        (int)a->n_rows, a->c_in, a->hidden, a->c_in, padded(a->hidden)};
  auto up = for_act<void (*)(FewArgs<T>)>(a->activation, [](auto act) { return gff_few_kernel<T, ROWS, 2, decltype(act)::value>; });
  hipLaunchKernelGGL(up, dim3((unsigned)ceil_div(u.N, kFewCols)), dim3(256), 0, s, u);
  const FewArgs<T> d = {(const T*)a->mid, {(const T*)a->w_down, nullptr}, nullptr, nullptr, (T*)a->out, (int)a->n_rows, a->hidden,
                        a->c_out, padded(a->hidden), a->c_out};
  hipLaunchKernelGGL((gff_few_kernel<T, ROWS, 1, 0>), dim3((unsigned)ceil_div(d.N, kFewCols)), dim3(256), 0, s, d);
}

template <typename T>
int gff_forward(const cgtp_gff_args* a, hipStream_t s) {
  if (few_rows(a)) {
    if (a->n_rows == 1) few_launch<T, 1>(a, s);
    else if constexpr (sizeof(T) == 4) few_launch<T, kFewRows>(a, s);
    return launch_status();
  }
  const Operands<T> o = operands_of<T>(a, false, s);
  const UpArgs<T> u = {o.x, o.wg, o.wu, (T*)a->gate, (T*)a->up, (T*)a->mid, a->n_rows, a->c_in, a->hidden, o.ldx, o.ldw, o.ldh};
  const int tile = o.mode == kLoose || small_tiles(ceil_div(a->n_rows, 128) * ceil_div(a->hidden, 64)) ? 64 : 128;
  auto up = for_act<void (*)(UpArgs<T>)>(a->activation, [&](auto act) {
    return for_tile<void (*)(UpArgs<T>)>(tile, o.mode, [](auto t, auto m) {
      return gff_up_kernel<T, decltype(t)::value, decltype(m)::value != kLoose, decltype(act)::value>;
    });
  });
  hipLaunchKernelGGL(up, dim3(tile_grid(ceil_div(a->n_rows, tile), ceil_div(a->hidden, tile / 2))), dim3(kGemmThreads), 0, s, u);
  rows_launch<T, false>(RowsArgs<T>{{(const T*)a->mid, nullptr}, {o.wd, nullptr}, (T*)a->out, nullptr, a->n_rows, o.ldh, o.ldd, 1,
                                    a->hidden, a->c_out, 1}, o.mode, a->workspace, s);
  return launch_status();
}

template <typename T>
int gff_backward(const cgtp_gff_args* a, hipStream_t s) {
  if (!a->grad_x && !a->grad_w_gate && !a->grad_w_up && !a->grad_w_down) return CGTP_OK;
  const Operands<T> o = operands_of<T>(a, true, s);
  if (a->n_rows > 0 && (a->grad_x || a->grad_w_gate || a->grad_w_up)) {
    const MidGradArgs<T> m = {o.gy, o.wd, (const T*)a->gate, (const T*)a->up, (T*)a->grad_gate, (T*)a->grad_up, a->n_rows, a->hidden,
                              a->c_out, o.ldd, o.ldd, o.ldh};
    const int tile = o.mode == kLoose || small_tiles(ceil_div(a->n_rows, 128) * ceil_div(a->hidden, 128)) ? 64 : 128;
    auto mid = for_act<void (*)(MidGradArgs<T>)>(a->activation, [&](auto act) {
      return for_tile<void (*)(MidGradArgs<T>)>(tile, o.mode, [](auto t, auto m) {
        return gff_mid_grad_kernel<T, decltype(t)::value, decltype(m)::value != kLoose, decltype(act)::value>;
      });
    });
    hipLaunchKernelGGL(mid, dim3(tile_grid(ceil_div(a->n_rows, tile), ceil_div(a->hidden, tile))), dim3(kGemmThreads), 0, s, m);
  }
  if (a->n_rows > 0 && a->grad_x)
    rows_launch<T, true>(RowsArgs<T>{{(const T*)a->grad_gate, (const T*)a->grad_up}, {o.wg, o.wu}, (T*)a->grad_x, nullptr, a->n_rows,
                                     o.ldh, o.ldw, 2, a->hidden, a->c_in, 1}, o.mode, a->workspace, s);
  const WeightShape shape = weight_shape(o.mode, a);
  WeightArgs<T> w = {};
  AddArgs<T> sum = {};
  w.parts = (float*)a->workspace;
  w.n_rows = a->n_rows;
  w.rows_per_split = shape.rows_per_split;
  w.splits = shape.splits;
  auto job = [&](const T* l, const T* r, void* out, int M, int N, int lda, int ldb) {
    if (!out) return;
    sum.out[w.jobs] = (T*)out;
    sum.first[w.jobs] = w.part_elems;
    w.job[w.jobs++] = {l, r, (T*)out, M, N, lda, ldb, w.tiles, (int)ceil_div(N, shape.tile), w.part_elems};
    w.tiles += (int)(ceil_div(M, shape.tile) * ceil_div(N, shape.tile));
    w.part_elems += (int64_t)M * N;
  };
  job(o.x, (const T*)a->grad_gate, a->grad_w_gate, a->c_in, a->hidden, o.ldx, o.ldh);
  job(o.x, (const T*)a->grad_up, a->grad_w_up, a->c_in, a->hidden, o.ldx, o.ldh);
  job((const T*)a->mid, o.gy, a->grad_w_down, a->hidden, a->c_out, o.ldh, o.ldd);
  if (w.jobs) {
    auto weight = for_tile<void (*)(WeightArgs<T>)>(shape.tile, o.mode, [](auto t, auto m) {
      return gff_weight_kernel<T, decltype(t)::value, decltype(m)::value>;
    });
    hipLaunchKernelGGL(weight, dim3(tile_grid(w.splits, w.tiles)), dim3(kGemmThreads), 0, s, w);
    if (w.splits > 1) {
      sum.parts = w.parts;
      sum.elems = w.part_elems;
      sum.outs = w.jobs;
      sum.splits = w.splits;
      add_launch(sum, s);
    }
  }
  return launch_status();
}

}  // namespace
}  // namespace cgtp

extern "C" {

int64_t cgtp_gff_workspace_bytes(const cgtp_gff_args* a, int backward) {
  using namespace cgtp;
  return gff_check(a) == CGTP_OK && a->n_rows > 0 ? workspace_of(a, backward != 0).all : 0;
}

int cgtp_gff_forward(const cgtp_gff_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = gff_check(a)) return rc;
  if (a->n_rows == 0) return CGTP_OK;
  if (!a->mid || !a->out || (!a->gate) != (!a->up)) return CGTP_ERR_NULL;
  if (!kept_aligned(a)) return CGTP_ERR_ALIGN;
  if (workspace_of(a, false).all > 0 && !a->workspace) return CGTP_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case CGTP_F32: return gff_forward<float>(a, s);
    case CGTP_BF16: return gff_forward<bf16_t>(a, s);
    default: return gff_forward<f16_t>(a, s);
  }
}

int cgtp_gff_backward(const cgtp_gff_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = gff_check(a)) return rc;
  if (a->n_rows > 0 && (!a->grad_out || !a->gate || !a->up || !a->mid || !a->grad_gate || !a->grad_up)) return CGTP_ERR_NULL;
  if (!kept_aligned(a)) return CGTP_ERR_ALIGN;
  if (cgtp_gff_workspace_bytes(a, 1) > 0 && !a->workspace) return CGTP_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case CGTP_F32: return gff_backward<float>(a, s);
    case CGTP_BF16: return gff_backward<bf16_t>(a, s);
    default: return gff_backward<f16_t>(a, s);
  }
}

}  // extern "C"
