// Gated feed-forward block on invariant channels (cgtp_gff_forward, cgtp_gff_backward):
//
//   g = x Wg,  u = x Wu,  m = act(g) * u,  y = m Wd
//   dm = dy Wd^T,  dg = dm * u * act'(g),  du = dm * act(g),
//   dx = dg Wg^T + du Wu^T,  dWg = x^T dg,  dWu = x^T du,  dWd = m^T dy
//
// x (rows, C_in), Wg, Wu (C_in, H), Wd (H, C_out).  Every product is formed in fp32; m, g, u, dg and du are rounded to the
// operands' type where they are stored, as operands of the next product: the same rounding the inputs have.
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

template <typename T>
struct UpArgs {
  const T *x, *wg, *wu;
  T *gate, *up, *mid;            // gate and up may be null (inference)
  int64_t n_rows;
  int C, H;
};

__device__ __forceinline__ int rows_left(int64_t n, int64_t from) { return (int)(n - from < kGemmTile ? n - from : kGemmTile); }

// g, u and m.  A tile is 128 rows x 64 hidden channels, of Wg and of Wu.
template <typename T, bool FAST, int ACT>
__global__ void __launch_bounds__(kGemmThreads, 3) gff_up_kernel(UpArgs<T> a) {
  __shared__ alignas(16) char lds[2 * kGemmTileBytes];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place((a.H + 63) / 64);
  const int64_t m0 = at.outer * kGemmTile;
  if (m0 >= a.n_rows) return;
  const int h0 = at.inner * 64;
  const GemmOperand<T> w = {{a.wg + h0, a.wu + h0}, a.H, {a.H - h0, a.H - h0}};
  const GemmOperand<T> x = {{a.x + m0 * a.C, nullptr}, a.C, {rows_left(a.n_rows, m0), 0}};
  f32x16_t acc[2][2];
  gemm_loop<T, FAST, true, false, true>(acc, lds, (a.C + D - 1) / D, [&](int64_t t, int64_t& k0, int64_t& depth) {
    k0 = t * D;
    depth = a.C;
    return x;
  }, [&](int64_t) { return w; });
  gemm_results<true, 4>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, const float (&g)[8], const float (&u)[8]) {
    const int left = a.H - h0 - c;
    if (r >= x.rows[0] || left <= 0) return;
    const int64_t to = (m0 + r) * a.H + h0 + c;
    float m[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = gff_act<T, ACT>(g[e]) * u[e];
    store_eight(a.mid + to, m, FAST ? 8 : left);
    if (a.gate) {
      store_eight(a.gate + to, g, FAST ? 8 : left);
      store_eight(a.up + to, u, FAST ? 8 : left);
    }
  });
}

template <typename T>
struct MidGradArgs {
  const T *gy, *wd, *gate, *up;
  T *g_gate, *g_up;
  int64_t n_rows;
  int H, C;
};

// dg and du from dm = dy Wd^T.
template <typename T, bool FAST, int ACT>
__global__ void __launch_bounds__(kGemmThreads, 3) gff_mid_grad_kernel(MidGradArgs<T> a) {
  __shared__ alignas(16) char lds[2 * kGemmTileBytes];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place((a.H + kGemmTile - 1) / kGemmTile);
  const int64_t m0 = at.outer * kGemmTile;
  if (m0 >= a.n_rows) return;
  const int h0 = at.inner * kGemmTile;
  const GemmOperand<T> wd = {{a.wd + (int64_t)h0 * a.C, nullptr}, a.C, {rows_left(a.H, h0), 0}};
  const GemmOperand<T> gy = {{a.gy + m0 * a.C, nullptr}, a.C, {rows_left(a.n_rows, m0), 0}};
  f32x16_t acc[2][2];
  gemm_loop<T, FAST, true, true, false>(acc, lds, (a.C + D - 1) / D, [&](int64_t t, int64_t& k0, int64_t& depth) {
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
    const int64_t from = (m0 + r) * a.H + h0 + c;
    pg[p % kAhead].load(a.gate + from, FAST ? 8 : left);
    pu[p % kAhead].load(a.up + from, FAST ? 8 : left);
  };
  gemm_results<false, kAhead>(acc, lds, fetch, [&](int p, int r, int c, const float (&dm)[8]) {
    const int left = a.H - h0 - c;
    if (r >= gy.rows[0] || left <= 0) return;
    const int64_t to = (m0 + r) * a.H + h0 + c;
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
    store_eight(a.g_gate + to, g, FAST ? 8 : left);
    store_eight(a.g_up + to, u, FAST ? 8 : left);
  });
}

// out = sum over segments of A_s B_s: y = m Wd (one segment), dx = dg Wg^T + du Wu^T (two).  A is contiguous along k.
template <typename T>
struct RowsArgs {
  const T *a[2], *b[2];
  T* out;
  int64_t n_rows, ldb;
  int segments, K, N;      // K: per segment
};
template <typename T, bool FAST, bool KB>
__global__ void __launch_bounds__(kGemmThreads, 3) gff_rows_kernel(RowsArgs<T> a) {
  __shared__ alignas(16) char lds[2 * kGemmTileBytes];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place((a.N + kGemmTile - 1) / kGemmTile);
  const int64_t m0 = at.outer * kGemmTile;
  if (m0 >= a.n_rows) return;
  const int n0 = at.inner * kGemmTile, tiles = (a.K + D - 1) / D, rows = rows_left(a.n_rows, m0), cols = rows_left(a.N, n0);
  f32x16_t acc[2][2];
  gemm_loop<T, FAST, true, KB, false>(acc, lds, (int64_t)tiles * a.segments, [&](int64_t t, int64_t& k0, int64_t& depth) {
    k0 = (t < tiles ? t : t - tiles) * D;
    depth = a.K;
    return GemmOperand<T>{{(t < tiles ? a.a[0] : a.a[1]) + m0 * a.K, nullptr}, a.K, {rows, 0}};
  }, [&](int64_t t) {
    const T* b = t < tiles ? a.b[0] : a.b[1];
    if (KB) return GemmOperand<T>{{b + n0 * a.ldb, nullptr}, a.ldb, {cols, 0}};
    return GemmOperand<T>{{b + n0, b + n0 + 64}, a.ldb, {cols, cols - 64}};
  });
  gemm_results<false, 8>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, const float (&v)[8]) {
    const int left = a.N - n0 - c;
    if (r < rows && left > 0) store_eight(a.out + (m0 + r) * a.N + n0 + c, v, FAST ? 8 : left);
  });
}

// Weight gradients out_j = A_j^T B_j over all rows: both operands contiguous along the tile's rows.  The rows are cut
// into `splits` ranges; a range's result is left in fp32 and the ranges are added in order by gff_add_kernel.
template <typename T>
struct WeightJob {
  const T *a, *b;
  T* out;
  int M, N, first_tile, tiles_n;      // first tile of the job among all jobs' tiles
  int64_t first_part;                 // first element of the job in a range's partial results
};
template <typename T>
struct WeightArgs {
  WeightJob<T> job[3];
  float* parts;
  int64_t n_rows, rows_per_split, part_elems;
  int jobs, tiles, splits;
};
template <typename T, bool FAST>
__global__ void __launch_bounds__(kGemmThreads, 3) gff_weight_kernel(WeightArgs<T> w) {
  __shared__ alignas(16) char lds[2 * kGemmTileBytes];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place(w.tiles);
  if (at.outer >= w.splits) return;
  const int which = w.jobs > 2 && at.inner >= w.job[2].first_tile ? 2 : w.jobs > 1 && at.inner >= w.job[1].first_tile ? 1 : 0;
  const WeightJob<T> job = w.job[which];
  const int tile = at.inner - job.first_tile;
  const int m0 = tile / job.tiles_n * kGemmTile, n0 = tile % job.tiles_n * kGemmTile;
  const int64_t r0 = at.outer * w.rows_per_split;
  const int64_t end = std::min(w.rows_per_split, w.n_rows - r0);
  const int rows = rows_left(job.M, m0), cols = rows_left(job.N, n0);
  const T *ja = job.a + r0 * job.M + m0, *jb = job.b + r0 * job.N + n0;
  const GemmOperand<T> pa = {{ja, ja + 64}, job.M, {rows, rows - 64}}, pb = {{jb, jb + 64}, job.N, {cols, cols - 64}};
  f32x16_t acc[2][2];
  gemm_loop<T, FAST, false, false, false>(acc, lds, (end + D - 1) / D, [&](int64_t t, int64_t& k0, int64_t& depth) {
    k0 = t * D;
    depth = end;
    return pa;
  }, [&](int64_t) { return pb; });
  gemm_results<false, 8>(acc, lds, [](int, int, int) {}, [&](int, int r, int c, const float (&v)[8]) {
    const int left = job.N - n0 - c;
    if (r >= rows || left <= 0) return;
    const int64_t to = (int64_t)(m0 + r) * job.N + n0 + c;
    if (w.splits > 1) store_eight(w.parts + at.outer * w.part_elems + job.first_part + to, v, FAST ? 8 : left);
    else store_eight(job.out + to, v, FAST ? 8 : left);
  });
}
template <typename T>
__global__ void __launch_bounds__(256) gff_add_kernel(WeightArgs<T> w) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= w.part_elems) return;
  float s = 0.f;
  for (int k = 0; k < w.splits; ++k) s += w.parts[k * w.part_elems + i];
  const int which = w.jobs > 2 && i >= w.job[2].first_part ? 2 : w.jobs > 1 && i >= w.job[1].first_part ? 1 : 0;
  const WeightJob<T> job = w.job[which];
  job.out[i - job.first_part] = (T)s;
}

// ---- launches -----------------------------------------------------------------------------------------------------
int gff_check(const cgtp_gff_args* a) {
  if (!a) return CGTP_ERR_NULL;
  if (a->dtype != CGTP_F32 && a->dtype != CGTP_BF16 && a->dtype != CGTP_F16) return CGTP_ERR_DTYPE;
  if (a->n_rows < 0 || a->n_rows > 0x7fffffff || a->c_in <= 0 || a->c_out <= 0 || a->hidden <= 0) return CGTP_ERR_SHAPE;
  // a grid has fewer than 2^32 threads, the weights' partial results an index of 31 bits
  if (((a->n_rows + 1023) / 1024) * ((a->hidden + 63) / 64) >= (1 << 20)) return CGTP_ERR_SHAPE;
  if ((int64_t)a->hidden * (2ll * a->c_in + a->c_out) > 0x7fffffff) return CGTP_ERR_SHAPE;
  if (a->c_in > 0x7fff || a->c_out > 0x7fff || a->hidden > 0x1ffff) return CGTP_ERR_SHAPE;
  if (a->activation < 0 || a->activation >= kActs) return CGTP_ERR_CONFIG;
  if (!a->w_gate || !a->w_up || !a->w_down) return CGTP_ERR_NULL;
  if (a->n_rows > 0 && !a->x) return CGTP_ERR_NULL;
  return CGTP_OK;
}

// Whether every row is a number of whole groups of eight elements, aligned, and a tile's offsets fit 31 bits: no access is cut.
bool whole_groups(const cgtp_gff_args* a) {
  const void* ptrs[] = {a->x, a->w_gate, a->w_up, a->w_down, a->gate, a->up, a->mid, a->out, a->grad_out, a->grad_gate, a->grad_up,
                        a->grad_x, a->grad_w_gate, a->grad_w_up, a->grad_w_down, a->workspace};
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  return a->c_in % 8 == 0 && a->hidden % 8 == 0 && a->c_out % 8 == 0;      // hidden < 2^17: 128 rows of it are below 2^26 bytes
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Ranges the rows are cut into for the weight gradients: three workgroups for each compute unit, at least eight k tiles each.
struct WeightShape { int splits; int64_t rows_per_split, part_elems; int tiles; };
WeightShape weight_shape(const cgtp_gff_args* a) {
  WeightShape s;
  const int64_t th = ceil_div(a->hidden, kGemmTile), ti = ceil_div(a->c_in, kGemmTile), to = ceil_div(a->c_out, kGemmTile);
  s.tiles = (int)(th * (2 * ti + to));
  s.part_elems = (int64_t)a->hidden * (2 * a->c_in + a->c_out);
  const int depth = a->dtype == CGTP_F32 ? 32 : 64;
  int64_t splits = std::max<int64_t>(1, 768 / s.tiles);
  splits = std::max<int64_t>(1, std::min(splits, ceil_div(a->n_rows, 8 * depth)));
  if (splits > 8) splits = splits / 8 * 8;           // a range's tiles run on one XCD: as many ranges for each of the eight
  s.rows_per_split = ceil_div(ceil_div(a->n_rows, splits), depth) * depth;
  s.splits = (int)std::max<int64_t>(1, ceil_div(a->n_rows, std::max<int64_t>(1, s.rows_per_split)));
  return s;
}

// The kernel of an activation: a branch on it for each element costs more than the activation.
template <typename Kernel, typename Of>
Kernel for_act(int act, Of&& of) {
  if (act == CGTP_ACT_SILU) return of(std::integral_constant<int, CGTP_ACT_SILU>{});
  if (act == CGTP_ACT_GELU) return of(std::integral_constant<int, CGTP_ACT_GELU>{});
  return of(std::integral_constant<int, CGTP_ACT_SIGMOID>{});
}

template <typename T>
int gff_forward(const cgtp_gff_args* a, hipStream_t s) {
  const bool fast = whole_groups(a);
  const int64_t mt = ceil_div(a->n_rows, kGemmTile);
  const UpArgs<T> u = {(const T*)a->x, (const T*)a->w_gate, (const T*)a->w_up, (T*)a->gate, (T*)a->up, (T*)a->mid, a->n_rows,
                       a->c_in, a->hidden};
  auto up = for_act<void (*)(UpArgs<T>)>(a->activation, [&](auto act) {
    return fast ? gff_up_kernel<T, true, decltype(act)::value> : gff_up_kernel<T, false, decltype(act)::value>;
  });
  hipLaunchKernelGGL(up, dim3(tile_grid(mt, ceil_div(a->hidden, 64))), dim3(kGemmThreads), 0, s, u);
  const RowsArgs<T> d = {{(const T*)a->mid, nullptr}, {(const T*)a->w_down, nullptr}, (T*)a->out, a->n_rows, a->c_out, 1, a->hidden,
                         a->c_out};
  auto down = fast ? gff_rows_kernel<T, true, false> : gff_rows_kernel<T, false, false>;
  hipLaunchKernelGGL(down, dim3(tile_grid(mt, ceil_div(a->c_out, kGemmTile))), dim3(kGemmThreads), 0, s, d);
  return launch_status();
}

template <typename T>
int gff_backward(const cgtp_gff_args* a, hipStream_t s) {
  const bool fast = whole_groups(a);
  const int64_t mt = ceil_div(a->n_rows, kGemmTile);
  if (a->n_rows > 0 && (a->grad_x || a->grad_w_gate || a->grad_w_up)) {
    const MidGradArgs<T> m = {(const T*)a->grad_out, (const T*)a->w_down, (const T*)a->gate, (const T*)a->up, (T*)a->grad_gate,
                              (T*)a->grad_up, a->n_rows, a->hidden, a->c_out};
    auto mid = for_act<void (*)(MidGradArgs<T>)>(a->activation, [&](auto act) {
      return fast ? gff_mid_grad_kernel<T, true, decltype(act)::value> : gff_mid_grad_kernel<T, false, decltype(act)::value>;
    });
    hipLaunchKernelGGL(mid, dim3(tile_grid(mt, ceil_div(a->hidden, kGemmTile))), dim3(kGemmThreads), 0, s, m);
  }
  if (a->n_rows > 0 && a->grad_x) {
    const RowsArgs<T> d = {{(const T*)a->grad_gate, (const T*)a->grad_up}, {(const T*)a->w_gate, (const T*)a->w_up},
                           (T*)a->grad_x, a->n_rows, a->hidden, 2, a->hidden, a->c_in};
    auto back = fast ? gff_rows_kernel<T, true, true>
                                                                         : gff_rows_kernel<T, false, true>;
    hipLaunchKernelGGL(back, dim3(tile_grid(mt, ceil_div(a->c_in, kGemmTile))), dim3(kGemmThreads), 0, s, d);
  }
  const WeightShape shape = weight_shape(a);
  WeightArgs<T> w = {};
  w.parts = (float*)a->workspace;
  w.n_rows = a->n_rows;
  w.rows_per_split = shape.rows_per_split;
  w.splits = shape.splits;
  auto job = [&](const void* l, const void* r, void* out, int M, int N) {
    if (!out) return;
    w.job[w.jobs++] = {(const T*)l, (const T*)r, (T*)out, M, N, w.tiles, (int)ceil_div(N, kGemmTile), w.part_elems};
    w.tiles += (int)(ceil_div(M, kGemmTile) * ceil_div(N, kGemmTile));
    w.part_elems += (int64_t)M * N;
  };
  job(a->x, a->grad_gate, a->grad_w_gate, a->c_in, a->hidden);
  job(a->x, a->grad_up, a->grad_w_up, a->c_in, a->hidden);
  job(a->mid, a->grad_out, a->grad_w_down, a->hidden, a->c_out);
  if (w.jobs) {
    auto weight = fast ? gff_weight_kernel<T, true> : gff_weight_kernel<T, false>;
    hipLaunchKernelGGL(weight, dim3(tile_grid(w.splits, w.tiles)), dim3(kGemmThreads), 0, s, w);
    if (w.splits > 1)
      hipLaunchKernelGGL(gff_add_kernel<T>, dim3((unsigned)ceil_div(w.part_elems, 256)), dim3(256), 0, s, w);
  }
  return launch_status();
}

}  // namespace
}  // namespace cgtp

extern "C" {

int64_t cgtp_gff_workspace_bytes(const cgtp_gff_args* a) {
  using namespace cgtp;
  if (gff_check(a) != CGTP_OK) return 0;
  const WeightShape s = weight_shape(a);
  return s.splits > 1 ? s.splits * s.part_elems * 4 : 0;
}

int cgtp_gff_forward(const cgtp_gff_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = gff_check(a)) return rc;
  if (a->n_rows == 0) return CGTP_OK;
  if (!a->mid || !a->out || (!a->gate) != (!a->up)) return CGTP_ERR_NULL;
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
  if (cgtp_gff_workspace_bytes(a) > 0 && !a->workspace) return CGTP_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case CGTP_F32: return gff_backward<float>(a, s);
    case CGTP_BF16: return gff_backward<bf16_t>(a, s);
    default: return gff_backward<f16_t>(a, s);
  }
}

}  // extern "C"
