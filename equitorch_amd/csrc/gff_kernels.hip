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

namespace cgtp {
namespace {

constexpr int kActs = 3;       // CGTP_ACT_SILU, CGTP_ACT_GELU, CGTP_ACT_SIGMOID

// act(g) and its derivative.  16-bit types take the hardware's exponential (1e-6 relative), fp32 the exact one.
template <typename T>
__device__ __forceinline__ float gff_sigmoid(float g) {
  if constexpr (sizeof(T) == 2) return 1.f / (1.f + __expf(-g));
  else return 1.f / (1.f + expf(-g));
}
template <typename T>
__device__ __forceinline__ float gff_act(int act, float g) {
  if (act == CGTP_ACT_GELU) return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
  const float s = gff_sigmoid<T>(g);
  return act == CGTP_ACT_SILU ? g * s : s;
}
template <typename T>
__device__ __forceinline__ float gff_act_grad(int act, float g, float& value) {
  if (act == CGTP_ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    value = g * cdf;
    return cdf + g * 0.3989422804014327f * expf(-0.5f * g * g);
  }
  const float s = gff_sigmoid<T>(g);
  if (act == CGTP_ACT_SILU) {
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

// Where a lane's results are within its wavefront's part.
struct LanePlace { int m, n; };       // of acc[i][j]: row 32 i + m, columns 32 j + n + 8 g + e
__device__ __forceinline__ LanePlace lane_place() {
  const int lane = threadIdx.x & 63;
  return {lane & 31, (lane >> 5) * 4};
}

template <typename T>
struct UpArgs {
  const T *x, *wg, *wu;
  T *gate, *up, *mid;            // gate and up may be null (inference)
  int64_t n_rows;
  int C, H, act;
};

// g, u and m.  A tile is 128 rows x 64 hidden channels, the columns of a wavefront 32 of Wg and the same 32 of Wu.
template <typename T>
__global__ void __launch_bounds__(kGemmThreads) gff_up_kernel(UpArgs<T> a) {
  __shared__ alignas(16) char lds[4 * kGemmTileBytes];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place((a.H + 63) / 64);
  const int64_t m0 = at.outer * kGemmTile;
  if (m0 >= a.n_rows) return;
  const int h0 = at.inner * 64;
  f32x16_t acc[2][2];
  gemm_loop<T, true, false>(
      acc, lds, (a.C + D - 1) / D,
      [&](auto& st, int64_t t) {
        st.load([&](int r, int64_t&) { return m0 + r < a.n_rows ? a.x + (m0 + r) * a.C : nullptr; }, t * D, a.C, 0);
      },
      [&](auto& st, int64_t t) {
        st.load([&](int r, int64_t& end) {
          const int h = h0 + (r >> 6) * 32 + (r & 31);
          end = a.H - h;
          return end > 0 ? ((r & 32) ? a.wu : a.wg) + h : nullptr;
        }, t * D, a.C, a.H);
      });
  const LanePlace lp = lane_place();
  const int wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + wm * 64 + 32 * i + lp.m;
    if (m >= a.n_rows) continue;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int h = h0 + wn * 32 + 8 * g + lp.n;
      if (h >= a.H) continue;
      T vg[4], vu[4], vm[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float fg = acc[i][0][4 * g + e], fu = acc[i][1][4 * g + e];
        vg[e] = (T)fg;
        vu[e] = (T)fu;
        vm[e] = (T)(gff_act<T>(a.act, fg) * fu);
      }
      const int64_t to = m * a.H + h;
      store_part<T, 4>(a.mid + to, vm, a.H - h);
      if (a.gate) {
        store_part<T, 4>(a.gate + to, vg, a.H - h);
        store_part<T, 4>(a.up + to, vu, a.H - h);
      }
    }
  }
}

template <typename T>
struct MidGradArgs {
  const T *gy, *wd, *gate, *up;
  T *g_gate, *g_up;
  int64_t n_rows;
  int H, C, act;
};

// dg and du from dm = dy Wd^T.
template <typename T>
__global__ void __launch_bounds__(kGemmThreads) gff_mid_grad_kernel(MidGradArgs<T> a) {
  __shared__ alignas(16) char lds[4 * kGemmTileBytes];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place((a.H + kGemmTile - 1) / kGemmTile);
  const int64_t m0 = at.outer * kGemmTile;
  if (m0 >= a.n_rows) return;
  const int h0 = at.inner * kGemmTile;
  f32x16_t acc[2][2];
  gemm_loop<T, true, true>(
      acc, lds, (a.C + D - 1) / D,
      [&](auto& st, int64_t t) {
        st.load([&](int r, int64_t&) { return m0 + r < a.n_rows ? a.gy + (m0 + r) * a.C : nullptr; }, t * D, a.C, 0);
      },
      [&](auto& st, int64_t t) {
        st.load([&](int r, int64_t&) { return h0 + r < a.H ? a.wd + (int64_t)(h0 + r) * a.C : nullptr; }, t * D, a.C, 0);
      });
  const LanePlace lp = lane_place();
  const int wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + wm * 64 + 32 * i + lp.m;
    if (m >= a.n_rows) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int h = h0 + wn * 64 + 32 * j + 8 * g + lp.n;
        if (h >= a.H) continue;
        const int64_t to = m * a.H + h;
        typedef Loose<T, 4> V4;
        typedef unsigned raw_t __attribute__((ext_vector_type(sizeof(T))));
        const V4 vg = __builtin_bit_cast(V4, load_part<raw_t, T>(a.gate + to, a.H - h));
        const V4 vu = __builtin_bit_cast(V4, load_part<raw_t, T>(a.up + to, a.H - h));
        T dg[4], du[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float dm = acc[i][j][4 * g + e];
          float value;
          const float slope = gff_act_grad<T>(a.act, (float)vg.v[e], value);
          dg[e] = (T)(dm * (float)vu.v[e] * slope);
          du[e] = (T)(dm * value);
        }
        store_part<T, 4>(a.g_gate + to, dg, a.H - h);
        store_part<T, 4>(a.g_up + to, du, a.H - h);
      }
  }
}

// out = sum over segments of A_s B_s: y = m Wd (one segment), dx = dg Wg^T + du Wu^T (two).  A is contiguous along k.
template <typename T>
struct RowsArgs {
  const T *a[2], *b[2];
  T* out;
  int64_t n_rows, ldb;
  int segments, K, N;            // per segment
};
template <typename T, bool KB>
__global__ void __launch_bounds__(kGemmThreads) gff_rows_kernel(RowsArgs<T> a) {
  __shared__ alignas(16) char lds[4 * kGemmTileBytes];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place((a.N + kGemmTile - 1) / kGemmTile);
  const int64_t m0 = at.outer * kGemmTile;
  if (m0 >= a.n_rows) return;
  const int n0 = at.inner * kGemmTile, tiles = (a.K + D - 1) / D;
  f32x16_t acc[2][2];
  gemm_loop<T, true, KB>(
      acc, lds, (int64_t)tiles * a.segments,
      [&](auto& st, int64_t t) {
        const T* p = t < tiles ? a.a[0] : a.a[1];
        if (t >= tiles) t -= tiles;
        st.load([&](int r, int64_t&) { return m0 + r < a.n_rows ? p + (m0 + r) * a.K : nullptr; }, t * D, a.K, 0);
      },
      [&](auto& st, int64_t t) {
        const T* p = t < tiles ? a.b[0] : a.b[1];
        if (t >= tiles) t -= tiles;
        st.load([&](int r, int64_t& end) {
          end = a.N - n0 - r;
          return end > 0 ? p + (KB ? (int64_t)(n0 + r) * a.ldb : n0 + r) : nullptr;
        }, t * D, a.K, a.ldb);
      });
  const LanePlace lp = lane_place();
  const int wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + wm * 64 + 32 * i + lp.m;
    if (m >= a.n_rows) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = n0 + wn * 64 + 32 * j + 8 * g + lp.n;
        if (n >= a.N) continue;
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)acc[i][j][4 * g + e];
        store_part<T, 4>(a.out + m * a.N + n, v, a.N - n);
      }
  }
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
template <typename T>
__global__ void __launch_bounds__(kGemmThreads) gff_weight_kernel(WeightArgs<T> w) {
  __shared__ alignas(16) char lds[4 * kGemmTileBytes];
  constexpr int D = GemmType<T>::kDepth;
  const TilePlace at = tile_place(w.tiles);
  if (at.outer >= w.splits) return;
  const int which = w.jobs > 2 && at.inner >= w.job[2].first_tile ? 2 : w.jobs > 1 && at.inner >= w.job[1].first_tile ? 1 : 0;
  const WeightJob<T> job = w.job[which];
  const int tile = at.inner - job.first_tile;
  const int m0 = tile / job.tiles_n * kGemmTile, n0 = tile % job.tiles_n * kGemmTile;
  const int64_t r0 = at.outer * w.rows_per_split;
  const int64_t depth = std::min(w.rows_per_split, w.n_rows - r0);
  f32x16_t acc[2][2];
  gemm_loop<T, false, false>(
      acc, lds, (depth + D - 1) / D,
      [&](auto& st, int64_t t) {
        st.load([&](int r, int64_t& end) {
          end = job.M - m0 - r;
          return end > 0 ? job.a + r0 * job.M + m0 + r : nullptr;
        }, t * D, depth, job.M);
      },
      [&](auto& st, int64_t t) {
        st.load([&](int r, int64_t& end) {
          end = job.N - n0 - r;
          return end > 0 ? job.b + r0 * job.N + n0 + r : nullptr;
        }, t * D, depth, job.N);
      });
  const LanePlace lp = lane_place();
  const int wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = m0 + wm * 64 + 32 * i + lp.m;
    if (m >= job.M) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = n0 + wn * 64 + 32 * j + 8 * g + lp.n;
        if (n >= job.N) continue;
        const int64_t to = (int64_t)m * job.N + n;
        if (w.splits > 1) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
          store_part<float, 4>(w.parts + at.outer * w.part_elems + job.first_part + to, v, job.N - n);
        } else {
          T v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (T)acc[i][j][4 * g + e];
          store_part<T, 4>(job.out + to, v, job.N - n);
        }
      }
  }
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

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Ranges the rows are cut into for the weight gradients: two workgroups for each compute unit, at least eight k tiles each.
struct WeightShape { int splits; int64_t rows_per_split, part_elems; int tiles; };
WeightShape weight_shape(const cgtp_gff_args* a) {
  WeightShape s;
  const int64_t th = ceil_div(a->hidden, kGemmTile), ti = ceil_div(a->c_in, kGemmTile), to = ceil_div(a->c_out, kGemmTile);
  s.tiles = (int)(th * (2 * ti + to));
  s.part_elems = (int64_t)a->hidden * (2 * a->c_in + a->c_out);
  const int depth = a->dtype == CGTP_F32 ? 32 : 64;
  int64_t splits = std::max<int64_t>(1, 512 / s.tiles);
  splits = std::max<int64_t>(1, std::min(splits, ceil_div(a->n_rows, 8 * depth)));
  s.rows_per_split = ceil_div(ceil_div(a->n_rows, splits), depth) * depth;
  s.splits = (int)std::max<int64_t>(1, ceil_div(a->n_rows, std::max<int64_t>(1, s.rows_per_split)));
  return s;
}

template <typename T>
int gff_forward(const cgtp_gff_args* a, hipStream_t s) {
  const int64_t mt = ceil_div(a->n_rows, kGemmTile);
  UpArgs<T> u = {(const T*)a->x, (const T*)a->w_gate, (const T*)a->w_up, (T*)a->gate, (T*)a->up, (T*)a->mid, a->n_rows,
                 a->c_in, a->hidden, a->activation};
  hipLaunchKernelGGL(gff_up_kernel<T>, dim3(tile_grid(mt, ceil_div(a->hidden, 64))), dim3(kGemmThreads), 0, s, u);
  RowsArgs<T> d = {{(const T*)a->mid, nullptr}, {(const T*)a->w_down, nullptr}, (T*)a->out, a->n_rows, a->c_out, 1, a->hidden,
                   a->c_out};
  hipLaunchKernelGGL((gff_rows_kernel<T, false>), dim3(tile_grid(mt, ceil_div(a->c_out, kGemmTile))), dim3(kGemmThreads), 0,
                     s, d);
  return launch_status();
}

template <typename T>
int gff_backward(const cgtp_gff_args* a, hipStream_t s) {
  const int64_t mt = ceil_div(a->n_rows, kGemmTile);
  if (a->n_rows > 0 && (a->grad_x || a->grad_w_gate || a->grad_w_up)) {
    MidGradArgs<T> m = {(const T*)a->grad_out, (const T*)a->w_down, (const T*)a->gate, (const T*)a->up, (T*)a->grad_gate,
                        (T*)a->grad_up, a->n_rows, a->hidden, a->c_out, a->activation};
    hipLaunchKernelGGL(gff_mid_grad_kernel<T>, dim3(tile_grid(mt, ceil_div(a->hidden, kGemmTile))), dim3(kGemmThreads), 0, s, m);
  }
  if (a->n_rows > 0 && a->grad_x) {
    RowsArgs<T> d = {{(const T*)a->grad_gate, (const T*)a->grad_up}, {(const T*)a->w_gate, (const T*)a->w_up}, (T*)a->grad_x,
                     a->n_rows, a->hidden, 2, a->hidden, a->c_in};
    hipLaunchKernelGGL((gff_rows_kernel<T, true>), dim3(tile_grid(mt, ceil_div(a->c_in, kGemmTile))), dim3(kGemmThreads), 0, s, d);
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
    hipLaunchKernelGGL(gff_weight_kernel<T>, dim3(tile_grid(w.splits, w.tiles)), dim3(kGemmThreads), 0, s, w);
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
