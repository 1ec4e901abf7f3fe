// Root-mean-square norm after a residual's addition (cgtp_add_rms_forward, cgtp_add_rms_backward):
//
//   t = x + residual, rounded to the residual's type,   r = (mean_c t^2 + eps)^-1/2,   out = t r w
//   u = w g,   grad t = g_t + r (u - t r^2 mean_c(u t)),   grad w = sum over rows of g t r
//
// with g, g_t the gradients of out and t.  The norm is that of t as it is stored, so that the backward, which reads t, has
// the forward's values.  8 bits: s = max_c |out| / 448 for each row, and out / s in e4m3.
//
// Bound by memory: every row is read once and stays in registers, eight elements (a chunk) a lane at a time.  A row of up to
// 64 chunks has the power of two of lanes that holds it, one chunk each, so that short rows share a wavefront; up to 1024
// channels a wavefront with two chunks a lane; longer ones a workgroup, with 256 threads of one to four chunks, or 512 of four or eight
// (which spill, above 16384 channels).  More chunks a lane leave too few wavefronts to hide the memory behind: 9765 rows of 4096 fp16
// channels, backward: 158 us with a wavefront and eight chunks, 71 with a workgroup and two; 26666 of 1500: 91 us with a wavefront and four, 76
// with a workgroup and one.  Loads need no alignment but the element's.  65536 rows of 256 channels, bf16 on an fp32 residual: forward
// 38.7 us (5.2 TB/s), backward 47.0 (5.4); 200003 rows of 512 in bf16 to 8 bits: 140 us (5.1 TB/s).
#include "elem.h"

#include <algorithm>

namespace cgtp {
namespace {

constexpr int kThreads = 256, kWaveChunks = 2;

template <typename U>
struct Chunk {
  static constexpr int N = 16 / (int)sizeof(U);
  __device__ static __forceinline__ void load(float (&d)[8], const U* p, int valid) {
    typedef U vec __attribute__((ext_vector_type(N)));
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      u32x4_t r = {0, 0, 0, 0};
      if (valid > i) r = load_part<u32x4_t, U>(p + i, valid - i);
      const vec v = __builtin_bit_cast(vec, r);
#pragma unroll
      for (int j = 0; j < N; ++j) d[i + j] = (float)v[j];
    }
  }
};

struct RmsArgs {
  const void *x, *residual, *weight;
  void *out, *total;
  float *rstd, *scale;
  const void *grad_out, *grad_total;
  void *grad_x, *grad_residual, *grad_weight;
  float* parts;
  int64_t n_rows;
  int c, group, weight_f32;      // group: lanes of a row, a power of two up to 64, or the workgroup's threads
  float eps;
};

// Sum over the lanes of a row, the same in every lane.  BLOCK: over the workgroup, `shared` has a place for each wavefront.
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, int group, float* shared) {
  for (int o = BLOCK ? 32 : group >> 1; o; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (BLOCK) {
    __syncthreads();               // the places are free again
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < (int)blockDim.x >> 6; ++i) v += shared[i];
  }
  return v;
}
// The largest of bit patterns of magnitudes, whose order is that of the numbers, with NaN above infinity.
template <bool BLOCK>
__device__ __forceinline__ unsigned row_max(unsigned v, int group, float* shared) {
  for (int o = BLOCK ? 32 : group >> 1; o; o >>= 1) v = std::max(v, (unsigned)__shfl_xor((int)v, o));
  if constexpr (BLOCK) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = __uint_as_float(v);
    __syncthreads();
    for (int i = 0; i < (int)blockDim.x >> 6; ++i) v = std::max(v, __float_as_uint(shared[i]));
  }
  return v;
}

// Where a lane's chunk of a row is.  A last chunk that the row does not fill is taken from the row's end: the columns that it shares with the
// chunk before are computed twice with the same bits, and only the sums leave the first `twice` of its elements out.  One by one
// its elements took as many accesses as a row of 1001 has altogether.
struct Place { int c, valid, twice; };
__device__ __forceinline__ Place place_of(int channels, int chunk) {
  Place p = {chunk * 8, channels - chunk * 8, 0};
  if (p.valid > 0 && p.valid < 8 && channels >= 8) p = {channels - 8, 8, 8 - p.valid};
  return p;
}

template <typename T>
__device__ __forceinline__ void load_weight(float (&w)[8], const RmsArgs& a, const Place& p) {
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = 1.f;
  if (!a.weight || p.valid <= 0) return;
  if (a.weight_f32) Chunk<float>::load(w, (const float*)a.weight + p.c, p.valid);
  else Chunk<T>::load(w, (const T*)a.weight + p.c, p.valid);
}

// Eight values of magnitude up to 448 in e4m3, to nearest.
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&v)[8], int valid) {
  uint8_t b[8];
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[i], v[i + 1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(v[i + 2], v[i + 3], r, true);
    __builtin_memcpy(b + i, &r, 4);
  }
  store_part<uint8_t, 8>(p, b, valid);
}

template <typename T, typename R, int CHUNKS, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : kThreads) add_rms_kernel(RmsArgs a) {
  __shared__ float shared[8];
  const int lanes = BLOCK ? (int)blockDim.x : a.group, lane = threadIdx.x & (lanes - 1);
  const int per_block = BLOCK ? 1 : kThreads / lanes;
  const T* x = (const T*)a.x;
  const R* residual = (const R*)a.residual;
  float w[CHUNKS][8];
  Place place[CHUNKS];
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k) {
    place[k] = place_of(a.c, k * lanes + lane);
    load_weight<T>(w[k], a, place[k]);
  }
  const float inv_c = 1.f / (float)a.c;
  for (int64_t first = (int64_t)blockIdx.x * per_block; first < a.n_rows; first += (int64_t)gridDim.x * per_block) {
    const int64_t row = first + (BLOCK ? 0 : (int)threadIdx.x / lanes);
    const bool in = row < a.n_rows;
    const int64_t at = row * a.c;
    float t[CHUNKS][8], sum = 0.f;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      const int c = place[k].c, valid = in ? place[k].valid : 0;
      Chunk<T>::load(t[k], x + at + c, valid);
      if (residual) {
        float r[8];
        Chunk<R>::load(r, residual + at + c, valid);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[k][e] = (float)(R)(t[k][e] + r[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = e < place[k].twice ? 0.f : t[k][e];
        sum = fmaf(v, v, sum);
      }
    }
    // total may be x or the residual: all of a row is read first, by all wavefronts that share it
    auto store_total = [&] {
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k)
        if (residual && a.total) store_eight((R*)a.total + at + place[k].c, t[k], in ? place[k].valid : 0);
    };
    if constexpr (!BLOCK) store_total();
    const float rstd = rsqrtf(row_sum<BLOCK>(sum, lanes, shared) * inv_c + a.eps);
    if constexpr (BLOCK) store_total();
    if (a.rstd && in && lane == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) t[k][e] = t[k][e] * rstd * w[k][e];
    if (!a.scale) {
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) store_eight((T*)a.out + at + place[k].c, t[k], in ? place[k].valid : 0);
    } else {
      unsigned top = 0;
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = std::max(top, __float_as_uint(t[k][e]) & 0x7fffffffu);
      const float most = __uint_as_float(row_max<BLOCK>(top, lanes, shared));
      // A row of zeros has scale 0; the scale of a tiny one is a normal number, so that its inverse is finite; a row with an
      // infinity or a NaN has scale NaN, whose inverse makes every value NaN.
      const float scale = most == 0.f ? 0.f : most < INFINITY ? std::max(most / 448.f, 0x1p-126f) : NAN;
      const float inverse = most == 0.f ? 0.f : 1.f / scale;
      if (in && lane == 0) a.scale[row] = scale;
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int valid = in ? place[k].valid : 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float q = t[k][e] * inverse;
          t[k][e] = q > 448.f ? 448.f : q < -448.f ? -448.f : q;
        }
        if (valid > 0) store_e4m3((uint8_t*)a.out + at + place[k].c, t[k], valid);
      }
    }
  }
}

// Rows are shared out over the workgroups by their number alone; a workgroup's sums of the weight's gradient are left in
// `parts`, or are the result where there is one workgroup.  The lanes of a wavefront that hold the same channels are
// added first, then the wavefronts in order.
template <typename T, typename R, int CHUNKS, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : kThreads) add_rms_grad_kernel(RmsArgs a) {
  __shared__ float shared[8];
  __shared__ float sums[BLOCK ? 1 : CHUNKS * 512];
  const int lanes = BLOCK ? (int)blockDim.x : a.group, lane = threadIdx.x & (lanes - 1);
  const int per_block = BLOCK ? 1 : kThreads / lanes;
  const R* total = (const R*)a.total;
  float w[CHUNKS][8], gw[CHUNKS][8];
  Place place[CHUNKS];
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k) {
    place[k] = place_of(a.c, k * lanes + lane);
    load_weight<T>(w[k], a, place[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[k][e] = 0.f;
  }
  const float inv_c = 1.f / (float)a.c;
  for (int64_t first = (int64_t)blockIdx.x * per_block; first < a.n_rows; first += (int64_t)gridDim.x * per_block) {
    const int64_t row = first + (BLOCK ? 0 : (int)threadIdx.x / lanes);
    const bool in = row < a.n_rows;
    const int64_t at = row * a.c;
    const float rstd = in ? a.rstd[row] : 0.f;
    float t[CHUNKS][8], u[CHUNKS][8], dot = 0.f;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      const int c = place[k].c, valid = in ? place[k].valid : 0;
      Chunk<R>::load(t[k], total + at + c, valid);
      Chunk<T>::load(u[k], (const T*)a.grad_out + at + c, valid);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[k][e] *= rstd;
        gw[k][e] = fmaf(u[k][e], t[k][e], gw[k][e]);        // of columns that are there twice: not taken below
        u[k][e] *= w[k][e];
        dot = fmaf(e < place[k].twice ? 0.f : u[k][e], t[k][e], dot);
      }
    }
    if (!a.grad_x && !a.grad_residual) continue;
    const float mean = row_sum<BLOCK>(dot, lanes, shared) * inv_c;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      const int c = place[k].c, valid = in ? place[k].valid : 0;
      if (a.grad_total) {
        float g[8];
        Chunk<R>::load(g, (const R*)a.grad_total + at + c, valid);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[k][e] = fmaf(rstd, u[k][e] - t[k][e] * mean, g[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[k][e] = rstd * (u[k][e] - t[k][e] * mean);
      }
      if (a.grad_x) store_eight((T*)a.grad_x + at + c, u[k], valid);
      if (a.grad_residual) store_eight((R*)a.grad_residual + at + c, u[k], valid);
    }
  }
  if (!a.grad_weight) return;
  float* part = a.parts + (int64_t)blockIdx.x * a.c;
  auto give = [&](int c, float v) {
    if (gridDim.x > 1) part[c] = v;
    else if (a.weight_f32) ((float*)a.grad_weight)[c] = v;
    else ((T*)a.grad_weight)[c] = (T)v;
  };
  if constexpr (BLOCK) {
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e >= place[k].twice && e < place[k].valid) give(place[k].c + e, gw[k][e]);
      }
  } else {
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        for (int o = lanes; o < 64; o <<= 1) gw[k][e] += __shfl_xor(gw[k][e], o);
    const int wave = threadIdx.x >> 6;
    for (int i = 0; i < kThreads / 64; ++i) {
      if (wave == i && (int)(threadIdx.x & 63) < lanes) {
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float* s = sums + (k * 8 + e) * lanes + lane;      // neighbouring lanes in neighbouring banks
            *s = i ? *s + gw[k][e] : gw[k][e];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < CHUNKS * lanes * 8; i += kThreads) {
      if (i >= a.c) continue;                                   // channel i: element i % 8 of chunk i / 8, the last one's behind the others
      const int k = i / 8 / lanes, l = i / 8 % lanes, e = (i & 7) + place_of(a.c, i / 8).twice;
      give(i, sums[(k * 8 + e) * lanes + l]);
    }
  }
}

// The workgroups' sums, in order: 32 threads for each of 32 channels, then one.
constexpr int kJoin = 32;
template <typename T>
__global__ void __launch_bounds__(kJoin * kJoin) add_rms_join_kernel(const float* parts, T* out, int n_parts, int c) {
  __shared__ float sums[kJoin][kJoin + 1];
  const int col = threadIdx.x % kJoin, slice = threadIdx.x / kJoin, at = blockIdx.x * kJoin + col;
  float s = 0.f;
  if (at < c)
#pragma unroll 8
    for (int i = slice; i < n_parts; i += kJoin) s += parts[(int64_t)i * c + at];
  sums[slice][col] = s;
  __syncthreads();
  if (slice || at >= c) return;
#pragma unroll
  for (int i = 1; i < kJoin; ++i) s += sums[i][col];
  out[at] = (T)s;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

struct RmsShape { int group, chunks, threads, rows; bool block; };      // rows of a workgroup at a time; block: the workgroup has one
RmsShape shape_of(int c) {
  const int chunks = (c + 7) / 8;
  RmsShape s = {64, 1, kThreads, 1, false};
  if (chunks <= 64) {
    for (s.group = 1; s.group < chunks;) s.group *= 2;
  } else if (chunks <= 64 * kWaveChunks) {
    s.chunks = kWaveChunks;
  } else {
    s.block = true;
    if (chunks > 4 * kThreads) s.threads = 512;
    while (s.threads * s.chunks < chunks) s.chunks *= 2;
    s.group = s.threads;
    return s;
  }
  s.rows = kThreads / s.group;
  return s;
}

// Workgroups of a launch: the forward's hold all rows or fill the GPU; the backward's leave a sum of the weight's gradient each.
int blocks_of(const RmsShape& s, int64_t n_rows, bool backward) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((n_rows + s.rows - 1) / s.rows, backward ? 1024 : 4096));
}

int rms_check(const cgtp_add_rms_args* a) {
  if (!a) return CGTP_ERR_NULL;
  auto float_type = [](int t) { return t == CGTP_F32 || t == CGTP_BF16 || t == CGTP_F16; };
  if (!float_type(a->dtype) || (a->residual_dtype != a->dtype && a->residual_dtype != CGTP_F32) ||
      (a->weight_dtype != a->dtype && a->weight_dtype != CGTP_F32))
    return CGTP_ERR_DTYPE;
  if (a->n_rows < 0 || a->n_rows > 0x7fffffff || a->channels <= 0 || a->channels > 0x7fff) return CGTP_ERR_SHAPE;
  // the kernels add it in 32 bits, where a number below the normal ones loses its bits, or is zero
  if (!(a->eps == 0 || (a->eps >= 0x1p-126 && a->eps <= 0x1.fffffep127))) return CGTP_ERR_CONFIG;
  return CGTP_OK;
}

RmsArgs kernel_args(const cgtp_add_rms_args* a, const RmsShape& s) {
  RmsArgs k = {};
  k.x = a->x;
  k.residual = a->residual;
  k.weight = a->weight;
  k.total = a->total;
  k.rstd = a->rstd;
  k.n_rows = a->n_rows;
  k.c = a->channels;
  k.group = s.group;
  k.weight_f32 = a->weight_dtype == CGTP_F32;
  k.eps = (float)a->eps;
  return k;
}

template <typename T, typename R, bool BACKWARD, int CHUNKS, bool BLOCK>
void launch(const RmsArgs& k, const RmsShape& s, hipStream_t stream) {
  const dim3 grid(blocks_of(s, k.n_rows, BACKWARD)), block(s.threads);
  if constexpr (BACKWARD) hipLaunchKernelGGL((add_rms_grad_kernel<T, R, CHUNKS, BLOCK>), grid, block, 0, stream, k);
  else hipLaunchKernelGGL((add_rms_kernel<T, R, CHUNKS, BLOCK>), grid, block, 0, stream, k);
}
static_assert(kWaveChunks == 2, "a wavefront's row has one chunk a lane or two");
template <typename T, typename R, bool BACKWARD>
void launch_of(const RmsArgs& k, const RmsShape& s, hipStream_t stream) {
  if (!s.block && s.chunks == 1) launch<T, R, BACKWARD, 1, false>(k, s, stream);
  else if (!s.block) launch<T, R, BACKWARD, kWaveChunks, false>(k, s, stream);
  else if (s.chunks == 1) launch<T, R, BACKWARD, 1, true>(k, s, stream);
  else if (s.chunks == 2) launch<T, R, BACKWARD, 2, true>(k, s, stream);
  else if (s.chunks == 4) launch<T, R, BACKWARD, 4, true>(k, s, stream);
  else launch<T, R, BACKWARD, 8, true>(k, s, stream);
}
template <bool BACKWARD>
void launch_types(const cgtp_add_rms_args* a, const RmsArgs& k, const RmsShape& s, hipStream_t stream) {
  const bool wide = a->residual_dtype == CGTP_F32;
  if (a->dtype == CGTP_F32) launch_of<float, float, BACKWARD>(k, s, stream);
  else if (a->dtype == CGTP_BF16) wide ? launch_of<bf16_t, float, BACKWARD>(k, s, stream) : launch_of<bf16_t, bf16_t, BACKWARD>(k, s, stream);
  else wide ? launch_of<f16_t, float, BACKWARD>(k, s, stream) : launch_of<f16_t, f16_t, BACKWARD>(k, s, stream);
}

template <typename T>
void join(const RmsArgs& k, int parts, hipStream_t stream) {
  hipLaunchKernelGGL(add_rms_join_kernel<T>, dim3(ceil_div(k.c, kJoin)), dim3(kJoin * kJoin), 0, stream, k.parts, (T*)k.grad_weight,
                     parts, k.c);
}

}  // namespace
}  // namespace cgtp

extern "C" {

int64_t cgtp_add_rms_workspace_bytes(const cgtp_add_rms_args* a) {
  using namespace cgtp;
  if (rms_check(a) != CGTP_OK || a->n_rows == 0 || !a->grad_weight) return 0;
  const int blocks = blocks_of(shape_of(a->channels), a->n_rows, true);
  return blocks > 1 ? (int64_t)blocks * a->channels * 4 : 0;
}

int cgtp_add_rms_forward(const cgtp_add_rms_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = rms_check(a)) return rc;
  if (a->n_rows == 0) return CGTP_OK;
  if (!a->x || !a->out) return CGTP_ERR_NULL;
  const RmsShape s = shape_of(a->channels);
  RmsArgs k = kernel_args(a, s);
  k.out = a->out;
  k.scale = a->scale;
  launch_types<false>(a, k, s, (hipStream_t)stream);
  return launch_status();
}

int cgtp_add_rms_backward(const cgtp_add_rms_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = rms_check(a)) return rc;
  if (!a->grad_x && !a->grad_residual && !a->grad_weight) return CGTP_OK;
  if (a->n_rows > 0 && (!a->total || !a->rstd || !a->grad_out)) return CGTP_ERR_NULL;
  if (cgtp_add_rms_workspace_bytes(a) > 0 && !a->workspace) return CGTP_ERR_WORKSPACE;
  const RmsShape s = shape_of(a->channels);
  RmsArgs k = kernel_args(a, s);
  k.grad_out = a->grad_out;
  k.grad_total = a->grad_total;
  k.grad_x = a->grad_x;
  k.grad_residual = a->grad_residual;
  k.grad_weight = a->grad_weight;
  k.parts = (float*)a->workspace;
  // without rows the one workgroup writes a gradient of zeros
  launch_types<true>(a, k, s, (hipStream_t)stream);
  const int blocks = blocks_of(s, a->n_rows, true);
  if (a->grad_weight && blocks > 1) {
    if (a->weight_dtype == CGTP_F32) join<float>(k, blocks, (hipStream_t)stream);
    else if (a->weight_dtype == CGTP_BF16) join<bf16_t>(k, blocks, (hipStream_t)stream);
    else join<f16_t>(k, blocks, (hipStream_t)stream);
  }
  return launch_status();
}

}  // extern "C"
