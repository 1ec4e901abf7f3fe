// AdamW step over many tensors at once (cgtp_adamw_step):
//
//   m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2,
//   p <- p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: 28 bytes an element in fp32 with states in 32 bits, 16 with states in 8.  The tensors' addresses are kernel
// arguments, so that a launch takes 52 to 64 tensors and nothing has to reach the GPU before it; a workgroup takes a chunk of one
// tensor.  The step's number is on the GPU (a recorded graph counts on when it is replayed): every workgroup reads it and
// works its factors out, and a launch behind them adds one.
//
// 8 bits: m and r = sqrt(v) in e4m3 with a scale for each 256 elements of a tensor, the largest magnitude / 448.  A wavefront has
// such a block in registers, four elements a lane.  m is rounded to nearest.  r is rounded up or down at random, in
// proportion: b2 = 0.999 changes v by a thousandth a step, a sixteenth of the way to the next value of three
// mantissa bits at most, and to nearest it would stay where it is for ever.  Above zero it never becomes zero, which m would
// be divided by.  The random bits are a hash of seed, tensor, step and element: the same in every run.  The step itself is taken on m and v
// before they are rounded.
#include "elem.h"

#include <algorithm>
#include <cmath>

namespace cgtp {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kBlock = CGTP_ADAMW_BLOCK;
static_assert(kBlock == 256, "four elements for each lane");

template <bool MASTER, bool EIGHT>
struct Entry {
  void* p;
  const void* g;
  void *m, *v;
  const float* step;
  void* more[2 * EIGHT + MASTER > 0 ? 2 * EIGHT + MASTER : 1];      // scales of m and v, then the copy in 32 bits
  unsigned n, number;             // number: the tensor's, for the random bits
  __device__ __forceinline__ float* m_scale() const { return (float*)more[0]; }
  __device__ __forceinline__ float* v_scale() const { return (float*)more[1]; }
  __device__ __forceinline__ float* master() const { return (float*)more[2 * EIGHT]; }
};
// As many tensors as 4 KB of arguments hold, no more than a wavefront finds its own among at once.
template <bool MASTER, bool EIGHT> constexpr int kAtOnce = std::min<int>(64, (4096 - 72) / (sizeof(Entry<MASTER, EIGHT>) + 4));
template <bool MASTER, bool EIGHT>
struct StepArgs {
  Entry<MASTER, EIGHT> entry[kAtOnce<MASTER, EIGHT>];
  unsigned first[kAtOnce<MASTER, EIGHT>];      // each one's first chunk among the launch's
  double lr, decay;
  const float* lr_ptr;            // null: lr
  float b1, b1_rest, log_b1, b2, b2_rest, log_b2, eps;      // b1_rest: with the sign of the step
  unsigned seed;
  int entries, blocks;            // blocks: of 256 elements, in a chunk
};
static_assert(sizeof(StepArgs<false, false>) <= 4096 && sizeof(StepArgs<false, true>) <= 4096 && sizeof(StepArgs<true, false>) <= 4096 &&
              sizeof(StepArgs<true, true>) <= 4096);

struct Factors {
  float keep, size, root;         // 1 - lr decay, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  unsigned key;
};

__device__ __forceinline__ unsigned mix(unsigned h) {
  h = (h ^ (h >> 16)) * 0x9C8F2D35u;
  h = (h ^ (h >> 15)) * 0xB5297A4Du;
  return h ^ (h >> 16);
}

// Four elements of a block from `left` on; WHOLE: all are there.
template <typename U, bool WHOLE>
__device__ __forceinline__ void load4(float (&d)[4], const U* p, int left) {
  typedef U vec __attribute__((ext_vector_type(4)));
  typedef unsigned raw_t __attribute__((ext_vector_type(sizeof(U))));
  if constexpr (WHOLE) {
    const vec v = __builtin_bit_cast(vec, *reinterpret_cast<const typename LooseOf<U, raw_t>::type*>(p));
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = e < left ? (float)p[e] : 0.f;
  }
}
template <typename U, bool WHOLE>
__device__ __forceinline__ void store4(U* p, const float (&s)[4], int left) {
  typedef U vec __attribute__((ext_vector_type(4)));
  typedef unsigned raw_t __attribute__((ext_vector_type(sizeof(U))));
  if constexpr (WHOLE) {
    vec v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (U)s[e];
    *reinterpret_cast<typename LooseOf<U, raw_t>::type*>(p) = __builtin_bit_cast(raw_t, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = (U)s[e];
  }
}
typedef unsigned loose_u32 __attribute__((aligned(1)));
template <bool WHOLE>
__device__ __forceinline__ unsigned load_codes(const uint8_t* p, int left) {
  if constexpr (WHOLE) return *reinterpret_cast<const loose_u32*>(p);
  unsigned r = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) r |= (unsigned)p[e] << (8 * e);
  return r;
}
template <bool WHOLE>
__device__ __forceinline__ void store_codes(uint8_t* p, unsigned codes, int left) {
  if constexpr (WHOLE) {
    *reinterpret_cast<loose_u32*>(p) = codes;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = (uint8_t)(codes >> (8 * e));
  }
}
__device__ __forceinline__ void decode(float (&d)[4], unsigned codes, float scale) {
  d[0] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 0) * scale;
  d[1] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 1) * scale;
  d[2] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 2) * scale;
  d[3] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 3) * scale;
}
__device__ __forceinline__ unsigned encode(const float (&s)[4]) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], r, true);
}

// The largest of all lanes' values, by moves within rows of sixteen and from row to row, in a scalar register.
__device__ __forceinline__ unsigned wave_max(unsigned v) {
  v = std::max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));      // from the lane before
  v = std::max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));      // two before
  v = std::max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));      // four
  v = std::max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));      // eight
  v = std::max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));      // rows 0 and 2 to the next
  v = std::max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));      // row 1 to rows 2 and 3
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
// The scale of a block: its largest magnitude / 448, 0 for zeros, a normal number else (whose inverse is finite), NaN where an
// element is not finite.  The order of the bit patterns is that of the magnitudes, NaN above infinity.
__device__ __forceinline__ float block_scale(const float (&s)[4], float& inverse) {
  unsigned top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = std::max(top, __float_as_uint(s[e]) & 0x7fffffffu);
  const float most = __uint_as_float(wave_max(top));
  const float scale = most == 0.f ? 0.f : most < INFINITY ? std::max(most * (1.f / 448.f), 0x1p-126f) : NAN;
  inverse = __builtin_amdgcn_rcpf(scale);      // to nearest: by what is left over
  inverse = most == 0.f ? 0.f : fmaf(fmaf(inverse, -scale, 1.f), inverse, inverse);
  return scale;
}

// A value of 0 .. 448 up or down to one of e4m3, by 20 random bits: added below the last bit that stays, which is then cut.  Below
// 2^-6 the values are the multiples of 2^-9, as they are between 2^-6 and 2^-5: those are rounded there.
__device__ __forceinline__ float at_random(float q, unsigned bits) {
  const float lift = q < 0x1p-6f ? 0x1p-6f : 0.f;
  const float r = __uint_as_float((__float_as_uint(q + lift) + bits) & 0xfff00000u) - lift;
  return q > 0.f ? std::max(r, 0x1p-9f) : 0.f;
}
// The root to a unit in the last place, small numbers brought among the normal ones first.
__device__ __forceinline__ float root(float v) {
  const bool small = v < 0x1p-96f;
  return __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v) * (small ? 0x1p-32f : 1.f);
}

// The same to nearest, as the reciprocal of a scale: the states in 8 bits are then, bit for bit, those of the formulas in elementary operations
// of 32 bits.  A last place of a root decides some roundings of it, and a block whose largest root is kept one value lower has that scale in all
// steps after.  115 million elements, bf16 with copies: 405 us, 401 with roots that err a unit in the last place.
__device__ __forceinline__ float near_root(float v) {
  const bool small = v < 0x1p-96f;
  const float w = small ? v * 0x1p64f : v, y = __builtin_amdgcn_rsqf(std::max(w, 0x1p-120f)), s = w * y;
  return fmaf(fmaf(-s, s, w) * 0.5f, y, s) * (small ? 0x1p-32f : 1.f);
}

// A value rounded to fp32 here: neither a product that a sum takes unrounded nor a result that goes on to 16 bits unrounded, so
// that what is stored in 16 and in 8 bits is the rounding of the number in 32 that the formula says.
__device__ __forceinline__ float rounded(float v) {
  asm("" : "+v"(v));
  return v;
}

// Four elements of one lane, as they are in memory.
template <typename T, bool MASTER, bool EIGHT>
struct Elements {
  float p[4], g[4], m[4], v[4];
  unsigned cm, cv;
  float sm, sv;
};
template <typename T, bool MASTER, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void load_block(Elements<T, MASTER, EIGHT>& x, const Entry<MASTER, EIGHT>& t, unsigned at, unsigned block) {
  const int left = (int)(t.n - at);
  if constexpr (MASTER) load4<float, WHOLE>(x.p, t.master() + at, left);
  else load4<T, WHOLE>(x.p, (const T*)t.p + at, left);
  load4<T, WHOLE>(x.g, (const T*)t.g + at, left);
  if constexpr (EIGHT) {
    x.cm = load_codes<WHOLE>((const uint8_t*)t.m + at, left);
    x.cv = load_codes<WHOLE>((const uint8_t*)t.v + at, left);
    x.sm = t.m_scale()[block];
    x.sv = t.v_scale()[block];
  } else {
    load4<float, WHOLE>(x.m, (const float*)t.m + at, left);
    load4<float, WHOLE>(x.v, (const float*)t.v + at, left);
  }
}
template <typename T, bool MASTER, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void step_block(Elements<T, MASTER, EIGHT>& x, const StepArgs<MASTER, EIGHT>& a, const Entry<MASTER, EIGHT>& t, const Factors& f,
                                           unsigned at, unsigned block) {
  const int left = (int)(t.n - at);
  float (&p)[4] = x.p, (&g)[4] = x.g, (&m)[4] = x.m, (&v)[4] = x.v;
  if constexpr (EIGHT) {
    decode(m, x.cm, x.sm);
    decode(v, x.cv, x.sv);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = rounded(v[e] * v[e]);
  }
  float r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = rounded(m[e] * a.b1) + rounded(g[e] * a.b1_rest);
    v[e] = rounded(v[e] * a.b2) + rounded(g[e] * g[e] * a.b2_rest);
    r[e] = EIGHT ? near_root(v[e]) : root(v[e]);
    // the reciprocal errs a unit in the last place
    p[e] = rounded(rounded(p[e] * f.keep) - rounded(f.size * (m[e] * __builtin_amdgcn_rcpf(rounded(r[e] * f.root) + a.eps))));
  }
  if constexpr (MASTER) store4<float, WHOLE>(t.master() + at, p, left);
  store4<T, WHOLE>((T*)t.p + at, p, left);
  if constexpr (EIGHT) {
    float inverse, q[4];
    const float m_scale = block_scale(m, inverse);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = __builtin_amdgcn_fmed3f(m[e] * inverse, -448.f, 448.f);
    store_codes<WHOLE>((uint8_t*)t.m + at, encode(q), left);
    const float v_scale = block_scale(r, inverse);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = at_random(std::min(r[e] * inverse, 448.f), mix(f.key + (at + e) * 0x9E3779B1u) >> 12);
    store_codes<WHOLE>((uint8_t*)t.v + at, encode(q), left);
    if ((threadIdx.x & 63) == 0) {
      t.m_scale()[block] = m_scale;
      t.v_scale()[block] = v_scale;
    }
  } else {
    store4<float, WHOLE>((float*)t.m + at, m, left);
    store4<float, WHOLE>((float*)t.v + at, v, left);
  }
}

template <typename T, bool MASTER, bool EIGHT>
__global__ void __launch_bounds__(kThreads) adamw_kernel(StepArgs<MASTER, EIGHT> a) {
  const int lane = threadIdx.x & 63;
  // the last tensor whose first chunk is not behind this one: every lane asks for one
  const unsigned long long before = __ballot(lane < a.entries && a.first[std::min(lane, kAtOnce<MASTER, EIGHT> - 1)] <= blockIdx.x);
  const int own = __popcll(before) - 1;
  const Entry<MASTER, EIGHT> t = a.entry[own];
  const unsigned first = (blockIdx.x - a.first[own]) * (unsigned)a.blocks, all = (t.n + kBlock - 1) / kBlock, end = std::min(first + a.blocks, all);
  unsigned b = __builtin_amdgcn_readfirstlane(first + (threadIdx.x >> 6));
  if (b >= end) return;
  // lanes beyond the end take part in the block's scale
  auto place = [&] { return b < t.n / kBlock ? b * kBlock + lane * 4 : std::min(b * kBlock + lane * 4, t.n); };
  Elements<T, MASTER, EIGHT> x;
  auto load = [&] {
    if (b < t.n / kBlock) load_block<T, MASTER, EIGHT, true>(x, t, place(), b);
    else load_block<T, MASTER, EIGHT, false>(x, t, place(), b);
  };
  load();                          // on its way while the factors are worked out (55 tensors of 3 million elements: 20 us -> 15 with one launch for two)
  Factors f;
  {
    const float now = *t.step + 1.f;
    const double lr = a.lr_ptr ? (double)*a.lr_ptr : a.lr;
    f.keep = (float)(1.0 - lr * a.decay);
    // 1 - b^t for b near 1 without the difference; in fp32: in 64 bits it took a chunk's wavefronts as long as its memory
    f.size = (float)lr / -expm1f(now * a.log_b1);
    f.root = 1.f / sqrtf(-expm1f(now * a.log_b2));
    f.key = mix(a.seed * 0x85157AF5u + t.number * 0x9E3779B1u + (unsigned)now * 0xC2B2AE63u);
  }
  for (;;) {
    if (b < t.n / kBlock) step_block<T, MASTER, EIGHT, true>(x, a, t, f, place(), b);
    else step_block<T, MASTER, EIGHT, false>(x, a, t, f, place(), b);
    if ((b += kWaves) >= end) return;
    load();
  }
}

constexpr int kSteps = 480;
struct CountArgs {
  float* step[kSteps];
  int n;
};
__global__ void __launch_bounds__(kSteps) adamw_count_kernel(CountArgs a) {
  if ((int)threadIdx.x < a.n) *a.step[threadIdx.x] += 1.f;
}

int adamw_check(const cgtp_adamw_args* a) {
  if (!a) return CGTP_ERR_NULL;
  if (a->dtype != CGTP_F32 && a->dtype != CGTP_BF16 && a->dtype != CGTP_F16) return CGTP_ERR_DTYPE;
  if (a->state_bits != 8 && a->state_bits != 32) return CGTP_ERR_CONFIG;
  if (a->n_tensors < 0) return CGTP_ERR_SHAPE;
  if (!(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1)) return CGTP_ERR_CONFIG;
  // it is added in 32 bits, and the sum's inverse is taken: where it is zero, or the inverse infinite, an element without a gradient would become NaN
  if (!(a->eps == 0 || (a->eps >= 0x1p-126 && a->eps <= 0x1.fffffep127))) return CGTP_ERR_CONFIG;
  if (a->n_tensors > 0 && !a->tensors) return CGTP_ERR_NULL;
  for (int64_t i = 0; i < a->n_tensors; ++i) {
    const cgtp_adamw_tensor& t = a->tensors[i];
    if (t.n < 0 || t.n > 0x7fffffff) return CGTP_ERR_SHAPE;
    if (!t.step) return CGTP_ERR_NULL;
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return CGTP_ERR_NULL;
    if (a->state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return CGTP_ERR_NULL;
    if (a->master && !t.master) return CGTP_ERR_NULL;
  }
  if (a->master && a->dtype == CGTP_F32) return CGTP_ERR_CONFIG;
  return CGTP_OK;
}

template <typename T, bool MASTER, bool EIGHT>
void adamw_launch(const cgtp_adamw_args* a, hipStream_t q) {
  StepArgs<MASTER, EIGHT> s = {};
  s.log_b1 = (float)std::log(a->beta1);
  s.log_b2 = (float)std::log(a->beta2);
  s.lr = a->lr;
  s.lr_ptr = a->lr_ptr;
  s.decay = a->weight_decay;
  s.b1 = (float)a->beta1;
  s.b1_rest = (float)(1.0 - a->beta1) * (a->maximize ? -1.f : 1.f);
  s.b2 = (float)a->beta2;
  s.b2_rest = (float)(1.0 - a->beta2);
  s.eps = (float)a->eps;
  s.seed = a->seed;
  int64_t all = 0;
  for (int64_t i = 0; i < a->n_tensors; ++i) all += (a->tensors[i].n + kBlock - 1) / kBlock;
  // Blocks of a chunk: eight for each wavefront of a workgroup, fewer where that leaves compute units idle.
  s.blocks = kWaves * (int)std::max<int64_t>(1, std::min<int64_t>(8, all / (kWaves * 1024)));
  unsigned chunks = 0;
  auto launch = [&] {
    if (s.entries) hipLaunchKernelGGL((adamw_kernel<T, MASTER, EIGHT>), dim3(chunks), dim3(kThreads), 0, q, s);
    s.entries = 0;
    chunks = 0;
  };
  for (int64_t i = 0; i < a->n_tensors; ++i) {
    const cgtp_adamw_tensor& t = a->tensors[i];
    if (t.n == 0) continue;
    // a grid has fewer than 2^32 threads
    const unsigned each = (unsigned)((t.n + kBlock * s.blocks - 1) / (kBlock * s.blocks));
    if (s.entries == kAtOnce<MASTER, EIGHT> || chunks + each >= (1u << 24)) launch();
    Entry<MASTER, EIGHT>& e = s.entry[s.entries];
    e = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.step, {}, (unsigned)t.n, (unsigned)t.number};
    if constexpr (EIGHT) {
      e.more[0] = t.exp_avg_scale;
      e.more[1] = t.exp_avg_sq_scale;
    }
    if constexpr (MASTER) e.more[2 * EIGHT] = t.master;
    s.first[s.entries++] = chunks;
    chunks += each;
  }
  launch();
}
template <typename T>
void adamw_launch(const cgtp_adamw_args* a, hipStream_t q) {
  const bool eight = a->state_bits == 8;
  if constexpr (sizeof(T) == 2)
    if (a->master) return eight ? adamw_launch<T, true, true>(a, q) : adamw_launch<T, true, false>(a, q);
  eight ? adamw_launch<T, false, true>(a, q) : adamw_launch<T, false, false>(a, q);
}

}  // namespace
}  // namespace cgtp

extern "C" {

int cgtp_adamw_step(const cgtp_adamw_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = adamw_check(a)) return rc;
  if (a->n_tensors == 0) return CGTP_OK;
  hipStream_t q = (hipStream_t)stream;
  if (a->dtype == CGTP_F32) adamw_launch<float>(a, q);
  else if (a->dtype == CGTP_BF16) adamw_launch<bf16_t>(a, q);
  else adamw_launch<f16_t>(a, q);
  CountArgs c;
  for (int64_t i = 0; i < a->n_tensors;) {
    for (c.n = 0; c.n < kSteps && i < a->n_tensors; ++i) c.step[c.n++] = a->tensors[i].step;
    hipLaunchKernelGGL(adamw_count_kernel, dim3(1), dim3(kSteps), 0, q, c);
  }
  return launch_status();
}

}  // extern "C"
