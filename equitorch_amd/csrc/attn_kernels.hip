// Attention among the nodes of a structure: entry points, and the kernels that add the heads' parts of the gradients of
// positions and slopes (attn_impl.h has the rest).
#include "attn_host.h"

#include <algorithm>
#include <cmath>

namespace cgtp {
namespace {

// Gradient of the positions of kPosNodes nodes: the parts of their rows (as queries) and of their heads of keys (as keys, where
// the positions are one tensor); and the queries' part of the gradient of every slope.  Eight lanes for a node, a head each at a
// time, added in a fixed order.
constexpr int kPosNodes = 128;
__device__ __forceinline__ void add_heads(const f32x4* part, int64_t node, int heads, int lane8, bool ok, float (&s)[3]) {
  for (int h = lane8; h < heads; h += 8) {
    if (!ok) continue;
    const f32x4 v = part[node * heads + h];
#pragma unroll
    for (int d = 0; d < 3; ++d) s[d] += v[d];
  }
}
__device__ __forceinline__ void write_pos(float* out, int64_t node, int lane8, bool ok, float (&s)[3]) {
#pragma unroll
  for (int d = 0; d < 3; ++d) s[d] = group_sum(s[d], 8);
  if (ok && lane8 < 3) out[node * 3 + lane8] = lane8 == 0 ? s[0] : lane8 == 1 ? s[1] : s[2];
}
__global__ void __launch_bounds__(1024) attn_pos_kernel(cgtp_attn_args a, AttnScratch w) {
  __shared__ float sums[1024];
  const int lane8 = threadIdx.x & 7, sub = threadIdx.x >> 3;
  const int64_t node = (int64_t)blockIdx.x * kPosNodes + sub;
  const bool ok = node < a.n_q;
  if (a.grad_pos_q) {
    float s[3] = {};
    add_heads(w.row_part, node, a.h_q, lane8, ok, s);
    if (a.same_pos) add_heads(w.key_part, node, a.h_kv, lane8, ok, s);
    write_pos(a.grad_pos_q, node, lane8, ok, s);
  }
  if (!a.grad_slope) return;
  for (int h0 = 0; h0 < a.h_q; h0 += 8) {
    const int h = h0 + lane8;
    __syncthreads();
    sums[lane8 * kPosNodes + sub] = ok && h < a.h_q ? w.row_part[node * a.h_q + h][3] : 0.f;
    __syncthreads();
    // a head's 128 values: 16 lanes take eight each
    if (threadIdx.x < 128) {
      const int which = threadIdx.x >> 4, l = threadIdx.x & 15;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += sums[which * kPosNodes + i * 16 + l];
      s = group_sum(s, 16);
      if (l == 0 && h0 + which < a.h_q) {
        if (gridDim.x == 1) a.grad_slope[h0 + which] = s;          // nothing to add it to
        else w.slope_part[(int64_t)(h0 + which) * gridDim.x + blockIdx.x] = s;
      }
    }
  }
}
__global__ void __launch_bounds__(1024) attn_pos_k_kernel(cgtp_attn_args a, AttnScratch w) {
  const int lane8 = threadIdx.x & 7;
  const int64_t node = (int64_t)blockIdx.x * kPosNodes + (threadIdx.x >> 3);
  float s[3] = {};
  add_heads(w.key_part, node, a.h_kv, lane8, node < a.n_k, s);
  write_pos(a.grad_pos_k, node, lane8, node < a.n_k, s);
}
// A workgroup per head: its blocks' parts, each thread every 256th in order, then the threads'.
__global__ void __launch_bounds__(256) attn_slope_kernel(float* out, const float* __restrict__ part, int blocks) {
  __shared__ float sums[4];
  float s = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < blocks; i += 256) s += part[(int64_t)blockIdx.x * blocks + i];
  s = group_sum(s, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) out[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

int64_t blocks_of(int64_t n) { return (n + kPosNodes - 1) / kPosNodes; }

// Rows that leave partial results.
int64_t q_parts(const cgtp_attn_args& a) { return (int64_t)a.n_q_slots * a.h_kv * cgtp_attn_rows(a.wide_q); }

// Workspace of the backward; every buffer starts at a multiple of 256 bytes.  The pieces' results of the two passes share a place.
struct AttnLayout { int64_t row_part, key_part, slope_part, parts, bytes; };
AttnLayout attn_layout(const cgtp_attn_args& a) {
  AttnLayout l;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t was = at; at += (bytes + 255) / 256 * 256; return was; };
  take(a.n_q * a.h_q * 4);
  l.row_part = take(a.slope ? a.n_q * a.h_q * 16 : 0);
  l.key_part = take(a.slope ? a.n_k * a.h_kv * 16 : 0);
  l.slope_part = take(a.slope ? blocks_of(a.n_q) * a.h_q * 4 : 0);
  l.parts = take(std::max(q_parts(a) * (a.dim + kQSums) * 4,
                          (int64_t)a.n_k_slots * a.h_kv * cgtp_attn_rows(a.wide_k) * (2 * a.dim + 4) * 4));
  l.bytes = at;
  return l;
}

int64_t forward_bytes(const cgtp_attn_args& a) { return (q_parts(a) * (a.dim + 2) * 4 + 255) / 256 * 256; }

int attn_check(const cgtp_attn_args* a) {
  if (!a) return CGTP_ERR_NULL;
  if (a->dtype != CGTP_F32 && a->dtype != CGTP_BF16 && a->dtype != CGTP_F16) return CGTP_ERR_DTYPE;
  // keys and rows are counted in 32 bits, up to four tiles of 64 beyond the last one
  constexpr int64_t kMost = 0x7fffffff - 1024;
  if (a->n_q < 0 || a->n_k < 0 || a->n_q > kMost || a->n_k > kMost) return CGTP_ERR_SHAPE;
  if (a->dim <= 0 || a->dim > 128 || a->h_kv <= 0 || a->h_q <= 0 || a->h_q % a->h_kv || a->h_q > 0x3fff) return CGTP_ERR_SHAPE;
  if (a->n_q * (a->h_q / a->h_kv) > kMost) return CGTP_ERR_SHAPE;
  // a grid has fewer than 2^32 threads
  if (a->n_q_items < 0 || a->n_q_joins < 0 || a->n_q_slots < 0 || a->n_k_items < 0 || a->n_k_joins < 0 || a->n_k_slots < 0)
    return CGTP_ERR_SHAPE;
  const int64_t heads = a->h_kv, group = a->h_q / a->h_kv;
  if (a->wide_q < 0 || a->wide_q > 2 || a->wide_k < 0 || a->wide_k > 1) return CGTP_ERR_CONFIG;
  if (a->n_q_items * heads >= (1 << 24) || (int64_t)a->n_k_items * a->h_kv >= (1 << 24)) return CGTP_ERR_SHAPE;
  if (a->n_q_joins * heads * cgtp_attn_rows(a->wide_q) >= (1 << 22) ||
      (int64_t)a->n_k_joins * a->h_kv * cgtp_attn_rows(a->wide_k) >= (1 << 22))
    return CGTP_ERR_SHAPE;
  if ((a->n_q_items && !a->q_items) || (a->n_q_joins && !a->q_joins)) return CGTP_ERR_NULL;
  if (a->n_q > 0 && (!a->q || !a->out)) return CGTP_ERR_NULL;
  if (a->n_k > 0 && (!a->k || !a->v)) return CGTP_ERR_NULL;
  if (a->slope && ((a->n_q > 0 && !a->pos_q) || (a->n_k > 0 && !a->pos_k))) return CGTP_ERR_NULL;
  return CGTP_OK;
}

// Rows that the kernels read where they are: whole aligned chunks of 16 bytes, and the rows of a tile (64 rows are at most 65
// queries' heads) within 31 bits.
bool in_place(const cgtp_attn_args& a, const void* p, int64_t node, int64_t head) {
  const int64_t size = elem_size(a.dtype), chunk = 16 / size, group = a.h_q / a.h_kv;
  return aligned16(p) && node % chunk == 0 && head % chunk == 0 && a.dim % chunk == 0 && node >= 0 && head >= 0 &&
         65 * node * size + group * head * size < (1ll << 31) - 512;
}

// A copy of an operand's rows, each in whole chunks with zeros at its end.  Read once and written once; reading such rows in the
// kernels' own loops took a third of their registers in code that is hardly ever run (20 structures of 1000 nodes, 4 heads
// of 128, bf16, aligned: forward 185 -> 151 us, step 797 -> 693 without it).
template <typename T>
__global__ void __launch_bounds__(256) attn_pack_kernel(const T* from, T* to, int64_t node, int64_t head, int64_t rows, int heads,
                                                        int dim, int chunks) {
  constexpr int N = 16 / sizeof(T);
  const int64_t step = (int64_t)gridDim.x * 256, n = rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
    const int64_t r = i / chunks;
    const int c = (int)(i - r * chunks) * N;
    reinterpret_cast<u32x4_t*>(to)[i] = load_part<u32x4_t, T>(from + r / heads * node + r % heads * head + c, dim - c);
  }
}

// The operands that are copied, one after the other from `at` on; returns where they end.  run: copy, else count.
int64_t pack(AttnLaunch& a, bool backward, int64_t at, bool run, hipStream_t s) {
  const int size = (int)elem_size(a.dtype), chunks = (a.dim * size + 15) / 16, width = chunks * 16 / size;
  auto take = [&](const void*& p, int64_t& node, int64_t& head, int64_t n, int heads) {
    const int64_t rows = n * heads;
    if (rows == 0 || in_place(a, p, node, head)) return;
    if (run) {
      char* to = (char*)a.workspace + at;
      const dim3 grid((unsigned)std::min<int64_t>((rows * chunks + 255) / 256, 1 << 16));
      if (size == 4)
        hipLaunchKernelGGL(attn_pack_kernel<float>, grid, dim3(256), 0, s, (const float*)p, (float*)to, node, head, rows, heads, a.dim, chunks);
      else       // 16 bits are copied as they are
        hipLaunchKernelGGL(attn_pack_kernel<bf16_t>, grid, dim3(256), 0, s, (const bf16_t*)p, (bf16_t*)to, node, head, rows, heads, a.dim, chunks);
      p = to;
      node = (int64_t)heads * width;
      head = width;
    }
    at += (rows * chunks * 16 + 255) / 256 * 256;
  };
  take(a.q, a.q_node, a.q_head, a.n_q, a.h_q);
  take(a.k, a.k_node, a.k_head, a.n_k, a.h_kv);
  take(a.v, a.v_node, a.v_head, a.n_k, a.h_kv);
  a.g_node = (int64_t)a.h_q * a.dim;
  a.g_head = a.dim;
  if (backward) take(a.grad_out, a.g_node, a.g_head, a.n_q, a.h_q);
  return at;
}
AttnLaunch launch_of(const cgtp_attn_args& args) {
  AttnLaunch a;
  static_cast<cgtp_attn_args&>(a) = args;
  return a;
}

template <typename T>
void launch_type(const AttnLaunch& a, const AttnScratch* w, hipStream_t s) {
  if (a.slope) a.cap > 0.f ? attn_launch<T, true, true>(a, w, s) : attn_launch<T, true, false>(a, w, s);
  else a.cap > 0.f ? attn_launch<T, false, true>(a, w, s) : attn_launch<T, false, false>(a, w, s);
}
// A cap that the kernels can form scale / cap and its square with.  Smaller ones are as good as this: scores all but equal.  Larger
// ones do not show before products q.k of 2^52, in scores that differ by more than any softmax tells apart.
float usable_cap(float scale, float cap) {
  if (!(cap > 0.f) || cap > std::fabs(scale) * 0x1p64f) return 0.f;
  return std::max(cap, std::max(std::fabs(scale), 1.f) * 0x1p-100f);
}
// copies: where they start in the workspace.
void launch(const cgtp_attn_args& args, const AttnScratch* w, int64_t copies, hipStream_t s) {
  AttnLaunch a = launch_of(args);
  a.cap = usable_cap(a.scale, a.cap);
  pack(a, w != nullptr, copies, true, s);
  if (a.dtype == CGTP_F32) launch_type<float>(a, w, s);
  else if (a.dtype == CGTP_BF16) launch_type<bf16_t>(a, w, s);
  else launch_type<f16_t>(a, w, s);
}

}  // namespace
}  // namespace cgtp

extern "C" {

int cgtp_attn_rows(int wide) { return wide == 1 ? 128 : 32; }

int64_t cgtp_attn_workspace_bytes(const cgtp_attn_args* a, int backward) {
  using namespace cgtp;
  if (attn_check(a) != CGTP_OK) return 0;
  AttnLaunch l = launch_of(*a);
  return pack(l, backward != 0, backward ? attn_layout(*a).bytes : forward_bytes(*a), false, nullptr);
}

int cgtp_attn_forward(const cgtp_attn_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = attn_check(a)) return rc;
  if (a->n_q == 0) return CGTP_OK;
  if (cgtp_attn_workspace_bytes(a, 0) > 0 && !a->workspace) return CGTP_ERR_WORKSPACE;
  if (!aligned16(a->workspace)) return CGTP_ERR_ALIGN;
  launch(*a, nullptr, forward_bytes(*a), (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? CGTP_OK : CGTP_ERR_LAUNCH;
}

int cgtp_attn_backward(const cgtp_attn_args* a, void* stream) {
  using namespace cgtp;
  if (int rc = attn_check(a)) return rc;
  if ((a->n_k_items && !a->k_items) || (a->n_k_joins && !a->k_joins)) return CGTP_ERR_NULL;
  if (a->n_q > 0 && (!a->lse || !a->grad_out)) return CGTP_ERR_NULL;
  const AttnLayout l = attn_layout(*a);
  if (cgtp_attn_workspace_bytes(a, 1) > 0 && !a->workspace) return CGTP_ERR_WORKSPACE;
  if (!aligned16(a->workspace)) return CGTP_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)a->workspace;
  const AttnScratch w = {(float*)ws, (f32x4*)(ws + l.row_part), (f32x4*)(ws + l.key_part), (float*)(ws + l.slope_part),
                         (float*)(ws + l.parts)};
  launch(*a, &w, l.bytes, s);
  if (a->slope) {
    const unsigned blocks = (unsigned)blocks_of(a->n_q);
    if (blocks && (a->grad_pos_q || a->grad_slope))
      hipLaunchKernelGGL(attn_pos_kernel, dim3(blocks), dim3(1024), 0, s, *a, w);
    if (a->grad_slope && blocks != 1)
      hipLaunchKernelGGL(attn_slope_kernel, dim3((unsigned)a->h_q), dim3(256), 0, s, a->grad_slope, (const float*)w.slope_part, (int)blocks);
    if (!a->same_pos && a->grad_pos_k && a->n_k > 0)
      hipLaunchKernelGGL(attn_pos_k_kernel, dim3((unsigned)blocks_of(a->n_k)), dim3(1024), 0, s, *a, w);
  }
  return hipGetLastError() == hipSuccess ? CGTP_OK : CGTP_ERR_LAUNCH;
}

}  // extern "C"
