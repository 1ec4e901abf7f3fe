// Kernels of the attention among the nodes of a structure for one element type, with or without distances and cap (the
// attn_<type>_*.hip: both are known when a kernel is compiled, a branch on them costs more than what it leaves out).
//
//   t_ij = log2(e) s_ij,  s_ij = cap tanh(scale q_i.k_j / cap) - slope_h |r_i - r_j|
//   out_i = sum_j 2^(t_ij - lse_i) v_j,  lse_i = log2 sum_j 2^t_ij
//   p_ij = 2^(t_ij - lse_i),  dp_ij = dout_i.v_j,  delta_i = dout_i.out_i,  ds_ij = p_ij (dp_ij - delta_i)
//   dv_j = sum_i p_ij dout_i,   du_ij = ds_ij (1 - tanh^2),   dq_i = scale sum_j du_ij k_j,  dk_j = scale sum_i du_ij q_i
//   dslope_h = -sum ds_ij |r_i - r_j|,   dr_i = -slope sum_j ds_ij (r_i - r_j) / |r_i - r_j|,  dr_j the opposite
//
// One pass over the keys with the running maximum and sum of each row (forward); the backward forms the scores again, once
// with the rows fixed (dq, dr_i, dslope) and once with the keys fixed (dk, dv, dr_j), so that every sum is held by one
// workgroup and no result depends on timing.
//
// A row is a (query, query head) pair of one head of keys: heads that share keys and values share the tiles in LDS, and a
// single query of a structure brings all its heads to one tile.  A wavefront owns 32 rows (or 32 keys) and forms the scores with
// the other operand's rows down the registers, so that a row's statistics take one exchange between the halves of the
// wavefront and the probabilities are the next product's operand as they lie.  Tiles never cross structures: what another
// structure holds, infinities and NaN included, is never read.  A key or row of a tile beyond its range is a zero in LDS (in
// the backward's scores the last one once more) and its probability zero.
#pragma once

#include "attn_tiles.h"
#include "attn_host.h"

namespace cgtp {
namespace {

constexpr float kLog2E = 1.4426950408889634f;
// Bounds of a squared distance in the backward, whose distance is d2 / sqrt(d2): a distance of zero gives 3e-19 and no direction, and a
// node so far off that d2 is infinite (-inf for its score in the forward, taking it out) the probability 0, not inf * 0.
constexpr float kNear2 = 1e-37f, kFar2 = 3e38f;

template <int NW> constexpr int kRowsOf = 32 * NW;
// Rows of a tile in LDS: 64 where four wavefronts move them, half of that for rows beyond 256 bytes, whose tiles on their way
// leave registers for one wavefront on a SIMD else (20 structures of 1000 nodes, 4 heads of 96, fp32: forward 364 -> 334 us,
// gradient of keys and values 738 -> 649).
template <typename T, int DP, int NW> constexpr int kBlockOf = NW == 1 || DP * sizeof(T) > 256 ? 32 : 64;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Scores of a block, in binary orders.  Without distances and cap the forward takes t = q.k, in units of `unit` orders (the
// scale, where that is positive); else t = linear q.k, or with a cap t = outer tanh(u), u = to_u q.k, and slope' times the
// distance is taken off when a score is used.
//
// tanh: 1 - 2 / (e^2u + 1) takes eleven issue slots and errs by 2^-24 of the cap, however small the score.  Scores are mostly far
// below their cap: where all of a wavefront's block have |u| <= kNear, the Taylor series does, in five slots (16-bit types: up to
// u^7, relative error 5e-6 at 0.35; fp32: up to u^9, 8e-9 at 0.25, and also for the small scores of a block with
// larger ones).  Forward of three structures of 2000 to 5000 nodes, 8 query heads on 4 of 64, bf16: 347 -> 330 us.
template <typename T, bool BIASED, bool CAPPED>
struct Score {
  static constexpr bool kWide = sizeof(T) == 4;
  float linear, unit, to_u, outer, by_outer, near, c[4];
  __device__ __forceinline__ explicit Score(const AttnLaunch& a) {
    linear = a.scale * kLog2E;
    unit = plain() ? linear : 1.f;
    if constexpr (CAPPED) {
      to_u = a.scale / a.cap;
      outer = a.cap * kLog2E;
      by_outer = 1.f / outer;
      near = kWide ? 0.25f : 0.35f;
      const float z = to_u * to_u;
      c[0] = linear * z * (-1.f / 3.f);
      c[1] = linear * z * z * (2.f / 15.f);
      c[2] = linear * z * z * z * (-17.f / 315.f);
      c[3] = linear * z * z * z * z * (62.f / 2835.f);
      // A cap far below the scale takes them past fp32.  The other form serves alone then: what it errs by is 2^-24 of that cap.
      if (!(fabsf(c[0]) + fabsf(c[1]) + fabsf(c[2]) + fabsf(c[3]) <= 1e38f)) near = -1.f;
    }
  }
  __device__ __forceinline__ bool plain() const { return !CAPPED && !BIASED && linear > 0.f; }
  __device__ __forceinline__ float series(float qk) const {
    const float z = qk * qk;
    float p = kWide ? fmaf(z, c[3], c[2]) : c[2];
    p = fmaf(z, p, c[1]);
    p = fmaf(z, p, c[0]);
    return qk * fmaf(z, p, linear);
  }
  // t from q.k; raw: left in units of `unit`.
  __device__ __forceinline__ void of(f32x16_t& t, bool raw = false) const {
    if constexpr (CAPPED) {
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(t[e]));
      if (__all(most * fabsf(to_u) <= near)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) t[e] = series(t[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float u = to_u * t[e], far = fmaf(-2.f * outer, __builtin_amdgcn_rcpf(exp2_fast(2.f * kLog2E * u) + 1.f), outer);
          t[e] = kWide && fabsf(u) <= near ? series(t[e]) : far;
        }
      }
    } else if (!raw) {
#pragma unroll
      for (int e = 0; e < 16; ++e) t[e] *= linear;
    }
  }
  __device__ __forceinline__ float less(float t, float slope, float dist) const { return BIASED ? fmaf(-slope, dist, t) : t; }
  // The gradient of t / linear with respect to q.k.
  __device__ __forceinline__ float through(float t) const {
    if constexpr (!CAPPED) return 1.f;
    const float th = t * by_outer;
    return fmaf(-th, th, 1.f);
  }
};
__device__ __forceinline__ float half_swap(float x) { return __shfl_xor(x, 32, kWave); }

struct Row {
  int query, head;     // of the tensors
  bool ok;
};
__device__ __forceinline__ Row row_of(const cgtp_attn_item& it, int r, int kv_head, int group) {
  Row o;
  o.ok = r < it.row_end;
  const int rr = o.ok ? r : it.row_begin;
  o.query = it.node + rr / group;
  o.head = kv_head * group + rr % group;
  return o;
}

// The keys of a tile, from k0 on, n of them.
template <typename T>
struct KeyRows {
  const T* base;
  int64_t node;
  int n;
  __device__ __forceinline__ KeyRows(const T* p, int64_t node, int64_t head, int hk, int k0, int n)
      : base(p + (int64_t)k0 * node + hk * head), node(node), n(n) {}
  __device__ __forceinline__ unsigned offset(int i) const { return i < n ? (unsigned)i * (unsigned)(node * sizeof(T)) : kNoRow; }
  // The last row again for those beyond: what has no part in a sum is a score like the others, not a zero times an infinity.
  __device__ __forceinline__ unsigned offset_again(int i) const { return offset(min(i, n - 1)); }
};
// The rows of a tile, from r0 on, n of them: query0 + (at + i) / group, head (at + i) % group of the kv head's.
template <typename T>
struct QueryRows {
  const T* base;       // first query's first head
  int64_t node, head;
  int n, at, group;
  float inv;
  __device__ __forceinline__ QueryRows(const T* p, int64_t node, int64_t head, int first_query, int hk, int group, int r0, int n)
      : node(node), head(head), n(n), at(r0 % group), group(group), inv(1.f / (float)group) {
    base = p + (int64_t)(first_query + r0 / group) * node + (int64_t)hk * group * head;
  }
  // Quotients of small numbers: (x + 1 / 2) / group is at least 1 / (2 group) away from an integer.
  __device__ __forceinline__ int query(int i) const { return (int)(((float)(at + i) + 0.5f) * inv); }
  __device__ __forceinline__ unsigned offset(int i) const {
    const int q = query(i), h = at + i - q * group;
    return i < n ? (unsigned)q * (unsigned)(node * sizeof(T)) + (unsigned)h * (unsigned)(head * sizeof(T)) : kNoRow;
  }
  __device__ __forceinline__ unsigned offset_again(int i) const { return offset(min(i, n - 1)); }
};

// One tile buffer of LDS where two would not leave room for two workgroups.
template <int BYTES> constexpr int kBuffers = 2 * BYTES <= 64 * 1024 ? 2 : 1;

// Wavefronts that share out the keys of one tile of rows (KS > 1): each has its own tiles in LDS and waits for nobody, the
// LDS taking one wavefront's accesses in order; their results are joined at the end.
template <int KS>
__device__ __forceinline__ void tile_sync() {
  if constexpr (KS == 1) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}
// A wavefront that moves its own tiles of long rows: both tiles of a step on their way at once would take half its registers, and
// two buffers of both the LDS of most wavefronts that a compute unit has room for.  One tile is fetched while the other
// one is worked on, into the same registers, and in the forward into the same place.  2000 structures of up to 20 nodes, 8 query
// heads on 2 of 128, fp32: forward 137 -> 92 us, step 546 -> 350; of 64: 60 -> 44 and 343 -> 186.
template <typename T, int DP, int NW> constexpr bool kLean = NW == 1 && DP * sizeof(T) > 128;

// Bytes of LDS for the tiles of a step (`lean`: how many of the two are there at a time), or for half the wavefronts' results of
// `sums` values for each lane.
template <typename T, int DP, int NW, int KS>
constexpr int attn_lds(int lean, int sums) {
  constexpr int one = kBlockOf<T, DP, NW> * AttnShape<T, DP>::kRow, tile = 2 * one;
  const int tiles = kLean<T, DP, NW> ? KS * lean * one : KS > 1 ? KS * tile : kBuffers<tile> * tile, join = KS > 1 ? KS / 2 * 64 * (16 * AttnShape<T, DP>::kOut + sums) * 4 : 0;
  return tiles > join ? tiles : join;
}
// Halves the number of wavefronts that hold results until one does: give(value place) and take of each value, `n` for a lane.
template <int KS, typename Give, typename Take>
__device__ __forceinline__ void join_waves(float* lds, int n, Give&& give, Take&& take) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int s = KS / 2; s >= 1; s >>= 1) {
    __syncthreads();
    float* at = lds + (wave % s) * n * 64 + lane;
    if (wave >= s && wave < 2 * s) give(at);
    __syncthreads();
    if (wave < s) take(at);
  }
}


// ---- forward ----------------------------------------------------------------------------------------------------
// Vector instructions bound it with distances: some 25 issue slots for a score (a root and an exponential take four each), 79 %
// of all slots used, the matrix cores 14 %.  300 structures of 40 to 250 nodes, 8 heads of 32, bf16, cap: 59 us; three of
// 2000 to 5000, 8 query heads on 4 of 64: 311 us.  Without distances and cap the matrix cores and LDS do: one of 12007, 16 query
// heads on 4 of 128, fp16: 1.35 to 1.43 ms, 830 to 877 TFLOP/s, 0.75 of what a large library product reaches.
//
// NW wavefronts of 32 rows share the tiles of keys (wide_q 1), or KS share out the keys of one tile of rows and join their
// results in LDS (wide_q 2: 64 readouts of one query over up to 400 keys, fp32, 30 us with one wavefront each, 15 so; one query
// of 8 heads on 2 of 64 over 200003 keys, bf16: 24 us, 4.3 TB/s of keys and values).
// Four wavefronts on a SIMD where a row is short and they wait for each other (20 structures of 1000 nodes, 4 heads of 32, bf16:
// 59 us with three, 50 so).
template <typename T, int DP, int NW, int KS, bool BIASED, bool CAPPED>
__global__ void __launch_bounds__(64 * NW * KS, sizeof(T) == 2 && DP <= 32 ? 4 : NW == 4 || DP * sizeof(T) <= 256 ? 2 : 1)
attn_fwd_kernel(AttnLaunch a, float* __restrict__ parts) {
  using S = AttnShape<T, DP>;
  constexpr int kBlock = kBlockOf<T, DP, NW>, kTile = kBlock * S::kRow, kBuf = KS > 1 || kLean<T, DP, NW> ? 1 : kBuffers<2 * kTile>;
  constexpr bool LEAN = kLean<T, DP, NW>;
  __shared__ alignas(16) char lds[attn_lds<T, DP, NW, KS>(1, 2)];
  __shared__ alignas(16) float all_pos[KS][2][3][kBlock];
  const int hk = blockIdx.x % a.h_kv, group = a.h_q / a.h_kv;
  const cgtp_attn_item it = a.q_items[blockIdx.x / a.h_kv];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6, tid = KS > 1 ? lane : (int)threadIdx.x;
  const int r = it.row_begin + (KS > 1 ? 0 : wave * 32) + (lane & 31), part = KS > 1 ? wave : 0;
  char* const tiles = lds + part * (LEAN ? 1 : 2) * kTile;
  auto& pos = all_pos[part];
  const Row row = row_of(it, r, hk, group);
  const Score<T, BIASED, CAPPED> sc(a);
  RowFrag<T, DP> q;
  q.load(row.ok ? (const T*)a.q + row.query * a.q_node + row.head * a.q_head : nullptr, a.dim);
  float x = 0.f, y = 0.f, z = 0.f, slope = 0.f;
  if (BIASED && row.ok) {
    x = a.pos_q[(int64_t)row.query * 3];
    y = a.pos_q[(int64_t)row.query * 3 + 1];
    z = a.pos_q[(int64_t)row.query * 3 + 2];
    slope = a.slope[row.head] * kLog2E;
  }
  AttnAcc<T, DP> acc;
#pragma unroll
  for (int o = 0; o < S::kOut; ++o)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[o][e] = 0.f;
  float top = -INFINITY, sum = 0.f;           // of the row's keys (top), of this lane's (sum)
  TileStage<T, DP, 64 * NW, kBlock> ks, other;
  auto& vs = LEAN ? ks : other;
  float ps[3] = {};
  auto fetch_v = [&](int k0) {
    const int n = it.k_end - k0;
    const KeyRows<T> vr((const T*)a.v, a.v_node, a.v_head, hk, k0, n);
    vs.load(vr.base, a.dim, [&](int i) { return vr.offset(i); });
  };
  auto fetch = [&](int k0) {
    const int n = it.k_end - k0;
    const KeyRows<T> kr((const T*)a.k, a.k_node, a.k_head, hk, k0, n);
    ks.load(kr.base, a.dim, [&](int i) { return kr.offset(i); });
    if (!LEAN) fetch_v(k0);
    if (BIASED && tid < kBlock)
#pragma unroll
      for (int d = 0; d < 3; ++d) ps[d] = tid < n ? a.pos_k[(int64_t)(k0 + tid) * 3 + d] : 0.f;
  };
  const int first = it.k_begin + part * kBlock;
  if (first < it.k_end) fetch(first);
  int buf = 0;
  for (int k0 = first; k0 < it.k_end; k0 += KS * kBlock, buf ^= 1) {
    const int n = it.k_end - k0;
    char* const k_tile = tiles + (kBuf == 2 ? buf : 0) * 2 * kTile;
    char* const v_tile = LEAN ? k_tile : k_tile + kTile;
    if (kBuf == 1) tile_sync<KS>();
    ks.store(k_tile);
    if (!LEAN) vs.store(v_tile);
    if (BIASED && tid < kBlock)
#pragma unroll
      for (int d = 0; d < 3; ++d) pos[buf][d][tid] = ps[d];
    tile_sync<KS>();
    if (LEAN) fetch_v(k0);
    else if (k0 + KS * kBlock < it.k_end) fetch(k0 + KS * kBlock);
    f32x16_t t[kBlock / 32];
    float most = top;
#pragma unroll
    for (int b = 0; b < kBlock / 32; ++b) {
      if (b * 32 >= n) continue;
      t[b] = rows_times<T, DP>(k_tile, 32 * b, q);
      sc.of(t[b], sc.plain());
      if constexpr (BIASED) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int at = 32 * b + 8 * g + 4 * half;
          const f32x4 px = *reinterpret_cast<const f32x4*>(&pos[buf][0][at]),
                      py = *reinterpret_cast<const f32x4*>(&pos[buf][1][at]),
                      pz = *reinterpret_cast<const f32x4*>(&pos[buf][2][at]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float dx = x - px[e], dy = y - py[e], dz = z - pz[e];
            t[b][4 * g + e] = sc.less(t[b][4 * g + e], slope, __builtin_amdgcn_sqrtf(dx * dx + dy * dy + dz * dz));
          }
          if (LEAN) __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (n < 32 * b + 32)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * b + 8 * (e >> 2) + 4 * half + (e & 3) >= n) t[b][e] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) most = fmaxf(most, t[b][e]);
    }
    most = fmaxf(most, half_swap(most));
    if (__any(most > top)) {
      const float by = top == most ? 1.f : exp2_fast((top - most) * sc.unit);      // equal: also both -inf
      sum *= by;
#pragma unroll
      for (int o = 0; o < S::kOut; ++o)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[o][e] *= by;
      top = most;
    }
    const float base = top == -INFINITY ? 0.f : fmaf(-top, sc.unit, (float)kUp<T>);
#pragma unroll
    for (int b = 0; b < kBlock / 32; ++b) {
      if (b * 32 >= n) continue;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        t[b][e] = exp2_fast(fmaf(t[b][e], sc.unit, base));
        sum += t[b][e];
      }
      if (LEAN) {
        tile_sync<KS>();
        vs.store(v_tile);
        tile_sync<KS>();
        if (k0 + KS * kBlock < it.k_end) fetch(k0 + KS * kBlock);
      }
      cols_times<T, DP>(acc, v_tile, 32 * b, t[b]);
    }
  }
  top = fmaf(top, sc.unit, (float)-kUp<T>);
  if constexpr (KS > 1) {
    join_waves<KS>(reinterpret_cast<float*>(lds), 16 * S::kOut + 2, [&](float* at) {
      at[0] = top;
      at[64] = sum;
#pragma unroll
      for (int i = 0; i < 16 * S::kOut; ++i) at[(2 + i) * 64] = acc[i / 16][i % 16];
    }, [&](const float* at) {
      const float top2 = at[0], most = fmaxf(top, top2);
      const float f1 = top == most ? 1.f : exp2_fast(top - most), f2 = top2 == most ? 1.f : exp2_fast(top2 - most);
      sum = sum * f1 + at[64] * f2;
#pragma unroll
      for (int i = 0; i < 16 * S::kOut; ++i) acc[i / 16][i % 16] = acc[i / 16][i % 16] * f1 + at[(2 + i) * 64] * f2;
      top = most;
    });
    if (wave) return;
  }
  sum += half_swap(sum);
  if (!row.ok) return;
  if (it.slot < 0) {
    const bool some = sum > 0.f || sum != sum;
    const int64_t at = (int64_t)row.query * a.h_q + row.head;
    const float by = some ? 1.f / sum : 0.f;
    store_cols<T, DP>((T*)a.out + at * a.dim, acc, by, a.dim);
    if (a.lse && half == 0) ((float*)a.lse)[at] = some ? top + __log2f(sum) : INFINITY;
  } else {
    float* p = parts + (((int64_t)it.slot * a.h_kv + hk) * kRowsOf<NW> + (r - it.row_begin)) * (a.dim + 2);
    store_cols<float, (DP < 32 ? 32 : DP)>(p, acc, 1.f, a.dim);
    if (half == 0) {
      p[a.dim] = top;
      p[a.dim + 1] = sum;
    }
  }
}

// Adds the parts of a row: a workgroup for each (tile, head of keys, row), its slots shared out over slices of threads.  A few
// slots in flight for each thread: bound by latency, 6 us for that query.
constexpr int kJoinThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) attn_fwd_join_kernel(AttnLaunch a, const float* __restrict__ parts, int rows) {
  const int heads = a.h_kv;
  __shared__ float acc[kJoinThreads], red[kJoinThreads / kWave];
  const int group = a.h_q / heads, rr = blockIdx.x % rows, hk = blockIdx.x / rows % heads;
  const cgtp_attn_item it = a.q_joins[blockIdx.x / rows / heads];
  const Row row = row_of(it, it.row_begin + rr, hk, group);
  if (!row.ok) return;
  const int tid = threadIdx.x, width = a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128, slices = kJoinThreads / width;
  const int64_t step = (int64_t)heads * rows * (a.dim + 2);
  const float* p = parts + (((int64_t)it.first * heads + hk) * rows + rr) * (a.dim + 2);
  float top = -INFINITY;
  for (int s = tid; s < it.count; s += kJoinThreads) top = fmaxf(top, p[s * step + a.dim]);
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / kWave; ++w) top = fmaxf(top, red[w]);
  const float base = top == -INFINITY ? 0.f : top;
  const int d = tid % width;
  float o = 0.f, sum = 0.f;
#pragma unroll 4
  for (int s = tid / width; s < it.count; s += slices) {
    const float* ps = p + s * step;
    const float by = exp2_fast(ps[a.dim] - base);
    sum += by * ps[a.dim + 1];
    o += by * (d < a.dim ? ps[d] : 0.f);
  }
  acc[tid] = o;
  __syncthreads();
  float total = 0.f;
  if (tid < width)
    for (int s = 0; s < slices; ++s) total += acc[s * width + tid];
  __syncthreads();
  acc[tid] = sum;
  __syncthreads();
  if (tid >= width) return;
  sum = 0.f;
  for (int s = 0; s < slices; ++s) sum += acc[s * width];
  const bool some = sum > 0.f || sum != sum;
  const int64_t at = (int64_t)row.query * a.h_q + row.head;
  if (d < a.dim) {
    const float o = some ? total / sum : 0.f;
    ((T*)a.out)[at * a.dim + d] = (T)o;
  }
  if (a.lse && tid == 0) ((float*)a.lse)[at] = some ? top + __log2f(sum) : INFINITY;
}

// The same where a row has few slots: an element to a thread.  Bound by memory: 30 us for the parts of three structures of 2000 to
// 5000 nodes.
template <typename T>
__global__ void __launch_bounds__(256) attn_fwd_join_few_kernel(AttnLaunch a, const float* __restrict__ parts, int rows) {
  const int heads = a.h_kv;
  const int group = a.h_q / heads, hk = blockIdx.x % heads, width = a.dim + 1;
  const cgtp_attn_item it = a.q_joins[blockIdx.x / heads];
  const int here = it.row_end - it.row_begin;
  const int64_t step = (int64_t)heads * rows * (a.dim + 2);
  for (int e = blockIdx.y * 256 + threadIdx.x; e < here * width; e += gridDim.y * 256) {
    const int r = e / width, d = e % width;
    const float* p = parts + (((int64_t)it.first * heads + hk) * rows + r) * (a.dim + 2);
    float top = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < it.count; ++k) top = fmaxf(top, p[k * step + a.dim]);
    const float base = top == -INFINITY ? 0.f : top;
    float o = 0.f, sum = 0.f;
#pragma unroll 4
    for (int k = 0; k < it.count; ++k) {
      const float by = exp2_fast(p[k * step + a.dim] - base);
      sum += by * p[k * step + a.dim + 1];
      o += by * p[k * step + d];             // the last element is not used
    }
    const bool some = sum > 0.f || sum != sum;
    const Row row = row_of(it, it.row_begin + r, hk, group);
    const int64_t at = (int64_t)row.query * a.h_q + row.head;
    if (d < a.dim) {
      o = some ? o / sum : 0.f;
      ((T*)a.out)[at * a.dim + d] = (T)o;
      } else if (a.lse) {
      ((float*)a.lse)[at] = some ? top + __log2f(sum) : INFINITY;
    }
  }
}

// A row's sums over its keys besides its gradient, and its delta.
struct QSums {
  float v[kQSums];
  __device__ __forceinline__ void finish(const AttnScratch& w, int64_t at, float slope, bool biased) const {
    const float off = v[8];
    w.delta[at] = v[9] + off;
    if (!biased) return;
    w.row_part[at] = f32x4{-slope * (v[0] - off * v[4]), -slope * (v[1] - off * v[5]), -slope * (v[2] - off * v[6]),
                           off * v[7] - v[3]};
  }
};

// ---- gradient with the rows fixed ---------------------------------------------------------------------------------
// Bound by vector instructions as the forward is (84 % of the slots): the score again, and the sums for positions and slopes.
// The two workloads above: 109 and 511 us.
template <typename T, int DP, int NW, int KS, bool BIASED, bool CAPPED>
__global__ void __launch_bounds__(64 * NW * KS, DP <= (sizeof(T) == 4 ? 64 : 96) ? 2 : 1)
attn_bwd_q_kernel(AttnLaunch a, AttnScratch w) {
  using S = AttnShape<T, DP>;
  constexpr int kBlock = kBlockOf<T, DP, NW>, kTile = kBlock * S::kRow, kBuf = KS > 1 || kLean<T, DP, NW> ? 1 : kBuffers<2 * kTile>;
  constexpr bool LEAN = kLean<T, DP, NW>;
  __shared__ alignas(16) char lds[attn_lds<T, DP, NW, KS>(2, 9)];
  __shared__ alignas(16) float all_pos[KS][2][3][kBlock];
  const int hk = blockIdx.x % a.h_kv, group = a.h_q / a.h_kv;
  const cgtp_attn_item it = a.q_items[blockIdx.x / a.h_kv];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6, tid = KS > 1 ? lane : (int)threadIdx.x;
  const int r = it.row_begin + (KS > 1 ? 0 : wave * 32) + (lane & 31), part = KS > 1 ? wave : 0;
  char* const tiles = lds + part * 2 * kTile;
  auto& pos = all_pos[part];
  const Row row = row_of(it, r, hk, group);
  const int64_t at = (int64_t)row.query * a.h_q + row.head;
  const Score<T, BIASED, CAPPED> sc(a);
  RowFrag<T, DP> q, g;
  q.load(row.ok ? (const T*)a.q + row.query * a.q_node + row.head * a.q_head : nullptr, a.dim);
  g.load(row.ok ? (const T*)a.grad_out + row.query * a.g_node + row.head * a.g_head : nullptr, a.dim);
  float delta = 0.f;
  {
    RowFrag<T, DP> o;
    o.template load<false>(row.ok ? (const T*)a.out + at * a.dim : nullptr, a.dim);
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      typedef T vec __attribute__((ext_vector_type(S::kChunk)));
      const vec go = __builtin_bit_cast(vec, g.f[s]), oo = __builtin_bit_cast(vec, o.f[s]);
#pragma unroll
      for (int j = 0; j < S::kChunk; ++j) delta = fmaf((float)go[j], (float)oo[j], delta);
    }
    delta += half_swap(delta);
  }
  const float lse = row.ok ? ((const float*)a.lse)[at] : INFINITY;
  float x = 0.f, y = 0.f, z = 0.f, slope = 0.f;
  if (BIASED && row.ok) {
    x = a.pos_q[(int64_t)row.query * 3];
    y = a.pos_q[(int64_t)row.query * 3 + 1];
    z = a.pos_q[(int64_t)row.query * 3 + 2];
    slope = a.slope[row.head];
  }
  const float slope2 = slope * kLog2E;
  AttnAcc<T, DP> acc;
#pragma unroll
  for (int o = 0; o < S::kOut; ++o)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[o][e] = 0.f;
  // Sums over the keys of ds (r_i - r_j) / |r_i - r_j| and of ds |r_i - r_j|; in 16-bit types also of ds, and of the others with
  // p for ds (kFix).  delta is against an output that was summed from rounded probabilities and rounded itself: the
  // exact one is delta + sum ds, and with it the gradients of positions and slopes, which are fp32, err as in fp32.  It is known
  // when the row is done: the row's own dq, rounded to 16 bits anyway, goes without.
  constexpr bool kFix = sizeof(T) == 2;
  QSums m = {};
  ColumnFit<T, DP> fit;
  TileStage<T, DP, 64 * NW, kBlock> ks, other;
  auto& vs = LEAN ? ks : other;
  float ps[3] = {};
  auto fetch_v = [&](int k0) {
    const int n = it.k_end - k0;
    const KeyRows<T> vr((const T*)a.v, a.v_node, a.v_head, hk, k0, n);
    vs.load(vr.base, a.dim, [&](int i) { return vr.offset(i); });
  };
  auto fetch = [&](int k0) {
    const int n = it.k_end - k0;
    const KeyRows<T> kr((const T*)a.k, a.k_node, a.k_head, hk, k0, n);
    ks.load(kr.base, a.dim, [&](int i) { return kr.offset_again(i); });
    if (!LEAN) fetch_v(k0);
    if (BIASED && tid < kBlock)
#pragma unroll
      for (int d = 0; d < 3; ++d) ps[d] = tid < n ? a.pos_k[(int64_t)(k0 + tid) * 3 + d] : 0.f;
  };
  const int first = it.k_begin + part * kBlock;
  if (first < it.k_end) fetch(first);
  int buf = 0;
  for (int k0 = first; k0 < it.k_end; k0 += KS * kBlock, buf ^= 1) {
    const int n = it.k_end - k0;
    char* const k_tile = tiles + (kBuf == 2 ? buf : 0) * 2 * kTile;
    char* const v_tile = k_tile + kTile;
    if (kBuf == 1) tile_sync<KS>();
    ks.store(k_tile);
    if (!LEAN) vs.store(v_tile);
    if (BIASED && tid < kBlock)
#pragma unroll
      for (int d = 0; d < 3; ++d) pos[buf][d][tid] = ps[d];
    tile_sync<KS>();
    if (LEAN) fetch_v(k0);
    else if (k0 + KS * kBlock < it.k_end) fetch(k0 + KS * kBlock);
#pragma unroll 1
    for (int b = 0; b < kBlock / 32; ++b) {
      if (b * 32 >= n) continue;
      f32x16_t t = rows_times<T, DP>(k_tile, 32 * b, q);
      sc.of(t);
      if (LEAN) {
        vs.store(v_tile);
        tile_sync<KS>();
        if (k0 + KS * kBlock < it.k_end) fetch(k0 + KS * kBlock);
      }
      f32x16_t ds = rows_times<T, DP>(v_tile, 32 * b, g);
      auto turn = [&](bool cut) {
#pragma unroll
        for (int gq = 0; gq < 4; ++gq) {
          const int first = 32 * b + 8 * gq + 4 * half;
          f32x4 px = {}, py = {}, pz = {};
          if constexpr (BIASED) {
            px = *reinterpret_cast<const f32x4*>(&pos[buf][0][first]);
            py = *reinterpret_cast<const f32x4*>(&pos[buf][1][first]);
            pz = *reinterpret_cast<const f32x4*>(&pos[buf][2][first]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * gq + e;
            float dx = 0.f, dy = 0.f, dz = 0.f, d2 = 0.f, inv = 0.f;
            if constexpr (BIASED) {
              dx = x - px[e];
              dy = y - py[e];
              dz = z - pz[e];
              d2 = __builtin_amdgcn_fmed3f(dx * dx + dy * dy + dz * dz, kNear2, kFar2);
              inv = __builtin_amdgcn_rsqf(d2);
            }
            float p = exp2_fast(sc.less(t[i], slope2, d2 * inv) - lse);
            if (cut && first + e >= n) p = 0.f;
            float d = p * (ds[i] - delta);
            if constexpr (BIASED) {
              const float u = d * inv;
              m.v[0] = fmaf(u, dx, m.v[0]);
              m.v[1] = fmaf(u, dy, m.v[1]);
              m.v[2] = fmaf(u, dz, m.v[2]);
              m.v[3] = fmaf(u, d2, m.v[3]);
              if constexpr (kFix) {
                const float near = p * inv;
                m.v[4] = fmaf(near, dx, m.v[4]);
                m.v[5] = fmaf(near, dy, m.v[5]);
                m.v[6] = fmaf(near, dz, m.v[6]);
                m.v[7] = fmaf(near, d2, m.v[7]);
                m.v[8] += d;
              }
            }
            if constexpr (CAPPED) d *= sc.through(t[i]);
            ds[i] = d;
          }
          __builtin_amdgcn_sched_barrier(0);      // keeps the next group's reads from LDS out of the registers
        }
      };
      if (n < 32 * b + 32) turn(true);
      else turn(false);
      fit.fit(ds, acc);
      cols_times<T, DP>(acc, k_tile, 32 * b, ds);
    }
  }
  if constexpr (KS > 1) {
    fit.settle(acc);
    join_waves<KS>(reinterpret_cast<float*>(lds), 16 * S::kOut + 9, [&](float* at) {
#pragma unroll
      for (int i = 0; i < 9; ++i) at[i * 64] = m.v[i];
#pragma unroll
      for (int i = 0; i < 16 * S::kOut; ++i) at[(9 + i) * 64] = acc[i / 16][i % 16];
    }, [&](const float* at) {
#pragma unroll
      for (int i = 0; i < 9; ++i) m.v[i] += at[i * 64];
#pragma unroll
      for (int i = 0; i < 16 * S::kOut; ++i) acc[i / 16][i % 16] += at[(9 + i) * 64];
    });
    if (wave) return;
  }
#pragma unroll
  for (int i = 0; i < (kFix ? 9 : 4); ++i) m.v[i] += half_swap(m.v[i]);
  m.v[9] = delta;
  if (!row.ok) return;
  if (lse == INFINITY) {                  // no key, or every score -inf: a key of infinities times a gradient of zero is none
#pragma unroll
    for (int i = 0; i < 9; ++i) m.v[i] = 0.f;
#pragma unroll
    for (int i = 0; i < 16 * S::kOut; ++i) acc[i / 16][i % 16] = 0.f;
  }
  const float grad_scale = fit.undo(a.scale);
  if (it.slot < 0) {
    if (a.grad_q) store_cols<T, DP>((T*)a.grad_q + at * a.dim, acc, grad_scale, a.dim);
    if (half == 0) m.finish(w, at, slope, BIASED);
  } else {
    float* p = w.parts + (((int64_t)it.slot * a.h_kv + hk) * kRowsOf<NW> + (r - it.row_begin)) * (a.dim + kQSums);
    store_cols<float, (DP < 32 ? 32 : DP)>(p, acc, grad_scale, a.dim);
    if (half == 0)
#pragma unroll
      for (int i = 0; i < kQSums; ++i) p[a.dim + i] = m.v[i];
  }
}

// Adds the parts of a tile's rows or keys, `width` values for each, elements from .. from + n - 1 of them: an element of the
// tile to a thread, its slots in order, the threads of the workgroups y of `ys`.  put(row or key, element, sum).
template <typename Put>
__device__ __forceinline__ void join_elements(const float* parts, const cgtp_attn_item& it, int head, int heads, int tile, int here,
                                              int width, int from, int n, int y, int ys, Put&& put) {
  const int64_t step = (int64_t)heads * tile * width;
  const float* p = parts + ((int64_t)it.first * heads + head) * tile * width + from;
  for (int e = y * 256 + threadIdx.x; e < here * n; e += ys * 256) {
    const int r = e / n, d = e % n;
    float s = 0.f;
#pragma unroll 4
    for (int k = 0; k < it.count; ++k) s += p[k * step + r * width + d];
    put(r, d, s);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) attn_bwd_q_join_kernel(AttnLaunch a, AttnScratch w, int tile) {
  __shared__ float sums[128][kQSums];
  const int group = a.h_q / a.h_kv, hk = blockIdx.x % a.h_kv, here_width = a.dim + kQSums;
  const cgtp_attn_item it = a.q_joins[blockIdx.x / a.h_kv];
  const int here = it.row_end - it.row_begin;
  if (a.grad_q)
    join_elements(w.parts, it, hk, a.h_kv, tile, here, here_width, 0, a.dim, blockIdx.y, gridDim.y, [&](int r, int d, float s) {
      const Row row = row_of(it, it.row_begin + r, hk, group);
      ((T*)a.grad_q)[((int64_t)row.query * a.h_q + row.head) * a.dim + d] = (T)s;
    });
  if (blockIdx.y) return;
  // one workgroup of a tile: the sums that end with a factor of the row
  join_elements(w.parts, it, hk, a.h_kv, tile, here, here_width, a.dim, kQSums, 0, 1, [&](int r, int d, float s) { sums[r][d] = s; });
  __syncthreads();
  if ((int)threadIdx.x >= here) return;
  const Row row = row_of(it, it.row_begin + threadIdx.x, hk, group);
  QSums m;
#pragma unroll
  for (int i = 0; i < kQSums; ++i) m.v[i] = sums[threadIdx.x][i];
  m.v[9] /= (float)it.count;            // delta: the same in every piece
  m.finish(w, (int64_t)row.query * a.h_q + row.head, a.slope ? a.slope[row.head] : 0.f, a.slope != nullptr);
}

// ---- gradient with the keys fixed ---------------------------------------------------------------------------------
// Bound by vector instructions; four sums of 32 x dim for a wavefront leave room for two of them on a SIMD up to dim 64.  The
// two workloads above: 111 and 549 us.  Taking two heads at a time, whose distances are the same, was within 5 % of
// this for short rows and slower for others (their sums spilled).
template <typename T, int DP, int NW, bool BIASED, bool CAPPED>
__global__ void __launch_bounds__(64 * NW, DP <= 64 ? 2 : 1)
attn_bwd_k_kernel(AttnLaunch a, AttnScratch w) {
  using S = AttnShape<T, DP>;
  constexpr int kBlock = kBlockOf<T, DP, NW>, kTile = kBlock * S::kRow, kBuf = kLean<T, DP, NW> ? 1 : kBuffers<2 * kTile>;
  constexpr bool LEAN = kLean<T, DP, NW>;
  __shared__ alignas(16) char tiles[kBuf][2][kTile];
  __shared__ alignas(16) float stat[2][6][kBlock];       // lse, delta, slope, position
  const int hk = blockIdx.x % a.h_kv, group = a.h_q / a.h_kv;
  const cgtp_attn_item it = a.k_items[blockIdx.x / a.h_kv];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const int key = it.k_begin + wave * 32 + (lane & 31);
  const bool ok = key < it.k_end;
  const Score<T, BIASED, CAPPED> sc(a);
  RowFrag<T, DP> k, v;
  k.load(ok ? (const T*)a.k + key * a.k_node + hk * a.k_head : nullptr, a.dim);
  v.load(ok ? (const T*)a.v + key * a.v_node + hk * a.v_head : nullptr, a.dim);
  float x = 0.f, y = 0.f, z = 0.f;
  if (BIASED && ok) {
    x = a.pos_k[(int64_t)key * 3];
    y = a.pos_k[(int64_t)key * 3 + 1];
    z = a.pos_k[(int64_t)key * 3 + 2];
  }
  AttnAcc<T, DP> gk, gv;
#pragma unroll
  for (int o = 0; o < S::kOut; ++o)
#pragma unroll
    for (int e = 0; e < 16; ++e) gk[o][e] = gv[o][e] = 0.f;
  float gx = 0.f, gy = 0.f, gz = 0.f;
  ColumnFit<T, DP> fit;
  TileStage<T, DP, 64 * NW, kBlock> qs, other;
  auto& gs = LEAN ? qs : other;
  float st[6] = {};
  auto fetch_g = [&](int r0) {
    const QueryRows<T> gr((const T*)a.grad_out, a.g_node, a.g_head, it.node, hk, group, r0, it.row_end - r0);
    gs.load(gr.base, a.dim, [&](int i) { return gr.offset(i); });
  };
  auto fetch = [&](int r0) {
    const QueryRows<T> qr((const T*)a.q, a.q_node, a.q_head, it.node, hk, group, r0, it.row_end - r0);
    qs.load(qr.base, a.dim, [&](int i) { return qr.offset_again(i); });
    if (!LEAN) fetch_g(r0);
    if (threadIdx.x < kBlock) {
      const Row o = row_of(it, r0 + threadIdx.x, hk, group);
      const int64_t at = (int64_t)o.query * a.h_q + o.head;
      st[0] = o.ok ? ((const float*)a.lse)[at] - kUp<T> : INFINITY;        // +inf: probability zero
      st[1] = o.ok ? w.delta[at] : 0.f;
      if constexpr (BIASED) {
        st[2] = o.ok ? a.slope[o.head] : 0.f;
#pragma unroll
        for (int d = 0; d < 3; ++d) st[3 + d] = o.ok ? a.pos_q[(int64_t)o.query * 3 + d] : 0.f;
      }
    }
  };
  if (it.row_begin < it.row_end) fetch(it.row_begin);
  int buf = 0;
  for (int r0 = it.row_begin; r0 < it.row_end; r0 += kBlock, buf ^= 1) {
    const int n = it.row_end - r0;
    char* const q_tile = tiles[kBuf == 2 ? buf : 0][0];
    char* const g_tile = tiles[kBuf == 2 ? buf : 0][1];
    if (kBuf == 1) __syncthreads();
    qs.store(q_tile);
    if (!LEAN) gs.store(g_tile);
    if (threadIdx.x < kBlock)
#pragma unroll
      for (int d = 0; d < 6; ++d) stat[buf][d][threadIdx.x] = st[d];
    __syncthreads();
    if (LEAN) fetch_g(r0);
    else if (r0 + kBlock < it.row_end) fetch(r0 + kBlock);
#pragma unroll 1
    for (int b = 0; b < kBlock / 32; ++b) {
      if (b * 32 >= n) continue;
      f32x16_t t = rows_times<T, DP>(q_tile, 32 * b, k);
      sc.of(t);
      if (LEAN) {
        gs.store(g_tile);
        __syncthreads();
        if (r0 + kBlock < it.row_end) fetch(r0 + kBlock);
      }
      f32x16_t ds = rows_times<T, DP>(g_tile, 32 * b, v);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int first = 32 * b + 8 * g + 4 * half;
        const f32x4 lse = *reinterpret_cast<const f32x4*>(&stat[buf][0][first]);
        const f32x4 delta = *reinterpret_cast<const f32x4*>(&stat[buf][1][first]);
        f32x4 slope = {}, px = {}, py = {}, pz = {};
        if constexpr (BIASED) {
          slope = *reinterpret_cast<const f32x4*>(&stat[buf][2][first]);
          px = *reinterpret_cast<const f32x4*>(&stat[buf][3][first]);
          py = *reinterpret_cast<const f32x4*>(&stat[buf][4][first]);
          pz = *reinterpret_cast<const f32x4*>(&stat[buf][5][first]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * g + e;
          float dx = 0.f, dy = 0.f, dz = 0.f, d2 = 0.f, inv = 0.f;
          if constexpr (BIASED) {
            dx = px[e] - x;
            dy = py[e] - y;
            dz = pz[e] - z;
            d2 = __builtin_amdgcn_fmed3f(dx * dx + dy * dy + dz * dz, kNear2, kFar2);
            inv = __builtin_amdgcn_rsqf(d2);
          }
          const float p = exp2_fast(sc.less(t[i], slope[e] * kLog2E, d2 * inv) - lse[e]);
          float d = p * (ds[i] - delta[e]);
          if constexpr (BIASED) {
            const float u = d * inv * slope[e];
            gx = fmaf(u, dx, gx);
            gy = fmaf(u, dy, gy);
            gz = fmaf(u, dz, gz);
          }
          if constexpr (CAPPED) d *= sc.through(t[i]);
          t[i] = p;
          ds[i] = d;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      fit.fit(ds, gk);
      cols_times<T, DP>(gv, g_tile, 32 * b, t);
      cols_times<T, DP>(gk, q_tile, 32 * b, ds);
    }
  }
  gx += half_swap(gx);
  gy += half_swap(gy);
  gz += half_swap(gz);
  if (!ok) return;
  const int64_t at = (int64_t)key * a.h_kv + hk;
  // p and ds were formed 2^kUp times as large
  constexpr float kDown = 1.f / (1 << kUp<T>);
  const float grad_scale = fit.undo(a.scale * kDown);
  if (it.slot < 0) {
    if (a.grad_k) store_cols<T, DP>((T*)a.grad_k + at * a.dim, gk, grad_scale, a.dim);
    if (a.grad_v) store_cols<T, DP>((T*)a.grad_v + at * a.dim, gv, kDown, a.dim);
    if (BIASED && half == 0) w.key_part[at] = f32x4{gx * kDown, gy * kDown, gz * kDown, 0.f};
  } else {
    float* p = w.parts + (((int64_t)it.slot * a.h_kv + hk) * kRowsOf<NW> + (key - it.k_begin)) * (2 * a.dim + 4);
    store_cols<float, (DP < 32 ? 32 : DP)>(p, gk, grad_scale, a.dim);
    store_cols<float, (DP < 32 ? 32 : DP)>(p + a.dim, gv, kDown, a.dim);
    if (half == 0) {
      p[2 * a.dim] = gx * kDown;
      p[2 * a.dim + 1] = gy * kDown;
      p[2 * a.dim + 2] = gz * kDown;
      p[2 * a.dim + 3] = 0.f;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) attn_bwd_k_join_kernel(cgtp_attn_args a, AttnScratch w, int tile) {
  const int hk = blockIdx.x % a.h_kv;
  const cgtp_attn_item it = a.k_joins[blockIdx.x / a.h_kv];
  join_elements(w.parts, it, hk, a.h_kv, tile, it.k_end - it.k_begin, 2 * a.dim + 4, 0, 2 * a.dim + 4, blockIdx.y, gridDim.y,
                [&](int key, int d, float s) {
    const int64_t at = (int64_t)(it.k_begin + key) * a.h_kv + hk;
    if (d < a.dim) {
      if (a.grad_k) ((T*)a.grad_k)[at * a.dim + d] = (T)s;
    } else if (d < 2 * a.dim) {
      if (a.grad_v) ((T*)a.grad_v)[at * a.dim + d - a.dim] = (T)s;
    } else if (a.slope) {
      ((float*)&w.key_part[at])[d - 2 * a.dim] = s;
    }
  });
}

// ---- launches -----------------------------------------------------------------------------------------------------
template <typename T, int DP, int NW, int KS, bool BIASED, bool CAPPED>
void q_launch(const AttnLaunch& a, const AttnScratch* w, hipStream_t s) {
  float* parts = (float*)a.workspace;
  const unsigned n = (unsigned)a.n_q_items * a.h_kv, joins = (unsigned)a.n_q_joins * a.h_kv;
  if (n) {
    const dim3 threads(64 * NW * KS);
    if (w) hipLaunchKernelGGL((attn_bwd_q_kernel<T, DP, NW, KS, BIASED, CAPPED>), dim3(n), threads, 0, s, a, *w);
    else hipLaunchKernelGGL((attn_fwd_kernel<T, DP, NW, KS, BIASED, CAPPED>), dim3(n), threads, 0, s, a, parts);
  }
  if (!joins) return;
  if (w) {
    hipLaunchKernelGGL((attn_bwd_q_join_kernel<T>), dim3(joins, 8), dim3(256), 0, s, a, *w, kRowsOf<NW>);
  } else if (a.n_q_slots > 16 * a.n_q_joins) {
    // a row's slots are shared out over a workgroup where they are many, else an element's slots are a thread's
    hipLaunchKernelGGL((attn_fwd_join_kernel<T>), dim3(joins * kRowsOf<NW>), dim3(kJoinThreads), 0, s, a, (const float*)parts,
                       kRowsOf<NW>);
  } else {
    hipLaunchKernelGGL((attn_fwd_join_few_kernel<T>), dim3(joins, 8), dim3(256), 0, s, a, (const float*)parts, kRowsOf<NW>);
  }
}
template <typename T, int DP, int NW, bool BIASED, bool CAPPED>
void k_launch(const AttnLaunch& a, const AttnScratch& w, hipStream_t s) {
  const unsigned n = (unsigned)a.n_k_items;
  const dim3 threads(64 * NW);
  if (n) {
    hipLaunchKernelGGL((attn_bwd_k_kernel<T, DP, NW, BIASED, CAPPED>), dim3(n * (unsigned)a.h_kv), threads, 0, s, a, w);
  }
  if (a.n_k_joins)
    hipLaunchKernelGGL((attn_bwd_k_join_kernel<T>), dim3((unsigned)a.n_k_joins * a.h_kv, 8), dim3(256), 0, s, a, w, kRowsOf<NW>);
}
template <typename T, int DP, bool BIASED, bool CAPPED>
void launch_dim(const AttnLaunch& a, const AttnScratch* w, hipStream_t s) {
  if (a.wide_q == 1) q_launch<T, DP, 4, 1, BIASED, CAPPED>(a, w, s);
  else if (a.wide_q == 2) q_launch<T, DP, 1, 4, BIASED, CAPPED>(a, w, s);
  else q_launch<T, DP, 1, 1, BIASED, CAPPED>(a, w, s);
  if (!w) return;
  if (a.wide_k) k_launch<T, DP, 4, BIASED, CAPPED>(a, *w, s);
  else k_launch<T, DP, 1, BIASED, CAPPED>(a, *w, s);
}

}  // namespace

template <typename T, bool BIASED, bool CAPPED>
void attn_launch(const AttnLaunch& a, const AttnScratch* w, hipStream_t s) {
  if (a.dim <= 16) launch_dim<T, 16, BIASED, CAPPED>(a, w, s);
  else if (a.dim <= 32) launch_dim<T, 32, BIASED, CAPPED>(a, w, s);
  else if (a.dim <= 64) launch_dim<T, 64, BIASED, CAPPED>(a, w, s);
  else if (a.dim <= 96) launch_dim<T, 96, BIASED, CAPPED>(a, w, s);
  else launch_dim<T, 128, BIASED, CAPPED>(a, w, s);
}

}  // namespace cgtp
