// Kernels of the attention with distances for dim <= 64 that take several heads at a time: the distance of a pair costs
// as many instructions as the rest of its score, and is the same for all heads.  A row is a query here, and a wavefront holds 32
// rows (or keys) of HEADS heads.  Vector instructions bound these kernels; counted in issue slots for a score (an
// exponential, reciprocal or root takes four), with a cap: forward 22, gradient of q 32, of k and v 32, where one head at a time
// takes 32, 48 and 41.  The scheduling barriers keep reads from LDS that would be needed later out of the registers.
//
// Rows are whole aligned chunks here (the launch refuses others).
//
// With a cap the score is taken without its constant part: t = -2 outer r - slope' |r_i - r_j|, r = 1 / (2^(inner q.k) + 1), which
// moves lse by as much; 1 - tanh^2 = 4 r (1 - r).
//
// In 16-bit types the output that the backward's delta is formed from has to be as good as fp32, for the gradients of
// positions and slopes are: the forward multiplies what rounding takes off the probabilities too, and leaves the output's
// own rounding error in out_low.
#pragma once

namespace cgtp {
namespace {

constexpr int kHeads = 2;      // four in the forward, dim <= 32: a wavefront for each SIMD instead of two, and 121 us where two take 74

// Scores of a block of 32 keys (or rows) from q.k, in binary orders.
template <bool CAPPED>
struct HeadScore {
  float linear, inner, outer2;
  __device__ __forceinline__ explicit HeadScore(const AttnLaunch& a) {
    linear = a.scale * kLog2E;
    inner = CAPPED ? 2.f * kLog2E * a.scale / a.cap : 0.f;
    outer2 = -2.f * a.cap * kLog2E;
  }
  // r: what a gradient needs of the cap.
  __device__ __forceinline__ float operator()(float qk, float slope, float dist, float& r) const {
    if constexpr (CAPPED) {
      r = __builtin_amdgcn_rcpf(exp2_fast(inner * qk) + 1.f);
      return fmaf(-slope, dist, outer2 * r);
    } else {
      return fmaf(-slope, dist, linear * qk);
    }
  }
};

// Distances of the lane's node from the 32 nodes of pos from `first` on, as a product of 32 x 32 lies.
__device__ __forceinline__ void distances(f32x16_t& dist, const float* pos, int stride, int first, float x, float y, float z) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int at = first + 8 * g + 4 * half;
    const f32x4 px = *reinterpret_cast<const f32x4*>(pos + at), py = *reinterpret_cast<const f32x4*>(pos + stride + at),
                pz = *reinterpret_cast<const f32x4*>(pos + 2 * stride + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float dx = x - px[e], dy = y - py[e], dz = z - pz[e];
      dist[4 * g + e] = __builtin_amdgcn_sqrtf(dx * dx + dy * dy + dz * dz);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}
// g += sum over the block of w (lane's node - node) / distance; a distance of zero gives nothing.
__device__ __forceinline__ void pull(float (&g)[3], const f32x16_t& w, const f32x16_t& dist, const float* pos, int stride, int first,
                                     float x, float y, float z) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int at = first + 8 * q + 4 * half;
    const f32x4 px = *reinterpret_cast<const f32x4*>(pos + at), py = *reinterpret_cast<const f32x4*>(pos + stride + at),
                pz = *reinterpret_cast<const f32x4*>(pos + 2 * stride + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float u = w[4 * q + e] * __builtin_amdgcn_rcpf(fmaxf(dist[4 * q + e], 1e-18f));
      g[0] = fmaf(u, x - px[e], g[0]);
      g[1] = fmaf(u, y - py[e], g[1]);
      g[2] = fmaf(u, z - pz[e], g[2]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

__device__ __forceinline__ bool beyond(int e, int first, int n) {
  return first + 8 * (e >> 2) + 4 * (int)((threadIdx.x & 63) >> 5) + (e & 3) >= n;
}

// Tiles of HEADS heads' keys and values (or queries and gradients) on their way to LDS: A from `a`, B from `b`, `tiles` of each.
template <typename T, int DP, int THREADS, int BLOCK, int HEADS>
struct HeadStage {
  TileStage<T, DP, THREADS, BLOCK> a[HEADS], b[HEADS];
  template <typename OfA, typename OfB>
  __device__ __forceinline__ void load(int dim, int tiles, OfA&& of_a, OfB&& of_b) {
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      if (j >= tiles) continue;
      const KeyRows<T> ra = of_a(j), rb = of_b(j);
      a[j].load_fast(ra.base, dim, [&](int i) { return ra.offset(i); });
      b[j].load_fast(rb.base, dim, [&](int i) { return rb.offset(i); });
    }
  }
  __device__ __forceinline__ void store(char* lds, int tiles) const {
    constexpr int kTile = BLOCK * AttnShape<T, DP>::kRow;
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      if (j >= tiles) continue;
      a[j].store(lds + 2 * j * kTile);
      b[j].store(lds + (2 * j + 1) * kTile);
    }
  }
};

// ---- forward ----------------------------------------------------------------------------------------------------
template <typename T, int DP, int NW, bool CAPPED>
__global__ void __launch_bounds__(64 * NW, 2) attn_heads_fwd_kernel(AttnLaunch a, float* __restrict__ parts) {
  using S = AttnShape<T, DP>;
  constexpr int HEADS = kHeads, kBlock = kBlockOf<NW>, kTile = kBlock * S::kRow, kBuf = kBuffers<2 * HEADS * kTile>;
  constexpr int kB = kBlock / 32;
  __shared__ alignas(16) char tiles[kBuf][2 * HEADS * kTile];
  __shared__ alignas(16) float pos[2][3][kBlock];
  const int groups = (a.h_q + HEADS - 1) / HEADS, h0 = blockIdx.x % groups * HEADS, group = a.h_q / a.h_kv;
  const cgtp_attn_item it = a.q_items[blockIdx.x / groups];
  const int here = min(HEADS, a.h_q - h0), hk0 = h0 / group;
  // Query heads of one head of keys among these: one, or all.
  const int per_log2 = min(group, HEADS) >> 1, n_tiles = (here + (1 << per_log2) - 1) >> per_log2;
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const int r = it.row_begin + wave * 32 + (lane & 31);
  const bool ok = r < it.row_end;
  const int64_t query = it.node + (ok ? r : it.row_begin);
  const HeadScore<CAPPED> score(a);
  RowFrag<T, DP> q[HEADS];
  AttnAcc<T, DP> acc[HEADS];
  float top[HEADS], sum[HEADS], slope[HEADS];
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    q[j].load_fast(ok && j < here ? (const T*)a.q + query * a.q_node + (h0 + j) * a.q_head : nullptr, a.dim);
    slope[j] = j < here ? a.slope[h0 + j] * kLog2E : 0.f;
    top[j] = -INFINITY;
    sum[j] = 0.f;
#pragma unroll
    for (int o = 0; o < S::kOut; ++o)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][o][e] = 0.f;
  }
  float x = 0.f, y = 0.f, z = 0.f;
  if (ok) {
    x = a.pos_q[query * 3];
    y = a.pos_q[query * 3 + 1];
    z = a.pos_q[query * 3 + 2];
  }
  HeadStage<T, DP, 64 * NW, kBlock, HEADS> stage;
  float ps[3] = {};
  auto fetch = [&](int k0) {
    const int n = it.k_end - k0;
    stage.load(a.dim, n_tiles, [&](int j) { return KeyRows<T>((const T*)a.k, a.k_node, a.k_head, hk0 + j, k0, n); },
               [&](int j) { return KeyRows<T>((const T*)a.v, a.v_node, a.v_head, hk0 + j, k0, n); });
    if (threadIdx.x < kBlock)
#pragma unroll
      for (int d = 0; d < 3; ++d) ps[d] = (int)threadIdx.x < n ? a.pos_k[(int64_t)(k0 + threadIdx.x) * 3 + d] : 0.f;
  };
  if (it.k_begin < it.k_end) fetch(it.k_begin);
  int buf = 0;
  for (int k0 = it.k_begin; k0 < it.k_end; k0 += kBlock, buf ^= 1) {
    const int n = it.k_end - k0;
    char* const tile = tiles[kBuf == 2 ? buf : 0];
    if (kBuf == 1) __syncthreads();
    stage.store(tile, n_tiles);
    if (threadIdx.x < kBlock)
#pragma unroll
      for (int d = 0; d < 3; ++d) pos[buf][d][threadIdx.x] = ps[d];
    __syncthreads();
    if (k0 + kBlock < it.k_end) fetch(k0 + kBlock);
    f32x16_t dist[kB];
#pragma unroll
    for (int b = 0; b < kB; ++b) distances(dist[b], pos[buf][0], kBlock, 32 * b, x, y, z);
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      if (j >= here) continue;
      const char* k_tile = tile + 2 * (j >> per_log2) * kTile;
      f32x16_t t[kB];
      float most = top[j];
#pragma unroll
      for (int b = 0; b < kB; ++b) {
        if (b * 32 >= n) continue;
        t[b] = rows_times<T, DP>(k_tile, 32 * b, q[j]);
        float r;
#pragma unroll
        for (int e = 0; e < 16; ++e) t[b][e] = score(t[b][e], slope[j], dist[b][e], r);
        if (n < 32 * b + 32)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (beyond(e, 32 * b, n)) t[b][e] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) most = fmaxf(most, t[b][e]);
      }
      most = fmaxf(most, half_swap(most));
      if (__any(most > top[j])) {
        const float by = top[j] == most ? 1.f : exp2_fast(top[j] - most);      // equal: also both -inf
        sum[j] *= by;
#pragma unroll
        for (int o = 0; o < S::kOut; ++o)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[j][o][e] *= by;
        top[j] = most;
      }
      const float base = top[j] == -INFINITY ? 0.f : top[j];
#pragma unroll
      for (int b = 0; b < kB; ++b) {
        if (b * 32 >= n) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          t[b][e] = exp2_fast(t[b][e] - base);
          sum[j] += t[b][e];
        }
        if (sizeof(T) == 2 && a.out_low) cols_times<T, DP, true>(acc[j], k_tile + kTile, 32 * b, t[b]);
        else cols_times<T, DP>(acc[j], k_tile + kTile, 32 * b, t[b]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const float total = sum[j] + half_swap(sum[j]);
    if (!ok || j >= here) continue;
    const int64_t at = query * a.h_q + h0 + j;
    if (it.slot < 0) {
      const bool some = total > 0.f || total != total;
      const float by = some ? 1.f / total : 0.f;
      store_cols_fast<T, DP>((T*)a.out + at * a.dim, acc[j], by, a.dim);
      if (sizeof(T) == 2 && a.out_low) {
#pragma unroll
        for (int o = 0; o < S::kOut; ++o)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[j][o][e] = acc[j][o][e] * by - (float)(T)(acc[j][o][e] * by);
        store_cols_fast<T, DP>((T*)a.out_low + at * a.dim, acc[j], 1.f, a.dim);
      }
      if (a.lse && half == 0) ((float*)a.lse)[at] = some ? top[j] + __log2f(total) : INFINITY;
    } else {
      float* p = parts + (((int64_t)it.slot * a.h_q + h0 + j) * kRowsOf<NW> + (r - it.row_begin)) * (a.dim + 2);
      store_cols<float, (DP < 32 ? 32 : DP)>(p, acc[j], 1.f, a.dim);
      if (half == 0) {
        p[a.dim] = top[j];
        p[a.dim + 1] = total;
      }
    }
  }
}

// ---- gradient with the rows fixed ---------------------------------------------------------------------------------
template <typename T, int DP, int NW, bool CAPPED>
__global__ void __launch_bounds__(64 * NW, 2) attn_heads_bwd_q_kernel(AttnLaunch a, AttnScratch w) {
  using S = AttnShape<T, DP>;
  constexpr int HEADS = kHeads, kBlock = kBlockOf<NW>, kTile = kBlock * S::kRow, kBuf = kBuffers<2 * HEADS * kTile>;
  __shared__ alignas(16) char tiles[kBuf][2 * HEADS * kTile];
  __shared__ alignas(16) float pos[2][3][kBlock];
  const int groups = (a.h_q + HEADS - 1) / HEADS, h0 = blockIdx.x % groups * HEADS, group = a.h_q / a.h_kv;
  const cgtp_attn_item it = a.q_items[blockIdx.x / groups];
  const int here = min(HEADS, a.h_q - h0), hk0 = h0 / group;
  // Query heads of one head of keys among these: one, or all.
  const int per_log2 = min(group, HEADS) >> 1, n_tiles = (here + (1 << per_log2) - 1) >> per_log2;
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const int r = it.row_begin + wave * 32 + (lane & 31);
  const bool ok = r < it.row_end;
  const int64_t query = it.node + (ok ? r : it.row_begin);
  const HeadScore<CAPPED> score(a);
  RowFrag<T, DP> q[HEADS], g[HEADS];
  AttnAcc<T, DP> acc[HEADS];
  float lse[HEADS], delta[HEADS], slope[HEADS], far[HEADS];      // far: sum of ds |r_i - r_j|
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const bool in = ok && j < here;
    const int64_t at = query * a.h_q + h0 + j;
    q[j].load_fast(in ? (const T*)a.q + query * a.q_node + (h0 + j) * a.q_head : nullptr, a.dim);
    g[j].load_fast(in ? (const T*)a.grad_out + at * a.dim : nullptr, a.dim);
    lse[j] = in ? ((const float*)a.lse)[at] : INFINITY;
    slope[j] = j < here ? a.slope[h0 + j] : 0.f;
    delta[j] = far[j] = 0.f;
#pragma unroll
    for (int part = 0; part < (sizeof(T) == 2 ? 2 : 1); ++part) {
      RowFrag<T, DP> o;
      o.load_fast(in ? (const T*)(part ? a.out_low : a.out) + at * a.dim : nullptr, a.dim);
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) {
        typedef T vec __attribute__((ext_vector_type(S::kChunk)));
        const vec go = __builtin_bit_cast(vec, g[j].f[s]), oo = __builtin_bit_cast(vec, o.f[s]);
#pragma unroll
        for (int e = 0; e < S::kChunk; ++e) delta[j] = fmaf((float)go[e], (float)oo[e], delta[j]);
      }
    }
    delta[j] += half_swap(delta[j]);
    if (in && half == 0 && it.first == 0) w.delta[at] = delta[j];
#pragma unroll
    for (int o = 0; o < S::kOut; ++o)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][o][e] = 0.f;
  }
  float x = 0.f, y = 0.f, z = 0.f, moved[3] = {};                // moved: sum of slope ds (r_i - r_j) / |r_i - r_j|
  if (ok) {
    x = a.pos_q[query * 3];
    y = a.pos_q[query * 3 + 1];
    z = a.pos_q[query * 3 + 2];
  }
  HeadStage<T, DP, 64 * NW, kBlock, HEADS> stage;
  float ps[3] = {};
  auto fetch = [&](int k0) {
    const int n = it.k_end - k0;
    stage.load(a.dim, n_tiles, [&](int j) { return KeyRows<T>((const T*)a.k, a.k_node, a.k_head, hk0 + j, k0, n); },
               [&](int j) { return KeyRows<T>((const T*)a.v, a.v_node, a.v_head, hk0 + j, k0, n); });
    if (threadIdx.x < kBlock)
#pragma unroll
      for (int d = 0; d < 3; ++d) ps[d] = (int)threadIdx.x < n ? a.pos_k[(int64_t)(k0 + threadIdx.x) * 3 + d] : 0.f;
  };
  if (it.k_begin < it.k_end) fetch(it.k_begin);
  int buf = 0;
  for (int k0 = it.k_begin; k0 < it.k_end; k0 += kBlock, buf ^= 1) {
    const int n = it.k_end - k0;
    char* const tile = tiles[kBuf == 2 ? buf : 0];
    if (kBuf == 1) __syncthreads();
    stage.store(tile, n_tiles);
    if (threadIdx.x < kBlock)
#pragma unroll
      for (int d = 0; d < 3; ++d) pos[buf][d][threadIdx.x] = ps[d];
    __syncthreads();
    if (k0 + kBlock < it.k_end) fetch(k0 + kBlock);
#pragma unroll 1
    for (int b = 0; b < kBlock / 32; ++b) {
      if (b * 32 >= n) continue;
      f32x16_t dist, weight;
      distances(dist, pos[buf][0], kBlock, 32 * b, x, y, z);
#pragma unroll
      for (int e = 0; e < 16; ++e) weight[e] = 0.f;
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        if (j >= here) continue;
        const char* k_tile = tile + 2 * (j >> per_log2) * kTile;
        f32x16_t t = rows_times<T, DP>(k_tile, 32 * b, q[j]);
        f32x16_t ds = rows_times<T, DP>(k_tile + kTile, 32 * b, g[j]);
        const float by = slope[j] * kLog2E;
        auto turn = [&](bool cut) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float c;
            const float s = score(t[e], by, dist[e], c);
            float p = exp2_fast(s - lse[j]);
            if (cut && beyond(e, 32 * b, n)) p = 0.f;
            float d = p * (ds[e] - delta[j]);
            far[j] = fmaf(d, dist[e], far[j]);
            weight[e] = fmaf(slope[j], d, weight[e]);
            if constexpr (CAPPED) d *= fmaf(-c, c, c);
            ds[e] = d;
          }
        };
        if (n < 32 * b + 32) turn(true);
        else turn(false);
        cols_times<T, DP>(acc[j], k_tile, 32 * b, ds);
        __builtin_amdgcn_sched_barrier(0);
      }
      pull(moved, weight, dist, pos[buf][0], kBlock, 32 * b, x, y, z);
    }
  }
#pragma unroll
  for (int d = 0; d < 3; ++d) moved[d] += half_swap(moved[d]);
  const float scale = CAPPED ? 4.f * a.scale : a.scale;
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    far[j] += half_swap(far[j]);
    if (!ok || j >= here) continue;
    const int64_t at = query * a.h_q + h0 + j;
    // the heads' common part of the position's gradient is the first head's
    const f32x4 part = j == 0 ? f32x4{-moved[0], -moved[1], -moved[2], -far[j]} : f32x4{0.f, 0.f, 0.f, -far[j]};
    if (it.slot < 0) {
      if (a.grad_q) store_cols_fast<T, DP>((T*)a.grad_q + at * a.dim, acc[j], scale, a.dim);
      if (half == 0) w.row_part[at] = part;
    } else {
      float* p = w.parts + (((int64_t)it.slot * a.h_q + h0 + j) * kRowsOf<NW> + (r - it.row_begin)) * (a.dim + kQSums);
      store_cols<float, (DP < 32 ? 32 : DP)>(p, acc[j], scale, a.dim);
      if (half == 0)
#pragma unroll
        for (int i = 0; i < kHeadSums; ++i) p[a.dim + i] = part[i];
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) attn_heads_bwd_q_join_kernel(AttnLaunch a, AttnScratch w, int tile) {
  const int h = blockIdx.x % a.h_q;
  const cgtp_attn_item it = a.q_joins[blockIdx.x / a.h_q];
  join_elements(w.parts, it, h, a.h_q, tile, it.row_end - it.row_begin, a.dim + kQSums, [&](int r, int d, float s) {
    const int64_t at = (int64_t)(it.node + it.row_begin + r) * a.h_q + h;
    if (d < a.dim) {
      if (a.grad_q) ((T*)a.grad_q)[at * a.dim + d] = (T)s;
    } else if (d < a.dim + kHeadSums) {
      ((float*)&w.row_part[at])[d - a.dim] = s;
    }
  });
}

// ---- gradient with the keys fixed ---------------------------------------------------------------------------------
// group 1: HEADS heads of keys.  Else one head of keys, whose query heads (an even number) come two at a time.
template <typename T, int DP, int NW, bool CAPPED, bool SHARED>
__global__ void __launch_bounds__(64 * NW, 2) attn_heads_bwd_k_kernel(AttnLaunch a, AttnScratch w) {
  using S = AttnShape<T, DP>;
  constexpr int HEADS = kHeads, SETS = SHARED ? 1 : HEADS;
  constexpr int kBlock = kBlockOf<NW>, kTile = kBlock * S::kRow, kBuf = kBuffers<2 * HEADS * kTile>;
  __shared__ alignas(16) char tiles[kBuf][2 * HEADS * kTile];
  __shared__ alignas(16) float stat[2][3 + 2 * HEADS][kBlock];       // position, then lse and delta of each head
  const int groups = (a.h_kv + SETS - 1) / SETS, hk0 = blockIdx.x % groups * SETS, group = a.h_q / a.h_kv;
  const cgtp_attn_item it = a.k_items[blockIdx.x / groups];
  const int sets = min(SETS, a.h_kv - hk0), here = SHARED ? HEADS : sets, rounds = SHARED ? group / HEADS : 1;
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const int key = it.k_begin + wave * 32 + (lane & 31);
  const bool ok = key < it.k_end;
  const HeadScore<CAPPED> score(a);
  RowFrag<T, DP> k[SETS], v[SETS];
  AttnAcc<T, DP> gk[SETS], gv[SETS];
#pragma unroll
  for (int j = 0; j < SETS; ++j) {
    const bool in = ok && j < sets;
    k[j].load_fast(in ? (const T*)a.k + key * a.k_node + (hk0 + j) * a.k_head : nullptr, a.dim);
    v[j].load_fast(in ? (const T*)a.v + key * a.v_node + (hk0 + j) * a.v_head : nullptr, a.dim);
#pragma unroll
    for (int o = 0; o < S::kOut; ++o)
#pragma unroll
      for (int e = 0; e < 16; ++e) gk[j][o][e] = gv[j][o][e] = 0.f;
  }
  float x = 0.f, y = 0.f, z = 0.f, moved[3] = {};
  if (ok) {
    x = a.pos_k[(int64_t)key * 3];
    y = a.pos_k[(int64_t)key * 3 + 1];
    z = a.pos_k[(int64_t)key * 3 + 2];
  }
  HeadStage<T, DP, 64 * NW, kBlock, HEADS> stage;
  float st[3 + 2 * HEADS] = {};
  // Step i: block of rows i / rounds, heads of round i % rounds.
  auto first_head = [&](int i) { return SHARED ? hk0 * group + i % rounds * HEADS : hk0; };
  auto fetch = [&](int i) {
    const int r0 = it.row_begin + i / rounds * kBlock, n = it.row_end - r0, h0 = first_head(i), q0 = it.node + r0;
    stage.load(a.dim, here, [&](int j) { return KeyRows<T>((const T*)a.q, a.q_node, a.q_head, h0 + j, q0, n); },
               [&](int j) { return KeyRows<T>((const T*)a.grad_out, (int64_t)a.h_q * a.dim, a.dim, h0 + j, q0, n); });
    if (threadIdx.x < kBlock) {
      const bool in = (int)threadIdx.x < n;
      const int64_t query = q0 + (in ? threadIdx.x : 0);
#pragma unroll
      for (int d = 0; d < 3; ++d) st[d] = in ? a.pos_q[query * 3 + d] : 0.f;
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        const bool there = in && j < here;
        st[3 + 2 * j] = there ? ((const float*)a.lse)[query * a.h_q + h0 + j] : INFINITY;       // +inf: probability zero
        st[4 + 2 * j] = there ? w.delta[query * a.h_q + h0 + j] : 0.f;
      }
    }
  };
  const int steps = (it.row_end - it.row_begin + kBlock - 1) / kBlock * rounds;
  if (steps > 0) fetch(0);
  int buf = 0;
  for (int i = 0; i < steps; ++i, buf ^= 1) {
    const int n = it.row_end - (it.row_begin + i / rounds * kBlock), h0 = first_head(i);
    char* const tile = tiles[kBuf == 2 ? buf : 0];
    if (kBuf == 1) __syncthreads();
    stage.store(tile, here);
    if (threadIdx.x < kBlock)
#pragma unroll
      for (int d = 0; d < 3 + 2 * HEADS; ++d) stat[buf][d][threadIdx.x] = st[d];
    __syncthreads();
    if (i + 1 < steps) fetch(i + 1);
#pragma unroll 1
    for (int b = 0; b < kBlock / 32; ++b) {
      if (b * 32 >= n) continue;
      f32x16_t dist, weight;
      distances(dist, stat[buf][0], kBlock, 32 * b, x, y, z);
#pragma unroll
      for (int e = 0; e < 16; ++e) weight[e] = 0.f;
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        if (j >= here) continue;
        const char* q_tile = tile + 2 * j * kTile;
        const float slope = a.slope[h0 + j], by = slope * kLog2E;
        f32x16_t t = rows_times<T, DP>(q_tile, 32 * b, k[SHARED ? 0 : j]);
        f32x16_t ds = rows_times<T, DP>(q_tile + kTile, 32 * b, v[SHARED ? 0 : j]);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int first = 32 * b + 8 * g + 4 * half;
          const f32x4 lse = *reinterpret_cast<const f32x4*>(&stat[buf][3 + 2 * j][first]);
          const f32x4 delta = *reinterpret_cast<const f32x4*>(&stat[buf][4 + 2 * j][first]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float c;
            const float s = score(t[4 * g + e], by, dist[4 * g + e], c);
            const float p = exp2_fast(s - lse[e]);
            float d = p * (ds[4 * g + e] - delta[e]);
            weight[4 * g + e] = fmaf(slope, d, weight[4 * g + e]);
            if constexpr (CAPPED) d *= fmaf(-c, c, c);
            t[4 * g + e] = p;
            ds[4 * g + e] = d;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        cols_times<T, DP>(gv[SHARED ? 0 : j], q_tile + kTile, 32 * b, t);
        cols_times<T, DP>(gk[SHARED ? 0 : j], q_tile, 32 * b, ds);
        __builtin_amdgcn_sched_barrier(0);
      }
      // of the key: the opposite of the rows' part, for (key - row) is the opposite of (row - key)
      pull(moved, weight, dist, stat[buf][0], kBlock, 32 * b, x, y, z);
    }
  }
#pragma unroll
  for (int d = 0; d < 3; ++d) moved[d] += half_swap(moved[d]);
  if (!ok) return;
  const float scale = CAPPED ? 4.f * a.scale : a.scale;
#pragma unroll
  for (int j = 0; j < SETS; ++j) {
    if (j >= sets) continue;
    const int64_t at = (int64_t)key * a.h_kv + hk0 + j;
    const f32x4 part = j == 0 ? f32x4{-moved[0], -moved[1], -moved[2], 0.f} : f32x4{0.f, 0.f, 0.f, 0.f};
    if (it.slot < 0) {
      if (a.grad_k) store_cols_fast<T, DP>((T*)a.grad_k + at * a.dim, gk[j], scale, a.dim);
      if (a.grad_v) store_cols_fast<T, DP>((T*)a.grad_v + at * a.dim, gv[j], 1.f, a.dim);
      if (half == 0) w.key_part[at] = part;
    } else {
      float* p = w.parts + (((int64_t)it.slot * a.h_kv + hk0 + j) * kRowsOf<NW> + (key - it.k_begin)) * (2 * a.dim + 4);
      store_cols<float, (DP < 32 ? 32 : DP)>(p, gk[j], scale, a.dim);
      store_cols<float, (DP < 32 ? 32 : DP)>(p + a.dim, gv[j], 1.f, a.dim);
      if (half == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[2 * a.dim + i] = part[i];
    }
  }
}

}  // namespace
}  // namespace cgtp
