// The gradient with the keys fixed for the attention with distances, dim <= 64, two heads at a time: the distance of a pair and
// what its gradient takes cost as many instructions as the rest of a score, and are the same for all heads.  A row is a query
// here, and a wavefront holds 32 keys of two heads, or of one head of keys with two of its query heads.  Vector instructions
// bound it (an exponential, reciprocal or root takes four issue slots): 300 structures of 40 to 250 nodes, 8 heads of 32, bf16:
// 118 us one head at a time, 102 so, three of 2000 to 5000, 8 query heads on 4 of 64: 618 and 510.  With the
// rows fixed the same saves nothing: two heads' queries, gradients and results leave too few
// registers for two wavefronts on a SIMD.
//
// The scheduling barriers keep reads from LDS that are needed later out of the registers.  Rows are whole aligned chunks
// (the launch refuses others).
#pragma once

namespace cgtp {
namespace {

constexpr int kHeads = 2;

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

// Tiles of HEADS heads' queries and gradients of the output on their way to LDS, `tiles` of each.
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
  const Score<T, true, CAPPED> score(a);
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
        score.of(t);
        f32x16_t ds = rows_times<T, DP>(q_tile + kTile, 32 * b, v[SHARED ? 0 : j]);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int first = 32 * b + 8 * g + 4 * half;
          const f32x4 lse = *reinterpret_cast<const f32x4*>(&stat[buf][3 + 2 * j][first]);
          const f32x4 delta = *reinterpret_cast<const f32x4*>(&stat[buf][4 + 2 * j][first]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = exp2_fast(score.less(t[4 * g + e], by, dist[4 * g + e]) - lse[e]);
            float d = p * (ds[4 * g + e] - delta[e]);
            weight[4 * g + e] = fmaf(slope, d, weight[4 * g + e]);
            if constexpr (CAPPED) d *= score.through(t[4 * g + e]);
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
  const float scale = a.scale;
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
