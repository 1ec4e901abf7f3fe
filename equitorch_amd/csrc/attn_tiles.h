// Tiles of the attention kernels in LDS and the matrix instructions over them.
//
// Every product has the form D = A B with 32 x 32 results: a lane holds column lane % 32 and, at index 4 g + e, row
// 8 g + 4 (lane / 32) + e.  A result can be the B operand of the next product as it lies in the registers: its rows become k,
// eight (16-bit) or one (fp32) of a lane's rows for each instruction, and A's k are taken in the same order.
//
// A tile of kBlock rows (nodes) is kept row by row, chunks of 16 bytes, chunk c of row r at a place that puts the eight rows a
// quarter wavefront reads into different groups of banks; for 16-bit types also column by column (RowsT), where the
// rows become k: a chunk there holds the eight rows of one lane and instruction.  fp32 needs no such copy: an
// instruction takes one row for each half of the wavefront, 32 neighbouring columns of it.
#pragma once

#include "elem.h"

namespace cgtp {



constexpr int kBlock = 64;                      // rows of a tile in LDS

template <typename T, int DP>
struct AttnShape {
  static constexpr int kChunk = 16 / (int)sizeof(T);          // elements of a chunk
  static constexpr int kChunks = DP / kChunk;                 // chunks of a row
  static constexpr int kSteps = kChunks / 2;                  // pairs of chunks: one per half wavefront
  static constexpr int kOut = (DP + 31) / 32;                 // 32-wide blocks of dim in a result
  static constexpr bool kTransposed = sizeof(T) == 2;
  static constexpr int kRowsBytes = kBlock * DP * (int)sizeof(T);
  static constexpr int kColsBytes = kTransposed ? kOut * 32 * kBlock * 2 : 0;
  __device__ static __forceinline__ int slot(int row, int c) {
    constexpr int kMix = kChunks % 8 == 0 ? 8 : kChunks % 4 == 0 ? 4 : 2;      // chunks that change places
    constexpr int kPer = kMix == 8 ? 1 : kMix == 4 ? 2 : 4;                    // rows before the pattern moves on
    return (row * kChunks + (c ^ ((row / kPer) & (kMix - 1)))) << 4;
  }
};

template <typename T>
__device__ __forceinline__ f32x16_t mma_pair(const u32x4_t& a, const u32x4_t& b, f32x16_t acc) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[j], fb[j], acc, 0, 0, 0);
  } else if constexpr (__is_same(T, f16_t)) {
    typedef f16_t v8 __attribute__((ext_vector_type(8)));
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), acc, 0, 0, 0);
  } else {
    typedef bf16_t v8 __attribute__((ext_vector_type(8)));
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), acc, 0, 0, 0);
  }
  return acc;
}

template <typename T, int DP> using AttnAcc = f32x16_t[AttnShape<T, DP>::kOut];

// A lane's part of one row as the B operand: chunk 2 s + lane / 32 at step s.  p null: zeros.
template <typename T, int DP>
struct RowFrag {
  u32x4_t f[AttnShape<T, DP>::kSteps];
  __device__ __forceinline__ void load(const T* p, int dim) {
    using S = AttnShape<T, DP>;
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      const int d = (2 * s + half) * S::kChunk;
      f[s] = u32x4_t{0, 0, 0, 0};
      if (p && d < dim) f[s] = load_part<u32x4_t, T>(p + d, dim - d);
    }
  }
};

// Rows row(0) .. row(kBlock - 1) (null: zeros) to LDS, row by row.
template <typename T, int DP, int THREADS, typename Row>
__device__ __forceinline__ void stage_rows(char* lds, int dim, Row&& row) {
  using S = AttnShape<T, DP>;
#pragma unroll
  for (int i = 0; i < (kBlock * S::kChunks + THREADS - 1) / THREADS; ++i) {
    const int id = i * THREADS + threadIdx.x, r = id / S::kChunks, c = id % S::kChunks;
    if (kBlock * S::kChunks % THREADS != 0 && id >= kBlock * S::kChunks) break;
    const T* p = row(r);
    u32x4_t v = {0, 0, 0, 0};
    if (p && c * S::kChunk < dim) v = load_part<u32x4_t, T>(p + c * S::kChunk, dim - c * S::kChunk);
    *reinterpret_cast<u32x4_t*>(lds + S::slot(r, c)) = v;
  }
}
// The same column by column (16-bit types): chunk c of column d holds rows 16 (c / 2) + 4 (c % 2) + {0 .. 3, 8 .. 11}.
template <typename T, int DP, int THREADS, typename Row>
__device__ __forceinline__ void stage_cols(char* lds, int dim, Row&& row) {
  using S = AttnShape<T, DP>;
  constexpr int kQuads = S::kOut * 8;           // groups of four columns
  constexpr int kTasks = kQuads * 8;
#pragma unroll
  for (int i = 0; i < (kTasks + THREADS - 1) / THREADS; ++i) {
    const int id = i * THREADS + threadIdx.x;
    if (kTasks % THREADS != 0 && id >= kTasks) break;
    const int c = id & 7, d = (id >> 3) * 4;
    u32x2_t t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const T* p = row(16 * (c >> 1) + 4 * (c & 1) + (j & 3) + 8 * (j >> 2));
      t[j] = u32x2_t{0, 0};
      if (p && d < dim) t[j] = load_part<u32x2_t, T>(p + d, dim - d);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x4_t v;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        v[w] = __builtin_amdgcn_perm(t[2 * w + 1][j >> 1], t[2 * w][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
      *reinterpret_cast<u32x4_t*>(lds + (d + j) * 128 + ((c ^ ((d + j) & 7)) << 4)) = v;
    }
  }
}

// D = rows of the tile (32 from `first` on) times the lanes' rows: 32 x 32 products over dim.
template <typename T, int DP>
__device__ __forceinline__ f32x16_t rows_times(const char* lds, int first, const RowFrag<T, DP>& b) {
  using S = AttnShape<T, DP>;
  const int lane = threadIdx.x & 63, r = first + (lane & 31), half = lane >> 5;
  f32x16_t acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s)
    acc = mma_pair<T>(*reinterpret_cast<const u32x4_t*>(lds + S::slot(r, 2 * s + half)), b.f[s], acc);
  return acc;
}

// acc[o] += columns 32 o .. of the 32 rows from `first` on, transposed, times p (rows by lanes' columns).  `rows` and `cols`
// are the two copies of the tile; only the one the type needs is read.
template <typename T, int DP>
__device__ __forceinline__ void cols_times(AttnAcc<T, DP>& acc, const char* rows, const char* cols, int first,
                                           const f32x16_t& p) {
  using S = AttnShape<T, DP>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  if constexpr (S::kTransposed) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      typedef T v8 __attribute__((ext_vector_type(8)));
      v8 b;
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = (T)p[8 * t + j];
      const int c = (first >> 3) + 2 * t + half;
#pragma unroll
      for (int o = 0; o < S::kOut; ++o) {
        const int d = 32 * o + (lane & 31);
        acc[o] = mma_pair<T>(*reinterpret_cast<const u32x4_t*>(cols + d * 128 + ((c ^ (d & 7)) << 4)),
                             __builtin_bit_cast(u32x4_t, b), acc[o]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int r = first + 8 * (e >> 2) + 4 * half + (e & 3);
#pragma unroll
      for (int o = 0; o < S::kOut; ++o) {
        const int d = 32 * o + (lane & 31);
        const bool in = DP % 32 == 0 || d < DP;
        const float v = *reinterpret_cast<const float*>(rows + S::slot(r, (in ? d : 0) >> 2) + ((d & 3) << 2));
        acc[o] = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? v : 0.f, p[e], acc[o], 0, 0, 0);
      }
    }
  }
}

// Results of a lane's column: its elements 32 o + 8 g + 4 (lane / 32) + e of dim, times `by`, to p.
template <typename T, int DP>
__device__ __forceinline__ void store_cols(T* p, const AttnAcc<T, DP>& acc, float by, int dim) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int o = 0; o < AttnShape<T, DP>::kOut; ++o)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * o + 8 * g + 4 * half;
      if (d >= dim) continue;
      T v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)(acc[o][4 * g + e] * by);
      store_part<T, 4>(p + d, v, dim - d);
    }
}

}  // namespace cgtp
