// Tiles of the attention kernels in LDS and the matrix instructions over them.
//
// Every product has the form D = A B with 32 x 32 results: a lane holds column lane % 32 and, at index 4 g + e, row
// 8 g + 4 (lane / 32) + e.  A result can be the B operand of the next product as it lies in the registers: its rows become k,
// eight (16-bit) or one (fp32) of a lane's rows for each instruction, and A's k are taken in the same order.
//
// A tile of 64 or 32 rows (nodes) lies in LDS row by row in chunks of 16 bytes, chunk c of row r at a place that puts the eight
// rows a quarter wavefront reads into different groups of banks.  Where the rows become k, 16-bit types read it through
// the LDS's transposing loads (four rows of 16 columns for each 16 lanes) and fp32 as it is, one row for each half of the
// wavefront: no second, transposed copy.
//
// A tile goes from memory through registers to LDS: loaded while the tile before it is worked on, stored after.  The loads are
// buffer loads with 32-bit offsets, whose range check turns what is beyond the structure into zeros.
#pragma once

#include "elem.h"

namespace cgtp {

constexpr unsigned kNoRow = 0x80000000u;        // an offset beyond every buffer

template <typename T, int DP>
struct AttnShape {
  static constexpr int kChunk = 16 / (int)sizeof(T);          // elements of a chunk
  static constexpr int kChunks = DP / kChunk;                 // chunks of a row
  static constexpr int kSteps = kChunks / 2;                  // pairs of chunks: one per half wavefront
  static constexpr int kOut = (DP + 31) / 32;                 // 32-wide blocks of dim in a result
  static constexpr int kRow = DP * (int)sizeof(T);            // bytes
  // Chunks that change places, and rows before the pattern moves on.  16-bit rows of 256 bytes all start at the same bank: four
  // neighbouring rows, read transposed at four neighbouring chunks, have to go to four groups of chunks (conflicts 37 -> 0 % of
  // the cycles, one structure of 12007 nodes, 16 query heads on 4 of 128, fp16, 1612 -> 1531 us; shorter rows gain nothing).
  static constexpr int kMix = sizeof(T) == 2 && kChunks % 16 == 0 ? 16 : kChunks % 8 == 0 ? 8 : kChunks % 4 == 0 ? 4 : 2;
  static constexpr int kPer = kMix >= 8 ? 1 : kMix == 4 ? 2 : 4;
  __device__ static __forceinline__ int mixed(int row, int c) {
    const int m = (row / kPer) & (kMix - 1);
    return c ^ (kMix == 16 ? (m & 3) << 2 | m >> 2 : m);
  }
  __device__ static __forceinline__ int slot(int row, int c) { return (row * kChunks + mixed(row, c)) << 4; }
};

template <typename T, int DP> using AttnAcc = f32x16_t[AttnShape<T, DP>::kOut];

// A lane's part of one row as the B operand: chunk 2 s + lane / 32 at step s.  p null: zeros.
template <typename T, int DP>
struct RowFrag {
  u32x4_t f[AttnShape<T, DP>::kSteps];
  template <bool WHOLE = true>      // 16 bytes at a time, aligned
  __device__ __forceinline__ void load(const T* p, int dim) {
    using S = AttnShape<T, DP>;
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      const int d = (2 * s + half) * S::kChunk;
      f[s] = u32x4_t{0, 0, 0, 0};
      if (p && d < dim) f[s] = WHOLE ? *reinterpret_cast<const u32x4_t*>(p + d) : load_part<u32x4_t, T>(p + d, dim - d);
    }
  }
};

// A tile between memory and LDS, moved by THREADS neighbouring threads.  Offset(i): bytes from `base` of row i, kNoRow for none.
template <typename T, int DP, int THREADS, int BLOCK>
struct TileStage {
  using S = AttnShape<T, DP>;
  static constexpr int kAll = BLOCK * S::kChunks, kEach = (kAll + THREADS - 1) / THREADS;
  u32x4_t reg[kEach];

  template <typename Offset>
  __device__ __forceinline__ void load(const T* base, int dim, Offset&& offset) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, kNoRow, 0x00027000);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int id = i * THREADS + (int)threadIdx.x % THREADS, r = id / S::kChunks, c = S::mixed(r, id % S::kChunks);
      if (kAll % THREADS != 0 && id >= kAll) break;
      const unsigned o = offset(r);
      reg[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
          rsrc, o == kNoRow || c * S::kChunk >= dim ? kNoRow : o + c * 16, 0, 0));
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int id = i * THREADS + (int)threadIdx.x % THREADS;
      if (kAll % THREADS != 0 && id >= kAll) break;
      *reinterpret_cast<u32x4_t*>(lds + id * 16) = reg[i];
    }
  }
};

// D = rows of the tile (32 from `first` on) times the lanes' rows: 32 x 32 products over dim.
template <typename T, int DP>
__device__ __forceinline__ f32x16_t rows_times(const char* lds, int first, const RowFrag<T, DP>& b) {
  using S = AttnShape<T, DP>;
  const int lane = threadIdx.x & 63, r = first + (lane & 31), half = lane >> 5;
  f32x16_t acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    acc = mma_pair<T>(*reinterpret_cast<const u32x4_t*>(lds + S::slot(r, 2 * s + half)), b.f[s], acc);
    if (sizeof(T) == 4 && s % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // not all of a row's reads at once in registers
  }
  return acc;
}

// Four rows of 16 columns, transposed: lane i of 16 reads four columns from 4 (i % 4) on of row i / 4, and gets column i.
__device__ __forceinline__ u32x2_t lds_transposed(const char* p) {
  typedef short v4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4 lds_v4;
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)p));
}

// acc[o] += columns 32 o .. of the tile's 32 rows from `first` on, transposed, times p (rows by lanes' columns).
template <typename T, int DP>
__device__ __forceinline__ void cols_times(AttnAcc<T, DP>& acc, const char* lds, int first, const f32x16_t& p) {
  using S = AttnShape<T, DP>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int r = first + 4 * half + ((lane & 15) >> 2), d = (lane & 16) + 4 * (lane & 3);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      typedef T v8 __attribute__((ext_vector_type(8)));
      v8 b;
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = (T)p[8 * t + j];
#pragma unroll
      for (int o = 0; o < S::kOut; ++o) {
        // DP = 16: the columns 16 .. 31 of the result do not exist; its lanes read the others again
        const int col = DP < 32 ? d & 15 : 32 * o + d;
        const u32x2_t x = lds_transposed(lds + S::slot(r + 16 * t, col >> 3) + (col & 7) * 2);
        const u32x2_t y = lds_transposed(lds + S::slot(r + 16 * t + 8, col >> 3) + (col & 7) * 2);
        acc[o] = mma_pair<T>(u32x4_t{x[0], x[1], y[0], y[1]}, __builtin_bit_cast(u32x4_t, b), acc[o]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int r = first + 8 * (e >> 2) + 4 * half + (e & 3);
#pragma unroll
      for (int o = 0; o < S::kOut; ++o) {
        const int d = DP < 32 ? lane & 15 : 32 * o + (lane & 31);
        const float v = *reinterpret_cast<const float*>(lds + S::slot(r, d >> 2) + ((d & 3) << 2));
        acc[o] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[e], acc[o], 0, 0, 0);
      }
      if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// fp16 operands.  Its normal numbers end at 2^-14 and 65504, and a probability is 1 / keys, a score's gradient as much of the incoming
// gradient, whatever that was scaled by.  So probabilities are 2^kUp times as large where they enter a product, and the
// gradients of a column's scores `by` times, a power of two that falls as larger ones come, along with the sum so far.  6000 keys
// and a gradient of 1e-3: dq and dk err 4e-4 of their norm in place of 8e-3.  It costs 5 to 15 % of a step (three structures of
// 2000 to 5000 nodes, 8 query heads on 4 of 64, fp16: 1330 us without it, 1400 so); the sum is multiplied every time, as a branch
// about it takes the gradient of keys and values 80 registers.  bf16 has fp32's range.
template <typename T> constexpr int kUp = __is_same(T, f16_t) ? 10 : 0;
template <typename T, int DP>
struct ColumnFit {
  static constexpr bool kOn = __is_same(T, f16_t);
  float by = kOn ? 0x1p100f : 1.f;
  // acc: the column's sum of such products so far.
  __device__ __forceinline__ void fit(f32x16_t& d, AttnAcc<T, DP>& acc) {
    if constexpr (kOn) {
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(d[e]));
      most = fmaxf(most, __shfl_xor(most, 32, kWave));
      // an infinity has the exponent 0, and no factor becomes larger
      const float now = most * by > 0x1p15f ? fminf(by, ldexpf(1.f, 13 - __builtin_amdgcn_frexp_expf(most))) : by;
      scale(acc, now * inverse(by));
      by = now;
#pragma unroll
      for (int e = 0; e < 16; ++e) d[e] *= by;
    }
  }
  __device__ __forceinline__ float undo(float x) const { return kOn ? x * inverse(by) : x; }
  __device__ __forceinline__ void settle(AttnAcc<T, DP>& acc) {
    if constexpr (kOn) {
      scale(acc, inverse(by));
      by = 1.f;
    }
  }

 private:
  __device__ static __forceinline__ float inverse(float power) { return ldexpf(1.f, 1 - __builtin_amdgcn_frexp_expf(power)); }
  __device__ static __forceinline__ void scale(AttnAcc<T, DP>& acc, float f) {
#pragma unroll
    for (int o = 0; o < AttnShape<T, DP>::kOut; ++o)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[o][e] *= f;
  }
};

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
