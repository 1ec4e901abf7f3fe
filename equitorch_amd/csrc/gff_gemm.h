// Matrix products of the gated feed-forward block on the matrix cores: tiles of 128 x 128, four wavefronts of 64 x 64 each,
// operands staged through registers into two LDS buffers.
//
// An operand is a matrix whose rows or whose columns are contiguous.  In LDS both look alike: per row of the tile eight chunks of
// 16 bytes along k, chunk c of row r at place c ^ (r & 7), so that the eight rows a quarter wavefront reads lie in eight
// different groups of banks.  An operand contiguous along its rows is transposed on the way in registers: a thread takes
// a chunk's worth of k for four neighbouring rows.
//
// 16-bit operands use 32 x 32 x 16 instructions; fp32 operands 32 x 32 x 2 ones, four per pair of chunks, whose k
// are taken in the order that lets a lane read its four in one access.
#pragma once

#include "elem.h"

namespace cgtp {



constexpr int kGemmTile = 128, kGemmThreads = 256, kGemmChunks = 8;
constexpr int kGemmTileBytes = kGemmTile * kGemmChunks * 16;

template <typename T> struct GemmType { static constexpr int kChunk = 16 / (int)sizeof(T), kDepth = kGemmChunks * kChunk; };

template <typename T>
__device__ __forceinline__ void mma_chunk(f32x16_t& acc, const u32x4_t& a, const u32x4_t& b) {
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
}

// One operand's tile in registers between memory and LDS.
template <typename T, bool K_CONTIGUOUS>
struct GemmStage {
  static constexpr int CH = GemmType<T>::kChunk;
  u32x4_t reg[4];

  // Where row r of the tile is: row(r) gives its pointer at k = 0 (K_CONTIGUOUS) or at (0, r), or null outside the matrix.
  // k0: first k of the tile; depth: end of k; ld: elements between rows of memory; end: number of columns of memory from
  // the pointer's own on that belong to this operand (row-contiguous only).
  template <typename Row>
  __device__ __forceinline__ void load(Row&& row, int64_t k0, int64_t depth, int64_t ld) {
    const int tid = threadIdx.x;
    if constexpr (K_CONTIGUOUS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int id = i * kGemmThreads + tid, r = id >> 3, c = id & 7;
        int64_t end;
        const T* p = row(r, end);
        const int64_t k = k0 + c * CH;
        reg[i] = u32x4_t{0, 0, 0, 0};
        if (p && k < depth) reg[i] = load_part<u32x4_t, T>(p + k, depth - k);
      }
    } else {
      const int c = tid & 7, r = (tid >> 3) * 4;
      int64_t end;
      const T* p = row(r, end);
      const int64_t k = k0 + c * CH;
      if constexpr (sizeof(T) == 4) {
        u32x4_t t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          t[i] = u32x4_t{0, 0, 0, 0};
          if (p && k + i < depth) t[i] = load_part<u32x4_t, T>(p + (k + i) * ld, end);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) reg[i] = u32x4_t{t[0][i], t[1][i], t[2][i], t[3][i]};
      } else {
        u32x2_t t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          t[i] = u32x2_t{0, 0};
          if (p && k + i < depth) t[i] = load_part<u32x2_t, T>(p + (k + i) * ld, end);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < 4; ++d)
            reg[i][d] = __builtin_amdgcn_perm(t[2 * d + 1][i >> 1], t[2 * d][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = K_CONTIGUOUS ? (i * kGemmThreads + tid) >> 3 : (tid >> 3) * 4 + i, c = tid & 7;
      *reinterpret_cast<u32x4_t*>(lds + r * 128 + ((c ^ (r & 7)) << 4)) = reg[i];
    }
  }
};

// acc[i][j] of wavefront (wm, wn): rows 64 wm + 32 i of the first operand, 64 wn + 32 j of the second.  A lane holds row lane % 32
// of the first and, at index 4 g + e, row 8 g + 4 (lane / 32) + e of the second: four neighbours for one store.
// first / second(k tile) load the next tile into their stage; tiles: number of k tiles, the same for all threads.
template <typename T, bool KA, bool KB, typename LoadA, typename LoadB>
__device__ __forceinline__ void gemm_loop(f32x16_t (&acc)[2][2], char* lds, int64_t tiles, LoadA&& load_a, LoadB&& load_b) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  if (tiles <= 0) return;
  GemmStage<T, KA> a;
  GemmStage<T, KB> b;
  load_a(a, (int64_t)0);
  load_b(b, (int64_t)0);
  const int ra = wm * 64 + (lane & 31), rb = wn * 64 + (lane & 31), half = lane >> 5, sw = lane & 7;
  for (int64_t t = 0; t < tiles; ++t) {
    char* la = lds + (t & 1) * 2 * kGemmTileBytes;
    char* lb = la + kGemmTileBytes;
    a.store(la);
    b.store(lb);
    __syncthreads();
    if (t + 1 < tiles) {
      load_a(a, t + 1);
      load_b(b, t + 1);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int at = ((2 * s + half) ^ sw) << 4;
      u32x4_t fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = *reinterpret_cast<const u32x4_t*>(la + (ra + 32 * i) * 128 + at);
        fb[i] = *reinterpret_cast<const u32x4_t*>(lb + (rb + 32 * i) * 128 + at);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) mma_chunk<T>(acc[i][j], fb[j], fa[i]);
    }
  }
}

}  // namespace cgtp
