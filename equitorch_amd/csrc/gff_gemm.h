// Matrix products of the gated feed-forward block on the matrix cores: tiles of 128 x 128, four wavefronts of 64 x 64 each, or
// of 64 x 64 where there would be too few of the others (TILE), operands brought through registers into one LDS buffer, the
// next tile loaded while one is worked on.
//
// An operand is a matrix whose k or whose rows are contiguous.  In LDS a tile is 8 TILE chunks of 16 bytes either way:
//   k contiguous    TILE rows of eight chunks along k, chunk c of row r at place c ^ (r / 2 & 7);
//   rows contiguous two halves of TILE / 2 rows, in each the rows of one k after the other, chunks exchanged by
//                   (k & 1) | (k << 1 & 4) | (k >> 2 & 2) where there are eight of them, which the transposing loads of
//                   16-bit types (four k of 32 rows for 32 lanes, k + 8 for the others) find in different banks.
// Neither has bank conflicts; with c ^ (r & 7) and (k & 3) | (k >> 1 & 4) they took 10 to 17 % of the cycles.
// 16-bit types use 32 x 32 x 16 instructions, fp32 32 x 32 x 2 ones, four for a pair of chunks, whose k are taken in the order
// that lets a lane read its four in one access.
//
// Aligned operands (16 bytes, rows of whole chunks) are read by buffer loads with 32-bit offsets, where an offset beyond the
// buffer gives zeros; others by element-aligned loads with the last chunk of a row cut.
#pragma once

#include "elem.h"

namespace cgtp {

constexpr int kGemmThreads = 256;
constexpr unsigned kOutside = 0x80000000u;

template <typename T> struct GemmType {
  static constexpr int kChunk = 16 / (int)sizeof(T), kDepth = 8 * kChunk;     // elements of a chunk; k of a tile
};

// An operand's tile.  k contiguous: `base` at the tile's first row, `ld` elements between rows, `rows` of them left.  Rows
// contiguous: base[i] at the first row of half i at k = 0, ld between k, rows[i] left.  The second half of a k-contiguous
// operand is not used.
template <typename T>
struct GemmOperand {
  const T* base[2];
  int64_t ld;
  int rows[2];
};

template <typename T, int TILE, bool K_CONTIGUOUS>
struct GemmStage {
  static constexpr int CH = GemmType<T>::kChunk, kEach = TILE / 32;
  static constexpr int kHalf = TILE / 2, kRow = kHalf / CH;       // rows contiguous: rows of a half, chunks of one k in it
  u32x4_t reg[kEach];

  __device__ static __forceinline__ int mix(int k) { return kRow >= 8 ? (k & 1) | ((k << 1) & 4) | ((k >> 2) & 2) : 0; }

  // k0: first k of the tile, depth: end of k.
  template <bool FAST>
  __device__ __forceinline__ void load(const GemmOperand<T>& p, int64_t k0, int64_t depth) {
    const int tid = threadIdx.x, left = (int)(depth - k0 < GemmType<T>::kDepth ? depth - k0 : GemmType<T>::kDepth);
    if constexpr (K_CONTIGUOUS) {
      const T* base = p.base[0] + k0;
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, kOutside, 0x00027000);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int id = i * kGemmThreads + tid, r = id >> 3, c = (id & 7) ^ ((r >> 1) & 7);
        const bool in = r < p.rows[0] && c * CH < left;
        if constexpr (FAST) {
          const unsigned at = (unsigned)r * (unsigned)(p.ld * sizeof(T)) + c * 16;
          reg[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, in ? at : kOutside, 0, 0));
        } else {
          reg[i] = u32x4_t{0, 0, 0, 0};
          if (in) reg[i] = load_part<u32x4_t, T>(base + r * p.ld + c * CH, left - c * CH);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int h = i / (kEach / 2), id = i % (kEach / 2) * kGemmThreads + tid, k = id / kRow, c = (id % kRow) ^ mix(k);
        const T* base = p.base[h] + k0 * p.ld;
        const bool in = k < left && c * CH < p.rows[h];
        if constexpr (FAST) {
          const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, kOutside, 0x00027000);
          const unsigned at = (unsigned)k * (unsigned)(p.ld * sizeof(T)) + c * 16;
          reg[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, in ? at : kOutside, 0, 0));
        } else {
          reg[i] = u32x4_t{0, 0, 0, 0};
          if (in) reg[i] = load_part<u32x4_t, T>(base + k * p.ld + c * CH, p.rows[h] - c * CH);
        }
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) *reinterpret_cast<u32x4_t*>(lds + (i * kGemmThreads + (int)threadIdx.x) * 16) = reg[i];
  }
  // Rows 32 `block` .. + 31 of the tile at the s-th pair of chunks of k.
  __device__ static __forceinline__ u32x4_t frag(const char* lds, int block, int s) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    if constexpr (K_CONTIGUOUS) {
      const int r = block * 32 + (lane & 31);
      return *reinterpret_cast<const u32x4_t*>(lds + r * 128 + (((2 * s + half) ^ ((r >> 1) & 7)) << 4));
    } else if constexpr (sizeof(T) == 2) {
      const char* h = lds + block * 32 / kHalf * (TILE * 64);
      const int k = 16 * s + 8 * half + ((lane & 15) >> 2), m = block * 32 % kHalf + (lane & 16) + 4 * (lane & 3);
      u32x4_t f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int kk = k + 4 * i;
        typedef short v4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) v4 lds_v4;
        const char* at = h + kk * (kRow * 16) + (((m >> 3) ^ mix(kk)) << 4) + (m & 7) * 2;
        const u32x2_t v = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)at));
        f[2 * i] = v[0];
        f[2 * i + 1] = v[1];
      }
      return f;
    } else {
      const char* h = lds + block * 32 / kHalf * (TILE * 64);
      const int k = 8 * s + 4 * half, m = block * 32 % kHalf + (lane & 31);
      u32x4_t f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int kk = k + j;
        f[j] = *reinterpret_cast<const unsigned*>(h + kk * (kRow * 16) + (((m >> 2) ^ mix(kk)) << 4) + (m & 3) * 4);
      }
      return f;
    }
  }
};

// B = TILE / 64 blocks of 32 each way for a wavefront (wm, wn).  acc[i][j]: rows 32 (B wm + i) of the first operand; of the second
// 32 (B wn + j), or with SPLIT 32 wn of half j (TILE = 128).  A lane holds row lane % 32 of the first and, at index 4 g + e, row 8 g + 4 (lane / 32) + e of the second.
// a(t, k0, depth) / b(t): the operands of tile t of k, and where its k begin and end; tiles: the same for all threads.
template <int TILE> using GemmAcc = f32x16_t[TILE / 64][TILE / 64];

template <typename T, int TILE, bool FAST, bool KA, bool KB, bool SPLIT, typename A, typename B>
__device__ __forceinline__ void gemm_loop(GemmAcc<TILE>& acc, char* lds, int64_t tiles, A&& a, B&& b) {
  constexpr int kB = TILE / 64;
  const int wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int i = 0; i < kB; ++i)
#pragma unroll
    for (int j = 0; j < kB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  if (tiles <= 0) return;
  GemmStage<T, TILE, KA> sa;
  GemmStage<T, TILE, KB> sb;
  auto fetch = [&](int64_t t) {
    int64_t k0, depth;
    const GemmOperand<T> pa = a(t, k0, depth), pb = b(t);
    sa.template load<FAST>(pa, k0, depth);
    sb.template load<FAST>(pb, k0, depth);
  };
  fetch(0);
  char* la = lds;
  char* lb = lds + TILE * 128;
  for (int64_t t = 0; t < tiles; ++t) {
    if (t) __syncthreads();         // the tile before has used the buffer
    sa.store(la);
    sb.store(lb);
    __syncthreads();
    if (t + 1 < tiles) fetch(t + 1);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u32x4_t fa[kB], fb[kB];
#pragma unroll
      for (int i = 0; i < kB; ++i) fa[i] = GemmStage<T, TILE, KA>::frag(la, kB * wm + i, s);
#pragma unroll
      for (int j = 0; j < kB; ++j) fb[j] = GemmStage<T, TILE, KB>::frag(lb, SPLIT ? 2 * j + wn : kB * wn + j, s);
#pragma unroll
      for (int i = 0; i < kB; ++i)
#pragma unroll
        for (int j = 0; j < kB; ++j) acc[i][j] = mma_pair<T>(fb[j], fa[i], acc[i][j]);
    }
  }
}

// Eight neighbouring elements as they come from memory.
template <typename T>
struct EightRaw {
  static constexpr int N = 16 / (int)sizeof(T);
  u32x4_t v[8 / N];
  __device__ __forceinline__ void load(const T* p, int valid) {
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      v[i] = u32x4_t{0, 0, 0, 0};
      if (valid > i * N) v[i] = load_part<u32x4_t, T>(p + i * N, valid - i * N);
    }
  }
  __device__ __forceinline__ void get(float (&to)[8]) const {
    typedef T vec __attribute__((ext_vector_type(N)));
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      const vec e = __builtin_bit_cast(vec, v[i]);
#pragma unroll
      for (int j = 0; j < N; ++j) to[i * N + j] = (float)e[j];
    }
  }
};

// The results through LDS in fp32, so that a row leaves in whole lines: each thread is handed, for TILE^2 / 2048 places i, eight
// neighbouring columns of a row: use(i, row, column, values).  SPLIT: column 32 wn + .. of half j is column TILE / 2 j + 32 wn +
// .., and use gets the same eight columns of both halves, for half as many places: use(i, row, column, first half, second
// half).  fetch(i, row, column) is called AHEAD places earlier.
template <int TILE, bool SPLIT, int AHEAD, typename Fetch, typename Use>
__device__ __forceinline__ void gemm_results(const GemmAcc<TILE>& acc, char* lds, Fetch&& fetch, Use&& use) {
  constexpr int kB = TILE / 64, kRow = TILE / (SPLIT ? 16 : 8), kPart = 64 * kRow / kGemmThreads, kPlaces = kB * kPart;
  constexpr int kCols = TILE / 4;
  auto place = [&](int i, int& r, int& c) {
    const int id = i % kPart * kGemmThreads + (int)threadIdx.x, at = id / kRow;       // row of the buffer
    r = (at >> 5) * (32 * kB) + (i / kPart) * 32 + (at & 31);
    c = id % kRow * 8;
    return at;
  };
  auto ahead = [&](int i) {
    int r, c;
    place(i, r, c);
    fetch(i, r, c);
  };
#pragma unroll
  for (int i = 0; i < AHEAD && i < kPlaces; ++i) ahead(i);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
  float* tile = reinterpret_cast<float*>(lds);           // 64 rows of kCols chunks, chunk c of row r at c ^ (r % kCols)
  auto chunk = [&](int r, int c) { return reinterpret_cast<f32x4*>(tile + r * TILE + ((c ^ (r & (kCols - 1))) << 2)); };
#pragma unroll
  for (int part = 0; part < kB; ++part) {                // rows 32 part .. + 31 of both wavefronts' rows
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kB; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = (SPLIT ? TILE / 2 * j + 32 * wn : 32 * kB * wn + 32 * j) + 8 * g + 4 * (lane >> 5);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[part][j][4 * g + e];
        *chunk(32 * wm + (lane & 31), n >> 2) = v;
      }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < kPart; ++p) {
      const int i = part * kPart + p;
      int r, c;
      const int at = place(i, r, c);
      float v[8];
      auto take = [&](int first, float (&to)[8]) {
        const f32x4 x = *chunk(at, first), y = *chunk(at, first + 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) { to[e] = x[e]; to[4 + e] = y[e]; }
      };
      take(c / 4, v);
      if constexpr (SPLIT) {
        float u[8];
        take(kCols / 2 + c / 4, u);
        use(i, r, c, v, u);
      } else {
        use(i, r, c, v);
      }
      if (i + AHEAD < kPlaces) ahead(i + AHEAD);
    }
  }
}

}  // namespace cgtp
