// Embedding of node kinds (cgtp_embed_forward) and its gradient (cgtp_embed_backward):
//
//   out[i, c] = scale * table[kind[i], c],        grad_table[t, c] = scale * sum_{i : kind[i] = t} grad_out[i, c]
//
// A kind outside 0 .. n_kinds - 1 gives a row of zeros and no gradient.  Both are bound by memory: the forward writes out
// and finds the table in cache, the backward reads grad_out once.
//
// The backward sums the rows of a kind in ascending order of their index cut at fixed places, so that its result does not
// depend on timing: no atomics.  The rows are sorted by kind first (stable counting sort by digits of eight bits, as
// many as n_kinds needs: one up to 255 kinds), then the sorted positions are cut into equal chunks whatever the kinds:
// a few kinds may hold most rows (elements), or most kinds a row or two (environments), and neither leaves compute
// units idle.  A run of equal kinds inside a chunk goes straight to the table; the run a chunk begins with and the one it
// ends with are left as fp32 partial sums (fp64 for fp64) and joined by the workgroup of the chunk where the run begins.
//
// A lane takes 16 bytes of a row, wherever it starts; where a row is not whole vectors its last one is taken from its end, and
// the columns that this vector shares with the one before are computed and written twice, with the same bits.
// Lookup and gradient of 1000003 rows of 201 channels, 30000 kinds, bf16: 605 us an element at a time, 290 so, 200 channels 265.
#include "elem.h"

#include <algorithm>

namespace cgtp {
namespace {

constexpr int64_t kMaxBlocks = 1 << 20;      // of grids that stride over their work


// ---- forward --------------------------------------------------------------------------------------------------
// A group of lanes per row, four rows at a time: the kinds, then the table's rows are on their way together.  1000003 rows of 256
// channels, 30011 kinds, bf16: 138 us, 3.7 TB/s written: bound by memory and by the gathers from the caches beside it (a fill
// alone reaches 6.8, a copy 5.1 both ways together).
template <typename T, int V>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const int64_t* __restrict__ kind, const T* __restrict__ table,
                                                        T* __restrict__ out, int64_t n_rows, int64_t n_kinds, int C,
                                                        typename AccOf<T>::type scale, int lpr_log2) {
  using A = typename AccOf<T>::type;
  constexpr int kRows = 4;
  const int sub = threadIdx.x & ((1 << lpr_log2) - 1), step = V << lpr_log2;
  const int64_t stride = (int64_t)gridDim.x * 256 >> lpr_log2;
  for (int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lpr_log2; row < n_rows; row += kRows * stride) {
    int64_t k[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) k[j] = row + j * stride < n_rows ? kind[row + j * stride] : -1;
    for (int at = sub * V; at < C; at += step) {
      const int c = min(at, C - V);
      A v[kRows][V];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const bool ok = (uint64_t)k[j] < (uint64_t)n_kinds;
        load_elems<T, V>(v[j], table + (ok ? k[j] : 0) * C + c);
#pragma unroll
        for (int e = 0; e < V; ++e) v[j][e] = ok ? v[j][e] * scale : A(0);
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (row + j * stride < n_rows) store_elems<T, V, true>(out + (row + j * stride) * C + c, v[j]);
    }
  }
}

// ---- sort by kind -----------------------------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave, kDigits = 256, kSortMaxBlocks = 256;

// The key of a position of the pass's input: from the kinds in the first pass (n_kinds for a kind out of range), from
// the last pass's output afterwards.
struct SortInput {
  const int64_t* kind;
  const int32_t *keys, *rows;
  int64_t n_kinds;
  __device__ __forceinline__ int key(int64_t i) const {
    if (keys) return keys[i];
    const int64_t k = kind[i];
    return (uint64_t)k < (uint64_t)n_kinds ? (int)k : (int)n_kinds;
  }
};

// Zeros, by threads `at` of `stride`.
__device__ __forceinline__ void clear_by(char* p, int64_t bytes, int64_t at, int64_t stride) {
  const int64_t words = (reinterpret_cast<uintptr_t>(p) & 15u) ? 0 : bytes / 16;
  for (int64_t i = at; i < words; i += stride) reinterpret_cast<uint4*>(p)[i] = uint4{0, 0, 0, 0};
  for (int64_t i = words * 16 + at; i < bytes; i += stride) p[i] = 0;
}

// Digits of every block's part; the first pass also clears the gradient (kinds without a row keep the zeros), with blocks that do
// nothing else where the table is large for the rows (300 rows of 30000 kinds, 256 channels fp32: 227 us without them).
__global__ void __launch_bounds__(kSortThreads) embed_digits_kernel(SortInput in, int32_t* __restrict__ digits,
                                                                    int64_t n_rows, int64_t per_block, int shift,
                                                                    char* __restrict__ clear, int64_t clear_bytes) {
  if (clear_bytes) clear_by(clear, clear_bytes, (int64_t)blockIdx.x * kSortThreads + threadIdx.x, (int64_t)gridDim.x * kSortThreads);
  const int64_t i0 = blockIdx.x * per_block;
  if (i0 >= n_rows) return;
  __shared__ int count[kDigits];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
  __syncthreads();
  const int64_t i1 = i0 + per_block < n_rows ? i0 + per_block : n_rows;
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kSortThreads) atomicAdd(&count[(in.key(i) >> shift) & 255], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) digits[(int64_t)blockIdx.x * kDigits + d] = count[d];
}

// Each block works out where its part's digits begin from the counts of all blocks, then moves its part in order: the rank of
// a key is the keys of its digit in earlier rounds, in earlier wavefronts and in earlier lanes (a ballot per bit).
__global__ void __launch_bounds__(kSortThreads) embed_scatter_kernel(SortInput in, const int32_t* __restrict__ digits,
                                                                     int32_t* __restrict__ keys_out,
                                                                     int32_t* __restrict__ rows_out, int64_t n_rows,
                                                                     int64_t per_block, int shift) {
  constexpr int kParts = kSortThreads / kDigits;
  __shared__ int count[kSortWaves][kDigits];
  __shared__ int base[kDigits], before[kParts][kDigits], total[kParts][kDigits], wave_total[kDigits / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  {
    const int d = tid % kDigits, part = tid / kDigits;
    int all = 0, mine = 0;
#pragma unroll 8
    for (int b = part; b < (int)gridDim.x; b += kParts) {
      const int n = digits[(int64_t)b * kDigits + d];
      all += n;
      mine += b < (int)blockIdx.x ? n : 0;
    }
    before[part][d] = mine;
    total[part][d] = all;
    __syncthreads();
    int scan = 0, sum = 0;
    if (tid < kDigits) {
      mine = 0;
      for (int p = 0; p < kParts; ++p) { sum += total[p][tid]; mine += before[p][tid]; }
      scan = sum;
      for (int off = 1; off < kWave; off <<= 1) {
        const int up = __shfl_up(scan, off, kWave);
        if (lane >= off) scan += up;
      }
      if (lane == kWave - 1) wave_total[wave] = scan;
    }
    __syncthreads();
    if (tid < kDigits) {
      for (int w = 0; w < wave; ++w) scan += wave_total[w];
      base[tid] = scan - sum + mine;
    }
  }
  const int64_t i0 = blockIdx.x * per_block, i1 = i0 + per_block < n_rows ? i0 + per_block : n_rows;
  for (int64_t r = i0; r < i1; r += kSortThreads) {
    for (int i = tid; i < kSortWaves * kDigits; i += kSortThreads) (&count[0][0])[i] = 0;
    __syncthreads();
    const int64_t i = r + tid;
    const bool ok = i < i1;
    const int key = ok ? in.key(i) : 0, d = (key >> shift) & 255;
    uint64_t same = __ballot(ok);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (ok && rank == 0) count[wave][d] = __popcll(same);
    __syncthreads();
    if (tid < kDigits) {
      int at = base[tid];
      for (int w = 0; w < kSortWaves; ++w) {
        const int n = count[w][tid];
        count[w][tid] = at;
        at += n;
      }
      base[tid] = at;
    }
    __syncthreads();
    if (ok) {
      const int to = count[wave][d] + rank;
      keys_out[to] = key;
      rows_out[to] = in.rows ? in.rows[i] : (int)i;
    }
    __syncthreads();
  }
}

// ---- sums over runs -----------------------------------------------------------------------------------------------
// What a chunk leaves to be joined: the kinds of its first and last run, whether they are one run.  Its partial sums are rows
// 2 c (first run) and 2 c + 1 (last run, unless it is the first).
struct ChunkRuns { int first, last, whole, reserved; };

// The same workload: 114 us, 4.5 TB/s of rows gathered from memory, eight on their way for each lane.
// A workgroup per chunk and block of columns.  Each group of lanes walks its own part of the chunk; the groups' first and last
// runs are joined in LDS.
template <typename T, int V>
__global__ void __launch_bounds__(256) embed_sum_kernel(const T* __restrict__ grad_out, const int32_t* __restrict__ keys,
                                                        const int32_t* __restrict__ rows, T* __restrict__ grad_table,
                                                        typename AccOf<T>::type* __restrict__ partial,
                                                        ChunkRuns* __restrict__ runs, int64_t n_rows, int n_kinds, int C,
                                                        typename AccOf<T>::type scale, int lpr_log2, int per_group) {
  using A = typename AccOf<T>::type;
  constexpr int kAhead = 8;
  __shared__ A head_sum[256 * V], tail_sum[256 * V];
  __shared__ int head_key[256], tail_key[256];           // tail_key -1: the group's part is one run; head_key -1: it is empty
  const int groups = 256 >> lpr_log2, lpr = 1 << lpr_log2;
  const int sub = threadIdx.x & (lpr - 1), g = threadIdx.x >> lpr_log2;
  const int at_c = (blockIdx.y * lpr + sub) * V, c = min(at_c, C - V);
  const bool col_ok = at_c < C;
  const int64_t p0 = ((int64_t)blockIdx.x * groups + g) * per_group;
  const int64_t p1 = p0 + per_group < n_rows ? p0 + per_group : n_rows;
  auto put = [&](int key, const A (&s)[V]) {
    if (!col_ok || key >= n_kinds) return;
    A o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = s[j] * scale;
    store_elems<T, V>(grad_table + (int64_t)key * C + c, o);
  };
  A acc[V];
  int cur = -1;
  bool in_head = true;
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = A(0);
  auto close = [&]() {                                   // the run of kind `cur` ends
    if (in_head) {
#pragma unroll
      for (int j = 0; j < V; ++j) head_sum[threadIdx.x * V + j] = acc[j];
      if (sub == 0) head_key[g] = cur;
      in_head = false;
    } else {
      put(cur, acc);
    }
  };
  for (int64_t p = p0; p < p1; p += kAhead) {
    int key[kAhead];
    A v[kAhead][V];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t at = p + j < p1 ? p + j : p1 - 1;
      key[j] = keys[at];
      load_elems<T, V>(v[j], grad_out + (int64_t)rows[at] * C + c);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (p + j >= p1) continue;
      if (key[j] != cur) {
        if (cur >= 0) close();
        cur = key[j];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = v[j][e];
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += v[j][e];
      }
    }
  }
  if (sub == 0) { tail_key[g] = -1; if (p0 >= p1) head_key[g] = -1; }
  if (p0 < p1) {
    if (in_head) {
      close();
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) tail_sum[threadIdx.x * V + j] = acc[j];
      if (sub == 0) tail_key[g] = cur;
    }
  }
  __syncthreads();
  if (threadIdx.x >= lpr) return;
  A* first_row = partial + (int64_t)blockIdx.x * 2 * C;
  in_head = true;
  cur = head_key[0];                                     // group 0 is never empty: the grid covers n_rows
  const int first_key = cur;
  auto leave = [&]() {
    if (in_head) {
      if (col_ok)
#pragma unroll
        for (int j = 0; j < V; ++j) first_row[c + j] = acc[j];
      in_head = false;
    } else {
      put(cur, acc);
    }
  };
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = A(0);
  for (int k = 0; k < groups && head_key[k] >= 0; ++k) {
    const int at = (k * lpr + sub) * V;
    if (head_key[k] != cur) {
      leave();
      cur = head_key[k];
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = head_sum[at + j];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += head_sum[at + j];
    }
    if (tail_key[k] >= 0) {
      leave();
      cur = tail_key[k];
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = tail_sum[at + j];
    }
  }
  const bool whole = in_head;
  if (col_ok)
#pragma unroll
    for (int j = 0; j < V; ++j) first_row[(whole ? 0 : C) + c + j] = acc[j];
  if (sub == 0 && blockIdx.y == 0) runs[blockIdx.x] = ChunkRuns{first_key, cur, whole ? 1 : 0, 0};
}

// Joins the runs that touch the ends of chunks: the workgroup of the chunk where such a run begins adds its parts.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) embed_join_kernel(const typename AccOf<T>::type* __restrict__ partial,
                                                         const ChunkRuns* __restrict__ runs, T* __restrict__ grad_table,
                                                         int n_chunks, int n_kinds, int C,
                                                         typename AccOf<T>::type scale, int lpr_log2) {
  using A = typename AccOf<T>::type;
  __shared__ A sums[THREADS];
  const int c0 = blockIdx.x;
  const ChunkRuns me = runs[c0];
  const int lpr = 1 << lpr_log2, groups = THREADS >> lpr_log2, sub = threadIdx.x & (lpr - 1), g = threadIdx.x >> lpr_log2;
  const int c = blockIdx.y * lpr + sub;
  const bool begins = c0 == 0 || runs[c0 - 1].last != me.first;
  if (begins && !me.whole && g == 0 && c < C && me.first < n_kinds)
    grad_table[(int64_t)me.first * C + c] = (T)(partial[(int64_t)c0 * 2 * C + c] * scale);
  if ((me.whole && !begins) || me.last >= n_kinds) return;
  int lo = c0, hi = n_chunks - 1;                        // last chunk that begins with this kind (kinds ascend), or c0
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (runs[mid].first <= me.last) lo = mid; else hi = mid - 1;
  }
  A s = A(0);
  if (c < C) {
    if (g == 0) s = partial[((int64_t)c0 * 2 + (me.whole ? 0 : 1)) * C + c];
    int k = c0 + 1 + g;
    for (; k + 3 * groups <= lo; k += 4 * groups) {
      const A a0 = partial[(int64_t)k * 2 * C + c], a1 = partial[(int64_t)(k + groups) * 2 * C + c],
              a2 = partial[(int64_t)(k + 2 * groups) * 2 * C + c], a3 = partial[(int64_t)(k + 3 * groups) * 2 * C + c];
      s += a0; s += a1; s += a2; s += a3;
    }
    for (; k <= lo; k += groups) s += partial[(int64_t)k * 2 * C + c];
  }
  sums[threadIdx.x] = s;
  __syncthreads();
  if (g != 0 || c >= C) return;
  for (int k = 1; k < groups; ++k) s += sums[k * lpr + sub];
  grad_table[(int64_t)me.last * C + c] = (T)(s * scale);
}

// Few rows: one launch in place of the sort, the sums and the join.  Every wavefront holds all the kinds, takes a row of the table
// at a time, finds who has its kind and sums them in ascending order, eight on their way.  256 rows of 100 kinds, 64 channels
// fp32, 5 us against 16 in four launches, all of one kind 17 against 13; of 30000 kinds, 256 channels, 8.5.
constexpr int kFewRows = 256;
template <typename T, int V>
__global__ void __launch_bounds__(256) embed_few_kernel(const int64_t* __restrict__ kind, const T* __restrict__ grad_out,
                                                        T* __restrict__ grad_table, int n_rows, int n_kinds, int C,
                                                        typename AccOf<T>::type scale) {
  using A = typename AccOf<T>::type;
  constexpr int kGroups = kFewRows / kWave, kAhead = 8;
  const int lane = threadIdx.x & (kWave - 1), waves = gridDim.x * (256 / kWave);
  int mine[kGroups];
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    const int i = q * kWave + lane;
    const int64_t k = i < n_rows ? kind[i] : -1;
    mine[q] = (uint64_t)k < (uint64_t)n_kinds ? (int)k : -1;
  }
  for (int64_t t = (blockIdx.x * 256 + (int)threadIdx.x) / kWave; t < n_kinds; t += waves) {
    uint64_t who[kGroups];
#pragma unroll
    for (int q = 0; q < kGroups; ++q) who[q] = __ballot(mine[q] == (int)t);
    for (int at = lane * V; at < C; at += kWave * V) {
      const int c = min(at, C - V);
      A acc[V];
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = A(0);
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        for (uint64_t m = who[q]; m;) {
          A v[kAhead][V];
          const int n = min(kAhead, __popcll(m));
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            if (j >= n) continue;
            load_elems<T, V>(v[j], grad_out + (int64_t)(q * kWave + __ffsll((unsigned long long)m) - 1) * C + c);
            m &= m - 1;
          }
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            if (j >= n) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += v[j][e];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] *= scale;
      store_elems<T, V>(grad_table + t * C + c, acc);
    }
  }
}

__global__ void __launch_bounds__(256) embed_clear_kernel(char* __restrict__ p, int64_t bytes) {
  clear_by(p, bytes, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

// ---- launches -----------------------------------------------------------------------------------------------------
int log2_up(int64_t n, int most) {
  int lg = 0;
  while (lg < most && ((int64_t)1 << lg) < n) ++lg;
  return lg;
}

// Sorted positions a group of lanes walks: long enough that partial sums stay a small part of what is read, short enough that
// there are about eight workgroups for each of the 256 compute units where there are rows for them.
int sum_per_group(int64_t n_rows, int groups) {
  int64_t n = n_rows / ((int64_t)groups * 2048);
  n = n < 16 ? 16 : n > 256 ? 256 : n;
  return (int)n & ~7;
}

struct EmbedPlan {
  int v, lpr_log2, groups, per_group, passes;
  int64_t chunks, blocks, per_block;
  int64_t keys[2], rows[2], digits, partial, runs, bytes;    // offsets into the workspace
};

template <typename T>
EmbedPlan embed_plan(int64_t n_rows, int64_t n_kinds, int C) {
  using A = typename AccOf<T>::type;
  EmbedPlan p;
  constexpr int VW = 16 / sizeof(T);
  p.v = C >= VW ? VW : 1;
  p.lpr_log2 = log2_up((C + p.v - 1) / p.v, 6);
  p.groups = 256 >> p.lpr_log2;
  p.per_group = sum_per_group(n_rows, p.groups);
  const int64_t per_chunk = (int64_t)p.groups * p.per_group;
  p.chunks = (n_rows + per_chunk - 1) / per_chunk;
  p.per_block = (n_rows + kSortMaxBlocks - 1) / kSortMaxBlocks;
  p.per_block = (p.per_block + kSortThreads - 1) / kSortThreads * kSortThreads;
  p.blocks = (n_rows + p.per_block - 1) / p.per_block;
  p.passes = 1;
  while (p.passes < 4 && (n_kinds >> (8 * p.passes)) > 0) ++p.passes;      // keys 0 .. n_kinds
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t was = at; at += (bytes + 255) / 256 * 256; return was; };
  for (int i = 0; i < 2; ++i) {
    p.keys[i] = take(n_rows * 4);
    p.rows[i] = take(n_rows * 4);
    if (p.passes == 1 && i == 0) { p.keys[1] = p.keys[0]; p.rows[1] = p.rows[0]; break; }
  }
  p.digits = take(p.blocks * kDigits * 4);
  p.partial = take(p.chunks * 2 * C * (int64_t)sizeof(A));
  p.runs = take(p.chunks * (int64_t)sizeof(ChunkRuns));
  p.bytes = at;
  return p;
}

int embed_check(int64_t n_rows, int64_t n_kinds, int C, int dtype) {
  if (elem_size(dtype) == 0) return CGTP_ERR_DTYPE;
  if (n_rows < 0 || n_rows > 0x7fffffff || n_kinds <= 0 || n_kinds >= 0x7fffffff || C <= 0 || C > 0x7fff) return CGTP_ERR_SHAPE;
  return CGTP_OK;
}

template <typename T>
int embed_forward(const int64_t* kind, const void* table, void* out, int64_t n_rows, int64_t n_kinds, int C, double scale,
                  hipStream_t stream) {
  constexpr int VW = 16 / sizeof(T);
  const bool vec = C >= VW;
  const int lpr_log2 = log2_up(vec ? (C + VW - 1) / VW : C, 8);
  // a row for each group while that leaves compute units idle, else four
  const int64_t threads = n_rows << lpr_log2;
  const int64_t blocks = std::min<int64_t>(threads < 2048 * 256 ? (threads + 255) / 256 : (threads + 1023) / 1024, kMaxBlocks);
  auto kern = vec ? embed_fwd_kernel<T, VW> : embed_fwd_kernel<T, 1>;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, kind, (const T*)table, (T*)out, n_rows, n_kinds, C,
                     (typename AccOf<T>::type)scale, lpr_log2);
  return launch_status();
}

template <typename T>
int embed_backward(const int64_t* kind, const void* grad_out, void* grad_table, void* workspace, int64_t n_rows,
                   int64_t n_kinds, int C, double scale, hipStream_t stream) {
  using A = typename AccOf<T>::type;
  if (n_rows <= kFewRows) {
    constexpr int VW = 16 / sizeof(T);
    auto few = C >= VW ? embed_few_kernel<T, VW> : embed_few_kernel<T, 1>;
    hipLaunchKernelGGL(few, dim3((unsigned)std::min<int64_t>((n_kinds + 3) / 4, 2048)), dim3(256), 0, stream, kind, (const T*)grad_out,
                       (T*)grad_table, (int)n_rows, (int)n_kinds, C, (A)scale);
    return launch_status();
  }
  const EmbedPlan p = embed_plan<T>(n_rows, n_kinds, C);
  char* ws = (char*)workspace;
  int32_t* digits = (int32_t*)(ws + p.digits);
  for (int pass = 0; pass < p.passes; ++pass) {
    const int from = (pass + 1) & 1, to = pass & 1;
    const SortInput in = {kind, pass ? (const int32_t*)(ws + p.keys[from]) : nullptr,
                          pass ? (const int32_t*)(ws + p.rows[from]) : nullptr, n_kinds};
    const int64_t clear = pass ? 0 : n_kinds * C * (int64_t)sizeof(T);
    const int64_t grid = std::max(p.blocks, std::min<int64_t>(512, clear >> 16));
    hipLaunchKernelGGL(embed_digits_kernel, dim3((unsigned)grid), dim3(kSortThreads), 0, stream, in, digits, n_rows, p.per_block,
                       8 * pass, (char*)grad_table, clear);
    hipLaunchKernelGGL(embed_scatter_kernel, dim3((unsigned)p.blocks), dim3(kSortThreads), 0, stream, in, digits,
                       (int32_t*)(ws + p.keys[to]), (int32_t*)(ws + p.rows[to]), n_rows, p.per_block, 8 * pass);
  }
  const int last = (p.passes - 1) & 1;
  const int32_t *keys = (const int32_t*)(ws + p.keys[last]), *rows = (const int32_t*)(ws + p.rows[last]);
  A* partial = (A*)(ws + p.partial);
  ChunkRuns* runs = (ChunkRuns*)(ws + p.runs);
  const int per_block = p.v << p.lpr_log2;
  auto kern = p.v == 1 ? embed_sum_kernel<T, 1> : embed_sum_kernel<T, 16 / sizeof(T)>;
  hipLaunchKernelGGL(kern, dim3((unsigned)p.chunks, (C + per_block - 1) / per_block), dim3(256), 0, stream,
                     (const T*)grad_out, keys, rows, (T*)grad_table, partial, runs, n_rows, (int)n_kinds, C, (A)scale,
                     p.lpr_log2, p.per_group);
  // With few chunks the longest run bounds this kernel, with many the workgroups that have next to nothing to join:
  // 60001 rows of 100 kinds 5.5 us with 1024 threads, 9.6 with 256; 1000003 rows of 30011 kinds 32 us and 15.
  const int lpr_log2 = log2_up(C, 6), threads = p.chunks <= 1024 ? 1024 : 256;
  hipLaunchKernelGGL((threads == 1024 ? embed_join_kernel<T, 1024> : embed_join_kernel<T, 256>),
                     dim3((unsigned)p.chunks, (C + (1 << lpr_log2) - 1) >> lpr_log2), dim3(threads), 0, stream,
                     (const A*)partial, (const ChunkRuns*)runs, (T*)grad_table, (int)p.chunks, (int)n_kinds, C, (A)scale,
                     lpr_log2);
  return launch_status();
}

}  // namespace
}  // namespace cgtp

extern "C" {

int64_t cgtp_embed_workspace_bytes(int64_t n_rows, int64_t n_kinds, int C, int dtype) {
  using namespace cgtp;
  if (embed_check(n_rows, n_kinds, C, dtype) != CGTP_OK || n_rows == 0) return 0;
  return dtype == CGTP_F64 ? embed_plan<double>(n_rows, n_kinds, C).bytes
         : dtype == CGTP_F32 ? embed_plan<float>(n_rows, n_kinds, C).bytes
                             : embed_plan<bf16_t>(n_rows, n_kinds, C).bytes;
}

int cgtp_embed_forward(const int64_t* kind, const void* table, void* out, int64_t n_rows, int64_t n_kinds, int C,
                       double scale, int dtype, void* stream) {
  using namespace cgtp;
  if (int rc = embed_check(n_rows, n_kinds, C, dtype)) return rc;
  if (n_rows == 0) return CGTP_OK;
  if (!kind || !table || !out) return CGTP_ERR_NULL;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case CGTP_F32: return embed_forward<float>(kind, table, out, n_rows, n_kinds, C, scale, s);
    case CGTP_F64: return embed_forward<double>(kind, table, out, n_rows, n_kinds, C, scale, s);
    case CGTP_BF16: return embed_forward<bf16_t>(kind, table, out, n_rows, n_kinds, C, scale, s);
    default: return embed_forward<f16_t>(kind, table, out, n_rows, n_kinds, C, scale, s);
  }
}

int cgtp_embed_backward(const int64_t* kind, const void* grad_out, void* grad_table, void* workspace, int64_t n_rows,
                        int64_t n_kinds, int C, double scale, int dtype, void* stream) {
  using namespace cgtp;
  if (int rc = embed_check(n_rows, n_kinds, C, dtype)) return rc;
  if (!grad_table) return CGTP_ERR_NULL;
  hipStream_t s = (hipStream_t)stream;
  if (n_rows == 0) {
    const int64_t bytes = n_kinds * C * elem_size(dtype);
    hipLaunchKernelGGL(embed_clear_kernel, dim3((unsigned)std::min<int64_t>((bytes + 4095) / 4096, kMaxBlocks)), dim3(256), 0, s, (char*)grad_table, bytes);
    return launch_status();
  }
  if (!kind || !grad_out) return CGTP_ERR_NULL;
  if (!workspace) return CGTP_ERR_WORKSPACE;
  switch (dtype) {
    case CGTP_F32: return embed_backward<float>(kind, grad_out, grad_table, workspace, n_rows, n_kinds, C, scale, s);
    case CGTP_F64: return embed_backward<double>(kind, grad_out, grad_table, workspace, n_rows, n_kinds, C, scale, s);
    case CGTP_BF16: return embed_backward<bf16_t>(kind, grad_out, grad_table, workspace, n_rows, n_kinds, C, scale, s);
    default: return embed_backward<f16_t>(kind, grad_out, grad_table, workspace, n_rows, n_kinds, C, scale, s);
  }
}

}  // extern "C"
