// Columns to expert-sorted rows and back.
//
// x[f][b] is feature-major (batch contiguous), rows[r][f] has the features of
// a row contiguous; row[j][b] is the row of column b's choice j (negative:
// none).  gather: rows[row[j][b]][.] = x[.][b].  combine: y[.][b] = sum_j
// weight[j][b] rows[row[j][b]][.] in fp32, rounded once.  Their gradients are a
// combination with unit weights, and (fused) d_rows = weight d_y with
// d_weight[j][b] = <rows[row[j][b]], d_y[.][b]>.
//
// All are transposes bound by HBM: a block turns tiles of 64 columns x 64 words
// in shared memory (a word is 4 bytes: one fp32 or two 16-bit features).  On the
// column side a thread moves four columns at once where the batch is aligned
// (one 16-byte or two 8-byte accesses), on the row side 16 lanes take a row's 64
// words, 16 bytes each where the rows are aligned.  Word w of column c lies in
// 16-byte chunk (w / 4) ^ (c / 4 mod 16) of the column's 256 bytes: whole chunks
// for the row side without conflicts, two-way conflicts for the column side.
// Measured: 2^20 columns of 256 bf16 features to two rows each in 253 us (1.63 GB,
// 6.4 TB/s, the rate of a plain copy); with one element a thread it was 394.  The
// combination of the same rows takes 471 us, its gradient 451 (2.7 GB, 6.0 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "device_math.cuh"
#include "operators.h"

namespace ponni_b200 {
namespace {

constexpr int kBlock = 256;
constexpr int kWarps = kBlock / 32;
constexpr int kTileCols = 64;
constexpr int kBackCols = 32;  // of combine_backward_kernel
constexpr int kTileWords = 64;
constexpr int kRowLanes = 16;  // lanes that take a row

// Place of word w of column c in the tile.
__device__ __forceinline__ int place(int c, int w) { return c * kTileWords + ((((w >> 2) ^ (c >> 2)) & 15) << 2) + (w & 3); }

template <class T> struct Word {  // 4 bytes of consecutive features
  static constexpr int n = 4 / sizeof(T);
  T v[n];
};

template <class T>
__device__ __forceinline__ void unpack(uint32_t u, float (&f)[Word<T>::n]) {
  Word<T> w;
  *reinterpret_cast<uint32_t*>(&w) = u;
#pragma unroll
  for (int i = 0; i < Word<T>::n; ++i) f[i] = Num<T>::to_c(w.v[i]);
}
template <class T>
__device__ __forceinline__ uint32_t pack(const float (&f)[Word<T>::n]) {
  Word<T> w;
#pragma unroll
  for (int i = 0; i < Word<T>::n; ++i) w.v[i] = Num<T>::from_c(f[i]);
  return *reinterpret_cast<uint32_t*>(&w);
}

// A word of a row: 4 bytes at once where the row starts on a 4-byte boundary
// and the word is whole, element by element otherwise.
template <class T>
__device__ __forceinline__ uint32_t load_word(const T* __restrict__ row, int f, int features, bool whole) {
  constexpr int n = Word<T>::n;
  if (whole && f + n <= features) return __ldg(reinterpret_cast<const unsigned*>(row + f));
  Word<T> w;
#pragma unroll
  for (int i = 0; i < n; ++i) w.v[i] = f + i < features ? row[f + i] : Num<T>::from_c(0.0f);
  return *reinterpret_cast<uint32_t*>(&w);
}
template <class T>
__device__ __forceinline__ void store_word(T* __restrict__ row, int f, int features, bool whole, uint32_t u) {
  constexpr int n = Word<T>::n;
  if (whole && f + n <= features) {
    *reinterpret_cast<uint32_t*>(row + f) = u;
    return;
  }
  Word<T> w;
  *reinterpret_cast<uint32_t*>(&w) = u;
#pragma unroll
  for (int i = 0; i < n; ++i)
    if (f + i < features) row[f + i] = w.v[i];
}

// Four columns of a word: n rows of x, four consecutive elements each, turned
// into one word a column.
template <class T>
__device__ __forceinline__ void turn_in(const T* __restrict__ x, int64_t ld, int f, int features, uint32_t (&u)[4]) {
  if constexpr (sizeof(T) == 4) {
    const uint4 v = f < features ? __ldg(reinterpret_cast<const uint4*>(x + f * ld)) : make_uint4(0, 0, 0, 0);
    u[0] = v.x;
    u[1] = v.y;
    u[2] = v.z;
    u[3] = v.w;
  } else {
    static_assert(sizeof(T) == 2, "16-bit features");
    const uint2 a = f < features ? __ldg(reinterpret_cast<const uint2*>(x + f * ld)) : make_uint2(0, 0);
    const uint2 b = f + 1 < features ? __ldg(reinterpret_cast<const uint2*>(x + (f + 1) * ld)) : make_uint2(0, 0);
    u[0] = __byte_perm(a.x, b.x, 0x5410);
    u[1] = __byte_perm(a.x, b.x, 0x7632);
    u[2] = __byte_perm(a.y, b.y, 0x5410);
    u[3] = __byte_perm(a.y, b.y, 0x7632);
  }
}
template <class T>
__device__ __forceinline__ void turn_out(T* __restrict__ y, int64_t ld, int f, int features, const uint32_t (&u)[4]) {
  if constexpr (sizeof(T) == 4) {
    if (f < features) *reinterpret_cast<uint4*>(y + f * ld) = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    if (f < features)
      *reinterpret_cast<uint2*>(y + f * ld) = make_uint2(__byte_perm(u[0], u[1], 0x5410), __byte_perm(u[2], u[3], 0x5410));
    if (f + 1 < features)
      *reinterpret_cast<uint2*>(y + (f + 1) * ld) =
          make_uint2(__byte_perm(u[0], u[1], 0x7632), __byte_perm(u[2], u[3], 0x7632));
  }
}

// Tile of x (COLS columns from c0, kTileWords words of features from f0)
// into shared memory; QUADS: the batch allows four columns at once.
template <class T, bool QUADS, int COLS>
__device__ __forceinline__ void load_tile(uint32_t* tile, const T* __restrict__ x, int64_t ld, int f0, int features,
                                          int64_t c0, int64_t batch) {
  constexpr int n = Word<T>::n;
  if (QUADS && c0 + COLS <= batch) {
    constexpr int kPer = kTileWords * (COLS / 4) / kBlock;
    uint32_t u[kPer][4];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int it = i * kBlock + threadIdx.x, q = it % (COLS / 4), w = it / (COLS / 4);
      turn_in<T>(x + c0 + 4 * q, ld, f0 + w * n, features, u[i]);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int it = i * kBlock + threadIdx.x, q = it % (COLS / 4), w = it / (COLS / 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) tile[place(4 * q + k, w)] = u[i][k];
    }
    return;
  }
  constexpr int kPer = kTileWords * COLS / kBlock;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i0 = 0; i0 < kPer; i0 += 8) {
    Word<T> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int it = (i0 + i) * kWarps + warp, c = it % (COLS / 32) * 32 + lane, w = it / (COLS / 32);
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const int f = f0 + w * n + k;
        v[i].v[k] = f < features && c0 + c < batch ? __ldg(x + f * ld + c0 + c) : Num<T>::from_c(0.0f);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int it = (i0 + i) * kWarps + warp, c = it % (COLS / 32) * 32 + lane, w = it / (COLS / 32);
      tile[place(c, w)] = *reinterpret_cast<uint32_t*>(&v[i]);
    }
  }
}

// The four words of a row that lane l of its 16 takes: neighbours where they
// are moved as 16 bytes, 16 apart otherwise.
template <bool VEC>
__device__ __forceinline__ int row_word(int l, int i) {
  return VEC ? 4 * l + i : l + kRowLanes * i;
}
template <class T, bool VEC>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int f0, int features, bool whole, int l, uint32_t (&u)[4]) {
  constexpr int n = Word<T>::n;
  if (VEC && f0 + (4 * l + 4) * n <= features) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + f0 + 4 * l * n));
    u[0] = v.x;
    u[1] = v.y;
    u[2] = v.z;
    u[3] = v.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int f = f0 + row_word<VEC>(l, i) * n;
    u[i] = f < features ? load_word<T>(row, f, features, whole) : 0u;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store_row(T* __restrict__ row, int f0, int features, bool whole, int l, const uint32_t (&u)[4]) {
  constexpr int n = Word<T>::n;
  if (VEC && f0 + (4 * l + 4) * n <= features) {
    *reinterpret_cast<uint4*>(row + f0 + 4 * l * n) = make_uint4(u[0], u[1], u[2], u[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int f = f0 + row_word<VEC>(l, i) * n;
    if (f < features) store_word<T>(row, f, features, whole, u[i]);
  }
}
template <bool VEC>
__device__ __forceinline__ void read_tile(const uint32_t* tile, int c, int l, uint32_t (&u)[4]) {
  if constexpr (VEC) {
    const uint4 v = *reinterpret_cast<const uint4*>(tile + place(c, 4 * l));
    u[0] = v.x;
    u[1] = v.y;
    u[2] = v.z;
    u[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = tile[place(c, row_word<VEC>(l, i))];
  }
}

// Rows that no choice fills: the ones past the last group.
template <class T>
__device__ __forceinline__ void zero_unused(T* __restrict__ rows, int64_t ld, int features, int64_t num_rows,
                                            const int* __restrict__ used, int64_t block, int64_t blocks) {
  const int64_t first = min((int64_t)max(*used, 0), num_rows);
  for (int64_t r = first + block; r < num_rows; r += blocks)
    for (int f = threadIdx.x; f < features; f += kBlock) rows[r * ld + f] = Num<T>::from_c(0.0f);
}

template <class T, bool QUADS, bool VEC>
__global__ void __launch_bounds__(kBlock)
    gather_kernel(const T* __restrict__ x, int64_t ld, int features, int64_t batch, int top_k,
                  const int* __restrict__ row, const int* __restrict__ used, T* __restrict__ rows, int64_t rows_ld,
                  int64_t num_rows, int whole) {
  __shared__ __align__(16) uint32_t tile[kTileCols * kTileWords];
  __shared__ int at[ops::kMaxTopK * kTileCols];
  constexpr int n = Word<T>::n;
  const int l = threadIdx.x % kRowLanes, g = threadIdx.x / kRowLanes;
  const int f0 = blockIdx.y * kTileWords * n;
  const int64_t c0 = blockIdx.x * (int64_t)kTileCols;
  for (int i = threadIdx.x; i < top_k * kTileCols; i += kBlock) {
    const int64_t c = c0 + i % kTileCols;
    const int r = c < batch ? row[i / kTileCols * batch + c] : -1;
    at[i] = r < num_rows ? r : -1;
  }
  load_tile<T, QUADS, kTileCols>(tile, x, ld, f0, features, c0, batch);
  __syncthreads();
#pragma unroll
  for (int c = g; c < kTileCols; c += kBlock / kRowLanes) {
    uint32_t u[4];
    read_tile<VEC>(tile, c, l, u);
    for (int j = 0; j < top_k; ++j) {
      const int r = at[j * kTileCols + c];
      if (r >= 0) store_row<T, VEC>(rows + r * rows_ld, f0, features, whole, l, u);
    }
  }
  if (blockIdx.y == 0) zero_unused<T>(rows, rows_ld, features, num_rows, used, blockIdx.x, gridDim.x);
}

// weight == nullptr: unit weights.
template <class T, bool QUADS, bool VEC>
__global__ void __launch_bounds__(kBlock)
    combine_kernel(const T* __restrict__ rows, int64_t rows_ld, int64_t num_rows, int features, int64_t batch, int top_k,
                   const int* __restrict__ row, const float* __restrict__ weight, T* __restrict__ y, int64_t ld,
                   int whole) {
  __shared__ __align__(16) uint32_t tile[kTileCols * kTileWords];
  __shared__ int at[ops::kMaxTopK * kTileCols];
  __shared__ float wt[ops::kMaxTopK * kTileCols];
  constexpr int n = Word<T>::n;
  constexpr int kGroups = kBlock / kRowLanes, kCols = kTileCols / kGroups;
  const int l = threadIdx.x % kRowLanes, g = threadIdx.x / kRowLanes;
  const int f0 = blockIdx.y * kTileWords * n;
  const int64_t c0 = blockIdx.x * (int64_t)kTileCols;
  for (int i = threadIdx.x; i < top_k * kTileCols; i += kBlock) {
    const int64_t c = c0 + i % kTileCols;
    const int r = c < batch ? row[i / kTileCols * batch + c] : -1;
    at[i] = r < num_rows ? r : -1;
    wt[i] = weight && c < batch ? weight[i / kTileCols * batch + c] : 1.0f;
  }
  __syncthreads();
  float acc[kCols][4][n] = {};
  for (int j = 0; j < top_k; ++j) {
    uint32_t u[kCols][4];
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      const int r = at[j * kTileCols + g + q * kGroups];
      if (r >= 0) load_row<T, VEC>(rows + r * rows_ld, f0, features, whole, l, u[q]);
    }
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      const int i = j * kTileCols + g + q * kGroups;
      if (at[i] >= 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v[n];
          unpack<T>(u[q][k], v);
#pragma unroll
          for (int h = 0; h < n; ++h) acc[q][k][h] = fmaf(wt[i], v[h], acc[q][k][h]);
        }
      }
    }
  }
#pragma unroll
  for (int q = 0; q < kCols; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k) tile[place(g + q * kGroups, row_word<VEC>(l, k))] = pack<T>(acc[q][k]);
  __syncthreads();
  if (QUADS && c0 + kTileCols <= batch) {
#pragma unroll
    for (int i = 0; i < kTileWords * (kTileCols / 4) / kBlock; ++i) {
      const int it = i * kBlock + threadIdx.x, q = it % (kTileCols / 4), w = it / (kTileCols / 4);
      uint32_t u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = tile[place(4 * q + k, w)];
      turn_out<T>(y + c0 + 4 * q, ld, f0 + w * n, features, u);
    }
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 4
  for (int it = warp; it < 2 * kTileWords; it += kWarps) {
    const int c = it % 2 * 32 + lane, w = it / 2;
    if (c0 + c >= batch) continue;
    const uint32_t u = tile[place(c, w)];
    const Word<T> v = *reinterpret_cast<const Word<T>*>(&u);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int f = f0 + w * n + i;
      if (f < features) y[f * ld + c0 + c] = v.v[i];
    }
  }
}

// A block holds its columns through all feature tiles, so that a dot product is
// summed by 16 lanes in a fixed order.  Bound by the latency of the row loads:
// 32 columns a block leave registers for four blocks an SM, and all row loads of
// a tile go out before it is turned (49999 x 1001 fp32, three rows a column: 402 us
// with 64 columns and two blocks, 348 with 32 and four, 280 with the early loads).
template <class T, int K, bool QUADS, bool VEC>
__global__ void __launch_bounds__(kBlock, 4)
    combine_backward_kernel(const T* __restrict__ dy, int64_t ld, const T* __restrict__ rows, int64_t rows_ld,
                            int64_t num_rows, int features, int64_t batch, const int* __restrict__ row,
                            const float* __restrict__ weight, const int* __restrict__ used, T* __restrict__ d_rows,
                            int64_t d_ld, float* __restrict__ d_weight, int whole, int d_whole) {
  __shared__ __align__(16) uint32_t tile[kBackCols * kTileWords];
  __shared__ int at[K * kBackCols];
  __shared__ float wt[K * kBackCols];
  constexpr int n = Word<T>::n, kGroups = kBlock / kRowLanes, kCols = kBackCols / kGroups;
  const int l = threadIdx.x % kRowLanes, g = threadIdx.x / kRowLanes;
  const int64_t c0 = blockIdx.x * (int64_t)kBackCols;
  for (int i = threadIdx.x; i < K * kBackCols; i += kBlock) {
    const int64_t c = c0 + i % kBackCols;
    const int r = c < batch ? row[i / kBackCols * batch + c] : -1;
    at[i] = r < num_rows ? r : -1;
    wt[i] = c < batch ? weight[i / kBackCols * batch + c] : 0.0f;
  }
  __syncthreads();
  float dot[kCols][K] = {};
  for (int f0 = 0; f0 < features; f0 += kTileWords * n) {
    // All row loads go out before the tile's (K <= 4: the registers allow it).
    constexpr bool kAhead = K <= 4;
    uint32_t u[kAhead ? K : 1][kCols][4];
    auto fetch = [&](int j) {
#pragma unroll
      for (int q = 0; q < kCols; ++q) {
        const int r = at[j * kBackCols + g + q * kGroups];
        if (r >= 0) load_row<T, VEC>(rows + r * rows_ld, f0, features, whole, l, u[kAhead ? j : 0][q]);
      }
    };
    if constexpr (kAhead) {
#pragma unroll
      for (int j = 0; j < K; ++j) fetch(j);
    }
    load_tile<T, QUADS, kBackCols>(tile, dy, ld, f0, features, c0, batch);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if constexpr (!kAhead) fetch(j);
#pragma unroll
      for (int q = 0; q < kCols; ++q) {
        const int c = g + q * kGroups, r = at[j * kBackCols + c];
        if (r < 0) continue;
        const float w = wt[j * kBackCols + c];
        uint32_t t[4], out[4];
        read_tile<VEC>(tile, c, l, t);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float d[n], v[n], o[n];
          unpack<T>(t[k], d);
          unpack<T>(u[kAhead ? j : 0][q][k], v);
#pragma unroll
          for (int h = 0; h < n; ++h) {
            dot[q][j] = fmaf(d[h], v[h], dot[q][j]);
            o[h] = w * d[h];
          }
          out[k] = pack<T>(o);
        }
        store_row<T, VEC>(d_rows + r * d_ld, f0, features, d_whole, l, out);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < kCols; ++q) {
    const int c = g + q * kGroups;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      float s = dot[q][j];
#pragma unroll
      for (int d = kRowLanes / 2; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (l == 0 && c0 + c < batch) d_weight[j * batch + c0 + c] = s;
    }
  }
  zero_unused<T>(d_rows, d_ld, features, num_rows, used, blockIdx.x, gridDim.x);
}

ponni_b200_status check_columns(const char* what, int dtype, const void* columns, int64_t ld, int features,
                                int64_t batch, int top_k, const void* row, const void* rows, int64_t rows_ld) {
  using namespace ops;
  const std::string at(what);
  if (!is_real_type(dtype)) return fail(PONNI_B200_ERR_UNSUPPORTED, at + ": values must be fp32, fp16 or bf16");
  if (!columns || !row || !rows || !aligned_to(element_bytes(dtype), columns, rows) || !aligned_to(4, row))
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": pointer is NULL or not aligned to its type");
  if (features < 1) return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": needs at least one feature");
  if (top_k < 1 || top_k > kMaxTopK) return fail(PONNI_B200_ERR_UNSUPPORTED, at + ": top_k must be 1 to 8");
  if (batch < 1 || batch > INT32_MAX / top_k)
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": batch must be nonzero and batch * top_k below 2^31");
  if (ld < batch || rows_ld < features)
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": row stride smaller than the row");
  return PONNI_B200_OK;
}

template <class T> bool whole_words(const void* p, int64_t ld) {
  return sizeof(T) == 4 || (reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld % 2 == 0);
}

bool whole_vectors(const void* p, int64_t ld, size_t z) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * z % 16 == 0;
}
// Four columns at once: 16 bytes of fp32, 8 of the 16-bit types.
bool whole_quads(const void* p, int64_t ld, size_t z) {
  return reinterpret_cast<uintptr_t>(p) % (4 * z) == 0 && ld % 4 == 0;
}

// f(QUADS, VEC) with the two flags as types.
template <class F>
void by_alignment(bool quads, bool vec, F&& f) {
  if (quads) vec ? f(std::true_type(), std::true_type()) : f(std::true_type(), std::false_type());
  else vec ? f(std::false_type(), std::true_type()) : f(std::false_type(), std::false_type());
}

template <class F>
ponni_b200_status by_type(int dtype, F&& f) {
  if (dtype == PONNI_B200_F32) return f(float());
  if (dtype == PONNI_B200_F16) return f(__half());
  return f(__nv_bfloat16());
}

}  // namespace
}  // namespace ponni_b200

using namespace ponni_b200;

extern "C" {

ponni_b200_status ponni_b200_gather_columns(int dtype, const void* x, int64_t ld, int features, int64_t batch, int top_k,
                                            const int32_t* row, const int32_t* num_used, void* rows, int64_t rows_ld,
                                            int device, void* stream) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    ponni_b200_status st = check_columns("gather_columns", dtype, x, ld, features, batch, top_k, row, rows, rows_ld);
    if (st) return st;
    if (!num_used || !ops::aligned_to(4, num_used))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "gather_columns: pointer is NULL or not aligned to its type");
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      const int per = kTileWords * Word<T>::n;
      const dim3 grid((unsigned)((batch + kTileCols - 1) / kTileCols), (unsigned)((features + per - 1) / per));
      if (grid.y > 65535) return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "gather_columns: too many features");
      by_alignment(whole_quads(x, ld, sizeof(T)), whole_vectors(rows, rows_ld, sizeof(T)), [&](auto q, auto v) {
        gather_kernel<T, q.value, v.value><<<grid, kBlock, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(x), ld, features, batch, top_k, row, num_used, static_cast<T*>(rows), rows_ld,
            batch * top_k, whole_words<T>(rows, rows_ld));
      });
      return ops::launched("gather_columns");
    });
  });
}

ponni_b200_status ponni_b200_combine_rows(int dtype, const void* rows, int64_t rows_ld, int features, int64_t batch,
                                          int top_k, const int32_t* row, const float* weight, void* y, int64_t ld,
                                          int device, void* stream) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    ponni_b200_status st = check_columns("combine_rows", dtype, y, ld, features, batch, top_k, row, rows, rows_ld);
    if (st) return st;
    if (!ops::aligned_to(4, weight))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "combine_rows: pointer not aligned to its type");
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      const int per = kTileWords * Word<T>::n;
      const dim3 grid((unsigned)((batch + kTileCols - 1) / kTileCols), (unsigned)((features + per - 1) / per));
      if (grid.y > 65535) return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "combine_rows: too many features");
      by_alignment(whole_quads(y, ld, sizeof(T)), whole_vectors(rows, rows_ld, sizeof(T)), [&](auto q, auto v) {
        combine_kernel<T, q.value, v.value><<<grid, kBlock, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(rows), rows_ld, batch * top_k, features, batch, top_k, row, weight, static_cast<T*>(y),
            ld, whole_words<T>(rows, rows_ld));
      });
      return ops::launched("combine_rows");
    });
  });
}

ponni_b200_status ponni_b200_combine_rows_backward(int dtype, const void* d_y, int64_t ld, const void* rows,
                                                   int64_t rows_ld, int features, int64_t batch, int top_k,
                                                   const int32_t* row, const float* weight, const int32_t* num_used,
                                                   void* d_rows, int64_t d_ld, float* d_weight, int device,
                                                   void* stream) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    ponni_b200_status st =
        check_columns("combine_rows_backward", dtype, d_y, ld, features, batch, top_k, row, rows, rows_ld);
    if (st) return st;
    if (!weight || !num_used || !d_rows || !d_weight || !ops::aligned_to(4, weight, num_used, d_weight) ||
        !ops::aligned_to(ops::element_bytes(dtype), d_rows))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT,
                       "combine_rows_backward: pointer is NULL or not aligned to its type");
    if (d_ld < features)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "combine_rows_backward: row stride smaller than the row");
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      const unsigned grid = (unsigned)((batch + kBackCols - 1) / kBackCols);
      cudaStream_t s = static_cast<cudaStream_t>(stream);
      const bool vec = whole_vectors(rows, rows_ld, sizeof(T)) && whole_vectors(d_rows, d_ld, sizeof(T));
      by_alignment(whole_quads(d_y, ld, sizeof(T)), vec, [&](auto q, auto v) {
        constexpr bool Q = decltype(q)::value, V = decltype(v)::value;
        switch (top_k) {
#define PB_CASE(K)                                                                                                    \
  case K:                                                                                                             \
    combine_backward_kernel<T, K, Q, V><<<grid, kBlock, 0, s>>>(                                                      \
        static_cast<const T*>(d_y), ld, static_cast<const T*>(rows), rows_ld, batch * K, features, batch, row, weight, \
        num_used, static_cast<T*>(d_rows), d_ld, d_weight, whole_words<T>(rows, rows_ld),                              \
        whole_words<T>(d_rows, d_ld));                                                                                 \
    break
          PB_CASE(1);
          PB_CASE(2);
          PB_CASE(3);
          PB_CASE(4);
          PB_CASE(5);
          PB_CASE(6);
          PB_CASE(7);
          PB_CASE(8);
#undef PB_CASE
        }
      });
      return ops::launched("combine_rows_backward");
    });
  });
}

}  // extern "C"
