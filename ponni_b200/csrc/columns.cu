// Columns to expert-sorted rows and back.
//
// x[f][b] is feature-major (batch contiguous), rows[r][f] has the features of
// a row contiguous; row[j][b] is the row of column b's choice j (negative:
// none).  gather: rows[row[j][b]][.] = x[.][b].  combine: y[.][b] = sum_j
// weight[j][b] rows[row[j][b]][.] in fp32, rounded once.  Their gradients are a
// combination with unit weights, and (fused) d_rows = weight d_y with
// d_weight[j][b] = <rows[row[j][b]], d_y[.][b]>.
//
// All are transposes bound by HBM: a block turns a tile of 64 columns in
// shared memory, in 4-byte words (one fp32 or two 16-bit features) with an odd
// pitch, so that both the column side (lanes along the batch) and the row
// side (lanes along the features) are free of bank conflicts.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "device_math.cuh"
#include "operators.h"

namespace ponni_b200 {
namespace {

constexpr int kBlock = 256;
constexpr int kWarps = kBlock / 32;
constexpr int kTileCols = 64;
constexpr int kTileWords = 64;
constexpr int kPitch = kTileWords + 1;

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

// Tile of x (kTileCols columns from c0, kTileWords words of features from f0)
// into shared memory [column][word].
template <class T>
__device__ __forceinline__ void load_tile(uint32_t* tile, const T* __restrict__ x, int64_t ld, int f0, int features,
                                          int64_t c0, int64_t batch) {
  constexpr int n = Word<T>::n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 4
  for (int w = warp; w < kTileWords; w += kWarps) {
#pragma unroll
    for (int h = 0; h < kTileCols / 32; ++h) {
      const int c = h * 32 + lane;
      Word<T> v;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const int f = f0 + w * n + i;
        v.v[i] = f < features && c0 + c < batch ? x[f * ld + c0 + c] : Num<T>::from_c(0.0f);
      }
      tile[c * kPitch + w] = *reinterpret_cast<uint32_t*>(&v);
    }
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

template <class T>
__global__ void __launch_bounds__(kBlock)
    gather_kernel(const T* __restrict__ x, int64_t ld, int features, int64_t batch, int top_k,
                  const int* __restrict__ row, const int* __restrict__ used, T* __restrict__ rows, int64_t rows_ld,
                  int64_t num_rows, int whole) {
  __shared__ uint32_t tile[kTileCols * kPitch];
  constexpr int n = Word<T>::n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int f0 = blockIdx.y * kTileWords * n;
  const int64_t c0 = blockIdx.x * (int64_t)kTileCols;
  load_tile<T>(tile, x, ld, f0, features, c0, batch);
  __syncthreads();
  for (int c = warp; c < kTileCols && c0 + c < batch; c += kWarps) {
    for (int j = 0; j < top_k; ++j) {
      const int r = row[j * batch + c0 + c];
      if (r < 0 || r >= num_rows) continue;
#pragma unroll
      for (int w = lane; w < kTileWords; w += 32)
        if (f0 + w * n < features) store_word<T>(rows + r * rows_ld, f0 + w * n, features, whole, tile[c * kPitch + w]);
    }
  }
  if (blockIdx.y == 0) zero_unused<T>(rows, rows_ld, features, num_rows, used, blockIdx.x, gridDim.x);
}

// weight == nullptr: unit weights.
template <class T>
__global__ void __launch_bounds__(kBlock)
    combine_kernel(const T* __restrict__ rows, int64_t rows_ld, int64_t num_rows, int features, int64_t batch, int top_k,
                   const int* __restrict__ row, const float* __restrict__ weight, T* __restrict__ y, int64_t ld,
                   int whole) {
  __shared__ uint32_t tile[kTileCols * kPitch];
  constexpr int n = Word<T>::n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int f0 = blockIdx.y * kTileWords * n;
  const int64_t c0 = blockIdx.x * (int64_t)kTileCols;
  for (int c = warp; c < kTileCols && c0 + c < batch; c += kWarps) {
    float acc[kTileWords / 32][n] = {};
    for (int j = 0; j < top_k; ++j) {
      const int r = row[j * batch + c0 + c];
      if (r < 0 || r >= num_rows) continue;
      const float wt = weight ? weight[j * batch + c0 + c] : 1.0f;
#pragma unroll
      for (int h = 0; h < kTileWords / 32; ++h) {
        const int f = f0 + (h * 32 + lane) * n;
        if (f < features) {
          float v[n];
          unpack<T>(load_word<T>(rows + r * rows_ld, f, features, whole), v);
#pragma unroll
          for (int i = 0; i < n; ++i) acc[h][i] = fmaf(wt, v[i], acc[h][i]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kTileWords / 32; ++h) tile[c * kPitch + h * 32 + lane] = pack<T>(acc[h]);
  }
  __syncthreads();
#pragma unroll 4
  for (int w = warp; w < kTileWords; w += kWarps) {
#pragma unroll
    for (int h = 0; h < kTileCols / 32; ++h) {
      const int c = h * 32 + lane;
      if (c0 + c >= batch) continue;
      const uint32_t u = tile[c * kPitch + w];
      const Word<T> v = *reinterpret_cast<const Word<T>*>(&u);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const int f = f0 + w * n + i;
        if (f < features) y[f * ld + c0 + c] = v.v[i];
      }
    }
  }
}

// A block holds its 64 columns through all feature tiles, so that a dot
// product is summed by one warp in a fixed order.
template <class T, int K>
__global__ void __launch_bounds__(kBlock)
    combine_backward_kernel(const T* __restrict__ dy, int64_t ld, const T* __restrict__ rows, int64_t rows_ld,
                            int64_t num_rows, int features, int64_t batch, const int* __restrict__ row,
                            const float* __restrict__ weight, const int* __restrict__ used, T* __restrict__ d_rows,
                            int64_t d_ld, float* __restrict__ d_weight, int whole, int d_whole) {
  __shared__ uint32_t tile[kTileCols * kPitch];
  constexpr int n = Word<T>::n, kCols = kTileCols / kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c0 = blockIdx.x * (int64_t)kTileCols;
  float dot[kCols][K] = {};
  for (int f0 = 0; f0 < features; f0 += kTileWords * n) {
    load_tile<T>(tile, dy, ld, f0, features, c0, batch);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      const int c = warp + q * kWarps;
      if (c0 + c < batch) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const int r = row[j * batch + c0 + c];
          if (r < 0 || r >= num_rows) continue;
          const float wt = weight[j * batch + c0 + c];
#pragma unroll
          for (int h = 0; h < kTileWords / 32; ++h) {
            const int f = f0 + (h * 32 + lane) * n;
            if (f < features) {
              float d[n], v[n], o[n];
              unpack<T>(tile[c * kPitch + h * 32 + lane], d);
              unpack<T>(load_word<T>(rows + r * rows_ld, f, features, whole), v);
#pragma unroll
              for (int i = 0; i < n; ++i) {
                dot[q][j] = fmaf(d[i], v[i], dot[q][j]);
                o[i] = wt * d[i];
              }
              store_word<T>(d_rows + r * d_ld, f, features, d_whole, pack<T>(o));
            }
          }
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < kCols; ++q) {
    const int c = warp + q * kWarps;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      float s = dot[q][j];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (lane == 0 && c0 + c < batch) d_weight[j * batch + c0 + c] = s;
    }
  }
  zero_unused<T>(d_rows, d_ld, features, num_rows, used, blockIdx.x, gridDim.x);
}

ponni_b200_status check_columns(const char* what, int dtype, const void* columns, int64_t ld, int features,
                                int64_t batch, int top_k, const void* row, const void* rows, int64_t rows_ld) {
  using namespace ops;
  const std::string at(what);
  if (!is_real_type(dtype)) return fail(PONNI_B200_ERR_UNSUPPORTED, at + ": values must be fp32, fp16 or bf16");
  if (!columns || !row || !rows) return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": pointer is NULL");
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
    if (!num_used) return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "gather_columns: pointer is NULL");
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      const int per = kTileWords * Word<T>::n;
      const dim3 grid((unsigned)((batch + kTileCols - 1) / kTileCols), (unsigned)((features + per - 1) / per));
      if (grid.y > 65535) return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "gather_columns: too many features");
      gather_kernel<T><<<grid, kBlock, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(x), ld, features, batch, top_k, row, num_used, static_cast<T*>(rows), rows_ld,
          batch * top_k, whole_words<T>(rows, rows_ld));
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
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      const int per = kTileWords * Word<T>::n;
      const dim3 grid((unsigned)((batch + kTileCols - 1) / kTileCols), (unsigned)((features + per - 1) / per));
      if (grid.y > 65535) return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "combine_rows: too many features");
      combine_kernel<T><<<grid, kBlock, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(rows), rows_ld, batch * top_k, features, batch, top_k, row, weight, static_cast<T*>(y),
          ld, whole_words<T>(rows, rows_ld));
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
    if (!weight || !num_used || !d_rows || !d_weight)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "combine_rows_backward: pointer is NULL");
    if (d_ld < features)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "combine_rows_backward: row stride smaller than the row");
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      const unsigned grid = (unsigned)((batch + kTileCols - 1) / kTileCols);
      cudaStream_t s = static_cast<cudaStream_t>(stream);
      switch (top_k) {
#define PB_CASE(K)                                                                                                   \
  case K:                                                                                                            \
    combine_backward_kernel<T, K><<<grid, kBlock, 0, s>>>(                                                         \
        static_cast<const T*>(d_y), ld, static_cast<const T*>(rows), rows_ld, batch * K, features, batch, row, weight, \
        num_used, static_cast<T*>(d_rows), d_ld, d_weight, whole_words<T>(rows, rows_ld),                             \
        whole_words<T>(d_rows, d_ld));                                                                                \
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
      return ops::launched("combine_rows_backward");
    });
  });
}

}  // extern "C"
