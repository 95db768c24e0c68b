// Products grouped by expert: rows r in [offset[e], offset[e+1]) times
// weights[e] (in x out, row-major), and the gradients.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "device_math.cuh"
#include "operators.h"

namespace ponni_b200 {
namespace {

constexpr int kTile = 64, kStep = 16, kBlock = 256;

// The groups as the kernels read them: kept within [0, rows] and ascending
// whatever the offsets hold; a violation is recorded.
__device__ __forceinline__ void group_of(const int* __restrict__ offset, int experts, int e, int64_t rows, int64_t& lo,
                                         int64_t& hi) {
  lo = min(max((int64_t)offset[e], (int64_t)0), rows);
  hi = min(max((int64_t)offset[e + 1], lo), rows);
}

// The first block's check of the offsets (the groups are clamped whatever they hold).
__device__ __forceinline__ void check_offsets(const int* __restrict__ offset, int experts, int64_t rows, int* error) {
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) {
    const int64_t o = offset[e], before = e ? offset[e - 1] : 0;
    if (o < before || o > rows || (e == 0 && o != 0)) atomicOr(error, 2);
  }
}

enum Mode { kForward, kRows, kWeights };

struct Args {
  const void* a;  // kForward: rows; kRows: d_out; kWeights: rows
  const void* b;  // kForward, kRows: weights; kWeights: d_out
  void* c;
  int64_t a_ld, b_ld, b_stride, c_ld;
  int64_t rows;
  const int* offset;
  const void* bias;
  int experts, inputs, outputs;
  int act, act_flags;
  float s0, s1;
  int* error;
};

template <class T, int MODE>
__global__ void __launch_bounds__(kBlock) simple_kernel(const Args p) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const T* a = static_cast<const T*>(p.a);
  const T* b = static_cast<const T*>(p.b);
  T* c = static_cast<T*>(p.c);
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_offsets(p.offset, p.experts, p.rows, p.error);
  int e = 0;
  int64_t lo = 0, hi = 0, m0 = 0;
  int m_end, n_end, k_end;
  if (MODE == kWeights) {
    e = blockIdx.z;
    group_of(p.offset, p.experts, e, p.rows, lo, hi);
    m0 = (int64_t)blockIdx.x * kTile;
    m_end = p.inputs;
    n_end = p.outputs;
    k_end = (int)(hi - lo);
  } else {
    int64_t t = blockIdx.x;  // tile of rows: the experts' tiles, then the rows in no group
    for (; e < p.experts; ++e) {
      group_of(p.offset, p.experts, e, p.rows, lo, hi);
      const int64_t tiles = (hi - lo + kTile - 1) / kTile;
      if (t < tiles) break;
      t -= tiles;
    }
    n_end = MODE == kForward ? p.outputs : p.inputs;
    k_end = MODE == kForward ? p.inputs : p.outputs;
    if (e == p.experts) {
      lo = min(max((int64_t)p.offset[p.experts], (int64_t)0), p.rows);
      hi = p.rows;
      k_end = 0;
    }
    m0 = t * kTile;
    if (m0 >= hi - lo) return;
    m_end = (int)(hi - lo);
  }
  const int n0 = blockIdx.y * kTile;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < k_end; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep; i += kBlock) {
      {
        const int m = MODE == kWeights ? i % kTile : i / kStep, k = MODE == kWeights ? i / kTile : i % kStep;
        float v = 0.0f;
        if (m0 + m < m_end && k0 + k < k_end)
          v = Num<T>::to_c(MODE == kWeights ? a[(lo + k0 + k) * p.a_ld + m0 + m] : a[(lo + m0 + m) * p.a_ld + k0 + k]);
        sa[k][m] = v;
      }
      {
        const int n = MODE == kRows ? i / kStep : i % kTile, k = MODE == kRows ? i % kStep : i / kTile;
        float v = 0.0f;
        if (n0 + n < n_end && k0 + k < k_end) {
          if (MODE == kForward) v = Num<T>::to_c(b[e * p.b_stride + (int64_t)(k0 + k) * p.b_ld + n0 + n]);
          if (MODE == kRows) v = Num<T>::to_c(b[e * p.b_stride + (int64_t)(n0 + n) * p.b_ld + k0 + k]);
          if (MODE == kWeights) v = Num<T>::to_c(b[(lo + k0 + k) * p.b_ld + n0 + n]);
        }
        sb[k][n] = v;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i;
      const int n = n0 + tx + 16 * j;
      if (m >= m_end || n >= n_end) continue;
      float v = acc[i][j];
      if (MODE == kForward && e < p.experts) {
        if (p.bias) v += Num<T>::to_c(static_cast<const T*>(p.bias)[(int64_t)e * p.outputs + n]);
        v = activation<float>(p.act, p.act_flags, v, p.s0, p.s1);
      }
      if (MODE == kWeights) c[((int64_t)e * p.inputs + m) * p.outputs + n] = Num<T>::from_c(v);
      else c[(lo + m) * p.c_ld + n] = Num<T>::from_c(v);
    }
}

// Column sums of an expert's rows.
template <class T>
__global__ void __launch_bounds__(kBlock)
    simple_bias_kernel(const T* __restrict__ d, int64_t ld, int64_t rows, const int* __restrict__ offset, int experts,
                       int outputs, T* __restrict__ out) {
  __shared__ float part[kBlock / 32][32];
  const int e = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.x * 32 + lane;
  int64_t lo, hi;
  group_of(offset, experts, e, rows, lo, hi);
  float s = 0.0f;
  if (n < outputs)
    for (int64_t r = lo + warp; r < hi; r += kBlock / 32) s += Num<T>::to_c(d[r * ld + n]);
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && n < outputs) {
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < kBlock / 32; ++w) t += part[w][lane];
    out[(int64_t)e * outputs + n] = Num<T>::from_c(t);
  }
}

template <class T>
ponni_b200_status launch_simple(int mode, const Args& p, cudaStream_t s) {
  const int64_t row_tiles = (p.rows + kTile - 1) / kTile + p.experts + 1;
  auto tiles = [](int n) { return (unsigned)((n + kTile - 1) / kTile); };
  if (tiles(p.inputs) > 65535 || tiles(p.outputs) > 65535)
    return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "expert_product: too many inputs or outputs");
  if (mode == kForward)
    simple_kernel<T, kForward><<<dim3((unsigned)row_tiles, tiles(p.outputs)), kBlock, 0, s>>>(p);
  else if (mode == kRows)
    simple_kernel<T, kRows><<<dim3((unsigned)row_tiles, tiles(p.inputs)), kBlock, 0, s>>>(p);
  else
    simple_kernel<T, kWeights><<<dim3(tiles(p.inputs), tiles(p.outputs), p.experts), kBlock, 0, s>>>(p);
  return ops::launched("expert_product");
}

template <class F>
ponni_b200_status by_type(int dtype, F&& f) {
  if (dtype == PONNI_B200_F32) return f(float());
  if (dtype == PONNI_B200_F16) return f(__half());
  return f(__nv_bfloat16());
}

ponni_b200_status check_product(const std::string& at, int dtype, const void* rows, int64_t rows_ld, int64_t num_rows,
                                const void* weights, int64_t w_ld, int64_t w_stride, const void* offset, int experts,
                                int inputs, int outputs) {
  using namespace ops;
  if (!is_real_type(dtype)) return fail(PONNI_B200_ERR_UNSUPPORTED, at + ": values must be fp32, fp16 or bf16");
  if (experts < 1 || experts > kMaxExperts)
    return fail(PONNI_B200_ERR_UNSUPPORTED, at + ": the number of experts must be 1 to 1024");
  if (inputs < 1 || outputs < 1) return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": needs inputs and outputs");
  if (num_rows < 0 || num_rows > INT32_MAX)
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": the number of rows must be below 2^31");
  if ((num_rows > 0 && !rows) || !weights || !offset)
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": pointer is NULL");
  if (rows_ld < inputs || w_ld < outputs || (experts > 1 && w_stride < (int64_t)inputs * w_ld - (w_ld - outputs)))
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": stride smaller than the row or the expert");
  return PONNI_B200_OK;
}

}  // namespace
}  // namespace ponni_b200

using namespace ponni_b200;

extern "C" {

int64_t ponni_b200_expert_product_workspace(int dtype, int64_t num_rows, int experts, int inputs, int outputs,
                                            int backward) {
  (void)dtype; (void)num_rows; (void)experts; (void)inputs; (void)outputs; (void)backward;
  return 0;
}

ponni_b200_status ponni_b200_expert_product(int dtype, const void* rows, int64_t rows_ld, int64_t num_rows,
                                            const void* weights, int64_t w_ld, int64_t w_stride, const void* bias,
                                            const int32_t* offset, int experts, int inputs, int outputs, int activation,
                                            int activation_flags, double scalar0, double scalar1, void* out,
                                            int64_t out_ld, void* workspace, int64_t workspace_bytes, int device,
                                            void* stream) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    ponni_b200_status st = check_product("expert_product", dtype, rows, rows_ld, num_rows, weights, w_ld, w_stride,
                                         offset, experts, inputs, outputs);
    if (st) return st;
    if (activation != -1 && (!is_pointwise(activation) || activation == PONNI_B200_BIAS))
      return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "expert_product: the activation must be an activation layer kind");
    if (num_rows == 0) return PONNI_B200_OK;
    if (!out) return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product: pointer is NULL");
    if (out_ld < outputs)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product: stride smaller than the row");
    Args p = {rows, weights, out, rows_ld, w_ld, w_stride, out_ld, num_rows, offset, bias, experts, inputs, outputs,
              activation < 0 ? EPI_NONE : activation, activation_flags, (float)scalar0, (float)scalar1, ops::error_word(device)};
    if (!p.error) return ops::fail(PONNI_B200_ERR_CUDA, "no operator error word on this device");
    return by_type(dtype, [&](auto t) { return launch_simple<decltype(t)>(kForward, p, static_cast<cudaStream_t>(stream)); });
  });
}

ponni_b200_status ponni_b200_expert_product_backward(int dtype, const void* d_out, int64_t d_out_ld, const void* rows,
                                                     int64_t rows_ld, int64_t num_rows, const void* weights,
                                                     int64_t w_ld, int64_t w_stride, const int32_t* offset, int experts,
                                                     int inputs, int outputs, void* d_rows, int64_t d_rows_ld,
                                                     void* d_weights, void* d_bias, void* workspace,
                                                     int64_t workspace_bytes, int device, void* stream) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    ponni_b200_status st = check_product("expert_product_backward", dtype, rows, rows_ld, num_rows, weights, w_ld,
                                         w_stride, offset, experts, inputs, outputs);
    if (st) return st;
    if (num_rows > 0 && !d_out)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product_backward: pointer is NULL");
    if (d_out_ld < outputs || (d_rows && d_rows_ld < inputs))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product_backward: stride smaller than the row");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      Args p = {d_out, weights, d_rows, d_out_ld, w_ld, w_stride, d_rows_ld, num_rows, offset, nullptr, experts, inputs,
                outputs, EPI_NONE, 0, 0.0f, 0.0f, ops::error_word(device)};
      if (!p.error) return ops::fail(PONNI_B200_ERR_CUDA, "no operator error word on this device");
      ponni_b200_status r = PONNI_B200_OK;
      if (d_rows && num_rows > 0) r = launch_simple<T>(kRows, p, s);
      if (!r && d_weights) {
        p.a = rows;
        p.a_ld = rows_ld;
        p.b = d_out;
        p.b_ld = d_out_ld;
        p.c = d_weights;
        r = launch_simple<T>(kWeights, p, s);
      }
      if (!r && d_bias) {
        simple_bias_kernel<T><<<dim3((outputs + 31) / 32, experts), kBlock, 0, s>>>(
            static_cast<const T*>(d_out), d_out_ld, num_rows, offset, experts, outputs, static_cast<T*>(d_bias));
        r = ops::launched("expert_product_backward");
      }
      return r;
    });
  });
}

}  // extern "C"
