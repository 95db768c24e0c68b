// Norm over many gradient tensors together, and clipping.
//
// norm = sqrt(sum over all tensors of g^2).  Where it is finite and above
// max_norm every g becomes g max_norm / norm, in place or packed into one flat
// vector in tensor order; otherwise the gradients stay as they are (packed:
// are copied).
//
// Bound by HBM: one read for the norm, one read and one write for the scaling
// (the read comes from L2 where the set fits it: the second pass goes through
// the chunks in reverse).  The tensors are cut into chunks once, when the set
// is made; a block sums its chunks in a fixed order and the partial sums are
// added in a fixed order, so the norm does not change from run to run.  Measured:
// 150 M values in 200 tensors, bf16 and fp32, 64 us for the norm (450 MB, 7.0 TB/s)
// and 188 us to pack them into fp32 (1.05 GB, 5.6 TB/s).
// Squares are summed in fp32 over one vector and in fp64 from there: a sum of
// 2^30 squares keeps fp32's full precision, and the fp32 part is redone in
// fp64 where it over- or underflows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <new>
#include <type_traits>
#include <utility>
#include <vector>

#include "device_math.cuh"
#include "operators.h"

struct ponni_b200_gradient_set {
  // A tensor's addresses, type and place in the packed vector.
  struct Extent {
    uintptr_t begin, end, reach;  // reach: the largest end up to here
    int64_t flat;
    int32_t dtype;
  };
  int device = 0;
  int64_t total = 0;
  int64_t num_chunks = 0;
  void* chunks = nullptr;       // device table
  std::vector<Extent> extents;  // by address
  bool overlap = false;         // two of them share elements
};

namespace ponni_b200 {
namespace {

constexpr int kBlock = 512;
constexpr int kMaxBlocks = 148 * 4;

struct Chunk {
  void* p;
  int64_t flat;   // element offset in the packed vector
  int32_t count;
  int32_t dtype;
};

// Vectors of 16 bytes.
template <class T> struct Vec {
  static constexpr int n = 16 / sizeof(T);
  T v[n];
};

__device__ __forceinline__ double square64(float x) { return (double)x * (double)x; }

template <class T>
__device__ __forceinline__ double squares(const T* __restrict__ p, int count) {
  using C = typename Num<T>::C;
  constexpr int n = Vec<T>::n;
  double s = 0.0;
  int done = 0;
  if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    const int vecs = count / n;
    const uint4* q = reinterpret_cast<const uint4*>(p);
    auto add = [&](const uint4& raw) {
      const Vec<T> v = *reinterpret_cast<const Vec<T>*>(&raw);
      if constexpr (sizeof(C) == 8) {
#pragma unroll
        for (int k = 0; k < n; ++k) s = fma((double)Num<T>::to_c(v.v[k]), (double)Num<T>::to_c(v.v[k]), s);
      } else {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < n; ++k) t = fmaf(Num<T>::to_c(v.v[k]), Num<T>::to_c(v.v[k]), t);
        if (t > 1e-30f && t < 1e38f) {
          s += t;
        } else {
#pragma unroll
          for (int k = 0; k < n; ++k) s += square64(Num<T>::to_c(v.v[k]));
        }
      }
    };
    int i = threadIdx.x;
    for (; i + 3 * kBlock < vecs; i += 4 * kBlock) {
      uint4 raw[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) raw[k] = __ldg(q + i + k * kBlock);
#pragma unroll
      for (int k = 0; k < 4; ++k) add(raw[k]);
    }
    for (; i < vecs; i += kBlock) add(__ldg(q + i));
    done = vecs * n;
  }
  for (int i = done + threadIdx.x; i < count; i += kBlock) {
    const double x = (double)Num<T>::to_c(p[i]);
    s = fma(x, x, s);
  }
  return s;
}

// Sum over the block, the same in every thread.
__device__ __forceinline__ double block_sum(double v, double* sums) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < kBlock / 32; ++i) t += sums[i];
  return t;
}

// This thread's part of the squares of the block's chunks.
__device__ __forceinline__ double chunk_squares(const Chunk* __restrict__ chunks, int64_t num_chunks) {
  double s = 0.0;
  for (int64_t i = blockIdx.x; i < num_chunks; i += gridDim.x) {
    const Chunk c = chunks[i];
    switch (c.dtype) {
      case PONNI_B200_F32: s += squares(static_cast<const float*>(c.p), c.count); break;
      case PONNI_B200_F64: s += squares(static_cast<const double*>(c.p), c.count); break;
      case PONNI_B200_F16: s += squares(static_cast<const __half*>(c.p), c.count); break;
      default: s += squares(static_cast<const __nv_bfloat16*>(c.p), c.count); break;
    }
  }
  return s;
}

__global__ void __launch_bounds__(kBlock)
    norm_kernel(const Chunk* __restrict__ chunks, int64_t num_chunks, double* __restrict__ partial) {
  __shared__ double sums[kBlock / 32];
  ops::let_successor_start();
  const double t = block_sum(chunk_squares(chunks, num_chunks), sums);
  if (threadIdx.x == 0) partial[blockIdx.x] = t;
}

// The factor, and as two of fp32: one far below 1 (a norm of 1e38 and more) would lose its
// precision below fp32's normal range or be zero, so 2^100 of it are taken off and put
// back behind the first product, which stays in range.
struct Scale {
  double exact;
  float first, second;
  __device__ explicit Scale(double s) : exact(s), first((float)s), second(1.0f) {
    if (s < 0x1p-100) {
      first = (float)(s * 0x1p100);
      second = 0x1p-100f;
    }
  }
};

template <class T, class O>
__device__ __forceinline__ O scaled(T x, const Scale& scale) {
  if constexpr (sizeof(T) == 8) return (O)Num<O>::from_c((typename Num<O>::C)((double)x * scale.exact));
  else if constexpr (sizeof(O) == 8) return (double)Num<T>::to_c(x) * scale.exact;
  else return Num<O>::from_c(Num<T>::to_c(x) * scale.first * scale.second);
}

template <class T, class O>
__device__ __forceinline__ void rescale(const T* p, O* out, int count, const Scale& scale) {
  constexpr int n = Vec<T>::n;
  int done = 0;
  if (sizeof(T) == sizeof(O) && reinterpret_cast<uintptr_t>(p) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
    const int vecs = count / n;
    const uint4* q = reinterpret_cast<const uint4*>(p);
    auto put = [&](const uint4& raw, int i) {
      const Vec<T> v = *reinterpret_cast<const Vec<T>*>(&raw);
      Vec<O> o;
#pragma unroll
      for (int k = 0; k < n; ++k) o.v[k] = scaled<T, O>(v.v[k], scale);
      reinterpret_cast<uint4*>(out)[i] = *reinterpret_cast<uint4*>(&o);
    };
    int i = threadIdx.x;
    for (; i + 3 * kBlock < vecs; i += 4 * kBlock) {
      uint4 raw[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) raw[k] = q[i + k * kBlock];
#pragma unroll
      for (int k = 0; k < 4; ++k) put(raw[k], i + k * kBlock);
    }
    for (; i < vecs; i += kBlock) put(q[i], i);
    done = vecs * n;
  }
  // Element by element (a packed vector leaves the tensors off the 16-byte
  // grid): coalesced on both sides, a batch of loads ahead of its stores.
  int i = done + threadIdx.x;
  auto batch = [&](auto size) {
    constexpr int B = decltype(size)::value;
    for (; i + (B - 1) * kBlock < count; i += B * kBlock) {
      T v[B];
#pragma unroll
      for (int k = 0; k < B; ++k) v[k] = p[i + k * kBlock];
#pragma unroll
      for (int k = 0; k < B; ++k) out[i + k * kBlock] = scaled<T, O>(v[k], scale);
    }
  };
  batch(std::integral_constant<int, 16>());
  batch(std::integral_constant<int, 4>());
  batch(std::integral_constant<int, 1>());
}

// flat_dtype < 0: in place.
template <class T>
__device__ __forceinline__ void rescale_to(const Chunk& c, void* flat, int flat_dtype, const Scale& scale) {
  const T* p = static_cast<const T*>(c.p);
  switch (flat_dtype) {
    case PONNI_B200_F32: rescale(p, static_cast<float*>(flat) + c.flat, c.count, scale); break;
    case PONNI_B200_F64: rescale(p, static_cast<double*>(flat) + c.flat, c.count, scale); break;
    case PONNI_B200_F16: rescale(p, static_cast<__half*>(flat) + c.flat, c.count, scale); break;
    case PONNI_B200_BF16: rescale(p, static_cast<__nv_bfloat16*>(flat) + c.flat, c.count, scale); break;
    default: rescale(p, static_cast<T*>(c.p), c.count, scale); break;
  }
}

// Scales (or packs) the block's chunks, the last ones first, by the norm over all.
__device__ __forceinline__ void clip_chunks(const Chunk* __restrict__ chunks, int64_t num_chunks, double norm,
                                            double max_norm, void* flat, int flat_dtype) {
  const bool clip = norm > max_norm && norm < (double)INFINITY;
  if (!clip && flat_dtype < 0) return;
  const Scale scale(clip ? max_norm / norm : 1.0);
  for (int64_t i = num_chunks - 1 - blockIdx.x; i >= 0; i -= gridDim.x) {
    const Chunk c = chunks[i];
    switch (c.dtype) {
      case PONNI_B200_F32: rescale_to<float>(c, flat, flat_dtype, scale); break;
      case PONNI_B200_F64: rescale_to<double>(c, flat, flat_dtype, scale); break;
      case PONNI_B200_F16: rescale_to<__half>(c, flat, flat_dtype, scale); break;
      default: rescale_to<__nv_bfloat16>(c, flat, flat_dtype, scale); break;
    }
  }
}

__global__ void __launch_bounds__(kBlock)
    clip_kernel(const Chunk* __restrict__ chunks, int64_t num_chunks, const double* __restrict__ partial,
                int num_partial, double max_norm, void* flat, int flat_dtype, float* __restrict__ norm_out) {
  __shared__ double sums[kBlock / 32];
  ops::let_successor_start();
  ops::wait_for_predecessor();
  double s = 0.0;
  for (int i = threadIdx.x; i < num_partial; i += kBlock) s += partial[i];
  const double norm = sqrt(block_sum(s, sums));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  clip_chunks(chunks, num_chunks, norm, max_norm, flat, flat_dtype);
}

// Both passes in one launch, by one cluster whose blocks read one another's
// sums: for sets of at most kOneClusterChunks chunks, where the second launch
// costs more than the work.
constexpr int kCluster = 8, kOneClusterChunks = 4 * kCluster;
__global__ void __launch_bounds__(kBlock)
    clip_one_cluster_kernel(const Chunk* __restrict__ chunks, int64_t num_chunks, double max_norm,
                            void* flat, int flat_dtype, float* __restrict__ norm_out) {
  __shared__ double sums[kBlock / 32];
  __shared__ double mine;
  const double t = block_sum(chunk_squares(chunks, num_chunks), sums);
  if (threadIdx.x == 0) mine = t;
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;\n" ::: "memory");
  double s = 0.0;
  for (int q = 0; q < (int)gridDim.x; ++q) {
    uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(&mine)), r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(q));
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];\n" : "=d"(v) : "r"(r) : "memory");
    s += v;
  }
  const double norm = sqrt(s);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  clip_chunks(chunks, num_chunks, norm, max_norm, flat, flat_dtype);
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;\n" ::: "memory");
}

// Whether the packed vector shares no element with a tensor, or the tensor lies in it just
// where its packed values go (gradients that are views of one vector): a thread then
// writes what it has read.
bool packs_apart(const ponni_b200_gradient_set& set, const void* flat, int flat_dtype) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(flat), z = ops::element_bytes(flat_dtype), hi = lo + set.total * z;
  auto at = std::partition_point(set.extents.begin(), set.extents.end(), [&](const auto& x) { return x.reach <= lo; });
  for (; at != set.extents.end() && at->begin < hi; ++at)
    if (at->end > lo && (at->dtype != flat_dtype || at->begin != lo + at->flat * z)) return false;
  return true;
}

}  // namespace
}  // namespace ponni_b200

using namespace ponni_b200;

extern "C" {

ponni_b200_status ponni_b200_gradient_set_create(const void* const* tensors, const int64_t* counts,
                                                 const int32_t* dtypes, int num_tensors, int device,
                                                 ponni_b200_gradient_set** out) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    if (!out) return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "gradient set: output pointer is NULL");
    *out = nullptr;
    if (num_tensors < 1 || !tensors || !counts || !dtypes)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "gradient set: needs at least one tensor");
    int64_t total = 0;
    for (int i = 0; i < num_tensors; ++i) {
      if (counts[i] < 0 || counts[i] > ((int64_t)1 << 40) || (counts[i] > 0 && !tensors[i]))
        return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "gradient set: bad pointer or size of a tensor");
      if (dtypes[i] < PONNI_B200_F32 || dtypes[i] > PONNI_B200_BF16)
        return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "gradient set: tensors must be fp32, fp64, fp16 or bf16");
      if (reinterpret_cast<uintptr_t>(tensors[i]) % ops::element_bytes(dtypes[i]) != 0)
        return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "gradient set: a tensor is not aligned to its type");
      total += counts[i];
    }
    // About eight chunks a block, 2048 to 16384 elements each.
    const int64_t per = std::min<int64_t>(16384, std::max<int64_t>(2048, total / (kMaxBlocks * 8) / 512 * 512));
    std::vector<Chunk> table;
    std::vector<ponni_b200_gradient_set::Extent> extents;
    int64_t flat = 0;
    for (int i = 0; i < num_tensors; ++i) {
      const int64_t z = ops::element_bytes(dtypes[i]);
      for (int64_t at = 0; at < counts[i]; at += per)
        table.push_back({static_cast<char*>(const_cast<void*>(tensors[i])) + at * z, flat + at,
                         (int32_t)std::min(per, counts[i] - at), dtypes[i]});
      const uintptr_t begin = reinterpret_cast<uintptr_t>(tensors[i]);
      if (counts[i]) extents.push_back({begin, begin + (uintptr_t)(counts[i] * z), 0, flat, dtypes[i]});
      flat += counts[i];
    }
    std::sort(extents.begin(), extents.end(), [](const auto& a, const auto& b) { return a.begin < b.begin; });
    bool overlap = false;
    uintptr_t reach = 0;
    for (auto& x : extents) {
      overlap |= x.begin < reach;
      x.reach = reach = std::max(reach, x.end);
    }
    ponni_b200_gradient_set* set = new (std::nothrow) ponni_b200_gradient_set;
    if (!set) return ops::fail(PONNI_B200_ERR_CUDA, "gradient set: out of host memory");
    set->device = device;
    set->total = total;
    set->num_chunks = (int64_t)table.size();
    set->extents = std::move(extents);
    set->overlap = overlap;
    if (!table.empty()) {
      cudaError_t e = cudaMalloc(&set->chunks, table.size() * sizeof(Chunk));
      // (A plain copy from pageable memory returns once the table is staged, and a stream that
      // does not wait for the default one could read it before it has arrived.)
      if (e == cudaSuccess)
        e = cudaMemcpyAsync(set->chunks, table.data(), table.size() * sizeof(Chunk), cudaMemcpyHostToDevice, nullptr);
      if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
      if (e != cudaSuccess) {
        if (set->chunks) cudaFree(set->chunks);
        delete set;
        cudaGetLastError();
        return ops::fail_cuda(e, "gradient set");
      }
    }
    *out = set;
    return PONNI_B200_OK;
  });
}

void ponni_b200_gradient_set_destroy(ponni_b200_gradient_set* set) {
  if (!set) return;
  {
    DeviceGuard guard(set->device);
    if (set->chunks && cudaFree(set->chunks) != cudaSuccess) cudaGetLastError();
  }
  delete set;
}

int64_t ponni_b200_gradient_set_count(const ponni_b200_gradient_set* set) { return set ? set->total : 0; }

int64_t ponni_b200_gradient_set_workspace(const ponni_b200_gradient_set* set) {
  return set ? (int64_t)kMaxBlocks * (int64_t)sizeof(double) : 0;
}

ponni_b200_status ponni_b200_gradient_set_clip(ponni_b200_gradient_set* set, double max_norm, void* flat, int flat_dtype,
                                               float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!set) return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "clip: gradient set is NULL");
  return ops::entry(set->device, [&]() -> ponni_b200_status {
    if (!(max_norm > 0.0)) return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "clip: max_norm must be positive");
    if (!norm || !ops::aligned_to(4, norm))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "clip: norm pointer is NULL or not aligned to 4 bytes");
    if (flat && (flat_dtype < PONNI_B200_F32 || flat_dtype > PONNI_B200_BF16))
      return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "clip: the packed vector must be fp32, fp64, fp16 or bf16");
    if (flat && !ops::aligned_to(ops::element_bytes(flat_dtype), flat))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "clip: the packed vector is not aligned to its type");
    if (!flat && set->overlap)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "clip: tensors of the set overlap, which only a packed vector allows");
    if (flat && !packs_apart(*set, flat, flat_dtype))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "clip: the packed vector overlaps a tensor of the set");
    if (!workspace || workspace_bytes < ponni_b200_gradient_set_workspace(set) ||
        reinterpret_cast<uintptr_t>(workspace) % 8 != 0)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "clip: workspace is too small or not aligned to 8 bytes");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>(set->num_chunks, kMaxBlocks));
    const Chunk* chunks = static_cast<const Chunk*>(set->chunks);
    double* partial = static_cast<double*>(workspace);
    cudaError_t e = cudaSuccess;
    if (set->num_chunks <= kOneClusterChunks) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = std::min(blocks, kCluster);
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(std::min(blocks, kCluster));
      cfg.blockDim = dim3(kBlock);
      cfg.stream = s;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, clip_one_cluster_kernel, chunks, set->num_chunks, max_norm, flat,
                             flat ? flat_dtype : -1, norm);
      return e == cudaSuccess ? PONNI_B200_OK : ops::fail_cuda(e, "clip");
    }
    norm_kernel<<<blocks, kBlock, 0, s>>>(chunks, set->num_chunks, partial);
    e = cudaGetLastError();
    if (e == cudaSuccess)
      e = ops::launch_after(clip_kernel, dim3(blocks), dim3(kBlock), 0, s, chunks, set->num_chunks,
                            (const double*)partial, blocks, max_norm, flat, flat ? flat_dtype : -1, norm);
    if (e != cudaSuccess) return ops::fail_cuda(e, "clip");
    return ops::launched("clip");
  });
}

}  // extern "C"
