// Softmax top-k routing of batch columns to experts, the expert-sorted row
// order that follows from it, and the gradient of the routing weights.
//
// logits x[e][b] (feature-major, batch contiguous).  Choices of column b: the
// top_k largest x[., b], ties to the lower expert; -inf and NaN are never
// chosen and add nothing to a sum.  With m the column's largest logit and
// t_e = exp(x_e - m) (1 where x_e = m, so that infinite logits share),
//   weight_j = t_{e_j} / sum t,   the sum over the chosen experts or over all.
// Rows: all (column, choice) pairs sorted by expert, then by column.
//
// One pass over the logits with the running maximum and sum; the choice is bound by
// the insertions' instructions, not by the logits' bytes: 131072 columns of 64 fp32
// logits, four choices, take 18.5 us to choose (34 MB: 5 us of HBM), 4 to scan
// the counts, 8.5 to place, their gradient 20 us (67 MB: 10 us; 16 with the exponential
// unit alone in place of expf, or where only chosen experts have a gradient).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "device_math.cuh"
#include "operators.h"

namespace ponni_b200 {
namespace {

constexpr int kBlock = 256;  // columns of a tile
constexpr int kWarps = kBlock / 32;

template <class T>
__device__ __forceinline__ float as_logit(T x) {
  const float v = Num<T>::to_c(x);
  return v == v ? v : -INFINITY;
}
// Raw logits of experts e0 .. e0 + N - 1; past the last one the last one's (the
// caller leaves them out).  No conditions around the loads: they go out together.
template <class T, int N>
__device__ __forceinline__ void load_logits(const T* __restrict__ x, int64_t ld, int e0, int experts, T (&raw)[N]) {
  if (e0 + N <= experts) {
    const T* p = x + (int64_t)e0 * ld;
#pragma unroll
    for (int u = 0; u < N; ++u) raw[u] = p[u * ld];
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u) raw[u] = x[(int64_t)min(e0 + u, experts - 1) * ld];
  }
}

// exp(v - best) for v <= best, 1 where they are equal (both may be infinite).
// best is at least -FLT_MAX, so that v = -inf gives 0.
__device__ __forceinline__ float from_best(float v, float best) { return v == best ? 1.0f : expf(v - best); }
// The same by the exponential unit alone, of a product rounded once: off by 2^-22 and 2^-24 of
// best - v, 5e-6 where that is 80.  For the terms of a sum of which the best is 1, and for
// results rounded to 16 bits (131072 columns, 64 experts, all weights: 31.7 us, with expf in
// the sum 35.8; their 16-bit gradient 20.4, 24.6).
__device__ __forceinline__ float near_best(float v, float best) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"((v - best) * 1.4426950408889634f));
  return v == best ? 1.0f : y;
}
__device__ __forceinline__ float at_least_finite(float best) { return fmaxf(best, -3.402823466e38f); }

// The K largest of `count` logits (rows of x, ld apart), largest first, and the
// sum of exp(x - best) over all of them.  Logits come in chunks of kChunk, the next
// chunk's loads ahead of this one's work.  Insertion has no branches: some lane of
// a warp inserts at nearly every expert.
constexpr int kChunk = 8;
template <class T, int K>
__device__ __forceinline__ void scan_logits(const T* __restrict__ x, int64_t ld, int count, bool over_all, int (&idx)[K],
                                            float (&top)[K], float& best, float& sum) {
#pragma unroll
  for (int j = 0; j < K; ++j) {
    top[j] = -INFINITY;
    idx[j] = -1;
  }
  sum = 0.0f;
  best = -3.402823466e38f;
  if (count < 1) return;
  T ahead[kChunk];
  load_logits<T, kChunk>(x, ld, 0, count, ahead);
  for (int e0 = 0; e0 < count; e0 += kChunk) {
    float v[kChunk];
#pragma unroll
    for (int u = 0; u < kChunk; ++u) v[u] = as_logit(ahead[u]);
    if (e0 + kChunk > count) {
#pragma unroll
      for (int u = 0; u < kChunk; ++u) v[u] = e0 + u < count ? v[u] : -INFINITY;
    }
    if (e0 + kChunk < count) load_logits<T, kChunk>(x, ld, e0 + kChunk, count, ahead);
    if (over_all) {
      float now = best;
#pragma unroll
      for (int u = 0; u < kChunk; ++u) now = fmaxf(now, v[u]);
      // In pairs, so that a term passes log2(kChunk) roundings and one for every further chunk.
      float t[kChunk];
#pragma unroll
      for (int u = 0; u < kChunk; ++u) t[u] = near_best(v[u], now);
#pragma unroll
      for (int d = 1; d < kChunk; d *= 2)
#pragma unroll
        for (int u = 0; u + d < kChunk; u += 2 * d) t[u] += t[u + d];
      sum = fmaf(sum, from_best(best, now), t[0]);
      best = now;
    }
#pragma unroll
    for (int u = 0; u < kChunk; ++u) {
      // Behind every entry that is at least as large (of equal logits the lower
      // expert stays first); the entries below move down one place.
      bool up[K];
#pragma unroll
      for (int j = 0; j < K; ++j) up[j] = v[u] > top[j];
#pragma unroll
      for (int j = K - 1; j >= 0; --j) {
        const bool shift = j > 0 && up[j > 0 ? j - 1 : 0];
        top[j] = shift ? top[j > 0 ? j - 1 : 0] : up[j] ? v[u] : top[j];
        idx[j] = shift ? idx[j > 0 ? j - 1 : 0] : up[j] ? e0 + u : idx[j];
      }
    }
  }
}

// Choice and weights of one column by G neighbouring lanes (all of the warp call
// it): each scans every G-th expert, then the lanes' lists are merged.  With G = 1
// the insertions of 256 experts alone take 23 us, and small batches have lanes to spare.
template <class T, int K, int G>
__device__ __forceinline__ void choose(const T* __restrict__ x, int64_t ld, int experts, bool over_all, int (&idx)[K],
                                       float (&w)[K]) {
  float top[K], best, sum;
  const int g = G > 1 ? threadIdx.x % G : 0;
  scan_logits<T, K>(x + g * ld, ld * G, (experts - g + G - 1) / G, over_all, idx, top, best, sum);
  if constexpr (G > 1) {
    int mine[K];
    float have[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      mine[j] = idx[j] < 0 ? -1 : idx[j] * G + g;
      have[j] = top[j];
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      float v = have[0];
      int i = mine[0];
#pragma unroll
      for (int d = 1; d < G; d <<= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, v, d);
        const int oi = __shfl_xor_sync(0xffffffffu, i, d);
        if (oi >= 0 && (i < 0 || ov > v || (ov == v && oi < i))) {
          v = ov;
          i = oi;
        }
      }
      top[j] = v;
      idx[j] = i;
      if (i >= 0 && i == mine[0]) {
#pragma unroll
        for (int q = 0; q + 1 < K; ++q) {
          mine[q] = mine[q + 1];
          have[q] = have[q + 1];
        }
        mine[K - 1] = -1;
        have[K - 1] = -INFINITY;
      }
    }
    if (over_all) {
      sum *= near_best(best, at_least_finite(top[0]));
#pragma unroll
      for (int d = 1; d < G; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    }
  }
  best = at_least_finite(top[0]);
#pragma unroll
  for (int j = 0; j < K; ++j) w[j] = idx[j] < 0 ? 0.0f : from_best(top[j], best);
  if (!over_all) {
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < K; ++j) sum += w[j];
  }
#pragma unroll
  for (int j = 0; j < K; ++j) w[j] = idx[j] < 0 ? 0.0f : w[j] / sum;
}

// Choices of this block's columns [c0, c1) and how many of them each expert
// took: counts[expert][block].
template <class T, int K, int G>
__global__ void __launch_bounds__(kBlock)
    choose_kernel(const T* __restrict__ x, int64_t ld, int experts, int64_t batch, int64_t per_block, int over_all,
                  int* __restrict__ expert, float* __restrict__ weight, int* __restrict__ counts) {
  extern __shared__ int hist[];
  ops::let_successor_start();
  for (int e = threadIdx.x; e < experts; e += kBlock) hist[e] = 0;
  __syncthreads();
  const int64_t c0 = blockIdx.x * per_block, c1 = min(batch, c0 + per_block);
  for (int64_t b0 = c0; b0 < c1; b0 += kBlock / G) {
    const int64_t b = b0 + threadIdx.x / G;
    int idx[K];
    float w[K];
    choose<T, K, G>(x + min(b, c1 - 1), ld, experts, over_all, idx, w);
    if (b < c1 && threadIdx.x % G == 0) {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        expert[j * batch + b] = idx[j];
        weight[j * batch + b] = w[j];
        if (idx[j] >= 0) atomicAdd(&hist[idx[j]], 1);
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kBlock) counts[(int64_t)e * gridDim.x + blockIdx.x] = hist[e];
}

// Exclusive scan of one value a thread over the block (kBlock threads);
// every thread also gets the total.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += o;
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const int t = warp_sums[i];
    if (i < warp) before += t;
    total += t;
  }
  __syncthreads();
  return before + s - v;
}

// counts[e][.] -> rows of expert e taken by earlier blocks; totals[e].
__global__ void __launch_bounds__(kBlock) scan_kernel(int* __restrict__ counts, int blocks, int* __restrict__ totals) {
  __shared__ int warp_sums[kWarps];
  ops::let_successor_start();
  ops::wait_for_predecessor();
  int* c = counts + (int64_t)blockIdx.x * blocks;
  int carry = 0;
  for (int i0 = 0; i0 < blocks; i0 += kBlock) {
    const int i = i0 + threadIdx.x;
    int total;
    const int before = block_scan(i < blocks ? c[i] : 0, warp_sums, total);
    if (i < blocks) c[i] = carry + before;
    carry += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Rows of the choices of columns [c0, c1), given the next row of each expert.
// Within a tile of kBlock columns the rank of a choice is the number of earlier
// columns that chose the same expert (at most once each): a lane mask per warp
// and expert in shared memory, zero on entry and on return.
__device__ __forceinline__ void place(const int* expert, int experts, int top_k, int64_t batch, int64_t c0, int64_t c1,
                                      int* next, unsigned* mask, int* row, int* column) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t t0 = c0; t0 < c1; t0 += kBlock) {
    const int64_t b = t0 + threadIdx.x;
    int es[ops::kMaxTopK];
#pragma unroll
    for (int j = 0; j < ops::kMaxTopK; ++j) es[j] = j < top_k && b < c1 ? expert[j * batch + b] : -1;
#pragma unroll
    for (int j = 0; j < ops::kMaxTopK; ++j)
      if (es[j] >= 0) atomicOr(&mask[warp * experts + es[j]], 1u << lane);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ops::kMaxTopK; ++j) {
      if (j >= top_k || b >= c1) continue;
      const int e = es[j];
      int r = -1;
      if (e >= 0) {
        r = next[e] + __popc(mask[warp * experts + e] & ((1u << lane) - 1u));
        for (int w = 0; w < warp; ++w) r += __popc(mask[w * experts + e]);
        column[r] = (int)b;
      }
      row[j * batch + b] = r;
    }
    __syncthreads();
    if (t0 + kBlock >= c1) break;
    for (int e = threadIdx.x; e < experts; e += kBlock) {
      int n = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        n += __popc(mask[w * experts + e]);
        mask[w * experts + e] = 0;
      }
      next[e] += n;
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kBlock)
    place_kernel(const int* __restrict__ expert, int experts, int top_k, int64_t batch, int64_t per_block,
                 const int* __restrict__ counts, const int* __restrict__ totals, int* __restrict__ row,
                 int* __restrict__ column, int* __restrict__ offset) {
  extern __shared__ int sm[];
  __shared__ int warp_sums[kWarps];
  int* next = sm;                                              // [experts]: next row of each expert
  unsigned* mask = reinterpret_cast<unsigned*>(sm + experts);  // [kWarps][experts]
  ops::let_successor_start();
  for (int i = threadIdx.x; i < kWarps * experts; i += kBlock) mask[i] = 0;
  ops::wait_for_predecessor();
  int carry = 0;
  for (int e0 = 0; e0 < experts; e0 += kBlock) {
    const int e = e0 + threadIdx.x;
    int total;
    const int before = carry + block_scan(e < experts ? totals[e] : 0, warp_sums, total);
    if (e < experts) {
      next[e] = before + counts[(int64_t)e * gridDim.x + blockIdx.x];
      if (blockIdx.x == 0) offset[e] = before;
    }
    carry += total;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offset[experts] = carry;
  for (int64_t i = carry + blockIdx.x * (int64_t)kBlock + threadIdx.x; i < batch * top_k;
       i += (int64_t)gridDim.x * kBlock)
    column[i] = -1;
  __syncthreads();
  const int64_t c0 = blockIdx.x * per_block;
  place(expert, experts, top_k, batch, c0, min(batch, c0 + per_block), next, mask, row, column);
}

// All of it in one launch, by one cluster of up to 8 blocks, for small batches:
// three dependent launches cost more than the work.  Up to kGrouped columns, kGroup lanes take a column.  The blocks read one another's counts through distributed shared memory.
constexpr int kMaxCluster = 8;
constexpr int64_t kOneCluster = kMaxCluster * kBlock;
constexpr int kGroup = 8;
constexpr int64_t kGrouped = 2 * kMaxCluster * kBlock / kGroup;
__device__ __forceinline__ int read_block(const int* p, int rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(rank));
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(v) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;\n" ::: "memory");
}
template <class T, int K, int G>
__global__ void __launch_bounds__(kBlock)
    route_one_cluster_kernel(const T* __restrict__ x, int64_t ld, int experts, int batch, int per_block, int over_all,
                             int* expert, float* __restrict__ weight, int* row, int* column, int* __restrict__ offset) {
  extern __shared__ int sm[];
  __shared__ int warp_sums[kWarps];
  int* hist = sm;                                                  // [experts]: this block's counts
  int* next = sm + experts;                                        // [experts]
  unsigned* mask = reinterpret_cast<unsigned*>(sm + 2 * experts);  // [kWarps][experts]
  const int rank = blockIdx.x, blocks = gridDim.x;
  for (int i = threadIdx.x; i < experts; i += kBlock) hist[i] = 0;
  for (int i = threadIdx.x; i < kWarps * experts; i += kBlock) mask[i] = 0;
  __syncthreads();
  const int c0 = rank * per_block, c1 = min(batch, c0 + per_block);
  for (int b0 = c0; b0 < c1; b0 += kBlock / G) {
    const int b = b0 + threadIdx.x / G;
    int idx[K];
    float w[K];
    choose<T, K, G>(x + min(b, c1 - 1), ld, experts, over_all, idx, w);
    if (b < c1 && threadIdx.x % G == 0) {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        expert[j * batch + b] = idx[j];
        weight[j * batch + b] = w[j];
        if (idx[j] >= 0) atomicAdd(&hist[idx[j]], 1);
      }
    }
  }
  __syncthreads();
  if (blocks > 1) cluster_barrier();
  int carry = 0;
  for (int e0 = 0; e0 < experts; e0 += kBlock) {
    const int e = e0 + threadIdx.x;
    int all = 0, earlier = 0, total;
    if (e < experts) {
      for (int q = 0; q < blocks; ++q) {
        const int n = blocks > 1 ? read_block(hist + e, q) : hist[e];
        all += n;
        earlier += q < rank ? n : 0;
      }
    }
    const int before = carry + block_scan(all, warp_sums, total);
    if (e < experts) {
      next[e] = before + earlier;
      if (rank == 0) offset[e] = before;
    }
    carry += total;
  }
  if (blocks > 1) cluster_barrier();  // the others have read this block's counts
  if (rank == 0 && threadIdx.x == 0) offset[experts] = carry;
  for (int i = carry + rank * kBlock + threadIdx.x; i < batch * K; i += blocks * kBlock) column[i] = -1;
  __syncthreads();
  place(expert, experts, K, batch, c0, c1, next, mask, row, column);
}

// d_x[e][b] = p_e (d_p_e - sum_j w_j d_w_j), d_p_e = d_w_j for the chosen
// experts and 0 for others; p is the softmax over all experts or over the
// chosen ones.  Over all: the first choice has t = 1, so p_e = t_e weight_0
// and no second sum is needed.
//
// A thread takes one column and kBackPart experts: all of them as if not
// chosen first (their logits loaded at once), then the chosen ones again.
constexpr int kBackPart = 16;
template <class T, int K>
__global__ void __launch_bounds__(kBlock)
    route_backward_kernel(const T* __restrict__ x, int64_t ld, int experts, int64_t batch, int over_all,
                          const int* __restrict__ expert, const float* __restrict__ weight,
                          const float* __restrict__ d_weight, T* __restrict__ dx, int64_t d_ld) {
  const int64_t b = blockIdx.x * (int64_t)kBlock + threadIdx.x;
  if (b >= batch) return;
  const int e0 = blockIdx.y * kBackPart;
  T raw[kBackPart];
  if (over_all) load_logits<T, kBackPart>(x + b, ld, e0, experts, raw);
  int idx[K];
  float w[K], g[K], mean = 0.0f;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    idx[j] = expert[j * batch + b];
    if (idx[j] >= experts) idx[j] = -1;
    w[j] = weight[j * batch + b];
    g[j] = idx[j] >= 0 ? w[j] * d_weight[j * batch + b] : 0.0f;
    mean += g[j];
  }
  const bool any = idx[0] >= 0;
  const float best = any && over_all ? as_logit(x[(int64_t)idx[0] * ld + b]) : 0.0f;
  const float scale = any ? -w[0] * mean : 0.0f;
  auto term = [&](float v) { return sizeof(T) == 2 ? near_best(v, best) : from_best(v, best); };
#pragma unroll
  for (int u = 0; u < kBackPart; ++u)
    if (e0 + u < experts)
      dx[(e0 + u) * d_ld + b] = Num<T>::from_c(over_all && any ? term(as_logit(raw[u])) * scale : 0.0f);
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (idx[j] >= e0 && idx[j] < e0 + kBackPart) dx[(int64_t)idx[j] * d_ld + b] = Num<T>::from_c(g[j] - w[j] * mean);
}

// Whether one cluster does all: 16 experts take 5 us with up to 2048 columns (7 in
// three launches, which also cost the host two launches more), 256 experts
// 12 us with 256 columns, but 35 with 1024 against 14 on all SMs.
bool one_cluster(int experts, int64_t batch) { return batch <= kGrouped / 2 || (batch <= kOneCluster && experts <= 64); }

// Columns of a block of the three-launch form: whole tiles for at most 592 blocks.
// Where the columns do not fill the SMs with work, kGroup lanes take a column and
// a tile is so much smaller (256 experts: 14.8 us against 44 with 4096 columns, 27
// against 44 with 16384; 16 experts: 9.9 against 7.0 with 16384).
bool spread(int experts, int64_t batch) { return batch <= (int64_t)128 * experts; }
int64_t columns_of_block(int experts, int64_t batch) {
  const int64_t tile = spread(experts, batch) ? kBlock / kGroup : kBlock;
  const int64_t tiles = (batch + tile - 1) / tile;
  return (tiles + 591) / 592 * tile;
}
int64_t blocks_of(int experts, int64_t batch) {
  const int64_t per = columns_of_block(experts, batch);
  return (batch + per - 1) / per;
}

// f(T, K) for the type and the number of choices.
template <class T, class F>
ponni_b200_status by_top_k(int top_k, F&& f) {
  switch (top_k) {
#define PB_CASE(K) \
  case K: return f(T(), std::integral_constant<int, K>())
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
  return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "route: top_k must be 1 to 8");
}
template <class F>
ponni_b200_status by_type(int dtype, int top_k, F&& f) {
  if (dtype == PONNI_B200_F32) return by_top_k<float>(top_k, f);
  if (dtype == PONNI_B200_F16) return by_top_k<__half>(top_k, f);
  return by_top_k<__nv_bfloat16>(top_k, f);
}

ponni_b200_status check_route(int dtype, const void* logits, int64_t ld, int experts, int top_k, int64_t batch,
                              int normalise) {
  using namespace ops;
  if (!is_real_type(dtype)) return fail(PONNI_B200_ERR_UNSUPPORTED, "route: logits must be fp32, fp16 or bf16");
  if (!logits || !aligned_to(element_bytes(dtype), logits))
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, "route: logits pointer is NULL or not aligned to its type");
  if (experts < 1 || experts > kMaxExperts)
    return fail(PONNI_B200_ERR_UNSUPPORTED, "route: the number of experts must be 1 to 1024");
  if (top_k < 1 || top_k > kMaxTopK || top_k > experts)
    return fail(PONNI_B200_ERR_UNSUPPORTED, "route: top_k must be 1 to 8 and at most the number of experts");
  if (batch < 1 || batch > INT32_MAX / top_k)
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, "route: batch must be nonzero and batch * top_k below 2^31");
  if (ld < batch) return fail(PONNI_B200_ERR_INVALID_ARGUMENT, "route: row stride smaller than the batch size");
  if (normalise != PONNI_B200_ROUTE_SELECTED && normalise != PONNI_B200_ROUTE_ALL)
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, "route: unknown normalisation");
  return PONNI_B200_OK;
}

}  // namespace
}  // namespace ponni_b200

using namespace ponni_b200;

extern "C" {

int64_t ponni_b200_route_workspace(int num_experts, int64_t batch) {
  if (num_experts < 1 || batch < 1 || one_cluster(num_experts, batch)) return 0;
  return (int64_t)num_experts * (blocks_of(num_experts, batch) + 1) * (int64_t)sizeof(int);
}

ponni_b200_status ponni_b200_route_columns(int dtype, const void* logits, int64_t ld, int num_experts, int top_k,
                                           int64_t batch, int normalise, int32_t* expert, float* weight, int32_t* row,
                                           int32_t* column, int32_t* offset, void* workspace, int64_t workspace_bytes,
                                           int device, void* stream) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    ponni_b200_status st = check_route(dtype, logits, ld, num_experts, top_k, batch, normalise);
    if (st) return st;
    if (!expert || !weight || !row || !column || !offset ||
        !ops::aligned_to(4, expert, weight, row, column, offset, workspace))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "route: output pointer is NULL or not aligned to 4 bytes");
    const int64_t need = ponni_b200_route_workspace(num_experts, batch);
    if (need && (!workspace || workspace_bytes < need))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "route: workspace is too small");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int all = normalise == PONNI_B200_ROUTE_ALL;
    const size_t place_smem = (size_t)num_experts * (kWarps + 1) * sizeof(int);
    return by_type(dtype, top_k, [&](auto t, auto k) -> ponni_b200_status {
      using T = decltype(t);
      constexpr int K = decltype(k)::value;
      const T* x = static_cast<const T*>(logits);
      if (one_cluster(num_experts, batch)) {
        const int64_t at_once = batch <= kGrouped ? kBlock / kGroup : kBlock;
        const int blocks = (int)std::min<int64_t>(kMaxCluster, (batch + at_once - 1) / at_once);
        const int per = (int)((batch + blocks - 1) / blocks);
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = blocks;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(blocks);
        cfg.blockDim = dim3(kBlock);
        cfg.dynamicSmemBytes = (size_t)num_experts * (kWarps + 2) * sizeof(int);
        cfg.stream = s;
        cfg.attrs = attr;
        cfg.numAttrs = blocks > 1 ? 1 : 0;
        auto kern = batch <= kGrouped ? route_one_cluster_kernel<T, K, kGroup> : route_one_cluster_kernel<T, K, 1>;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, x, ld, num_experts, (int)batch, per, all, expert, weight, row,
                                                 column, offset);
        return e == cudaSuccess ? PONNI_B200_OK : ops::fail_cuda(e, "route_columns");
      }
      const int64_t per_block = columns_of_block(num_experts, batch);
      const int blocks = (int)blocks_of(num_experts, batch);
      int* counts = static_cast<int*>(workspace);
      int* totals = counts + (int64_t)num_experts * blocks;
      auto choose = spread(num_experts, batch) ? choose_kernel<T, K, kGroup> : choose_kernel<T, K, 1>;
      choose<<<blocks, kBlock, num_experts * sizeof(int), s>>>(x, ld, num_experts, batch, per_block, all, expert, weight,
                                                             counts);
      cudaError_t e = cudaGetLastError();
      if (e == cudaSuccess)
        e = ops::launch_after(scan_kernel, dim3(num_experts), dim3(kBlock), 0, s, counts, blocks, totals);
      if (e == cudaSuccess)
        e = ops::launch_after(place_kernel, dim3(blocks), dim3(kBlock), place_smem, s, (const int*)expert, num_experts,
                              top_k, batch, per_block, (const int*)counts, (const int*)totals, row, column, offset);
      return e == cudaSuccess ? PONNI_B200_OK : ops::fail_cuda(e, "route_columns");
    });
  });
}

ponni_b200_status ponni_b200_route_columns_backward(int dtype, const void* logits, int64_t ld, int num_experts,
                                                    int top_k, int64_t batch, int normalise, const int32_t* expert,
                                                    const float* weight, const float* d_weight, void* d_logits,
                                                    int64_t d_ld, int device, void* stream) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    ponni_b200_status st = check_route(dtype, logits, ld, num_experts, top_k, batch, normalise);
    if (st) return st;
    if (!expert || !weight || !d_weight || !d_logits || !ops::aligned_to(4, expert, weight, d_weight) ||
        !ops::aligned_to(ops::element_bytes(dtype), d_logits))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "route backward: pointer is NULL or not aligned to its type");
    if (d_ld < batch)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "route backward: row stride smaller than the batch size");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((batch + kBlock - 1) / kBlock), (unsigned)((num_experts + kBackPart - 1) / kBackPart));
    const int all = normalise == PONNI_B200_ROUTE_ALL;
    return by_type(dtype, top_k, [&](auto t, auto k) -> ponni_b200_status {
      using T = decltype(t);
      route_backward_kernel<T, decltype(k)::value><<<grid, kBlock, 0, s>>>(
          static_cast<const T*>(logits), ld, num_experts, batch, all, expert, weight, d_weight,
          static_cast<T*>(d_logits), d_ld);
      return ops::launched("route_columns_backward");
    });
  });
}

}  // extern "C"
