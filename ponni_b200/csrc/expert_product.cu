// Products grouped by expert: rows r in [offset[e], offset[e+1]) times
// weights[e] (inputs x outputs, row-major as in Matvec), with bias and
// activation, and the gradients
//   kForward  out[r]      = act(rows[r] W_e + b_e)       M rows,   N outputs, K inputs
//   kRows     d_rows[r]   = d_out[r] W_e^T               M rows,   N inputs,  K outputs
//   kWeights  d_W_e       = rows_e^T d_out_e             M inputs, N outputs, K rows of the group
// as tcgen05 products of 128 x BN tiles, K in blocks of 64.
//
// Operands are read where they lie: the groups' rows start anywhere, but rows
// are the outer index of every operand, so a tile starts at any row with an
// aligned innermost coordinate, and whichever index is contiguous decides
// between K-major and MN-major shared-memory tiles (no transposed copies):
//            A                    B
//   kForward rows     K-major     W_e     MN-major
//   kRows    d_out    K-major     W_e     K-major
//   kWeights rows     MN-major    d_out   MN-major
// A row tile that runs past its group computes on the next group's rows and
// does not store them; in kWeights the rows past the group are the
// contraction, so the last K block's are zeroed in shared memory (both
// operands: the neighbour's values may be infinite).
//
// fp32 operands are split exactly into three bf16 parts x = x0 + x1 + x2, the nearest
// each time, and six products are kept (x1 y2, x2 y1 and x2 y2 are dropped: together below 2^-23
// of the magnitude, near 2^-25 on average, of either sign).  Each K
// block of 64 goes into its own TMEM accumulator, the five small products first,
// and is added to the tile's sum in fp32 registers: the tensor core truncates
// when it accumulates, so long sums in TMEM drift by a part of 2^-24 for
// every step (16-bit products are added up every kSegment blocks).  These products are bound by shared memory: a block's 24 MMAs of
// 128 x 128 x 16 read 192 KB and its copies write 96 KB, 2250 cycles at 128 bytes a
// cycle against 1536 of the tensor cores.  (K blocks of 32 and twice the stages are
// 10% slower.)
//
// One persistent CTA per SM: a TMA producer, an MMA warp and sixteen epilogue
// warps.  Every role walks the same tile sequence, which it derives from the
// offsets (read once into shared memory): no host copy of the group sizes.
// Measured alone: 32768 rows, 32 experts of 2048 x 2048 bf16 with SiLU in 208 to
// 232 us (1.2 PFLOP/s; tensor pipe 78% active at the power limit's 1.39 GHz),
// 2^20 rows, 8 experts of 256 x 256 in 174 us without activation (6.2 TB/s), 203 to 222 with
// SiLU, 384 rows, 64 experts of 1024 x 2048 in 53 to 59 us (4.6 to 5.1 TB/s).
//
// A few rows for each expert (serving) are bound by the weights' bytes and by
// latency: few_rows_kernel streams the weights once, without tensor cores.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "device_math.cuh"
#include "expert_tiles.h"
#include "operators.h"
#include "tc_common.cuh"

PONNI_B200_SKIP_ARRIVE_FLAG(ge)

namespace ponni_b200 {
namespace {
using namespace tc;

using namespace grouped;

// K blocks of a 16-bit product that are summed in one accumulator before the epilogue adds
// them to its fp32 sum.  The tensor core truncates as it accumulates: 32 blocks drift by 2^-16
// of the sum at most, a thirty-second of fp16's rounding, whole groups of 2^20 rows would by
// 2^-8.  (16384 rows, 4 experts of 8192 -> 2048: 365 us, 367 with 16 blocks, 364 without
// segments; 2048 -> 2048, where 16 blocks make two segments: 197 us against 195.)
constexpr int kSegment = 32;
constexpr int kEpiWarps = 16;
constexpr int kBlock = 32 * (2 + kEpiWarps);
constexpr int kEpiPitch = 48;  // bytes of a staged output row segment of 32 (+16: conflict-free)
constexpr int kEpiBytes = kEpiWarps * 32 * kEpiPitch;
constexpr int kBiasBytes = kEpiWarps * 64 * 4;

struct Args {
  const void* a;  // kForward: rows; kRows: d_out; kWeights: rows (as the caller gave them)
  const void* b;  // kForward, kRows: weights; kWeights: d_out
  void* c;
  float* partial;  // kWeights, split: fp32 sums of every unit [unit][inputs][outputs]
  int64_t a_ld, b_ld, b_stride, c_ld;
  int64_t rows;
  const int* offset;
  const void* bias;
  int experts, inputs, outputs;
  int act, act_flags;
  float s0, s1;
  int unit_rows;  // kWeights: rows of a unit (a multiple of kBK); 0: a group is one unit
  int vec;        // c may be written 16 bytes at a time
  int bulk;       // and by the copy engine (map_c)
  int boxes;      // of output staging a warp
  int stages;
  int device;
  int* error;
};

// CG: CTAs that share a tile.  With two (cta_group::2) the tile is 256 x BN, each
// CTA holds its 128 rows of A, half of B's columns and its 128 rows of the sums.
template <int P, int BN, int CG> struct Shape {
  static constexpr int b_rows = BN / CG;
  static constexpr int a_bytes = P * kBM * kBK * 2;
  static constexpr int b_bytes = P * b_rows * kBK * 2;
  static constexpr int stage_bytes = a_bytes + b_bytes;
  static constexpr int acc_cols = BN <= 128 ? 128 : 256;
  static constexpr int acc_bufs = 512 / acc_cols;
  // Epilogue warps: four lane quarters (a warp reads the TMEM lanes of its
  // number modulo 4) times `parts` strips of columns.
  static constexpr int parts = BN >= 128 ? 4 : 2;
  // Groups of warps, which take tiles by their accumulators (Turns).  Only where a tile is
  // one accumulator (16-bit operands).
  static constexpr int groups = 4 / parts;
  static_assert(groups == 1 || (P == 1 && acc_bufs % groups == 0), "an accumulator belongs to one group");
  // K blocks that are summed in one accumulator.  (Groups of warps: all of a tile's; the host gives
  // them sums of at most kSegment blocks.)
  static constexpr int segment = P == 3 ? 1 : groups > 1 ? 1 << 30 : kSegment;
  static constexpr int part_cols = BN / parts;
  // Output staging of a warp: boxes of 32 rows x 64 bytes for the copy engine
  // (16-bit operands in pairs or 64 wide), else its rows of 32 bytes: the boxes cost
  // the single 128-wide tiles stages, and with them 10% on weight-bound products.
  static constexpr bool bulk_store = P == 1 && (CG == 2 || BN == 64);
};

// Staging bytes.  Products of up to 8 K blocks, which store a tile after little else,
// get two boxes a warp (256 -> 128: 131 us against 142 with one); longer ones
// one box and a stage more (64 us against 61 for 16384 rows, 1024 -> 2048).
template <class S>
__host__ __device__ constexpr int epi_bytes(int boxes) {
  return S::bulk_store ? kEpiWarps * 2048 * boxes : kEpiBytes;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// The same in a pair: the bytes are counted on a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
      "%4}], [%5];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// 8 accumulator columns of this thread's TMEM lane, from `taddr` on and back.
__device__ __forceinline__ void tmem_add8(uint32_t taddr, float* v) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    f2::add(v[i], v[i + 1], v[i], v[i + 1], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(taddr),
               "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
               "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
               "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
               : "memory");
}

// Arrival on another CTA's barrier after reading tensor memory, which the tcgen05
// fence before it orders: no release of this thread's stores, which would cost
// half a microsecond each.
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int x, int y, int z, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n\t"
               "cp.async.bulk.commit_group;\n" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(z), "r"(src)
               : "memory");
}
// All but the last N stores of this thread have read their source.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tma_store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }

// Check of the offsets by one block (the groups are clamped whatever they hold).
__device__ __forceinline__ void check_offsets(const int* __restrict__ offset, int experts, int64_t rows, int* error) {
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) {
    const int64_t o = offset[e], before = e ? offset[e - 1] : 0;
    if (o < before || o > rows || (e == 0 && o != 0)) atomicOr(error, 2);
  }
}
__device__ __forceinline__ int clamped(int o, int lo, int64_t rows) { return (int)min(max((int64_t)o, (int64_t)lo), rows); }

// Bounds of all groups into shared memory, by the whole block, which may use them on return.
__device__ __forceinline__ void read_bounds(int* edge, const int* __restrict__ offset, int experts, int64_t rows) {
  bool descends = false;
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) {
    const int b = bound(offset[e], rows);
    edge[e] = b;
    descends |= e > 0 && b < bound(offset[e - 1], rows);
  }
  if (__syncthreads_or(descends)) {
    if (threadIdx.x == 0) ascending(edge, experts);
    __syncthreads();
  }
}

// Which of up to 32 lines of an operand hold a NaN, as a mask; by the whole warp.
__device__ __forceinline__ unsigned nan_lines(const float* p, int lines, int64_t line_step, int terms, int64_t term_step) {
  const int lane = threadIdx.x & 31;
  if (term_step != 1) {  // a line a lane
    bool nan = false;
    const float* q = p + min(lane, lines - 1) * line_step;
#pragma unroll 8
    for (int k = 0; k < terms; ++k) nan |= q[k * term_step] != q[k * term_step];
    return __ballot_sync(0xffffffffu, nan);
  }
  unsigned mask = 0;
  for (int i = 0; i < lines; ++i) {
    bool nan = false;
    const float* q = p + i * line_step;
#pragma unroll 8
    for (int k = lane; k < terms; k += 32) nan |= q[k] != q[k];
    mask |= (__any_sync(0xffffffffu, nan) ? 1u : 0u) << i;
  }
  return mask;
}

// 32 columns of 32 rows (a row a lane, from row m on) straight from the fp32 operands: taken
// where the split parts gave NaN, because an infinite value times another's zero part
// is NaN where the plain product is infinite.  Rows and columns that hold a NaN are NaN all
// the same and found first: 8192 rows of 1024 -> 1024 with one NaN in each take 640 us, without 135,
// and 38 ms if they are all summed one by one.  Of the others all columns are summed at once, so
// that a term costs one load of the row and 32 broadcast ones: a tile of 16384 terms takes 17 ms (180 one
// column after the other).  Sums of more than kPlainTerms terms stay NaN: a tile of them
// would come near the other roles' bounded waits.
constexpr int kPlainTerms = 65536;
template <int MODE>
__device__ __noinline__ void plain_sums(const Args& p, int e, int lo, int hi, int m, int m_valid, int n, int n_valid,
                                        float (&x)[32]) {
  const float* a = static_cast<const float*>(p.a);
  const float* b = static_cast<const float*>(p.b);
  int64_t a_row = p.a_ld, a_step = 1, b_step = p.b_ld, b_col = 1;
  int terms = p.inputs;
  if (MODE == kWeights) {
    a += lo * p.a_ld + m;
    b += lo * p.b_ld + n;
    a_row = 1;
    a_step = p.a_ld;
    terms = hi - lo;
  } else {
    a += (int64_t)(lo + m) * p.a_ld;
    b += e * p.b_stride + (MODE == kForward ? n : n * p.b_ld);
    if (MODE == kRows) {
      b_step = 1;
      b_col = p.b_ld;
      terms = p.outputs;
    }
  }
  const int row = min((int)(threadIdx.x & 31), m_valid - 1);
  n_valid = min(n_valid, 32);
  const unsigned rows = nan_lines(a, m_valid, a_row, terms, a_step);
  const unsigned cols = nan_lines(b, n_valid, b_col, terms, b_step);
  bool wanted = false;
#pragma unroll
  for (int i = 0; i < 32; ++i) wanted |= i < n_valid && x[i] != x[i] && !(cols >> i & 1u);
  if (!__any_sync(0xffffffffu, wanted && !(rows >> row & 1u))) return;
  a += row * a_row;
  float s[32] = {};
  for (int k = 0; k < terms; ++k) {
    const float v = a[k * a_step];
    const float* w = b + k * b_step;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n_valid) s[i] = fmaf(v, w[i * b_col], s[i]);
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = x[i] != x[i] ? s[i] : x[i];
}

// Activations of results that are rounded to 16 bits: exp and reciprocal by the
// fast units, each within 2^-21 of its value, subnormal values as zero.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float fast_sigmoid(float x) { return fast_rcp(1.0f + fast_exp2(-kLog2e * x)); }
// 0.5 x (1 + erf(x / sqrt 2)) with the error function of Abramowitz and Stegun
// 7.1.26 (erf within 1.5e-7): erfc(y) = (a1 t + ... + a5 t^5) exp(-y^2),
// t = 1 / (1 + 0.3275911 y), y >= 0.
__device__ __forceinline__ float fast_gelu(float x) {
  const float y = fabsf(x) * 0.70710678118654752f;
  const float t = fast_rcp(fmaf(0.3275911f, y, 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float c = 0.5f * p * t * fast_exp2(-kLog2e * y * y);  // erfc(y) / 2
  return x * (x > 0.0f ? 1.0f - c : c);
}

template <class T>
__device__ __forceinline__ float activate_one(int kind, int flags, float x, float s0, float s1) {
  if constexpr (sizeof(T) == 2) {
    if (kind == EPI_SILU) return x * fast_sigmoid(x);
    if (kind == EPI_SIGMOID) return fast_sigmoid(x);
    if (kind == EPI_GELU && !(flags & 0x2)) return fast_gelu(x);
  }
  return activation<float>(kind, flags, x, s0, s1);
}

// Out of line: the exact formulas, unrolled into a kernel for 32 values, cost
// more in instruction fetches than in work.
template <class T>
__device__ __noinline__ float4 activate4(float4 v, int kind, int flags, float s0, float s1) {
  v.x = activate_one<T>(kind, flags, v.x, s0, s1);
  v.y = activate_one<T>(kind, flags, v.y, s0, s1);
  v.z = activate_one<T>(kind, flags, v.z, s0, s1);
  v.w = activate_one<T>(kind, flags, v.w, s0, s1);
  return v;
}

// SiLU and exact GELU of 32 values whose results are rounded to 16 bits.  The
// special-function unit bounds the epilogue of narrow products (256 -> 256: two of
// its operations a value would take 139 of the 256 us measured with them), so two
// values share one reciprocal: 1/a = b (1/ab) (213 us; 219 with two reciprocals,
// 226 with half of the exponentials by polynomial).  That needs ab finite and keeps no NaN
// from its neighbour: false, and nothing done, where a value is NaN or below -43 (exponentials
// up to 2^62.1); such rows take activate_one, as a few rows do.  (The check costs 2%, 244 us
// against 240; the same without it by scaled reciprocals takes as long.)
__device__ __forceinline__ float min_or_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float least_of(const float (&v)[32]) {
  float least[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int i = 4; i < 32; ++i) least[i % 4] = min_or_nan(least[i % 4], v[i]);
  return min_or_nan(min_or_nan(least[0], least[1]), min_or_nan(least[2], least[3]));
}
__device__ __forceinline__ bool fast_silu32(float (&v)[32]) {
  if (!(least_of(v) >= -43.0f)) return false;
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    float a, b;
    f2::mul(a, b, v[i], v[i + 1], -kLog2e, -kLog2e);
    f2::add(a, b, fast_exp2(a), fast_exp2(b), 1.0f, 1.0f);
    const float r = fast_rcp(a * b);
    f2::mul(a, b, b, a, r, r);
    f2::mul(v[i], v[i + 1], v[i], v[i + 1], a, b);
  }
  return true;
}
__device__ __forceinline__ void fast_gelu32(float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    float y, z, s, t, p, q;
    f2::mul(y, z, fabsf(v[i]), fabsf(v[i + 1]), 0.70710678118654752f, 0.70710678118654752f);
    y = fminf(y, 1e9f);
    z = fminf(z, 1e9f);
    f2::fma(s, t, y, z, 0.3275911f, 0.3275911f, 1.0f, 1.0f);
    const float r = fast_rcp(s * t);
    f2::mul(s, t, t, s, r, r);
    f2::fma(p, q, s, t, 1.061405429f, 1.061405429f, -1.453152027f, -1.453152027f);
    f2::fma(p, q, p, q, s, t, 1.421413741f, 1.421413741f);
    f2::fma(p, q, p, q, s, t, -0.284496736f, -0.284496736f);
    f2::fma(p, q, p, q, s, t, 0.254829592f, 0.254829592f);
    f2::mul(p, q, p, q, s, t);
    f2::mul(s, t, y, z, -kLog2e, -kLog2e);
    f2::mul(s, t, s, t, y, z);
    f2::mul(p, q, p, q, 0.5f, 0.5f);
    f2::mul(p, q, p, q, fast_exp2(s), fast_exp2(t));  // erfc(|x| / sqrt 2) / 2
    v[i] *= v[i] > 0.0f ? 1.0f - p : p;
    v[i + 1] *= v[i + 1] > 0.0f ? 1.0f - q : q;
  }
}

template <class T>
__device__ __forceinline__ void activate_all(float (&v)[32], int kind, int flags, float s0, float s1) {
  if (kind == EPI_NONE) return;
  if (kind == EPI_RELU) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = v[i] > 0.0f ? v[i] : 0.0f;
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (kind == EPI_SILU && fast_silu32(v)) return;
    if (kind == EPI_GELU && !(flags & 0x2)) return fast_gelu32(v);
  } else if (kind == EPI_SILU && least_of(v) >= -80.0f) {
    // As activation() has it where no exponential overflows, in line: 2^20 rows of 256 -> 256 in
    // 1590 us against 2050, 1465 with an approximate division.
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = v[i] / (1.0f + expf(-v[i]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 r = activate4<T>(make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]), kind, flags, s0, s1);
    v[i] = r.x;
    v[i + 1] = r.y;
    v[i + 2] = r.z;
    v[i + 3] = r.w;
  }
}

// 32 columns of this warp's 32 rows (one row a lane) to global memory through
// the warp's staging rows: 32 contiguous bytes (a sector) of a row at a time.
template <class O>
__device__ __forceinline__ void store_rows(const float (&v)[32], unsigned char* stage, O* c, int64_t ld, int m_valid,
                                           int n_valid, bool vec) {
  constexpr int kCols = 32 / sizeof(O), kPasses = 32 / kCols, kPer = 16 / sizeof(O);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    alignas(16) O o[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) o[i] = Num<O>::from_c(v[pass * kCols + i]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<uint4*>(stage + lane * kEpiPitch)[i] = reinterpret_cast<const uint4*>(o)[i];
    __syncwarp();
    const int col0 = pass * kCols;
    if (vec && col0 + kCols <= n_valid) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = i * 16 + (lane >> 1), ch = lane & 1;
        const uint4 u = *reinterpret_cast<const uint4*>(stage + r * kEpiPitch + ch * 16);
        if (r < m_valid) *reinterpret_cast<uint4*>(c + r * ld + col0 + ch * kPer) = u;
      }
    } else {
#pragma unroll 4
      for (int i = 0; i < kCols; ++i) {
        const int r = i * (32 / kCols) + lane / kCols, col = lane % kCols;
        const O u = reinterpret_cast<const O*>(stage + r * kEpiPitch)[col];
        if (r < m_valid && col0 + col < n_valid) c[r * ld + col0 + col] = u;
      }
    }
    __syncwarp();
  }
}

template <class T, int MODE, int P, int BN, int CG>
__global__ void __launch_bounds__(kBlock, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_c, const Args p) {
  using S = Shape<P, BN, CG>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t bars[3 * kMaxStages + 2 * 4 + 1];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  static_assert(sizeof bars + sizeof tmem_slot + sizeof abort_word + 16 <= kStaticBytes, "static shared memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_raw + (base - raw);
  unsigned char* epi = base_ptr + p.stages * S::stage_bytes;
  const int epi_total = epi_bytes<S>(p.boxes);
  float* bias_s = reinterpret_cast<float*>(epi + epi_total);
  int* edge = reinterpret_cast<int*>(epi + epi_total + kBiasBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto peer_full = [&](int s) { return bar0 + 8u * (2 * kMaxStages + s); };  // the other CTA's stage, told to the first
  auto acc_full = [&](int b) { return bar0 + 8u * (3 * kMaxStages + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (3 * kMaxStages + 4 + b); };
  const uint32_t drain = bar0 + 8u * (3 * kMaxStages + 8);
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  volatile int* abort_flag = &abort_word;

  ops::let_successor_start();
  if (tid == 0) {
    abort_word = 0;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
      mbar_init(peer_full(s), 1);
    }
    for (int b = 0; b < S::acc_bufs; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), CG * 4 * S::parts);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 1) {
    if constexpr (CG == 2) tmem_alloc_pair(smem_u32(&tmem_slot), 512);
    else tmem_alloc(smem_u32(&tmem_slot), 512);
  }
  ops::wait_for_predecessor();
  if (blockIdx.x == 0) check_offsets(p.offset, p.experts, p.rows, p.error);
  tc_fence_before();
  read_bounds(edge, p.offset, p.experts, p.rows);
  if constexpr (CG == 2) cluster_sync();  // the barriers exist before the other CTA's arrivals
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  Tiles<MODE, BN, CG> tiles({p.experts, p.inputs, p.outputs, p.unit_rows}, edge, blockIdx.x / CG, gridDim.x / CG, (int)rank);
  Tile v;
  int64_t issued = 0;  // stages filled so far (thread 0)
  if (warp == 0) {
    // ------------------------------------------------------- producer ----
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 1;  // empty barriers: the first pass finds them free
      bool ok = true;
      while (ok && tiles.next(v)) {
        for (int kb = 0; kb < v.k_blocks; ++kb) {
          if (!wait_phase_abort(empty(s), ph, abort_flag, PONNI_B200_WAIT_LIMIT)) {
            ok = false;
            break;
          }
          const uint32_t a = base + (uint32_t)s * S::stage_bytes, b = a + S::a_bytes;
          const int k0 = kb * kBK, b0 = v.n0 + (int)rank * S::b_rows;
          // A pair's loads are counted on the first CTA's barrier, except for a
          // K block whose tail each CTA has to clear first.
          const bool apart = CG == 1 || (MODE == kWeights && v.hi - v.lo - k0 < kBK);
          const uint32_t bar = CG == 2 && !apart ? mapa_shared(full(s), 0) : full(s);
          if (rank == 0 || apart) mbar_expect_tx(full(s), apart ? S::stage_bytes : CG * S::stage_bytes);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int z) {
            if constexpr (CG == 2) tma_load_3d_pair(dst, map, x, y, z, bar);
            else tma_load_3d(dst, map, x, y, z, bar);
          };
#pragma unroll
          for (int q = 0; q < P; ++q) {
            const uint32_t aq = a + q * (kBM * kBK * 2), bq = b + q * (S::b_rows * kBK * 2);
            if (MODE != kWeights) {
              load(aq, &map_a, k0, v.lo + v.m0, q);
            } else {
#pragma unroll
              for (int j = 0; j < kBM / 64; ++j) load(aq + j * 8192, &map_a, v.m0 + 64 * j, v.lo + k0, q);
            }
            if (MODE == kRows) {
              load(bq, &map_b, k0, b0, q * p.experts + v.e);
            } else {
#pragma unroll
              for (int j = 0; j < S::b_rows / 64; ++j) {
                if (MODE == kForward) load(bq + j * 8192, &map_b, b0 + 64 * j, k0, q * p.experts + v.e);
                else load(bq + j * 8192, &map_b, b0 + 64 * j, v.lo + k0, q);
              }
            }
          }
          ++issued;
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      if (!ok) atomicOr(p.error, 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA ----
    constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr bool a_mn = MODE == kWeights, b_mn = MODE != kRows;
    constexpr uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_mn ? 1u : 0u) << 15) |
                               ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(CG * kBM >> 4) << 24);
    // MN-major: 64-element chunks 8192 bytes apart (leading offset), groups of
    // 8 k 1024 apart; K-major: rows of 128 bytes, groups of 8 rows 1024 apart.
    const uint64_t da = smem_desc(base, a_mn ? 8192 : 16, 1024), db = smem_desc(base, b_mn ? 8192 : 16, 1024);
    const uint32_t a_hi = (uint32_t)(da >> 32), b_hi = (uint32_t)(db >> 32), a_lo0 = (uint32_t)da, b_lo0 = (uint32_t)db;
    constexpr uint32_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;  // 16 k further, in 16-byte units
    int s = 0, buf = 0;
    uint32_t ph = 0, acc_ph = 1;
    bool ok = true, skip = PONNI_B200_SKIP_ARRIVE();
    // Rows of the next group in the unit's last K block: not part of this sum.
    auto clear_tail = [&](int kb) {
      const int valid = v.hi - v.lo - kb * kBK;
      unsigned char* stage = base_ptr + s * S::stage_bytes;
      for (int ch = 0; ch < S::stage_bytes / 8192; ++ch)
        for (int i = valid * 8 + lane; i < kBK * 8; i += 32)
          *reinterpret_cast<uint4*>(stage + ch * 8192 + i * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
    };
    auto mma = [&](uint32_t d, uint32_t alo, uint32_t blo, uint32_t accumulate) {
      if constexpr (CG == 2) umma_f16_pair_warp(d, alo, a_hi, blo, b_hi, idesc, accumulate);
      else umma_f16_desc_warp(d, alo, a_hi, blo, b_hi, idesc, accumulate);
    };
    auto commit = [&](uint32_t bar) {
      if constexpr (CG == 2) umma_commit_pair_warp(bar);  // to both CTAs
      else umma_commit_warp(bar);
    };
    auto next_stage = [&]() {
      if (++s == p.stages) {
        s = 0;
        ph ^= 1u;
      }
    };
    uint32_t tail_ph = 0;  // a bit per stage: phase of its next apart load
    if (CG == 2 && rank == 1) {
      // The second CTA of a pair issues nothing; it clears its tails and tells the first.
      while (MODE == kWeights && ok && tiles.next(v)) {
        for (int kb = 0; kb < v.k_blocks; ++kb) {
          if (v.hi - v.lo - kb * kBK < kBK) {
            ok = wait_phase_abort(full(s), tail_ph >> s & 1u, abort_flag, PONNI_B200_WAIT_LIMIT);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tail_ph ^= 1u << s;
            clear_tail(kb);
            if (lane == 0) mbar_arrive_cluster(mapa_shared(peer_full(s), 0));  // releases the cleared rows
          }
          next_stage();
        }
      }
      if (!ok && lane == 0) atomicOr(p.error, 1);
    } else {
      while (ok && tiles.next(v)) {
        for (int kb = 0; kb < v.k_blocks; ++kb) {
          const uint32_t d = tmem + (uint32_t)(buf * S::acc_cols);
          if (kb % S::segment == 0) {
            ok = wait_phase_abort(acc_empty(buf), acc_ph, abort_flag, PONNI_B200_WAIT_LIMIT);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
          ok = wait_phase_abort(full(s), ph, abort_flag, PONNI_B200_WAIT_LIMIT);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (MODE == kWeights && v.hi - v.lo - kb * kBK < kBK) {
            clear_tail(kb);
            if (CG == 2) {
              ok = wait_phase_abort_cluster(peer_full(s), tail_ph >> s & 1u, abort_flag, PONNI_B200_WAIT_LIMIT);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              tail_ph ^= 1u << s;
            }
          }
          tc_fence_after();
          const uint32_t stage = (uint32_t)s * S::stage_bytes;
          const uint32_t a0 = a_lo0 + (stage >> 4), b0 = b_lo0 + ((stage + S::a_bytes) >> 4);
          if constexpr (P == 1) {
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) mma(d, a0 + k * a_step, b0 + k * b_step, (kb % S::segment > 0 || k > 0) ? 1u : 0u);
          } else {
            constexpr uint32_t ap = kBM * kBK * 2 / 16, bp = S::b_rows * kBK * 2 / 16;
            constexpr int qa[6] = {1, 0, 2, 0, 1, 0}, qb[6] = {1, 2, 0, 1, 0, 0};
#pragma unroll
            for (int q = 0; q < 6; ++q)
#pragma unroll
              for (int k = 0; k < kBK / 16; ++k)
                mma(d, a0 + qa[q] * ap + k * a_step, b0 + qb[q] * bp + k * b_step, (q > 0 || k > 0) ? 1u : 0u);
          }
          commit(empty(s));
          if (kb % S::segment == S::segment - 1 || kb == v.k_blocks - 1) {
            if (!skip) commit(acc_full(buf));
            skip = false;
            if (++buf == S::acc_bufs) {
              buf = 0;
              acc_ph ^= 1u;
            }
          }
          next_stage();
        }
      }
      if (!ok) {
        if (lane == 0) atomicOr(p.error, 1);
        commit(drain);  // the MMAs issued so far, before TMEM is freed
        (void)mbar_wait_bounded(drain, 0);
      }
    }
  } else {
    // ------------------------------------------------------- epilogue ----
    const int quarter = warp & 3, part = ((warp - 2) >> 2) % S::parts, w = warp - 2;
    const int group = ((warp - 2) >> 2) / S::parts;
    Turns<S::groups> turns;
    constexpr int kChunks = S::part_cols / 32;
    unsigned char* stage = epi + w * (epi_total / kEpiWarps);
    int box = 0;  // of the store boxes
    float* bias_w = bias_s + w * 64;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int n_end = MODE == kRows ? p.inputs : p.outputs;
    int buf = 0, bias_e = -1, bias_n = -1;  // the strip whose bias lies in bias_w
    uint32_t acc_ph = 0;
    bool ok = true;
    auto wait_acc = [&]() -> bool {
      int got = 0;
      if (lane == 0) got = wait_phase_abort(acc_full(buf), acc_ph, abort_flag, PONNI_B200_WAIT_LIMIT) ? 1 : 0;
      got = __shfl_sync(0xffffffffu, got, 0);
      tc_fence_after();
      return got != 0;
    };
    auto next_acc = [&]() {
      if (++buf == S::acc_bufs) {
        buf = 0;
        acc_ph ^= 1u;
      }
    };
    auto release_acc = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) arrive_remote(mapa_shared(acc_empty(buf), 0));
        else mbar_arrive(acc_empty(buf));
      }
      next_acc();
    };
    while (ok && tiles.next(v)) {
      if (!turns.mine(group, v.k_blocks > 0, buf)) {
        if (v.k_blocks > 0) next_acc();
        continue;
      }
      const int m_end = MODE == kWeights ? p.inputs : v.hi - v.lo;
      const int row0 = v.m0 + quarter * 32, m_valid = min(32, m_end - row0);
      const int col0 = v.n0 + part * S::part_cols;
      if (MODE == kForward && p.bias && (v.e != bias_e || v.n0 != bias_n)) {
        bias_e = v.e;
        bias_n = v.n0;
        const T* bias = static_cast<const T*>(p.bias) + (int64_t)v.e * p.outputs;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const int n = col0 + i * 32 + lane;
          bias_w[i * 32 + lane] = n < n_end ? Num<T>::to_c(bias[n]) : 0.0f;
        }
        __syncwarp();
      }
      auto finish = [&](float (&x)[32], int c) {
        const int n = col0 + c * 32, n_valid = n_end - n;
        if (n_valid <= 0 || m_valid <= 0) return;
        if constexpr (P == 3) {
          bool nan = false;
#pragma unroll
          for (int i = 0; i < 32; ++i) nan |= x[i] != x[i];
          const int terms = MODE == kForward ? p.inputs : MODE == kRows ? p.outputs : v.hi - v.lo;
          if (__any_sync(0xffffffffu, nan && lane < m_valid) && terms <= kPlainTerms) {
            float y[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = x[i];
            plain_sums<MODE>(p, v.e, v.lo, v.hi, row0, m_valid, n, n_valid, y);
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = y[i];
          }
        }
        if (MODE == kForward) {
          if (p.bias) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 b = *reinterpret_cast<const float4*>(bias_w + c * 32 + i);
              f2::add(x[i], x[i + 1], x[i], x[i + 1], b.x, b.y);
              f2::add(x[i + 2], x[i + 3], x[i + 2], x[i + 3], b.z, b.w);
            }
          }
          activate_all<T>(x, p.act, p.act_flags, p.s0, p.s1);
        }
        if constexpr (S::bulk_store) {
          if (p.bulk && (MODE == kWeights || m_valid == 32)) {  // (rows past the weights' end are clipped)
            // 64-byte rows, 16-byte chunks swizzled by row / 2 as the tensor map has it.
            if (lane == 0) {
              if (p.boxes == 2) tma_store_wait_read<1>();
              else tma_store_wait_read<0>();
            }
            __syncwarp();
            const uint32_t dst = smem_u32(stage) + (uint32_t)box * 2048;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              st_shared_v4(dst + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4), pack2(x[8 * i], x[8 * i + 1], (T*)0),
                           pack2(x[8 * i + 2], x[8 * i + 3], (T*)0), pack2(x[8 * i + 4], x[8 * i + 5], (T*)0),
                           pack2(x[8 * i + 6], x[8 * i + 7], (T*)0));
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              if (MODE == kWeights) tma_store_3d(&map_c, n, row0, v.e, dst);
              else tma_store_3d(&map_c, n, v.lo + row0, 0, dst);
            }
            box ^= p.boxes - 1;
            return;
          }
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
        }
        if (MODE == kWeights) {
          if (p.unit_rows)
            store_rows<float>(x, stage, p.partial + (v.slot * p.inputs + row0) * p.outputs + n, p.outputs, m_valid,
                              n_valid, p.vec);
          else
            store_rows<T>(x, stage, static_cast<T*>(p.c) + ((int64_t)v.e * p.inputs + row0) * p.outputs + n, p.outputs,
                          m_valid, n_valid, p.vec);
        } else {
          store_rows<T>(x, stage, static_cast<T*>(p.c) + (int64_t)(v.lo + row0) * p.c_ld + n, p.c_ld, m_valid, n_valid,
                        p.vec);
        }
      };
      if (P == 1 && v.k_blocks > 0) {
        if (!(ok = wait_acc())) break;
        if (v.k_blocks > S::segment) {
          // A long sum: the accumulators of its segments added up, and put back in place of the last one.
          float sum[S::part_cols] = {};
#pragma unroll 1
          for (int kb = S::segment;; kb += S::segment) {
            const uint32_t t = tmem + lane_base + (uint32_t)(buf * S::acc_cols + part * S::part_cols);
#pragma unroll
            for (int i = 0; i < S::part_cols; i += 8) tmem_add8(t + i, sum + i);
            if (kb >= v.k_blocks) break;
            release_acc();
            if (!(ok = wait_acc())) break;
          }
          if (!ok) break;
          const uint32_t t = tmem + lane_base + (uint32_t)(buf * S::acc_cols + part * S::part_cols);
#pragma unroll
          for (int i = 0; i < S::part_cols; i += 8) tmem_st8(t + i, sum + i);
          asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
        }
        const uint32_t t = tmem + lane_base + (uint32_t)(buf * S::acc_cols + part * S::part_cols);
        // One chunk at a time: both at once is slower (239 against 202 us for 256 -> 256
        // without activation), the stores then come in bursts.
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
          float x[32];
          tmem_ld32(t + c * 32, x);
          if (c == kChunks - 1) release_acc();
          finish(x, c);
        }
      } else {
        float acc[kChunks][32] = {};
        if constexpr (P == 3) {
          for (int kb = 0; kb < v.k_blocks; ++kb) {
            if (!(ok = wait_acc())) break;
            const uint32_t t = tmem + lane_base + (uint32_t)(buf * S::acc_cols + part * S::part_cols);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              float x[32];
              tmem_ld32(t + c * 32, x);
              f2::add_n(acc[c], x);
            }
            release_acc();
          }
          if (!ok) break;
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) finish(acc[c], c);
      }
    }
    if (S::bulk_store && lane == 0) tma_store_wait_all();
    if (!ok && lane == 0) atomicOr(p.error, 1);
  }
  if (MODE != kWeights) {
    // Rows in no group.
    const int64_t used = clamped(p.offset[p.experts], 0, p.rows);
    const int n_end = MODE == kRows ? p.inputs : p.outputs;
    T* c = static_cast<T*>(p.c);
    for (int64_t r = used + blockIdx.x; r < p.rows; r += gridDim.x)
      for (int n = tid; n < n_end; n += kBlock) c[r * p.c_ld + n] = Num<T>::from_c(0.0f);
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) {
    // A role gave up: wait (bounded) for the copies in flight before the CTA ends.
    if (rank == 0) {
      for (int64_t i = issued > p.stages ? issued - p.stages : 0; i < issued; ++i)
        if (!mbar_wait_bounded(full((int)(i % p.stages)), (uint32_t)(i / p.stages) & 1u)) break;
    } else {  // counted by the other CTA: a millisecond is a thousand copies' time
      for (const long long t0 = clock64(); clock64() - t0 < 2000000;) __nanosleep(1000);
    }
  }
  if constexpr (CG == 2) cluster_sync();  // the pair's MMAs and copies, which use both CTAs' memory, are complete
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------ few rows ----
// Forward for groups of a few rows: a work item is up to 8 rows of a group (16 of
// fp32, whose thread holds half the columns), a
// block takes 128 columns and one of the cluster's slices of K.  A thread holds
// the sums of a vector of columns (16 bytes of weights: one load serves all of
// the item's rows) for every 8th or 16th k; the k groups are added in shared
// memory, the slices through the cluster's distributed shared memory, in a
// fixed order.  The rows of the item lie in shared memory as fp32.  Measured: two
// rows by two experts of 2048 x 1024 bf16 in 8.3 us alone (8.4 MB; launch and one
// pass's latency), one row by each of 64 experts of 1024 x 2048 fp32 in 92 us
// (5.8 TB/s).
constexpr int kFewThreads = 256, kFewCols = 128, kFewFloats = 8192;

template <class T> struct Few {
  static constexpr int vec = 16 / sizeof(T);           // columns of a thread
  static constexpr int lanes = kFewCols / vec;         // threads side by side
  static constexpr int groups = kFewThreads / lanes;   // k groups of the block
  static constexpr int rows = sizeof(T) == 4 ? 16 : 8;  // of an item
};

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Sums of RB rows over k in [0, kn) of the weights at w (row stride w_ld).
template <class T, int RB, bool VEC>
__device__ __forceinline__ void few_sums(const T* __restrict__ w, int64_t w_ld, int kn, int cols, const float* xs,
                                         float (&acc)[RB][Few<T>::vec]) {
  constexpr int V = Few<T>::vec, G = Few<T>::groups, U = RB * V > 32 ? 4 : 8;
  const int g = threadIdx.x / Few<T>::lanes;
  auto load = [&](int k) -> uint4 {
    const T* p = w + (int64_t)k * w_ld;
    if constexpr (VEC) {
      return cols >= V ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
    } else {
      alignas(16) T v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = i < cols ? p[i] : Num<T>::from_c(0.0f);
      return *reinterpret_cast<uint4*>(v);
    }
  };
  auto add = [&](const uint4& u, int k) {
    const T* t = reinterpret_cast<const T*>(&u);
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Num<T>::to_c(t[i]);
    float xr[RB];
    if constexpr (RB % 4 == 0) {
#pragma unroll
      for (int r = 0; r < RB; r += 4) {
        const float4 q = *reinterpret_cast<const float4*>(xs + k * RB + r);
        xr[r] = q.x;
        xr[r + 1] = q.y;
        xr[r + 2] = q.z;
        xr[r + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int r = 0; r < RB; ++r) xr[r] = xs[k * RB + r];
    }
    // Packed over two rows: their values come side by side out of shared memory.
    if constexpr (RB == 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) acc[0][i] = fmaf(f[i], xr[0], acc[0][i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int r = 0; r < RB; r += 2)
          f2::fma(acc[r][i], acc[r + 1][i], xr[r], xr[r + 1], f[i], f[i], acc[r][i], acc[r + 1][i]);
    }
  };
  int k = g;
  for (; k + (U - 1) * G < kn; k += U * G) {
    uint4 u[U];
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = load(k + i * G);
#pragma unroll
    for (int i = 0; i < U; ++i) add(u[i], k + i * G);
  }
  for (; k < kn; k += G) add(load(k), k);
}

template <class T, int RB, bool VEC>
__device__ void few_item(const Args& p, int e, int64_t row0, int n_rows, int n0, int slice, int slices, float* sm) {
  constexpr int V = Few<T>::vec, L = Few<T>::lanes, W = kFewThreads / 32;
  const int tid = threadIdx.x, x = tid % L, lane = tid & 31, warp = tid >> 5;
  const int per = (p.inputs + slices - 1) / slices, k_lo = slice * per, k_hi = min(p.inputs, k_lo + per);
  const T* rows = static_cast<const T*>(p.a) + row0 * p.a_ld;
  const int cols = p.outputs - (n0 + x * V);
  const T* w = static_cast<const T*>(p.b) + e * p.b_stride + (cols > 0 ? n0 + x * V : 0);
  float acc[RB][V] = {};
  constexpr int kStep = kFewFloats / RB < 1024 ? kFewFloats / RB : 1024;
  for (int k0 = k_lo; k0 < k_hi; k0 += kStep) {
    const int kn = min(kStep, k_hi - k0);
    __syncthreads();
    // A thread brings four k of up to four rows at a time and writes the rows of a
    // k side by side.
    constexpr int G = RB < 4 ? RB : 4, kAcross = kFewThreads / (RB / G);
    const int r0 = tid / kAcross * G;
    for (int k = tid % kAcross; k < kn; k += 4 * kAcross) {
      T v[4][G];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < G; ++r)
          v[j][r] = rows[min(r0 + r, n_rows - 1) * p.a_ld + k0 + min(k + j * kAcross, kn - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (k + j * kAcross >= kn) break;
        float* dst = sm + (k + j * kAcross) * RB + r0;
        float f[G];
#pragma unroll
        for (int r = 0; r < G; ++r) f[r] = r0 + r < n_rows ? Num<T>::to_c(v[j][r]) : 0.0f;
        if constexpr (G == 4) *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
        else if constexpr (G == 2) *reinterpret_cast<float2*>(dst) = make_float2(f[0], f[1]);
        else dst[0] = f[0];
      }
    }
    __syncthreads();
    few_sums<T, RB, VEC>(w + (int64_t)k0 * p.b_ld, p.b_ld, kn, cols, sm, acc);
  }
  if (L == 16) {
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[r][i] += __shfl_xor_sync(0xffffffffu, acc[r][i], 16);
  }
  // sm: [RB][kFewCols] sums of the block in front; behind them [W][H][kFewCols]
  // sums of the warps, H rows at a time.
  constexpr int H = RB < 4 ? RB : 4;
  float* part = sm + RB * kFewCols;
  static_assert((RB + W * H) * kFewCols <= kFewFloats, "sums of the warps");
  __syncthreads();
#pragma unroll
  for (int h = 0; h < RB; h += H) {
    if (lane < L) {
#pragma unroll
      for (int r = 0; r < H; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) part[(warp * H + r) * kFewCols + x * V + i] = acc[h + r][i];
    }
    __syncthreads();
    for (int i = tid; i < H * kFewCols; i += kFewThreads) {
      float s = 0.0f;
#pragma unroll
      for (int q = 0; q < W; ++q) s += part[q * H * kFewCols + i];
      sm[h * kFewCols + i] = s;
    }
    __syncthreads();
  }
  if (slices > 1) cluster_sync();
  T* out = static_cast<T*>(p.c) + row0 * p.c_ld;
  for (int i = slice * kFewThreads + tid; i < n_rows * kFewCols; i += slices * kFewThreads) {
    const int r = i / kFewCols, n = n0 + i % kFewCols;
    float s = 0.0f;
    if (slices > 1) {
      for (int q = 0; q < slices; ++q) s += ld_cluster(mapa_shared(smem_u32(sm + i), q));
    } else {
      s = sm[i];
    }
    if (n < p.outputs) {
      if (p.bias) s += Num<T>::to_c(static_cast<const T*>(p.bias)[(int64_t)e * p.outputs + n]);
      out[r * p.c_ld + n] = Num<T>::from_c(activate_one<T>(p.act, p.act_flags, s, p.s0, p.s1));
    }
  }
  if (slices > 1) cluster_sync();  // the others may still read this block's sums
}

template <class T, bool VEC>
__global__ void __launch_bounds__(kFewThreads, 2) few_rows_kernel(const Args p, int slices) {
  __shared__ __align__(16) float sm[kFewFloats];
  constexpr int kFewRows = Few<T>::rows;
  __shared__ int found[3];
  ops::let_successor_start();
  ops::wait_for_predecessor();
  const int tid = threadIdx.x, lane = tid & 31;
  const int strip = blockIdx.x / slices, slice = blockIdx.x % slices;
  if (tid < 32) {
    // The item's group: items in expert order, kFewRows rows each.
    int base = 0, e = -1, row0 = 0, n = 0;
    for (int e0 = 0; e0 < p.experts && e < 0; e0 += 32) {
      const int i = e0 + lane;
      int lo = 0, hi = 0;
      if (i < p.experts) {
        lo = clamped(p.offset[i], 0, p.rows);
        hi = clamped(p.offset[i + 1], lo, p.rows);
      }
      const int c = (hi - lo + kFewRows - 1) / kFewRows;
      int s = c;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, s, d);
        if (lane >= d) s += o;
      }
      const int first = base + s - c, want = (int)blockIdx.y;
      const unsigned hit = __ballot_sync(0xffffffffu, want >= first && want < first + c);
      if (hit) {
        const int src = __ffs(hit) - 1;
        e = e0 + src;
        row0 = __shfl_sync(0xffffffffu, lo + (want - first) * kFewRows, src);
        n = min(kFewRows, __shfl_sync(0xffffffffu, hi, src) - row0);
      }
      base += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) {
      found[0] = e;
      found[1] = row0;
      found[2] = n;
    }
  }
  if (blockIdx.x == 0 && blockIdx.y == 0) check_offsets(p.offset, p.experts, p.rows, p.error);
  if (blockIdx.y == 0) {
    const int64_t used = clamped(p.offset[p.experts], 0, p.rows);
    for (int64_t r = used + blockIdx.x; r < p.rows; r += gridDim.x)
      for (int n = tid; n < p.outputs; n += kFewThreads) static_cast<T*>(p.c)[r * p.c_ld + n] = Num<T>::from_c(0.0f);
  }
  __syncthreads();
  const int e = found[0], n = found[2];
  if (e < 0) return;  // the whole cluster: it has one item
  const int n0 = strip * kFewCols;
  if (n == 1) few_item<T, 1, VEC>(p, e, found[1], n, n0, slice, slices, sm);
  else if (n == 2) few_item<T, 2, VEC>(p, e, found[1], n, n0, slice, slices, sm);
  else if (n <= 4) few_item<T, 4, VEC>(p, e, found[1], n, n0, slice, slices, sm);
  else if (Few<T>::rows == 8 || n <= 8) few_item<T, 8, VEC>(p, e, found[1], n, n0, slice, slices, sm);
  else if constexpr (Few<T>::rows == 16) few_item<T, 16, VEC>(p, e, found[1], n, n0, slice, slices, sm);
}

// d_W_e = sum of its units' partial sums, in order.
template <class T>
__global__ void __launch_bounds__(256)
    sum_units_kernel(const float* __restrict__ partial, T* __restrict__ c, const int* __restrict__ offset, int experts,
                     int64_t rows, int unit_rows, int64_t per_expert) {
  __shared__ int64_t first_s;
  const int64_t most = slots(rows, unit_rows, experts);  // (offsets out of order would give more)
  ops::wait_for_predecessor();
  const int e = blockIdx.y;
  auto units_of = [&](int i) {
    const int l = clamped(offset[i], 0, rows);
    return units(clamped(offset[i + 1], l, rows) - l, unit_rows);
  };
  if (threadIdx.x < 32) {
    int64_t n = 0;
    for (int i = threadIdx.x; i < e; i += 32) n += units_of(i);
    for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
    if (threadIdx.x == 0) first_s = n;
  }
  __syncthreads();
  const int64_t first = min(first_s, most);
  const int n = (int)min(units_of(e), most - first);
  const float* src = partial + first * per_expert;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < per_expert; i += (int64_t)gridDim.x * 256) {
    float s = 0.0f;
#pragma unroll 4
    for (int u = 0; u < n; ++u) s += src[u * per_expert + i];
    c[e * per_expert + i] = Num<T>::from_c(s);
  }
}

// d_b_e: column sums of a group's rows.  A block sums one of `parts` equal parts
// of a group's rows over one strip of columns (16 bytes a lane where the rows
// allow it, else one element), in a fixed order; several parts are added by
// sum_parts_kernel.  d_out was just read by the products, so this reads L2.
template <class T, int V>
__global__ void __launch_bounds__(256)
    bias_gradient_kernel(const T* __restrict__ d, int64_t ld, int64_t rows, const int* __restrict__ offset, int outputs,
                         int parts, float* __restrict__ partial, T* __restrict__ out) {
  constexpr int kLanes = V > 1 ? 16 : 32, kGroups = 256 / kLanes, kCols = kLanes * V;
  __shared__ float sums[kGroups][kCols + 1];
  ops::let_successor_start();
  const int e = blockIdx.y, x = threadIdx.x % kLanes, y = threadIdx.x / kLanes, n = blockIdx.x * kCols + x * V;
  const int lo = clamped(offset[e], 0, rows), hi = clamped(offset[e + 1], lo, rows);
  const int64_t per = ((int64_t)hi - lo + parts - 1) / parts;
  const int64_t r0 = lo + blockIdx.z * per, r1 = min((int64_t)hi, r0 + per);
  float s[V] = {};
  if (n < outputs) {
    const T* p = d + n;
    if constexpr (V > 1) {
#pragma unroll 4
      for (int64_t r = r0 + y; r < r1; r += kGroups) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + r * ld));
        const T* v = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] += Num<T>::to_c(v[i]);
      }
    } else {
#pragma unroll 8
      for (int64_t r = r0 + y; r < r1; r += kGroups) s[0] += Num<T>::to_c(p[r * ld]);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) sums[y][x * V + i] = s[i];
  __syncthreads();
  for (int i = threadIdx.x; i < kCols; i += 256) {
    const int c = blockIdx.x * kCols + i;
    if (c >= outputs) break;
    float t = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) t += sums[g][i];
    if (parts == 1) out[(int64_t)e * outputs + c] = Num<T>::from_c(t);
    else partial[((int64_t)blockIdx.z * gridDim.y + e) * outputs + c] = t;
  }
}

template <class T>
__global__ void __launch_bounds__(256)
    sum_parts_kernel(const float* __restrict__ partial, T* __restrict__ out, int64_t n, int parts) {
  ops::wait_for_predecessor();
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.0f;
#pragma unroll 4
    for (int q = 0; q < parts; ++q) s += partial[q * n + i];
    out[i] = Num<T>::from_c(s);
  }
}

// ------------------------------------------------------------- staging ----
// An operand that the copy engine cannot read (fp32, or a base or stride off
// the 16-byte grid) is laid out in the workspace first: rows of `pitch`
// elements, fp32 as three bf16 planes.
struct Stage {
  const void* src;
  void* dst;
  int64_t rows, ld, group_rows, group_stride;  // source row r: (r / group_rows) * group_stride + (r % group_rows) * ld
  int cols, pitch;
  int vec;  // the source's rows start on 16-byte boundaries
};
struct Stages {
  Stage s[3];
  int n;
};

// Parts of two values, packed (x in the lower halves): each part is the nearest bf16 value to
// what the ones before leave, so that the products that are dropped are small and of either
// sign (parts cut off instead are four times as far off, always towards zero).
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&h)[3]) {
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    h[q] = pack2(x, y, (__nv_bfloat16*)0);
    if (q < 2) f2::sub(x, y, x, y, __uint_as_float(h[q] << 16), __uint_as_float(h[q] & 0xFFFF0000u));
  }
}
// What would round up past the largest bf16 is cut off in its first part; infinities and NaN
// stay whole in it.
constexpr uint32_t kLastRounded = 0x7F7F7FFFu;  // magnitude bits of the largest value that split_pair takes
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ void split_extreme(float x, float y, uint32_t (&h)[3]) {
  float v[2] = {x, y};
  uint32_t first[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool finite = magnitude(v[i]) < 0x7F800000u;
    first[i] = v[i] != v[i] ? 0x7FC00000u
               : magnitude(v[i]) > kLastRounded ? __float_as_uint(v[i]) & 0xFFFF0000u
                                                : (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v[i])) << 16;
    v[i] = finite ? v[i] - __uint_as_float(first[i]) : 0.0f;
  }
  split_pair(v[0], v[1], h);
  h[2] = h[1];
  h[1] = h[0];
  h[0] = pack_hi16(first[0], first[1]);
}

// A thread lays out 8 elements: one 16-byte store a plane.  (Two elements a thread,
// coalesced on both sides, issues more instructions than it saves: 29 to 47 us
// against 26 for two operands of 20011 x 301 and 20011 x 257.)
template <class T>
__global__ void __launch_bounds__(256) stage_kernel(const Stages all) {
  ops::let_successor_start();
  ops::wait_for_predecessor();
  const Stage& s = all.s[blockIdx.y];
  const int vecs = s.pitch / 8;
  int tx = 1;
  while (tx < vecs && tx < 256) tx *= 2;  // threads along a row
  const int x = threadIdx.x % tx, y = threadIdx.x / tx, ty = 256 / tx;
  const int64_t plane = s.rows * (int64_t)s.pitch;
  for (int64_t r = blockIdx.x * (int64_t)ty + y; r < s.rows; r += (int64_t)gridDim.x * ty) {
    const T* src = static_cast<const T*>(s.src) +
                   (s.group_rows == s.rows ? r * s.ld : r / s.group_rows * s.group_stride + r % s.group_rows * s.ld);
    for (int c = x; c < vecs; c += tx) {
      alignas(16) T v[8];
      if (s.vec && c * 8 + 8 <= s.cols) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
          reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(src + c * 8) + i);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c * 8 + i < s.cols ? __ldg(src + c * 8 + i) : Num<T>::from_c(0.0f);
      }
      if constexpr (sizeof(T) == 4) {
        uint32_t h[4][3], most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, magnitude(v[i]));
#pragma unroll
        for (int i = 0; i < 4; ++i) split_pair(v[2 * i], v[2 * i + 1], h[i]);
        if (most > kLastRounded) {
#pragma unroll
          for (int i = 0; i < 4; ++i) split_extreme(v[2 * i], v[2 * i + 1], h[i]);
        }
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(s.dst) + r * s.pitch + c * 8;
#pragma unroll
        for (int q = 0; q < 3; ++q)
          *reinterpret_cast<uint4*>(dst + q * plane) = make_uint4(h[0][q], h[1][q], h[2][q], h[3][q]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<T*>(s.dst) + r * s.pitch + c * 8) = *reinterpret_cast<uint4*>(v);
      }
    }
  }
}

// ---------------------------------------------------------------- host ----
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// An operand as the tensor maps describe it: [depth][rows][cols] of 16-bit
// elements (depth: planes, experts, or planes of experts).
struct Operand {
  const void* p;
  int64_t ld, stride;  // elements
  int64_t cols, rows, depth;
};

// box_cols: 64 elements of an operand (128-byte swizzle) or 32 of an output (64-byte).
ponni_b200_status make_map(CUtensorMap& map, const Operand& o, bool half, int box_rows, int box_cols = 64) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return ops::fail(PONNI_B200_ERR_CUDA, "expert_product: the driver has no tensor maps");
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.depth};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.depth > 1 ? o.stride : o.ld) * 2};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  if (strides[0] >= (1ull << 40) || strides[1] >= (1ull << 40) ||
      enc(&map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p),
          dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "expert_product: operand sizes or strides beyond the copy engine's");
  return PONNI_B200_OK;
}

bool on_grid(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * 2 % 16 == 0; }

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t staged_bytes(int dtype, int64_t rows, int cols) {
  return pad256(rows * pad8(cols) * (dtype == PONNI_B200_F32 ? 6 : 2));
}

// Tile width.  An MMA of 128 x 64 takes as long as one of 128 x 128 (58 and 64
// cycles for 16 k), so 64 is for products of at most 64 columns, whose sums (`terms` at
// most) fit one segment: its two groups of epilogue warps cannot share an accumulator's
// sums (2^18 rows, 64 experts, gradient of 1024 x 64: 119 us with 128 columns, 115 with 64
// and sums that drift; 20000 rows, 20 experts of 512 x 48: 21.5 and 19.5); 256 halves the
// reads of the row tile against 128 and is taken unless its padding costs over
// an eighth more columns, or the rows are so few that the weights' traffic
// decides (at most half a tile of rows a group): 128 then spreads them more evenly
// over the SMs.
int tile_width(int n, int64_t terms, int64_t rows, int experts, bool weights) {
  if (n <= 64 && terms <= kSegment * kBK) return 64;
  if (n <= 128 || (!weights && rows <= (int64_t)64 * experts)) return 128;
  auto padded = [&](int w) { return (int64_t)(n + w - 1) / w * w; };
  return padded(256) * 8 > padded(128) * 9 ? 128 : 256;
}

// Whether two CTAs share a tile of 256 rows: half the weight traffic, but more
// rows of padding at the end of a group.  16-bit rows x 1024 x 1024, 16 experts:
// 23.1 us against 22.2 in pairs with 256 rows each, 24.3 / 28.4 with 512, 39.7 / 36.6
// with 1024, 128.5 / 117.2 with 4096; the weight gradient has no such padding (31.1 /
// 28.8 with 512).  fp32 spends its time on the parts' traffic and the sums of every K
// block: 969.8 / 1060 with 4096 rows each, 4245 / 4170 with 16384.
bool use_pairs(int64_t rows, int experts, int mode, bool parts) {
  const int64_t least = parts ? 8192 : mode == kWeights ? 256 : 768;
  return rows >= least * experts;
}

struct TileShape {
  int columns, ctas;  // of a tile; its rows are 128 a CTA
};
TileShape tile_shape(int dtype, int mode, int64_t rows, int experts, int inputs, int outputs) {
  const bool parts = dtype == PONNI_B200_F32;
  const int64_t terms = mode == kForward ? inputs : mode == kRows ? outputs : rows;
  TileShape t = {tile_width(mode == kRows ? inputs : outputs, terms, rows, experts, mode == kWeights), 1};
  if (t.columns > 64 && use_pairs(rows, experts, mode, parts)) t.ctas = 2;
  if (parts && t.ctas == 1) t.columns = 128;
  return t;
}

// Rows of a unit of d_W: whole groups where their tiles fill the SMs twice or the
// groups are short (2048 rows on average, 512 of fp32: a split costs another
// launch, 9.5 us against 19 for 16 experts of 256 x 256 with 64 and 128 rows each);
// else so many that the tiles make about three waves (two leave the SMs a third
// idle where the last is ragged, more waves cost partial sums, 8 bytes an element of
// W_e and unit): 1024 rows at least, 256 of fp32, whose K blocks take four times as long.
int unit_rows_of(int dtype, int64_t rows, int experts, int inputs, int outputs, int sms) {
  const bool parts = dtype == PONNI_B200_F32;
  const TileShape t = tile_shape(dtype, kWeights, rows, experts, inputs, outputs);
  const int64_t m = t.ctas * kBM;
  const int64_t per = ((inputs + m - 1) / m) * ((outputs + t.columns - 1) / t.columns), slots = sms / t.ctas;
  if (per * experts >= 2 * slots || rows <= (int64_t)(parts ? 512 : 2048) * experts) return 0;
  const int64_t units = std::max<int64_t>(1, 3 * slots / per - experts / 2);  // a group's last unit is half full
  const int64_t unit = std::max<int64_t>(parts ? 256 : 1024, ((rows + units - 1) / units + kBK - 1) / kBK * kBK);
  return unit < rows ? (int)std::min<int64_t>(unit, 1 << 30) : 0;
}
int64_t partial_bytes(int dtype, int64_t rows, int experts, int inputs, int outputs, int sms) {
  const int unit = unit_rows_of(dtype, rows, experts, inputs, outputs, sms);
  return unit ? pad256(slots(rows, unit, experts) * inputs * outputs * 4) : 0;
}

// Parts of a group's rows in the bias gradient: about four blocks an SM, of 128
// rows at least on average.
int bias_parts(int64_t rows, int experts, int outputs, int sms) {
  const int64_t strips = (int64_t)experts * ((outputs + 127) / 128);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(64, rows / experts / 128), 4 * sms / strips));
}
int64_t bias_bytes(int64_t rows, int experts, int outputs, int sms) {
  const int parts = bias_parts(rows, experts, outputs, sms);
  return parts > 1 ? pad256((int64_t)parts * experts * outputs * 4) : 0;
}

// Hands out the caller's workspace.
struct Space {
  char* at;
  int64_t left;
  void* take(int64_t bytes) {
    if (bytes > left || !at) return nullptr;
    void* p = at;
    at += bytes;
    left -= bytes;
    return p;
  }
};

template <class T, int MODE, int P, int BN, int CG>
ponni_b200_status launch_shape(const Operand& a, const Operand& b, Args p, int sms, int64_t tiles, cudaStream_t stream) {
  using S = Shape<P, BN, CG>;
  CUtensorMap map_a, map_b, map_c;
  std::memset(&map_c, 0, sizeof map_c);
  constexpr bool half = std::is_same<T, __half>::value;
  ponni_b200_status st = make_map(map_a, a, half, MODE == kWeights ? 64 : kBM);
  if (!st) st = make_map(map_b, b, half, MODE == kRows ? S::b_rows : 64);
  p.bulk = S::bulk_store && p.vec && !p.unit_rows;
  if (!st && p.bulk) {
    const int64_t n = MODE == kRows ? p.inputs : p.outputs;
    const Operand c = MODE == kWeights ? Operand{p.c, n, n * p.inputs, n, p.inputs, p.experts}
                                       : Operand{p.c, p.c_ld, 0, n, p.rows, 1};
    st = make_map(map_c, c, half, 32, 32);
  }
  if (st) return st;
  const int k = MODE == kForward ? p.inputs : p.outputs;
  p.boxes = MODE != kWeights && k <= 8 * kBK ? 2 : 1;
  const int epi = epi_bytes<S>(p.boxes);
  const Memory memory = memory_of(S::stage_bytes, epi + kBiasBytes, p.experts);
  p.stages = memory.stages;
  auto kern = product_kernel<T, MODE, P, BN, CG>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = ops::allow_smem(reinterpret_cast<const void*>(kern), kDynamicBytes, p.device, allowed);
  if (e != cudaSuccess) return ops::fail_cuda(e, "expert_product");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(CG * std::max<int64_t>(1, std::min<int64_t>(sms / CG, tiles))));
  cfg.blockDim = dim3(kBlock);
  cfg.dynamicSmemBytes = memory.bytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, map_a, map_b, map_c, p);
  return e == cudaSuccess ? PONNI_B200_OK : ops::fail_cuda(e, "expert_product");
}

template <class T, int MODE>
ponni_b200_status launch_product(const Operand& a, const Operand& b, const Args& p, int sms, cudaStream_t stream) {
  constexpr int P = sizeof(T) == 4 ? 3 : 1;
  const int n = MODE == kRows ? p.inputs : p.outputs;
  const TileShape shape = tile_shape(P == 3 ? PONNI_B200_F32 : PONNI_B200_BF16, MODE, p.rows, p.experts, p.inputs, p.outputs);
  const int w = shape.columns, cg = shape.ctas, m = cg * kBM;
  const int64_t m_tiles = MODE == kWeights
                              ? (int64_t)((p.inputs + m - 1) / m) * (p.experts + (p.unit_rows ? p.rows / p.unit_rows : 0))
                              : p.rows / m + std::min<int64_t>(p.experts, p.rows);
  const int64_t tiles = m_tiles * ((n + w - 1) / w);
  if constexpr (P == 1) {
    if (w == 64) return launch_shape<T, MODE, P, 64, 1>(a, b, p, sms, tiles, stream);
  }
  if (w == 128)
    return cg == 2 ? launch_shape<T, MODE, P, 128, 2>(a, b, p, sms, tiles, stream)
                   : launch_shape<T, MODE, P, 128, 1>(a, b, p, sms, tiles, stream);
  if (cg == 2) return launch_shape<T, MODE, P, 256, 2>(a, b, p, sms, tiles, stream);
  if constexpr (P == 1) return launch_shape<T, MODE, P, 256, 1>(a, b, p, sms, tiles, stream);
  return ops::fail(PONNI_B200_ERR_UNSUPPORTED, "expert_product: no tile shape");
}

// Whether few_rows_kernel takes a forward product.  fp32: up to 48 rows a group on
// average; the tensor-core path has to lay out split copies of all weights first
// (64 experts of 1024 x 2048: 92 / 116 / 173 / 297 / 424 us with 1 / 8 / 16 / 32 / 48
// rows each against 415 to 434; 8 of 2048 x 1024: 13 / 24 / 71 with 1 / 16 / 48
// against 75).  16 bits: up to 8 rows where the 128-column tiles do not fill the SMs
// (8 experts of 2048 x 1024: 10.1 / 9.5 / 13.8 / 22.3 us with 1 / 4 / 8 / 12 rows each
// against 15.4 to 17.6; one expert of 2048 x 2048: 5.3 to 9.9 with 1 to 16 against
// 14.1); where they do, the tensor cores stream the weights as fast with any number
// of rows (64 experts of 1024 x 2048: 49.5 to 52 us against 54 with one row each, 94 with 8).
bool few_rows(int dtype, int64_t rows, int experts, int outputs, int sms) {
  if (dtype == PONNI_B200_F32) return rows <= (int64_t)48 * experts;
  const int64_t tiles = std::min<int64_t>(rows, experts) * ((outputs + 127) / 128);
  return tiles < sms && rows <= (int64_t)8 * (experts + 1);
}

template <class T>
ponni_b200_status launch_few(const Args& p, int sms, cudaStream_t stream) {
  const bool vec = reinterpret_cast<uintptr_t>(p.b) % 16 == 0 && p.b_ld * sizeof(T) % 16 == 0 &&
                   (p.experts == 1 || p.b_stride * sizeof(T) % 16 == 0) && p.outputs * sizeof(T) % 16 == 0;
  const int64_t strips = (p.outputs + kFewCols - 1) / kFewCols;
  const int64_t items = std::min<int64_t>(p.experts, p.rows) + p.rows / Few<T>::rows;
  // Slices of K until there are two blocks an SM, of 128 k at least.
  int slices = 1;
  while (slices < 8 && items * strips * slices < 2 * sms && p.inputs / (2 * slices) >= 128) slices *= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = slices;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(strips * slices), (unsigned)items);
  cfg.blockDim = dim3(kFewThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, few_rows_kernel<T, true>, p, slices)
                            : cudaLaunchKernelEx(&cfg, few_rows_kernel<T, false>, p, slices);
  return e == cudaSuccess ? PONNI_B200_OK : ops::fail_cuda(e, "expert_product");
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
  if (inputs < 1 || outputs < 1 || inputs > (1 << 24) || outputs > (1 << 24))
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": inputs and outputs must be 1 to 2^24");
  if (num_rows < 0 || num_rows > INT32_MAX - 65536)
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": the number of rows must be below 2^31 - 65536");
  if ((num_rows > 0 && !rows) || !weights || !offset || !aligned_to(element_bytes(dtype), rows, weights) ||
      !aligned_to(4, offset))
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": pointer is NULL or not aligned to its type");
  if (rows_ld < inputs || w_ld < outputs || (experts > 1 && w_stride < (int64_t)(inputs - 1) * w_ld + outputs))
    return fail(PONNI_B200_ERR_INVALID_ARGUMENT, at + ": stride smaller than the row or the expert");
  return PONNI_B200_OK;
}

// The operand as the product reads it: in place, or through the workspace.
ponni_b200_status operand(Operand& o, Stages& stages, Space& space, int dtype, const void* p, int64_t ld, int64_t stride,
                          int64_t rows, int cols, int64_t depth) {
  const int planes = dtype == PONNI_B200_F32 ? 3 : 1;
  if (planes == 1 && on_grid(p, ld) && (depth == 1 || stride % 8 == 0)) {
    o = {p, ld, stride, cols, rows, depth};
    return PONNI_B200_OK;
  }
  const int64_t pitch = pad8(cols);
  void* dst = space.take(staged_bytes(dtype, rows * depth, cols));
  if (!dst) return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product: workspace is too small");
  o = {dst, pitch, rows * pitch, cols, rows, depth * planes};
  const int64_t z = ops::element_bytes(dtype);
  const bool vec = reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * z % 16 == 0 && (depth == 1 || stride * z % 16 == 0);
  stages.s[stages.n++] = {p, dst, rows * depth, ld, rows, stride, cols, (int)pitch, vec};
  return PONNI_B200_OK;
}

template <class T>
ponni_b200_status run_stages(const Stages& st, int sms, cudaStream_t s) {
  if (!st.n) return PONNI_B200_OK;
  int64_t most = 1;
  for (int i = 0; i < st.n; ++i) {
    most = std::max(most, (st.s[i].rows * st.s[i].pitch + 2047) / 2048);
  }
  stage_kernel<T><<<dim3((unsigned)std::min<int64_t>(most, sms * 8), st.n), 256, 0, s>>>(st);
  return ops::launched("expert_product");
}

}  // namespace
}  // namespace ponni_b200

using namespace ponni_b200;

extern "C" {

int64_t ponni_b200_expert_product_workspace(int dtype, int64_t num_rows, int experts, int inputs, int outputs,
                                            int aligned, int backward, int device) {
  if (num_rows < 0 || experts < 1 || inputs < 1 || outputs < 1) return 0;
  int64_t n = 0;
  if (!backward && few_rows(dtype, num_rows, experts, outputs, ops::num_sms(device))) return 0;
  if (dtype == PONNI_B200_F32 || !aligned) {
    n += staged_bytes(dtype, num_rows, inputs) + staged_bytes(dtype, (int64_t)experts * inputs, outputs);
    if (backward) n += staged_bytes(dtype, num_rows, outputs);
  }
  if (backward)
    n += partial_bytes(dtype, num_rows, experts, inputs, outputs, ops::num_sms(device)) +
         bias_bytes(num_rows, experts, outputs, ops::num_sms(device));
  return n;
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
    if (!out || !ops::aligned_to(ops::element_bytes(dtype), out, bias) || !ops::aligned_to(256, workspace))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product: pointer is NULL or not aligned");
    if (out_ld < outputs)
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product: stride smaller than the row");
    Args p = {};
    p.a = rows;
    p.b = weights;
    p.c = out;
    p.a_ld = rows_ld;
    p.b_ld = w_ld;
    p.b_stride = w_stride;
    p.c_ld = out_ld;
    p.rows = num_rows;
    p.offset = offset;
    p.bias = bias;
    p.experts = experts;
    p.inputs = inputs;
    p.outputs = outputs;
    p.act = activation < 0 ? EPI_NONE : activation;
    p.act_flags = activation_flags;
    p.s0 = (float)scalar0;
    p.s1 = (float)scalar1;
    p.device = device;
    p.error = ops::error_word(device);
    if (!p.error) return ops::fail(PONNI_B200_ERR_CUDA, "no operator error word on this device");
    const int sms = ops::num_sms(device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (few_rows(dtype, num_rows, experts, outputs, sms)) return by_type(dtype, [&](auto t) { return launch_few<decltype(t)>(p, sms, s); });
    Stages stages = {};
    Space space = {static_cast<char*>(workspace), workspace_bytes};
    Operand a, b;
    st = operand(a, stages, space, dtype, rows, rows_ld, 0, num_rows, inputs, 1);
    if (!st) st = operand(b, stages, space, dtype, weights, w_ld, w_stride, inputs, outputs, experts);
    if (st) return st;
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      p.vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_ld * sizeof(T) % 16 == 0;
      ponni_b200_status r = run_stages<T>(stages, sms, s);
      return r ? r : launch_product<T, kForward>(a, b, p, sms, s);
    });
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
    if ((num_rows > 0 && !d_out) || !ops::aligned_to(ops::element_bytes(dtype), d_out, d_rows, d_weights, d_bias) ||
        !ops::aligned_to(256, workspace))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product_backward: pointer is NULL or not aligned");
    if (d_out_ld < outputs || (d_rows && d_rows_ld < inputs))
      return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product_backward: stride smaller than the row");
    const int sms = ops::num_sms(device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int* error = ops::error_word(device);
    if (!error) return ops::fail(PONNI_B200_ERR_CUDA, "no operator error word on this device");
    if (num_rows == 0) {  // the gradients of experts without rows
      const size_t z = ops::element_bytes(dtype);
      cudaError_t e = cudaSuccess;
      if (d_weights) e = cudaMemsetAsync(d_weights, 0, z * experts * inputs * outputs, s);
      if (e == cudaSuccess && d_bias) e = cudaMemsetAsync(d_bias, 0, z * experts * outputs, s);
      return e == cudaSuccess ? PONNI_B200_OK : ops::fail_cuda(e, "expert_product_backward");
    }
    Stages stages = {};
    Space space = {static_cast<char*>(workspace), workspace_bytes};
    Operand x, w, d;
    if (d_rows || d_weights) st = operand(d, stages, space, dtype, d_out, d_out_ld, 0, num_rows, outputs, 1);
    if (!st && d_rows) st = operand(w, stages, space, dtype, weights, w_ld, w_stride, inputs, outputs, experts);
    if (!st && d_weights) st = operand(x, stages, space, dtype, rows, rows_ld, 0, num_rows, inputs, 1);
    const int unit = unit_rows_of(dtype, num_rows, experts, inputs, outputs, sms);
    void* partial = nullptr;
    if (!st && d_weights && unit) {
      partial = space.take(partial_bytes(dtype, num_rows, experts, inputs, outputs, sms));
      if (!partial) st = ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product_backward: workspace is too small");
    }
    const int parts = bias_parts(num_rows, experts, outputs, sms);
    float* bias_partial = nullptr;
    if (!st && d_bias && parts > 1) {
      bias_partial = static_cast<float*>(space.take(bias_bytes(num_rows, experts, outputs, sms)));
      if (!bias_partial) st = ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT, "expert_product_backward: workspace is too small");
    }
    if (st) return st;
    return by_type(dtype, [&](auto t) -> ponni_b200_status {
      using T = decltype(t);
      Args p = {};
      p.rows = num_rows;
      p.offset = offset;
      p.experts = experts;
      p.inputs = inputs;
      p.outputs = outputs;
      p.device = device;
      p.error = error;
      ponni_b200_status r = run_stages<T>(stages, sms, s);
      if (!r && d_rows) {
        Args q = p;
        q.a = d_out;
        q.a_ld = d_out_ld;
        q.b = weights;
        q.b_ld = w_ld;
        q.b_stride = w_stride;
        q.c = d_rows;
        q.c_ld = d_rows_ld;
        q.vec = reinterpret_cast<uintptr_t>(d_rows) % 16 == 0 && d_rows_ld * sizeof(T) % 16 == 0;
        r = launch_product<T, kRows>(d, w, q, sms, s);
      }
      if (!r && d_weights) {
        Args q = p;
        q.a = rows;
        q.a_ld = rows_ld;
        q.b = d_out;
        q.b_ld = d_out_ld;
        q.c = d_weights;
        q.partial = static_cast<float*>(partial);
        q.unit_rows = unit;
        const size_t z = unit ? 4 : sizeof(T);
        q.vec = reinterpret_cast<uintptr_t>(unit ? partial : d_weights) % 16 == 0 && outputs * z % 16 == 0;
        r = launch_product<T, kWeights>(x, d, q, sms, s);
        if (!r && unit) {
          const int64_t per = (int64_t)inputs * outputs;
          const unsigned blocks = (unsigned)std::min<int64_t>((per + 255) / 256, std::max(1, sms * 8 / experts));
          const cudaError_t e =
              ops::launch_after(sum_units_kernel<T>, dim3(blocks, experts), dim3(256), 0, s, (const float*)partial,
                                static_cast<T*>(d_weights), offset, experts, num_rows, unit, per);
          if (e != cudaSuccess) r = ops::fail_cuda(e, "expert_product_backward");
        }
      }
      if (!r && d_bias) {
        constexpr int V = 16 / sizeof(T);
        const bool vec = reinterpret_cast<uintptr_t>(d_out) % 16 == 0 && d_out_ld % V == 0 && outputs % V == 0;
        const int cols = vec ? 16 * V : 32;
        const dim3 grid((outputs + cols - 1) / cols, experts, parts);
        auto kern = vec ? bias_gradient_kernel<T, V> : bias_gradient_kernel<T, 1>;
        kern<<<grid, 256, 0, s>>>(static_cast<const T*>(d_out), d_out_ld, num_rows, offset, outputs, parts, bias_partial,
                                  static_cast<T*>(d_bias));
        r = ops::launched("expert_product_backward");
        if (!r && parts > 1) {
          const int64_t n = (int64_t)experts * outputs;
          const cudaError_t e = ops::launch_after(sum_parts_kernel<T>, dim3((unsigned)std::min<int64_t>((n + 255) / 256, sms * 4)),
                                                  dim3(256), 0, s, (const float*)bias_partial, static_cast<T*>(d_bias), n, parts);
          if (e != cudaSuccess) r = ops::fail_cuda(e, "expert_product_backward");
        }
      }
      return r;
    });
  });
}

}  // extern "C"
