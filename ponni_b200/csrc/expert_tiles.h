// The tile sequence of the products grouped by expert (expert_product.cu), which
// every role of the kernel derives for itself, and which epilogue warps take a
// tile.  Plain index arithmetic, compiled for the host too (tests/cpp/test_expert_tiles.cpp).
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define PONNI_B200_HD __host__ __device__ __forceinline__
#else
#define PONNI_B200_HD inline
#endif

namespace ponni_b200 {
namespace grouped {

enum Mode { kForward, kRows, kWeights };

constexpr int kBM = 128, kBK = 64;

struct Tile {
  int e, m0, n0;
  int lo, hi;    // kForward, kRows: the group's rows; kWeights: the unit's
  int k_blocks;
  int64_t slot;  // kWeights, split: the unit's partial sums
};

struct Sizes {
  int experts, inputs, outputs;
  int unit_rows;  // kWeights: rows of a unit (a multiple of kBK); 0: a group is one unit
};

// A bound of a group as the caller's offset has it, kept within the rows.
PONNI_B200_HD int bound(int offset, int64_t rows) { return offset < 0 ? 0 : offset > rows ? (int)rows : offset; }
// Bounds that descend somewhere (which is reported) become a running maximum: the
// groups stay disjoint, so that all of them together have no more units than slots().
PONNI_B200_HD void ascending(int* edge, int experts) {
  for (int e = 1; e <= experts; ++e)
    if (edge[e] < edge[e - 1]) edge[e] = edge[e - 1];
}
// Units of a group (the sum of both may pass 2^31).
PONNI_B200_HD int64_t units(int64_t rows, int64_t unit_rows) { return (rows + unit_rows - 1) / unit_rows; }
// Units of all groups at most: every group's last one may be short.
PONNI_B200_HD int64_t slots(int64_t rows, int unit_rows, int experts) { return rows / unit_rows + experts; }

// The tile sequence of a CTA (pair): tile `first`, then every `step`-th one, of
// all tiles: experts in order, row tiles innermost (neighbours share the weight
// tile).  m0 is the first row of CTA `rank` of the pair.
template <int MODE, int BN, int CG> struct Tiles {
  const int* edge;  // bounds of the groups (bound, ascending): group e is [edge[e], edge[e + 1])
  int experts, m_tiles, n_tiles, k_blocks, unit_rows, rank;
  int e = 0;
  int64_t t, step, base = 0;

  PONNI_B200_HD Tiles(const Sizes& p, const int* edge_, int64_t first, int64_t step_, int rank_)
      : edge(edge_), experts(p.experts), unit_rows(p.unit_rows), rank(rank_), t(first), step(step_) {
    const int n = MODE == kRows ? p.inputs : p.outputs, k = MODE == kForward ? p.inputs : p.outputs;
    m_tiles = (p.inputs + CG * kBM - 1) / (CG * kBM);
    n_tiles = (n + BN - 1) / BN;
    k_blocks = (k + kBK - 1) / kBK;
  }
  PONNI_B200_HD int64_t count(int i) const {
    const int rows = edge[i + 1] - edge[i];
    if (MODE != kWeights) return (int64_t)((rows + CG * kBM - 1) / (CG * kBM)) * n_tiles;
    return (unit_rows ? units(rows, unit_rows) : 1) * m_tiles * n_tiles;
  }
  PONNI_B200_HD bool next(Tile& v) {
    int64_t c = 0;
    while (e < experts && t >= base + (c = count(e))) {
      base += c;
      ++e;
    }
    if (e >= experts) return false;
    const int64_t local = t - base;
    t += step;
    v.e = e;
    v.lo = edge[e];
    v.hi = edge[e + 1];
    if (MODE != kWeights) {
      const int m = (v.hi - v.lo + CG * kBM - 1) / (CG * kBM);
      v.n0 = (int)(local / m) * BN;
      v.m0 = (int)(local % m) * CG * kBM;
      v.k_blocks = k_blocks;
    } else {
      const int per = m_tiles * n_tiles;
      const int unit = (int)(local / per), i = (int)(local % per);
      v.m0 = i % m_tiles * CG * kBM;
      v.n0 = i / m_tiles * BN;
      v.slot = base / per + unit;
      if (unit_rows) {
        v.lo += unit * unit_rows;
        if (v.hi - v.lo > unit_rows) v.hi = v.lo + unit_rows;  // (their sum may pass 2^31)
      }
      v.k_blocks = (v.hi - v.lo + kBK - 1) / kBK;
    }
    if (CG == 2) v.m0 += kBM * rank;
    return true;
  }
};

// Which of GROUPS groups of epilogue warps takes a tile.  A parity wait tells a
// barrier's next phase from the present one, not from the one after the next, so a
// group may not wait for a use of an accumulator before the use before it is
// over.  Tiles therefore go by the accumulator that they use: with an even number of
// them each belongs to one group, which has waited for its use before.  Tiles without
// sums (experts without rows) use none; they are dealt out by a count of their own.
template <int GROUPS> struct Turns {
  int empty = 0;
  PONNI_B200_HD bool mine(int group, bool sums, int buf) {
    return GROUPS == 1 || (sums ? buf : empty++) % GROUPS == group;
  }
};

// Shared memory of the kernel.  A block has 227 KB, static and dynamic together;
// kStaticBytes of them cover the static part (barriers, the TMEM address).  The launch asks
// for `bytes`, and the kernel is allowed kDynamicBytes.
constexpr int kStaticBytes = 512, kDynamicBytes = 232448 - kStaticBytes, kMaxStages = 8;
struct Memory {
  int stages, bytes;
};
// Stages of `stage_bytes` beside `other` bytes and the groups' bounds; 1024 bytes align the first stage.
inline Memory memory_of(int stage_bytes, int other, int experts) {
  const int fixed = 1024 + other + (experts + 1) * (int)sizeof(int), fit = (kDynamicBytes - fixed) / stage_bytes;
  const int stages = fit < kMaxStages ? fit : kMaxStages;
  return {stages, fixed + stages * stage_bytes};
}

}  // namespace grouped
}  // namespace ponni_b200
