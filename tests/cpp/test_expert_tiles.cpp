// Host checks of the grouped product's tile sequence (ponni_b200/csrc/expert_tiles.h).
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "expert_tiles.h"

using namespace ponni_b200::grouped;

static int failures = 0;
#define CHECK(c, ...)                            \
  do {                                           \
    if (!(c)) {                                  \
      if (++failures < 20) {                     \
        std::printf("%s: ", #c);                 \
        std::printf(__VA_ARGS__);                \
        std::printf("\n");                       \
      }                                          \
    }                                            \
  } while (0)

using Groups = std::vector<int>;  // bounds
static Groups groups_of(const std::vector<int>& rows) {
  Groups g = {0};
  for (int r : rows) g.push_back(g.back() + r);
  return g;
}

// Accumulators complete in the order of the CTA's tiles.  A wait for use n of an
// accumulator by its parity is safe once use n - 1 is known to be over: the same
// group has waited for that use or for a later accumulator of the sequence.
template <int BN, int GROUPS, int BUFS>
static void check_waits(const Sizes& p, const Groups& g, int ctas) {
  for (int cta = 0; cta < ctas; ++cta)
    for (int group = 0; group < GROUPS; ++group) {
      Tiles<kWeights, BN, 1> tiles(p, g.data(), cta, ctas, 0);
      Turns<GROUPS> turns;
      Tile v;
      int64_t sums = 0, known = -1;  // accumulators so far; the last one known to be complete
      while (tiles.next(v)) {
        const int64_t at = sums;
        const bool mine = turns.mine(group, v.k_blocks > 0, (int)(at % BUFS));
        if (v.k_blocks > 0) ++sums;
        if (!mine || v.k_blocks == 0) continue;
        CHECK(known >= at - BUFS, "%d experts, CTA %d, group %d: accumulator %lld awaited while %lld is the last known",
              p.experts, cta, group, (long long)at, (long long)known);
        known = at;
      }
    }
}

// Every tile of every CTA is taken by one group.
template <int BN, int GROUPS, int BUFS>
static void check_taken(const Sizes& p, const Groups& g, int ctas) {
  for (int cta = 0; cta < ctas; ++cta) {
    std::vector<int> taken;
    for (int group = 0; group < GROUPS; ++group) {
      Tiles<kWeights, BN, 1> tiles(p, g.data(), cta, ctas, 0);
      Turns<GROUPS> turns;
      Tile v;
      int64_t sums = 0;
      size_t i = 0;
      while (tiles.next(v)) {
        if (taken.size() <= i) taken.push_back(0);
        taken[i++] += turns.mine(group, v.k_blocks > 0, (int)(sums % BUFS));
        if (v.k_blocks > 0) ++sums;
      }
    }
    for (int t : taken) CHECK(t == 1, "a tile of CTA %d is taken %d times", cta, t);
  }
}

static void empty_groups() {
  // Empty and long groups in an order that gives one group of warps four accumulators in a row.
  check_waits<64, 2, 4>({8, 18944, 64, 0}, groups_of({4096, 0, 4096, 0, 4096, 0, 4096, 4096}), 148);
  std::mt19937 rng(1);
  for (int experts : {2, 16, 64, 128, 256, 1024})
    for (double empty : {0.0, 0.2, 0.5, 0.9})
      for (int inputs : {64, 300, 1024, 2048})
        for (int round = 0; round < 5; ++round) {
          std::vector<int> rows(experts);
          for (int& r : rows) r = std::uniform_real_distribution<>(0, 1)(rng) < empty ? 0 : 1 + (int)(rng() % 300);
          const Groups g = groups_of(rows);
          const Sizes p = {experts, inputs, 64, 0};
          check_waits<64, 2, 4>(p, g, 148);
          check_taken<64, 2, 4>(p, g, 148);
        }
}

// All tiles together cover every group's rows and columns once.
template <int MODE, int BN, int CG>
static void check_cover(const Sizes& p, const Groups& g, int ctas) {
  const int m_all = MODE == kWeights ? (p.inputs + kBM - 1) / kBM : 0;
  const int n_tiles = ((MODE == kRows ? p.inputs : p.outputs) + BN - 1) / BN;
  int64_t want = 0, got = 0;
  for (int e = 0; e < p.experts; ++e) {
    const int rows = g[e + 1] - g[e];
    if (MODE != kWeights) want += (int64_t)((rows + kBM - 1) / kBM) * n_tiles;
    else want += (int64_t)m_all * n_tiles * (p.unit_rows ? (rows + p.unit_rows - 1) / p.unit_rows : 1);
  }
  std::vector<char> seen;
  for (int cta = 0; cta < ctas * CG; ++cta) {
    Tiles<MODE, BN, CG> tiles(p, g.data(), cta / CG, ctas, cta % CG);
    Tile v;
    while (tiles.next(v)) {
      const int m_end = MODE == kWeights ? p.inputs : v.hi - v.lo;
      CHECK(v.e >= 0 && v.e < p.experts && v.lo >= g[v.e] && v.hi <= g[v.e + 1] && v.m0 % kBM == 0, "expert %d", v.e);
      if (v.m0 < m_end) ++got;
    }
  }
  CHECK(got == want, "%lld tiles, not %lld", (long long)got, (long long)want);
}

static void cover() {
  const Groups g = groups_of({0, 1, 128, 129, 0, 1000, 255, 256, 257, 0});
  for (int inputs : {1, 128, 300})
    for (int outputs : {1, 64, 129, 700}) {
      check_cover<kForward, 128, 1>({10, inputs, outputs, 0}, g, 7);
      check_cover<kForward, 256, 2>({10, inputs, outputs, 0}, g, 7);
      check_cover<kRows, 64, 1>({10, inputs, outputs, 0}, g, 7);
      check_cover<kWeights, 128, 2>({10, inputs, outputs, 0}, g, 7);
      check_cover<kWeights, 64, 1>({10, inputs, outputs, 128}, g, 7);
    }
}

// Offsets of any kind: every tile lies within the rows, every unit has its slot.
static void offsets_out_of_order() {
  std::mt19937 rng(2);
  for (int experts : {1, 2, 9, 64, 1024})
    for (int rows : {1, 5000, 100000})
      for (int round = 0; round < 20; ++round) {
        const int unit = 256;
        std::vector<int> edge(experts + 1);
        for (int e = 0; e <= experts; ++e) {
          int o = round == 0 ? (e % 2) * rows : (int)(rng() % (2 * rows)) - rows / 2;
          if (round == 1) o = e % 2 ? INT32_MAX : INT32_MIN;
          edge[e] = bound(o, rows);
        }
        ascending(edge.data(), experts);
        Tiles<kWeights, 128, 1> tiles({experts, 128, 128, unit}, edge.data(), 0, 1, 0);
        Tile v;
        while (tiles.next(v))
          CHECK(v.lo >= 0 && v.lo <= v.hi && v.hi <= rows && v.slot >= 0 && v.slot < slots(rows, unit, experts),
                "%d experts, %d rows: rows %d to %d in slot %lld of %lld", experts, rows, v.lo, v.hi, (long long)v.slot,
                (long long)slots(rows, unit, experts));
      }
}

// Groups near the largest number of rows, in long units.
static void long_groups() {
  const int most = INT32_MAX - 65536, unit = 715000000 / kBK * kBK;
  const Groups g = {0, 100, 1900000000, most};
  Tiles<kWeights, 128, 1> tiles({3, 128, 128, unit}, g.data(), 0, 1, 0);
  Tile v;
  int64_t rows = 0;
  while (tiles.next(v)) {
    CHECK(v.lo >= g[v.e] && v.lo < v.hi && v.hi <= g[v.e + 1] && v.hi - v.lo <= unit, "rows %d to %d", v.lo, v.hi);
    CHECK(v.k_blocks == (v.hi - v.lo + kBK - 1) / kBK, "%d blocks", v.k_blocks);
    rows += v.hi - v.lo;
  }
  CHECK(rows == most, "%lld rows", (long long)rows);
}

// Every launch asks for no more than the kernel is allowed, for every number of experts:
// stages of 24 to 96 KB (tile shapes), staging of 24, 32 and 64 KB, a bias strip a warp.
static void memory() {
  for (int stage : {24576, 32768, 49152, 98304})
    for (int epi : {24576, 32768, 65536})
      for (int experts = 1; experts <= 1024; ++experts) {
        if (stage == 98304 && epi > 24576) continue;  // (fp32 parts: the small staging)
        const Memory m = memory_of(stage, epi + 4096, experts);
        CHECK(m.stages >= 1 && m.bytes <= kDynamicBytes && m.bytes + kStaticBytes <= 227 * 1024,
              "%d experts, stages of %d: %d bytes", experts, stage, m.bytes);
      }
}

int main() {
  memory();
  offsets_out_of_order();
  long_groups();
  empty_groups();
  cover();
  if (failures) std::printf("%d failures\n", failures);
  return failures != 0;
}
