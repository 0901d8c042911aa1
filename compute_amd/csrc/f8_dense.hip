// Dense product over 8-bit floating-point blocks: the choice of a kernel, and the tiles with direct loads
// (f8_dense_tiles.h has the kernel; f8_dense_staged.hip its form for unaligned operands).
#include "f8_dense_tiles.h"

namespace mx {
namespace {
using namespace f8;

using Tile256x256 = DenseTile<4, 2, 8, 2>;  // columns x rows
using Tile256x128 = DenseTile<4, 2, 4, 3>;
using Tile128x128 = DenseTile<2, 4, 2, 3>;  // (with one more buffer the smaller tiles are up to 5% slower)
using Tile128x64 = DenseTile<2, 2, 2, 3>;   // three: two workgroups a CU
using Tile64x128 = DenseTile<1, 4, 2, 3>;
using Tile64x64 = DenseTile<1, 2, 2, 4>;

enum class DensePlan { kSkinny, kTiles, kStaged };
struct DenseChoice {
  DensePlan plan;
  int tile, slices;
};

// The tile and the number of K slices that take the least time by the times of their parts: a launch 3 us; a
// round of workgroups its first loads and its stores 4.5 us, and a step of 128 k (below, us, with every CU at work); for sums
// that meet in scratch 1.2 us, 0.3 us a slice and their bytes, out and back, at 14 TB/s (they mostly stay in the
// caches).  Against sweeps of all of them at 28 shapes (profiles/f8_tile_sweeps.txt, with the steps measured by themselves) the choice
// is within 3% of the best at 26, and 10% behind at 200 and 256 rows of 4096 x 4096, for instance (us, columns x rows, slices, bfloat16
// results)
//   [97,4096] x 14336     128x128 in two 20.4, 64x128 in two 20.9, 128x64 21.0, 256x128 in three 24.5
//   [256,4096] x 4096     128x64 in two 15.6, 64x128 in two 16.1, 128x128 in three 16.7 (the choice: in four 17.2)
//   [512,4096] x 11008    256x128 35.5, 256x256 in two 44.1, 128x64 46.9
//   [2048,4096] x 4096    256x128 42.2, 256x256 51.3, 128x128 56.8
//   [4096,4096] x 4096    256x256 66.6 (2.06 PFLOP/s), 256x128 84.2, 128x128 117
//   [2048,4096] x 14336   256x256 119, 256x128 154, 128x64 200
struct TileCost {
  int cols, rows, threads, slots;  // threads of a workgroup, workgroups at once on 256 CUs
  float step, wide_step;  // (float32 results)
  float alone, wide_alone;  // with at most one workgroup a CU
  bool staged;              // also built for chunks through registers
};
constexpr float kNever = 1e9f;  // not built: bfloat16 operands of eight groups have no registers, and two workgroups of half
                                // the 128 x 128 tile take less than its 1.34 a step (and 1.20 alone), whatever the sizes
constexpr TileCost kTileCosts[] = {{256, 256, 512, 256, 1.82f, kNever, 1.82f, kNever, false},
                                   {256, 128, 512, 256, 1.10f, 2.05f, 1.10f, 2.05f, false},
                                   {128, 128, 512, 256, 0.73f, kNever, 0.58f, kNever, true},
                                   {128, 64, 256, 512, 0.80f, 1.15f, 0.44f, 0.76f, true},
                                   {64, 128, 256, 512, 0.80f, 1.15f, 0.43f, 0.74f, false},
                                   {64, 64, 128, 512, 0.65f, 1.05f, 0.40f, 0.68f, true}};

DenseChoice dense_plan(const F8DenseDesc& d) {
  if (skinny_fits(d)) return {DensePlan::kSkinny, 0, 1};
  // The direct loads take whole aligned 16-byte chunks of rows and 32-bit offsets; others come through registers.
  const bool direct = d.K == 0 || (d.K % 16 == 0 && (d.oi || d.N % 16 == 0) && aligned16(d.x) && aligned16(d.w) && d.K <= 1 << 21 &&
                                   d.N <= 1 << 21);
  const bool wide = d.out_dt == MX_DTYPE_FLOAT32;
  const int64_t KB = blocks(d.K);
  DenseChoice best{direct ? DensePlan::kTiles : DensePlan::kStaged, 1, 1};
  double least = 1e30;
  for (int t = 0; t < (int)(sizeof(kTileCosts) / sizeof(kTileCosts[0])); ++t) {
    const TileCost& c = kTileCosts[t];
    if (!direct && !c.staged) continue;
    const int64_t tiles = ((d.M + c.rows - 1) / c.rows) * ((d.N + c.cols - 1) / c.cols);
    for (int S = 1; S <= 16 && S <= KB; ++S) {
      const int64_t per = (KB + S - 1) / S, used = (KB + per - 1) / per;  // slices that are not empty
      const double part = (double)tiles * (double)used * c.rows * c.cols * 4;
      if (tiles * S * c.threads > kMaxWorkItems) continue;
      if (S > 1 && (used != S || tiles > (int64_t)(kScratchCounterBytes / 4) || part > 64e6)) continue;
      const bool alone = tiles * S <= 256;
      const double step = wide ? (alone ? c.wide_alone : c.wide_step) : alone ? c.alone : c.step;
      const double us = 3 + (double)((tiles * S + c.slots - 1) / c.slots) * (4.5 + (double)per * step) + (S > 1 ? 1.2 + 0.3 * S + 2 * part / 14e6 : 0);
      if (us < least) {
        least = us;
        best.tile = t;
        best.slices = S;
      }
    }
  }
  return best;
}

const char* kernel_name(DensePlan p) {
  return p == DensePlan::kSkinny ? "f8_dense_skinny" : p == DensePlan::kTiles ? "f8_dense_tiles" : "f8_dense_staged";
}

}  // namespace

std::string f8_product_plan(const F8DenseDesc& d) {
  const DenseChoice c = dense_plan(d);
  if (c.plan == DensePlan::kSkinny) return kernel_name(c.plan);
  const TileCost& t = kTileCosts[c.tile];
  return std::string(kernel_name(c.plan)) + " " + std::to_string(t.cols) + "x" + std::to_string(t.rows) + " slices " + std::to_string(c.slices);
}

bool f8_product_takes_float(const F8DenseDesc& d) { return skinny_fits(d); }

int f8_product_run(mx_backend* b, const F8DenseDesc& d) {
  if (d.M == 0 || d.N == 0) return MX_OK;
  DenseArgs a = dense_args(d);
  const DenseChoice choice = dense_plan(d);
  const char* name = kernel_name(choice.plan);
  if (choice.plan == DensePlan::kSkinny) return skinny_run(b, d, name);
  const bool wide = d.out_dt == MX_DTYPE_FLOAT32;
  a.vec_out = wide ? d.N % 4 == 0 && aligned16(d.out) : d.oi ? d.N % 8 == 0 && aligned16(d.out) : d.N % 4 == 0 && ((uintptr_t)d.out & 7) == 0;
  if (choice.plan == DensePlan::kStaged) return staged_run(b, name, a, wide, choice.tile, choice.slices);
  if (wide) {
    switch (choice.tile) {
      case 1: return run_dense_tiles<Tile256x128, true, true>(b, name, a, choice.slices);
      case 3: return run_dense_tiles<Tile128x64, true, true>(b, name, a, choice.slices);
      case 4: return run_dense_tiles<Tile64x128, true, true>(b, name, a, choice.slices);
      default: return run_dense_tiles<Tile64x64, true, true>(b, name, a, choice.slices);
    }
  }
  switch (choice.tile) {
    case 0: return run_dense_tiles<Tile256x256, false, true>(b, name, a, choice.slices);
    case 1: return run_dense_tiles<Tile256x128, false, true>(b, name, a, choice.slices);
    case 2: return run_dense_tiles<Tile128x128, false, true>(b, name, a, choice.slices);
    case 3: return run_dense_tiles<Tile128x64, false, true>(b, name, a, choice.slices);
    case 4: return run_dense_tiles<Tile64x128, false, true>(b, name, a, choice.slices);
    default: return run_dense_tiles<Tile64x64, false, true>(b, name, a, choice.slices);
  }
}

}  // namespace mx
