// Dense product over 4-bit floating-point blocks: the choice of a kernel, and operands brought into the form that it loads.
#include <cmath>

#include "f4_dense.h"

namespace mx {
namespace {
using namespace f4;

enum class Kind { kTiles, kWide, kSkinny, kColumns };
struct Choice {
  Kind kind;
  int tile, cols, rows, slices;  // skinny: tile is the shape, rows those of a group
};

// The tile and the number of K slices that take the least time by the times of their parts, measured over the tiles and slices of
// 11 to 17 products each (profiles/f4_tile_sweeps.txt): a launch 3 us; a round of workgroups its first loads and its stores
// (fixed) and its steps (256 of k on the 4-bit matrix cores, 64 on the bf16 ones), which take longer with every CU at work; for
// sums that meet in scratch 1.8 us, 0.3 us a slice and their bytes, out and back, at 14 TB/s.  For instance (us, columns x rows, slices):
//   codes [2048,4096] x 4096     256x128 25.0, 256x256 31.2, 128x128 32.0       [2048,4096] x 11008   256x256 64.9, 256x128 68.1
//         [512,4096] x 4096      128x64 11.2, 64x64 14.6, 128x128 15.9          [64,14336] x 4096     128x64 in four 13.7, whole 26.4
//   bf16  [2048,4096] x 4096     256x128 59.6, 128x128 62.1, 256x256 77         [64,4096] x 4096      64x64 in four 12.4, whole 25.5
//         [4096,4096] x 4096     256x256 110, 256x128 125, 128x128 128
struct TileCost {
  int cols, rows, threads, slots;   // threads of a workgroup, workgroups at once on 256 CUs
  float fixed, step, alone;         // us; a step with a workgroup on each CU at most (of two a CU), or on 160 of them
};
constexpr TileCost kTileCosts[] = {{256, 256, 512, 256, 4.5f, 1.95f, 1.27f},
                                   {256, 128, 512, 256, 3.4f, 1.15f, 0.87f},
                                   {128, 128, 512, 256, 2.0f, 0.77f, 0.66f},
                                   {128, 64, 256, 256, 1.9f, 0.43f, 0.38f},
                                   {64, 64, 128, 512, 1.5f, 0.66f, 0.41f}};
// By weights [N, K] or [K, N] (whose codes take another way through LDS), and x as one bf16 array or as three.
constexpr TileCost kWideCosts[2][2][5] = {{{{256, 256, 512, 256, 3.0f, 1.80f, 1.40f},
                                            {256, 128, 512, 256, 2.8f, 1.08f, 0.97f},
                                            {128, 128, 256, 512, 2.0f, 1.17f, 0.77f},
                                            {128, 64, 256, 512, 1.4f, 0.88f, 0.65f},
                                            {64, 64, 128, 512, 1.3f, 0.78f, 0.60f}},
                                           {{0, 0, 0, 0, 0, 0, 0},
                                            {256, 64, 512, 256, 2.5f, 1.50f, 1.25f},
                                            {0, 0, 0, 0, 0, 0, 0},
                                            {128, 64, 256, 256, 1.5f, 0.95f, 0.93f},
                                            {64, 64, 128, 256, 1.3f, 0.88f, 0.88f}}},
                                          {{{256, 256, 512, 256, 3.0f, 1.62f, 1.04f},
                                            {256, 128, 512, 256, 2.7f, 0.85f, 0.59f},
                                            {128, 128, 256, 512, 2.0f, 0.90f, 0.47f},
                                            {128, 64, 256, 512, 0.9f, 0.58f, 0.36f},
                                            {64, 64, 128, 512, 0.8f, 0.48f, 0.35f}},
                                           {{256, 128, 512, 256, 3.5f, 2.45f, 1.75f},
                                            {256, 64, 512, 256, 2.0f, 1.32f, 1.05f},
                                            {0, 0, 0, 0, 0, 0, 0},
                                            {128, 64, 256, 512, 1.5f, 1.46f, 0.86f},
                                            {64, 64, 128, 512, 1.3f, 1.04f, 0.76f}}}};

Choice cheapest(const F4DenseDesc& d, Kind kind, const TileCost (&costs)[5], int step) {
  const int64_t steps = (d.K + step - 1) / step;
  Choice best{kind, -1, 0, 0, 1};
  double least = 1e30;
  for (int t = 0; t < 5; ++t) {
    const TileCost& c = costs[t];
    if (c.cols == 0) continue;
    // Experts' rows are not known here: half a tile is lost to each, and each of them has one.
    const double experts = (double)std::min(d.E, d.M);
    const double tm = d.offsets ? std::max(experts, (double)d.M / c.rows + experts / 2) : (double)((d.M + c.rows - 1) / c.rows);
    const double tiles = tm * (double)((d.N + c.cols - 1) / c.cols);
    for (int S = 1; S <= (d.offsets ? 1 : 16) && (S == 1 || S <= steps); ++S) {
      const int64_t per = (steps + S - 1) / S, used = per ? (steps + per - 1) / per : 1;  // slices that are not empty
      const double part = tiles * S * c.rows * c.cols * 4;
      if (S > 1 && (used != S || tiles > kScratchCounterBytes / 4 || part > 128e6)) continue;
      if ((double)most_tiles(d, c.rows) * (double)((d.N + c.cols - 1) / c.cols) * S * c.threads > (double)kMaxWorkItems) continue;
      const double us = std::ceil(tiles * S / c.slots) * (c.fixed + (double)per * (tiles * S <= (c.slots == 256 ? 160 : 256) ? c.alone : c.step)) +
                        (S > 1 ? 1.8 + 0.3 * S + 2 * part / 14e6 : 0);
      if (us < least) {
        least = us;
        best = Choice{kind, t, c.cols, c.rows, S};
      }
    }
  }
  return best;
}

// Few rows: measured against the tiles (us; skinny, tiles)
//   bf16   64 rows of 32 experts, [2048] x 1536     17.3  20.8     codes   14.5  15.1
//          32 rows of 8 experts, [4096] x 14336     83    84               72    56
//          16 rows, [4096] x 4096                   7.4   12.0              5.1   9.0
bool few_rows(const F4DenseDesc& d) {
  if (!d.oi || d.K == 0) return false;
  if (d.offsets == nullptr) return d.M <= skinny_rows(d);
  return d.M <= (d.x_dt == MX_DTYPE_BFLOAT16 ? 4 : 2) * d.E;
}

// Waves and columns of a workgroup (us; waves x operands of 16 columns):
//   bf16 1 row   [4096] x 4096     8x1 4.7, 4x4 10.2      [4096] x 11008    4x1 8.2, 8x1 9.0, 4x4 10.6      x 114688  4x1 46.1, 4x4 46.6
//        16 rows [4096] x 4096     8x1 7.5, 4x4 12.7      [4096] x 11008    4x4 13.1, 4x1 17.2              [2048] x 32001  4x4 12.5, 4x1 21
//   codes 16 rows                  8x1 5.2, 4x4 10.0                        4x4 10.5, 4x1 10.6                 1 row x 114688  4x4 44, 4x1 51
//   experts, 32 of [2048] x 1536   2x2 17.3, 4x4 18.9     8 of [4096] x 14336   4x4 61.8, 2x2 65.5
int skinny_shape(const F4DenseDesc& d) {
  constexpr int k2x2 = 0, k8x1 = 1, k4x1 = 2, k4x4 = 3;  // cases of run_shape
  const int64_t strips = d.E * ((d.N + 15) / 16);
  if (strips < 512) return k8x1;
  if (d.offsets == nullptr && d.x_dt == MX_DTYPE_BFLOAT16 && d.M <= 2) return k4x1;
  if (d.offsets) return d.K <= 2048 ? k2x2 : k4x4;
  return strips >= 1536 || (d.x_dt != MX_DTYPE_F4E2M1FN && d.M > 4) ? k4x4 : k4x1;
}

// Few rows against w [K, N]: a workgroup's rows, and slices of K: a power of two (uneven ones wait for each other) whose empty ones are
// dropped, enough for 320 workgroups and for 16 steps each at most, of four steps at least.  Measured (us; slices, tiles; more of them in
// profiles/f4_tile_sweeps.txt):
//   bf16  1 row  [4096] x 4096     9.0 in 16, 10.3 in 8, tiles 15.3      [4096] x 11008   12.2 in 16, 11.8 in 8, tiles 20.9
//                [14336] x 4096    14.6 in 32, 15.8 in 16, tiles 28.8    [2048] x 32000   11.5 in 8, 11.7 in 4, tiles 21.9
//         4 rows [4096] x 11008    19.3 in 16, tiles 21.0                [4096] x 4096    14.9 in 16 (12.1 in 8 with one row a workgroup), tiles 15.2
//         3 rows [1536] x 384      13.7 in 4, tiles 9.2: four rows a workgroup cost more than they save where there are few columns
//   experts, 64 rows of 32, [2048] x 1536  27.7 in four (19.0 with one row a workgroup), tiles 30.8 (float32 27.7, 47)
//            32 rows of 8, [4096] x 14336  117 in four, 128 in two, tiles 112              2 rows of 8     28 in eight, tiles 46
bool few_columns(const F4DenseDesc& d, Choice* c) {
  if (d.oi || d.K == 0 || d.M > (d.offsets ? 4 * d.E : 4)) return false;
  const int rows = d.offsets || d.M > 2 ? 4 : (int)d.M;
  constexpr int64_t kLeast = 4, kMost = 16, kMostSlices = 32;
  const int64_t steps = (d.K + kColumnsStep - 1) / kColumnsStep, tn = (d.N + kColumnsOfGroup - 1) / kColumnsOfGroup;
  const int64_t live = (d.offsets ? std::min(d.E, d.M) : 1) * tn, tiles = most_tiles(d, rows) * tn;
  int64_t S = 1;
  while (S < kMostSlices && 2 * S * kLeast <= steps && (S * live < 320 || S * kMost < steps)) S *= 2;
  if (tiles > (int64_t)kScratchCounterBytes / 4 || (double)tiles * (double)S * rows * kColumnsOfGroup * 4 > 128e6) S = 1;
  if ((double)tiles * (double)S * kColumnsThreads > (double)kMaxWorkItems) return false;
  const int64_t per = (steps + S - 1) / S;
  S = (steps + per - 1) / per;  // 65 steps in 16 would be 13 slices of five
  *c = {Kind::kColumns, rows, kColumnsOfGroup, rows, (int)S};
  return true;
}

Choice choose(const F4DenseDesc& d) {  // of a result that has rows and columns
  Choice columns;
  if (few_columns(d, &columns)) return columns;
  if (few_rows(d)) return {Kind::kSkinny, skinny_shape(d), 0, skinny_rows(d), 1};
  if (d.x_dt == MX_DTYPE_F4E2M1FN && d.oi && d.K > 0) return cheapest(d, Kind::kTiles, kTileCosts, 256);
  return cheapest(d, Kind::kWide, kWideCosts[d.oi][d.x_dt == MX_DTYPE_FLOAT32 && d.K > 0], 64);  // (K = 0: no parts of x)
}

const char* kernel_name(Kind k) {
  return k == Kind::kTiles ? "f4_tiles" : k == Kind::kWide ? "f4_wide" : k == Kind::kColumns ? "f4_columns" : "f4_skinny";
}

bool aligned4(const void* p) { return ((uintptr_t)p & 3) == 0; }
size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Memory of a call's own, given back when the call is queued (the pool is ordered by the backend's stream).
class Room {
 public:
  explicit Room(mx_backend* b) : b_(b) {}
  ~Room() {
    for (int i = 0; i < n_; ++i) dev_free(b_, p_[i]);
  }
  int take(size_t bytes, uint8_t** out) {
    void* p = nullptr;
    MX_TRY(dev_alloc(b_, bytes, &p));
    p_[n_++] = p;
    *out = (uint8_t*)p;
    return MX_OK;
  }

 private:
  mx_backend* b_;
  void* p_[3];
  int n_ = 0;
};

// Codes [rows, n] with scales [rows, ceil(n / 32)] as rows of a multiple of 128 values, zeros behind, once the jobs have run.
int padded_codes(Room& room, PadRows& jobs, int64_t rows, int64_t n, const uint8_t** codes, const uint8_t** scale) {
  const int64_t wide = round_up(n, 128);
  uint8_t* to = nullptr;
  const size_t first = round256((size_t)rows * (wide / 2));
  MX_TRY(room.take(first + (size_t)rows * (wide / kBlock), &to));
  jobs.add(*codes, to, rows, n / 2, wide / 2);
  jobs.add(*scale, to + first, rows, blocks(n), wide / kBlock);
  *codes = to;
  *scale = to + first;
  return MX_OK;
}

int run_prepared(mx_backend* b, F4DenseDesc d, const Choice& c) {
  Room room(b);
  PadRows jobs;
  const int64_t K = d.K;
  // Weights: whole aligned rows of chunks and of words of scales, along the dimension that their blocks run along.
  int64_t& along = d.oi ? d.K : d.N;
  const bool columns = c.kind == Kind::kColumns;  // (takes words of codes, and bytes of scales)
  const bool whole = columns ? along % 8 == 0 && aligned4(d.w) : along % 128 == 0 && aligned16(d.w) && aligned4(d.w_scale);
  const int64_t w_values = whole ? along : round_up(along, 128);
  if (K > 0 && !whole) MX_TRY(padded_codes(room, jobs, d.E * (d.oi ? d.N : K), along, &d.w, &d.w_scale));
  WideX x{1, 2 * K, 0, w_values};
  if (columns && d.x_dt != MX_DTYPE_F4E2M1FN) {
    x.pitch = 2 * K;
  } else if (d.x_dt == MX_DTYPE_F4E2M1FN && c.kind != Kind::kWide && !columns) {  // codes as they are: rows like w's
    const uint8_t* codes = (const uint8_t*)d.x;
    if (K % 128 != 0 || !aligned16(codes) || !aligned4(d.x_scale)) MX_TRY(padded_codes(room, jobs, d.M, K, &codes, &d.x_scale));
    d.x = codes;
    d.K = w_values;
    x.pitch = w_values / 2;
  } else if (K > 0 && (d.x_dt != MX_DTYPE_BFLOAT16 || K % 8 != 0 || !aligned16(d.x))) {
    const int64_t pitch = round_up(K, 64);
    x.parts = d.x_dt == MX_DTYPE_FLOAT32 ? 3 : 1;
    x.pitch = 2 * pitch;
    x.part = (int64_t)round256((size_t)(d.M * x.pitch));
    uint8_t* to = nullptr;
    MX_TRY(room.take((size_t)x.parts * x.part, &to));
    MX_TRY(bf16_rows(b, d, to, pitch, x.part));
    d.x = to;
  }
  if (jobs.n > 0) MX_TRY(pad_rows(b, jobs));
  switch (c.kind) {
    case Kind::kTiles: return tiles_run(b, kernel_name(c.kind), d, c.tile, c.slices);
    case Kind::kWide: return wide_run(b, kernel_name(c.kind), d, x, c.tile, c.slices);
    case Kind::kColumns: return columns_run(b, kernel_name(c.kind), d, ColumnsX{d.x_dt == MX_DTYPE_FLOAT32, x.pitch / 2, w_values}, c.rows, c.slices);
    default: return skinny_run(b, kernel_name(c.kind), d, x, c.tile);
  }
}

}  // namespace

std::string f4_dense_plan(const F4DenseDesc& d) {
  if (d.M == 0 || d.N == 0) return "nothing";
  const Choice c = choose(d);
  if (c.kind == Kind::kSkinny) return kernel_name(c.kind);
  if (c.tile < 0) return "too large";
  return std::string(kernel_name(c.kind)) + " " + std::to_string(c.cols) + "x" + std::to_string(c.rows) + " slices " + std::to_string(c.slices);
}

int f4_dense_run(mx_backend* b, const F4DenseDesc& d) {
  if (d.M == 0 || d.N == 0) return MX_OK;
  const Choice c = choose(d);
  if (c.tile < 0) return set_error(MX_ERR_INVALID, "F4Dense: a result of more tiles than a launch holds");
  return run_prepared(b, d, c);
}

}  // namespace mx
