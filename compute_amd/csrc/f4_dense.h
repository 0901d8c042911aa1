// What the kernels of the dense product over 4-bit floating-point blocks share: the product of one weight matrix, and that of
// rows sorted by expert with the weights of each.
#pragma once

#include <algorithm>

#include "f4_common.h"
#include "lds_loads.h"
#include "mxrt_internal.h"

namespace mx {
namespace f4 {

struct DenseArgs {
  const uint8_t* x;  // codes or floats
  const uint8_t* xs;
  const uint8_t* w;
  const uint8_t* ws;
  const void* bias;
  void* out;
  const int32_t* offsets;  // of the experts' rows, or null: one matrix
  int M, K, N, KB, E;
  int ldx, ldw;       // f4_wide.h: bytes of a row of x, values of a row of w,
  int64_t x_part;     // and bytes of a part of x
  int b_dt, out_dt, act;
  int tiles_n, tiles_m, vec_out;
  int64_t first;      // few rows: the launch's first workgroup
  int S, kps;         // slices of K of a tile, steps of a slice
  char* part;         // [tile][slice] sums (S > 1)
  uint32_t* arrived;  // [tile], zero between launches
};

inline DenseArgs dense_args(const F4DenseDesc& d) {
  return DenseArgs{(const uint8_t*)d.x, d.x_scale, d.w, d.w_scale, d.bias, d.out, d.offsets, (int)d.M, (int)d.K, (int)d.N,
                   (int)blocks(d.K), (int)d.E, 0, 0, 0, d.b_dt, d.out_dt, d.act, 0, 0, 0, 0, 1, 0, nullptr, nullptr};
}

// The rows of a tile: first .. first + per - 1, of which those from `end` on are not its own.  Expert E: the rows behind the
// last expert's, which are zero in the result.
struct TileRows {
  int expert, first, end;
};

// Experts' rows start tiles of their own, so the tiles of `per` rows are numbered through the experts.  Their lengths are known here
// only; offsets are brought into [0, M] and ascending order, so that any offsets stay in the arrays.
__device__ __forceinline__ void expert_rows(const DenseArgs& a, int e, int& lo, int& hi) {  // e == E: those behind the last; past it none
  auto offset = [&](int i) { return i <= 0 ? 0 : i > a.E ? a.M : min(max(a.offsets[i], 0), a.M); };
  lo = offset(e);
  hi = e > a.E ? lo : max(offset(e + 1), lo);
}
// All tiles (at most M / per + E + 1, of ascending offsets; not more than `most` in any case): 64 experts a lane each.
__device__ __forceinline__ int count_tiles(const DenseArgs& a, int per, int most) {
  if (a.offsets == nullptr) return most;
  int64_t all = 0;
  for (int base = 0; base <= a.E; base += 64) {
    int lo, hi;
    expert_rows(a, base + (int)threadIdx.x % 64, lo, hi);
    all += (hi - lo + per - 1) / per;
  }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) all += __shfl_xor(all, d);
  return __builtin_amdgcn_readfirstlane((int)(all < most ? all : most));
}
// Tile t: the running sum of the experts' tiles finds the one that holds it.  False past the last tile.  Sums stop at kTop, which is
// past every t (rows < 2^30, four or more to a tile), so that no offsets overflow them; those before the tile found are exact.
__device__ __forceinline__ bool locate_rows(const DenseArgs& a, int t, int per, TileRows& r) {
  if (a.offsets == nullptr) {
    r = TileRows{0, t * per, a.M};
    return r.first < a.M;
  }
  constexpr int kTop = (1 << 30) - 1;
  const int lane = threadIdx.x % 64;
  int before = 0;
  for (int base = 0; base <= a.E; base += 64) {
    int lo, hi;
    expert_rows(a, base + lane, lo, hi);
    int sum = (hi - lo + per - 1) / per;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum = min(sum + o, kTop);
    }
    const uint64_t holds = __ballot(before + sum > t);
    if (holds != 0) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)holds) - 1);
      const int start = before + (l == 0 ? 0 : __builtin_amdgcn_readlane(sum, l - 1));
      r.expert = base + l;
      r.first = __builtin_amdgcn_readlane(lo, l) + (t - start) * per;
      r.end = __builtin_amdgcn_readlane(hi, l);
      return r.first < r.end;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// Tiles of `per` rows that a launch has to have.
inline int64_t most_tiles(const F4DenseDesc& d, int per) {
  return d.offsets == nullptr ? (d.M + per - 1) / per : d.M / per + d.E + 1;
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// A wave's results: 64 columns from n0 of the rows m0 .. end - 1.  Lane (i = lane % 32, g = lane / 32) has, of each row 32 b + i,
// the columns 32 c + 8 t + 4 g and three more in registers 4 t of operand c; a store of its own would touch 32 rows, so they go through the wave's part of LDS (32 rows of 64 floats and four more) and out as whole
// lines.  LIVE: with bias and activation (not the zeros behind the last expert).
constexpr int kOutPitch = 64 + 4;
constexpr int kGeluF32 = -1;  // among the activations: GELU of float32 results
template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == kGeluF32)
    return gelu_f32(v);
  else
    return act_fast(v, ACT);
}
template <int ACT, bool LIVE, int TB>
__device__ __forceinline__ void store_rows(const DenseArgs& a, const f32x16 (&acc)[2][TB], float* out, int m0, int end, int n0, int expert) {
  const int lane = threadIdx.x % 64, i = lane % 32, g = lane / 32;
  const int n = n0 + 8 * (lane % 8);  // the columns that the lane stores, of the rows lane / 8 and on
  float bias[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) bias[r] = LIVE && a.bias && n + r < a.N ? load_f(a.bias, (int64_t)expert * a.N + n + r, a.b_dt) : 0.0f;
  const bool f32 = a.out_dt == MX_DTYPE_FLOAT32;
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    if (m0 + 32 * b >= end) break;
    // One wave writes and reads: its LDS operations keep their order.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        *(f32x4*)(out + i * kOutPitch + 32 * c + 8 * t + 4 * g) = f32x4{acc[c][b][4 * t], acc[c][b][4 * t + 1], acc[c][b][4 * t + 2], acc[c][b][4 * t + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int in = 8 * p + lane / 8, m = m0 + 32 * b + in;
      const f32x4 lo = *(const f32x4*)(out + in * kOutPitch + 8 * (lane % 8)), hi = *(const f32x4*)(out + in * kOutPitch + 8 * (lane % 8) + 4);
      if (m >= end) continue;
      float v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = LIVE ? activate<ACT>((r < 4 ? lo[r % 4] : hi[r % 4]) + bias[r]) : 0.0f;
      const int64_t at = (int64_t)m * a.N + n;
      if (!f32 && a.vec_out) {  // rows on 16 bytes, N a multiple of 8
        u32x4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x2 two = {v[2 * r], v[2 * r + 1]};
          o[r] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
        }
        if (n < a.N) *(u32x4*)((uint16_t*)a.out + at) = o;
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          f8::store4(a.out, at + 4 * q, a.N - n - 4 * q, a.vec_out, a.out_dt, f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]});
      }
    }
  }
}

template <int TB>
__device__ __forceinline__ void store_activated_rows(const DenseArgs& a, const f32x16 (&acc)[2][TB], float* out, int m0, int end, int n0, int expert) {
  if (expert == a.E) return store_rows<MX_ACT_NONE, false, TB>(a, acc, out, m0, end, n0, expert);
  switch (a.act) {
    case MX_ACT_GELU:  // (a choice for each value slowed both: [2048,4096] x 14336 in codes with bf16 results 96 us instead of 89)
      if (a.out_dt == MX_DTYPE_FLOAT32) return store_rows<kGeluF32, true, TB>(a, acc, out, m0, end, n0, expert);
      return store_rows<MX_ACT_GELU, true, TB>(a, acc, out, m0, end, n0, expert);
    case MX_ACT_RELU: return store_rows<MX_ACT_RELU, true, TB>(a, acc, out, m0, end, n0, expert);
    case MX_ACT_SILU: return store_rows<MX_ACT_SILU, true, TB>(a, acc, out, m0, end, n0, expert);
    case MX_ACT_HARDSWISH: return store_rows<MX_ACT_HARDSWISH, true, TB>(a, acc, out, m0, end, n0, expert);
    case MX_ACT_TANH: return store_rows<MX_ACT_TANH, true, TB>(a, acc, out, m0, end, n0, expert);
    default: return store_rows<MX_ACT_NONE, true, TB>(a, acc, out, m0, end, n0, expert);
  }
}

// Whether results go out as whole aligned vectors.
inline bool vector_results(const F4DenseDesc& d) {
  if (d.out_dt == MX_DTYPE_FLOAT32) return d.N % 4 == 0 && aligned16(d.out);
  return d.N % 8 == 0 && aligned16(d.out);
}

// The slices of a tile's K meet in scratch, stored and loaded with the agent-scope coherence bit (sc1): the slices may run on
// different XCDs.  The last to arrive adds them in order and goes on (true); it leaves the counter at zero.  word: a word of
// LDS that nothing else uses any more.
template <int THREADS, int TB>
__device__ __forceinline__ bool join_slices(const DenseArgs& a, f32x16 (&acc)[2][TB], int tile, int slice, int* word) {
  constexpr int kSc1 = 16, kPartBytes = 2 * TB * THREADS * 64;
  const __amdgpu_buffer_rsrc_t prs =
      __builtin_amdgcn_make_buffer_rsrc(a.part + (int64_t)tile * a.S * kPartBytes, 0, a.S * kPartBytes, 0x00027000);
  auto at = [&](int sl, int c, int b, int t) { return (uint32_t)(sl * kPartBytes + (((c * TB + b) * 4 + t) * THREADS + (int)threadIdx.x) * 16); };
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 v = {acc[c][b][4 * t], acc[c][b][4 * t + 1], acc[c][b][4 * t + 2], acc[c][b][4 * t + 3]};
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), prs, at(slice, c, b, t), 0, kSc1);
      }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = __hip_atomic_fetch_add(&a.arrived[tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool last = before + 1u == (uint32_t)a.S;
    *word = last;
    if (last) __hip_atomic_store(&a.arrived[tile], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (*word == 0) return false;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[c][b] = f32x16{};
  constexpr int kTogether = TB == 1 ? 4 : 1;  // slices in flight at a time
#pragma unroll kTogether
  for (int sl = 0; sl < a.S; ++sl)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, at(sl, c, b, t), 0, kSc1));
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[c][b][4 * t + r] += v[r];
        }
  return true;
}

// The place of a workgroup: runs of 4 tiles of n by all tiles of m, so that a run's workgroups share their rows of x and w in
// an L2; a tile's slices are neighbours.  Only tiles that are there are dealt out (a launch holds the most that could be): with
// places for the others an XCD may get more tiles than it has CUs (777 x 2 rows of eight experts, [1536] x 2048: 33 on one, 80 us instead of 55).
struct TilePlace {
  int mt, nt, tile, slice;
};
__device__ __forceinline__ bool tile_place(const DenseArgs& a, int per, TilePlace& p) {
  const int tiles_m = count_tiles(a, per, a.tiles_m), items = tiles_m * a.tiles_n * a.S;
  if ((int)blockIdx.x >= items) return false;
  const int it = f8::xcd_order((int)blockIdx.x, items);
  p.tile = it / a.S;
  p.slice = it - p.tile * a.S;
  const int run = 4 * tiles_m, q = p.tile / run, cols = min(4, a.tiles_n - 4 * q), in = p.tile - q * run;
  p.nt = 4 * q + in % cols;
  p.mt = in / cols;
  return true;
}

// Sets the grid of a launch of ROWS x COLS tiles with K cut into slices of whole steps; scratch for the slices' sums.
inline int set_tiles(mx_backend* b, const F4DenseDesc& d, DenseArgs& a, int rows, int cols, int threads, int step, int slices, unsigned* grid) {
  const int64_t tm = most_tiles(d, rows), tn = (d.N + cols - 1) / cols, steps = (d.K + step - 1) / step;
  a.tiles_m = (int)tm;
  a.tiles_n = (int)tn;
  a.kps = (int)std::max<int64_t>((steps + slices - 1) / slices, 1);
  a.S = (int)std::max<int64_t>((steps + a.kps - 1) / a.kps, 1);  // K = 0: one slice without a step, act(bias)
  if (tm * tn * a.S * threads > kMaxWorkItems) return set_error(MX_ERR_INVALID, "F4Dense: a result of more tiles than a launch holds");
  a.vec_out = vector_results(d);
  if (a.S > 1) {
    void* scratch = nullptr;
    MX_TRY(ensure_scratch(b, kScratchCounterBytes + (size_t)(tm * tn * a.S) * rows * cols * 4, &scratch));
    a.arrived = (uint32_t*)scratch;
    a.part = (char*)scratch + kScratchCounterBytes;
  }
  *grid = (unsigned)(tm * tn * a.S);
  return MX_OK;
}

// Tiles on the 4-bit matrix cores (f4_tiles.hip): x and w in codes [.., K], K a multiple of 128, codes on 16 bytes, scales on 4.
int tiles_run(mx_backend* b, const char* name, const F4DenseDesc& d, int tile, int slices);

// Tiles on the bf16 matrix cores (f4_wide.hip): d.x as bf16 rows on 16 bytes, or as the three parts of float32 rows; rows of w of a
// multiple of 128 values along their last dimension, codes on 16 bytes, scales on 4.
struct WideX {
  int parts;
  int64_t pitch, part;  // bytes of a row, and from one part to the next
  int64_t w_values;     // of a row of w
};
int wide_run(mx_backend* b, const char* name, const F4DenseDesc& d, const WideX& x, int tile, int slices);

// Few rows (f4_skinny.hip), w [N, K] as above; x as above, or codes with rows like w's.  A group of rows has skinny_rows at most;
// shape: waves and columns of a workgroup.
inline int skinny_rows(const F4DenseDesc& d) { return d.x_dt == MX_DTYPE_FLOAT32 ? 5 : 16; }
int skinny_run(mx_backend* b, const char* name, const F4DenseDesc& d, const WideX& x, int shape);

// Few rows, w [K, N] (f4_columns.hip): x as float32 or bf16 rows of `pitch` values, rows of w of w_values, a multiple of eight, codes on
// four bytes.  rows: 1, 2 or 4 of a workgroup.
constexpr int kColumnsOfGroup = 512, kColumnsStep = 64, kColumnsThreads = 512;
struct ColumnsX {
  bool f32;
  int64_t pitch, w_values;
};
int columns_run(mx_backend* b, const char* name, const F4DenseDesc& d, const ColumnsX& x, int rows, int slices);

// Rows of bytes to rows of `pitch` bytes (a multiple of four; 16 where it is one of 16: `to` on as much), zeros behind, of up to kMost
// arrays; x to bf16 rows (three parts of float32) of `pitch` values (f4_prepare.hip).
struct PadRows {
  static constexpr int kMost = 4;
  struct Job {
    const uint8_t* from;
    uint8_t* to;
    int bytes, pitch, unit;
    int64_t units, group;  // units of the array, and its first workgroup
  };
  Job job[kMost];
  int n = 0;
  int64_t groups = 0;
  void add(const uint8_t* from, uint8_t* to, int64_t rows, int64_t bytes, int64_t pitch);
};
int pad_rows(mx_backend* b, const PadRows& jobs);
int bf16_rows(mx_backend* b, const F4DenseDesc& d, uint8_t* to, int64_t pitch, int64_t part);

}  // namespace f4
}  // namespace mx
