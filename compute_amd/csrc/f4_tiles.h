// Dense product over 4-bit floating-point blocks, both operands in codes with blocks along K, on the 4-bit matrix cores:
//   y[m, n] = act(sum_k x[m, k] * w[n, k] + bias[n]).
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes 32 codes of a row from each lane with the scale byte of their block, and adds to the
// float32 total directly: the block is the instruction's own.  Its sums are float32 sums (e2m1 products are multiples of 1/4
// up to 36, so that nothing of a block is cut off; measured equal to 64 bits on random codes, 1.1e-7 of the terms with scales over 40
// binades), so float32 and bfloat16 results come from the same instructions.
//
// Operand layout.  Lane (i = lane % 32, g = lane / 32) of an instruction (32x32x64) holds one block of row (or column) i; the sum does
// not depend on which block a lane stands for as long as both operands agree.  A step is 256 of k, 128 bytes of a row: lane g has
// its blocks 4 g to 4 g + 3, one for each of four instructions, whose scale bytes are a word.
//
// Tiles.  A workgroup of WN x WM waves computes 64 WN columns (n) x 32 TB WM rows (m), a wave 64 x 32 TB of it.  w is the first
// operand, so that a lane's sixteen results of a tile are of one row.
//
// Staging.  Codes move from memory straight into LDS, BUF - 1 steps ahead, 16 bytes a lane.  The resources end with their arrays:
// rows past M or N are zeros; chunks past K in the last step are sent past the end.  Rows are 128 bytes in LDS; chunk c of row r lies
// at c ^ (r >> 1 & 7): the 16 lanes that a 16-byte read takes at a time (0-3, 12-15, 20-23, 24-27, and the rest) are eight pairs of
// rows that meet every bank once.
//   Scales are 8 bytes of a row a step, but a cache line moves whole: a word of each row a step took as many lines as the codes
//   and more time than the MFMAs (2.6 us a step of 256 x 256).  So they come for Q steps (two or four) at once, 8 Q bytes of
//   a row, into two buffers, a load of 128 / Q rows from each wave beside its codes' loads.  Rows lie 8 Q bytes apart in LDS too, so
//   that four lanes (Q = 4) or two read their words from one bank: such conflicts are 41 and 24 of 100 LDS cycles.  In a copy whose
//   scale addresses were free of them (and its scales wrong) 6 and 4 were left, and the kernels took 5 and 2 of 100 cycles less.
//
// Schedule.  A step is TB groups of eight MFMAs, one operand of x against the wave's two of w, in four pieces of one block each.
// Operands of x are read a group ahead.  The step's barrier stands before its last group, whose operands are in registers:
// behind it begin the requests of the step BUF ahead, into the buffer just left, and under that group travel the first
// operands of the next step, all of w's among them.  The requests are spread over pieces; a piece's loads take one addition
// each, their resources are the whole call's.
//
// Measured: 8192 x 8192 x 8192 in 274 to 285 us (4.0 PFLOP/s), [2048,4096] x 14336 with SiLU 76, [2048,4096] x 4096 26.5.  A step of 256 x 256 takes
// 1.95 us on 256 CUs: MFMAs alone 0.85 at 2.4 GHz, 1.45 without loads at the clock that all CUs hold, the rest the loads beside
// the operands' reads.
#pragma once

#include <algorithm>

#include "f4_dense.h"

namespace mx {
namespace f4 {
namespace {

using f8::kPastEnd;
using f8::lds_addr;
using f8::lds_barrier;
using f8::lds_load16;
using f8::lds_read16;
using f8::make_resource;
using f8::Resource;
using f8::wait_loads;

typedef __attribute__((address_space(3))) const uint32_t lds_u32;

constexpr int kStepK = 256, kStepBytes = kStepK / 2;  // of a row a step

// Q: steps whose scales are loaded together.
template <int WN_, int WM_, int TB_, int BUF_, int Q_>
struct Tile4 {
  static constexpr int WN = WN_, WM = WM_, TB = TB_, BUF = BUF_, Q = Q_, kWaves = WN * WM, kThreads = 64 * kWaves;
  static constexpr int kCols = 64 * WN, kRows = 32 * TB * WM;
  static constexpr int kXBytes = kRows * kStepBytes, kWBytes = kCols * kStepBytes, kScaleBytes = 8 * Q * (kRows + kCols);
  static constexpr int kX = 0, kW = BUF * kXBytes, kScale = kW + BUF * kWBytes, kLds = kScale + 2 * kScaleBytes;
  static constexpr int XL = kXBytes / (1024 * kWaves), WL = kWBytes / (1024 * kWaves);  // loads of a wave a step
  static constexpr int kScaleLoads = kScaleBytes / 1024, SL = (kScaleLoads + kWaves - 1) / kWaves;  // and of Q steps' scales
  static constexpr int kLoads = XL + WL;
  static_assert(Q == 2 || Q == 4, "whole loads of scales");
  static_assert(SL <= Q + 2 - BUF, "the loads of Q steps' scales fit between the last use of their buffer and the first of theirs");
  static_assert(kXBytes % (1024 * kWaves) == 0 && kWBytes % (1024 * kWaves) == 0 && kRows % (128 / Q) == 0, "whole loads");
  static_assert(kWaves >= 2, "the rows of a wave's loads differ by multiples of 16: one chunk order for all of them");
  static_assert(kLds <= 160 * 1024 && kWaves * 32 * 4 * (64 + 4) <= kLds, "LDS of a CU; the results' part of it");
};

// The block J of two operands: the first half of the registers is all that 4-bit operands take.
template <int J>
__device__ __forceinline__ f32x16 mfma_f4(const u32x4& a, uint32_t sa, const u32x4& b, uint32_t sb, const f32x16& c) {
  const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, J, (int)sa, J, (int)sb);
}

template <class Tile>
__global__ __launch_bounds__(Tile::kThreads, 2) void f4_tiles_kernel(DenseArgs a) {
  constexpr int TB = Tile::TB, Q = Tile::Q, kWaves = Tile::kWaves, XL = Tile::XL, SL = Tile::SL, kLoads = Tile::kLoads;
  constexpr bool kOne = TB == 1;  // the next step's operand of x travels while the present one is in use
  static_assert(kOne || TB % 2 == 0, "operands of x alternate");
  extern __shared__ __align__(1024) uint8_t lds[];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = lane % 32, g = lane / 32;
  const uint32_t base = lds_addr(lds);
  TilePlace place;
  TileRows rows;
  if (!tile_place(a, Tile::kRows, place) || !locate_rows(a, place.mt, Tile::kRows, rows)) return;
  const int m0 = rows.first, n0 = place.nt * Tile::kCols;
  const int wn = wave / Tile::WM, wm = wave % Tile::WM;
  f32x16 acc[2][TB] = {};
  const int steps = (a.K + kStepK - 1) / kStepK, s0 = place.slice * a.kps, s1 = min(steps, s0 + a.kps);  // the slice's steps
  if (rows.expert < a.E && s0 < s1) {
    const uint32_t row_bytes = (uint32_t)a.K / 2;
    const int64_t row = (int64_t)rows.expert * a.N + n0;
    const Resource xr = make_resource(a.x + (int64_t)m0 * row_bytes, (int64_t)(a.M - m0) * row_bytes);
    const Resource wr = make_resource(a.w + row * row_bytes, (int64_t)(a.N - n0) * row_bytes);
    const Resource xsr = make_resource(a.xs + (int64_t)m0 * a.KB, (int64_t)(a.M - m0) * a.KB);
    const Resource wsr = make_resource(a.ws + row * a.KB, (int64_t)(a.N - n0) * a.KB);
    // A load of codes is eight rows of 128 bytes, a wave's loads 8 kWaves rows apart.
    const int chunk = (lane % 8) ^ ((8 * wave + lane / 8) >> 1 & 7);
    const bool half = a.K % kStepK != 0;  // the last step has the first half of a row's bytes
    const uint32_t off = (uint32_t)(8 * wave + lane / 8) * row_bytes + 16 * chunk, tail = half && chunk >= 4 ? kPastEnd : 0u;
    const uint32_t s_off = (uint32_t)(lane / (Q / 2)) * (uint32_t)a.KB + 16 * (lane % (Q / 2));
    // The `part`-th of a wave's loads of the scales of steps s0 + Q t and on: 128 / Q rows, x's before w's.
    auto request_scales = [&](int t, int part) __attribute__((always_inline)) {
      if (part * kWaves + wave >= Tile::kScaleLoads) return;
      const int r = 128 / Q * (part * kWaves + wave);
      const uint32_t at = 8 * (uint32_t)(s0 + Q * t) + (uint32_t)(r < Tile::kRows ? r : r - Tile::kRows) * (uint32_t)a.KB;
      lds_load16(r < Tile::kRows ? xsr : wsr, s_off + at, base + Tile::kScale + (t & 1) * Tile::kScaleBytes + 8 * Q * r);
    };
    // Loads `from` to `to` of a wave's kLoads of a step.  (Steps past the last are requested like any other, from wherever they
    // lie within the arrays, and not used.)  With the codes of step s comes a load of scales: those of Q steps are needed
    // behind the barrier of the step before them, which waits for what came with their first; their buffer is free behind the
    // barrier of the step 2 Q before that first, behind which the codes of the step BUF later are requested.  The waits count the
    // loads of codes alone: with one of scales among the last ones they wait for a load more.
    auto request = [&](int s, uint32_t buf, int from, int to) __attribute__((always_inline)) {
      const uint32_t o = off | (s == steps - 1 ? tail : 0u);
#pragma unroll
      for (int j = from; j < to; ++j) {
        const bool x = j < XL;
        const int q = x ? j : j - XL;
        if (j == XL) {
          const int u = s - s0 + 1 - Tile::BUF;  // (Q / 2 = log2 Q; shifts round down)
          if (u >= 0 && (u & (Q - 1)) < SL) request_scales((u >> (Q / 2)) + 1, u & (Q - 1));
        }
        lds_load16(x ? xr : wr, o + ((uint32_t)s * kStepBytes + 8 * kWaves * q * row_bytes),
                   base + (x ? Tile::kX + buf * Tile::kXBytes : Tile::kW + buf * Tile::kWBytes) + 1024 * (wave + kWaves * q));
      }
    };
    constexpr int kSpread = TB == 1 ? 4 : TB == 2 ? 6 : 9;  // pieces that carry loads, from the barrier on
    auto loads_before = [](int p) constexpr { return p < kSpread ? (p * kLoads + kSpread - 1) / kSpread : kLoads; };
    constexpr int kBehind = loads_before(4);  // those behind the barrier

    // Operand reads: four blocks, and a word of their scale bytes.
    const int x_row = 32 * TB * wm + i, w_row = 64 * wn + i;
    const uint32_t xa = base + Tile::kX + x_row * kStepBytes + 16 * ((4 * g) ^ (x_row >> 1 & 7));
    const uint32_t wa = base + Tile::kW + w_row * kStepBytes + 16 * ((4 * g) ^ (w_row >> 1 & 7));
    const uint32_t sxa = base + Tile::kScale + 8 * Q * x_row + 4 * g, swa = base + Tile::kScale + 8 * Q * (Tile::kRows + w_row) + 4 * g;
    // The scales of a step, and a mask of those that the last step has: what lies past K belongs to another row.
    const uint32_t has_last = half && g == 1 ? 0u : ~0u;
    uint32_t s_step, s_has;
    auto scales_of = [&](int s) __attribute__((always_inline)) {
      const int u = s - s0;
      s_step = (u >> (Q / 2) & 1) * Tile::kScaleBytes + 8 * (u & (Q - 1));
      s_has = s == steps - 1 ? has_last : ~0u;
    };
    u32x4 wv[2][4], wo[2][4], xo[2][4];
    uint32_t sw[2], swo[2], sx[2];
    auto read_w = [&](int c, int q, uint32_t buf) __attribute__((always_inline)) {
      wo[c][q] = lds_read16((wa ^ (16 * q)) + buf * Tile::kWBytes + 32 * kStepBytes * c);
      if (q == 0) swo[c] = *(lds_u32*)(swa + s_step + 256 * Q * c) & s_has;
    };
    auto read_x = [&](int to, int q, int b, uint32_t buf) __attribute__((always_inline)) {
      xo[to][q] = lds_read16((xa ^ (16 * q)) + buf * Tile::kXBytes + 32 * kStepBytes * b);
      if (q == 0) sx[to] = *(lds_u32*)(sxa + s_step + 256 * Q * b) & s_has;
    };

#pragma unroll
    for (int j = 0; j < SL; ++j) request_scales(0, j);
#pragma unroll
    for (int j = 0; j < Tile::BUF - 1; ++j) request(s0 + j, j, 0, kLoads);
    request(s0 + Tile::BUF - 1, Tile::BUF - 1, 0, kBehind);
    wait_loads<(Tile::BUF - 2) * kLoads + kBehind>();
    lds_barrier();
    scales_of(s0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      read_w(0, q, 0);
      read_w(1, q, 0);
      read_x(kOne ? 1 : 0, q, 0, 0);
    }
    uint32_t cur = 0, left = Tile::BUF - 1;  // the step's buffer and the one before it
    for (int s = s0; s < s1; ++s) {
      const uint32_t next = cur + 1 == Tile::BUF ? 0 : cur + 1;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int q = 0; q < 4; ++q) wv[c][q] = wo[c][q];
        sw[c] = swo[c];
      }
      if constexpr (kOne) {
#pragma unroll
        for (int q = 0; q < 4; ++q) xo[0][q] = xo[1][q];
        sx[0] = sx[1];
      }
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        if (b == TB - 1) {
          wait_loads<(Tile::BUF - 2) * kLoads>();
          lds_barrier();
          scales_of(s + 1);
        }
        const uint32_t sv = sx[b % 2];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (b + 1 < TB) {
            read_x((b + 1) % 2, q, b + 1, cur);
          } else {
            read_w(0, q, next);
            read_w(1, q, next);
            read_x(kOne ? 1 : 0, q, 0, next);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (q == 0) acc[c][b] = mfma_f4<0>(wv[c][0], sw[c], xo[b % 2][0], sv, acc[c][b]);
            if (q == 1) acc[c][b] = mfma_f4<1>(wv[c][1], sw[c], xo[b % 2][1], sv, acc[c][b]);
            if (q == 2) acc[c][b] = mfma_f4<2>(wv[c][2], sw[c], xo[b % 2][2], sv, acc[c][b]);
            if (q == 3) acc[c][b] = mfma_f4<3>(wv[c][3], sw[c], xo[b % 2][3], sv, acc[c][b]);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);  // LDS read
            __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // VALU
          }
          __builtin_amdgcn_sched_barrier(0);
          const bool behind = b == TB - 1;
          const int at = behind ? q : 4 * (b + 1) + q;
          request(behind ? s + Tile::BUF : s + Tile::BUF - 1, behind ? cur : left, loads_before(at), loads_before(at + 1));
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      left = cur;
      cur = next;
    }
    wait_loads<0>();  // of the steps past the last: LDS is the results' from here on
  }
  if (a.S > 1 && !join_slices<Tile::kThreads, TB>(a, acc, place.tile, place.slice, (int*)lds)) return;
  __syncthreads();
  store_activated_rows<TB>(a, acc, (float*)lds + wave * 32 * kOutPitch, m0 + 32 * TB * wm, rows.end, n0 + 64 * wn, rows.expert);
}

template <class Tile>
int run_f4_tiles(mx_backend* b, const char* name, const F4DenseDesc& d, int slices) {
  DenseArgs a = dense_args(d);
  unsigned grid = 0;
  MX_TRY(set_tiles(b, d, a, Tile::kRows, Tile::kCols, Tile::kThreads, kStepK, slices, &grid));
  auto k = f4_tiles_kernel<Tile>;
  MX_CHECK_HIP(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, Tile::kLds));
  return launch(b, name, [&] { dispatch(k, dim3(grid), dim3(Tile::kThreads), Tile::kLds, b->stream, a); });
}

}  // namespace
}  // namespace f4
}  // namespace mx
