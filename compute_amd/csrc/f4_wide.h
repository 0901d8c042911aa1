// Dense product over 4-bit floating-point blocks on the bf16 matrix cores, for x in floats, and for weights whose blocks do not lie
// along K:
//   y[m, n] = act(sum_k x[m, k] * (code[k, n] * s) + bias[n]).
//
// code * s has two significant bits and is exact in bf16, so v_mfma_f32_32x32x16_bf16 multiplies exact values and sums them in
// float32.  x comes as P arrays of bf16 rows: itself (P = 1), or the three parts of float32 values, h + m + l exactly, made before
// (P = 3: three products); f4_prepare.hip makes them, and whole aligned rows of whatever is not so.
//
// Operand layout.  Lane (i = lane % 32, g = lane / 32) of an instruction holds eight k of row (or column) i; the sum does not
// depend on which k a position stands for as long as both operands agree: the q-th of a step's four instructions takes
// k = 32 g + 8 q .. + 7 from lanes g, so that a lane's share of a step is one block of a row.
//
// Tiles.  A workgroup of WN x 2 waves computes 64 WN columns (n) x 64 TB rows (m), a wave 64 x 32 TB of it, 64 of k a step.  w is the
// first operand, so that a lane's sixteen results of a tile are of one row.
//
// LDS, all of it loaded straight from memory, BUF - 1 steps ahead, 16 bytes a lane; rows past M or N are zeros by their arrays' ends,
// chunks of x past K are sent past the end.
//   x: rows of 128 bytes (64 k); chunk c of row r lies at c ^ (r >> 1 & 7).
//   w [N, K] (OI): rows of 32 bytes of codes, a lane's share one chunk, widened after the read with one scale; chunk c of row r lies at
//     c ^ (r >> 3 & 1).  Scales come for eight steps at once, 16 bytes of a row, into two buffers (f4_wide_schedule.h).
//   w [K, N] (!OI): the blocks run across k, so that a lane's eight k have scales of their own.  Codes ([k][32 WN bytes], chunk c of
//     row k at c ^ swizzle) become bf16 values a step ahead, a chunk a thread, and lie in LDS once more, [k][n], in two buffers; they
//     come out through the transposing read, four k of 16 columns at a time.  Of row k the pair of chunks p (16 columns) lies at
//     p ^ pair_swizzle(k) and its halves are exchanged where k & 8: a write of 16 lanes (16 rows of one chunk) and a read of 32 (four
//     rows of two pairs) meet every bank once.  The codes of a step travel with the x of the step before.
//
// Schedule.  A step is TB groups of 8 P MFMAs, one operand of x (and its parts) against the wave's two of w, in four pieces.  Operands
// of x are read a group ahead.  The step's barrier stands before its last group, whose operands are in registers: behind it
// begin the requests of the step BUF ahead, into the buffer just left, and under that group travel the first operands of the
// next step, all of w's among them.
//
// Measured, bf16: 8192 x 8192 x 8192 in 818 us with w [N, K] (1.34 PFLOP/s), 930 with w [K, N]; [2048,14336] x 4096, w [K, N], 223.  The matrix cores
// are busy half of the time; the rest is the widening (of w [K, N] twice through LDS) and the loads.
#pragma once

#include "f4_dense.h"
#include "f4_wide_schedule.h"

namespace mx {
namespace f4 {
namespace {

using f8::kPastEnd;
using f8::lds_addr;
using f8::lds_barrier;
using f8::lds_load16;
using f8::lds_load4;
using f8::lds_read16;
using f8::lds_u32x4_rw;
using f8::make_resource;
using f8::Resource;
using f8::wait_loads;

typedef __attribute__((address_space(3))) const uint8_t lds_u8;

constexpr int kStep = 64;  // k of a step
static_assert(kStep == 2 * kBlock, "two scales of a row a step");

template <int WN_, int TB_, int BUF_, int P_, bool OI_>
struct WideTile {
  static constexpr int WN = WN_, WM = 2, TB = TB_, BUF = BUF_, P = P_, kWaves = WN * WM, kThreads = 64 * kWaves;
  static constexpr bool OI = OI_;
  static constexpr int kCols = 64 * WN, kRows = 32 * TB * WM;
  static constexpr int kPartBytes = kRows * 128, kXBytes = P * kPartBytes, kWBytes = kCols * 32, kWideBytes = OI ? 0 : kCols * 128;
  static constexpr int kScaleBytes = OI ? 16 * kCols : 256 * ((kCols + 127) / 128);  // of eight steps, or of one
  static constexpr int kX = 0, kW = BUF * kXBytes, kWide = kW + BUF * kWBytes, kScale = kWide + 2 * kWideBytes;
  static constexpr int kLds = kScale + (OI ? 2 : BUF) * kScaleBytes;
  static constexpr int XL = kXBytes / (1024 * kWaves), kLoads = XL + 1;  // loads of a wave a step (without scales)
  static_assert(kXBytes % (1024 * kWaves) == 0 && kPartBytes % (1024 * kWaves) == 0 && kWBytes == 1024 * kWaves, "whole loads");
  static_assert(kLds <= 160 * 1024 && kWaves * 32 * 4 * kOutPitch <= kLds, "LDS of a CU; the results' part of it");
};

template <int COLS>
__device__ __forceinline__ int pair_swizzle(int k) {
  if constexpr (COLS >= 128)
    return 2 * (k & 3) ^ (k >> 2 & 1);
  else  // two rows meet all banks: four pairs a row
    return 2 * (k >> 1 & 1) ^ (k >> 2 & 1);
}
// Rows of codes [K, N]: 128, 64 or 32 bytes; a read of 16 lanes takes one chunk of 16 rows.
template <int COLS>
__device__ __forceinline__ int code_swizzle(int k) {
  return COLS == 256 ? k >> 1 & 7 : COLS == 128 ? k >> 2 & 3 : k >> 3 & 1;
}

template <class Tile>
__global__ __launch_bounds__(Tile::kThreads, 2) void f4_wide_kernel(DenseArgs a) {
  constexpr int TB = Tile::TB, P = Tile::P, kWaves = Tile::kWaves, XL = Tile::XL, kLoads = Tile::kLoads, BUF = Tile::BUF, kCols = Tile::kCols;
  constexpr bool OI = Tile::OI, kOne = TB == 1;  // kOne: the next step's operand of x travels while the present one is in use
  static_assert(kOne || TB % 2 == 0, "operands of x alternate");
  extern __shared__ __align__(1024) uint8_t lds[];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = lane % 32, g = lane / 32;
  const uint32_t base = lds_addr(lds);
  TilePlace place;
  TileRows rows;
  if (!tile_place(a, Tile::kRows, place) || !locate_rows(a, place.mt, Tile::kRows, rows)) return;
  const int m0 = rows.first, n0 = place.nt * kCols;
  const int wn = wave / 2, wm = wave % 2;
  f32x16 acc[2][TB] = {};
  const int steps = (a.K + kStep - 1) / kStep, s0 = place.slice * a.kps, s1 = min(steps, s0 + a.kps);  // the slice's steps
  if (rows.expert < a.E && s0 < s1) {
    const uint32_t w_row_bytes = (uint32_t)a.ldw / 2, s_row_bytes = (uint32_t)a.ldw / kBlock;
    const int64_t w_rows = OI ? a.N : a.K, w_bytes = w_rows * w_row_bytes, s_bytes = w_rows * s_row_bytes;  // of an expert
    const int64_t w0 = OI ? (int64_t)n0 * w_row_bytes : n0 / 2, ws0 = OI ? (int64_t)n0 * s_row_bytes : n0 / kBlock & ~3;
    Resource xr[P];
#pragma unroll
    for (int p = 0; p < P; ++p) xr[p] = make_resource(a.x + p * a.x_part + (int64_t)m0 * a.ldx, (int64_t)(a.M - m0) * a.ldx);
    // A load of x is eight rows of 128 bytes, a wave's loads of a part 8 kWaves rows apart.
    const int chunk = (lane % 8) ^ ((8 * wave + lane / 8) >> 1 & 7);
    const uint32_t x_off = (uint32_t)(8 * wave + lane / 8) * (uint32_t)a.ldx + 16 * chunk;
    const uint32_t x_tail = 8 * chunk >= a.K - (steps - 1) * kStep ? kPastEnd : 0u;
    // A load of w is 1024 bytes: rows of 32 (OI), or of 32 WN.
    constexpr int kRowLanes = OI ? 2 : 2 * Tile::WN;
    const int w_row = (64 / kRowLanes) * wave + lane / kRowLanes;
    const uint32_t w_off = (uint32_t)w_row * w_row_bytes + 16 * ((lane % kRowLanes) ^ (OI ? w_row >> 3 & 1 : code_swizzle<kCols>(w_row)));
    const uint8_t* we = a.w + rows.expert * w_bytes + w0;
    const uint8_t* se = a.ws + rows.expert * s_bytes + ws0;
    const Resource wr = make_resource(we, w_bytes - w0), sr = make_resource(se, s_bytes - ws0);  // (OI)
    // OI: the scales of group t of eight steps, a load of 64 rows.  !OI: those of step t, words of four blocks of the 64 rows of k.
    auto request_scales = [&](int t, uint32_t buf) __attribute__((always_inline)) {
      if constexpr (OI) {
        if (wave < kCols / 64)
          lds_load16(sr, (uint32_t)(64 * wave + lane) * s_row_bytes + (uint32_t)scales_at(s0, t),
                     base + Tile::kScale + (t & 1) * Tile::kScaleBytes + 1024 * wave);
      } else {
        const int64_t moved = (int64_t)t * kStep * s_row_bytes;
        if (wave < (kCols + 127) / 128)
          lds_load4(make_resource(se + moved, s_bytes - ws0 - moved), (uint32_t)lane * s_row_bytes + 4 * wave,
                    base + Tile::kScale + buf * Tile::kScaleBytes + 256 * wave);
      }
    };
    auto request_codes = [&](int s, uint32_t buf) __attribute__((always_inline)) {
      const uint32_t to = base + Tile::kW + buf * Tile::kWBytes + 1024 * wave;
      if constexpr (OI) {
        lds_load16(wr, w_off + (uint32_t)s * 32, to);
      } else {
        const int64_t moved = (int64_t)s * kStep * w_row_bytes;
        lds_load16(make_resource(we + moved, w_bytes - w0 - moved), w_off, to);
      }
    };
    // Loads `from` to `to` of a wave's kLoads of a step: x, and the codes of the step (OI) or of the one behind it.  (Steps past the
    // last are requested like any other, from wherever they lie within the arrays, and not used.)  The waits count these; with
    // loads of scales among the last ones they wait for more.
    auto request = [&](int s, uint32_t buf, int from, int to) __attribute__((always_inline)) {
      const uint32_t o = x_off | (s == steps - 1 ? x_tail : 0u);
#pragma unroll
      for (int j = from; j < to; ++j) {
        if (j == 0) {
          if constexpr (OI) {
            if (const int t = scales_with(s, s0, BUF)) request_scales(t, 0);
          } else {
            request_scales(s + 1, buf);
          }
        }
        if (j < XL) {
          constexpr int kPer = XL / P;  // loads of a part
          const int p = j / kPer, q = j % kPer;
          lds_load16(xr[p], o + ((uint32_t)s * 128 + (uint32_t)(8 * kWaves * q) * (uint32_t)a.ldx),
                     base + Tile::kX + buf * Tile::kXBytes + p * Tile::kPartBytes + 1024 * (wave + kWaves * q));
        } else {
          request_codes(OI ? s : s + 1, buf);
        }
      }
    };
    static_assert(BUF <= kScaleSteps, "scales of eight steps arrive before their first");
    constexpr int kPieces = 4 * TB, kSpread = kPieces <= kLoads ? kPieces : kLoads;  // pieces that carry loads, from the barrier on
    auto loads_before = [](int p) constexpr { return p < kSpread ? (p * kLoads + kSpread - 1) / kSpread : kLoads; };
    constexpr int kBehind = loads_before(4);  // those behind the barrier

    // Operand reads.
    const int x_row = 32 * TB * wm + i, w_col = 64 * wn + i;
    const uint32_t xa = base + Tile::kX + x_row * 128 + 16 * ((4 * g) ^ (x_row >> 1 & 7));
    const uint32_t wa = base + Tile::kW + w_col * 32 + 16 * (g ^ (w_col >> 3 & 1)), swa = base + Tile::kScale + 16 * w_col + g;
    bf16x8 wv[2][4];
    u32x4 wo[2], wt[2][4], xo[2][P][4];  // wo: codes of the next step's operands; wt: their values, transposed
    uint32_t so[2];
    auto read_w = [&](int c, int q, int s, uint32_t buf) __attribute__((always_inline)) {  // s: the step
      if constexpr (OI) {
        if (q != 0) return;
        wo[c] = lds_read16(wa + buf * Tile::kWBytes + 1024 * c);
        so[c] = *(lds_u8*)(swa + (scales_group(s, s0) & 1) * Tile::kScaleBytes + scales_byte(s, s0) + 512 * c);
      } else {
        u32x2 half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int l = lane % 16, k = 32 * g + 8 * q + 4 * h + l / 4, pair = 4 * wn + 2 * c + i / 16;
          half[h] = f8::read_tr16(base + Tile::kWide + (s & 1) * Tile::kWideBytes + k * 2 * kCols + 32 * (pair ^ pair_swizzle<kCols>(k)) +
                                  16 * ((l % 4 / 2) ^ (k >> 3 & 1)) + 8 * (l % 2));
        }
        wt[c][q] = u32x4{half[0][0], half[0][1], half[1][0], half[1][1]};
      }
    };
    auto read_x = [&](int to, int q, int b, uint32_t buf) __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < P; ++p) xo[to][p][q] = lds_read16((xa ^ (16 * q)) + buf * Tile::kXBytes + p * Tile::kPartBytes + 32 * 128 * b);
    };
    // !OI: the codes of a step (in raw buffer `buf`) to their values, a chunk a thread: row k, 32 columns.
    u32x4 raw;
    uint32_t raw_scale;
    const int ck = threadIdx.x % 64, cc = threadIdx.x / 64;
    auto read_codes = [&](uint32_t buf) __attribute__((always_inline)) {
      raw = lds_read16(base + Tile::kW + buf * Tile::kWBytes + ck * 32 * Tile::WN + 16 * (cc ^ code_swizzle<kCols>(ck)));
      const int block = kCols == 64 ? (n0 / kBlock & 3) + cc : cc;
      raw_scale = *(lds_u8*)(base + Tile::kScale + buf * Tile::kScaleBytes + 256 * (block / 4) + 4 * ck + block % 4);
    };
    auto write_values = [&](int s) __attribute__((always_inline)) {
      const float f = scale_operand(raw_scale);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(lds_u32x4_rw*)(base + Tile::kWide + (s & 1) * Tile::kWideBytes + ck * 2 * kCols + 32 * ((2 * cc + e / 2) ^ pair_swizzle<kCols>(ck)) +
                         16 * ((e & 1) ^ (ck >> 3 & 1))) = __builtin_bit_cast(u32x4, widen8(raw[e], f));
    };

    if constexpr (OI) {
      request_scales(0, 0);
    } else {
      request_scales(s0, BUF - 1);
      request_codes(s0, BUF - 1);
    }
#pragma unroll
    for (int j = 0; j < BUF - 1; ++j) request(s0 + j, j, 0, kLoads);
    if constexpr (OI) {
      request(s0 + BUF - 1, BUF - 1, 0, kBehind);
      wait_loads<(BUF - 2) * kLoads + kBehind>();
      lds_barrier();
    } else {
      wait_loads<(BUF - 2) * kLoads>();
      lds_barrier();
      read_codes(BUF - 1);
      write_values(s0);
      lds_barrier();
      request(s0 + BUF - 1, BUF - 1, 0, kBehind);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      read_w(0, q, s0, 0);
      read_w(1, q, s0, 0);
      read_x(kOne ? 1 : 0, q, 0, 0);
    }
    uint32_t cur = 0, left = BUF - 1;  // the step's buffer and the one before it
    for (int s = s0; s < s1; ++s) {
      const uint32_t next = cur + 1 == BUF ? 0 : cur + 1;
      if constexpr (!OI) read_codes(cur);  // of the next step
      uint32_t sw[2];
      u32x4 wc[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if constexpr (OI) {
          wc[c] = wo[c];
          sw[c] = so[c];
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) wv[c][q] = __builtin_bit_cast(bf16x8, wt[c][q]);
        }
      }
      if constexpr (kOne) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int q = 0; q < 4; ++q) xo[0][p][q] = xo[1][p][q];
        if constexpr (!OI) write_values(s + 1);
      }
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        if (b == TB - 1) {
          wait_loads<(BUF - 2) * kLoads>();
          lds_barrier();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (OI) {
            if (b == 0)
#pragma unroll
              for (int c = 0; c < 2; ++c) wv[c][q] = widen8(wc[c][q], scale_operand(sw[c]));
          } else if constexpr (!kOne) {
            if (b == 0 && q == 2) write_values(s + 1);
          }
          if (b + 1 < TB) {
            read_x((b + 1) % 2, q, b + 1, cur);
          } else {
            read_w(0, q, s + 1, next);
            read_w(1, q, s + 1, next);
            read_x(kOne ? 1 : 0, q, 0, next);
          }
#pragma unroll
          for (int p = P - 1; p >= 0; --p)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              acc[c][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wv[c][q], __builtin_bit_cast(bf16x8, xo[b % 2][p][q]), acc[c][b], 0, 0, 0);
#pragma unroll
          for (int c = 0; c < 2 * P; ++c) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);  // LDS read
            __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);  // VALU
          }
          __builtin_amdgcn_sched_barrier(0);
          const bool behind = b == TB - 1;
          const int at = behind ? q : 4 * (b + 1) + q;
          request(behind ? s + BUF : s + BUF - 1, behind ? cur : left, loads_before(at), loads_before(at + 1));
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
int run_f4_wide(mx_backend* b, const char* name, const F4DenseDesc& d, const WideX& x, int slices) {
  DenseArgs a = dense_args(d);
  a.ldx = (int)x.pitch;
  a.ldw = (int)x.w_values;
  a.x_part = x.part;
  unsigned grid = 0;
  MX_TRY(set_tiles(b, d, a, Tile::kRows, Tile::kCols, Tile::kThreads, kStep, slices, &grid));
  auto k = f4_wide_kernel<Tile>;
  MX_CHECK_HIP(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, Tile::kLds));
  return launch(b, name, [&] { dispatch(k, dim3(grid), dim3(Tile::kThreads), Tile::kLds, b->stream, a); });
}

}  // namespace
}  // namespace f4
}  // namespace mx
