// Dense product over 4-bit floating-point blocks for few rows (decode), weights [N, K]: up to 16 rows of codes or bf16 values, or five of
// float32 values, of one matrix or of each expert.
//
// The weights are read once and are nearly all the bytes, so the work is to keep them coming: a workgroup owns 16 C columns,
// its waves take the units of 256 k in turn, and a wave keeps up to 2 kAhead units in flight straight into the registers of the
// MFMA (lane (i = lane % 16, g = lane / 16): the blocks g and 4 + g of a unit of column i, 16 lines of 128 bytes an instruction pair).
// There is no barrier before the end and nothing to share but x.  The waves' sums are added through LDS in wave order.
//
// x in codes: v_mfma_scale_f32_16x16x128_f8f6f4, two a unit, each lane's blocks with their scale bytes.  x in bf16: eight
// v_mfma_f32_16x16x32_bf16, the weights widened in registers; float32 values are three bf16 parts (f4_prepare.hip), each a row of the
// operand, whose results are added at the end: no more instructions than for bf16, and five rows instead of sixteen.
//   One or two rows of bf16 (PARTS 8): eight loads a unit of 16 bytes for a few lanes cost more than the weights' three, so that
//   lane (i, g) loads one chunk, the (i % 8)-th of row i / 8, and an instruction takes the lanes whose chunk it is and zeros from
//   the others: a chunk's results stay in a row of their own and are added at the end.
//
// Measured: 1 row of bf16, [4096] x 11008, 8.2 us (2.9 TB/s of weights; 24 MB are four units a wave, so that starting the waves is
// as much as the bytes); 64 rows of 32 experts, [2048] x 1536, 14.1 (3.8 TB/s).
#include <algorithm>

#include "f4_dense.h"

namespace mx {
namespace f4 {
namespace {

constexpr int kUnit = 256;

struct SkinnyArgs {
  DenseArgs d;
  int strips, per;  // strips of columns, rows of a group
};

template <bool CODES, int PARTS, int NW, int C>
__global__ __launch_bounds__(64 * NW) void f4_skinny_kernel(SkinnyArgs s) {
  constexpr int kAhead = CODES || PARTS == 8 ? 2 : 1;  // units requested at once, with as many in flight from before
  constexpr bool kSpread = PARTS == 8;
  constexpr int kX = CODES ? 2 : kSpread ? 1 : 8;  // 16-byte chunks of x of a lane and unit
  const DenseArgs& a = s.d;
  __shared__ f32x4 sums[NW][C][64];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = lane % 16, g = lane / 16;
  // Groups that are there are dealt out in runs to the XCDs (a launch holds the most that could be).
  const int64_t items = (int64_t)count_tiles(a, s.per, a.tiles_m) * s.strips, of = items - a.first;
  if ((int64_t)blockIdx.x >= of) return;
  const int64_t at = a.first + f8::xcd_order((int)blockIdx.x, of < (int64_t)gridDim.x ? (int)of : (int)gridDim.x);
  const int group = (int)(at / s.strips), n0 = 16 * C * (int)(at - (int64_t)group * s.strips);
  TileRows rows;
  if (!locate_rows(a, group, s.per, rows)) return;
  const int count = min(s.per, rows.end - rows.first);
  f32x4 acc[C] = {};
  if (rows.expert < a.E) {
    const int row_bytes = a.ldw / 2, row_scales = a.ldw / kBlock;
    const uint8_t* wrow[C];
    const uint8_t* wsrow[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int64_t n = (int64_t)rows.expert * a.N + min(n0 + 16 * c + i, a.N - 1);
      wrow[c] = a.w + n * row_bytes + 16 * g;
      wsrow[c] = a.ws + n * row_scales;
    }
    const int m = i / PARTS;  // the lane's row of x
    const bool row = m < count;
    const int64_t xm = rows.first + min(m, count - 1);
    const uint8_t* xrow = a.x + (PARTS == 3 ? (i % 3) * a.x_part : 0) + xm * a.ldx + (CODES ? 16 : 64) * g + (kSpread ? 256 * (i / 4 % 2) + 16 * (i % 4) : 0);
    const uint8_t* xsrow = CODES ? a.xs + xm * row_scales : nullptr;

    struct Unit {
      u32x4 w[C][2], x[kX];
      u32x2 sw[C], sx;
    };
    // A unit, whole or the last, which may have the first half only (rows of w and codes are multiples of 128; those of x in
    // bf16 end where they end, in whole chunks).
    auto request = [&](int u, bool whole) __attribute__((always_inline)) {
      Unit o;
      const bool second = whole || u * kUnit + 128 < a.ldw;
      const u32x4 zero = {0u, 0u, 0u, 0u};
      auto scales = [&](const uint8_t* p) __attribute__((always_inline)) {
        return u32x2{*(const uint32_t*)p, second ? *(const uint32_t*)(p + 4) : 0u};
      };
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint8_t* p = wrow[c] + (int64_t)u * (kUnit / 2);
        o.w[c][0] = *(const u32x4*)p;
        o.w[c][1] = second ? *(const u32x4*)(p + 64) : zero;
        o.sw[c] = scales(wsrow[c] + u * (kUnit / kBlock));
      }
#pragma unroll
      for (int q = 0; q < kX; ++q) o.x[q] = zero;
      o.sx = u32x2{0u, 0u};
      if (row) {
        const uint8_t* p = xrow + (int64_t)u * (CODES ? kUnit / 2 : 2 * kUnit);
#pragma unroll
        for (int q = 0; q < kX; ++q) {
          if constexpr (CODES) {
            if (q == 0 || second) o.x[q] = *(const u32x4*)(p + 64 * q);
          } else if constexpr (kSpread) {
            if (whole || u * kUnit + 128 * (i / 4 % 2) + 32 * g + 8 * (i % 4) < a.K) o.x[q] = *(const u32x4*)p;
          } else {
            if (whole || u * kUnit + 128 * (q / 4) + 32 * g + 8 * (q % 4) < a.K) o.x[q] = *(const u32x4*)(p + 256 * (q / 4) + 16 * (q % 4));
          }
        }
        if constexpr (CODES) o.sx = scales(xsrow + u * (kUnit / kBlock));
      }
      return o;
    };
    auto multiply = [&](const Unit& o) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (CODES) {
          const i32x8 x = {(int)o.x[h][0], (int)o.x[h][1], (int)o.x[h][2], (int)o.x[h][3], 0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const i32x8 w = {(int)o.w[c][h][0], (int)o.w[c][h][1], (int)o.w[c][h][2], (int)o.w[c][h][3], 0, 0, 0, 0};
            acc[c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc[c], 4, 4, 0, (int)(o.sw[c][h] >> (8 * g)), 0, (int)(o.sx[h] >> (8 * g)));
          }
        } else {
          u32x4 x[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[q][e] = !kSpread ? o.x[kSpread ? 0 : 4 * h + q][e] : i % 8 == 4 * h + q ? o.x[0][e] : 0u;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float f = scale_operand(o.sw[c][h] >> (8 * g) & 255u);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(o.w[c][h][q], f), __builtin_bit_cast(bf16x8, x[q]), acc[c], 0, 0, 0);
          }
        }
      }
    };
    // Whole units wave, wave + NW, ..: groups of kAhead, the next requested before the present is multiplied.
    const int whole = a.K / kUnit, units = (a.K + kUnit - 1) / kUnit, mine = whole > wave ? (whole - wave + NW - 1) / NW : 0;
    Unit unit[2][kAhead];
    auto fetch = [&](int set, int first) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (first + j < mine) unit[set][j] = request(wave + NW * (first + j), true);
    };
    auto products = [&](int set, int first) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (first + j < mine) multiply(unit[set][j]);
    };
    fetch(0, 0);
    for (int first = 0; first < mine; first += 2 * kAhead) {
      fetch(1, first + kAhead);
      products(0, first);
      fetch(0, first + 2 * kAhead);
      products(1, first + kAhead);
    }
    if (whole < units && wave == whole % NW) multiply(request(whole, false));
  }
#pragma unroll
  for (int c = 0; c < C; ++c) sums[wave][c][lane] = acc[c];
  __syncthreads();
  const bool live = rows.expert < a.E;
  for (int o = threadIdx.x; o < 16 * C * count; o += 64 * NW) {
    const int m = o / (16 * C), n = o % (16 * C);
    if (n0 + n >= a.N) continue;
    float v = 0.0f;
#pragma unroll
    for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
      for (int q = 0; q < NW; ++q) v += sums[q][n / 16][16 * (n % 16 / 4) + PARTS * m + p][n % 4];
    if (live) {
      if (a.bias) v += load_f(a.bias, (int64_t)rows.expert * a.N + n0 + n, a.b_dt);
      v = act_result(v, a.act, a.out_dt == MX_DTYPE_FLOAT32);
    }
    store_f(a.out, (int64_t)(rows.first + m) * a.N + n0 + n, a.out_dt, v);
  }
}

template <bool CODES, int PARTS, int NW, int C>
int run(mx_backend* b, const char* name, const F4DenseDesc& d, const WideX& x) {
  SkinnyArgs s{dense_args(d), 0, PARTS == 8 ? 2 : skinny_rows(d)};
  s.d.ldx = (int)x.pitch;
  s.d.x_part = x.part;
  s.d.ldw = (int)x.w_values;
  s.strips = (int)((d.N + 16 * C - 1) / (16 * C));
  s.d.tiles_m = (int)most_tiles(d, s.per);
  return launch_runs(b, name, (int64_t)s.d.tiles_m * s.strips, 64 * NW, [&](int64_t first, unsigned count) {
    s.d.first = first;
    dispatch(f4_skinny_kernel<CODES, PARTS, NW, C>, dim3(count), dim3(64 * NW), 0, b->stream, s);
  });
}

template <bool CODES, int PARTS>
int run_shape(mx_backend* b, const char* name, const F4DenseDesc& d, const WideX& x, int shape) {
  switch (shape) {
    case 0: return run<CODES, PARTS, 2, 2>(b, name, d, x);
    case 1: return run<CODES, PARTS, 8, 1>(b, name, d, x);
    case 2: return run<CODES, PARTS, 4, 1>(b, name, d, x);
    default: return run<CODES, PARTS, 4, 4>(b, name, d, x);
  }
}

}  // namespace

int skinny_run(mx_backend* b, const char* name, const F4DenseDesc& d, const WideX& x, int shape) {
  if (d.x_dt == MX_DTYPE_F4E2M1FN) return run_shape<true, 1>(b, name, d, x, shape);
  if (x.parts == 3) return run_shape<false, 3>(b, name, d, x, shape);
  return d.M <= 2 ? run_shape<false, 8>(b, name, d, x, shape) : run_shape<false, 1>(b, name, d, x, shape);
}

}  // namespace f4
}  // namespace mx
