// Dense product over 8-bit floating-point blocks for up to 16 rows (decode), weights [N, K].
//
// The weights are read once and are nearly all the bytes, so the work is to keep them coming: a workgroup
// owns 16 or 32 columns (C operands of 16), its waves take the blocks of 128 k in turn, and a wave keeps up to 2 kAhead blocks in flight
// straight into the registers that the MFMA reads (lane (i, g): 32 codes of column i from 32 g; 16 segments of
// 128 bytes an instruction pair).  There is no LDS on the way, no
// barrier before the end and nothing to share but x.  The waves' sums are added through LDS in wave order.
//
// [1, 4096] x [4096, 11008] reads 45 MB in 9.7 to 10.7 us (4.2 to 4.6 TB/s; a large copy moves 4.9); run_skinny has more.
//
// x: codes with their scales, each lane (i, g) its own 32 codes of row i; or up to four rows of float values, which
// each wave makes into codes for its own blocks, 16 lanes a row, as the quantiser does, and passes to the MFMA's
// lanes through LDS of its own.  A wave's blocks are read by no other wave of the workgroup; every workgroup repeats
// the conversion of the whole x, which is why it stops at four rows (one pass of the wave).
#include <algorithm>

#include "f8_dense.h"

namespace mx {
namespace f8 {
namespace {

enum XKind { kCodes, kBf16, kF32 };

constexpr int kAhead = 2;        // blocks requested at once, with as many in flight from before
constexpr int kFloatRows = 4;    // rows that a wave converts in one pass
constexpr int kPitch = kBlock + 16;

template <int X, bool WIDE, int NW, int C>
__global__ __launch_bounds__(64 * NW) void f8_skinny_kernel(DenseArgs a) {
  constexpr bool kFloat = X != kCodes;
  __shared__ __align__(16) uint8_t codes[kFloat ? NW : 1][kFloat ? kFloatRows * kPitch : 16];
  __shared__ float scales[kFloat ? NW : 1][kFloatRows];
  __shared__ f32x4 sums[NW][C][64];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = lane % 16, g = lane / 16;
  const int n0 = 16 * C * (a.first + xcd_order((int)blockIdx.x, (int)gridDim.x));
  const uint8_t* wrow[C];
#pragma unroll
  for (int c = 0; c < C; ++c) wrow[c] = a.w + (int64_t)min(n0 + 16 * c + i, a.N - 1) * a.K + 32 * g;
  const uint8_t* xrow = a.x + (int64_t)min(i, a.M - 1) * a.K + 32 * g;
  const float* sw = a.w_scale + (int64_t)(n0 / kBlock) * a.KB;
  const bool row = i < a.M;
  const int fr = g, fk = 8 * i;  // float x: the lane's row and first value of a block

  struct Block {
    u32x4 w[C][2], x[X == kBf16 ? 1 : 2];
    float sw, sx;
  };
  auto request = [&](int kb, bool whole) __attribute__((always_inline)) {
    Block o;
    const int k = kb * kBlock, left = a.K - k;  // whole: at least a block
    auto load = [&](const uint8_t* p, int n) __attribute__((always_inline)) { return whole ? load16_any(p) : load16(p, n); };
#pragma unroll
    for (int c = 0; c < C; ++c) {
      o.w[c][0] = load(wrow[c] + k, left - 32 * g);
      o.w[c][1] = load(wrow[c] + k + 16, left - 32 * g - 16);
    }
    o.sw = sw[kb];
    o.x[0] = u32x4{0u, 0u, 0u, 0u};
    if constexpr (X != kBf16) o.x[1] = o.x[0];
    o.sx = 0.0f;
    if constexpr (!kFloat) {
      if (row) {
        o.x[0] = load(xrow + k, left - 32 * g);
        o.x[1] = load(xrow + k + 16, left - 32 * g - 16);
        o.sx = a.x_scale[(int64_t)i * a.KB + kb];
      }
    } else if (fr < a.M) {
      constexpr int E = X == kBf16 ? 2 : 4;
      const uint8_t* p = (const uint8_t*)a.xf + ((int64_t)fr * a.K + k + fk) * E;
      o.x[0] = load(p, (left - fk) * E);
      if constexpr (X == kF32) o.x[1] = load(p + 16, (left - fk) * E - 16);
    }
    return o;
  };
  // Codes and row scale of a block for the MFMA's lane.
  auto operand = [&](const Block& blk, float& sx) __attribute__((always_inline)) {
    if constexpr (!kFloat) {
      sx = blk.sx;
      return join(blk.x[0], blk.x[1]);
    } else {
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (X == kF32) {
          v[e] = __uint_as_float(blk.x[0][e]);
          v[4 + e] = __uint_as_float(blk.x[1][e]);
        } else {
          v[2 * e] = __uint_as_float(blk.x[0][e] << 16);
          v[2 * e + 1] = __uint_as_float(blk.x[0][e] & 0xffff0000u);
        }
      }
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, finite_bits(v[e]));
      const int e2 = scale_exponent(row_max(top));
      const float inv = pow2(-e2);
      if (fr < a.M) {
        *(u32x2*)(codes[wave] + fr * kPitch + fk) =
            u32x2{encode4(scaled(v[0], inv), scaled(v[1], inv), scaled(v[2], inv), scaled(v[3], inv)),
                  encode4(scaled(v[4], inv), scaled(v[5], inv), scaled(v[6], inv), scaled(v[7], inv))};
        if (i == 0) scales[wave][fr] = pow2(e2);
      }
      // One wave writes and reads: its LDS operations keep their order.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      i32x8 o = {0, 0, 0, 0, 0, 0, 0, 0};
      sx = 0.0f;
      if (row) {
        o = read32(codes[wave] + i * kPitch + 32 * g);
        sx = scales[wave][i];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      return o;
    }
  };

  f32x4 acc[C] = {};
  auto multiply = [&](const Block& blk) __attribute__((always_inline)) {
    float sx;
    const i32x8 xo = operand(blk, sx);
    const float sc = sx * blk.sw;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const f32x4 t = block_sum<WIDE>(join(blk.w[c][0], blk.w[c][1]), xo);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[c][r] = fmaf(t[r], sc, acc[c][r]);
    }
  };
  // Whole blocks wave, wave + NW, ..: groups of kAhead, the next requested before the present is multiplied.
  const int whole = a.K / kBlock, mine = whole > wave ? (whole - wave + NW - 1) / NW : 0;
  Block blk[2][kAhead];
  auto group = [&](int set, int first) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (first + j < mine) blk[set][j] = request(wave + NW * (first + j), true);
  };
  auto products = [&](int set, int first) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (first + j < mine) multiply(blk[set][j]);
  };
  group(0, 0);
  for (int first = 0; first < mine; first += 2 * kAhead) {
    group(1, first + kAhead);
    products(0, first);
    group(0, first + 2 * kAhead);
    products(1, first + kAhead);
  }
  if (whole < a.KB && wave == whole % NW) multiply(request(whole, false));  // the short last block
#pragma unroll
  for (int c = 0; c < C; ++c) sums[wave][c][lane] = acc[c];
  __syncthreads();
  for (int o = threadIdx.x; o < 16 * C * a.M; o += 64 * NW) {
    const int m = o / (16 * C), n = o % (16 * C);
    if (n0 + n >= a.N) continue;
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < NW; ++q) v += sums[q][n / 16][16 * (n % 16 / 4) + m][n % 4];
    if (a.bias) v += load_f(a.bias, n0 + n, a.b_dt);
    store_f(a.out, (int64_t)m * a.N + n0 + n, a.out_dt, act_fast(v, a.act));
  }
}

// Waves of a workgroup and operands of columns.  Measured (us, bf16 results; waves x operands 4x1, 4x2, 8x1, 16x1; profiles/f8_tile_sweeps.txt):
//   one bf16 row   [4096] x 11008    9.7  11.3  10.3  12.0      16 rows  [2048] x 32001, f32   19.8  15.6  21.2  29.3
//                  [4096] x 4096     6.3   7.7   5.2   4.6               [4096] x 14336         19.7  15.5  19.7  22.0
//                  [14336] x 4096   18.5  20.1  12.6  11.9               [4096] x 4096           6.8   8.7   6.5   6.7
//                                                              8 rows    [14336] x 4096         15.2  21.2  14.1  14.1
// From 768 strips the CUs are full with two operands, which share the lanes' x (as many bytes as the weights with 16
// rows); from 512 with four waves; below, the waves have to come from K, and with more rows their sums cost more.
template <int X, bool WIDE>
int run_skinny(mx_backend* b, const char* name, DenseArgs a) {
  auto go = [&](auto k, int waves, int c) {
    return launch_runs(b, name, ((int64_t)a.N + 16 * c - 1) / (16 * c), 64 * waves, [&](int64_t first, unsigned count) {
      a.first = (int)first;
      dispatch(k, dim3(count), dim3(64 * waves), 0, b->stream, a);
    });
  };
  const int strips = (int)(((int64_t)a.N + 15) / 16);
  if (a.M <= kFloatRows) {  // float rows and their codes alike: the same order of sums, the same bits
    if (strips < 512) return go(f8_skinny_kernel<X, WIDE, 16, 1>, 16, 1);
  } else if constexpr (X == kCodes) {
    if (strips >= 768) return go(f8_skinny_kernel<X, WIDE, 4, 2>, 4, 2);
    if (strips < 512) return go(f8_skinny_kernel<X, WIDE, 8, 1>, 8, 1);
  }
  return go(f8_skinny_kernel<X, WIDE, 4, 1>, 4, 1);
}

}  // namespace

bool skinny_fits(const F8DenseDesc& d) {
  return d.oi && d.K > 0 && d.M <= (d.x_dt == MX_DTYPE_F8E4M3FN ? 16 : kFloatRows);
}

int skinny_run(mx_backend* b, const F8DenseDesc& d, const char* name) {
  DenseArgs a = dense_args(d);
  const bool wide = d.out_dt == MX_DTYPE_FLOAT32;
  switch (d.x_dt) {
    case MX_DTYPE_FLOAT32: return wide ? run_skinny<kF32, true>(b, name, a) : run_skinny<kF32, false>(b, name, a);
    case MX_DTYPE_BFLOAT16: return wide ? run_skinny<kBf16, true>(b, name, a) : run_skinny<kBf16, false>(b, name, a);
    default: return wide ? run_skinny<kCodes, true>(b, name, a) : run_skinny<kCodes, false>(b, name, a);
  }
}

}  // namespace f8
}  // namespace mx
