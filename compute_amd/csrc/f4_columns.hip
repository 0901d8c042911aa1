// Dense product over 4-bit floating-point blocks for few rows (decode), weights [K, N]: up to four rows of one matrix or of each expert.
//
// The blocks run across k here, so that a matrix instruction would need the codes turned and widened through LDS (f4_wide.h); with a few
// rows the work is the weights' bytes, and plain FMAs keep up.  A lane owns eight columns, a word of codes of each k with one scale:
// four conversions and eight FMAs a row of x, which is float32 here (bf16 exactly, and float32 itself: no parts).  A wave covers 512
// columns, two lines of a row of w, and takes eight k at a time, the next eight requested before they are multiplied.  A workgroup's
// eight waves share the k of its slice of K; their sums meet in LDS in wave order, the slices' in scratch in slice order.
//   1 row of bf16, [4096] x 11008, 12.0 us (20.9 by the tiles of f4_wide.h): a launch, the first loads, 4 us of FMAs and conversions, and
// the join of the slices.  Four rows, 18.9: a workgroup multiplies R rows whatever it has of them.  64 rows of 32 experts,
// [2048] x 1536, 27.7 (R = 4, most experts with a row or two).  Eight rows: the FMAs take longer than the tiles.
#include <algorithm>

#include "f4_dense.h"

namespace mx {
namespace f4 {
namespace {

constexpr int kWaves = 8, kThreads = kColumnsThreads, kCols = kColumnsOfGroup, kRows = 8, kStep = kColumnsStep;  // kRows: k of a wave and step
constexpr int kChunk = 512;  // k of x in LDS at a time
constexpr int kAhead = 1;    // steps requested before one is multiplied (two: no faster for one row, 33 against 26 us for experts)
static_assert(kThreads == 64 * kWaves && kStep == kRows * kWaves, "waves of a workgroup");
static_assert(kCols == 64 * 8 && kCols == kThreads, "a word of codes a lane; a column a thread at the end");
static_assert(kChunk % kStep == 0 && kChunk == kThreads, "whole steps; a value of each row a thread");

template <bool F32, int R>
__global__ __launch_bounds__(kThreads) void f4_columns_kernel(DenseArgs a) {
  __shared__ __align__(16) float x[R][kChunk];
  __shared__ __align__(16) float sums[2][kWaves][kCols];
  __shared__ int word;
  const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
  TilePlace place;
  TileRows rows;
  if (!tile_place(a, R, place) || !locate_rows(a, place.mt, R, rows)) return;
  const int count = min(R, rows.end - rows.first), n0 = kCols * place.nt;
  const bool live = rows.expert < a.E;
  if (!live && place.slice != 0) return;
  float acc[R][8] = {};
  if (live) {
    const int steps = (a.K + kStep - 1) / kStep, s0 = place.slice * a.kps, s1 = min(steps, s0 + a.kps);
    const int64_t w_pitch = a.ldw / 2, s_pitch = (a.ldw + kBlock - 1) / kBlock;
    const uint8_t *w = a.w + rows.expert * (a.K * w_pitch), *ws = a.ws + rows.expert * (a.K * s_pitch);
    const int col = n0 + 8 * lane < a.ldw ? n0 + 8 * lane : 0;  // lanes past the last column read the first and store nothing
    struct Codes {
      uint32_t w[kRows], s[kRows];
    };
    auto request = [&](int s) __attribute__((always_inline)) {  // k past the last are the last, against zeros of x
      Codes o;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int k = min(kStep * s + kRows * wave + r, a.K - 1);
        o.w[r] = *(const uint32_t*)(w + k * w_pitch + col / 2);
        o.s[r] = ws[k * s_pitch + col / kBlock];
      }
      return o;
    };
    Codes codes[kAhead + 1] = {};
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (s0 + q < s1) codes[q] = request(s0 + q);
    auto step = [&](int s, const Codes& o) __attribute__((always_inline)) {
      const int in = kStep * (s - s0) % kChunk;
      if (in == 0) {
        __syncthreads();
        const int k = kStep * s + t;
#pragma unroll
        for (int m = 0; m < R; ++m) {
          const int64_t at = (int64_t)(rows.first + min(m, count - 1)) * a.ldx + min(k, a.K - 1);
          const float v = F32 ? ((const float*)a.x)[at] : bf16_to_f32(((const uint16_t*)a.x)[at]);
          x[m][t] = m < count && k < a.K ? v : 0.0f;
        }
        __syncthreads();
      }
#pragma unroll
      for (int h = 0; h < kRows / 4; ++h) {
        f32x4 xv[R];
#pragma unroll
        for (int m = 0; m < R; ++m) xv[m] = *(const f32x4*)&x[m][in + kRows * wave + 4 * h];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t c = o.w[4 * h + r];
          const float f = scale_operand(o.s[4 * h + r]);
          const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 1),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, f, 3)};
#pragma unroll
          for (int m = 0; m < R; ++m)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[m][j] = fmaf(xv[m][r], v[j / 2][j % 2], acc[m][j]);
        }
      }
    };
    for (int s = s0; s < s1; s += kAhead + 1)
#pragma unroll
      for (int q = 0; q <= kAhead; ++q) {
        if (s + q + kAhead < s1) codes[(q + kAhead) % (kAhead + 1)] = request(s + q + kAhead);
        if (s + q < s1) step(s + q, codes[q]);
      }
  }
  float sum[R];
#pragma unroll
  for (int m = 0; m < R; ++m) {  // a barrier a row: the buffer written next was read before the last one
    *(f32x4*)&sums[m % 2][wave][8 * lane] = f32x4{acc[m][0], acc[m][1], acc[m][2], acc[m][3]};
    *(f32x4*)&sums[m % 2][wave][8 * lane + 4] = f32x4{acc[m][4], acc[m][5], acc[m][6], acc[m][7]};
    __syncthreads();
    sum[m] = 0.0f;
#pragma unroll
    for (int q = 0; q < kWaves; ++q) sum[m] += sums[m % 2][q][t];
  }
  if (live && a.S > 1) {  // the slices' sums, as in join_slices
    constexpr int kSc1 = 16, kPart = R * kCols * 4;
    const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(a.part + (int64_t)place.tile * a.S * kPart, 0, a.S * kPart, 0x00027000);
    auto at = [&](int slice, int m) { return (uint32_t)(slice * kPart + (m * kCols + t) * 4); };
#pragma unroll
    for (int m = 0; m < R; ++m) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(sum[m]), prs, at(place.slice, m), 0, kSc1);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t == 0) {
      const uint32_t before = __hip_atomic_fetch_add(&a.arrived[place.tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const bool last = before + 1u == (uint32_t)a.S;
      word = last;
      if (last) __hip_atomic_store(&a.arrived[place.tile], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (word == 0) return;
#pragma unroll
    for (int m = 0; m < R; ++m) sum[m] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < a.S; ++s)
#pragma unroll
      for (int m = 0; m < R; ++m) sum[m] += __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, at(s, m), 0, kSc1));
  }
  const int n = n0 + t;
  if (n >= a.N) return;
  const float bias = live && a.bias ? load_f(a.bias, (int64_t)rows.expert * a.N + n, a.b_dt) : 0.0f;
#pragma unroll
  for (int m = 0; m < R; ++m)
    if (m < count) store_f(a.out, (int64_t)(rows.first + m) * a.N + n, a.out_dt, live ? act_result(sum[m] + bias, a.act, a.out_dt == MX_DTYPE_FLOAT32) : 0.0f);
}

template <bool F32>
int run(mx_backend* b, const char* name, const F4DenseDesc& d, const ColumnsX& x, int rows, int slices) {
  DenseArgs a = dense_args(d);
  a.ldx = (int)x.pitch;
  a.ldw = (int)x.w_values;
  unsigned grid = 0;
  MX_TRY(set_tiles(b, d, a, rows, kCols, kThreads, kStep, slices, &grid));
  auto k = rows == 1 ? f4_columns_kernel<F32, 1> : rows == 2 ? f4_columns_kernel<F32, 2> : f4_columns_kernel<F32, 4>;
  return launch(b, name, [&] { dispatch(k, dim3(grid), dim3(kThreads), 0, b->stream, a); });
}

}  // namespace

int columns_run(mx_backend* b, const char* name, const F4DenseDesc& d, const ColumnsX& x, int rows, int slices) {
  return x.f32 ? run<true>(b, name, d, x, rows, slices) : run<false>(b, name, d, x, rows, slices);
}

}  // namespace f4
}  // namespace mx
