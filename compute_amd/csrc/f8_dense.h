// What the kernels of the dense product over 8-bit floating-point blocks share.
#pragma once

#include "f8_common.h"
#include "mxrt_internal.h"

namespace mx {
namespace f8 {

struct DenseArgs {
  const uint8_t* x;  // codes
  const void* xf;    // or float values
  const float* x_scale;
  const uint8_t* w;
  const float* w_scale;
  const void* bias;
  void* out;
  int M, K, N, KB, NB;
  int b_dt, out_dt, act, oi;
  int tiles_n, vec_out;
  int first;          // few rows: the launch's first strip of columns
  int S, kps;         // slices of K of a tile, blocks of a slice
  char* part;         // [tile][slice] sums (S > 1)
  uint32_t* arrived;  // [tile], zero between launches
};

__device__ __forceinline__ f32x4 mfma_f8(const i32x8& a, const i32x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// The sum of products of one block.
template <bool WIDE>
__device__ __forceinline__ f32x4 block_sum(const i32x8& a, const i32x8& b) {
  f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8((uint32_t)a[2 * j], (uint32_t)a[2 * j + 1]),
                                                  widen8((uint32_t)b[2 * j], (uint32_t)b[2 * j + 1]), t, 0, 0, 0);
    return t;
  } else {
    return mfma_f8(a, b, t);
  }
}

inline DenseArgs dense_args(const F8DenseDesc& d) {
  const bool codes = d.x_dt == MX_DTYPE_F8E4M3FN;
  return DenseArgs{codes ? (const uint8_t*)d.x : nullptr, codes ? nullptr : d.x, d.x_scale, d.w, d.w_scale, d.bias, d.out,
                   (int)d.M, (int)d.K, (int)d.N, (int)blocks(d.K), (int)blocks(d.N), d.b_dt, d.out_dt, d.act, d.oi, 0, 0, 0, 1, 0, nullptr, nullptr};
}

// Up to 16 rows, weights [N, K] (f8_skinny.hip); float x up to four rows.
bool skinny_fits(const F8DenseDesc& d);
int skinny_run(mx_backend* b, const F8DenseDesc& d, const char* name);
// Tiles whose operands come through registers (f8_dense_staged.hip).
int staged_run(mx_backend* b, const char* name, const DenseArgs& a, bool wide, int tile, int slices);

}  // namespace f8
}  // namespace mx
