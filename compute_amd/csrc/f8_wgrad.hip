// Weight gradient of a dense layer from its input kept in 8-bit floating-point blocks:
//   dW[k, n] = sum_m (x[m, k] * s[m, k / 128]) * dy[m, n], summed in float32 over the tokens m.
//
// The scales vary along the summed axis, so they belong to the operands: a value code * s is formed
// in bf16 on its way into LDS, which is exact for the quantiser's powers of two (a code has four
// significant bits), and multiplied by dy on the bf16 matrix cores.  float32 dy is three bf16 parts
// cut from its bits, h + m + l = dy exactly (eight bits each; parts below 2^-133 are lost), and three
// products.
//
// Both operands lie with the summed axis slowest in memory; the MFMA wants it fastest, so LDS holds
// them transposed.
#include <algorithm>

#include "f8_common.h"
#include "mxrt_internal.h"

namespace mx {
namespace {
using namespace f8;

struct WGradArgs {
  const uint8_t* x;
  const float* x_scale;
  const void* dy;
  void* out;
  int M, K, N, KB;
  int out_dt, oi;
  int tiles_n;
};

__device__ __forceinline__ f32x4 mfma_bf16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The bf16 parts of a float32 value, each the top 16 bits of what the ones before it left.  An
// infinity or NaN is its first part.
__device__ __forceinline__ void parts_of(float v, uint16_t (&p)[3]) {
  const uint32_t h = __float_as_uint(v) & 0xffff0000u;
  const bool special = (h & 0x7f800000u) == 0x7f800000u;
  const float r1 = special ? 0.0f : v - __uint_as_float(h);
  const uint32_t m = __float_as_uint(r1) & 0xffff0000u;
  const float r2 = r1 - __uint_as_float(m);
  p[0] = (uint16_t)(h >> 16);
  if (special && (__float_as_uint(v) & 0x7fffffu)) p[0] |= 0x40;  // a NaN stays one
  p[1] = (uint16_t)(m >> 16);
  p[2] = (uint16_t)(__float_as_uint(r2) >> 16);
}

// Any sizes, alignment and layout: 64 (k) x 64 (n) tiles, tokens in steps of 32.
constexpr int kAnyTile = 64, kAnyThreads = 256, kAnyStep = 32, kAnyPitch = kAnyStep + 8;

template <bool F32>
__global__ __launch_bounds__(kAnyThreads) void f8_wgrad_any_kernel(WGradArgs a) {
  constexpr int P = F32 ? 3 : 1;
  __shared__ __align__(16) uint16_t xs[kAnyTile * kAnyPitch], ds[P][kAnyTile * kAnyPitch];
  const int k0 = (int)(blockIdx.x / (unsigned)a.tiles_n) * kAnyTile, n0 = (int)(blockIdx.x % (unsigned)a.tiles_n) * kAnyTile;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, i = lane % 16, g = lane / 16;
  f32x4 acc[4] = {};
  for (int m0 = 0; m0 < a.M; m0 += kAnyStep) {
    __syncthreads();
    for (int c = threadIdx.x; c < kAnyTile * kAnyStep; c += kAnyThreads) {
      const int m = m0 + c / kAnyTile, j = c % kAnyTile;
      float v = 0.0f;
      if (m < a.M && k0 + j < a.K)
        v = decode4(a.x[(int64_t)m * a.K + k0 + j]).x * a.x_scale[(int64_t)m * a.KB + (k0 + j) / kBlock];
      xs[j * kAnyPitch + c / kAnyTile] = f32_to_bf16(v);
      const bool in = m < a.M && n0 + j < a.N;
      const int64_t at = in ? (int64_t)m * a.N + n0 + j : 0;
      if constexpr (F32) {
        uint16_t p[3];
        parts_of(in ? ((const float*)a.dy)[at] : 0.0f, p);
#pragma unroll
        for (int q = 0; q < 3; ++q) ds[q][j * kAnyPitch + c / kAnyTile] = p[q];
      } else {
        ds[0][j * kAnyPitch + c / kAnyTile] = in ? ((const uint16_t*)a.dy)[at] : (uint16_t)0;
      }
    }
    __syncthreads();
    const u32x4 xa = *(const u32x4*)(xs + (16 * wave + i) * kAnyPitch + 8 * g);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int q = P - 1; q >= 0; --q)
        acc[c] = mfma_bf16(xa, *(const u32x4*)(ds[q] + (16 * c + i) * kAnyPitch + 8 * g), acc[c]);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int n = n0 + 16 * c + i;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = k0 + 16 * wave + 4 * g + r;
      if (n < a.N && k < a.K) store_f(a.out, a.oi ? (int64_t)n * a.K + k : (int64_t)k * a.N + n, a.out_dt, acc[c][r]);
    }
  }
}

}  // namespace

const char* f8_wgrad_name(const F8WGradDesc&) { return "f8_wgrad_any"; }

int f8_wgrad_run(mx_backend* b, const F8WGradDesc& d) {
  if (d.K == 0 || d.N == 0) return MX_OK;
  WGradArgs a{d.x, d.x_scale, d.dy, d.out, (int)d.M, (int)d.K, (int)d.N, (int)blocks(d.K), d.out_dt, d.oi, 0};
  const int64_t tk = (d.K + kAnyTile - 1) / kAnyTile, tn = (d.N + kAnyTile - 1) / kAnyTile;
  if (tk * tn >= (int64_t)1 << 31) return set_error(MX_ERR_INVALID, "F8WeightGradient: more than 2^31 workgroups");
  a.tiles_n = (int)tn;
  auto k = d.dy_dt == MX_DTYPE_FLOAT32 ? f8_wgrad_any_kernel<true> : f8_wgrad_any_kernel<false>;
  return launch(b, f8_wgrad_name(d), [&] {
    dispatch(k, dim3((unsigned)(tk * tn)), dim3(kAnyThreads), 0, b->stream, a);
  });
}

}  // namespace mx
