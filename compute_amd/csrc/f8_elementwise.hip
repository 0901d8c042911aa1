// Quantisation into 8-bit floating-point blocks, and the gradient of an activation from its input
// kept in that form.  Both are one pass over their data and bound by HBM.
//
// Quantisation.  With a the largest finite magnitude of a block, its scale s is the smallest power of
// two with a <= 448 s and a code is x / s rounded to nearest even.  A power of two costs nothing in a
// floating format (a code keeps its four significant bits wherever it lies in the range; the block's
// smallest values lose one binade of about 17), the division is exact, so every implementation of the
// definition gives the same codes, and a value read back, code * s, is exact in bf16.
//
// A row of 16 lanes holds a block of 128 values, eight a lane (one 16-byte load of bf16, two of f32,
// one 8-byte store of codes), so that the maximum of a block takes four DPP steps and no LDS.
//
// Activation gradient.  z' = dy * act'(z) (and, gated, dy * up * act'(z) and dy * act(z)) with z and up
// decoded from their codes: 1 or 2 bytes of codes, dy and one or two results per value.  A lane takes
// eight consecutive values, which share a scale.
#include <algorithm>

#include "f8_common.h"
#include "mxrt_internal.h"

namespace mx {
namespace {
using namespace f8;

constexpr int kThreads = 256;
constexpr int kPerLane = 8;                        // values of a lane
constexpr int kLanes = kBlock / kPerLane;          // lanes of a block: a DPP row
constexpr int kGroups = kThreads / kLanes;         // blocks of a workgroup

// Eight consecutive values from element `at`, of which the first n are in the row; the rest 0.
// VEC: rows and array start on 16 bytes, so all eight are in the row or none; otherwise whole chunks still go as vectors,
// from any address ([2048, 14335] bf16 quantised 42 us value by value).
template <bool F32, bool VEC>
__device__ __forceinline__ void load8(const void* p, int64_t at, int n, float (&v)[8]) {
  if (VEC ? n > 0 : n >= 8) {
    const uint8_t* q = (const uint8_t*)p + at * (F32 ? 4 : 2);
    if constexpr (F32) {
      const u32x4 a = VEC ? *(const u32x4*)q : load16_any(q), b = VEC ? *(const u32x4*)(q + 16) : load16_any(q + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
    } else {
      const u32x4 a = VEC ? *(const u32x4*)q : load16_any(q);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(a[i] << 16), v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = !VEC && i < n ? (F32 ? ((const float*)p)[at + i] : bf16_to_f32(((const uint16_t*)p)[at + i])) : 0.0f;
  }
}

template <bool F32, bool VEC>
__device__ __forceinline__ void store8(void* p, int64_t at, int n, const float (&v)[8]) {
  if (VEC ? n > 0 : n >= 8) {
    uint8_t* q = (uint8_t*)p + at * (F32 ? 4 : 2);
    u32x4 o[F32 ? 2 : 1];
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i / 4][i % 4] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 two = {v[2 * i], v[2 * i + 1]};
        o[0][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
      }
    }
#pragma unroll
    for (int h = 0; h < (F32 ? 2 : 1); ++h) {
      if constexpr (VEC)
        *(u32x4*)(q + 16 * h) = o[h];
      else
        __builtin_memcpy(q + 16 * h, &o[h], 16);
    }
  } else if (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) {
        if constexpr (F32)
          ((float*)p)[at + i] = v[i];
        else
          ((uint16_t*)p)[at + i] = f32_to_bf16(v[i]);
      }
  }
}

template <bool VEC>
__device__ __forceinline__ void store_codes8(uint8_t* p, int64_t at, int n, const float (&v)[8], float inv) {
  const u32x2 c = {encode4(scaled(v[0], inv), scaled(v[1], inv), scaled(v[2], inv), scaled(v[3], inv)),
                   encode4(scaled(v[4], inv), scaled(v[5], inv), scaled(v[6], inv), scaled(v[7], inv))};
  if constexpr (VEC) {
    if (n > 0) *(u32x2*)(p + at) = c;
  } else if (n >= 8) {
    __builtin_memcpy(p + at, &c, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[at + i] = (uint8_t)(c[i / 4] >> (8 * (i % 4)));
  }
}

__device__ __forceinline__ uint32_t largest8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, finite_bits(v[i]));
  return m;
}

// One scale per 128 values of a row: block t of the M * KB blocks is row t / KB's.  A launch holds the workgroups from
// `first` on.
template <bool F32, bool VEC>
__global__ __launch_bounds__(kThreads) void f8_quantize_rows_kernel(const void* x, uint8_t* codes, float* scale, int K,
                                                                    int KB, int64_t total, int64_t first) {
  const int64_t t = (first + blockIdx.x) * kGroups + threadIdx.x / kLanes;
  if (t >= total) return;
  const int64_t row = t / KB;
  const int k0 = (int)(t - row * KB) * kBlock + (int)(threadIdx.x % kLanes) * kPerLane;
  const int n = K - k0;
  const int64_t at = row * K + k0;
  float v[8];
  load8<F32, VEC>(x, at, n, v);
  const int e = scale_exponent(row_max(largest8(v)));
  store_codes8<VEC>(codes, at, n, v, pow2(-e));
  if (threadIdx.x % kLanes == 0) scale[t] = pow2(e);
}

// One scale per 128 x 128 block: a workgroup's, its values held in registers between the passes.
template <bool F32, bool VEC>
__global__ __launch_bounds__(kThreads) void f8_quantize_tiles_kernel(const void* x, uint8_t* codes, float* scale, int M,
                                                                     int K, int KB, unsigned first) {
  constexpr int kPasses = kBlock / kGroups;
  __shared__ uint32_t part[kThreads / 64];
  const unsigned at = first + blockIdx.x;  // fewer than 2^32 blocks in 2^45 values
  const int rb = (int)(at / (unsigned)KB), cb = (int)(at % (unsigned)KB);
  const int k0 = cb * kBlock + (int)(threadIdx.x % kLanes) * kPerLane;
  const int n = K - k0;
  float v[kPasses][8];
  uint32_t m = 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = rb * kBlock + p * kGroups + (int)(threadIdx.x / kLanes);
    load8<F32, VEC>(x, (int64_t)row * K + k0, row < M ? n : 0, v[p]);
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p) m = max(m, largest8(v[p]));
  m = row_max(m);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = m;
  __syncthreads();
  for (int i = 0; i < kThreads / 64; ++i) m = max(m, part[i]);
  const int e = scale_exponent(m);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = rb * kBlock + p * kGroups + (int)(threadIdx.x / kLanes);
    store_codes8<VEC>(codes, (int64_t)row * K + k0, row < M ? n : 0, v[p], pow2(-e));
  }
  if (threadIdx.x == 0) scale[(int64_t)rb * KB + cb] = pow2(e);
}

// act(z) and its slope.  GELU in bf16: with x = |z| / sqrt(2) and t = 1 / (1 + 0.415 x), erfc(x) = p(t) exp(-x^2), p a polynomial
// of six terms fitted to exp(x^2) erfc(x) by linear programming: within 1.4e-7 of erfc and, so that the tail's values keep
// bf16's bits, within 3.8e-5 of its own size.  Its exponential is that of the normal density: one exp and one reciprocal for value and
// slope, and the small side of the normal distribution without a cancellation.  With OCML's erfc the kernel took 62 us
// for [2048, 14336], twice the time of its bytes.  float32 takes OCML's all the same: 4.4e-8 of the norm off
// instead of 1.2e-7 with a polynomial, for 55 to 62 us instead of 49 ([2048, 14336]; gated 77 both).
template <int ACT, bool F32>
__device__ __forceinline__ void act_and_slope(float z, float& a, float& s) {
  if constexpr (ACT == MX_ACT_GELU) {
    const float e = __expf(-0.5f * z * z);
    float small;
    if constexpr (F32) {
      small = 0.5f * erfcf(0.70710678118654752f * fabsf(z));
    } else {
      const float t = __builtin_amdgcn_rcpf(fmaf(0.2934493f, fabsf(z), 1.0f));
      float p = fmaf(-0.171013132f, t, 0.523574352f);
      p = fmaf(p, t, -0.132057682f);
      p = fmaf(p, t, 0.332223147f);
      p = fmaf(p, t, 0.211444676f);
      p = fmaf(p, t, 0.235828385f);
      small = 0.5f * p * t * e;
    }
    const float cdf = z < 0.0f ? small : 1.0f - small;
    a = z * cdf;
    s = fmaf(z * 0.39894228040143268f, e, cdf);
  } else if constexpr (ACT == MX_ACT_RELU) {
    a = z < 0.0f ? 0.0f : z;
    s = z > 0.0f ? 1.0f : z == z ? 0.0f : z;
  } else if constexpr (ACT == MX_ACT_SILU) {
    const float g = __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    a = z * g;
    s = g * fmaf(z, 1.0f - g, 1.0f);
  } else if constexpr (ACT == MX_ACT_HARDSWISH) {
    float v = z * (1.0f / 6.0f) + 0.5f;
    v = v > 0.0f ? v : v == v ? 0.0f : v;
    v = v < 1.0f ? v : v == v ? 1.0f : v;
    a = z * v;
    s = z <= -3.0f ? 0.0f : z >= 3.0f ? 1.0f : fmaf(z, 1.0f / 3.0f, 0.5f);
  } else if constexpr (ACT == MX_ACT_TANH) {
    a = tanhf(z);
    // 1 - tanh^2 = 4 e / (1 + e)^2 with e = exp(-2 |z|), without the cancellation
    const float e = __expf(-2.0f * fabsf(z)), d = __builtin_amdgcn_rcpf(1.0f + e);
    s = 4.0f * e * d * d;
  } else {
    a = z;
    s = 1.0f;
  }
}

template <bool VEC>
__device__ __forceinline__ void load_codes8(const uint8_t* p, int64_t at, int n, float scale, float (&v)[8]) {
  u32x2 c = {0u, 0u};
  if constexpr (VEC) {
    if (n > 0) c = *(const u32x2*)(p + at);
  } else if (n >= 8) {
    __builtin_memcpy(&c, p + at, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) c[i / 4] |= (uint32_t)p[at + i] << (8 * (i % 4));
  }
  const f32x4 a = decode4(c.x), b = decode4(c.y);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = a[i] * scale, v[4 + i] = b[i] * scale;
}

struct ActGradArgs {
  const uint8_t *z, *up;
  const float *z_scale, *up_scale;
  const void* dy;
  void *dz, *dup;
  int N, NB;
  int64_t total, first;  // blocks; the launch's first workgroup
};

template <bool F32, bool VEC, bool GATED, int ACT>
__global__ __launch_bounds__(kThreads) void f8_act_grad_kernel(ActGradArgs a) {
  const int64_t t = (a.first + blockIdx.x) * kGroups + threadIdx.x / kLanes;
  if (t >= a.total) return;
  const int64_t row = t / a.NB;
  const int n0 = (int)(t - row * a.NB) * kBlock + (int)(threadIdx.x % kLanes) * kPerLane;
  const int n = a.N - n0;
  const int64_t at = row * a.N + n0;
  float z[8], up[8], dy[8], dz[8], dup[8];
  load_codes8<VEC>(a.z, at, n, a.z_scale[t], z);
  if constexpr (GATED) load_codes8<VEC>(a.up, at, n, a.up_scale[t], up);
  load8<F32, VEC>(a.dy, at, n, dy);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float act, slope;
    act_and_slope<ACT, F32>(z[i], act, slope);
    dz[i] = (GATED ? dy[i] * up[i] : dy[i]) * slope;
    dup[i] = dy[i] * act;
  }
  store8<F32, VEC>(a.dz, at, n, dz);
  if constexpr (GATED) store8<F32, VEC>(a.dup, at, n, dup);
}

template <bool F32, bool VEC, bool GATED>
auto act_grad_kernel(int act) {
  switch (act) {
    case MX_ACT_GELU: return f8_act_grad_kernel<F32, VEC, GATED, MX_ACT_GELU>;
    case MX_ACT_RELU: return f8_act_grad_kernel<F32, VEC, GATED, MX_ACT_RELU>;
    case MX_ACT_SILU: return f8_act_grad_kernel<F32, VEC, GATED, MX_ACT_SILU>;
    case MX_ACT_HARDSWISH: return f8_act_grad_kernel<F32, VEC, GATED, MX_ACT_HARDSWISH>;
    case MX_ACT_TANH: return f8_act_grad_kernel<F32, VEC, GATED, MX_ACT_TANH>;
    default: return f8_act_grad_kernel<F32, VEC, GATED, MX_ACT_NONE>;
  }
}

bool aligned8(const void* p) { return ((uintptr_t)p & 7) == 0; }

}  // namespace

int f8_quantize_run(mx_backend* b, const F8QuantizeDesc& d) {
  if (d.M == 0 || d.K == 0) return MX_OK;
  const bool f32 = d.x_dt == MX_DTYPE_FLOAT32;
  const bool vec = d.K % kPerLane == 0 && aligned16(d.x) && aligned8(d.codes);
  const int64_t KB = blocks(d.K);
  if (d.rows == 1) {
    const int64_t total = d.M * KB, grid = (total + kGroups - 1) / kGroups;
    auto k = f32 ? (vec ? f8_quantize_rows_kernel<true, true> : f8_quantize_rows_kernel<true, false>)
                 : (vec ? f8_quantize_rows_kernel<false, true> : f8_quantize_rows_kernel<false, false>);
    return launch_runs(b, "f8_quantize_rows", grid, kThreads, [&](int64_t first, unsigned count) {
      dispatch(k, dim3(count), dim3(kThreads), 0, b->stream, d.x, d.codes, d.scale, (int)d.K, (int)KB, total, first);
    });
  }
  const int64_t grid = blocks(d.M) * KB;
  auto k = f32 ? (vec ? f8_quantize_tiles_kernel<true, true> : f8_quantize_tiles_kernel<true, false>)
               : (vec ? f8_quantize_tiles_kernel<false, true> : f8_quantize_tiles_kernel<false, false>);
  return launch_runs(b, "f8_quantize_tiles", grid, kThreads, [&](int64_t first, unsigned count) {
    dispatch(k, dim3(count), dim3(kThreads), 0, b->stream, d.x, d.codes, d.scale, (int)d.M, (int)d.K, (int)KB, (unsigned)first);
  });
}

int f8_act_grad_run(mx_backend* b, const F8ActGradDesc& d) {
  if (d.M == 0 || d.N == 0) return MX_OK;
  const bool f32 = d.dy_dt == MX_DTYPE_FLOAT32, gated = d.up != nullptr;
  const bool vec = d.N % kPerLane == 0 && aligned8(d.z) && aligned8(d.up) && aligned16(d.dy) && aligned16(d.dz) && aligned16(d.dup);
  const int64_t NB = blocks(d.N), total = d.M * NB, grid = (total + kGroups - 1) / kGroups;
  ActGradArgs a{d.z, d.up, d.z_scale, d.up_scale, d.dy, d.dz, d.dup, (int)d.N, (int)NB, total, 0};
  auto k = f32 ? (vec ? (gated ? act_grad_kernel<true, true, true>(d.act) : act_grad_kernel<true, true, false>(d.act))
                      : (gated ? act_grad_kernel<true, false, true>(d.act) : act_grad_kernel<true, false, false>(d.act)))
               : (vec ? (gated ? act_grad_kernel<false, true, true>(d.act) : act_grad_kernel<false, true, false>(d.act))
                      : (gated ? act_grad_kernel<false, false, true>(d.act) : act_grad_kernel<false, false, false>(d.act)));
  return launch_runs(b, gated ? "f8_act_grad_gated" : "f8_act_grad", grid, kThreads, [&](int64_t first, unsigned count) {
    a.first = first;
    dispatch(k, dim3(count), dim3(kThreads), 0, b->stream, a);
  });
}

}  // namespace mx
