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

// A workgroup of four waves computes 32 T (k) x 32 T (n), a wave 16 T x 16 T of it; tokens in steps of S.
//
// Per step the codes and dy travel through registers, requested one step ahead: 16 codes a chunk, scaled
// to bf16 (32 bytes of LDS), and 8 values of dy.  LDS keeps both as they lie in memory, [token][column],
// in two buffers; the operands, eight consecutive tokens of a column per lane, come out through the
// transposing read, four tokens at a time.  A row's 32-byte pieces are XOR-ed with (token & 3) | (token
// >> 3 & 1) << 2, so that the 32 lanes of a half-wave, which read 8 rows of one piece, touch every bank
// once.
//
// Columns past K or N hold whatever lies there: they meet only results that are not stored.  Tokens past
// M are zeros in both operands.  WHOLE: rows are whole chunks; otherwise a chunk may start anywhere and
// run into the next row, and only the array's own end is looked at.
template <int T, int S, bool F32, bool OI, bool WHOLE>
__global__ __launch_bounds__(256, 1) void f8_wgrad_kernel(WGradArgs a) {
  constexpr int P = F32 ? 3 : 1, W = 32 * T;           // parts of dy, columns of a tile
  constexpr int kRow = 2 * W;                          // bytes of a row in LDS
  constexpr int kBuf = S * kRow;                       // one operand (part) of a step
  constexpr int CX = S * W / 16 / 256;                 // chunks of x a thread stages
  constexpr int CD = S * W / 8 / 256;                  // chunks of dy
  static_assert(CX * 16 * 256 == S * W && CD * 8 * 256 == S * W, "whole chunks");
  extern __shared__ __align__(1024) uint8_t lds[];     // [2][1 + P][S][W] bf16
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, i = lane % 16, g = lane / 16;
  const int tiles_k = (a.K + W - 1) / W;
  int kt, nt;
  {
    // Runs of 4 tiles of k by all tiles of n: a run's workgroups share their rows of x and dy in an L2.
    const int t = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int per = 4 * a.tiles_n, q = t / per, rows = min(4, tiles_k - 4 * q), in = t - q * per;
    kt = 4 * q + in % rows;
    nt = in / rows;
  }
  const int k0 = kt * W, n0 = nt * W;
  const int64_t x_total = (int64_t)a.M * a.K, dy_total = (int64_t)a.M * a.N;

  u32x4 xr[CX], dr[CD][F32 ? 2 : 1];
  float sr[CX];
  auto request = [&](int m0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < CX; ++j) {
      const int c = tid + 256 * j, m = m0 + c / (W / 16), k = k0 + 16 * (c % (W / 16));
      const int mc = min(m, a.M - 1);
      const int64_t row = (int64_t)mc * a.K;
      if constexpr (WHOLE) {
        xr[j] = *(const u32x4*)(a.x + row + min(k, a.K - 16));
      } else {
        const int64_t at = row + min(k, a.K - 1);
        xr[j] = load16(a.x + at, x_total - at);
      }
      sr[j] = a.x_scale[(int64_t)mc * a.KB + min(k / kBlock, a.KB - 1)];
      if (m >= a.M) xr[j] = u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int j = 0; j < CD; ++j) {
      const int c = tid + 256 * j, m = m0 + c / (W / 8), n = n0 + 8 * (c % (W / 8));
      const int64_t row = (int64_t)min(m, a.M - 1) * a.N;
      constexpr int E = F32 ? 4 : 2;
      const uint8_t* p = (const uint8_t*)a.dy;
#pragma unroll
      for (int h = 0; h < (F32 ? 2 : 1); ++h) {
        if constexpr (WHOLE) {
          dr[j][h] = *(const u32x4*)(p + E * (row + min(n, a.N - 8)) + 16 * h);
        } else {
          const int64_t at = row + min(n, a.N - 1) + 4 * h;
          dr[j][h] = load16(p + E * at, E * (dy_total - at));
        }
        if (m >= a.M) dr[j][h] = u32x4{0u, 0u, 0u, 0u};
      }
    }
  };
  auto swizzled = [](int m, int piece) { return m * kRow + 32 * (piece ^ ((m & 3) | (m >> 3 & 1) << 2)); };
  auto stage = [&](int buf) __attribute__((always_inline)) {
    uint8_t* xb = lds + buf * (1 + P) * kBuf;
#pragma unroll
    for (int j = 0; j < CX; ++j) {
      const int c = tid + 256 * j;
      u32x4 o[2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const f32x4 v = decode4(xr[j][w]);
        const f32x2 lo = {v[0] * sr[j], v[1] * sr[j]}, hi = {v[2] * sr[j], v[3] * sr[j]};
        o[w / 2][2 * (w % 2)] = __builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2));
        o[w / 2][2 * (w % 2) + 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2));
      }
      uint8_t* q = xb + swizzled(c / (W / 16), c % (W / 16));
      *(u32x4*)q = o[0];
      *(u32x4*)(q + 16) = o[1];
    }
#pragma unroll
    for (int j = 0; j < CD; ++j) {
      const int c = tid + 256 * j, piece = c % (W / 8);
      uint8_t* q = xb + kBuf + swizzled(c / (W / 8), piece / 2) + 16 * (piece % 2);
      if constexpr (F32) {
        uint16_t p[8][3];
#pragma unroll
        for (int e = 0; e < 8; ++e) parts_of(__uint_as_float(dr[j][e / 4][e % 4]), p[e]);
#pragma unroll
        for (int t = 0; t < 3; ++t) {
          u32x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (uint32_t)p[2 * e][t] | (uint32_t)p[2 * e + 1][t] << 16;
          *(u32x4*)(q + t * kBuf) = o;
        }
      } else {
        *(u32x4*)q = dr[j][0];
      }
    }
  };

  // Operand reads: token 8 g + 4 h + i / 4 of a half step, columns 16 t + 4 (i % 4) ..
  const int wk = wave / 2, wn = wave % 2;
  const uint32_t base = lds_addr(lds);
  auto read_base = [&](int w) { return base + (uint32_t)swizzled(8 * g + i / 4, w * T) + 8 * (i % 4); };
  const uint32_t xa = read_base(wk), da = read_base(wn) + kBuf;
  auto operand = [&](uint32_t at, int t, int off) __attribute__((always_inline)) {
    const uint32_t p = (at ^ (uint32_t)(32 * t)) + (uint32_t)off;
    const u32x2 lo = read_tr16(p), hi = read_tr16(p + 4 * kRow);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  static_assert(T == 4 || T == 8, "a wave's pieces start on a multiple of its own T, so an XOR with t < T picks one");

  f32x4 acc[T][T] = {};
  auto multiply = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < S / 32; ++h) {
      const int off = buf * (1 + P) * kBuf + h * 32 * kRow;
      u32x4 xo[T], dv;
#pragma unroll
      for (int t = 0; t < T; ++t) xo[t] = operand(xa, t, off);
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int n = 0; n < T; ++n) {
          dv = operand(da, n, off + p * kBuf);
#pragma unroll
          for (int t = 0; t < T; ++t) {
            if constexpr (OI)
              acc[t][n] = mfma_bf16(dv, xo[t], acc[t][n]);
            else
              acc[t][n] = mfma_bf16(xo[t], dv, acc[t][n]);
          }
        }
    }
  };

  const int steps = (a.M + S - 1) / S;
  if (steps > 0) {
    request(0);
    stage(0);
    lds_barrier();
    for (int s = 0; s < steps; s += 2) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (s + b < steps) {
          const bool more = s + b + 1 < steps;
          if (more) request((s + b + 1) * S);
          multiply(b);
          if (more) stage(1 - b);
          lds_barrier();
        }
      }
    }
  }

  // Result (t, n): rows 4 g + r and column i of its 16 x 16; OI: rows are columns of dy.
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int n = 0; n < T; ++n) {
      const int k = k0 + 16 * (wk * T + t) + (OI ? i : 4 * g), c = n0 + 16 * (wn * T + n) + (OI ? 4 * g : i);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kk = k + (OI ? 0 : r), cc = c + (OI ? r : 0);
        if (kk < a.K && cc < a.N) store_f(a.out, OI ? (int64_t)cc * a.K + kk : (int64_t)kk * a.N + cc, a.out_dt, acc[t][n][r]);
      }
    }
}

template <int T, int S, bool F32>
int run_tiles(mx_backend* b, const char* name, WGradArgs a, bool whole) {
  constexpr int W = 32 * T, P = F32 ? 3 : 1, kLds = 2 * (1 + P) * S * W * 2;
  const int64_t tk = (a.K + W - 1) / W, tn = (a.N + W - 1) / W;
  if (tk * tn >= (int64_t)1 << 31) return set_error(MX_ERR_INVALID, "F8WeightGradient: more than 2^31 workgroups");
  a.tiles_n = (int)tn;
  auto k = a.oi ? (whole ? f8_wgrad_kernel<T, S, F32, true, true> : f8_wgrad_kernel<T, S, F32, true, false>)
                : (whole ? f8_wgrad_kernel<T, S, F32, false, true> : f8_wgrad_kernel<T, S, F32, false, false>);
  MX_CHECK_HIP(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
  return launch(b, name, [&] { dispatch(k, dim3((unsigned)(tk * tn)), dim3(256), kLds, b->stream, a); });
}

enum class Plan { kF32, kBf16, kBf16Large };

Plan plan_of(const F8WGradDesc& d) {
  if (d.dy_dt == MX_DTYPE_FLOAT32) return Plan::kF32;
  const int64_t tiles = ((d.K + 255) / 256) * ((d.N + 255) / 256);
  return tiles >= 192 ? Plan::kBf16Large : Plan::kBf16;
}

}  // namespace

const char* f8_wgrad_name(const F8WGradDesc& d) {
  switch (plan_of(d)) {
    case Plan::kF32: return "f8_wgrad_f32_128";
    case Plan::kBf16: return "f8_wgrad_bf16_128";
    default: return "f8_wgrad_bf16_256";
  }
}

int f8_wgrad_run(mx_backend* b, const F8WGradDesc& d) {
  if (d.K == 0 || d.N == 0) return MX_OK;
  const WGradArgs a{d.x, d.x_scale, d.dy, d.out, (int)d.M, (int)d.K, (int)d.N, (int)blocks(d.K), d.out_dt, d.oi, 0};
  const bool whole = d.K % 16 == 0 && d.N % 8 == 0 && aligned16(d.x) && aligned16(d.dy);
  const char* name = f8_wgrad_name(d);
  switch (plan_of(d)) {
    case Plan::kF32: return run_tiles<4, 32, true>(b, name, a, whole);
    case Plan::kBf16: return run_tiles<4, 64, false>(b, name, a, whole);
    default: return run_tiles<8, 64, false>(b, name, a, whole);
  }
}

}  // namespace mx
