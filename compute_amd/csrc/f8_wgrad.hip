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
  int out_dt, oi, vec_out;
  int tiles_n;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma_bf16(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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

// A workgroup computes W (k) x W (n) in WK x WN waves of 32 TK x 32 TN; tokens in steps of S.
template <int WK_, int WN_, int TK_, int TN_, int S_, int OCC>
struct Tile {
  static constexpr int WK = WK_, WN = WN_, TK = TK_, TN = TN_, S = S_, W = 32 * TK * WK, kThreads = 64 * WK * WN, kOccupancy = OCC;
  static_assert(W == 32 * TN * WN, "square tiles");
};
//
// Staging.  The codes and dy of a step travel through registers, requested a step ahead: 16 codes a chunk,
// scaled to bf16 (32 bytes of LDS), and 8 values of dy.  LDS keeps both as they lie in memory,
// [token][column], in two buffers; the operands, eight consecutive tokens of a column per lane, come out
// through the transposing read, four tokens at a time.  A row's 32-byte pieces are XOR-ed with
// 2 (token & 3), so that the 32 lanes of a half-wave, which read four rows of two neighbouring pieces,
// touch every bank once.
//
// Schedule.  A step is G groups of TK MFMAs, one operand of dy against the wave's TK operands of x.  An
// operand of dy is read kRing - 1 groups ahead of its use and the x operands of the next 16 tokens
// during the present ones.  The step's barrier stands before its last kRing - 1 groups, whose operands
// are then in registers: under them travel the first operands of the next step.  A chunk of the next step
// is staged, and that of the step after requested into its registers, in the groups before the barrier.
//
// Columns past K or N hold whatever lies there: they meet only results that are not stored.  Tokens past
// M are zeros in both operands (a step past the last is staged like any other and not used).  WHOLE: rows
// are whole chunks below 2^24 columns, read through buffer resources that end with the array, so that
// what lies past it reads as zero; otherwise a chunk may start anywhere and run into the next row, and the
// tokens and the array's end are looked at.
// A window on an array that moves a step at a time: what lies past the array's end reads as zero.
struct Window {
  const uint8_t* p;
  int64_t left;
  __device__ __forceinline__ void move(int64_t bytes) {
    p += bytes;
    left -= bytes;
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t resource() const {
    const uint32_t hi = (uint32_t)(left >> 32);
    const uint32_t n = (int32_t)hi < 0 ? 0u : hi ? 0xffffffffu : (uint32_t)left;
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)n, 0x00027000);
  }
};

template <class Tile, bool F32, bool OI, bool WHOLE>
__global__ __launch_bounds__(Tile::kThreads, Tile::kOccupancy) void f8_wgrad_kernel(WGradArgs a) {
  constexpr int TK = Tile::TK, TN = Tile::TN, S = Tile::S, kThreads = Tile::kThreads;
  constexpr int P = F32 ? 3 : 1, W = Tile::W;          // parts of dy, columns of a tile
  constexpr int kRow = 2 * W;                          // bytes of a row in LDS
  constexpr int kBuf = S * kRow;                       // one operand (part) of a step
  constexpr int kStep = (1 + P) * kBuf;                // LDS of a step
  constexpr int CX = S * W / 16 / kThreads;            // chunks of x a thread stages
  constexpr int CD = S * W / 8 / kThreads;             // chunks of dy
  constexpr int RX = kThreads / (W / 16), RD = kThreads / (W / 8);  // rows between a thread's chunks
  constexpr int kParts = S / 16, kPart = P * TN, G = kParts * kPart;
  constexpr int kRing = 4, kLast = kRing - 1;          // groups after the barrier
  constexpr int kPieces = 2 * CX + CD;                 // staged at a time: half a chunk of x or one of dy
  constexpr int kStageGroups = G - kLast < kPieces ? G - kLast : kPieces, kStageFrom = G - kLast - kStageGroups;
  static_assert(2 * CX == CD, "pieces alternate between x and dy");
  constexpr int kPerGroup = (kPieces + kStageGroups - 1) / kStageGroups;
  constexpr int H = F32 ? 2 : 1, E = F32 ? 4 : 2;      // loads of a dy chunk, bytes of a value
  static_assert(CX * 16 * kThreads == S * W && CD * 8 * kThreads == S * W, "whole chunks");
  static_assert(kParts % 2 == 0 && kPart >= TK, "the sets of x operands alternate, and one is read while the other is used");
  static_assert(G % kRing == 0, "the ring's slots are the same in every step");
  static_assert((kStep & (kStep - 1)) == 0, "the buffers alternate by an XOR");
  static_assert((TK & (TK - 1)) == 0 && (TN & (TN - 1)) == 0, "a wave's pieces start on a multiple of their number: an XOR picks one");
  extern __shared__ __align__(1024) uint8_t lds[];     // [2][1 + P][S][W] bf16
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, i = lane % 32, g = lane / 32;
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
  const int xrow = tid / (W / 16), xk = k0 + 16 * (tid % (W / 16));  // the thread's first chunk of a step
  const int drow = tid / (W / 8), dn = n0 + 8 * (tid % (W / 8));
  const int kb = min(xk / kBlock, a.KB - 1);

  u32x4 xr[CX], dr[CD][H];
  float sr[CX];
  // WHOLE: byte offsets of the thread's chunks within a step (below 64 rows of 2^26 bytes), and the
  // windows of the step requested next.
  uint32_t x_off[CX], s_off[CX], d_off[CD];
#pragma unroll
  for (int j = 0; j < CX; ++j) {
    x_off[j] = (uint32_t)(xrow + j * RX) * (uint32_t)a.K + (uint32_t)min(xk, a.K - 16);
    s_off[j] = 4 * ((uint32_t)(xrow + j * RX) * (uint32_t)a.KB + (uint32_t)kb);
  }
#pragma unroll
  for (int j = 0; j < CD; ++j) d_off[j] = E * ((uint32_t)(drow + j * RD) * (uint32_t)a.N + (uint32_t)min(dn, a.N - 8));
  Window xw{a.x, x_total}, sw{(const uint8_t*)a.x_scale, (int64_t)a.M * a.KB * 4}, dw{(const uint8_t*)a.dy, dy_total * E};
  auto advance = [&]() __attribute__((always_inline)) {
    xw.move((int64_t)S * a.K);
    sw.move((int64_t)S * a.KB * 4);
    dw.move((int64_t)S * a.N * E);
  };
  auto request = [&](int m0, int piece) __attribute__((always_inline)) {
    if (piece % 2 == 0) {
      const int j = piece / 4;
      if (piece % 4 == 0) return;  // the first half of a chunk: the second still stands in the registers
      if constexpr (WHOLE) {
        xr[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(xw.resource(), x_off[j], 0, 0));
        sr[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sw.resource(), s_off[j], 0, 0));
      } else {
        const int64_t row = min(m0 + xrow + j * RX, a.M - 1), at = row * a.K + min(xk, a.K - 1);
        xr[j] = load16(a.x + at, x_total - at);
        sr[j] = a.x_scale[row * a.KB + kb];
      }
    } else {
      const int j = piece / 2;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        if constexpr (WHOLE) {
          dr[j][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(dw.resource(), d_off[j], 16 * h, 0));
        } else {
          const int64_t at = (int64_t)min(m0 + drow + j * RD, a.M - 1) * a.N + min(dn, a.N - 1) + 4 * h;
          dr[j][h] = load16((const uint8_t*)a.dy + E * at, E * (dy_total - at));
        }
      }
    }
  };
  // Piece of the step from m0 into LDS at `step`.
  auto swizzled = [](int m, int piece) { return m * kRow + 32 * (piece ^ (2 * (m & 3))); };
  auto stage = [&](int m0, uint32_t step, int piece) __attribute__((always_inline)) {
    uint8_t* xb = lds + step;
    if (piece % 2 == 0) {
      const int j = piece / 4, half = piece / 2 % 2;
      if (!WHOLE && half == 0 && m0 + xrow + j * RX >= a.M) xr[j] = u32x4{0u, 0u, 0u, 0u};
      u32x4 o;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const f32x4 v = decode4(xr[j][2 * half + w]);
        const float s = sr[j];
        const f32x2 lo = {v[0] * s, v[1] * s}, hi = {v[2] * s, v[3] * s};
        o[2 * w] = __builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2));
        o[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2));
      }
      *(u32x4*)(xb + swizzled(xrow + j * RX, tid % (W / 16)) + 16 * half) = o;
    } else {
      const int j = piece / 2, c = tid % (W / 8);
#pragma unroll
      for (int h = 0; h < H; ++h)
        if (!WHOLE && m0 + drow + j * RD >= a.M) dr[j][h] = u32x4{0u, 0u, 0u, 0u};
      uint8_t* q = xb + kBuf + swizzled(drow + j * RD, c / 2) + 16 * (c % 2);
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

  // Operand reads: token 8 g + 4 h + (lane % 16) / 4 of 16, columns 32 t + 16 (i / 16) + 4 (lane % 4) ..
  const int wk = wave / Tile::WN, wn = wave % Tile::WN;
  const uint32_t base = lds_addr(lds);
  auto read_base = [&](int piece) { return base + (uint32_t)swizzled(8 * g + lane % 16 / 4, piece + i / 16) + 8 * (lane % 4); };
  const uint32_t xa = read_base(2 * wk * TK), da = read_base(2 * wn * TN) + kBuf;
  auto operand = [&](uint32_t at, int t, int off) __attribute__((always_inline)) {
    const uint32_t p = (at ^ (uint32_t)(64 * t)) + (uint32_t)off;
    const u32x2 lo = read_tr16(p), hi = read_tr16(p + 4 * kRow);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  u32x4 xo[2][TK], dv[kRing];
  auto read_x = [&](int set, int t, uint32_t step, int part) __attribute__((always_inline)) {
    xo[set][t] = operand(xa + step, t, part * 16 * kRow);
  };
  auto read_dy = [&](int q, uint32_t step) __attribute__((always_inline)) {  // of group q of a step
    dv[q % kRing] = operand(da + step, q % TN, (q / TN % P) * kBuf + q / (TN * P) * 16 * kRow);
  };

  f32x16 acc[TK][TN] = {};
  if (a.M > 0) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) request(0, p);
    if constexpr (WHOLE) advance();
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      stage(0, 0, p);
      request(S, p);
    }
    lds_barrier();
#pragma unroll
    for (int t = 0; t < TK; ++t) read_x(0, t, 0, 0);
#pragma unroll
    for (int q = 0; q < kLast; ++q) read_dy(q, 0);
    uint32_t cur = 0;
    for (int m0 = 0; m0 < a.M; m0 += S) {
      const uint32_t next = cur ^ kStep;
      if constexpr (WHOLE) advance();
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const int part = q / kPart, set = part % 2;
        if (q == G - kLast) lds_barrier();
        // Operands of later groups.
        if (q + kLast < G)
          read_dy(q + kLast, cur);
        else
          read_dy(q + kLast - G, next);
        if (part + 1 < kParts && q % kPart < TK) read_x(1 - set, q % kPart, cur, part + 1);
        constexpr int kTail = kLast < kPart ? kLast : kPart;  // groups of the last 16 tokens behind the barrier
        if (q >= G - kTail) {
          constexpr int per = (TK + kTail - 1) / kTail;
#pragma unroll
          for (int e = 0; e < per; ++e) {
            const int t = (q - (G - kTail)) * per + e;
            if (t < TK) read_x(0, t, next, 0);
          }
        }
        if (q >= kStageFrom && q < G - kLast) {
#pragma unroll
          for (int e = 0; e < kPerGroup; ++e) {
            const int p = (q - kStageFrom) * kPerGroup + e;
            if (p < kPieces) {
              stage(m0 + S, next, p);
              request(m0 + 2 * S, p);
            }
          }
        }
#pragma unroll
        for (int t = 0; t < TK; ++t) {
          if constexpr (OI)
            acc[t][q % TN] = mfma_bf16(xo[set][t], dv[q % kRing], acc[t][q % TN]);
          else
            acc[t][q % TN] = mfma_bf16(dv[q % kRing], xo[set][t], acc[t][q % TN]);
        }
        if constexpr (WHOLE) {
#pragma unroll
          for (int t = 0; t < TK; ++t) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
            __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);  // VALU
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      cur = next;
    }
  }

  // Result (t, n): of its 32 x 32 the lane holds column i and rows 8 q + 4 g .. + 3.  The operand whose
  // columns are contiguous in the output is the first, so that four results go out in one store.
#pragma unroll
  for (int t = 0; t < TK; ++t)
#pragma unroll
    for (int n = 0; n < TN; ++n) {
      const int kf = k0 + 32 * (wk * TK + t), nf = n0 + 32 * (wn * TN + n);
      const int row = (OI ? nf : kf) + i, rows = OI ? a.N : a.K, cols = OI ? a.K : a.N;
      if (row >= rows) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = (OI ? kf : nf) + 8 * q + 4 * g;
        const f32x4 v = {acc[t][n][4 * q], acc[t][n][4 * q + 1], acc[t][n][4 * q + 2], acc[t][n][4 * q + 3]};
        store4(a.out, (int64_t)row * cols + col, cols - col, a.vec_out, a.out_dt, v);
      }
    }
}

template <class Tile, bool F32>
int run_tiles(mx_backend* b, const char* name, WGradArgs a, bool whole) {
  constexpr int W = Tile::W, P = F32 ? 3 : 1, kLds = 2 * (1 + P) * Tile::S * W * 2;
  const int64_t tk = (a.K + W - 1) / W, tn = (a.N + W - 1) / W;
  if (tk * tn >= (int64_t)1 << 31) return set_error(MX_ERR_INVALID, "F8WeightGradient: more than 2^31 workgroups");
  a.tiles_n = (int)tn;
  auto k = a.oi ? (whole ? f8_wgrad_kernel<Tile, F32, true, true> : f8_wgrad_kernel<Tile, F32, true, false>)
                : (whole ? f8_wgrad_kernel<Tile, F32, false, true> : f8_wgrad_kernel<Tile, F32, false, false>);
  MX_CHECK_HIP(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
  return launch(b, name, [&] { dispatch(k, dim3((unsigned)(tk * tn)), dim3(Tile::kThreads), kLds, b->stream, a); });
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
  const WGradArgs a{d.x, d.x_scale, d.dy, d.out, (int)d.M, (int)d.K, (int)d.N, (int)blocks(d.K), d.out_dt, d.oi,
                    (d.oi ? d.K : d.N) % 4 == 0 && ((uintptr_t)d.out & (d.out_dt == MX_DTYPE_FLOAT32 ? 15 : 7)) == 0, 0};
  const bool whole = d.K % 16 == 0 && d.N % 8 == 0 && d.K <= 1 << 24 && d.N <= 1 << 24 && aligned16(d.x) && aligned16(d.dy);
  const char* name = f8_wgrad_name(d);
  switch (plan_of(d)) {
    case Plan::kF32: return run_tiles<Tile<2, 2, 2, 2, 32, 2>, true>(b, name, a, whole);
    case Plan::kBf16: return run_tiles<Tile<2, 2, 2, 2, 64, 2>, false>(b, name, a, whole);
    default: return run_tiles<Tile<4, 2, 2, 4, 64, 2>, false>(b, name, a, whole);
  }
}

}  // namespace mx
