// Dense product over 8-bit floating-point blocks:
//   y[m, n] = act(sum_b sx[m, b] * sw[b, n / 128] * (sum_{k in block b} x[m, k] * w[k, n]) + bias[n]).
//
// A block of 128 codes is one v_mfma_f32_16x16x128_f8f6f4, whose sum starts from zero and enters the
// float32 total with the block's two scales: acc += t * (sx * sw).
//
// Precision.  The matrix cores add the products of 8-bit operands in groups of eight, aligned to the
// group's largest and cut off 13 bits below it (measured with single products, for every 8-bit form
// of the instruction); groups are added in float32.  On random codes of mixed exponents a sum of 128
// is 4.4e-5 off in norm.  That is 1/38 of the rounding of a bfloat16 result, which therefore takes
// these instructions at 4.4 PFLOP/s.  A float32 result (WIDE) takes the codes as bfloat16 values, which
// are exact, through v_mfma_f32_16x16x32_bf16, whose sums are good to 2^-23 of their terms, at half the
// rate.
//
// Operand layout.  Lane (i = lane % 16, g = lane / 16) of the instruction holds 32 consecutive codes of
// row (or column) i, those from 32 g; the sum does not depend on which k a position stands for as
// long as both operands agree.  WIDE: four instructions, each over eight of a lane's 32 codes.  The
// result: column i, rows 4 g .. 4 g + 3.
#include <algorithm>

#include "f8_dense.h"

namespace mx {
namespace {
using namespace f8;

// Any sizes, alignment and layout: 64 x 64 tiles, both operands staged in LDS as rows of 128 codes.
constexpr int kAnyTile = 64, kAnyThreads = 256, kAnyPitch = kBlock + 16;

template <bool WIDE>
__global__ __launch_bounds__(kAnyThreads) void f8_dense_any_kernel(DenseArgs a) {
  __shared__ __align__(16) uint8_t xs[kAnyTile * kAnyPitch], ws[kAnyTile * kAnyPitch];
  const int m0 = (int)(blockIdx.x / (unsigned)a.tiles_n) * kAnyTile, n0 = (int)(blockIdx.x % (unsigned)a.tiles_n) * kAnyTile;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, i = lane % 16, g = lane / 16;
  f32x4 acc[4] = {};
  for (int kb = 0; kb < a.KB; ++kb) {
    const int k0 = kb * kBlock;
    __syncthreads();
    for (int c = threadIdx.x; c < kAnyTile * 8; c += kAnyThreads) {
      const int r = c / 8, k = k0 + 16 * (c % 8);
      const bool in = m0 + r < a.M;
      *(u32x4*)(xs + r * kAnyPitch + 16 * (c % 8)) = load16(a.x + (in ? (int64_t)(m0 + r) * a.K + k : 0), in ? a.K - k : 0);
    }
    if (a.oi) {
      for (int c = threadIdx.x; c < kAnyTile * 8; c += kAnyThreads) {
        const int r = c / 8, k = k0 + 16 * (c % 8);
        const bool in = n0 + r < a.N;
        *(u32x4*)(ws + r * kAnyPitch + 16 * (c % 8)) = load16(a.w + (in ? (int64_t)(n0 + r) * a.K + k : 0), in ? a.K - k : 0);
      }
    } else {
      for (int c = threadIdx.x; c < kBlock * 4; c += kAnyThreads) {
        const int r = c / 4, n = n0 + 16 * (c % 4);
        const bool in = k0 + r < a.K;
        const u32x4 v = load16(a.w + (in ? (int64_t)(k0 + r) * a.N + n : 0), in ? a.N - n : 0);
#pragma unroll
        for (int j = 0; j < 16; ++j) ws[(16 * (c % 4) + j) * kAnyPitch + r] = (uint8_t)(v[j / 4] >> (8 * (j % 4)));
      }
    }
    __syncthreads();
    float sx[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + 16 * wave + 4 * g + r;
      sx[r] = m < a.M ? a.x_scale[(int64_t)m * a.KB + kb] : 0.0f;
    }
    const float sw = a.oi ? a.w_scale[(int64_t)(n0 / kBlock) * a.KB + kb] : a.w_scale[(int64_t)kb * a.NB + n0 / kBlock];
    const i32x8 xa = read32(xs + (16 * wave + i) * kAnyPitch + 32 * g);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const i32x8 wb = read32(ws + (16 * c + i) * kAnyPitch + 32 * g);
      const f32x4 t = block_sum<WIDE>(xa, wb);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[c][r] = fmaf(t[r], sx[r] * sw, acc[c][r]);
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int n = n0 + 16 * c + i;
    if (n >= a.N) continue;
    const float bias = a.bias ? load_f(a.bias, n, a.b_dt) : 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + 16 * wave + 4 * g + r;
      if (m < a.M) store_f(a.out, (int64_t)m * a.N + n, a.out_dt, act_fast(acc[c][r] + bias, a.act));
    }
  }
}

// -------------------------------------------------------------------------------------------------
// Tiles for bfloat16 results.  A workgroup of WN x WM waves computes 64 WN columns (n) x 16 TB WM rows (m), a wave
// 64 x 16 TB of it, one block of 128 k a step.
//
// Roles.  w is the first operand, so that a lane's four results of a tile are four columns of one row: the scale
// of a tile is then one value a lane, sx of its row times the wave's sw.
//
// Staging.  Codes and scales move from memory straight into LDS (buffer_load ... lds, 16 or 4 bytes a lane), a step
// ahead, into two buffers.  The resources end with their arrays, and past the end LDS gets zeros: rows past M or N and,
// for w [K, N], rows past K need nothing more.  The last block's chunks past K are sent past the end by their offset.
//   x, and w [N, K] (OI): rows of 128 bytes.  A lane reads its 32 codes as two 16-byte chunks; chunk c of row r lies at
//     c ^ (r >> 1 & 7) for x, whose operands are 16 consecutive rows, and at c ^ ((r >> 1 & 1) | (r >> 4 & 3) << 1) for
//     w: operand a of a wave is the rows 16 (i / 4) + 4 a + i % 4 of its 64, which leaves a lane with 16 consecutive
//     columns over its four operands.  Either way 16 lanes meet every bank once.
//   w [K, N] (!OI): 128 rows of k, 64 WN columns, read through the transposing read, eight k at a time; 16-byte chunk c
//     of row k lies at c ^ (2 (k & 7) | (k >> 5 & 1)).
//
// Schedule.  A step is TB groups of four MFMAs, one operand of x against the wave's four of w.  An operand of x is
// read kRing - 1 groups ahead; a group's sums enter the total during the next group.  The step's barrier stands before
// its last kRing - 1 groups, whose operands are in registers: behind it the step after the next is requested into the
// buffer just left, and w's operands are read again as the last group leaves them.
struct Resource {
  i32x4 d;
};
__device__ __forceinline__ Resource make_resource(const void* p, int64_t bytes) {
  constexpr int64_t kMost = 0x7fffffff;  // offsets from 2^31 on are past the end
  const uint64_t at = (uint64_t)(uintptr_t)p;
  return Resource{i32x4{(int)(uint32_t)at, (int)((uint32_t)(at >> 32) & 0xffffu), (int)(bytes < 0 ? 0 : bytes < kMost ? bytes : kMost), 0x00027000}};
}
constexpr uint32_t kPastEnd = 0x80000000u;

// 16 (or 4) bytes a lane from offset voff of a resource, lane l's to LDS address `to` + 16 l (4 l); past the
// resource's end zeros.  Issued as assembly: the compiler neither waits for it nor knows that it writes LDS, so the
// kernel waits itself (wait_loads) before the barrier that publishes a step, and before it ends.
__device__ __forceinline__ void lds_load16(const Resource& r, uint32_t voff, uint32_t to) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(voff), "s"(to), "s"(r.d)
      : "memory");
}
__device__ __forceinline__ void lds_load4(const Resource& r, uint32_t voff, uint32_t to) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %1, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(voff), "s"(to), "s"(r.d)
      : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) const float lds_float;
__device__ __forceinline__ u32x4 lds_read16(uint32_t at) { return *(lds_u32x4*)at; }
__device__ __forceinline__ float lds_read_float(uint32_t at) { return *(lds_float*)at; }

template <int WN_, int WM_, int TB_>
struct DenseTile {
  static constexpr int WN = WN_, WM = WM_, TB = TB_, kWaves = WN * WM, kThreads = 64 * kWaves;
  static constexpr int kCols = 64 * WN, kRows = 16 * TB * WM;
  static constexpr int kXBytes = kRows * kBlock, kWBytes = kCols * kBlock, kScaleBytes = 4 * kRows + 256;
  static constexpr int kX = 0, kW = 2 * kXBytes, kScale = kW + 2 * kWBytes, kLds = kScale + 2 * kScaleBytes;
  static_assert(kXBytes % (1024 * kWaves) == 0 && kWBytes % (1024 * kWaves) == 0, "whole loads");
  static_assert(kRows % 64 == 0 && kRows / 64 < kWaves, "a wave a load of row scales, and one of the weight's");
};

template <int ACT, bool OI, int TB>
__device__ __forceinline__ void store_results(const DenseArgs& a, const f32x4 (&acc)[4][TB], int m0, int n0) {
  const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
  float bias[4][4];
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + (OI ? 16 * g + 4 * c : 16 * c + 4 * g) + r;
      bias[c][r] = a.bias && n < a.N ? load_f(a.bias, n, a.b_dt) : 0.0f;
    }
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    const int m = m0 + 16 * b + i;
    if (m >= a.M) continue;
    u32x2 o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = act_fast(acc[c][b][r] + bias[c][r], ACT);
      const f32x2 lo = {v[0], v[1]}, hi = {v[2], v[3]};
      o[c] = u32x2{__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2)),
                   __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2))};
    }
    uint16_t* row = (uint16_t*)a.out + (int64_t)m * a.N;
    if (OI && a.vec_out) {  // rows on 16 bytes, N a multiple of 8
      const int n = n0 + 16 * g;
      if (n < a.N) *(u32x4*)(row + n) = u32x4{o[0][0], o[0][1], o[1][0], o[1][1]};
      if (n + 8 < a.N) *(u32x4*)(row + n + 8) = u32x4{o[2][0], o[2][1], o[3][0], o[3][1]};
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = n0 + (OI ? 16 * g + 4 * c : 16 * c + 4 * g);
        if (a.vec_out) {
          if (n < a.N) *(u32x2*)(row + n) = o[c];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < a.N) row[n + r] = (uint16_t)(o[c][r / 2] >> (16 * (r % 2)));
        }
      }
    }
  }
}

template <class Tile, bool OI>
__global__ __launch_bounds__(Tile::kThreads, 2) void f8_dense_tiles_kernel(DenseArgs a) {
  constexpr int TB = Tile::TB, kWaves = Tile::kWaves;
  constexpr int kRing = 2, kLast = kRing - 1;
  constexpr int XL = Tile::kXBytes / (1024 * kWaves), WL = Tile::kWBytes / (1024 * kWaves);  // loads a wave a step
  static_assert(TB % kRing == 0, "the ring's slots are the same in every step");
  extern __shared__ __align__(1024) uint8_t lds[];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = lane % 16, g = lane / 16;
  const uint32_t base = lds_addr(lds);
  int mt, nt;
  {
    // Runs of 4 tiles of n by all tiles of m: a run's workgroups share their rows of x and w in an L2.
    const int tiles_m = (int)gridDim.x / a.tiles_n;
    const int t = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int per = 4 * tiles_m, q = t / per, cols = min(4, a.tiles_n - 4 * q), in = t - q * per;
    nt = 4 * q + in % cols;
    mt = in / cols;
  }
  const int m0 = mt * Tile::kRows, n0 = nt * Tile::kCols;

  // Loads: the wave's lanes' offsets within a step, and what moves with it.
  uint32_t x_off[XL], w_off[WL];
  const int x_chunk = (lane % 8) ^ ((wave & 1) * 4 + lane / 16);               // (row >> 1) & 7
  const int w_chunk = (lane % 8) ^ ((lane / 16 & 1) | (wave / 2 & 3) << 1);    // OI
#pragma unroll
  for (int j = 0; j < XL; ++j) x_off[j] = (uint32_t)(8 * (wave + kWaves * j) + lane / 8) * (uint32_t)a.K + 16 * x_chunk;
  constexpr int kLanesRow = Tile::kCols / 16;  // !OI: lanes of a row of k
#pragma unroll
  for (int j = 0; j < WL; ++j) {
    if constexpr (OI) {
      w_off[j] = (uint32_t)(8 * (wave + kWaves * j) + lane / 8) * (uint32_t)a.K + 16 * w_chunk;
    } else {
      const int k = (64 / kLanesRow) * (wave + kWaves * j) + lane / kLanesRow;
      w_off[j] = (uint32_t)k * (uint32_t)a.N + 16 * ((lane % kLanesRow) ^ (((2 * (k & 7)) | (k >> 5 & 1)) % kLanesRow));
    }
  }
  const uint8_t* xp = a.x + (int64_t)m0 * a.K;
  const int64_t x_left = (int64_t)(a.M - m0) * a.K;
  const uint8_t* wp = OI ? a.w + (int64_t)n0 * a.K : a.w + n0;
  const int64_t w_left = OI ? (int64_t)(a.N - n0) * a.K : (int64_t)a.K * a.N - n0;
  // Waves below kRows / 64 load 64 row scales each, the others (all the same) the weight's of the tile's columns.
  const bool row_scales = wave < Tile::kRows / 64;
  const uint8_t* sp = (const uint8_t*)(row_scales ? a.x_scale + (int64_t)(m0 + 64 * wave) * a.KB : a.w_scale);
  const int64_t s_left = 4 * (row_scales ? (int64_t)(a.M - m0 - 64 * wave) * a.KB : (int64_t)a.KB * a.NB);
  const uint32_t nb = (uint32_t)min(n0 / kBlock + lane % ((Tile::kCols + kBlock - 1) / kBlock), a.NB - 1);
  const uint32_t s_off = 4 * (row_scales ? (uint32_t)lane * (uint32_t)a.KB : OI ? nb * (uint32_t)a.KB : nb);
  const uint32_t s_step = row_scales || OI ? 4 : 4 * (uint32_t)a.NB;
  const uint32_t s_to = base + Tile::kScale + (row_scales ? 256 * wave : 4 * Tile::kRows);
  // The last block's chunks past K are sent past the end.  (A block past the last is requested like any other, from
  // wherever it lies, and not used.)
  const int last = a.K - (a.KB - 1) * kBlock;
  const uint32_t x_tail = 16 * x_chunk >= last ? kPastEnd : 0u, w_tail = OI && 16 * w_chunk >= last ? kPastEnd : 0u;
  auto request = [&](int kb, uint32_t buf) __attribute__((always_inline)) {
    const Resource xr = make_resource(xp + (int64_t)kb * kBlock, x_left - (int64_t)kb * kBlock);
    const Resource sr = make_resource(sp + (int64_t)kb * s_step, s_left - (int64_t)kb * s_step);
    const uint32_t xt = kb == a.KB - 1 ? x_tail : 0u, wt = kb == a.KB - 1 ? w_tail : 0u;
#pragma unroll
    for (int j = 0; j < XL; ++j)
      lds_load16(xr, x_off[j] | xt, base + Tile::kX + buf * Tile::kXBytes + 1024 * (wave + kWaves * j));
    const int64_t moved = (int64_t)kb * kBlock * (OI ? 1 : a.N);
    const Resource wr = make_resource(wp + moved, w_left - moved);
#pragma unroll
    for (int j = 0; j < WL; ++j)
      lds_load16(wr, w_off[j] | wt, base + Tile::kW + buf * Tile::kWBytes + 1024 * (wave + kWaves * j));
    lds_load4(sr, s_off, s_to + buf * Tile::kScaleBytes);
  };

  // Operand reads.
  const int wn = wave / Tile::WM, wm = wave % Tile::WM;
  const int x_row = 16 * TB * wm + i, x_first = (2 * g) ^ (i >> 1 & 7);
  const uint32_t xa = base + Tile::kX + x_row * kBlock + 16 * x_first;
  uint32_t wa;
  if constexpr (OI) {
    const int r = 64 * wn + 16 * (i / 4) + i % 4, first = (2 * g) ^ ((i % 4) / 2 | (i / 4) << 1);
    wa = base + Tile::kW + r * kBlock + 16 * first;
  } else {
    const int k = 32 * g + i / 2;
    wa = base + Tile::kW + k * Tile::kCols + 16 * ((4 * wn) ^ ((2 * (k & 7) | (k >> 5 & 1)) % kLanesRow)) + 8 * (i % 2);
  }
  const uint32_t sxa = base + Tile::kScale + 4 * x_row, swa = base + Tile::kScale + 4 * Tile::kRows + 4 * (64 * wn / kBlock);
  i32x8 wo[4], xo[kRing];
  float sx[kRing];
  auto read_w = [&](int c, uint32_t buf) __attribute__((always_inline)) {
    const uint32_t at = wa + buf * Tile::kWBytes;
    if constexpr (OI) {
      wo[c] = join(lds_read16(at + 4 * kBlock * c), lds_read16((at ^ 16) + 4 * kBlock * c));
    } else {
      const uint32_t p = at ^ (uint32_t)(16 * c);
      const u32x2 k0 = read_tr8(p), k1 = read_tr8(p + 8 * Tile::kCols), k2 = read_tr8(p + 16 * Tile::kCols), k3 = read_tr8(p + 24 * Tile::kCols);
      wo[c] = i32x8{(int)k0[0], (int)k0[1], (int)k1[0], (int)k1[1], (int)k2[0], (int)k2[1], (int)k3[0], (int)k3[1]};
    }
  };
  auto read_x = [&](int b, uint32_t buf) __attribute__((always_inline)) {
    const uint32_t at = xa + buf * Tile::kXBytes;
    xo[b % kRing] = join(lds_read16(at + 16 * kBlock * b), lds_read16((at ^ 16) + 16 * kBlock * b));
    sx[b % kRing] = lds_read_float(sxa + buf * Tile::kScaleBytes + 64 * b);
  };

  f32x4 acc[4][TB] = {}, t[2][4] = {};
  float st[2] = {};
  if (a.KB > 0) {
    request(0, 0);
    wait_loads();
    lds_barrier();
    request(1, 1);
    float sw = lds_read_float(swa);
#pragma unroll
    for (int c = 0; c < 4; ++c) read_w(c, 0);
#pragma unroll
    for (int b = 0; b < kLast; ++b) read_x(b, 0);
    uint32_t cur = 0;
    for (int kb = 0; kb < a.KB; ++kb) {
      const uint32_t next = cur ^ 1;
      float sw_next = 0.0f;
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        if (b == TB - kLast) {
          wait_loads();
          lds_barrier();
          request(kb + 2, cur);
          sw_next = lds_read_float(swa + next * Tile::kScaleBytes);
        }
        if (b + kLast < TB)
          read_x(b + kLast, cur);
        else
          read_x(b + kLast - TB, next);
        st[b % 2] = sx[b % kRing] * sw;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          t[b % 2][c] = mfma_f8(wo[c], xo[b % kRing], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
          if (b == TB - 1) read_w(c, next);
        }
        constexpr int kBefore = TB - 1;
        const int p = b == 0 ? kBefore : b - 1;  // the group before (of the step before: t starts as zeros)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[c][p][r] = fmaf(t[1 - b % 2][c][r], st[1 - b % 2], acc[c][p][r]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS read
          __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // VALU
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      sw = sw_next;
      cur = next;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[c][TB - 1][r] = fmaf(t[1][c][r], st[1], acc[c][TB - 1][r]);
    wait_loads();  // of the block past the last: LDS is the next workgroup's when this one ends
  }
  static_assert(TB % 2 == 0, "the last group's sums lie in t[1]");
  const int mw = m0 + 16 * TB * wm, nw = n0 + 64 * wn;
  switch (a.act) {
    case MX_ACT_GELU: store_results<MX_ACT_GELU, OI, TB>(a, acc, mw, nw); break;
    case MX_ACT_RELU: store_results<MX_ACT_RELU, OI, TB>(a, acc, mw, nw); break;
    case MX_ACT_SILU: store_results<MX_ACT_SILU, OI, TB>(a, acc, mw, nw); break;
    case MX_ACT_HARDSWISH: store_results<MX_ACT_HARDSWISH, OI, TB>(a, acc, mw, nw); break;
    case MX_ACT_TANH: store_results<MX_ACT_TANH, OI, TB>(a, acc, mw, nw); break;
    default: store_results<MX_ACT_NONE, OI, TB>(a, acc, mw, nw); break;
  }
}

template <class Tile>
int run_dense_tiles(mx_backend* b, const char* name, DenseArgs a) {
  const int64_t tm = ((int64_t)a.M + Tile::kRows - 1) / Tile::kRows, tn = ((int64_t)a.N + Tile::kCols - 1) / Tile::kCols;
  if (tm * tn >= (int64_t)1 << 31) return set_error(MX_ERR_INVALID, "F8Dense: more than 2^31 workgroups");
  a.tiles_n = (int)tn;
  auto k = a.oi ? f8_dense_tiles_kernel<Tile, true> : f8_dense_tiles_kernel<Tile, false>;
  MX_CHECK_HIP(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, Tile::kLds));
  return launch(b, name, [&] { dispatch(k, dim3((unsigned)(tm * tn)), dim3(Tile::kThreads), Tile::kLds, b->stream, a); });
}

using Tile256 = DenseTile<4, 2, 8>;  // 256 x 256
using Tile128 = DenseTile<4, 2, 4>;  // 256 columns x 128 rows

enum class DensePlan { kAny, kSkinny, kTiles256, kTiles128 };

DensePlan dense_plan(const F8DenseDesc& d) {
  if (skinny_fits(d)) return DensePlan::kSkinny;
  // The direct loads take whole aligned 16-byte chunks of rows and 32-bit offsets.
  const bool chunks = d.K % 16 == 0 && (d.oi || d.N % 16 == 0) && aligned16(d.x) && aligned16(d.w) && d.K <= 1 << 21 && d.N <= 1 << 21;
  if (!chunks || d.out_dt != MX_DTYPE_BFLOAT16 || d.K == 0) return DensePlan::kAny;
  const int64_t t256 = ((d.M + 255) / 256) * ((d.N + 255) / 256);
  return t256 >= 192 ? DensePlan::kTiles256 : DensePlan::kTiles128;
}

}  // namespace

const char* f8_product_name(const F8DenseDesc& d) {
  switch (dense_plan(d)) {
    case DensePlan::kSkinny: return "f8_dense_skinny";
    case DensePlan::kTiles256: return "f8_dense_tiles_256";
    case DensePlan::kTiles128: return "f8_dense_tiles_128";
    default: return "f8_dense_any";
  }
}

bool f8_product_takes_float(const F8DenseDesc& d) { return skinny_fits(d); }

int f8_product_run(mx_backend* b, const F8DenseDesc& d) {
  if (d.M == 0 || d.N == 0) return MX_OK;
  DenseArgs a = dense_args(d);
  const char* name = f8_product_name(d);
  switch (dense_plan(d)) {
    case DensePlan::kSkinny: return skinny_run(b, d, name);
    case DensePlan::kTiles256:
    case DensePlan::kTiles128: {
      const bool large = dense_plan(d) == DensePlan::kTiles256;
      a.vec_out = d.oi ? d.N % 8 == 0 && aligned16(d.out) : d.N % 4 == 0 && ((uintptr_t)d.out & 7) == 0;
      return large ? run_dense_tiles<Tile256>(b, name, a) : run_dense_tiles<Tile128>(b, name, a);
    }
    default: break;
  }
  const int64_t tm = (d.M + kAnyTile - 1) / kAnyTile, tn = (d.N + kAnyTile - 1) / kAnyTile;
  if (tm * tn >= (int64_t)1 << 31) return set_error(MX_ERR_INVALID, "F8Dense: more than 2^31 workgroups");
  a.tiles_n = (int)tn;
  auto k = d.out_dt == MX_DTYPE_FLOAT32 ? f8_dense_any_kernel<true> : f8_dense_any_kernel<false>;
  return launch(b, name, [&] {
    dispatch(k, dim3((unsigned)(tm * tn)), dim3(kAnyThreads), 0, b->stream, a);
  });
}

}  // namespace mx
