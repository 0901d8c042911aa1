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
#include "f8_wgrad_schedule.h"
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
  int tiles_n, slices, tokens;  // slices of the tokens of a tile, tokens of a slice
  char* part;                   // [tile][slice] sums (slices > 1)
  uint32_t* arrived;            // [tile], zero between launches
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

// Staging.  The codes and dy of a step travel through registers, requested a step ahead: 16 codes a chunk,
// scaled to bf16 (32 bytes of LDS), and 8 values of dy.  LDS keeps both as they lie in memory,
// [token][column], in two buffers; the operands, eight consecutive tokens of a column per lane, come out
// through the transposing read, four tokens at a time.  A row's 32-byte pieces are XOR-ed with
// 2 (token & 3), so that the 32 lanes of a half-wave, which read four rows of two neighbouring pieces,
// touch every bank once.
//
// Schedule (f8_wgrad_schedule.h).  A step is groups of TK MFMAs, one operand of dy against the wave's TK operands of x.  An
// operand of dy is read kLast groups ahead of its use and the x operands of the next 16 tokens
// during the present ones.  The step's barrier stands before its last kLast groups, whose operands
// are then in registers: under them travel the first operands of the next step.  A chunk of the next step
// is staged, and that of the step after requested into its registers, in the groups before the barrier.
//
// Columns past K or N hold whatever lies there: they meet only results that are not stored.  Tokens past
// M are zeros in both operands, their scales too (a step past the last is staged like any other and not used).  WHOLE: rows
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

template <class Tile, bool OI, bool WHOLE>
__global__ __launch_bounds__(Tile::kThreads, Tile::kOccupancy) void f8_wgrad_kernel(WGradArgs a) {
  constexpr int TK = Tile::TK, TN = Tile::TN, S = Tile::S, P = Tile::P, kThreads = Tile::kThreads;
  constexpr bool F32 = P == 3;
  constexpr int WX = Tile::kK, WD = Tile::kN;          // columns of the operands
  constexpr int kXRow = 2 * WX, kDRow = 2 * WD;        // bytes of a row in LDS
  constexpr int kXBuf = S * kXRow, kDBuf = S * kDRow;  // x and a part of dy of a step
  constexpr int kStep = kXBuf + P * kDBuf;             // LDS of a step
  constexpr int CX = Tile::kXChunks, CD = Tile::kDChunks;  // chunks of x and dy that a thread stages
  constexpr int RX = kThreads / (WX / 16), RD = kThreads / (WD / 8);  // rows between a thread's chunks
  constexpr int kParts = Tile::kParts, kPart = Tile::kPart, G = Tile::kGroups, kRing = Tile::kRing, kLast = Tile::kLast;
  constexpr int kPieces = Tile::kPieces;
  auto x_before = [](int p) constexpr { return (p * 2 * CX + kPieces - 1) / kPieces; };  // pieces of x among the first p
  constexpr int H = F32 ? 2 : 1, E = F32 ? 4 : 2;      // loads of a dy chunk, bytes of a value
  static_assert(kStep % 1024 == 0, "the buffers differ above the bits of a piece");
  static_assert((TK & (TK - 1)) == 0 && (TN & (TN - 1)) == 0, "a wave's pieces start on a multiple of their number: an XOR picks one");
  extern __shared__ __align__(1024) uint8_t lds[];     // [2]: x [S][WX], then the parts of dy [P][S][WD], bf16
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, i = lane % 32, g = lane / 32;
  int kt, nt, tile, slice;
  {
    // Runs of 4 tiles of k by all tiles of n: a run's workgroups share their rows of x and dy in an L2.  A tile's
    // slices of the tokens are neighbours.
    const int it = xcd_order((int)blockIdx.x, (int)gridDim.x), t = it / a.slices;
    tile = t;
    slice = it - t * a.slices;
    const int tiles_k = (int)gridDim.x / a.slices / a.tiles_n;
    const int per = 4 * a.tiles_n, q = t / per, rows = min(4, tiles_k - 4 * q), in = t - q * per;
    kt = 4 * q + in % rows;
    nt = in / rows;
  }
  const int k0 = kt * WX, n0 = nt * WD;
  const int from = slice * a.tokens, to = min(a.M, from + a.tokens);  // the slice's tokens
  const int64_t x_total = (int64_t)a.M * a.K, dy_total = (int64_t)a.M * a.N;
  const int xrow = tid / (WX / 16), xk = k0 + 16 * (tid % (WX / 16));  // the thread's first chunk of a step
  const int drow = tid / (WD / 8), dn = n0 + 8 * (tid % (WD / 8));
  const int kb = min(xk / kBlock, a.KB - 1);

  u32x4 xr[CX], dr[CD][H];
  float sr[CX];
  // Byte offsets of the thread's chunks within a step (below 64 rows of 2^26 bytes), and the windows of the
  // step requested next.
  uint32_t x_off[CX], s_off[CX], d_off[CD];
#pragma unroll
  for (int j = 0; j < CX; ++j) {
    x_off[j] = (uint32_t)(xrow + j * RX) * (uint32_t)a.K + (uint32_t)min(xk, a.K - (WHOLE ? 16 : 1));
    s_off[j] = 4 * ((uint32_t)(xrow + j * RX) * (uint32_t)a.KB + (uint32_t)kb);
  }
#pragma unroll
  for (int j = 0; j < CD; ++j) d_off[j] = E * ((uint32_t)(drow + j * RD) * (uint32_t)a.N + (uint32_t)min(dn, a.N - (WHOLE ? 8 : 1)));
  // (A slice's windows end with its tokens.)
  Window xw{a.x + (int64_t)from * a.K, (int64_t)(to - from) * a.K};
  Window sw{(const uint8_t*)(a.x_scale + (int64_t)from * a.KB), (int64_t)(to - from) * a.KB * 4};
  Window dw{(const uint8_t*)a.dy + (int64_t)from * a.N * E, (int64_t)(to - from) * a.N * E};
  auto advance = [&]() __attribute__((always_inline)) {
    xw.move((int64_t)S * a.K);
    sw.move((int64_t)S * a.KB * 4);
    dw.move((int64_t)S * a.N * E);
  };
  auto request = [&](auto inside, int m0, int piece) __attribute__((always_inline)) {
    constexpr bool kInside = decltype(inside)::value;
    if (x_before(piece + 1) > x_before(piece)) {
      const int j = x_before(piece) / 2;
      if (x_before(piece) % 2 == 0) return;  // the first half of a chunk: the second still stands in the registers
      if constexpr (WHOLE) {
        xr[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(xw.resource(), x_off[j], 0, 0));
        sr[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sw.resource(), s_off[j], 0, 0));
      } else if constexpr (kInside) {
        xr[j] = load16_any(xw.p + x_off[j]);
        sr[j] = *(const float*)(sw.p + s_off[j]);
      } else {
        const int64_t row = min(m0 + xrow + j * RX, a.M - 1), at = row * a.K + min(xk, a.K - 1);
        xr[j] = load16(a.x + at, x_total - at);
        sr[j] = a.x_scale[row * a.KB + kb];
      }
    } else {
      const int j = piece - x_before(piece);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        if constexpr (WHOLE) {
          dr[j][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(dw.resource(), d_off[j], 16 * h, 0));
        } else if constexpr (kInside) {
          dr[j][h] = load16_any(dw.p + d_off[j] + 16 * h);
        } else {
          const int64_t at = (int64_t)min(m0 + drow + j * RD, a.M - 1) * a.N + min(dn, a.N - 1) + 4 * h;
          dr[j][h] = load16((const uint8_t*)a.dy + E * at, E * (dy_total - at));
        }
      }
    }
  };
  // Piece of the step from m0 into LDS at `step`.
  auto swizzled = [](int row, int m, int piece) { return m * row + 32 * (piece ^ (2 * (m & 3))); };
  auto stage = [&](auto inside, int m0, uint32_t step, int piece) __attribute__((always_inline)) {
    constexpr bool kMask = !WHOLE && !decltype(inside)::value;
    uint8_t* xb = lds + step;
    if (x_before(piece + 1) > x_before(piece)) {
      const int j = x_before(piece) / 2, half = x_before(piece) % 2;
      if (kMask && half == 0 && m0 + xrow + j * RX >= to) xr[j] = u32x4{0u, 0u, 0u, 0u}, sr[j] = 0.0f;
      u32x4 o;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const f32x4 v = decode4(xr[j][2 * half + w]);
        const float s = sr[j];
        const f32x2 lo = {v[0] * s, v[1] * s}, hi = {v[2] * s, v[3] * s};
        o[2 * w] = __builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2));
        o[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2));
      }
      *(u32x4*)(xb + swizzled(kXRow, xrow + j * RX, tid % (WX / 16)) + 16 * half) = o;
    } else {
      const int j = piece - x_before(piece), c = tid % (WD / 8);
#pragma unroll
      for (int h = 0; h < H; ++h)
        if (kMask && m0 + drow + j * RD >= to) dr[j][h] = u32x4{0u, 0u, 0u, 0u};
      uint8_t* q = xb + kXBuf + swizzled(kDRow, drow + j * RD, c / 2) + 16 * (c % 2);
      if constexpr (F32) {
        uint16_t p[8][3];
#pragma unroll
        for (int e = 0; e < 8; ++e) parts_of(__uint_as_float(dr[j][e / 4][e % 4]), p[e]);
#pragma unroll
        for (int t = 0; t < 3; ++t) {
          u32x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (uint32_t)p[2 * e][t] | (uint32_t)p[2 * e + 1][t] << 16;
          *(u32x4*)(q + t * kDBuf) = o;
        }
      } else {
        *(u32x4*)q = dr[j][0];
      }
    }
  };

  // Operand reads: token 8 g + 4 h + (lane % 16) / 4 of 16, columns 32 t + 16 (i / 16) + 4 (lane % 4) ..
  const int wk = wave / Tile::WN, wn = wave % Tile::WN;
  const uint32_t base = lds_addr(lds);
  auto read_base = [&](int row, int piece) { return base + (uint32_t)swizzled(row, 8 * g + lane % 16 / 4, piece + i / 16) + 8 * (lane % 4); };
  const uint32_t xa = read_base(kXRow, 2 * wk * TK), da = read_base(kDRow, 2 * wn * TN) + kXBuf;
  auto operand = [&](uint32_t at, int row, int t, int off) __attribute__((always_inline)) {
    const uint32_t p = (at ^ (uint32_t)(64 * t)) + (uint32_t)off;
    const u32x2 lo = read_tr16(p), hi = read_tr16(p + 4 * row);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  u32x4 xo[2][TK], dv[kRing];
  auto read_x = [&](int set, int t, uint32_t step, int part) __attribute__((always_inline)) {
    xo[set][t] = operand(xa + step, kXRow, t, part * 16 * kXRow);
  };
  auto read_dy = [&](int q, uint32_t step) __attribute__((always_inline)) {  // of group q of a step
    dv[q % kRing] = operand(da + step, kDRow, q % TN, (q / TN % P) * kDBuf + q / (TN * P) * 16 * kDRow);
  };

  f32x16 acc[TK][TN] = {};
  uint32_t cur = 0;
  // The step from token m0.  inside (WHOLE: always): what it stages lies before `to` and what it requests in the array,
  // a chunk past a row's end included.
  auto step = [&](auto inside, int m0) __attribute__((always_inline)) {
      const uint32_t next = kStep - cur;
      advance();
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const int part = q / kPart, set = part % 2;
        if (q == Tile::kBarrier) lds_barrier();
        // Operands of later groups.
        if (q + kLast < G)
          read_dy(q + kLast, cur);
        else
          read_dy(q + kLast - G, next);
        if (part + 1 < kParts && q % kPart < Tile::kXGroups) {
#pragma unroll
          for (int e = 0; e < Tile::kXPer; ++e) {
            const int t = q % kPart * Tile::kXPer + e;
            if (t < TK) read_x(1 - set, t, cur, part + 1);
          }
        }
        if (q >= G - Tile::kNextGroups) {
#pragma unroll
          for (int e = 0; e < Tile::kNextPer; ++e) {
            const int t = (q - (G - Tile::kNextGroups)) * Tile::kNextPer + e;
            if (t < TK) read_x(0, t, next, 0);
          }
        }
        if (q >= Tile::kStageFrom && q < Tile::kBarrier) {
#pragma unroll
          for (int e = 0; e < Tile::kPerGroup; ++e) {
            const int p = (q - Tile::kStageFrom) * Tile::kPerGroup + e;
            if (p < kPieces) {
              stage(inside, m0 + S, next, p);
              request(inside, m0 + 2 * S, p);
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
        if constexpr (WHOLE || decltype(inside)::value) {
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
  };
  if (from < to) {
    constexpr std::integral_constant<bool, WHOLE> edge{};
#pragma unroll
    for (int p = 0; p < kPieces; ++p) request(edge, from, p);
    advance();
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      stage(edge, from, 0, p);
      request(edge, from + S, p);
    }
    lds_barrier();
#pragma unroll
    for (int t = 0; t < TK; ++t) read_x(0, t, 0, 0);
#pragma unroll
    for (int q = 0; q < kLast; ++q) read_dy(q, 0);
    int m0 = from;
    if constexpr (!WHOLE) {
      const int64_t most = min(a.K, a.N);
      if (a.K <= 1 << 24 && a.N <= 1 << 24)
        for (; m0 + 3 * S <= to && (int64_t)(a.M - (m0 + 3 * S)) * most >= 16; m0 += S) step(std::true_type{}, m0);
    }
    for (; m0 < to; m0 += S) step(edge, m0);
  }

  if (a.slices > 1) {
    // The slices' sums meet in scratch, stored and loaded with the agent-scope coherence bit (sc1): the slices may run
    // on different XCDs.  The last to arrive adds them in order and goes on; it leaves the counter at zero.
    __shared__ int s_last;
    constexpr int kSc1 = 16;
    const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc((char*)a.part + (int64_t)tile * a.slices * Tile::kPartBytes, 0,
                                                                         a.slices * Tile::kPartBytes, 0x00027000);
    auto at = [&](int sl, int t, int n, int q) {
      return (uint32_t)(sl * Tile::kPartBytes + (((t * TN + n) * 4 + q) * kThreads + tid) * 16);
    };
#pragma unroll
    for (int t = 0; t < TK; ++t)
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 v = {acc[t][n][4 * q], acc[t][n][4 * q + 1], acc[t][n][4 * q + 2], acc[t][n][4 * q + 3]};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), prs, at(slice, t, n, q), 0, kSc1);
        }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      const uint32_t before = __hip_atomic_fetch_add(&a.arrived[tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = before + 1u == (uint32_t)a.slices;
      if (s_last) __hip_atomic_store(&a.arrived[tile], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
#pragma unroll
    for (int t = 0; t < TK; ++t)
#pragma unroll
      for (int n = 0; n < TN; ++n) acc[t][n] = f32x16{};
    constexpr int kTogether = TK * TN <= 4 ? 2 : 1;  // slices in flight at a time
#pragma unroll kTogether
    for (int sl = 0; sl < a.slices; ++sl)
#pragma unroll
      for (int t = 0; t < TK; ++t)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, at(sl, t, n, q), 0, kSc1));
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[t][n][4 * q + r] += v[r];
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

template <class Tile>
int run_tiles(mx_backend* b, const char* name, WGradArgs a, bool whole, int slices) {
  constexpr int kLds = 2 * 2 * Tile::S * (Tile::kK + Tile::P * Tile::kN);
  const int64_t tk = (a.K + Tile::kK - 1) / Tile::kK, tn = (a.N + Tile::kN - 1) / Tile::kN;
  const int steps = (a.M + Tile::S - 1) / Tile::S, per = (steps + slices - 1) / slices;
  a.tokens = std::max(per, 1) * Tile::S;
  a.slices = std::max((a.M + a.tokens - 1) / a.tokens, 1);
  a.tiles_n = (int)tn;
  if (tk * tn * a.slices * Tile::kThreads > kMaxWorkItems)
    return set_error(MX_ERR_INVALID, "F8WeightGradient: a result of more tiles than a launch holds");
  if (a.slices > 1) {
    void* scratch = nullptr;
    MX_TRY(ensure_scratch(b, kScratchCounterBytes + (size_t)(tk * tn * a.slices) * Tile::kPartBytes, &scratch));
    a.arrived = (uint32_t*)scratch;
    a.part = (char*)scratch + kScratchCounterBytes;
  }
  auto k = a.oi ? (whole ? f8_wgrad_kernel<Tile, true, true> : f8_wgrad_kernel<Tile, true, false>)
                : (whole ? f8_wgrad_kernel<Tile, false, true> : f8_wgrad_kernel<Tile, false, false>);
  MX_CHECK_HIP(hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
  return launch(b, name, [&] { dispatch(k, dim3((unsigned)(tk * tn * a.slices)), dim3(Tile::kThreads), kLds, b->stream, a); });
}

struct Choice {
  bool large;  // 256 x 256 tiles
  int slices;
};

// The tile and the number of token slices that take the least time by the times of their parts: a launch 3 us; a
// round of workgroups its first loads and its stores, and its steps (the 128 x 128 tiles run two to a CU); for sums that
// meet in scratch 3 us and 1.2 a slice.  Against sweeps at 16 shapes (profiles/f8_tile_sweeps.txt) the choice is within 2% of the
// best, and 5% behind for 64 tokens of 4096 x 4096.  Measured (us; 256 x 256 | 128 x 128 by slices 1, 2, 3, 4, 6, 8):
//   bf16  2048 x 4096 x 14336    262 | 328         4096 x 1024 x 1024    66 (in 3) | 49 31 26 24 30 31
//         2048 x 4096 x 4096      71 |  95          333 x 1536 x 384     19 | 9.0 11 11 -  13
//         2048 x 2048 x 2048      54 |  31 34 42
//   f32    333 x 1536 x 384       36 | 17.2 15.1 14.0 13.8 15.0    4000 x 512 x 512     111 (in 6) | 139 76 55 44 34 31 (29 in 12)
//         2048 x 2048 x 2048      95 (in 3) | 80 71 77
//         2048 x 4096 x 14336    711 | 855              515 x 7552 x 10528   289 | 356
//         4096 x 4096 x 4096     365 | 467               63 x 7808 x 7296     76 | 64
// Tiles of 128 x 256 and 256 x 128, two workgroups a CU, took 291 and 294 us for the first when 256 x 256 took 265.
Choice plan_of(const F8WGradDesc& d) {
  const bool f32 = d.dy_dt == MX_DTYPE_FLOAT32;
  Choice best{false, 1};
  double least = 1e30;
  for (int large = 0; large < 2; ++large) {
    const int side = large ? 256 : 128, S = f32 ? 32 : 64, slots = large ? 256 : 512;
    const int64_t tiles = ((d.K + side - 1) / side) * ((d.N + side - 1) / side), steps = (d.M + S - 1) / S;
    for (int slices = 1; slices <= 16 && slices <= std::max<int64_t>(steps, 1); ++slices) {
      const int64_t per = (steps + slices - 1) / slices;
      const double part = (double)tiles * slices * side * side * 4;
      if (tiles * slices * (large ? WGradTile256::kThreads : WGradTile128::kThreads) > kMaxWorkItems) continue;
      if (slices > 1 && ((steps + per - 1) / per != slices || tiles > (int64_t)(kScratchCounterBytes / 4) || part > 64e6)) continue;
      const bool alone = tiles * slices <= 256;  // at most one workgroup a CU
      const double step = large ? (f32 ? 2.6 : 1.72) : f32 ? (alone ? 1.28 : 1.9) : alone ? 0.83 : 1.2;
      const double us = 3 + (double)((tiles * slices + slots - 1) / slots) * ((large ? 11 : alone ? 2 : 5) + (double)per * step) + (slices > 1 ? 3 + 1.2 * slices : 0);
      if (us < least) {
        least = us;
        best = {large != 0, slices};
      }
    }
  }
  return best;
}

const char* kernel_name(const F8WGradDesc& d) { return d.dy_dt == MX_DTYPE_FLOAT32 ? "f8_wgrad_f32" : "f8_wgrad_bf16"; }

}  // namespace

std::string f8_wgrad_plan(const F8WGradDesc& d) {
  const Choice c = plan_of(d);
  return std::string(kernel_name(d)) + (c.large ? " 256x256" : " 128x128") + " slices " + std::to_string(c.slices);
}

int f8_wgrad_run(mx_backend* b, const F8WGradDesc& d) {
  if (d.K == 0 || d.N == 0) return MX_OK;
  const bool vec = (d.oi ? d.K : d.N) % 4 == 0 && ((uintptr_t)d.out & (d.out_dt == MX_DTYPE_FLOAT32 ? 15 : 7)) == 0;
  const WGradArgs a{d.x, d.x_scale, d.dy, d.out, (int)d.M, (int)d.K, (int)d.N, (int)blocks(d.K), d.out_dt, d.oi, vec, 0, 1, 0, nullptr, nullptr};
  const bool whole = d.K % 16 == 0 && d.N % 8 == 0 && d.K <= 1 << 24 && d.N <= 1 << 24 && aligned16(d.x) && aligned16(d.dy);
  const char* name = kernel_name(d);
  const Choice c = plan_of(d);
  if (d.dy_dt == MX_DTYPE_FLOAT32)
    return c.large ? run_tiles<WGradTile256F32>(b, name, a, whole, c.slices) : run_tiles<WGradTile128F32>(b, name, a, whole, c.slices);
  return c.large ? run_tiles<WGradTile256>(b, name, a, whole, c.slices) : run_tiles<WGradTile128>(b, name, a, whole, c.slices);
}

}  // namespace mx
