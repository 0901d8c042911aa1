// Device helpers of the operators on 8-bit floating-point blocks: e4m3 codes with one float32 scale
// for every 128 consecutive values of a row, or for every 128 x 128 block of a weight matrix.
#pragma once

#include <type_traits>

#include "device_common.h"

namespace mx {
namespace f8 {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;

constexpr int kBlock = MX_F8_BLOCK;

inline int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 32 consecutive codes, an operand of the 16x16x128 MFMA, from 16-byte aligned memory.
__device__ __forceinline__ i32x8 join(const u32x4& lo, const u32x4& hi) {
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
__device__ __forceinline__ i32x8 read32(const uint8_t* p) { return join(*(const u32x4*)p, *(const u32x4*)(p + 16)); }

// The four values of a word of codes (v_cvt_pk_f32_fp8: exact, NaN codes to NaN).
__device__ __forceinline__ f32x4 decode4(uint32_t w) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return f32x4{a.x, a.y, b.x, b.y};
}

// Eight codes as the bf16 values they stand for (exact), an operand of the bf16 16x16x32 MFMA.
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four values, at most 448 in magnitude, to codes (round to nearest even; NaN to a NaN code).
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// 16 bytes from any address.
__device__ __forceinline__ u32x4 load16_any(const uint8_t* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// 16 bytes from p, of which the first n are there (the rest 0).  p may be any byte.
__device__ __forceinline__ u32x4 load16(const uint8_t* p, int64_t n) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (n >= 16) {
    __builtin_memcpy(&v, p, 16);
  } else {
    for (int i = 0; i < n; ++i) v[i / 4] |= (uint32_t)p[i] << (8 * (i % 4));
  }
  return v;
}

// Four consecutive results from element `at`, of which the first n are in the row; vec: they are whole and aligned.
// (Unaligned ones still go as one store: value by value an instruction writes 4 bytes to each of 64 places.)
__device__ __forceinline__ void store4(void* out, int64_t at, int n, bool vec, int dt, const f32x4& v) {
  if (vec ? n > 0 : n >= 4) {
    if (dt == MX_DTYPE_FLOAT32) {
      if (vec)
        *(f32x4*)((float*)out + at) = v;
      else
        __builtin_memcpy((float*)out + at, &v, 16);
    } else {
      const f32x2 lo = {v[0], v[1]}, hi = {v[2], v[3]};
      const u32x2 o = {__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2)),
                       __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2))};
      if (vec)
        *(u32x2*)((uint16_t*)out + at) = o;
      else
        __builtin_memcpy((uint16_t*)out + at, &o, 8);
    }
  } else if (!vec) {
#pragma unroll
    for (int r = 0; r < 3; ++r)
      if (r < n) store_f(out, at + r, dt, v[r]);
  }
}

// Workgroup barrier ordering LDS only: global loads in flight stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// LDS byte address of a shared-memory pointer.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

// Transposing LDS reads: every 16 lanes read a block of 16 columns, lane l's eight bytes lying at its
// own address, and lane i gets column i.  16-bit values: four rows, of which lane l holds row l / 4,
// columns 4 (l % 4) ..; codes: eight rows, lane l row l / 2, columns 8 (l % 2) ...
__device__ __forceinline__ u32x2 read_tr16(uint32_t addr) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)addr));
}
__device__ __forceinline__ u32x2 read_tr8(uint32_t addr) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)addr));
}

// Workgroup b of n to a work item such that each XCD (the hardware deals workgroups to the eight in
// turn) takes a contiguous run of items.
__device__ __forceinline__ int xcd_order(int b, int n) {
  constexpr int kXcds = 8;
  const int x = b % kXcds, q = n / kXcds, r = n % kXcds;
  return x * q + (x < r ? x : r) + b / kXcds;
}

// The magnitude bits of a finite value, 0 of an infinity or NaN: they compare as integers.
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

// The exponent of a block's scale from its largest magnitude's bits: the smallest e >= -126 with
// a <= 448 * 2^e.  a = 1.f * 2^(E - 127) and 448 = 1.75 * 2^8, so e = E - 135, and one more where
// 1.f > 1.75.  0 (a scale of 1) where a is 0.  At most 120, so that 2^e and 2^-e are normal floats.
__device__ __forceinline__ int scale_exponent(uint32_t a) {
  const int e = (int)(a >> 23) - 135 + ((a & 0x7fffffu) > 0x600000u ? 1 : 0);
  return a == 0 ? 0 : max(e, -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// v / s for s = 2^-e as v * inv, exact (or below any code); NaN where v is not finite, as the format
// holds no infinity.
__device__ __forceinline__ float scaled(float v, float inv) {
  return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : v * inv;
}

// The largest of 16 lanes' values (a row of the wave), in every lane of the row.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  auto step = [&](auto ctrl) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true);
    v = v > o ? v : o;
  };
  step(std::integral_constant<int, 0xB1>{});   // quad_perm 1,0,3,2
  step(std::integral_constant<int, 0x4E>{});   // quad_perm 2,3,0,1
  step(std::integral_constant<int, 0x141>{});  // row_half_mirror
  step(std::integral_constant<int, 0x140>{});  // row_mirror
  return v;
}

}  // namespace f8
}  // namespace mx
