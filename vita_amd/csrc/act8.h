// 8-bit activation checkpoints: device helpers shared by act8.hip and addnorm.hip.
//
// A row is cut into groups of 32 neighbours.  A group has one power-of-two scale 2^e (kept as the byte e + 127, e8m0) and 32
// e4m3 codes; a stored value is code * 2^e.  e is the smallest integer in [-117, 119] with amax / 2^e <= 448, amax over the
// group's FINITE values, so no finite value saturates except above 1.75 * 2^127, where e stops so that code * 2^e stays finite.
// At the other end e >= -117 keeps the smallest nonzero value, 2^-9 * 2^e, a normal number.  A power of two costs up to one
// bit of the codes' range against an arbitrary fp32 scale and buys exactness: code * 2^e has 4 significant bits, so it is exact
// in bf16 and a matrix product on restored values adds no rounding of its own.
//
// Rounding to e4m3 is the hardware's (v_cvt_pk_fp8_f32, nearest, ties to even); value / 2^e is a multiplication by a power of
// two and exact (below 2^-126 it may round, far under half of the smallest code).  NaN and infinities become the NaN code.
//
// A lane holds 8 neighbouring values, 4 neighbouring lanes a group: amax is two DPP steps inside a quad.
#pragma once
#include "common.h"

#define ACT8_GROUP 32
#define ACT8_MAX_COLS (1 << 20)

__device__ __forceinline__ uint32_t act8_quad_max(uint32_t v) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);    // quad_perm [1,0,3,2]
  v = v > a ? v : a;
  const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);    // quad_perm [2,3,0,1]
  return v > b ? v : b;
}
// scale byte of a group from the bits of its amax: amax = m * 2^E, 1 <= m < 2 -> e = E - 8, one more when m > 1.75
// (adding 0x1fffff carries into the exponent exactly then)
__device__ __forceinline__ uint32_t act8_scale_byte(uint32_t amax) {
  int c = (int)((amax + 0x1fffffu) >> 23) - 8;
  c = c < 10 ? 10 : c;
  return (uint32_t)(c > 246 ? 246 : c);
}
__device__ __forceinline__ float act8_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
__device__ __forceinline__ float act8_inv_scale(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }

// Bits of the largest magnitude whose group the plain path may code: above it lie NaN, infinities and amax > 1.75 * 2^127, where e is
// at its end and values saturate
#define ACT8_TOP 0x7f600000u

// the 8 values of a lane (all 4 lanes of the quad call it) over their group's scale: t, the scale byte and the bits of the largest magnitude
__device__ __forceinline__ void act8_scaled(const float (&v)[8], float (&t)[8], uint32_t& byte, uint32_t& m) {
  m = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) { const uint32_t a = __builtin_bit_cast(uint32_t, v[r]) & 0x7fffffffu; m = m > a ? m : a; }
  m = act8_quad_max(m);
  if (__builtin_expect(m > ACT8_TOP, 0)) {      // the four lanes of a quad together
    m = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const uint32_t a = __builtin_bit_cast(uint32_t, v[r]) & 0x7fffffffu;
      if (a < 0x7f800000u) m = m > a ? m : a;
    }
    m = act8_quad_max(m);
    byte = act8_scale_byte(m);
    const float inv = act8_inv_scale(byte);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      t[r] = __builtin_amdgcn_fmed3f(v[r] * inv, -448.f, 448.f);
      if ((__builtin_bit_cast(uint32_t, v[r]) & 0x7f800000u) == 0x7f800000u) t[r] = __builtin_nanf("");
    }
  } else {
    byte = act8_scale_byte(m);
    const float inv = act8_inv_scale(byte);
#pragma unroll
    for (int r = 0; r < 8; ++r) t[r] = v[r] * inv;
  }
}
__device__ __forceinline__ u32x2 act8_codes(const float (&t)[8]) {
  u32x2 q;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * h], t[4 * h + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * h + 2], t[4 * h + 3], w, true);
    q[h] = (uint32_t)w;
  }
  return q;
}
// the 8 values of a lane (all 4 lanes of the quad call it) -> their codes; byte = the group's scale byte
__device__ __forceinline__ u32x2 act8_encode(const float (&v)[8], uint32_t& byte) {
  float t[8];
  uint32_t m;
  act8_scaled(v, t, byte, m);
  return act8_codes(t);
}
// Whether a value over its scale lies within w steps of 2^-23 of a border between two codes (normal ones: 3 bits of the mantissa, a border
// half a step behind each), or a group's maximum within w of the border between two scales (1.75 2^k)
__device__ __forceinline__ uint32_t act8_off_border(float t, uint32_t w) { return (__builtin_bit_cast(uint32_t, t) + 0x80000u + w) & 0xfffffu; }     // <= 2 w
__device__ __forceinline__ bool act8_near_scale(uint32_t m, uint32_t w) { return (m & 0x7fffffu) - 0x600000u + w <= 2 * w; }
__device__ __forceinline__ void act8_decode(u32x2 q, uint32_t byte, float (&v)[8]) {
  typedef float f32x2v __attribute__((ext_vector_type(2)));
  const float s = act8_scale(byte);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2v a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
    v[4 * h] = a[0] * s; v[4 * h + 1] = a[1] * s; v[4 * h + 2] = b[0] * s; v[4 * h + 3] = b[1] * s;
  }
}

// ---- 8 neighbouring columns [c, c + 8) of a row with d real columns; columns >= d read as 0 and are never touched.  whole: the row has
// two more behind it, so that all 8 are inside the matrix' memory wherever c < d; what stands behind d comes back as it is then.
struct Raw8 { u32x4 a, b; };      // bf16 rows use a only
template <bool F32>
__device__ __forceinline__ Raw8 raw_load8(const void* row, int c, int d, bool whole = false) {
  Raw8 w;
  w.a = w.b = u32x4{0, 0, 0, 0};
  if (c + 8 <= d || (whole && c < d)) {
    if (F32) {
      w.a = *reinterpret_cast<const u32x4*>((const float*)row + c);
      w.b = *reinterpret_cast<const u32x4*>((const float*)row + c + 4);
    } else {
      w.a = *reinterpret_cast<const u32x4*>((const uint16_t*)row + c);
    }
  } else if (c < d) {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (c + r < d) {
        if (F32) {
          if (r < 4) w.a[r & 3] = ((const uint32_t*)row)[c + r];
          else w.b[r & 3] = ((const uint32_t*)row)[c + r];
        } else w.a[r >> 1] |= (uint32_t)((const uint16_t*)row)[c + r] << (16 * (r & 1));
      }
  }
  return w;
}
template <bool F32>
__device__ __forceinline__ void raw_values8(const Raw8& w, float (&v)[8]) {
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    if (F32) v[r] = __builtin_bit_cast(float, r < 4 ? w.a[r & 3] : w.b[r & 3]);
    else v[r] = __builtin_bit_cast(float, (r & 1) ? (w.a[r >> 1] & 0xffff0000u) : (w.a[r >> 1] << 16));
  }
}
__device__ __forceinline__ u32x4 pack_bf16x8(const float (&v)[8]) {      // four v_cvt_pk_bf16_f32
  bf16x8 o;
#pragma unroll
  for (int r = 0; r < 8; ++r) o[r] = (__bf16)v[r];
  return __builtin_bit_cast(u32x4, o);
}
// 8 neighbouring floats of a vector of d (gamma, beta), `fill` behind its end and for NULL; al: 16-byte aligned
__device__ __forceinline__ void vec_load8(const float* p, int c, int d, bool al, float fill, float (&v)[8]) {
  if (p && al && c + 8 <= d) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p + c), b = *reinterpret_cast<const f32x4*>(p + c + 4);
#pragma unroll
    for (int r = 0; r < 4; ++r) { v[r] = a[r]; v[4 + r] = b[r]; }
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = p && c + r < d ? p[c + r] : fill;
  }
}
// columns [c, c + 8) of a row of `ld` columns (ld % 8 == 0 for bf16, % 4 for fp32): all 8, or those below ld
__device__ __forceinline__ void store8(void* row, int c, int64_t ld, bool f32, const float (&v)[8]) {
  if (f32) {
    if (c < ld) *reinterpret_cast<f32x4*>((float*)row + c) = f32x4{v[0], v[1], v[2], v[3]};
    if (c + 4 < ld) *reinterpret_cast<f32x4*>((float*)row + c + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else if (c < ld) {
    *reinterpret_cast<u32x4*>((uint16_t*)row + c) = pack_bf16x8(v);
  }
}

// ---- one column to a lane: 64 neighbouring columns of a wave, a group is one half of it
template <bool F32>
__device__ __forceinline__ float load1(const void* row, int c, int d) {
  if (c >= d) return 0.f;
  return F32 ? ((const float*)row)[c] : bf16_bits_to_f32(((const uint16_t*)row)[c]);
}
__device__ __forceinline__ void store1(void* row, int c, int64_t ld, bool f32, float v) {
  if (c >= ld) return;
  if (f32) ((float*)row)[c] = v; else ((uint16_t*)row)[c] = f32_to_bf16_bits(v);
}
__device__ __forceinline__ uint8_t act8_encode1(float v, uint32_t& byte) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
  uint32_t m = a < 0x7f800000u ? a : 0u;
  m = act8_quad_max(m);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) { const uint32_t b = (uint32_t)__shfl_xor((int)m, o, 64); m = m > b ? m : b; }
  byte = act8_scale_byte(m);
  float t = __builtin_amdgcn_fmed3f(v * act8_inv_scale(byte), -448.f, 448.f);
  if (a >= 0x7f800000u) t = __builtin_nanf("");
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(t, t, 0, false);
}
__device__ __forceinline__ float act8_decode1(uint8_t q, uint8_t byte) {
  return __builtin_amdgcn_cvt_f32_fp8((int)q, 0) * act8_scale(byte);
}

// host: a [rows][ld] matrix of a VITA_DT_* type that the kernels may read / write in 16-byte pieces
static inline bool act8_mat_ok(const void* p, int64_t ld, int64_t d, int32_t dtype) {
  if (dtype != VITA_DT_BF16 && dtype != VITA_DT_F32) return false;
  return p && ld >= d && ld % (dtype == VITA_DT_BF16 ? 8 : 4) == 0 && ((uintptr_t)p & 15) == 0;
}
// host: codes and scale bytes of [rows][d]
static inline bool act8_codes_ok(const void* q, int64_t ldq, const void* scale, int64_t lds, int64_t d) {
  const int64_t g = (d + ACT8_GROUP - 1) / ACT8_GROUP;
  return q && scale && ldq >= g * ACT8_GROUP && ldq % 16 == 0 && ((uintptr_t)q & 15) == 0 && lds >= g;
}
