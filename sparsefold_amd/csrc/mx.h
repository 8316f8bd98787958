// Microscaled numbers on the device: 4 lanes hold 8 elements each of a block of 32.
#pragma once

#include "sf_common.h"

struct MxFp8 {
  static constexpr int kFormat = SF_FORMAT_MXFP8, kBytes = 8;          // of 8 codes
  static constexpr int kPower = 8;                                      // exponent of the largest power of two
  typedef u32x2 Codes;
  // 8 elements that the scale has been taken out of.  The instruction rounds to the nearest, ties to even; past 448 it would
  // give NaN, so that is clamped before.
  static __device__ __forceinline__ Codes encode(const float (&y)[8]) {
    Codes c;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = __builtin_amdgcn_fmed3f(y[4 * w + e], -448.f, 448.f);
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
      c[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], p, true);
    }
    return c;
  }
  static __device__ __forceinline__ void decode(Codes c, float (&y)[8]) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], true);
      y[4 * w] = a[0]; y[4 * w + 1] = a[1]; y[4 * w + 2] = b[0]; y[4 * w + 3] = b[1];
    }
  }
};

struct MxFp4 {
  static constexpr int kFormat = SF_FORMAT_MXFP4, kBytes = 4;
  static constexpr int kPower = 2;
  typedef uint32_t Codes;
  static __device__ __forceinline__ Codes encode(const float (&y)[8]) {    // (saturates by itself)
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[0], y[1], 1.f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], 1.f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[4], y[5], 1.f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[6], y[7], 1.f, 3);
    return c;
  }
  static __device__ __forceinline__ void decode(Codes c, float (&y)[8]) {
    const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1),
                p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);
    y[0] = p0[0]; y[1] = p0[1]; y[2] = p1[0]; y[3] = p1[1]; y[4] = p2[0]; y[5] = p2[1]; y[6] = p3[0]; y[7] = p3[1];
  }
};

// The scale byte of a block from the bits of its largest magnitude: the exponent of a float is its bits 23 up, so
// floor(log2) needs no logarithm; subnormal and zero magnitudes have the exponent field 0.  255: not finite.
template <class F>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const int e = (int)(top >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - F::kPower, 0);
}
// What takes the scale out of the elements, 2^(127 - byte): exact, but for results far below the smallest code.
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return byte == 255 ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// The block's largest magnitude (as bits, which order like the numbers, NaN above infinity) from 4 lanes' 8 elements.
__device__ __forceinline__ uint32_t mx_block_top(const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));    // quad_perm 1, 0, 3, 2
  return max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));   // quad_perm 2, 3, 0, 1
}

// Codes of a lane's 8 elements of a block, and its scale byte.
template <class F>
__device__ __forceinline__ typename F::Codes mx_encode(const float (&x)[8], uint32_t& byte) {
  byte = mx_scale_byte<F>(mx_block_top(x));
  const float inv = mx_inverse(byte);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = byte == 255 ? 0.f : x[e] * inv;
  return F::encode(y);
}

// Element types of rows: 8 consecutive elements from and to 16-byte aligned memory, one element.
struct RowBf16 {
  typedef uint16_t T;
  static constexpr int kDtype = SF_DTYPE_BF16;
  static __device__ __forceinline__ float load(const T* p) { return bf2f(*p); }
  static __device__ __forceinline__ void store(T* p, float v) { *p = f2bf(v); }
  static __device__ __forceinline__ float round(float v) { return bf2f(f2bf(v)); }
  static __device__ __forceinline__ void unpack(u32x4 w, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[2 * e] = bflo(w[e]); x[2 * e + 1] = bfhi(w[e]); }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[8]) {
    return u32x4{pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7])};
  }
};
struct RowFp16 {
  typedef uint16_t T;
  typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
  static constexpr int kDtype = SF_DTYPE_F16;
  static __device__ __forceinline__ float load(const T* p) { return (float)__builtin_bit_cast(_Float16, *p); }
  static __device__ __forceinline__ void store(T* p, float v) { *p = __builtin_bit_cast(uint16_t, (_Float16)v); }
  static __device__ __forceinline__ float round(float v) { return (float)(_Float16)v; }
  static __device__ __forceinline__ void unpack(u32x4 w, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = w[e];                               // (a bit cast of the element itself takes the vector's first bytes)
      const f16x2 p = __builtin_bit_cast(f16x2, u);
      x[2 * e] = (float)p[0];
      x[2 * e + 1] = (float)p[1];
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[2 * e], x[2 * e + 1]}, f16x2));
    return w;
  }
};
struct RowFp32 {
  typedef float T;
  static constexpr int kDtype = SF_DTYPE_F32;
  static __device__ __forceinline__ float load(const T* p) { return *p; }
  static __device__ __forceinline__ void store(T* p, float v) { *p = v; }
  static __device__ __forceinline__ float round(float v) { return v; }
};

// 8 elements as loaded, so that they wait for nothing until they are taken.
template <class E>
struct Raw8 {
  u32x4 w;
  __device__ __forceinline__ void load(const typename E::T* p) { w = ld16(p); }
  __device__ __forceinline__ void get(float (&x)[8]) const { E::unpack(w, x); }
  static __device__ __forceinline__ void store(typename E::T* p, const float (&x)[8]) { st16(p, E::pack(x)); }
};
template <>
struct Raw8<RowFp32> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const f32x4*>(p);
    b = *reinterpret_cast<const f32x4*>(p + 4);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
  }
  static __device__ __forceinline__ void store(float* p, const float (&x)[8]) {
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  }
};
