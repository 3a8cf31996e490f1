// 8-bit activations: what a forward pass keeps of a row tensor for its backward pass.
//
// A block is 32 consecutive channels of a row (the last block of a row may be shorter). With a the
// largest finite |x| of the block and s the least whole number >= -126 with a <= 448 2^s, value x is
// kept as the e4m3 code of x / 2^s (nearest, halves to even; 448 is e4m3's largest number, so no code
// overflows) and read back as code * 2^s. The scale is the byte s + 127, the exponent field of 2^s as
// fp32, so both directions multiply by an exact power of two. NaN and infinities become NaN. Finite values
// from 1.9375 * 2^127 on, at the end of the types' range, are nearest to 256 * 2^120 and read back as infinities.
#pragma once

#include "ffk_device.h"

namespace ffk {

constexpr int kActBlock = 32;

// |v| where v is finite, else 0.
__device__ __forceinline__ float finite_abs(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
  return __uint_as_float(u < 0x7f800000u ? u : 0u);
}

// The scale byte of a block whose largest finite magnitude is top: 448 = 1.75 * 2^8, so the exponent
// field of top less 8, one more where its mantissa is past 1.75.
__device__ __forceinline__ uint32_t act_scale(float top) {
  const uint32_t u = __float_as_uint(top);
  const int byte = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(byte < 1 ? 1 : byte);
}
// 2^s and 2^-s of a scale byte in [1, 247].
__device__ __forceinline__ float act_unit(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float act_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ float lanes_max4(float v) {
  v = fmaxf(v, dpp_f<kDppXor1>(v));
  return fmaxf(v, dpp_f<kDppXor2>(v));
}
// Largest of a block's lanes: 32 / VE lanes of VE values each (every lane gets it).
template <int VE>
__device__ __forceinline__ float block_max(float v) {
  static_assert(VE == 1 || VE == 4 || VE == 8, "values a lane holds of a block");
  v = lanes_max4(v);
  if constexpr (VE <= 4) v = fmaxf(v, dpp_f<kDppHalfMirror>(v));
  if constexpr (VE == 1) {
    v = fmaxf(v, dpp_f<kDppMirror>(v));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// Four values times inv as e4m3 codes, value 0 in the low byte.
__device__ __forceinline__ uint32_t act_code4(float a, float b, float c, float d, float inv) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  p = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, p, true);
  return (uint32_t)p;
}
// The four values of a word of codes.
__device__ __forceinline__ void act_value4(uint32_t codes, float unit, float* v) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  v[0] = lo[0] * unit;
  v[1] = lo[1] * unit;
  v[2] = hi[0] * unit;
  v[3] = hi[1] * unit;
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// VE consecutive channels of a kept row as a lane holds them, VE = 8 or 4 (16 bytes of T) or 1:
// of the tensor itself (CODES false) or of an 8-bit activation.
template <typename T, bool CODES, int VE>
struct KeptPiece;

template <typename T, int VE>
struct KeptPiece<T, false, VE> {
  typedef T vec __attribute__((__vector_size__(VE * sizeof(T))));
  vec v;
  // row: the row's index; c: the piece's first channel
  __device__ __forceinline__ void load(const void* x, const uint8_t*, int64_t row, int c, int cols, int) {
    v = *reinterpret_cast<const vec*>(static_cast<const T*>(x) + row * cols + c);
  }
  __device__ __forceinline__ void values(float* o) const {
#pragma unroll
    for (int e = 0; e < VE; ++e) o[e] = (float)v[e];
  }
};
template <typename T>
struct KeptPiece<T, false, 1> {
  T v;
  __device__ __forceinline__ void load(const void* x, const uint8_t*, int64_t row, int c, int cols, int) {
    v = static_cast<const T*>(x)[row * cols + c];
  }
  __device__ __forceinline__ void values(float* o) const { o[0] = (float)v; }
};
template <typename T, int VE>
struct KeptPiece<T, true, VE> {
  uint32_t v[VE / 4];
  uint8_t scale;
  __device__ __forceinline__ void load(const void* x, const uint8_t* scales, int64_t row, int c, int cols,
                                       int blocks) {
    const uint8_t* p = static_cast<const uint8_t*>(x) + row * cols + c;
    if constexpr (VE == 8) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(p);
      v[0] = w[0];
      v[1] = w[1];
    } else {
      v[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    scale = scales[row * blocks + c / kActBlock];
  }
  __device__ __forceinline__ void values(float* o) const {
#pragma unroll
    for (int e = 0; e < VE / 4; ++e) act_value4(v[e], act_unit(scale), o + 4 * e);
  }
};
template <typename T>
struct KeptPiece<T, true, 1> {
  uint8_t v, scale;
  __device__ __forceinline__ void load(const void* x, const uint8_t* scales, int64_t row, int c, int cols,
                                       int blocks) {
    v = static_cast<const uint8_t*>(x)[row * cols + c];
    scale = scales[row * blocks + c / kActBlock];
  }
  __device__ __forceinline__ void values(float* o) const {
    o[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false)[0] * act_unit(scale);
  }
};

// VE fp32 values of a lane as the block's codes: every lane of the block calls it together; valid is
// false for the lanes past the end of the row. The block's first lane writes the scale.
template <int VE>
__device__ __forceinline__ void act_store(const float* v, bool valid, bool first, uint8_t* codes, uint8_t* scale) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < VE; ++e) top = fmaxf(top, valid ? finite_abs(v[e]) : 0.f);
  const uint32_t byte = act_scale(block_max<VE>(top));
  const float inv = act_inverse(byte);
  if (!valid) return;
  if constexpr (VE == 8) {
    u32x2 w;
    w[0] = act_code4(v[0], v[1], v[2], v[3], inv);
    w[1] = act_code4(v[4], v[5], v[6], v[7], inv);
    __builtin_nontemporal_store(w, reinterpret_cast<u32x2*>(codes));
  } else if constexpr (VE == 4) {
    __builtin_nontemporal_store(act_code4(v[0], v[1], v[2], v[3], inv), reinterpret_cast<uint32_t*>(codes));
  } else {
    *codes = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, 0.f, 0, false) & 0xff);
  }
  if (first) *scale = (uint8_t)byte;
}

}  // namespace ffk
