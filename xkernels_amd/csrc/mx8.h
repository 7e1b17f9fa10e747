// Activations held in 8 bits: e4m3 values [M, K] (bytes) with one e8m0 byte for
// each block of 32 along a row, value = e4m3 * 2^(byte - 127).
#pragma once

#include "common.h"

namespace xk {

constexpr int kMx8Block = 32;

// The e8m0 byte of a block: the least exponent e in [-127, 127] with
// amax * 2^-e <= 448 = 1.75 * 2^8, from amax = 1.f * 2^(E-127): e = E - 135, one
// more where 1.f > 1.75. An amax of 0 or up to 1.75 * 2^-119 gives byte 0.
__device__ __forceinline__ uint32_t mx8_scale_byte(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int byte = int(b >> 23) - 8 + int((b & 0x7FFFFFu) > 0x600000u);
  return uint32_t(byte < 0 ? 0 : byte);
}

// 2^(byte - 127); byte 0 is the denormal 2^-127, byte 255 (which no checkpoint
// holds) NaN.
__device__ __forceinline__ float mx8_scale(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255u ? 0x7FC00000u : byte << 23);
}
// 2^(127 - byte) for byte <= 247 (the largest that mx8_scale_byte gives): a normal number.
__device__ __forceinline__ float mx8_inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// 4 values (unscaled) of a word, lowest byte first.
__device__ __forceinline__ void mx8_unpack4(uint32_t w, float* v) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
  v[0] = a[0];
  v[1] = a[1];
  v[2] = b[0];
  v[3] = b[1];
}

// The least byte with which an e4m3 value can pass the largest finite value of bf16 and
// fp32 (448 * 2^119 does not, 256 * 2^120 does).
constexpr uint32_t kMx8Top = 247;

// 8 scaled values of two words. bf16: v_cvt_scalef32_pk_bf16_fp8, which applies the
// exponent field of its scale operand (byte 0: 2^-127); a reserved byte 255 makes
// every value NaN first. A value past the type's range becomes its largest finite one, as
// act_restore has it; e4m3 has no infinity, so an infinity here is such a value.
__device__ __forceinline__ void mx8_unpack8(uint32_t w0, uint32_t w1, uint32_t byte, float* v) {
  const float s = mx8_scale(byte);
  mx8_unpack4(w0, v);
  mx8_unpack4(w1, v + 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= s;
  if (byte >= kMx8Top) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(v[i]) == __builtin_inff()) v[i] = copysignf(3.4028234663852886e38f, v[i]);
  }
}
__device__ __forceinline__ void mx8_unpack8(uint32_t w0, uint32_t w1, uint32_t byte, uint16_t* v) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  if (byte == 255u) w0 = w1 = 0x7F7F7F7Fu;
  const float s = __uint_as_float((byte == 255u ? 127u : byte) << 23);
  b2* o = reinterpret_cast<b2*>(v);
  o[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false);
  o[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
  o[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false);
  o[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
  if (byte >= kMx8Top) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((v[i] & 0x7FFFu) == 0x7F80u) --v[i];
  }
}

}  // namespace xk
