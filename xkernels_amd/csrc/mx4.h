// Values in MXFP4: e2m1 codes, two a byte (the lower k in the low half), with one e8m0
// byte for each block of 32 along a row, value = e2m1 * 2^(byte - 127). A row of K
// values is ceil(K / 32) whole blocks of 16 bytes, the last one filled up with zeros.
#pragma once

#include "common.h"

namespace xk {

constexpr int kMx4Block = 32;
constexpr uint32_t kMx4Nan = 255;  // e8m0's NaN: the whole block

// The e8m0 byte of a block: the least exponent e in [-127, 127] with amax * 2^-e <= 6 =
// 1.5 * 2^2, from amax = 1.f * 2^(E-127): e = E - 129, one more where 1.f > 1.5. An
// amax of 0 or up to 1.5 * 2^-125 gives byte 0; the largest finite one gives 253. An infinity
// or a NaN, which e2m1 cannot hold, makes the block NaN.
__device__ __forceinline__ uint32_t mx4_scale_byte(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b >= 0x7F800000u) return kMx4Nan;
  const int byte = int(b >> 23) - 2 + int((b & 0x7FFFFFu) > 0x400000u);
  return uint32_t(byte < 0 ? 0 : byte);
}
// 2^(127 - byte) for byte <= 253: a normal number. (A NaN block's codes are zeros.)
__device__ __forceinline__ float mx4_inverse_scale(uint32_t byte) {
  return byte == kMx4Nan ? 0.f : __uint_as_float((254u - byte) << 23);
}
// 2^(byte - 127)
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == kMx4Nan ? 0x7FC00000u : byte << 23);
}

// 8 values of magnitude <= 6 to the nearest codes (ties to the even one), lowest nibble first.
__device__ __forceinline__ uint32_t mx4_pack8(const float* v) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.0f, 3);
}
__device__ __forceinline__ void mx4_unpack8(uint32_t w, float* v) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
           c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
  v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
}

// Rows of `from` scales that are to lie `to` apart, filled up with 127 (no rows: nothing to do).
struct ScaleRows {
  const uint8_t* src = nullptr;
  uint8_t* dst = nullptr;
  int64_t rows = 0, from = 0, to = 0;
};

// Codes and scales (rows lds apart, filled up with 127) of x; in the same launch scales of another
// operand are widened.
int launch_mxfp4_quantize(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales,
                          int64_t lds, const ScaleRows& wide, hipStream_t stream);
int launch_mxfp4_widen(const ScaleRows& a, const ScaleRows& b, hipStream_t stream);

}  // namespace xk
