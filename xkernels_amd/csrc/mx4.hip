// Values to MXFP4 (format in mx4.h) and back.
//
// One pass each way, HBM bound: a lane owns half a block, 16 values, whose loads are 16
// bytes each; the block's largest magnitude takes one lane exchange. A power of two as
// scale makes the division exact, so the one rounding is the value's, to e2m1.
#include <algorithm>

#include "mx4.h"

namespace xk {
namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 16;  // values a lane owns

template <typename T> struct val;
template <> struct val<uint16_t> {
  __device__ __forceinline__ static float get(uint16_t b) { return bf16_to_f32(b); }
  __device__ __forceinline__ static uint16_t put(float f) { return f32_to_bf16(f); }
  static constexpr float kMax = 3.3895313892515355e38f;
};
template <> struct val<_Float16> {
  __device__ __forceinline__ static float get(_Float16 h) { return float(h); }
  __device__ __forceinline__ static _Float16 put(float f) { return _Float16(f); }
  static constexpr float kMax = 65504.f;
};
template <> struct val<float> {
  __device__ __forceinline__ static float get(float f) { return f; }
  __device__ __forceinline__ static float put(float f) { return f; }
  static constexpr float kMax = 3.4028234663852886e38f;
};

// A lane's values; n of them lie in the row (fewer than 16, also none, in a row's last block).
template <typename T> __device__ __forceinline__ void load_piece(const T* p, int n, T* v) {
  if (n >= kPiece) {
    __builtin_memcpy(v, p, kPiece * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) v[i] = i < n ? p[i] : T(0);
  }
}
template <typename T> __device__ __forceinline__ void store_piece(T* p, int n, const T* v) {
  if (n >= kPiece) {
    __builtin_memcpy(p, v, kPiece * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      if (i < n) p[i] = v[i];
  }
}

// Half blocks are numbered row by row: both lanes of a block are always in the same round.
// The scales' rows lie lds apart, the places behind the row's blocks are filled with 127.
template <typename T>
__global__ void __launch_bounds__(kThreads)
mx4_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t M, int64_t K, int64_t blocks,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t lds) {
  const int64_t halves = 2 * blocks, total = M * halves;
  for (int64_t q = int64_t(blockIdx.x) * kThreads + threadIdx.x; q < total; q += int64_t(gridDim.x) * kThreads) {
    const int64_t row = q / halves, half = q - row * halves;
    const int64_t k0 = half * kPiece;
    const int n = int(min(int64_t(kPiece), max(int64_t(0), K - k0)));
    __attribute__((aligned(16))) T v[kPiece];
    load_piece(x + row * ldx + k0, n, v);
    float f[kPiece];
    uint32_t top = 0;  // the largest magnitude as bits: infinities and NaN are above all numbers
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      f[i] = val<T>::get(v[i]);
      top = max(top, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    }
    top = max(top, uint32_t(__shfl_xor(int(top), 1)));
    const uint32_t byte = mx4_scale_byte(__uint_as_float(top));
    const float inv = mx4_inverse_scale(byte);
#pragma unroll
    for (int i = 0; i < kPiece; ++i) f[i] = byte == kMx4Nan ? 0.f : f[i] * inv;
    uint32_t w[2] = {mx4_pack8(f), mx4_pack8(f + 8)};
    __builtin_memcpy(codes + q * 8, w, 8);
    if ((half & 1) == 0) scales[row * lds + half / 2] = uint8_t(byte);
    if (half == halves - 1)
      for (int64_t b = blocks; b < lds; ++b) scales[row * lds + b] = 127;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
mx4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t M, int64_t K,
                      int64_t blocks, T* __restrict__ out) {
  const int64_t halves = 2 * blocks, total = M * halves;
  for (int64_t q = int64_t(blockIdx.x) * kThreads + threadIdx.x; q < total; q += int64_t(gridDim.x) * kThreads) {
    const int64_t row = q / halves, half = q - row * halves;
    const int64_t k0 = half * kPiece;
    const int n = int(min(int64_t(kPiece), K - k0));
    if (n <= 0) continue;
    uint32_t w[2];
    __builtin_memcpy(w, codes + q * 8, 8);
    const float s = mx4_scale(scales[row * blocks + half / 2]);
    float f[kPiece];
    mx4_unpack8(w[0], f);
    mx4_unpack8(w[1], f + 8);
    __attribute__((aligned(16))) T v[kPiece];
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      const float a = f[i] * s;
      const float c = fminf(fmaxf(a, -val<T>::kMax), val<T>::kMax);
      v[i] = val<T>::put(a == a ? c : a);
    }
    store_piece(out + row * K + k0, n, v);
  }
}

int grid_for(int64_t pieces) { return int(std::min<int64_t>(cdiv(pieces, kThreads), 256 * 64)); }

template <typename T>
void quantize_typed(const void* x, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales, int64_t lds,
                    hipStream_t stream) {
  const int64_t blocks = cdiv(K, kMx4Block);
  hipLaunchKernelGGL((mx4_quantize_kernel<T>), dim3(grid_for(M * 2 * blocks)), dim3(kThreads), 0, stream,
                     static_cast<const T*>(x), ldx, M, K, blocks, codes, scales, lds);
}

template <typename T>
void dequantize_typed(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out,
                      hipStream_t stream) {
  const int64_t blocks = cdiv(K, kMx4Block);
  hipLaunchKernelGGL((mx4_dequantize_kernel<T>), dim3(grid_for(M * 2 * blocks)), dim3(kThreads), 0, stream, codes,
                     scales, M, K, blocks, static_cast<T*>(out));
}

}  // namespace

int launch_mxfp4_quantize(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales,
                          int64_t lds, hipStream_t stream) {
  if (dtype == XK_DT_BF16) quantize_typed<uint16_t>(x, ldx, M, K, codes, scales, lds, stream);
  else if (dtype == XK_DT_FP16) quantize_typed<_Float16>(x, ldx, M, K, codes, scales, lds, stream);
  else quantize_typed<float>(x, ldx, M, K, codes, scales, lds, stream);
  XK_CHECK_LAUNCH("mxfp4_quantize");
  return XK_OK;
}

int launch_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, int dtype, void* out,
                            hipStream_t stream) {
  if (dtype == XK_DT_BF16) dequantize_typed<uint16_t>(codes, scales, M, K, out, stream);
  else if (dtype == XK_DT_FP16) dequantize_typed<_Float16>(codes, scales, M, K, out, stream);
  else dequantize_typed<float>(codes, scales, M, K, out, stream);
  XK_CHECK_LAUNCH("mxfp4_dequantize");
  return XK_OK;
}

}  // namespace xk
