// Activation checkpoints in 8 bits (format in mx8.h) and back.
//
// One pass each way, HBM bound: a lane owns 16 values, half a block, so that its
// loads and its store of 16 bytes are as wide as they get; the block's largest
// magnitude takes one lane exchange. Powers of two as scales make the division
// exact: the one rounding is the value's, to e4m3 (nearest even,
// v_cvt_pk_fp8_f32), and a restored value is exact in bf16, fp16 and fp32 down to
// their least steps. 16,384 x 7,168 bf16: 75 us to 8 bits (356 MB, 4.7 TB/s), 66 back
// (5.4), where large copies run at 5.1 to 5.4.
//
// Infinities and NaN have no place in e4m3 but its NaN: they become NaN and do not
// count towards the block's scale. A value whose restored neighbour passes the
// output type's largest finite value (the nearest e4m3 to the top of fp16's or
// bf16's range does) is restored to that largest value.
#include <algorithm>

#include "mx8.h"

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

// A piece's values: n of them lie in the row (n < 16 only in a row's last block).
template <typename T, bool WIDE>
__device__ __forceinline__ void load_piece(const T* p, int n, T* v) {
  if (WIDE && n == kPiece) {
    const u32x4* s = reinterpret_cast<const u32x4*>(p);
    u32x4* d = reinterpret_cast<u32x4*>(v);
#pragma unroll
    for (int i = 0; i < int(kPiece * sizeof(T) / 16); ++i) d[i] = s[i];
  } else if (n == kPiece) {
    __builtin_memcpy(v, p, kPiece * sizeof(T));  // wide accesses at any alignment
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) v[i] = i < n ? p[i] : T(0);
  }
}
template <typename T, bool WIDE>
__device__ __forceinline__ void store_piece(T* p, int n, const T* v) {
  if (WIDE && n == kPiece) {
    const u32x4* s = reinterpret_cast<const u32x4*>(v);
    u32x4* d = reinterpret_cast<u32x4*>(p);
#pragma unroll
    for (int i = 0; i < int(kPiece * sizeof(T) / 16); ++i) d[i] = s[i];
  } else if (n == kPiece) {
    __builtin_memcpy(p, v, kPiece * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      if (i < n) p[i] = v[i];
  }
}

// Pieces are numbered row by row, two to a block, the last block's filled up.
// The rows' pieces are a grid-stride loop of pairs, so both lanes of a block are
// always in the same round.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
act_checkpoint_kernel(const T* __restrict__ x, int64_t ldx, int64_t M, int64_t K, int64_t row_pieces,
                      uint8_t* __restrict__ values, uint8_t* __restrict__ scales) {
  const int64_t total = M * row_pieces;
  for (int64_t q = int64_t(blockIdx.x) * kThreads + threadIdx.x; q < total; q += int64_t(gridDim.x) * kThreads) {
    const int64_t row = q / row_pieces, piece = q - row * row_pieces;
    const int64_t k0 = piece * kPiece;
    const int n = int(min(int64_t(kPiece), max(int64_t(0), K - k0)));
    __attribute__((aligned(16))) T v[kPiece];
    load_piece<T, WIDE>(x + row * ldx + k0, n, v);
    float f[kPiece], amax = 0.f;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      f[i] = val<T>::get(v[i]);
      const float a = fabsf(f[i]);
      amax = a <= 3.4028234663852886e38f ? fmaxf(amax, a) : amax;  // neither inf nor NaN
    }
    amax = fmaxf(amax, __shfl_xor(amax, 1));
    const uint32_t byte = mx8_scale_byte(amax);
    const float inv = mx8_inverse_scale(byte);
    __attribute__((aligned(16))) uint32_t w[kPiece / 4];
#pragma unroll
    for (int i = 0; i < kPiece / 4; ++i) {
      float s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = f[4 * i + j];
        s[j] = fabsf(a) <= 3.4028234663852886e38f ? a * inv : __builtin_nanf("");
      }
      int r = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
      w[i] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], r, true));
    }
    if (n > 0) store_piece<uint8_t, WIDE>(values + row * K + k0, n, reinterpret_cast<const uint8_t*>(w));
    if ((piece & 1) == 0) scales[row * (row_pieces / 2) + piece / 2] = uint8_t(byte);
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
act_restore_kernel(const uint8_t* __restrict__ values, const uint8_t* __restrict__ scales, int64_t M, int64_t K,
                   int64_t row_pieces, T* __restrict__ out) {
  const int64_t total = M * row_pieces;
  for (int64_t q = int64_t(blockIdx.x) * kThreads + threadIdx.x; q < total; q += int64_t(gridDim.x) * kThreads) {
    const int64_t row = q / row_pieces, piece = q - row * row_pieces;
    const int64_t k0 = piece * kPiece;
    const int n = int(min(int64_t(kPiece), K - k0));
    if (n <= 0) continue;
    __attribute__((aligned(16))) uint8_t b[kPiece];
    load_piece<uint8_t, WIDE>(values + row * K + k0, n, b);
    const float s = mx8_scale(scales[row * (row_pieces / 2) + piece / 2]);
    __attribute__((aligned(16))) T v[kPiece];
#pragma unroll
    for (int i = 0; i < kPiece / 4; ++i) {
      float f[4];
      mx8_unpack4(reinterpret_cast<const uint32_t*>(b)[i], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = f[j] * s;
        const float c = fminf(fmaxf(a, -val<T>::kMax), val<T>::kMax);
        v[4 * i + j] = val<T>::put(a == a ? c : a);
      }
    }
    store_piece<T, WIDE>(out + row * K + k0, n, v);
  }
}

int grid_for(int64_t pieces) { return int(std::min<int64_t>(cdiv(pieces, kThreads), 256 * 64)); }

template <typename T>
void checkpoint_typed(const void* x, int64_t ldx, int64_t M, int64_t K, uint8_t* values, uint8_t* scales,
                      hipStream_t stream) {
  const int64_t row_pieces = 2 * cdiv(K, kMx8Block);
  const bool wide = K % 16 == 0 && (ldx * sizeof(T)) % 16 == 0 &&
                    (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(values)) % 16 == 0;
  const dim3 grid(grid_for(M * row_pieces));
  const T* p = static_cast<const T*>(x);
  if (wide)
    hipLaunchKernelGGL((act_checkpoint_kernel<T, true>), grid, dim3(kThreads), 0, stream, p, ldx, M, K, row_pieces,
                       values, scales);
  else
    hipLaunchKernelGGL((act_checkpoint_kernel<T, false>), grid, dim3(kThreads), 0, stream, p, ldx, M, K, row_pieces,
                       values, scales);
}

template <typename T>
void restore_typed(const uint8_t* values, const uint8_t* scales, int64_t M, int64_t K, void* out,
                   hipStream_t stream) {
  const int64_t row_pieces = 2 * cdiv(K, kMx8Block);
  const bool wide =
      K % 16 == 0 && (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(values)) % 16 == 0;
  const dim3 grid(grid_for(M * row_pieces));
  T* p = static_cast<T*>(out);
  if (wide)
    hipLaunchKernelGGL((act_restore_kernel<T, true>), grid, dim3(kThreads), 0, stream, values, scales, M, K,
                       row_pieces, p);
  else
    hipLaunchKernelGGL((act_restore_kernel<T, false>), grid, dim3(kThreads), 0, stream, values, scales, M, K,
                       row_pieces, p);
}

}  // namespace

int launch_act_checkpoint(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* values,
                          uint8_t* scales, hipStream_t stream) {
  if (dtype == XK_DT_BF16) checkpoint_typed<uint16_t>(x, ldx, M, K, values, scales, stream);
  else if (dtype == XK_DT_FP16) checkpoint_typed<_Float16>(x, ldx, M, K, values, scales, stream);
  else checkpoint_typed<float>(x, ldx, M, K, values, scales, stream);
  XK_CHECK_LAUNCH("act_checkpoint");
  return XK_OK;
}

int launch_act_restore(const uint8_t* values, const uint8_t* scales, int64_t M, int64_t K, int dtype, void* out,
                       hipStream_t stream) {
  if (dtype == XK_DT_BF16) restore_typed<uint16_t>(values, scales, M, K, out, stream);
  else if (dtype == XK_DT_FP16) restore_typed<_Float16>(values, scales, M, K, out, stream);
  else restore_typed<float>(values, scales, M, K, out, stream);
  XK_CHECK_LAUNCH("act_restore");
  return XK_OK;
}

}  // namespace xk
