// Values to MXFP4 (format in mx4.h) and back.
//
// One pass each way, HBM bound. To 4 bits a lane owns half a block, 16 values, whose loads are 16
// bytes each; the block's largest magnitude takes one lane exchange. Back, a lane owns 16
// bytes of the result, so that a wave's stores are one run of 1 KB. A power of two as scale
// makes the division exact, so the one rounding is the value's, to e2m1. Rows are told apart by
// a division a lane, which whole blocks in rows without a gap do not need. 16,384 x 7,168 bf16: 69 us to
// 4 bits (297 MB), 50 back, 119 together (5.0 TB/s; a large copy runs at 5.2).
#include <algorithm>
#include <type_traits>

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
// Scales in rows of `to`, filled up with 127, from rows of `from` (see launch_mxfp4_quantize).
__device__ __forceinline__ void widen(const ScaleRows& w, int64_t first, int64_t step) {
  for (int64_t q = first; q < w.rows * w.to; q += step) {
    const int64_t row = q / w.to, b = q - row * w.to;
    w.dst[q] = b < w.from ? w.src[row * w.from + b] : 127;
  }
}

__global__ void __launch_bounds__(kThreads) mx4_widen_kernel(ScaleRows a, ScaleRows b) {
  const int64_t first = int64_t(blockIdx.x) * kThreads + threadIdx.x, step = int64_t(gridDim.x) * kThreads;
  widen(a, first, step);
  widen(b, first, step);
}

// Half blocks are numbered row by row: both lanes of a block are always in the same round.
// The scales' rows lie lds apart, the places behind the row's blocks are filled with 127. FLAT: rows
// without a gap of whole blocks, one after the other. There are fewer than 2^31.
// Workgroups from `own` on widen other scales.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(kThreads)
mx4_quantize_kernel(const T* __restrict__ x, int64_t ldx, uint32_t total, int64_t K, uint32_t halves,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t lds, int own, ScaleRows wide) {
  if (int(blockIdx.x) >= own) {
    widen(wide, int64_t(blockIdx.x - own) * kThreads + threadIdx.x, int64_t(gridDim.x - own) * kThreads);
    return;
  }
  for (uint32_t q = blockIdx.x * kThreads + threadIdx.x; q < total; q += uint32_t(own) * kThreads) {
    const uint32_t r = FLAT ? 0 : q / halves, half = q - r * halves;
    const int64_t row = r;
    const int64_t k0 = int64_t(half) * kPiece;
    const int n = FLAT ? kPiece : int(min(int64_t(kPiece), max(int64_t(0), K - k0)));
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
    __builtin_memcpy(codes + int64_t(q) * 8, w, 8);
    if ((half & 1) == 0) scales[row * lds + half / 2] = uint8_t(byte);
    if (!FLAT && half == halves - 1)
      for (int64_t b = halves / 2; b < lds; ++b) scales[row * lds + b] = 127;
  }
}

template <typename T, bool FLAT>
__global__ void __launch_bounds__(kThreads)
mx4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t total, int64_t K,
                      uint32_t pieces, T* __restrict__ out) {
  constexpr int PER = 16 / sizeof(T);  // values of a lane
  typedef std::conditional_t<PER == 8, uint32_t, uint16_t> W;
  for (uint32_t q = blockIdx.x * kThreads + threadIdx.x; q < total; q += gridDim.x * kThreads) {
    const uint32_t r = FLAT ? 0 : q / pieces, piece = q - r * pieces;
    const int64_t row = r;
    const int64_t k0 = int64_t(piece) * PER;
    const int n = FLAT ? PER : int(min(int64_t(PER), K - k0));
    if (n <= 0) continue;
    const uint32_t w = load_unaligned<W>(codes + int64_t(q) * (PER / 2));
    const float s = mx4_scale(scales[q / (kMx4Block / PER)]);
    float f[8];
    mx4_unpack8(w, f);
    __attribute__((aligned(16))) T v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float a = f[i] * s;
      const float c = fminf(fmaxf(a, -val<T>::kMax), val<T>::kMax);
      v[i] = val<T>::put(a == a ? c : a);
    }
    T* to = out + row * K + k0;
    if (n == PER) {
      __builtin_memcpy(to, v, 16);
    } else {
#pragma unroll
      for (int i = 0; i < PER - 1; ++i)
        if (i < n) to[i] = v[i];
    }
  }
}

int grid_for(int64_t pieces) { return int(std::min<int64_t>(cdiv(pieces, kThreads), 256 * 64)); }

template <typename T>
void quantize_typed(const void* x, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales, int64_t lds,
                    const ScaleRows& wide, hipStream_t stream) {
  const int64_t blocks = cdiv(K, kMx4Block), total = M * 2 * blocks;
  const int own = grid_for(total), more = wide.rows > 0 ? grid_for(cdiv(wide.rows * wide.to, 8)) : 0;
  const dim3 grid(own + more), block(kThreads);
  const T* p = static_cast<const T*>(x);
  const bool flat = K % kMx4Block == 0 && (ldx == K || M == 1) && lds == blocks;
  if (flat)
    hipLaunchKernelGGL((mx4_quantize_kernel<T, true>), grid, block, 0, stream, p, ldx, uint32_t(total), K,
                       uint32_t(2 * blocks), codes, scales, lds, own, wide);
  else
    hipLaunchKernelGGL((mx4_quantize_kernel<T, false>), grid, block, 0, stream, p, ldx, uint32_t(total), K,
                       uint32_t(2 * blocks), codes, scales, lds, own, wide);
}

template <typename T>
void dequantize_typed(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out,
                      hipStream_t stream) {
  const int64_t pieces = cdiv(K, kMx4Block) * kMx4Block / (16 / int64_t(sizeof(T))), total = M * pieces;
  const dim3 grid(grid_for(total)), block(kThreads);
  T* to = static_cast<T*>(out);
  if (K % kMx4Block == 0)
    hipLaunchKernelGGL((mx4_dequantize_kernel<T, true>), grid, block, 0, stream, codes, scales, uint32_t(total), K,
                       uint32_t(pieces), to);
  else
    hipLaunchKernelGGL((mx4_dequantize_kernel<T, false>), grid, block, 0, stream, codes, scales, uint32_t(total), K,
                       uint32_t(pieces), to);
}

}  // namespace

int launch_mxfp4_quantize(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales,
                          int64_t lds, const ScaleRows& wide, hipStream_t stream) {
  if (dtype == XK_DT_BF16) quantize_typed<uint16_t>(x, ldx, M, K, codes, scales, lds, wide, stream);
  else if (dtype == XK_DT_FP16) quantize_typed<_Float16>(x, ldx, M, K, codes, scales, lds, wide, stream);
  else quantize_typed<float>(x, ldx, M, K, codes, scales, lds, wide, stream);
  XK_CHECK_LAUNCH("mxfp4_quantize");
  return XK_OK;
}

int launch_mxfp4_widen(const ScaleRows& a, const ScaleRows& b, hipStream_t stream) {
  if (a.rows + b.rows == 0) return XK_OK;
  const int64_t pieces = cdiv(std::max(a.rows * a.to, b.rows * b.to), 8);
  hipLaunchKernelGGL(mx4_widen_kernel, dim3(grid_for(pieces)), dim3(kThreads), 0, stream, a, b);
  XK_CHECK_LAUNCH("mxfp4_widen");
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
