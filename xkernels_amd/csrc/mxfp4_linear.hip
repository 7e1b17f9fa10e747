// The product of two MXFP4 operands: out[m, n] = sum over blocks b of 2^(sx + sw) times the
// block's sum of e2m1 products (+ bias[n]), in fp32 on the scaled matrix instructions,
// rounded once. Activations that come in 16 or 32 bits are quantised first, in a pass
// of their own.
#include <algorithm>

#include "dense_tile.h"
#include "mx4.h"

namespace xk {

int launch_mxfp4_quantize(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales,
                          int64_t lds, hipStream_t stream);

namespace {

using namespace dense;

int64_t pad4(int64_t n) { return (n + 3) & ~int64_t(3); }
int64_t aligned(int64_t bytes) { return (bytes + 255) & ~int64_t(255); }

template <typename T> struct val;
template <> struct val<uint16_t> {
  __device__ __forceinline__ static float get(uint16_t b) { return bf16_to_f32(b); }
  __device__ __forceinline__ static uint16_t put(float f) { return f32_to_bf16(f); }
};
template <> struct val<_Float16> {
  __device__ __forceinline__ static float get(_Float16 h) { return float(h); }
  __device__ __forceinline__ static _Float16 put(float f) { return _Float16(f); }
};
template <> struct val<float> {
  __device__ __forceinline__ static float get(float f) { return f; }
  __device__ __forceinline__ static float put(float f) { return f; }
};

template <typename T> struct Store {
  T* out;
  const T* bias;
  int64_t M, N;
  template <int WT, int XT>
  __device__ __forceinline__ void operator()(const f32x4 (&acc)[WT][XT], int64_t m, int64_t n, int lane) const {
    struct four { T v[4]; };
    n += (lane >> 4) * 4;
#pragma unroll
    for (int a = 0; a < WT; ++a) {
      const int64_t left = N - n - a * 16;
      float add[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) add[i] = bias != nullptr && i < left ? val<T>::get(bias[n + a * 16 + i]) : 0.f;
#pragma unroll
      for (int b = 0; b < XT; ++b) {
        const int64_t row = m + b * 16 + (lane & 15);
        if (row >= M) continue;
        T* to = out + row * N + n + a * 16;
        four v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v.v[i] = val<T>::put(acc[a][b][i] + add[i]);
        if (left >= 4) {
          store_unaligned(to, v);
        } else {
#pragma unroll
          for (int i = 0; i < 3; ++i)
            if (i < left) to[i] = v.v[i];
        }
      }
    }
  }
};

// Scales whose rows do not start at 4 bytes, in rows that do.
__global__ void __launch_bounds__(256)
pad_scales(const uint8_t* __restrict__ src, int64_t rows, int64_t blocks, int64_t lds, uint8_t* __restrict__ dst) {
  const int64_t total = rows * lds;
  for (int64_t q = int64_t(blockIdx.x) * 256 + threadIdx.x; q < total; q += int64_t(gridDim.x) * 256) {
    const int64_t row = q / lds, b = q - row * lds;
    dst[q] = b < blocks ? src[row * blocks + b] : 127;
  }
}

const uint8_t* take_scales(const uint8_t* s, int64_t rows, int64_t blocks, char*& ws, hipStream_t stream) {
  const int64_t lds = pad4(blocks);
  if (lds == blocks) return s;
  uint8_t* to = reinterpret_cast<uint8_t*>(ws);
  ws += aligned(rows * lds);
  const int grid = int(std::min<int64_t>(cdiv(rows * lds, 256), 256 * 32));
  hipLaunchKernelGGL(pad_scales, dim3(grid), dim3(256), 0, stream, s, rows, blocks, lds, to);
  return to;
}

template <typename T>
void typed(const Product& p, const void* bias, void* out, hipStream_t stream) {
  launch_tile<Form::kFp4, Lay::kRowsOfK, Lay::kRowsOfK, 128, 128, 64, 64, false>(
      p, Store<T>{static_cast<T*>(out), static_cast<const T*>(bias), p.M, p.N}, stream);
}

}  // namespace

int64_t mxfp4_linear_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  const int64_t blocks = cdiv(K, kMx4Block), lds = pad4(blocks);
  return aligned(M * blocks * 16) + aligned(M * lds) + (lds == blocks ? 0 : aligned(N * lds));
}

int launch_mxfp4_linear(const void* x, int dtype, int64_t ldx, const uint8_t* x_scales, int64_t M, int64_t K,
                        const uint8_t* codes, const uint8_t* scales, int64_t N, const void* bias, void* out,
                        int out_dtype, void* workspace, hipStream_t stream) {
  const int64_t blocks = cdiv(K, kMx4Block), lds = pad4(blocks);
  char* ws = static_cast<char*>(workspace);
  const uint8_t *xc = static_cast<const uint8_t*>(x), *xs;
  if (x_scales == nullptr) {
    uint8_t* c = reinterpret_cast<uint8_t*>(ws);
    ws += aligned(M * blocks * 16);
    uint8_t* s = reinterpret_cast<uint8_t*>(ws);
    ws += aligned(M * lds);
    if (int rc = launch_mxfp4_quantize(x, dtype, ldx, M, K, c, s, lds, stream)) return rc;
    xc = c;
    xs = s;
  } else {
    xs = take_scales(x_scales, M, blocks, ws, stream);
  }
  const uint8_t* wsc = take_scales(scales, N, blocks, ws, stream);
  Product p{};
  p.x = Side{reinterpret_cast<const char*>(xc), blocks * 16, M, xs, lds};
  p.w = Side{reinterpret_cast<const char*>(codes), blocks * 16, N, wsc, lds};
  p.M = M;
  p.N = N;
  p.k_bytes = blocks * 16;
  p.blocks = blocks;
  p.chunks = int(cdiv(blocks, 8));
  if (out_dtype == XK_DT_BF16) typed<uint16_t>(p, bias, out, stream);
  else if (out_dtype == XK_DT_FP16) typed<_Float16>(p, bias, out, stream);
  else typed<float>(p, bias, out, stream);
  XK_CHECK_LAUNCH("mxfp4_linear");
  return XK_OK;
}

}  // namespace xk
