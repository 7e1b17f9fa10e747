// The product of two MXFP4 operands: out[m, n] = sum over blocks b of 2^(sx + sw) times the
// block's sum of e2m1 products (+ bias[n]), in fp32 on the scaled matrix instructions,
// rounded once. Up to 16 rows are one launch, which quantises activations in 16 or 32 bits as it
// reads them; of more rows they are quantised first, in a pass of their own: tiles that did it would
// read four times the bytes, once for every column of tiles.
//
// bf16 in and out, the quantising pass included: one row 7168 -> 4096 8.4 us (its launch; 16 MB), 4,096 rows
// 73 to 78 (3.1 to 3.3 PFLOP/s; the way from L2 to LDS: the scales leave X two places there, as W has, so a
// chunk's barrier waits for every load, and the matrix unit is busy half the time), 16,384 rows 2048 -> 7168
// 171 to 178 (2.8; tiles of 8 chunks, 235 MB of results).
#include <algorithm>

#include "dense_rows.h"

namespace xk {

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

template <typename T, bool BIAS> struct Store {
  static constexpr bool kFetches = BIAS;
  T* out;
  const T* bias;
  int64_t N;
  struct Spot {
    T* out;
    const T* bias;
    int ld, left;  // columns from the spot on
    template <bool WHOLE> __device__ __forceinline__ f32x4 fetch(int, int col) const {
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = WHOLE || col + i < left ? val<T>::get(bias[col + i]) : 0.f;
      return v;
    }
    template <bool WHOLE> __device__ __forceinline__ void put(int row, int col, f32x4 sum, f32x4 add = {}) const {
      struct four { T v[4]; } v;
      T* to = out + uint32_t(row * ld + col);
#pragma unroll
      for (int i = 0; i < 4; ++i) v.v[i] = val<T>::put(BIAS ? sum[i] + add[i] : sum[i]);
      if (WHOLE || left - col >= 4) {
        store_unaligned(to, v);
      } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (col + i < left) to[i] = v.v[i];
      }
    }
  };
  __device__ __forceinline__ Spot spot(int64_t m, int64_t n) const {
    return Spot{out + m * N + n, bias + n, int(N), int(N - n)};
  }
};

// Scales whose rows do not start at 4 bytes lie in rows that do (`rows` says which those are to be).
const uint8_t* take_scales(const uint8_t* s, int64_t n, int64_t blocks, char*& ws, ScaleRows& rows) {
  const int64_t lds = pad4(blocks);
  if (lds == blocks) return s;
  rows = ScaleRows{s, reinterpret_cast<uint8_t*>(ws), n, blocks, lds};
  ws += aligned(n * lds);
  return rows.dst;
}

struct Call {
  const void* x;
  int dtype;
  int64_t ldx;
  const uint8_t* x_scales;
  int64_t M, K;
  const uint8_t *codes, *scales;
  int64_t N;
};

template <typename EPI> int cut(const Call& c, const EPI& store, char* ws, hipStream_t stream) {
  const int64_t blocks = cdiv(c.K, kMx4Block), lds = pad4(blocks);
  const char* codes = reinterpret_cast<const char*>(c.codes);
  if (c.M <= kFewRows) {
    const Rows w{codes, blocks * 16, c.N, c.scales, blocks};
    const Rows x{static_cast<const char*>(c.x), c.x_scales ? blocks * 16 : c.ldx * (c.dtype == XK_DT_FP32 ? 4 : 2), c.M,
                 c.x_scales, blocks};
    if (c.x_scales != nullptr)
      launch_rows<Form::kFp4, void, false>(x, w, c.M, c.N, blocks, 0, store, stream);
    else if (c.dtype == XK_DT_BF16)
      launch_rows<Form::kFp4, uint16_t, false>(x, w, c.M, c.N, blocks, c.K, store, stream);
    else if (c.dtype == XK_DT_FP16)
      launch_rows<Form::kFp4, _Float16, false>(x, w, c.M, c.N, blocks, c.K, store, stream);
    else
      launch_rows<Form::kFp4, float, false>(x, w, c.M, c.N, blocks, c.K, store, stream);
    return XK_OK;
  }
  const char* xc = static_cast<const char*>(c.x);
  const uint8_t* xs;
  ScaleRows wide, x_wide;
  const uint8_t* wsc = take_scales(c.scales, c.N, blocks, ws, wide);
  int rc;
  if (c.x_scales == nullptr) {
    uint8_t* to = reinterpret_cast<uint8_t*>(ws);
    ws += aligned(c.M * blocks * 16);
    uint8_t* s = reinterpret_cast<uint8_t*>(ws);
    ws += aligned(c.M * lds);
    rc = launch_mxfp4_quantize(c.x, c.dtype, c.ldx, c.M, c.K, to, s, lds, wide, stream);
    xc = reinterpret_cast<const char*>(to);
    xs = s;
  } else {
    xs = take_scales(c.x_scales, c.M, blocks, ws, x_wide);
    rc = launch_mxfp4_widen(wide, x_wide, stream);
  }
  if (rc) return rc;
  Product p{};
  p.x = Side{xc, blocks * 16, c.M, xs, lds};
  p.w = Side{codes, blocks * 16, c.N, wsc, lds};
  p.M = c.M;
  p.N = c.N;
  p.k_bytes = blocks * 16;
  p.blocks = blocks;
  p.chunks = int(cdiv(blocks, 8));
  launch_tiles<Form::kFp4, Lay::kRowsOfK, Lay::kRowsOfK, false>(p, store, ws, stream);
  return XK_OK;
}

template <typename T> int typed(const Call& c, void* out, const void* bias, char* ws, hipStream_t stream) {
  T* o = static_cast<T*>(out);
  const T* b = static_cast<const T*>(bias);
  return b != nullptr ? cut(c, Store<T, true>{o, b, c.N}, ws, stream) : cut(c, Store<T, false>{o, b, c.N}, ws, stream);
}

}  // namespace

int64_t mxfp4_linear_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= kFewRows) return 0;
  const int64_t blocks = cdiv(K, kMx4Block), lds = pad4(blocks);
  return aligned(M * blocks * 16) + aligned(M * lds) + (lds == blocks ? 0 : aligned(N * lds)) +
         sums_bytes(plan_tiles(true, M, N, cdiv(blocks, 8), false));
}

int launch_mxfp4_linear(const void* x, int dtype, int64_t ldx, const uint8_t* x_scales, int64_t M, int64_t K,
                        const uint8_t* codes, const uint8_t* scales, int64_t N, const void* bias, void* out,
                        int out_dtype, void* workspace, hipStream_t stream) {
  const Call c{x, dtype, ldx, x_scales, M, K, codes, scales, N};
  char* ws = static_cast<char*>(workspace);
  const int rc = out_dtype == XK_DT_BF16   ? typed<uint16_t>(c, out, bias, ws, stream)
                 : out_dtype == XK_DT_FP16 ? typed<_Float16>(c, out, bias, ws, stream)
                                           : typed<float>(c, out, bias, ws, stream);
  if (rc) return rc;
  XK_CHECK_LAUNCH("mxfp4_linear");
  return XK_OK;
}

}  // namespace xk
