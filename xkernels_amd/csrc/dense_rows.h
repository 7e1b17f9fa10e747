// The dense products of few rows of X (up to 16): out[m, n] = sum_k X(m, k) W(n, k), where the
// weights' bytes are what counts.
//
//   * A workgroup owns 16 rows of W, its 8 waves take chunks of 128 bytes of k in turn
//     and add up through LDS in a fixed order: one launch, no partial results in memory, and
//     N / 16 workgroups keep all CUs loading.
//   * W and X go from memory straight to MFMA operands, a lane 32 bytes of a row. X is read
//     again by every workgroup, from L2. Rows past the last are read as the last: sums of
//     theirs go nowhere.
//   * Rows start at any address; only a row's last, short chunk is read by the value.
//   * MXFP4: activations in 16 or 32 bits are quantised on the way, a lane its blocks.
//   * Up to 8 rows X may be pairs of values, each with what its rounding left, as rows 8 to 15 of
//     the same operands: no more loads and products. (7168 x 2048, weights from memory: one token 21.3
//     -> 21.7 us, 8 tokens 24.5 -> 26.5; with the rest as an operand of its own 23.0 and 27.5, and 16 tokens
//     28.8 -> 32.9.)
//   * The order of a turn's loads and products is the compiler's, which takes 62 registers: all loads ahead of the
//     products take 154, and fewer waves, and were slower (23.0 -> 24.6 us).
#pragma once

#include "dense_tile.h"
#include "mx4.h"

namespace xk {
namespace dense {

constexpr int kRowWaves = 8;

// Where rows' values lie: `ld` bytes apart, of MXFP4 codes with scales, or of values to quantise, or
// of pairs, whose second parts lie `low` bytes behind the first ones (0: no pairs).
struct Rows {
  const char* p;
  int64_t ld, rows;
  const uint8_t* s;
  int64_t lds, low = 0;
};

// 16 bytes of a row from byte k of its `bytes`, zeros behind them.
__device__ __forceinline__ u32x4 row_end(const char* row, int64_t k, int64_t bytes) {
  if (k + 16 <= bytes) return load_unaligned<u32x4>(row + k);
  __attribute__((aligned(16))) uint16_t v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + 2 * i < bytes ? reinterpret_cast<const uint16_t*>(row + k)[i] : uint16_t(0);
  return *reinterpret_cast<const u32x4*>(v);
}

// The lane's two blocks of a chunk (32 bytes of codes) and their scales.
struct Blocks {
  u32x4 v[2];
  uint32_t s;  // a byte each
};

// Values to blocks. SRC: uint16_t (bf16), _Float16 or float.
template <typename SRC> __device__ __forceinline__ float src_value(SRC v) {
  if constexpr (sizeof(SRC) == 4) return v;
  else if constexpr (std::is_same_v<SRC, _Float16>) return float(v);
  else return bf16_to_f32(v);
}
template <typename SRC> struct Values { SRC v[2][kMx4Block]; };
template <typename SRC> __device__ __forceinline__ Blocks quantised(const Values<SRC>& x) {
  Blocks r;
  r.s = 0;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    float f[kMx4Block];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kMx4Block; ++i) {
      f[i] = src_value(x.v[b][i]);
      top = max(top, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    }
    const uint32_t byte = mx4_scale_byte(__uint_as_float(top));
    const float inv = mx4_inverse_scale(byte);
#pragma unroll
    for (int i = 0; i < kMx4Block; ++i) f[i] = byte == kMx4Nan ? 0.f : f[i] * inv;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[b][i] = mx4_pack8(f + 8 * i);
    r.s |= byte << (8 * b);
  }
  return r;
}

// F: of W. SRC: void where X is of F too, else the type of values that are quantised.
// K: 16-bit values, or MXFP4 blocks, of a row; `x_values`: the values of a row that are quantised.
template <Form F, typename SRC, bool PAIRED, typename EPI>
__global__ void __launch_bounds__(kRowWaves * 64)
dense_rows(Rows x, Rows w, int64_t M, int64_t N, int64_t K, int64_t x_values, EPI epi) {
  constexpr bool FP4 = F == Form::kFp4, QUANT = !std::is_void_v<SRC>;
  constexpr int MOST = QUANT ? 2 : 8;  // chunks at a time
  typedef std::conditional_t<QUANT, SRC, uint16_t> S;
  __shared__ f32x4 sums[kRowWaves][64];
  const int lane = threadIdx.x & 63, wave = uniform(int(threadIdx.x) >> 6), c = lane & 15, q = lane >> 4;
  const int64_t n0 = int64_t(blockIdx.x) * (PAIRED ? 8 : 16);
  // the lane's row of W: pairs have 8 gate rows and the 8 up rows of the same columns
  const int64_t wr = PAIRED ? min(n0 + (c & 7), N - 1) + (c >= 8 ? N : 0) : min(n0 + c, N - 1);
  const char* wp = w.p + wr * w.ld;
  const uint8_t* wsp = FP4 ? w.s + wr * w.lds : nullptr;
  const bool both = x.low != 0;
  const int64_t xr = min(int64_t(both ? c & 7 : c), M - 1);
  const char* xp = x.p + xr * x.ld + (c >= 8 ? x.low : 0);
  const uint8_t* xsp = FP4 && !QUANT ? x.s + xr * x.lds : nullptr;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};

  const int64_t bytes = FP4 ? K * 16 : K * 2;
  // whole chunks; values that are quantised end with the row's last whole chunk of them
  const int full = int(QUANT ? x_values / (8 * kMx4Block) : bytes / kChunk);
  const int all = int(cdiv(bytes, kChunk));
  auto load = [&](const char* row, const uint8_t* s, int chunk, Blocks& o) __attribute__((always_inline)) {
    const char* p = row + int64_t(chunk) * kChunk + q * 32;
    o.v[0] = load_unaligned<u32x4>(p);
    o.v[1] = load_unaligned<u32x4>(p + 16);
    if constexpr (FP4) o.s = load_unaligned<uint16_t>(s + int64_t(chunk) * 8 + q * 2);
  };
  auto load_values = [&](const char* row, int chunk, Values<S>& o) __attribute__((always_inline)) {
    __builtin_memcpy(&o, row + (int64_t(chunk) * 8 + q * 2) * kMx4Block * sizeof(S), sizeof(o));
  };
  auto math = [&](const Blocks& wv, const Blocks& xv) __attribute__((always_inline)) {
    if constexpr (FP4) {
      acc = mma4<0>(wv.v[0], wv.s, xv.v[0], xv.s, acc);
      acc = mma4<1>(wv.v[1], wv.s, xv.v[1], xv.s, acc);
    } else {
      acc = mma<F>(wv.v[0], xv.v[0], acc);
      acc = mma<F>(wv.v[1], xv.v[1], acc);
    }
  };
  int chunk = wave;
  // U chunks: all their loads, then their products
  auto batch = [&](auto COUNT) __attribute__((always_inline)) {
    constexpr int U = decltype(COUNT)::value;
    Blocks wv[U];
    std::conditional_t<QUANT, Values<S>, Blocks> xv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(wp, wsp, chunk + u * kRowWaves, wv[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (QUANT) load_values(xp, chunk + u * kRowWaves, xv[u]);
      else load(xp, xsp, chunk + u * kRowWaves, xv[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (QUANT) math(wv[u], quantised(xv[u]));
      else math(wv[u], xv[u]);
    }
    chunk += U * kRowWaves;
  };
  while (chunk + (MOST - 1) * kRowWaves < full) batch(std::integral_constant<int, MOST>{});
  if (MOST > 4 && chunk + 3 * kRowWaves < full) batch(std::integral_constant<int, 4>{});
  if (MOST > 2 && chunk + kRowWaves < full) batch(std::integral_constant<int, 2>{});
  if (chunk < full) batch(std::integral_constant<int, 1>{});
  if (chunk < all) {  // the row's short chunk
    Blocks wv, xv;
    const int64_t k = int64_t(chunk) * kChunk + q * 32;
    auto load_end = [&](const char* row, const uint8_t* s, Blocks& o) __attribute__((always_inline)) {
      o.v[0] = row_end(row, k, bytes);
      o.v[1] = row_end(row, k + 16, bytes);
      if constexpr (FP4) {  // (a scale of 1 where there is no block)
        const int64_t at = int64_t(chunk) * 8 + q * 2;
        o.s = (at < K ? s[at] : 127u) | (at + 1 < K ? s[at + 1] : 127u) << 8;
      }
    };
    load_end(wp, wsp, wv);
    if constexpr (QUANT) {
      Values<S> v;
      const int64_t at = (int64_t(chunk) * 8 + q * 2) * kMx4Block;
      const S* row = reinterpret_cast<const S*>(xp);
#pragma unroll
      for (int i = 0; i < 2 * kMx4Block; ++i) v.v[i / kMx4Block][i % kMx4Block] = at + i < x_values ? row[at + i] : S(0);
      xv = quantised(v);
    } else {
      load_end(xp, xsp, xv);
    }
    math(wv, xv);
  }

  sums[wave][lane] = acc;
  __syncthreads();
  if (wave > 0 || c >= M || (PAIRED && q >= 2)) return;
  auto total = [&](int at) __attribute__((always_inline)) {
    f32x4 t = sums[0][at];
#pragma unroll
    for (int v = 1; v < kRowWaves; ++v) t += sums[v][at];
    return t;
  };
  f32x4 t = total(lane);
  if (both) {  // (what is not finite comes from the first parts or from W, which has it in both sums)
    const f32x4 rest = total(lane + 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = fabsf(t[i]) < __builtin_inff() ? t[i] + rest[i] : t[i];
  }
  finish<EPI, PAIRED>(epi.spot(0, n0), c, q * 4, t, PAIRED ? total((lane + 32) & 63) : f32x4{});
}

// More rows are cheaper in tiles with slices of k (32 x 4096 x 4096: 10 and 4 us, where two row
// tiles here took 15).
constexpr int64_t kFewRows = 16, kPairRows = 8;

template <Form F, typename SRC, bool PAIRED, typename EPI>
void launch_rows(const Rows& x, const Rows& w, int64_t M, int64_t N, int64_t K, int64_t x_values, const EPI& epi,
                 hipStream_t stream) {
  hipLaunchKernelGGL((dense_rows<F, SRC, PAIRED, EPI>), dim3(int(cdiv(N, PAIRED ? 8 : 16))), dim3(kRowWaves * 64), 0, stream,
                     x, w, M, N, K, x_values, epi);
}

}  // namespace dense
}  // namespace xk
