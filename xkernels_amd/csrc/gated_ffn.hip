// The gated feed-forward block in 16 bits and its gradients:
//   g = x Wg^T, u = x Wu^T, h = silu(min(g, L)) clamp(u, -L, L), out = h W2^T
//   dh = dy W2, gc = min(g, L), uc = clamp(u, -L, L), s = 1 / (1 + e^-gc)
//   dg = dh uc s (1 + gc (1 - s)) [g <= L],  du = dh gc s [|u| <= L]
//   dx = [dg du] W13,  dW13 = [dg du]^T x,  dW2 = dy^T h
// Each product is a launch of the tile kernel (two with slices of k), or, for up to 16 tokens,
// of the kernel for few rows; the activation runs in the epilogue of the gate/up product,
// its gradient in that of dh. h, dg and du are rounded to the type once, as operands of
// the next product: their roundings add up like those of the outputs themselves (in bf16 outputs are 2.3e-3
// from 64 bits, their own rounding is 1.7e-3 of that). Up to 8 tokens the forward keeps what
// h's rounding left as well, in operand rows that would be empty: outputs are 1.7e-3 off. In
// fp16 all this is so within its range: h, dg and du past 65,504 are infinities, below 6e-5 they lose bits.
//
// bf16, 7168 x 2048: one token 22 us with the weights from memory (88 MB at 4.1 TB/s, two launches; 19 to 20 in calls
// on the same weights, parts of which are in caches then), 4,096 tokens 279 to 292 (1.24 to 1.29
// PFLOP/s, power and the way from L2 to LDS), forward and gradients of 8,192 tokens 1,749 to 1,827
// (1.18 to 1.24); 64 tokens of 4096 x 2048 29 us, in four dependent launches.
#include <algorithm>

#include "dense_rows.h"

namespace xk {
namespace {

using namespace dense;

int64_t pad8(int64_t n) { return (n + 7) & ~int64_t(7); }
int64_t aligned(int64_t bytes) { return (bytes + 255) & ~int64_t(255); }

template <Form F> struct num;
template <> struct num<Form::kBf16> {
  typedef uint16_t type;
  __device__ __forceinline__ static float get(uint16_t b) { return bf16_to_f32(b); }
  __device__ __forceinline__ static uint16_t put(float f) { return f32_to_bf16(f); }
};
template <> struct num<Form::kFp16> {
  typedef _Float16 type;
  __device__ __forceinline__ static float get(_Float16 h) { return float(h); }
  __device__ __forceinline__ static _Float16 put(float f) { return _Float16(f); }
};

// 4 consecutive values, of which n (any number) are within the row.
template <typename T> struct four { T v[4]; };
template <typename T> __device__ __forceinline__ void store_four(T* p, const four<T>& v, int64_t n) {
  if (n >= 4) {
    store_unaligned(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < n) p[i] = v.v[i];
  }
}
// out[m, n] in the type.
template <Form F> struct Store {
  static constexpr bool kFetches = false;
  typedef typename num<F>::type T;
  T* out;
  int64_t ld, N;
  struct Spot {
    T* out;
    int ld, left;  // columns from the spot on
    template <bool WHOLE> __device__ __forceinline__ void put(int row, int col, f32x4 sum) const {
      four<T> v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v.v[i] = num<F>::put(sum[i]);
      store_four(out + uint32_t(row * ld + col), v, WHOLE ? 4 : left - col);
    }
  };
  __device__ __forceinline__ Spot spot(int64_t m, int64_t n) const { return Spot{out + m * ld + n, int(ld), int(N - n)}; }
};

// The activation's parts. `limit` is an infinity where there is none.
__device__ __forceinline__ bool past(float v, float limit) { return v > limit; }  // (NaN is not)
// min(g, L) and clamp(u, -L, L); NaN stays NaN
__device__ __forceinline__ float below(float g, float limit) { return past(g, limit) ? limit : g; }
__device__ __forceinline__ float within(float u, float limit) { return past(fabsf(u), limit) ? copysignf(limit, u) : u; }
// (the reciprocal is within a step of fp32, as a division is; of an infinity it is 0)
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

// 4 consecutive fp32 values, of which n are within the row.
__device__ __forceinline__ void store_sums(float* p, f32x4 v, int n) {
  if (n >= 4) {
    store_unaligned(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < n) p[i] = v[i];
  }
}
__device__ __forceinline__ f32x4 load_sums(const float* p, int n) {
  if (n >= 4) return load_unaligned<f32x4>(p);
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
  return v;
}

// h = silu(g) u, in rows ldh apart whose places past the I columns are zeros, and
// gate_up [M, 2 I] (either may be null). The sums are kept in fp32: rounded, they would add their
// errors to every gradient (dW2 then is 3.4e-3 off, with them as they are 2.3e-3, the result's own
// rounding alone 1.7e-3; the time of a step of 8,192 tokens does not show it).
// LOW: what h's rounding left goes `low` values behind it, unless that is 0.
template <Form F, bool LOW = false> struct Gate {
  static constexpr bool kFetches = false;
  typedef typename num<F>::type T;
  T* h;
  float* gate_up;
  int64_t ldh, I;
  float limit;
  int64_t low = 0;
  struct Spot {
    T* h;
    float *g, *u;
    int ldh, ldg, left;
    float limit;
    int64_t low;
    template <bool WHOLE> __device__ __forceinline__ void put(int row, int col, f32x4 gs, f32x4 us) const {
      if (!WHOLE && col >= left) return;
      if (h != nullptr) {
        four<T> v, rest;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float gc = below(gs[i], limit), uc = within(us[i], limit), a = gc * sigmoid(gc) * uc;
          v.v[i] = WHOLE || col + i < left ? num<F>::put(a) : T(0);
          if constexpr (LOW) {  // (of a value past the type's finite ones nothing is left)
            const float off = a - num<F>::get(v.v[i]);
            rest.v[i] = col + i < left && fabsf(off) < 1e38f ? num<F>::put(off) : T(0);
          }
        }
        T* at = h + uint32_t(row * ldh + col);
        store_unaligned(at, v);  // (rows end at a multiple of 8)
        if constexpr (LOW) if (low != 0) store_unaligned(at + low, rest);
        if (!WHOLE && col + 4 >= left && (left & 7) <= 4 && (left & 7) > 0) store_unaligned(at + 4, four<T>{});
      }
      if (g != nullptr) {
        const uint32_t at = uint32_t(row * ldg + col);
        store_sums(g + at, gs, WHOLE ? 4 : left - col);
        store_sums(u + at, us, WHOLE ? 4 : left - col);
      }
    }
  };
  __device__ __forceinline__ Spot spot(int64_t m, int64_t j) const {
    float* g = gate_up == nullptr ? nullptr : gate_up + m * 2 * I + j;
    return Spot{h == nullptr ? nullptr : h + m * ldh + j, g, g + I, int(ldh), int(2 * I), int(I - j), limit, low};
  }
};

// From dh and gate_up [M, 2 I]: d [M, 2 I] = [dg du] and h [M, I], rows ldd and ldh apart with
// zeros behind them.
template <Form F> struct GateGrad {
  static constexpr bool kFetches = true;
  typedef typename num<F>::type T;
  const float* gate_up;
  T *d, *h;
  int64_t ldd, ldh, I;
  float limit;
  struct Kept {
    f32x4 g, u;
  };
  struct Spot {
    const float *g, *u;
    T *dg, *du, *h;
    int ldg, ldd, ldh, left;
    float limit;
    template <bool WHOLE> __device__ __forceinline__ Kept fetch(int row, int col) const {
      const uint32_t at = uint32_t(row * ldg + col);
      return Kept{load_sums(g + at, WHOLE ? 4 : left - col), load_sums(u + at, WHOLE ? 4 : left - col)};
    }
    template <bool WHOLE> __device__ __forceinline__ void put(int row, int col, f32x4 dh, const Kept& kept) const {
      if (!WHOLE && col >= left) return;
      four<T> gr, ur, v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float gs = kept.g[i], us = kept.u[i];
        const bool g_over = past(gs, limit), u_over = past(fabsf(us), limit);
        const float gc = g_over ? limit : gs, uc = u_over ? copysignf(limit, us) : us;
        const float s = sigmoid(gc), silu = gc * s, slope = fmaf(silu, 1.0f - s, s);
        gr.v[i] = num<F>::put(g_over ? 0.f : dh[i] * uc * slope);
        ur.v[i] = num<F>::put(u_over ? 0.f : dh[i] * silu);
        v.v[i] = WHOLE || col + i < left ? num<F>::put(silu * uc) : T(0);
      }
      const uint32_t at = uint32_t(row * ldd + col);
      store_four(dg + at, gr, WHOLE ? 4 : left - col);
      store_four(du + at, ur, WHOLE ? 4 : left - col);
      T* hat = h + uint32_t(row * ldh + col);
      store_unaligned(hat, v);  // (rows end at a multiple of 8)
      if (col + 4 >= left) {    // a row's last columns: the zeros behind them
        if ((left & 7) <= 4 && (left & 7) > 0) store_unaligned(hat + 4, four<T>{});
        T* end = du + uint32_t(row * ldd + left);
        for (int c = 0; c < ldd - ldg; ++c) end[c] = T(0);
      }
    }
  };
  __device__ __forceinline__ Spot spot(int64_t m, int64_t j) const {
    const float* g = gate_up + m * 2 * I + j;
    T* dg = d + m * ldd + j;
    return Spot{g, g + I, dg, dg + I, h + m * ldh + j, int(2 * I), int(ldd), int(ldh), int(I - j), limit};
  }
};

// Up to 4 matrices of n values a row, ld apart, to rows of n8 = pad8(n) with zeros behind them.
struct Copies {
  const uint16_t* src[4];
  uint16_t* dst[4];
  int64_t ld[4], n[4], end[4];  // end: in pieces of 8, of the copies up to this one
  int count = 0;
};
__global__ void __launch_bounds__(256) pad_rows(Copies c) {
  for (int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x; t < c.end[c.count - 1]; t += int64_t(gridDim.x) * 256) {
    int i = 0;
    while (t >= c.end[i]) ++i;
    const int64_t q = i ? t - c.end[i - 1] : t, n = c.n[i], pieces = (n + 7) / 8;
    const int64_t row = q / pieces, k = (q - row * pieces) * 8;
    const uint16_t* s = c.src[i] + row * c.ld[i] + k;
    __attribute__((aligned(16))) uint16_t v[8];
    if (k + 8 <= n) {
      __builtin_memcpy(v, s, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < n ? s[j] : uint16_t(0);
    }
    *reinterpret_cast<u32x4*>(c.dst[i] + q * 8) = *reinterpret_cast<const u32x4*>(v);
  }
}
void launch_copies(const Copies& c, hipStream_t stream) {
  if (c.count == 0) return;
  const int grid = int(std::min<int64_t>(cdiv(c.end[c.count - 1], 256), 256 * 32));
  hipLaunchKernelGGL(pad_rows, dim3(grid), dim3(256), 0, stream, c);
}

// A matrix [rows, n] of 16-bit values, rows ld apart, whose rows start at 16 bytes.
struct Matrix {
  const void* p;
  int64_t rows, n, ld;
  Side of_k() const { return Side{static_cast<const char*>(p), ld * 2, rows, nullptr, 0}; }
  // its columns as the rows of an operand
  Side columns() const { return Side{static_cast<const char*>(p), ld * 2, pad8(n), nullptr, 0}; }
};

// Takes the matrix as it is, or, where its width keeps rows from 16 bytes, as a copy with wider rows.
Matrix take(const void* p, int64_t rows, int64_t n, int64_t ld, char*& ws, Copies& copies) {
  if (n % 8 == 0 || rows == 0) return Matrix{p, rows, n, ld};
  const int64_t n8 = pad8(n);
  const int i = copies.count++;
  copies.src[i] = static_cast<const uint16_t*>(p);
  copies.dst[i] = reinterpret_cast<uint16_t*>(ws);
  copies.ld[i] = ld;
  copies.n[i] = n;
  copies.end[i] = rows * (n8 / 8) + (i ? copies.end[i - 1] : 0);
  ws += aligned(rows * n8 * 2);
  return Matrix{copies.dst[i], rows, n, n8};
}
int64_t taken_bytes(int64_t rows, int64_t n) { return n % 8 == 0 ? 0 : aligned(rows * pad8(n) * 2); }

int64_t chunks_of(int64_t k) { return cdiv(k, 64); }

// out = X W^T of k8 values a row of a side that lies so, k_rows of one that does not
Product product(const Side& x, const Side& w, int64_t M, int64_t N, int64_t k8, int64_t k_rows) {
  Product p{};
  p.x = x;
  p.w = w;
  p.M = M;
  p.N = N;
  p.k_bytes = k8 * 2;
  p.k_rows = k_rows;
  p.chunks = int(chunks_of(std::max(k8, k_rows)));
  return p;
}
Rows rows_of(const void* p, int64_t rows, int64_t ld) { return Rows{static_cast<const char*>(p), ld * 2, rows, nullptr, 0}; }

template <Form F>
int forward(const void* x, int64_t ldx, int64_t M, int64_t H, const void* w13, const void* w2, int64_t I, float limit,
            void* out, void* gate_up, void* workspace, hipStream_t stream) {
  typedef typename num<F>::type T;
  constexpr Lay R = Lay::kRowsOfK;
  limit = limit > 0.f ? limit : __builtin_inff();
  char* ws = static_cast<char*>(workspace);
  T* h = reinterpret_cast<T*>(ws);
  const int64_t ldh = pad8(I);
  const Store<F> store{static_cast<T*>(out), H, H};
  if (M <= kFewRows) {
    const int64_t low = M <= kPairRows ? M * ldh : 0;
    const Gate<F, true> gate{h, static_cast<float*>(gate_up), ldh, I, limit, low};
    Rows hr = rows_of(h, M, ldh);
    hr.low = low * 2;
    launch_rows<F, void, true>(rows_of(x, M, ldx), rows_of(w13, 2 * I, H), M, I, H, 0, gate, stream);
    launch_rows<F, void, false>(hr, rows_of(w2, H, I), M, H, I, 0, store, stream);
  } else {
    ws += aligned(M * ldh * 2);
    const Gate<F> gate{h, static_cast<float*>(gate_up), ldh, I, limit};
    Copies copies;
    const Matrix xm = take(x, M, H, ldx, ws, copies), m13 = take(w13, 2 * I, H, H, ws, copies),
                 m2 = take(w2, H, I, I, ws, copies), hm{h, M, I, ldh};
    launch_copies(copies, stream);
    launch_tiles<F, R, R, true>(product(xm.of_k(), m13.of_k(), M, I, pad8(H), 0), gate, ws, stream);
    launch_tiles<F, R, R, false>(product(hm.of_k(), m2.of_k(), M, H, ldh, 0), store, ws, stream);
  }
  XK_CHECK_LAUNCH("gated_ffn");
  return XK_OK;
}

template <Form F>
int backward(const void* dy, int64_t ldg, const void* x, int64_t ldx, int64_t M, int64_t H, const void* w13,
             const void* w2, int64_t I, const void* gate_up, float limit, void* dx, void* dw13, void* dw2,
             void* workspace, hipStream_t stream) {
  typedef typename num<F>::type T;
  constexpr Lay R = Lay::kRowsOfK, C = Lay::kColumns;
  limit = limit > 0.f ? limit : __builtin_inff();
  char* ws = static_cast<char*>(workspace);
  T* h = reinterpret_cast<T*>(ws);
  ws += aligned(M * pad8(I) * 2);
  T* d = reinterpret_cast<T*>(ws);
  ws += aligned(M * pad8(2 * I) * 2);
  Copies copies;
  const Matrix xm = take(x, M, H, ldx, ws, copies), m13 = take(w13, 2 * I, H, H, ws, copies),
               m2 = take(w2, H, I, I, ws, copies), gm = take(dy, M, H, ldg, ws, copies);
  launch_copies(copies, stream);
  const Matrix hm{h, M, I, pad8(I)}, dm{d, M, 2 * I, pad8(2 * I)};
  if (M > 0) {
    if (gate_up == nullptr) {
      gate_up = ws;
      const Gate<F> gate{nullptr, reinterpret_cast<float*>(ws), 0, I, limit};
      ws += aligned(M * 2 * I * 4);
      launch_tiles<F, R, R, true>(product(xm.of_k(), m13.of_k(), M, I, pad8(H), 0), gate, ws, stream);
    }
    const GateGrad<F> grad{static_cast<const float*>(gate_up), d, h, dm.ld, hm.ld, I, limit};
    launch_tiles<F, R, C, false>(product(gm.of_k(), m2.columns(), M, I, pad8(H), H), grad, ws, stream);
    launch_tiles<F, R, C, false>(product(dm.of_k(), m13.columns(), M, H, pad8(2 * I), 2 * I),
                                 Store<F>{static_cast<T*>(dx), H, H}, ws, stream);
  }
  launch_tiles<F, C, C, false>(product(dm.columns(), xm.columns(), 2 * I, H, 0, M), Store<F>{static_cast<T*>(dw13), H, H},
                               ws, stream);
  launch_tiles<F, C, C, false>(product(gm.columns(), hm.columns(), H, I, 0, M), Store<F>{static_cast<T*>(dw2), I, I}, ws,
                               stream);
  XK_CHECK_LAUNCH("gated_ffn_backward");
  return XK_OK;
}

// the slices' sums of a product of k values
int64_t sums_of(int64_t M, int64_t N, int64_t k, bool paired) {
  return M > 0 ? aligned(sums_bytes(plan_tiles(false, M, N, chunks_of(k), paired))) : 0;
}

}  // namespace

int64_t gated_ffn_workspace_bytes(int64_t M, int64_t H, int64_t I) {
  const int64_t h = aligned(M * pad8(I) * (M <= kPairRows ? 4 : 2));
  if (M <= kFewRows) return h;
  return h + taken_bytes(M, H) + taken_bytes(2 * I, H) + taken_bytes(H, I) +
         std::max(sums_of(M, I, pad8(H), true), sums_of(M, H, pad8(I), false));
}
int64_t gated_ffn_backward_workspace_bytes(int64_t M, int64_t H, int64_t I, int recompute) {
  const int64_t k1 = pad8(H), k2 = pad8(2 * I);
  int64_t sums = std::max(std::max(sums_of(M, I, k1, false), sums_of(M, H, k2, false)),
                          std::max(sums_of(2 * I, H, M, false), sums_of(H, I, M, false)));
  if (recompute) sums = std::max(sums, sums_of(M, I, k1, true)) + aligned(M * 2 * I * 4);
  return aligned(M * pad8(I) * 2) + aligned(M * k2 * 2) + taken_bytes(M, H) * 2 + taken_bytes(2 * I, H) +
         taken_bytes(H, I) + sums;
}

int launch_gated_ffn(const void* x, int dtype, int64_t ldx, int64_t M, int64_t H, const void* w13, const void* w2,
                     int64_t I, float limit, void* out, void* gate_up, void* ws, hipStream_t stream) {
  return dtype == XK_DT_BF16 ? forward<Form::kBf16>(x, ldx, M, H, w13, w2, I, limit, out, gate_up, ws, stream)
                             : forward<Form::kFp16>(x, ldx, M, H, w13, w2, I, limit, out, gate_up, ws, stream);
}

int launch_gated_ffn_backward(const void* dy, int dtype, int64_t ldg, const void* x, int64_t ldx, int64_t M, int64_t H,
                              const void* w13, const void* w2, int64_t I, const void* gate_up, float limit, void* dx,
                              void* dw13, void* dw2, void* ws, hipStream_t stream) {
  return dtype == XK_DT_BF16
             ? backward<Form::kBf16>(dy, ldg, x, ldx, M, H, w13, w2, I, gate_up, limit, dx, dw13, dw2, ws, stream)
             : backward<Form::kFp16>(dy, ldg, x, ldx, M, H, w13, w2, I, gate_up, limit, dx, dw13, dw2, ws, stream);
}

}  // namespace xk
