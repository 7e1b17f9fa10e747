// The router's training step: the balance loss with its per-expert counts, and the
// gradient of the logits.
//
// With V the T rows that the mask leaves (all without one), p = softmax(logits) in
// fp32 and c_e the number of slots of V on expert e:
//   loss = E / (T^2 k) sum_e c_e sum_{m in V} p_me,
//   d loss / d z_mi = E / (T^2 k) p_mi (c_i - sum_e p_me c_e)    (c constant),
// and through the router's weights (renormalised: a softmax of the selected logits)
//   dz_i += sum_{j: e_j = i} w_j (u_j - sum_l w_l u_l),  w_j = p_{e_j} / sum_l p_{e_l}, or
//   dz_i += p_i (sum_{j: e_j = i} u_j - sum_j p_{e_j} u_j)       (not renormalised).
//
// Both directions are one pass over the logits, HBM bound for large batches (M * E
// values in, and out in the backward) and launches for small ones. The forward
// keeps each workgroup's column sums in registers over its rows and leaves one
// plane of sums and counts per workgroup; a second launch adds the planes in
// order, eights of them in 64 bits, so results do not depend on scheduling (counts are whole
// numbers; the probabilities' sums have a fixed order). No sum in 32 bits is longer
// than kLaneRows: a term that is always the same rounds the same way every time, and
// the error would grow with the batch. The backward forms p again rather than
// read it: M * E exponentials cost less than M * E more values from memory.
// Up to kOneWgRows rows the forward is one workgroup and one launch.
#include <algorithm>

#include "router_rows.h"

namespace xk {
namespace {

constexpr int kThreads = 256;
constexpr int kRowThreads = 512;    // of a forward's workgroup: few planes, many rows on their way
constexpr int kOneWg = 1024;        // threads of the one workgroup of a small batch, and of the sums
constexpr int64_t kOneWgRows = 256; // rows up to which it is one workgroup's work
constexpr int kFastExperts = 512, kFastTopk = 16;
constexpr int kGradWgs = 1024;      // most workgroups of the gradient: each forms the counts' mean once
constexpr int kPlanes = 512;        // workgroups of the forward: 16 waves a CU, more past 2^20 rows
constexpr int kLaneRows = 64;       // most rows of a 16-lane row of the forward

__device__ __forceinline__ float row_max(float x) {
  row_steps([&](auto from) { x = fmaxf(x, __uint_as_float(from(__float_as_uint(x)))); });
  return x;
}
__device__ __forceinline__ float row_sum(float x) {
  row_steps([&](auto from) { x += __uint_as_float(from(__float_as_uint(x))); });
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off);
  return x;
}

// (exact for whole numbers, as the counts are)
__device__ __forceinline__ double row_sum(double x) {
  row_steps([&](auto from) {
    const uint64_t b = __double_as_longlong(x);
    const uint64_t lo = from(uint32_t(b)), hi = from(uint32_t(b >> 32));
    x += __longlong_as_double(hi << 32 | lo);
  });
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off);
  return x;
}

template <typename T> __device__ __forceinline__ T to_out(float f);
template <> __device__ __forceinline__ uint16_t to_out<uint16_t>(float f) { return f32_to_bf16(f); }
template <> __device__ __forceinline__ _Float16 to_out<_Float16>(float f) { return _Float16(f); }
template <> __device__ __forceinline__ float to_out<float>(float f) { return f; }

// e^x for x <= 0 or NaN, to 2 steps of fp32 and to fp32's least step: 2^(x log2 e) as
// 2^n 2^f, n the nearest whole number (the low bits of a sum with 1.5 * 2^23) and f what
// is left, with log2 e in two parts, by v_exp_f32 (whose own results below the least
// normal number would be 0).
__device__ __forceinline__ float exp_neg(float x) {
  x = __builtin_elementwise_maximum(x, -104.f);  // (NaN stays)
  constexpr float kWhole = 12582912.f;
  const float t = fmaf(x, 1.44269502f, kWhole);
  const float f = fmaf(x, 1.92596303e-8f, fmaf(x, 1.44269502f, kWhole - t));
  return __builtin_ldexpf(__builtin_amdgcn_exp2f(f), int(__float_as_uint(t) - __float_as_uint(kWhole)));
}

// A row on its 16 lanes: lane i holds the 8-expert pieces i, i + 16, ...; z the logits
// (-inf past E).
template <typename T, int PIECES, bool WIDE>
__device__ __forceinline__ void load_row(const T* g, int E, int i16, float* z) {
#pragma unroll
  for (int c = 0; c < PIECES; ++c) {
    const int e0 = (c * 16 + i16) * 8;
    if (WIDE) {
      if (e0 < E) {
        piece8<T>::load(g + e0, z + 8 * c);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[8 * c + i] = -__builtin_inff();
      }
    } else if (e0 + 8 <= E) {
      __attribute__((aligned(16))) T v[8];
      __builtin_memcpy(v, g + e0, sizeof(v));  // a wide access at any alignment
      piece8<T>::load(v, z + 8 * c);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[8 * c + i] = e0 + i < E ? logit_at<T>(g + e0 + i) : -__builtin_inff();
    }
  }
}
// z becomes e^(z - mx); the sum over the row is returned. (Past E: e^-inf = 0 but where
// mx is infinite, and then the row is NaN.)
template <int N> __device__ __forceinline__ float row_exp(float* z, float& mx) {
  mx = z[0];
#pragma unroll
  for (int j = 1; j < N; ++j) mx = fmaxf(mx, z[j]);
  mx = row_max(mx);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    z[j] = exp_neg(z[j] - mx);
    sum += z[j];
  }
  return row_sum(sum);
}

// Scratch: planes of column sums and counts, the rows counted per plane, the
// loss's parts and their ticket.
struct BalanceScratch {
  float* sums;     // [planes, E]
  int32_t* cnt;    // [planes, E]
  int32_t* rows;   // [planes]
  double* parts;   // [blocks of the last kernel]
  int32_t* ticket;
  float* stat;     // [M, 2] for rows past kFastExperts: maximum and 1 / sum
};

// loss = E / (T^2 k) * total in 64 bits: T = 0 gives 0.
__device__ __forceinline__ float loss_of(double total, int64_t E, int64_t T, int64_t k) {
  return T == 0 ? 0.f : float(total * double(E) / (double(T) * double(T) * double(k)));
}

// One workgroup's rows: column sums of p over them in registers, then over the
// workgroup's rows of lanes in LDS. ONE: the whole batch, loss included.
//
// bf16, k = 8: M = 65,536, E = 384 18 us (50 MB and 2 of ids, 2.9 TB/s; some 15 VALU
// operations for each of 25 M logits, about 12 us, and the loads, 10, which begin only
// when the row before is done); 8,192 x 256 5.3; one workgroup, 200 x 48 fp32, 6.8.
template <typename T, int PIECES, bool WIDE, bool ONE>
__global__ void __launch_bounds__(ONE ? kOneWg : kRowThreads)
balance_rows(const T* __restrict__ logits, const int32_t* __restrict__ ids, const uint8_t* __restrict__ mask,
             int64_t M, int E, int k, BalanceScratch s, float* __restrict__ loss, int32_t* __restrict__ counts,
             int32_t* __restrict__ tokens) {
  constexpr int N = PIECES * 8, kT = ONE ? kOneWg : kRowThreads, kWaves = kT / 64;
  __shared__ float lds_sum[kWaves][PIECES * 128];
  __shared__ int lds_cnt[PIECES * 128];
  __shared__ int lds_rows;
  __shared__ double lds_part[kWaves];
  const int tid = threadIdx.x, i16 = tid & 15;
  for (int e = tid; e < E; e += kT) lds_cnt[e] = 0;
  if (tid == 0) {
    lds_rows = 0;
    if (!ONE && blockIdx.x == 0) *s.ticket = 0;  // for the launch that follows
  }
  __syncthreads();
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  int rows = 0;
  for (int64_t row = int64_t(blockIdx.x) * (kT / 16) + (tid >> 4); row < M; row += int64_t(gridDim.x) * (kT / 16)) {
    if (mask != nullptr && mask[row] == 0) continue;  // whole 16-lane rows
    ++rows;
    for (int j = i16; j < k; j += 16) {
      const int id = ids[row * k + j];
      if (id >= 0 && id < E) atomicAdd(&lds_cnt[id], 1);
    }
    float p[N], mx;
    load_row<T, PIECES, WIDE>(logits + row * E, E, i16, p);
    const float inv = 1.f / row_exp<N>(p, mx);
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = fmaf(p[j], inv, acc[j]);
  }
  if (i16 == 0 && rows) atomicAdd(&lds_rows, rows);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    acc[j] += __shfl_xor(acc[j], 16);
    acc[j] += __shfl_xor(acc[j], 32);
  }
  if ((tid & 63) < 16)
#pragma unroll
    for (int j = 0; j < N; ++j) lds_sum[tid >> 6][((j >> 3) * 16 + i16) * 8 + (j & 7)] = acc[j];
  __syncthreads();
  double part = 0.0;
  for (int e = tid; e < E; e += kT) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) t += lds_sum[w][e];
    const int c = lds_cnt[e];
    if (ONE) {
      counts[e] = c;
      part += double(c) * double(t);
    } else {
      s.sums[int64_t(blockIdx.x) * E + e] = t;
      s.cnt[int64_t(blockIdx.x) * E + e] = c;
    }
  }
  if (!ONE) {
    if (tid == 0) s.rows[blockIdx.x] = lds_rows;
    return;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) part += __shfl_xor(part, off);
  if ((tid & 63) == 0) lds_part[tid >> 6] = part;
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += lds_part[w];
    *loss = loss_of(total, E, lds_rows, k);
    *tokens = lds_rows;
  }
}

// Adds the planes: 16 columns a workgroup, 64 threads a column, eight planes' loads in
// flight each; the workgroup that arrives last adds the loss's parts in order.
// COUNTED: counts[] is complete. 5.1 to 5.9 us: a launch, two dependent rounds of loads
// and the ticket.
template <bool COUNTED>
__global__ void __launch_bounds__(kOneWg)
balance_finish(int planes, int64_t E, int64_t k, BalanceScratch s, float* __restrict__ loss,
               int32_t* __restrict__ counts, int32_t* __restrict__ tokens) {
  constexpr int kParts = kOneWg / 16, kAhead = 8;
  __shared__ float lds_p[kParts][16];
  __shared__ int lds_c[kParts][16];
  __shared__ int lds_rows[kOneWg / 64];
  const int tid = threadIdx.x, col = tid & 15, part = tid >> 4;
  const int64_t e = int64_t(blockIdx.x) * 16 + col;
  double p = 0.0;
  int c = 0;
  for (int g0 = part; g0 < planes; g0 += kParts * kAhead) {
    float pv[kAhead];
    int cv[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int g = g0 + j * kParts;
      const bool in = g < planes && e < E;
      pv[j] = in ? s.sums[int64_t(g) * E + e] : 0.f;
      cv[j] = in && !COUNTED ? s.cnt[int64_t(g) * E + e] : 0;
    }
    float eight = 0.f;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      eight += pv[j];
      c += cv[j];
    }
    p += double(eight);
  }
  lds_p[part][col] = float(p);
  lds_c[part][col] = c;
  int rows = 0;
  for (int g = tid; g < planes; g += kOneWg) rows += s.rows[g];
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) rows += __shfl_xor(rows, off);
  if ((tid & 63) == 0) lds_rows[tid >> 6] = rows;
  __syncthreads();
  if (tid >= 64) return;
  int T = 0;
#pragma unroll
  for (int w = 0; w < kOneWg / 64; ++w) T += lds_rows[w];
  double dot = 0.0;
  if (tid < 16 && e < E) {
    double ps = 0.0;
    int cs = 0;
#pragma unroll 2
    for (int i = 0; i < kParts; i += 8) {
      float eight = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        eight += lds_p[i + j][col];
        cs += lds_c[i + j][col];
      }
      ps += double(eight);
    }
    if (COUNTED) cs = counts[e];
    else counts[e] = cs;
    dot = double(cs) * ps;
  }
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) dot += __shfl_xor(dot, off);
  int at = 0;
  if (tid == 0) {
    __hip_atomic_store(&s.parts[blockIdx.x], dot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    at = __hip_atomic_fetch_add(s.ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (__builtin_amdgcn_readfirstlane(at) != int(gridDim.x) - 1) return;
  double total = 0.0;
  for (int i = tid; i < int(gridDim.x); i += 64)
    total += __hip_atomic_load(&s.parts[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) total += __shfl_xor(total, off);
  if (tid == 0) {
    *loss = loss_of(total, E, T, k);
    *tokens = T;
  }
}

// ------------------------------------------------- rows past kFastExperts ----
// 8,192 x 600: 9 us and, for the columns, 76: up to 64 planes, each thread's rows one
// after another (65,536 rows 650 us in all).
// Maximum and 1 / sum of each row (a wave each); counts[] and the ticket cleared.
template <typename T>
__global__ void __launch_bounds__(kThreads)
row_stats(const T* __restrict__ logits, const uint8_t* __restrict__ mask, int64_t M, int64_t E, BalanceScratch s,
          int32_t* __restrict__ counts) {
  const int lane = threadIdx.x & 63;
  const int64_t t0 = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  for (int64_t e = t0; e < E; e += int64_t(gridDim.x) * kThreads) counts[e] = 0;
  if (t0 == 0) *s.ticket = 0;
  for (int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); row < M; row += int64_t(gridDim.x) * 4) {
    if (mask != nullptr && mask[row] == 0) continue;
    const T* g = logits + row * E;
    float mx = -__builtin_inff(), sum = 0.f;
    for (int64_t e = lane; e < E; e += 64) mx = fmaxf(mx, logit_at<T>(g + e));
    mx = wave_max(mx);
    for (int64_t e = lane; e < E; e += 64) sum += expf(logit_at<T>(g + e) - mx);
    sum = wave_sum(sum);
    if (lane == 0) {
      s.stat[2 * row] = mx;
      s.stat[2 * row + 1] = 1.f / sum;
    }
  }
}

// Column sums: a thread per expert, a plane per part of the rows, in 64 bits (a part may
// be long).
template <typename T>
__global__ void __launch_bounds__(kThreads)
balance_columns(const T* __restrict__ logits, const int32_t* __restrict__ ids, const uint8_t* __restrict__ mask,
                int64_t M, int64_t E, int64_t k, int64_t rows_per_plane, BalanceScratch s,
                int32_t* __restrict__ counts) {
  const int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t first = int64_t(blockIdx.y) * rows_per_plane, end = min(M, first + rows_per_plane);
  double sum = 0.0;
  int rows = 0;
  for (int64_t row = first; row < end; ++row) {
    if (mask != nullptr && mask[row] == 0) continue;
    ++rows;
    if (e < E) sum += double(expf(logit_at<T>(logits + row * E + e) - s.stat[2 * row]) * s.stat[2 * row + 1]);
    if (blockIdx.x == 0)
      for (int64_t j = threadIdx.x; j < k; j += kThreads) {
        const int id = ids[row * k + j];
        if (id >= 0 && id < E) atomicAdd(&counts[id], 1);
      }
  }
  if (e < E) s.sums[int64_t(blockIdx.y) * E + e] = float(sum);
  if (blockIdx.x == 0 && threadIdx.x == 0) s.rows[blockIdx.y] = rows;
}

// ---------------------------------------------------------------- backward ----
struct RouterGrad {
  const int32_t* ids;
  const uint8_t* mask;
  const int32_t* counts;      // with grad_loss
  const int32_t* tokens;      // nullable: every row counts
  const float* grad_loss;     // nullable
  const float* grad_weights;  // nullable
  int renorm;
};

// E / (T^2 k) * grad_loss; 0 without one or without rows.
__device__ __forceinline__ float loss_factor(const RouterGrad& a, int64_t M, int64_t E, int64_t k) {
  if (a.grad_loss == nullptr) return 0.f;
  const double T = a.tokens != nullptr ? double(*a.tokens) : double(M);
  return T > 0.0 ? float(double(*a.grad_loss) * double(E) / (T * T * double(k))) : 0.f;
}

template <typename T, int PIECES>
__device__ __forceinline__ void put_row(const float* p, T* row, int i16) {
#pragma unroll
  for (int cc = 0; cc < PIECES; ++cc) {
    __attribute__((aligned(16))) T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_out<T>(p[8 * cc + i]);
#pragma unroll
    for (int h = 0; h < int(sizeof(T)) / 2; ++h)
      reinterpret_cast<u32x4*>(row + (cc * 16 + i16) * 8)[h] = reinterpret_cast<const u32x4*>(v)[h];
  }
}

// The counts less their mean: as p sums to 1, c_i - sum p c is the same of either,
// and near-uniform counts (as a balanced router has) no longer cancel. The difference
// is formed in 64 bits: counts summed over many batches have more than fp32's 24. A row's
// gradient goes through LDS on its way out: the selected experts' slots, on the lane
// of their number, put their values there, and whole pieces leave.
//
// bf16, k = 8: M = 65,536, E = 384 30 us (100 MB and 4 of ids and weights, 3.5 TB/s,
// and as much VALU work as the forward's, after each row's loads), 8,192 x 256 7.0.
template <typename T, int PIECES, bool WIDE>
__global__ void __launch_bounds__(kThreads)
router_grad_rows(const T* __restrict__ logits, int64_t M, int E, int k, RouterGrad a, T* __restrict__ grad) {
  constexpr int N = PIECES * 8, ROW = PIECES * 128;
  __shared__ __attribute__((aligned(16))) T rows_lds[kThreads / 16][ROW];
  __shared__ union { int count; float over; } experts[ROW];  // the counts, then less their mean
  const int tid = threadIdx.x, i16 = tid & 15;
  const bool with_loss = a.grad_loss != nullptr, with_weights = a.grad_weights != nullptr;
  T* mine = rows_lds[tid >> 4];
  for (int e = tid; e < ROW; e += kThreads) experts[e].count = with_loss && e < E ? a.counts[e] : 0;
  __syncthreads();
  double mean = 0.0;
#pragma unroll
  for (int j = 0; j < N; ++j) mean += double(experts[((j >> 3) * 16 + i16) * 8 + (j & 7)].count);
  mean = row_sum(mean) / double(E);
  __syncthreads();
  for (int e = tid; e < ROW; e += kThreads) experts[e].over = float(double(experts[e].count) - mean);
  __syncthreads();
  float c[N];
#pragma unroll
  for (int j = 0; j < N; ++j) c[j] = experts[((j >> 3) * 16 + i16) * 8 + (j & 7)].over;
  const float factor = loss_factor(a, M, E, k);
  for (int64_t row = int64_t(blockIdx.x) * (kThreads / 16) + (tid >> 4); row < M;
       row += int64_t(gridDim.x) * (kThreads / 16)) {
    const T* g = logits + row * E;
    T* out = grad + row * E;
    const bool on = a.mask == nullptr || a.mask[row] != 0;  // the same on a row's 16 lanes
    float p[N];
    if (on) {
      int id = -1;
      float u = 0.f, z_id = -__builtin_inff();
      if (with_weights && i16 < k) {  // lane t holds slot t
        id = a.ids[row * k + i16];
        if (id < 0 || id >= E) id = -1;
        u = a.grad_weights[row * k + i16];
      }
      load_row<T, PIECES, WIDE>(g, E, i16, p);
      if (id >= 0) z_id = logit_at<T>(g + id);
      float mx, pc = 0.f, q = 0.f;
      const float inv = 1.f / row_exp<N>(p, mx);
      if (with_loss) {
#pragma unroll
        for (int j = 0; j < N; ++j) pc = fmaf(p[j], c[j], pc);
        pc = row_sum(pc) * inv;
      }
      float slot = 0.f, p_id = 0.f;
      if (with_weights) {
        p_id = id >= 0 ? exp_neg(z_id - mx) * inv : 0.f;
        if (a.renorm) {  // a softmax of the slots' logits
          const float top = row_max(z_id);
          const float w = id >= 0 ? exp_neg(z_id - top) : 0.f;
          const float scale = 1.f / row_sum(w);
          const float wu = row_sum(id >= 0 ? w * u : 0.f) * scale;
          slot = id >= 0 ? w * scale * (u - wu) : 0.f;
        } else {
          slot = id >= 0 ? p_id * u : 0.f;
          q = row_sum(slot);
        }
      }
      const float f = factor * inv, qi = q * inv;
#pragma unroll
      for (int j = 0; j < N; ++j) p[j] = with_loss ? p[j] * fmaf(f, c[j] - pc, -qi) : -p[j] * qi;
      put_row<T, PIECES>(p, mine, i16);
      wave_lds_fence();  // a slot's value replaces another lane's
      if (with_weights) {
        // every slot of one expert forms the same sum, in slot order
        float add = 0.f;
        for (int l = 0; l < k; ++l) {
          const float v = __shfl(slot, (tid & 48) + l);
          const int other = __shfl(id, (tid & 48) + l);
          if (other == id) add += v;
        }
        if (id >= 0) mine[id] = to_out<T>((with_loss ? p_id * fmaf(factor, experts[id].over - pc, -q) : -p_id * q) + add);
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) p[j] = 0.f;
      put_row<T, PIECES>(p, mine, i16);
    }
    wave_lds_fence();
#pragma unroll
    for (int cc = 0; cc < PIECES; ++cc) {
      const int e0 = (cc * 16 + i16) * 8;
      if (WIDE) {
        if (e0 < E)
#pragma unroll
          for (int h = 0; h < int(sizeof(T)) / 2; ++h)
            reinterpret_cast<u32x4*>(out + e0)[h] = reinterpret_cast<const u32x4*>(mine + e0)[h];
      } else if (e0 + 8 <= E) {
        __builtin_memcpy(out + e0, mine + e0, 8 * sizeof(T));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e0 + i < E) out[e0 + i] = mine[e0 + i];
      }
    }
    wave_lds_fence();
  }
}

// Any E and k: a wave per row, the row read again for each pass and its probabilities
// formed in each (8,192 rows: E = 600, k = 8 31 us, E = 256, k = 24 22).
template <typename T>
__global__ void __launch_bounds__(kThreads)
router_grad_any(const T* __restrict__ logits, int64_t M, int64_t E, int64_t k, RouterGrad a, T* __restrict__ grad) {
  const int lane = threadIdx.x & 63;
  const bool with_loss = a.grad_loss != nullptr;
  double mean = 0.0;
  if (with_loss) {
    for (int64_t e = lane; e < E; e += 64) mean += double(a.counts[e]);
    mean = wave_sum(mean) / double(E);
  }
  auto over = [&](int64_t e) { return float(double(a.counts[e]) - mean); };
  const float factor = loss_factor(a, M, E, k);
  for (int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); row < M; row += int64_t(gridDim.x) * 4) {
    const T* g = logits + row * E;
    T* out = grad + row * E;
    if (a.mask != nullptr && a.mask[row] == 0) {
      for (int64_t e = lane; e < E; e += 64) out[e] = to_out<T>(0.f);
      continue;
    }
    float mx = -__builtin_inff(), sum = 0.f;
    for (int64_t e = lane; e < E; e += 64) mx = fmaxf(mx, logit_at<T>(g + e));
    mx = wave_max(mx);
    for (int64_t e = lane; e < E; e += 64) sum += expf(logit_at<T>(g + e) - mx);
    sum = wave_sum(sum);
    auto prob = [&](int64_t e) { return expf(logit_at<T>(g + e) - mx) / sum; };
    float pc = 0.f, q = 0.f, ps = 0.f, wu = 0.f, top = -__builtin_inff();
    if (with_loss) {
      for (int64_t e = lane; e < E; e += 64) pc += prob(e) * over(e);
      pc = wave_sum(pc);
    }
    if (a.grad_weights != nullptr) {
      if (a.renorm) {  // a softmax of the slots' logits
        for (int64_t j = lane; j < k; j += 64) {
          const int id = a.ids[row * k + j];
          if (id >= 0 && id < E) top = fmaxf(top, logit_at<T>(g + id));
        }
        top = wave_max(top);
      }
      for (int64_t j = lane; j < k; j += 64) {
        const int id = a.ids[row * k + j];
        if (id < 0 || id >= E) continue;
        const float pj = a.renorm ? expf(logit_at<T>(g + id) - top) : prob(id);
        ps += pj;
        q += pj * a.grad_weights[row * k + j];
      }
      ps = wave_sum(ps);
      q = wave_sum(q);
      if (a.renorm) {
        wu = q / ps;
        q = 0.f;
      }
    }
    auto base = [&](int64_t e) {
      return prob(e) * (with_loss ? fmaf(factor, over(e) - pc, -q) : -q);
    };
    for (int64_t e = lane; e < E; e += 64) out[e] = to_out<T>(base(e));
    if (a.grad_weights == nullptr) continue;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // the row's stores first (vmcnt 0)
    for (int64_t j = lane; j < k; j += 64) {
      const int id = a.ids[row * k + j];
      if (id < 0 || id >= E) continue;
      const float w = a.renorm ? expf(logit_at<T>(g + id) - top) / ps : prob(id);
      float add = 0.f;
      for (int64_t l = 0; l < k; ++l)
        if (a.ids[row * k + l] == id) add += w * (a.grad_weights[row * k + l] - wu);
      out[id] = to_out<T>(base(id) + add);
    }
  }
}

int planes_for(int64_t M, int64_t E) {
  if (E <= kFastExperts)
    return int(std::max(std::min<int64_t>(kPlanes, cdiv(M, kRowThreads / 16)), cdiv(M, kRowThreads / 16 * kLaneRows)));
  return int(std::max<int64_t>(1, std::min<int64_t>(64, cdiv(M, 16))));
}
int64_t up(int64_t x) { return (x + 255) / 256 * 256; }

template <typename T, int PIECES>
void launch_balance_rows(const T* g, const int32_t* ids, const uint8_t* mask, int64_t M, int E, int k, int planes,
                         const BalanceScratch& s, float* loss, int32_t* counts, int32_t* tokens,
                         hipStream_t stream) {
  const bool wide = E % 8 == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0;
  const bool one = M <= kOneWgRows;
#define XK_ROWS(W, O)                                                                                             \
  hipLaunchKernelGGL((balance_rows<T, PIECES, W, O>), dim3(O ? 1 : planes), dim3(O ? kOneWg : kRowThreads), 0, stream, g, \
                     ids, mask, M, E, k, s, loss, counts, tokens)
  if (one && wide) XK_ROWS(true, true);
  else if (one) XK_ROWS(false, true);
  else if (wide) XK_ROWS(true, false);
  else XK_ROWS(false, false);
#undef XK_ROWS
}

template <typename T>
int balance_typed(const void* logits, const int32_t* ids, const uint8_t* mask, int64_t M, int64_t E, int64_t k,
                  BalanceScratch s, float* loss, int32_t* counts, int32_t* tokens, hipStream_t stream) {
  const T* g = static_cast<const T*>(logits);
  const int planes = planes_for(M, E);
  if (E <= kFastExperts) {
    const int e = int(E), kk = int(k);
    if (E <= 128) launch_balance_rows<T, 1>(g, ids, mask, M, e, kk, planes, s, loss, counts, tokens, stream);
    else if (E <= 256) launch_balance_rows<T, 2>(g, ids, mask, M, e, kk, planes, s, loss, counts, tokens, stream);
    else if (E <= 384) launch_balance_rows<T, 3>(g, ids, mask, M, e, kk, planes, s, loss, counts, tokens, stream);
    else launch_balance_rows<T, 4>(g, ids, mask, M, e, kk, planes, s, loss, counts, tokens, stream);
    XK_CHECK_LAUNCH("balance_rows");
    if (M <= kOneWgRows) return XK_OK;
    hipLaunchKernelGGL((balance_finish<false>), dim3(unsigned(cdiv(E, 16))), dim3(kOneWg), 0, stream, planes, E, k,
                       s, loss, counts, tokens);
  } else {
    const int64_t per = std::max<int64_t>(1, cdiv(M, planes));
    hipLaunchKernelGGL((row_stats<T>), dim3(unsigned(std::min<int64_t>(2048, std::max<int64_t>(cdiv(M, 4), cdiv(E, kThreads))))),
                       dim3(kThreads), 0, stream, g, mask, M, E, s, counts);
    XK_CHECK_LAUNCH("row_stats");
    hipLaunchKernelGGL((balance_columns<T>), dim3(unsigned(cdiv(E, kThreads)), planes), dim3(kThreads), 0, stream, g,
                       ids, mask, M, E, k, per, s, counts);
    XK_CHECK_LAUNCH("balance_columns");
    hipLaunchKernelGGL((balance_finish<true>), dim3(unsigned(cdiv(E, 16))), dim3(kOneWg), 0, stream, planes, E, k,
                       s, loss, counts, tokens);
  }
  XK_CHECK_LAUNCH("balance_finish");
  return XK_OK;
}

template <typename T, int PIECES>
void launch_grad_rows(const T* g, int64_t M, int E, int k, const RouterGrad& a, T* grad, hipStream_t stream) {
  const bool wide = E % 8 == 0 && (reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(grad)) % 16 == 0;
  const dim3 grid(unsigned(std::min<int64_t>(kGradWgs, cdiv(M, kThreads / 16))));
  if (wide)
    hipLaunchKernelGGL((router_grad_rows<T, PIECES, true>), grid, dim3(kThreads), 0, stream, g, M, E, k, a, grad);
  else
    hipLaunchKernelGGL((router_grad_rows<T, PIECES, false>), grid, dim3(kThreads), 0, stream, g, M, E, k, a, grad);
}

template <typename T>
int grad_typed(const void* logits, int64_t M, int64_t E, int64_t k, const RouterGrad& a, void* grad,
               hipStream_t stream) {
  const T* g = static_cast<const T*>(logits);
  T* o = static_cast<T*>(grad);
  if (E <= kFastExperts && k <= kFastTopk) {
    if (E <= 128) launch_grad_rows<T, 1>(g, M, int(E), int(k), a, o, stream);
    else if (E <= 256) launch_grad_rows<T, 2>(g, M, int(E), int(k), a, o, stream);
    else if (E <= 384) launch_grad_rows<T, 3>(g, M, int(E), int(k), a, o, stream);
    else launch_grad_rows<T, 4>(g, M, int(E), int(k), a, o, stream);
  } else {
    hipLaunchKernelGGL((router_grad_any<T>), dim3(unsigned(std::min<int64_t>(4096, cdiv(M, 4)))), dim3(kThreads), 0,
                       stream, g, M, E, k, a, o);
  }
  XK_CHECK_LAUNCH("router_grad");
  return XK_OK;
}

}  // namespace

int64_t balance_workspace_bytes(int64_t M, int64_t E) {
  if (M <= kOneWgRows && E <= kFastExperts) return 0;  // one workgroup
  const int64_t planes = planes_for(std::max<int64_t>(M, 1), E);
  return up(planes * E * 4) * 2 + up(planes * 4) + up(cdiv(E, 16) * 8) + up(4) +
         (E > kFastExperts ? up(M * 8) : 0);
}

int launch_balance_loss(const void* logits, int dtype, int64_t M, int64_t E, const int32_t* ids, int64_t k,
                        const uint8_t* mask, float* loss, int32_t* counts, int32_t* tokens, void* workspace,
                        hipStream_t stream) {
  const int64_t planes = planes_for(std::max<int64_t>(M, 1), E);
  char* w = static_cast<char*>(workspace);
  BalanceScratch s;
  s.sums = reinterpret_cast<float*>(w); w += up(planes * E * 4);
  s.cnt = reinterpret_cast<int32_t*>(w); w += up(planes * E * 4);
  s.rows = reinterpret_cast<int32_t*>(w); w += up(planes * 4);
  s.parts = reinterpret_cast<double*>(w); w += up(cdiv(E, 16) * 8);
  s.ticket = reinterpret_cast<int32_t*>(w); w += up(4);
  s.stat = reinterpret_cast<float*>(w);
  if (dtype == XK_DT_BF16)
    return balance_typed<uint16_t>(logits, ids, mask, M, E, k, s, loss, counts, tokens, stream);
  if (dtype == XK_DT_FP16)
    return balance_typed<_Float16>(logits, ids, mask, M, E, k, s, loss, counts, tokens, stream);
  return balance_typed<float>(logits, ids, mask, M, E, k, s, loss, counts, tokens, stream);
}

int launch_router_backward(const void* logits, int dtype, int64_t M, int64_t E, const int32_t* ids, int64_t k,
                           const uint8_t* mask, const int32_t* counts, const int32_t* tokens, const float* grad_loss,
                           const float* grad_weights, int renorm, void* grad, hipStream_t stream) {
  const RouterGrad a{ids, mask, counts, tokens, grad_loss, grad_weights, renorm};
  if (dtype == XK_DT_BF16) return grad_typed<uint16_t>(logits, M, E, k, a, grad, stream);
  if (dtype == XK_DT_FP16) return grad_typed<_Float16>(logits, M, E, k, a, grad, stream);
  return grad_typed<float>(logits, M, E, k, a, grad, stream);
}

}  // namespace xk
