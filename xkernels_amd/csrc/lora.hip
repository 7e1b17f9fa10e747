// Low-rank adapters of many requests beside a shared projection, and their
// gradients. With a = adapter of row m (rows without one keep the base):
//   h[m] = x[m] A[a]^T                     (shrink:  [M, K] -> [M, r], fp32)
//   y[m] = base[m] + s[a] h[m] B[a]^T      (expand:  [M, r] -> [M, N])
//   g[m] = s[a] dy[m] B[a]                 (shrink over N)
//   dx[m] = g[m] A[a]                      (expand to K)
//   dA[i] = sum_m g[m]^T x[m],  dB[i] = sum_m s[i] dy[m]^T h[m]     (wgrad)
// A [L, r, K], B [L, N, r].
//
// A row's r values cost 2 r (K + N) operations against K + 2 N values of traffic:
// HBM bound for every r taken here (up to 128). So each kernel reads its long rows
// once, in 16-byte pieces straight into MFMA operands, and the adapters' weights,
// which many rows share, come from L2.
//
// Rows are sorted by adapter into tiles of 64 (the library's align); batches of up to
// kFew rows instead let each workgroup find its tile of 16 itself, one launch
// less. Contractions over a long axis are split over workgroups into planes, which
// the next kernel adds in order: no atomics, results do not depend on scheduling.
//
// Precision: bf16 operands, fp32 sums. What stands between two products (h, g) is
// kept in fp32 and enters the second product as the bf16 pair hi + lo (2^-17
// relative): an operand of 16 ranks fills half of an MFMA's 32 contraction
// places, so the pair costs no further instruction. fp32 tensors run on fp32 MFMAs.
#include <algorithm>
#include <type_traits>

#include "mx8.h"

namespace xk {

int64_t align_workspace_bytes(int64_t numel, int num_experts);
int launch_align(const int32_t* ids, int64_t numel, int num_experts, int block_size, const int32_t* emap,
                 int num_global, int32_t* sorted_ids, int32_t* expert_ids, int32_t* num_post,
                 int32_t* expert_offsets, void* workspace, int64_t workspace_bytes, hipStream_t stream,
                 int* clear = nullptr, int nclear = 0, int clear_stride = 1);

namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;      // rows of a sorted tile
constexpr int kFewTile = 16;   // rows of a tile that a workgroup finds itself
constexpr int kFew = 256;      // rows up to which they do (a thread per row)
constexpr int kMaxRank = 128;
constexpr int kCols = 128;     // columns of a wgrad workgroup

// ------------------------------------------------------------- operands ----
// frag: 8 contraction values of one operand row. half: 16 ranks as an operand, of
// which a lane holds 8 (bf16: lanes 32..63 once more, for the pair's other part) or
// 4 (fp32).
template <typename T> struct mm;
template <> struct mm<uint16_t> {
  typedef bf16x8 frag;
  typedef bf16x8 half;
  static constexpr int kHalf = 8;
  __device__ __forceinline__ static f32x4 mma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 mma_half(half a, half b, f32x4 c) { return mma(a, b, c); }
  __device__ __forceinline__ static int rank0(int lane) { return ((lane >> 4) & 1) * 8; }
};
template <> struct mm<float> {
  struct alignas(16) frag { float v[8]; };
  typedef f32x4 half;
  static constexpr int kHalf = 4;
  __device__ __forceinline__ static f32x4 mma(const frag& a, const frag& b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static f32x4 mma_half(half a, half b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static int rank0(int lane) { return (lane >> 4) * 4; }
};

// n values at p (n <= 8; the rest zero). VEC: whole ones are 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ typename mm<T>::frag load_frag(const T* p, int n) {
  typename mm<T>::frag f;
  T* v = reinterpret_cast<T*>(&f);
  if (VEC && n >= 8) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i)
      reinterpret_cast<u32x4*>(&f)[i] = reinterpret_cast<const u32x4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T(0);
  }
  return f;
}
template <typename T>
__device__ __forceinline__ typename mm<T>::frag zero_frag() {
  typename mm<T>::frag f;
#pragma unroll
  for (int i = 0; i < int(sizeof(T)) / 2; ++i) reinterpret_cast<u32x4*>(&f)[i] = u32x4{0, 0, 0, 0};
  return f;
}
// n of a lane's ranks of a half operand at p.
template <typename T, bool VEC>
__device__ __forceinline__ typename mm<T>::half load_half(const T* p, int n) {
  typename mm<T>::half f;
  if (VEC && n >= mm<T>::kHalf) {
    *reinterpret_cast<u32x4*>(&f) = *reinterpret_cast<const u32x4*>(p);
  } else {
    T* v = reinterpret_cast<T*>(&f);
#pragma unroll
    for (int i = 0; i < mm<T>::kHalf; ++i) v[i] = i < n ? p[i] : T(0);
  }
  return f;
}

// What hi leaves of v; 0 where hi is infinite or NaN and says it all.
__device__ __forceinline__ float rest_of(float v, float hi) {
  const float rest = v - hi;
  return fabsf(rest) <= 3.4028234663852886e38f ? rest : 0.f;
}

__device__ __forceinline__ bf16x8 split_part(const float* v, bool low) {
  bf16x8 f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __bf16 hi = static_cast<__bf16>(v[i]);
    f[i] = low ? static_cast<__bf16>(rest_of(v[i], static_cast<float>(hi))) : hi;
  }
  return f;
}

// ----------------------------------------------------------------- rows ----
struct Rows {  // sorted tiles, or (sorted == nullptr) at most kFew rows unsorted
  const int32_t* ids;
  int64_t M;
  int L;
  const int32_t* sorted;
  const int32_t* tile_adapter;
  const int32_t* num_post;
};

// The tile of up to 16 rows that row j leads: rows of one adapter in ascending
// order, cut into sixteens; returns its adapter, or -1 where j leads none. rows[]
// holds M past the last one. Every thread of the workgroup calls it.
__device__ __forceinline__ int few_tile(const Rows& a, int j, int* rows) {
  __shared__ uint64_t masks[kThreads / 64];
  const int t = threadIdx.x, M = int(a.M);
  const int want = a.ids[j];
  if (t < kFewTile) rows[t] = M;
  const bool match = t < M && a.ids[t] == want;
  const uint64_t mine = __ballot(match);
  if ((t & 63) == 0) masks[t >> 6] = mine;
  __syncthreads();
  if (want < 0 || want >= a.L) return -1;
  int before_j = 0, before_t = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const uint64_t m = masks[w];
    const int nj = min(64, max(0, j - 64 * w)), nt = min(64, max(0, t - 64 * w));
    before_j += __popcll(nj == 64 ? m : m & ((uint64_t(1) << nj) - 1));
    before_t += __popcll(nt == 64 ? m : m & ((uint64_t(1) << nt) - 1));
  }
  if (before_j % kFewTile != 0) return -1;
  if (match && before_t >= before_j && before_t < before_j + kFewTile) rows[before_t - before_j] = t;
  __syncthreads();
  return want;
}

// --------------------------------------------------------------- shrink ----
// acc[t] += 16 ranks x 16 rows over [k0, k1): lane's row x + (row lane & 15).
template <typename T, int RT, bool VEC>
__device__ __forceinline__ void shrink_range(const T* xr, bool valid, const T* ar, int64_t K, int r, int64_t k0,
                                             int64_t k1, int lane, f32x4 (&acc)[RT]) {
  const int g8 = (lane >> 4) * 8, rank = lane & 15;
  int64_t k = k0;
#pragma unroll 4
  for (; k + 32 <= k1; k += 32) {
    const typename mm<T>::frag xf = valid ? load_frag<T, VEC>(xr + k + g8, 8) : zero_frag<T>();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const bool in = 16 * t + rank < r;
      const typename mm<T>::frag af = in ? load_frag<T, VEC>(ar + int64_t(16 * t + rank) * K + k + g8, 8) : zero_frag<T>();
      acc[t] = mm<T>::mma(af, xf, acc[t]);
    }
  }
  if (k < k1) {
    const int n = int(min(int64_t(8), max(int64_t(0), k1 - k - g8)));
    const typename mm<T>::frag xf = valid ? load_frag<T, VEC>(xr + k + g8, n) : zero_frag<T>();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const bool in = 16 * t + rank < r;
      const typename mm<T>::frag af = in ? load_frag<T, VEC>(ar + int64_t(16 * t + rank) * K + k + g8, n) : zero_frag<T>();
      acc[t] = mm<T>::mma(af, xf, acc[t]);
    }
  }
}

// planes[s, m, 0 .. 16 RT): the sums over slice s of K. Sorted tiles: a wave per 16
// rows. Few rows: the waves share a tile and a quarter of the slice each.
template <typename T, int RT, bool VEC, bool FEW>
__global__ void __launch_bounds__(kThreads)
lora_shrink(Rows rows, const T* __restrict__ x, int64_t ldx, int64_t K, const T* __restrict__ a, int r,
            int64_t slice, float* __restrict__ planes) {
  constexpr int RP = RT * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t k0 = int64_t(blockIdx.y) * slice, k1 = min(K, k0 + slice);
  f32x4 acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float* plane = planes + int64_t(blockIdx.y) * rows.M * RP;
  if (FEW) {
    __shared__ int tile_rows[kFewTile];
    __shared__ f32x4 red[3][RT][64];
    const int adapter = few_tile(rows, blockIdx.x, tile_rows);
    if (adapter < 0) return;
    const int64_t m = tile_rows[lane & 15];
    const bool valid = m < rows.M;
    const int64_t quarter = slice / 4, w0 = min(k1, k0 + wave * quarter), w1 = min(k1, w0 + quarter);
    shrink_range<T, RT, VEC>(valid ? x + m * ldx : x, valid, a + int64_t(adapter) * r * K, K, r, w0, w1, lane, acc);
    if (wave > 0)
#pragma unroll
      for (int t = 0; t < RT; ++t) red[wave - 1][t][lane] = acc[t];
    __syncthreads();
    if (wave > 0 || !valid) return;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const f32x4 v = ((acc[t] + red[0][t][lane]) + red[1][t][lane]) + red[2][t][lane];
      *reinterpret_cast<f32x4*>(plane + m * RP + 16 * t + (lane >> 4) * 4) = v;
    }
  } else {
    const int64_t pos = int64_t(blockIdx.x) * kTile;
    if (pos >= *rows.num_post) return;
    const int adapter = rows.tile_adapter[blockIdx.x];
    const int64_t m = rows.sorted[pos + wave * 16 + (lane & 15)];
    const bool valid = m < rows.M;
    if (__ballot(valid) == 0) return;
    shrink_range<T, RT, VEC>(valid ? x + m * ldx : x, valid, a + int64_t(adapter) * r * K, K, r, k0, k1, lane, acc);
    if (!valid) return;
#pragma unroll
    for (int t = 0; t < RT; ++t)
      *reinterpret_cast<f32x4*>(plane + m * RP + 16 * t + (lane >> 4) * 4) = acc[t];
  }
}

// Ranks [0, 16 RT) of row m: the planes' sum in order, zeros from r on. pitch: the
// planes' own 16 RT, or r (a caller's [M, r] tensor, one plane).
struct Ranks {
  const float* planes;
  int64_t plane_stride;
  int count, pitch, r;
};
__device__ __forceinline__ f32x4 ranks4(const Ranks& u, int64_t m, int rank) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  const float* p = u.planes + m * u.pitch + rank;
  if (u.pitch % 4 == 0 && rank + 4 <= u.pitch && (reinterpret_cast<uintptr_t>(u.planes) & 15) == 0) {
    for (int s = 0; s < u.count; ++s) v += *reinterpret_cast<const f32x4*>(p + s * u.plane_stride);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (rank + i >= u.r) v[i] = 0.f;  // the planes hold 0 * x there: NaN for an infinite x
  } else {
    for (int s = 0; s < u.count; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (rank + i < u.r) v[i] += p[s * u.plane_stride + i];
  }
  return v;
}

// --------------------------------------------------------------- expand ----
// out[m, n] = base[m, n] + s sum_r h[m, r] b[n, r] for a tile of rows and a chunk of
// columns. The weights are the MFMA's rows and the tile's rows its columns, so a
// lane ends up with consecutive columns of one row; two 16-column products with
// interleaved fours give it 8 of them, 16 bytes of bf16.
template <typename T, int RT, bool VEC, bool FEW>
__global__ void __launch_bounds__(kThreads)
lora_expand(Rows rows, int64_t tiles, Ranks h, const T* __restrict__ b, const float* __restrict__ scaling,
            const T* __restrict__ base, int64_t ldbase, int64_t N, int64_t chunk, T* __restrict__ out,
            float* __restrict__ hidden) {
  constexpr int RP = RT * 16, BM = FEW ? kFewTile : kTile, BT = BM / 16, PITCH = RP + 4;
  __shared__ int tile_rows[BM];
  __shared__ __attribute__((aligned(16))) float hs[BM * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
  const int64_t c0 = int64_t(blockIdx.y) * chunk, c1 = min(N, c0 + chunk);
  int adapter;
  if (FEW) {
    adapter = few_tile(rows, blockIdx.x, tile_rows);
    if (tid == 0 && adapter < 0) {  // a row without an adapter is its own workgroup's
      const int id = rows.ids[blockIdx.x];
      tile_rows[0] = id < 0 || id >= rows.L ? int(blockIdx.x) : int(rows.M);
    }
    __syncthreads();
  } else if (int64_t(blockIdx.x) < tiles) {
    const int64_t pos = int64_t(blockIdx.x) * kTile;
    if (pos >= *rows.num_post) return;
    adapter = rows.tile_adapter[blockIdx.x];
    if (tid < BM) tile_rows[tid] = rows.sorted[pos + tid];
    __syncthreads();
  } else {  // the rows without an adapter among 64 in the batch's order
    adapter = -1;
    if (tid < BM) {
      const int64_t m = (int64_t(blockIdx.x) - tiles) * kTile + tid;
      const int id = m < rows.M ? rows.ids[m] : 0;
      tile_rows[tid] = m < rows.M && (id < 0 || id >= rows.L) ? int(m) : int(rows.M);
    }
    __syncthreads();
  }
  if (adapter < 0) {
    for (int i = 0; i < (FEW ? 1 : BM); ++i) {
      const int64_t m = tile_rows[i];
      if (m >= rows.M) continue;
      if (hidden != nullptr && blockIdx.y == 0)
        for (int j = tid; j < h.r; j += kThreads) hidden[m * h.r + j] = 0.f;
      for (int64_t n = c0 + tid * 8; n < c1; n += kThreads * 8) {
        const int cnt = int(min(int64_t(8), c1 - n));
        const typename mm<T>::frag v = base != nullptr ? load_frag<T, VEC>(base + m * ldbase + n, cnt) : zero_frag<T>();
        T* o = out + m * N + n;
        if (VEC && cnt == 8) {
#pragma unroll
          for (int j = 0; j < int(sizeof(T)) / 2; ++j)
            reinterpret_cast<u32x4*>(o)[j] = reinterpret_cast<const u32x4*>(&v)[j];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < cnt) o[j] = reinterpret_cast<const T*>(&v)[j];
        }
      }
    }
    return;
  }
  const float s = scaling != nullptr ? scaling[adapter] : 1.f;
  for (int q = tid; q < BM * (RP / 4); q += kThreads) {
    const int i = q / (RP / 4), rank = (q % (RP / 4)) * 4;
    const int64_t m = tile_rows[i];
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (m < rows.M) {
      v = ranks4(h, m, rank);
      if (hidden != nullptr && blockIdx.y == 0)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (rank + j < h.r) hidden[m * h.r + rank + j] = v[j];
    }
    *reinterpret_cast<f32x4*>(hs + i * PITCH + rank) = v * s;
  }
  __syncthreads();
  const int rank0 = mm<T>::rank0(lane);
  typename mm<T>::half hf[BT][RT];
  int64_t m[BT];
#pragma unroll
  for (int i = 0; i < BT; ++i) {
    m[i] = tile_rows[16 * i + (lane & 15)];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float* p = hs + (16 * i + (lane & 15)) * PITCH + 16 * t + rank0;
      if constexpr (std::is_same<T, float>::value) {
        hf[i][t] = *reinterpret_cast<const f32x4*>(p);
      } else {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p[j];
        hf[i][t] = split_part(v, g >= 2);
      }
    }
  }
  const T* bw = b + int64_t(adapter) * N * h.r;
  const int nr = 8 * ((lane & 15) >> 2) + (lane & 3);  // this lane's weight row among 32, less 4 for the second product
  for (int64_t n0 = c0 + wave * 32; n0 < c1; n0 += kThreads / 64 * 32) {
    const int64_t nb = n0 + g * 8;
    const int cnt = int(min(int64_t(8), max(int64_t(0), c1 - nb)));
    typename mm<T>::frag bs[BT];
#pragma unroll
    for (int i = 0; i < BT; ++i)
      bs[i] = base != nullptr && m[i] < rows.M && cnt > 0 ? load_frag<T, VEC>(base + m[i] * ldbase + nb, cnt)
                                                           : zero_frag<T>();
    f32x4 acc[BT][2];
#pragma unroll
    for (int i = 0; i < BT; ++i) acc[i][0] = acc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t n = n0 + nr + 4 * e;
        const int left = n < c1 ? h.r - 16 * t - rank0 : 0;
        const typename mm<T>::half wf = load_half<T, VEC>(bw + n * h.r + 16 * t + rank0, left);
#pragma unroll
        for (int i = 0; i < BT; ++i) acc[i][e] = mm<T>::mma_half(wf, hf[i][t], acc[i][e]);
      }
    }
#pragma unroll
    for (int i = 0; i < BT; ++i) {
      if (m[i] >= rows.M || cnt == 0) continue;
      typename mm<T>::frag o;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const T bv = reinterpret_cast<const T*>(&bs[i])[j];
        io<T>::store(reinterpret_cast<T*>(&o) + j, io<T>::load(&bv) + acc[i][j >> 2][j & 3]);
      }
      T* p = out + m[i] * N + nb;
      if (VEC && cnt == 8) {
#pragma unroll
        for (int j = 0; j < int(sizeof(T)) / 2; ++j)
          reinterpret_cast<u32x4*>(p)[j] = reinterpret_cast<const u32x4*>(&o)[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < cnt) p[j] = reinterpret_cast<const T*>(&o)[j];
      }
    }
  }
}

// ------------------------------------------------------------ transpose ----
// out[l, c, r] = in[l, r, c] for the adapters that rows use (offsets differ).
template <typename T>
__global__ void __launch_bounds__(kThreads)
transpose_used(const T* __restrict__ in, int64_t R, int64_t C, int64_t col_tiles, const int32_t* __restrict__ offsets,
               T* __restrict__ out) {
  __shared__ T tile[64][65];
  const int l = blockIdx.y;
  if (offsets[l] == offsets[l + 1]) return;
  const int64_t r0 = int64_t(blockIdx.x) / col_tiles * 64, c0 = int64_t(blockIdx.x) % col_tiles * 64;
  const T* src = in + int64_t(l) * R * C;
  T* dst = out + int64_t(l) * R * C;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  for (int i = ty; i < 64; i += 4)
    if (r0 + i < R && c0 + tx < C) tile[i][tx] = src[(r0 + i) * C + c0 + tx];
  __syncthreads();
  for (int i = ty; i < 64; i += 4)
    if (c0 + i < C && r0 + tx < R) dst[(c0 + i) * R + r0 + tx] = tile[tx][i];
}

// ---------------------------------------------------------------- wgrad ----
// out[i] = sum over adapter i's rows of u[m, :]^T v[m, :]: u the ranks (r of them), v a
// long row (C columns). Positions of the sorted order are cut into windows; a
// workgroup takes one adapter's part of one window and kCols columns. An adapter
// inside one window writes its gradient; one over several leaves a plane for each,
// which wgrad_reduce adds in order (and which writes zeros for adapters without rows).
struct Side {
  Ranks u;
  const float* scaling;    // per adapter, nullable
  const void* v;           // [M, C] of T, or e4m3 bytes with `scales`
  const uint8_t* scales;
  int64_t ldv, C;
  void* out;               // by_rank: [L, r, C]; else [L, C, r]
  int by_rank;
  float* partial;          // [2 windows, 16 RT, C]
};

// Window j's plane for adapter range [off0, off1): at most one adapter that goes
// on past a window starts in it, and at most one comes in from the window before.
__device__ __forceinline__ int64_t plane_of(int64_t off0, int64_t window, int64_t seg) {
  return 2 * window + (off0 >= window * seg ? 1 : 0);
}

template <typename T, bool VEC>
__device__ __forceinline__ typename mm<T>::frag load_row_piece(const Side& sd, int64_t m, int64_t c, int n) {
  if (sd.scales == nullptr) return load_frag<T, VEC>(static_cast<const T*>(sd.v) + m * sd.ldv + c, n);
  typename mm<T>::frag f = zero_frag<T>();
  if (n <= 0) return f;
  const uint8_t* q = static_cast<const uint8_t*>(sd.v) + m * sd.ldv + c;
  __attribute__((aligned(8))) uint8_t b[8];
  if (VEC && n >= 8) {
    *reinterpret_cast<uint64_t*>(b) = *reinterpret_cast<const uint64_t*>(q);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = i < n ? q[i] : 0;
  }
  const float s = mx8_scale(sd.scales[m * cdiv(sd.C, kMx8Block) + c / kMx8Block]);
  float w[8];
  mx8_unpack4(reinterpret_cast<const uint32_t*>(b)[0], w);
  mx8_unpack4(reinterpret_cast<const uint32_t*>(b)[1], w + 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) io<T>::store(reinterpret_cast<T*>(&f) + i, i < n ? w[i] * s : 0.f);
  return f;
}

template <typename T, int RT, bool VEC>
__global__ void __launch_bounds__(kThreads)
lora_wgrad(Side side_a, Side side_b, int a_chunks, const int32_t* __restrict__ sorted,
           const int32_t* __restrict__ offsets, int L, int64_t M, int64_t seg) {
  constexpr int RP = RT * 16, KB = 32, VP = kCols + 8, UP = KB + 8;
  constexpr bool F32 = std::is_same<T, float>::value;
  __shared__ __attribute__((aligned(16))) T vt[KB * VP];
  __shared__ __attribute__((aligned(16))) T ut[(F32 ? 1 : 2) * RP * UP];  // [part][rank][row]
  const bool is_a = int(blockIdx.y) < a_chunks;
  const Side& sd = is_a ? side_a : side_b;
  const int64_t c0 = int64_t(is_a ? blockIdx.y : blockIdx.y - a_chunks) * kCols;
  // pair (adapter, window) number blockIdx.x: adapter i takes the numbers from
  // offsets[i] / seg + i, one per window that it touches
  const int64_t want = blockIdx.x;
  int lo = 0, hi = L - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (offsets[mid] / seg + mid <= want) lo = mid; else hi = mid - 1;
  }
  const int64_t off0 = offsets[lo], off1 = offsets[lo + 1], window = want - lo;
  if (off0 == off1 || window < off0 / seg || window > (off1 - 1) / seg) return;
  const int64_t p0 = max(off0, window * seg), p1 = min(off1, (window + 1) * seg);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
  const float s = sd.scaling != nullptr ? sd.scaling[lo] : 1.f;
  f32x4 acc[2][RT];
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[e][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int64_t p = p0; p < p1; p += KB) {
    if (sorted[p] >= M) break;  // padding ends an adapter's positions
    for (int q = tid; q < KB * (kCols / 8); q += kThreads) {
      const int row = q / (kCols / 8), c = (q % (kCols / 8)) * 8;
      const int64_t m = sorted[p + row];
      const int n = int(min(int64_t(8), max(int64_t(0), sd.C - c0 - c)));
      const typename mm<T>::frag f = m < M ? load_row_piece<T, VEC>(sd, m, c0 + c, n) : zero_frag<T>();
#pragma unroll
      for (int i = 0; i < int(sizeof(T)) / 2; ++i)
        reinterpret_cast<u32x4*>(vt + row * VP + c)[i] = reinterpret_cast<const u32x4*>(&f)[i];
    }
    for (int q = tid; q < KB * (RP / 4); q += kThreads) {
      const int row = q / (RP / 4), rank = (q % (RP / 4)) * 4;
      const int64_t m = sorted[p + row];
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (m < M) v = ranks4(sd.u, m, rank) * s;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (F32) {
          ut[(rank + i) * UP + row] = v[i];
        } else {
          const uint16_t hi16 = f32_to_bf16(v[i]);
          ut[(rank + i) * UP + row] = hi16;
          ut[(RP + rank + i) * UP + row] = f32_to_bf16(rest_of(v[i], bf16_to_f32(hi16)));
        }
      }
    }
    __syncthreads();
    typename mm<T>::frag vf[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        reinterpret_cast<T*>(&vf[e])[j] = vt[(8 * g + j) * VP + wave * 32 + e * 16 + (lane & 15)];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int part = 0; part < (F32 ? 1 : 2); ++part) {
        const typename mm<T>::frag uf = load_frag<T, true>(ut + (part * RP + 16 * t + (lane & 15)) * UP + 8 * g, 8);
#pragma unroll
        for (int e = 0; e < 2; ++e) acc[e][t] = mm<T>::mma(uf, vf[e], acc[e][t]);
      }
    }
    __syncthreads();
  }
  const bool whole = off0 / seg == (off1 - 1) / seg;
  float* plane = whole ? nullptr : sd.partial + plane_of(off0, window, seg) * RP * sd.C;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int64_t c = c0 + wave * 32 + e * 16 + (lane & 15);
    if (c >= sd.C) continue;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rank = 16 * t + 4 * g + i;
        if (rank >= sd.u.r) continue;
        if (whole) {
          T* o = static_cast<T*>(sd.out) + int64_t(lo) * sd.u.r * sd.C;
          io<T>::store(o + (sd.by_rank ? rank * sd.C + c : c * sd.u.r + rank), acc[e][t][i]);
        } else {
          plane[rank * sd.C + c] = acc[e][t][i];
        }
      }
  }
}

// Adds the planes of adapters over several windows; zeros for adapters without rows.
template <typename T>
__global__ void __launch_bounds__(kThreads)
wgrad_reduce(Side side_a, Side side_b, int a_blocks, int RP, const int32_t* __restrict__ offsets, int64_t seg) {
  const bool is_a = int(blockIdx.x) < a_blocks;
  const Side& sd = is_a ? side_a : side_b;
  const int i = blockIdx.y;
  const int64_t off0 = offsets[i], off1 = offsets[i + 1];
  const int64_t w0 = off0 / seg, w1 = off1 > off0 ? (off1 - 1) / seg : w0 - 1;
  if (w1 == w0) return;
  const int64_t q = int64_t(is_a ? blockIdx.x : blockIdx.x - a_blocks) * kThreads + threadIdx.x;
  const int r = sd.u.r;
  if (q >= r * sd.C) return;
  const int64_t rank = q / sd.C, c = q % sd.C;
  float v = 0.f;
  for (int64_t w = w0; w <= w1; ++w) v += sd.partial[(plane_of(off0, w, seg) * RP + rank) * sd.C + c];
  io<T>::store(static_cast<T*>(sd.out) + int64_t(i) * r * sd.C + (sd.by_rank ? q : c * r + rank), v);
}

// ----------------------------------------------------------------- host ----
int64_t up(int64_t x) { return (x + 255) / 256 * 256; }
int rank_tiles(int r) { return r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : 8; }

// Scratch of the sort by adapter.
struct Sort {
  int64_t sorted, tile_adapter, num_post, offsets, inner, inner_bytes, tiles, total;
  Sort(int64_t M, int L) {
    const int64_t most = M + int64_t(L + 1) * (kTile - 1);
    // a tile holds a row, and all but an adapter's last are full
    tiles = std::min<int64_t>(M / kTile + L, M);
    int64_t o = 0;
    sorted = o; o += up(most * 4);
    tile_adapter = o; o += up(cdiv(most, kTile) * 4);
    num_post = o; o += up(4);
    offsets = o; o += up(int64_t(L + 1) * 4);
    inner = o; inner_bytes = align_workspace_bytes(M, L); o += up(inner_bytes);
    total = o;
  }
};

// Slices of a contraction over C: workgroups for every CU a few times over, slices
// long enough to pay for their plane.
struct Slices {
  int64_t len;
  int count;
  Slices(int64_t C, int64_t tiles, bool few) {
    const int64_t want = std::max<int64_t>(1, cdiv(few ? 512 : 1024, std::max<int64_t>(tiles, 1)));
    const int64_t least = few ? 256 : 512;
    const int64_t n = std::max<int64_t>(1, std::min(want, cdiv(C, least)));
    const int64_t unit = few ? 128 : 32;
    len = cdiv(cdiv(C, n), unit) * unit;
    count = int(cdiv(C, len));
  }
};

int64_t chunk_of(int64_t N, int64_t tiles, bool few) {
  const int64_t want = std::max<int64_t>(1, cdiv(few ? 512 : 1024, std::max<int64_t>(tiles, 1)));
  const int64_t n = std::max<int64_t>(1, std::min(want, cdiv(N, few ? 128 : 256)));
  return cdiv(cdiv(N, n), 128) * 128;
}

template <typename F> void with_ranks(int r, F&& f) {
  switch (rank_tiles(r)) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    default: f(std::integral_constant<int, 8>{}); break;
  }
}

bool aligned16(std::initializer_list<const void*> ps) {
  uintptr_t b = 0;
  for (const void* p : ps) b |= reinterpret_cast<uintptr_t>(p);
  return b % 16 == 0;
}

template <typename T>
void run_shrink(const Rows& rows, int64_t tiles, bool few, const T* x, int64_t ldx, int64_t K, const T* a, int r,
                const Slices& sl, float* planes, hipStream_t stream) {
  const bool vec = K % 8 == 0 && ldx % 8 == 0 && aligned16({x, a});
  const dim3 grid(unsigned(few ? rows.M : tiles), sl.count);
  with_ranks(r, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
#define XK_SHRINK(V, F) \
  hipLaunchKernelGGL((lora_shrink<T, RT, V, F>), grid, dim3(kThreads), 0, stream, rows, x, ldx, K, a, r, sl.len, planes)
    if (vec && few) XK_SHRINK(true, true);
    else if (vec) XK_SHRINK(true, false);
    else if (few) XK_SHRINK(false, true);
    else XK_SHRINK(false, false);
#undef XK_SHRINK
  });
}

template <typename T>
void run_expand(const Rows& rows, int64_t tiles, bool few, const Ranks& h, const T* b, const float* scaling,
                const T* base, int64_t ldbase, int64_t N, T* out, float* hidden, hipStream_t stream) {
  const bool vec = N % 8 == 0 && h.r % 8 == 0 && (base == nullptr || ldbase % 8 == 0) && aligned16({b, base, out});
  const int64_t chunk = chunk_of(N, tiles, few);
  const dim3 grid(unsigned(few ? rows.M : tiles + cdiv(rows.M, kTile)), unsigned(cdiv(N, chunk)));
  with_ranks(h.r, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
#define XK_EXPAND(V, F)                                                                                          \
  hipLaunchKernelGGL((lora_expand<T, RT, V, F>), grid, dim3(kThreads), 0, stream, rows, tiles, h, b, scaling, base, \
                     ldbase, N, chunk, out, hidden)
    if (vec && few) XK_EXPAND(true, true);
    else if (vec) XK_EXPAND(true, false);
    else if (few) XK_EXPAND(false, true);
    else XK_EXPAND(false, false);
#undef XK_EXPAND
  });
}

int sort_rows(const int32_t* ids, int64_t M, int L, const Sort& so, char* ws, Rows* rows, hipStream_t stream) {
  rows->sorted = reinterpret_cast<int32_t*>(ws + so.sorted);
  rows->tile_adapter = reinterpret_cast<int32_t*>(ws + so.tile_adapter);
  rows->num_post = reinterpret_cast<int32_t*>(ws + so.num_post);
  return launch_align(ids, M, L, kTile, nullptr, 0, reinterpret_cast<int32_t*>(ws + so.sorted),
                      reinterpret_cast<int32_t*>(ws + so.tile_adapter), reinterpret_cast<int32_t*>(ws + so.num_post),
                      reinterpret_cast<int32_t*>(ws + so.offsets), ws + so.inner, so.inner_bytes, stream);
}

struct ForwardPlan {
  bool few;
  Sort sort;
  int64_t tiles;
  Slices slices;
  int64_t planes, total;
  ForwardPlan(int64_t M, int64_t K, int L, int r)
      : few(M <= kFew), sort(M, L), tiles(few ? std::min<int64_t>(M, M / kFewTile + L) : sort.tiles),
        slices(K, tiles, few) {
    planes = few ? 0 : sort.total;
    total = planes + up(int64_t(slices.count) * M * rank_tiles(r) * 16 * 4);
  }
};

// Windows of the sorted positions: enough for the CUs, none shorter than 256 rows.
struct Windows {
  int64_t seg, count;
  Windows(int64_t M, int L, int64_t chunks) {
    const int64_t most = M + int64_t(L) * (kTile - 1);
    const int64_t n = std::max<int64_t>(1, std::min(cdiv(1024, chunks), cdiv(most, 256)));
    seg = cdiv(cdiv(most, n), kTile) * kTile;
    count = cdiv(most, seg);
  }
};

struct BackwardPlan {
  Sort sort;
  Slices slices;
  int64_t a_chunks, b_chunks;
  Windows win;
  int64_t at, bt, planes, part_a, part_b, total;
  BackwardPlan(int64_t M, int64_t K, int64_t N, int L, int r, int64_t elem)
      : sort(M, L), slices(N, sort.tiles, false), a_chunks(cdiv(K, kCols)), b_chunks(cdiv(N, kCols)),
        win(M, L, a_chunks + b_chunks) {
    const int64_t RP = rank_tiles(r) * 16;
    at = sort.total;
    bt = at + up(int64_t(L) * r * K * elem);
    planes = bt + up(int64_t(L) * r * N * elem);
    part_a = planes + up(int64_t(slices.count) * M * RP * 4);
    part_b = part_a + (win.count > 1 ? up(2 * win.count * RP * K * 4) : 0);
    total = part_b + (win.count > 1 ? up(2 * win.count * RP * N * 4) : 0);
  }
};

template <typename T>
int forward_typed(const T* x, int64_t ldx, int64_t M, int64_t K, const T* a, const T* b, int L, int64_t N, int r,
                  const int32_t* ids, const float* scaling, const T* base, int64_t ldbase, T* out, float* hidden,
                  char* ws, hipStream_t stream) {
  const ForwardPlan plan(M, K, L, r);
  Rows rows{ids, M, L, nullptr, nullptr, nullptr};
  if (!plan.few)
    if (int rc = sort_rows(ids, M, L, plan.sort, ws, &rows, stream)) return rc;
  float* planes = reinterpret_cast<float*>(ws + plan.planes);
  run_shrink<T>(rows, plan.tiles, plan.few, x, ldx, K, a, r, plan.slices, planes, stream);
  XK_CHECK_LAUNCH("lora_shrink");
  const int RP = rank_tiles(r) * 16;
  run_expand<T>(rows, plan.tiles, plan.few, Ranks{planes, M * RP, plan.slices.count, RP, r}, b, scaling, base, ldbase, N,
                out, hidden, stream);
  XK_CHECK_LAUNCH("lora_expand");
  return XK_OK;
}

template <typename T>
int backward_typed(const T* dy, int64_t lddy, const void* x, int64_t ldx, const uint8_t* x_scales, int64_t M, int64_t K,
                   const T* a, const T* b, int L, int64_t N, int r, const int32_t* ids, const float* scaling,
                   const float* hidden, T* dx, T* da, T* db, char* ws, hipStream_t stream) {
  const BackwardPlan plan(M, K, N, L, r, sizeof(T));
  const int RP = rank_tiles(r) * 16;
  Rows rows{ids, M, L, nullptr, nullptr, nullptr};
  if (int rc = sort_rows(ids, M, L, plan.sort, ws, &rows, stream)) return rc;
  const int32_t* offsets = reinterpret_cast<const int32_t*>(ws + plan.sort.offsets);
  T* at = reinterpret_cast<T*>(ws + plan.at);
  T* bt = reinterpret_cast<T*>(ws + plan.bt);
  float* planes = reinterpret_cast<float*>(ws + plan.planes);
  const auto transpose = [&](const T* in, int64_t R, int64_t C, T* out) {
    const int64_t ct = cdiv(C, 64);
    hipLaunchKernelGGL((transpose_used<T>), dim3(unsigned(cdiv(R, 64) * ct), L), dim3(kThreads), 0, stream, in, R, C, ct,
                       offsets, out);
  };
  const Ranks g{planes, M * RP, plan.slices.count, RP, r};
  const Side sa{g, scaling, x, x_scales, ldx, K, da, 1, reinterpret_cast<float*>(ws + plan.part_a)};
  const Side sb{Ranks{hidden, 0, 1, r, r}, scaling, dy, nullptr, lddy, N, db, 0, reinterpret_cast<float*>(ws + plan.part_b)};
  const int64_t ab = cdiv(r * K, kThreads), bb = cdiv(r * N, kThreads);
  const auto reduce = [&]() {
    hipLaunchKernelGGL((wgrad_reduce<T>), dim3(unsigned(ab + bb), L), dim3(kThreads), 0, stream, sa, sb, int(ab), RP,
                       offsets, plan.win.seg);
    XK_CHECK_LAUNCH("wgrad_reduce");
    return XK_OK;
  };
  if (M == 0) return reduce();  // no adapter has rows: zeros
  transpose(b, N, r, bt);
  XK_CHECK_LAUNCH("lora transpose");
  transpose(a, r, K, at);
  XK_CHECK_LAUNCH("lora transpose");
  run_shrink<T>(rows, plan.sort.tiles, false, dy, lddy, N, bt, r, plan.slices, planes, stream);
  XK_CHECK_LAUNCH("lora_shrink");
  run_expand<T>(rows, plan.sort.tiles, false, g, at, scaling, static_cast<const T*>(nullptr), 0, K, dx,
                static_cast<float*>(nullptr), stream);
  XK_CHECK_LAUNCH("lora_expand");
  // (8-byte pieces of 8-bit rows are aligned where 16-byte ones of T are)
  const bool vec = K % 8 == 0 && N % 8 == 0 && ldx % 8 == 0 && lddy % 8 == 0 && aligned16({dy, x});
  const dim3 grid(unsigned(plan.win.count + L), unsigned(plan.a_chunks + plan.b_chunks));
  with_ranks(r, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    if (vec)
      hipLaunchKernelGGL((lora_wgrad<T, RT, true>), grid, dim3(kThreads), 0, stream, sa, sb, int(plan.a_chunks),
                         rows.sorted, offsets, L, M, plan.win.seg);
    else
      hipLaunchKernelGGL((lora_wgrad<T, RT, false>), grid, dim3(kThreads), 0, stream, sa, sb, int(plan.a_chunks),
                         rows.sorted, offsets, L, M, plan.win.seg);
  });
  XK_CHECK_LAUNCH("lora_wgrad");
  return reduce();
}

}  // namespace

int lora_max_rank() { return kMaxRank; }

int64_t lora_workspace_bytes(int64_t M, int64_t K, int64_t L, int64_t r) {
  return ForwardPlan(M, K, int(L), int(r)).total;
}

int64_t lora_backward_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t L, int64_t r, int dtype) {
  return BackwardPlan(M, K, N, int(L), int(r), dtype == XK_DT_FP32 ? 4 : 2).total;
}

int launch_lora(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, const void* a, const void* b, int64_t L,
                int64_t N, int64_t r, const int32_t* ids, const float* scaling, const void* base, int64_t ldbase,
                void* out, float* hidden, void* ws, hipStream_t stream) {
  if (dtype == XK_DT_BF16)
    return forward_typed(static_cast<const uint16_t*>(x), ldx, M, K, static_cast<const uint16_t*>(a),
                         static_cast<const uint16_t*>(b), int(L), N, int(r), ids, scaling,
                         static_cast<const uint16_t*>(base), ldbase, static_cast<uint16_t*>(out), hidden,
                         static_cast<char*>(ws), stream);
  return forward_typed(static_cast<const float*>(x), ldx, M, K, static_cast<const float*>(a),
                       static_cast<const float*>(b), int(L), N, int(r), ids, scaling, static_cast<const float*>(base),
                       ldbase, static_cast<float*>(out), hidden, static_cast<char*>(ws), stream);
}

int launch_lora_backward(const void* dy, int dtype, int64_t lddy, const void* x, int64_t ldx, const uint8_t* x_scales,
                         int64_t M, int64_t K, const void* a, const void* b, int64_t L, int64_t N, int64_t r,
                         const int32_t* ids, const float* scaling, const float* hidden, void* dx, void* da, void* db,
                         void* ws, hipStream_t stream) {
  if (dtype == XK_DT_BF16)
    return backward_typed(static_cast<const uint16_t*>(dy), lddy, x, ldx, x_scales, M, K, static_cast<const uint16_t*>(a),
                          static_cast<const uint16_t*>(b), int(L), N, int(r), ids, scaling, hidden,
                          static_cast<uint16_t*>(dx), static_cast<uint16_t*>(da), static_cast<uint16_t*>(db),
                          static_cast<char*>(ws), stream);
  return backward_typed(static_cast<const float*>(dy), lddy, x, ldx, x_scales, M, K, static_cast<const float*>(a),
                        static_cast<const float*>(b), int(L), N, int(r), ids, scaling, hidden, static_cast<float*>(dx),
                        static_cast<float*>(da), static_cast<float*>(db), static_cast<char*>(ws), stream);
}

}  // namespace xk
