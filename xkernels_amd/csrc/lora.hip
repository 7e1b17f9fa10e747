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
// bf16 is HBM bound for every r taken here (up to 128), fp32, with an eighth of the
// operations a second, to about r = 90 (4,096 x 4,096 -> 4,096, r = 128: 157 us for 216 MB
// and 56 us of products). So each kernel reads its long rows
// once, in 16-byte pieces straight into MFMA operands, and the adapters' weights,
// which many rows share, come from L2.
//
// Rows are sorted by adapter into tiles of 64 (lora_prepare); batches of up to kFew
// rows instead let each workgroup find its tile of 16 itself, one launch less (5 us,
// as much as either of the others). Contractions over a long axis are split over
// workgroups into planes, which the next kernel adds in order: no atomics, results
// do not depend on scheduling.
//
// Precision: bf16 operands, fp32 sums. What stands between two products (h, g) is
// kept in fp32 and enters the second product as the bf16 pair hi + lo (2^-17
// relative, where a bf16 result rounds by 2^-8): an operand of 16 ranks fills half of
// an MFMA's 32 contraction places, so the pair costs no further instruction. fp32
// tensors run on fp32 MFMAs.
//
// Times beside the kernels are of single launches on one MI355X, whose device copies
// run at 5.1 TB/s (1 GiB) to 7 (within the last level's cache).
#include <algorithm>
#include <type_traits>

#include "int4_common.h"
#include "mx8.h"

namespace xk {

namespace {

// Kernels of MFMAs ask for two waves a SIMD at least (the second launch bound), with
// which their sums stay in registers that other instructions reach.
constexpr int kThreads = 256;
constexpr int kXcds = 8;
constexpr int kTile = 64;      // rows of a sorted tile
constexpr int kFewTile = 16;   // rows of a tile that a workgroup finds itself
constexpr int kFew = 256;      // rows up to which they do (a thread per row)
constexpr int kMaxRank = 128;
// Workgroups of a CU asked of the compiler, and counted on by Shares. The unaligned bf16
// forms get there by spilling: 36 bytes a lane for RT = 1, 12 for RT = 4 (4,096 x 4,097 ->
// 2,881, r = 16: 21 us, aligned 12).
template <int RT> constexpr int kExpandPlaces = RT == 1 ? 4 : RT <= 4 ? 3 : 2;
// The same of the weight gradients (fp32, 24 adapters of rank 8 on 2,422 rows, 6,552 and
// 7,168 columns: 53 us with three, 65 with two).
template <typename T, int RT> constexpr int kWgradPlaces = sizeof(T) == 4 && RT == 1 ? 3 : 2;
constexpr int kMaxAdapters = 1024;
constexpr int kSortThreads = 1024;             // and rows a round of the sort
constexpr int64_t kOneLaunchRows = 65536;      // rows up to which each sorting workgroup counts the whole batch
constexpr int kMostChunks = 512;               // else a launch counts first, for at most so many workgroups

// ------------------------------------------------------------- operands ----
// frag: 8 contraction values of one operand row.
template <typename T> struct mm;
template <> struct mm<uint16_t> {
  typedef bf16x8 frag;
  __device__ __forceinline__ static f32x4 mma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct mm<float> {
  struct alignas(16) frag { float v[8]; };
  __device__ __forceinline__ static f32x4 mma(const frag& a, const frag& b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
  }
};

// 8 values at p. VEC: widths are whole aligned pieces, one load and no condition, so
// that loads stay in flight: the caller moves a pointer past the end to one that
// can be read and drops or blanks what comes of it. Else n values and zeros: whole
// pieces unaligned, a row's last one value by value.
template <typename T, bool VEC>
__device__ __forceinline__ typename mm<T>::frag load_frag(const T* p, int64_t n) {
  typename mm<T>::frag f;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i)
      reinterpret_cast<u32x4*>(&f)[i] = reinterpret_cast<const u32x4*>(p)[i];
  } else if (n >= 8) {
    f = load_unaligned<typename mm<T>::frag>(p);
  } else {
    T* v = reinterpret_cast<T*>(&f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T(0);
  }
  return f;
}
// 16 bytes the same way: n values of PER.
template <typename T> __device__ __forceinline__ u32x4 load_piece(const T* p, int64_t n) {
  constexpr int PER = 16 / sizeof(T);
  if (n >= PER) return load_unaligned<u32x4>(p);
  u32x4 w;
#pragma unroll
  for (int i = 0; i < PER; ++i) reinterpret_cast<T*>(&w)[i] = i < n ? p[i] : T(0);
  return w;
}
template <typename T, typename V> __device__ __forceinline__ void store_values(T* p, int64_t n, const V& v) {
  constexpr int ALL = sizeof(V) / sizeof(T);
  if (n >= ALL) {
    store_unaligned(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < ALL; ++i)
      if (i < n) p[i] = reinterpret_cast<const T*>(&v)[i];
  }
}
template <typename T>
__device__ __forceinline__ void blank_unless_frag(bool keep, typename mm<T>::frag& f) {
#pragma unroll
  for (int i = 0; i < int(sizeof(T)) / 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x4& w = reinterpret_cast<u32x4*>(&f)[i];
      w[j] = keep ? w[j] : 0u;
    }
}
template <typename T>
__device__ __forceinline__ typename mm<T>::frag zero_frag() {
  typename mm<T>::frag f;
#pragma unroll
  for (int i = 0; i < int(sizeof(T)) / 2; ++i) reinterpret_cast<u32x4*>(&f)[i] = u32x4{0, 0, 0, 0};
  return f;
}
// v as hi + lo. Where v rounds to an infinity hi is bf16's largest value, so that a finite v
// leaves the difference to lo, and an infinity itself. (By its bits: limits in registers
// cost the expansion of up to 16 ranks 12 bytes a lane of scratch.)
__device__ __forceinline__ bf16x8 split_part(const float* v, bool low) {
  bf16x8 f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint16_t bits = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v[i]));
    bits -= (bits & 0x7FFFu) == 0x7F80u;
    const __bf16 hi = __builtin_bit_cast(__bf16, bits);
    f[i] = low ? static_cast<__bf16>(v[i] - static_cast<float>(hi)) : hi;
  }
  return f;
}

// The expansion's contraction, over ranks. bf16, up to 16 of them: one MFMA takes the
// weights twice, against hi and lo. More: blocks of 32 ranks, the weights' operand
// serves an MFMA with hi and one with lo (half the loads). fp32: blocks of 16.
template <typename T, int RT> struct rank_blocks {
  static constexpr bool kBoth = RT == 1;
  static constexpr int kRanks = kBoth ? 16 : 32, kBlocks = kBoth ? 1 : RT / 2;
  typedef bf16x8 weight;
  struct hidden { bf16x8 part[kBoth ? 1 : 2]; };
  __device__ __forceinline__ static int rank0(int lane) { return (kBoth ? (lane >> 4) & 1 : lane >> 4) * 8; }
  __device__ __forceinline__ static hidden make(const float* p, int lane) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j];
    hidden h;
    if constexpr (kBoth) {
      h.part[0] = split_part(v, lane >= 32);
    } else {
      h.part[0] = split_part(v, false);
      h.part[1] = split_part(v, true);
    }
    return h;
  }
  template <bool VEC> __device__ __forceinline__ static weight load(const uint16_t* p, int n) {
    return load_frag<uint16_t, VEC>(p, n);
  }
  __device__ __forceinline__ static void blank_unless(bool keep, weight& w) { blank_unless_frag<uint16_t>(keep, w); }
  __device__ __forceinline__ static f32x4 mma(const weight& w, const hidden& h, f32x4 c) {
    c = mm<uint16_t>::mma(w, h.part[0], c);
    if constexpr (!kBoth) c = mm<uint16_t>::mma(w, h.part[1], c);
    return c;
  }
  __device__ __forceinline__ static f32x4 mma(const hidden& h, const weight& w, f32x4 c) {
    c = mm<uint16_t>::mma(h.part[0], w, c);
    if constexpr (!kBoth) c = mm<uint16_t>::mma(h.part[1], w, c);
    return c;
  }
};
template <int RT> struct rank_blocks<float, RT> {
  static constexpr int kRanks = 16, kBlocks = RT;
  typedef f32x4 weight;
  typedef f32x4 hidden;
  __device__ __forceinline__ static int rank0(int lane) { return (lane >> 4) * 4; }
  __device__ __forceinline__ static hidden make(const float* p, int) { return *reinterpret_cast<const f32x4*>(p); }
  __device__ __forceinline__ static void blank_unless(bool keep, weight& w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = keep ? w[i] : 0.f;
  }
  template <bool VEC> __device__ __forceinline__ static weight load(const float* p, int n) {
    if constexpr (VEC) return *reinterpret_cast<const f32x4*>(p);
    weight w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = i < n ? p[i] : 0.f;
    return w;
  }
  __device__ __forceinline__ static f32x4 mma(const weight& w, const hidden& h, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], h[j], c, 0, 0, 0);
    return c;
  }
};

// ----------------------------------------------------------------- rows ----
struct Rows {
  const int32_t* ids;
  int64_t M;
  int L;
  // more than kFew rows: sorted by adapter, the rows without one last, each group
  // filled up with M to whole tiles
  const int32_t* sorted;        // [tiles, 64] row numbers
  const int32_t* tile_adapter;  // [tiles]: L for rows without an adapter, -1 for unused tiles
  const int32_t* end;           // positions in use
};

// This workgroup's place in an order in which each XCD has a run of its own (they take
// workgroups in turn): tiles of one adapter, whose weights they read again and
// again, lie next to each other and so share that XCD's L2 (expansion of M = 16,384,
// N = 7,168, 8 adapters of r = 64, 0.9 MB each: 99 us, in launch order 112).
__device__ __forceinline__ unsigned xcd_block() {
  const unsigned xcd = blockIdx.x % kXcds, each = gridDim.x / kXcds, more = gridDim.x % kXcds;
  return xcd * each + min(xcd, more) + blockIdx.x / kXcds;
}

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

// ----------------------------------------------------------------- sort ----
// A stable sort of the rows by adapter into tiles: 5.5 us for 300 rows, 6 for 4,096,
// 9.7 for 16,384, with the weights' transposes 10; chains of dependent steps. Past
// kOneLaunchRows every workgroup walks all parts' counts: 131,072 rows 4.8 + 7.5 us with
// 32 adapters, 4.6 + 56 with 1,024 (128 parts of 1,025). Group L holds the rows without an
// adapter. A workgroup places rounds of 1,024 rows of its part of the batch; what
// lies before it, and the groups' sizes, it counts itself over the whole batch (64 KB
// of ids at 16,384 rows, from L2: one launch where counting apart needs two) up to
// kOneLaunchRows, past which lora_count leaves counts of every part.
struct SortOut {
  int32_t* sorted;
  int32_t* tile_adapter;
  int32_t* offsets;  // [L + 2]: where the groups' positions begin, and their end
  int32_t* counts;   // [chunks, L + 1], with lora_count
  int64_t tiles;
};

__device__ __forceinline__ int group_of(int id, int L) { return id >= 0 && id < L ? id : L; }

// cnt[g] += lanes of group g (those with `in`, the wave's first lane among them if
// any is); runs of one group, as requests' rows are, cost one add.
__device__ __forceinline__ void count_groups(int* cnt, int g, bool in) {
  const uint64_t active = __ballot(in);
  if (active == 0) return;
  const int first = __builtin_amdgcn_readfirstlane(g);
  if (__ballot(in && g == first) == active) {
    if ((threadIdx.x & 63) == 0) atomicAdd(&cnt[first], __popcll(active));
  } else if (in) {
    atomicAdd(&cnt[g], 1);
  }
}

__global__ void __launch_bounds__(kSortThreads)
lora_count(const int32_t* __restrict__ ids, int64_t M, int L, int64_t part, int32_t* __restrict__ counts) {
  __shared__ int cnt[kMaxAdapters + 1];
  for (int g = threadIdx.x; g <= L; g += kSortThreads) cnt[g] = 0;
  __syncthreads();
  const int64_t first = int64_t(blockIdx.x) * part, end = min(M, first + part);
  for (int64_t i = first; i < end; i += kSortThreads) {
    const bool in = i + threadIdx.x < end;
    count_groups(cnt, in ? group_of(ids[i + threadIdx.x], L) : 0, in);
  }
  __syncthreads();
  for (int g = threadIdx.x; g <= L; g += kSortThreads) counts[int64_t(blockIdx.x) * (L + 1) + g] = cnt[g];
}

__device__ __forceinline__ void sort_part(const int32_t* __restrict__ ids, int64_t M, int L, int64_t part, int chunks,
                                          bool counted, SortOut o) {
  __shared__ int total[kMaxAdapters + 1], before[kMaxAdapters + 1], off[kMaxAdapters + 2];
  __shared__ int wave_sum[kSortThreads / 64];
  __shared__ __attribute__((aligned(16))) uint8_t in_wave[(kMaxAdapters + 1) * 16];  // [group][wave]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, G = L + 1;
  const int64_t first = int64_t(blockIdx.x) * part, end = min(M, first + part);
  for (int g = tid; g < G; g += kSortThreads) total[g] = before[g] = 0;
  __syncthreads();
  if (counted) {
    for (int64_t q = tid; q < int64_t(chunks) * G; q += kSortThreads) {
      const int c = int(q / G), g = int(q - int64_t(c) * G), n = o.counts[q];
      if (n == 0) continue;
      atomicAdd(&total[g], n);
      if (c < int(blockIdx.x)) atomicAdd(&before[g], n);
    }
  } else {
    // (part is a multiple of kSortThreads, so a round is before it or not as a whole)
    constexpr int kAhead = 8;
    for (int64_t i0 = 0; i0 < M; i0 += kAhead * kSortThreads) {
      int id[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t i = i0 + j * kSortThreads + tid;
        id[j] = i < M ? ids[i] : 0;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t i = i0 + j * kSortThreads + tid;
        count_groups(i - tid < first ? before : total, group_of(id[j], L), i < M);
      }
    }
  }
  __syncthreads();
  if (!counted) {  // total: what lies before too
    for (int g = tid; g < G; g += kSortThreads) total[g] += before[g];
    __syncthreads();
  }
  // positions of the groups: a prefix sum of the sizes in whole tiles (at most 1,025
  // of them: the last thread takes two)
  int mine = 0;
  const int per = G > kSortThreads ? 2 : 1;
  for (int j = 0; j < per; ++j)
    if (tid * per + j < G) mine += (total[tid * per + j] + kTile - 1) / kTile * kTile;
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(sum, d);
    if (lane >= d) sum += v;
  }
  if (lane == 63) wave_sum[wave] = sum;
  __syncthreads();
  int at = sum - mine;
  for (int w = 0; w < wave; ++w) at += wave_sum[w];
  for (int j = 0; j < per; ++j) {
    const int g = tid * per + j;
    if (g > G) break;
    off[g] = at;
    if (g < G) at += (total[g] + kTile - 1) / kTile * kTile;
  }
  if (per == 1 && tid == G - 1) off[G] = at;
  __syncthreads();
  if (blockIdx.x == 0)
    for (int g = tid; g <= G; g += kSortThreads) o.offsets[g] = off[g];
  // this part's rows
  const int bits = 32 - __clz(L);
  for (int64_t i = first; i < end; i += kSortThreads) {
    for (int q = tid; q < G * 4; q += kSortThreads) reinterpret_cast<uint32_t*>(in_wave)[q] = 0;
    __syncthreads();
    const int64_t row = i + tid;
    const bool in = row < end;
    const int g = in ? group_of(ids[row], L) : 0;
    uint64_t peers = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((g >> b) & 1);
      peers &= (g >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(peers & ((uint64_t(1) << lane) - 1));
    if (in && rank == 0) in_wave[g * 16 + wave] = uint8_t(__popcll(peers));
    __syncthreads();
    if (in) {
      const uint8_t* c = in_wave + g * 16;
      int ahead = 0;
      for (int w = 0; w < wave; ++w) ahead += c[w];
      o.sorted[off[g] + before[g] + ahead + rank] = int(row);
    }
    if (i + kSortThreads >= end) break;
    __syncthreads();
    for (int q = tid; q < G; q += kSortThreads) {
      int n = 0;
      for (int w = 0; w < 16; ++w) n += in_wave[q * 16 + w];
      before[q] += n;
    }
    __syncthreads();
  }
  // the tiles' adapters and what fills them up, the tiles dealt out to the workgroups
  for (int64_t t = int64_t(blockIdx.x) * (kSortThreads / kTile) + tid / kTile; t < o.tiles;
       t += int64_t(chunks) * (kSortThreads / kTile)) {
    const int64_t pos = t * kTile + tid % kTile;
    int g = -1;
    if (pos < off[G]) {
      int lo = 0, hi = G - 1;  // the last group that begins at or before pos holds it (empty ones end there)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= pos) lo = mid; else hi = mid - 1;
      }
      g = lo;
    }
    if (tid % kTile == 0) o.tile_adapter[t] = g;
    if (g < 0 || pos - off[g] >= total[g]) o.sorted[pos] = int(M);
  }
}

// out[l, c, r] = in[l, r, c]. A thread takes 8 values along r, which it writes in 16
// bytes (bf16), unaligned where rows of `out` are no whole pieces.
template <typename T>
__device__ __forceinline__ void transpose_part(const T* __restrict__ in, int64_t L, int64_t R, int64_t C,
                                               T* __restrict__ out, int64_t first, int64_t threads) {
  const int64_t pieces = cdiv(R, 8), total = L * pieces * C;
  for (int64_t q = first; q < total; q += threads) {
    // neighbouring threads: along the shorter of the two, so that the wide side's
    // accesses run through whole lines
    int64_t l = q / (pieces * C), rest = q - l * (pieces * C), c, p;
    if (R < C) {
      c = rest / pieces;
      p = rest - c * pieces;
    } else {
      p = rest / C;
      c = rest - p * C;
    }
    const T* src = in + (l * R + p * 8) * C + c;
    T* dst = out + (l * C + c) * R + p * 8;
    const int n = int(min(int64_t(8), R - p * 8));
    __attribute__((aligned(16))) T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? src[j * C] : T(0);
    if (n == 8 && R % 8 == 0) {
#pragma unroll
      for (int j = 0; j < int(sizeof(T)) / 2; ++j) reinterpret_cast<u32x4*>(dst)[j] = reinterpret_cast<u32x4*>(v)[j];
    } else if (n == 8) {
#pragma unroll
      for (int j = 0; j < int(sizeof(T)) / 2; ++j) store_unaligned(dst + j * 16 / sizeof(T), reinterpret_cast<u32x4*>(v)[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) dst[j] = v[j];
    }
  }
}

// The sort, in `chunks` workgroups; for the backward more of them transpose the
// weights, as the contractions there run along their other axis. (The gradients
// of all adapters are written anyhow, as many bytes.)
template <typename T>
__global__ void __launch_bounds__(kSortThreads)
lora_prepare(const int32_t* __restrict__ ids, int64_t M, int L, int64_t part, int chunks, int counted, SortOut o,
             const T* __restrict__ a, const T* __restrict__ b, int64_t K, int64_t N, int r, T* __restrict__ at,
             T* __restrict__ bt) {
  if (int(blockIdx.x) < chunks) {
    sort_part(ids, M, L, part, chunks, counted != 0, o);
    return;
  }
  const int64_t first = int64_t(blockIdx.x - chunks) * kSortThreads + threadIdx.x;
  const int64_t threads = int64_t(gridDim.x - chunks) * kSortThreads;
  transpose_part<T>(a, L, r, K, at, first, threads);
  transpose_part<T>(b, L, N, r, bt, first, threads);
}

// --------------------------------------------------------------- shrink ----
// planes[s, m, 0 .. 16 RT): the sums over slice s of K for a tile's rows.
//
// An operand loaded straight from memory has its 16 bytes a lane in 16 rows, and the
// vector cache serves 16 bytes of such a load a cycle where neighbouring lanes' 64
// bytes could be one: 9.8 TB/s over the chip. x can be read that way (it is read
// once), the weights beside it, which every 16 rows read again, cannot. So they go
// through LDS, whole rows at a time, for the 16 rows of each of the four waves.
//
// Bound by HBM and the write-backs of what the launches before left in the caches:
// M = 8,192, K = 4,096, r = 16 17.7 us (67 MB, 3.8 TB/s), 4,096 x 7,168, r = 32 14.8
// (59 MB, 4.0), 16,384 x 2,048, r = 64 31 (2.2; 22 where the launch before wrote its
// 235 MB past the caches). A second round of x on its way, or twice the slices,
// measured the same. fp32: 4,096 x 7,168, r = 32 35 (117 MB, 3.4), 8,192 x 4,096, r = 16 58.
template <typename T> constexpr int kStepK = 256 / sizeof(T);  // contraction values a round

template <typename T, int RT, bool VEC>
__global__ void __launch_bounds__(kThreads, 2)
lora_shrink(Rows rows, const T* __restrict__ x, int64_t ldx, int64_t K, const T* __restrict__ a, int r,
            int64_t slice, float* __restrict__ planes) {
  constexpr int RP = RT * 16, KS = kStepK<T>, PER = 16 / sizeof(T), PPR = KS / PER;  // pieces of 16 bytes a row
  constexpr int NA = RP * PPR / kThreads, PITCH = KS + PER, NX = KS / 32;
  __shared__ __attribute__((aligned(16))) T as[2][RP * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g8 = (lane >> 4) * 8;
  const int adapter = rows.tile_adapter[blockIdx.x];
  const int64_t m = rows.sorted[int64_t(blockIdx.x) * kTile + 16 * wave + (lane & 15)];
  if (adapter < 0 || adapter >= rows.L) return;
  const int64_t k0 = int64_t(blockIdx.y) * slice, k1 = min(K, k0 + slice);
  // rows past the batch and ranks past r read others' values in their place: what
  // comes of them stays in their own sums, which are not used
  const T* xr = x + min(m, rows.M - 1) * ldx;
  const T* ar[NA];
#pragma unroll
  for (int j = 0; j < NA; ++j)
    ar[j] = a + (int64_t(adapter) * r + min((tid + j * kThreads) / PPR, r - 1)) * K;
  const int ap = (tid % PPR) * PER;  // this thread's piece of a row (kThreads is a multiple of PPR)
  u32x4 an[NA];
  typename mm<T>::frag xn[NX];
  auto fetch = [&](int64_t k) {
#pragma unroll
    for (int j = 0; j < NA; ++j) {
      if constexpr (VEC) {
        an[j] = *reinterpret_cast<const u32x4*>(ar[j] + min(k + ap, K - PER));
        if (k + ap >= k1) an[j] = u32x4{0, 0, 0, 0};
      } else {
        an[j] = load_piece(ar[j] + k + ap, k1 - k - ap);
      }
    }
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      const int64_t at = k + 32 * j + g8;
      xn[j] = load_frag<T, VEC>(xr + (VEC ? min(at, K - 8) : at), k1 - at);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int j = 0; j < NA; ++j)
      *reinterpret_cast<u32x4*>(&as[buf][((tid + j * kThreads) / PPR) * PITCH + ap]) = an[j];
  };
  f32x4 acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  fetch(k0);
  for (int64_t k = k0, buf = 0; k < k1; k += KS, buf ^= 1) {
    put(int(buf));
    typename mm<T>::frag xc[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      xc[j] = xn[j];
      if (VEC && k + KS > k1) blank_unless_frag<T>(k + 32 * j + g8 < k1, xc[j]);  // (the weights there are 0)
    }
    if (k + KS < k1) fetch(k + KS);
    lds_sync();  // one a round: a buffer is written again two rounds on
#pragma unroll
    for (int j = 0; j < NX; ++j)
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const typename mm<T>::frag af = load_frag<T, true>(&as[buf][(16 * t + (lane & 15)) * PITCH + 32 * j + g8], 8);
        acc[t] = mm<T>::mma(af, xc[j], acc[t]);
      }
  }
  if (m >= rows.M) return;
  float* plane = planes + (int64_t(blockIdx.y) * rows.M + m) * RP + (lane >> 4) * 4;
#pragma unroll
  for (int t = 0; t < RT; ++t) *reinterpret_cast<f32x4*>(plane + 16 * t) = acc[t];
}

// The same for few rows: a 16-row tile, found here, a quarter of the slice a wave,
// weights straight to operands (they are read once); the quarters meet in LDS. A launch
// and its loads' latency: M = 1, K = 7,168, r = 16 4.0 us, 64 rows of 32 adapters 6.2.
template <typename T, int RT, bool VEC>
__global__ void __launch_bounds__(kThreads, 2)
lora_shrink_few(Rows rows, const T* __restrict__ x, int64_t ldx, int64_t K, const T* __restrict__ a, int r,
                int64_t slice, float* __restrict__ planes) {
  constexpr int RP = RT * 16;
  __shared__ int tile_rows[kFewTile];
  __shared__ f32x4 red[3][RT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g8 = (lane >> 4) * 8, rank = lane & 15;
  const int adapter = few_tile(rows, blockIdx.x, tile_rows);
  if (adapter < 0) return;
  const int64_t m = tile_rows[rank], k0 = int64_t(blockIdx.y) * slice, k1 = min(K, k0 + slice);
  const T* xr = x + min(m, rows.M - 1) * ldx + g8;
  const T* ar[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) ar[t] = a + (int64_t(adapter) * r + min(16 * t + rank, r - 1)) * K + g8;
  f32x4 acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t quarter = slice / 4, w0 = min(k1, k0 + wave * quarter), w1 = min(k1, w0 + quarter);
  const int64_t whole = w0 + (w1 - w0) / 32 * 32;
  int64_t k = w0;
  for (; k + 128 <= whole; k += 128) {  // four steps' loads in flight
    typename mm<T>::frag xf[4], af[4][RT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      xf[j] = load_frag<T, VEC>(xr + k + 32 * j, 8);
#pragma unroll
      for (int t = 0; t < RT; ++t) af[j][t] = load_frag<T, VEC>(ar[t] + k + 32 * j, 8);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[t] = mm<T>::mma(af[j][t], xf[j], acc[t]);
  }
  for (; k < whole; k += 32) {
    const typename mm<T>::frag xf = load_frag<T, VEC>(xr + k, 8);
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = mm<T>::mma(load_frag<T, VEC>(ar[t] + k, 8), xf, acc[t]);
  }
  if (whole < w1) {  // K's last, not whole 32
    const int64_t n = w1 - whole - g8, at = VEC && n <= 0 ? -g8 : whole;
    typename mm<T>::frag xf = load_frag<T, VEC>(xr + at, n);
    if (VEC) blank_unless_frag<T>(n > 0, xf);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      typename mm<T>::frag af = load_frag<T, VEC>(ar[t] + at, n);
      if (VEC) blank_unless_frag<T>(n > 0, af);
      acc[t] = mm<T>::mma(af, xf, acc[t]);
    }
  }
  if (wave > 0)
#pragma unroll
    for (int t = 0; t < RT; ++t) red[wave - 1][t][lane] = acc[t];
  __syncthreads();
  if (wave > 0 || m >= rows.M) return;
  float* plane = planes + (int64_t(blockIdx.y) * rows.M + m) * RP + (lane >> 4) * 4;
#pragma unroll
  for (int t = 0; t < RT; ++t)
    *reinterpret_cast<f32x4*>(plane + 16 * t) = ((acc[t] + red[0][t][lane]) + red[1][t][lane]) + red[2][t][lane];
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
    int s = 0;
    for (; s + 8 <= u.count; s += 8) {  // 8 loads in flight, added in order
      f32x4 w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const f32x4*>(p + (s + i) * u.plane_stride);
#pragma unroll
      for (int i = 0; i < 8; ++i) v += w[i];
    }
    for (; s < u.count; ++s) v += *reinterpret_cast<const f32x4*>(p + s * u.plane_stride);
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
// columns.

// s * h of a tile's N rows into LDS, fp32; the first chunk's workgroup leaves h itself.
// With fewer values than threads the planes are dealt out in PARTS, added in order.
template <int RP, int PITCH, int N>
__device__ __forceinline__ void stage_ranks(const Ranks& h, const int* tile_rows, int64_t M, float s, float* hs,
                                            float* hidden) {
  constexpr int VALUES = N * (RP / 4), PARTS = VALUES < kThreads ? kThreads / VALUES : 1;
  __shared__ f32x4 part_sums[PARTS > 1 ? PARTS - 1 : 1][PARTS > 1 ? VALUES : 1];
  f32x4 first = {0.f, 0.f, 0.f, 0.f};
  if (PARTS > 1) {
    const int q = threadIdx.x % VALUES, part = threadIdx.x / VALUES;
    const int64_t m = tile_rows[q / (RP / 4)];
    Ranks mine = h;
    mine.planes += part * h.count / PARTS * h.plane_stride;
    mine.count = (part + 1) * h.count / PARTS - part * h.count / PARTS;
    if (m < M) first = ranks4(mine, m, (q % (RP / 4)) * 4);
    if (part > 0) part_sums[part - 1][q] = first;
    __syncthreads();
  }
  for (int q = threadIdx.x; q < VALUES; q += kThreads) {
    const int i = q / (RP / 4), rank = (q % (RP / 4)) * 4;
    const int64_t m = tile_rows[i];
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (m < M) {
      if (PARTS > 1) {
        v = first;
#pragma unroll
        for (int j = 1; j < PARTS; ++j) v += part_sums[j - 1][q];
      } else {
        v = ranks4(h, m, rank);
      }
      if (hidden != nullptr)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (rank + j < h.r) hidden[m * h.r + rank + j] = v[j];
    }
    *reinterpret_cast<f32x4*>(hs + i * PITCH + rank) = v * s;
  }
}

// Rows without an adapter: the base, or zeros.
template <typename T, bool VEC>
__device__ __forceinline__ void copy_rows(const int* tile_rows, int n_rows, int64_t M, const T* base, int64_t ldbase,
                                          int64_t N, int64_t c0, int64_t c1, T* out, float* hidden, int r) {
  if (hidden != nullptr)
    for (int q = threadIdx.x; q < n_rows * r; q += kThreads)
      if (tile_rows[q / r] < M) hidden[int64_t(tile_rows[q / r]) * r + q % r] = 0.f;
  const int pieces = int(cdiv(c1 - c0, 8)), total = n_rows * pieces;
  for (int q0 = threadIdx.x; q0 < total; q0 += 4 * kThreads) {  // 4 pieces in flight
    typename mm<T>::frag v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = q0 + j * kThreads;
      v[j] = zero_frag<T>();
      if (q >= total || base == nullptr) continue;
      const int64_t m = tile_rows[q / pieces], n = c0 + int64_t(q % pieces) * 8;
      if (m < M) v[j] = load_frag<T, VEC>(base + m * ldbase + n, c1 - n);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = q0 + j * kThreads;
      if (q >= total) continue;
      const int64_t m = tile_rows[q / pieces], n = c0 + int64_t(q % pieces) * 8;
      if (m >= M) continue;
      T* o = out + m * N + n;
      if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T)) / 2; ++i)
          reinterpret_cast<u32x4*>(o)[i] = reinterpret_cast<const u32x4*>(&v[j])[i];
      } else {
        store_values(o, c1 - n, v[j]);
      }
    }
  }
}

// Sorted tiles: 16 rows a wave. The rows are the MFMA's rows and the weights its
// columns, column l of product t being 16 bytes' worth * l + t: a lane ends up with 16
// bytes of consecutive columns of four rows, and 16 lanes with 256 of a row, so base
// and output move in whole lines. The weights of a round go through LDS for all four
// waves (product t's rows together), the next round's on their way meanwhile, as is
// its base: loads and stores leave a wave's counter in order, so neither is waited
// for right after a store. `out` may be `base`: a lane's values of it are read before
// they are written, and no other lane uses them.
//
// HBM bound: M = 16,384, N = 7,168, r = 64 with a base 101 us (470 MB, 4.7 TB/s; a copy
// of as much 87), r = 32 without one 53 (235 MB, 4.4). 4,096 x 4,096, r = 32 19 (67 MB,
// 3.5 TB/s, where copies of that size run at 6.9: a tile's chunks begin with its ranks'
// planes). fp32 35 (134 MB, 3.8).
template <typename T, int RT, bool VEC>
__global__ void __launch_bounds__(kThreads, kExpandPlaces<RT>)
lora_expand(Rows rows, Ranks h, const T* __restrict__ b, int wide, const float* __restrict__ scaling,
            const T* base, int64_t ldbase, int64_t N, int chunks, T* out, float* __restrict__ hidden_out) {
  constexpr int RP = RT * 16, HP = RP + 4, PER = 16 / sizeof(T), BN = 16 * PER;
  constexpr int PPR = RP / PER, WP = RP + PER, NW = BN * PPR / kThreads;  // pieces of a weight row, its pitch, pieces a thread
  constexpr int kWeightBytes = 2 * BN * WP * sizeof(T), kHiddenBytes = kTile * HP * 4;
  constexpr bool kBaseFirst = sizeof(T) == 2;
  typedef rank_blocks<T, RT> rb;
  __shared__ int tile_rows[kTile];
  __shared__ __attribute__((aligned(16))) unsigned char lds[kWeightBytes > kHiddenBytes ? kWeightBytes : kHiddenBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
  const int64_t per_tile = cdiv(N, BN), rounds = int64_t(*rows.end / kTile) * per_tile;
  const unsigned block = xcd_block();
  int64_t at, until;
  if (chunks > 0) {  // a tile's chunk
    const int64_t tile = block / chunks, chunk = block % chunks;
    at = tile * per_tile + per_tile * chunk / chunks;
    until = min(rounds, tile * per_tile + per_tile * (chunk + 1) / chunks);
  } else {
    at = rounds * block / gridDim.x;
    until = rounds * (block + 1) / gridDim.x;
  }
  for (int64_t step; at < until; at += step) {
    const int64_t tile = at / per_tile, c0 = (at - tile * per_tile) * BN;
    step = min(until - at, per_tile - (at - tile * per_tile));
    const int64_t c1 = min(N, c0 + step * BN);
    const int adapter = rows.tile_adapter[tile];
    float* hidden = c0 == 0 ? hidden_out : nullptr;
    __syncthreads();  // the tile before
    if (tid < kTile) tile_rows[tid] = rows.sorted[tile * kTile + tid];
    __syncthreads();
    if (adapter >= rows.L) {
      copy_rows<T, VEC>(tile_rows, kTile, rows.M, base, ldbase, N, c0, c1, out, hidden, h.r);
      continue;
    }
    const T* bw = b + int64_t(adapter) * N * h.r;
    u32x4 wn[NW];
    auto fetch_weights = [&](int64_t n0) {
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        const int q = tid + j * kThreads, rank = (q % PPR) * PER;
        const int64_t n = min(n0 + q / PPR, N - 1);  // (columns past N are not written)
        if (wide) {  // (r a multiple of 8, the weights aligned)
          wn[j] = *reinterpret_cast<const u32x4*>(bw + n * h.r + (rank < h.r ? rank : 0));
          if (rank >= h.r) wn[j] = u32x4{0, 0, 0, 0};
        } else {
          wn[j] = load_piece(bw + n * h.r + rank, h.r - rank);
        }
      }
    };
    T* ws = reinterpret_cast<T*>(lds);
    auto put_weights = [&](int buf) {
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        const int q = tid + j * kThreads, row = q / PPR;
        *reinterpret_cast<u32x4*>(ws + (buf * BN + (row % PER) * 16 + row / PER) * WP + (q % PPR) * PER) = wn[j];
      }
    };
    fetch_weights(c0);
    float* hs = reinterpret_cast<float*>(lds);
    stage_ranks<RP, HP, kTile>(h, tile_rows, rows.M, scaling != nullptr ? scaling[adapter] : 1.f, hs, hidden);
    __syncthreads();
    typename rb::hidden hf[rb::kBlocks];
#pragma unroll
    for (int t = 0; t < rb::kBlocks; ++t)
      hf[t] = rb::make(hs + (16 * wave + (lane & 15)) * HP + rb::kRanks * t + rb::rank0(lane), lane);
    const int64_t col = PER * (lane & 15);
    const T* br[4];
    T* orow[4];
    bool in[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = tile_rows[16 * wave + 4 * g + i];
      in[i] = m < rows.M;
      br[i] = base != nullptr ? base + min(m, rows.M - 1) * ldbase : nullptr;
      orow[i] = out + min(m, rows.M - 1) * N + col;
    }
    u32x4 bn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) bn[i] = u32x4{0, 0, 0, 0};
    auto fetch_base = [&](int64_t n0) {
      if (base == nullptr) return;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (VEC) {
          bn[i] = *reinterpret_cast<const u32x4*>(br[i] + min(n0 + col, N - PER));
        } else {
          bn[i] = load_piece(br[i] + n0 + col, c1 - n0 - col);
        }
      }
    };
    fetch_base(c0);
    __syncthreads();  // hs has been read
    int buf = 0;
    for (int64_t n0 = c0; n0 < c1; n0 += BN, buf ^= 1) {
      put_weights(buf);
      if (n0 + BN < c1) fetch_weights(n0 + BN);
      lds_sync();  // one a round: a buffer is written again two rounds on
      // bf16: from the base on (what its 24 bits lose of small products is far below the
      // result's half step); fp32: the base last, as no later rounding hides that loss
      f32x4 acc[PER];
      u32x4 bc[kBaseFirst ? 1 : 4];
#pragma unroll
      for (int t = 0; t < PER; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T bv = reinterpret_cast<const T*>(&bn[i])[t];
          acc[t][i] = kBaseFirst ? io<T>::load(&bv) : 0.f;
        }
      }
      if constexpr (!kBaseFirst)
#pragma unroll
        for (int i = 0; i < 4; ++i) bc[i] = bn[i];
      if (n0 + BN < c1) fetch_base(n0 + BN);
#pragma unroll
      for (int t = 0; t < PER; ++t)
#pragma unroll
        for (int q = 0; q < rb::kBlocks; ++q) {
          const typename rb::weight wf = *reinterpret_cast<const typename rb::weight*>(
              ws + (buf * BN + t * 16 + (lane & 15)) * WP + rb::kRanks * q + rb::rank0(lane));
          acc[t] = rb::mma(hf[q], wf, acc[t]);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!in[i]) continue;
        u32x4 o;
#pragma unroll
        for (int t = 0; t < PER; ++t) {
          float v = acc[t][i];
          if constexpr (!kBaseFirst) v += __uint_as_float(bc[i][t]);
          io<T>::store(reinterpret_cast<T*>(&o) + t, v);
        }
        if constexpr (VEC) {
          if (n0 + col < c1) *reinterpret_cast<u32x4*>(orow[i] + n0) = o;
        } else {
          store_values(orow[i] + n0, c1 - n0 - col, o);
        }
      }
    }
    }
}

// Few rows: a 16-row tile, found here, the chunk's columns a quarter a wave, weights
// (read once) straight to operands (M = 1, N = 4,096, r = 16: 4.7 us, 64 rows 7). They are the MFMA's rows here; two products with
// interleaved fours give a lane 8 consecutive columns of a row.
template <typename T, int RT, bool VEC>
__global__ void __launch_bounds__(kThreads, 2)
lora_expand_few(Rows rows, Ranks h, const T* __restrict__ b, int wide, const float* __restrict__ scaling,
                const T* base, int64_t ldbase, int64_t N, int64_t chunk, T* out, float* __restrict__ hidden) {
  constexpr int RP = RT * 16, PITCH = RP + 4;
  typedef rank_blocks<T, RT> rb;
  __shared__ int tile_rows[kFewTile];
  __shared__ __attribute__((aligned(16))) float hs[kFewTile * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
  const int64_t c0 = int64_t(blockIdx.y) * chunk, c1 = min(N, c0 + chunk);
  if (blockIdx.y != 0) hidden = nullptr;
  const int adapter = few_tile(rows, blockIdx.x, tile_rows);
  if (adapter < 0) {  // a row without an adapter is its own workgroup's
    const int id = rows.ids[blockIdx.x];
    if (id >= 0 && id < rows.L) return;
    const int mine = int(blockIdx.x);
    copy_rows<T, VEC>(&mine, 1, rows.M, base, ldbase, N, c0, c1, out, hidden, h.r);
    return;
  }
  const int64_t w0 = c0 + wave * (chunk / 4), w1 = min(c1, w0 + chunk / 4);
  const int64_t m = tile_rows[lane & 15];
  const int rank0 = rb::rank0(lane);
  const T* bw = b + int64_t(adapter) * N * h.r + rank0;
  const T* br = base != nullptr ? base + min(m, rows.M - 1) * ldbase : nullptr;
  const int nr = 8 * ((lane & 15) >> 2) + (lane & 3);  // this lane's weight row among 32, less 4 for the second product
  typename rb::weight wf[rb::kBlocks][2];
  typename mm<T>::frag bs = zero_frag<T>();
  auto fetch = [&](int64_t n0) {  // (VEC: columns past N read the last ones again, for columns that are not written)
#pragma unroll
    for (int t = 0; t < rb::kBlocks; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t n = n0 + nr + 4 * e;
        const int left = h.r - rb::kRanks * t - rank0;
        if (wide) wf[t][e] = rb::template load<true>(bw + min(n, N - 1) * h.r + (left > 0 ? rb::kRanks * t : -rank0), 0);
        else wf[t][e] = rb::template load<false>(bw + n * h.r + rb::kRanks * t, n < w1 ? left : 0);
      }
    const int64_t nb = n0 + g * 8;
    if (base != nullptr) bs = load_frag<T, VEC>(br + (VEC ? min(nb, N - 8) : nb), w1 - nb);
  };
  if (w0 < w1) fetch(w0);  // on their way while the ranks are summed
  stage_ranks<RP, PITCH, kFewTile>(h, tile_rows, rows.M, scaling != nullptr ? scaling[adapter] : 1.f, hs, hidden);
  __syncthreads();
  typename rb::hidden hf[rb::kBlocks];
#pragma unroll
  for (int t = 0; t < rb::kBlocks; ++t) hf[t] = rb::make(hs + (lane & 15) * PITCH + rb::kRanks * t + rank0, lane);
  for (int64_t n0 = w0; n0 < w1; n0 += 32) {
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int t = 0; t < rb::kBlocks; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        rb::blank_unless(rb::kRanks * t + rank0 < h.r, wf[t][e]);
        acc[e] = rb::mma(wf[t][e], hf[t], acc[e]);
      }
    typename mm<T>::frag o;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const T bv = reinterpret_cast<const T*>(&bs)[j];
      io<T>::store(reinterpret_cast<T*>(&o) + j, io<T>::load(&bv) + acc[j >> 2][j & 3]);
    }
    if (n0 + 32 < w1) fetch(n0 + 32);
    const int64_t nb = n0 + g * 8, cnt = w1 - nb;
    if (m >= rows.M || cnt <= 0) continue;
    T* p = out + m * N + nb;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < int(sizeof(T)) / 2; ++j)
        reinterpret_cast<u32x4*>(p)[j] = reinterpret_cast<const u32x4*>(&o)[j];
    } else {
      store_values(p, cnt, o);
    }
  }
}

// ---------------------------------------------------------------- wgrad ----
// out[i] = sum over adapter i's rows of u[m, :]^T v[m, :]: u the ranks (r of them), v a
// long row (C columns). Positions of the sorted order are cut into even windows, as
// many as make one workgroup for each place on the chip; a workgroup takes a window,
// adapter by adapter, and a strip of columns. An adapter inside one window writes
// its gradient; one over several leaves a plane for each, which wgrad_reduce adds in
// order (and which writes zeros for adapters without rows).
//
// The contraction runs over rows, along which neither operand is contiguous. u comes
// packed as MFMA operands (lora_pack). v goes through LDS: a wave takes 32 rows at a
// time into registers, the next 32 on their way meanwhile, writes them row by row
// and reads them back transposed (ds_read_b64_tr_b16: 4 rows of a lane's column). A
// wave's tile is its own, so the loop has no barrier; the waves' sums meet at the end.
// Contraction place 8 g + j is row 4 g + j for j < 4, else 16 + 4 g + j - 4: with a
// row pitch of 32 bytes past a multiple of 256 the transposed reads of half a wave then
// fall on distinct banks.
//
// Both gradients in one launch. HBM, two workgroups a CU (their sums and two tiles of
// rows fill the registers): M = 8,192, K = 7,168, N = 4,096, r = 16 43 us (184 MB, 4.3 TB/s;
// fp32 99, 369 MB, 3.7), 16,384 x (7,168 of 8 bits + 2,048), r = 32 49 to 57 (184 MB, 3.2 to
// 3.8); 300 rows of 2 x 2,880, r = 8 5.3.
struct Side {
  const void* packed;      // [positions / 32, parts, RT, 64 lanes, 8] of T: u as operands
  const void* v;           // [M, C] of T, or e4m3 bytes with `scales`
  const uint8_t* scales;
  int64_t ldv, C;
  void* out;               // by_rank: [L, r, C]; else [L, C, r]
  int by_rank;
  float* partial;          // [2 windows, 16 RT, C]
};

template <typename T> constexpr int kParts = std::is_same<T, float>::value ? 1 : 2;

// Packs 64 positions' ranks: blockIdx.y 0 sums g's planes, scales them, keeps the sum
// for the expansion and packs it; 1 packs scaling * hidden. Three dependent loads: 4.4 us
// for 8,192 rows of r = 16, 7 for 16,384 of 32.
template <typename T, int RT>
__global__ void __launch_bounds__(kThreads)
lora_pack(Rows rows, Ranks g, Ranks h, const float* __restrict__ scaling, float* __restrict__ g_sum,
          T* __restrict__ packed_g, T* __restrict__ packed_h) {
  constexpr int RP = RT * 16, PITCH = RP + 1;
  __shared__ float u[kTile * PITCH];
  const int64_t pos = int64_t(blockIdx.x) * kTile;
  const int adapter = rows.tile_adapter[blockIdx.x];
  if (adapter < 0 || adapter >= rows.L) return;
  const bool is_g = blockIdx.y == 0;
  const float s = scaling != nullptr ? scaling[adapter] : 1.f;
  for (int q = threadIdx.x; q < kTile * (RP / 4); q += kThreads) {
    const int i = q / (RP / 4), rank = (q % (RP / 4)) * 4;
    const int64_t m = rows.sorted[pos + i];
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (m < rows.M) {
      v = ranks4(is_g ? g : h, m, rank) * s;
      if (is_g) *reinterpret_cast<f32x4*>(g_sum + m * RP + rank) = v;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) u[i * PITCH + rank + j] = v[j];
  }
  __syncthreads();
  T* out = (is_g ? packed_g : packed_h) + pos * RP * kParts<T>;
  for (int q = threadIdx.x; q < 2 * RP * 4; q += kThreads) {  // a lane's 8 places of a rank, of 2 x 32 rows
    const int p8 = q & 3, rank = (q >> 2) % RP, tile = (q >> 2) / RP;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = u[(32 * tile + 4 * p8 + (j & 3) + (j >> 2) * 16) * PITCH + rank];
    T* o = out + tile * kParts<T> * RP * 32 + ((rank >> 4) * 64 + 16 * p8 + (rank & 15)) * 8;  // lane 16 p8 + rank % 16
    if constexpr (std::is_same<T, float>::value) {
      *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      *reinterpret_cast<bf16x8*>(o) = split_part(v, false);
      *reinterpret_cast<bf16x8*>(o + RP * 32) = split_part(v, true);
    }
  }
}

// Window j's plane for adapter range [off0, off1): at most one adapter that goes
// on past a window starts in it, and at most one comes in from the window before.
__device__ __forceinline__ int plane_of(int off0, int window, int seg) {
  return 2 * window + (off0 >= window * seg ? 1 : 0);
}

// 16 e4m3 bytes (n of them a row's) and their block's scale.
struct Piece8 {
  u32x4 q;
  uint32_t scale;
};

// Column tiles of a wgrad workgroup: 128 accumulators a lane at most.
template <typename T, int RT> constexpr int kColTiles = (std::is_same<T, float>::value ? 4 : 8) / (RT == 8 ? 2 : 1);

template <typename T, int RT, bool VEC, bool Q8>
__device__ __forceinline__ void wgrad_strip(const Side& sd, int r, const int32_t* __restrict__ sorted, int64_t M,
                                            int64_t c0, int p0, int p1, int64_t out_at, float* plane,
                                            unsigned char* lds) {
  constexpr int RP = RT * 16, CT = kColTiles<T, RT>, BC = CT * 16, PITCH = BC + 32 / sizeof(T), PARTS = kParts<T>;
  constexpr bool F32 = std::is_same<T, float>::value;
  constexpr int PER = Q8 ? 16 : 8, PIECES = BC / PER, RPI = 64 / PIECES, NI = 32 / RPI;  // rows an instruction, instructions a tile
  // (opaque: else what every adapter's pass has alike is formed before the loop over
  // them and held in registers through it)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63, wave = tid >> 6, g = lane >> 4;
  T* vt = reinterpret_cast<T*>(lds) + wave * 32 * PITCH;
  f32x4 acc[CT][RT];
#pragma unroll
  for (int e = 0; e < CT; ++e)
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[e][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  typedef typename std::conditional<Q8, Piece8, typename mm<T>::frag>::type piece;
  constexpr int DEPTH = RT <= 2 ? 2 : 1;  // tiles on their way
  piece vs[DEPTH][NI];
  const int64_t col = c0 + (lane % PIECES) * PER;
  const int n = int(min(int64_t(PER), max(int64_t(0), sd.C - col)));
  const int64_t col_at = VEC ? min(col, sd.C - PER) : col;  // (columns past C are not written)
  const int64_t blocks = cdiv(sd.C, kMx8Block);
  uint32_t helds[DEPTH];  // bit i: piece i is a row of the batch's
  auto fetch = [&](int row, piece (&v)[NI], uint32_t& held) __attribute__((always_inline)) {  // the 32 rows whose numbers lanes 0 .. 31 hold
    held = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int64_t m = __shfl(row, i * RPI + lane / PIECES);
      held |= m < M ? 1u << i : 0u;
      const int64_t at = min(m, M - 1);
      if constexpr (Q8) {
        const uint8_t* q = static_cast<const uint8_t*>(sd.v) + at * sd.ldv + col_at;
        if constexpr (VEC) {
          v[i].q = *reinterpret_cast<const u32x4*>(q);
          v[i].scale = sd.scales[at * blocks + col_at / kMx8Block];
        } else {
          v[i].q = load_piece(q, n);
          v[i].scale = n > 0 ? sd.scales[at * blocks + col / kMx8Block] : 127;
        }
      } else {
        v[i] = load_frag<T, VEC>(static_cast<const T*>(sd.v) + at * sd.ldv + col_at, n);
      }
    }
  };
  // row numbers are read a tile ahead of the rows; padding (M) ends an adapter's positions
  constexpr int kStep = 32 * (kThreads / 64);
  int p = p0 + __builtin_amdgcn_readfirstlane(wave) * 32;
  auto row_at = [&](int p) { return p < p1 ? sorted[p + (lane & 31)] : int(M); };
  auto any = [&](int row) { return __builtin_amdgcn_readfirstlane(row) < M; };
  // u's operands of the rows, which up to 32 ranks leave registers to read ahead
  constexpr bool kAhead = PARTS * RT <= 4;
  typename mm<T>::frag uf[PARTS][RT];
  auto fetch_u = [&](int p) __attribute__((always_inline)) {
    const T* up = static_cast<const T*>(sd.packed) + int64_t(p) * RP * PARTS + lane * 8;
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
      for (int t = 0; t < RT; ++t) uf[part][t] = load_frag<T, true>(up + (part * RT + t) * 512, 8);
  };
  // tile d of the DEPTH next: its rows are fetched if there are any
  bool more[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) {
    const int row = row_at(p + d * kStep);
    more[d] = any(row);
    if (more[d]) fetch(row, vs[d], helds[d]);
  }
  int next = row_at(p + DEPTH * kStep);
  if (more[0] && kAhead) fetch_u(p);
  auto tile = [&](piece (&v)[NI], uint32_t& held, bool& again, bool follows) __attribute__((always_inline)) {
    if (!kAhead) fetch_u(p);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      // (rows that fill a tile up have ranks of 0, which an infinity must not meet)
      const bool keep = held >> i & 1;
      T* at = vt + (i * RPI + lane / PIECES) * PITCH + (lane % PIECES) * PER;
      if constexpr (Q8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          typename mm<T>::frag f;
          mx8_unpack8(v[i].q[2 * h], v[i].q[2 * h + 1], v[i].scale, reinterpret_cast<T*>(&f));
          blank_unless_frag<T>(keep, f);
#pragma unroll
          for (int j = 0; j < int(sizeof(T)) / 2; ++j)
            reinterpret_cast<u32x4*>(at + 8 * h)[j] = reinterpret_cast<const u32x4*>(&f)[j];
        }
      } else {
        blank_unless_frag<T>(keep, v[i]);
#pragma unroll
        for (int j = 0; j < int(sizeof(T)) / 2; ++j)
          reinterpret_cast<u32x4*>(at)[j] = reinterpret_cast<const u32x4*>(&v[i])[j];
      }
    }
    wave_lds_fence();
    typename mm<T>::frag uc[PARTS][RT];
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
      for (int t = 0; t < RT; ++t) uc[part][t] = uf[part][t];
    p += kStep;
    again = any(next);
    if (again) fetch(next, v, held);
    if (follows && kAhead) fetch_u(p);
    next = row_at(p + DEPTH * kStep);
#pragma unroll
    for (int e = 0; e < CT; ++e) {
      typename mm<T>::frag vf;
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) vf.v[j] = vt[(4 * g + (j & 3) + (j >> 2) * 16) * PITCH + e * 16 + (lane & 15)];
      } else {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 lds_s4;
        T* at = vt + (4 * g + ((lane & 15) >> 2)) * PITCH + e * 16 + (lane & 3) * 4;
        const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at);
        const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 16 * PITCH));
        vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
      }
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[e][t] = mm<T>::mma(uc[part][t], vf, acc[e][t]);
    }
    wave_lds_fence();
  };
  while (more[0]) {
    if constexpr (DEPTH == 1) {
      bool again;
      tile(vs[0], helds[0], again, any(next));
      more[0] = again;
    } else {
      tile(vs[0], helds[0], more[0], more[1]);
      if (!more[1]) break;
      tile(vs[1], helds[1], more[1], more[0]);
    }
  }
  // the waves' sums, 16 ranks at a time, added in wave order by all threads and written in
  // 16 bytes: of a rank's columns, or (out [L, C, r]) of a column's ranks. (The code of a
  // part is kept short: a short adapter's whole pass is one run through it. 59 rows,
  // r = 64: 15 us, 30 with a quarter of the columns at a time, added by one wave.)
  constexpr int ITEM = 65;  // f32x4s from one column tile's to the next: a rank's pieces fall on all banks
  f32x4* red = reinterpret_cast<f32x4*>(lds);  // [4 waves][CT][ITEM]
  const float* redf = reinterpret_cast<const float*>(lds);
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    if (16 * t >= r) break;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < CT; ++e) red[(wave * CT + e) * ITEM + lane] = acc[e][t];
    __syncthreads();
    if (plane != nullptr || sd.by_rank) {
      constexpr int OUT = 16 / sizeof(T), ROW = BC / OUT;
      const int k = tid / ROW, c_in = tid % ROW * OUT, rank = 16 * t + k;
      const int64_t c = c0 + c_in, at = int64_t(rank) * sd.C + c;
      if (k >= 16 || rank >= r || c >= sd.C) continue;
      float v[OUT];
#pragma unroll
      for (int x = 0; x < OUT; ++x) {
        const int col = c_in + x, item = ((col >> 4) * ITEM + (k >> 2) * 16 + (col & 15)) * 4 + (k & 3);
        v[x] = 0.f;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) v[x] += redf[w * CT * ITEM * 4 + item];
      }
      if (plane != nullptr) {
#pragma unroll
        for (int x = 0; x < OUT; x += 4) store_values(plane + at + x, sd.C - c - x, f32x4{v[x], v[x + 1], v[x + 2], v[x + 3]});
      } else {
        u32x4 o;
#pragma unroll
        for (int x = 0; x < OUT; ++x) io<T>::store(reinterpret_cast<T*>(&o) + x, v[x]);
        store_values(static_cast<T*>(sd.out) + out_at + at, sd.C - c, o);
      }
    } else {
      struct four { T v[4]; };
#pragma unroll 1
      for (int e = wave; e < CT; e += kThreads / 64) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) sum += red[(w * CT + e) * ITEM + lane];
        const int64_t c = c0 + e * 16 + (lane & 15);
        const int rank = 16 * t + 4 * g;
        four o;
#pragma unroll
        for (int x = 0; x < 4; ++x) io<T>::store(&o.v[x], sum[x]);
        if (c < sd.C) store_values(static_cast<T*>(sd.out) + out_at + c * r + rank, r - rank, o);
      }
    }
  }
}

template <typename T, int RT, bool VEC, bool Q8>
__global__ void __launch_bounds__(kThreads, (kWgradPlaces<T, RT>))
lora_wgrad(Side side_a, Side side_b, int r, int a_strips, const int32_t* __restrict__ sorted,
           const int32_t* __restrict__ offsets, int L, int64_t M, int seg) {
  constexpr int RP = RT * 16, BC = kColTiles<T, RT> * 16, PITCH = BC + 32 / sizeof(T);
  constexpr int kTileBytes = 4 * 32 * PITCH * sizeof(T), kRedBytes = 4 * (BC / 16) * 65 * 16;
  __shared__ __attribute__((aligned(16))) unsigned char lds[kTileBytes > kRedBytes ? kTileBytes : kRedBytes];
  const bool is_a = int(blockIdx.y) < a_strips;
  const Side sd = is_a ? side_a : side_b;
  const int64_t c0 = int64_t(is_a ? blockIdx.y : blockIdx.y - a_strips) * BC;
  const int window = blockIdx.x, first = window * seg, end = min(offsets[L], first + seg);
  if (first >= end) return;
  int i = 0, hi = L - 1;  // the last adapter that begins at or before the window
  while (i < hi) {
    const int mid = (i + hi + 1) >> 1;
    if (offsets[mid] <= first) i = mid; else hi = mid - 1;
  }
  for (int off0 = offsets[i], off1; i < L && off0 < end; ++i, off0 = off1) {
    off1 = offsets[i + 1];
    if (off0 == off1) continue;
    const bool whole = off0 >= first && off1 <= first + seg;
    float* plane = whole ? nullptr : sd.partial + int64_t(plane_of(off0, window, seg)) * RP * sd.C;
    const int64_t out_at = int64_t(i) * r * sd.C;
    const int p0 = max(off0, first), p1 = min(off1, end);
    if (Q8 && is_a) wgrad_strip<T, RT, VEC, Q8>(sd, r, sorted, M, c0, p0, p1, out_at, plane, lds);
    else wgrad_strip<T, RT, VEC, false>(sd, r, sorted, M, c0, p0, p1, out_at, plane, lds);
    __syncthreads();  // the LDS of the sums is the next one's tiles
  }
}

// Adds the planes of adapters over several windows; zeros for adapters without rows
// (4 adapters of 8,192 rows, r = 16: 4.8 us).
template <typename T>
__global__ void __launch_bounds__(kThreads)
wgrad_reduce(Side side_a, Side side_b, int r, int a_blocks, int RP, const int32_t* __restrict__ offsets, int seg) {
  const bool is_a = int(blockIdx.x) < a_blocks;
  const Side& sd = is_a ? side_a : side_b;
  const int i = blockIdx.y;
  const int off0 = offsets[i], off1 = offsets[i + 1];
  const int w0 = off0 / seg, w1 = off1 > off0 ? (off1 - 1) / seg : w0 - 1;
  if (w1 == w0) return;
  const int64_t q = int64_t(is_a ? blockIdx.x : blockIdx.x - a_blocks) * kThreads + threadIdx.x;
  if (q >= r * sd.C) return;
  const int64_t rank = q / sd.C, c = q % sd.C;
  float v = 0.f;
  for (int w = w0; w <= w1; ++w) v += sd.partial[(int64_t(plane_of(off0, w, seg)) * RP + rank) * sd.C + c];
  io<T>::store(static_cast<T*>(sd.out) + int64_t(i) * r * sd.C + (sd.by_rank ? q : c * r + rank), v);
}

// ----------------------------------------------------------------- host ----
int64_t up(int64_t x) { return (x + 255) / 256 * 256; }
int rank_tiles(int r) { return r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : 8; }

// Scratch of the sort by adapter.
struct Sort {
  int64_t tiles, part;
  int chunks;
  bool counted;
  int64_t sorted, tile_adapter, offsets, counts, total;
  Sort(int64_t M, int L) {
    // the groups' last tiles hold a row at least, the others are full
    tiles = std::min<int64_t>(M / kTile + L + 1, M);
    counted = M > kOneLaunchRows;
    part = cdiv(cdiv(M, counted ? kMostChunks : kOneLaunchRows / kSortThreads), kSortThreads) * kSortThreads;
    part = std::max<int64_t>(part, kSortThreads);
    chunks = int(std::max<int64_t>(1, cdiv(M, part)));
    int64_t o = 0;
    sorted = o; o += up(tiles * kTile * 4);
    tile_adapter = o; o += up(tiles * 4);
    offsets = o; o += up(int64_t(L + 2) * 4);
    counts = o; o += counted ? up(int64_t(chunks) * (L + 1) * 4) : 0;
    total = o;
  }
};

// Slices of a contraction over C: workgroups for every CU a few times over, slices
// long enough to pay for their plane.
struct Slices {
  int64_t len;
  int count;
  Slices(int64_t C, int64_t tiles, bool few) {
    const int64_t want = std::max<int64_t>(1, cdiv(few ? 512 : 768, std::max<int64_t>(tiles, 1)));
    const int64_t least = few ? 512 : tiles < 64 ? 256 : 1024;
    const int64_t n = std::max<int64_t>(1, std::min(want, cdiv(C, least)));
    const int64_t unit = 128;
    len = cdiv(cdiv(C, n), unit) * unit;
    count = int(cdiv(C, len));
  }
};

// Columns of a few rows' expansion workgroup.
int64_t chunk_of(int64_t N, int64_t tiles) {
  const int64_t n = std::max<int64_t>(1, std::min(cdiv(512, std::max<int64_t>(tiles, 1)), cdiv(N, 128)));
  return cdiv(cdiv(N, n), 128) * 128;
}

// Workgroups of an expansion. The chip has places for 4, 3 or 2 a CU (a tile's
// registers and LDS). Six tiles' worth of them or more: each tile in that many
// chunks, of two rounds at least (a workgroup begins with 3 to 4 us of reading
// its ranks). Else one even share for each place: a second round of workgroups for a
// few left over costs as much as the first (M = 16,384, N = 7,168, r = 64, 265 tiles
// of ragged requests: 128 us in 3 chunks, 109 us in shares).
struct Shares {
  int chunks;
  unsigned grid;
  Shares(int64_t N, int64_t tiles, int r, int64_t elem) {
    const int64_t places = 256 * (rank_tiles(r) == 1 ? 4 : rank_tiles(r) <= 4 ? 3 : 2), per_tile = cdiv(N, 256 / elem);
    const int64_t each = places / tiles;
    chunks = each >= 6 ? int(std::min(each, cdiv(per_tile, 2))) : 0;
    grid = unsigned(chunks > 0 ? tiles * chunks : places);
  }
};

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
#define XK_SHRINK(NAME, V) \
  hipLaunchKernelGGL((NAME<T, RT, V>), grid, dim3(kThreads), 0, stream, rows, x, ldx, K, a, r, sl.len, planes)
    if (vec && few) XK_SHRINK(lora_shrink_few, true);
    else if (vec) XK_SHRINK(lora_shrink, true);
    else if (few) XK_SHRINK(lora_shrink_few, false);
    else XK_SHRINK(lora_shrink, false);
#undef XK_SHRINK
  });
}

template <typename T>
void run_expand(const Rows& rows, int64_t tiles, bool few,  const Ranks& h, const T* b, const float* scaling,
                const T* base, int64_t ldbase, int64_t N, T* out, float* hidden, hipStream_t stream) {
  const bool vec = N % 8 == 0 && (base == nullptr || ldbase % 8 == 0) && aligned16({base, out});
  const int wide = h.r % 8 == 0 && aligned16({b});
  const int64_t chunk = chunk_of(N, tiles);
  const dim3 grid(unsigned(rows.M), unsigned(cdiv(N, chunk)));
  const Shares sh(N, tiles, h.r, sizeof(T));
  with_ranks(h.r, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
#define XK_EXPAND_FEW(V)                                                                                          \
  hipLaunchKernelGGL((lora_expand_few<T, RT, V>), grid, dim3(kThreads), 0, stream, rows, h, b, wide, scaling, base, \
                     ldbase, N, chunk, out, hidden)
#define XK_EXPAND(V)                                                                                               \
  hipLaunchKernelGGL((lora_expand<T, RT, V>), dim3(sh.grid), dim3(kThreads), 0, stream, rows, h, b, wide, scaling, base, \
                     ldbase, N, sh.chunks, out, hidden)
    if (vec && few) XK_EXPAND_FEW(true);
    else if (vec) XK_EXPAND(true);
    else if (few) XK_EXPAND_FEW(false);
    else XK_EXPAND(false);
#undef XK_EXPAND_FEW
#undef XK_EXPAND
  });
}

// Sorts the rows and, with a and b, transposes the weights.
template <typename T>
int prepare(const int32_t* ids, int64_t M, int L, const Sort& so, char* ws, Rows* rows, const T* a, const T* b, int64_t K,
            int64_t N, int r, T* at, T* bt, hipStream_t stream) {
  const SortOut o{reinterpret_cast<int32_t*>(ws + so.sorted), reinterpret_cast<int32_t*>(ws + so.tile_adapter),
                  reinterpret_cast<int32_t*>(ws + so.offsets), reinterpret_cast<int32_t*>(ws + so.counts), so.tiles};
  rows->sorted = o.sorted;
  rows->tile_adapter = o.tile_adapter;
  rows->end = o.offsets + L + 1;
  if (so.counted) {
    hipLaunchKernelGGL(lora_count, dim3(so.chunks), dim3(kSortThreads), 0, stream, ids, M, L, so.part, o.counts);
    XK_CHECK_LAUNCH("lora_count");
  }
  // a transposed piece a thread: latency (2 adapters 3,952 -> 6,867, r = 64: 7.4 us, with
  // two pieces 9.1)
  const int64_t pieces = a == nullptr ? 0 : int64_t(L) * (cdiv(r, 8) * K + cdiv(N, 8) * r);
  const int64_t more = std::min<int64_t>(512, cdiv(pieces, kSortThreads));
  hipLaunchKernelGGL((lora_prepare<T>), dim3(unsigned(so.chunks + more)), dim3(kSortThreads), 0, stream, ids, M, L,
                     so.part, so.chunks, int(so.counted), o, a, b, K, N, r, at, bt);
  XK_CHECK_LAUNCH("lora_prepare");
  return XK_OK;
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

// Windows of the sorted positions: one workgroup for each place that registers and
// LDS leave on the chip, so that all run at once and for as long, a tile at least: short
// adapters then lie in windows of their own rather than one after the other (80 rows of
// 4 adapters, r = 64: 8.1 us, with two tiles at least 13.3).
struct Windows {
  int seg;
  int64_t count;
  Windows(int64_t tiles, int64_t strips, int each) {
    const int64_t places = 256 * each;
    const int64_t n = std::max<int64_t>(1, std::min(places / strips, tiles));
    seg = int(std::max<int64_t>(1, cdiv(tiles, n)) * kTile);
    count = std::max<int64_t>(1, cdiv(tiles * kTile, seg));
  }
};

struct BackwardPlan {
  Sort sort;
  Slices slices;
  int64_t a_strips, b_strips;
  Windows win;
  int64_t at, bt, planes, g_sum, packed_g, packed_h, part_a, part_b, total;
  BackwardPlan(int64_t M, int64_t K, int64_t N, int L, int r, int64_t elem)
      : sort(M, L), slices(N, sort.tiles, false), a_strips(cdiv(K, strip(r, elem))), b_strips(cdiv(N, strip(r, elem))),
        win(sort.tiles, a_strips + b_strips, elem == 4 && r <= 16 ? kWgradPlaces<float, 1> : kWgradPlaces<uint16_t, 1>) {
    const int64_t RP = rank_tiles(r) * 16, packed = sort.tiles * kTile * RP * 4;  // two bf16 or one fp32
    at = sort.total;
    bt = at + up(int64_t(L) * r * K * elem);
    planes = bt + up(int64_t(L) * r * N * elem);
    g_sum = planes + up(int64_t(slices.count) * M * RP * 4);
    packed_g = g_sum + up(M * RP * 4);
    packed_h = packed_g + up(packed);
    part_a = packed_h + up(packed);
    part_b = part_a + (win.count > 1 ? up(2 * win.count * RP * K * 4) : 0);
    total = part_b + (win.count > 1 ? up(2 * win.count * RP * N * 4) : 0);
  }
  static int64_t strip(int r, int64_t elem) {
    return 16 * (rank_tiles(r) == 8 ? 2 : 4) * (elem == 2 ? 2 : 1);
  }
};

template <typename T>
int forward_typed(const T* x, int64_t ldx, int64_t M, int64_t K, const T* a, const T* b, int L, int64_t N, int r,
                  const int32_t* ids, const float* scaling, const T* base, int64_t ldbase, T* out, float* hidden,
                  char* ws, hipStream_t stream) {
  const ForwardPlan plan(M, K, L, r);
  Rows rows{ids, M, L, nullptr, nullptr, nullptr};
  if (!plan.few)
    if (int rc = prepare<T>(ids, M, L, plan.sort, ws, &rows, nullptr, nullptr, K, N, r, nullptr, nullptr, stream))
      return rc;
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
  const int32_t* offsets = reinterpret_cast<const int32_t*>(ws + plan.sort.offsets);
  T* at = reinterpret_cast<T*>(ws + plan.at);
  T* bt = reinterpret_cast<T*>(ws + plan.bt);
  float* planes = reinterpret_cast<float*>(ws + plan.planes);
  if (int rc = prepare<T>(ids, M, L, plan.sort, ws, &rows, a, b, K, N, r, at, bt, stream)) return rc;
  const Ranks g{planes, M * RP, plan.slices.count, RP, r};
  const Ranks h{hidden, 0, 1, r, r};
  float* g_sum = reinterpret_cast<float*>(ws + plan.g_sum);
  T* packed_g = reinterpret_cast<T*>(ws + plan.packed_g);
  T* packed_h = reinterpret_cast<T*>(ws + plan.packed_h);
  const Side sa{packed_g, x, x_scales, ldx, K, da, 1, reinterpret_cast<float*>(ws + plan.part_a)};
  const Side sb{packed_h, dy, nullptr, lddy, N, db, 0, reinterpret_cast<float*>(ws + plan.part_b)};
  const int64_t ab = cdiv(r * K, kThreads), bb = cdiv(r * N, kThreads);
  const auto reduce = [&]() {
    hipLaunchKernelGGL((wgrad_reduce<T>), dim3(unsigned(ab + bb), L), dim3(kThreads), 0, stream, sa, sb, r, int(ab), RP,
                       offsets, plan.win.seg);
    XK_CHECK_LAUNCH("wgrad_reduce");
    return XK_OK;
  };
  if (M == 0) return reduce();  // no adapter has rows: zeros
  run_shrink<T>(rows, plan.sort.tiles, false, dy, lddy, N, bt, r, plan.slices, planes, stream);
  XK_CHECK_LAUNCH("lora_shrink");
  with_ranks(r, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    hipLaunchKernelGGL((lora_pack<T, RT>), dim3(unsigned(plan.sort.tiles), 2), dim3(kThreads), 0, stream, rows, g, h,
                       scaling, g_sum, packed_g, packed_h);
  });
  XK_CHECK_LAUNCH("lora_pack");
  const int64_t unit = x_scales != nullptr ? 16 : 8;  // values of a piece of x
  const bool vec = K % unit == 0 && ldx % unit == 0 && N % 8 == 0 && lddy % 8 == 0 && aligned16({dy, x});
  const dim3 grid(unsigned(plan.win.count), unsigned(plan.a_strips + plan.b_strips));
  with_ranks(r, [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
#define XK_WGRAD(V, Q)                                                                                           \
  hipLaunchKernelGGL((lora_wgrad<T, RT, V, Q>), grid, dim3(kThreads), 0, stream, sa, sb, r, int(plan.a_strips), \
                     rows.sorted, offsets, L, M, plan.win.seg)
    if (vec && x_scales != nullptr) XK_WGRAD(true, true);
    else if (vec) XK_WGRAD(true, false);
    else if (x_scales != nullptr) XK_WGRAD(false, true);
    else XK_WGRAD(false, false);
#undef XK_WGRAD
  });
  XK_CHECK_LAUNCH("lora_wgrad");
  // (after the weights' gradients, which read grad_out while it is still in the last
  // level's cache; dx would push it out)
  run_expand<T>(rows, plan.sort.tiles, false, Ranks{g_sum, 0, 1, RP, r}, at, static_cast<const float*>(nullptr),
                static_cast<const T*>(nullptr), 0, K, dx, static_cast<float*>(nullptr), stream);
  XK_CHECK_LAUNCH("lora_expand");
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
