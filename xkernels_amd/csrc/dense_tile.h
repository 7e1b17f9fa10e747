// The tile kernel of the dense products: out[m, n] = sum_k X(m, k) W(n, k) in fp32, of
// 16-bit operands (bf16 or fp16) or MXFP4 ones, with an epilogue of the caller's.
//
//   * Operands lie k-contiguous (kRowsOfK: [rows, k], as activations and weights do) or
//     k by k (kColumns: [k, rows], as both operands of a weight's gradient do). Either
//     way a chunk of 128 bytes of k a row (64 values of 16 bits, 256 of 4) comes to LDS
//     by direct loads of 16 bytes a lane, double buffered.
//   * LDS holds kRowsOfK chunks as rows of 8 pieces of 16 bytes, permuted by the row's
//     low bits; an operand of v_mfma 16x16x32 (16 bits) or 16x16x128 (4 bits) is one
//     ds_read_b128 either way, so the three formats share every address. kColumns chunks
//     lie as [64 k][rows], units of 16 rows permuted by k, and are read through the
//     transposing ds_read_b64_tr_b16.
//   * The W side is the MFMA's first operand, so a lane's four sums are consecutive n of
//     one m, which the epilogue writes together.
//   * Past a tensor's end the buffer loads give zeros; a row's last chunk, where it is
//     short, is cut off lane by lane.
#pragma once

#include "int4_common.h"

namespace xk {
namespace dense {

enum class Form { kBf16, kFp16, kFp4 };
enum class Lay { kRowsOfK, kColumns };

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 128;     // bytes of k a row and chunk
constexpr int kCut = 1 << 30;   // added to an offset: past every buffer's end (records stay below)

// One side of the product, as the kernel reads it.
struct Side {
  const char* p;       // 16-byte aligned
  int64_t ld;          // bytes from row to row (kRowsOfK) or from k to k (kColumns), a multiple of 16
  int64_t rows;        // m or n
  const uint8_t* s;    // MXFP4: e8m0 scales, 4-byte aligned
  int64_t lds;         // bytes from row to row of s, a multiple of 4
};

__device__ __forceinline__ uint32_t records(int64_t bytes) {
  return bytes <= 0 ? 0u : uint32_t(bytes < kCut ? bytes : int64_t(kCut));
}

// 4-byte form of dma_16: lane i's 4 bytes land at lds + 4 i.
__device__ __forceinline__ void dma_4(i32x4 rsrc, const void* lds, int voff, int soff) {
  const uint32_t m0 = uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)));
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :
               : "s"(m0), "v"(voff), "s"(rsrc), "s"(uniform(soff))
               : "memory", "m0");
}

// Which row of an operand lies in LDS row r of a tile that starts at r0.
struct Straight {
  static constexpr bool kPaired = false;
};
// Gate and up rows of one weight [2 half, k]: of each wave's WAVE rows the first half are gate
// rows, the other the up rows of the same columns, so both sums of a column meet in a lane.
template <int WAVE> struct Paired {
  static constexpr bool kPaired = true;
  static constexpr int kWave = WAVE;
};

template <Form F, Lay L, int ROWS, int WAVES, typename MAP = Straight> struct Loader {
  static constexpr int kBytes = ROWS * kChunk;
  static constexpr int kInstr = ROWS * kChunk / 1024 / WAVES;  // loads of 1 KiB a wave and chunk
  static constexpr int kPitch = L == Lay::kRowsOfK ? kChunk : 2 * ROWS;
  static constexpr int kKRows = 64;  // k of a kColumns chunk
  static_assert(kInstr >= 1, "a wave loads 1 KiB at a time");
  static_assert(L == Lay::kRowsOfK || (F != Form::kFp4 && ROWS >= 128), "kColumns: 16 bits, 8 units a row");

  const char* base;
  const char* base2;  // Paired: the up rows
  int64_t left, left2, step;
  int off[kInstr], piece;

  // `half`: Paired: the rows of a half.
  // `extent`: the side's k, in bytes of a row (kRowsOfK) or a number (kColumns)
  __device__ __forceinline__ void init(const Side& s, int64_t r0, int64_t extent, int64_t k0, int wave, int lane,
                                       int64_t half = 0) {
    if constexpr (L == Lay::kRowsOfK) {
      piece = (lane & 7) ^ (lane >> 3);
      base = s.p + r0 * s.ld + k0 * kChunk;
      const int64_t rows = MAP::kPaired ? half : s.rows;
      left = (rows - 1 - r0) * s.ld + extent - k0 * kChunk;
      if constexpr (MAP::kPaired) {
        base2 = base + half * s.ld;
        left2 = left;
      }
      step = kChunk;
#pragma unroll
      for (int i = 0; i < kInstr; ++i) {
        int row = (wave * kInstr + i) * 8 + (lane >> 3);
        if constexpr (MAP::kPaired) row = row / MAP::kWave * (MAP::kWave / 2) + row % (MAP::kWave / 2);
        off[i] = int(row * s.ld) + piece * 16;
      }
    } else {
      piece = 0;
      base = s.p + r0 * 2 + k0 * kKRows * s.ld;
      left = (extent - 1 - k0 * kKRows) * s.ld + (s.rows - r0) * 2;
      step = kKRows * s.ld;
#pragma unroll
      for (int i = 0; i < kInstr; ++i) {
        const int at = ((wave * kInstr + i) * 64 + lane) * 16, k = at / kPitch, unit = at % kPitch / 32;
        off[i] = int(k * s.ld) + (unit ^ flip(k)) * 32 + (at & 16);
      }
    }
  }
  // which way the 32-byte units of k are permuted: the 8 k of a half wave's transposing read
  // (0 .. 3 and 8 .. 11 of 16) fall on all banks
  __device__ __forceinline__ static int flip(int k) { return (k & 3) | ((k >> 1) & 4); }

  // Issues the next chunk's loads to `lds`; `cut` (kRowsOfK): pieces left of a short chunk, else 8.
  __device__ __forceinline__ void issue(char* lds, int wave, int cut) {
    const i32x4 r = make_rsrc(base, records(left));
    i32x4 r2;
    if constexpr (MAP::kPaired) r2 = make_rsrc(base2, records(left2));
#pragma unroll
    for (int i = 0; i < kInstr; ++i) {
      int o = off[i];
      if (L == Lay::kRowsOfK && cut < 8) o |= piece >= cut ? kCut : 0;
      char* at = lds + (wave * kInstr + i) * 1024;
      if constexpr (MAP::kPaired) {
        const bool up = (wave * kInstr + i) * 8 % MAP::kWave >= MAP::kWave / 2;
        dma_16(up ? r2 : r, at, o, 0);
      } else {
        dma_16(r, at, o, 0);
      }
    }
    base += step;
    left -= step;
    if constexpr (MAP::kPaired) {
      base2 += step;
      left2 -= step;
    }
  }
};

// The scales of an MXFP4 operand: 8 bytes a row and chunk.
template <int ROWS, int WAVES> struct ScaleLoader {
  static constexpr int kBytes = ROWS * 8;
  static constexpr int kTotal = ROWS / 32;  // loads of 256 bytes
  static constexpr int kInstr = (kTotal + WAVES - 1) / WAVES;
  const uint8_t* base;
  int64_t left;
  int off[kInstr], word;
  __device__ __forceinline__ void init(const Side& s, int64_t r0, int64_t blocks, int64_t k0, int wave, int lane) {
    word = lane & 1;
    base = s.s + r0 * s.lds + k0 * 8;
    left = (s.rows - 1 - r0) * s.lds + (blocks + 3) / 4 * 4 - k0 * 8;
#pragma unroll
    for (int i = 0; i < kInstr; ++i) off[i] = int(((wave * kInstr + i) * 32 + (lane >> 1)) * s.lds) + word * 4;
  }
  // `cut`: words left of a short chunk, else 2
  __device__ __forceinline__ void issue(char* lds, int wave, int cut) {
    const i32x4 r = make_rsrc(base, records(left));
#pragma unroll
    for (int i = 0; i < kInstr; ++i)
      if (wave * kInstr + i < kTotal) dma_4(r, lds + (wave * kInstr + i) * 256, off[i] | (word >= cut ? kCut : 0), 0);
    base += 8;
    left -= 8;
  }
};

// One operand fragment: 16 rows, step s of 2 of a chunk.
template <Form F, Lay L, int ROWS> struct Reader {
  static constexpr int kPitch = L == Lay::kRowsOfK ? kChunk : 2 * ROWS;
  int at0, at1;  // kRowsOfK: of each step; kColumns: at0, to which a fragment's unit is xored
  __device__ __forceinline__ void init(int row0, int lane) {
    const int c = lane & 15, q = lane >> 4;
    if constexpr (L == Lay::kRowsOfK) {
      // 16 bits: step s reads piece 4 s + q, 4 bits: block 2 q + s (any order of k will do that
      // both operands share)
      const int p0 = F == Form::kFp4 ? 2 * q : q, p1 = F == Form::kFp4 ? 2 * q + 1 : 4 + q;
      at0 = (row0 + c) * kChunk + ((p0 ^ (c & 7)) << 4);
      at1 = (row0 + c) * kChunk + ((p1 ^ (c & 7)) << 4);
    } else {
      at0 = (8 * q + (c >> 2)) * kPitch + (((row0 >> 4) ^ ((c >> 2) | (q & 1) << 2)) << 5) + (c & 3) * 8;
      at1 = 0;
    }
  }
  // fragment t (row0 + 16 t .. + 15); row0 is a multiple of 16 times the wave's fragments
  __device__ __forceinline__ u32x4 read(const char* lds, int t, int s) const {
    if constexpr (L == Lay::kRowsOfK) {
      return *reinterpret_cast<const u32x4*>(lds + (s ? at1 : at0) + t * 16 * kChunk);
    } else {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4 lds_s4;
      const char* p = lds + (at0 ^ (t << 5)) + s * 32 * kPitch;
      const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
      const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 4 * kPitch));
      return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

template <Form F> __device__ __forceinline__ f32x4 mma(u32x4 w, u32x4 x, f32x4 acc) {
  if constexpr (F == Form::kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), acc, 0,
                                                  0, 0);
}
// 4 bits; byte S of each scale word
template <int S> __device__ __forceinline__ f32x4 mma4(u32x4 w, uint32_t ws, u32x4 x, uint32_t xs, f32x4 acc) {
  const i32x8 a = {int(w[0]), int(w[1]), int(w[2]), int(w[3]), 0, 0, 0, 0};
  const i32x8 b = {int(x[0]), int(x[1]), int(x[2]), int(x[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, S, int(ws), S, int(xs));
}

// What a launch works on. Grid: tiles of the product, one after the other.
struct Product {
  Side x, w;
  int64_t M, N;      // N: of the output's columns (Paired: those of a half)
  int64_t k_bytes;   // of a row of a kRowsOfK side (a multiple of 16)
  int64_t k_rows;    // of a kColumns side: the number of k
  int64_t blocks;    // MXFP4: blocks of a row
  int chunks;        // of k
  int tiles_m, tiles_n;
};

// Tile `id` of the launch: XCD i (workgroups go round the 8 of them) takes a run of
// consecutive tiles, ordered in bands of kBand row tiles, so that its 4 MB of L2 sees few
// rows of X and W at a time.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_of(int id, int total, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int xcd = id & 7, local = id >> 3, share = total >> 3, rest = total & 7;
  const int t = xcd * share + min(xcd, rest) + local;
  const int band = t / (kBand * tiles_n), in = t - band * kBand * tiles_n;
  const int height = min(kBand, tiles_m - band * kBand);
  tn = in / height;
  tm = band * kBand + in - tn * height;
}

// EPI: struct with `template <int WT, int XT> void operator()(const f32x4 (&acc)[WT][XT], int64_t m, int64_t n, int lane)`:
// the sums of the wave's rows m .. and columns n .. (fragment t of either side 16 t further, Paired: n of
// the gate's first half of the fragments).
template <Form F, Lay LX, Lay LW, int BM, int BN, int WM, int WN, bool PAIRED, typename EPI>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64)
dense_tile(Product p, EPI epi) {
  constexpr int WAVES = BM / WM * (BN / WN), XT = WM / 16, WT = WN / 16;
  constexpr bool FP4 = F == Form::kFp4;
  using XLoad = Loader<F, LX, BM, WAVES>;
  using WLoad = Loader<F, LW, BN, WAVES, std::conditional_t<PAIRED, Paired<WN>, Straight>>;
  using XScale = ScaleLoader<BM, WAVES>;
  using WScale = ScaleLoader<BN, WAVES>;
  constexpr int STAGE = XLoad::kBytes + WLoad::kBytes + (FP4 ? XScale::kBytes + WScale::kBytes : 0);
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  const int lane = threadIdx.x & 63, wave = uniform(int(threadIdx.x) >> 6);
  const int wn = wave % (BN / WN), wm = wave / (BN / WN);
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, tm, tn);
  const int64_t m0 = int64_t(tm) * BM, n0 = int64_t(tn) * (PAIRED ? BN / 2 : BN);

  XLoad xl;
  WLoad wl;
  xl.init(p.x, m0, LX == Lay::kRowsOfK ? p.k_bytes : p.k_rows, 0, wave, lane);
  wl.init(p.w, n0, LW == Lay::kRowsOfK ? p.k_bytes : p.k_rows, 0, wave, lane, p.N);
  XScale xsl;
  WScale wsl;
  if constexpr (FP4) {
    xsl.init(p.x, m0, p.blocks, 0, wave, lane);
    wsl.init(p.w, n0, p.blocks, 0, wave, lane);
  }
  auto issue = [&](int i) __attribute__((always_inline)) {
    char* at = lds + (i & 1) * STAGE;
    const int64_t left = LX == Lay::kRowsOfK ? p.k_bytes - int64_t(i) * kChunk : kChunk;
    const int cut = left < kChunk ? int(left >> 4) : 8;
    xl.issue(at, wave, cut);
    wl.issue(at + XLoad::kBytes, wave, cut);
    if constexpr (FP4) {
      const int words = left < kChunk ? int((p.blocks - int64_t(i) * 8 + 3) >> 2) : 2;
      xsl.issue(at + XLoad::kBytes + WLoad::kBytes, wave, words);
      wsl.issue(at + XLoad::kBytes + WLoad::kBytes + XScale::kBytes, wave, words);
    }
  };
  Reader<F, LX, BM> xr;
  Reader<F, LW, BN> wr;
  xr.init(wm * WM, lane);
  wr.init(wn * WN, lane);

  f32x4 acc[WT][XT];
#pragma unroll
  for (int a = 0; a < WT; ++a)
#pragma unroll
    for (int b = 0; b < XT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (p.chunks > 0) issue(0);
  for (int i = 0; i < p.chunks; ++i) {
    // chunk i has landed, and every wave has read chunk i - 1, whose place chunk i + 1 takes
    XK_WAIT_VMCNT(0);
    lds_sync();
    if (i + 1 < p.chunks) issue(i + 1);
    const char* xb = lds + (i & 1) * STAGE;
    const char* wb = xb + XLoad::kBytes;
    uint32_t xs[XT], ws[WT];
    if constexpr (FP4) {
      const char* sb = wb + WLoad::kBytes + (lane & 15) * 8 + (lane >> 4) * 2;
#pragma unroll
      for (int b = 0; b < XT; ++b) xs[b] = *reinterpret_cast<const uint16_t*>(sb + (wm * WM + b * 16) * 8);
#pragma unroll
      for (int a = 0; a < WT; ++a)
        ws[a] = *reinterpret_cast<const uint16_t*>(sb + XScale::kBytes + (wn * WN + a * 16) * 8);
    }
    static_for<2>([&](auto S) __attribute__((always_inline)) {
      constexpr int s = decltype(S)::value;
      u32x4 wf[WT], xf[XT];
#pragma unroll
      for (int a = 0; a < WT; ++a) wf[a] = wr.read(wb, a, s);
#pragma unroll
      for (int b = 0; b < XT; ++b) xf[b] = xr.read(xb, b, s);
#pragma unroll
      for (int b = 0; b < XT; ++b)
#pragma unroll
        for (int a = 0; a < WT; ++a) {
          if constexpr (FP4) acc[a][b] = mma4<s>(wf[a], ws[a], xf[b], xs[b], acc[a][b]);
          else acc[a][b] = mma<F>(wf[a], xf[b], acc[a][b]);
        }
    });
  }
  epi(acc, m0 + wm * WM, n0 + wn * (PAIRED ? WN / 2 : WN), lane);
}

template <Form F, Lay LX, Lay LW, int BM, int BN, int WM, int WN, bool PAIRED, typename EPI>
void launch_tile(Product p, const EPI& epi, hipStream_t stream) {
  p.tiles_m = int(cdiv(p.M, BM));
  p.tiles_n = int(cdiv(p.N, PAIRED ? BN / 2 : BN));
  auto* fn = &dense_tile<F, LX, LW, BM, BN, WM, WN, PAIRED, EPI>;
  hipLaunchKernelGGL(fn, dim3(p.tiles_m * p.tiles_n), dim3(BM / WM * (BN / WN) * 64), 0, stream, p, epi);
}

}  // namespace dense
}  // namespace xk
