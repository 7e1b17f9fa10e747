// The tile kernel of the dense products: out[m, n] = sum_k X(m, k) W(n, k) in fp32, of
// 16-bit operands (bf16 or fp16) or MXFP4 ones, with an epilogue of the caller's.
//
//   * Operands lie k-contiguous (kRowsOfK: [rows, k], as activations and weights do) or
//     k by k (kColumns: [k, rows], as both operands of a weight's gradient do). Either
//     way a chunk of 128 bytes of k a row (64 values of 16 bits, 256 of 4) comes to LDS
//     by direct loads of 16 bytes a lane.
//   * LDS holds kRowsOfK chunks as rows of 8 pieces of 16 bytes, permuted by the row's
//     low bits; an operand of v_mfma 16x16x32 (16 bits) or 16x16x128 (4 bits) is one
//     ds_read_b128 either way, so the three formats share every address. kColumns chunks
//     lie as [64 k][rows], units of 16 rows permuted by k, and are read through the
//     transposing ds_read_b64_tr_b16. Neither has bank conflicts.
//   * A wave owns 64 rows x BN / 2 (or BN / 4) columns. While it multiplies one half of a
//     chunk it reads the other half's fragments, W's into the registers that are done
//     with, so the matrix unit waits for LDS only behind a barrier, of which there is one a
//     chunk; and it issues the loads of later chunks between the products. X has three
//     places in LDS and W two (160 KB at 256 x 256), so loads stay in flight across the
//     barrier.
//   * A workgroup stays for tile after tile and sends for the next one's first chunks before
//     it writes a tile out.
//   * The W side is the MFMA's first operand, so a lane's four sums are consecutive n of
//     one m, which the epilogue writes together.
//   * Past a tensor's end the buffer loads give zeros; a row's last chunk, where it is
//     short, is cut off lane by lane. Behind the last chunk the loop loads nothing in the
//     same way, so it has one form.
#pragma once

#include <algorithm>

#include "int4_common.h"

namespace xk {
namespace dense {

enum class Form { kBf16, kFp16, kFp4 };
enum class Lay { kRowsOfK, kColumns };

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 128;    // bytes of k a row and chunk: two MFMAs'
constexpr int kCut = 1 << 30;  // added to an offset: past every buffer's end (records stay below)

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

// Direct-to-LDS loads: lane i's 16 (4) bytes from voff + soff land at LDS address `lds` + 16 i
// (4 i), zeros where they are past the buffer. Inline assembly with its wait states, as dma_16 is,
// and the LDS address as the number that it is. The kernel waits for them itself.
__device__ __forceinline__ void to_lds_16(i32x4 rsrc, uint32_t lds, int voff, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(uniform(lds)), "v"(voff), "s"(rsrc), "s"(uniform(soff))
               : "memory", "m0");
}
__device__ __forceinline__ void to_lds_4(i32x4 rsrc, uint32_t lds, int voff, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :
               : "s"(uniform(lds)), "v"(voff), "s"(rsrc), "s"(uniform(soff))
               : "memory", "m0");
}

// Chunks [first, end) of a slice of k.
struct Range {
  int first, end;
};
__device__ __forceinline__ Range range_of(int slice, int slices, int chunks) {
  const int share = chunks / slices, rest = chunks - share * slices;
  const int first = slice * share + min(slice, rest);
  return Range{first, first + share + (slice < rest)};
}

// Loads one side's chunks. PAIR: the rows of W are gate and up rows of one weight [2 half, k]: of
// each PAIR rows in LDS (a wave's) the first half are gate rows, the other the up rows of
// the same columns, so both sums of a column meet in a lane. 0: rows as they come.
template <Form F, Lay L, int ROWS, int WAVES, int PAIR = 0> struct Loader {
  static constexpr int kBytes = ROWS * kChunk;
  static constexpr int kInstr = ROWS * kChunk / 1024 / WAVES;  // loads of 1 KiB a wave and chunk
  static constexpr int kPitch = L == Lay::kRowsOfK ? kChunk : 2 * ROWS;
  static constexpr int kKRows = 64;  // k of a kColumns chunk
  static_assert(kInstr * 1024 * WAVES == kBytes, "a wave loads 1 KiB at a time");
  static_assert(L == Lay::kRowsOfK || (F != Form::kFp4 && kInstr == 4 && (ROWS == 256 || ROWS == 128)), "kColumns: 16 bits");

  i32x4 rsrc, up;     // up: PAIR's up rows; kColumns: 4 k further
  int soff;           // kRowsOfK: k of the chunk. kColumns: the descriptor moves on
  int left;           // kRowsOfK: pieces of 16 bytes left of a row. kColumns: chunks left,
  uint32_t last;      // and the bytes from the last one's start to the tensor's end
  const char* base;
  int64_t step;
  // kColumns: a lane's places 4 k apart differ by no more than that
  static constexpr int kBit = ROWS == 256 ? 2 : 1;  // of i, that says which of the two
  static constexpr int kOff = L == Lay::kRowsOfK ? kInstr : kInstr / 2;
  int off[kOff], piece;

  // `extent`: the side's k, in bytes of a row (kRowsOfK) or a number (kColumns); `half`: PAIR's.
  __device__ __forceinline__ void init(const Side& s, int64_t r0, int64_t extent, Range c, int wave, int lane,
                                       int64_t half = 0) {
    if constexpr (L == Lay::kRowsOfK) {
      piece = (lane & 7) ^ (lane >> 3);
      // 4 bits: a lane of step s is to find block 2 q + s, whose scales lie together, where it finds
      // piece 4 s + q of 16 bits
      if constexpr (F == Form::kFp4) piece = (piece & 3) * 2 + (piece >> 2);
      // (a row past the last starts past the end, whatever the chunk)
      const uint32_t n = records(((PAIR ? half : s.rows) - 1 - r0) * s.ld + extent);
      rsrc = make_rsrc(s.p + r0 * s.ld, n);
      if constexpr (PAIR != 0) up = make_rsrc(s.p + (r0 + half) * s.ld, n);
      soff = c.first * kChunk;
      left = min(int(extent >> 4), c.end * 8) - c.first * 8;
#pragma unroll
      for (int i = 0; i < kInstr; ++i) {
        int row = (wave * kInstr + i) * 8 + (lane >> 3);
        if constexpr (PAIR != 0) row = row / PAIR * (PAIR / 2) + row % (PAIR / 2);
        off[i] = int(row * s.ld) + piece * 16;
      }
    } else {
      piece = soff = 0;
      base = s.p + r0 * 2 + int64_t(c.first) * kKRows * s.ld;
      step = kKRows * s.ld;
      left = c.end - c.first;
      last = records((extent - 1 - int64_t(c.end - 1) * kKRows) * s.ld + (s.rows - r0) * 2);
      describe();
#pragma unroll
      for (int j = 0; j < kOff; ++j) {
        const int i = kBit == 2 ? j : 2 * j;
        const int at = ((wave * kInstr + i) * 64 + lane) * 16, k = at / kPitch, unit = at % kPitch / 32;
        off[j] = int(k * s.ld) + (unit ^ flip(k)) * 32 + (at & 16);
      }
    }
  }
  __device__ __forceinline__ void describe() {
    // (a chunk with two more behind it reads nothing past the end: of its last k at most 512 bytes from the
    // tile's first row on, and 64 k and more follow, of 16 bytes at least)
    const uint32_t four = uint32_t(4 * step / kKRows),
                   n = left > 2 ? uint32_t(kCut) : left == 2 ? min(last + uint32_t(step), uint32_t(kCut)) : left == 1 ? last : 0u;
    rsrc = make_rsrc(base, n);
    up = make_rsrc(base + four, n > four ? n - four : 0u);
  }
  // which way the 32-byte units of k are permuted: the 8 k of a half wave's transposing read
  // (0 .. 3 and 8 .. 11 of 16) fall on all banks
  __device__ __forceinline__ static int flip(int k) { return (k & 3) | ((k >> 1) & 4); }

  // Load i of the next chunk to the wave's place in LDS.
  __device__ __forceinline__ void issue(uint32_t lds, int wave, int i) {
    if constexpr (L == Lay::kColumns) {
      to_lds_16(i & kBit ? up : rsrc, lds + i * 1024, off[kBit == 2 ? i & 1 : i >> 1], 0);
      return;
    }
    const int o = off[i < kOff ? i : 0] | (piece >= left ? kCut : 0);
    if (PAIR != 0 && (wave * kInstr + i) * 8 % (PAIR ? PAIR : 1) >= PAIR / 2) to_lds_16(up, lds + i * 1024, o, soff);
    else to_lds_16(rsrc, lds + i * 1024, o, soff);
  }
  __device__ __forceinline__ void advance() {
    if constexpr (L == Lay::kRowsOfK) {
      soff += kChunk;
      left -= 8;
    } else {
      base += step;
      --left;
      describe();
    }
  }
};

// The scales of an MXFP4 operand: 8 bytes a row and chunk, in loads of 256 bytes for 32 rows.
template <int ROWS, int WAVES> struct ScaleLoader {
  static constexpr int kBytes = ROWS * 8;
  static constexpr int kLoads = ROWS / 32;
  static_assert(kLoads == WAVES, "a load a wave");
  i32x4 rsrc;
  int soff, off, word, left;
  __device__ __forceinline__ void init(const Side& s, int64_t r0, int64_t blocks, Range c, int wave, int lane) {
    word = lane & 1;
    rsrc = make_rsrc(s.s + r0 * s.lds, records((s.rows - 1 - r0) * s.lds + (blocks + 3) / 4 * 4));
    off = int((wave * 32 + (lane >> 1)) * s.lds) + word * 4;
    soff = c.first * 8;
    left = min(int((blocks + 3) >> 2), c.end * 2) - c.first * 2;
  }
  __device__ __forceinline__ void issue(uint32_t lds) {
    to_lds_4(rsrc, lds, off | (word >= left ? kCut : 0), soff);
    soff += 8;
    left -= 2;
  }
};

// One operand fragment: 16 rows, step S of 2 of a chunk, of which lane group q has k = 32 S + 8 q .. + 7 (16 bits)
// or block 2 q + S (4 bits; any order of k will do that both operands share).
template <Form F, Lay L, int ROWS> struct Reader {
  static constexpr int kPitch = L == Lay::kRowsOfK ? kChunk : 2 * ROWS;
  int at0, at1;  // kRowsOfK: of each step; kColumns: of a unit's first byte, and the way units are permuted
  int unit;
  __device__ __forceinline__ void init(int row0, int lane) {
    const int c = lane & 15, q = lane >> 4;
    unit = row0 >> 4;
    if constexpr (L == Lay::kRowsOfK) {
      at0 = (row0 + c) * kChunk + ((q ^ (c & 7)) << 4);
      at1 = (row0 + c) * kChunk + (((4 + q) ^ (c & 7)) << 4);
    } else {
      at0 = (8 * q + (c >> 2)) * kPitch + (c & 3) * 8;
      at1 = ((c >> 2) | (q & 1) << 2) << 5;
    }
  }
  // Keeps the compiler from holding every fragment's address in registers over the loop.
  __device__ __forceinline__ void forget() {
    if constexpr (L == Lay::kColumns) asm volatile("" : "+v"(at1));
  }
  // fragment t: rows row0 + 16 t .. + 15
  template <int S> __device__ __forceinline__ u32x4 read(const char* lds, int t) const {
    if constexpr (L == Lay::kRowsOfK) {
      return *reinterpret_cast<const u32x4*>(lds + (S ? at1 : at0) + t * 16 * kChunk);
    } else {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4 lds_s4;
      const char* p = lds + at0 + (((unit + t) << 5) ^ at1) + S * 32 * kPitch;
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

// What a launch works on.
struct Product {
  Side x, w;
  int64_t M, N;      // N: of the output's columns (pairs: those of a half)
  int64_t k_bytes;   // of a row of a kRowsOfK side (a multiple of 16)
  int64_t k_rows;    // of a kColumns side: the number of k
  int64_t blocks;    // MXFP4: blocks of a row
  int chunks;        // of k
  // Tiles from `full` on are cut into `slices` of k, whose sums go to `sums` for dense_finish.
  int tiles_m, tiles_n, full, slices;
  f32x4* sums;
};

// Tile `id` of the launch: XCD i (workgroups go round the 8 of them) takes a run of
// consecutive tiles, ordered in bands of kBand row tiles, so that its 4 MB of L2 sees few
// rows of X and W at a time.
constexpr int kBand = 4;
constexpr int kWavesN = 2;  // side by side in a tile's columns
__device__ __forceinline__ void tile_of(int id, int total, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int xcd = id & 7, local = id >> 3, share = total >> 3, rest = total & 7;
  const int t = xcd * share + min(xcd, rest) + local;
  const int band = t / (kBand * tiles_n), in = t - band * kBand * tiles_n;
  const int height = min(kBand, tiles_m - band * kBand);
  tn = in / height;
  tm = band * kBand + in - tn * height;
}

// EPI: a struct whose `spot(m, n)` gives, for a wave's first row and column (pairs: of a half), a struct with
// `template <bool WHOLE> void put(int row, int col, f32x4 v)`: the sums of row m + row and columns
// n + col .. + 3, or, for pairs, `put(row, col, f32x4 g, f32x4 u)`; col is a multiple of 4, row and col are
// below 256. WHOLE: they lie within the output, else they may lie past its last column (not its
// last row). Addresses come from the wave's place and 32-bit offsets, and whole tiles have no checks:
// a tile's epilogue is code that nothing hides (16384 x 7168 x 2048 in 4 bits: 293 us with checks
// in every tile, 194 without). With EPI::kFetches, put takes a last argument, what
// `fetch<WHOLE>(row, col)` read from memory for it: the tile kernel calls that ahead.
template <Form F, Lay LX, Lay LW, int BM, int BN, bool DEEP, bool PAIRED, typename EPI>
__global__ void __launch_bounds__(BM / 64 * kWavesN * 64)
dense_tile(Product p, EPI epi) {
  constexpr int WAVES = BM / 64 * kWavesN, WN = BN / kWavesN, XT = 4, WT = WN / 16;
  constexpr bool FP4 = F == Form::kFp4;
  // (224 columns are loaded as 256: whole loads for every wave)
  constexpr int W_ROWS = BN == 224 ? 256 : BN;
  static_assert(!PAIRED || BN == W_ROWS, "pairs: whole tiles");
  using XLoad = Loader<F, LX, BM, WAVES>;
  using WLoad = Loader<F, LW, W_ROWS, WAVES, PAIRED ? WN : 0>;
  using XScale = ScaleLoader<BM, WAVES>;
  using WScale = ScaleLoader<W_ROWS, WAVES>;
  // X lies in XRING places in turn, W in WRING: while chunk c is read, the chunks up to c + WRING - 1
  // and, of X, c + XRING - 1 are on their way, so the loads never run dry. 256 rows: 3 and 2
  // (4 bits: the scales leave 2 and 2); DEEP, for a workgroup alone on its CU: 5 and 5 (4 and 4).
  constexpr int XRING = DEEP ? (FP4 ? 4 : 5) : FP4 ? 2 : 3, WRING = DEEP ? XRING : 2;
  constexpr int XI = XLoad::kInstr, WI = WLoad::kInstr;
  static_assert(XRING == WRING || XRING == WRING + 1, "the order of loads that publish() counts on");
  constexpr int W_AT = XRING * XLoad::kBytes, S_AT = W_AT + WRING * WLoad::kBytes;
  constexpr int SCALES = FP4 ? XScale::kBytes + WScale::kBytes : 0;
  __shared__ __attribute__((aligned(1024))) char lds[S_AT + WRING * SCALES];
  const int lane = threadIdx.x & 63, wave = uniform(int(threadIdx.x) >> 6);
  const int wn = wave % kWavesN, wm = wave / kWavesN;
  XLoad xl;
  WLoad wl;
  XScale xsl;
  WScale wsl;
  int64_t m0, n0;
  int C, part;  // chunks, and which of the slices' sums (-1: a whole tile)
  // the lane's number, for what is worked out between tiles and not to be held during one
  auto lane_again = [&]() __attribute__((always_inline)) {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
  };
  auto open = [&](int job) __attribute__((always_inline)) {
    const int lane = lane_again();
    Range range{0, p.chunks};
    part = job - p.full;
    if (part >= 0) {
      job = p.full + part / p.slices;
      range = range_of(part % p.slices, p.slices, p.chunks);
    }
    C = range.end - range.first;
    int tm, tn;
    tile_of(job, p.tiles_m * p.tiles_n, p.tiles_m, p.tiles_n, tm, tn);
    m0 = int64_t(tm) * BM;
    n0 = int64_t(tn) * (PAIRED ? BN / 2 : BN);
    xl.init(p.x, m0, LX == Lay::kRowsOfK ? p.k_bytes : p.k_rows, range, wave, lane);
    wl.init(p.w, n0, LW == Lay::kRowsOfK ? p.k_bytes : p.k_rows, range, wave, lane, p.N);
    if constexpr (FP4) {
      xsl.init(p.x, m0, p.blocks, range, wave, lane);
      wsl.init(p.w, n0, p.blocks, range, wave, lane);
    }
  };
  // the next loads' places
  const uint32_t lds0 = uniform(uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds)));
  const uint32_t x_to = lds0 + wave * XI * 1024, w_to = lds0 + W_AT + wave * WI * 1024, s_to = lds0 + S_AT + wave * 256;
  int x_at = 0, w_at = 0, s_at = 0;
  auto issue_x = [&](int i) __attribute__((always_inline)) { xl.issue(x_to + x_at, wave, i); };
  auto issue_w = [&](int i) __attribute__((always_inline)) { wl.issue(w_to + w_at, wave, i); };
  auto issue_s = [&]() __attribute__((always_inline)) {
    xsl.issue(s_to + s_at);
    wsl.issue(s_to + s_at + XScale::kBytes);
    s_at = s_at == (WRING - 1) * SCALES ? 0 : s_at + SCALES;
  };
  auto next_x = [&]() __attribute__((always_inline)) {
    xl.advance();
    x_at = x_at == (XRING - 1) * XLoad::kBytes ? 0 : x_at + XLoad::kBytes;
  };
  auto next_w = [&]() __attribute__((always_inline)) {
    wl.advance();
    w_at = w_at == (WRING - 1) * WLoad::kBytes ? 0 : w_at + WLoad::kBytes;
  };
  Reader<F, LX, BM> xr;
  Reader<F, LW, W_ROWS> wr;
  xr.init(wm * 64, lane);
  wr.init(wn * WN, lane);
  const int sx_at = S_AT + (wm * 64 + (lane & 15)) * 8 + (lane >> 4) * 2,
            sw_at = S_AT + XScale::kBytes + (wn * WN + (lane & 15)) * 8 + (lane >> 4) * 2;

  f32x4 acc[WT][XT];
  // Fragments of the step at hand and, as its W fragments are used up, of the next. W's last one
  // has places of its own in both steps, so that every read is out well before a barrier.
  constexpr int KEEP = WT - 1, XLATE = XRING == 2;  // (two places of X: its loads go out as early as W's)
  u32x4 wf[KEEP], we[2], xf[2][XT];
  uint32_t ws[WT], xs[XT], xsn[XT];
  int cx = 0, cw = 0, cs = 0;  // where the chunk to read lies

  // Step S of the chunk in registers, while step 1 - S is read: of the same chunk (S = 0), or of
  // the next one (S = 1); a later chunk of W (S = 1) and of X (S = 0) go out, in the step's first half,
  // so that they have longest until the barrier that waits for them (4096 x 7168 x 2048 forward: 279 us,
  // spread over the whole step 297, all at once 287).
  auto step = [&](auto STEP, auto READ, auto MATH) __attribute__((always_inline)) {
    constexpr int s = decltype(STEP)::value, n = 1 - s;
    constexpr bool read = decltype(READ)::value, math = decltype(MATH)::value;
    const char* xb = lds + cx;
    const char* wb = lds + W_AT + cw;
    auto w_of = [&](int a) __attribute__((always_inline)) -> u32x4& { return a < KEEP ? wf[a] : we[s]; };
    if constexpr (read) {
      xr.forget();
      wr.forget();
#pragma unroll
      for (int b = 0; b < XT; ++b) xf[n][b] = xr.template read<n>(xb, b);
      if constexpr (FP4 && n == 0) {
#pragma unroll
        for (int b = 0; b < XT; ++b) xsn[b] = *reinterpret_cast<const uint16_t*>(lds + cs + sx_at + b * 128);
      }
      we[n] = wr.template read<n>(wb, KEEP);
    }
#pragma unroll
    for (int a = 0; a < WT; ++a) {
      if constexpr (math) {
#pragma unroll
        for (int b = 0; b < XT; ++b) {
          if constexpr (FP4) acc[a][b] = mma4<s>(w_of(a), ws[a], xf[s][b], xs[b], acc[a][b]);
          else acc[a][b] = mma<F>(w_of(a), xf[s][b], acc[a][b]);
        }
      }
      if constexpr (read && s == 1) {
        if (FP4 && a == 0) issue_s();
#pragma unroll
        for (int i = 0; i < WI; ++i)
          if (a == (XLATE ? 0 : i * WT / WI / 2)) issue_w(i);
      }
      if constexpr (read && s == XLATE) {
#pragma unroll
        for (int i = 0; i < XI; ++i)
          if (a == (XLATE ? 1 : i * WT / XI / 2)) issue_x(i);
      }
      if constexpr (read) {
        if (a < KEEP) wf[a] = wr.template read<n>(wb, a);
        if constexpr (FP4 && n == 0) ws[a] = *reinterpret_cast<const uint16_t*>(lds + cs + sw_at + a * 128);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (FP4 && read && n == 0) {
#pragma unroll
      for (int b = 0; b < XT; ++b) xs[b] = xsn[b];
    }
    if constexpr (read && s == 1) next_w();
    if constexpr (read && s == XLATE) next_x();
  };
  // Behind it: all of the next chunk has landed, for every wave, and every wave has read the
  // one before it.
  auto publish = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    constexpr int CHUNK = XI + WI + (FP4 ? 2 : 0);  // a wave's loads of a chunk
    XK_WAIT_VMCNT((WRING - 2) * CHUNK + (XRING > WRING ? XI : 0));
    lds_sync();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto turn = [&]() __attribute__((always_inline)) {  // to the next chunk's places
    cx = cx == (XRING - 1) * XLoad::kBytes ? 0 : cx + XLoad::kBytes;
    cw = cw == (WRING - 1) * WLoad::kBytes ? 0 : cw + WLoad::kBytes;
    if constexpr (FP4) cs = cs == (WRING - 1) * SCALES ? 0 : cs + SCALES;
  };
  constexpr std::integral_constant<int, 0> S0{};
  constexpr std::integral_constant<int, 1> S1{};
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  auto send = [&]() __attribute__((always_inline)) {  // a tile's first chunks
    x_at = w_at = s_at = 0;
#pragma unroll
    for (int r = 0; r < WRING - 1; ++r) {
      if constexpr (FP4) issue_s();
#pragma unroll
      for (int i = 0; i < WI; ++i) issue_w(i);
      next_w();
#pragma unroll
      for (int i = 0; i < XI; ++i) issue_x(i);
      next_x();
    }
    if constexpr (XRING > WRING) {
#pragma unroll
      for (int i = 0; i < XI; ++i) issue_x(i);
      next_x();
    }
  };
  const int jobs = p.full + (p.tiles_m * p.tiles_n - p.full) * p.slices;
  int job = blockIdx.x;
  open(job);
  send();
  while (true) {
#pragma unroll
    for (int a = 0; a < WT; ++a)
#pragma unroll
      for (int b = 0; b < XT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    cx = cw = cs = 0;
    if (C > 0) {
      publish();
      // chunk c's turn: step 1 of c - 1 and step 0 of c, reading both steps of c
      step(S1, yes, no);
      step(S0, yes, yes);
      publish();
      turn();
      for (int c = 1; c < C; ++c) {
        step(S1, yes, yes);
        step(S0, yes, yes);
        publish();
        turn();
      }
      step(S1, no, yes);
    }
    // the loads of nothing have landed: they are the wave's own, as are the places of the next
    // ones (and at the end the LDS may be another workgroup's)
    XK_WAIT_VMCNT(0);
    const int l = lane_again(), done = part;
    const int rows_left = int(min(p.M - m0 - wm * 64, int64_t(64)));
    const auto spot = epi.spot(m0 + wm * 64, n0 + wn * (PAIRED ? WN / 2 : WN));
    const bool whole_tile = m0 + BM <= p.M && n0 + (PAIRED ? BN / 2 : BN) <= p.N;
    job += gridDim.x;
    if (job < jobs) {
      open(job);
      send();
    }
    // Up to 4 fragments of 16 rows at a time go through LDS (the wave's part of X's last place, which
    // no load is bound for yet) and come back row by row: whole pieces of a row leave together,
    // and the epilogue's code is there once for 16 of its calls (code that runs once comes from
    // memory: the checked form of GateGrad, unrolled, took a 128 x 128 tile 20 us). Pieces are
    // permuted by the row.
    f32x4* own = reinterpret_cast<f32x4*>(lds + (XRING - 1) * XLoad::kBytes + wave * 4096);
    static_assert(XLoad::kBytes == WAVES * 4096, "4 KB of an X place a wave");
    auto put_all = [&](auto WHOLE) __attribute__((always_inline)) {
      constexpr bool whole = decltype(WHOLE)::value;
      constexpr int AT = PAIRED ? WT / 2 : WT, STRIDE = PAIRED ? 2 : 4;  // fragments of columns, and at a time
      constexpr int LANES = PAIRED ? 8 : 16, ROWS = 64 / LANES;          // to a row, and rows of a wave at a time
      constexpr int TIMES = (AT + STRIDE - 1) / STRIDE * XT;
      const int unit = l & (LANES - 1);
      auto stage = [&](int t) __attribute__((always_inline)) {
        const int a0 = t / XT * STRIDE, b = t % XT, c = l & 15, q = l >> 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int a = PAIRED ? a0 + (e & 1) + (e >> 1) * (WT / 2) : a0 + e;
          if (a < WT) own[c * 16 + ((e * 4 + q) ^ c)] = acc[a][b];
        }
        wave_lds_fence();
      };
      // whether the lane has something to write in row `row` of turn t
      auto holds = [&](int t, int row) __attribute__((always_inline)) {
        return (whole || t % XT * 16 + row < rows_left) && (PAIRED || unit < (WT - t / XT * STRIDE) * 4);
      };
      if constexpr (EPI::kFetches) if constexpr (whole) {
        static_assert(!PAIRED, "no pairs with values of memory");
        // two rows of a turn at a time, the next two's values on their way
        constexpr int HALVES = 16 / ROWS / 2;
        decltype(spot.template fetch<whole>(0, 0)) held[2][2];
        auto fetch = [&](int h) __attribute__((always_inline)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int t = h / HALVES, row = l / LANES + (h % HALVES * 2 + r) * ROWS;
            if (holds(t, row)) held[h & 1][r] = spot.template fetch<whole>(t % XT * 16 + row, t / XT * STRIDE * 16 + unit * 4);
          }
        };
        fetch(0);
#pragma unroll
        for (int h = 0; h < TIMES * HALVES; ++h) {
          const int t = h / HALVES;
          if (h + 1 < TIMES * HALVES) fetch(h + 1);
          if (h % HALVES == 0) stage(t);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int row = l / LANES + (h % HALVES * 2 + r) * ROWS;
            if (holds(t, row))
              spot.template put<whole>(t % XT * 16 + row, t / XT * STRIDE * 16 + unit * 4, own[row * 16 + (unit ^ row)],
                                       held[h & 1][r]);
          }
          wave_lds_fence();
          __builtin_amdgcn_sched_barrier(0);
        }
        return;
      }
#pragma unroll
      for (int t = 0; t < TIMES; ++t) {
        stage(t);
        const int col = t / XT * STRIDE * 16 + unit * 4;
#pragma unroll 1
        for (int row = l / LANES; row < 16; row += ROWS) {
          if (!holds(t, row)) continue;
          const int at = t % XT * 16 + row;
          const f32x4 v = own[row * 16 + (unit ^ row)];
          if constexpr (PAIRED) spot.template put<whole>(at, col, v, own[row * 16 + ((unit + 8) ^ row)]);
          else if constexpr (EPI::kFetches) spot.template put<whole>(at, col, v, spot.template fetch<whole>(at, col));
          else spot.template put<whole>(at, col, v);
        }
        wave_lds_fence();
      }
    };
    if (done >= 0) {
      f32x4* to = p.sums + (int64_t(done) * WAVES + wave) * (WT * XT * 64) + l;
#pragma unroll
      for (int b = 0; b < XT; ++b) {
        if (b * 16 >= rows_left) break;  // (rows past the last are not added up either)
#pragma unroll
        for (int a = 0; a < WT; ++a) to[(a * XT + b) * 64] = acc[a][b];
      }
    } else if (whole_tile) {
      put_all(yes);
    } else {
      put_all(no);
    }
    if (job >= jobs) break;
  }
}

// One group of sums to the epilogue, outside the tile kernel.
template <typename EPI, bool PAIRED, typename SPOT>
__device__ __forceinline__ void finish(const SPOT& spot, int row, int col, f32x4 v, f32x4 u) {
  if constexpr (PAIRED) spot.template put<false>(row, col, v, u);
  else if constexpr (EPI::kFetches) spot.template put<false>(row, col, v, spot.template fetch<false>(row, col));
  else spot.template put<false>(row, col, v);
}

// Adds up the slices of tiles full .., in their order, for the epilogue: a workgroup a wave's
// 16 columns (pairs: both 16s) x 64 rows.
template <int BM, int BN, bool PAIRED, typename EPI>
__global__ void __launch_bounds__(256)
dense_finish(Product p, EPI epi) {
  constexpr int WAVES = BM / 64 * kWavesN, WN = BN / kWavesN, XT = 4, WT = WN / 16, AT = PAIRED ? WT / 2 : WT;
  const int lane = threadIdx.x & 63, b = uniform(int(threadIdx.x) >> 6);
  const int a = blockIdx.x % AT, wave = blockIdx.x / AT % WAVES, rest = blockIdx.x / AT / WAVES;
  const int wn = wave % kWavesN, wm = wave / kWavesN;
  int tm, tn;
  tile_of(p.full + rest, p.tiles_m * p.tiles_n, p.tiles_m, p.tiles_n, tm, tn);
  const int64_t m = int64_t(tm) * BM + wm * 64 + b * 16;
  const int64_t n = int64_t(tn) * (PAIRED ? BN / 2 : BN) + wn * (PAIRED ? WN / 2 : WN) + a * 16;
  const int row = lane & 15, col = (lane >> 4) * 4;
  if (m + row >= p.M) return;
  constexpr int64_t plane = int64_t(WAVES) * WT * XT * 64;
  const f32x4* at = p.sums + int64_t(rest) * p.slices * plane + (int64_t(wave) * WT + a) * XT * 64 + b * 64 + lane;
  f32x4 v = *at, u = {};
  if constexpr (PAIRED) u = at[WT / 2 * XT * 64];
  for (int s = 1; s < p.slices; ++s) {
    v += at[s * plane];
    if constexpr (PAIRED) u += at[s * plane + WT / 2 * XT * 64];
  }
  finish<EPI, PAIRED>(epi.spot(m, n), row, col, v, u);
}

// ---------------------------------------------------------------- launches ----

// How a product is cut up.
struct Plan {
  int rows, cols;  // of a tile
  int full;        // tiles that are not cut; a multiple of the workgroups at a time
  int slices;      // of k, that the other tiles are cut into
  int64_t rest;    // the other tiles
};
inline int64_t sums_bytes(const Plan& plan) {
  return plan.slices > 1 ? plan.rest * plan.slices * plan.rows * plan.cols * 4 : 0;
}

// The cheapest of the tiles and slices, in microseconds as measured (16 bits; MXFP4; the 16-bit
// figures with loads spread over whole steps: the present order takes 2 to 6 % off):
//   * 256 x 256, a workgroup a CU: 1.47 (2.3) a chunk, however many CUs are busy
//     (8192 x 4096 x 7168: 333 us; 4096 x 4096 x 7168 in 4 bits: 67);
//   * 256 x 224 takes 0.96 of that, and fewer rounds where it divides the columns better
//     (8192 x 7168 x 4096, 4 rounds of either: 376 us, with 256 x 256 391);
//   * 128 x 128: two workgroups a CU 0.88 (1.7) a chunk each, one alone 0.75 (0.77), with more
//     places in LDS (8192 x 4096 x 7168: 392 us; 512 x 4096 x 4096: 39 us, where 256 x 256 takes 98; 2048 x 2048 in
//     4 bits, 28 chunks 28.6 us, 8 chunks 13.2);
//   * slices of k, for all tiles where they leave CUs idle or for those of the last round: the
//     sums written and read at 3 TB/s, and another launch of 4 us and half a one for each slice
//     (64 x 4096 x 4096: 30 us, with 8 slices 11 and 4; 64 x 4096 x 2048: 4 slices 11 and 4, 8 slices
//     14 and 5); without them 3 us for results written by few workgroups.
inline Plan plan_tiles(bool fp4, int64_t M, int64_t N, int64_t chunks, bool paired) {
  const int64_t cols = paired ? 2 * N : N;
  const double big = fp4 ? 2.3 : 1.47, two = fp4 ? 1.7 : 0.88, one = 0.75;
  Plan best{};
  double least = 1e300;
  auto offer = [&](int bm, int bn, int64_t places, double chunk, double alone) {
    const int64_t tiles = cdiv(M, bm) * cdiv(cols, bn), full = tiles / places * places, rest = tiles - full;
    for (int s = 1; s <= 32 && (s == 1 || (rest * s <= places && 2 * s <= chunks)); s *= 2) {
      const double each = rest == 0 ? 0 : full == 0 && rest * s <= 256 ? alone : chunk;
      Plan plan{bm, bn, int(s > 1 ? full : tiles), s, s > 1 ? rest : 0};
      const double us = 4 + double(full / places) * chunk * chunks + each * double(cdiv(chunks, s)) +
                        (s > 1 ? 4 + 0.5 * s + double(sums_bytes(plan)) * std::min<int64_t>(M, bm) / bm / 3e6 : 0) +
                        (s == 1 && full == 0 && rest <= 256 ? 3 : 0);
      if (us < least) {
        least = us;
        best = plan;
      }
    }
  };
  offer(256, 256, 256, big, big);
  if (!paired) offer(256, 224, 256, 0.96 * big, 0.96 * big);
  offer(128, 128, 512, two, one);
  return best;
}

template <Form F, Lay LX, Lay LW, int BM, int BN, bool DEEP, bool PAIRED, typename EPI>
void launch_cut(Product p, int64_t places, const EPI& epi, hipStream_t stream) {
  p.tiles_m = int(cdiv(p.M, BM));
  p.tiles_n = int(cdiv(p.N, PAIRED ? BN / 2 : BN));
  const int64_t rest = int64_t(p.tiles_m) * p.tiles_n - p.full, jobs = p.full + rest * p.slices;
  hipLaunchKernelGGL((dense_tile<F, LX, LW, BM, BN, DEEP, PAIRED, EPI>), dim3(int(std::min(jobs, places))),
                     dim3(BM / 64 * kWavesN * 64), 0, stream, p, epi);
  if (rest > 0)
    hipLaunchKernelGGL((dense_finish<BM, BN, PAIRED, EPI>),
                       dim3(int(rest * (BM / 64 * kWavesN) * (BN / kWavesN / 16 / (PAIRED ? 2 : 1)))), dim3(256), 0, stream,
                       p, epi);
}

// The product with its epilogue; `scratch` (16-byte aligned) holds the plan's sums_bytes.
template <Form F, Lay LX, Lay LW, bool PAIRED, typename EPI>
void launch_tiles(Product p, const EPI& epi, void* scratch, hipStream_t stream) {
  const Plan plan = plan_tiles(F == Form::kFp4, p.M, p.N, p.chunks, PAIRED);
  p.full = plan.full;
  p.slices = plan.slices;
  p.sums = static_cast<f32x4*>(scratch);
  if (plan.rows == 128) {
    // deep where every workgroup has a CU to itself
    if (plan.full + plan.rest * plan.slices <= 256)
      launch_cut<F, LX, LW, 128, 128, true, PAIRED>(p, 256, epi, stream);
    else
      launch_cut<F, LX, LW, 128, 128, false, PAIRED>(p, 512, epi, stream);
  } else if (plan.cols == 224) {
    if constexpr (!PAIRED) launch_cut<F, LX, LW, 256, 224, false, false>(p, 256, epi, stream);
  } else {
    launch_cut<F, LX, LW, 256, 256, false, PAIRED>(p, 256, epi, stream);
  }
}

}  // namespace dense
}  // namespace xk
