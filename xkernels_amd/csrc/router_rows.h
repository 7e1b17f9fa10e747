// Router rows on 16 lanes each: loads of 8 logits and reductions over the lanes of
// a row, shared by the selection (topk_softmax.hip) and the training kernels
// (router_train.hip).
#pragma once

#include "common.h"

namespace xk {

template <typename T>
__device__ __forceinline__ float logit_at(const T* p);
template <>
__device__ __forceinline__ float logit_at<uint16_t>(const uint16_t* p) {  // bf16 bits
  return __uint_as_float(uint32_t(*p) << 16);
}
template <>
__device__ __forceinline__ float logit_at<_Float16>(const _Float16* p) {
  return float(*p);
}
template <>
__device__ __forceinline__ float logit_at<float>(const float* p) {
  return *p;
}

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xF, 0xF, false);
}
// f over the partners of an all-reduce of 16 lanes: neighbours, pairs, the
// mirrored half row, the mirrored row.
template <typename F> __device__ __forceinline__ void row_steps(F&& f) {
  f([](uint32_t x) { return dpp<0xB1>(x); });
  f([](uint32_t x) { return dpp<0x4E>(x); });
  f([](uint32_t x) { return dpp<0x141>(x); });
  f([](uint32_t x) { return dpp<0x140>(x); });
}

template <typename T> struct piece8 {};  // 8 logits in 16-byte loads
template <> struct piece8<uint16_t> {
  __device__ __forceinline__ static void load(const uint16_t* g, float* v) {
    const u32x4 r = *reinterpret_cast<const u32x4*>(g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
    }
  }
};
template <> struct piece8<_Float16> {
  __device__ __forceinline__ static void load(const _Float16* g, float* v) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const h8 r = *reinterpret_cast<const h8*>(g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(r[i]);
  }
};
template <> struct piece8<float> {
  __device__ __forceinline__ static void load(const float* g, float* v) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 r = reinterpret_cast<const f32x4*>(g)[h];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * h + i] = r[i];
    }
  }
};

}  // namespace xk
