// ifx_rope.h -- loads, stores and index arithmetic of the kernels that rotate
// and append (rope_append.hip, rope_append_q8.hip).
#pragma once

#include "ifx_attn.h"

namespace ifx {

// Eight values of a row, as they lie in memory.
template <int SRC>
struct Raw8 {
  u32x4 u[SRC == IFX_ATTN_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *p, int64_t at) {
    const char *c = static_cast<const char *>(p) + at * (SRC == IFX_ATTN_F32 ? 4 : 2);
    u[0] = ldg<u32x4>(c);
    if constexpr (SRC == IFX_ATTN_F32) u[1] = ldg<u32x4>(c + 16);
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    if constexpr (SRC == IFX_ATTN_F32) {
      const f32x4 v = __builtin_bit_cast(f32x4, u[0]), w = __builtin_bit_cast(f32x4, u[1]);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
      x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = SRC == IFX_ATTN_F16 ? F16::value(u[0][i] & 0xFFFFu) : BF16::value(u[0][i] & 0xFFFFu);
        x[2 * i + 1] = SRC == IFX_ATTN_F16 ? F16::value(u[0][i] >> 16) : BF16::value(u[0][i] >> 16);
      }
    }
  }
};

template <class T>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7])};
}

// Two neighbouring values of a row.
template <int SRC>
__device__ __forceinline__ float2 load2(const void *p, int64_t at) {
  if constexpr (SRC == IFX_ATTN_F32) return ldg<float2>(static_cast<const float *>(p) + at);
  const uint32_t u = ldg<uint32_t>(static_cast<const uint16_t *>(p) + at);
  return SRC == IFX_ATTN_F16 ? make_float2(F16::value(u & 0xFFFFu), F16::value(u >> 16))
                             : make_float2(BF16::value(u & 0xFFFFu), BF16::value(u >> 16));
}

// floor(x / d) for 0 <= x < 2^24 with r = 1 / d: the product is off by less than 1.
__device__ __forceinline__ int quotient(int x, int d, float r) {
  const int q = static_cast<int>(static_cast<float>(x) * r), rest = x - q * d;
  return q + (rest >= d) - (rest < 0);
}

}  // namespace ifx
