// ifx_attn_q8.h -- what the kernels of the 8-bit cache (rope_append_q8.hip,
// attn_rows_q8.hip, attn_tile_q8.hip) and their entry points share.
#pragma once

#include "ifx_attention_q8.h"
#include "ifx_attn.h"

namespace ifx {

struct AppendQ8Args {
  AppendArgs a;
  uint32_t *scales;
  int kv_parts;  // parts that K's and V's heads are each shared out in
};
hipError_t launch_rope_append_q8(const AppendQ8Args &a, int src_dtype, int q_dtype, hipStream_t s);

struct ReadArgs {
  const void *k, *v;
  const uint32_t *scales;
  const int32_t *slots;
  void *k_out, *v_out;
  int64_t k_stride, v_stride;
  int N, Hkv, D, page_shift, num_slots;
};
hipError_t launch_read_rows_q8(const ReadArgs &a, int out_dtype, hipStream_t s);

hipError_t launch_attn_rows_q8(const AttnArgs &a, int D, int max_rows, int blocks, int items,
                               hipStream_t s);
hipError_t launch_attn_tile_q8(const AttnArgs &a, int D, int items, hipStream_t s);

// 16 or 4 bytes a lane from memory to 64 consecutive places in LDS.
__device__ __forceinline__ void to_lds16(const void *from, u32x4 *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
__device__ __forceinline__ void to_lds4(const void *from, u32x4 *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)to, 4, 0, 0);
}

// Waits until at most N of this wave's loads are on their way: loads end in
// order, so all before its last N have ended.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "six bits count them");
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4 << 14));
  __builtin_amdgcn_sched_barrier(0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Scales of a token and head: K's in the low half, V's in the high one.
__device__ __forceinline__ float k_scale(uint32_t s) { return __builtin_bit_cast(float, s << 16); }
__device__ __forceinline__ float v_scale(uint32_t s) {
  return __builtin_bit_cast(float, s & 0xFFFF0000u);
}

// Four codes as fp16, exactly: code + 128 in the low bits of 1024, less 1152.
__device__ __forceinline__ u32x2 codes_f16(uint32_t w) {
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  const uint32_t x = w ^ 0x80808080u;
  const v2 less = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  const v2 lo = __builtin_bit_cast(v2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + less;
  const v2 hi = __builtin_bit_cast(v2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + less;
  return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}
__device__ __forceinline__ u32x4 codes_f16(u32x2 w) {
  const u32x2 a = codes_f16(w.x), b = codes_f16(w.y);
  return u32x4{a.x, a.y, b.x, b.y};
}
// Eight of a piece's sixteen: the first (i = 0) or the last.
__device__ __forceinline__ u32x4 codes_f16(u32x4 p, int i) {
  return codes_f16(i ? u32x2{p.z, p.w} : u32x2{p.x, p.y});
}

// Q of a row as fp16 operands: as it is, or of bf16 times a power of two that
// takes the row's largest value to [2^13, 2^14).  f: the lane's part of the row;
// lanes LANES apart hold the rest of it.  Returns what scores are multiplied by.
template <int LANES, int NS>
__device__ __forceinline__ float row_to_f16(u32x4 (&f)[NS], int dtype, float c) {
  if (dtype == IFX_ATTN_F16) return c;
  float top = 0.0f;
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      top = fmaxf(top, fmaxf(fabsf(BF16::value(f[s][j] & 0xFFFFu)), fabsf(BF16::value(f[s][j] >> 16))));
#pragma unroll
  for (int d = LANES; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const int e = min(max(static_cast<int>(__builtin_bit_cast(uint32_t, top) >> 23), 64), 253);
  const float up = __builtin_bit_cast(float, static_cast<uint32_t>(267 - e) << 23);
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      f[s][j] = F16::pack(BF16::value(f[s][j] & 0xFFFFu) * up, BF16::value(f[s][j] >> 16) * up);
  return fminf(c * __builtin_bit_cast(float, static_cast<uint32_t>(e - 13) << 23), 3.0e38f);
}

// The running maximum of a row's scores and, a power of two, the size of V's
// scales that it has met.  Exponents are taken relative to `less`, so that a
// probability times V's scale is at most 2^(kShift + kLag).
struct Level {
  float m, size, less;
  __device__ __forceinline__ Level() : m(-__builtin_inff()), size(0x1p-80f), less(0.0f) {}
  // whether scores up to mt and scales up to vt need another level
  __device__ __forceinline__ bool above(float mt, float vt, float c) const {
    return (mt - m) * c > kLag || vt > size;
  }
  // raises it; what earlier sums are multiplied by
  __device__ __forceinline__ float raise(float mt, float vt, float c) {
    const float mn = fmaxf(m, mt);
    float sn = size;
    if (vt > size)  // the next power of two
      sn = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, vt) + 0x7FFFFFu) & 0x7F800000u);
    const float e = power(sn), was = power(size);
    const float w = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c + (was - e));
    m = mn, size = sn;
    less = m == -__builtin_inff() ? 0.0f : m * c - F16::kShift + e;
    return w;
  }
  static __device__ __forceinline__ float power(float size) {
    return static_cast<float>(static_cast<int>(__builtin_bit_cast(uint32_t, size) >> 23) - 127);
  }
  // of sums that met nothing: -inf
  __device__ __forceinline__ float of_sums() const { return m == -__builtin_inff() ? m : less; }
};

}  // namespace ifx
