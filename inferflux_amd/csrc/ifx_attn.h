// ifx_attn.h -- what the attention kernels (kv_plan.hip, rope_append.hip,
// attn_rows.hip, attn_tile.hip) and their entry points (attention_api.hip)
// share.
#pragma once

#include <atomic>

#include "ifx_attention.h"
#include "ifx_common.h"

namespace ifx {

constexpr float kLog2e = 1.44269504088896340736f;

// 16-bit element types: the MFMA operand, the conversion of two fp32 values
// (round to nearest even) into one dword, and of one back.
struct F16 {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a),
                                                  __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    const v2 r = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, r);
  }
  static __device__ __forceinline__ float value(uint32_t bits16) { return h2f(bits16); }
  // Probabilities are 2^(x - max + kShift): fp16 has 2^-24 as its smallest
  // step, and a long row of keys far below the maximum would otherwise lose
  // what they weigh together.  Up to 2^(kShift + kLag) = 2^14 is reached, in
  // fp16's range.
  static constexpr float kShift = 6.0f;
};
struct BF16 {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a),
                                                   __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    const v2 r = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, r);
  }
  static __device__ __forceinline__ float value(uint32_t bits16) {
    return __builtin_bit_cast(float, bits16 << 16);
  }
  static constexpr float kShift = 0.0f;
};

template <int DT>
struct ElemOf;
template <>
struct ElemOf<IFX_ATTN_F16> {
  typedef F16 type;
};
template <>
struct ElemOf<IFX_ATTN_BF16> {
  typedef BF16 type;
};
template <int DT>
using Elem = typename ElemOf<DT>::type;

// The running maximum of a row is raised only when a tile's exceeds it by
// more than 2^kLag in the exponent: sums and products are rescaled then and
// not for every tile, and the result is the same, as all terms of a row carry
// the same factor.
constexpr float kLag = 8.0f;

// value(v) of lane l ^ 32 beside the lane's own: (lanes 0-31's, lanes 32-63's).
__device__ __forceinline__ void both_halves(float v, float &low, float &high) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  low = __builtin_bit_cast(float, static_cast<uint32_t>(r[0]));
  high = __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}
__device__ __forceinline__ float halves_max(float v) {
  float a, b;
  both_halves(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float halves_sum(float v) {
  float a, b;
  both_halves(v, a, b);
  return a + b;
}

// Key of A-operand row m of a 32-key product S^T = K Q^T.  The 32x32 result
// holds rows 8 (r / 4) + 4 h + r % 4 in register r of lane half h; with bits 2
// and 3 of the row number exchanged, register r of half h is key
// 16 (r / 8) + 8 h + r % 8, which is the B-operand order of the next product
// O^T = V^T P^T: the probabilities are its operand as they stand, without a
// move between lanes.
__device__ __forceinline__ int key_of_row(int m) {
  return (m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1);
}

// Four consecutive values of an output row, rounded once.
__device__ __forceinline__ void store4(void *row, int dtype, int at, f32x4 v) {
  if (dtype == IFX_ATTN_F32) {
    __builtin_memcpy(static_cast<float *>(row) + at, &v, 16);
  } else {
    const u32x2 p = dtype == IFX_ATTN_F16 ? u32x2{F16::pack(v.x, v.y), F16::pack(v.z, v.w)}
                                          : u32x2{BF16::pack(v.x, v.y), BF16::pack(v.z, v.w)};
    __builtin_memcpy(static_cast<uint16_t *>(row) + at, &p, 8);
  }
}
__device__ __forceinline__ int dtype_bytes(int dtype) { return dtype == IFX_ATTN_F32 ? 4 : 2; }

// Buffer accesses that other XCDs see / that see what they wrote (sc1: past
// this XCD's L2), for split sums exchanged within one launch.
constexpr int kAuxDevice = 16;
__device__ __forceinline__ void st_dev4(rsrc_t r, uint32_t byte, f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, byte, 0, kAuxDevice);
}
__device__ __forceinline__ f32x4 ld_dev4(rsrc_t r, uint32_t byte) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, byte, 0, kAuxDevice));
}

// Weight of sums taken under maximum m in a total under `top` >= m.  Sums that
// saw nothing (m = -inf) are 0, or not a number if all their scores were not:
// both are kept by a weight of 0.
__device__ __forceinline__ float weight(float m, float top, float c) {
  return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - top) * c);
}

// Allows a kernel dynamic LDS beyond 64 KB, once per device (`done`: one flag
// word per kernel).
hipError_t allow_lds(const void *kernel, int bytes, std::atomic<uint64_t> &done);

struct PlanArgs {
  const int32_t *ctx_len, *new_len;
  int32_t *block_table;
  const int32_t *free_pages, *free_count;
  int32_t *cu_q, *kv_len, *positions, *slots, *free_left, *status;
  int table_width, free_capacity, page_shift, B, max_tokens;
};
constexpr int kPlanTokens = 1024;  // tokens a workgroup places
hipError_t launch_plan_batch(const PlanArgs &a, hipStream_t s);

struct AppendArgs {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  const int32_t *positions, *slots;
  const double *inv_freq;
  void *q_out, *k_cache, *v_cache;
  int rot_dim, interleaved, T, Hq, Hkv, D, page_shift, num_slots;
};
hipError_t launch_rope_append(const AppendArgs &a, int src_dtype, int cache_dtype, hipStream_t s);

// Attention over a paged cache (k, v: cache; table) or over packed rows.
struct AttnArgs {
  const void *q, *k, *v;
  void *out;
  int64_t q_stride, k_stride, v_stride, out_stride;  // elements
  const int32_t *table, *cu, *kv_len;
  int64_t num_pages;
  int table_width, page_shift;
  int B, T, Hq, Hkv, G;
  int causal, window, out_dtype;
  float c;     // scale * log2(e)
  int chunk;   // attn_rows: keys of a split
  int splits;  // attn_rows: most splits of a request, grid and workspace slots
  int goal;    // attn_tile: about this many workgroups for a key/value head
  uint32_t *cnt;
  float *part;
  uint32_t part_bytes;
};

// Query rows of one key/value head: row r of a request is query head r % G of
// the group and new token r / G.
constexpr int kRowsMax = 32;   // rows of a request that attn_rows takes
constexpr int kRowKeys = 128;  // attn_rows: keys that a workgroup's waves take at a time
constexpr int kTileKeys = 64;  // attn_tile: keys of a stage

// attn_rows: keys of a split, the plan's, or more where a request is longer than the plan
// was told, so that a.splits of them always suffice.
__device__ __forceinline__ int split_chunk(const AttnArgs &a, int keys) {
  if (keys <= static_cast<int64_t>(a.chunk) * a.splits) return a.chunk;
  return (keys / a.splits / kRowKeys + 1) * kRowKeys;
}

hipError_t launch_attn_rows(const AttnArgs &a, int dtype, int D, int max_rows, hipStream_t s);
hipError_t launch_attn_tile(const AttnArgs &a, int dtype, int D, bool paged, int tiles,
                            hipStream_t s);
int attn_tile_rows(int D);
int attn_tile_min_keys();  // of a split
int64_t attn_tile_slot_bytes(int D);

}  // namespace ifx
