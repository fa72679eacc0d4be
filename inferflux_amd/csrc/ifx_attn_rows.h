// ifx_attn_rows.h -- what the attention kernels of requests with few query rows
// (attn_rows.hip, attn_rows_q8.hip) do with their sums: the four waves' are
// added in LDS, the chunks' of a request through the workspace.
#pragma once

#include <type_traits>

#include "ifx_attn.h"

namespace ifx {

constexpr int kRowWaves = 4;

// LDS of the waves' maxima and sums.
struct RowSums {
  float m[kRowWaves][32], l[kRowWaves][32];
};

// Of a wave the lanes with the same n hold row n, one of them (lead) besides the
// others its maximum m and sum l; exponents are (s - m) c.  put(scale): the
// lane writes its part of the row's sums, times scale, to red[wave][D / 4][R][4].
// red later holds [chunk][row].  slot_bytes: of a chunk's place in the workspace.
// The R rows are those from row0 on of the request, its row block number `block`,
// whose keys are cut into ns chunks, this one z.  none(t): whether the rows of new
// token t see nothing.  kAtOnce: chunks whose sums a thread reads at a time, 4
// registers each.  GROUPED: for many rows, of several places at a time.  A tree of
// 64 nodes, 3000 keys, 16 / 2 heads of 128: 23.1 us with it and 24.9 without, over the
// 8-bit cache 22.2 and 24.8; 49 rows of 450 keys, 28 / 4 heads of 256, 22.4 and 31.0.
// Single tokens, which have no such places, lost 0.3 by the longer code.
template <int D, int kAtOnce = 24, bool GROUPED = true, class Put, class None>
__device__ __forceinline__ void rows_finish(const AttnArgs &a, const Split &split, float *red,
                                            RowSums &sums, int n, bool lead, float m, float l,
                                            float c, uint32_t slot_bytes, int R, int block, int z, int ns,
                                            int kvh, Put put, None none) {
  constexpr uint32_t kOut = 1u << 30;  // an offset past the workspace's end: reads zeros
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q0 = split.req.q0, row0 = block * 32;

  // the four waves' sums, in the waves' order
  if (lead) {
    sums.m[wave][n] = m;
    sums.l[wave][n] = l;
  }
  __syncthreads();
  float top = sums.m[0][n];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) top = fmaxf(top, sums.m[w][n]);
  if (n < R) put(weight(m, top, c));
  float lt = 0.0f;  // of row n
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    const float mw = sums.m[w][n];
    lt += sums.l[w][n] * weight(mw, top, c);
  }
  __syncthreads();  // all waves have read sums.m / sums.l
  if (wave == 0 && lead) {
    sums.m[0][n] = top;
    sums.l[0][n] = lt;
  }
  __syncthreads();

  const int elems = R * (D / 4);  // groups of four dims of a row
  const int head0 = kvh * a.G;
  if (ns == 1) {
    for (int i = tid; i < elems; i += 256) {
      const int r = i % R, d4 = i / R;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kRowWaves; ++w) v += ldg<f32x4>(red + ((w * (D / 4) + d4) * R + r) * 4);
      const int row = row0 + r, t = row / a.G;
      // a row that sees no key is 0; one whose keys all weigh nothing is not a number
      const float inv = 1.0f / sums.l[0][r];
      v = none(t) ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v * inv;
      char *o = static_cast<char *>(a.out) +
                ((q0 + t) * a.out_stride + static_cast<int64_t>(head0 + row % a.G) * D) *
                    dtype_bytes(a.out_dtype);
      store4(o, a.out_dtype, d4 * 4, v);
    }
    return;
  }

  // split: this chunk's sums to its slot, (m, l) of its rows behind them
  const rsrc_t part = make_rsrc(a.part, a.part_bytes);
  const uint32_t first = split.slot * a.Hkv + (block * a.Hkv + kvh) * split.ns;  // the block's slots
  const uint32_t slot0 = first * slot_bytes;
  const uint32_t slot = slot0 + z * slot_bytes;
  for (int i = tid; i < elems; i += 256) {
    const int r = i % R, d4 = i / R;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) v += ldg<f32x4>(red + ((w * (D / 4) + d4) * R + r) * 4);
    st_dev4(part, slot + i * 16, v);
  }
  if (tid < R) st_dev4(part, slot + (elems + tid) * 16, f32x4{sums.m[0][tid], sums.l[0][tid], 0.0f, 0.0f});
  wait_own_memory();
  uint32_t *cnt = a.cnt + first;
  if (!split_arrive_last(cnt, ns)) return;
  // [chunk][row] maximum, then weight, and sum: the waves' sums are no longer needed
  float2 *ml = reinterpret_cast<float2 *>(red);
  const auto weights = [&]() __attribute__((always_inline)) {
    const int r = tid >> 3, j = tid & 7;  // eight lanes for a row
    float mx = -__builtin_inff(), sum = 0.0f;
    if (r < R) {
      for (int y0 = j; y0 < ns; y0 += 32) {
        f32x4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int y = y0 + 8 * i;
          u[i] = ld_dev4(part, y < ns ? slot0 + y * slot_bytes + (elems + r) * 16 : kOut);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int y = y0 + 8 * i;
          if (y < ns) {
            ml[y * R + r] = make_float2(u[i].x, u[i].y);
            mx = fmaxf(mx, u[i].x);
          }
        }
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      for (int y = j; y < ns; y += 8) {
        const float2 u = ml[y * R + r];
        const float w = weight(u.x, mx, c);
        ml[y * R + r].x = w;
        sum += u.y * w;
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor(sum, o);
      if (j == 0) sums.l[0][r] = 1.0f / sum;
    }
  };
  // Reads past the L2 take a microsecond: a thread's first sums are on their way
  // while the chunks' weights are formed, and where there are few chunks those of
  // GROUPS of its places at a time.
  const auto add = [&](auto groups_c) __attribute__((always_inline)) {
    constexpr int GROUPS = decltype(groups_c)::value, kY = kAtOnce / GROUPS;
    f32x4 v[GROUPS][kY];
    auto read = [&](int i, int y0) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int y = 0; y < kY; ++y)
          v[g][y] = ld_dev4(part, i + 256 * g < elems && y0 + y < ns
                                      ? slot0 + (y0 + y) * slot_bytes + (i + 256 * g) * 16 : kOut);
    };
    read(tid, 0);
    __builtin_amdgcn_sched_barrier(0);
    weights();
    __syncthreads();
    for (int i0 = tid; i0 < elems; i0 += 256 * GROUPS) {
      f32x4 o[GROUPS] = {};
      for (int y0 = 0; y0 < ns; y0 += kY) {
        if (i0 != tid || y0) read(i0, y0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int r = (i0 + 256 * g) % R;
#pragma unroll
          for (int y = 0; y < kY; ++y) o[g] += v[g][y] * (y0 + y < ns ? ml[(y0 + y) * R + r].x : 0.0f);
        }
      }
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int i = i0 + 256 * g;
        if (i >= elems) break;
        const int r = i % R, d4 = i / R, row = row0 + r, t = row / a.G;
        const f32x4 x = none(t) ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o[g] * sums.l[0][r];
        char *to = static_cast<char *>(a.out) +
                   ((q0 + t) * a.out_stride + static_cast<int64_t>(head0 + row % a.G) * D) *
                       dtype_bytes(a.out_dtype);
        store4(to, a.out_dtype, d4 * 4, x);
      }
    }
  };
  if (GROUPED && ns * 4 <= kAtOnce && elems > 512)
    add(std::integral_constant<int, 4>{});
  else if (GROUPED && ns * 2 <= kAtOnce && elems > 256)
    add(std::integral_constant<int, 2>{});
  else
    add(std::integral_constant<int, 1>{});
  split_reset(cnt);
}

// put of 32-row accumulators: acc[d][r] of lane half h is dim 32 d + 8 (r / 4) + 4 h + r % 4.
template <int D>
__device__ __forceinline__ void put_rows32(float *red, const f32x16 (&acc)[D / 32], float scale, int R) {
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = acc[d][4 * g + r] * scale;
      __builtin_memcpy(red + ((wave * (D / 4) + 8 * d + 2 * g + h) * R + n) * 4, &v, 16);
    }
}

}  // namespace ifx
