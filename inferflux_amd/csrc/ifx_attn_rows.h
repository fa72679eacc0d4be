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

// The largest maximum of the four waves' rows n, behind which all waves have written
// to `sums`.  Of a wave the lanes with the same n hold row n, one of them (lead)
// besides the others its maximum m and sum l; exponents are (s - m) c.
__device__ __forceinline__ float rows_top(RowSums &sums, int wave, int n, bool lead, float m, float l) {
  if (lead) {
    sums.m[wave][n] = m;
    sums.l[wave][n] = l;
  }
  __syncthreads();
  float top = sums.m[0][n];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) top = fmaxf(top, sums.m[w][n]);
  return top;
}

// The sums of a block's chunks in the workspace.
struct ChunkSums {
  rsrc_t part;  // up to the last chunk's end: what is read of further ones is zeros
  uint32_t slot0, slot_bytes;  // bytes: of the first chunk's, of each
  int ns, R, elems;            // chunks, rows, groups of four dims of a row
  static constexpr uint32_t kOut = 1u << 30;  // an offset past the workspace's end: reads zeros
  __device__ __forceinline__ f32x4 read(int y, int i) const {
    return ld_dev4(part, i < elems ? slot0 + y * slot_bytes + i * 16 : kOut);
  }
};

// [chunk][row] maximum, then weight, and sum to ml; the rows' totals, inverted, to
// sums.l[0].
__device__ __forceinline__ void chunk_weights(ChunkSums k, float2 *ml, RowSums &sums, float c) {
  const int r = threadIdx.x >> 3, j = threadIdx.x & 7;  // eight lanes for a row
  if (r >= k.R) return;
  float mx = -__builtin_inff(), sum = 0.0f;
  for (int y0 = j; y0 < k.ns; y0 += 32) {
    f32x4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int y = y0 + 8 * i;
      u[i] = ld_dev4(k.part, y < k.ns ? k.slot0 + y * k.slot_bytes + (k.elems + r) * 16 : ChunkSums::kOut);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int y = y0 + 8 * i;
      if (y < k.ns) {
        ml[y * k.R + r] = make_float2(u[i].x, u[i].y);
        mx = fmaxf(mx, u[i].x);
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  for (int y = j; y < k.ns; y += 8) {
    const float2 u = ml[y * k.R + r];
    const float w = weight(u.x, mx, c);
    ml[y * k.R + r].x = w;
    sum += u.y * w;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor(sum, o);
  if (j == 0) sums.l[0][r] = 1.0f / sum;
}

// Where a block's rows are written.
struct RowsOut {
  int q0, row0, head0;
  template <int D>
  __device__ __forceinline__ void write(const AttnArgs &a, int r, int d4, f32x4 v) const {
    const int row = row0 + r, t = row / a.G;
    char *to = static_cast<char *>(a.out) +
               ((q0 + t) * a.out_stride + static_cast<int64_t>(head0 + row % a.G) * D) *
                   dtype_bytes(a.out_dtype);
    store4(to, a.out_dtype, d4 * 4, v);
  }
};

// Adds the chunks' sums.  Reads past the L2 take a microsecond: a thread's first
// sums are on their way while the chunks' weights are formed, and where there are
// few chunks those of GROUPS of its places at a time.
template <int D, int GROUPS, int kAtOnce, class None>
__device__ __forceinline__ void add_chunks(const AttnArgs &a, ChunkSums k, float2 *ml, RowSums &sums,
                                           float c, RowsOut out, None none) {
  constexpr int kY = kAtOnce / GROUPS;
  const int tid = threadIdx.x;
  f32x4 v[GROUPS][kY];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
#pragma unroll
    for (int y = 0; y < kY; ++y) v[g][y] = k.read(y, tid + 256 * g);
  __builtin_amdgcn_sched_barrier(0);
  chunk_weights(k, ml, sums, c);
  __syncthreads();
  for (int i0 = tid; i0 < k.elems; i0 += 256 * GROUPS) {
    f32x4 o[GROUPS] = {};
    for (int y0 = 0; y0 < k.ns; y0 += kY) {
      if (i0 != tid || y0) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
          for (int y = 0; y < kY; ++y) v[g][y] = k.read(y0 + y, i0 + 256 * g);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int r = (i0 + 256 * g) % k.R;
#pragma unroll
        for (int y = 0; y < kY; ++y) o[g] += v[g][y] * (y0 + y < k.ns ? ml[(y0 + y) * k.R + r].x : 0.0f);
      }
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int i = i0 + 256 * g;
      if (i >= k.elems) break;
      const int r = i % k.R, d4 = i / k.R;
      out.write<D>(a, r, d4, none((out.row0 + r) / a.G) ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o[g] * sums.l[0][r]);
    }
  }
}

// Behind rows_top, and behind the waves' writing of their sums times weight(m, top, c)
// to red[wave][D / 4][R][4] (put_rows32).  red later holds [chunk][row].  slot_bytes:
// of a chunk's place in the workspace.  The R rows are those from row0 on of the
// request, its row block number `block`, whose keys are cut into ns chunks, this one
// z.  none(t): whether the rows of new token t see nothing.  kAtOnce: chunks whose
// sums a thread reads at a time, 4 registers each.  GROUPED: for many rows, of several
// places at a time.  A tree of 64 nodes, 3000 keys, 16 / 2 heads of 128: 17.7 us with
// it and 21.0 without, over the 8-bit cache 17.0 and 20.5; 49 rows of 450 keys, 28 / 4
// heads of 256, 22.3 and 31.0.  Single tokens have no such places and gain nothing.
//
// In functions with values as arguments, not closures: accumulators that a closure
// held by reference took 12 vector registers more, which with heads of 64 left two
// waves a SIMD instead of three: 16.5 us instead of 14.1 for 8 requests of 300 to 4000
// keys, 32 / 8 heads, 133 instead of 118 for 32 of 500 to 24000, 12 / 12 heads.
template <int D, int kAtOnce = 24, bool GROUPED = true, class None>
__device__ __forceinline__ void rows_finish(const AttnArgs &a, const Split &split, float *red,
                                            RowSums &sums, int n, bool lead, float top, float c,
                                            uint32_t slot_bytes, int R, int block, int z, int ns,
                                            int kvh, None none) {
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RowsOut out = {split.req.q0, block * 32, kvh * a.G};

  // the four waves' sums, in the waves' order
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
  if (ns == 1) {
    for (int i = tid; i < elems; i += 256) {
      const int r = i % R, d4 = i / R;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kRowWaves; ++w) v += ldg<f32x4>(red + ((w * (D / 4) + d4) * R + r) * 4);
      // a row that sees no key is 0; one whose keys all weigh nothing is not a number
      const float inv = 1.0f / sums.l[0][r];
      out.write<D>(a, r, d4, none((out.row0 + r) / a.G) ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v * inv);
    }
    return;
  }

  // split: this chunk's sums to its slot, (m, l) of its rows behind them
  const uint32_t first = split.slot * a.Hkv + (block * a.Hkv + kvh) * split.ns;  // the block's slots
  const ChunkSums k = {make_rsrc(a.part, min(a.part_bytes, (first + ns) * slot_bytes)), first * slot_bytes,
                       slot_bytes, ns, R, elems};
  const uint32_t slot = k.slot0 + z * slot_bytes;
  for (int i = tid; i < elems; i += 256) {
    const int r = i % R, d4 = i / R;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) v += ldg<f32x4>(red + ((w * (D / 4) + d4) * R + r) * 4);
    st_dev4(k.part, slot + i * 16, v);
  }
  if (tid < R) st_dev4(k.part, slot + (elems + tid) * 16, f32x4{sums.m[0][tid], sums.l[0][tid], 0.0f, 0.0f});
  wait_own_memory();
  uint32_t *cnt = a.cnt + first;
  if (!split_arrive_last(cnt, ns)) return;
  float2 *ml = reinterpret_cast<float2 *>(red);  // the waves' sums are no longer needed
  if (GROUPED && ns * 4 <= kAtOnce && elems > 512)
    add_chunks<D, 4, kAtOnce>(a, k, ml, sums, c, out, none);
  else if (GROUPED && ns * 2 <= kAtOnce && elems > 256)
    add_chunks<D, 2, kAtOnce>(a, k, ml, sums, c, out, none);
  else
    add_chunks<D, 1, kAtOnce>(a, k, ml, sums, c, out, none);
  split_reset(cnt);
}

// 32-row accumulators times scale to red[wave][D / 4][R][4]: acc[d][r] of lane half h
// is dim 32 d + 8 (r / 4) + 4 h + r % 4.
template <int D>
__device__ __forceinline__ void put_rows32(float *red, const f32x16 (&acc)[D / 32], float scale, int R,
                                           int n, int h, int wave) {
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
