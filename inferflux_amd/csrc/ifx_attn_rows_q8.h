// ifx_attn_rows_q8.h -- a chunk of keys of the 8-bit cache for up to 32 query
// rows: what attn_rows_q8.hip runs for all its requests, and attn_tile_q8.hip for
// those of a batch that have few rows.
#pragma once

#include "ifx_attn_q8.h"
#include "ifx_attn_rows.h"
#include "ifx_attn_work.h"

namespace ifx {

// Key of A-operand row m of S^T = K Q^T: with register r of lane half h as key
// 16 h + r, the probabilities of a half are those of one piece of V's 16 tokens.
__device__ __forceinline__ int key_of_row16(int m) {
  return (m & 3) | ((m >> 1) & 0xC) | ((m & 4) << 2);
}

constexpr int kStep = 32 * kRowWaves;  // keys from a wave's tile to its next
constexpr int kDepth = 2;              // tiles that are on their way or worked on
// 16-byte places of a tile in LDS: K, V, and 64 dwords of scales (32 keys', twice).
template <int D>
constexpr int tile_pieces() {
  return 2 * (D / 32) * 64 + 16;
}

// LDS of rows32_q8's tiles: [wave][tile][piece].
template <int D>
constexpr int rows32_bytes() {
  return kRowWaves * kDepth * tile_pieces<D>() * 16;
}

__device__ __forceinline__ bool rows_work(const AttnArgs &a, float *reqs, int lds_rows, int blocks, RowsWork &w) {
  return rows_work(a, find_item<1, kRowsRoot>(a, reinterpret_cast<int2 *>(reqs), blockIdx.x / a.Hkv,
                                   [&](const Request &r) { return rows_units(a, r, blocks); }),
                   kRowKeys, lds_rows, w);
}

// What a lane's row sees.
struct RowSight {
  bool tree;
  Sight<false> line;
  Sight<true> nodes;
  __device__ __forceinline__ RowSight(const AttnArgs &a, const RowsWork &w, int tok)
      : tree(w.tree), line{a.window > 0 ? max(0, w.ctx + tok - a.window + 1) : 0, w.ctx + tok, w.ctx, 0},
        nodes{0, 0, w.ctx, 0} {
    if (tree) nodes.bits = node_bits(a, w.q0 + tok, w.nq);
  }
  __device__ __forceinline__ bool sees(int key) const { return tree ? nodes.sees(key) : line.sees(key); }
};
// Whether some row may not see all of the 32 keys from k0 on.
__device__ __forceinline__ bool in_part(const AttnArgs &a, const RowsWork &w, int k0) {
  return k0 + 31 >= w.ctx + !w.tree || (a.window > 0 && k0 < w.ctx + w.nq - a.window);
}
// Whether the rows of new token t see nothing.
__device__ __forceinline__ bool row_sees_nothing(const AttnArgs &a, const RowsWork &w, int t) {
  return w.tree ? Sight<true>{0, 0, w.ctx, node_bits(a, w.q0 + t, w.nq)}.nothing() : w.ctx + t < 0;
}

// The pages of the two 16-key halves of a wave's tiles, as the table has them: of
// 64 tiles at a time, a lane each.
struct Pages {
  const int32_t *table;
  int sh, wmax, last, first, entry0, entry1;
  __device__ __forceinline__ Pages(const AttnArgs &a, int b, int kfirst)
      : table(a.table + static_cast<int64_t>(b) * a.table_width), sh(a.page_shift),
        wmax(a.table_width - 1), last(static_cast<int>(a.num_pages) - 1), first(kfirst) {}
  __device__ __forceinline__ void read(int t) {
    const int64_t k = first + static_cast<int64_t>(t + (threadIdx.x & 63)) * kStep;
    entry0 = table[min(k >> sh, static_cast<int64_t>(wmax))];
    entry1 = table[min((k + 16) >> sh, static_cast<int64_t>(wmax))];
    wait_loads<0>();  // here, so that no later use of them waits for tiles
  }
  __device__ __forceinline__ int page0(int t) const {
    return min(max(__builtin_amdgcn_readlane(entry0, t & 63), 0), last);
  }
  __device__ __forceinline__ int page1(int t) const {
    return min(max(__builtin_amdgcn_readlane(entry1, t & 63), 0), last);
  }
};

// red: at first [wave][tile][piece], then [wave][D / 4][row][4], then a chunk's
// weights; 16-byte aligned.  slot_bytes: of a chunk's place in the workspace.
template <int D>
__device__ __forceinline__ void rows32_q8(const AttnArgs &a, const RowsWork &w, float *red, RowSums &sums,
                                          uint32_t slot_bytes, int kvh) {
  constexpr int ND = D / 32, NS = D / 16;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int sh = a.page_shift, P = 1 << sh;

  const int row = row_of_lane(w, n), tok = row / a.G, head = kvh * a.G + row % a.G;
  const RowSight sight(a, w, tok);
  u32x4 qf[NS];
  {  // of step s the dims 32 (s / 2) + 16 h + 8 (s % 2), as K's pieces hold them
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + (w.q0 + tok) * a.q_stride +
                        static_cast<int64_t>(head) * D + 16 * h;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = ldg<u32x4>(q + 32 * (s >> 1) + 8 * (s & 1));
  }

  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
  Level level;
  float l = 0.0f;

  // ---- tiles: memory to LDS past the registers, each lane's pieces to its own
  // places, so that no wave waits for another
  const int kn = key_of_row16(n);  // the key of a tile whose K this lane takes
  const int64_t page_bytes = (static_cast<int64_t>(a.Hkv) * D) << sh;
  const uint8_t *K = static_cast<const uint8_t *>(a.k) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint8_t *V = static_cast<const uint8_t *>(a.v) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint32_t *S = a.scales + (static_cast<int64_t>(kvh) << sh);
  constexpr int kPieces = tile_pieces<D>(), kLoads = 2 * ND + 1;  // of a tile
  u32x4 *ring = reinterpret_cast<u32x4 *>(red) + wave * kDepth * kPieces;
  const int kfirst = w.zbeg + 32 * wave, tiles = (w.zend - kfirst + kStep - 1) / kStep;
  Pages pages(a, w.b, kfirst);
  auto issue = [&](int t) __attribute__((always_inline)) {
    if (t && (t & 63) == 0) pages.read(t);
    const int k0 = kfirst + t * kStep, pg0 = pages.page0(t), pg1 = pages.page1(t);
    u32x4 *to = ring + (t & (kDepth - 1)) * kPieces;
    const uint8_t *kp = K + (kn & 16 ? pg1 : pg0) * page_bytes +
                        ((((k0 + kn) & (P - 1)) + (h << sh)) * 16);
#pragma unroll
    for (int i = 0; i < ND; ++i) to_lds16(kp + ((i * 32) << sh), to + i * 64);
    const uint32_t *sp = S + ((static_cast<int64_t>(n & 16 ? pg1 : pg0) * a.Hkv) << sh) +
                         ((k0 + n) & (P - 1));
    to_lds4(sp, to + 2 * ND * 64);
    const uint8_t *vp = V + (h ? pg1 : pg0) * page_bytes + ((k0 + 16 * h) & (P - 1)) * D + n * 16;
#pragma unroll
    for (int d = 0; d < ND; ++d) to_lds16(vp + d * 512, to + (ND + d) * 64);
  };

  pages.read(0);  // and the rows of Q are here
  const float c = row_to_f16<32>(qf, a.q_dtype, a.c);
#pragma unroll
  for (int t = 0; t < kDepth; ++t)
    if (t < tiles) issue(t);
#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    const int k0 = kfirst + t * kStep;
    const u32x4 *from = ring + (t & (kDepth - 1)) * kPieces;
    if (t + 1 < tiles)
      wait_loads<(kDepth - 1) * kLoads>();
    else
      wait_loads<0>();
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const u32x4 k = from[i * 64 + lane];
      s = F16::mfma32(codes_f16(k, 0), qf[2 * i], s);
      s = F16::mfma32(codes_f16(k, 1), qf[2 * i + 1], s);
    }
    float sv[16];
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const u32x4 f = from[2 * ND * 64 + 4 * h + (r >> 2)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[r + j] *= k_scale(f[j]);
        sv[r + j] = v_scale(f[j]);
      }
    }
    if (in_part(a, w, k0)) {  // what the row does not see, a page's unwritten slots among it
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool sees = sight.sees(k0 + 16 * h + r);
        s[r] = sees ? s[r] : -__builtin_inff();
        sv[r] = sees ? sv[r] : 0.0f;
      }
    }
    float mt = s[0], vt = sv[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]), vt = fmaxf(vt, sv[r]);
    mt = halves_max(mt), vt = halves_max(vt);
    if (__any(level.above(mt, vt, c))) {
      const float less = level.raise(mt, vt, c);
      l *= less;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= less;
    }
    u32x4 pf[2];
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -level.less));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], c, -level.less));
      sum += p0 + p1;
      pf[r >> 3][(r & 7) >> 1] = F16::pack(p0 * sv[r], p1 * sv[r + 1]);
    }
    l += sum;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const u32x4 v = from[(ND + d) * 64 + lane];
      acc[d] = F16::mfma32(codes_f16(v, 0), pf[0], acc[d]);
      acc[d] = F16::mfma32(codes_f16(v, 1), pf[1], acc[d]);
    }
    __builtin_amdgcn_sched_barrier(0);  // the tile's places are read
    if (t + kDepth < tiles) issue(t + kDepth);
  }

  l = halves_sum(l);
  const float level_of = level.of_sums(), top = rows_top(sums, wave, n, h == 0, level_of, l);
  if (n < w.R) put_rows32<D>(red, acc, weight(level_of, top, 1.0f), w.R, n, h, wave);
  rows_finish<D>(a, w.split, red, sums, n, h == 0, top, 1.0f, slot_bytes, w.R, w.block, w.z, w.ns, kvh,
                 [&](int t) { return row_sees_nothing(a, w, t); });
}

}  // namespace ifx
