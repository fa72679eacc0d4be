// ifx_attn_tile.h -- what the attention kernels of many query rows
// (attn_tile.hip, attn_tile_q8.hip) do with their sums: written as they are,
// or added to those of a row tile's other chunks of keys through the workspace.
#pragma once

#include "ifx_attn.h"

namespace ifx {

constexpr int kTileWaves = 4;                // of a workgroup
constexpr int kQueryRows = 32 * kTileWaves;   // its query rows
// Bytes of the workspace that a wave's sums of a chunk take, and the workgroup's.
template <int D>
constexpr uint32_t tile_wave_bytes() {
  return 32 * D * 4 + 64 * 4 * 2;
}
template <int D>
constexpr uint32_t tile_slot_bytes() {
  return kTileWaves * tile_wave_bytes<D>();
}

// Lane n of each half of a wave holds row 128 tile + 32 wave + n of the
// request's R: maximum m and sum l, and in acc the dims
// 32 d + 8 (r / 4) + 4 h + r % 4.  Exponents are (s - m) c.  nothing(t):
// whether the rows of new token t see no key.
template <int D, bool SPLIT, class Nothing>
__device__ __forceinline__ void tile_finish(const AttnArgs &a, const Split &split,
                                            const f32x16 (&acc)[D / 32], float m, float l, float c,
                                            int tile, int z, int ns, int kvh, int R,
                                            Nothing nothing) {
  constexpr int ND = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = tile * kQueryRows;
  const int q0 = __builtin_amdgcn_readfirstlane(split.req.q0);
  int row = min(row0 + 32 * wave + n, R - 1), tok = row / a.G;
  int head = kvh * a.G + row - tok * a.G;

  l = halves_sum(l);
  bool none = nothing(tok);  // the row sees no key
  bool own = row0 + 32 * wave + n < R;
  auto write_dims = [&](int d, const f32x4 *v, float scale) __attribute__((always_inline)) {  // of one dim tile
    if (!own) return;
    char *o = static_cast<char *>(a.out) +
              ((q0 + tok) * a.out_stride + static_cast<int64_t>(head) * D) * dtype_bytes(a.out_dtype);
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4(o, a.out_dtype, 32 * d + 8 * g + 4 * h, none ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v[g] * scale);
  };
  auto write = [&](float scale) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      f32x4 v[4];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i >> 2][i & 3] = acc[d][i];
      write_dims(d, v, scale);
    }
  };
  if (!SPLIT || ns == 1) return write(1.0f / l);

  // split: this chunk's sums to its slot, every lane in its own places; the
  // last workgroup of the tile adds the chunks in their order, lane by lane.
  // Lanes without a row have their places behind the buffer's end: they write
  // nothing and read zeros.
  const rsrc_t part = make_rsrc(a.part, a.part_bytes);
  constexpr uint32_t kWaveBytes = tile_wave_bytes<D>(), kSlotBytes = tile_slot_bytes<D>();
  const uint32_t first = split.slot * a.Hkv + (tile * a.Hkv + kvh) * split.ns;  // the tile's slots
  constexpr uint32_t kOut = 1u << 30;
  const uint32_t out = row0 + 32 * wave + n < R ? 0 : kOut;
  uint32_t mine = (first * kSlotBytes + wave * kWaveBytes + lane * 16) | out;
  uint32_t mine_ml = (first * kSlotBytes + wave * kWaveBytes + 32 * D * 4 + lane * 8) | out;
  {
    const uint32_t at = mine + z * kSlotBytes;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        st_dev4(part, at + (4 * d + g) * 1024,
                f32x4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]});
    __builtin_amdgcn_raw_buffer_store_b64(
        __builtin_bit_cast(u32x2, make_float2(m, l)), part, mine_ml + z * kSlotBytes, 0, kAuxDevice);
  }
  wait_own_memory();
  uint32_t *cnt = a.cnt + first;
  if (!split_arrive_last(cnt, ns)) return;
  const bool few = R - row0 <= 32;  // all rows are the first wave's: the waves share the dims
  if (few) {
    row = min(row0 + n, R - 1), tok = row / a.G, head = kvh * a.G + row - tok * a.G;
    own = row0 + n < R;
    none = nothing(tok);
    const uint32_t at = first * kSlotBytes | (own ? 0 : kOut);
    mine = at + lane * 16, mine_ml = at + 32 * D * 4 + lane * 8;
  }
  auto ml_of = [&](int y) {  // of chunk y, and past the last of none
    return __builtin_bit_cast(
        float2, __builtin_amdgcn_raw_buffer_load_b64(
                    part, y < ns ? mine_ml + y * kSlotBytes : kOut, 0, kAuxDevice));
  };
  // Reads past the L2 take a microsecond: several at a time
  float top = -__builtin_inff(), total = 0.0f;
  for (int y0 = 0; y0 < ns; y0 += 8) {
    float2 ml[8];
#pragma unroll
    for (int y = 0; y < 8; ++y) ml[y] = ml_of(y0 + y);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      const float my = y0 + y < ns ? ml[y].x : -__builtin_inff();
      const float mn = fmaxf(top, my);
      total = __builtin_fmaf(total, weight(top, mn, c), ml[y].y * weight(my, mn, c));
      top = mn;
    }
  }
  // N dim tiles from d on, four chunks at a time
  auto add_chunks = [&](int d, auto n_c) __attribute__((always_inline)) {
    constexpr int N = decltype(n_c)::value;
    f32x4 o[4 * N] = {};
    for (int y0 = 0; y0 < ns; y0 += 4) {
      float2 ml[4];
      f32x4 v[4][4 * N];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        ml[y] = ml_of(y0 + y);
        const uint32_t at = y0 + y < ns ? mine + (y0 + y) * kSlotBytes + d * 4096 : kOut;
#pragma unroll
        for (int g = 0; g < 4 * N; ++g) v[y][g] = ld_dev4(part, at + g * 1024);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float w = y0 + y < ns ? weight(ml[y].x, top, c) : 0.0f;
#pragma unroll
        for (int g = 0; g < 4 * N; ++g) o[g] += v[y][g] * w;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) write_dims(d + i, o + 4 * i, 1.0f / total);
  };
  using one = std::integral_constant<int, 1>;
  using two = std::integral_constant<int, 2>;
  if (few || D == 64) {  // (D = 64: registers of three waves a SIMD)
#pragma unroll 1
    for (int d = few ? wave : 0; d < ND; d += few ? kTileWaves : 1) add_chunks(d, one{});
  } else {
#pragma unroll 1
    for (int d = 0; d + 1 < ND; d += 2) add_chunks(d, two{});
    if constexpr (ND % 2) add_chunks(ND - 1, one{});
  }
  split_reset(cnt);
}

}  // namespace ifx
