// ifx_attn.h -- what the attention kernels (kv_plan.hip, rope_append.hip,
// attn_rows.hip, attn_tile.hip) and their entry points (attention_api.hip)
// share.
#pragma once

#include <atomic>

#include "ifx_attention.h"
#include "ifx_common.h"

namespace ifx {

constexpr float kLog2e = 1.44269504088896340736f;

// Probabilities are rounded to the caches' type for the product with V: its
// MFMA takes 16-bit operands, in fp32 it runs at a sixteenth of the rate, and
// two 16-bit parts of each would be half as many products again.  The row sums
// take them unrounded.  Against 64 bits an output is off by 0.0020 to 0.0023 of
// its size in bf16 and 0.00023 to 0.00028 in fp16, where rounding the output
// alone leaves 0.0017 and 0.0002.
//
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
  int goal;    // paged: work items of a key/value head (find_item)
  uint32_t *cnt;
  float *part;
  uint32_t part_bytes;
};

// Query rows of one key/value head: row r of a request is query head r % G of
// the group and new token r / G.
//
// Rows of a request that attn_rows takes: what one of its MFMA tiles holds.  It
// is made for decode steps, and drafts of many tokens would gain from a lower
// bound where there are several requests.  us with attn_rows / attn_tile:
//   16 / 2 heads of 128, rows     8          16         24         32
//     1 request of 3000 keys  10.1/18.3  12.3/18.3  14.9/18.4  17.5/18.5
//     8                       12.4/19.5  15.7/19.4  19.6/19.6  23.8/19.9
//     32 of 6000              39.5/38.7  43.3/39.0  48.1/39.5  45.0/40.1
//   40 / 8 heads, rows            5          15         20         30
//     1 request of 3000 keys   9.6/18.1  12.3/18.3  14.5/18.4  17.3/18.6
//     8                       26.1/26.6  29.6/26.8  33.0/26.9  37.3/27.6
//     32 of 6000               144/152    150/152    155/154    162/154
constexpr int kRowsMax = 32;
constexpr int kRowKeys = 128;  // attn_rows: keys of a stage, 32 for each wave
constexpr int kTileKeys = 64;  // attn_tile: keys of a stage

// Inclusive sums over the lanes, in the vector unit's own lane moves: shifts by
// 1, 2, 4, 8 within 16 lanes, then the last lane of each 16 to the next, and of
// the first 32 to the others.
struct Add {
  template <class V>
  __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ int operator()(int a, int b) const { return max(a, b); }
};
template <int CTRL, int ROWS, class Op, class V>
__device__ __forceinline__ V with_moved(V v) {  // lanes that get none: with 0
  return Op()(v, __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false)));
}
template <class Op = Add, class V>
__device__ __forceinline__ V wave_scan(V v) {
  v = with_moved<0x111, 0xF, Op>(v);
  v = with_moved<0x112, 0xF, Op>(v);
  v = with_moved<0x114, 0xF, Op>(v);
  v = with_moved<0x118, 0xF, Op>(v);
  v = with_moved<0x142, 0xA, Op>(v);
  return with_moved<0x143, 0xC, Op>(v);
}
template <class Op = Add, class V>
__device__ __forceinline__ V wave_sum(V v) {
  return __builtin_bit_cast(
      V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan<Op>(v)), 63));
}

struct Request {
  int q0, nq, kv;  // first new token, new tokens, tokens
};
__device__ __forceinline__ Request request_of(const AttnArgs &a, int b) {
  const int c0 = min(max(a.cu[b], 0), a.T), c1 = min(max(a.cu[b + 1], 0), a.T);
  return {c0, max(c1 - c0, 0), min(max(a.kv_len[b], 0), a.table_width << a.page_shift)};
}

// ceil(x / d) for 0 <= x <= 2^24 with r = 1 / d: the product is off by less than 1.
__device__ __forceinline__ int ceil_div(int x, int d, float r) {
  const int q = static_cast<int>(static_cast<float>(x) * r), rest = x - q * d;
  return q + (rest > 0) + (rest > d) - (rest <= -d);
}

// Chunks of a request of x stages: of `chunk` (r = 1 / chunk), or of least at least.
template <int LEAST>
__device__ __forceinline__ int chunks_of(int x, int chunk, float r) {
  return min(ceil_div(x, chunk, r), max(x / LEAST, 1));
}

// A piece of paged work: item `item` (chunk major) of request b's `tiles` row
// tiles x ns chunks of `chunk` stages.  chunk is 0 where there is no such item.
struct Split {
  int chunk, ns, slot;  // ns: of the request; slot: of the split sums of its first tile
  int b, item, tiles;
  Request req;
};

// Item i of the batch (for one key/value head).  No list of work is built
// beforehand: the workgroups' waves find it, each for itself, from the
// requests' {row tiles, stages}, work(request); beyond 64 requests by way of
// LDS (reqs).  The work is cut so that about a.goal items of one length come
// out.  At most a.goal items belong to split tiles: all items are no more, or
// else chunks are so long that a request of s > c stages, cut in less than
// s / c + 1 < 2 s / c of them, leaves no more.  Lane l has requests l, l + 64,
// ...: their places in LDS are neighbours' (with consecutive ones a lane, 1024
// prompts of 30 to 60 tokens of 16 / 2 heads took 283 us; 177 now).
template <int MIN_CHUNK, class Work>
__device__ __forceinline__ Split find_item(const AttnArgs &a, int2 *reqs, int i, Work work) {
  const int lane = threadIdx.x & 63, B = a.B, goal = a.goal;
  Request req = {0, 0, 0};
  int2 mine = {0, 1};  // the lane's first request, `lane`; 64 on from there its others
  Split f = {};
  if (B == 1) {  // nothing to be weighed against each other
    f.req = request_of(a, 0);
    const int2 r = work(f.req);
    f.chunk = r.y, f.ns = 1, f.item = i, f.tiles = r.x;
    if (goal >= r.x && r.x > 0) {
      const int share = r.x == 1 ? goal : goal / r.x;  // chunks of a tile
      f.chunk = max(MIN_CHUNK, ceil_div(r.y, share, __builtin_amdgcn_rcpf(static_cast<float>(share))));
      f.ns = chunks_of<MIN_CHUNK>(r.y, f.chunk, __builtin_amdgcn_rcpf(static_cast<float>(f.chunk)));
      f.chunk = (r.y + f.ns - 1) / f.ns;  // of equal length
    }
    f.chunk = i < r.x * f.ns ? __builtin_amdgcn_readfirstlane(f.chunk) : 0;
    f.ns = __builtin_amdgcn_readfirstlane(f.ns);
    return f;
  }
  if (B <= 64) {
    if (lane < B) {
      req = request_of(a, lane);
      mine = work(req);
    }
  } else {
    for (int b = threadIdx.x; b < B; b += blockDim.x) reqs[b] = work(request_of(a, b));
    __syncthreads();
    mine = reqs[lane];
  }
  auto each = [&](auto f) __attribute__((always_inline)) {
    f(mine);
#pragma unroll 4
    for (int b = lane + 64; b < B; b += 64) f(reqs[b]);
  };
  int chunk = 1 << 25;
  float inv = 1.0f / chunk;
  if (goal > 0) {
    float stages = 0.0f, tiles = 0.0f;
    each([&](int2 r) {
      tiles += static_cast<float>(r.x);
      stages += static_cast<float>(r.x) * static_cast<float>(r.y);
    });
    const float share = min(wave_sum(stages) / goal, 2e7f);
    chunk = max(MIN_CHUNK, static_cast<int>(ceilf(share)));
    bool fits = false;
    if (wave_sum(tiles) < goal) {
      for (int tries = 0; tries < 3 && !fits; ++tries) {
        float items = 0.0f;
        inv = __builtin_amdgcn_rcpf(static_cast<float>(chunk));
        each([&](int2 r) { items += static_cast<float>(r.x * chunks_of<MIN_CHUNK>(r.y, chunk, inv)); });
        items = wave_sum(items);
        fits = items <= goal;
        if (!fits) chunk = max(chunk + 1, static_cast<int>(chunk * (items / goal)));
      }
    }
    if (!fits) chunk = max(chunk, static_cast<int>(2.0f * share) + 1);
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    inv = __builtin_amdgcn_rcpf(static_cast<float>(chunk));
  }
  int items = 0, slots = 0;
  each([&](int2 r) {
    const int ns = chunks_of<MIN_CHUNK>(r.y, chunk, inv);
    items += r.x * ns;
    slots += ns > 1 ? r.x * ns : 0;
  });
  int at = wave_scan(items) - items, slot = wave_scan(slots) - slots;
  const uint64_t has = __ballot(i >= at && i < at + items);
  if (!has) return f;
  const int who = __builtin_ctzll(has);
  at = __builtin_amdgcn_readlane(at, who), slot = __builtin_amdgcn_readlane(slot, who);
  int row = 0;  // of 64 requests
  if (B > 64) {  // which of lane who's: a lane for each
    const int b = who + 64 * lane;
    mine = b < B ? reqs[b] : make_int2(0, 1);
    const int ns = chunks_of<MIN_CHUNK>(mine.y, chunk, inv);
    items = mine.x * ns, slots = ns > 1 ? items : 0;
    const int to = at + wave_scan(items), slot_to = slot + wave_scan(slots);
    row = __builtin_ctzll(__ballot(i < to));
    at = __builtin_amdgcn_readlane(to - items, row);
    slot = __builtin_amdgcn_readlane(slot_to - slots, row);
  }
  const int which = B > 64 ? row : who;
  f.b = who + 64 * row;
  f.tiles = __builtin_amdgcn_readlane(mine.x, which);
  const int stages = __builtin_amdgcn_readlane(mine.y, which);
  f.ns = __builtin_amdgcn_readfirstlane(chunks_of<MIN_CHUNK>(stages, chunk, inv));
  f.chunk = (stages + f.ns - 1) / f.ns;  // of equal length
  f.slot = slot;
  f.item = i - at;
  if (B <= 64) {
    f.req = {__builtin_amdgcn_readlane(req.q0, who), __builtin_amdgcn_readlane(req.nq, who),
             __builtin_amdgcn_readlane(req.kv, who)};
  } else {
    f.req = request_of(a, f.b);
    __syncthreads();  // reqs is read
  }
  return f;
}

// Row tile i of packed prompts (for one key/value head), found as above.
// Causal: the requests' last tiles first, so the longest first, whichever
// request they are of; N(t) = sum of max(tiles - t, 0) tiles have an index of t
// or more, so tile i has the largest t of N(t) > i.  Not causal: in order.
struct Tile {
  int b, tile;  // b is -1 where there is no such tile
  Request req;
};
template <class Tiles>
__device__ __forceinline__ Tile find_tile(const AttnArgs &a, int *reqs, int i, Tiles tiles_of) {
  const int lane = threadIdx.x & 63, B = a.B;
  auto request = [&](int b) {
    const int c0 = min(max(a.cu[b], 0), a.T), c1 = min(max(a.cu[b + 1], 0), a.T);
    return Request{c0, max(c1 - c0, 0), max(c1 - c0, 0)};
  };
  Tile f = {-1, 0, {0, 0, 0}};
  if (B == 1) {
    f.req = request(0);
    f.tile = tiles_of(f.req) - 1 - i;
    f.b = f.tile < 0 ? -1 : 0;
    return f;
  }
  int mine = 0;  // tiles of the lane's first request
  if (B <= 64) {
    if (lane < B) {
      f.req = request(lane);
      mine = tiles_of(f.req);
    }
  } else {
    for (int b = threadIdx.x; b < B; b += blockDim.x) reqs[b] = tiles_of(request(b));
    __syncthreads();
    mine = reqs[lane];
  }
  auto over = [&](int t) {  // the lane's tiles with an index of t or more
    int n = max(mine - t, 0);
#pragma unroll 4
    for (int b = lane + 64; b < B; b += 64) n += max(reqs[b] - t, 0);
    return n;
  };
  int t = 0, has = over(0);  // the lane's candidates
  if (a.causal) {
    if (wave_sum(has) <= i) return f;
    int most = mine;
#pragma unroll 4
    for (int b = lane + 64; b < B; b += 64) most = max(most, reqs[b]);
    most = wave_sum<Max>(most);
    for (int bit = 1 << (31 - __builtin_clz(most)); bit; bit >>= 1)
      if (wave_sum(over(t + bit)) > i) t += bit;
    i -= wave_sum(over(t + 1));  // among the requests that have a tile t
    has = over(t) - over(t + 1);
  }
  const int at = wave_scan(has) - has;
  const uint64_t lanes = __ballot(i >= at && i < at + has);
  if (!lanes) return f;
  const int who = __builtin_ctzll(lanes);
  i -= __builtin_amdgcn_readlane(at, who);
  if (B <= 64) {
    f.b = who;
    f.req = {__builtin_amdgcn_readlane(f.req.q0, who), __builtin_amdgcn_readlane(f.req.nq, who),
             __builtin_amdgcn_readlane(f.req.kv, who)};
  } else {  // which of lane who's requests: a lane for each
    const int b = who + 64 * lane, tiles = b < B ? reqs[b] : 0;
    const int n = a.causal ? tiles > t : tiles, to = wave_scan(n);
    const int row = __builtin_ctzll(__ballot(i < to));
    f.b = who + 64 * row;
    i -= __builtin_amdgcn_readlane(to - n, row);
    f.req = request(f.b);
    __syncthreads();  // reqs is read
  }
  f.tile = a.causal ? t : i;
  return f;
}

hipError_t launch_attn_rows(const AttnArgs &a, int dtype, int D, int max_rows, int items,
                            hipStream_t s);
int attn_rows_max_goal(int max_rows);
hipError_t launch_attn_tile(const AttnArgs &a, int dtype, int D, bool paged, int items,
                            hipStream_t s);
int attn_tile_rows(int D);
int attn_tile_min_keys();  // of a split
int64_t attn_tile_slot_bytes(int D);

}  // namespace ifx
