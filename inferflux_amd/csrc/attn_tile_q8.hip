// attn_tile_q8.hip -- attention over the 8-bit paged cache of many query rows:
// chunks of new tokens, wide trees of drafts, mixed batches.
//
//   s_j = sk_j q . ck_j,  p_j = 2^(c s_j - m),  l = sum p_j,
//   o = sum (p_j sv_j) cv_j / l;  ck, cv: codes, sk, sv: scales
//
// Work is shared as in attn_tile: 128 rows of a key/value head a workgroup, 32 a
// wave, stages of 64 keys in LDS, both products transposed.  A stage's codes are
// copied to LDS past the registers while the stage before is multiplied; then each
// wave takes a quarter of them to fp16, in LDS too, for all four.
//
// Bound by the vector units and LDS beside the matrix cores: 375 vector
// instructions and 32 products of 32x32x16 for a wave's stage, LDS read and written
// for about as long.  512 tokens behind 7430, 40 / 8 heads of 128: 126 us, 640
// TFLOP/s (the 16-bit cache's: 94), and 146 where the same launches in a row have
// lowered the card's clock.  36 registers (one request) or 17 (several) of D = 128, 105
// of D = 256, are kept in scratch memory over the stages; none of them is used in one
// that its rows see whole.  Tried: codes in registers instead of LDS 133
// to 146, stages of 32 keys 145, three workgroups a CU of 168 registers 213 (they
// spill), codes taken to fp16 between the products 126; the same without any scales
// (which is no attention, but a bound) 119; two stages of codes on their way 129.
//
// Requests of up to 32 rows of a key/value head, single tokens next to chunks or
// trees, would leave three of the four waves idle: their chunks go through
// rows32_q8, where the waves share the keys.  24 trees of 1 to 38 nodes behind 110
// to 7302 tokens, 40 / 8 heads, with their plan: 58 us with it and 75 without; 32 of 2
// to 23 nodes behind 107 to 7471 71 and 73; 16 single tokens and 8 chunks of 17 to 182
// tokens 50 and 68, of 16 / 2 heads 36 and 38.  A request without new tokens is no
// work: as many idle ones of 20000 keys beside such batches change their times by
// less than 3 %.
#include "ifx_attn_rows_q8.h"
#include "ifx_attn_tile.h"

namespace ifx {

namespace {

#define IFX_INLINE __attribute__((always_inline))

constexpr int kThreads = 64 * kTileWaves;
constexpr int TK = kTileKeys;
constexpr int kMinChunk = 8;  // stages of a chunk at least (attn_tile)

// Waits for this wave's LDS accesses and then for the workgroup's other waves;
// copies from memory stay on their way.
__device__ __forceinline__ void group_barrier() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

constexpr int kScales = 2 * TK + 4;  // of a stage: K's, V's, the largest of V's

// Keys of few rows that count as a stage of a row tile, as they take about as long:
// with 128 / 160 / 192 / 224 / 256 the batches above take 59/59/60/58/63 us (24
// trees), 73/71/71/71/71 (32 trees) and 53/56/51/50/50 (40 / 8 heads' mixed step).
constexpr int kFewKeys = 224;

// LDS: fp16 K and V of a stage, its codes and scales; or the tiles of few rows and
// their waves' sums, of which a request's chunks' weights take the place.
template <int D, bool MIXED>
constexpr int tile_bytes() {
  constexpr int sums = kRowWaves * D * 4 * kRowsMax;
  constexpr int rows = rows32_bytes<D>() > sums ? rows32_bytes<D>() : sums;
  constexpr int stages = 2 * TK * D * 3 + 256 + kScales * 4;
  return MIXED && rows > stages ? rows : stages;
}
// Keys of a request that goes through rows32_q8: the weights of its chunks, of
// kMinChunk units at least, have their place.
template <int D, bool MIXED>
constexpr int few_most() {
  return MIXED ? tile_bytes<D, true>() / (kRowsMax * 8) * kMinChunk * kFewKeys : -1;
}

}  // namespace

// MIXED: of several requests, of which some may have few rows.
template <int D, bool MIXED = false>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void k_attn_tile_q8(const AttnArgs a) {
  constexpr int ND = D / 32, NS = D / 16;
  constexpr int kPieces = TK * D / 8;           // 16-byte pieces of fp16, of K and of V
  constexpr int kRaw = TK * D / 16;             // of codes
  constexpr int NL = (kRaw + kThreads - 1) / kThreads;
  extern __shared__ u32x4 lds[];                // fp16 [K, V][kPieces], codes and scales as copied, kScales
  u32x4 *raw = lds + 2 * kPieces;               // [K, V][kRaw], 64 dwords
  float *scales = reinterpret_cast<float *>(raw + 2 * kRaw + 16);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // kept, and not the thread's number
  const int n = lane & 31, h = lane >> 5;
  const int kvh = blockIdx.x % a.Hkv;

  const Split split = find_item<kMinChunk, 0>(
      a, reinterpret_cast<int2 *>(lds), blockIdx.x / a.Hkv, [&](const Request &r) {
        return tile_units_q8(a, r, kQueryRows, kFewKeys, few_most<D, MIXED>());
      });
  if (split.chunk == 0) return;
  if constexpr (MIXED) {
    if (few_rows(a, split.req, few_most<D, true>())) {
      __shared__ RowSums sums;
      RowsWork w;
      if (rows_work(a, split, kFewKeys, kRowsMax, w))
        rows32_q8<D>(a, w, reinterpret_cast<float *>(lds), sums, tile_slot_bytes<D>(), kvh);
      return;
    }
  }
  // the same in all lanes, and kept in scalar registers
  const int b = __builtin_amdgcn_readfirstlane(split.b);
  const int z = __builtin_amdgcn_readfirstlane(split.item / split.tiles);
  const int tile = __builtin_amdgcn_readfirstlane(split.tiles - 1 - split.item % split.tiles);
  const int q0 = __builtin_amdgcn_readfirstlane(split.req.q0);
  const int nq = __builtin_amdgcn_readfirstlane(split.req.nq);
  const int kv = __builtin_amdgcn_readfirstlane(split.req.kv), R = nq * a.G;
  const int row0 = tile * kQueryRows, ctx = kv - nq;
  const bool tree = a.masks != nullptr;

  // keys that any row of the workgroup sees
  const int tok_a = row0 / a.G, tok_z = (min(row0 + kQueryRows, R) - 1) / a.G;
  const int kend = tree ? kv : ctx + tok_z + 1;
  const int kbeg = a.window > 0 ? max(0, ctx + tok_a - a.window + 1) & ~(TK - 1) : 0;
  // stages [full_a, full_z) all of its rows see whole
  const int full_a = a.window > 0 ? (max(0, ctx + tok_z - a.window + 1) + TK - 1) & ~(TK - 1) : 0;
  const int full_z = max(0, tree ? ctx : ctx + tok_a + 1) & ~(TK - 1);
  const int chunk = __builtin_amdgcn_readfirstlane(split.chunk) * TK;
  const int ns = kend > kbeg ? (kend - kbeg + chunk - 1) / chunk : 1;
  if (z >= ns) return;
  const int zbeg = kbeg + z * chunk, zend = min(zbeg + chunk, kend);

  // this lane's row; rows behind the last repeat it
  const int row = min(row0 + 32 * wave + n, R - 1), tok = row / a.G;
  const int head = kvh * a.G + row - tok * a.G;
  const Sight<false> line = {a.window > 0 ? max(0, ctx + tok - a.window + 1) : 0, ctx + tok, ctx, 0};
  Sight<true> nodes = {0, 0, ctx, 0};
  if (tree) nodes.bits = node_bits(a, q0 + tok, nq);
  const bool idle = row0 + 32 * wave >= R;  // the wave has no rows, it only copies

  u32x4 qf[NS];
  {
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + (q0 + tok) * a.q_stride +
                        static_cast<int64_t>(head) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = ldg<u32x4>(q + 16 * s);
  }
  const float c = row_to_f16<32>(qf, a.q_dtype, a.c);
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
  Level level;
  float l = 0.0f;

  // ---- stages: codes from memory to LDS, and from there as fp16 to LDS
  const int sh = a.page_shift, P = 1 << sh;
  const int32_t *table = a.table + static_cast<int64_t>(b) * a.table_width;
  const int wmax = a.table_width - 1, last_page = static_cast<int>(a.num_pages) - 1;
  const uint32_t page_bytes = static_cast<uint32_t>(a.Hkv * D) << sh;
  const uint8_t *K = static_cast<const uint8_t *>(a.k) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint8_t *V = static_cast<const uint8_t *>(a.v) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint32_t *S = a.scales + (static_cast<int64_t>(kvh) << sh);
  // the page of key k0 + lane, as the table has it: read a stage ahead
  auto entry_of = [&](int k0) { return table[min((k0 + lane) >> sh, wmax)]; };
  // Copies a stage's codes to LDS past the registers, each lane's pieces to its
  // own places, and wave 0 the scales.
  auto issue = [&](int k0, int entry) IFX_INLINE {
    const int page = min(max(entry, 0), last_page);
    const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_bytes;
    const uint8_t *kp = K + at + ((k0 + lane) & (P - 1)) * 16;
    if (wave == 0)
      to_lds4(S + ((static_cast<int64_t>(page) * a.Hkv) << sh) + ((k0 + lane) & (P - 1)), raw + 2 * kRaw);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int p0 = (i * kTileWaves + wave) * 64, p = p0 + lane;  // 64 pieces
      if (kRaw % kThreads && p0 >= kRaw) break;
      to_lds16(kp + ((p0 >> 6) << sh) * 16, raw + p0);
      const int g = p / D, dim = p - g * D;
      const uint32_t pg = static_cast<uint32_t>(__shfl(page, 16 * g));
      to_lds16(V + static_cast<uint64_t>(pg) * page_bytes + ((k0 + 16 * g) & (P - 1)) * D + dim * 16,
               raw + kRaw + p0);
    }
  };
  // The codes that this wave copied as fp16.
  auto convert = [&]() IFX_INLINE {
    u32x4 *sk = lds, *sv = sk + kPieces;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int p0 = (i * kTileWaves + wave) * 64, p = p0 + lane;
      if (kRaw % kThreads && p0 >= kRaw) break;
      const int g = p / D, dim = p - g * D;
      const u32x4 rk = raw[p], rv = raw[kRaw + p];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sk[(p0 >> 6) * 2 * TK + e * TK + lane] = codes_f16(rk, e);
        sv[(2 * g + e) * D + dim] = codes_f16(rv, e);
      }
    }
    if (wave == 0) {
      const uint32_t rs = reinterpret_cast<const uint32_t *>(raw + 2 * kRaw)[lane];
      scales[lane] = k_scale(rs);
      scales[TK + lane] = v_scale(rs);
      float top = v_scale(rs);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
      if (lane == 0) scales[2 * TK] = top;
    }
  };

  // One stage.  The matrix cores get the fragments of K, then of V, in one
  // sequence: fragment i + kAhead is on its way from LDS while i is multiplied.
  // edge: some rows see only a part of it.
  const int kn = key_of_row(n);
  const f32x16 none_yet = {};
  auto stage = [&](int k0, auto edge_c) IFX_INLINE {
    constexpr bool edge = decltype(edge_c)::value;
    constexpr int kAhead = 3;
    const u32x4 *sk = lds + h * TK + kn, *sv = lds + kPieces + h * D + n;
    const float *ks = scales + 8 * h, *vs = ks + TK;
    u32x4 f[4 * NS];  // K of both halves, V: at most kAhead + 1 are alive
    auto frag = [&](int i) IFX_INLINE {
      if (i < 2 * NS)
        f[i] = sk[2 * (i % NS) * TK + 32 * (i / NS)];
      else if (i < 4 * NS)
        f[i] = sv[2 * ((i - 2 * NS) / ND) * D + 32 * ((i - 2 * NS) % ND)];
    };
    auto at = [](int sub, int r) { return 32 * sub + 16 * (r >> 3) + (r & 7); };  // key of register r, less 8 h
    f32x16 s[2];
    float mt[2] = {-__builtin_inff(), -__builtin_inff()};
    float vt = edge ? 0.0f : scales[2 * TK];
    // what the lane's row sees of the keys of its half of the wave: bit 32 sub + 16 (r / 8) + r % 8
    uint64_t sees = 0;
    if constexpr (edge) sees = (tree ? nodes.of_64(k0) : line.of_64(k0)) >> (8 * h);
    auto mask = [&](int key) IFX_INLINE {  // all bits where it sees it
      const uint32_t half = static_cast<uint32_t>(key < 32 ? sees : sees >> 32);
      return static_cast<uint32_t>(static_cast<int32_t>(half << (31 - (key & 31))) >> 31);
    };
    auto and_mask = [&](float v, uint32_t m) IFX_INLINE {
      return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & m);
    };
    // four scores of a half, scaled and masked
    auto scale4 = [&](int sub, int r) IFX_INLINE {
      const f32x4 k4 = *reinterpret_cast<const f32x4 *>(ks + at(sub, r));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = s[sub][r + j] * k4[j];
        if constexpr (edge) {
          const uint32_t m = mask(at(sub, r) + j);
          x = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & m) | (0xFF800000u & ~m));
          vt = fmaxf(vt, and_mask(vs[at(sub, r) + j], m));
        }
        s[sub][r + j] = x;
      }
      mt[0] = fmaxf(fmaxf(mt[0], s[sub][r]), s[sub][r + 1]);
      mt[1] = fmaxf(fmaxf(mt[1], s[sub][r + 2]), s[sub][r + 3]);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) frag(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) {
      frag(i + kAhead);
      s[i / NS] = F16::mfma32(f[i], qf[i % NS], i % NS ? s[i / NS] : none_yet);
      // the first half's scores beside the second half's products
      constexpr int kFrom = NS + NS / 4, kSteps = 2 * NS - kFrom;
      if (i >= kFrom) {
#pragma unroll
        for (int r = (i - kFrom) * 4 / kSteps; r < (i - kFrom + 1) * 4 / kSteps; ++r) scale4(0, 4 * r);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 16; r += 4) scale4(1, r);
    const float top = halves_max(fmaxf(mt[0], mt[1]));
    if constexpr (edge) vt = halves_max(vt);
    if (__any(level.above(top, vt, c))) {
      const float less = level.raise(top, vt, c);
      l *= less;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= less;
    }
    u32x4 pf[4];
    float sum[2] = {l, 0.0f};
    auto weigh4 = [&](int sub, int r) IFX_INLINE {
      f32x4 v4 = *reinterpret_cast<const f32x4 *>(vs + at(sub, r));
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r + j], c, -level.less));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r + j + 1], c, -level.less));
        sum[0] += p0;
        sum[1] += p1;
        if constexpr (edge) {
          v4[j] = and_mask(v4[j], mask(at(sub, r) + j));
          v4[j + 1] = and_mask(v4[j + 1], mask(at(sub, r) + j + 1));
        }
        pf[2 * sub + (r >> 3)][((r & 7) + j) >> 1] = F16::pack(p0 * v4[j], p1 * v4[j + 1]);
      }
    };
#pragma unroll
    for (int r = 0; r < 16; r += 4) weigh4(0, r);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) {
      frag(2 * NS + i + kAhead);
      acc[i % ND] = F16::mfma32(f[2 * NS + i], pf[i / ND], acc[i % ND]);
      if (i < NS) {  // the second half's weights beside the first half's products
#pragma unroll
        for (int r = i * 4 / NS; r < (i + 1) * 4 / NS; ++r) weigh4(1, 4 * r);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    l = sum[0] + sum[1];
  };

  if (zbeg < zend) {
    int entry = entry_of(zbeg);
    issue(zbeg, entry);
    entry = entry_of(zbeg + TK);
    int k0 = zbeg;
    auto stages = [&](int until, auto edge_c) IFX_INLINE {
      for (; k0 < until; k0 += TK) {
        wait_loads<0>();
        group_barrier();  // the stage before is multiplied
        convert();
        __builtin_amdgcn_sched_barrier(0);  // the codes' places are read
        if (k0 + TK < zend) {
          issue(k0 + TK, entry);
          entry = entry_of(k0 + 2 * TK);
        }
        group_barrier();  // this stage is in LDS
        if (!idle) stage(k0, edge_c);
      }
    };
    // stages that all rows of the workgroup see whole, between those that some
    // see in part: where windows begin, and at the causal end
    int until = a.window > 0 ? min(full_a, zend) : zbeg;
    while (true) {
      stages(until, std::true_type{});
      if (k0 >= zend) break;
      stages(min(full_z, zend), std::false_type{});
      until = zend;
    }
  }

  tile_finish<D, true>(a, split, acc, level.of_sums(), l, 1.0f, tile, z, ns, kvh, R, [&](int t) {
    return tree ? Sight<true>{0, 0, ctx, node_bits(a, q0 + t, nq)}.nothing() : ctx + t < 0;
  });
}

namespace {
template <int D, bool MIXED>
hipError_t launch_tile(const AttnArgs &a, int items, hipStream_t s) {
  constexpr int requests = MIXED ? IFX_ATTN_MAX_BATCH * 8 : 0;
  constexpr int bytes = tile_bytes<D, MIXED>() > requests ? tile_bytes<D, MIXED>() : requests;
  if constexpr (bytes > 65536 - 2048) {  // what a launch may ask for without more ado
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const hipError_t e = allow_lds(reinterpret_cast<const void *>(&k_attn_tile_q8<D, MIXED>), bytes, done);
      if (e != hipSuccess) return e;
    }
  }
  if constexpr (MIXED)
    IFX_LAUNCH(k_attn_tile_q8, (D, true), dim3(a.Hkv * items), dim3(kThreads), bytes, s, a);
  else
    IFX_LAUNCH(k_attn_tile_q8, (D), dim3(a.Hkv * items), dim3(kThreads), bytes, s, a);
  return last_error();
}
template <int D>
hipError_t launch_tile(const AttnArgs &a, int items, hipStream_t s) {
  return a.B > 1 ? launch_tile<D, true>(a, items, s) : launch_tile<D, false>(a, items, s);
}
}  // namespace

hipError_t launch_attn_tile_q8(const AttnArgs &a, int D, int items, hipStream_t s) {
  switch (D) {
    case 64: return launch_tile<64>(a, items, s);
    case 96: return launch_tile<96>(a, items, s);
    case 128: return launch_tile<128>(a, items, s);
    default: return launch_tile<256>(a, items, s);
  }
}

}  // namespace ifx
