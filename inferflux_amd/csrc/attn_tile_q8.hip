// attn_tile_q8.hip -- attention over the 8-bit paged cache of many query rows:
// chunks of new tokens, wide trees of drafts, mixed batches.
//
//   s_j = sk_j q . ck_j,  p_j = 2^(c s_j - m),  l = sum p_j,
//   o = sum (p_j sv_j) cv_j / l;  ck, cv: codes, sk, sv: scales
//
// Bound by the vector units beside the matrix cores.  Work is shared as in
// attn_tile: 128 rows of a key/value head a workgroup, 32 a wave, stages of 64
// keys in LDS, both products transposed.  A stage's codes are taken to fp16
// once for all four waves, on their way from registers, where they have waited
// for the stage before, to LDS.
#include "ifx_attn_q8.h"
#include "ifx_attn_tile.h"

namespace ifx {

namespace {

#define IFX_INLINE __attribute__((always_inline))

constexpr int kThreads = 64 * kTileWaves;
constexpr int TK = kTileKeys;
constexpr int kMinChunk = 8;  // stages of a chunk at least (attn_tile)

}  // namespace

template <int D>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void k_attn_tile_q8(const AttnArgs a) {
  constexpr int ND = D / 32, NS = D / 16;
  constexpr int kPieces = TK * D / 8;           // 16-byte pieces of fp16, of K and of V
  constexpr int kRaw = TK * D / 16;             // of codes
  constexpr int NL = (kRaw + kThreads - 1) / kThreads;
  extern __shared__ u32x4 lds[];                // [2 stages][K, V][kPieces], [2][K, V scales][64]
  float *scales = reinterpret_cast<float *>(lds + 4 * kPieces);
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.Hkv;

  const Split split = find_item<kMinChunk>(
      a, reinterpret_cast<int2 *>(lds), blockIdx.x / a.Hkv, [&](const Request &r) {
        int keys = r.kv;  // that a tile sees
        if (a.window > 0) keys = min<int64_t>(keys, static_cast<int64_t>(a.window) + kQueryRows + TK);
        return make_int2((r.nq * a.G + kQueryRows - 1) / kQueryRows, max(1, (keys + TK - 1) / TK));
      });
  if (split.chunk == 0) return;
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

  // ---- stages: memory to registers, and from there as fp16 to LDS
  const int sh = a.page_shift, P = 1 << sh;
  const int32_t *table = a.table + static_cast<int64_t>(b) * a.table_width;
  const int wmax = a.table_width - 1, last_page = static_cast<int>(a.num_pages) - 1;
  const uint32_t page_bytes = static_cast<uint32_t>(a.Hkv * D) << sh;
  const uint8_t *K = static_cast<const uint8_t *>(a.k) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint8_t *V = static_cast<const uint8_t *>(a.v) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint32_t *S = a.scales + (static_cast<int64_t>(kvh) << sh);
  // the page of key k0 + lane, as the table has it: read a stage ahead
  auto entry_of = [&](int k0) { return table[min((k0 + lane) >> sh, wmax)]; };
  u32x4 rk[NL], rv[NL];
  uint32_t rs = 0;
  auto load = [&](int k0, int entry) IFX_INLINE {
    const int page = min(max(entry, 0), last_page);
    const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_bytes;
    const uint8_t *kp = K + at + ((k0 + lane) & (P - 1)) * 16;
    if (wave == 0)
      rs = S[((static_cast<int64_t>(page) * a.Hkv) << sh) + ((k0 + lane) & (P - 1))];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int p0 = (i * kTileWaves + wave) * 64, p = p0 + lane;  // 64 pieces
      if (kRaw % kThreads && p0 >= kRaw) break;
      rk[i] = ldg<u32x4>(kp + ((p0 >> 6) << sh) * 16);
      const int g = p / D, dim = p - g * D;
      const uint32_t pg = static_cast<uint32_t>(__shfl(page, 16 * g));
      rv[i] = ldg<u32x4>(V + static_cast<uint64_t>(pg) * page_bytes + ((k0 + 16 * g) & (P - 1)) * D + dim * 16);
    }
  };
  auto store = [&](int buf) IFX_INLINE {
    u32x4 *sk = lds + buf * 2 * kPieces, *sv = sk + kPieces;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int p0 = (i * kTileWaves + wave) * 64, p = p0 + lane;
      if (kRaw % kThreads && p0 >= kRaw) break;
      const int g = p / D, dim = p - g * D;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sk[(p0 >> 6) * 2 * TK + e * TK + lane] = codes_f16(rk[i], e);
        sv[(2 * g + e) * D + dim] = codes_f16(rv[i], e);
      }
    }
    if (wave == 0) {
      scales[buf * 2 * TK + lane] = k_scale(rs);
      scales[buf * 2 * TK + TK + lane] = v_scale(rs);
    }
  };

  const int kn = key_of_row(n);
  auto stage = [&](int k0, int buf, bool edge) IFX_INLINE {
    const u32x4 *sk = lds + buf * 2 * kPieces, *sv = sk + kPieces;
    const float *ks = scales + buf * 2 * TK, *vs = ks + TK;
    f32x16 s[2];
    float w[2][16];
    float mt = -__builtin_inff(), vt = 0.0f;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[sub][r] = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        s[sub] = F16::mfma32(sk[(2 * i + h) * TK + 32 * sub + kn], qf[i], s[sub]);
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int at = 32 * sub + 16 * (r >> 3) + 8 * h + (r & 7);
        const f32x4 k4 = ldg<f32x4>(ks + at), v4 = ldg<f32x4>(vs + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[sub][r + j] *= k4[j];
          w[sub][r + j] = v4[j];
          if (edge) {
            const bool sees = tree ? nodes.sees(k0 + at + j) : line.sees(k0 + at + j);
            s[sub][r + j] = sees ? s[sub][r + j] : -__builtin_inff();
            w[sub][r + j] = sees ? v4[j] : 0.0f;
          }
          mt = fmaxf(mt, s[sub][r + j]), vt = fmaxf(vt, w[sub][r + j]);
        }
      }
    }
    mt = halves_max(mt), vt = halves_max(vt);
    if (__any(level.above(mt, vt, c))) {
      const float less = level.raise(mt, vt, c);
      l *= less;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= less;
    }
    u32x4 pf[4];
    float sum = 0.0f;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r], c, -level.less));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r + 1], c, -level.less));
        sum += p0 + p1;
        pf[2 * sub + (r >> 3)][(r & 7) >> 1] = F16::pack(p0 * w[sub][r], p1 * w[sub][r + 1]);
      }
    l += sum;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] = F16::mfma32(sv[(2 * ks + h) * D + 32 * d + n], pf[ks], acc[d]);
  };

  if (zbeg < zend) {
    int entry = entry_of(zbeg);
    load(zbeg, entry);
    entry = entry_of(zbeg + TK);
    store(0);
    int buf = 0;
    for (int k0 = zbeg; k0 < zend; k0 += TK, buf ^= 1) {
      __syncthreads();  // this stage is in LDS, and no wave reads the other one
      const bool more = k0 + TK < zend;
      if (more) {
        load(k0 + TK, entry);
        entry = entry_of(k0 + 2 * TK);
      }
      if (!idle) {
        if (k0 < full_a || k0 >= full_z)
          stage(k0, buf, true);
        else
          stage(k0, buf, false);
      }
      if (more) store(buf ^ 1);
    }
  }

  tile_finish<D, true>(a, split, acc, level.of_sums(), l, 1.0f, tile, z, ns, kvh, R, [&](int t) {
    return tree ? Sight<true>{0, 0, ctx, node_bits(a, q0 + t, nq)}.nothing() : ctx + t < 0;
  });
}

namespace {
template <int D>
hipError_t launch_tile(const AttnArgs &a, int items, hipStream_t s) {
  constexpr int stages = 2 * 2 * TK * D * 2 + 2 * 2 * TK * 4, requests = IFX_ATTN_MAX_BATCH * 8;
  constexpr int bytes = stages > requests ? stages : requests;
  if constexpr (bytes > 65536 - 256) {
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const hipError_t e = allow_lds(reinterpret_cast<const void *>(&k_attn_tile_q8<D>), bytes, done);
      if (e != hipSuccess) return e;
    }
  }
  IFX_LAUNCH(k_attn_tile_q8, (D), dim3(a.Hkv * items), dim3(kThreads), bytes, s, a);
  return last_error();
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
