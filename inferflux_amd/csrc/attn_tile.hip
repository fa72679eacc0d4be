// attn_tile.hip -- attention of many query rows: chunks of new tokens over the
// paged cache, and whole prompts packed one after the other.
//
//   s_j = c q . k_j (c = scale log2 e), p_j = 2^(s_j - m), l = sum p_j,
//   o = sum p_j v_j / l, in one pass over the keys with the running m and l
//
// Bound by the MFMA rate and the exponentials beside it.  The rows of a
// key/value head are its group's query heads for every new token, so a
// workgroup's 128 rows read K and V once for all G heads.  Each wave keeps 32
// rows: Q as operand registers, O^T as accumulators; K and V pass through LDS
// in stages of 64 keys, double buffered, the next stage's loads in flight
// during the products.  Both products are taken transposed (S^T = K Q^T,
// O^T = V^T P^T): a lane then holds one row's scores, its maximum and sum need
// no more than one exchange between lane halves, and the probabilities are the
// next product's operand as they stand (key_of_row).
#include "ifx_attn.h"

namespace ifx {

namespace {

constexpr int kNW = 4;             // waves of a workgroup
constexpr int kRows = 32 * kNW;    // its query rows
constexpr int TK = kTileKeys;

// LDS places, in 16-byte pieces of 8 values.
//
// A paged stage is a copy of the cache's order: K [D / 8][64 keys], V
// [8 key groups][D].  Lanes read neighbouring pieces.
//
// A stage of packed rows keeps rows: K and V [64 keys][D / 8 pieces], with the
// pieces of a row exchanged by an XOR of the row number, chosen so that the 16
// lanes that a read serves at a time reach 16 different piece columns (256
// bytes: all banks).  K's lanes differ in the row, V's transposing reads take
// four rows of four neighbouring pieces.
template <int D>
__device__ __forceinline__ int swap_k(int m) {  // m: the A-operand row of the key
  return D == 64 ? (m >> 1) & 7 : D == 96 ? (m >> 2) & 3 : m & 15;
}
template <int D>
__device__ __forceinline__ int swap_v(int key) {
  return D == 64 ? (key & 2) << 1 : D == 96 ? 0 : (key & 3) << 2;
}

}  // namespace

template <int DT, int D, bool PAGED>
__global__ __launch_bounds__(64 * kNW, D == 256 ? 1 : 2) void k_attn_tile(const AttnArgs a) {
  using T = Elem<DT>;
  constexpr int ND = D / 32, NS = D / 16, NP = D / 8;
  constexpr int kPieces = TK * NP;              // of K, and of V, a stage
  constexpr int NL = kPieces / (64 * kNW);      // pieces a thread loads, each
  extern __shared__ u32x4 lds[];                // [2 stages][K, V][kPieces]
  __shared__ int found[3];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.Hkv, z = blockIdx.y;

  // Which request's rows: request b owns the row tiles from
  // floor(cu[b] G / kRows) + b on, at least as many as it needs, so that no
  // tile list has to be built.  Late tiles (long key ranges) come first.
  const int tile = (gridDim.x - 1 - blockIdx.x) / a.Hkv;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  for (int b = tid; b < a.B; b += 64 * kNW) {
    const int c0 = min(max(a.cu[b], 0), a.T), c1 = min(max(a.cu[b + 1], 0), a.T);
    const int t0 = c0 * a.G / kRows + b, t1 = c1 * a.G / kRows + b + 1;
    if (t0 <= tile && tile < t1 && (tile - t0) * kRows < (c1 - c0) * a.G) {
      found[0] = b;
      found[1] = c0;
      found[2] = c1;
    }
  }
  __syncthreads();
  const int b = __builtin_amdgcn_readfirstlane(found[0]);
  if (b < 0) return;
  const int q0 = __builtin_amdgcn_readfirstlane(found[1]);
  const int nq = __builtin_amdgcn_readfirstlane(found[2]) - q0;
  const int R = nq * a.G;
  const int row0 = (tile - (q0 * a.G / kRows + b)) * kRows;  // the workgroup's first
  const int kv = PAGED ? min(max(a.kv_len[b], 0), a.table_width << a.page_shift) : nq;
  const int ctx = kv - nq;  // position of the request's first row

  // keys that any row of the workgroup sees
  const int tok_a = row0 / a.G, tok_z = (min(row0 + kRows, R) - 1) / a.G;
  const int kend = a.causal ? ctx + tok_z + 1 : kv;
  const int kbeg = a.window > 0 ? max(0, ctx + tok_a - a.window + 1) & ~(TK - 1) : 0;
  const int chunk = split_chunk(a, kend - kbeg, TK);
  const int ns = kend > kbeg ? (kend - kbeg + chunk - 1) / chunk : 1;
  if (z >= ns) return;
  const int zbeg = kbeg + z * chunk, zend = min(zbeg + chunk, kend);

  // this lane's row sees [lo, hi]; rows behind the last repeat it
  const int row = min(row0 + 32 * wave + n, R - 1), tok = row / a.G;
  const int head = kvh * a.G + row - tok * a.G;
  const int hi = a.causal ? ctx + tok : kv - 1;
  const int lo = a.window > 0 ? max(0, ctx + tok - a.window + 1) : 0;
  // over the wave's rows: all see [lo_z, hi_a], some [lo_a, hi_z]
  const int hi_a = __builtin_amdgcn_readlane(hi, 0), hi_z = __builtin_amdgcn_readlane(hi, 31);
  const int lo_a = __builtin_amdgcn_readlane(lo, 0), lo_z = __builtin_amdgcn_readlane(lo, 31);

  u32x4 qf[NS];
  {
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + (q0 + tok) * a.q_stride +
                        static_cast<int64_t>(head) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = ldg<u32x4>(q + 16 * s);
  }
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
  float m = -__builtin_inff(), l = 0.0f;

  // ---- stages: loads to registers, then to LDS
  u32x4 kreg[NL], vreg[NL];
  const int sh = a.page_shift, P = 1 << sh;
  const int32_t *table = PAGED ? a.table + static_cast<int64_t>(b) * a.table_width : nullptr;
  const int wmax = a.table_width - 1, last_page = static_cast<int>(a.num_pages) - 1;
  const int64_t page_elems = (static_cast<int64_t>(a.Hkv) * D) << sh;
  const uint16_t *K = static_cast<const uint16_t *>(a.k) +
                      (PAGED ? (static_cast<int64_t>(kvh) * D) << sh
                             : q0 * a.k_stride + static_cast<int64_t>(kvh) * D);
  const uint16_t *V = static_cast<const uint16_t *>(a.v) +
                      (PAGED ? (static_cast<int64_t>(kvh) * D) << sh
                             : q0 * a.v_stride + static_cast<int64_t>(kvh) * D);
  auto page_of = [&](int k0) {  // of key k0 + lane
    return min(max(table[min((k0 + lane) >> sh, wmax)], 0), last_page);
  };
  auto load = [&](int k0, int page) {
    if constexpr (PAGED) {
      const uint16_t *kp = K + page * page_elems + ((k0 + lane) & (P - 1)) * 8;
#pragma unroll
      for (int i = 0; i < NL; ++i)  // piece (NP / NL ... ): 64 keys of one dim group
        kreg[i] = ldg<u32x4>(kp + (static_cast<int64_t>((i * kNW + wave) * 8) << sh));
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int p = i * 64 * kNW + tid, g = p / D, dim = p - g * D;
        const int64_t e = __shfl(page, 8 * g) * page_elems;
        vreg[i] = ldg<u32x4>(V + e + ((k0 + 8 * g) & (P - 1)) * D + dim * 8);
      }
      if (k0 + TK > kv) {  // slots behind the last token: no value may come from them
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int key = k0 + 8 * ((i * 64 * kNW + tid) / D);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            vreg[i][j] &= (key + 2 * j < kv ? 0xFFFFu : 0u) | (key + 2 * j + 1 < kv ? 0xFFFF0000u : 0u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int p = i * 64 * kNW + tid, key = p / NP, c = p - key * NP;
        const int64_t r = min(k0 + key, kv - 1);
        kreg[i] = ldg<u32x4>(K + r * a.k_stride + c * 8);
        vreg[i] = ldg<u32x4>(V + r * a.v_stride + c * 8);
      }
    }
  };
  auto store = [&](int buf) {
    u32x4 *sk = lds + buf * 2 * kPieces, *sv = sk + kPieces;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int p = i * 64 * kNW + tid;
      if constexpr (PAGED) {
        sk[p] = kreg[i];
        sv[p] = vreg[i];
      } else {
        const int key = p / NP, c = p - key * NP;
        sk[key * NP + (c ^ swap_k<D>(key_of_row(key & 31)))] = kreg[i];
        sv[key * NP + (c ^ swap_v<D>(key))] = vreg[i];
      }
    }
  };

  // ---- operands from LDS
  const int kn = key_of_row(n);
  auto k_at = [&](const u32x4 *sk, int sub, int s) {
    const int key = 32 * sub + kn, c = 2 * s + h;
    return PAGED ? sk[c * TK + key] : sk[key * NP + (c ^ swap_k<D>(n))];
  };
  auto v_at = [&](const u32x4 *sv, int ks, int d) -> u32x4 {
    if constexpr (PAGED) {
      return sv[(2 * ks + h) * D + 32 * d + n];
    } else {
      // each group of 16 lanes reads four rows of 16 dims and gets, transposed,
      // four keys of one dim a lane
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 *lds4;
      const int i = lane & 15, dim = 32 * d + (lane & 16) + 4 * (i & 3);
      u32x4 r;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int key = 16 * ks + 8 * h + 4 * w + (i >> 2);
        const u32x4 *piece = sv + key * NP + ((dim >> 3) ^ swap_v<D>(key));
        const u32x2 t = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (lds4)(reinterpret_cast<const char *>(piece) + 8 * (i & 1))));
        r[2 * w] = t.x;
        r[2 * w + 1] = t.y;
      }
      return r;
    }
  };
  auto v_one = [&](const u32x4 *sv, int key, int dim) {  // one value, for the rare path
    const uint16_t *e = reinterpret_cast<const uint16_t *>(
        PAGED ? sv + (key >> 3) * D + dim : sv + key * NP + ((dim >> 3) ^ swap_v<D>(key)));
    return T::value(e[PAGED ? key & 7 : dim & 7]);
  };

  auto step = [&](int k0, const u32x4 *sk, const u32x4 *sv, auto edge_c) {
    constexpr bool EDGE = decltype(edge_c)::value;
    f32x16 s[2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[sub][r] = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i) s[sub] = T::mfma32(k_at(sk, sub, i), qf[i], s[sub]);
      if constexpr (EDGE) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + 32 * sub + 16 * (r >> 3) + 8 * h + (r & 7);
          s[sub][r] = key >= lo && key <= hi ? s[sub][r] : -__builtin_inff();
        }
      }
    }
    float mt = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = fmaxf(fmaxf(mt, s[0][r]), s[1][r]);
    mt = halves_max(mt);
    if (__any((mt - m) * a.c > kLag)) {
      const float mn = fmaxf(m, mt);
      const float w = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * a.c);
      l *= w;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= w;
      m = mn;
    }
    const float mc = m == -__builtin_inff() ? 0.0f : m * a.c - T::kShift;
    u32x4 pf[4];
    float sum = 0.0f;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r], a.c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r + 1], a.c, -mc));
        sum += p0 + p1;
        pf[2 * sub + (r >> 3)][(r & 7) >> 1] = T::pack(p0, p1);
      }
    l += sum;

    if constexpr (EDGE) {
      // A masked key's probability is 0, but 0 times an infinity or NaN is not:
      // a product of V with zeros shows whether the stage holds one.  Then the
      // stage is added key by key, so that a row takes only what it sees.
      f32x16 probe;
#pragma unroll
      for (int r = 0; r < 16; ++r) probe[r] = 0.0f;
      const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) probe = T::mfma32(v_at(sv, ks, d), zero, probe);
      float any = probe[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) any += probe[r];
      if (__any(any != 0.0f)) {
#pragma unroll 1
        for (int i = 0; i < TK; ++i) {
          const int key = k0 + i, w = (i & 7) >> 1;
          const u32x4 pk = i < 16 ? pf[0] : i < 32 ? pf[1] : i < 48 ? pf[2] : pf[3];
          const uint32_t pd = w == 0 ? pk[0] : w == 1 ? pk[1] : w == 2 ? pk[2] : pk[3];
          const uint32_t mine = (pd >> (16 * (i & 1))) & 0xFFFFu;
          const float p = T::value(static_cast<uint32_t>(
              __shfl(static_cast<int>(mine), n + 32 * ((i >> 3) & 1))));
          const bool seen = key >= lo && key <= hi;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float v = v_one(sv, i, 32 * d + 8 * (r >> 2) + 4 * h + (r & 3));
              acc[d][r] = seen ? __builtin_fmaf(p, v, acc[d][r]) : acc[d][r];
            }
        }
        return;
      }
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] = T::mfma32(v_at(sv, ks, d), pf[ks], acc[d]);
  };

  if (zbeg < zend) {
    int page = 0;
    if constexpr (PAGED) page = page_of(zbeg);
    load(zbeg, page);
    if constexpr (PAGED) page = page_of(zbeg + TK);
    store(0);
    int buf = 0;
    for (int k0 = zbeg; k0 < zend; k0 += TK, buf ^= 1) {
      __syncthreads();  // this stage is in LDS, and no wave reads the other one
      const bool more = k0 + TK < zend;
      if (more) {
        load(k0 + TK, page);
        if constexpr (PAGED) page = page_of(k0 + 2 * TK);
      }
      const u32x4 *sk = lds + buf * 2 * kPieces, *sv = sk + kPieces;
      if (k0 <= hi_z && k0 + TK > lo_a) {
        if (k0 >= lo_z && k0 + TK - 1 <= hi_a)
          step(k0, sk, sv, std::false_type{});
        else
          step(k0, sk, sv, std::true_type{});
      }
      if (more) store(buf ^ 1);
    }
  }

  l = halves_sum(l);
  const bool none = hi < lo;  // the row sees no key
  auto write = [&](float inv) {
    if (row0 + 32 * wave + n >= R) return;
    char *o = static_cast<char *>(a.out) +
              ((q0 + tok) * a.out_stride + static_cast<int64_t>(head) * D) * dtype_bytes(a.out_dtype);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = none ? 0.0f : acc[d][4 * g + r] * inv;
        store4(o, a.out_dtype, 32 * d + 8 * g + 4 * h, v);
      }
  };
  if (ns == 1) return write(1.0f / l);

  // split: this chunk's sums to its slot, every lane in its own places; the
  // last workgroup of the tile adds the chunks in their order, lane by lane
  const rsrc_t part = make_rsrc(a.part, a.part_bytes);
  constexpr uint32_t kWaveBytes = 32 * D * 4 + 64 * 4 * 2, kSlotBytes = kNW * kWaveBytes;
  const uint32_t unit = static_cast<uint32_t>(tile) * a.Hkv + kvh;
  const uint32_t mine = unit * a.splits * kSlotBytes + wave * kWaveBytes + lane * 16;
  const uint32_t mine_ml = unit * a.splits * kSlotBytes + wave * kWaveBytes + 32 * D * 4 + lane * 8;
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
  uint32_t *cnt = a.cnt + unit;
  if (!split_arrive_last(cnt, ns)) return;
  float top = -__builtin_inff(), total = 0.0f;
  for (int y = 0; y < ns; ++y) {
    const float2 ml = __builtin_bit_cast(
        float2, __builtin_amdgcn_raw_buffer_load_b64(part, mine_ml + y * kSlotBytes, 0, kAuxDevice));
    const float mn = fmaxf(top, ml.x);
    total = total * weight(top, mn, a.c) + ml.y * weight(ml.x, mn, a.c);
    top = mn;
  }
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
  for (int y = 0; y < ns; ++y) {
    const float2 ml = __builtin_bit_cast(
        float2, __builtin_amdgcn_raw_buffer_load_b64(part, mine_ml + y * kSlotBytes, 0, kAuxDevice));
    const float w = weight(ml.x, top, a.c);
    const uint32_t at = mine + y * kSlotBytes;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 v = ld_dev4(part, at + (4 * d + g) * 1024);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[d][4 * g + r] += v[r] * w;
      }
  }
  write(1.0f / total);
  split_reset(cnt);
}

namespace {
template <int DT, int D, bool PAGED>
hipError_t launch_tile(const AttnArgs &a, int tiles, hipStream_t s) {
  constexpr int bytes = 2 * 2 * TK * D * 2;
  if constexpr (bytes > 65536 - 256) {
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const hipError_t e =
          allow_lds(reinterpret_cast<const void *>(&k_attn_tile<DT, D, PAGED>), bytes, done);
      if (e != hipSuccess) return e;
    }
  }
  IFX_LAUNCH(k_attn_tile, (DT, D, PAGED), dim3(a.Hkv * tiles, a.splits), dim3(64 * kNW), bytes, s, a);
  return last_error();
}
template <int DT>
hipError_t launch_tile(const AttnArgs &a, int D, bool paged, int tiles, hipStream_t s) {
  switch (D) {
    case 64: return paged ? launch_tile<DT, 64, true>(a, tiles, s) : launch_tile<DT, 64, false>(a, tiles, s);
    case 96: return paged ? launch_tile<DT, 96, true>(a, tiles, s) : launch_tile<DT, 96, false>(a, tiles, s);
    case 128: return paged ? launch_tile<DT, 128, true>(a, tiles, s) : launch_tile<DT, 128, false>(a, tiles, s);
    default: return paged ? launch_tile<DT, 256, true>(a, tiles, s) : launch_tile<DT, 256, false>(a, tiles, s);
  }
}
}  // namespace

int attn_tile_rows(int) { return kRows; }
int64_t attn_tile_slot_bytes(int D) { return kNW * (32 * D * 4 + 64 * 4 * 2); }

hipError_t launch_attn_tile(const AttnArgs &a, int dtype, int D, bool paged, int tiles,
                            hipStream_t s) {
  return dtype == IFX_ATTN_F16 ? launch_tile<IFX_ATTN_F16>(a, D, paged, tiles, s)
                               : launch_tile<IFX_ATTN_BF16>(a, D, paged, tiles, s);
}

}  // namespace ifx
