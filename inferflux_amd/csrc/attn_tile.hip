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

// LDS places, in 16-byte pieces of 8 values.  Copies go from memory to LDS
// past the registers.
//
// A paged stage is a copy of the cache's order: K [D / 8][64 keys], V
// [8 key groups][D].  Lanes read neighbouring pieces.
//
// A stage of packed rows keeps rows: K and V [64 keys][D / 8 pieces], with the
// pieces of a row exchanged by an XOR of the row number, chosen so that the 16
// lanes that a read serves at a time reach 16 different piece columns (256
// bytes: all banks).  K's lanes differ in the row, V's transposing reads take
// four rows of four neighbouring pieces.
// 16 bytes a lane from memory to 64 consecutive places in LDS.
__device__ __forceinline__ void to_lds(const void *from, u32x4 *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

__device__ __forceinline__ void to_lds(rsrc_t from, int voff, int soff, u32x4 *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 16,
                                           voff, soff, 0, 0);
}

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
  // stages [full_a, full_z) all of its rows see whole
  const int full_a = a.window > 0 ? (max(0, ctx + tok_z - a.window + 1) + TK - 1) & ~(TK - 1) : 0;
  const int full_z = max(0, a.causal ? ctx + tok_a + 1 : kv) & ~(TK - 1);
  int ns = 1, zbeg = kbeg, zend = kend;  // prompts are not split
  if constexpr (PAGED) {
    const int chunk = split_chunk(a, kend - kbeg, TK);
    if (kend > kbeg) ns = (kend - kbeg + chunk - 1) / chunk;
    if (z >= ns) return;
    zbeg = kbeg + z * chunk, zend = min(zbeg + chunk, kend);
  }

  // this lane's row sees [lo, hi]; rows behind the last repeat it
  const int row = min(row0 + 32 * wave + n, R - 1), tok = row / a.G;
  const int head = kvh * a.G + row - tok * a.G;
  const int hi = a.causal ? ctx + tok : kv - 1;
  const int lo = a.window > 0 ? max(0, ctx + tok - a.window + 1) : 0;
  const int hi_z = __builtin_amdgcn_readlane(hi, 31);  // some of the wave's rows see [lo_a, hi_z]
  const int lo_a = __builtin_amdgcn_readlane(lo, 0);

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

  // ---- stages: memory to LDS, 1 KB (64 pieces) an instruction
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
  // packed rows: where the piece that this lane loads first lies in a stage.
  // Its next ones lie whole groups of rows further, 16 or 32, with the same
  // exchange of pieces (kSame)
  constexpr bool kSame = D == 64 || D == 128;
  const int k_row = static_cast<int>(a.k_stride) * 2, v_row = static_cast<int>(a.v_stride) * 2;
  int k_off = 0, v_off = 0;
  if constexpr (!PAGED && kSame) {
    const int p = wave * 64 + lane, key = p / NP, c = p - key * NP;
    k_off = key * k_row + (c ^ swap_k<D>(key_of_row(key))) * 16;
    v_off = key * v_row + (c ^ swap_v<D>(key)) * 16;
  }
  // of key k0 + lane, as the table has it: it is read a stage ahead and looked
  // at only when that stage's loads are issued
  auto entry_of = [&](int k0) { return table[min((k0 + lane) >> sh, wmax)]; };
  auto load = [&](int k0, int entry, int buf) {
    const int page = min(max(entry, 0), last_page);
    u32x4 *sk = lds + buf * 2 * kPieces, *sv = sk + kPieces;
    if constexpr (PAGED) {
      const uint16_t *kp = K + page * page_elems + ((k0 + lane) & (P - 1)) * 8;
#pragma unroll
      for (int i = 0; i < NL; ++i) {  // the 64 keys' pieces of one dim group
        const int c = i * kNW + wave;
        to_lds(kp + (static_cast<int64_t>(c * 8) << sh), sk + c * TK);
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int p0 = (i * kNW + wave) * 64;
        if constexpr (D % 64 == 0) {  // 64 dims of one key group
          const int g = p0 / D;
          const int64_t e = __builtin_amdgcn_readlane(page, 8 * g) * page_elems;
          const uint16_t *vp = V + e + ((k0 + 8 * g) & (P - 1)) * D + (p0 - g * D) * 8;
          to_lds(vp + lane * 8, sv + p0);
        } else {
          const int p = p0 + lane, g = p / D, dim = p - g * D;
          const int64_t e = __shfl(page, 8 * g) * page_elems;
          to_lds(V + e + ((k0 + 8 * g) & (P - 1)) * D + dim * 8, sv + p0);
        }
      }
    } else {
      // the stage's rows; those behind the request's last read as 0
      const int rows = min(kv - k0, TK);
      const rsrc_t rk = make_rsrc(K + k0 * a.k_stride, rows * k_row);
      const rsrc_t rv = make_rsrc(V + k0 * a.v_stride, rows * v_row);
#pragma unroll
      for (int i = 0; i < NL; ++i) {  // 64 places in order, each with the piece that belongs there
        const int p0 = (i * kNW + wave) * 64;
        if constexpr (kSame) {
          to_lds(rk, k_off, i * (kNW * 64 / NP) * k_row, sk + p0);
          to_lds(rv, v_off, i * (kNW * 64 / NP) * v_row, sv + p0);
        } else {
          const int p = p0 + lane, key = p / NP, c = p - key * NP;
          to_lds(rk, key * k_row + (c ^ swap_k<D>(key_of_row(key & 31))) * 16, 0, sk + p0);
          to_lds(rv, key * v_row + (c ^ swap_v<D>(key)) * 16, 0, sv + p0);
        }
      }
    }
  };

  // ---- operands from LDS
  // Byte offsets of this lane's pieces; what changes with the step, dim tile or
  // key group is an immediate, or XORed in where pieces are exchanged.
  const int kn = key_of_row(n), ti = lane & 15;
  const int k_lane = PAGED ? (h * TK + kn) * 16 : kn * NP * 16;
  const int k_swap = PAGED ? 0 : (h ^ swap_k<D>(n)) * 16;
  // packed rows: V is read transposing: each group of 16 lanes reads four rows
  // of 16 dims and gets four keys of one dim a lane
  const int v_lane = PAGED ? (h * D + n) * 16
                           : (8 * h + (ti >> 2)) * NP * 16 + ((lane & 16) >> 3) * 16 + (ti & 3) * 8;
  const int v_swap = PAGED ? 0 : swap_v<D>(ti >> 2) * 16;
  auto k_at = [&](const char *sk, int sub, int s) {
    const char *p = PAGED ? sk + (k_lane + (2 * s * TK + 32 * sub) * 16)
                          : sk + ((k_swap ^ (32 * s)) + k_lane) + 32 * sub * NP * 16;
    return *reinterpret_cast<const u32x4 *>(p);
  };
  auto v_at = [&](const char *sv, int ks, int d) -> u32x4 {
    if constexpr (PAGED) {
      return *reinterpret_cast<const u32x4 *>(sv + (v_lane + (2 * ks * D + 32 * d) * 16));
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 *lds4;
      const char *p = sv + ((v_swap ^ (64 * d)) + v_lane) + 16 * ks * NP * 16;
      const u32x2 t = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p));
      const u32x2 u = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * NP * 16)));
      return u32x4{t.x, t.y, u.x, u.y};
    }
  };
  // the same without what lies behind the last token: a page's unwritten slots
  auto v_in = [&](int k0, const char *sv, int ks, int d) -> u32x4 {
    u32x4 r = v_at(sv, ks, d);
    if constexpr (PAGED) {
      const int key = k0 + 16 * ks + 8 * h;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[j] &= (key + 2 * j < kv ? 0xFFFFu : 0u) | (key + 2 * j + 1 < kv ? 0xFFFF0000u : 0u);
    }
    return r;
  };
  auto v_one = [&](const char *sv, int key, int dim) {  // one value, for the rare path
    const int piece = PAGED ? (key >> 3) * D + dim : key * NP + ((dim >> 3) ^ swap_v<D>(key));
    return T::value(reinterpret_cast<const uint16_t *>(sv + piece * 16)[PAGED ? key & 7 : dim & 7]);
  };

  // One stage. The matrix cores get the fragments of K, then of V, in one
  // sequence (frag): fragment i + kAhead is on its way from LDS while i is used.
  auto raise = [&](float mt) {  // the running maximum, where it is far enough behind
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
    return m == -__builtin_inff() ? 0.0f : m * a.c - T::kShift;
  };
  auto step = [&](const char *sk, const char *sv) {
    constexpr int kAhead = 4;
    f32x16 s[2];
    u32x4 f[4 * NS];  // K of both halves, V: at most kAhead + 1 are alive
    auto frag = [&](int i) {
      if (i < 2 * NS)
        f[i] = k_at(sk, i / NS, i % NS);
      else if (i < 4 * NS)
        f[i] = v_at(sv, (i - 2 * NS) / ND, (i - 2 * NS) % ND);
    };
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.0f;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) frag(i);
    __builtin_amdgcn_sched_barrier(0);
    float mt = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) {
      frag(i + kAhead);
      s[i / NS] = T::mfma32(f[i], qf[i % NS], s[i / NS]);
      // the first half's maximum beside the second half's products
      constexpr int kFrom = NS + NS / 4, kSteps = 2 * NS - kFrom;
      if (i >= kFrom) {
#pragma unroll
        for (int r = (i - kFrom) * 8 / kSteps; r < (i - kFrom + 1) * 8 / kSteps; ++r)
          mt = fmaxf(fmaxf(mt, s[0][2 * r]), s[0][2 * r + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 16; r += 2) mt = fmaxf(fmaxf(mt, s[1][r]), s[1][r + 1]);
    const float mc = raise(mt);
    u32x4 pf[4];
    auto weigh = [&](int sub, int r) {  // keys 2r and 2r + 1 of a half
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][2 * r], a.c, -mc));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][2 * r + 1], a.c, -mc));
      l += p0 + p1;
      pf[2 * sub + (r >> 2)][r & 3] = T::pack(p0, p1);
    };
#pragma unroll
    for (int r = 0; r < 8; ++r) weigh(0, r);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) {
      frag(2 * NS + i + kAhead);
      acc[i % ND] = T::mfma32(f[2 * NS + i], pf[i / ND], acc[i % ND]);
      if (i < NS) {  // the second half's weights beside the first half's products
#pragma unroll
        for (int r = i * 8 / NS; r < (i + 1) * 8 / NS; ++r) weigh(1, r);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // One stage of which some rows see only a part.
  auto edge_step = [&](int k0, const char *sk, const char *sv) {
    f32x16 s[2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[sub][r] = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i) s[sub] = T::mfma32(k_at(sk, sub, i), qf[i], s[sub]);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = k0 + 32 * sub + 16 * (r >> 3) + 8 * h + (r & 7);
        s[sub][r] = key >= lo && key <= hi ? s[sub][r] : -__builtin_inff();
      }
    }
    float mt = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = fmaxf(fmaxf(mt, s[0][r]), s[1][r]);
    const float mc = raise(mt);
    u32x4 pf[4];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r], a.c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r + 1], a.c, -mc));
        l += p0 + p1;
        pf[2 * sub + (r >> 3)][(r & 7) >> 1] = T::pack(p0, p1);
      }

    __builtin_amdgcn_sched_barrier(0);

    // A masked key's probability is 0, but 0 times an infinity or NaN is not: a
    // product of V with zeros shows whether the stage holds one.  Then the
    // stage is added key by key, so that a row takes only what it sees.
    f32x16 probe;
#pragma unroll
    for (int r = 0; r < 16; ++r) probe[r] = 0.0f;
    const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < ND; ++d) probe = T::mfma32(v_in(k0, sv, ks, d), zero, probe);
    __builtin_amdgcn_sched_barrier(0);
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
            __builtin_amdgcn_sched_barrier(0);
          }
      }
      return;
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] = T::mfma32(v_in(k0, sv, ks, d), pf[ks], acc[d]);
  };

  if (zbeg < zend) {
    int entry = 0;
    if constexpr (PAGED) entry = entry_of(zbeg);
    load(zbeg, entry, 0);
    if constexpr (PAGED) entry = entry_of(zbeg + TK);
    int k0 = zbeg, buf = 0;
    auto stages = [&](int until, auto edge_c) {
      for (; k0 < until; k0 += TK, buf ^= 1) {
        wait_own_memory();
        __syncthreads();  // this stage is in LDS, and no wave reads the other one
        if (k0 + TK < zend) {
          load(k0 + TK, entry, buf ^ 1);
          if constexpr (PAGED) entry = entry_of(k0 + 2 * TK);
        }
        const char *sk = reinterpret_cast<const char *>(lds + buf * 2 * kPieces);
        const char *sv = sk + kPieces * 16;
        if constexpr (decltype(edge_c)::value) {
          if (k0 <= hi_z && k0 + TK > lo_a) edge_step(k0, sk, sv);
        } else {
          step(sk, sv);
        }
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
  if (!PAGED || ns == 1) return write(1.0f / l);

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
