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
//
// Measured at 40 query and 8 key/value heads of 128: a causal prompt of 8111
// tokens in 630 us, 1.07 PFLOP/s (a large 16-bit matrix product reaches 1.2 on
// the same card), and in up to 737 where the card has lowered its clock; there
// the matrix cores are busy for 56 % of the time and the vector units for 47 %.
// A chunk of 512 tokens over 7430 cached ones in 90 us.  What took longer, for
// that prompt, on the way: stages through registers 3207 us, as they
// spill; fragments read where they are needed 701, when kAhead of them on their
// way took 657; V transposed in registers 800; 64 rows a wave 2600, for the
// moves between the halves of the register file; 8 waves in two groups half a
// stage apart 671.
//
// Registers: 256 a wave, two workgroups a CU.  D = 64 does with 168, three a
// CU: 8111 tokens of 40 / 8 heads took 370 us, with two 387, with four 1330
// (spills).  D = 256 needs 512: 4111 tokens of 16 / 2 heads in 241 us (fp16) or
// 276 (bf16).
#include "ifx_attn.h"

namespace ifx {

namespace {

// Lambdas that are calls would keep what they capture in memory.
#define IFX_INLINE __attribute__((always_inline))

constexpr int kNW = 4;           // waves of a workgroup
constexpr int kRows = 32 * kNW;  // its query rows
constexpr int TK = kTileKeys;
// Stages of a chunk at least: beside them it takes 6 us for its first loads and
// its sums' exchange, as much as 5 stages.  A mixed batch (16 decode steps, 8
// chunks): 32 us with 4 or 6, 28 with 8, 30 with 12; 60 tokens over 3000: 23,
// 23, 25, 30.
constexpr int kMinChunk = 8;

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

// The same from a range of memory; places behind its end get 0.  The whole
// offset is the lanes': the range check does not count a scalar one.
__device__ __forceinline__ void to_lds(rsrc_t from, int off, u32x4 *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 16,
                                           off, 0, 0, 0);
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
__global__ __launch_bounds__(64 * kNW, D == 256 ? 1 : D == 64 ? 3 : 2) void k_attn_tile(const AttnArgs a) {
  using T = Elem<DT>;
  constexpr int ND = D / 32, NS = D / 16, NP = D / 8;
  constexpr int kPieces = TK * NP;              // of K, and of V, a stage
  constexpr int NL = kPieces / (64 * kNW);      // pieces a thread loads, each
  extern __shared__ u32x4 lds[];                // [2 stages][K, V][kPieces]
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.Hkv;

  int b, tile, z = 0;  // request, its row tile, its chunk of the keys
  Split split = {};
  if constexpr (PAGED) {
    split = find_item<kMinChunk>(
        a, reinterpret_cast<int2 *>(lds), blockIdx.x / a.Hkv, [&](const Request &r) {
          int keys = r.kv;  // that a tile sees
          if (a.window > 0) keys = min<int64_t>(keys, static_cast<int64_t>(a.window) + kRows + TK);
          return make_int2((r.nq * a.G + kRows - 1) / kRows, max(1, (keys + TK - 1) / TK));
        });
    if (split.chunk == 0) return;
    b = split.b, z = split.item / split.tiles;
    tile = split.tiles - 1 - (split.item - z * split.tiles);  // late tiles first
  } else {
    const Tile found = find_tile(a, reinterpret_cast<int *>(lds), blockIdx.x / a.Hkv,
                                 [&](const Request &r) { return (r.nq * a.G + kRows - 1) / kRows; });
    if (found.b < 0) return;
    b = found.b, tile = found.tile, split.req = found.req;
  }
  // the same in all lanes, and kept in scalar registers
  b = __builtin_amdgcn_readfirstlane(b), tile = __builtin_amdgcn_readfirstlane(tile);
  z = __builtin_amdgcn_readfirstlane(z);
  const int q0 = __builtin_amdgcn_readfirstlane(split.req.q0);
  const int nq = __builtin_amdgcn_readfirstlane(split.req.nq);
  const int kv = __builtin_amdgcn_readfirstlane(split.req.kv), R = nq * a.G;
  const int row0 = tile * kRows;  // the workgroup's first
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
    const int chunk = __builtin_amdgcn_readfirstlane(split.chunk) * TK;
    if (kend > kbeg) ns = (kend - kbeg + chunk - 1) / chunk;
    if (z >= ns) return;
    zbeg = kbeg + z * chunk, zend = min(zbeg + chunk, kend);
  }

  // this lane's row sees [lo, hi]; rows behind the last repeat it
  int row = min(row0 + 32 * wave + n, R - 1), tok = row / a.G;
  int head = kvh * a.G + row - tok * a.G;
  const int hi = a.causal ? ctx + tok : kv - 1;
  const int lo = a.window > 0 ? max(0, ctx + tok - a.window + 1) : 0;
  const int hi_z = __builtin_amdgcn_readlane(hi, 31);  // some of the wave's rows see [lo_a, hi_z]
  const int lo_a = __builtin_amdgcn_readlane(lo, 0);
  const bool idle = row0 + 32 * wave >= R;  // the wave has no rows, it only copies

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
  const uint32_t page_bytes = static_cast<uint32_t>(a.Hkv * D * 2) << sh;
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
  // the page of key k0 + lane, as the table has it: it is read a stage ahead and
  // looked at only when that stage's copies are issued
  auto entry_of = [&](int k0) { return table[min((k0 + lane) >> sh, wmax)]; };
  auto page_of = [&](int entry) { return min(max(entry, 0), last_page); };
  // One stage's copies: where they come from, and the i-th (of 2 NL) of this wave.
  struct Source {
    const char *kp;  // paged K: this lane's key
    int page, k0, buf;
    rsrc_t rk, rv;   // packed rows: those behind the request's last read as 0
  };
  auto source = [&](int k0, int entry, int buf) IFX_INLINE {
    Source f;
    f.k0 = k0, f.buf = buf;
    if constexpr (PAGED) {
      f.page = page_of(entry);
      f.kp = reinterpret_cast<const char *>(K) +
             static_cast<uint64_t>(static_cast<uint32_t>(f.page)) * page_bytes +
             ((k0 + lane) & (P - 1)) * 16;
    } else {
      const int rows = min(kv - k0, TK);
      f.rk = make_rsrc(K + k0 * a.k_stride, rows * k_row);
      f.rv = make_rsrc(V + k0 * a.v_stride, rows * v_row);
    }
    return f;
  };
  auto copy = [&](const Source &f, int j) IFX_INLINE {
    const int i = j >> 1, n0 = i * kNW + wave;  // 64 pieces
    u32x4 *sk = lds + f.buf * 2 * kPieces + n0 * 64, *sv = sk + kPieces;
    if constexpr (PAGED) {
      if ((j & 1) == 0) {  // K: the 64 keys' pieces of one dim group
        to_lds(f.kp + ((n0 * 16) << sh), sk);
      } else if constexpr (D % 64 == 0) {  // V: 64 dims of one key group
        const int g = n0 * 64 / D;
        const uint32_t pg = __builtin_amdgcn_readlane(f.page, 8 * g);
        to_lds(reinterpret_cast<const char *>(V) + static_cast<uint64_t>(pg) * page_bytes +
                   (((f.k0 + 8 * g) & (P - 1)) * D + (n0 * 64 - g * D) * 8) * 2 + lane * 16,
               sv);
      } else {
        const int p = n0 * 64 + lane, g = p / D, dim = p - g * D;
        const uint32_t pg = __shfl(f.page, 8 * g);
        to_lds(reinterpret_cast<const char *>(V) + static_cast<uint64_t>(pg) * page_bytes +
                   (((f.k0 + 8 * g) & (P - 1)) * D + dim * 8) * 2,
               sv);
      }
    } else if constexpr (kSame) {  // 64 places in order, each with the piece that belongs there
      const bool is_k = (j & 1) == 0;
      int off = is_k ? k_off : v_off;
      if (i) asm volatile("" : "+v"(off));  // the sum is formed here, not kept in a register
      to_lds(is_k ? f.rk : f.rv, off + i * (kNW * 64 / NP) * (is_k ? k_row : v_row), is_k ? sk : sv);
    } else {
      const int p = n0 * 64 + lane, key = p / NP, c = p - key * NP;
      if ((j & 1) == 0)
        to_lds(f.rk, key * k_row + (c ^ swap_k<D>(key_of_row(key & 31))) * 16, sk);
      else
        to_lds(f.rv, key * v_row + (c ^ swap_v<D>(key)) * 16, sv);
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
  auto k_at = [&](const char *sk, int sub, int s, int swap) IFX_INLINE {
    const char *p = PAGED ? sk + (k_lane + (2 * s * TK + 32 * sub) * 16)
                          : sk + ((swap ^ (32 * s)) + k_lane) + 32 * sub * NP * 16;
    return *reinterpret_cast<const u32x4 *>(p);
  };
  auto v_at = [&](const char *sv, int ks, int d) IFX_INLINE -> u32x4 {
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
  auto v_in = [&](int k0, const char *sv, int ks, int d) IFX_INLINE -> u32x4 {
    u32x4 r = v_at(sv, ks, d);
    if constexpr (PAGED) {
      const int key = k0 + 16 * ks + 8 * h;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[j] &= (key + 2 * j < kv ? 0xFFFFu : 0u) | (key + 2 * j + 1 < kv ? 0xFFFF0000u : 0u);
    }
    return r;
  };
  // Raises the running maximum where a stage's is far enough above it; what the
  // exponents are then taken relative to.
  auto raise = [&](float mt) IFX_INLINE {
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
  // One stage.  The matrix cores get the fragments of K, then of V, in one
  // sequence: fragment i + kAhead is on its way from LDS while i is multiplied.
  // next(j), j < 2 NL, issues the next stage's copies, one at a time between the
  // first products: a wave waits at its next copy until the last is under way.
  const f32x16 none_yet = {};
  auto step = [&](const char *sk, const char *sv, auto next) IFX_INLINE {
    constexpr int kAhead = 4;
    f32x16 s[2];
    u32x4 f[4 * NS];  // K of both halves, V: at most kAhead + 1 are alive
    int swap = k_swap;
    asm volatile("" : "+v"(swap));  // offsets formed anew in every stage, not kept in registers
    auto frag = [&](int i) {
      if (i < 2 * NS)
        f[i] = k_at(sk, i / NS, i % NS, swap);
      else if (i < 4 * NS)
        f[i] = v_at(sv, (i - 2 * NS) / ND, (i - 2 * NS) % ND);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) frag(i);
    if constexpr (!PAGED) {
#pragma unroll
      for (int j = 0; j < 2 * NL; ++j) next(j);
    }
    __builtin_amdgcn_sched_barrier(0);
    float mt[2] = {-__builtin_inff(), -__builtin_inff()};
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) {
      frag(i + kAhead);
      s[i / NS] = T::mfma32(f[i], qf[i % NS], i % NS ? s[i / NS] : none_yet);
      if constexpr (PAGED) {
#pragma unroll
        for (int j = i * NL / NS; j < (i + 1) * NL / NS; ++j) next(j);
      }
      // the first half's maximum beside the second half's products
      constexpr int kFrom = NS + NS / 4, kSteps = 2 * NS - kFrom;
      if (i >= kFrom) {
#pragma unroll
        for (int r = (i - kFrom) * 8 / kSteps; r < (i - kFrom + 1) * 8 / kSteps; ++r)
          mt[r & 1] = fmaxf(fmaxf(mt[r & 1], s[0][2 * r]), s[0][2 * r + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) mt[r & 1] = fmaxf(fmaxf(mt[r & 1], s[1][2 * r]), s[1][2 * r + 1]);
    const float mc = raise(fmaxf(mt[0], mt[1]));
    u32x4 pf[4];
    float sum[2] = {l, 0.0f};
    auto weigh = [&](int sub, int r) {  // keys 2r and 2r + 1 of a half
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][2 * r], a.c, -mc));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][2 * r + 1], a.c, -mc));
      sum[0] += p0;
      sum[1] += p1;
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
    l = sum[0] + sum[1];
  };

  // One stage of which some rows see only a part.
  bool tainted = false;
  auto edge_step = [&](int k0, const char *sk, const char *sv) IFX_INLINE {
    f32x16 s[2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
      for (int i = 0; i < NS; ++i)
        s[sub] = T::mfma32(k_at(sk, sub, i, k_swap), qf[i], i ? s[sub] : none_yet);
      __builtin_amdgcn_sched_barrier(0);  // a few fragments at a time: registers
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
    // A masked key's probability is 0, but 0 times an infinity or NaN is not: a
    // product of V with zeros shows whether the stage holds one.
    f32x16 probe = none_yet;
    const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const u32x4 v = v_in(k0, sv, ks, d);
        probe = T::mfma32(v, zero, probe);
        acc[d] = T::mfma32(v, pf[ks], acc[d]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    float any = probe[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) any += probe[r];
    tainted |= __any(any != 0.0f) != 0;
  };

  if (zbeg < zend) {
    int entry = 0, k0 = zbeg, buf = 0;
    if constexpr (PAGED) entry = entry_of(zbeg);
    {
      const Source f = source(zbeg, entry, 0);
#pragma unroll
      for (int j = 0; j < 2 * NL; ++j) copy(f, j);
    }
    if constexpr (PAGED) entry = entry_of(zbeg + TK);
    // Stages up to `until`.  (`last`: a stage among them may have no successor.)
    auto stages = [&](int until, auto edge_c, auto last_c) IFX_INLINE {
      for (; k0 < until; k0 += TK, buf ^= 1) {
        wait_own_memory();
        __syncthreads();  // this stage is in LDS, and no wave reads the other one
        const bool more = !decltype(last_c)::value || k0 + TK < zend;
        const Source f = source(more ? k0 + TK : zbeg, entry, buf ^ 1);
        if constexpr (PAGED) entry = entry_of(k0 + 2 * TK);
        auto next = [&](int j) {
          if (more) copy(f, j);
        };
        const char *sk = reinterpret_cast<const char *>(lds + buf * 2 * kPieces);
        const char *sv = sk + kPieces * 16;
        if (decltype(edge_c)::value || idle) {
#pragma unroll
          for (int j = 0; j < 2 * NL; ++j) next(j);
          if constexpr (decltype(edge_c)::value)
            if (!idle && k0 <= hi_z && k0 + TK > lo_a) edge_step(k0, sk, sv);
        } else {
          step(sk, sv, next);
        }
      }
    };
    // stages that all rows of the workgroup see whole, between those that some
    // see in part: where windows begin, and at the causal end
    using yes = std::true_type;
    using no = std::false_type;
    int until = a.window > 0 ? min(full_a, zend) : zbeg;
    while (true) {
      stages(until, yes{}, yes{});
      if (k0 >= zend) break;
      stages(min(full_z, zend - TK), no{}, no{});
      stages(min(full_z, zend), no{}, yes{});
      until = zend;
    }
  }

  // A wave that met an infinity or NaN in the values of a stage that its rows
  // see in part takes its rows again, key by key from memory, each lane its
  // row's half of the dims, so that a row takes only what it sees.  Rare and
  // slow (about a microsecond a key).
  if (tainted) {
    auto dim_of = [&](int i) { return 32 * (i >> 4) + 8 * (i >> 2 & 3) + 4 * h; };  // of i .. i + 3
    float q[ND * 16];
    const uint16_t *qp = static_cast<const uint16_t *>(a.q) + (q0 + tok) * a.q_stride +
                         static_cast<int64_t>(head) * D;
#pragma unroll
    for (int i = 0; i < ND * 16; ++i) q[i] = T::value(qp[dim_of(i) + (i & 3)]);
#pragma unroll
    for (int i = 0; i < ND * 16; ++i) acc[i >> 4][i & 15] = 0.0f;
    m = -__builtin_inff(), l = 0.0f;
#pragma unroll 1
    for (int key = zbeg; key < zend; ++key) {
      const char *kp, *vp;
      if constexpr (PAGED) {
        const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(
                                page_of(table[min(key >> sh, wmax)]))) * page_bytes;
        kp = reinterpret_cast<const char *>(K) + at + (key & (P - 1)) * 16;
        vp = reinterpret_cast<const char *>(V) + at + ((key & (P - 1) & ~7) * D + (key & 7)) * 2;
      } else {
        kp = reinterpret_cast<const char *>(K + key * a.k_stride);
        vp = reinterpret_cast<const char *>(V + key * a.v_stride);
      }
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < ND * 16; i += 4) {
        const int dim = dim_of(i);
        const u32x2 k4 = ldg<u32x2>(kp + (PAGED ? ((dim & ~7) * 2 << sh) + (dim & 7) * 2 : dim * 2));
        x = __builtin_fmaf(q[i], T::value(k4.x & 0xFFFFu), x);
        x = __builtin_fmaf(q[i + 1], T::value(k4.x >> 16), x);
        x = __builtin_fmaf(q[i + 2], T::value(k4.y & 0xFFFFu), x);
        x = __builtin_fmaf(q[i + 3], T::value(k4.y >> 16), x);
      }
      x = halves_sum(x);
      const bool seen = key >= lo && key <= hi;
      const float mn = seen ? fmaxf(m, x) : m;
      const float w = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * a.c);
      const float rel = mn == -__builtin_inff() ? 0.0f : mn * a.c - T::kShift;
      const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.c, -rel));
      m = mn;
      l = l * w + (seen && h == 0 ? pr : 0.0f);  // the halves' are added below
#pragma unroll
      for (int i = 0; i < ND * 16; ++i) {
        const float v = T::value(*reinterpret_cast<const uint16_t *>(
            vp + (dim_of(i) + (i & 3)) * (PAGED ? 16 : 2)));
        const float o = acc[i >> 4][i & 15] * w;
        acc[i >> 4][i & 15] = seen ? __builtin_fmaf(pr, v, o) : o;
      }
    }
  }

  l = halves_sum(l);
  bool none = hi < lo;  // the row sees no key
  bool own = row0 + 32 * wave + n < R;
  auto write_dims = [&](int d, const f32x4 *v, float scale) IFX_INLINE {  // of one dim tile
    if (!own) return;
    char *o = static_cast<char *>(a.out) +
              ((q0 + tok) * a.out_stride + static_cast<int64_t>(head) * D) * dtype_bytes(a.out_dtype);
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4(o, a.out_dtype, 32 * d + 8 * g + 4 * h, none ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v[g] * scale);
  };
  auto write = [&](float scale) IFX_INLINE {
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      f32x4 v[4];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i >> 2][i & 3] = acc[d][i];
      write_dims(d, v, scale);
    }
  };
  if (!PAGED || ns == 1) return write(1.0f / l);

  // split: this chunk's sums to its slot, every lane in its own places; the
  // last workgroup of the tile adds the chunks in their order, lane by lane.
  // Lanes without a row have their places behind the buffer's end: they write
  // nothing and read zeros.
  const rsrc_t part = make_rsrc(a.part, a.part_bytes);
  constexpr uint32_t kWaveBytes = 32 * D * 4 + 64 * 4 * 2, kSlotBytes = kNW * kWaveBytes;
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
    none = a.causal && ctx + tok < 0;  // a row that sees any sees itself
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
      total = total * weight(top, mn, a.c) + ml[y].y * weight(my, mn, a.c);
      top = mn;
    }
  }
  // N dim tiles from d on, four chunks at a time
  auto add_chunks = [&](int d, auto n_c) IFX_INLINE {
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
        const float w = y0 + y < ns ? weight(ml[y].x, top, a.c) : 0.0f;
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
    for (int d = few ? wave : 0; d < ND; d += few ? kNW : 1) add_chunks(d, one{});
  } else {
#pragma unroll 1
    for (int d = 0; d + 1 < ND; d += 2) add_chunks(d, two{});
    if constexpr (ND % 2) add_chunks(ND - 1, one{});
  }
  split_reset(cnt);
}

namespace {
template <int DT, int D, bool PAGED>
hipError_t launch_tile(const AttnArgs &a, int items, hipStream_t s) {
  constexpr int bytes = 2 * 2 * TK * D * 2;
  if constexpr (bytes > 65536 - 256) {
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const hipError_t e =
          allow_lds(reinterpret_cast<const void *>(&k_attn_tile<DT, D, PAGED>), bytes, done);
      if (e != hipSuccess) return e;
    }
  }
  IFX_LAUNCH(k_attn_tile, (DT, D, PAGED), dim3(a.Hkv * items), dim3(64 * kNW), bytes, s, a);
  return last_error();
}
template <int DT>
hipError_t launch_tile(const AttnArgs &a, int D, bool paged, int items, hipStream_t s) {
  switch (D) {
    case 64: return paged ? launch_tile<DT, 64, true>(a, items, s) : launch_tile<DT, 64, false>(a, items, s);
    case 96: return paged ? launch_tile<DT, 96, true>(a, items, s) : launch_tile<DT, 96, false>(a, items, s);
    case 128: return paged ? launch_tile<DT, 128, true>(a, items, s) : launch_tile<DT, 128, false>(a, items, s);
    default: return paged ? launch_tile<DT, 256, true>(a, items, s) : launch_tile<DT, 256, false>(a, items, s);
  }
}
}  // namespace

int attn_tile_rows(int) { return kRows; }
int attn_tile_min_keys() { return kMinChunk * TK; }
int64_t attn_tile_slot_bytes(int D) { return kNW * (32 * D * 4 + 64 * 4 * 2); }

hipError_t launch_attn_tile(const AttnArgs &a, int dtype, int D, bool paged, int items,
                            hipStream_t s) {
  return dtype == IFX_ATTN_F16 ? launch_tile<IFX_ATTN_F16>(a, D, paged, items, s)
                               : launch_tile<IFX_ATTN_BF16>(a, D, paged, items, s);
}

}  // namespace ifx
