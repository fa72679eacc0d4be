// attn_rows_q8.hip -- attention over the 8-bit paged cache of requests with few
// query rows (at most 32 = new tokens x query heads of a group, or some blocks of
// 32: decode steps, drafts).
//
//   s_j = sk_j q . ck_j,  p_j = 2^(c s_j - m),  l = sum p_j,
//   o = sum (p_j sv_j) cv_j / l;  ck, cv: codes, sk, sv: scales
//
// Bound by HBM, at half the 16-bit cache's bytes, or for few requests by latency.
// As in attn_rows a wave takes every fourth 32 keys of a chunk, and the rows of the
// key/value head are the columns of both products, transposed.  Codes go from the
// cache to LDS past the registers, each lane's to places that it alone reads, so
// that no wave waits for another; from there they are taken to fp16, exactly, half
// a vector instruction a code.  K's scales meet the scores, V's the probabilities,
// of which there are 32 times fewer than codes.
//
// Codes held in registers until their turn instead spilled: 270 us for 32 requests
// of 404.5 MB (40 / 8 heads of 128, 531 to 22591 keys) against 99, and 85 with the
// 16x16 products below: 4.8 TB/s, where a kernel that only copied the tiles took
// 82 and the 16-bit cache's takes 148.  One request of 3000 keys, 16 / 2 heads:
// 10.3 us.  768 to 2048 work items instead of 1024: the same.
#include "ifx_attn_rows_q8.h"

namespace ifx {

namespace {

// Rows of the 16x16 products, which take half the 32x32 ones' work and room: 32
// requests of 5 rows, 404.5 MB, 82 us with them and 99 without.
constexpr int kFewRows = 16;

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(F16::v8, a),
                                                __builtin_bit_cast(F16::v8, b), c, 0, 0, 0);
}

// Over the four lanes of the same lane % 16.
__device__ __forceinline__ void both_sixteens(float v, float &x, float &y) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  x = __builtin_bit_cast(float, static_cast<uint32_t>(r[0]));
  y = __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}
__device__ __forceinline__ float quarters_max(float v) {
  float x, y;
  both_sixteens(v, x, y);
  return halves_max(fmaxf(x, y));
}
__device__ __forceinline__ float quarters_sum(float v) {
  float x, y;
  both_sixteens(v, x, y);
  return halves_sum(x + y);
}

}  // namespace

template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_rows_q8(const AttnArgs a, int lds_rows, int blocks) {
  // Aligned, as copies of 16 bytes a lane to LDS need it: behind 1028 bytes of
  // other data they left parts of pieces wrong where many workgroups ran.
  extern __shared__ __attribute__((aligned(16))) float red[];
  __shared__ RowSums sums;
  RowsWork w;
  if (rows_work(a, red, lds_rows, blocks, w))
    rows32_q8<D>(a, w, red, sums, lds_rows * (D + 4) * 4, blockIdx.x % a.Hkv);
}

// At most 16 rows: the same with 16x16 products, so that half as many scores are
// weighed, and registers and LDS for twice as many workgroups.  Lane (m, g),
// m = lane % 16, g = lane / 16, holds row m: of S^T the keys 8 g + 4 i + r
// (register r of product i), which are the B operand of O^T = V^T P^T as they
// stand; of O^T the dims 16 d + 4 g + r.
template <int D>
__global__ __launch_bounds__(256, D == 256 ? 2 : 4) void k_attn_rows16_q8(const AttnArgs a, int lds_rows,
                                                                             int blocks) {
  constexpr int ND = D / 32, NB = D / 16;
  // at first the requests, then [wave][piece], then [wave][D / 4][row][4]
  extern __shared__ __attribute__((aligned(16))) float red[];
  __shared__ RowSums sums;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.Hkv;
  const int sh = a.page_shift, P = 1 << sh;
  RowsWork w;
  if (!rows_work(a, red, lds_rows, blocks, w)) return;

  const int row = row_of_lane(w, m), tok = row / a.G, head = kvh * a.G + row % a.G;
  const RowSight sight(a, w, tok);
  u32x4 qf[ND];
  {  // steps 2 i and 2 i + 1: the dims 64 i + 16 g + 0 .. 7 and + 8 .. 15, a piece of
     // K; a last step alone: 8 g .. + 7 of the last 32
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + (w.q0 + tok) * a.q_stride +
                        static_cast<int64_t>(head) * D;
#pragma unroll
    for (int s = 0; s < ND; ++s)
      qf[s] = ldg<u32x4>(q + (s + 1 == ND && ND % 2 ? 32 * s + 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1)));
  }
  f32x4 acc[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Level level;
  float l = 0.0f;

  // ---- a tile: memory to LDS past the registers, K [D / 16][32 keys], in the
  // order in which the products take them, V [2][D], scales [32]
  const int64_t page_bytes = (static_cast<int64_t>(a.Hkv) * D) << sh;
  const uint8_t *K = static_cast<const uint8_t *>(a.k) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint8_t *V = static_cast<const uint8_t *>(a.v) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint32_t *S = a.scales + (static_cast<int64_t>(kvh) << sh);
  u32x4 *tk = reinterpret_cast<u32x4 *>(red) + wave * tile_pieces<D>(), *tv = tk + ND * 64;
  u32x4 *ts = tv + ND * 64;
  const int kfirst = w.zbeg + 32 * wave, tiles = (w.zend - kfirst + kStep - 1) / kStep;
  Pages pages(a, w.b, kfirst);
  const int kl = (lane >> 2 & 3) * 8 + (lane >> 4 & 1) * 4 + (lane & 3);  // the key that a lane copies
  auto issue_k = [&](int t) __attribute__((always_inline)) {
    if (t && (t & 63) == 0) pages.read(t);
    const int k0 = kfirst + t * kStep, pg0 = pages.page0(t), pg1 = pages.page1(t);
    const uint8_t *kp = K + (kl & 16 ? pg1 : pg0) * page_bytes +
                        ((((k0 + kl) & (P - 1)) + ((lane >> 5) << sh)) * 16);
#pragma unroll
    for (int i = 0; i < ND; ++i) to_lds16(kp + ((i * 32) << sh), tk + i * 64);
    const int n = lane & 31;
    to_lds4(S + ((static_cast<int64_t>(n & 16 ? pg1 : pg0) * a.Hkv) << sh) + ((k0 + n) & (P - 1)), ts);
  };
  auto issue_v = [&](int t) __attribute__((always_inline)) {
    const int k0 = kfirst + t * kStep, pg0 = pages.page0(t), pg1 = pages.page1(t);
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const int p = i * 64 + lane, half = p >= D, dim = p - (half ? D : 0);
      to_lds16(V + (half ? pg1 : pg0) * page_bytes + ((k0 + 16 * half) & (P - 1)) * D + dim * 16, tv + i * 64);
    }
  };

  pages.read(0);  // and the rows of Q are here
  const float c = row_to_f16<16>(qf, a.q_dtype, a.c);
  if (tiles > 0) {
    issue_k(0);
    issue_v(0);
  }
#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    const int k0 = kfirst + t * kStep;
    const bool more = t + 1 < tiles;
    wait_loads<ND>();  // K and the scales; V's are behind them
    f32x4 s[2] = {};
#pragma unroll
    for (int i = 0; i < (ND + 1) / 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (2 * i + 1 < ND) {
          const u32x4 k = tk[(4 * i + g) * 32 + 16 * e + m];
          s[e] = mfma16(codes_f16(k, 0), qf[2 * i], s[e]);
          s[e] = mfma16(codes_f16(k, 1), qf[2 * i + 1], s[e]);
        } else {
          const u32x2 k = reinterpret_cast<const u32x2 *>(tk + (4 * i + (g >> 1)) * 32 + 16 * e + m)[g & 1];
          s[e] = mfma16(codes_f16(k), qf[2 * i], s[e]);
        }
      }
    float sv[2][4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const u32x4 f = ts[2 * g + e];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[e][r] *= k_scale(f[r]);
        sv[e][r] = v_scale(f[r]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // K's and the scales' places are read
    if (more) issue_k(t + 1);
    if (in_part(a, w, k0)) {  // what the row does not see, a page's unwritten slots among it
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool sees = sight.sees(k0 + 8 * g + 4 * e + r);
          s[e][r] = sees ? s[e][r] : -__builtin_inff();
          sv[e][r] = sees ? sv[e][r] : 0.0f;
        }
    }
    float mt = s[0][0], vt = sv[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mt = fmaxf(mt, s[i >> 2][i & 3]), vt = fmaxf(vt, sv[i >> 2][i & 3]);
    mt = quarters_max(mt), vt = quarters_max(vt);
    if (__any(level.above(mt, vt, c))) {
      const float less = level.raise(mt, vt, c);
      l *= less;
#pragma unroll
      for (int d = 0; d < NB; ++d) acc[d] *= less;
    }
    u32x4 pf;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][2 * (i & 1)], c, -level.less));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][2 * (i & 1) + 1], c, -level.less));
      l += p0 + p1;
      pf[i] = F16::pack(p0 * sv[i >> 1][2 * (i & 1)], p1 * sv[i >> 1][2 * (i & 1) + 1]);
    }
    if (more)
      wait_loads<ND + 1>();  // V; the next tile's K and scales are behind it
    else
      wait_loads<0>();
#pragma unroll
    for (int d = 0; d < NB; ++d) {
      const u32x2 v = reinterpret_cast<const u32x2 *>(tv + (g >> 1) * D + 16 * d + m)[g & 1];
      acc[d] = mfma16(codes_f16(v), pf, acc[d]);
    }
    __builtin_amdgcn_sched_barrier(0);  // V's places are read
    if (more) issue_v(t + 1);
  }

  l = quarters_sum(l);
  const float level_of = level.of_sums(), top = rows_top(sums, wave, m, g == 0, level_of, l);
  if (m < w.R) {
    const float scale = weight(level_of, top, 1.0f);
#pragma unroll
    for (int d = 0; d < NB; ++d) {
      const f32x4 v = acc[d] * scale;
      __builtin_memcpy(red + ((wave * (D / 4) + 4 * d + g) * w.R + m) * 4, &v, 16);
    }
  }
  rows_finish<D, 16, D == 256>(a, w.split, red, sums, m, g == 0, top, 1.0f, lds_rows * (D + 4) * 4, w.R,
                               w.block, w.z, w.ns, kvh, [&](int t) { return row_sees_nothing(a, w, t); });
}

namespace {
template <int D, bool FEW>
hipError_t launch_rows(const AttnArgs &a, int max_rows, int blocks, int items, hipStream_t s) {
  constexpr int row_bytes = kRowWaves * D * 4;  // LDS of a row: the waves' sums
  constexpr int rows = FEW ? kFewRows : kRowsMax;
  constexpr int ring_bytes = FEW ? kRowWaves * tile_pieces<D>() * 16 : rows32_bytes<D>();
  constexpr int most = ring_bytes > row_bytes * rows ? ring_bytes : row_bytes * rows;
  if constexpr (most > 65536 - 2048) {  // what a launch may ask for without more ado
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const void *kernel = FEW ? reinterpret_cast<const void *>(&k_attn_rows16_q8<D>)
                               : reinterpret_cast<const void *>(&k_attn_rows_q8<D>);
      const hipError_t e = allow_lds(kernel, most, done);
      if (e != hipSuccess) return e;
    }
  }
  // the tiles; before them the requests, after them the waves' sums, and then the
  // chunks' weights and sums
  int bytes = ring_bytes;
  for (const int need : {row_bytes * max_rows, a.B * 8, a.goal * max_rows * 8})
    if (bytes < need) bytes = need;
  const dim3 grid(a.Hkv * items), block(64 * kRowWaves);
  if constexpr (FEW)
    IFX_LAUNCH(k_attn_rows16_q8, (D), grid, block, bytes, s, a, max_rows, blocks);
  else
    IFX_LAUNCH(k_attn_rows_q8, (D), grid, block, bytes, s, a, max_rows, blocks);
  return last_error();
}
template <int D>
hipError_t launch_rows(const AttnArgs &a, int max_rows, int blocks, int items, hipStream_t s) {
  return max_rows <= kFewRows ? launch_rows<D, true>(a, max_rows, blocks, items, s)
                              : launch_rows<D, false>(a, max_rows, blocks, items, s);
}
}  // namespace

hipError_t launch_attn_rows_q8(const AttnArgs &a, int D, int max_rows, int blocks, int items,
                               hipStream_t s) {
  switch (D) {
    case 64: return launch_rows<64>(a, max_rows, blocks, items, s);
    case 96: return launch_rows<96>(a, max_rows, blocks, items, s);
    case 128: return launch_rows<128>(a, max_rows, blocks, items, s);
    default: return launch_rows<256>(a, max_rows, blocks, items, s);
  }
}

}  // namespace ifx
