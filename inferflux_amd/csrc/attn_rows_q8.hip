// attn_rows_q8.hip -- attention over the 8-bit paged cache of requests with few
// query rows (at most 32 = new tokens x query heads of a group: decode steps,
// drafts).
//
//   s_j = sk_j q . ck_j,  p_j = 2^(c s_j - m),  l = sum p_j,
//   o = sum (p_j sv_j) cv_j / l;  ck, cv: codes, sk, sv: scales
//
// Bound by HBM: as attn_rows, with half its bytes.  The codes go from the cache
// into registers, half a kilobyte a half-wave, and are taken to fp16 operands
// there, one vector instruction a code; K's scales meet the scores, V's the
// probabilities, of which there are 32 times fewer than codes.  The next
// tile's loads are on their way during a tile's products.
#include "ifx_attn_q8.h"
#include "ifx_attn_rows.h"

namespace ifx {

namespace {

// Key of A-operand row m of S^T = K Q^T: with register r of lane half h as key
// 16 h + r, the probabilities of a half are those of one piece of V's 16 tokens.
__device__ __forceinline__ int key_of_row16(int m) {
  return (m & 3) | ((m >> 1) & 0xC) | ((m & 4) << 2);
}

}  // namespace

template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_rows_q8(const AttnArgs a, int lds_rows) {
  constexpr int ND = D / 32, NS = D / 16;
  extern __shared__ float red[];  // [wave][D / 4][row][4]; at first the requests
  __shared__ RowSums sums;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.Hkv;
  const int sh = a.page_shift, P = 1 << sh;

  // the workgroup's request and chunk of its keys
  const Split split = find_item<1>(
      a, reinterpret_cast<int2 *>(red), blockIdx.x / a.Hkv, [&](const Request &r) {
        int keys = r.kv;
        if (a.window > 0) keys = min<int64_t>(keys, static_cast<int64_t>(a.window) + r.nq + kRowKeys);
        return make_int2(r.nq > 0 ? 1 : 0, max(1, (keys + kRowKeys - 1) / kRowKeys));
      });
  if (split.chunk == 0) return;
  const int b = split.b, z = split.item;
  const int q0 = split.req.q0, nq = split.req.nq, kv = split.req.kv, R = min(nq * a.G, lds_rows);
  const int ctx = kv - nq;  // position of the first row; below 0 it sees nothing
  const bool tree = a.masks != nullptr;
  const int lo0 = a.window > 0 ? max(0, ctx - a.window + 1) : 0;
  const int kbeg = lo0 & ~(kRowKeys - 1), kend = kv;
  const int chunk = split.chunk * kRowKeys;
  const int ns = kend > kbeg ? (kend - kbeg + chunk - 1) / chunk : 1;
  if (z >= ns) return;
  const int zbeg = kbeg + z * chunk, zend = min(zbeg + chunk, kend);

  // this lane's row; rows behind the last repeat it
  const int row = min(n, R - 1), tok = row / a.G, head = kvh * a.G + row % a.G;
  const Sight<false> line = {a.window > 0 ? max(0, ctx + tok - a.window + 1) : 0, ctx + tok, ctx, 0};
  Sight<true> nodes = {0, 0, ctx, 0};
  if (tree) nodes.bits = node_bits(a, q0 + tok, nq);
  u32x4 qf[NS];
  {  // of step s the dims 32 (s / 2) + 16 h + 8 (s % 2), as K's pieces hold them
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + (q0 + tok) * a.q_stride +
                        static_cast<int64_t>(head) * D + 16 * h;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = ldg<u32x4>(q + 32 * (s >> 1) + 8 * (s & 1));
  }
  const float c = row_to_f16(qf, a.q_dtype, a.c);

  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
  Level level;
  float l = 0.0f;

  const int kn = key_of_row16(n);  // the key of a tile whose K this lane loads
  const int32_t *table = a.table + static_cast<int64_t>(b) * a.table_width;
  const int last_page = static_cast<int>(a.num_pages) - 1, wmax = a.table_width - 1;
  const int64_t page_bytes = (static_cast<int64_t>(a.Hkv) * D) << sh;
  const uint8_t *K = static_cast<const uint8_t *>(a.k) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint8_t *V = static_cast<const uint8_t *>(a.v) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint32_t *S = a.scales + (static_cast<int64_t>(kvh) << sh);

  // A tile's codes and scales as they lie in the cache.
  struct Raw {
    u32x4 k[ND], v[ND], s[4];
  };
  // The pages of a tile's two 16-key halves, as the table has them: read a tile
  // ahead, looked at when that tile's loads are issued.
  int next0 = 0, next1 = 0;
  auto entries = [&](int k0) {
    next0 = table[min(k0 >> sh, wmax)];
    next1 = table[min((k0 + 16) >> sh, wmax)];
  };
  auto load = [&](Raw &f, int k0) __attribute__((always_inline)) {
    const int pg0 = min(max(next0, 0), last_page), pg1 = min(max(next1, 0), last_page);
    entries(k0 + 32 * kRowWaves);
    const uint8_t *kp = K + (kn & 16 ? pg1 : pg0) * page_bytes +
                        ((((k0 + kn) & (P - 1)) + (h << sh)) * 16);
#pragma unroll
    for (int i = 0; i < ND; ++i) f.k[i] = ldg<u32x4>(kp + ((i * 32) << sh));
    const int pg = h ? pg1 : pg0, at = (k0 + 16 * h) & (P - 1);
    const uint32_t *sp = S + ((static_cast<int64_t>(pg) * a.Hkv) << sh) + at;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.s[i] = ldg<u32x4>(sp + 4 * i);
    const uint8_t *vp = V + pg * page_bytes + at * D + n * 16;
#pragma unroll
    for (int d = 0; d < ND; ++d) f.v[d] = ldg<u32x4>(vp + d * 512);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto tile = [&](const Raw &f, int k0) __attribute__((always_inline)) {
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i) s = F16::mfma32(codes_f16(f.k[i >> 1], i & 1), qf[i], s);
    float sv[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] *= k_scale(f.s[r >> 2][r & 3]);
      sv[r] = v_scale(f.s[r >> 2][r & 3]);
    }
    if (k0 + 31 >= ctx + !tree || (a.window > 0 && k0 < ctx + nq - a.window)) {
      // what the row does not see, a page's unwritten slots among it
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = k0 + 16 * h + r;
        const bool sees = tree ? nodes.sees(key) : line.sees(key);
        s[r] = sees ? s[r] : -__builtin_inff();
        sv[r] = sees ? sv[r] : 0.0f;
      }
    }
    float mt = s[0], vt = sv[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]), vt = fmaxf(vt, sv[r]);
    mt = halves_max(mt), vt = halves_max(vt);
    if (__any(level.above(mt, vt, c))) {
      const float w = level.raise(mt, vt, c);
      l *= w;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= w;
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
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] = F16::mfma32(codes_f16(f.v[d], ks), pf[ks], acc[d]);
  };

  constexpr int kStep = 32 * kRowWaves;
  int k0 = zbeg + 32 * wave;
  if (k0 < zend) {
    Raw f, g;  // in turn: one's loads are on their way while the other is worked on
    entries(k0);
    load(f, k0);
    while (true) {
      if (k0 + kStep >= zend) {
        tile(f, k0);
        break;
      }
      load(g, k0 + kStep);
      tile(f, k0);
      k0 += kStep;
      if (k0 + kStep >= zend) {
        tile(g, k0);
        break;
      }
      load(f, k0 + kStep);
      tile(g, k0);
      k0 += kStep;
    }
  }

  rows_finish<D>(a, split, red, sums, acc, level.of_sums(), l, 1.0f, lds_rows, R, ns, kvh, [&](int t) {
    return tree ? Sight<true>{0, 0, ctx, node_bits(a, q0 + t, nq)}.nothing() : ctx + t < 0;
  });
}

namespace {
constexpr int kMaxLds = 65536 - 2048;  // what a launch may ask for without more ado

template <int D>
hipError_t launch_rows(const AttnArgs &a, int max_rows, int items, hipStream_t s) {
  constexpr int row_bytes = kRowWaves * D * 4;  // LDS of a row: the waves' sums
  if constexpr (row_bytes * kRowsMax > kMaxLds) {
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const hipError_t e = allow_lds(reinterpret_cast<const void *>(&k_attn_rows_q8<D>),
                                     row_bytes * kRowsMax, done);
      if (e != hipSuccess) return e;
    }
  }
  // the waves' sums; before them the requests, after them the chunks' weights and sums
  int bytes = row_bytes * max_rows;
  if (bytes < a.B * 8) bytes = a.B * 8;
  if (bytes < a.goal * max_rows * 8) bytes = a.goal * max_rows * 8;
  IFX_LAUNCH(k_attn_rows_q8, (D), dim3(a.Hkv * items), dim3(64 * kRowWaves), bytes, s, a, max_rows);
  return last_error();
}
}  // namespace

hipError_t launch_attn_rows_q8(const AttnArgs &a, int D, int max_rows, int items, hipStream_t s) {
  switch (D) {
    case 64: return launch_rows<64>(a, max_rows, items, s);
    case 96: return launch_rows<96>(a, max_rows, items, s);
    case 128: return launch_rows<128>(a, max_rows, items, s);
    default: return launch_rows<256>(a, max_rows, items, s);
  }
}

}  // namespace ifx
