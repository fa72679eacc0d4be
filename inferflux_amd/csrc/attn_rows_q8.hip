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

constexpr int kStep = 32 * kRowWaves;  // keys from a wave's tile to its next
constexpr int kDepth = 2;              // tiles that are on their way or worked on
// 16-byte places of a tile in LDS: K, V, and 64 dwords of scales (32 keys', twice).
template <int D>
constexpr int tile_pieces() {
  return 2 * (D / 32) * 64 + 16;
}

// 16 or 4 bytes a lane from memory to 64 consecutive places in LDS.
__device__ __forceinline__ void to_lds16(const void *from, u32x4 *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
__device__ __forceinline__ void to_lds4(const void *from, u32x4 *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)to, 4, 0, 0);
}

// Waits until at most N of this wave's loads are on their way: loads end in
// order, so all before its last N have ended.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "six bits count them");
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4 << 14));
  __builtin_amdgcn_sched_barrier(0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

}  // namespace

template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_rows_q8(const AttnArgs a, int lds_rows) {
  constexpr int ND = D / 32, NS = D / 16;
  // at first the requests, then [wave][tile][piece], then [wave][D / 4][row][4]
  extern __shared__ float red[];
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

  // ---- tiles: memory to LDS past the registers, each lane's pieces to its own
  // places, so that no wave waits for another
  const int kn = key_of_row16(n);  // the key of a tile whose K this lane takes
  const int32_t *table = a.table + static_cast<int64_t>(b) * a.table_width;
  const int last_page = static_cast<int>(a.num_pages) - 1, wmax = a.table_width - 1;
  const int64_t page_bytes = (static_cast<int64_t>(a.Hkv) * D) << sh;
  const uint8_t *K = static_cast<const uint8_t *>(a.k) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint8_t *V = static_cast<const uint8_t *>(a.v) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint32_t *S = a.scales + (static_cast<int64_t>(kvh) << sh);
  constexpr int kPieces = tile_pieces<D>(), kLoads = 2 * ND + 1;  // of a tile
  u32x4 *ring = reinterpret_cast<u32x4 *>(red) + wave * kDepth * kPieces;
  const int kfirst = zbeg + 32 * wave;
  const int tiles = (zend - kfirst + kStep - 1) / kStep;
  // The pages of the tiles' two 16-key halves, as the table has them: of 64 tiles
  // at a time, a lane each.
  int entry0 = 0, entry1 = 0;
  auto issue = [&](int t) __attribute__((always_inline)) {
    if ((t & 63) == 0) {
      const int k = kfirst + (t + lane) * kStep;
      entry0 = table[min(k >> sh, wmax)];
      entry1 = table[min((k + 16) >> sh, wmax)];
    }
    const int k0 = kfirst + t * kStep;
    const int pg0 = min(max(__builtin_amdgcn_readlane(entry0, t & 63), 0), last_page);
    const int pg1 = min(max(__builtin_amdgcn_readlane(entry1, t & 63), 0), last_page);
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

  rows_finish<D>(a, split, red, sums, acc, level.of_sums(), l, 1.0f, lds_rows, R, ns, kvh, [&](int t) {
    return tree ? Sight<true>{0, 0, ctx, node_bits(a, q0 + t, nq)}.nothing() : ctx + t < 0;
  });
}

namespace {
template <int D>
hipError_t launch_rows(const AttnArgs &a, int max_rows, int items, hipStream_t s) {
  constexpr int row_bytes = kRowWaves * D * 4;  // LDS of a row: the waves' sums
  constexpr int ring_bytes = kRowWaves * kDepth * tile_pieces<D>() * 16;
  constexpr int most = ring_bytes > row_bytes * kRowsMax ? ring_bytes : row_bytes * kRowsMax;
  if constexpr (most > 65536 - 2048) {  // what a launch may ask for without more ado
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const hipError_t e = allow_lds(reinterpret_cast<const void *>(&k_attn_rows_q8<D>), most, done);
      if (e != hipSuccess) return e;
    }
  }
  // the tiles; before them the requests, after them the waves' sums, and then the
  // chunks' weights and sums
  int bytes = ring_bytes;
  for (const int need : {row_bytes * max_rows, a.B * 8, a.goal * max_rows * 8})
    if (bytes < need) bytes = need;
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
