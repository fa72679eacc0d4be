// attn_rows.hip -- paged attention of requests with few query rows (at most
// 32 = new tokens x query heads of a group: decode steps), and of trees of drafts
// with more, in blocks of 32.
//
//   s_j = c q . k_j (c = scale log2 e), p_j = 2^(s_j - m), l = sum p_j,
//   o = sum p_j v_j / l
//
// Bound by HBM: every key and value of the request is read once for 2 x 32
// (padded) x D multiply-adds an element, well under the MFMA rate.  So what
// counts is bytes in flight.  The cache's layout is the MFMA operand order:
// each wave reads its 32 keys' K and V straight into operand registers with
// contiguous 16-byte loads, 16 KB a wave at D = 128, and nothing passes
// through LDS.  Waves take tiles of 32 keys in turn, each with its own running
// maximum and sums; they meet once, in LDS, at the end.  The keys of all
// requests are cut into chunks of about one length (find_item); the last
// workgroup of a request and head to finish adds the chunks in their order.
//
// Measured: 32 requests of 531 to 22591 keys, 40 query and 8 key/value heads of
// 128 (796 MB), 148 us, 5.4 TB/s (matrix cores busy for 7 % of the time, vector
// units for 13); with chunks as long as the longest request's
// eighth, 187.  One request of 3000 keys, 16 and 2 heads: 9.6 us, of them 1 to
// find the work, 1.4 for the keys, 1.7 for the waves' and 4 for the chunks' sums.
#include "ifx_attn_rows.h"

namespace ifx {

namespace {

constexpr int kWaves = kRowWaves;

// The four dwords of an 8-key piece with the keys outside [lo, hi] cleared.
struct PieceMask {
  uint32_t m[4];
};
__device__ __forceinline__ PieceMask piece_mask(int key, int lo, int hi) {
  PieceMask r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k0 = key + 2 * j, k1 = k0 + 1;
    r.m[j] = (k0 >= lo && k0 <= hi ? 0xFFFFu : 0u) | (k1 >= lo && k1 <= hi ? 0xFFFF0000u : 0u);
  }
  return r;
}

}  // namespace

// TREE: rows see the cached tokens and the nodes of their masks; more than 32
// are blocks of 32, the keys of each split by themselves, `most` blocks of a request
// at most.
template <int DT, int D, bool TREE = false>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_rows(const AttnArgs a, int lds_rows, int most) {
  using T = Elem<DT>;
  constexpr int ND = D / 32, NS = D / 16;
  extern __shared__ float red[];  // [wave][D / 4][row][4]; at first the requests
  __shared__ RowSums sums;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.Hkv;
  const int sh = a.page_shift, P = 1 << sh;

  // the workgroup's request and chunk of its keys
  const Split split = find_item<1, TREE ? kRowsRoot : 0>(
      a, reinterpret_cast<int2 *>(red), blockIdx.x / a.Hkv, [&](const Request &r) {
        int keys = r.kv;
        if (a.window > 0) keys = min<int64_t>(keys, static_cast<int64_t>(a.window) + r.nq + kRowKeys);
        const int blocks = TREE ? min((r.nq * a.G + 31) / 32, most) : r.nq > 0 ? 1 : 0;
        return make_int2(blocks, max(1, (keys + kRowKeys - 1) / kRowKeys));
      });
  if (split.chunk == 0) return;
  const int b = split.b, z = TREE ? split.item / split.tiles : split.item;
  const int block = TREE ? split.item - z * split.tiles : 0, row0 = 32 * block;
  const int q0 = split.req.q0, nq = split.req.nq, kv = split.req.kv, R = min(nq * a.G - row0, lds_rows);
  const int ctx = kv - nq;  // position of the first row; below 0 it sees nothing
  const int lo0 = a.window > 0 ? max(0, ctx - a.window + 1) : 0;
  const int kbeg = lo0 & ~(kRowKeys - 1), kend = kv;  // the last row sees kv - 1
  const int chunk = split.chunk * kRowKeys;
  const int ns = kend > kbeg ? (kend - kbeg + chunk - 1) / chunk : 1;
  if (z >= ns) return;
  const int zbeg = kbeg + z * chunk, zend = min(zbeg + chunk, kend);

  // this lane's row: what it sees is [lo, hi]; rows behind the last repeat it
  const int row = row0 + min(n, R - 1), tok = row / a.G, head = kvh * a.G + row % a.G;
  Sight<TREE> sight = {0, ctx + tok, ctx, 0};
  if constexpr (TREE)
    sight.bits = node_bits(a, q0 + tok, nq);
  else if (a.window > 0)
    sight.lo = max(0, sight.hi - a.window + 1);
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

  const int kn = key_of_row(n);  // the key of a tile whose K this lane loads
  const int32_t *table = a.table + static_cast<int64_t>(b) * a.table_width;
  const int last_page = static_cast<int>(a.num_pages) - 1;
  const int64_t page_elems = (static_cast<int64_t>(a.Hkv) * D) << sh;
  const uint16_t *K = static_cast<const uint16_t *>(a.k) + ((static_cast<int64_t>(kvh) * D) << sh);
  const uint16_t *V = static_cast<const uint16_t *>(a.v) + ((static_cast<int64_t>(kvh) * D) << sh);
  const int wmax = a.table_width - 1;

  // The pages of a tile's two 16-key halves, as the table has them: read a tile
  // ahead, looked at when that tile's loads are issued.
  int next0 = 0, next1 = 0;
  auto entries = [&](int k0) {
    next0 = table[min(k0 >> sh, wmax)];
    next1 = table[min((k0 + 16) >> sh, wmax)];
  };
  entries(zbeg + 32 * wave);
  for (int k0 = zbeg + 32 * wave; k0 < zend; k0 += 32 * kWaves) {
    const int pg0 = min(max(next0, 0), last_page);
    const int pg1 = min(max(next1, 0), last_page);
    entries(k0 + 32 * kWaves);
    const int64_t e0 = pg0 * page_elems, e1 = pg1 * page_elems;
    u32x4 kf[NS], vf[2][ND];
    {
      const uint16_t *kp = K + (kn & 16 ? e1 : e0) + ((k0 + kn) & (P - 1)) * 8 + ((h * 8) << sh);
#pragma unroll
      for (int s = 0; s < NS; ++s) kf[s] = ldg<u32x4>(kp + ((s * 16) << sh));
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const uint16_t *vp = V + (ks ? e1 : e0) +
                             (((k0 + 16 * ks) & (P - 1)) + 8 * h) * D + n * 8;
#pragma unroll
        for (int d = 0; d < ND; ++d) vf[ks][d] = ldg<u32x4>(vp + d * 256);
      }
    }
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i) s = T::mfma32(kf[i], qf[i], s);

    const bool edge = k0 + 31 > ctx - TREE || (a.window > 0 && k0 < ctx + nq - a.window);
    if (edge) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = k0 + 16 * (r >> 3) + 8 * h + (r & 7);
        s[r] = sight.sees(key) ? s[r] : -__builtin_inff();
      }
      // values that no row sees: the pages' unwritten slots among them
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const PieceMask pm = piece_mask(k0 + 16 * ks + 8 * h, lo0, kv - 1);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[ks][d][j] &= pm.m[j];
      }
    }
    float mt = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]);
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
    u32x4 pf[2];
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -mc));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], a.c, -mc));
      sum += p0 + p1;
      pf[r >> 3][(r & 7) >> 1] = T::pack(p0, p1);
    }
    l += sum;

    bool apart = false;  // an infinity or NaN in V that some rows see and others do not
    if (edge && (TREE || nq > 1)) {
      f32x16 probe;
#pragma unroll
      for (int r = 0; r < 16; ++r) probe[r] = 0.0f;
      const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) probe = T::mfma32(vf[ks][d], zero, probe);
      float any = probe[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) any += probe[r];
      apart = __any(any != 0.0f);
    }
    if (!apart) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = T::mfma32(vf[ks][d], pf[ks], acc[d]);
    } else {
      // key by key, so that a row takes only the values that it sees
#pragma unroll 1
      for (int i = 0; i < 32; ++i) {
        const int key = k0 + i, w = (i & 7) >> 1;
        const u32x4 pk = i < 16 ? pf[0] : pf[1];
        const uint32_t pd = w == 0 ? pk[0] : w == 1 ? pk[1] : w == 2 ? pk[2] : pk[3];
        const uint32_t mine = (pd >> (16 * (i & 1))) & 0xFFFFu;
        const float p = T::value(static_cast<uint32_t>(
            __shfl(static_cast<int>(mine), n + 32 * ((i >> 3) & 1))));
        if (key < lo0 || key >= kv) continue;
        const bool seen = sight.sees(key);
        const uint16_t *vp = V + (i < 16 ? e0 : e1) + ((key & (P - 1)) & ~7) * D + (key & 7);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float v = T::value(vp[(32 * d + 8 * (r >> 2) + 4 * h + (r & 3)) * 8]);
            acc[d][r] = seen ? __builtin_fmaf(p, v, acc[d][r]) : acc[d][r];
          }
      }
    }
  }

  l = halves_sum(l);
  const float top = rows_top(sums, wave, n, h == 0, m, l);
  if (n < R) put_rows32<D>(red, acc, weight(m, top, a.c), R, n, h, wave);
  const uint32_t slot_bytes = lds_rows * (D + 4) * 4;
  rows_finish<D, 24, TREE>(a, split, red, sums, n, h == 0, top, a.c, slot_bytes, R, block, z, ns, kvh, [&](int t) {
    if constexpr (TREE)
      return Sight<true>{0, 0, ctx, node_bits(a, q0 + t, nq)}.nothing();
    else
      return ctx + t < 0;
  });
}

namespace {
constexpr int kMaxLds = 65536 - 2048;  // what a launch may ask for without more ado

template <int DT, int D, bool TREE>
hipError_t launch_rows(const AttnArgs &a, int max_rows, int blocks, int items, hipStream_t s) {
  constexpr int row_bytes = kWaves * D * 4;  // LDS of a row: the waves' sums
  if constexpr (row_bytes * kRowsMax > kMaxLds) {
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const hipError_t e = allow_lds(reinterpret_cast<const void *>(&k_attn_rows<DT, D, TREE>),
                                     row_bytes * kRowsMax, done);
      if (e != hipSuccess) return e;
    }
  }
  // the waves' sums; before them the requests, after them the chunks' weights and sums
  int bytes = row_bytes * max_rows;
  if (bytes < a.B * 8) bytes = a.B * 8;
  if (bytes < a.goal * max_rows * 8) bytes = a.goal * max_rows * 8;
  if constexpr (TREE)
    IFX_LAUNCH(k_attn_rows, (DT, D, true), dim3(a.Hkv * items), dim3(64 * kWaves), bytes, s, a, max_rows, blocks);
  else
    IFX_LAUNCH(k_attn_rows, (DT, D), dim3(a.Hkv * items), dim3(64 * kWaves), bytes, s, a, max_rows, blocks);
  return last_error();
}
template <int DT, bool TREE>
hipError_t launch_rows(const AttnArgs &a, int D, int max_rows, int blocks, int items, hipStream_t s) {
  switch (D) {
    case 64: return launch_rows<DT, 64, TREE>(a, max_rows, blocks, items, s);
    case 96: return launch_rows<DT, 96, TREE>(a, max_rows, blocks, items, s);
    case 128: return launch_rows<DT, 128, TREE>(a, max_rows, blocks, items, s);
    default: return launch_rows<DT, 256, TREE>(a, max_rows, blocks, items, s);
  }
}
template <int DT>
hipError_t launch_rows(const AttnArgs &a, int D, int max_rows, int blocks, int items, hipStream_t s) {
  return a.masks ? launch_rows<DT, true>(a, D, max_rows, blocks, items, s)
                 : launch_rows<DT, false>(a, D, max_rows, blocks, items, s);
}
}  // namespace

int attn_rows_max_goal(int max_rows) { return kMaxLds / 8 / max_rows; }

hipError_t launch_attn_rows(const AttnArgs &a, int dtype, int D, int max_rows, int blocks, int items,
                            hipStream_t s) {
  return dtype == IFX_ATTN_F16 ? launch_rows<IFX_ATTN_F16>(a, D, max_rows, blocks, items, s)
                               : launch_rows<IFX_ATTN_BF16>(a, D, max_rows, blocks, items, s);
}

}  // namespace ifx
