// attn_rows.hip -- paged attention of requests with few query rows (at most
// 32 = new tokens x query heads of a group: decode steps).
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
#include "ifx_attn.h"

namespace ifx {

namespace {

constexpr int kWaves = 4;
constexpr uint32_t kOut = 1u << 30;  // an offset past the workspace's end: reads zeros

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

template <int DT, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_rows(const AttnArgs a, int lds_rows) {
  using T = Elem<DT>;
  constexpr int ND = D / 32, NS = D / 16;
  extern __shared__ float red[];  // [wave][D / 4][row][4]; at first the requests
  __shared__ float red_m[kWaves][32], red_l[kWaves][32];
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
  const int lo0 = a.window > 0 ? max(0, ctx - a.window + 1) : 0;
  const int kbeg = lo0 & ~(kRowKeys - 1), kend = kv;  // the last row sees kv - 1
  const int chunk = split.chunk * kRowKeys;
  const int ns = kend > kbeg ? (kend - kbeg + chunk - 1) / chunk : 1;
  if (z >= ns) return;
  const int zbeg = kbeg + z * chunk, zend = min(zbeg + chunk, kend);

  // this lane's row: what it sees is [lo, hi]; rows behind the last repeat it
  const int row = min(n, R - 1), tok = row / a.G, head = kvh * a.G + row % a.G;
  const int hi = ctx + tok, lo = a.window > 0 ? max(0, hi - a.window + 1) : 0;
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

    const bool edge = k0 + 31 > ctx || (a.window > 0 && k0 < ctx + nq - a.window);
    if (edge) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = k0 + 16 * (r >> 3) + 8 * h + (r & 7);
        s[r] = key >= lo && key <= hi ? s[r] : -__builtin_inff();
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
    if (edge && nq > 1) {
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
        const bool seen = key >= lo && key <= hi;
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

  // the four waves' sums, in the waves' order
  l = halves_sum(l);
  if (h == 0) {
    red_m[wave][n] = m;
    red_l[wave][n] = l;
  }
  __syncthreads();
  float top = red_m[0][n];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, red_m[w][n]);
  const float scale = weight(m, top, a.c);
  if (n < R) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[d][4 * g + r] * scale;
        __builtin_memcpy(red + ((wave * (D / 4) + 8 * d + 2 * g + h) * R + n) * 4, &v, 16);
      }
  }
  float lt = 0.0f;  // of row n
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float mw = red_m[w][n];
    lt += red_l[w][n] * weight(mw, top, a.c);
  }
  __syncthreads();  // all waves have read red_m / red_l
  if (wave == 0 && h == 0) {
    red_m[0][n] = top;
    red_l[0][n] = lt;
  }
  __syncthreads();

  const int elems = R * (D / 4);  // groups of four dims of a row
  const int head0 = kvh * a.G;
  if (ns == 1) {
    for (int i = tid; i < elems; i += 256) {
      const int r = i % R, d4 = i / R;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v += ldg<f32x4>(red + ((w * (D / 4) + d4) * R + r) * 4);
      const int t = r / a.G;
      // a row that sees no key is 0; one whose keys all weigh nothing is not a number
      const float inv = ctx + t < 0 ? 0.0f : 1.0f / red_l[0][r];
      v = ctx + t < 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : v * inv;
      char *o = static_cast<char *>(a.out) +
                ((q0 + t) * a.out_stride + static_cast<int64_t>(head0 + r % a.G) * D) *
                    dtype_bytes(a.out_dtype);
      store4(o, a.out_dtype, d4 * 4, v);
    }
    return;
  }

  // split: this chunk's sums to its slot, (m, l) of its rows behind them
  const rsrc_t part = make_rsrc(a.part, a.part_bytes);
  const uint32_t slot_bytes = lds_rows * (D + 4) * 4;
  const uint32_t first = split.slot * a.Hkv + kvh * split.ns;  // the request's slots
  const uint32_t slot0 = first * slot_bytes;
  const uint32_t slot = slot0 + z * slot_bytes;
  for (int i = tid; i < elems; i += 256) {
    const int r = i % R, d4 = i / R;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += ldg<f32x4>(red + ((w * (D / 4) + d4) * R + r) * 4);
    st_dev4(part, slot + i * 16, v);
  }
  if (tid < R) st_dev4(part, slot + (elems + tid) * 16, f32x4{red_m[0][tid], red_l[0][tid], 0.0f, 0.0f});
  wait_own_memory();
  uint32_t *cnt = a.cnt + first;
  if (!split_arrive_last(cnt, ns)) return;
  // Reads past the L2 take a microsecond: a thread's first sums are on their way
  // while the chunks' weights are formed.
  constexpr int kAtOnce = 24;
  f32x4 v[kAtOnce];
  auto read = [&](int i, int y0) __attribute__((always_inline)) {
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y)
      v[y] = ld_dev4(part, i < elems && y0 + y < ns ? slot0 + (y0 + y) * slot_bytes + i * 16 : kOut);
  };
  read(tid, 0);
  __builtin_amdgcn_sched_barrier(0);
  // [chunk][row] maximum, then weight, and sum: the waves' sums are no longer needed
  float2 *ml = reinterpret_cast<float2 *>(red);
  {
    const int r = tid >> 3, j = tid & 7;  // eight lanes for a row
    float mx = -__builtin_inff(), sum = 0.0f;
    if (r < R) {
      for (int y0 = j; y0 < ns; y0 += 32) {
        f32x4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int y = y0 + 8 * i;
          u[i] = ld_dev4(part, y < ns ? slot0 + y * slot_bytes + (elems + r) * 16 : kOut);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int y = y0 + 8 * i;
          if (y < ns) {
            ml[y * R + r] = make_float2(u[i].x, u[i].y);
            mx = fmaxf(mx, u[i].x);
          }
        }
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      for (int y = j; y < ns; y += 8) {
        const float2 u = ml[y * R + r];
        const float w = weight(u.x, mx, a.c);
        ml[y * R + r].x = w;
        sum += u.y * w;
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor(sum, o);
      if (j == 0) red_l[0][r] = 1.0f / sum;
    }
  }
  __syncthreads();
  for (int i = tid; i < elems; i += 256) {
    const int r = i % R, d4 = i / R, t = r / a.G;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int y0 = 0; y0 < ns; y0 += kAtOnce) {
      if (i != tid || y0) read(i, y0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int y = 0; y < kAtOnce; ++y) o += v[y] * (y0 + y < ns ? ml[(y0 + y) * R + r].x : 0.0f);
    }
    o = ctx + t < 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * red_l[0][r];
    char *to = static_cast<char *>(a.out) +
               ((q0 + t) * a.out_stride + static_cast<int64_t>(head0 + r % a.G) * D) *
                   dtype_bytes(a.out_dtype);
    store4(to, a.out_dtype, d4 * 4, o);
  }
  split_reset(cnt);
}

namespace {
constexpr int kMaxLds = 65536 - 2048;  // what a launch may ask for without more ado

template <int DT, int D>
hipError_t launch_rows(const AttnArgs &a, int max_rows, int items, hipStream_t s) {
  constexpr int row_bytes = kWaves * D * 4;  // LDS of a row: the waves' sums
  if constexpr (row_bytes * kRowsMax > kMaxLds) {
    static std::atomic<uint64_t> done{0};
    if (!dry_run()) {
      const hipError_t e = allow_lds(reinterpret_cast<const void *>(&k_attn_rows<DT, D>),
                                     row_bytes * kRowsMax, done);
      if (e != hipSuccess) return e;
    }
  }
  // the waves' sums; before them the requests, after them the chunks' weights and sums
  int bytes = row_bytes * max_rows;
  if (bytes < a.B * 8) bytes = a.B * 8;
  if (bytes < a.goal * max_rows * 8) bytes = a.goal * max_rows * 8;
  IFX_LAUNCH(k_attn_rows, (DT, D), dim3(a.Hkv * items), dim3(64 * kWaves), bytes, s, a, max_rows);
  return last_error();
}
template <int DT>
hipError_t launch_rows(const AttnArgs &a, int D, int max_rows, int items, hipStream_t s) {
  switch (D) {
    case 64: return launch_rows<DT, 64>(a, max_rows, items, s);
    case 96: return launch_rows<DT, 96>(a, max_rows, items, s);
    case 128: return launch_rows<DT, 128>(a, max_rows, items, s);
    default: return launch_rows<DT, 256>(a, max_rows, items, s);
  }
}
}  // namespace

int attn_rows_max_goal(int max_rows) { return kMaxLds / 8 / max_rows; }

hipError_t launch_attn_rows(const AttnArgs &a, int dtype, int D, int max_rows, int items,
                            hipStream_t s) {
  return dtype == IFX_ATTN_F16 ? launch_rows<IFX_ATTN_F16>(a, D, max_rows, items, s)
                               : launch_rows<IFX_ATTN_BF16>(a, D, max_rows, items, s);
}

}  // namespace ifx
