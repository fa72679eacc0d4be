// attention_api.hip -- the C entry points of include/ifx_attention.h:
// validation, the split of keys over workgroups, and the launches.
#include <climits>
#include <cmath>

#include "ifx_attn.h"
#include "ifx_qgemm.h"

namespace ifx {

hipError_t allow_lds(const void *kernel, int bytes, std::atomic<uint64_t> &done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
  e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace ifx

namespace {

using namespace ifx;

int status_of(hipError_t e) { return e == hipSuccess ? IFX_OK : -static_cast<int>(e); }

// log2 of a page size the cache can have, else -1.
int page_shift_of(int page_size) {
  for (int sh = 4; sh <= 8; ++sh)
    if (page_size == 1 << sh) return sh;
  return -1;
}

bool is_elem(int dtype) { return dtype == IFX_ATTN_F16 || dtype == IFX_ATTN_BF16; }
bool is_out(int dtype) { return dtype == IFX_ATTN_F32 || is_elem(dtype); }

// Head counts, head size and rows that the attention kernels take: the rows of
// a key/value head (T x group) and the grids stay within 31 bits.
bool heads_ok(int B, int T, int Hq, int Hkv, int D) {
  if (B < 1 || B > IFX_ATTN_MAX_BATCH || T < 0 || Hkv < 1 || Hq < Hkv || Hq % Hkv) return false;
  if (D != 64 && D != 96 && D != 128 && D != 256) return false;
  if (static_cast<int64_t>(Hkv) * D >= (1 << 22)) return false;  // bytes of a page: 32 bits
  const int64_t rows = static_cast<int64_t>(T) * (Hq / Hkv);
  return rows < (1 << 30) && (rows / 32 + B) * Hkv < (1 << 23);
}

// scale log2 e is what the kernels multiply by.
bool scale_ok(float scale) { return scale > 0.0f && std::isfinite(scale * kLog2e); }

// Positions are below 2^30: a window as wide is none, and position - window
// stays within 32 bits, also of rows before the first key (above -2^30).
int window_of(int window) { return window < (1 << 30) ? window : 0; }

// Split sums: units (a request's or row tile's key/value head) that can be
// split, their counters at the start of the workspace.  The counters' place is
// the same for every shape, as one workspace serves calls of many shapes and
// only they have to be zero between calls.
constexpr int kMaxUnits = 8192;
constexpr int64_t kCntBytes = kMaxUnits * 4;

struct PagedPlan {
  bool rows;         // attn_rows, else attn_tile
  int goal, items;   // AttnArgs; workgroups of a key/value head
  int64_t bytes;     // of workspace
};

// How ifx_attn_paged's keys are split over workgroups: about `goal` work items
// for each key/value head, whose lengths the workgroups find (find_item).
//
// attn_tile: as many as are resident, two a CU (D = 64: three, D = 256: one).
// A chunk of 512 tokens over 7430 keys, 40 / 8 heads of 128: 143 us with 256,
// 115 with 384, 95 with 512, 107 with 768, 101 with 1000.
//
// attn_rows: two rounds of those that are resident at two a CU (D = 256: four
// rounds at one), as requests differ in length.  32 requests of 531 to 22591
// keys, 40 / 8 heads of 128: 162 us with 512, 150 with 768, 148 with 1024, 150
// with 1536, 153 with 2048.
//
// Fewer where the split sums would not fit the largest workspace.
PagedPlan plan_paged(int B, int T, int Hq, int Hkv, int D, int max_q, int max_kv) {
  PagedPlan p{};
  const int G = Hq / Hkv;
  const int64_t rows = static_cast<int64_t>(max_q) * G;
  p.rows = rows <= kRowsMax;
  // row tiles, stages of the longest request that a split must have, bytes of a slot
  const int64_t tiles = p.rows ? B : static_cast<int64_t>(T) * G / attn_tile_rows(D) + B;
  const int unit = p.rows ? kRowKeys : attn_tile_min_keys();
  const int64_t slot = p.rows ? rows * (D + 4) * 4 : attn_tile_slot_bytes(D);
  const int all = p.rows ? 1024 : D == 256 ? 256 : D == 64 ? 768 : 512;
  int64_t goal = all / Hkv;
  const int64_t use = tiles * ((static_cast<int64_t>(max_kv) + unit - 1) / unit);
  const int64_t fit = (IFX_ATTN_WORKSPACE_BYTES - kCntBytes) / slot / Hkv;
  if (goal > use) goal = use;
  if (goal > fit) goal = fit;
  if (goal > kMaxUnits / Hkv) goal = kMaxUnits / Hkv;
  if (p.rows && goal > attn_rows_max_goal(static_cast<int>(rows)))
    goal = attn_rows_max_goal(static_cast<int>(rows));
  if (max_kv <= (p.rows ? unit : 2 * unit - kTileKeys)) goal = 0;  // one chunk each
  p.goal = static_cast<int>(goal);
  p.items = static_cast<int>(tiles + goal);
  p.bytes = goal ? kCntBytes + goal * Hkv * slot : 0;
  return p;
}

}  // namespace

extern "C" {

int ifx_plan_batch(const int32_t *ctx_len, const int32_t *new_len, int32_t *block_table,
                   int table_width, const int32_t *free_pages, int free_capacity,
                   const int32_t *free_count, int page_size, int B, int max_tokens, int32_t *cu_q,
                   int32_t *kv_len, int32_t *positions, int32_t *slots, int32_t *free_left,
                   int32_t *status, void *stream) {
  const int sh = page_shift_of(page_size);
  if (sh < 0 || B < 1 || B > IFX_ATTN_MAX_BATCH || table_width < 1 || free_capacity < 0 ||
      max_tokens < 0 || max_tokens > (1 << 30))
    return IFX_BAD_GEOMETRY;
  if (!ctx_len || !new_len || !block_table || !free_count || !cu_q || !kv_len || !free_left ||
      !status || (free_capacity && !free_pages) || (max_tokens && (!positions || !slots)))
    return IFX_NULL_POINTER;
  // every workgroup reads the inputs: an output in their place would be read
  // by some after others have written it
  const void *in[] = {ctx_len, new_len, free_count, free_pages};
  const void *out[] = {cu_q, kv_len, positions, slots, free_left, status};
  for (const void *o : out)
    for (const void *i : in)
      if (o && o == i) return IFX_BAD_GEOMETRY;
  const PlanArgs a{ctx_len, new_len, block_table, free_pages, free_count, cu_q, kv_len, positions,
                   slots, free_left, status, table_width, free_capacity, sh, B, max_tokens};
  return status_of(launch_plan_batch(a, static_cast<hipStream_t>(stream)));
}

int ifx_rope_append(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                    const void *v, int64_t v_stride, int src_dtype, const int32_t *positions,
                    const int32_t *slots, const double *inv_freq, int rot_dim, int interleaved,
                    int T, int Hq, int Hkv, int D, void *q_out, int64_t q_out_stride,
                    void *k_cache, void *v_cache, int cache_dtype, int64_t num_pages,
                    int page_size, void *stream) {
  if (!is_out(src_dtype) || !is_elem(cache_dtype)) return IFX_UNSUPPORTED_TYPE;
  const int sh = page_shift_of(page_size);
  if (sh < 0 || num_pages < 1 || num_pages > (INT_MAX >> sh)) return IFX_BAD_GEOMETRY;
  if (T < 0 || T > (1 << 27) - 8 || Hq < 1 || Hkv < 1 || Hq > 65536 || Hkv > 65536 || D < 8 ||
      D > 256 || D % 8 || rot_dim < 0 || rot_dim > D || rot_dim % 16)
    return IFX_BAD_GEOMETRY;
  const int64_t qn = static_cast<int64_t>(Hq) * D, kn = static_cast<int64_t>(Hkv) * D;
  if (q_stride < qn || k_stride < kn || v_stride < kn || q_out_stride < qn) return IFX_BAD_GEOMETRY;
  if (T == 0) return IFX_OK;
  if (!q || !k || !v || !slots || !q_out || !k_cache || !v_cache ||
      (rot_dim && (!positions || !inv_freq)))
    return IFX_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15)
    return IFX_BAD_GEOMETRY;
  const AppendArgs a{q, k, v, q_stride, k_stride, v_stride, q_out_stride, positions, slots,
                     inv_freq, q_out, k_cache, v_cache, rot_dim, interleaved != 0, T, Hq, Hkv, D,
                     sh, static_cast<int>(num_pages << sh)};
  return status_of(launch_rope_append(a, src_dtype, cache_dtype, static_cast<hipStream_t>(stream)));
}

int64_t ifx_attn_paged_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int max_q,
                                       int max_kv) {
  if (!heads_ok(B, T, Hq, Hkv, D) || max_q < 1 || max_kv < 1) return 0;
  return plan_paged(B, T, Hq, Hkv, D, max_q, max_kv).bytes;
}

int ifx_attn_paged(const void *q, int64_t q_stride, int dtype, const void *k_cache,
                   const void *v_cache, int64_t num_pages, int page_size,
                   const int32_t *block_table, int table_width, const int32_t *cu_q,
                   const int32_t *kv_len, int B, int T, int Hq, int Hkv, int D, int max_q,
                   int max_kv, float scale, int window, void *out, int64_t out_stride,
                   int out_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  if (!is_elem(dtype) || !is_out(out_dtype)) return IFX_UNSUPPORTED_TYPE;
  const int sh = page_shift_of(page_size);
  if (sh < 0 || num_pages < 1 || num_pages > (INT_MAX >> sh) || table_width < 1 ||
      table_width > ((1 << 30) >> sh))  // positions and the stages behind them fit an int
    return IFX_BAD_GEOMETRY;
  if (!heads_ok(B, T, Hq, Hkv, D) || max_q < 1 || max_kv < 1 || window < 0 ||
      !scale_ok(scale))
    return IFX_BAD_GEOMETRY;
  const int64_t qn = static_cast<int64_t>(Hq) * D;
  if (q_stride < qn || out_stride < qn) return IFX_BAD_GEOMETRY;
  if (T == 0) return IFX_OK;
  if (!q || !k_cache || !v_cache || !block_table || !cu_q || !kv_len || !out)
    return IFX_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15)
    return IFX_BAD_GEOMETRY;
  const PagedPlan p = plan_paged(B, T, Hq, Hkv, D, max_q, max_kv);
  if (p.bytes) {
    if (!workspace) return IFX_NULL_POINTER;
    if (workspace_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255))
      return IFX_BAD_GEOMETRY;
  }
  AttnArgs a{};
  a.q = q, a.k = k_cache, a.v = v_cache, a.out = out;
  a.q_stride = q_stride, a.out_stride = out_stride;
  a.table = block_table, a.cu = cu_q, a.kv_len = kv_len;
  a.num_pages = num_pages, a.table_width = table_width, a.page_shift = sh;
  a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv;
  a.causal = 1, a.window = window_of(window), a.out_dtype = out_dtype;
  a.c = scale * kLog2e;
  a.goal = p.goal;
  if (p.bytes) {
    a.cnt = static_cast<uint32_t *>(workspace);
    a.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + kCntBytes);
    a.part_bytes = static_cast<uint32_t>(p.bytes - kCntBytes);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.rows) return status_of(launch_attn_rows(a, dtype, D, max_q * a.G, p.items, s));
  return status_of(launch_attn_tile(a, dtype, D, true, p.items, s));
}

int ifx_attn_prompt(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                    const void *v, int64_t v_stride, int dtype, const int32_t *cu_len, int B,
                    int T, int Hq, int Hkv, int D, int max_len, int causal, int window,
                    float scale, void *out, int64_t out_stride, int out_dtype, void *stream) {
  if (!is_elem(dtype) || !is_out(out_dtype)) return IFX_UNSUPPORTED_TYPE;
  if (!heads_ok(B, T, Hq, Hkv, D) || max_len < 1 || window < 0 || (window > 0 && !causal) ||
      !scale_ok(scale))
    return IFX_BAD_GEOMETRY;
  const int64_t qn = static_cast<int64_t>(Hq) * D, kn = static_cast<int64_t>(Hkv) * D;
  // 64 rows of K or V are addressed by 32-bit offsets
  if (q_stride < qn || k_stride < kn || v_stride < kn || out_stride < qn ||
      k_stride >= (1 << 23) || v_stride >= (1 << 23))
    return IFX_BAD_GEOMETRY;
  if (T == 0) return IFX_OK;
  if (!q || !k || !v || !cu_len || !out) return IFX_NULL_POINTER;
  AttnArgs a{};
  a.q = q, a.k = k, a.v = v, a.out = out;
  a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride, a.out_stride = out_stride;
  a.cu = cu_len;
  a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv;
  a.causal = causal != 0, a.window = window_of(window), a.out_dtype = out_dtype;
  a.c = scale * kLog2e;
  const int tiles = static_cast<int>(static_cast<int64_t>(T) * a.G / attn_tile_rows(D)) + B;
  return status_of(launch_attn_tile(a, dtype, D, false, tiles, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
