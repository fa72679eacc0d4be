// attention_api.hip -- the C entry points of include/ifx_attention.h and
// include/ifx_attention_q8.h, and the attention's of include/ifx_drafts.h:
// validation, the split of keys over workgroups, and the launches.
#include <climits>
#include <cmath>

#include "ifx_attn_q8.h"
#include "ifx_drafts_impl.h"
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

// Geometry and pointers of an append; sets its number of slots.
int append_args(AppendArgs &a, int64_t num_pages) {
  const int sh = a.page_shift;
  if (sh < 0 || num_pages < 1 || num_pages > (INT_MAX >> sh)) return IFX_BAD_GEOMETRY;
  if (a.T < 0 || a.T > (1 << 27) - 8 || a.Hq < 1 || a.Hkv < 1 || a.Hq > 65536 || a.Hkv > 65536 ||
      a.D < 8 || a.D > 256 || a.D % 8 || a.rot_dim < 0 || a.rot_dim > a.D || a.rot_dim % 16)
    return IFX_BAD_GEOMETRY;
  const int64_t qn = static_cast<int64_t>(a.Hq) * a.D, kn = static_cast<int64_t>(a.Hkv) * a.D;
  if (a.q_stride < qn || a.k_stride < kn || a.v_stride < kn || a.q_out_stride < qn)
    return IFX_BAD_GEOMETRY;
  if (a.T == 0) return IFX_OK;
  if (!a.q || !a.k || !a.v || !a.slots || !a.q_out || !a.k_cache || !a.v_cache ||
      (a.rot_dim && (!a.positions || !a.inv_freq)))
    return IFX_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & 15)
    return IFX_BAD_GEOMETRY;
  a.num_slots = static_cast<int>(num_pages << sh);
  return IFX_OK;
}

// Positions are below 2^30: a window as wide is none, and position - window
// stays within 32 bits, also of rows before the first key (above -2^30).
int window_of(int window) { return window < (1 << 30) ? window : 0; }

// Split sums: units (a request's or row tile's key/value head) that can be
// split, their counters at the start of the workspace.  The counters' place is
// the same for every shape, as one workspace serves calls of many shapes and
// only they have to be zero between calls.
constexpr int kMaxUnits = kSplitUnits;
constexpr int64_t kCntBytes = kSplitCntBytes;

struct PagedPlan {
  bool rows;         // attn_rows, else attn_tile
  int row_slots;     // attn_rows: rows of a workgroup
  int blocks;        // attn_rows: of max_q rows
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
// Blocks of rows: as many workgroups as CUs.  us with 256 / 512 / 1024, 3000 keys:
// 16 / 2 heads, 160 rows 16.7 with each, 512 rows 17.7/18.7/18.8, 8-bit 16.9/18.7/18.6;
// 40 / 8 heads, 150 rows, 8-bit 16.0/18.4/18.6; 12000 keys, 16 / 2 heads, 160 rows 26.2
// with each, 512 rows 34.7/33.9/34.0.
//
// Fewer where the split sums would not fit the largest workspace.
//
// Trees over the 16-bit cache go to attn_rows with up to 32 rows for a few units
// (requests times key/value heads), 24 for some, else 16.  us with attn_tile /
// attn_rows, 3000 keys, heads of 128, the caches from memory:
//   40 / 8 heads, 20 rows  2 requests 23.4/17.5, 4 25.2/22.6, 8 38.7/36.4, 16 50.7/54.6
//                 30 rows  1 22.2/17.3, 2 23.3/19.0, 4 25.1/24.9, 8 39.3/39.9, 16 51.9/58.4
//   16 / 2 heads, 24 rows  8 23.5/18.2, 32 39.3/31.2
// Over the 8-bit cache all of up to 32 rows go to attn_rows; from 17 on many of them
// would be sooner done in attn_tile's way for few rows (32 requests of 30 rows, 40 / 8
// heads, 43 against 59).
//
// More rows as blocks of 32 of attn_rows, where attn_tile's workgroups would leave
// much of the chip idle (both read the keys once for each block or tile): up to 112
// blocks, over the 8-bit cache 256 if a unit has no more than 8.  us with attn_tile /
// in blocks, 3000 keys, by blocks of all units:
//   16-bit  1 head of K    640 rows   20 29.5/17.0,  80 31.1/24.1;  1024 128 31.9/42.7
//           16 / 2 heads   160 rows   10 29.2/16.7,  40 30.8/20.8;  512 128 32.6/34.0
//           40 / 8 heads   100 rows   32 29.7/18.9,  64 31.5/23.9, 128 33.2/35.2
//                          200 rows   56 30.1/22.5, 112 31.9/34.4, 224 45.4/53.8
//   8-bit   1 head of K   1024 rows   32 32.6/16.4, 128 34.5/36.8;  640 320 48.5/51.7
//           16 / 2 heads   160 rows   10 32.1/16.0,  40 33.3/17.9, 160 45.5/37.8
//           40 / 8 heads   100 rows   32 31.6/17.2, 128 33.8/26.6, 512 56.1/57.2
//                          200 rows   56 32.6/18.7, 224 45.6/37.2, 896 82.6/100.9
//                          640 rows  160 50.8/71.3 (7000 keys)
enum PagedKind { kPaged16, kTree16, kPaged8 };
PagedPlan plan_paged(PagedKind kind, int B, int T, int Hq, int Hkv, int D, int max_q, int max_kv) {
  PagedPlan p{};
  const int G = Hq / Hkv;
  const int64_t rows = static_cast<int64_t>(max_q) * G, units = static_cast<int64_t>(B) * Hkv;
  p.rows = rows <= (kind != kTree16 ? kRowsMax : units <= 16 ? kRowsMax : units <= 64 ? 24 : 16);
  const int64_t each = (rows + kRowsMax - 1) / kRowsMax;  // blocks of a unit
  const bool blocks = !p.rows && kind != kPaged16 && rows > kRowsMax &&
                      (units * each <= 112 || (kind == kPaged8 && each <= 8 && units * each <= 256));
  p.rows |= blocks;
  // row tiles, stages of the longest request that a split must have, bytes of a slot
  const int64_t tiles = p.rows && !blocks
                            ? B
                            : static_cast<int64_t>(T) * G / (blocks ? kRowsMax : attn_tile_rows(D)) + B;
  const int unit = p.rows ? kRowKeys : attn_tile_min_keys();
  p.blocks = static_cast<int>(each);
  p.row_slots = static_cast<int>(rows < kRowsMax ? rows : kRowsMax);
  const int64_t slot = p.rows ? p.row_slots * (D + 4) * 4 : attn_tile_slot_bytes(D);
  const int all = blocks ? 256 : p.rows ? 1024 : D == 256 ? 256 : D == 64 ? 768 : 512;
  int64_t goal = all / Hkv;
  const int64_t use = tiles * ((static_cast<int64_t>(max_kv) + unit - 1) / unit);
  const int64_t fit = (IFX_ATTN_WORKSPACE_BYTES - kCntBytes) / slot / Hkv;
  if (goal > use) goal = use;
  if (goal > fit) goal = fit;
  if (goal > kMaxUnits / Hkv) goal = kMaxUnits / Hkv;
  if (p.rows && goal > attn_rows_max_goal(p.row_slots))
    goal = attn_rows_max_goal(p.row_slots);
  if (max_kv <= (p.rows ? unit : 2 * unit - kTileKeys)) goal = 0;  // one chunk each
  p.goal = static_cast<int>(goal);
  p.items = static_cast<int>(tiles + goal);
  p.bytes = goal ? kCntBytes + goal * Hkv * slot : 0;
  return p;
}

// masks: the nodes that rows of trees see, or null.  scales: of the 8-bit cache,
// null for the 16-bit one.
int attn_paged(const void *q, int64_t q_stride, int dtype, const void *k_cache,
               const void *v_cache, const void *scales, int64_t num_pages, int page_size,
               const int32_t *block_table, int table_width, const int32_t *cu_q,
               const int32_t *kv_len, const uint64_t *masks, int B, int T, int Hq, int Hkv, int D,
               int max_q, int max_kv, float scale, int window, void *out, int64_t out_stride,
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
  const PagedPlan p = plan_paged(scales ? kPaged8 : masks ? kTree16 : kPaged16, B, T, Hq, Hkv, D,
                                 max_q, max_kv);
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
  a.masks = masks, a.scales = static_cast<const uint32_t *>(scales), a.q_dtype = dtype;
  a.c = scale * kLog2e;
  a.goal = p.goal;
  if (p.bytes) {
    a.cnt = static_cast<uint32_t *>(workspace);
    a.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + kCntBytes);
    a.part_bytes = static_cast<uint32_t>(p.bytes - kCntBytes);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (scales)
    return status_of(p.rows ? launch_attn_rows_q8(a, D, p.row_slots, p.blocks, p.items, s)
                            : launch_attn_tile_q8(a, D, p.items, s));
  if (p.rows) return status_of(launch_attn_rows(a, dtype, D, p.row_slots, p.blocks, p.items, s));
  return status_of(launch_attn_tile(a, dtype, D, true, p.items, s));
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
  AppendArgs a{q, k, v, q_stride, k_stride, v_stride, q_out_stride, positions, slots, inv_freq,
               q_out, k_cache, v_cache, rot_dim, interleaved != 0, T, Hq, Hkv, D,
               page_shift_of(page_size), 0};
  const int rc = append_args(a, num_pages);
  if (rc || T == 0) return rc;
  return status_of(launch_rope_append(a, src_dtype, cache_dtype, static_cast<hipStream_t>(stream)));
}

int ifx_rope_append_q8(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                       const void *v, int64_t v_stride, int src_dtype, const int32_t *positions,
                       const int32_t *slots, const double *inv_freq, int rot_dim, int interleaved,
                       int T, int Hq, int Hkv, int D, void *q_out, int64_t q_out_stride,
                       int q_dtype, void *k_cache, void *v_cache, void *scales, int64_t num_pages,
                       int page_size, void *stream) {
  if (!is_out(src_dtype) || !is_elem(q_dtype)) return IFX_UNSUPPORTED_TYPE;
  AppendQ8Args b{{q, k, v, q_stride, k_stride, v_stride, q_out_stride, positions, slots,
                  inv_freq, q_out, k_cache, v_cache, rot_dim, interleaved != 0, T, Hq, Hkv, D,
                  page_shift_of(page_size), 0},
                 static_cast<uint32_t *>(scales), 0};
  if (D % 32) return IFX_BAD_GEOMETRY;
  const int rc = append_args(b.a, num_pages);
  if (rc || T == 0) return rc;
  if (!scales) return IFX_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(scales) & 15) return IFX_BAD_GEOMETRY;
  return status_of(launch_rope_append_q8(b, src_dtype, q_dtype, static_cast<hipStream_t>(stream)));
}

int ifx_read_rows_q8(const void *k_cache, const void *v_cache, const void *scales,
                     int64_t num_pages, int page_size, const int32_t *slots, int N, int Hkv, int D,
                     void *k_out, int64_t k_stride, void *v_out, int64_t v_stride, int out_dtype,
                     void *stream) {
  if (!is_out(out_dtype)) return IFX_UNSUPPORTED_TYPE;
  const int sh = page_shift_of(page_size);
  const int64_t row = static_cast<int64_t>(Hkv) * D;
  if (sh < 0 || num_pages < 1 || num_pages > (INT_MAX >> sh) || N < 0 || N >= (1 << 27) ||
      Hkv < 1 || Hkv > 65536 || D < 32 || D > 256 || D % 32 || k_stride < row || v_stride < row)
    return IFX_BAD_GEOMETRY;
  if (N == 0) return IFX_OK;
  if (!k_cache || !v_cache || !scales || !slots || !k_out || !v_out) return IFX_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(scales)) & 15)
    return IFX_BAD_GEOMETRY;
  const ReadArgs a{k_cache, v_cache, static_cast<const uint32_t *>(scales), slots, k_out, v_out,
                   k_stride, v_stride, N, Hkv, D, sh, static_cast<int>(num_pages << sh)};
  return status_of(launch_read_rows_q8(a, out_dtype, static_cast<hipStream_t>(stream)));
}

int64_t ifx_attn_paged_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int max_q,
                                       int max_kv) {
  if (!heads_ok(B, T, Hq, Hkv, D) || max_q < 1 || max_kv < 1) return 0;
  return plan_paged(kPaged16, B, T, Hq, Hkv, D, max_q, max_kv).bytes;
}

int ifx_attn_paged(const void *q, int64_t q_stride, int dtype, const void *k_cache,
                   const void *v_cache, int64_t num_pages, int page_size,
                   const int32_t *block_table, int table_width, const int32_t *cu_q,
                   const int32_t *kv_len, int B, int T, int Hq, int Hkv, int D, int max_q,
                   int max_kv, float scale, int window, void *out, int64_t out_stride,
                   int out_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  return attn_paged(q, q_stride, dtype, k_cache, v_cache, nullptr, num_pages, page_size, block_table,
                    table_width, cu_q, kv_len, nullptr, B, T, Hq, Hkv, D, max_q, max_kv, scale,
                    window, out, out_stride, out_dtype, workspace, workspace_bytes, stream);
}

int64_t ifx_attn_tree_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int max_q,
                                      int max_kv) {
  if (!heads_ok(B, T, Hq, Hkv, D) || max_q < 1 || max_q > IFX_TREE_MAX_NODES || max_kv < 1) return 0;
  return plan_paged(kTree16, B, T, Hq, Hkv, D, max_q, max_kv).bytes;
}

int ifx_attn_tree(const void *q, int64_t q_stride, int dtype, const void *k_cache,
                  const void *v_cache, int64_t num_pages, int page_size,
                  const int32_t *block_table, int table_width, const int32_t *cu_q,
                  const int32_t *kv_len, const uint64_t *masks, int B, int T, int Hq, int Hkv,
                  int D, int max_q, int max_kv, float scale, void *out, int64_t out_stride,
                  int out_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  if (max_q > IFX_TREE_MAX_NODES) return IFX_BAD_GEOMETRY;
  if (T && !masks) return IFX_NULL_POINTER;
  return attn_paged(q, q_stride, dtype, k_cache, v_cache, nullptr, num_pages, page_size, block_table,
                    table_width, cu_q, kv_len, masks, B, T, Hq, Hkv, D, max_q, max_kv, scale, 0,
                    out, out_stride, out_dtype, workspace, workspace_bytes, stream);
}

int64_t ifx_attn_paged_q8_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int max_q,
                                          int max_kv) {
  if (!heads_ok(B, T, Hq, Hkv, D) || max_q < 1 || max_kv < 1) return 0;
  return plan_paged(kPaged8, B, T, Hq, Hkv, D, max_q, max_kv).bytes;
}

int ifx_attn_paged_q8(const void *q, int64_t q_stride, int q_dtype, const void *k_cache,
                      const void *v_cache, const void *scales, int64_t num_pages, int page_size,
                      const int32_t *block_table, int table_width, const int32_t *cu_q,
                      const int32_t *kv_len, const uint64_t *masks, int B, int T, int Hq, int Hkv,
                      int D, int max_q, int max_kv, float scale, int window, void *out,
                      int64_t out_stride, int out_dtype, void *workspace, int64_t workspace_bytes,
                      void *stream) {
  if (masks && (window || max_q > IFX_TREE_MAX_NODES)) return IFX_BAD_GEOMETRY;
  if (T && !scales) return IFX_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(scales) & 15) return IFX_BAD_GEOMETRY;
  return attn_paged(q, q_stride, q_dtype, k_cache, v_cache, scales, num_pages, page_size,
                    block_table, table_width, cu_q, kv_len, masks, B, T, Hq, Hkv, D, max_q, max_kv,
                    scale, window, out, out_stride, out_dtype, workspace, workspace_bytes, stream);
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
