// kv_plan.hip -- one serving step's block tables, slots, positions and row
// offsets from the requests' lengths, on the device.
//
// With c_b tokens cached and n_b new ones, P tokens a page:
//   held_b = ceil(c_b / P), need_b = ceil((c_b + n_b) / P) - held_b,
//   cu_b = sum_{a < b} n_a, off_b = sum_{a < b} need_a;
// new token t of request b (cu_b <= t < cu_{b+1}) stands at position
// p = c_b + t - cu_b, in page w = p / P of the request: the table's entry if
// w < held_b, else free_pages[free_count - 1 - (off_b + w - held_b)].
//
// Bound by latency: a launch, one dependent read of the lengths, one of the
// tables.  So a single launch does it all: every workgroup scans the B
// lengths itself (two arrays, 32 KB at most, from L2) instead of waiting for
// another to do it, and then places its own span of tokens by a binary search among the
// row offsets in LDS.  A new page's table entry is written by the thread that
// places the page's first token: no thread reads an entry that another
// writes, because entries below held_b are only read.  Measured: 32 decode
// requests 3.1 us, 300 requests with 43000 new tokens 5.8 us.
#include <climits>

#include "ifx_attn.h"

namespace ifx {

namespace {

__device__ __forceinline__ int64_t shfl_up64(int64_t v, int d) {
  const int lo = __shfl_up(static_cast<int>(v), d);
  const int hi = __shfl_up(static_cast<int>(v >> 32), d);
  return (static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo);
}

}  // namespace

// LDS: cu[B + 1], off[B], ctx[B] (int32), then the scan's scratch.
__global__ __launch_bounds__(1024) void k_plan_batch(const PlanArgs a) {
  extern __shared__ int32_t lds[];
  int32_t *cu = lds, *off = cu + a.B + 1, *cx = off + a.B;
  __shared__ int64_t part[2][16];
  __shared__ int64_t base[2];
  __shared__ int flags;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wave = tid >> 6;
  const int sh = a.page_shift, P = 1 << sh;
  if (tid == 0) {
    base[0] = base[1] = 0;
    flags = 0;
  }
  __syncthreads();
  const int avail = min(max(a.free_count[0], 0), a.free_capacity);
  for (int b0 = 0; b0 < a.B; b0 += nt) {
    const int b = b0 + tid;
    int c = 0, n = 0, bad = 0;
    if (b < a.B) {
      c = a.ctx_len[b];
      n = a.new_len[b];
      if (c < 0 || n < 0 || c > INT_MAX - n) {
        bad = IFX_PLAN_BAD_LENGTH;
        c = n = 0;
      }
    }
    const int64_t total = (static_cast<int64_t>(c) + n + P - 1) >> sh;
    if (total > a.table_width) bad |= IFX_PLAN_NARROW;
    int64_t toks = n, need = total - ((static_cast<int64_t>(c) + P - 1) >> sh);
    const int64_t own_t = toks, own_n = need;
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t t = shfl_up64(toks, d), u = shfl_up64(need, d);
      if (lane >= d) {
        toks += t;
        need += u;
      }
    }
    if (lane == 63) {
      part[0][wave] = toks;
      part[1][wave] = need;
    }
    if (bad) atomicOr(&flags, bad);
    __syncthreads();
    int64_t bt = base[0], bn = base[1];
    for (int w = 0; w < wave; ++w) {
      bt += part[0][w];
      bn += part[1][w];
    }
    // saturated: only read where the whole plan fits 31 bits
    if (b < a.B) {
      cu[b] = static_cast<int32_t>(min(bt + toks - own_t, static_cast<int64_t>(INT_MAX)));
      off[b] = static_cast<int32_t>(min(bn + need - own_n, static_cast<int64_t>(INT_MAX)));
      cx[b] = c;
    }
    __syncthreads();
    if (tid == nt - 1) {
      base[0] = bt + toks;
      base[1] = bn + need;
    }
    __syncthreads();
  }
  const int64_t tokens = base[0], taken = base[1];
  int st = flags;
  if (taken > avail) st |= IFX_PLAN_NO_PAGES;
  if (tokens > a.max_tokens) st |= IFX_PLAN_NO_ROOM;
  const int T = st ? 0 : static_cast<int>(tokens);
  if (blockIdx.x == 0) {
    for (int b = tid; b < a.B; b += nt) {
      a.cu_q[b] = st ? 0 : cu[b];
      a.kv_len[b] = a.ctx_len[b] + (st ? 0 : a.new_len[b]);
    }
    if (tid == 0) {
      a.cu_q[a.B] = T;
      a.free_left[0] = st ? a.free_count[0] : avail - static_cast<int>(taken);
      a.status[0] = st;
    }
  }
  const int t0 = blockIdx.x * kPlanTokens;
  const int t1 = min(t0 + kPlanTokens, a.max_tokens);
  for (int t = t0 + tid; t < t1; t += nt) {
    int pos = 0, slot = -1;
    if (t < T) {
      int lo = 0, hi = a.B - 1;  // the last request whose first row is <= t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t)
          lo = mid;
        else
          hi = mid - 1;
      }
      const int c = cx[lo];
      pos = c + (t - cu[lo]);
      const int w = pos >> sh, held = (c + P - 1) >> sh;
      int32_t *entry = a.block_table + static_cast<int64_t>(lo) * a.table_width + w;
      int page;
      if (w < held) {
        page = *entry;
      } else {
        page = a.free_pages[avail - 1 - (off[lo] + w - held)];
        if ((pos & (P - 1)) == 0) *entry = page;
      }
      // a page number that no cache can have gives no slot
      if (page >= 0 && page <= (INT_MAX >> sh)) slot = (page << sh) + (pos & (P - 1));
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
}

hipError_t launch_plan_batch(const PlanArgs &a, hipStream_t s) {
  // one request a thread where a single pass over them is enough
  const int nt = a.B <= 256 ? 256 : 1024;
  const int grid = a.max_tokens > kPlanTokens ? (a.max_tokens + kPlanTokens - 1) / kPlanTokens : 1;
  const size_t lds = sizeof(int32_t) * (3 * static_cast<size_t>(a.B) + 1);
  IFX_LAUNCH0(k_plan_batch, dim3(grid), dim3(nt), lds, s, a);
  return last_error();
}

}  // namespace ifx
