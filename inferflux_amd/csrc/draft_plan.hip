// draft_plan.hip -- positions and masks of trees of drafted tokens, and what a
// batch keeps of them once they are verified.
//
//   mask_i = {i} + mask_parent(i),  position_i = ctx + |mask_i| - 1
//
// Bound by latency: a launch, the reads of the lengths, then of the parents; 2.2 us
// for one tree of 61 nodes and 2.4 for 32 in a row of launches, up to 5 where the
// lengths are read from memory.  A request is a wave, its nodes the
// lanes: the masks of all nodes grow twice as far towards the root with each of
// six exchanges between lanes, where a walk would take a node's depth of them.
#include "ifx_drafts_impl.h"

namespace ifx {

namespace {

constexpr int kTreeWaves = 4;

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
  const uint32_t lo = __shfl(static_cast<int>(v), lane), hi = __shfl(static_cast<int>(v >> 32), lane);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

}  // namespace

__global__ __launch_bounds__(64 * kTreeWaves) void k_plan_tree(const TreeArgs a) {
  const int lane = threadIdx.x & 63;
  const int b = blockIdx.x * kTreeWaves + (threadIdx.x >> 6);
  // rows behind the last request's
  const int end = min(max(a.cu[a.B], 0), a.T);
  for (int t = end + blockIdx.x * blockDim.x + threadIdx.x; t < a.T; t += gridDim.x * blockDim.x) {
    a.positions[t] = 0;
    a.masks[t] = 0;
  }
  if (b >= a.B) return;
  const int r0 = min(max(a.cu[b], 0), a.T), n = max(min(max(a.cu[b + 1], 0), a.T) - r0, 0);
  const int ctx = a.kv_len[b] - n;
  const int parent = lane < n ? a.parents[r0 + lane] : -1;
  const bool has = parent >= 0 && parent < lane;
  uint64_t mask = 1ull << lane;
  int up = has ? parent : lane;  // 2^k nodes towards the root, or where that ends
  bool more = has;
#pragma unroll
  for (int k = 1; k < kMaxNodes; k <<= 1) {
    const uint64_t above = shfl64(mask, up);
    const int far = __shfl(up, up);
    const bool on = __shfl(static_cast<int>(more), up) != 0;
    if (more) {
      mask |= above;
      up = far;
      more = on;
    }
  }
  if (lane < n) {
    a.positions[r0 + lane] = ctx + __popcll(mask) - 1;
    a.masks[r0 + lane] = mask;
  }
  for (int t = kMaxNodes + lane; t < n; t += 64) {
    a.positions[r0 + t] = 0;
    a.masks[r0 + t] = 0;
  }
}

hipError_t launch_plan_tree(const TreeArgs &a, hipStream_t s) {
  IFX_LAUNCH0(k_plan_tree, dim3((a.B + kTreeWaves - 1) / kTreeWaves), dim3(64 * kTreeWaves), 0, s, a);
  return last_error();
}

// One workgroup: a page's place among the free ones depends on how many all
// requests behind its own give back.
__global__ __launch_bounds__(1024) void k_plan_kept(const KeptArgs a) {
  constexpr int kEach = IFX_ATTN_MAX_BATCH / 1024;  // requests of a thread
  __shared__ int64_t part[16];
  __shared__ int given[IFX_ATTN_MAX_BATCH], behind[IFX_ATTN_MAX_BATCH];  // pages of a request, of those behind it
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sh = a.page_shift, P = 1 << sh;
  const int room = a.table_width << sh;
  auto of = [&](int b, int &kept, int &held) {  // tokens kept, pages held
    const int n = max(a.cu[b + 1] - a.cu[b], 0), kv = min(max(a.kv_len[b], 0), room);
    const int take = n ? min(max(a.accepted[b], -1) + 1, n) : 0;
    kept = max(kv - n + take, 0);
    held = (kv + P - 1) >> sh;
    return held - ((kept + P - 1) >> sh);
  };
  int give[kEach];
  int64_t own = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = tid * kEach + i;
    give[i] = 0;
    if (b < a.B) {
      int kept, held;
      give[i] = of(b, kept, held);
      a.ctx_len[b] = kept;
    }
    own += give[i];
  }
  int64_t to = own;  // of the wave's threads up to this one
  for (int d = 1; d < 64; d <<= 1) {
    const int lo = __shfl_up(static_cast<int>(to), d), hi = __shfl_up(static_cast<int>(to >> 32), d);
    if (lane >= d) to += (static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo);
  }
  if (lane == 63) part[wave] = to;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) to += part[w];
    total += part[w];
  }
  const int count = min(max(a.free_count[0], 0), a.free_capacity);
  const bool fits = total <= a.free_capacity - count;
  if (tid == 0) {
    a.free_left[0] = fits ? count + static_cast<int>(total) : a.free_count[0];
    a.status[0] = fits ? 0 : IFX_KEPT_NO_SPACE;
  }
  if (!fits) return;
  to -= own;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    to += give[i];
    given[tid * kEach + i] = give[i];
    behind[tid * kEach + i] = static_cast<int>(total - to);
  }
  __syncthreads();
  // the last request's last page first; a wave takes a request
  for (int b = wave; b < a.B; b += 16) {
    const int n = given[b];
    if (!n) continue;
    int kept, held;
    of(b, kept, held);
    for (int i = lane; i < n; i += 64)
      a.free_pages[count + behind[b] + i] = a.table[static_cast<int64_t>(b) * a.table_width + held - 1 - i];
  }
}

hipError_t launch_plan_kept(const KeptArgs &a, hipStream_t s) {
  IFX_LAUNCH0(k_plan_kept, dim3(1), dim3(1024), 0, s, a);
  return last_error();
}

}  // namespace ifx
