// keep_path.hip -- moves the K and V of the drafted nodes that a request keeps
// behind the tokens that were in its cache.
//
//   token ctx + i <- node path[i], 0 < i <= accepted
//
// Bound by latency: a few tokens' rows, 2.7 us for one request of 61 nodes, 2 heads
// of 128, 4.3 for 32 requests and 8 heads (0.9 MB).  The lengths, then the table, then the
// rows, whose reads are on their way eight nodes at a time.  A thread has one
// piece of K or one dim of V and moves it for all nodes in their order: as
// path[i] >= i grows with i, a place that it writes is not read after that, and
// no other thread touches its piece.
#include "ifx_drafts_impl.h"

namespace ifx {

// E: values of a 16-byte piece, 8 of 16 bits or 16 of 8.
template <int E>
__global__ __launch_bounds__(256) void k_keep_path(const KeepArgs a) {
  using V = typename std::conditional<E == 8, uint16_t, uint8_t>::type;
  constexpr int kAtOnce = 8;
  __shared__ int from[kMaxNodes], to[kMaxNodes];  // slots; from = -1: nothing moves
  const int tid = threadIdx.x, b = blockIdx.x / a.Hkv, head = blockIdx.x - b * a.Hkv;
  const int sh = a.page_shift, P = 1 << sh;
  const int r0 = min(max(a.cu[b], 0), a.T), rows = max(min(max(a.cu[b + 1], 0), a.T) - r0, 0);
  const int n = min(rows, a.max_q), moves = min(a.accepted[b], n - 1);
  if (moves <= 0) return;
  if (tid <= moves) {
    const int ctx = a.kv_len[b] - rows, node = a.path[r0 + tid];
    const int32_t *table = a.table + static_cast<int64_t>(b) * a.table_width;
    auto slot = [&](int64_t token) -> int {
      if (token < 0 || token >= static_cast<int64_t>(a.table_width) << sh) return -1;
      const int page = table[token >> sh];
      if (page < 0 || page >= a.num_pages) return -1;
      return (page << sh) + static_cast<int>(token & (P - 1));
    };
    const int src = node > tid && node < n ? slot(static_cast<int64_t>(ctx) + node) : -1;
    const int dst = slot(static_cast<int64_t>(ctx) + tid);
    from[tid] = dst < 0 || tid == 0 ? -1 : src;
    to[tid] = dst;
  }
  __syncthreads();
  const int pieces = a.D / E;
  // moves one value of type T: at(slot) is its address
  auto move = [&](auto *base, auto at) {
    using T = typename std::remove_pointer<decltype(base)>::type;
    for (int i0 = 1; i0 <= moves; i0 += kAtOnce) {
      T v[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        if (i0 + i <= moves && from[i0 + i] >= 0) v[i] = base[at(from[i0 + i])];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        if (i0 + i <= moves && from[i0 + i] >= 0) base[at(to[i0 + i])] = v[i];
    }
  };
  auto block = [&](int slot) { return static_cast<int64_t>(slot >> sh) * a.Hkv + head; };
  for (int u = tid; u < a.D + pieces + (E == 16); u += 256) {
    if (u < a.D) {
      move(static_cast<V *>(a.v), [&](int slot) {
        const int t = slot & (P - 1);
        return ((block(slot) << sh) + (t & ~(E - 1))) * a.D + u * E + (t & (E - 1));
      });
    } else if (u < a.D + pieces) {
      move(static_cast<u32x4 *>(a.k), [&](int slot) {
        return ((block(slot) * pieces + (u - a.D)) << sh) + (slot & (P - 1));
      });
    } else {
      move(static_cast<uint32_t *>(a.scales), [&](int slot) {
        return (block(slot) << sh) + (slot & (P - 1));
      });
    }
  }
}

hipError_t launch_keep_path(const KeepArgs &a, int elem_bytes, hipStream_t s) {
  if (elem_bytes == 2)
    IFX_LAUNCH(k_keep_path, (8), dim3(a.B * a.Hkv), dim3(256), 0, s, a);
  else
    IFX_LAUNCH(k_keep_path, (16), dim3(a.B * a.Hkv), dim3(256), 0, s, a);
  return last_error();
}

}  // namespace ifx
