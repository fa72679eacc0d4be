// verify_drafts.hip -- which drafted nodes the target's probabilities accept,
// and the token drawn behind them.
//
//   without the drafter's probabilities, from node i with u uniform: to the
//   first child c with u < sum of p_i over the children up to c; w = p_i
//   without the children's tokens
//   with them (a chain): on where u q_i(x) < p_i(x); w = max(p_i - q_i, 0)
//   token = the smallest v with w_0 + ... + w_v > u' sum(w)
//
// Bound by latency for few requests, by HBM for many: one row of p (and of q)
// a request, 0.6 MB of 32 bits for 151936 tokens, and the walk before it, whose
// reads depend on each other only through the tokens.  So a single launch does
// it all: rows are cut into chunks, a workgroup each, and every wave walks for
// itself, the nodes' probabilities gathered by its lanes at once.  A chunk's
// sum goes to the workspace; the last workgroup of a request to finish finds
// the chunk that the token is in, and the token by reading that chunk again.
//
// Sums are 64 bits, added in an order that does not depend on who is last.  In
// 32 bits a row's 10^5 sums are off by as much as the tokens between them
// weigh, and the token drawn would depend on the split.
#include "ifx_drafts_impl.h"

namespace ifx {

namespace {

constexpr int kThreads = 256;
constexpr int kStep = kThreads * 4;  // values that a workgroup reads at a time
constexpr int kAhead = 4;            // such reads on their way
constexpr int kAtOnce = 4;           // and where the token is looked for

// Four values of a row from `at` on.
template <int DT>
__device__ __forceinline__ f32x4 read4(const void *row, int at) {
  if constexpr (DT == IFX_ATTN_F32) return ldg<f32x4>(static_cast<const float *>(row) + at);
  const u32x2 u = ldg<u32x2>(static_cast<const uint16_t *>(row) + at);
  using T = Elem<DT == IFX_ATTN_F32 ? IFX_ATTN_F16 : DT>;
  return f32x4{T::value(u.x & 0xFFFFu), T::value(u.x >> 16), T::value(u.y & 0xFFFFu), T::value(u.y >> 16)};
}
// Negative values and NaN are 0.
__device__ __forceinline__ f32x4 clean(f32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = v[i] > 0.0f ? v[i] : 0.0f;
  return v;
}
// The same, and 0 past the row's end.
template <int DT>
__device__ __forceinline__ f32x4 probs4(const void *row, int at, int V) {
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (at + 3 < V) {
    v = read4<DT>(row, at);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < V) {
        if constexpr (DT == IFX_ATTN_F32)
          v[i] = static_cast<const float *>(row)[at + i];
        else
          v[i] = Elem<DT>::value(static_cast<const uint16_t *>(row)[at + i]);
      }
  }
  return clean(v);
}
template <int DT>
__device__ __forceinline__ float prob(const void *row, int at) {
  float v;
  if constexpr (DT == IFX_ATTN_F32)
    v = static_cast<const float *>(row)[at];
  else
    v = Elem<DT>::value(static_cast<const uint16_t *>(row)[at]);
  return v > 0.0f ? v : 0.0f;
}
template <int DT>
__device__ __forceinline__ const void *row_of(const void *p, int64_t stride, int row) {
  return static_cast<const char *>(p) + row * stride * (DT == IFX_ATTN_F32 ? 4 : 2);
}

__device__ __forceinline__ double lane64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(b), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(b >> 32), lane);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
// Inclusive sums over the lanes, as wave_scan's, of 64 bits.
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_moved(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = dpp<CTRL, ROWS>(0u, static_cast<uint32_t>(b));
  const uint32_t hi = dpp<CTRL, ROWS>(0u, static_cast<uint32_t>(b >> 32));
  return v + __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ double scan64(double v) {
  v = add_moved<0x111, 0xF>(v);
  v = add_moved<0x112, 0xF>(v);
  v = add_moved<0x114, 0xF>(v);
  v = add_moved<0x118, 0xF>(v);
  v = add_moved<0x142, 0xA>(v);
  return add_moved<0x143, 0xC>(v);
}

// The workgroup's threads in order hold weights of `mine` each: the first at
// which their sum passes share * total + target, or else the last that holds any;
// -1 if none does.  before: the sum of those before it.
struct Place {
  int thread;
  bool passed;
  double before, total;
};
__device__ __forceinline__ Place find_place(double mine, double share, double target, double *sums,
                                            int *found) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const double to = scan64(mine);
  if (lane == 63) sums[wave] = to;
  if (tid < 2) found[tid] = tid ? -1 : INT_MAX;
  __syncthreads();
  double before = 0.0, total = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w == wave) before = total;
    total += sums[w];
  }
  target += share * total;
  const bool over = mine > 0.0 && before + to > target, any = mine > 0.0;
  const uint64_t o = __ballot(over), s = __ballot(any);
  if (lane == 0) {
    if (o) atomicMin(&found[0], 64 * wave + __builtin_ctzll(o));
    if (s) atomicMax(&found[1], 64 * wave + 63 - __builtin_clzll(s));
  }
  __syncthreads();
  const bool passed = found[0] != INT_MAX;
  const int at = passed ? found[0] : found[1];
  if (tid == at) sums[kThreads / 64] = before + (to - mine);
  __syncthreads();
  return {at, passed, sums[kThreads / 64], total};
}

}  // namespace

template <int DT>
__global__ __launch_bounds__(kThreads, 4) void k_verify(const VerifyArgs a) {
  __shared__ double sums[kThreads / 64 + 1], whole[kThreads / 64];
  __shared__ int found[2];  // find_place's, which clears it without waiting for who still reads it
  __shared__ int place_token;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.chunks, z = blockIdx.x - b * a.chunks;
  const int r0 = min(max(a.cu[b], 0), a.T), rows = max(min(max(a.cu[b + 1], 0), a.T) - r0, 0);
  const int n = min(rows, a.max_q);
  if (n == 0) {
    if (z == 0 && tid == 0) a.accepted[b] = -1;
    return;
  }

  // ---- the walk: lane j is node j
  const bool is = lane < n;
  const int token = is ? a.tokens[r0 + lane] : -1;
  int parent = lane - 1;
  if (a.parents) parent = is ? a.parents[r0 + lane] : -1;
  if (!is || parent < 0 || parent >= lane) parent = -1;
  const float u = is ? a.accept_u[r0 + lane] : 0.0f;
  const bool known = parent >= 0 && token >= 0 && token < a.V;
  const float p = known ? prob<DT>(row_of<DT>(a.target, a.target_stride, r0 + parent), token) : 0.0f;
  uint64_t walked = 1, children = 0;  // children: of the last node walked
  int last = 0;
  if (a.drafter) {
    const float q = known ? prob<DT>(row_of<DT>(a.drafter, a.drafter_stride, r0 + parent), token) : 0.0f;
    const float up = __shfl(u, lane > 0 ? lane - 1 : 0);
    const uint64_t taken =
        __ballot(known && static_cast<double>(up) * static_cast<double>(q) < static_cast<double>(p)) >> 1;
    last = min(static_cast<int>(__builtin_ctzll(~taken)), n - 1);
    walked = last == 63 ? ~0ull : (2ull << last) - 1;
    children = last + 1 < n;
  } else {
    while (true) {
      children = __ballot(parent == last);
      const double ul = static_cast<double>(
          __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, u), last)));
      int to = -1;
      double sum = 0.0;
      for (uint64_t left = children; left; left &= left - 1) {
        const int c = __builtin_ctzll(left);
        const int x = __builtin_amdgcn_readlane(token, c);
        if (__ballot(token == x) & children & ((1ull << c) - 1)) continue;
        sum += lane64(static_cast<double>(p), c);
        if (ul < sum) {
          to = c;
          break;
        }
      }
      if (to < 0) break;
      last = to;
      walked |= 1ull << to;
    }
  }

  // ---- the chunk's share of what the next token is drawn from
  const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
  const void *pr = row_of<DT>(a.target, a.target_stride, r0 + last);
  const void *qr = nullptr;
  if (a.drafter && children) qr = row_of<DT>(a.drafter, a.drafter_stride, r0 + last);
  const uint64_t gone = a.drafter ? 0 : children;
  // weights of four tokens from `at` on; near: the children with tokens of the chunk
  auto weights = [&](f32x4 v, f32x4 q, int at, uint64_t near,
                     double (&w)[4]) __attribute__((always_inline)) {
    if (qr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = fmax(static_cast<double>(v[i]) - static_cast<double>(q[i]), 0.0);
      return;
    }
    for (uint64_t left = near; left; left &= left - 1) {
      const int x = __builtin_amdgcn_readlane(token, __builtin_ctzll(left)) - at;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = x == i ? 0.0f : v[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = static_cast<double>(v[i]);
  };
  auto near_of = [&](int from) {
    return gone & __ballot(token >= from && token - from < a.chunk);
  };
  {
    const int from = z * a.chunk, to = min(from + a.chunk, a.V);
    const uint64_t near = near_of(from);
    double sum = 0.0, all = 0.0;
    auto add = [&](f32x4 v, f32x4 q, int at) __attribute__((always_inline)) {
      double w[4];
      weights(v, q, at, near, w);
      sum += (w[0] + w[1]) + (w[2] + w[3]);
      all += (static_cast<double>(v[0]) + static_cast<double>(v[1])) +
             (static_cast<double>(v[2]) + static_cast<double>(v[3]));
    };
    int at = from + tid * 4;
    for (; at - tid * 4 + kAhead * kStep <= to; at += kAhead * kStep) {  // several reads on their way
      f32x4 v[kAhead], q[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) v[i] = read4<DT>(pr, at + i * kStep);
      if (qr) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) q[i] = read4<DT>(qr, at + i * kStep);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) add(clean(v[i]), qr ? clean(q[i]) : none, at + i * kStep);
    }
    for (; at < to; at += kStep)
      add(probs4<DT>(pr, at, a.V), qr ? probs4<DT>(qr, at, a.V) : none, at);
    sum = scan64(sum), all = scan64(all);
    if (lane == 63) {
      sums[wave] = sum;
      whole[wave] = all;
    }
    __syncthreads();
    if (tid == 0) {
      double s = 0.0, t = 0.0;
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w) s += sums[w], t += whole[w];
      double *out = a.part + (static_cast<int64_t>(b) * a.chunks + z) * 2;
      __hip_atomic_store(out, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(out + 1, t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  wait_own_memory();
  if (!split_arrive_last(a.cnt + b, a.chunks)) return;

  // ---- the request's last workgroup: the chunk, the token, the outputs
  double sum = 0.0, all = 0.0;
  if (tid < a.chunks) {
    double *in = a.part + (static_cast<int64_t>(b) * a.chunks + tid) * 2;
    sum = __hip_atomic_load(in, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    all = __hip_atomic_load(in + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const bool some = __syncthreads_or(sum > 0.0);
  const double mine = some ? sum : all;
  const double share = fmax(static_cast<double>(a.sample_u[b]), 0.0);
  const Place chunk = find_place(mine, share, 0.0, sums, found);
  int drawn = -1;
  if (chunk.thread >= 0) {
    const int from = chunk.thread * a.chunk, to = min(from + a.chunk, a.V);
    const uint64_t near = some ? near_of(from) : 0;
    if (!some) qr = nullptr;
    const double rest = fmax(share * chunk.total - chunk.before, 0.0);
    double run = 0.0;
    bool passed = false;
    // 16 tokens a thread, one behind the other, read all at once
    for (int base = from; base < to && !passed; base += kThreads * 4 * kAtOnce) {
      const int at = base + tid * 4 * kAtOnce;
      f32x4 v[kAtOnce], q[kAtOnce];
      if (base + kThreads * 4 * kAtOnce <= a.V) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) v[i] = read4<DT>(pr, at + 4 * i);
        if (qr) {
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) q[i] = read4<DT>(qr, at + 4 * i);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) v[i] = clean(v[i]), q[i] = qr ? clean(q[i]) : none;
      } else {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          v[i] = probs4<DT>(pr, at + 4 * i, a.V);
          q[i] = qr ? probs4<DT>(qr, at + 4 * i, a.V) : none;
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)  // the next chunk's, whose children `near` has not
        if (at + 4 * i >= to) v[i] = q[i] = none;
      double own = 0.0;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        double w[4];
        weights(v[i], q[i], at + 4 * i, near, w);
        own += (w[0] + w[1]) + (w[2] + w[3]);
      }
      const Place place = find_place(own, 0.0, rest - run, sums, found);
      if (tid == place.thread) {
        double sum = place.before;
        int token = -1;
        bool done = false;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          double w[4];
          weights(v[i], q[i], at + 4 * i, near, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sum += w[j];
            if (!done && w[j] > 0.0) {
              token = at + 4 * i + j;
              done = sum > rest - run;
            }
          }
        }
        place_token = token;
      }
      __syncthreads();
      // rounding apart the sum passes `rest` in one of them; else the last weight's
      if (place.thread >= 0) drawn = place_token;
      passed = place.passed;
      run += place.total;
    }
  }
  if (wave == 0) {
    const int accepted = __popcll(walked) - 1;
    if (lane == 0) a.accepted[b] = accepted;
    // row i: the i-th node walked, and the token of the one behind it
    int node = -1, next = -1;
    uint64_t left = walked;
    for (int i = 0; i <= accepted; ++i, left &= left - 1) {
      const int c = __builtin_ctzll(left);
      const int x = __builtin_amdgcn_readlane(token, c);
      if (lane == i) node = c;
      if (lane == i - 1) next = x;
    }
    if (lane == accepted) next = drawn;
    for (int t = lane; t < rows; t += 64) {
      a.path[r0 + t] = t < 64 ? node : -1;
      a.emitted[r0 + t] = t < 64 ? next : -1;
    }
  }
  split_reset(a.cnt + b);
}

// Chunks of a row: enough workgroups for four a CU, of whole rounds of kAhead
// steps, as many as a workgroup has threads at most.  us for 1 / 4 / 16 / 32 / 48 /
// 64 rows of 151936 values:
//   for 512 workgroups   7.9 / 9.3 / 13.9 / 16.8 / 20.7 / 24.8
//       1024             7.9 / 9.3 / 15.0 / 15.9 / 18.4 / 21.1
//       1024, of steps   9.0 / 14.2 / 17.7 / 19.1 / 18.5 / 21.7
void verify_split(int B, int V, int *chunks, int *chunk) {
  constexpr int kRound = kAhead * kStep;
  const int64_t rounds = (static_cast<int64_t>(V) + kRound - 1) / kRound;
  int64_t want = 1024 / B;
  if (want < 1) want = 1;
  if (want > kThreads) want = kThreads;
  const int64_t each = (rounds + want - 1) / want;
  *chunk = static_cast<int>(each * kRound);
  *chunks = static_cast<int>((rounds + each - 1) / each);
}

hipError_t launch_verify(const VerifyArgs &a, int prob_dtype, hipStream_t s) {
  const dim3 grid(a.B * a.chunks), block(kThreads);
  if (prob_dtype == IFX_ATTN_F32)
    IFX_LAUNCH(k_verify, (IFX_ATTN_F32), grid, block, 0, s, a);
  else if (prob_dtype == IFX_ATTN_F16)
    IFX_LAUNCH(k_verify, (IFX_ATTN_F16), grid, block, 0, s, a);
  else
    IFX_LAUNCH(k_verify, (IFX_ATTN_BF16), grid, block, 0, s, a);
  return last_error();
}

}  // namespace ifx
