// rope_append.hip -- rotates the new tokens' Q and K and writes K and V into
// the paged cache (layout: ifx_attention.h).
//
//   y_i = x_i cos(a) - x_j sin(a),  y_j = x_j cos(a) + x_i sin(a),
//   a = position * inv_freq
//
// Bound by HBM: every value is read once and written once.  The angle is
// formed in fp64 as turns and reduced to half a turn there (a position of
// 10^5 would leave an fp32 angle 10^-2 off), its sine and cosine in fp32: one
// pair per position and frequency, shared by all heads through LDS.
#include "ifx_attn.h"

namespace ifx {

namespace {

template <int SRC>
__device__ __forceinline__ void load8(const void *p, int64_t at, float (&x)[8]) {
  if constexpr (SRC == IFX_ATTN_F32) {
    const float *f = static_cast<const float *>(p) + at;
    const f32x4 a = ldg<f32x4>(f), b = ldg<f32x4>(f + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const u32x4 u = ldg<u32x4>(static_cast<const uint16_t *>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = SRC == IFX_ATTN_F16 ? F16::value(u[i] & 0xFFFFu) : BF16::value(u[i] & 0xFFFFu);
      x[2 * i + 1] = SRC == IFX_ATTN_F16 ? F16::value(u[i] >> 16) : BF16::value(u[i] >> 16);
    }
  }
}

template <class T>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7])};
}

template <int SRC>
__device__ __forceinline__ float load1(const void *p, int64_t at) {
  if constexpr (SRC == IFX_ATTN_F32) return static_cast<const float *>(p)[at];
  const uint32_t u = static_cast<const uint16_t *>(p)[at];
  return SRC == IFX_ATTN_F16 ? F16::value(u) : BF16::value(u);
}

}  // namespace

// A workgroup takes NTOK consecutive tokens.  Units of Q and K are pieces of 8
// values (and their partners' piece where pairs lie half a rotation apart);
// K's units run over the tokens first, so that neighbouring lanes write
// neighbouring 16-byte pieces of the cache.  V's pieces hold 8 tokens of one
// dim, so a lane gathers the tokens of one piece: the token that begins a run
// of consecutive slots within a piece writes the whole run, from whichever
// workgroup holds it, with one 16-byte store where the run fills the piece.
template <int DT, int SRC, int NTOK>
__global__ __launch_bounds__(256) void k_rope_append(const AppendArgs a) {
  using T = Elem<DT>;
  __shared__ float2 turn[NTOK * 128];
  __shared__ int slot_of[NTOK + 8];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * NTOK;
  const int half = a.rot_dim >> 1, pieces = a.D >> 3, sh = a.page_shift, P = 1 << sh;
  // slots of the tokens, of the one before them (entry 0) and of those a run
  // can reach behind them
  for (int i = tid; i < NTOK + 8; i += 256) {
    const int t = t0 - 1 + i;
    const int s = t >= 0 && t < a.T ? a.slots[t] : -1;
    slot_of[i] = static_cast<uint32_t>(s) < static_cast<uint32_t>(a.num_slots) ? s : -1;
  }
  for (int i = tid; i < NTOK * half; i += 256) {
    const int t = t0 + i / half;
    if (t < a.T) {
      const double turns = a.positions[t] * a.inv_freq[i % half] * 0.15915494309189533577;
      const float x = static_cast<float>(2.0 * (turns - rint(turns)));
      float sn, cs;
      sincospif(x, &sn, &cs);
      turn[i] = make_float2(cs, sn);
    }
  }
  __syncthreads();

  // Q and K: unit = (token, head, piece); a piece below rot_dim / 2 takes its
  // partner along, the partner's own unit does nothing
  const int heads = a.Hq + a.Hkv;
  const int units = NTOK * heads * pieces;
  for (int u = tid; u < units; u += 256) {
    int t, head, pc;
    if (u < NTOK * a.Hq * pieces) {  // Q: the row's order
      pc = u % pieces;
      head = u / pieces % a.Hq;
      t = u / (pieces * a.Hq);
    } else {  // K: tokens first
      const int w = u - NTOK * a.Hq * pieces;
      t = w % NTOK;
      pc = w / NTOK % pieces;
      head = a.Hq + w / (NTOK * pieces);
    }
    const int slot = slot_of[t + 1];
    if (slot < 0) continue;
    const bool is_q = head < a.Hq;
    const int hh = is_q ? head : head - a.Hq;
    const void *src = is_q ? a.q : a.k;
    const int64_t at = (t0 + t) * (is_q ? a.q_stride : a.k_stride) +
                       static_cast<int64_t>(hh) * a.D + pc * 8;
    const float2 *tw = turn + t * half;
    float x[8], y[8];
    bool two = false;
    if (a.interleaved || pc * 8 >= a.rot_dim) {
      load8<SRC>(src, at, x);
      if (pc * 8 < a.rot_dim) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 w = tw[pc * 4 + i];
          const float p = x[2 * i], r = x[2 * i + 1];
          x[2 * i] = p * w.x - r * w.y;
          x[2 * i + 1] = r * w.x + p * w.y;
        }
      }
    } else {
      if (pc * 8 >= half) continue;
      load8<SRC>(src, at, x);
      load8<SRC>(src, at + half, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 w = tw[pc * 8 + i];
        const float p = x[i], r = y[i];
        x[i] = p * w.x - r * w.y;
        y[i] = r * w.x + p * w.y;
      }
      two = true;
    }
    if (is_q) {
      uint16_t *o = static_cast<uint16_t *>(a.q_out) + (t0 + t) * a.q_out_stride +
                    static_cast<int64_t>(hh) * a.D + pc * 8;
      const u32x4 px = pack8<T>(x);
      __builtin_memcpy(o, &px, 16);
      if (two) {
        const u32x4 py = pack8<T>(y);
        __builtin_memcpy(o + half, &py, 16);
      }
    } else {
      const int64_t chunk = static_cast<int64_t>(slot >> sh) * a.Hkv + hh;
      u32x4 *o = static_cast<u32x4 *>(a.k_cache) + (chunk * pieces << sh) + (slot & (P - 1));
      o[pc << sh] = pack8<T>(x);
      if (two) o[(pc + (half >> 3)) << sh] = pack8<T>(y);
    }
  }

  // V: unit = (run, head, dim), lanes along the dims
  for (int t = 0; t < NTOK; ++t) {
    const int slot = slot_of[t + 1];
    if (slot < 0) continue;
    const int before = slot_of[t];
    if (before >= 0 && before + 1 == slot && (slot & 7) != 0) continue;  // within a run
    int n = 1;
    while (((slot + n) & 7) != 0 && slot_of[t + 1 + n] == slot + n) ++n;
    const int64_t page = slot >> sh;
    const int in_page = slot & (P - 1);
    for (int i = tid; i < a.Hkv * a.D; i += 256) {
      const int hh = i / a.D, dim = i - hh * a.D;
      uint16_t *o = static_cast<uint16_t *>(a.v_cache) +
                    ((((page * a.Hkv + hh) << sh) + (in_page & ~7)) * a.D + dim * 8) +
                    (in_page & 7);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = e < n ? load1<SRC>(a.v, (t0 + t + e) * a.v_stride + i) : 0.0f;
      const u32x4 p = pack8<T>(x);
      if (n == 8) {
        *reinterpret_cast<u32x4 *>(o) = p;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) o[e] = static_cast<uint16_t>(p[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
}

namespace {
template <int DT, int SRC>
void launch(const AppendArgs &a, hipStream_t s) {
  if (a.T >= 2048) {
    IFX_LAUNCH(k_rope_append, (DT, SRC, 8), dim3((a.T + 7) / 8), dim3(256), 0, s, a);
  } else {
    IFX_LAUNCH(k_rope_append, (DT, SRC, 1), dim3(a.T), dim3(256), 0, s, a);
  }
}
template <int DT>
void launch(const AppendArgs &a, int src_dtype, hipStream_t s) {
  switch (src_dtype) {
    case IFX_ATTN_F32: return launch<DT, IFX_ATTN_F32>(a, s);
    case IFX_ATTN_F16: return launch<DT, IFX_ATTN_F16>(a, s);
    default: return launch<DT, IFX_ATTN_BF16>(a, s);
  }
}
}  // namespace

hipError_t launch_rope_append(const AppendArgs &a, int src_dtype, int cache_dtype, hipStream_t s) {
  if (cache_dtype == IFX_ATTN_F16)
    launch<IFX_ATTN_F16>(a, src_dtype, s);
  else
    launch<IFX_ATTN_BF16>(a, src_dtype, s);
  return last_error();
}

}  // namespace ifx
