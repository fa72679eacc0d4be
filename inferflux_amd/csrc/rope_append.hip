// rope_append.hip -- rotates the new tokens' Q and K and writes K and V into
// the paged cache (layout: ifx_attention.h).
//
//   y_i = x_i cos(a) - x_j sin(a),  y_j = x_j cos(a) + x_i sin(a),
//   a = position * inv_freq
//
// Every value is read once and written once, and at prompts' sizes HBM would be
// the bound; what holds it up is that a workgroup's first rows are asked for
// only behind its slots, positions, angles and a barrier, with two units a
// thread to hide that, and that lanes of neighbouring pieces read their angles
// from the same LDS banks (15 cycles an instruction).  The angle is
// formed in fp64 as turns and reduced to half a turn there (a position of
// 10^5 would leave an fp32 angle 10^-2 off), its sine and cosine in fp32: one
// pair per position and frequency, shared by all heads through LDS.
//
// Measured: 5299 tokens of 40 query and 8 key/value heads of 128, fp16 (152 MB):
// 43 us from memory, 3.5 TB/s, and 27 where the rows are still in the caches
// (vector units busy for 39 % of the time); 8 tokens of 16 and 2 heads, fp32: a
// kernel of 3.9 us.
#include "ifx_rope.h"

namespace ifx {

// A workgroup takes NTOK consecutive tokens, and of them a part: K and V
// (blockIdx.y 0) or some of Q's units.  Units of Q and K are pieces of 8 values
// (and their partners' piece where pairs lie half a rotation apart); K's units
// run over the tokens first, so that neighbouring lanes write neighbouring
// 16-byte pieces of the cache.  V's pieces hold 8 tokens of one dim, so a lane
// gathers the tokens of two dims' pieces: the token that begins a run of
// consecutive slots within a piece writes the whole run, from whichever
// workgroup holds it, with 16-byte stores where the run fills the piece.
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

  // Q and K: unit = (token, head, c): piece c and its partner, or behind the
  // pairs a piece alone
  const bool q_part = blockIdx.y > 0;
  const int heads = q_part ? a.Hq : a.Hkv;
  const int pairs = a.interleaved ? 0 : half >> 3, per_head = pieces - pairs;
  const int units = NTOK * heads * per_head;
  const int share = q_part ? (units + gridDim.y - 2) / (gridDim.y - 1) : units;
  const int u_begin = q_part ? (blockIdx.y - 1) * share : 0, u_end = min(u_begin + share, units);
  const float per_head_inv = 1.0f / per_head, heads_inv = 1.0f / heads;
  for (int u = u_begin + tid; u < u_end; u += 256) {
    const int v = q_part ? u : u / NTOK, w = quotient(v, per_head, per_head_inv);
    const int c = v - w * per_head;
    const int t = q_part ? quotient(w, heads, heads_inv) : u % NTOK;
    const int head = q_part ? w - t * heads : w, pc = c < pairs ? c : c + pairs;
    const int slot = slot_of[t + 1];
    if (slot < 0) continue;
    const bool two = c < pairs;
    Raw8<SRC> lo, hi;
    const int64_t at = (t0 + t) * (q_part ? a.q_stride : a.k_stride) +
                       static_cast<int64_t>(head) * a.D + pc * 8;
    lo.load(q_part ? a.q : a.k, at);
    if (two) hi.load(q_part ? a.q : a.k, at + half);
    const float2 *tw = turn + t * half;
    float x[8], y[8];
    lo.values(x);
    if (two) {
      hi.values(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 w = tw[pc * 8 + i];
        const float p = x[i], r = y[i];
        x[i] = p * w.x - r * w.y;
        y[i] = r * w.x + p * w.y;
      }
    } else if (pc * 8 < a.rot_dim) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 w = tw[pc * 4 + i];
        const float p = x[2 * i], r = x[2 * i + 1];
        x[2 * i] = p * w.x - r * w.y;
        x[2 * i + 1] = r * w.x + p * w.y;
      }
    }
    if (q_part) {
      uint16_t *o = static_cast<uint16_t *>(a.q_out) + (t0 + t) * a.q_out_stride +
                    static_cast<int64_t>(head) * a.D + pc * 8;
      const u32x4 px = pack8<T>(x);
      __builtin_memcpy(o, &px, 16);
      if (two) {
        const u32x4 py = pack8<T>(y);
        __builtin_memcpy(o + half, &py, 16);
      }
    } else {
      const int64_t chunk = static_cast<int64_t>(slot >> sh) * a.Hkv + head;
      u32x4 *o = static_cast<u32x4 *>(a.k_cache) + (chunk * pieces << sh) + (slot & (P - 1));
      o[pc << sh] = pack8<T>(x);
      if (two) o[(pc + pairs) << sh] = pack8<T>(y);
    }
  }
  if (q_part) return;

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
    for (int i = tid * 2; i < a.Hkv * a.D; i += 512) {
      const int hh = i / a.D, dim = i - hh * a.D;
      uint16_t *o = static_cast<uint16_t *>(a.v_cache) +
                    ((((page * a.Hkv + hh) << sh) + (in_page & ~7)) * a.D + dim * 8) +
                    (in_page & 7);
      float x[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 v = e < n ? load2<SRC>(a.v, (t0 + t + e) * a.v_stride + i) : make_float2(0.0f, 0.0f);
        x[e] = v.x, y[e] = v.y;
      }
      const u32x4 p = pack8<T>(x), r = pack8<T>(y);
      if (n == 8) {
        *reinterpret_cast<u32x4 *>(o) = p;
        *reinterpret_cast<u32x4 *>(o + 8) = r;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) {
            o[e] = static_cast<uint16_t>(p[e >> 1] >> (16 * (e & 1)));
            o[8 + e] = static_cast<uint16_t>(r[e >> 1] >> (16 * (e & 1)));
          }
      }
    }
  }
}

namespace {
template <int DT, int SRC>
void launch(const AppendArgs &a, hipStream_t s) {
  // One token a workgroup hides its chain of dependent steps best, eight share
  // K's and V's cache lines.  us with one / eight, rows in the caches, heads of 128:
  //   tokens               32       256       512       1024       2048       5299
  //   16 / 2, fp16     4.4/5.9   4.8/6.1   5.4/6.2   6.4/6.8  10.0/7.5  20.5/13.6
  //   16 / 2, fp32     3.9/5.3   4.3/5.5   4.8/5.6   6.0/6.1   9.6/7.1  21.7/15.5
  //   40 / 8, fp16     5.6/8.0   6.6/8.4   9.5/9.2  11.9/11.2 19.6/14.3 44.8/25.4
  //   40 / 8, fp32     4.4/6.8   5.5/7.2   7.8/7.8  13.3/9.5  25.2/15.4 59.1/35.3
  // They meet at 500 to 1200 tokens; from 2048 on eight are faster by a quarter
  // at least for all of these.
  if (a.T >= 2048) {
    // 5299 tokens as above, from memory: 54 us with one part for all, 45 with 2 for
    // Q, 43 with 5
    IFX_LAUNCH(k_rope_append, (DT, SRC, 8), dim3((a.T + 7) / 8, 6), dim3(256), 0, s, a);
  } else {
    IFX_LAUNCH(k_rope_append, (DT, SRC, 1), dim3(a.T, 2), dim3(256), 0, s, a);
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
