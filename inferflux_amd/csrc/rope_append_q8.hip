// rope_append_q8.hip -- rotates the new tokens' Q and K, writes K and V into the
// 8-bit paged cache (layout: ifx_attention_q8.h), and reads tokens back.
//
//   y_i = x_i cos(a) - x_j sin(a),  y_j = x_j cos(a) + x_i sin(a),
//   a = position * inv_freq;  s = the smallest bf16 >= max |y| / 127,
//   code_i = rint(y_i / s)
//
// K is rotated in fp64, and a code is that of the exact value but for fp64's last
// bits: an fp32 angle's error of 1e-7 would move one code in 30000, and a value read
// back by a whole step.  The quotients are first taken in fp32, by a reciprocal,
// which is off by less than 1e-4 of a step; only a wave in which a value of K lies
// within that of a border divides in fp64, and what is left of V after the nearest
// code is exact in fp32.
//
// Few tokens: bound by latency, 4.6 us for 8 tokens of 16 / 2 heads of 128, the
// read of them 3.3.  Many: 5299 tokens of fp16, 40 / 8 heads of 128, take 33 us for
// 130 MB and the read of them 11 us for 44 MB, where a copy of as many bytes takes
// 25 and 8.4: what keeps the append from that is V's transposed bytes and K's
// fp64, angles among it.
#include "ifx_attn_q8.h"
#include "ifx_rope.h"

namespace ifx {

namespace {

// Bits of the smallest bf16 s with 127 s >= top (15 significant bits: exact in
// fp32); of NaN where top is not finite.
__device__ __forceinline__ uint32_t scale_bits(float top) {
  if (!(top <= 3.4028234e38f)) return 0x7FC0u;
  uint32_t s = __builtin_bit_cast(uint32_t, top / 127.0f) >> 16;
  if (__builtin_bit_cast(float, s << 16) * 127.0f < top) ++s;
  return s;
}

// The largest over the 8, 16 or 32 lanes that share a row.
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, dpp<0xB1>(0u, v));   // quad_perm [1,0,3,2]
  v = max(v, dpp<0x4E>(0u, v));   // quad_perm [2,3,0,1]
  v = max(v, dpp<0x141>(0u, v));  // row_half_mirror
  if constexpr (LANES > 8) v = max(v, dpp<0x140>(0u, v));  // row_mirror
  if constexpr (LANES > 16) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
  return v;
}
template <int LANES>
__device__ __forceinline__ double row_max(double v) {
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) v = fmax(v, __shfl_xor(v, d));
  return v;
}

// A dim's codes of N tokens to their slots: those that follow each other within a
// piece together, in stores as wide as their places are aligned.  The slots are
// the same for all lanes, and so are the branches.
template <int N>
__device__ __forceinline__ void store_tokens(uint8_t *dims, int D, int Hkv, int head, int sh,
                                             const int *slot_of, const uint8_t *codes) {
  const uint64_t all = *reinterpret_cast<const uint64_t *>(codes);
  for (int t = 0; t < N;) {
    const int slot = __builtin_amdgcn_readfirstlane(slot_of[t]);
    if (slot < 0) {
      ++t;
      continue;
    }
    const int tok = slot & ((1 << sh) - 1);
    uint8_t *o = dims + (((static_cast<int64_t>(slot >> sh) * Hkv + head) << sh) + (tok & ~15)) * D + (tok & 15);
    auto follow = [&](int n) {  // whether n tokens from t on lie there, one behind the other
      bool yes = t + n <= N && (slot & (n - 1)) == 0;
      for (int i = 1; i < n && yes; ++i) yes = __builtin_amdgcn_readfirstlane(slot_of[t + i]) == slot + i;
      return yes;
    };
    const uint64_t v = all >> (8 * t);
    if (follow(8)) {
      *reinterpret_cast<uint64_t *>(o) = v;
      t += 8;
    } else if (follow(4)) {
      *reinterpret_cast<uint32_t *>(o) = static_cast<uint32_t>(v);
      t += 4;
    } else if (follow(2)) {
      *reinterpret_cast<uint16_t *>(o) = static_cast<uint16_t>(v);
      t += 2;
    } else {
      *o = static_cast<uint8_t>(v);
      ++t;
    }
  }
}

// Scales below are divided by in fp64: their reciprocals pass fp32's range.
constexpr float kLeast = 0x1p-100f;

}  // namespace

// A workgroup takes NTOK consecutive tokens, and of them a part: some of K's
// heads (blockIdx.y below kv_parts), of V's (the next kv_parts) or of Q's units,
// pieces of 8 values (and their partners' where pairs lie half a rotation apart).
// A row of K or V is shared by LANES lanes, a piece of 8 values each.
template <int DT, int SRC, int LANES, int NTOK>
__global__ __launch_bounds__(256) void k_rope_append_q8(const AppendQ8Args args) {
  using T = Elem<DT>;
  const AppendArgs &a = args.a;
  // cosine and sine: [token][i % 8][i / 8], so that neighbouring pieces' are neighbours
  __shared__ union {
    float2 q[NTOK * 128];
    double2 k[NTOK * 128];
  } turn;
  __shared__ int slot_of[NTOK];
  const int tid = threadIdx.x, t0 = blockIdx.x * NTOK;
  const int half = a.rot_dim >> 1, angles = half >> 3;  // half: a multiple of 8
  const int pieces = a.D >> 3, sh = a.page_shift, P = 1 << sh;
  const int kv_parts = args.kv_parts, y = blockIdx.y;
  const bool q_part = y >= 2 * kv_parts, is_v = !q_part && y >= kv_parts;
  if (tid < NTOK) {
    const int t = t0 + tid, s = t < a.T ? a.slots[t] : -1;
    slot_of[tid] = static_cast<uint32_t>(s) < static_cast<uint32_t>(a.num_slots) ? s : -1;
  }
  for (int i = tid; i < NTOK * half && !is_v; i += 256) {
    const int tok = i / half, t = t0 + tok, f = i - tok * half;
    if (t < a.T) {
      const double turns = a.positions[t] * a.inv_freq[f] * 0.15915494309189533577;
      const double x = 2.0 * (turns - rint(turns));
      const int to = tok * half + (f & 7) * angles + (f >> 3);
      if (q_part) {
        float sn, cs;
        sincospif(static_cast<float>(x), &sn, &cs);
        turn.q[to] = make_float2(cs, sn);
      } else {
        double sn, cs;
        sincospi(x, &sn, &cs);
        turn.k[to] = make_double2(cs, sn);
      }
    }
  }
  __syncthreads();

  if (q_part) {
    const int pairs = a.interleaved ? 0 : angles, per_head = pieces - pairs;
    const int units = NTOK * a.Hq * per_head, parts = gridDim.y - 2 * kv_parts;
    const int share = (units + parts - 1) / parts;
    const int u0 = (y - 2 * kv_parts) * share, u1 = min(u0 + share, units);
    const float per_head_inv = 1.0f / per_head, heads_inv = 1.0f / a.Hq;
    for (int u = u0 + tid; u < u1; u += 256) {
      const int w = quotient(u, per_head, per_head_inv), c = u - w * per_head;
      const int t = quotient(w, a.Hq, heads_inv), head = w - t * a.Hq;
      if (slot_of[t] < 0) continue;
      const int pc = c < pairs ? c : c + pairs;
      const bool two = c < pairs;
      Raw8<SRC> lo, hi;
      const int64_t at = (t0 + t) * a.q_stride + static_cast<int64_t>(head) * a.D + pc * 8;
      lo.load(a.q, at);
      if (two) hi.load(a.q, at + half);
      const float2 *tw = turn.q + t * half;
      float x[8], y[8];
      lo.values(x);
      uint16_t *o = static_cast<uint16_t *>(a.q_out) + (t0 + t) * a.q_out_stride +
                    static_cast<int64_t>(head) * a.D + pc * 8;
      if (two) {
        hi.values(y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 r = tw[i * angles + pc];
          const float p = x[i], s = y[i];
          x[i] = p * r.x - s * r.y;
          y[i] = s * r.x + p * r.y;
        }
        const u32x4 py = pack8<T>(y);
        __builtin_memcpy(o + half, &py, 16);
      } else if (pc * 8 < a.rot_dim) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 r = tw[((pc * 4 + i) & 7) * angles + (pc >> 1)];
          const float p = x[2 * i], s = x[2 * i + 1];
          x[2 * i] = p * r.x - s * r.y;
          x[2 * i + 1] = s * r.x + p * r.y;
        }
      }
      const u32x4 px = pack8<T>(x);
      __builtin_memcpy(o, &px, 16);
    }
    return;
  }

  // K or V: row = (token, head), tokens fastest.  All lanes take as many turns, as
  // rows are reduced across them.
  constexpr int kRows = 256 / LANES, kHeads = NTOK > 1 ? kRows / NTOK : 1;
  uint8_t *by_dim = reinterpret_cast<uint8_t *>(&turn);  // V: [head][dim][token], of kHeads
  const int c = tid & (LANES - 1), rows = NTOK * a.Hkv;
  const int part_rows = ((rows + kRows - 1) / kRows + kv_parts - 1) / kv_parts * kRows;  // whole turns
  const int from = (is_v ? y - kv_parts : y) * part_rows, until = min(from + part_rows, rows);
  const void *src = is_v ? a.v : a.k;
  const int64_t stride = is_v ? a.v_stride : a.k_stride;
  const bool turned = !is_v && c * 8 < a.rot_dim, paired = turned && !a.interleaved;
  const bool first = c < angles;  // of its pair
  const int other = first ? c + angles : c - angles;
  for (int r = from + tid / LANES; r - tid / LANES < until; r += kRows) {
    const int t = r % NTOK, head = r / NTOK;
    const int slot = r < rows && c < pieces ? slot_of[t] : -1;
    Raw8<SRC> lo = {}, hi = {};
    if (slot >= 0) {
      const int64_t row = (t0 + t) * stride + static_cast<int64_t>(head) * a.D;
      lo.load(src, row + c * 8);
      if (paired) hi.load(src, row + other * 8);
    }
    float v[8];
    double y[8];  // of K
    lo.values(v);
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = v[i];
      const double2 *tw = turn.k + t * half;
      if (paired) {
        float z[8];
        hi.values(z);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double2 w = tw[i * angles + (first ? c : other)];
          y[i] = y[i] * w.x + (first ? -w.y : w.y) * static_cast<double>(z[i]);
        }
      } else if (turned) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const double2 w = tw[((c * 4 + (i >> 1)) & 7) * angles + (c >> 1)];
          const double p = y[i], q = y[i + 1];
          y[i] = p * w.x - q * w.y;
          y[i + 1] = q * w.x + p * w.y;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(y[i]);
    }
    uint32_t most = 0;  // as bits: infinities and, above them, NaN win
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
    const float top = __builtin_bit_cast(float, row_max<LANES>(most));
    uint32_t bits = scale_bits(top);
    float s = __builtin_bit_cast(float, bits << 16);
    if (!is_v && __any(127.0f * s == top)) {  // the value itself may be above that
      double exact = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) exact = fmax(exact, fabs(y[i]));
      exact = row_max<LANES>(exact);
      if (127.0 * static_cast<double>(s) < exact && bits < 0x7F80u) s = __builtin_bit_cast(float, ++bits << 16);
    }
    const float inv = __builtin_amdgcn_rcpf(s);
    int code[8];
    bool near = s < kLeast;  // whether a value may lie on the other side of a border
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = v[i] * inv, n = rintf(q);
      code[i] = static_cast<int>(n);
      if (is_v) {
        // what is left of v is exact in fp32: n s has 15 bits
        const float left = fabsf(__builtin_fmaf(-n, s, v[i])), border = 0.5f * s;
        if (left > border || (left == border && (code[i] & 1))) code[i] += v[i] > n * s ? 1 : -1;
      } else {
        near |= fabsf(q - n) > 0.4999f;
      }
    }
    if (__any(near)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        code[i] = static_cast<int>(rint((is_v ? static_cast<double>(v[i]) : y[i]) / static_cast<double>(s)));
    }
    const bool some = s > 0.0f;  // not a row of zeros, nor one that reads as NaN
    if (NTOK > 1 && is_v) {
      // by way of LDS, so that a lane has a dim's codes of all tokens
      uint8_t *mine = by_dim + (head % kHeads) * LANES * 8 * NTOK + c * 8 * NTOK + t;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[i * NTOK] = static_cast<uint8_t>(some ? code[i] : 0);
      if (slot >= 0 && c == 0)
        reinterpret_cast<uint16_t *>(args.scales)[
            (((static_cast<int64_t>(slot >> sh) * a.Hkv + head) << sh) + (slot & (P - 1))) * 2 + 1] =
            static_cast<uint16_t>(bits);
      __syncthreads();
      const int head0 = (r - tid / LANES) / NTOK;
      for (int i = tid; i < kHeads * LANES * 8; i += 256) {
        const int h = i / (LANES * 8), dim = i - h * LANES * 8;
        if (head0 + h >= a.Hkv || dim >= a.D) continue;
        store_tokens<NTOK>(static_cast<uint8_t *>(a.v_cache) + dim * 16, a.D, a.Hkv, head0 + h, sh,
                           slot_of, by_dim + i * NTOK);
      }
      __syncthreads();
      continue;
    }
    if (slot < 0) continue;
    const int64_t block = static_cast<int64_t>(slot >> sh) * a.Hkv + head;
    const int tok = slot & (P - 1);
    if (c == 0)
      reinterpret_cast<uint16_t *>(args.scales)[((block << sh) + tok) * 2 + is_v] =
          static_cast<uint16_t>(bits);
    if (is_v) {
      uint8_t *o = static_cast<uint8_t *>(a.v_cache) + ((block << sh) + (tok & ~15)) * a.D + c * 128 +
                   (tok & 15);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i * 16] = static_cast<uint8_t>(some ? code[i] : 0);
    } else {
      uint8_t *o = static_cast<uint8_t *>(a.k_cache) + ((block * (a.D >> 4) + (c >> 1)) << sh) * 16 +
                   tok * 16 + (c & 1) * 8;
      u32x2 w = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i >> 2] |= static_cast<uint32_t>(code[i] & 0xFF) << (8 * (i & 3));
      *reinterpret_cast<u32x2 *>(o) = some ? w : u32x2{0u, 0u};
    }
  }
}

// A wave reads 16 tokens' K or V, 64 values of each: neighbouring lanes four
// pieces of 16 values, so that a row is written in whole lines, and four lanes
// further the next token, so that its codes, in V bytes of one piece, are near.
template <int OUT>
__global__ __launch_bounds__(256) void k_read_rows_q8(const ReadArgs a) {
  const int row_pieces = a.Hkv * (a.D >> 4), groups = (row_pieces + 3) >> 2;
  const int sh = a.page_shift, P = 1 << sh, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t units = static_cast<int64_t>((a.N + 15) >> 4) * groups * 2;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + wave; i < units; i += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t w = i / groups;
    const int u = static_cast<int>(i - w * groups) * 4 + (lane & 3);  // piece of the row
    const bool is_v = w & 1;
    const int row = static_cast<int>(w >> 1) * 16 + (lane >> 2);
    if (row >= a.N || u >= row_pieces) continue;
    const int head = u / (a.D >> 4), c = u - head * (a.D >> 4);
    const int slot = a.slots[row];
    float x[16] = {};
    if (static_cast<uint32_t>(slot) < static_cast<uint32_t>(a.num_slots)) {
      const int64_t block = static_cast<int64_t>(slot >> sh) * a.Hkv + head;
      const int tok = slot & (P - 1);
      const uint32_t s = a.scales[(block << sh) + tok];
      const float scale = is_v ? v_scale(s) : k_scale(s);
      if (is_v) {
        const int8_t *p = static_cast<const int8_t *>(a.v) + ((block << sh) + (tok & ~15)) * a.D +
                          c * 256 + (tok & 15);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = static_cast<float>(p[e * 16]) * scale;
      } else {
        const u32x4 p = static_cast<const u32x4 *>(a.k)[((block * (a.D >> 4) + c) << sh) + tok];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[e] = static_cast<float>(static_cast<int8_t>(p[e >> 2] >> (8 * (e & 3)))) * scale;
      }
    }
    char *o = static_cast<char *>(is_v ? a.v_out : a.k_out) +
              (row * (is_v ? a.v_stride : a.k_stride) + static_cast<int64_t>(u) * 16) *
                  (OUT == IFX_ATTN_F32 ? 4 : 2);
    if constexpr (OUT == IFX_ATTN_F32) {
#pragma unroll
      for (int e = 0; e < 16; e += 4) store4(o, OUT, e, f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]});
    } else {
      using T = Elem<OUT == IFX_ATTN_F32 ? IFX_ATTN_F16 : OUT>;
#pragma unroll
      for (int e = 0; e < 16; e += 8) {
        const u32x4 w8 = {T::pack(x[e], x[e + 1]), T::pack(x[e + 2], x[e + 3]),
                          T::pack(x[e + 4], x[e + 5]), T::pack(x[e + 6], x[e + 7])};
        __builtin_memcpy(o + e * 2, &w8, 16);
      }
    }
  }
}

namespace {
// Eight tokens a workgroup, whose V is written eight bytes at a time rather than
// byte by byte, from where there are workgroups enough for the chip.  us of an
// append and a read with one token / with eight, heads of 128, fp16 rows:
//    8 /  1 heads  256 tokens 7.5/8.0, 512 9.2/8.2, 1024 13.3/8.5, 2048 21.4/10.0
//   16 /  2        256 8.0/8.2, 512 10.0/8.6, 1024 14.7/9.2, 4096 40.5/17.3
//   40 /  8        128 7.8/8.3, 192 8.9/8.6, 512 13.4/11.1, 4096 62.8/40.2
//   48 / 16         64 8.3/8.3, 128 9.0/8.7, 512 17.8/14.3, 2048 46.7/32.6
//   32 / 32         64 10.8/8.5, 256 16.3/13.3, 1024 41.0/29.8, 2048 86.6/50.0
// Of K's and V's heads as few a workgroup as fill the chip, as each makes the
// angles anew: with a turn / two / four of the workgroup's lanes over them
//   40 /  8 heads  512 tokens 11.1/13.3/19.2, 2048 24.1/22.5/24.6, 4096 44.5/41.7/40.2
//   32 / 32        512 19.7/20.3/24.1, 1024 31.2/29.8/31.7, 2048 58.7/52.8/50.0
// and of Q with 512 / 1024 / 1536 / 2560 units of them
//   40 /  8 heads  2048 tokens 22.6/22.2/21.6/23.2, 4096 40.5/39.6/39.0/38.1, 5299 52.5/52.5/51.2/51.9
template <int DT, int SRC, int LANES>
void launch(AppendQ8Args a, hipStream_t s) {
  const AppendArgs &p = a.a;
  if (static_cast<int64_t>(p.T) * (p.Hq + 2 * p.Hkv) >= 7168) {
    const int turns = (8 * p.Hkv * LANES + 255) / 256;  // of K's heads
    const int64_t groups = static_cast<int64_t>(p.T + 7) / 8 * turns;
    const int each = groups < 1024 ? 1 : groups < 2048 ? 2 : 4;
    const int units = 8 * p.Hq * ((p.D >> 3) - (p.interleaved ? 0 : p.rot_dim >> 4));
    const int share = each == 1 ? 512 : 1536;  // of Q's units
    a.kv_parts = (turns + each - 1) / each;
    IFX_LAUNCH(k_rope_append_q8, (DT, SRC, LANES, 8),
               dim3((p.T + 7) / 8, 2 * a.kv_parts + (units + share - 1) / share), dim3(256), 0, s, a);
  } else {
    a.kv_parts = 1;
    IFX_LAUNCH(k_rope_append_q8, (DT, SRC, LANES, 1), dim3(p.T, 3), dim3(256), 0, s, a);
  }
}
template <int DT, int SRC>
void launch(const AppendQ8Args &a, hipStream_t s) {
  if (a.a.D <= 64) return launch<DT, SRC, 8>(a, s);
  if (a.a.D <= 128) return launch<DT, SRC, 16>(a, s);
  return launch<DT, SRC, 32>(a, s);
}
template <int DT>
void launch(const AppendQ8Args &a, int src_dtype, hipStream_t s) {
  switch (src_dtype) {
    case IFX_ATTN_F32: return launch<DT, IFX_ATTN_F32>(a, s);
    case IFX_ATTN_F16: return launch<DT, IFX_ATTN_F16>(a, s);
    default: return launch<DT, IFX_ATTN_BF16>(a, s);
  }
}
}  // namespace

hipError_t launch_rope_append_q8(const AppendQ8Args &a, int src_dtype, int q_dtype, hipStream_t s) {
  if (q_dtype == IFX_ATTN_F16)
    launch<IFX_ATTN_F16>(a, src_dtype, s);
  else
    launch<IFX_ATTN_BF16>(a, src_dtype, s);
  return last_error();
}

hipError_t launch_read_rows_q8(const ReadArgs &a, int out_dtype, hipStream_t s) {
  const int64_t units = static_cast<int64_t>((a.N + 15) >> 4) * ((a.Hkv * (a.D >> 4) + 3) >> 2) * 2;
  const int64_t need = (units + 3) / 4;  // a wave each
  const dim3 grid(static_cast<uint32_t>(need < 16384 ? need : 16384));
  if (out_dtype == IFX_ATTN_F32)
    IFX_LAUNCH(k_read_rows_q8, (IFX_ATTN_F32), grid, dim3(256), 0, s, a);
  else if (out_dtype == IFX_ATTN_F16)
    IFX_LAUNCH(k_read_rows_q8, (IFX_ATTN_F16), grid, dim3(256), 0, s, a);
  else
    IFX_LAUNCH(k_read_rows_q8, (IFX_ATTN_BF16), grid, dim3(256), 0, s, a);
  return last_error();
}

}  // namespace ifx
