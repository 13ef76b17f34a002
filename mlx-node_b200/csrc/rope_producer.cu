// Per-head RMS norm of queries and keys, rotation by a plan and cache write, for every head
// size, block size and cache type of the library.
//
//   y = x * w / sqrt(mean(x^2) + eps)            (no norm: y = x)
//   (a, b) -> g (a cos t - b sin t, b cos t + a sin t),  t = position * f_i
//
// A row stays in fp32 from the load to the one rounding to the 16-bit type.  The phase is
// position * turn[i] modulo 2^64 in units of 2^-64 turns (RopeTable): reduced exactly, its top
// 32 bits as a signed number are the angle within half a turn.
//
// HBM-bound for chunks, latency-bound for single tokens; in between the instructions count, so
// that every index is a shift and every address of a loop a constant step.  Two kinds of CTAs, both
// over `tokens` tokens - 16 for chunks, so that pool stores fill sectors; down to one for small
// batches, so that the rows spread over the SMs:
//   queries    up to 16 query heads of the tokens; nothing is shared, no barrier
//   keys       up to 4 kv heads: the key rows, the value rows and the pool write, staged in shared
//              memory
// (more heads to a CTA where it has few tokens: what a CTA does once - addresses, the plan's entries,
// sines - costs as much as three rows).
// A row belongs to D / 8 lanes of a warp, 16 bytes each; the next two rows of a group of lanes are
// on their way while two are computed.  A lane computes the sines and cosines of its own elements
// once per token, in registers, and folds the norm's weights into them.  The rotation's partner
// elements sit in the same lane (interleaved pairs), in another lane of the group (halves of a
// multiple of 8 elements: a shuffle) or, for the odd sizes, are read again from global memory.  The
// value chunk is a transpose of the rows: where a CTA's 16 tokens fill an aligned run of slots it is
// stored in runs of tokens out of ldmatrix.trans (FP8: byte permutes), otherwise element by element.
// Measured on one B200, the same inputs over and over: 8192 tokens, 32/8 heads of 128, keys kept, 218 MB in
// 50.0 us (4.4 TB/s) where the slots begin with a block; 53.4 where they begin inside one, 52.1 as packed
// prompts of 300-900 tokens, 51.4 with blocks of 8 tokens (the element-wise write); 47.5 with interleaved pairs; 89.7
// with 90 of the 128 elements rotated (partners read again).  2049 tokens, 64/8 heads, FP8 write, 84 MB in 20.7 us,
// 21.3 from inside a block; with changing inputs 50.6 and 22.7.  64 tokens in a graph 6.0 us in a row and 6.1 with a
// block and a position each; one token 4.3.
#include <algorithm>
#include <type_traits>

#include "prompt_path.cuh"

namespace pa {

namespace {

constexpr int kThreads = 256;
constexpr int kTokMax = 16;
enum { PAIR_LANE = 0, PAIR_SHUFFLE = 1, PAIR_MEMORY = 2 };

template <bool F16>
__device__ __forceinline__ void unpack8(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = elem_value<F16>(w[i] & 0xffffu);
    x[2 * i + 1] = elem_value<F16>(w[i] >> 16);
  }
}
__device__ __forceinline__ bool has_exponent15(uint2 b) {
  return ((((b.x & 0x78787878u) + 0x08080808u) | ((b.y & 0x78787878u) + 0x08080808u)) & 0x80808080u) != 0u;
}
// Two fp32 values at a time: 2049 tokens, 32/8 heads, 18.0 -> 16.5 us, 8192 tokens 50.7 -> 49.5 (rows that
// rotate interleaved pairs and the FP8 division keep single ones: 22.7 us on an FP8 chunk, 24.5 in twos).
__device__ __forceinline__ uint64_t pair64(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair64(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// quantise8 for the common cases, bit for bit.  Elements whose scaled magnitudes are in [2^-6, 240) take
// the hardware's E4M3 conversion, which rounds that range to nearest even like the cache format does.
// Smaller ones (one lane in thirty for normal values of deviation 12 to 24) have their bytes replaced
// by the format's: a multiple of 2^-9, rounded half up, masked to three bits, zero below 2^-9.  Eight
// elements with any larger one, an infinity or a NaN go to the format's own encoder, and only they can
// hold an exponent field of 15 (`odd`).
// x / scale is rounded to fp32 as IEEE division does, by Markstein's correction (IBM J. Res. Dev. 34,
// 1990): with y the correctly rounded reciprocal, q = x y and
// q + (x - q scale) y is the correctly rounded quotient as long as nothing under- or overflows.
// `scale` in [2^-60, 2^60] and a quotient of at least 2^-10 make sure of that; below it the bytes are
// zeros with the element's sign either way.  8192 tokens, 64/8 heads: 78 us with eight elements in the
// format's encoder for one small one, 73.4 so.
template <bool F16>
__device__ __forceinline__ uint2 quantise_row8(uint4 v, float scale, float recip, bool &odd) {
  constexpr uint32_t kSmall = F16 ? 0x2400u : 0x3c80u, kLarge = F16 ? 0x5b80u : 0x4370u;  // 2^-6, 240
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t r[4], least = 0xffffffffu, most = 0u;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float x0 = elem_value<F16>(w[i] & 0xffffu), x1 = elem_value<F16>(w[i] >> 16);
    float q0 = x0 * recip, q1 = x1 * recip;
    q0 = fmaf(fmaf(-q0, scale, x0), recip, q0);
    q1 = fmaf(fmaf(-q1, scale, x1), recip, q1);
    r[i] = pack2<F16>(q0, q1);  // to the 16-bit type first, as the plain write does
    least = min_u16x2(least, r[i] & 0x7fff7fffu);
    most = max_u16x2(most, r[i] & 0x7fff7fffu);
  }
  odd = recip == 0.f || (most & 0xffffu) >= kLarge || (most >> 16) >= kLarge;
  if (odd) {
    const uint2 b = quantise8<F16>(v, scale);
    odd = has_exponent15(b);
    return b;
  }
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint16_t h;
    if (F16) asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h) : "r"(r[i]));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(elem_value<F16>(r[i] >> 16)), "f"(elem_value<F16>(r[i] & 0xffffu)));
    o[i] = h;
  }
  if ((least & 0xffffu) < kSmall || (least >> 16) < kSmall) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float t = fabsf(elem_value<F16>(r[i >> 1] >> (i & 1) * 16 & 0xffffu));
      // (the sign is the element's: the correction turns -0 into 0)
      const uint32_t byte = (w[i >> 1] >> (i & 1) * 16 + 8 & 0x80u) | (t < 0x1p-9f ? 0u : (uint32_t)(int)fmaf(t, 512.f, 0.5f) & 7u);
      if (t < 0x1p-6f) o[i >> 1] = i & 1 ? (o[i >> 1] & 0xffu) | byte << 8 : (o[i >> 1] & 0xff00u) | byte;
    }
  }
  return make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16);
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// GW: lanes of a row, a power of two of at least D / 8.
// BATCH: rows that a group of lanes computes while as many more are on their way: 2, or 1 where a
// group has no more (less code to fetch on a path whose time is the latency of one pass through it).
// (64 registers, so that an SM holds four CTAs: two rows ahead measured 50.8 us on a 8192-token prompt
// and 22.4 on an FP8 chunk of 2049 (same inputs each time), four without looking ahead 51.3 and 26.3, three CTAs of 80 registers
// and four rows ahead 49.6 and 28.7.  At 64 registers the form with two rows ahead spills, in stores per thread: 32 to
// 64 bytes with 16-bit pools, 56 to 88 with FP8, 124 to 144 where partners are read again.)
template <int GW, bool F16, bool FP8, int PAIR, int BATCH>
__global__ void __launch_bounds__(kThreads, BATCH == 1 ? 3 : 4)
rope_norm_cache_kernel(const __grid_constant__ RotateParams p, int tok_log, int q_heads, int kv_heads, int kv_ctas) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int tokens = 1 << tok_log, D = p.D, dims = p.rope.dims, half = dims >> 1;
  constexpr int kElem = FP8 ? 1 : 2;  // bytes of a pool element
  const int v_row = D * kElem + 16;   // bytes of a staged value row, padded against bank conflicts
  __shared__ int64_t slot_s[kTokMax];

  // the attention kernel that follows may set up (it reads no pool data before its own wait)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x;
  const bool keys = (int)blockIdx.y < kv_ctas;
  const int h = keys ? blockIdx.y * kv_heads : (blockIdx.y - kv_ctas) * q_heads;  // first head
  const int n_heads = keys ? min(kv_heads, p.Hkv - h) : min(q_heads, p.Hq - h);   // rows of a token
  uint8_t *const k_s = smem;                                  // [head][token][D]
  uint8_t *const v_s = k_s + kv_heads * tokens * D * kElem;   // [head][token][v_row]
  const int64_t t0 = (int64_t)blockIdx.x << tok_log;
  const int n_tok = (int)min((int64_t)tokens, p.num_tokens - t0);
  const bool write = keys && p.slot_mapping != nullptr;
  auto recip_of = [](float x) { return x >= 0x1p-60f && x <= 0x1p60f ? __frcp_rn(x) : 0.f; };  // 0: not to be used
  const float k_recip = FP8 ? recip_of(p.k_scale) : 0.f, v_recip = FP8 ? recip_of(p.v_scale) : 0.f;

  // ---- this group's rows: of one token, every `share`-th row ------------------------------
  constexpr int kGroups = kThreads / GW;
  const int group = tid / GW, gl = tid % GW, e0 = gl * 8;
  const uint32_t lanes = (GW == 32 ? 0xffffffffu : (1u << (GW % 32)) - 1u) << ((tid & 31) / GW * GW);  // this group's
  const bool in_row = e0 < D;
  const int share_log = kGroups >> tok_log ? 31 - __clz(kGroups >> tok_log) : 0;  // log2(groups of a token)
  const int first = group & ((1 << share_log) - 1);
  int tok = group >> share_log;
  const elem16 *const x_in = (keys ? p.k : p.q) + (t0 * (keys ? p.k_stride : p.q_stride) + (int64_t)h * D + e0);
  const int64_t x_stride = keys ? p.k_stride : p.q_stride;
  const elem16 *const weight = keys ? p.k_norm_w : p.q_norm_w;
  const elem16 *src;  // this lane's piece of the token's first row
  uint4 raw[BATCH];
  auto load_rows = [&](uint4 (&raw)[BATCH], int r0) {
#pragma unroll
    for (int b = 0; b < BATCH; b++) {
      const int r = r0 + (b << share_log);
      raw[b] = make_uint4(0, 0, 0, 0);
      if (in_row && tok < n_tok && r < n_heads) raw[b] = *reinterpret_cast<const uint4 *>(src + r * D);
    }
  };
  src = x_in + tok * x_stride;
  load_rows(raw, first);
  const bool turns = e0 < dims;  // this lane has elements that rotate (PAIR_SHUFFLE: all of them or none)
  // the piece with the partners of this lane's elements (PAIR_SHUFFLE), in lanes
  const int other = PAIR != PAIR_SHUFFLE || !turns ? gl : e0 < half ? gl + (half >> 3) : gl - (half >> 3);
  auto partner = [&](int d) { return PAIR == PAIR_LANE ? d ^ 1 : d < half ? d + half : d - half; };

  // The plan's entries of this lane's elements (of its four pairs, when they are interleaved).  An
  // indexed constant load takes a cycle and more per distinct address of a warp; through a generic
  // address it is an ordinary load.
  constexpr int kTurns = PAIR == PAIR_LANE ? 4 : 8;
  uint32_t turn_lo[kTurns], turn_hi[kTurns];
  if (PAIR == PAIR_MEMORY) {
#pragma unroll
    for (int i = 0; i < kTurns; i++) {
      const int d = e0 + i;
      turn_lo[i] = turn_hi[i] = 0;
      if (d < dims)
        asm("ld.v2.u32 {%0, %1}, [%2];" : "=r"(turn_lo[i]), "=r"(turn_hi[i]) : "l"(p.rope.turn + (d < half ? d : d - half)));
    }
  } else {
    const uint64_t *at = p.rope.turn + (!turns ? 0 : PAIR == PAIR_LANE ? e0 >> 1 : e0 < half ? e0 : e0 - half);
#pragma unroll
    for (int i = 0; i < kTurns; i += 2)
      asm("ld.v4.u32 {%0, %1, %2, %3}, [%4];"
          : "=r"(turn_lo[i]), "=r"(turn_hi[i]), "=r"(turn_lo[i + 1]), "=r"(turn_hi[i + 1])
          : "l"(at + i));
  }

  // ---- slots and values ---------------------------------------------------------------------
  if (write) {
    if (tid < tokens) {
      int64_t s = -1;
      if (tid < n_tok) {
        s = p.slot_mapping[t0 + tid];
        if (s >= ((int64_t)p.num_blocks << p.bs_log)) {
          atomicOr(p.err, kErrSlotRange);
          s = -1;
        }
      }
      slot_s[tid] = s;
    }
    for (int vt = tok; vt < n_tok && in_row; vt += kGroups) {
      const elem16 *const v = p.v + (t0 + vt) * p.v_stride + h * D + e0;
      uint8_t *const dst = v_s + vt * v_row + e0 * kElem;
      const int dst_head = tokens * v_row;
      if (FP8) {
        for (int r0 = first; r0 < n_heads; r0 += 4 << share_log) {  // four rows on their way at once
          uint4 rows[4];
#pragma unroll
          for (int b = 0; b < 4; b++) {
            const int r = r0 + (b << share_log);
            if (r < n_heads) rows[b] = *reinterpret_cast<const uint4 *>(v + r * D);
          }
#pragma unroll
          for (int b = 0; b < 4; b++) {
            const int r = r0 + (b << share_log);
            if (r >= n_heads) break;
            bool odd;
            *reinterpret_cast<uint2 *>(dst + r * dst_head) = quantise_row8<F16>(rows[b], p.v_scale, v_recip, odd);
            if (odd && p.slot_mapping[t0 + vt] >= 0) atomicOr(p.special, 1u);
          }
        }
      } else {
        for (int r = first; r < n_heads; r += 1 << share_log)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + r * dst_head)), "l"(v + r * D) : "memory");
      }
    }
  }

  // ---- norm and rotation: y_e = inv (x_e A_e + x_partner B_e) ------------------------------------
  const float inv_d = 1.f / (float)D;
  // one row of this group: its piece in `r`, the piece's address (PAIR_MEMORY) in `row`
  auto turn_row = [&](uint4 r, const elem16 *row, const float (&A)[8], const float (&B)[8]) {
    float x[8], z[8];
    unpack8<F16>(r, x);
    float inv = 1.f;
    if (weight) {
      uint64_t ss2 = 0;
#pragma unroll
      for (int i = 0; i < 8; i += 2) ss2 = fma2(pair64(x[i], x[i + 1]), pair64(x[i], x[i + 1]), ss2);
      float ss, ss_odd;
      unpair64(ss2, ss, ss_odd);
      ss += ss_odd;
#pragma unroll
      for (int o = GW / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
      inv = rsqrtf(fmaf(ss, inv_d, p.eps));
    }
    // the partner's value, 0 for an element that does not rotate (its B is 0, and 0 * inf is not)
    if (PAIR == PAIR_LANE) {
#pragma unroll
      for (int i = 0; i < 8; i++) z[i] = e0 + i < dims ? x[i ^ 1] : 0.f;
    } else if (PAIR == PAIR_SHUFFLE) {
      uint4 o;
      o.x = __shfl_sync(lanes, r.x, other, GW);
      o.y = __shfl_sync(lanes, r.y, other, GW);
      o.z = __shfl_sync(lanes, r.z, other, GW);
      o.w = __shfl_sync(lanes, r.w, other, GW);
      if (!turns) o = make_uint4(0, 0, 0, 0);
      unpack8<F16>(o, z);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) z[i] = in_row && e0 + i < dims ? elem_value<F16>(row[partner(e0 + i) - e0]) : 0.f;
      __syncwarp(lanes);  // the row may be rotated in place: all of it has been read
    }
    uint32_t out[4];
    const uint64_t inv2 = pair64(inv, inv);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (PAIR == PAIR_LANE) {  // (a swapped pair would have to be moved into place)
        out[i >> 1] = pack2<F16>(fmaf(x[i], A[i], z[i] * B[i]) * inv, fmaf(x[i + 1], A[i + 1], z[i + 1] * B[i + 1]) * inv);
        continue;
      }
      const uint64_t zb = mul2(pair64(z[i], z[i + 1]), pair64(B[i], B[i + 1]));
      float y0, y1;
      unpair64(mul2(fma2(pair64(x[i], x[i + 1]), pair64(A[i], A[i + 1]), zb), inv2), y0, y1);
      out[i >> 1] = pack2<F16>(y0, y1);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
  };
  for (;;) {
    if (tok < n_tok && first < n_heads) {
      // Sine and cosine for this lane's elements.  The phase's top word is within half a turn, where
      // the hardware's sine and cosine are off by at most 2^-20.9 absolute: nothing against the
      // half step of 2^-9 or 2^-12 that the result is rounded by.
      const int64_t t = t0 + tok;
      const int32_t pos = p.positions[t];
      float A[8], B[8];
#pragma unroll
      for (int i = 0; i < kTurns; i++) {
        // top word of (64-bit position) * entry modulo 2^64
        uint32_t phase = __umulhi((uint32_t)pos, turn_lo[i]) + (uint32_t)pos * turn_hi[i];
        phase -= (uint32_t)(pos >> 31) & turn_lo[i];
        const float angle = (float)(int32_t)phase * 1.46291807926715968e-9f;  // 2 pi / 2^32
        const float cn = __cosf(angle) * p.rope.gain, sn = __sinf(angle) * p.rope.gain;
        if (PAIR == PAIR_LANE) {
          const bool on = e0 + 2 * i < dims;
          A[2 * i] = A[2 * i + 1] = on ? cn : 1.f;
          B[2 * i] = on ? -sn : 0.f;
          B[2 * i + 1] = on ? sn : 0.f;
        } else {
          const bool on = e0 + i < dims;
          A[i] = on ? cn : 1.f;
          B[i] = on ? (e0 + i < half ? -sn : sn) : 0.f;
        }
      }
      if (weight && in_row) {  // A *= w, B *= the partner's w
        float w[8];
        unpack8<F16>(*reinterpret_cast<const uint4 *>(weight + e0), w);
#pragma unroll
        for (int i = 0; i < 8; i++) A[i] *= w[i];
        if (PAIR == PAIR_LANE) {
#pragma unroll
          for (int i = 0; i < 8; i++) B[i] *= w[i ^ 1];
        } else if (PAIR == PAIR_SHUFFLE) {
          unpack8<F16>(*reinterpret_cast<const uint4 *>(weight + other * 8), w);
#pragma unroll
          for (int i = 0; i < 8; i++) B[i] *= w[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (e0 + i < dims) B[i] *= elem_value<F16>(weight[partner(e0 + i)]);
        }
      }
      elem16 *const dst = keys ? p.k_out ? p.k_out + t * p.k_out_stride + (int64_t)h * D + e0 : nullptr
                               : p.q_out + t * p.q_out_stride + (int64_t)h * D + e0;
      for (int base = first; base < n_heads; base += BATCH << share_log) {
        // the next batch is on its way while this one is computed
        uint4 next[BATCH];
        if (BATCH > 1) load_rows(next, base + (BATCH << share_log));
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
          const int r = base + (b << share_log);
          if (r >= n_heads) break;
          const uint4 out = turn_row(raw[b], src + r * D, A, B);
          if (in_row && dst) *reinterpret_cast<uint4 *>(dst + r * D) = out;
          if (in_row && write) {
            uint8_t *st = k_s + ((r * tokens + tok) * D + e0) * kElem;
            if (FP8) {
              bool odd;
              *reinterpret_cast<uint2 *>(st) = quantise_row8<F16>(out, p.k_scale, k_recip, odd);
              if (odd && p.slot_mapping[t] >= 0) atomicOr(p.special, 1u);
            } else {
              *reinterpret_cast<uint4 *>(st) = out;
            }
          }
        }
        if (BATCH == 1) load_rows(next, base + (BATCH << share_log));
#pragma unroll
        for (int b = 0; b < BATCH; b++) raw[b] = next[b];
      }
    }
    // fewer groups than tokens (rows of 32 lanes): a group takes a second token
    tok += kGroups;
    if (tok >= tokens) break;
    src = x_in + tok * x_stride;
    load_rows(raw, first);
  }
  if (!write) return;
  if (!FP8) asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();

  // ---- pool write, token index fastest across threads: a thread keeps its token ----------------
  const int wt = tid & (tokens - 1), bs = 1 << p.bs_log;
  const int64_t slot = slot_s[wt];
  const int off = (int)(slot & (bs - 1));
  const int chunk_bytes = (D << p.bs_log) * kElem;
  const int64_t chunk0 = ((slot >> p.bs_log) * p.Hkv + h) * (int64_t)chunk_bytes;
  // an aligned run of 16 slots (two blocks of 8 tokens are not one)
  const bool run = __all_sync(0xffffffffu, tokens == kTokMax && bs >= kTokMax && slot >= 0 && slot == slot_s[0] + wt && (slot_s[0] & 15) == 0);
  const int warp = tid >> 5, lane = tid & 31;
  if (slot >= 0) {
    uint8_t *const dst = static_cast<uint8_t *>(p.k_pool) + chunk0 + off * 16;
    for (int r = 0; r < n_heads; r++)
      for (int c = tid >> tok_log; c < D * kElem / 16; c += kThreads >> tok_log)
        *reinterpret_cast<uint4 *>(dst + r * chunk_bytes + c * bs * 16) =
            *reinterpret_cast<const uint4 *>(k_s + (r * tokens + wt) * D * kElem + c * 16);
  }
  uint8_t *const v_dst = static_cast<uint8_t *>(p.v_pool) + chunk0;
  if (run && !FP8) {
    // matrices 0 and 1 hold 8 dimensions, 2 and 3 the next 8; row r of matrix m is token
    // (r / 2) * 4 + 2 (m % 2) + r % 2, so that a lane ends up with four tokens of a dimension
    const int m = lane >> 3, mr = lane & 7, mt = (mr >> 1) * 4 + (m & 1) * 2 + (mr & 1);
    const int run_off = (int)(slot_s[0] & (bs - 1)) * 2 + (lane & 3) * 8;
    for (int r = 0; r < n_heads; r++)
      for (int d0 = warp * 16; d0 < D; d0 += kThreads / 2) {
        uint32_t w[4];
        ldmatrix_x4_trans(w, smem_u32(v_s) + (r * tokens + mt) * v_row + (d0 + (m >> 1) * 8) * 2);
        uint8_t *dst = v_dst + r * chunk_bytes + run_off;
        const int d = d0 + (lane >> 2);
        *reinterpret_cast<uint2 *>(dst + d * bs * 2) = make_uint2(w[0], w[1]);
        if (d + 8 < D) *reinterpret_cast<uint2 *>(dst + (d + 8) * bs * 2) = make_uint2(w[2], w[3]);
      }
  } else if (run) {
    // four tokens x four dimensions of bytes per thread
    for (int i = tid; i < n_heads * D; i += kThreads) {
      const int r = i / kHeadSize, tq = i & 3, d = (i % kHeadSize >> 2) * 4;  // FP8 caches have head size 128
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] = *reinterpret_cast<const uint32_t *>(v_s + (r * tokens + tq * 4 + k) * v_row + d);
      const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);  // dimensions 0, 1
      const uint32_t c = __byte_perm(w[0], w[1], 0x7362), e = __byte_perm(w[2], w[3], 0x7362);  // dimensions 2, 3
      uint8_t *dst = v_dst + r * chunk_bytes + (int)(slot_s[0] & (bs - 1)) + tq * 4 + d * bs;
      *reinterpret_cast<uint32_t *>(dst) = __byte_perm(a, b, 0x5410);
      *reinterpret_cast<uint32_t *>(dst + bs) = __byte_perm(a, b, 0x7632);
      *reinterpret_cast<uint32_t *>(dst + 2 * bs) = __byte_perm(c, e, 0x5410);
      *reinterpret_cast<uint32_t *>(dst + 3 * bs) = __byte_perm(c, e, 0x7632);
    }
  } else if (slot >= 0) {
    for (int r = 0; r < n_heads; r++)
      for (int d = tid >> tok_log; d < D; d += kThreads >> tok_log) {
        const uint8_t *from = v_s + (r * tokens + wt) * v_row + d * kElem;
        uint8_t *to = v_dst + r * chunk_bytes + (d * bs + off) * kElem;
        if (FP8) *to = *from;
        else *reinterpret_cast<elem16 *>(to) = *reinterpret_cast<const elem16 *>(from);
      }
  }
}

// Heads of a CTA and the grid for `tokens` tokens to a CTA.
struct Shape {
  int q_heads, kv_heads, kv_ctas;
  dim3 grid;
  size_t smem;
};
Shape shape_of(const RotateParams &p, int tok_log, bool fp8) {
  const int tokens = 1 << tok_log, gw = p.D <= 32 ? 4 : p.D <= 64 ? 8 : p.D <= 128 ? 16 : 32;
  const int share = std::max((kThreads / gw) >> tok_log, 1);  // groups of a token
  const int head_bytes = tokens * (p.D * (fp8 ? 2 : 4) + 16);
  Shape s;
  // 16 query and 4 kv heads (half of both: FP8 chunk of 2049 tokens, 64/8 heads, 22.7 -> 24.6 us; two kv
  // heads: 8192-token prompt, 32/8 heads, 50.6 -> 55; 32 query heads: FP8, 32768 tokens, 64/8 heads, 279 -> 270,
  // but the prompt 50.6 -> 55)
  s.q_heads = std::min(p.Hq, std::max(16, share));
  s.kv_heads = std::max(1, std::min({p.Hkv, std::max(4, share), 40960 / head_bytes}));
  s.kv_ctas = (p.Hkv + s.kv_heads - 1) / s.kv_heads;
  s.grid = dim3((unsigned)((p.num_tokens + tokens - 1) >> tok_log), (unsigned)(s.kv_ctas + (p.Hq + s.q_heads - 1) / s.q_heads));
  s.smem = (size_t)s.kv_heads * head_bytes;
  return s;
}

template <int GW, bool FP8, bool F16, int PAIR>
cudaError_t launch_pair(const RotateParams &p, int tok_log, cudaStream_t st) {
  const Shape s = shape_of(p, tok_log, FP8);
  const int share = (kThreads / GW) >> tok_log;
  auto go = [&](auto kernel) { kernel<<<s.grid, kThreads, s.smem, st>>>(p, tok_log, s.q_heads, s.kv_heads, s.kv_ctas); };
  if (share >= s.q_heads && share >= s.kv_heads) go(rope_norm_cache_kernel<GW, F16, FP8, PAIR, 1>);
  else go(rope_norm_cache_kernel<GW, F16, FP8, PAIR, 2>);
  return cudaGetLastError();
}
template <int GW, bool FP8, bool F16>
cudaError_t launch_group(const RotateParams &p, int tok_log, cudaStream_t st) {
  if (p.rope.interleaved) return launch_pair<GW, FP8, F16, PAIR_LANE>(p, tok_log, st);
  if (p.rope.dims % 16 == 0) return launch_pair<GW, FP8, F16, PAIR_SHUFFLE>(p, tok_log, st);
  return launch_pair<GW, FP8, F16, PAIR_MEMORY>(p, tok_log, st);
}

}  // namespace

cudaError_t launch_rope_norm_cache(const RotateParams &p, bool f16, bool fp8, int num_sms, cudaStream_t st) {
  if (p.num_tokens <= 0) return cudaSuccess;
  // two CTAs per SM before a CTA takes more than one token
  int tok_log = 4;
  for (; tok_log > 0; tok_log--) {
    const Shape s = shape_of(p, tok_log, fp8);
    if ((int64_t)s.grid.x * s.grid.y >= 2 * num_sms) break;
  }
  auto go = [&](auto f16_tag) {
    constexpr bool F16 = decltype(f16_tag)::value;
    if (fp8) return launch_group<16, true, F16>(p, tok_log, st);
    if (p.D <= 32) return launch_group<4, false, F16>(p, tok_log, st);
    if (p.D <= 64) return launch_group<8, false, F16>(p, tok_log, st);
    if (p.D <= 128) return launch_group<16, false, F16>(p, tok_log, st);
    return launch_group<32, false, F16>(p, tok_log, st);
  };
  const cudaError_t e = f16 ? go(std::true_type{}) : go(std::false_type{});
  __atomic_fetch_add(&g_launch_count, 1ull, __ATOMIC_RELAXED);
  return e;
}

}  // namespace pa
