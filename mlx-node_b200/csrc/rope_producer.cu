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
// HBM-bound for chunks, latency-bound for single tokens.  A CTA takes `tokens` tokens (16 for
// chunks, so that pool stores fill sectors; down to one for small batches, so that the rows
// spread over the SMs) of one kv head: its key row, its value row and the G query rows.  A row
// belongs to D / 8 lanes of a warp, 16 bytes each; rows of a group of lanes are loaded four
// at a time before the first is used.  Sines and cosines are computed once per (token, pair) into
// shared memory.  The rotation's partner elements sit in the same lane (interleaved pairs), in
// another lane of the group (halves of a multiple of 8 elements: a shuffle) or, for the odd
// sizes, are read again from global memory.
#include "prompt_path.cuh"

namespace pa {

namespace {

constexpr int kThreads = 256;
constexpr int kTokMax = 16;
constexpr int kBatch = 4;  // rows in flight per group of lanes
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

// GW: lanes of a row, a power of two of at least D / 8.
template <int GW, bool F16, bool FP8, int PAIR>
__global__ void __launch_bounds__(kThreads, 3) rope_norm_cache_kernel(const __grid_constant__ RotateParams p, int tok_log) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int tokens = 1 << tok_log, D = p.D, half = p.rope.dims >> 1, G = p.Hq / p.Hkv, pieces = D >> 3;
  const int v_row = D + (FP8 ? 8 : 2);  // elements (FP8: bytes) of a staged value row, padded against bank conflicts
  float2 *const cs = reinterpret_cast<float2 *>(smem);                   // [tokens][half]
  uint8_t *const k_s = smem + (size_t)tokens * ((half + 1) & ~1) * 8;    // [tokens][D] elements or bytes
  uint8_t *const v_s = k_s + (size_t)tokens * D * (FP8 ? 1 : 2);         // [tokens][v_row]
  __shared__ int64_t slot_s[kTokMax];

  // the attention kernel that follows may set up (it reads no pool data before its own wait)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int h = blockIdx.y, tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x << tok_log;
  const int n_tok = (int)min((int64_t)tokens, p.num_tokens - t0);
  const bool write = p.slot_mapping != nullptr;

  // ---- this group's rows: token, then every `share`-th of (key, G queries) -------------
  constexpr int kGroups = kThreads / GW;
  const int group = tid / GW, gl = tid % GW, e0 = gl * 8;
  const int share = kGroups >= tokens ? kGroups >> tok_log : 1;  // groups of a token
  const bool in_row = e0 < D;
  auto row_src = [&](int64_t t, int r) {
    return r == 0 ? p.k + t * p.k_stride + (int64_t)h * D : p.q + t * p.q_stride + (int64_t)(h * G + r - 1) * D;
  };
  uint4 raw[kBatch];
  auto load_batch = [&](int tok, int r0) {
#pragma unroll
    for (int b = 0; b < kBatch; b++) {
      const int r = r0 + b * share;
      raw[b] = make_uint4(0, 0, 0, 0);
      if (in_row && tok < n_tok && r <= G) raw[b] = *reinterpret_cast<const uint4 *>(row_src(t0 + tok, r) + e0);
    }
  };
  int tok = group / share;
  const int r_first = group % share;
  load_batch(tok, r_first);
  uint4 qw = make_uint4(0, 0, 0, 0), kw = qw;
  if (in_row && p.q_norm_w) qw = *reinterpret_cast<const uint4 *>(p.q_norm_w + e0);
  if (in_row && p.k_norm_w) kw = *reinterpret_cast<const uint4 *>(p.k_norm_w + e0);

  // ---- slots, values, sines -------------------------------------------------------------
  if (tid < kTokMax) {
    int64_t s = -1;
    if (write && tid < n_tok) {
      s = p.slot_mapping[t0 + tid];
      if (s >= ((int64_t)p.num_blocks << p.bs_log)) {
        atomicOr(p.err, kErrSlotRange);
        s = -1;
      }
    }
    slot_s[tid] = s;
  }
  if (write) {
    for (int i = tid; i < n_tok * pieces; i += kThreads) {
      const int vt = i / pieces, c = i - vt * pieces;
      const uint4 v = *reinterpret_cast<const uint4 *>(p.v + (t0 + vt) * p.v_stride + (int64_t)h * D + c * 8);
      if (FP8) {
        const uint2 b = quantise8<F16>(v, p.v_scale);
        if (has_exponent15(b) && p.slot_mapping[t0 + vt] >= 0) atomicOr(p.special, 1u);
        *reinterpret_cast<uint2 *>(v_s + vt * v_row + c * 8) = b;
      } else {
        uint32_t *d = reinterpret_cast<uint32_t *>(v_s + (vt * v_row + c * 8) * 2);
        d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
      }
    }
  }
  for (int i = tid; i < n_tok * half; i += kThreads) {
    const int ct = i / half, f = i - ct * half;
    const uint64_t phase = (uint64_t)(int64_t)p.positions[t0 + ct] * p.rope.turn[f];
    float sn, cn;
    sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &sn, &cn);
    cs[ct * half + f] = make_float2(cn * p.rope.gain, sn * p.rope.gain);
  }
  __syncthreads();

  // ---- norm and rotation --------------------------------------------------------------------
  const int step = kGroups >= tokens ? tokens : kGroups;  // a group takes tokens `step` apart
  for (; tok < tokens; tok += step) {
    if (tok != group / share) load_batch(tok, r_first);
    // sine and cosine of this lane's elements (of its four pairs, when they are interleaved)
    float co[8], si[8];
    if (tok < n_tok) {
#pragma unroll
      for (int i = 0; i < (PAIR == PAIR_LANE ? 4 : 8); i++) {
        const int d = PAIR == PAIR_LANE ? e0 + 2 * i : e0 + i;
        float2 c = make_float2(1.f, 0.f);
        if (d < 2 * half) c = cs[tok * half + (PAIR == PAIR_LANE ? d >> 1 : d < half ? d : d - half)];
        co[i] = c.x;
        si[i] = PAIR == PAIR_LANE || d >= half ? c.y : -c.y;  // halves: first a cos - b sin, second b cos + a sin
      }
    }
    const int64_t t = t0 + tok;
    // the same number of rounds for every group of a warp: they meet at the shuffles
    for (int r0 = r_first; r0 - r_first <= G; r0 += kBatch * share) {
      if (r0 != r_first) load_batch(tok, r0);
#pragma unroll
      for (int b = 0; b < kBatch; b++) {
        const int r = r0 + b * share;
        // (shuffles below: groups of one warp may hold different rows, or none)
        const bool have = in_row && tok < n_tok && r <= G;
        const bool is_k = r == 0, norm = is_k ? p.k_norm_w != nullptr : p.q_norm_w != nullptr;
        float x[8], y[8];
        unpack8<F16>(raw[b], x);
        float inv = 1.f;
        if (p.q_norm_w || p.k_norm_w) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
          for (int o = GW / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          if (norm) {
            inv = rsqrtf(ss / (float)D + p.eps);
            float w[8];
            unpack8<F16>(is_k ? kw : qw, w);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] *= inv * w[i];
          }
        }
        if (PAIR == PAIR_LANE) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            y[2 * i] = x[2 * i] * co[i] - x[2 * i + 1] * si[i];
            y[2 * i + 1] = x[2 * i + 1] * co[i] + x[2 * i] * si[i];
          }
        } else if (PAIR == PAIR_SHUFFLE) {
          const int other = e0 < half ? gl + (half >> 3) : gl - (half >> 3);  // used below 2 * half only
          const bool turns = e0 < 2 * half;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float z = __shfl_sync(0xffffffffu, x[i], turns ? other : gl, GW);
            y[i] = turns ? fmaf(x[i], co[i], z * si[i]) : x[i];
          }
        } else {
          const elem16 *src = row_src(t, r), *w = is_k ? p.k_norm_w : p.q_norm_w;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int d = e0 + i;
            y[i] = x[i];
            if (have && d < 2 * half) {
              const int o = d < half ? d + half : d - half;
              float z = elem_value<F16>(src[o]);
              if (norm) z *= inv * elem_value<F16>(w[o]);
              y[i] = fmaf(x[i], co[i], z * si[i]);
            }
          }
          __syncwarp();  // the row may be rotated in place: all of it has been read
        }
        if (have) {
          const uint4 out = make_uint4(pack2<F16>(y[0], y[1]), pack2<F16>(y[2], y[3]), pack2<F16>(y[4], y[5]), pack2<F16>(y[6], y[7]));
          if (!is_k) {
            *reinterpret_cast<uint4 *>(p.q_out + t * p.q_out_stride + (int64_t)(h * G + r - 1) * D + e0) = out;
          } else {
            if (p.k_out) *reinterpret_cast<uint4 *>(p.k_out + t * p.k_out_stride + (int64_t)h * D + e0) = out;
            if (write && FP8) {
              const uint2 q8 = quantise8<F16>(out, p.k_scale);
              if (has_exponent15(q8) && slot_s[tok] >= 0) atomicOr(p.special, 1u);
              *reinterpret_cast<uint2 *>(k_s + tok * D + e0) = q8;
            } else if (write) {
              *reinterpret_cast<uint4 *>(k_s + (tok * D + e0) * 2) = out;
            }
          }
        }
      }
    }
  }
  if (!write) return;
  __syncthreads();

  // ---- pool write, token index fastest across threads ---------------------------------------
  const int bs = 1 << p.bs_log;
  constexpr int X = FP8 ? 16 : 8;  // elements of a 16-byte key piece
  for (int i = tid; i < (D / X) << tok_log; i += kThreads) {
    const int wt = i & (tokens - 1), c = i >> tok_log;
    const int64_t slot = slot_s[wt];
    if (slot < 0) continue;
    const int64_t chunk = ((slot >> p.bs_log) * p.Hkv + h) * (int64_t)D << p.bs_log;
    const int off = (int)(slot & (bs - 1));
    uint8_t *dst = static_cast<uint8_t *>(p.k_pool) + (chunk + (int64_t)(c * bs + off) * X) * (FP8 ? 1 : 2);
    *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(k_s + wt * D * (FP8 ? 1 : 2) + c * 16);
  }
  for (int i = tid; i < D << tok_log; i += kThreads) {
    const int wt = i & (tokens - 1), d = i >> tok_log;
    const int64_t slot = slot_s[wt];
    if (slot < 0) continue;
    const int64_t at = (((slot >> p.bs_log) * p.Hkv + h) * (int64_t)D << p.bs_log) + (int64_t)d * bs + (slot & (bs - 1));
    if (FP8) static_cast<uint8_t *>(p.v_pool)[at] = v_s[wt * v_row + d];
    else static_cast<elem16 *>(p.v_pool)[at] = *reinterpret_cast<const elem16 *>(v_s + (wt * v_row + d) * 2);
  }
}

template <int GW, bool FP8>
cudaError_t launch_group(const RotateParams &p, bool f16, int tok_log, dim3 grid, size_t smem, cudaStream_t st) {
  const int half = p.rope.dims / 2;
  auto go = [&](auto kernel) { kernel<<<grid, kThreads, smem, st>>>(p, tok_log); };
  if (p.rope.interleaved) {
    if (f16) go(rope_norm_cache_kernel<GW, true, FP8, PAIR_LANE>);
    else go(rope_norm_cache_kernel<GW, false, FP8, PAIR_LANE>);
  } else if (half % 8 == 0) {
    if (f16) go(rope_norm_cache_kernel<GW, true, FP8, PAIR_SHUFFLE>);
    else go(rope_norm_cache_kernel<GW, false, FP8, PAIR_SHUFFLE>);
  } else {
    if (f16) go(rope_norm_cache_kernel<GW, true, FP8, PAIR_MEMORY>);
    else go(rope_norm_cache_kernel<GW, false, FP8, PAIR_MEMORY>);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope_norm_cache(const RotateParams &p, bool f16, bool fp8, int num_sms, cudaStream_t st) {
  if (p.num_tokens <= 0) return cudaSuccess;
  // about two CTAs per SM before a CTA takes more than one token
  int tok_log = 0;
  while (tok_log < 4 && (p.num_tokens * p.Hkv >> (tok_log + 1)) >= 2 * num_sms) tok_log++;
  const int tokens = 1 << tok_log, half = p.rope.dims / 2;
  const dim3 grid((unsigned)((p.num_tokens + tokens - 1) >> tok_log), (unsigned)p.Hkv);
  const size_t smem = (size_t)tokens * (((half + 1) & ~1) * 8 + (fp8 ? 2 * p.D + 8 : 4 * p.D + 4));
  cudaError_t e;
  if (fp8) e = launch_group<16, true>(p, f16, tok_log, grid, smem, st);
  else if (p.D <= 32) e = launch_group<4, false>(p, f16, tok_log, grid, smem, st);
  else if (p.D <= 64) e = launch_group<8, false>(p, f16, tok_log, grid, smem, st);
  else if (p.D <= 128) e = launch_group<16, false>(p, f16, tok_log, grid, smem, st);
  else e = launch_group<32, false>(p, f16, tok_log, grid, smem, st);
  __atomic_fetch_add(&g_launch_count, 1ull, __ATOMIC_RELAXED);
  return e;
}

}  // namespace pa
