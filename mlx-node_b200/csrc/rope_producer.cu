// Per-head RMS norm of queries and keys, rotation by a plan and cache write, for every head
// size, block size and cache type of the library.
//
//   y = x * w / sqrt(mean(x^2) + eps)            (no norm: y = x)
//   (a, b) -> g (a cos t - b sin t, b cos t + a sin t),  t = position * f_i
//
// A row stays in fp32 from the load to the one rounding to the 16-bit type.  The phase is
// position * turn[i] modulo 2^64 in units of 2^-64 turns (RopeTable): reduced exactly, its top
// 32 bits as a signed number are the angle within half a turn.
#include "prompt_path.cuh"

namespace pa {

namespace {

// One CTA per (token, kv head): a warp per row.
template <bool F16, bool FP8>
__global__ void __launch_bounds__(128) rope_norm_cache_kernel(const RotateParams p) {
  __shared__ float2 cs[kMaxRopePairs];
  __shared__ float row_s[4][256];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = p.D, half = p.rope.dims >> 1, G = p.Hq / p.Hkv;
  for (int i = tid; i < half; i += 128) {
    const uint64_t phase = (uint64_t)(int64_t)p.positions[t] * p.rope.turn[i];
    float sn, cn;
    sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &sn, &cn);
    cs[i] = make_float2(cn * p.rope.gain, sn * p.rope.gain);
  }
  int64_t slot = -1;
  if (p.slot_mapping) {
    slot = p.slot_mapping[t];
    if (slot >= ((int64_t)p.num_blocks << p.bs_log)) {
      if (tid == 0) atomicOr(p.err, kErrSlotRange);
      slot = -1;
    }
  }
  const int64_t blk = slot >> p.bs_log;
  const int off = (int)(slot & ((1 << p.bs_log) - 1));
  __syncthreads();
  constexpr int X = FP8 ? 16 : 8;
  auto pool_k = [&](int d) { return (((blk * p.Hkv + h) * (int64_t)(D / X) + d / X) << p.bs_log) * X + off * X + d % X; };
  auto pool_v = [&](int d) { return (((blk * p.Hkv + h) * (int64_t)D + d) << p.bs_log) + off; };
  auto quant = [&](uint32_t bits, float scale) -> uint32_t {
    const uint32_t b = quantise8<F16>(make_uint4(bits, 0, 0, 0), scale).x & 0xffu;
    if ((b & 0x78u) == 0x78u) atomicOr(p.special, 1u);
    return b;
  };
  for (int r = warp; r <= G + 1; r += 4) {
    if (r == G + 1) {
      if (slot >= 0)
        for (int d = lane; d < D; d += 32) {
          const uint32_t e = p.v[t * p.v_stride + (int64_t)h * D + d];
          if (FP8) static_cast<uint8_t *>(p.v_pool)[pool_v(d)] = (uint8_t)quant(e, p.v_scale);
          else static_cast<elem16 *>(p.v_pool)[pool_v(d)] = (elem16)e;
        }
      break;
    }
    const bool is_k = r == 0;
    const elem16 *src = is_k ? p.k + t * p.k_stride + (int64_t)h * D : p.q + t * p.q_stride + (int64_t)(h * G + r - 1) * D;
    const elem16 *w = is_k ? p.k_norm_w : p.q_norm_w;
    float ss = 0.f;
    for (int d = lane; d < D; d += 32) {
      const float x = elem_value<F16>(src[d]);
      row_s[warp][d] = x;
      ss += x * x;
    }
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = 1.0f / sqrtf(ss / D + p.eps);
    __syncwarp();
    if (w)
      for (int d = lane; d < D; d += 32) row_s[warp][d] *= inv * elem_value<F16>(w[d]);
    __syncwarp();
    for (int d = lane; d < D; d += 32) {
      float y = row_s[warp][d];
      if (d < 2 * half) {
        const int i = p.rope.interleaved ? d >> 1 : (d < half ? d : d - half);
        const bool second = p.rope.interleaved ? d & 1 : d >= half;
        const float o = row_s[warp][p.rope.interleaved ? d ^ 1 : (second ? d - half : d + half)];
        y = second ? y * cs[i].x + o * cs[i].y : y * cs[i].x - o * cs[i].y;
      }
      const elem16 e = to_elem<F16>(y);
      if (!is_k) {
        p.q_out[t * p.q_out_stride + (int64_t)(h * G + r - 1) * D + d] = e;
      } else {
        if (p.k_out) p.k_out[t * p.k_out_stride + (int64_t)h * D + d] = e;
        if (slot >= 0) {
          if (FP8) static_cast<uint8_t *>(p.k_pool)[pool_k(d)] = (uint8_t)quant(e, p.k_scale);
          else static_cast<elem16 *>(p.k_pool)[pool_k(d)] = e;
        }
      }
    }
    __syncwarp();
  }
}

}  // namespace

cudaError_t launch_rope_norm_cache(const RotateParams &p, bool f16, bool fp8, int num_sms, cudaStream_t st) {
  (void)num_sms;
  if (p.num_tokens <= 0) return cudaSuccess;
  const dim3 grid((unsigned)p.num_tokens, (unsigned)p.Hkv);
  if (f16 && fp8) rope_norm_cache_kernel<true, true><<<grid, 128, 0, st>>>(p);
  else if (f16) rope_norm_cache_kernel<true, false><<<grid, 128, 0, st>>>(p);
  else if (fp8) rope_norm_cache_kernel<false, true><<<grid, 128, 0, st>>>(p);
  else rope_norm_cache_kernel<false, false><<<grid, 128, 0, st>>>(p);
  __atomic_fetch_add(&g_launch_count, 1ull, __ATOMIC_RELAXED);
  return cudaGetLastError();
}

}  // namespace pa
