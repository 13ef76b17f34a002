// Read-back of cached keys and values through block tables into packed 16-bit rows.
#include "prompt_path.cuh"

namespace pa {

namespace {

// A cache byte's value: exponent field 15 is infinity (mantissa 0) or NaN, field 0 subnormal.
__device__ __forceinline__ float fp8_value(uint32_t b) {
  const uint32_t e = (b >> 3) & 15u, m = b & 7u;
  float f = e == 0 ? m * 0x1p-9f
                   : e == 15 ? (m ? __uint_as_float(0x7FC00000u) : INFINITY)
                             : __uint_as_float((e + 120u) << 23 | m << 20);
  return b & 0x80u ? -f : f;
}

// One CTA per (16-token unit, kv head): a thread per element.
template <bool F16, bool FP8>
__global__ void __launch_bounds__(256) gather_cache_kernel(const GatherParams p) {
  const int h = blockIdx.y, unit = blockIdx.x;
  int lo = 0, hi = p.S;  // the last sequence with units[s] <= unit
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.units[mid] <= unit) lo = mid;
    else hi = mid;
  }
  const int s = lo, len = p.cu[s + 1] - p.cu[s], start = p.start[s];
  const int64_t tok0 = ((int64_t)(start >> 4) + unit - p.units[s]) * 16;
  constexpr int X = FP8 ? 16 : 8;
  for (int e = threadIdx.x; e < 16 * p.D; e += 256) {
    const int64_t tok = tok0 + e / p.D;
    const int d = e % p.D;
    if (tok < start || tok >= (int64_t)start + len) continue;
    const uint32_t blk = (uint32_t)p.block_tables[(int64_t)s * p.MB + (tok >> p.bs_log)];
    if (blk >= p.num_blocks) {
      atomicOr(p.err, kErrBlockRange);
      continue;
    }
    const int off = (int)(tok & ((1 << p.bs_log) - 1));
    const int64_t chunk = (int64_t)blk * p.Hkv + h;
    const int64_t ki = ((chunk * (p.D / X) + d / X) << p.bs_log) * X + off * X + d % X;
    const int64_t vi = ((chunk * p.D + d) << p.bs_log) + off;
    const int64_t row = p.cu[s] + (tok - start);
    elem16 k, v;
    if (FP8) {
      k = to_elem<F16>(fp8_value(static_cast<const uint8_t *>(p.k_pool)[ki]) * p.k_scale);
      v = to_elem<F16>(fp8_value(static_cast<const uint8_t *>(p.v_pool)[vi]) * p.v_scale);
    } else {
      k = static_cast<const elem16 *>(p.k_pool)[ki];
      v = static_cast<const elem16 *>(p.v_pool)[vi];
    }
    p.key[row * p.key_stride + (int64_t)h * p.D + d] = k;
    p.value[row * p.value_stride + (int64_t)h * p.D + d] = v;
  }
}

}  // namespace

cudaError_t launch_gather_cache(const GatherParams &p, bool f16, bool fp8, cudaStream_t st) {
  if (p.units[p.S] <= 0) return cudaSuccess;
  const dim3 grid((unsigned)p.units[p.S], (unsigned)p.Hkv);
  if (fp8 && f16) gather_cache_kernel<true, true><<<grid, 256, 0, st>>>(p);
  else if (fp8) gather_cache_kernel<false, true><<<grid, 256, 0, st>>>(p);
  else gather_cache_kernel<false, false><<<grid, 256, 0, st>>>(p);
  __atomic_fetch_add(&g_launch_count, 1ull, __ATOMIC_RELAXED);
  return cudaGetLastError();
}

}  // namespace pa
