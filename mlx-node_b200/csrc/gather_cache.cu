// Read-back of cached keys and values through block tables into packed 16-bit rows.
//
// HBM-bound: every pool byte of the ranges is read once, every row byte written once, no
// arithmetic but an FP8 cache's decode * scale.  What the layout asks for is a transpose: a value
// chunk holds the tokens of one head dimension side by side, a row the dimensions of one token.
//
// A warp takes one 16-token unit (aligned in the sequence, so that whole 16-byte pieces of the
// pool are fetched whatever the range) of one kv head, 64 dimensions at a time: all its 16-byte
// loads are issued before the first is used, 4 KB in flight per warp.  Keys go straight through: lane l
// holds piece l % 4 of token l / 4, so that loads are 128-byte lines and stores 64-byte runs.  Values
// pass through 2 KB of shared memory and come out of it by
// ldmatrix.trans, whose row addresses are permuted so that the four registers of a lane are
// eight consecutive dimensions of one token, in the same lane order as the keys.
#include "prompt_path.cuh"

namespace pa {

namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ uint4 ld_stream(const void *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Four cache bytes -> four 16-bit elements of value * scale: fp8x4_to_f16 leaves value / 256,
// exactly, and `scale256` holds 256 * scale; one rounding.
template <bool F16>
__device__ __forceinline__ uint2 dequant4(uint32_t w, float scale256) {
  uint32_t lo, hi;
  fp8x4_to_f16<true>(w, lo, hi);
  return make_uint2(pack2<F16>(elem_value<true>(lo & 0xffffu) * scale256, elem_value<true>(lo >> 16) * scale256),
                    pack2<F16>(elem_value<true>(hi & 0xffffu) * scale256, elem_value<true>(hi >> 16) * scale256));
}

// DC: head dimensions a warp has in flight (32 or 64); more are taken in turns.  64 registers, 32 warps
// on an SM in CTAs of four that come and go; stores marked streaming, as nothing here is read again.
// 8 sequences of 2000-8192 tokens, 8 heads of 128: 298 MB in 52.0 us = 5.7 TB/s (CTAs of eight warps,
// 128 dimensions, plain stores: 59.7); the FP8 ranges 247 MB in 46.7 us (57.0).
template <int DC, bool F16, bool FP8>
__global__ void __launch_bounds__(kWarps * 32, 8) gather_cache_kernel(const __grid_constant__ GatherParams p) {
  __shared__ __align__(128) uint4 v_s[kWarps][DC * 2];  // 16-byte pieces (dimension, token half)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t job = (int64_t)blockIdx.x * kWarps + warp;  // unit, then kv head
  const int unit = (int)(job / p.Hkv), h = (int)(job - (int64_t)unit * p.Hkv);
  if (unit >= p.units[p.S]) return;
  int s = 0, hi = p.S;  // the last sequence with units[s] <= unit
  while (hi - s > 1) {
    const int mid = (s + hi) >> 1;
    if (p.units[mid] <= unit) s = mid;
    else hi = mid;
  }
  const int64_t start = p.start[s], end = start + (p.cu[s + 1] - p.cu[s]);
  const int64_t tok0 = ((start >> 4) + unit - p.units[s]) * 16;
  const int bs = 1 << p.bs_log, D = p.D;
  const int32_t *table = p.block_tables + (int64_t)s * p.MB;

  // chunk and first offset of each half of the unit (blocks of 8 tokens: two chunks)
  int64_t chunk[2];
  bool have[2];
  const int off0 = (int)(tok0 & (bs - 1));
#pragma unroll
  for (int th = 0; th < 2; th++) {
    const int64_t t = tok0 + 8 * th;
    have[th] = t < end && t + 8 > start;
    chunk[th] = 0;
    if (have[th]) {
      const uint32_t id = (uint32_t)table[t >> p.bs_log];
      if (id < p.num_blocks) {
        chunk[th] = (int64_t)id * p.Hkv + h;
      } else {
        have[th] = false;
        if (lane == 0) atomicOr(p.err, kErrBlockRange);
      }
    }
  }
  const int off1 = p.bs_log == 3 ? 0 : off0 + 8;
  const int tok = lane >> 2, q = lane & 3;
  bool row_ok[2];
  elem16 *k_row[2], *v_row[2];
#pragma unroll
  for (int th = 0; th < 2; th++) {
    const int64_t t = tok0 + 8 * th + tok, row = p.cu[s] + (t - start);
    row_ok[th] = have[th] && t >= start && t < end;
    k_row[th] = p.key + row * p.key_stride + (int64_t)h * D;
    v_row[th] = p.value + row * p.value_stride + (int64_t)h * D;
  }
  const uint32_t vs = smem_u32(v_s[warp]);
  // Piece (d, half) at slot 2 d + half with bits 0 and 2 flipped by the dimension's octet: the
  // eight rows that one ldmatrix phase reads then lie in eight different 16-byte banks.
  auto v_slot = [](int d, int half) {
    const int o = (d >> 3) & 3;
    return (2 * d + half) ^ ((o & 1) | ((o & 2) << 1));
  };

  for (int d0 = 0; d0 < D; d0 += DC) {
    if constexpr (!FP8) {
      const elem16 *kp = static_cast<const elem16 *>(p.k_pool), *vp = static_cast<const elem16 *>(p.v_pool);
      uint4 k[2][DC / 32], v[DC / 16];
#pragma unroll
      for (int th = 0; th < 2; th++)
#pragma unroll
        for (int j = 0; j < DC / 32; j++) {
          const int d = d0 + j * 32 + q * 8;
          if (d < D && have[th])
            k[th][j] = ld_stream(kp + ((chunk[th] * D) << p.bs_log) + (int64_t)(d * bs) + ((th ? off1 : off0) + tok) * 8);
        }
#pragma unroll
      for (int i = 0; i < DC / 16; i++) {
        const int d = d0 + i * 16 + (lane >> 1), half = lane & 1;
        v[i] = make_uint4(0, 0, 0, 0);
        if (d < D && (half ? have[1] : have[0]))
          v[i] = ld_stream(vp + (((half ? chunk[1] : chunk[0]) * D) << p.bs_log) + (int64_t)d * bs + (half ? off1 : off0));
      }
#pragma unroll
      for (int i = 0; i < DC / 16; i++) v_s[warp][v_slot(i * 16 + (lane >> 1), lane & 1)] = v[i];
#pragma unroll
      for (int th = 0; th < 2; th++)
#pragma unroll
        for (int j = 0; j < DC / 32; j++) {
          const int d = d0 + j * 32 + q * 8;
          if (d < D && row_ok[th]) __stcs(reinterpret_cast<uint4 *>(k_row[th] + d), k[th][j]);
        }
    } else {
      const uint8_t *kp = static_cast<const uint8_t *>(p.k_pool), *vp = static_cast<const uint8_t *>(p.v_pool);
      const float ks = p.k_scale * kFp8Unbias, vsc = p.v_scale * kFp8Unbias;
      uint4 k[2][DC / 64], v[DC / 32];
#pragma unroll
      for (int th = 0; th < 2; th++)
#pragma unroll
        for (int j = 0; j < DC / 64; j++) {
          const int d = d0 + j * 64 + q * 16;
          if (have[th])
            k[th][j] = ld_stream(kp + ((chunk[th] * D) << p.bs_log) + (int64_t)d * bs + ((th ? off1 : off0) + tok) * 16);
        }
#pragma unroll
      for (int i = 0; i < DC / 32; i++) {
        const int d = d0 + i * 32 + lane;
        v[i] = make_uint4(0, 0, 0, 0);
        // FP8 blocks have 16 or 32 tokens: a unit's 16 bytes are in one chunk
        if (have[0] || have[1])
          v[i] = ld_stream(vp + (((have[0] ? chunk[0] : chunk[1]) * D) << p.bs_log) + (int64_t)d * bs + off0);
      }
#pragma unroll
      for (int i = 0; i < DC / 32; i++) {
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const uint2 a = dequant4<F16>(w[2 * half], vsc), b = dequant4<F16>(w[2 * half + 1], vsc);
          v_s[warp][v_slot(i * 32 + lane, half)] = make_uint4(a.x, a.y, b.x, b.y);
        }
      }
#pragma unroll
      for (int th = 0; th < 2; th++)
#pragma unroll
        for (int j = 0; j < DC / 64; j++)
          if (row_ok[th]) {
            elem16 *dst = k_row[th] + d0 + j * 64 + q * 16;
            const uint2 a = dequant4<F16>(k[th][j].x, ks), b = dequant4<F16>(k[th][j].y, ks),
                        c = dequant4<F16>(k[th][j].z, ks), e = dequant4<F16>(k[th][j].w, ks);
            __stcs(reinterpret_cast<uint4 *>(dst), make_uint4(a.x, a.y, b.x, b.y));
            __stcs(reinterpret_cast<uint4 *>(dst + 8), make_uint4(c.x, c.y, e.x, e.y));
          }
    }
    __syncwarp();
    // matrix m, row r of a load: dimension (r / 2) * 8 + 2 m + r % 2 of the 32, so that register m
    // of lane (tok, q) is dimensions 8 q + 2 m and 8 q + 2 m + 1 of token tok
    const int r = lane & 7, dm = (r >> 1) * 8 + (lane >> 3) * 2 + (r & 1);
#pragma unroll
    for (int th = 0; th < 2; th++)
#pragma unroll
      for (int j = 0; j < DC / 32; j++) {
        uint32_t w[4];
        ldmatrix_x4_trans(w, vs + v_slot(j * 32 + dm, th) * 16);
        const int d = d0 + j * 32 + q * 8;
        if (d < D && row_ok[th]) __stcs(reinterpret_cast<uint4 *>(v_row[th] + d), make_uint4(w[0], w[1], w[2], w[3]));
      }
    __syncwarp();
  }
}

}  // namespace

cudaError_t launch_gather_cache(const GatherParams &p, bool f16, bool fp8, cudaStream_t st) {
  const int64_t jobs = (int64_t)p.units[p.S] * p.Hkv;
  if (jobs <= 0) return cudaSuccess;
  if ((jobs + kWarps - 1) / kWarps > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const unsigned grid = (unsigned)((jobs + kWarps - 1) / kWarps);
  if (fp8 && f16) gather_cache_kernel<64, true, true><<<grid, kWarps * 32, 0, st>>>(p);
  else if (fp8) gather_cache_kernel<64, false, true><<<grid, kWarps * 32, 0, st>>>(p);
  else if (p.D <= 32) gather_cache_kernel<32, false, false><<<grid, kWarps * 32, 0, st>>>(p);
  else gather_cache_kernel<64, false, false><<<grid, kWarps * 32, 0, st>>>(p);
  __atomic_fetch_add(&g_launch_count, 1ull, __ATOMIC_RELAXED);
  return cudaGetLastError();
}

}  // namespace pa
