// Causal attention of packed prompts over contiguous keys and values.
#include "prompt_path.cuh"

namespace pa {

namespace {

// One row - a (query token, query head) - by one warp: 32 keys at a time, a lane per key for
// the logits, the online softmax across the warp, then a lane per D/32 output dimensions.
template <bool F16>
__device__ void attend_row(const PromptParams &p, int s, int token, int head, elem16 *out) {
  const int lane = threadIdx.x & 31, D = p.D, h = head / p.G;
  const int q_len = p.cu_q[s + 1] - p.cu_q[s], kv_len = p.cu_kv[s + 1] - p.cu_kv[s];
  const int keys = kv_len - q_len + token + 1;
  const elem16 *q = p.q + (int64_t)(p.cu_q[s] + token) * p.q_stride + (int64_t)head * D;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int j0 = 0; j0 < keys; j0 += 32) {
    const int j = j0 + lane;
    float x = -INFINITY;
    if (j < keys) {
      const elem16 *k = p.k + (int64_t)(p.cu_kv[s] + j) * p.k_stride + (int64_t)h * D;
      float dot = 0.f;
      for (int d = 0; d < D; d += 8) {
        const uint4 a = *reinterpret_cast<const uint4 *>(q + d), b = *reinterpret_cast<const uint4 *>(k + d);
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          dot = fmaf(elem_value<F16>(aw[i] & 0xffffu), elem_value<F16>(bw[i] & 0xffffu), dot);
          dot = fmaf(elem_value<F16>(aw[i] >> 16), elem_value<F16>(bw[i] >> 16), dot);
        }
      }
      x = dot * p.scale;
      if (p.softcap != 1.0f) x = tanhf(x / p.softcap) * p.softcap;
    }
    float mx = x;
    for (int i = 16; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
    const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.f : m_new;
    const float keep = m == -INFINITY ? 0.f : expf(m - base);
    const float w = j < keys ? expf(x - base) : 0.f;
    float sum = w;
    for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    l = l * keep + sum;
    m = m_new;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] *= keep;
    for (int jj = 0; jj < 32 && j0 + jj < keys; jj++) {
      const float wj = __shfl_sync(0xffffffffu, w, jj);
      const elem16 *v = p.v + (int64_t)(p.cu_kv[s] + j0 + jj) * p.v_stride + (int64_t)h * D;
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i * 32 + lane < D) o[i] = fmaf(wj, elem_value<F16>(v[i * 32 + lane]), o[i]);
    }
  }
  const float inv = keys > 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i * 32 + lane < D) out[i * 32 + lane] = to_elem<F16>(keys > 0 ? o[i] * inv : 0.f);
}

template <bool F16>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const PromptParams p) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t total = (int64_t)(p.cu_q[p.S] - p.cu_q[0]) * p.Hq;
  if (row >= total) return;
  const int t = p.cu_q[0] + (int)(row / p.Hq), head = (int)(row % p.Hq);
  int lo = 0, hi = p.S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid] <= t) lo = mid;
    else hi = mid;
  }
  attend_row<F16>(p, lo, t - p.cu_q[lo], head, p.out + (int64_t)t * p.out_stride + (int64_t)head * p.D);
}

}  // namespace

size_t prompt_workspace_bytes(int num_sms, int head_size) {
  const size_t rows = head_size <= 128 ? 256 : 128;
  return (size_t)2 * std::min(num_sms, kMaxPlanCtas) * rows * (head_size + 2) * 4;
}
cudaError_t prompt_configure() { return cudaSuccess; }

cudaError_t launch_prompt_attention(const PromptParams &p, bool f16, int num_sms, void *workspace, unsigned *err,
                                    cudaStream_t st) {
  (void)num_sms, (void)workspace, (void)err;
  const int64_t rows = (int64_t)(p.cu_q[p.S] - p.cu_q[0]) * p.Hq;
  if (rows <= 0) return cudaSuccess;
  const unsigned grid = (unsigned)((rows + 3) / 4);
  if (f16) prompt_rows_kernel<true><<<grid, 128, 0, st>>>(p);
  else prompt_rows_kernel<false><<<grid, 128, 0, st>>>(p);
  __atomic_fetch_add(&g_launch_count, 1ull, __ATOMIC_RELAXED);
  return cudaGetLastError();
}

}  // namespace pa
