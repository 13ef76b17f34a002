// Launch parameters of the prompt-path kernels: rotation + cache write (rope_producer.cu),
// cache read-back (gather_cache.cu) and packed prompt attention (prompt_attention.cu).
#pragma once
#include "pa_common.cuh"
#include "prompt_host.hpp"

namespace pa {

struct RotateParams {
  const elem16 *q, *k, *v;
  elem16 *q_out, *k_out;                 // k_out may be null
  const elem16 *q_norm_w, *k_norm_w;     // null: no norm
  const int32_t *positions;
  const int64_t *slot_mapping;           // null: no cache write
  void *k_pool, *v_pool;
  int64_t num_tokens, q_stride, q_out_stride, k_stride, k_out_stride, v_stride;
  int Hq, Hkv, D;
  int bs_log;                            // log2 of the pool's block size
  uint32_t num_blocks;
  float eps;
  float k_scale, v_scale;                // FP8 pools
  unsigned *err, *special;
  RopeTable rope;
};
cudaError_t launch_rope_norm_cache(const RotateParams &p, bool f16, bool fp8, int num_sms, cudaStream_t st);

// Ranges of up to kMaxPlanSeqs sequences of one read-back launch.
struct GatherParams {
  const void *k_pool, *v_pool;
  elem16 *key, *value;
  const int32_t *block_tables;           // row 0 = the launch's first sequence
  int64_t key_stride, value_stride;
  int Hkv, D, MB, S;
  int bs_log;
  uint32_t num_blocks;
  float k_scale, v_scale;
  unsigned *err;
  int32_t start[kMaxPlanSeqs];           // first token of each range
  int32_t cu[kMaxPlanSeqs + 1];          // output rows
  int32_t units[kMaxPlanSeqs + 1];       // 16-token units (aligned in the sequence) before each sequence
};
cudaError_t launch_gather_cache(const GatherParams &p, bool f16, bool fp8, cudaStream_t st);

struct PromptParams {
  elem16 *out;
  const elem16 *q, *k, *v;
  int64_t q_stride, k_stride, v_stride, out_stride;
  int Hq, Hkv, G, D, S;
  float scale, softcap;
  int32_t cu_q[kMaxPlanSeqs + 1], cu_kv[kMaxPlanSeqs + 1];
};
size_t prompt_workspace_bytes(int num_sms, int head_size);
// Sequences [0, p.S) with the plan of their work.
cudaError_t launch_prompt_attention(const PromptParams &p, bool f16, int num_sms, void *workspace,
                                    unsigned *err, cudaStream_t st);
cudaError_t prompt_configure();

template <bool F16>
__device__ __forceinline__ float elem_value(uint32_t bits16) {
  if (F16) {
    float f;
    asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"((uint16_t)bits16));
    return f;
  }
  return __uint_as_float(bits16 << 16);
}

}  // namespace pa
