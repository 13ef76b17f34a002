// Causal attention of packed prompts over contiguous keys and values: tcgen05 tensor cores,
// accumulators in TMEM, every operand brought in by tensor-map copies, sm_100a.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i k_j - m_i),  j <= kv_len - q_len + i
//
// with m_i any number near the row's largest logit (it cancels).  One pass over the keys: reference
// and running sum are kept in fp32 per row, the reference in units of log2.  It is the maximum of
// the first tile, and stale after that: a tile's probabilities are taken against the reference of
// the tiles before it, and it moves - before the next tile - only when the tile's sum of
// probabilities exceeded 2^8, by log2 of that sum, which is the tile's maximum plus seven at most.
// So no maximum is taken in the loop, and the accumulator is rarely rescaled.
// Probabilities are rounded to the 16-bit type because the tensor cores take both operands of
// P.V in one 16-bit type; their sum is taken before the rounding.
//
// Work: an item is up to 256 rows of one (sequence, kv head), a row being a (query token, head
// of the group) pair, so that every key tile is read once for the whole group: two 128-row
// query tiles that share each 128-key tile (head sizes above 128: one query tile, the
// accumulator takes all the columns two would).  An item of one query tile - single tokens, drafts,
// the end of a prompt - gives the second tile's place to every other key tile: two accumulators with
// references of their own, added at the end, so that the tensor cores and the softmax overlap there
// too.  The line of items is cut into one piece of
// equal cost per CTA (plan_prompt); an item that a cut splits leaves fp32 partial results in
// the workspace, joined in CTA order by prompt_join_kernel, so that few rows over long keys
// use every SM and the same call gives the same bits.
//
// Roles (warps):
//   8 per query tile  softmax: two threads per row, each 64 of a tile's 128 logits, so that a
//                     scheduler has two warps of a tile in flight while the other query tile
//                     is in the tensor cores.  The two tell each other their sums through
//                     shared memory and read them a tile later, when the barriers of the P.V in
//                     between have ordered them: no barrier of their own
//   1                 copies: Q per item, K and V tiles into two rings
//   1                 issues every tcgen05.mma (two more idle: register budgets move between
//                     warpgroups of four)
// TMEM (512 columns): logits S0 | S1 (128 each), outputs O0 | O1.  P overwrites the first half
// of the thread's own logit columns and is the A operand of O += P.V.
// K tiles and Q are K-major with the 128-byte swizzle; a V tile lands the same way - rows of
// tokens - and is read as an MN-major B operand, so nothing is transposed on the way.
//
// S_i(j+1) overwrites P_i(j), and the tensor cores order only MMAs of one accumulator and
// shape, so it is issued after P_i(j).V(j) has signalled completion; the other query tile's
// work fills the pipe meanwhile.
//
// A probability of a masked key is exactly 0, but 0 * NaN is NaN: a row whose result is not
// finite is checked for masked values that are not, and then recomputed by itself over the keys
// that it sees (repair_row).  So is a bf16 row that is not finite after a sum above 2^16 (a logit
// 11 above everything in the tiles before); a sum that overflows makes its row NaN (reciprocal).  The check
// costs a comparison per output element.
//
// That recomputation is one warp's scalar work and slow: 0.78 s for a row of a million keys of 256
// dimensions, and where every row of a prompt of 4096 (8 heads of 128) jumps by 100 nats, 271 ms instead of
// 62 us.  It takes jumps of 84 to 88.7 nats - the sum's or a probability's exponent - and more over everything before
// in the row, or a NaN or infinity in a value that the row's last key tiles hold and the row does not see.  f16 jumps are settled in the
// loop (redo_tile).
//
// Bound by the chain of one query tile (S - softmax - P.V - S), 3200 cycles per 128 keys of both
// query tiles against 2350 of tensor pipe; measured on several B200s, with the same and
// with changing inputs: 8192-token prompt, 32/8 heads of 128, bf16, 467-550 us (1.0-1.18 PFLOP/s); seven f16 prompts of 700-2500 260-311 us; two
// chunks of 1024 over 4096 160-173 us; eight sequences of 1-5 tokens over 4000-16000 keys 75-81 us (4.4-4.8 TB/s).
// The 8192-token prompt in other forms: f16 530 us, softcap 1230 (a tanhf per logit), head size 64 412 us, 16/4
// heads of 192 429 and of 256 517 (f16 613).  The two-tile kernels hold 96 registers a thread and spill: 20 bytes
// of reloads in bf16, 136 in f16, which keeps what redo_tile needs.
//
// Every wait is bounded; on expiry the CTA raises the error word, every role leaves its loop,
// copies in flight are drained and TMEM is freed.
#include <cuda.h>

#include <type_traits>

#include "prompt_path.cuh"
#include "tile_common.cuh"

namespace pa {

namespace {

using namespace tile;

constexpr int kBox = 128 * 128;  // one operand slab: 128 rows x 64 elements

template <int NBOX>
struct Geo {
  static constexpr int QT = NBOX <= 2 ? 2 : 1;          // query tiles of an item
  static constexpr int NK = NBOX == 1 ? 5 : NBOX <= 3 ? 2 : 1;  // ring depths, tiles of NBOX slabs
  static constexpr int NV = NBOX == 1 ? 5 : NBOX == 2 ? 2 : 1;
  static constexpr int kTile = NBOX * kBox;
  static constexpr int kSoft = 8 * QT;                  // softmax warps
  static constexpr int kThreads = (kSoft + 4) * 32;     // whole warpgroups
  static constexpr int B_QFULL = 0, B_QEMPTY = 1, B_KFULL = 2, B_KEMPTY = B_KFULL + NK, B_VFULL = B_KEMPTY + NK,
                       B_VEMPTY = B_VFULL + NV, B_SFULL = B_VEMPTY + NV, B_PREADY = B_SFULL + QT,
                       B_PHALF = B_PREADY + QT, B_PVDONE = B_PHALF + QT, kBars = B_PVDONE + QT;
  static constexpr int kXch = 5 * QT * 2 * 128 * 4;     // [slot][query tile][half][row] floats
  static constexpr int kWalk = kThreads / 32 * 16;       // a PlanPos per warp
  static constexpr int kWords = 8 * QT * 4 + 16;        // a meeting word per softmax warp, the beat
  static constexpr int kSmem = 1024 + (QT + NK + NV) * kTile + kXch + kWalk + kWords + kBars * 8 + 16;
  static_assert(kSmem <= 232448, "shared memory per CTA");
};

struct PromptLaunch {
  PromptParams p;
  PlanPos begin[kMaxPlanCtas + 1];
  float *ws;       // two partial slots per CTA, each [D + 3][128 * QT] floats: O, reference, sum, far
  unsigned *err;
  int32_t sub_tokens, tile_tokens;
};

// Where a CTA is on the line of items; every role walks it for itself.
struct Seg {
  int s, h, qt, kt0, kt1, n;  // key tiles [kt0, kt1) of the item's n
  int q_len, kv_len, q0, tiles;
};
// The position lives in shared memory, one per warp: it is touched once per item and would
// otherwise hold registers through the softmax.
template <bool WARP>  // a whole warp walks, or one lane
__device__ __forceinline__ bool walk_next(const PromptLaunch &L, PlanPos *at, Seg &g) {
  if (WARP) __syncwarp();
  struct {
    PlanPos p, e;
  } w = {*at, L.begin[blockIdx.x + 1]};
  if (w.p.seq == w.e.seq && w.p.head == w.e.head && w.p.qt == w.e.qt && w.p.kt >= w.e.kt) return false;
  g.s = w.p.seq;
  g.h = w.p.head;
  g.qt = w.p.qt;
  g.q_len = L.p.cu_q[g.s + 1] - L.p.cu_q[g.s];
  g.kv_len = L.p.cu_kv[g.s + 1] - L.p.cu_kv[g.s];
  g.q0 = g.qt * L.tile_tokens;
  const int q1 = min(g.q_len, g.q0 + L.tile_tokens);
  g.tiles = q1 - g.q0 > L.sub_tokens ? 2 : 1;
  const int keys = max(g.kv_len - g.q_len + q1, 0);
  g.n = (keys + kKeyTile - 1) / kKeyTile;
  g.kt0 = w.p.kt;
  const bool cut = w.e.seq == g.s && w.e.head == g.h && w.e.qt == g.qt;
  g.kt1 = cut ? w.e.kt : g.n;
  w.p.kt = 0;
  if (cut) {
    w.p = w.e;
  } else if (q1 < g.q_len) {
    w.p.qt++;
  } else {
    w.p.qt = 0;
    if (++w.p.head == L.p.Hkv) {
      w.p.head = 0;
      for (w.p.seq++; w.p.seq < L.p.S && L.p.cu_q[w.p.seq + 1] == L.p.cu_q[w.p.seq];) w.p.seq++;
    }
  }
  if (WARP) __syncwarp();  // every lane has read it
  *at = w.p;
  return true;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle (layout 2, version 1).  The low word holds the
// address and the leading byte offset, both in units of 16 bytes, so that a step along an operand is
// an addition to it.  Q and K: K-major, groups of 8 rows 1024 B apart.  A V tile as the B operand of
// P.V: MN-major (the head dimension contiguous), slabs of 64 dimensions kBox apart, groups of 8 tokens
// 1024 B apart.
constexpr uint32_t kDescHigh = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t k_major_low(uint32_t smem_addr) { return ((smem_addr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint32_t mn_major_low(uint32_t smem_addr) {
  return ((smem_addr >> 4) & 0x3FFFu) | ((uint32_t)(kBox >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(kDescHigh), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
      "r"(a_tmem), "r"(b_low), "r"(kDescHigh), "r"(idesc), "r"(acc)
      : "memory");
}
// fp32 accumulator, M = 128; bit 16: B is MN-major
__device__ __forceinline__ uint32_t mma_desc(bool f16, uint32_t n, bool b_mn) {
  return (1u << 4) | (f16 ? 0u : ((1u << 7) | (1u << 10))) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// wait_bar with a second chance: a softmax warp that recomputes rows by itself (repair_row) counts them
// in `beat`, and the roles that wait for it meanwhile start their second anew with every count.
__device__ __forceinline__ bool wait_live(uint32_t bar, uint32_t parity, volatile int *abort_flag, volatile uint32_t *beat) {
  if (mbar_try_wait(bar, parity)) return true;
  long long t0 = clock64();
  uint32_t seen = *beat;
  int spins = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++spins & 63) == 0) {
      if (*abort_flag) return false;
      if (*beat != seen) {
        seen = *beat;
        t0 = clock64();
      } else if (clock64() - t0 > (1ll << 31)) {
        *abort_flag = 1;
        return false;
      }
    }
  }
  return true;
}

__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// Dynamic shared memory from its first 1024-byte line on, and in it the meeting words of the softmax warps; the beat
// follows them.
__device__ __forceinline__ uint8_t *aligned_smem() {
  extern __shared__ uint8_t smem_raw[];
  return smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
}
template <int NBOX>
__device__ __forceinline__ uint32_t *meeting_words() {
  using Z = Geo<NBOX>;
  return reinterpret_cast<uint32_t *>(aligned_smem() + (Z::QT + Z::NK + Z::NV) * Z::kTile + Z::kXch + Z::kWalk);
}

// One row - a (query token, query head) - by one warp over exactly the keys it sees: 32 keys
// at a time, a lane per key for the logits, the online softmax across the warp, then a lane per
// output dimension.  Writes the 8-column pieces whose bit is set in `pieces`; counts every 16384 keys in
// the beat of a CTA of Geo<NBOX> (0: nobody waits), as millions of keys take longer than a wait's second.
// (The beat's place is found again here: handed over as an argument it cost the f16 loop registers, 380 instead of
// 136 bytes of reloads and 305 instead of 300 us on packed prompts.)
template <bool F16, int NBOX>
__device__ __noinline__ void repair_row(const PromptParams &p, int s, int token, int head, uint32_t pieces) {
  const int lane = threadIdx.x & 31, D = p.D, h = head / p.G;
  const int q_len = p.cu_q[s + 1] - p.cu_q[s], kv_len = p.cu_kv[s + 1] - p.cu_kv[s];
  const int keys = kv_len - q_len + token + 1;
  const elem16 *q = p.q + (int64_t)(p.cu_q[s] + token) * p.q_stride + (int64_t)head * D;
  elem16 *out = p.out + (int64_t)(p.cu_q[s] + token) * p.out_stride + (int64_t)head * D;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int j0 = 0; j0 < keys; j0 += 32) {
    if constexpr (NBOX > 0)
      if ((j0 & 16383) == 0 && lane == 0) atomicAdd(meeting_words<NBOX>() + 8 * Geo<NBOX>::QT, 1u);
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
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: zeros; NaN stays
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i * 32 + lane < D && (pieces >> (i * 4 + (lane >> 3)) & 1u)) out[i * 32 + lane] = to_elem<F16>(o[i] * inv);
}

// Whether a value outside the keys that a row sees, but inside the key tiles that its item
// reads, is not finite (the tiles run on into the rows of the next sequences).
__device__ __noinline__ bool masked_value_not_finite(const PromptParams &p, int s, int token, int h, int n_tiles, bool f16) {
  const int lane = threadIdx.x & 31;
  const int q_len = p.cu_q[s + 1] - p.cu_q[s], kv_len = p.cu_kv[s + 1] - p.cu_kv[s];
  const int first = max(kv_len - q_len + token + 1, 0);
  const int64_t end = min((int64_t)n_tiles * kKeyTile, (int64_t)p.cu_kv[p.S] - p.cu_kv[s]);
  const uint32_t top = f16 ? 0x7C00u : 0x7F80u;  // the exponent of infinity and NaN
  bool bad = false;
  for (int64_t j = first; j < end; j++) {
    const elem16 *v = p.v + (p.cu_kv[s] + j) * p.v_stride + (int64_t)h * p.D;
    for (int d = lane; d < p.D; d += 32) bad |= (v[d] & top) == top;
  }
  return __any_sync(0xffffffffu, bad);
}

// f16: the rare case that a logit of the current tile is so far above the reference that its probability
// would leave the type's range: the two warps of a set
// of rows meet and settle on the tile's own maximum before the tile's P.V may start.  One of them
// found the case before it stored its probabilities and takes them again from the logits; the other
// may have stored and announced its own (`stored`) and scales those.  Neither can run ahead: P.V
// waits for the first one's announcement.  The meetings are words in shared memory with a bounded
// wait, so that a CTA that has given up elsewhere does not hang here.
struct Redo {
  float ref, l, sum;
};
__device__ __forceinline__ void redo_meet(uint32_t mine, uint32_t other, uint32_t stamp, volatile int *abort_flag) {
  __threadfence_block();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(mine), "r"(stamp) : "memory");
  const long long t0 = clock64();
  for (;;) {
    uint32_t w;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(w) : "r"(other) : "memory");
    if (__all_sync(0xffffffffu, (int)(w - stamp) >= 0 || *abort_flag)) break;
    if (clock64() - t0 > (1ll << 31)) *abort_flag = 1;
  }
  __threadfence_block();
  __syncwarp();
}
// 32-column chunks of O: the first half of them is one thread's of a row, the rest the other's.
__device__ __forceinline__ int chunk_begin(int D, int half) { return half ? (((D + 31) >> 5) + 1) >> 1 : 0; }
__device__ __forceinline__ int chunk_end(int D, int half) { return half ? (D + 31) >> 5 : (((D + 31) >> 5) + 1) >> 1; }

// 1 / x of a sum of probabilities, NaN for one that has left fp32: bf16 sums may, with every probability and
// weighted sum inside it still, and 1 / inf = 0 would turn the row into zeros that look like a result.  NaN
// sticks to the row's sum and reaches every column of it, whatever later tiles, places and pieces add, and the row is
// recomputed at the end.
__device__ __forceinline__ float reciprocal(float x) { return 1.f / x + (x - x); }

// O of this half's columns, times a factor per row.
__device__ __forceinline__ void scale_o(uint32_t o_t, int D, int half, float factor) {
#pragma unroll 1
  for (int ch = chunk_begin(D, half); ch < chunk_end(D, half); ch++) {
    uint32_t r[32];
    tmem_ld32(o_t + ch * 32, r);
    tmem_wait_ld32(r);
#pragma unroll
    for (int e = 0; e < 32; e++) r[e] = __float_as_uint(__uint_as_float(r[e]) * factor);
    tmem_st32(o_t + ch * 32, r);
  }
}
template <bool CAP, bool F16>
__device__ __noinline__ Redo redo_tile(uint32_t s_t, uint32_t o_t, int D, int half, float c, float cap_in, float cap_out, float ref,
                                       float l, float sum, uint32_t sum_slot, uint32_t mx_slot, uint32_t l_slot, uint32_t word_mine, uint32_t stamp, bool valid,
                                       bool stored, bool rescale, int left, volatile int *abort_flag) {
  auto logits = [&](int ch, uint32_t (&r)[16]) {
    tmem_ld16(s_t + ch * 16, r);
    tmem_wait_ld16(r);
#pragma unroll
    for (int e = 0; e < 16; e++) {
      float x = __uint_as_float(r[e]);
      if (CAP) x = tanhf(x * cap_in) * cap_out;
      r[e] = __float_as_uint(ch * 16 + e >= left ? -INFINITY : x * c);
    }
  };
  // how far this half is above the reference: its maximum, or what its sum says of it
  float mx = -INFINITY;
  if (stored) {
    mx = ref + log2f(sum);
  } else {
#pragma unroll 1
    for (int ch = 0; ch < 4; ch++) {
      uint32_t r[16];
      logits(ch, r);
#pragma unroll
      for (int e = 0; e < 16; e++) mx = fmaxf(mx, __uint_as_float(r[e]));
    }
  }
  // (the slot of the tile before: both warps have read it)
  asm volatile("st.volatile.shared.f32 [%0], %1;" ::"r"(mx_slot), "f"(mx) : "memory");
  redo_meet(word_mine, word_mine ^ 16, stamp, abort_flag);
  float theirs;
  asm volatile("ld.volatile.shared.f32 %0, [%1];" : "=f"(theirs) : "r"(mx_slot ^ 512) : "memory");
  const float to = fmaxf(ref, fmaxf(mx, theirs));
  float factor = 1.f;
  if (valid && to > ref) {
    factor = fast_exp2(ref - to);
    ref = to;
  }
  if (rescale) scale_o(o_t, D, half, factor);
  if (stored) {
    uint32_t r[32];
    tmem_ld32(s_t, r);
    tmem_wait_ld32(r);
#pragma unroll
    for (int e = 0; e < 32; e++)
      r[e] = pack2<F16>(elem_value<F16>(r[e] & 0xffffu) * factor, elem_value<F16>(r[e] >> 16) * factor);
    tmem_st32(s_t, r);
    sum *= factor;
  } else {
    sum = 0.f;
#pragma unroll 1
    for (int ch = 0; ch < 4; ch++) {
      uint32_t r[16], t[8];
      logits(ch, r);
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const float pe = fast_exp2(__uint_as_float(r[e]) - ref);
        sum += pe;
        r[e] = __float_as_uint(pe);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) t[e] = pack2<F16>(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
      // columns that have been read already: chunk ch goes over logits 8 ch .. 8 ch + 7
      tmem_st8(s_t + ch * 8, t);
    }
  }
  tmem_wait_st();
  tc_fence_before();
  asm volatile("st.volatile.shared.f32 [%0], %1;" ::"r"(sum_slot), "f"(sum) : "memory");
  if (stored) asm volatile("st.volatile.shared.f32 [%0], %1;" ::"r"(l_slot), "f"(l * factor) : "memory");
  redo_meet(word_mine, word_mine ^ 16, stamp + 1, abort_flag);
  tc_fence_after();
  return Redo{ref, l * factor, sum};
}

__device__ __forceinline__ uint64_t pair64(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpair64(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <int NBOX, bool CAP, bool F16>
__global__ void __launch_bounds__(Geo<NBOX>::kThreads, 1)
prompt_attention_kernel(const __grid_constant__ PromptLaunch L, const __grid_constant__ CUtensorMap q_map,
                        const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using Z = Geo<NBOX>;
  uint8_t *gen = aligned_smem();
  const uint32_t base = smem_u32(gen);
  const uint32_t q_s = base, k_s = q_s + Z::QT * Z::kTile, v_s = k_s + Z::NK * Z::kTile;
  float *xch = reinterpret_cast<float *>(gen + (Z::QT + Z::NK + Z::NV) * Z::kTile);
  PlanPos *const at = reinterpret_cast<PlanPos *>(reinterpret_cast<uint8_t *>(xch) + Z::kXch) + (threadIdx.x >> 5);
  uint32_t *const words = meeting_words<NBOX>();
  volatile uint32_t *const beat = words + 8 * Z::QT;
  uint64_t *bars = reinterpret_cast<uint64_t *>(words + 8 * Z::QT + 4);
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + Z::kBars);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  const PromptParams &p = L.p;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.G, D = p.D;
  // the launch that joins partial results may be set up; it waits for this grid's end itself
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    mbar_init(bar(Z::B_QFULL), 1);
    mbar_init(bar(Z::B_QEMPTY), 1);
    for (int i = 0; i < Z::NK; i++) mbar_init(bar(Z::B_KFULL + i), 1), mbar_init(bar(Z::B_KEMPTY + i), 1);
    for (int i = 0; i < Z::NV; i++) mbar_init(bar(Z::B_VFULL + i), 1), mbar_init(bar(Z::B_VEMPTY + i), 1);
    for (int i = 0; i < Z::QT; i++) {
      mbar_init(bar(Z::B_SFULL + i), 1);
      mbar_init(bar(Z::B_PREADY + i), 8);
      mbar_init(bar(Z::B_PHALF + i), 8);
      mbar_init(bar(Z::B_PVDONE + i), 1);
    }
    for (int i = 0; i <= 8 * Z::QT; i++) words[i] = 0;
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == Z::kSoft + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_holder)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  // set up while the kernel ahead was finishing; what it wrote is read, and what it read written, from
  // here on only
  asm volatile("griddepcontrol.wait;" ::: "memory");
  bool failed = false;
  Seg g;
  if (lane == 0) *at = L.begin[blockIdx.x];
  __syncwarp();

  // Two threads per row and two query tiles make 640 threads of 96 registers; the softmax needs a
  // few more: 16 warps x 104 + 4 x 56 = 60416 of the 61440 that the launch holds.
  if (warp >= Z::kSoft) {
    if (Z::QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == Z::kSoft) {
      // =========================== copies ==============================================
      if (lane == 0) {
        uint32_t items = 0, tiles = 0;  // items and key tiles fetched so far
        while (!failed && walk_next<false>(L, at, g)) {
          if (g.kt0 >= g.kt1) continue;
          if (items > 0 && !wait_live(bar(Z::B_QEMPTY), (items - 1) & 1, abort_flag, beat)) { failed = true; break; }
          mbar_expect_tx(bar(Z::B_QFULL), (uint32_t)(g.tiles * NBOX * L.sub_tokens * G) * 128u);
          for (int i = 0; i < g.tiles; i++)
            for (int b = 0; b < NBOX; b++)
              tma_load_3d(q_s + (i * NBOX + b) * kBox, &q_map, b * 64, g.h * G, p.cu_q[g.s] + g.q0 + i * L.sub_tokens,
                          bar(Z::B_QFULL));
          items++;
          for (int t = g.kt0; t < g.kt1; t++, tiles++) {
            const int row = p.cu_kv[g.s] + t * kKeyTile;
            const int ks = tiles % Z::NK, vs = tiles % Z::NV;
            if (tiles >= Z::NK && !wait_live(bar(Z::B_KEMPTY + ks), (tiles / Z::NK - 1) & 1, abort_flag, beat)) { failed = true; break; }
            mbar_expect_tx(bar(Z::B_KFULL + ks), Z::kTile);
            for (int b = 0; b < NBOX; b++)
              tma_load_3d(k_s + ks * Z::kTile + b * kBox, &k_map, b * 64, g.h, row, bar(Z::B_KFULL + ks));
            if (tiles >= Z::NV && !wait_live(bar(Z::B_VEMPTY + vs), (tiles / Z::NV - 1) & 1, abort_flag, beat)) { failed = true; break; }
            mbar_expect_tx(bar(Z::B_VFULL + vs), Z::kTile);
            for (int b = 0; b < NBOX; b++)
              tma_load_3d(v_s + vs * Z::kTile + b * kBox, &v_map, b * 64, g.h, row, bar(Z::B_VFULL + vs));
          }
        }
      }
      __syncwarp();
    } else if (warp == Z::kSoft + 1) {
      // =========================== MMA issue ===========================================
      // The whole warp walks the loop so that descriptors and addresses stay warp-uniform; one
      // elected lane issues.  Its waits end alike for every lane.
      auto wait_all = [&](uint32_t b, uint32_t parity) { return __all_sync(0xffffffffu, wait_live(b, parity, abort_flag, beat)) != 0; };
      const uint32_t idesc_s = mma_desc(F16, 128, false), idesc_pv = mma_desc(F16, (uint32_t)(D + 15) & ~15u, true);
      const int ksteps = (D + 15) >> 4;
      const bool leader = elect_one();
      uint32_t items = 0, tiles = 0;
      uint32_t cnt[Z::QT];  // logit tiles issued for each query tile
#pragma unroll
      for (int i = 0; i < Z::QT; i++) cnt[i] = 0;
      auto issue_s = [&](int i, int q, uint32_t t) {
        const uint32_t a = k_major_low(q_s + q * Z::kTile), b = k_major_low(k_s + (t % Z::NK) * Z::kTile), d = tmem + i * 128;
#pragma unroll
        for (int kk = 0; kk < NBOX * 4; kk++) {
          const uint32_t off = ((kk >> 2) * kBox + (kk & 3) * 32) >> 4;
          if (leader && kk < ksteps) mma_ss(d, a + off, b + off, idesc_s, kk > 0 ? 1u : 0u);
        }
        if (leader) tc_commit(bar(Z::B_SFULL + i));
      };
      // P_i.V(t), as the softmax announces it (the issuing warp waits): bf16 in two halves, the first
      // while the second half's probabilities are still being taken
      auto issue_pv = [&](int i, uint32_t t, uint32_t acc) {
        const uint32_t b = mn_major_low(v_s + (t % Z::NV) * Z::kTile), a = tmem + i * 128, d = tmem + 256 + i * 128;
        if (!F16) {
          if (!wait_all(bar(Z::B_PHALF + i), (cnt[i] - 1) & 1)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 8; kk++)
            if (leader && !(kk & 2)) mma_ts(d, a + (kk >> 2) * 64 + (kk & 3) * 8, b + kk * 128, idesc_pv, kk > 0 ? 1u : acc);
        }
        if (!wait_all(bar(Z::B_PREADY + i), (cnt[i] - 1) & 1)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 8; kk++)
          if (leader && (F16 || (kk & 2)))
            mma_ts(d, a + (kk >> 2) * 64 + (kk & 3) * 8, b + kk * 128, idesc_pv, !F16 || kk > 0 ? 1u : acc);
        if (leader) tc_commit(bar(Z::B_PVDONE + i));
        return true;
      };
      // S_i = Q_q . K(t) into its buffer, once P_i.V of the tile before it is through with it
      auto next_s = [&](int i, int q, uint32_t t) {
        if (cnt[i] > 0 && !wait_all(bar(Z::B_PVDONE + i), (cnt[i] - 1) & 1)) return false;
        tc_fence_after();
        issue_s(i, q, t);
        cnt[i]++;
        return true;
      };
      auto k_full = [&](uint32_t t) { return wait_all(bar(Z::B_KFULL + t % Z::NK), (t / Z::NK) & 1); };
      auto v_full = [&](uint32_t t) { return wait_all(bar(Z::B_VFULL + t % Z::NV), (t / Z::NV) & 1); };
      while (!failed && walk_next<true>(L, at, g)) {
        const int n = g.kt1 - g.kt0;
        if (n <= 0) continue;
        if (!wait_all(bar(Z::B_QFULL), items & 1) || !k_full(tiles)) { failed = true; break; }
        if constexpr (Z::QT == 2) if (g.tiles == 1) {
          // one query tile: key tile j in place j % 2
          failed = !next_s(0, 0, tiles);
          if (!failed && leader) tc_commit(bar(Z::B_KEMPTY + tiles % Z::NK));
          if (!failed && n > 1) {
            failed = !k_full(tiles + 1) || !next_s(1, 0, tiles + 1);
            if (!failed && leader) tc_commit(bar(Z::B_KEMPTY + (tiles + 1) % Z::NK));
          }
          if (!failed && n <= 2 && leader) tc_commit(bar(Z::B_QEMPTY));
          for (int j0 = 0; j0 < n && !failed; j0 += 2) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int j = j0 + i;
              const uint32_t t = tiles + j;
              if (j >= n || failed) continue;
              if (!v_full(t) || !issue_pv(i, t, j > 1 ? 1u : 0u)) { failed = true; continue; }
              if (leader) tc_commit(bar(Z::B_VEMPTY + t % Z::NV));
              if (j + 2 < n) {
                if (!k_full(t + 2) || !next_s(i, 0, t + 2)) { failed = true; continue; }
                if (leader) {
                  tc_commit(bar(Z::B_KEMPTY + (t + 2) % Z::NK));
                  if (j + 3 == n) tc_commit(bar(Z::B_QEMPTY));
                }
              }
            }
            __syncwarp();
          }
          tiles += n;
          items++;
          continue;
        }
#pragma unroll
        for (int i = 0; i < Z::QT; i++)
          if (i < g.tiles && !failed) failed = !next_s(i, i, tiles);
        if (failed) break;
        if (leader) {
          tc_commit(bar(Z::B_KEMPTY + tiles % Z::NK));
          if (n == 1) tc_commit(bar(Z::B_QEMPTY));
        }
        for (int j = 0; j < n && !failed; j++) {
          const uint32_t t = tiles + j;
          const bool more = j + 1 < n;
          // waited for while the softmax has the tile, not between its announcement and P.V
          if (!v_full(t) || (more && !k_full(t + 1))) { failed = true; break; }
#pragma unroll
          for (int i = 0; i < Z::QT; i++) {
            if (i >= g.tiles || failed) continue;
            if (!issue_pv(i, t, j > 0 ? 1u : 0u)) { failed = true; continue; }
            const bool last = i + 1 == g.tiles;
            if (last && leader) tc_commit(bar(Z::B_VEMPTY + t % Z::NV));
            if (more) {
              if (!next_s(i, i, t + 1)) { failed = true; continue; }
              if (last && leader) {
                tc_commit(bar(Z::B_KEMPTY + (t + 1) % Z::NK));
                if (j + 2 == n) tc_commit(bar(Z::B_QEMPTY));
              }
            }
          }
          __syncwarp();
        }
        tiles += n;
        items++;
      }
    }
  } else {
    // =========================== softmax + epilogue ==================================
    if (Z::QT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int i = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
    const int row = quad * 32 + lane;  // row of the query tile = TMEM lane
    const int tok_in = row / G, head_in = row - tok_in * G;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t s_t = tmem + lane_base + i * 128 + half * 64;
    const uint32_t o_t = tmem + lane_base + 256 + i * 128;
    const int sync_id = 1 + i * 4 + quad;  // the two warps that share these rows
    // this thread's word of the exchange; the other half's is 512 bytes on or back (the area is aligned)
    const uint32_t mine = smem_u32(xch) + ((i * 2 + half) * 128 + row) * 4;
    constexpr uint32_t kSlot = Z::QT * 2 * 128 * 4;
    const uint32_t word_mine = smem_u32(words + warp);  // the other warp's: ^ 16
    // slots 0 and 1: the sums of even and odd tiles; slot 2: an item's sum;
    // slot 3: the maxima of an item's first tile
    uint32_t cnt = 0;  // logit tiles seen
    const float c = p.scale * kLog2e;
    // soft-capping: x -> tanh(x*scale/cap)*cap/scale, so that x*c is the capped logit
    const float cap_in = p.scale / p.softcap, cap_out = p.softcap / p.scale;
    // Sums of up to this much against the stale reference are taken as they are.  f16 ends at 2^16; bf16 has
    // fp32's range, and its probabilities are announced before the sum is known.
    // (bf16: beyond this a row that comes out not finite is recomputed, see `far`.  Its weighted sums are as
    // far above the result as the sum is above 1: below this, values of up to 2^110 stay in fp32.)
    constexpr float kFar = F16 ? 32768.f : 65536.f;
    auto put = [&](uint32_t slot, float x) { asm volatile("st.volatile.shared.f32 [%0], %1;" ::"r"(mine + slot * kSlot), "f"(x) : "memory"); };
    auto get = [&](uint32_t slot) {
      float y;
      asm volatile("ld.volatile.shared.f32 %0, [%1];" : "=f"(y) : "r"((mine ^ 512) + slot * kSlot) : "memory");
      return y;
    };
    // Waits for a barrier that cannot complete before both warps of these rows have announced tile
    // cnt - 1; meanwhile the other one may call for a meeting about that tile (redo_tile).
    auto wait_pending = [&](uint32_t b, uint32_t parity, auto &&join) {
      if (__all_sync(0xffffffffu, mbar_try_wait(b, parity))) return;
      long long t0 = clock64();
      uint32_t seen = *beat;
      bool met = false;
      while (!__all_sync(0xffffffffu, mbar_try_wait(b, parity))) {
        uint32_t w;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(w) : "r"(word_mine ^ 16) : "memory");
        if (!met && __any_sync(0xffffffffu, w == 2 * cnt)) {
          join();
          met = true;
        }
        if (*abort_flag) failed = true;
        if (*beat != seen) seen = *beat, t0 = clock64();
        if (clock64() - t0 > (1ll << 31)) failed = true, *abort_flag = 1;
        if (__any_sync(0xffffffffu, failed)) {
          failed = true;
          return;
        }
      }
    };
    // After a wait that ran out these warps keep going through the motions (every further wait
    // returns at once): two of them share each row's barrier, and one that left would leave
    // the other waiting at it.
    while (walk_next<true>(L, at, g)) {
      // one query tile, two places: this one takes every other key tile from `start` on
      const bool both_places = Z::QT == 2 && g.tiles == 1;
      const int step = both_places ? 2 : 1, start = g.kt0 + (both_places ? i : 0);
      if (i >= g.tiles && !(both_places && start < g.kt1)) continue;
      const int token = g.q0 + (both_places ? 0 : i * L.sub_tokens) + tok_in;  // within the sequence
      const bool valid = tok_in < L.sub_tokens && token < g.q_len;
      const int lim = valid ? g.kv_len - g.q_len + token + 1 : 0x7fffffff;  // keys the row sees
      int min_lim = lim;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) min_lim = min(min_lim, __shfl_xor_sync(0xffffffffu, min_lim, o));
      float ref = 0.f, l = 0.f, sum = 0.f;  // ref: 0 while the row has seen nothing
      bool behind = false;  // tile cnt - 1 is this item's, and the other warp may yet call a meeting about it
      int left = 0;         // columns of the tile from here on are masked
      bool far = false;     // bf16: a sum was so large that an overflow may be this kernel's own
      [[maybe_unused]] auto redo = [&](bool stored, bool rescale) {
        const uint32_t tile = stored ? cnt - 1 : cnt;
        const Redo r = redo_tile<CAP, F16>(s_t, o_t, D, half, c, cap_in, cap_out, ref, l, sum, mine + (tile & 1) * kSlot,
                                           mine + (~tile & 1) * kSlot, mine + 2 * kSlot, word_mine, 2 * (tile + 1), valid, stored, rescale, left,
                                           abort_flag);
        ref = r.ref;
        sum = r.sum;
        l = r.l;
      };
      for (int t = start; t < g.kt1; t += step, cnt++) {
        const bool first = t == start;
        if (first || !F16) {
          failed |= !wait_live(bar(Z::B_SFULL + i), cnt & 1, abort_flag, beat);
          __syncwarp();
        } else {
          wait_pending(bar(Z::B_SFULL + i), cnt & 1, [&] {
            if (behind) redo(true, t > start + step);
          });
        }
        tc_fence_after();
        const int key0 = t * kKeyTile + half * 64;
        const bool need_mask = key0 + 64 > min_lim;
        left = lim - key0;
        auto cap_and_mask = [&](uint32_t (&r)[16], int col0, bool mask) {
          if (CAP) {
#pragma unroll
            for (int e = 0; e < 16; e++) r[e] = __float_as_uint(tanhf(__uint_as_float(r[e]) * cap_in) * cap_out);
          }
          if (mask) {
#pragma unroll
            for (int e = 0; e < 16; e++)
              if (col0 + e >= left) r[e] = 0xff800000u;
          }
        };
        if (first) {  // the first tile sets the reference
          float mx = -INFINITY;
#pragma unroll 1
          for (int ch = 0; ch < 4; ch++) {
            uint32_t r[16];
            tmem_ld16(s_t + ch * 16, r);
            tmem_wait_ld16(r);
            cap_and_mask(r, ch * 16, need_mask);
#pragma unroll
            for (int e = 0; e < 16; e++) mx = fmaxf(mx, __uint_as_float(r[e]));
          }
          put(3, mx);
          pair_sync(sync_id);
          mx = fmaxf(mx, get(3));
          ref = mx == -INFINITY ? 0.f : mx * c;
        } else {
          // both halves of a row see the same sum of the tile before and decide alike
          const float both = sum + get((cnt - 1) & 1);
          if (__any_sync(0xffffffffu, valid && both > 256.f)) {
            float factor = 1.f;
            if (valid && both > 256.f) {
              factor = reciprocal(both);
              ref += log2f(both);
            }
            // O holds the tiles before this one: S of this tile was issued after their P.V
            scale_o(o_t, D, half, factor);
            l *= factor;
          }
        }
        uint32_t pr[32];  // the row half's probabilities, packed
        auto pass = [&](auto masked) {
          constexpr bool MASK = decltype(masked)::value;
          const uint64_t c2 = pair64(c, c), ref2 = pair64(-ref, -ref);
          uint64_t acc0 = 0, acc1 = 0;
          // 16 columns at a time: a load takes some forty cycles, which the scheduler's other warps fill
#pragma unroll
          for (int ch = 0; ch < 4; ch++) {
            uint32_t r[16];
            tmem_ld16(s_t + ch * 16, r);
            tmem_wait_ld16(r);
            cap_and_mask(r, ch * 16, MASK);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const uint64_t x = fma2(pair64(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), c2, ref2);
              float p0, p1;
              unpair64(x, p0, p1);
              p0 = fast_exp2(p0);
              p1 = fast_exp2(p1);
              if (e & 2) acc1 = add2(acc1, pair64(p0, p1));
              else acc0 = add2(acc0, pair64(p0, p1));
              pr[ch * 8 + (e >> 1)] = pack2<F16>(p0, p1);
            }
            if (!F16 && ch == 1) tmem_st16(s_t, reinterpret_cast<uint32_t (&)[16]>(pr[0]));
            if (!F16 && ch == 2) {  // the first half has been on its way for a quarter of the pass
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(Z::B_PHALF + i));
            }
          }
          float x0, x1;
          unpair64(add2(acc0, acc1), x0, x1);
          sum = x0 + x1;
        };
        if (need_mask) pass(std::true_type{});
        else pass(std::false_type{});
        if constexpr (F16) {
          behind = true;
          if (__any_sync(0xffffffffu, valid && sum > kFar)) {
            redo(false, !first);
            behind = false;
          } else {
            put(cnt & 1, sum);
            tmem_st32(s_t, pr);
            tmem_wait_st();
            tc_fence_before();
          }
        } else {
          far |= sum > kFar;
          tmem_st16(s_t + 16, reinterpret_cast<uint32_t (&)[16]>(pr[16]));
          put(cnt & 1, sum);
          tmem_wait_st();
          tc_fence_before();
        }
        l += sum;
        if (t + step >= g.kt1) {  // read after P.V of this tile, for which both warps have arrived
          put(2, l);
          if (!F16) put(4, far ? 1.f : 0.f);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(Z::B_PREADY + i));
      }
      const int64_t q_row = p.cu_q[g.s] + token;
      const bool whole = g.kt0 == 0 && g.kt1 == g.n;
      elem16 *orow = p.out + q_row * p.out_stride + (int64_t)(g.h * G + head_in) * D;
      if (g.n == 0) {  // no key for any row of the item
        if (valid)
          for (int e = chunk_begin(D, half) * 32; e < min(chunk_end(D, half) * 32, D); e += 8)
            *reinterpret_cast<uint4 *>(orow + e) = make_uint4(0, 0, 0, 0);
        continue;
      }
      if (F16) {
        wait_pending(bar(Z::B_PVDONE + i), (cnt - 1) & 1, [&] {
          if (behind) redo(true, g.kt1 > start + step);
        });
      } else {
        failed |= !wait_live(bar(Z::B_PVDONE + i), (cnt - 1) & 1, abort_flag, beat);
        __syncwarp();
      }
      tc_fence_after();
      {
        const float l_other = get(2);
        l = half == 0 ? l + l_other : l_other + l;
        if (!F16) far |= get(4) != 0.f;
      }
      const bool two = both_places && g.kt0 + 1 < g.kt1;
      if constexpr (!F16) {
        // What is joined with other parts of its item - the other place, or pieces of other CTAs - is
        // weighted by 2^(reference - largest reference), and a reference that a jump in the last key tile left
        // behind by more than fp32's exponents would take its part, of a sum as large, with it.
        if ((two || g.kt1 - g.kt0 < g.n) && __any_sync(0xffffffffu, valid && far)) {
          float factor = 1.f;
          if (valid && far) {
            factor = reciprocal(l);
            ref += log2f(l);
            l *= factor;
          }
          scale_o(o_t, D, half, factor);
          tmem_wait_st();
        }
      }
      if (two) {
        // place 1 hands its reference and sum to place 0, which reads both accumulators
        auto quad_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(9 + quad) : "memory"); };
        if (i == 1) {
          put(0, l == 0.f ? -INFINITY : ref);
          put(1, l);
          if (!F16) put(3, far ? 1.f : 0.f);
          tc_fence_before();
          quad_sync();
          quad_sync();  // O_1 has been read
          continue;
        }
        quad_sync();
        tc_fence_after();
        float ref1, l1;
        asm volatile("ld.volatile.shared.f32 %0, [%1];" : "=f"(ref1) : "r"(mine + 1024) : "memory");
        asm volatile("ld.volatile.shared.f32 %0, [%1];" : "=f"(l1) : "r"(mine + 1024 + kSlot) : "memory");
        if (!F16) {
          float far1;
          asm volatile("ld.volatile.shared.f32 %0, [%1];" : "=f"(far1) : "r"(mine + 1024 + 3 * kSlot) : "memory");
          far |= far1 != 0.f;
        }
        // a place whose keys the row does not see counts for nothing (its P was 0, its P.V may be NaN)
        const float top = fmaxf(l == 0.f ? -INFINITY : ref, ref1);
        const float f0 = l == 0.f ? 0.f : fast_exp2(ref - top);  // O = f0 O_0 + f1 O_1
        const float f1 = l1 == 0.f ? 0.f : fast_exp2(ref1 - top);
        l = f0 * l + f1 * l1;
        if (top != -INFINITY) ref = top;
#pragma unroll 1
        for (int ch = chunk_begin(D, half); ch < chunk_end(D, half); ch++) {
          uint32_t r[32], r1[32];
          tmem_ld32(o_t + ch * 32, r);
          tmem_ld32(o_t + 128 + ch * 32, r1);
          tmem_wait_ld32(r);
          tmem_wait_ld32(r1);
#pragma unroll
          for (int e = 0; e < 32; e++) {
            const float a = f0 == 0.f ? 0.f : f0 * __uint_as_float(r[e]), b = f1 == 0.f ? 0.f : f1 * __uint_as_float(r1[e]);
            r[e] = __float_as_uint(a + b);
          }
          tmem_st32(o_t + ch * 32, r);
        }
        tmem_wait_st();
        tc_fence_before();
        quad_sync();
      }
      const float inv = whole ? (l == 0.f ? 0.f : reciprocal(l)) : 1.f;
      constexpr int kRows = 128 * Z::QT;
      float *part = L.ws + (size_t)(2 * blockIdx.x + (g.kt0 > 0 ? 0 : 1)) * (D + 3) * kRows + i * 128 + row;
      bool finite = true;
      const int c0 = chunk_begin(D, half), c1 = chunk_end(D, half);
      if (whole) {
        // A thread has 64 bytes of its own row per chunk; four threads trade 16-byte pieces so that a
        // store covers 64 bytes of eight rows instead of 16 bytes of thirty-two (a row apiece cost
        // 4096 cycles of line accesses per item).
        elem16 *row_at[4];
        bool row_ok[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int src = (lane & ~3) + k;
          row_at[k] = reinterpret_cast<elem16 *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(orow), src)) + (lane & 3) * 8;
          row_ok[k] = __shfl_sync(0xffffffffu, valid, src);
        }
        const uint64_t inv2 = pair64(inv, inv);
        uint64_t odd2 = 0;
        for (int ch = c0; ch < c1; ch++) {
          uint32_t r[32];
          tmem_ld32(o_t + ch * 32, r);
          tmem_wait_ld32(r);
          uint32_t w[4][4];  // piece, word
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const uint64_t y = fma2(pair64(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), inv2, 0);
            // 0 unless something is infinite or NaN (columns beyond D hold what an earlier item left: not
            // looked at)
            if (ch * 32 + e < D) odd2 = fma2(y, 0, odd2);
            float y0, y1;
            unpair64(y, y0, y1);
            w[e >> 3][(e >> 1) & 3] = pack2<F16>(y0, y1);
          }
          // 4 x 4 transpose of pieces over four lanes: piece b of lane a to piece a of lane b
#pragma unroll
          for (int bit = 1; bit <= 2; bit <<= 1) {
            const bool up = lane & bit;
#pragma unroll
            for (int a = 0; a < 4; a++) {
              if (a & bit) continue;
#pragma unroll
              for (int k = 0; k < 4; k++) {
                const uint32_t give = up ? w[a][k] : w[a | bit][k];
                const uint32_t got = __shfl_xor_sync(0xffffffffu, give, bit);
                if (up) w[a][k] = got;
                else w[a | bit][k] = got;
              }
            }
          }
#pragma unroll
          for (int k = 0; k < 4; k++)
            if (row_ok[k] && ch * 32 + (lane & 3) * 8 < D)
              *reinterpret_cast<uint4 *>(row_at[k] + ch * 32) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
        }
        float odd0, odd1;
        unpair64(odd2, odd0, odd1);
        finite = odd0 == 0.f && odd1 == 0.f;
      } else {
        for (int ch = c0; ch < c1; ch++) {
          uint32_t r[32];
          tmem_ld32(o_t + ch * 32, r);
          tmem_wait_ld32(r);
          if (valid) {
#pragma unroll
            for (int e = 0; e < 32; e++)
              if (ch * 32 + e < D) part[(ch * 32 + e) * kRows] = __uint_as_float(r[e]);
          }
          __syncwarp();
        }
      }
      if (!whole && valid && half == 0) {
        part[(size_t)D * kRows] = l == 0.f ? -INFINITY : ref;  // a row that sees no key of this piece
        part[(size_t)(D + 1) * kRows] = l;
        part[(size_t)(D + 2) * kRows] = far ? 1.f : 0.f;
      }
      tc_fence_before();
      uint32_t odd = __ballot_sync(0xffffffffu, valid && !finite);
      __syncwarp();
      while (odd) {
        const int src = __ffs(odd) - 1;
        odd &= odd - 1;
        const int tk = __shfl_sync(0xffffffffu, token, src), hd = g.h * G + __shfl_sync(0xffffffffu, head_in, src);
        const bool own = __shfl_sync(0xffffffffu, far, src);  // the row overflowed here and not in its values
        if (own || masked_value_not_finite(p, g.s, tk, g.h, g.n, F16)) {
          // pieces of eight columns, four to a chunk
          const uint32_t below = (uint32_t)((1ull << (c0 * 4)) - 1), upto = (uint32_t)((1ull << (c1 * 4)) - 1);
          repair_row<F16, NBOX>(p, g.s, tk, hd, upto & ~below);
        }
        if (lane == 0) atomicAdd(const_cast<uint32_t *>(beat), 1u);
      }
    }
  }

  if (failed) atomicOr(L.err, kErrTimeout);
  // ---- teardown -------------------------------------------------------------------
  // A role that gave up may have left copies in flight towards this CTA's shared memory; the
  // CTA must not exit before they have landed.
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && warp == Z::kSoft) {
    const long long t0 = clock64();
    while (clock64() - t0 < (1ll << 22)) {
    }  // ~2 ms: far longer than any copy takes; nothing below reads shared memory
  }
  __syncthreads();
  if (warp == Z::kSoft + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

struct JoinLaunch {
  PromptParams p;
  const float *ws;
  int32_t sub_tokens, tile_tokens, rows;  // rows of a partial slot: 128 per query tile
  PlanPos item[kMaxPlanCtas];             // .kt unused
  int32_t first[kMaxPlanCtas], last[kMaxPlanCtas];
};

// Joins the partial results of the items that were cut: out = sum_c w_c O_c / sum_c w_c l_c with
// w_c = 2^(m_c - max m), pieces in CTA order.  A CTA takes 32 rows of an item: its warps fetch the
// pieces' maxima and sums side by side, the weights go to shared memory, and then a warp takes
// 8 dimensions of the rows at a time, the loads of four pieces in flight.  Partials are stored
// dimension-major, so that loads are whole lines.  Bound by latency: launch, sums, rows.
template <bool F16>
__global__ void __launch_bounds__(256) prompt_join_kernel(const __grid_constant__ JoinLaunch J) {
  extern __shared__ float join_smem[];  // the pieces' references, then their sums
  __shared__ int far_s[32];
  const PromptParams &p = J.p;
  const PlanPos it = J.item[blockIdx.x];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.D, G = p.G;
  const int row = blockIdx.y * 32 + lane;  // 128 per query tile
  const int tile_i = row >> 7, tok_in = (row & 127) / G, head_in = (row & 127) - tok_in * G;
  const int q_len = p.cu_q[it.seq + 1] - p.cu_q[it.seq], kv_len = p.cu_kv[it.seq + 1] - p.cu_kv[it.seq];
  const int q0 = it.qt * J.tile_tokens, token = q0 + tile_i * J.sub_tokens + tok_in;
  const bool valid = tok_in < J.sub_tokens && token < q_len;
  if (!__any_sync(0xffffffffu, valid)) return;  // the same rows in every warp
  const int n = (max(kv_len - q_len + min(q_len, q0 + J.tile_tokens), 0) + kKeyTile - 1) / kKeyTile;
  const int first = J.first[blockIdx.x], pieces = J.last[blockIdx.x] - first + 1;
  float(*const m_s)[32] = reinterpret_cast<float(*)[32]>(join_smem), (*const l_s)[32] = m_s + pieces;
  const size_t slot = (size_t)(D + 3) * J.rows;
  if (warp == 0) far_s[lane] = 0;
  __syncthreads();
  // the first piece begins the item: the second slot of its CTA; the others the first
  const float *const at = J.ws + (size_t)(2 * first) * slot + row;
  auto part = [&](int c) { return at + (size_t)(c == 0 ? 1 : 2 * c) * slot; };
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the attention kernel is through
#pragma unroll 4
  for (int c = warp; c < pieces; c += 8) {
    m_s[c][lane] = valid ? part(c)[(size_t)D * J.rows] : -INFINITY;
    l_s[c][lane] = valid ? part(c)[(size_t)(D + 1) * J.rows] : 0.f;
    if (valid && part(c)[(size_t)(D + 2) * J.rows] != 0.f) far_s[lane] = 1;
  }
  __syncthreads();
  float mx = -INFINITY, l = 0.f;
  for (int c = 0; c < pieces; c++) mx = fmaxf(mx, m_s[c][lane]);
  const float base = mx == -INFINITY ? 0.f : mx;
  for (int c = 0; c < pieces; c++) l += fast_exp2(m_s[c][lane] - base) * l_s[c][lane];
  const float inv = l == 0.f ? 0.f : reciprocal(l);
  elem16 *orow = p.out + (int64_t)(p.cu_q[it.seq] + token) * p.out_stride + (int64_t)(it.head * G + head_in) * D;
  for (int d = warp * 8; d < D; d += 64) {
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < pieces; c += 4) {
      float x[4][8];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        // a row that sees no key of a piece has nothing there to add
        const bool have = c + k < pieces && m_s[min(c + k, pieces - 1)][lane] != -INFINITY;
        const float *src = part(c + k) + (size_t)d * J.rows;
#pragma unroll
        for (int e = 0; e < 8; e++) x[k][e] = have ? src[(size_t)e * J.rows] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float wgt = fast_exp2(m_s[min(c + k, pieces - 1)][lane] - base);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = fmaf(wgt, x[k][e], o[e]);
      }
    }
    bool finite = true;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      o[k] *= inv;
      finite &= fabsf(o[k]) < INFINITY;
    }
    if (valid)
      *reinterpret_cast<uint4 *>(orow + d) =
          make_uint4(pack2<F16>(o[0], o[1]), pack2<F16>(o[2], o[3]), pack2<F16>(o[4], o[5]), pack2<F16>(o[6], o[7]));
    uint32_t odd = __ballot_sync(0xffffffffu, valid && !finite);
    __syncwarp();
    while (odd) {
      const int src = __ffs(odd) - 1;
      odd &= odd - 1;
      const int tk = __shfl_sync(0xffffffffu, token, src), hd = it.head * G + __shfl_sync(0xffffffffu, head_in, src);
      if (far_s[src] || masked_value_not_finite(p, it.seq, tk, it.head, n, F16)) repair_row<F16, 0>(p, it.seq, tk, hd, 1u << (d >> 3));
    }
  }
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn g_encode = nullptr;  // set by prompt_configure, before any call

// Rows of [heads][D] as {D, heads, rows}; a box of 64 dimensions, `heads_box` heads, `rows_box`
// rows lands as lines of 128 bytes with the 128-byte swizzle.  Out-of-range elements read 0.
bool encode_rows(CUtensorMap *map, const void *ptr, int D, int heads, int64_t rows, int64_t stride, int heads_box,
                 int rows_box) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads_box, (cuuint32_t)rows_box}, steps[3] = {1, 1, 1};
  return g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(ptr), dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A launch whose CTAs may be set up before the kernel ahead on the stream has finished.
template <typename... Args>
cudaError_t launch_dependent(void (*kernel)(Args...), dim3 grid, int threads, int smem, cudaStream_t st, const Args &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  __atomic_fetch_add(&g_launch_count, 1ull, __ATOMIC_RELAXED);
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int NBOX>
cudaError_t launch_boxes(const PromptLaunch &L, const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm,
                         bool f16, int ctas, cudaStream_t st) {
  const bool cap = L.p.softcap != 1.0f;
  cudaError_t e = cudaSuccess;
  auto go = [&](auto kernel) { e = launch_dependent(kernel, dim3(ctas), Geo<NBOX>::kThreads, Geo<NBOX>::kSmem, st, L, qm, km, vm); };
  if (cap && f16) go(prompt_attention_kernel<NBOX, true, true>);
  else if (cap) go(prompt_attention_kernel<NBOX, true, false>);
  else if (f16) go(prompt_attention_kernel<NBOX, false, true>);
  else go(prompt_attention_kernel<NBOX, false, false>);
  return e;
}

}  // namespace

size_t prompt_workspace_bytes(int num_sms, int head_size) {
  const size_t rows = head_size <= 128 ? 256 : 128;
  return (size_t)2 * std::min(num_sms, kMaxPlanCtas) * rows * (head_size + 3) * 4;
}

cudaError_t prompt_configure() {
  cudaError_t e = cudaSuccess;
  auto set = [&](auto kernel, int bytes) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  };
  auto set4 = [&](auto k0, auto k1, auto k2, auto k3, int bytes) {
    set(k0, bytes), set(k1, bytes), set(k2, bytes), set(k3, bytes);
  };
  set4(prompt_attention_kernel<1, false, false>, prompt_attention_kernel<1, false, true>,
       prompt_attention_kernel<1, true, false>, prompt_attention_kernel<1, true, true>, Geo<1>::kSmem);
  set4(prompt_attention_kernel<2, false, false>, prompt_attention_kernel<2, false, true>,
       prompt_attention_kernel<2, true, false>, prompt_attention_kernel<2, true, true>, Geo<2>::kSmem);
  set4(prompt_attention_kernel<3, false, false>, prompt_attention_kernel<3, false, true>,
       prompt_attention_kernel<3, true, false>, prompt_attention_kernel<3, true, true>, Geo<3>::kSmem);
  set4(prompt_attention_kernel<4, false, false>, prompt_attention_kernel<4, false, true>,
       prompt_attention_kernel<4, true, false>, prompt_attention_kernel<4, true, true>, Geo<4>::kSmem);
  if (e != cudaSuccess) return e;
  void *fn = nullptr;
  cudaDriverEntryPointQueryResult qres;
  e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
  if (e != cudaSuccess) return e;
  if (!fn || qres != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
  __atomic_store_n(&g_encode, reinterpret_cast<EncodeFn>(fn), __ATOMIC_RELEASE);
  return cudaSuccess;
}

cudaError_t launch_prompt_attention(const PromptParams &p, bool f16, int num_sms, void *workspace, unsigned *err,
                                    cudaStream_t st) {
  const PromptShape shape = prompt_shape(p.D, p.G);
  PromptPlan plan;
  plan_prompt(p.cu_q, p.cu_kv, 0, p.S, p.Hkv, shape, num_sms, kMinPiece, kMinTilesPerCta, &plan);
  if (plan.num_ctas == 0) return cudaSuccess;
  PromptLaunch L;
  L.p = p;
  std::copy(plan.begin, plan.begin + plan.num_ctas + 1, L.begin);
  L.ws = static_cast<float *>(workspace);
  L.err = err;
  L.sub_tokens = shape.sub_tokens;
  L.tile_tokens = shape.tile_tokens;
  CUtensorMap qm, km, vm;
  bool ok = encode_rows(&qm, p.q, p.D, p.Hq, p.cu_q[p.S], p.q_stride, p.G, shape.sub_tokens);
  if (p.cu_kv[p.S] > p.cu_kv[0]) {
    ok = ok && encode_rows(&km, p.k, p.D, p.Hkv, p.cu_kv[p.S], p.k_stride, 1, kKeyTile) &&
         encode_rows(&vm, p.v, p.D, p.Hkv, p.cu_kv[p.S], p.v_stride, 1, kKeyTile);
  } else {
    km = vm = qm;  // no key anywhere: never read
  }
  if (!ok) return cudaErrorInvalidValue;
  cudaError_t e = cudaSuccess;
  switch ((p.D + 63) / 64) {
    case 1: e = launch_boxes<1>(L, qm, km, vm, f16, plan.num_ctas, st); break;
    case 2: e = launch_boxes<2>(L, qm, km, vm, f16, plan.num_ctas, st); break;
    case 3: e = launch_boxes<3>(L, qm, km, vm, f16, plan.num_ctas, st); break;
    default: e = launch_boxes<4>(L, qm, km, vm, f16, plan.num_ctas, st); break;
  }
  if (e != cudaSuccess || plan.num_split == 0) return e;
  JoinLaunch J;
  J.p = p;
  J.ws = L.ws;
  J.sub_tokens = shape.sub_tokens;
  J.tile_tokens = shape.tile_tokens;
  J.rows = shape.tile_tokens > shape.sub_tokens ? 256 : 128;
  int most = 0, pieces = 0;  // rows of the largest item that is cut, pieces of the one cut most often
  for (int k = 0; k < plan.num_split; k++) {
    J.item[k] = plan.begin[plan.split_last[k]];
    J.first[k] = plan.split_first[k];
    J.last[k] = plan.split_last[k];
    pieces = std::max(pieces, plan.split_last[k] - plan.split_first[k] + 1);
    const int left = p.cu_q[J.item[k].seq + 1] - p.cu_q[J.item[k].seq] - J.item[k].qt * shape.tile_tokens;
    most = std::max(most, left > shape.sub_tokens ? J.rows : std::min(left, shape.sub_tokens) * p.G);
  }
  const dim3 grid((unsigned)plan.num_split, (unsigned)(most + 31) / 32);
  const int smem = pieces * 2 * 32 * 4;  // 40 KB for an item over all CTAs
  return f16 ? launch_dependent(prompt_join_kernel<true>, grid, 256, smem, st, J)
             : launch_dependent(prompt_join_kernel<false>, grid, 256, smem, st, J);
}

}  // namespace pa
