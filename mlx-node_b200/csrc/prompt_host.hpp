// Host side of the prompt-path entry points (rotation + cache write, packed prompt
// attention, cache read-back): argument checks, the rotation table and the partition of the
// attention's work.  No CUDA call in here, so that all of it can be checked without a device.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/paged_attn_b200.h"

namespace pa {

// An error code with its message, or OK.
struct ArgError {
  pa_status code = PA_OK;
  const char *what = "";
  explicit operator bool() const { return code != PA_OK; }
};
inline ArgError bad_arg(const char *what) { return ArgError{PA_ERR_INVALID_ARG, what}; }

inline bool ptr16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---- rotation table ---------------------------------------------------------------------
constexpr int kMaxRopePairs = 128;

// Frequencies as turns per position in 64-bit fixed point: entry i is
// frac(f_i / (2 pi)) * 2^64.  position * entry modulo 2^64 is then the phase of that
// position in units of 2^-64 turns, exact for every 32-bit position up to the entry's own
// rounding (2^31 * 2^-65 turns): an fp32 or even fp64 product of a far position and a
// frequency would lose the low bits that the sine depends on.
struct alignas(16) RopeTable {
  uint64_t turn[kMaxRopePairs];
  float gain;       // multiplies cosine and sine
  int32_t dims;     // elements rotated, even
  int32_t interleaved;
};

inline ArgError check_rope_config(const PaRopeConfig &c) {
  if (c.rope_dims == 0 || (c.rope_dims & 1u) || c.rope_dims > 2u * kMaxRopePairs)
    return bad_arg("rope_dims must be even and in [2, 256]");
  if (c.interleaved > 1u) return bad_arg("interleaved must be 0 or 1");
  if (!(c.base > 0.f) || !std::isfinite(c.base)) return bad_arg("base must be finite and > 0");
  if (c.scaling > PA_ROPE_YARN) return bad_arg("unknown scaling");
  if (!(c.attention_factor >= 0.f) || !std::isfinite(c.attention_factor))
    return bad_arg("attention_factor must be finite and >= 0 (0 = the scaling's own)");
  if (c.scaling != PA_ROPE_PLAIN && (!(c.factor > 0.f) || !std::isfinite(c.factor)))
    return bad_arg("factor must be finite and > 0");
  if (c.scaling >= PA_ROPE_BANDS && c.original_max_position == 0)
    return bad_arg("original_max_position must be > 0 for this scaling");
  if (c.scaling == PA_ROPE_BANDS &&
      (!(c.low_freq_factor > 0.f) || !(c.high_freq_factor > c.low_freq_factor) || !std::isfinite(c.high_freq_factor)))
    return bad_arg("low_freq_factor must be > 0 and below high_freq_factor");
  if (c.scaling == PA_ROPE_YARN &&
      (!(c.beta_slow > 0.f) || !(c.beta_fast > c.beta_slow) || !std::isfinite(c.beta_fast) || !(c.base > 1.f)))
    return bad_arg("beta_slow must be > 0 and below beta_fast, and base above 1");
  return {};
}

// Radians per position of pair i, and the gain, of a checked configuration.
inline long double rope_frequency(const PaRopeConfig &c, int i) {
  const long double two_pi = 6.283185307179586476925286766559005768L;
  const int half = (int)c.rope_dims / 2;
  const long double f = std::pow((long double)c.base, -(long double)i / half);
  switch (c.scaling) {
    case PA_ROPE_LINEAR:
      return f / c.factor;
    case PA_ROPE_BANDS: {
      // turns the pair makes over the trained length: few -> slowed down by `factor`, many ->
      // kept, in between a blend
      const long double turns = c.original_max_position * f / two_pi;
      long double keep = (turns - c.low_freq_factor) / ((long double)c.high_freq_factor - c.low_freq_factor);
      keep = std::min(1.0L, std::max(0.0L, keep));
      return f * keep + f / c.factor * (1 - keep);
    }
    case PA_ROPE_YARN: {
      // the same idea as a ramp over the pair's index between the indexes that make
      // beta_fast and beta_slow turns
      auto where = [&](long double turns) {
        return half * std::log(c.original_max_position / (turns * two_pi)) / std::log((long double)c.base);
      };
      const long double lo = std::max(std::floor(where(c.beta_fast)), 0.0L);
      const long double hi = std::min(std::ceil(where(c.beta_slow)), (long double)c.rope_dims - 1);
      long double slow = (i - lo) / std::max(hi - lo, 0.001L);
      slow = std::min(1.0L, std::max(0.0L, slow));
      return f / c.factor * slow + f * (1 - slow);
    }
    default:
      return f;
  }
}

inline void build_rope_table(const PaRopeConfig &c, RopeTable *t) {
  const long double two_pi = 6.283185307179586476925286766559005768L;
  t->dims = (int32_t)c.rope_dims;
  t->interleaved = (int32_t)c.interleaved;
  t->gain = c.attention_factor;
  if (t->gain == 0.f)
    t->gain = c.scaling == PA_ROPE_YARN && c.factor > 1.f ? (float)(0.1L * std::log((long double)c.factor) + 1.0L) : 1.f;
  for (int i = 0; i < kMaxRopePairs; i++) {
    t->turn[i] = 0;
    if (i >= (int)c.rope_dims / 2) continue;
    long double turns = rope_frequency(c, i) / two_pi;
    turns -= std::floor(turns);
    const long double scaled = std::floor(std::ldexp(turns, 64) + 0.5L);
    t->turn[i] = scaled >= std::ldexp(1.0L, 64) ? 0u : (uint64_t)scaled;
  }
}

// ---- argument checks ----------------------------------------------------------------------
inline ArgError check_rotate_args(const PagedAttnConfig &cfg, const RopeTable *rope, const void *q_out,
                                  const void *k_out, const void *q, const void *k, const void *v,
                                  const void *q_norm_weight, const void *k_norm_weight, float eps,
                                  const int32_t *positions, const int64_t *slot_mapping, int64_t num_tokens,
                                  int32_t num_q_heads, int64_t q_stride, int64_t q_out_stride, int64_t k_stride,
                                  int64_t k_out_stride, int64_t v_stride) {
  const int64_t D = cfg.head_size, Hkv = cfg.num_kv_heads;
  if (!rope) return bad_arg("rope plan is null");
  if (rope->dims > D) return bad_arg("the plan rotates more elements than a head has");
  if (!q_out || !q || !k || !positions) return bad_arg("null tensor pointer");
  if (!slot_mapping && !k_out) return bad_arg("slot_mapping and k_out are both null: the keys would go nowhere");
  if (slot_mapping && !v) return bad_arg("v is null");
  if (num_q_heads <= 0 || num_q_heads % Hkv) return bad_arg("num_q_heads must be a positive multiple of num_kv_heads");
  if (Hkv + num_q_heads > 65535) return bad_arg("more than 65535 heads");
  if (!(eps >= 0.f) || !std::isfinite(eps)) return bad_arg("eps must be finite and >= 0");
  const int64_t q_row = num_q_heads * D, kv_row = Hkv * D;
  if (q_stride < q_row || q_out_stride < q_row || k_stride < kv_row || (k_out && k_out_stride < kv_row) ||
      (slot_mapping && v_stride < kv_row) || ((q_stride | q_out_stride | k_stride) & 7) ||
      (k_out && (k_out_stride & 7)) || (slot_mapping && (v_stride & 7)))
    return bad_arg("row strides must cover a row and be multiples of 8");
  if (!ptr16(q) || !ptr16(q_out) || !ptr16(k) || !ptr16(k_out) || !ptr16(v) || !ptr16(q_norm_weight) ||
      !ptr16(k_norm_weight))
    return bad_arg("tensors must be 16-byte aligned");
  if (num_tokens > ((int64_t)1 << 31)) return bad_arg("num_tokens too large");
  return {};
}

// Rows rotated in place have to come back to where they were read: with another stride a row's result
// lands on rows that other lanes have yet to read.
inline ArgError check_rotate_in_place(const void *q_out, const void *k_out, const void *q, const void *k,
                                      const void *v, int64_t num_tokens, int64_t q_stride, int64_t q_out_stride,
                                      int64_t k_stride, int64_t k_out_stride) {
  if (num_tokens > 1 && q_out == q && q_out_stride != q_stride) return bad_arg("q rotated in place needs one stride");
  if (num_tokens > 1 && k_out && k_out == k && k_out_stride != k_stride)
    return bad_arg("k rotated in place needs one stride");
  if (q_out == k || q_out == v || q_out == k_out || (k_out && (k_out == q || k_out == v)))
    return bad_arg("outputs may be no other tensor of the call");
  return {};
}

inline ArgError check_cu(const int32_t *cu, int32_t n, const char *what) {
  if (cu[0] < 0) return bad_arg(what);
  for (int32_t i = 0; i < n; i++)
    if (cu[i + 1] < cu[i]) return bad_arg(what);
  return {};
}

inline ArgError check_prompt_args(const PagedAttnConfig &cfg, const void *out, const void *q, const void *k,
                                  const void *v, const int32_t *cu_q, const int32_t *cu_kv, int32_t num_seqs,
                                  int32_t num_q_heads, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                  int64_t out_stride, float scale, float softcap, const void *workspace,
                                  size_t workspace_bytes, size_t need_bytes) {
  const int64_t D = cfg.head_size, Hkv = cfg.num_kv_heads;
  if (num_q_heads <= 0 || num_q_heads % Hkv) return bad_arg("num_q_heads must be a positive multiple of num_kv_heads");
  if (num_q_heads / Hkv > 128) return ArgError{PA_ERR_UNSUPPORTED, "more than 128 query heads per kv head"};
  if (!cu_q) return bad_arg("cu_q_lens is null");
  if (ArgError e = check_cu(cu_q, num_seqs, "cu_q_lens must be non-negative and non-decreasing")) return e;
  if (cu_kv)
    if (ArgError e = check_cu(cu_kv, num_seqs, "cu_kv_lens must be non-negative and non-decreasing")) return e;
  const int32_t *ckv = cu_kv ? cu_kv : cu_q;
  if (cu_q[num_seqs] == cu_q[0]) return {};  // no query anywhere: nothing else is looked at
  if (!out || !q || (ckv[num_seqs] > ckv[0] && (!k || !v))) return bad_arg("null tensor pointer");
  const int64_t q_row = num_q_heads * D, kv_row = Hkv * D;
  if (q_stride < q_row || out_stride < q_row || k_stride < kv_row || v_stride < kv_row ||
      ((q_stride | out_stride | k_stride | v_stride) & 7))
    return bad_arg("row strides must cover a row and be multiples of 8");
  if (q_stride >= ((int64_t)1 << 38) || k_stride >= ((int64_t)1 << 38) || v_stride >= ((int64_t)1 << 38))
    return bad_arg("row strides must be below 2^38 elements");
  if (!ptr16(out) || !ptr16(q) || !ptr16(k) || !ptr16(v)) return bad_arg("tensors must be 16-byte aligned");
  if (!(scale > 0.f) || !(softcap > 0.f) || !std::isfinite(scale) || !std::isfinite(softcap))
    return bad_arg("scale and softcap must be finite and > 0");
  if (softcap != 1.0f && !std::isfinite(softcap / scale)) return bad_arg("softcap / scale must be finite");
  if (cu_q[num_seqs] > INT32_MAX - 1024 || ckv[num_seqs] > INT32_MAX - 1024)
    return bad_arg("more than 2^31 - 1024 query or key rows");
  if (!workspace || workspace_bytes < need_bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return bad_arg("workspace missing, too small or not 256-byte aligned");
  return {};
}

// The output in an input's place: a row that is recomputed reads its query after other lanes have written
// there, and every row its keys and values after the rows of other CTAs.
inline ArgError check_prompt_in_place(const void *out, const void *q, const void *k, const void *v) {
  if (out && (out == q || out == k || out == v)) return bad_arg("out may not be one of the inputs");
  return {};
}

inline ArgError check_gather_args(const PagedAttnConfig &cfg, const void *key, const void *value,
                                  const int32_t *block_tables, const int32_t *starts, const int32_t *cu,
                                  int32_t num_seqs, int32_t max_blocks, int64_t key_stride, int64_t value_stride) {
  if (!cu) return bad_arg("cu_lens is null");
  if (ArgError e = check_cu(cu, num_seqs, "cu_lens must be non-negative and non-decreasing")) return e;
  if (cu[num_seqs] == cu[0]) return {};
  if (!key || !value || !block_tables) return bad_arg("null tensor pointer");
  if (max_blocks <= 0) return bad_arg("max_blocks_per_seq must be > 0");
  for (int32_t i = 0; i < num_seqs; i++) {
    const int64_t first = starts ? starts[i] : 0, len = cu[i + 1] - cu[i];
    if (first < 0) return bad_arg("starts must be >= 0");
    if (len > 0 && first + len > (int64_t)max_blocks * cfg.block_size)
      return bad_arg("a range ends beyond the sequence's row of the block table");
  }
  const int64_t row = (int64_t)cfg.num_kv_heads * cfg.head_size;
  if (key_stride < row || value_stride < row || ((key_stride | value_stride) & 7))
    return bad_arg("row strides must cover a row and be multiples of 8");
  if (!ptr16(key) || !ptr16(value)) return bad_arg("tensors must be 16-byte aligned");
  return {};
}

// ---- partition of the prompt attention -------------------------------------------------------
// An item is one tile of query tokens of one (sequence, kv head); its work is the key tiles
// that the tile's last query sees.  Items are laid end to end - sequence, then kv head, then
// query tile - and the line is cut into one piece per CTA, pieces of equal cost.  A cut may
// fall inside an item: the CTAs on both sides then leave partial results that a second
// launch joins.  A cut closer than `min_piece` key tiles to an item's end moves there.
constexpr int kKeyTile = 128;     // keys of a tile
constexpr int kTileRows = 128;    // (token, head) rows of a query tile: one tensor-memory lane each
constexpr int kMaxPlanSeqs = 256; // sequences of one launch
constexpr int kMaxPlanCtas = 160;

struct PlanPos {
  int32_t seq, head, qt, kt;  // sequence, kv head, query tile, first key tile
};
inline bool operator==(const PlanPos &a, const PlanPos &b) {
  return a.seq == b.seq && a.head == b.head && a.qt == b.qt && a.kt == b.kt;
}

constexpr int kMinPiece = 2;         // a piece of an item is at least this many key tiles
constexpr int kMinTilesPerCta = 2;   // and a CTA gets work worth this many
// Costs in sixteenths of the time of a key tile with two query tiles (fitted to the CTAs' own times:
// an item costs two key tiles besides its tiles; one query tile alone runs two key tiles at a time,
// except with head sizes above 128).
constexpr int kCostTwo = 16, kCostOne = 9, kCostItem = 31, kCostZero = 4;

struct PromptShape {
  int32_t tile_tokens;  // query tokens of an item: tiles * (128 / group)
  int32_t sub_tokens;   // query tokens of one 128-row tile
  int32_t cost_one;     // of a key tile with one query tile
};
inline PromptShape prompt_shape(int head_size, int group) {
  PromptShape s;
  s.sub_tokens = kTileRows / group;
  s.tile_tokens = s.sub_tokens * (head_size <= 128 ? 2 : 1);
  s.cost_one = head_size <= 128 ? kCostOne : kCostTwo;
  return s;
}

// Key tiles that the queries [q0, q1) of a sequence see.
inline int32_t plan_key_tiles(int32_t q_len, int32_t kv_len, int32_t q1) {
  const int64_t keys = (int64_t)kv_len - q_len + q1;
  return keys <= 0 ? 0 : (int32_t)((std::min<int64_t>(keys, kv_len) + kKeyTile - 1) / kKeyTile);
}

struct PromptPlan {
  int32_t num_ctas = 0;
  PlanPos begin[kMaxPlanCtas + 1];  // CTA c works on [begin[c], begin[c + 1]); no piece is empty
  int32_t num_split = 0;
  int32_t split_first[kMaxPlanCtas];  // first and last CTA of each item that is cut
  int32_t split_last[kMaxPlanCtas];
};

// Plans sequences [s0, s1) of the batch (at most kMaxPlanSeqs).
inline void plan_prompt(const int32_t *cu_q, const int32_t *cu_kv, int32_t s0, int32_t s1, int32_t num_kv_heads,
                        PromptShape shape, int32_t max_ctas, int32_t min_piece, int32_t min_tiles_per_cta,
                        PromptPlan *plan) {
  plan->num_ctas = plan->num_split = 0;
  // prefix costs of the query tiles of each sequence (the same for each of its heads)
  std::vector<int64_t> prefix, group, base;
  std::vector<size_t> at;
  int64_t total = 0;
  for (int32_t s = s0; s < s1; s++) {
    const int32_t ql = cu_q[s + 1] - cu_q[s], kl = cu_kv[s + 1] - cu_kv[s];
    at.push_back(prefix.size());
    base.push_back(total);
    int64_t sum = 0;
    for (int32_t q = 0; q < ql;) {
      prefix.push_back(sum);
      const int32_t q1 = std::min(ql - q, shape.tile_tokens) + q;
      const int32_t n = plan_key_tiles(ql, kl, q1);
      sum += n == 0 ? kCostZero : kCostItem + (int64_t)n * (q1 - q > shape.sub_tokens ? kCostTwo : shape.cost_one);
      q = q1;
    }
    prefix.push_back(sum);
    group.push_back(sum);
    total += sum * num_kv_heads;
  }
  if (total == 0) return;
  const int64_t least = (int64_t)min_tiles_per_cta * kCostTwo;
  const int64_t ctas = std::max<int64_t>(1, std::min<int64_t>(std::min(max_ctas, kMaxPlanCtas), total / std::max<int64_t>(least, 1)));
  const PlanPos end{s1, 0, 0, 0};
  auto next_item = [&](PlanPos p) {
    const int32_t ql = cu_q[p.seq + 1] - cu_q[p.seq];
    p.kt = 0;
    if ((int64_t)(p.qt + 1) * shape.tile_tokens < ql) {
      p.qt++;
      return p;
    }
    p.qt = 0;
    if (++p.head < num_kv_heads) return p;
    p.head = 0;
    for (p.seq++; p.seq < s1 && cu_q[p.seq + 1] == cu_q[p.seq];) p.seq++;
    return p.seq < s1 ? p : end;
  };
  int32_t s = s0, n = 0;
  for (int64_t c = 0; c < ctas; c++) {
    // the position of share c of the total
    const int64_t r0 = total * c / ctas;
    while (group[s - s0] == 0 || r0 >= base[s - s0] + group[s - s0] * num_kv_heads) s++;
    int64_t r = r0 - base[s - s0];
    PlanPos p{s, (int32_t)(r / group[s - s0]), 0, 0};
    r -= (int64_t)p.head * group[s - s0];
    const int32_t ql = cu_q[s + 1] - cu_q[s], kl = cu_kv[s + 1] - cu_kv[s];
    const int64_t *pre = prefix.data() + at[s - s0];
    const int32_t tiles = (ql + shape.tile_tokens - 1) / shape.tile_tokens;
    p.qt = (int32_t)(std::upper_bound(pre, pre + tiles, r) - pre) - 1;
    r -= pre[p.qt];
    const int64_t q0 = (int64_t)p.qt * shape.tile_tokens;
    const int32_t q1 = (int32_t)std::min<int64_t>(q0 + shape.tile_tokens, ql);
    const int32_t kts = plan_key_tiles(ql, kl, q1);
    const int32_t unit = q1 - q0 > shape.sub_tokens ? kCostTwo : shape.cost_one;
    const int64_t kt = kts == 0 || r <= kCostItem / 2 ? 0 : std::max<int64_t>(0, (r - kCostItem + unit / 2) / unit);
    if (c > 0) {
      if (kt < min_piece) p.kt = 0;
      else if (kts - kt < min_piece) p = next_item(p);
      else p.kt = (int32_t)kt;
    }
    if (p == end || (n > 0 && plan->begin[n - 1] == p)) continue;
    plan->begin[n++] = p;
  }
  plan->begin[n] = end;
  plan->num_ctas = n;
  for (int32_t c = 1; c < n; c++) {
    const PlanPos &p = plan->begin[c];
    if (p.kt == 0) continue;
    int32_t k = plan->num_split - 1;
    if (k >= 0) {
      const PlanPos &o = plan->begin[plan->split_last[k]];
      if (o.seq == p.seq && o.head == p.head && o.qt == p.qt) {
        plan->split_last[k] = c;
        continue;
      }
    }
    k = plan->num_split++;
    plan->split_first[k] = c - 1;
    plan->split_last[k] = c;
  }
}

}  // namespace pa
