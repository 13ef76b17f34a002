// Host side of the prompt-path entry points, checked without a device: the partition of the
// attention's work covers every (item, key tile) exactly once, the rotation table's phases
// are exact, and the argument checks refuse what they should.
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <tuple>

#include "../mlx-node_b200/csrc/prompt_host.hpp"

using namespace pa;

static int failures = 0;
#define EXPECT(c)                                                   \
  do {                                                              \
    if (!(c)) {                                                     \
      std::printf("line %d: %s\n", __LINE__, #c);                   \
      failures++;                                                   \
    }                                                               \
  } while (0)

// Walks the plan the way a CTA does and counts the key tiles of every item.
static void check_plan(const std::vector<int32_t> &ql, const std::vector<int32_t> &kl, int heads, int head_size,
                       int group, int ctas, int min_piece, int min_tiles) {
  std::vector<int32_t> cq{0}, ck{0};
  for (size_t i = 0; i < ql.size(); i++) cq.push_back(cq.back() + ql[i]), ck.push_back(ck.back() + kl[i]);
  const PromptShape shape = prompt_shape(head_size, group);
  PromptPlan plan;
  const int S = (int)ql.size();
  plan_prompt(cq.data(), ck.data(), 0, S, heads, shape, ctas, min_piece, min_tiles, &plan);
  std::map<std::tuple<int, int, int>, std::vector<std::pair<int, int>>> seen;
  std::map<std::tuple<int, int, int>, std::set<int>> by;
  for (int c = 0; c < plan.num_ctas; c++) {
    PlanPos p = plan.begin[c];
    const PlanPos e = plan.begin[c + 1];
    EXPECT(!(p == e));
    int guard = 0;
    while (!(p == e) && guard++ < 1000000) {
      const int32_t q1 = std::min(ql[p.seq], (p.qt + 1) * shape.tile_tokens);
      const int32_t n = plan_key_tiles(ql[p.seq], kl[p.seq], q1);
      const bool cut = e.seq == p.seq && e.head == p.head && e.qt == p.qt;
      const int32_t k1 = cut ? e.kt : n;
      EXPECT(p.kt < k1 || (n == 0 && p.kt == 0));
      seen[{p.seq, p.head, p.qt}].push_back({p.kt, k1});
      by[{p.seq, p.head, p.qt}].insert(c);
      if (cut) break;
      p.kt = 0;
      if ((p.qt + 1) * shape.tile_tokens < ql[p.seq]) p.qt++;
      else {
        p.qt = 0;
        if (++p.head == heads) {
          p.head = 0;
          for (p.seq++; p.seq < S && ql[p.seq] == 0;) p.seq++;
        }
      }
    }
  }
  size_t items = 0, split = 0;
  for (int s = 0; s < S; s++)
    for (int q = 0; q * shape.tile_tokens < ql[s]; q++)
      for (int h = 0; h < heads; h++) {
        items++;
        auto &v = seen[{s, h, q}];
        const int n = plan_key_tiles(ql[s], kl[s], std::min(ql[s], (q + 1) * shape.tile_tokens));
        EXPECT(!v.empty() && v.front().first == 0 && v.back().second == n);
        for (size_t i = 1; i < v.size(); i++) EXPECT(v[i].first == v[i - 1].second);
        if (v.size() > 1) split++;
      }
  EXPECT(seen.size() == items);
  EXPECT((int)split == plan.num_split);
  for (int k = 0; k < plan.num_split; k++) {
    const PlanPos &p = plan.begin[plan.split_last[k]];
    const auto &c = by[{p.seq, p.head, p.qt}];
    EXPECT(*c.begin() == plan.split_first[k] && *c.rbegin() == plan.split_last[k]);
    EXPECT((int)c.size() == plan.split_last[k] - plan.split_first[k] + 1);
  }
}

int main() {
  // ---- partition -----------------------------------------------------------------------
  check_plan({1}, {1}, 1, 128, 1, 148, 2, 3);
  check_plan({0, 0}, {5, 0}, 2, 128, 4, 148, 2, 3);
  check_plan({5}, {0}, 2, 64, 4, 148, 2, 3);
  check_plan({300}, {200}, 2, 128, 4, 148, 1, 1);
  check_plan({8192}, {8192}, 8, 128, 4, 148, 2, 3);
  check_plan({1, 1, 3}, {16000, 4000, 32000}, 8, 128, 8, 148, 2, 3);
  check_plan({1024, 1024}, {5120, 5120}, 8, 256, 4, 148, 2, 3);
  std::mt19937 rng(7);
  for (int it = 0; it < 800; it++) {
    std::vector<int32_t> ql, kl;
    const int S = 1 + rng() % 12;
    for (int s = 0; s < S; s++) {
      ql.push_back(rng() % 4 == 0 ? 0 : rng() % (rng() % 3 ? 40 : 2000));
      kl.push_back(rng() % 5 == 0 ? rng() % (ql.back() + 1) : ql.back() + rng() % 5000);
    }
    const int heads[] = {32, 64, 80, 128, 192, 256};
    check_plan(ql, kl, 1 + rng() % 8, heads[rng() % 6], 1 + rng() % 128, 1 + rng() % 160, 1 + rng() % 6, rng() % 8);
  }
  // ---- rotation table --------------------------------------------------------------------
  {
    PaRopeConfig c{128, 0, 1e6f, PA_ROPE_PLAIN, 1.f, 0, 0.f, 0.f, 0.f, 0.f, 0.f};
    EXPECT(!check_rope_config(c));
    RopeTable t;
    build_rope_table(c, &t);
    EXPECT(t.gain == 1.f && t.dims == 128);
    const long double two_pi = 6.283185307179586476925286766559005768L;
    const int64_t positions[] = {0, 1, -1, 1000003, 2147483647, -2147483647 - 1};
    for (int i = 0; i < 64; i++)
      for (int64_t pos : positions) {
        const uint64_t phase = (uint64_t)pos * t.turn[i];
        long double want = std::fmod((long double)pos * (rope_frequency(c, i) / two_pi), 1.0L);
        long double got = std::ldexp((long double)(int64_t)phase, -64);
        long double d = got - want;
        d -= std::floor(d + 0.5L);
        // the entry is off by half a unit of 2^-64 turns, and the product of the right-hand
        // side by half a step of a 64-bit mantissa: 2^31 * 2^-65 + 2^31 * 2^-64
        EXPECT(std::fabs(d) <= 0x1p-32L);
      }
    PaRopeConfig bad = c;
    bad.rope_dims = 7; EXPECT(check_rope_config(bad));
    bad.rope_dims = 0; EXPECT(check_rope_config(bad));
    bad.rope_dims = 258; EXPECT(check_rope_config(bad));
    bad = c; bad.interleaved = 2; EXPECT(check_rope_config(bad));
    bad = c; bad.base = 0.f; EXPECT(check_rope_config(bad));
    bad = c; bad.base = INFINITY; EXPECT(check_rope_config(bad));
    bad = c; bad.base = NAN; EXPECT(check_rope_config(bad));
    bad = c; bad.scaling = 4; EXPECT(check_rope_config(bad));
    bad = c; bad.scaling = PA_ROPE_LINEAR; bad.factor = 0.f; EXPECT(check_rope_config(bad));
    bad = c; bad.scaling = PA_ROPE_BANDS; bad.low_freq_factor = 1.f; bad.high_freq_factor = 4.f; EXPECT(check_rope_config(bad));
    bad.original_max_position = 8192; EXPECT(!check_rope_config(bad));
    bad.high_freq_factor = 1.f; EXPECT(check_rope_config(bad));
    bad = c; bad.scaling = PA_ROPE_YARN; bad.original_max_position = 4096; bad.beta_fast = 32.f; EXPECT(check_rope_config(bad));
    bad.beta_slow = 1.f; EXPECT(!check_rope_config(bad));
    bad.base = 1.f; EXPECT(check_rope_config(bad));
    bad = c; bad.attention_factor = -1.f; EXPECT(check_rope_config(bad));
  }
  // ---- argument checks -------------------------------------------------------------------
  {
    const PagedAttnConfig cfg{16, 8, 128, 2, 1, 1};
    void *const p = reinterpret_cast<void *>(0x10000), *const odd = reinterpret_cast<void *>(0x10008);
    RopeTable t{};
    t.dims = 128;
    const int32_t *pos = static_cast<const int32_t *>(p);
    const int64_t *slots = static_cast<const int64_t *>(p);
    auto rotate = [&](const RopeTable *r, const void *qo, const void *ko, const void *q, const void *v, float eps,
                      const int64_t *sl, int64_t n, int hq, int64_t qs, int64_t ks) {
      return check_rotate_args(cfg, r, qo, ko, q, p, v, p, nullptr, eps, pos, sl, n, hq, qs, 512, ks, 256, 256).code;
    };
    EXPECT(rotate(&t, p, p, p, p, 1e-6f, slots, 4, 4, 512, 256) == PA_OK);
    EXPECT(rotate(&t, p, nullptr, p, p, 1e-6f, slots, 4, 4, 512, 256) == PA_OK);
    EXPECT(rotate(&t, p, p, p, nullptr, 1e-6f, nullptr, 4, 4, 512, 256) == PA_OK);
    EXPECT(rotate(nullptr, p, p, p, p, 1e-6f, slots, 4, 4, 512, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, nullptr, p, p, p, 1e-6f, slots, 4, 4, 512, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, nullptr, p, p, 1e-6f, nullptr, 4, 4, 512, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, p, p, nullptr, 1e-6f, slots, 4, 4, 512, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, p, odd, p, 1e-6f, slots, 4, 4, 512, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, p, p, p, -1.f, slots, 4, 4, 512, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, p, p, p, NAN, slots, 4, 4, 512, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, p, p, p, 1e-6f, slots, 4, 3, 512, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, p, p, p, 1e-6f, slots, 4, 4, 504, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, p, p, p, 1e-6f, slots, 4, 4, 516, 256) == PA_ERR_INVALID_ARG);
    EXPECT(rotate(&t, p, p, p, p, 1e-6f, slots, (int64_t)1 << 40, 4, 512, 256) == PA_ERR_INVALID_ARG);
    t.dims = 130;
    EXPECT(rotate(&t, p, p, p, p, 1e-6f, slots, 4, 4, 512, 256) == PA_ERR_INVALID_ARG);

    const int32_t cu[] = {0, 5, 9}, down[] = {0, 5, 4}, neg[] = {-1, 5, 9};
    auto prompt = [&](const void *q, const void *k, const int32_t *cq, const int32_t *ck, int hq, int64_t qs, float scale,
                      float cap, const void *ws, size_t have) {
      return check_prompt_args(cfg, p, q, k, p, cq, ck, 2, hq, qs, 256, 256, 512, scale, cap, ws, have, 1000).code;
    };
    EXPECT(prompt(p, p, cu, nullptr, 4, 512, 1.f, 1.f, p, 1000) == PA_OK);
    EXPECT(prompt(p, p, cu, cu, 4, 512, 1.f, 30.f, p, 2000) == PA_OK);
    EXPECT(prompt(p, p, nullptr, cu, 4, 512, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, down, cu, 4, 512, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, neg, 4, 512, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(nullptr, p, cu, cu, 4, 512, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, nullptr, cu, cu, 4, 512, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, odd, cu, cu, 4, 512, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, cu, 5, 768, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, cu, 2 * 129, 1 << 20, 1.f, 1.f, p, 1000) == PA_ERR_UNSUPPORTED);
    EXPECT(prompt(p, p, cu, cu, 4, 508, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, cu, 4, 512, 0.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, cu, 4, 512, NAN, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, cu, 4, 512, 1.f, -1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, cu, 4, 512, 1.f, 1.f, p, 999) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, cu, 4, 512, 1.f, 1.f, odd, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, cu, cu, 4, 512, 1e-38f, 30.f, p, 1000) == PA_ERR_INVALID_ARG);  // softcap / scale
    const int32_t huge[] = {0, 5, INT32_MAX};
    EXPECT(prompt(p, p, cu, huge, 4, 512, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    EXPECT(prompt(p, p, huge, huge, 4, 512, 1.f, 1.f, p, 1000) == PA_ERR_INVALID_ARG);
    const int32_t none[] = {0, 0, 0}, later[] = {7, 7, 7};
    EXPECT(prompt(p, nullptr, cu, later, 4, 512, 1.f, 1.f, p, 1000) == PA_OK);
    EXPECT(prompt(nullptr, nullptr, none, cu, 4, 512, 1.f, 1.f, nullptr, 0) == PA_OK);
    EXPECT(prompt(p, nullptr, cu, none, 4, 512, 1.f, 1.f, p, 1000) == PA_OK);

    const int32_t starts[] = {3, 0}, minus[] = {-1, 0}, late[] = {60, 0};
    auto gather = [&](const void *key, const int32_t *st, const int32_t *c, int mb, int64_t ks) {
      return check_gather_args(cfg, key, p, pos, st, c, 2, mb, ks, 256).code;
    };
    EXPECT(gather(p, nullptr, cu, 1, 256) == PA_OK);
    EXPECT(gather(p, starts, cu, 1, 256) == PA_OK);
    EXPECT(gather(p, minus, cu, 1, 256) == PA_ERR_INVALID_ARG);
    EXPECT(gather(p, late, cu, 4, 256) == PA_ERR_INVALID_ARG);  // 60 + 5 > 64
    EXPECT(gather(p, late, cu, 5, 256) == PA_OK);
    EXPECT(gather(p, starts, down, 1, 256) == PA_ERR_INVALID_ARG);
    EXPECT(gather(p, starts, cu, 0, 256) == PA_ERR_INVALID_ARG);
    EXPECT(gather(odd, starts, cu, 1, 256) == PA_ERR_INVALID_ARG);
    EXPECT(gather(p, starts, cu, 1, 248) == PA_ERR_INVALID_ARG);
    EXPECT(gather(nullptr, starts, cu, 1, 256) == PA_ERR_INVALID_ARG);
    EXPECT(gather(nullptr, nullptr, none, 1, 256) == PA_OK);
  }
  std::printf(failures ? "%d failures\n" : "ok\n", failures);
  return failures ? 1 : 0;
}
