// Sanitizer check of how much hxm_tree_attention launches and keeps
// (hexagon-mlir_amd/csrc/host_logic.h): the pieces of any batch against attn_step_grid and
// attn_step_slots of what attn_span says, and that no sequence of a batch taken for whole is cut.
// Built with g++ -fsanitize=address,undefined by tests/test_draft_scratch_host.py; prints
// "draft scratch ok" and exits 0 when every check holds.
#include <algorithm>
#include <climits>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../hexagon-mlir_amd/csrc/host_logic.h"

static int failures = 0;
#define CHECK(cond, ...)                    \
  do {                                      \
    if (!(cond)) {                          \
      std::fprintf(stderr, __VA_ARGS__);    \
      std::fputc('\n', stderr);             \
      if (++failures > 20) std::exit(1);    \
    }                                       \
  } while (0)

static std::mt19937_64 rng(23);
static int64_t pick(int64_t lo, int64_t hi) {
  return lo + static_cast<int64_t>(rng() % static_cast<uint64_t>(hi - lo + 1));
}

static int tight = 0;  // batches that come within a workgroup of each head of the bound

static void check_batch(const std::vector<int32_t>& lens, int64_t heads, int64_t window,
                        int64_t capacity, uint32_t groups) {
  const int64_t batch = static_cast<int64_t>(lens.size());
  const int64_t span = hxm::attn_span(capacity, window);
  const int64_t grid = hxm::attn_step_grid(batch, heads, span, groups);
  const int64_t most = hxm::attn_step_slots(batch, heads, span, groups);
  CHECK(span <= capacity && grid >= batch * heads && most <= grid, "bounds out of order");
  if (batch > hxm::kAttnCutBatch) return;
  std::vector<uint32_t> w(lens.size());
  uint64_t total = 0;
  for (size_t b = 0; b < lens.size(); ++b) {
    const int32_t n = lens[b] > capacity ? 0 : std::max(lens[b], 0);
    const int32_t lo = window > 0 ? static_cast<int32_t>(std::max<int64_t>(0, n - window)) : 0;
    w[b] = hxm::attn_units(n, lo);
    CHECK(w[b] <= 1 || static_cast<int64_t>(w[b]) <= hxm::ceil_div(span, hxm::kAttnUnit),
          "%u units of %d tokens, window %lld, span %lld", w[b], n, (long long)window,
          (long long)span);
    total += w[b];
  }
  const uint32_t share = hxm::attn_share(total, static_cast<uint64_t>(heads), groups);
  uint32_t size = 0;
  auto pieces_of = [&] {
    uint64_t p = 0;
    for (uint32_t u : w) p += hxm::attn_cut(u, size);
    return p;
  };
  bool fits = false;
  for (uint32_t k = 0; batch <= 64 && k < hxm::kAttnSteps && !fits; ++k) {
    size = hxm::attn_step_size(share, k);
    fits = pieces_of() * heads <= groups;
  }
  if (!fits) size = hxm::attn_fine_size(share);
  const int64_t pieces = static_cast<int64_t>(pieces_of()) * heads;
  int64_t slots = 0;
  for (uint32_t u : w) {
    const uint32_t c = hxm::attn_cut(u, size);
    if (c > 1) slots += c * heads;
  }
  CHECK(pieces <= grid, "%lld pieces for %lld workgroups (%lld sequences, %lld heads, span %lld)",
        (long long)pieces, (long long)grid, (long long)batch, (long long)heads, (long long)span);
  CHECK(slots <= most, "%lld partial results for %lld", (long long)slots, (long long)most);
  if (span <= hxm::kAttnWhole * hxm::kAttnUnit) CHECK(slots == 0, "a whole sequence is cut");
  tight += grid - pieces < heads;
}

int main() {
  for (uint32_t groups : {hxm::kAttnGroups, 2 * hxm::kAttnGroups}) {
    for (int64_t heads : {1, 2, 3, 8, 32, 64, 127, 128, 129, 255, 256, 257, 1000})
      for (int64_t batch : {1, 2, 3, 4, 7, 16, 32, 63, 64, 65, 256, 257})
        for (int64_t window : {0, 1, 480, 481, 482, 513, 1055, 4096, 1 << 20, 1 << 30})
          for (int64_t top : {1, 511, 512, 513, 640, 16384, 1 << 20, 1 << 30}) {
            std::vector<int32_t> lens(batch, static_cast<int32_t>(top));
            check_batch(lens, heads, window, top, groups);
            std::fill(lens.begin() + 1, lens.end(), 1);
            check_batch(lens, heads, window, top, groups);
            for (auto& l : lens) l = static_cast<int32_t>(pick(-1, top));
            check_batch(lens, heads, window, top, groups);
          }
    for (int i = 0; i < 200000; ++i) {
      const int64_t batch = pick(1, pick(0, 7) ? 64 : 300), heads = pick(1, pick(0, 1) ? 16 : 300);
      const int64_t top = int64_t(1) << pick(0, pick(0, 3) ? 15 : 30);
      std::vector<int32_t> lens(batch);
      const int64_t few = pick(1, top);
      for (auto& l : lens) l = static_cast<int32_t>(pick(0, 3) ? few : pick(-1, top));
      check_batch(lens, heads, pick(0, 1) ? 0 : pick(1, top), pick(0, 3) ? top : top / 2 + 1,
                  groups);
    }
  }
  CHECK(tight > 1000, "only %d batches near the bound", tight);
  // 5 sequences of 3 tiles, 25 nodes with a window of 1000; 4 of 16 over 32768 tokens.
  CHECK(hxm::attn_step_slots(5, 3, hxm::attn_span(16384, 1024), 512) == 75, "a window's scratch");
  CHECK(hxm::attn_step_slots(4, 16, hxm::attn_span(32768, 0), 512) == 512, "a few long sequences'");
  CHECK(hxm::attn_step_slots(64, 4, 1 << 20, 512) == 512, "half as many pairs as workgroups");
  CHECK(hxm::attn_step_slots(64, 5, 1 << 20, 512) == 1536 + 320, "and more of them");
  CHECK(hxm::attn_step_slots(256, 1000, 1 << 20, 512) == 6 * 512, "the most");
  if (failures) return 1;
  std::puts("draft scratch ok");
  return 0;
}
