// Sanitizer check of the host arithmetic of the operators of a step with drafted tokens
// (hexagon-mlir_amd/csrc/host_logic.h): the cut of a batch in small steps, and
// layer_twins_disjoint against a marking of every element.  Built with
// g++ -fsanitize=address,undefined by tests/test_draft_host.py; prints "draft logic ok" and
// exits 0 when every check holds.
#include <algorithm>
#include <climits>
#include <cstdlib>
#include <random>
#include <set>
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

static std::mt19937_64 rng(22);
static int64_t pick(int64_t lo, int64_t hi) {
  return lo + static_cast<int64_t>(rng() % static_cast<uint64_t>(hi - lo + 1));
}

// A batch cut in small steps for `groups` workgroups, as the tree's kernel does, all workgroups
// at once.
static void check_cut(const std::vector<int32_t>& lens, int64_t heads, int32_t window,
                      int64_t capacity, uint32_t groups) {
  const size_t batch = lens.size();
  std::vector<int32_t> n(batch), lo(batch);
  std::vector<uint32_t> w(batch);
  uint64_t total = 0;
  for (size_t b = 0; b < batch; ++b) {
    n[b] = lens[b] > capacity ? 0 : std::max(lens[b], 0);
    lo[b] = window > 0 ? std::max(0, n[b] - window) : 0;
    w[b] = hxm::attn_units(n[b], lo[b]);
    total += w[b];
    CHECK(total < (uint64_t(1) << 32) || batch > 256, "units of 64 sequences pass 32 bits");
  }
  const int64_t grid = hxm::attn_grid(static_cast<int64_t>(batch), heads, capacity, groups);
  if (static_cast<int64_t>(batch) > hxm::kAttnCutBatch) return;  // a sequence a piece
  // What the host takes for whole is.
  if (capacity <= hxm::kAttnWhole * hxm::kAttnUnit)
    for (uint32_t u : w) CHECK(hxm::attn_cut(u, 2) <= 1, "a short sequence is cut");
  const uint32_t share = hxm::attn_share(total, heads, groups);
  uint32_t size = 0;
  bool fits = false;
  auto pieces_of = [&] {
    uint64_t p = 0;
    for (uint32_t u : w) p += hxm::attn_cut(u, size);
    return p;
  };
  if (batch <= 64)
    for (int k = 0; k < hxm::kAttnSteps && !fits; ++k) {
      const uint32_t last = size;
      size = hxm::attn_step_size(share, static_cast<uint32_t>(k));
      CHECK(size >= last && size >= share, "sizes go down");
      fits = pieces_of() * heads <= groups;
    }
  if (!fits) size = hxm::attn_fine_size(share);
  const uint64_t pieces = pieces_of();
  CHECK(static_cast<int64_t>(pieces * heads) <= grid, "%llu pieces of %lld heads, grid %lld",
        (unsigned long long)pieces, (long long)heads, (long long)grid);
  uint64_t slots = 0;
  for (size_t b = 0; b < batch; ++b) {
    const uint32_t c = hxm::attn_cut(w[b], size);
    CHECK(c >= 1, "sequence without a piece");
    if (c > 1) slots += c;
    const int64_t step = static_cast<int64_t>((w[b] + c - 1) / c) * hxm::kAttnUnit;
    const int64_t from = lo[b] & ~static_cast<int32_t>(hxm::kAttnTile - 1);
    CHECK(from + (c - 1) * step <= INT32_MAX - step, "a piece's end passes 32 bits");
    int64_t at = from;
    for (uint32_t i = 0; i < c && c < 100000; ++i) {
      const int64_t begin = from + i * step,
                    end = i + 1 < c ? std::min<int64_t>(n[b], begin + step) : n[b];
      CHECK(begin == at, "piece %u begins at %lld, not %lld", i, (long long)begin, (long long)at);
      CHECK(end > begin || n[b] == 0, "piece %u of %u of %d tokens is empty", i, c, n[b]);
      at = end;
    }
    if (c < 100000) CHECK(at == n[b], "pieces end at %lld of %d", (long long)at, n[b]);
  }
  CHECK(slots * heads <= 2 * hxm::kAttnFine * groups,
        "%llu partial results of %lld heads", (unsigned long long)slots, (long long)heads);
}

static void check_attention(uint32_t groups) {
  for (int64_t heads : {1, 2, 3, 8, 32, 64, 128, 255, 256, 257, 1000, 65535}) {
    for (int32_t len : {0, 1, 31, 32, 33, 127, 128, 129, 512, 513, 640, 1024, 4096, 32768, 1 << 20,
                        1 << 30})
      for (int64_t batch : {1, 2, 7, 63, 64, 65, 130, 255, 256, 257}) {
        if (batch * heads > (1 << 24)) continue;
        check_cut(std::vector<int32_t>(batch, len), heads, 0, len > 0 ? len : 32, groups);
        check_cut(std::vector<int32_t>(batch, len), heads, 1000, int64_t(1) << 30, groups);
        std::vector<int32_t> one(batch, 1);
        one[batch / 2] = len;
        check_cut(one, heads, 0, int64_t(1) << 30, groups);
      }
  }
  check_cut(std::vector<int32_t>(256, 1 << 12), 65535, 0, 1 << 12, groups);
  check_cut(std::vector<int32_t>(256, 1 << 30), 65535, 0, int64_t(1) << 30, groups);
  for (int i = 0; i < 4000; ++i) {
    const int64_t batch = pick(1, pick(0, 3) ? 80 : 300), heads = pick(1, pick(0, 1) ? 16 : 200);
    const int64_t top = int64_t(1) << pick(0, pick(0, 3) ? 15 : 30);
    std::vector<int32_t> lens(batch);
    const bool skew = pick(0, 1);
    for (auto& l : lens)
      l = static_cast<int32_t>(pick(0, 9) == 0 ? pick(-2, 1)
                                               : pick(0, skew && pick(0, 7) ? top / 64 : top));
    const int64_t capacity = pick(0, 3) ? top : top / 2 + 1;
    check_cut(lens, heads, pick(0, 1) ? 0 : static_cast<int32_t>(pick(1, top)), capacity, groups);
  }
}

static void check_layers() {
  int admitted = 0;
  for (int i = 0; i < 60000; ++i) {
    const int64_t width = pick(1, 3), eb = 2, delta = pick(-120, 120);
    int64_t n[4], s[4];
    for (int d = 0; d < 4; ++d) n[d] = pick(1, 3), s[d] = pick(0, 40);
    const uintptr_t a = 4096, b = static_cast<uintptr_t>(4096 + delta);
    std::set<int64_t> seen;
    bool apart = true;
    for (uintptr_t base : {a, b})
      for (int64_t at = 0; at < n[0] * n[1] * n[2] * n[3]; ++at) {
        int64_t rest = at, off = 0;
        for (int d = 0; d < 4; ++d) off += rest % n[d] * s[d], rest /= n[d];
        for (int64_t e = 0; e < width * eb; ++e)
          apart = seen.insert(static_cast<int64_t>(base) + off * eb + e).second && apart;
      }
    const bool says = hxm::layer_twins_disjoint(a, b, n, s, width, eb);
    admitted += says;
    if (says) CHECK(apart, "layer_twins_disjoint admits what collides, %lld apart", (long long)delta);
  }
  CHECK(admitted > 300, "only %d admitted", admitted);
  // Keys and values side by side in a row, a page and a layer; odd bytes; the range's ends.
  const int64_t n[4] = {3, 4, 2, 16};
  const int64_t row[4] = {16384, 4096, 2048, 128}, page[4] = {16384, 4096, 1024, 64},
                layer[4] = {16384, 2048, 1024, 64};
  CHECK(hxm::layer_twins_disjoint(4096, 4096 + 128, n, row, 64, 2), "side by side in a row");
  CHECK(hxm::layer_twins_disjoint(4096 + 4096, 4096, n, page, 64, 2), "in a page, the other way");
  CHECK(hxm::layer_twins_disjoint(4096, 4096 + 16384, n, layer, 64, 2), "in a layer");
  CHECK(!hxm::layer_twins_disjoint(4096, 4096 + 126, n, row, 64, 2), "rows that meet");
  CHECK(!hxm::layer_twins_disjoint(4096, 4096, n, row, 64, 2), "itself");
  CHECK(!hxm::layer_twins_disjoint(4096, 4097 + 128, n, row, 64, 2), "half an element off");
  CHECK(hxm::layer_twins_disjoint(0, UINTPTR_MAX - 1, n, row, 64, 2), "ends of the range");
}

int main() {
  check_attention(hxm::kAttnGroups);
  check_attention(2 * hxm::kAttnGroups);
  check_layers();
  if (failures) return 1;
  std::puts("draft logic ok");
  return 0;
}
