// Sanitizer check of the host-only arithmetic of the decoder-layer operators
// (hexagon-mlir_amd/csrc/host_logic.h): built with g++ -fsanitize=address,undefined
// by tests/test_decoder_host.py.  The overlap rules are compared with a marking
// of every element, the division by multiplication with the division, and paged attention's
// cut of a batch is walked piece by piece as its kernel walks it: every token in
// one piece, every piece in the launched grid, every partial result in its
// workspace.  Prints "decoder logic ok" and exits 0 when every check holds.
#include <algorithm>
#include <climits>
#include <cstdlib>
#include <cstring>
#include <random>
#include <set>
#include <string>
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

static std::mt19937_64 rng(20);
static int64_t pick(int64_t lo, int64_t hi) {
  return lo + static_cast<int64_t>(rng() % static_cast<uint64_t>(hi - lo + 1));
}

static void check_fast_div() {
  auto one = [](uint32_t n, uint32_t d, const hxm::FastDiv& f) {
    const uint32_t q = static_cast<uint32_t>((static_cast<uint64_t>(n) * f.mul) >> f.shift);
    CHECK(q == n / d, "fast_div %u / %u gives %u", n, d, q);
  };
  auto with = [&](uint32_t d) {
    const hxm::FastDiv f = hxm::fast_div(d);
    for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 2 * d - 1, 0x7ffffffeu, 0x7fffffffu})
      if (n <= 0x7fffffffu) one(n, d, f);
    for (int i = 0; i < 200; ++i) one(static_cast<uint32_t>(rng()) >> 1, d, f);
    for (int i = 0; i < 50; ++i) {
      const uint64_t q = rng() % (0x7fffffffu / d + 1);
      for (int64_t n : {static_cast<int64_t>(q * d) - 1, static_cast<int64_t>(q * d)})
        if (n >= 0 && n <= 0x7fffffff) one(static_cast<uint32_t>(n), d, f);
    }
  };
  for (uint32_t d = 1; d <= 300; ++d) with(d);
  for (uint32_t p = 1; p < 31; ++p)
    for (int o = -1; o <= 1; ++o)
      if ((1u << p) + o >= 1) with((1u << p) + o);
  with(0x7fffffffu);
  for (int i = 0; i < 2000; ++i) with(1 + static_cast<uint32_t>(rng() % 0x7fffffffu));
}

static void check_strides_disjoint() {
  for (int i = 0; i < 40000; ++i) {
    int64_t n[3], s[3];
    const int dims = static_cast<int>(pick(0, 3));
    const int64_t width = pick(1, 4);
    for (int d = 0; d < 3; ++d) n[d] = pick(1, 4), s[d] = pick(0, 20);
    std::set<int64_t> seen;
    bool apart = true;
    for (int64_t a = 0; a < (dims > 0 ? n[0] : 1); ++a)
      for (int64_t b = 0; b < (dims > 1 ? n[1] : 1); ++b)
        for (int64_t c = 0; c < (dims > 2 ? n[2] : 1); ++c)
          for (int64_t e = 0; e < width; ++e) {
            const int64_t at = (dims > 0 ? a * s[0] : 0) + (dims > 1 ? b * s[1] : 0) +
                               (dims > 2 ? c * s[2] : 0) + e;
            apart = seen.insert(at).second && apart;
          }
    // The rule may refuse what happens not to collide, never admit what does; nested
    // strides it must admit.
    if (hxm::strides_disjoint(n, s, dims, width))
      CHECK(apart, "strides_disjoint admits %lld,%lld,%lld at %lld,%lld,%lld width %lld",
            (long long)n[0], (long long)n[1], (long long)n[2], (long long)s[0], (long long)s[1],
            (long long)s[2], (long long)width);
    int64_t nested[3], span = width;
    for (int d = 0; d < 3; ++d) nested[d] = span + pick(0, 3), span += nested[d] * (n[d] - 1);
    CHECK(hxm::strides_disjoint(n, nested, 3, width), "strides_disjoint refuses nested strides");
  }
  const int64_t far[3] = {INT32_MAX, 65535, INT32_MAX},
                wide[3] = {int64_t(1) << 40, int64_t(1) << 40, int64_t(1) << 40};
  CHECK(!hxm::strides_disjoint(far, wide, 3, 256), "equal strides are not apart");
}

static void check_matrices_disjoint() {
  for (int i = 0; i < 40000; ++i) {
    const int64_t rows = pick(0, 4), ca = pick(0, 5), cb = pick(0, 5), eb = pick(0, 1) ? 2 : 4;
    const int64_t lda = ca + pick(0, 12), ldb = pick(0, 1) ? lda : cb + pick(0, 12);
    if (ldb < cb) continue;
    const uintptr_t a = 1000, b = 1000 + static_cast<uintptr_t>(pick(-120, 120) * 2);
    std::set<int64_t> seen;
    bool apart = true;
    for (int64_t r = 0; r < rows; ++r)
      for (int64_t e = 0; e < ca * eb; ++e) seen.insert(static_cast<int64_t>(a) + r * lda * eb + e);
    for (int64_t r = 0; r < rows; ++r)
      for (int64_t e = 0; e < cb * eb; ++e)
        apart = apart && !seen.count(static_cast<int64_t>(b) + r * ldb * eb + e);
    if (hxm::matrices_disjoint(a, lda, b, ldb, rows, ca, cb, eb))
      CHECK(apart, "matrices_disjoint admits ld %lld %lld, cols %lld %lld, %lld rows",
            (long long)lda, (long long)ldb, (long long)ca, (long long)cb, (long long)rows);
  }
  // Columns [0, 8) and [8, 16) of one matrix, and whole buffers one after the other.
  CHECK(hxm::matrices_disjoint(4096, 16, 4096 + 16, 16, 100, 8, 8, 2), "columns side by side");
  CHECK(!hxm::matrices_disjoint(4096, 16, 4096 + 14, 16, 100, 8, 8, 2), "columns that meet");
  CHECK(hxm::matrices_disjoint(4096, 8, 4096 + 1600, 9, 100, 8, 9, 2), "one after the other");
  CHECK(!hxm::matrices_disjoint(4096, 8, 4096 + 1598, 9, 100, 8, 9, 2), "one into the other");
}

// A batch cut as find_piece of the kernel does, all workgroups at once.
static void check_cut(const std::vector<int32_t>& lens, int64_t heads, int32_t window,
                      int64_t capacity) {
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
  const int64_t grid = hxm::attn_grid(static_cast<int64_t>(batch), heads, capacity);
  if (static_cast<int64_t>(batch) > hxm::kAttnCutBatch) {  // a sequence a piece
    CHECK(grid == static_cast<int64_t>(batch) * heads, "grid of a batch that is not cut");
    return;
  }
  const uint32_t share = hxm::attn_share(total, heads);
  uint32_t size = 0;
  bool fits = false;
  auto pieces_of = [&] {
    uint64_t p = 0;
    for (uint32_t u : w) p += hxm::attn_cut(u, size);
    return p;
  };
  if (batch <= 64)
    for (uint32_t k = 0; k < 4 && !fits; ++k) {
      size = hxm::attn_size(share, k);
      fits = pieces_of() * heads <= hxm::kAttnGroups;
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
  CHECK(slots * heads <= 2 * hxm::kAttnFine * hxm::kAttnGroups,
        "%llu partial results of %lld heads", (unsigned long long)slots, (long long)heads);
}

static void check_attention() {
  for (int64_t heads : {1, 2, 3, 8, 32, 64, 128, 255, 256, 257, 1000, 65535}) {
    for (int32_t len : {0, 1, 31, 32, 33, 127, 128, 129, 512, 513, 640, 1024, 4096, 32768, 1 << 20,
                        1 << 30})
      for (int64_t batch : {1, 2, 7, 63, 64, 65, 130, 255, 256, 257}) {
        if (batch * heads > (1 << 24)) continue;
        check_cut(std::vector<int32_t>(batch, len), heads, 0, len > 0 ? len : 32);
        check_cut(std::vector<int32_t>(batch, len), heads, 1000, int64_t(1) << 30);
        std::vector<int32_t> one(batch, 1);
        one[batch / 2] = len;
        check_cut(one, heads, 0, int64_t(1) << 30);
      }
  }
  check_cut(std::vector<int32_t>(256, 1 << 12), 65535, 0, 1 << 12);
  check_cut(std::vector<int32_t>(256, 1 << 30), 65535, 0, int64_t(1) << 30);
  for (int i = 0; i < 4000; ++i) {
    const int64_t batch = pick(1, pick(0, 3) ? 80 : 300), heads = pick(1, pick(0, 1) ? 16 : 200);
    const int64_t top = int64_t(1) << pick(0, pick(0, 3) ? 15 : 30);
    std::vector<int32_t> lens(batch);
    const bool skew = pick(0, 1);
    for (auto& l : lens)
      l = static_cast<int32_t>(pick(0, 9) == 0 ? pick(-2, 1)
                                               : pick(0, skew && pick(0, 7) ? top / 64 : top));
    const int64_t capacity = pick(0, 3) ? top : top / 2 + 1;
    check_cut(lens, heads, pick(0, 1) ? 0 : static_cast<int32_t>(pick(1, top)), capacity);
  }
}

int main() {
  check_fast_div();
  check_strides_disjoint();
  check_matrices_disjoint();
  check_attention();
  if (failures) return 1;
  std::printf("decoder logic ok\n");
  return 0;
}
