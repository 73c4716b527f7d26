// Sanitizer check of twins_disjoint (hexagon-mlir_amd/csrc/host_logic.h): built with
// g++ -fsanitize=address,undefined by tests/test_decoder_host.py and compared with a
// marking of every element.  Prints "overlap logic ok" and exits 0 when every check holds.
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

static std::mt19937_64 rng(21);
static int64_t pick(int64_t lo, int64_t hi) {
  return lo + static_cast<int64_t>(rng() % static_cast<uint64_t>(hi - lo + 1));
}

int main() {
  int admitted = 0;
  for (int i = 0; i < 60000; ++i) {
    const int dims = static_cast<int>(pick(0, 3));
    const int64_t width = pick(1, 4), eb = 2, delta = pick(-90, 90);
    int64_t n[3] = {1, 1, 1}, s[3] = {0, 0, 0};
    for (int d = 0; d < dims; ++d) n[d] = pick(1, 4), s[d] = pick(0, 24);
    const uintptr_t a = 4096, b = static_cast<uintptr_t>(4096 + delta);
    std::set<int64_t> seen;
    bool apart = true;
    for (uintptr_t base : {a, b})
      for (int64_t x = 0; x < n[0]; ++x)
        for (int64_t y = 0; y < n[1]; ++y)
          for (int64_t z = 0; z < n[2]; ++z)
            for (int64_t e = 0; e < width * eb; ++e)
              apart = seen.insert(static_cast<int64_t>(base) +
                                  (x * s[0] + y * s[1] + z * s[2]) * eb + e).second && apart;
    const bool says = hxm::twins_disjoint(a, b, n, s, dims, width, eb);
    admitted += says;
    // May refuse what happens not to collide, never admit what does.
    if (says)
      CHECK(apart, "twins_disjoint admits %lld,%lld,%lld at %lld,%lld,%lld width %lld, %lld apart",
            (long long)n[0], (long long)n[1], (long long)n[2], (long long)s[0], (long long)s[1],
            (long long)s[2], (long long)width, (long long)delta);
  }
  CHECK(admitted > 1000, "only %d admitted", admitted);
  // Heads of q, k and v side by side; either order; odd bytes; the ends of the address range.
  const int64_t n[2] = {100, 8}, s[2] = {8 * 192, 192};
  CHECK(hxm::twins_disjoint(4096, 4096 + 128, n, s, 2, 64, 2), "k after q");
  CHECK(hxm::twins_disjoint(4096 + 256, 4096, n, s, 2, 64, 2), "v after q, the other way");
  CHECK(!hxm::twins_disjoint(4096, 4096 + 126, n, s, 2, 64, 2), "k into q");
  CHECK(!hxm::twins_disjoint(4096, 4096 + 258, n, s, 2, 64, 2), "k into the next q");
  CHECK(!hxm::twins_disjoint(4096, 4096, n, s, 2, 64, 2), "itself");
  CHECK(!hxm::twins_disjoint(4096, 4097 + 128, n, s, 2, 64, 2), "half an element off");
  CHECK(hxm::twins_disjoint(0, UINTPTR_MAX - 1, n, s, 2, 64, 2), "ends of the range");
  CHECK(!hxm::twins_disjoint(4096, 8192, n, s, 4, 64, 2), "four dims are not its own");
  if (failures) return 1;
  std::printf("overlap logic ok\n");
  return 0;
}
