// Launch shape of omni_adapter_linear: for every spread of the tokens over the adapters (and over no adapter) the row
// blocks fit the grid, and the parts of the reduction cover it once.
#include <stdarg.h>

#include <random>

#include "../../omni_infer_amd/csrc/host_logic.h"

void omni_set_error(const char* fmt, ...) { (void)fmt; }

#define CHECK(c)                                                                        \
  do {                                                                                  \
    if (!(c)) {                                                                         \
      printf("%s fails: T=%d n=%d H=%d r=%d S=%d\n", #c, T, n, H, r, S);                \
      return 1;                                                                         \
    }                                                                                   \
  } while (0)

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
  for (int it = 0; it < 20000; ++it) {
    const int T = it % 3 ? pick(1, 200) : pick(1, 20000), n = pick(1, it % 2 ? 8 : 256);
    const int H = 8 * pick(1, it % 5 ? 200 : 2000), r = 8 * pick(1, 32), S = pick(1, 4);
    const omni_host::AdapterPlan p = omni_host::adapter_plan(T, n, H, r, S);
    CHECK(p.row_tiles == 1 || p.row_tiles == 4);
    CHECK(p.row_tiles == 1 || r <= 128);  // what the second launch keeps in shared memory
    CHECK(p.ksplit >= 1 && p.ksplit <= 16 && p.col_blocks >= 1);
    CHECK(p.rank_block == 16 || p.rank_block == 32 || p.rank_block == 64 || p.rank_block == 128);
    // the tokens at random, all but a few alone, or all with one adapter
    std::vector<int> c(n + 1, 0);
    const int kind = pick(0, 2);
    for (int t = 0; t < T; ++t) ++c[kind == 0 ? pick(0, n) : kind == 1 ? (t < n ? t : n) : 0];
    int blocks = 0, none = 0;
    const int bm = 16 * p.row_tiles;
    for (int g = 0; g < n; ++g) blocks += (c[g] + bm - 1) / bm;
    none = (c[n] + bm - 1) / bm;
    CHECK(blocks <= p.tiles_max);
    CHECK(blocks + none <= p.tiles_max + 1);
    const int chunks = (H + 63) / 64, per = (chunks + p.ksplit - 1) / p.ksplit;
    CHECK((int64_t)per * p.ksplit >= chunks);
  }
  puts("ok");
  return 0;
}
