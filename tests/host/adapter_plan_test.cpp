// Launch shape of omni_adapter_linear: for every spread of the tokens over the adapters (and over no adapter) the row
// blocks fit the grid, and the parts of the reduction cover it once.
#include <stdarg.h>

#include <random>

#include "../../omni_infer_amd/csrc/host_logic.h"

void omni_set_error(const char* fmt, ...) { (void)fmt; }

#define CHECK(c)                                                                        \
  do {                                                                                  \
    if (!(c)) {                                                                         \
      printf("%s fails: T=%d n=%d H=%d r=%d S=%d N=%d\n", #c, T, n, H, r, S, N);                \
      return 1;                                                                         \
    }                                                                                   \
  } while (0)

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
  for (int it = 0; it < 20000; ++it) {
    const int T = it % 3 ? pick(1, 200) : pick(1, 20000), n = pick(1, it % 2 ? 8 : 256);
    const int H = 8 * pick(1, it % 5 ? 200 : 2000), r = 8 * pick(1, 32), S = pick(1, 4), N = 8 * pick(1, 2000);
    const omni_host::AdapterPlan p = omni_host::adapter_plan(T, n, H, r, S, N);
    CHECK(p.row_tiles == 1 || (p.row_tiles == 8 && p.rank_block >= 64));
    CHECK(p.out_row_tiles == 1 || p.out_row_tiles == 2);
    CHECK(!p.fused || (r <= 64 && p.row_tiles == 1 && p.out_row_tiles == 1 && p.ksplit == 1));
    CHECK(p.ksplit >= 1 && p.ksplit <= 16 && p.unit_blocks >= 1);
    CHECK(p.rank_block == 16 || p.rank_block == 32 || p.rank_block == 64 || p.rank_block == 128);
    // the tokens at random, all but a few alone, or all with one adapter
    std::vector<int> c(n + 1, 0);
    const int kind = pick(0, 2);
    for (int t = 0; t < T; ++t) ++c[kind == 0 ? pick(0, n) : kind == 1 ? (t < n ? t : n) : 0];
    for (int out = 0; out < 2; ++out) {
      const int bm = 16 * (out ? p.out_row_tiles : p.row_tiles), most = out ? p.out_tiles_max : p.tiles_max;
      int blocks = 0;
      for (int g = 0; g < n; ++g) blocks += (c[g] + bm - 1) / bm;
      CHECK(blocks <= most);
      CHECK(blocks + (c[n] + bm - 1) / bm <= most + 1);
    }
    const int chunks = (H + 63) / 64, per = (chunks + p.ksplit - 1) / p.ksplit;
    CHECK((int64_t)per * p.ksplit >= chunks);
  }
  puts("ok");
  return 0;
}
