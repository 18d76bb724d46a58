// Which kernels omni_adapter_linear launches: for every line "T n H r S N" of the input, or without any for many drawn
// shapes, the first and the second product's kernel, and the parts of the reduction.
#include <stdarg.h>

#include <random>
#include <set>
#include <string>

#include "../../omni_infer_amd/csrc/host_logic.h"

void omni_set_error(const char* fmt, ...) { (void)fmt; }

static std::string kernels(int T, int n, int H, int r, int S, int N, int& parts) {
  const omni_host::AdapterPlan p = omni_host::adapter_plan(T, n, H, r, S, N);
  parts = p.ksplit;
  const std::string ranks = r <= 16 ? "16" : r <= 32 ? "32" : r <= 64 ? "64" : "256";
  if (p.fused) return "one_launch_" + ranks;
  return std::string(p.row_tiles == 8 ? "tile_" : "rows_") + std::to_string(p.rank_block) + " out" +
         std::to_string(p.out_row_tiles) + "_" + (r <= 32 ? "32" : ranks);
}

int main(int argc, char**) {
  int T, n, H, r, S, N, parts;
  if (argc > 1) {
    while (scanf("%d %d %d %d %d %d", &T, &n, &H, &r, &S, &N) == 6) {
      const std::string k = kernels(T, n, H, r, S, N, parts);
      printf("%s parts %d\n", k.c_str(), parts);
    }
    return 0;
  }
  std::set<std::string> seen;
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
  for (int it = 0; it < 300000; ++it) {
    T = 1 << pick(0, 14), T += pick(0, T), n = pick(1, it % 2 ? 8 : 256), r = 8 * pick(1, 32), S = pick(1, 4);
    H = 8 * pick(1, 2000), N = 8 * pick(S, 2000);
    seen.insert(kernels(T, n, H, r, S, N, parts));
  }
  for (const std::string& k : seen) puts(k.c_str());
  return 0;
}
