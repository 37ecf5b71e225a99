// Host check of csrc/fp8_cut.h, compiled and run by test_fp8_cut_cpu.py: for a grid of products, on GPUs of several sizes, every step of every item is done once, by
// as many CTAs as the arrival counter of a cut item waits for, and the parts they leave lie within the workspace that a product of that many rows is given.
// Prints the rows, workspace bytes and form of each product asked for as an argument triple M N K, after the grid.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "fp8_cut.h"

using namespace hb;

static int fail(const F8Gpu& g, int M, int N, int K, const F8Cut& c, const char* what, long long v) {
  printf("M=%d N=%d K=%d on %d SMs, %d CTAs, %d clusters: rows %d split %d: %s (%lld)\n", M, N, K, g.sm_count, g.max_ctas, g.clusters, c.rows, c.split, what, v);
  return 1;
}

static int check(const F8Gpu& g, int M, int N, int K) {
  const F8Cut cut = f8_cut(g, M, N, K);
  const long long room = (long long)f8_part_bytes(f8_most_rows(M));
  const uint32_t KB = f8_blocks(K), n_nt = (N + 255) / 256;
  const int nt = (M + cut.rows - 1) / cut.rows;
  const uint32_t items = nt * n_nt;
  std::vector<uint32_t> done(items, 0u);
  if (cut.rows == F8S_ROWS) {                                    // split items meet in shared memory: no parts
    const uint32_t G = f8_grid(g, cut.rows, cut.split);
    for (uint32_t c = 0; c < G; ++c) {
      F8Rounds s;
      s.init(items, KB, G, c, false, cut.split);
      int item, k0, k1;
      while (s.next(item, k0, k1)) { if (k1 <= k0) return fail(g, M, N, K, cut, "empty segment", c); done[item] += k1 - k0; }
    }
  } else {
    const int ctas = cut.rows == F8P_ROWS ? 2 : 1;
    const uint32_t G = f8_grid(g, cut.rows, ctas) / ctas;
    const long long part = 256ll * (ctas == 2 ? 128 : cut.rows) * 4;   // bytes of one
    std::vector<uint32_t> arrived(G, 0u);
    for (uint32_t c = 0; c < G; ++c) {
      F8Sched s;
      s.init(items, KB, G, c, ctas == 1, ctas == 2 ? F8P_SLACK : 0u);
      const uint32_t run = s.start(c);
      int item, k0, k1;
      while (s.next(item, k0, k1)) {
        if (k1 <= k0) return fail(g, M, N, K, cut, "empty segment", c);
        done[item] += k1 - k0;
        if ((uint32_t)(k1 - k0) == KB) continue;
        const uint32_t s0 = (uint32_t)item * KB, first = s.owner(s0), last = s.owner(s0 + KB - 1);
        if (c < first || c > last || last >= G) return fail(g, M, N, K, cut, "owner", c);
        for (int r = 0; r < ctas; ++r) {
          const long long end = (((long long)ctas * c + r) * 2 + (c == first && run != s0 ? 1 : 0) + 1) * part;
          if (end > room) return fail(g, M, N, K, cut, "a part ends behind the workspace", end - room);
        }
        if (ctas * first + ctas - 1 >= 2u * F8_MAX_CTAS) return fail(g, M, N, K, cut, "counter", first);
        if (++arrived[first] == last - first + 1) arrived[first] = 0u;
      }
    }
    for (uint32_t c = 0; c < G; ++c) if (arrived[c]) return fail(g, M, N, K, cut, "a counter is left", c);
  }
  for (uint32_t i = 0; i < items; ++i) if (done[i] != KB) return fail(g, M, N, K, cut, "steps of an item", i);
  return 0;
}

int main(int argc, char** argv) {
  const int Ms[] = {1, 16, 17, 32, 33, 48, 64, 96, 127, 128, 129, 200, 256, 257, 300, 512, 1000};
  const int Ns[] = {1, 64, 256, 257, 512, 640, 1024, 2048, 4100, 5120, 7168, 17408};
  const int Ks[] = {16, 128, 2048, 2064, 4096, 12288, 12816, 13312, 14400, 15376, 16384, 17408, 20480, 32768, 131072, 1 << 20, 1 << 23};
  const F8Gpu gpus[] = {{148, 0, 37}, {148, 0, 32}, {148, 0, 36}, {132, 0, 33}, {160, 0, 40}, {148, 1, 37}, {148, 2, 37}, {148, 3, 37}, {148, 7, 37}, {148, 64, 37}, {148, 147, 37}};
  for (const F8Gpu& g : gpus)
    for (int M : Ms)
      for (int N : Ns)
        for (int K : Ks)
          if (check(g, M, N, K)) return 1;
  srand(1);
  for (int i = 0; i < 200000; ++i) {
    const int M = 1 + rand() % 400, N = 1 + rand() % (rand() % 2 ? 3000 : 20000), K = 16 * (1 + rand() % 2000);
    if (check(gpus[rand() % 11], M, N, K)) return 1;
  }
  for (int i = 1; i + 2 < argc; i += 3) {
    const int M = atoi(argv[i]);
    const F8Cut c = f8_cut(gpus[0], M, atoi(argv[i + 1]), atoi(argv[i + 2]));
    printf("%d %zu %d\n", c.rows, f8_part_bytes(f8_most_rows(M)), c.split);
  }
  return 0;
}
