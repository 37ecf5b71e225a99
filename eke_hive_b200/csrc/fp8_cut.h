// How a product on 8-bit floats is cut into items, steps and forms, and the room its parts take: plain arithmetic, the same for the host that sizes the
// workspace and launches, for the kernels, and for a test without a GPU.
#pragma once
#include <cstddef>
#include <cstdint>
#include <initializer_list>

#ifdef __CUDACC__
#define HB_HD __host__ __device__ __forceinline__
#else
#define HB_HD inline
#endif

namespace hb {

constexpr int F8_B = 128;                              // values a scale covers
HB_HD constexpr int f8_blocks(int n) { return (n + F8_B - 1) / F8_B; }

constexpr int F8_MAX_CTAS = 160;                       // grid at most; the workspace holds two partial items of each
constexpr int F8S_ROWS = 128, F8P_ROWS = 256;          // rows of x a tile of the many-row kernel may have: one CTA, a pair
constexpr uint32_t F8S_WHOLE = 16;                     // steps up to which an item of single CTAs stays whole: putting its sums together takes some 8 (two CTAs) or 12 (four)
constexpr uint32_t F8P_SLACK = 40;                     // steps that cutting has to save: leaving and adding up parts takes a pair some 20 us

// The steps of a CTA, the same for all its warps: segments (item, first step, end).
struct F8Sched {                                       // (32 bits: at most 320 items of at most 2^16 steps, or 2^24 steps, times 160 CTAs)
  uint32_t KB, G, me, dp, sk, U, Gs, end, u, u1, i;
  // runs: no rounds, the whole list in equal runs (as long as its steps can be counted so): a CTA stays with an expert.  Else rounds, and of what they leave over
  // items are cut where that saves more than `slack` steps
  HB_HD void init(uint32_t items, uint32_t KB_, uint32_t G_, uint32_t me_, bool runs, uint32_t slack) {
    KB = KB_; G = G_; me = me_;
    const uint32_t waves = items / G, rem = items - waves * G;
    const bool all = runs && (unsigned long long)items * KB < (1ull << 24);
    const bool cut = rem != 0u && (unsigned long long)(G - rem) * KB > (unsigned long long)slack * G;
    dp = all ? 0u : !cut ? waves + (rem != 0u) : waves > 0u ? waves - 1u : 0u;   // rounds of whole items, after the cut ones
    sk = all || cut ? items - dp * G : 0u;
    U = sk * KB; end = items;
    const uint32_t some = U > 1u ? U : 1u;
    Gs = G < some ? G : some;                                                  // CTAs that get a run of steps: none is empty
    u = start(me); u1 = start(me + 1u);
    i = 0u;
  }
  HB_HD uint32_t start(uint32_t c) const { return c >= Gs ? U : c * U / Gs; }
  HB_HD bool next(int& item, int& kb0, int& kb1) {
    if (u < u1) {
      item = (int)(u / KB); kb0 = (int)(u - (uint32_t)item * KB);
      const uint32_t to = (uint32_t)kb0 + (u1 - u);
      kb1 = (int)(to < KB ? to : KB);
      u += (uint32_t)(kb1 - kb0);
      return true;
    }
    if (i >= dp) return false;
    item = (int)(sk + i * G + me); kb0 = 0; kb1 = (int)KB; ++i;
    return (uint32_t)item < end;
  }
  HB_HD uint32_t owner(uint32_t step) const { return ((step + 1u) * Gs - 1u) / U; }
};
// Steps of a CTA of the one-CTA form of the many-row kernel: rounds of whole items, then the items left over, each split among the CTAs of a cluster where there are
// enough clusters.
struct F8Rounds {
  uint32_t KB, G, me, dp, rem, split, i;
  HB_HD void init(uint32_t items, uint32_t KB_, uint32_t G_, uint32_t me_, bool, uint32_t cluster) {
    KB = KB_; G = G_; me = me_;
    dp = items / G; rem = items - dp * G;
    split = rem * cluster <= G && KB > F8S_WHOLE ? cluster : 1u;
    i = 0u;
  }
  HB_HD bool splits() const { return split > 1u && me / split < rem; }         // the same for all CTAs of a cluster
  HB_HD bool next(int& item, int& kb0, int& kb1) {
    if (i > dp) return false;
    if (i++ < dp) { item = (int)((i - 1u) * G + me); kb0 = 0; kb1 = (int)KB; return true; }
    const uint32_t t = me / split, r = me - t * split;
    if (t >= rem) return false;
    item = (int)(dp * G + t); kb0 = (int)(KB * r / split); kb1 = (int)(KB * (r + 1u) / split);
    return true;
  }
};

// What the forms run on: SMs, CTAs a context may use (0: all), clusters of four CTAs of the one-CTA form that are resident at once.
struct F8Gpu { int sm_count, max_ctas, clusters; };
// CTAs of a launch: one an SM, in whole clusters of cl.  Not all SMs are in reach of clusters of four.
inline int f8_grid(const F8Gpu& g, int rows, int cl) {
  int n = g.max_ctas > 0 && g.max_ctas < g.sm_count ? g.max_ctas : g.sm_count;
  if (n > F8_MAX_CTAS) n = F8_MAX_CTAS;
  if (cl == 4 && rows == F8S_ROWS && n > 4 * g.clusters) n = 4 * g.clusters;
  return n < cl ? cl : n / cl * cl;
}
// sums of cut items: two of each CTA.  (A row of x a lane: in pairs alone.)
inline size_t f8_part_bytes(int rows) { return (size_t)F8_MAX_CTAS * 2 * 256 * (rows == F8P_ROWS ? 128 : rows == F8S_ROWS ? 32 : rows) * 4; }
// Rows of the largest tile that a dense product of M rows may take, whatever N, K and the GPU: what its workspace is sized for.
inline int f8_most_rows(int M) { return M <= 16 ? 16 : M <= 32 ? 32 : M <= F8S_ROWS ? F8S_ROWS : F8P_ROWS; }
// How a dense product is cut.  Up to 32 rows a weight row a lane (17408 x 5120, 32 rows: 24 us; a row of x a lane: 28).  More: a row of x a lane, tiles of 128 rows
// of single CTAs or, from 129 rows on, of 256 of pairs, by the steps the longest CTA takes.  Single: rounds of whole items, what is left over split among the two or four
// CTAs of a cluster where there are that many, at the price of some 8 and 12 steps (128 rows of 4096 x 4096: 21 us whole, 17 in two, 15 in four; 2048 x 512: 6.4, 9.3, 10.3).
// Pairs: a step takes a tenth less, as an SM pulls less out of L2 (512 rows of 18944 x 4096: 42 us, single CTAs 44; 5120 x 17408, where half the pairs' work is left over
// and cut through the workspace: 62 and 74; 2048 rows of 5120 x 5120, split in two: 65 and 63).  Up to 128 rows half of a pair's tile would be empty (64 rows of
// 4096 x 1536: 10.3 us, single CTAs 10.2; 64 or 128 rows of 7168 x 2048 the same within 1 %), and no parts are left: a pair's take 42 MB, the workspace of so few rows has 10.
struct F8Cut { int rows, split; };
inline F8Cut f8_cut(const F8Gpu& g, int M, int N, int K) {
  const int most = f8_most_rows(M);
  if (most < F8S_ROWS) return {most, 1};
  const long long KB = f8_blocks(K), n_nt = ((long long)N + 255) / 256;
  F8Cut best{F8S_ROWS, 1};
  long long least = 0;
  for (int c : {1, 2, 4}) {
    const long long G = f8_grid(g, F8S_ROWS, c), items = (M + F8S_ROWS - 1) / F8S_ROWS * n_nt, rem = items % G;
    if (c > 1 && (rem * c > G || KB <= F8S_WHOLE)) continue;
    const long long steps = items / G * KB + (rem == 0 ? 0 : c == 1 ? KB : (KB + c - 1) / c + (c == 2 ? 8 : 12));
    if (c == 1 || steps < least) { least = steps; best.split = c; }
  }
  if (most < F8P_ROWS) return best;
  const long long G = f8_grid(g, F8P_ROWS, 2) / 2, items = (M + F8P_ROWS - 1) / F8P_ROWS * n_nt, rem = items % G, cut = (KB * rem + G - 1) / G + F8P_SLACK;
  const long long steps = items / G * KB + (rem == 0 ? 0 : cut < KB ? cut : KB);
  return 9 * steps < 10 * least ? F8Cut{F8P_ROWS, 2} : best;
}

}  // namespace hb
