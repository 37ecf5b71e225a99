// Routing limited to groups of experts.  With l the logits of a row,
//   s = sigmoid(l) or softmax(l) over all experts,  c = s + bias,
//   a group's value = the sum of its group_top (1 or 2) largest c; the topk_group groups of the largest values stay,
//   the k experts of the largest c among theirs are picked, best first (ties: the smaller index, for groups and experts),
//   w = s of the pick, divided by (the picks' sum + 1e-20) when renorm is set, times scale.
// The selection is that of exact arithmetic as far as 64 bits tell: scores, sums and comparisons are fp64.
#include "hb_common.cuh"
#include "hb_kernels.h"

namespace hb {

constexpr int RG_WARPS = 4;

struct RouteGroupedArgs {
  const float* logits; int ld, M, E, k, n_group, topk_group, group_top, sigmoid, renorm; const float* bias; float scale; int32_t* ids; float* w;
};

// a before b: the larger value, the smaller index among equals; NaN comes after everything
__device__ __forceinline__ bool rg_before(double a, int ia, double b, int ib) { return a > b || (a == b && ia < ib); }

__global__ void __launch_bounds__(RG_WARPS * 32) route_grouped_kernel(const RouteGroupedArgs a) {
  extern __shared__ double rg_sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, m = blockIdx.x * RG_WARPS + warp;
  griddep_wait();
  if (m >= a.M) return;
  double* c = rg_sm + (size_t)warp * a.E;
  const float* lr = a.logits + (size_t)m * a.ld;
  auto logit = [&](int e) -> double { const float v = lr[e]; return v == v ? (double)v : -INFINITY; };   // NaN counts as -inf
  double mx = -INFINITY, sum = 0.0;
  if (!a.sigmoid) {
    for (int e = lane; e < a.E; e += 32) mx = fmax(mx, logit(e));
    for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    for (int e = lane; e < a.E; e += 32) sum += exp(logit(e) - mx);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  auto score = [&](int e) -> double {
    if (a.sigmoid) return 1.0 / (1.0 + exp(-logit(e)));
    return mx == -INFINITY ? 0.0 : exp(logit(e) - mx) / sum;                 // a row without a finite logit: all scores 0
  };
  for (int e = lane; e < a.E; e += 32) {
    const double v = score(e) + (a.bias ? (double)a.bias[e] : 0.0);
    c[e] = v == v ? v : -INFINITY;                                               // NaN is picked last
  }
  __syncwarp();
  const int size = a.E / a.n_group;
  uint32_t keep = 0xffffffffu;
  if (a.topk_group < a.n_group) {
    double v = -INFINITY;
    if (lane < a.n_group) {
      double t1 = -INFINITY, t2 = -INFINITY;
      for (int i = 0; i < size; ++i) { const double x = c[lane * size + i]; if (x > t1) { t2 = t1; t1 = x; } else if (x > t2) t2 = x; }
      v = a.group_top == 2 && size > 1 ? t1 + t2 : t1;
    }
    int rank = 0;
    for (int g = 0; g < a.n_group; ++g) rank += rg_before(__shfl_sync(0xffffffffu, v, g), g, v, lane);
    keep = __ballot_sync(0xffffffffu, lane < a.n_group && rank < a.topk_group);
  }
  uint32_t gone = 0u;                                                            // bit j: expert lane + 32 j is not to be had
  for (int j = 0, e = lane; e < a.E; ++j, e += 32) if (!((keep >> (e / size)) & 1u)) gone |= 1u << j;
  int id = 0;
  for (int r = 0; r < a.k; ++r) {
    double b = -INFINITY; int at = 0x7fffffff;
    for (int j = 0, e = lane; e < a.E; ++j, e += 32) {
      if ((gone >> j) & 1u) continue;
      if (at == 0x7fffffff || rg_before(c[e], e, b, at)) { b = c[e]; at = e; }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, b, o); const int oa = __shfl_xor_sync(0xffffffffu, at, o);
      if (oa != 0x7fffffff && (at == 0x7fffffff || rg_before(ob, oa, b, at))) { b = ob; at = oa; }
    }
    if ((at & 31) == lane) gone |= 1u << (at >> 5);
    if (lane == r) id = at;
  }
  double s = lane < a.k ? score(id) : 0.0, tot = 0.0;
  if (!(s == s)) s = 0.0;
  for (int r = 0; r < a.k; ++r) tot += __shfl_sync(0xffffffffu, s, r);
  if (a.renorm) s /= tot + 1e-20;
  if (lane < a.k) { a.ids[(size_t)m * a.k + lane] = id; a.w[(size_t)m * a.k + lane] = (float)(s * (double)a.scale); }
}

}  // namespace hb

using namespace hb;

extern "C" int hb_route_grouped_topk(hb_ctx* ctx, const float* logits, int ld, int M, int E, int k, int n_group, int topk_group, int group_top, int score,
                                     const float* bias, int renorm, float scale, int32_t* ids, float* w, void* stream) {
  if (!ctx) return HB_ERR_INVALID;
  if (M == 0) return HB_OK;
  HB_REQUIRE(ctx, logits && ids && w, HB_ERR_INVALID, "route_grouped_topk: NULL argument");
  HB_REQUIRE(ctx, M > 0 && E > 0 && E <= HB_MAX_EXPERTS && ld >= E && k >= 1 && k <= 16, HB_ERR_UNSUPPORTED,
             "route_grouped_topk: M=%d E=%d (1..%d) ld=%d (>= E) k=%d (1..16)", M, E, HB_MAX_EXPERTS, ld, k);
  HB_REQUIRE(ctx, n_group >= 1 && n_group <= 32 && E % n_group == 0 && topk_group >= 1 && topk_group <= n_group && k <= topk_group * (E / n_group),
             HB_ERR_UNSUPPORTED, "route_grouped_topk: n_group=%d (1..32, a divisor of E=%d) topk_group=%d (1..n_group) k=%d (at most the experts of the groups kept)",
             n_group, E, topk_group, k);
  HB_REQUIRE(ctx, (group_top == 1 || group_top == 2) && (score == HB_SCORE_SOFTMAX || score == HB_SCORE_SIGMOID), HB_ERR_INVALID,
             "route_grouped_topk: group_top=%d (1 or 2) score=%d", group_top, score);
  RouteGroupedArgs a{logits, ld, M, E, k, n_group, topk_group, group_top, score == HB_SCORE_SIGMOID, renorm, bias, scale, ids, w};
  return hb_launch(ctx, "route_grouped", !(ctx->flags & HB_FLAG_NO_PDL), route_grouped_kernel, dim3((M + RG_WARPS - 1) / RG_WARPS), dim3(RG_WARPS * 32),
                   (size_t)RG_WARPS * E * 8, reinterpret_cast<cudaStream_t>(stream), a);
}
