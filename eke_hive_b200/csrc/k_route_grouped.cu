// Routing limited to groups of experts.  With l the logits of a row,
//   s = sigmoid(l) or softmax(l) over all experts,  c = s + bias,
//   a group's value = the sum of its group_top (1 or 2) largest c; the topk_group groups of the largest values stay,
//   the k experts of the largest c among theirs are picked, best first (ties: the smaller index, for groups and experts),
//   w = s of the pick, divided by (the picks' sum + 1e-20) when renorm is set, times scale.
// The selection is that of 64-bit arithmetic.
#include <type_traits>

#include "hb_common.cuh"
#include "hb_kernels.h"

namespace hb {

// One warp takes a row.  The scores are worked out in fp32 with an error bound, and so is the selection; wherever two neighbours of the result (two
// picks next to each other, the last pick and the best expert left out that is not its equal by its inputs, the last group kept and the best one dropped) are
// closer than their bounds, and are not equal by their inputs, 64 bits decide: between experts for the candidates alone, a lane each; between groups for the groups' values; for scores at the end of
// fp32's range the warp does the whole row again.  64 bits for every row took 37 us for 8192 rows of 256 experts (this way 15)
// and 12 us for one (6).
constexpr int RG_WARPS = 4;

struct RouteGroupedArgs {
  const float* logits; int ld, M, E, k, n_group, topk_group, group_top, sigmoid, renorm; const float* bias; float scale; int32_t* ids; float* w;
};

// A bias in the range of finite values, NaN the lowest: no sum of two is NaN, whose order would be nobody's.
__device__ __forceinline__ float rg_bias(const RouteGroupedArgs& a, int e) {
  constexpr float top = 3.402823466e38f;
  return a.bias ? fminf(fmaxf(__ldg(a.bias + e), -top), top) : 0.f;
}

// a before b: the larger value, the smaller index among equals
__device__ __forceinline__ bool rg_before(double a, int ia, double b, int ib) { return a > b || (a == b && ia < ib); }

// A row in 64 bits; c: E doubles of shared memory of the warp's own.  Lane l < k gets pick l.
__device__ __noinline__ void route_grouped_row64(const RouteGroupedArgs& a, const float* lr, double* c, int lane, int& id, float& w) {
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
    return mx == -INFINITY ? 0.0 : exp(logit(e) - mx) / sum;                     // a row without a finite logit: all scores 0
  };
  for (int e = lane; e < a.E; e += 32) {
    const double v = score(e) + (double)rg_bias(a, e);
    c[e] = v == v ? v : -INFINITY;
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
  id = 0;
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
  double s = lane < a.k ? score(id) : 0.0, tot = 0.0;                            // (NaN in a softmax row with +inf)
  for (int r = 0; r < a.k; ++r) tot += __shfl_sync(0xffffffffu, s, r);
  if (a.renorm) s /= tot + 1e-20;
  w = (float)(s * (double)a.scale);
}

__device__ __forceinline__ uint32_t rg_key(float v) {                            // orders like the value; 0 is below everything
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float rg_exp(float x) {                               // e^x, off by 2 + 1.2 |x| steps; 0 below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504088896341f));
  return r;
}
__device__ __forceinline__ float rg_rcp(float x) {                               // 1 / x, off by a step
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rg_val(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// The groups a row keeps (a bit each), in 64 bits: where fp32 does not settle the last one kept.  c: E doubles of the warp's own; mx: the row's largest logit.
__device__ __noinline__ uint32_t route_grouped_keep64(const RouteGroupedArgs& a, const float* lr, double* c, float mx, int lane) {
  double scale = 1.0;                                                            // of exp(l - max): without a bias it changes no order
  if (!a.sigmoid) {
    double sum = 0.0;
    for (int e = lane; e < a.E; e += 32) { const float v = __ldg(lr + e); const double p = v == v ? exp((double)v - (double)mx) : 0.0; c[e] = p; sum += p; }
    if (a.bias) {
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      scale = 1.0 / sum;
    }
  }
  for (int e = lane; e < a.E; e += 32) {
    double s;
    if (a.sigmoid) { const float v = __ldg(lr + e); s = v == v ? 1.0 / (1.0 + exp(-(double)v)) : 0.0; }
    else s = a.bias ? c[e] * scale : c[e];
    c[e] = a.bias ? s + (double)rg_bias(a, e) : s;
  }
  __syncwarp();
  const int size = a.E / a.n_group;
  double v = -INFINITY;
  for (int g = 0; g < a.n_group; ++g) {                                          // a group at a time by all lanes
    double t1 = -INFINITY, t2 = -INFINITY;
    for (int i = lane; i < size; i += 32) { const double x = c[g * size + i]; t2 = fmax(t2, fmin(t1, x)); t1 = fmax(t1, x); }
    for (int o = 16; o > 0; o >>= 1) {
      const double o1 = __shfl_xor_sync(0xffffffffu, t1, o), o2 = __shfl_xor_sync(0xffffffffu, t2, o);
      t2 = fmax(fmax(t2, o2), fmin(t1, o1)); t1 = fmax(t1, o1);
    }
    if (lane == g) v = a.group_top == 2 && size > 1 ? t1 + t2 : t1;
  }
  int rank = 0;
  for (int g = 0; g < a.n_group; ++g) rank += rg_before(__shfl_sync(0xffffffffu, v, g), g, v, lane);
  __syncwarp();
  return __ballot_sync(0xffffffffu, lane < a.n_group && rank < a.topk_group);
}

// The row in fp32; R: experts a lane holds (e = lane + 32 j).  Returns false where fp32 does not settle the selection.
template <int R, bool SIG>
__device__ __forceinline__ bool route_grouped_row32(const RouteGroupedArgs& a, const float* lr, float* c, int lane, int& id, float& w) {
  float s[R]; uint32_t key[R];
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane + 32 * j;
    s[j] = e < a.E ? fmaxf(__ldg(lr + e), -INFINITY) : -INFINITY;                // (NaN gives way)
    if (!SIG) mx = fmaxf(mx, s[j]);
  }
  // Error of a score, against the other scores of the row, with rg_exp off by 2 + 1.2 |x| steps and rg_rcp by one.
  // sigmoid: the exponential counts 1 - s times: relative 2^-18 down to logits of -20 (err() sees to it), absolute (a bias beside it) 3.5 steps of 1.
  // softmax: l - max = -d is off by half a step of d besides, the sum (the same for all) by some 20 steps.  Without a bias the sum does not count: relative
  // 2^-17 for d < 20.  With one: e^-d (2 + 1.7 d) + 20 steps of the largest score.
  float eps = a.bias ? 0x1p-21f : 0x1p-18f, low = 0x1p-28f;
  float inv_sum = 1.f;
  bool safe = true;
  if (SIG) {
#pragma unroll
    for (int j = 0; j < R; ++j) s[j] = rg_rcp(1.f + rg_exp(-s[j]));
  } else {
    mx = rg_val(__reduce_max_sync(0xffffffffu, rg_key(mx)));
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < R; ++j) { s[j] = rg_exp(s[j] - mx); sum += s[j]; }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float r = __frcp_rn(sum);
    inv_sum = r; low = r * 0x1p-28f;
#pragma unroll
    for (int j = 0; j < R; ++j) s[j] *= r;
    eps = a.bias ? r * 0x1p-18f : 0x1p-17f;
    safe = mx > -INFINITY && mx < INFINITY;
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int e = lane + 32 * j;
    const float v = e < a.E ? s[j] + rg_bias(a, e) : 0.f;
    if (e < a.E) c[lane + 36 * j] = v;                                           // (four words aside every 32: a group's lanes below meet no bank conflicts)
    key[j] = e < a.E ? rg_key(v) : 0u;
  }
  __syncwarp();
  // bound of the error of a value v = score + bias
  auto err = [&](float v) { return a.bias ? fmaf(fabsf(v), 0x1p-23f, eps) : v > low ? v * (eps + 0x1p-23f) : INFINITY; };
  if (a.topk_group < a.n_group) {
    const int size = a.E / a.n_group;
    int T = 1, lg = 0;                                                           // lanes a group gets: a power of two
    while (2 * T * a.n_group <= 32) { T *= 2; ++lg; }
    const int g = lane >> lg, t = lane & (T - 1);
    float t1 = -INFINITY, t2 = -INFINITY;
    if (g < a.n_group) {
#pragma unroll 4
      for (int i = t; i < size; i += T) { const int e = g * size + i; const float x = c[e + (e >> 5) * 4]; t2 = fmaxf(t2, fminf(t1, x)); t1 = fmaxf(t1, x); }
    }
    for (int o = T >> 1; o > 0; o >>= 1) {
      const float o1 = __shfl_xor_sync(0xffffffffu, t1, o), o2 = __shfl_xor_sync(0xffffffffu, t2, o);
      t2 = fmaxf(fmaxf(t2, o2), fminf(t1, o1)); t1 = fmaxf(t1, o1);
    }
    const bool two = a.group_top == 2 && size > 1;
    float v = two ? t1 + t2 : t1, ve = two ? err(t1) + err(t2) + fabsf(v) * 0x1p-23f : err(t1);
    v = __shfl_sync(0xffffffffu, v, (lane << lg) & 31); ve = __shfl_sync(0xffffffffu, ve, (lane << lg) & 31);   // lane g: group g
    int rank = 0;
    for (int i = 0; i < a.n_group; ++i) { const float ov = __shfl_sync(0xffffffffu, v, i); rank += ov > v || (ov == v && i < lane); }
    const bool in = lane < a.n_group;
    uint32_t keep = __ballot_sync(0xffffffffu, in && rank < a.topk_group);
    // the lowest a kept group can be against the highest a dropped one can be
    const float lo = rg_val(__reduce_min_sync(0xffffffffu, in && rank < a.topk_group ? rg_key(v - ve) : 0xffffffffu));
    const float hi = rg_val(__reduce_max_sync(0xffffffffu, in && rank >= a.topk_group ? rg_key(v + ve) : 0u));
    if (safe && !(lo > hi)) keep = route_grouped_keep64(a, lr, reinterpret_cast<double*>(c), mx, lane);
    if ((size & 31) == 0) {                                                      // whole runs of 32 experts: the same group in all lanes
      int g = 0, left = size >> 5;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (!((keep >> (g & 31)) & 1u)) key[j] = 0u;
        if (--left == 0) { ++g; left = size >> 5; }
      }
    } else {
      const uint32_t mul = 0xffffffffu / (uint32_t)size + 1u;                    // e / size for e < 2^10
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const uint32_t e = lane + 32 * j;
        if (!((keep >> ((size == 1 ? e : __umulhi(e, mul)) & 31u)) & 1u)) key[j] = 0u;
      }
    }
  }
  // k picks and the best one left out, lane r the r-th
  uint32_t mykey = 0u; id = 0;
  uint32_t bound = 0u; int listed = 0;
  bool rounds = false;                                                           // picked one by one: what has been picked is out of key[]
  auto pick = [&](int r) -> uint32_t {
    uint32_t best = 0u; int at = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) if (key[j] > best) { best = key[j]; at = j; }
    const uint32_t m = __reduce_max_sync(0xffffffffu, best);
    const uint32_t e = __reduce_min_sync(0xffffffffu, best == m && m ? (uint32_t)(lane + 32 * at) : 0x7fffffffu);
    if (lane == r) { mykey = m; id = (int)e; }
    if ((e & 31u) == (uint32_t)lane && m) {
#pragma unroll
      for (int j = 0; j < R; ++j) if (j == (int)(e >> 5)) key[j] = 0u;
    }
    return m;
  };
  // The (k + 1)-th largest of the lanes' own largest is a bound that k + 1 experts reach; those that reach it are listed, a lane each, and count how many come
  // before them (as in router.cuh).  Lists longer than a warp, and fewer than k + 1 lanes with anything left: k + 1 rounds over all.
  {
    uint32_t best = 0u;
#pragma unroll
    for (int j = 0; j < R; ++j) best = max(best, key[j]);
#pragma unroll 1
    for (int r = 0; r <= a.k; ++r) { bound = __reduce_max_sync(0xffffffffu, best); if (best == bound) best = 0u; }
    int n = 0;
    __syncwarp();
    uint32_t* list = reinterpret_cast<uint32_t*>(c);
    if (bound > 0u) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const uint32_t b = __ballot_sync(0xffffffffu, key[j] >= bound);
        const int at = n + __popc(b & ((1u << lane) - 1u));
        if (key[j] >= bound && at < 32) { list[at] = key[j]; list[32 + at] = (uint32_t)(lane + 32 * j); }
        n += __popc(b);
      }
    }
    if (bound > 0u && n <= 32) {
      __syncwarp();
      const uint32_t ck = lane < n ? list[lane] : 0u, ci = list[32 + lane];
      int rank = 0;
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const uint32_t ok = __shfl_sync(0xffffffffu, ck, i), oi = __shfl_sync(0xffffffffu, ci, i);
        rank += ok > ck || (ok == ck && oi < ci);
      }
      __syncwarp();
      if (lane < n) { list[rank] = ck; list[32 + rank] = ci; }
      __syncwarp();
      if (lane < n) { mykey = list[lane]; id = (int)list[32 + lane]; }
      listed = n;
      __syncwarp();
    } else {
      rounds = true;
#pragma unroll 1
      for (int r = 0; r <= a.k; ++r) pick(r);
    }
  }
  auto inputs = [&](float& l, float& b) {                                        // of the lane's pick
    l = mykey ? __ldg(lr + id) : -INFINITY;
    if (!(l == l)) l = -INFINITY;
    b = mykey ? rg_bias(a, id) : 0.f;
  };
  float l, b;
  inputs(l, b);
  const float v = rg_val(mykey), vn = __shfl_down_sync(0xffffffffu, v, 1);
  const float ln = __shfl_down_sync(0xffffffffu, l, 1), bn = __shfl_down_sync(0xffffffffu, b, 1);
  const bool next = __shfl_down_sync(0xffffffffu, mykey, 1) != 0u;               // (there may be no expert left to be left out)
  const bool same = l == ln && b == bn;
  bool close = lane < a.k && next && !(v - vn > err(v) + err(vn)) && !same;
  if (__any_sync(0xffffffffu, lane == a.k - 1 && next && same)) {
    // A tie at the border settles nothing about those behind it: the last pick has to stand clear of the best one left out that is not its equal
    const uint32_t kk = __shfl_sync(0xffffffffu, mykey, a.k - 1);
    const float lk = __shfl_sync(0xffffffffu, l, a.k - 1), bk = __shfl_sync(0xffffffffu, b, a.k - 1);
    uint32_t rest = __reduce_max_sync(0xffffffffu, lane >= a.k && mykey && !(l == lk && b == bk) ? mykey : 0u);
    if (rest == 0u) {                                                            // (what is listed comes before all that is not)
#pragma unroll
      for (int j = 0; j < R; ++j) {
        uint32_t x = rounds || key[j] < bound ? key[j] : 0u;                     // neither picked nor listed
        if (x == kk) {
          const int e = lane + 32 * j;
          const float xl = fmaxf(__ldg(lr + e), -INFINITY);
          if (xl == lk && rg_bias(a, e) == bk) x = 0u;
        }
        rest = max(rest, x);
      }
      rest = __reduce_max_sync(0xffffffffu, rest);
    }
    const float vk = rg_val(kk), vr = rg_val(rest);
    close = close || (rest != 0u && !(vk - vr > err(vk) + err(vr)));
  }
  safe = safe && !__any_sync(0xffffffffu, lane < a.k && mykey == 0u);
  if (!safe) return false;
  if (__any_sync(0xffffffffu, close)) {
    // Neighbours too close for fp32: everyone that may belong among the picks, a lane each, put in order in 64 bits
    const float vk = __shfl_sync(0xffffffffu, v, a.k - 1), vb = rg_val(bound);
    int n = a.k + 1;
    if (!rounds && vk - vb > err(vk) + err(vb)) n = listed;                      // the list has them all
    else {
      if (!rounds) {
        mykey = 0u; id = 0;
        for (int r = 0; r <= a.k; ++r) pick(r);
      }
      for (bool more = true; more;) {
        const uint32_t kl = __shfl_sync(0xffffffffu, mykey, n - 1);
        if (kl == 0u) { --n; break; }
        if (vk - rg_val(kl) > err(vk) + err(rg_val(kl))) break;
        if (n == 32) return false;
        pick(n++);
      }
    }
    inputs(l, b);
    double d = 0.0;
    if (SIG) d = 1.0 / (1.0 + exp(-(double)l));
    else {
      d = exp((double)l - (double)mx);                                           // without a bias the sum changes no order
      if (a.bias) {
        double sum = 0.0;
        for (int e = lane; e < a.E; e += 32) { const float x = __ldg(lr + e); if (x == x) sum += exp((double)x - (double)mx); }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        d /= sum;
      }
    }
    d += (double)b;
    int rank = 0;
    for (int i = 0; i < n; ++i) { const double od = __shfl_sync(0xffffffffu, d, i); const int oi = __shfl_sync(0xffffffffu, id, i); rank += rg_before(od, oi, d, id); }
    __syncwarp();
    int* ids = reinterpret_cast<int*>(c);
    if (lane < n) { ids[rank] = id; ids[32 + rank] = (int)mykey; }
    __syncwarp();
    if (lane < a.k) { id = ids[lane]; mykey = (uint32_t)ids[32 + lane]; }
    __syncwarp();
    inputs(l, b);
  }
  float sc = 0.f;
  if (lane < a.k) sc = SIG ? __frcp_rn(1.f + expf(-l)) : expf(l - mx) * inv_sum;   // the picks' own, as exactly as fp32 has them
  if (__any_sync(0xffffffffu, lane < a.k && l > -INFINITY && sc < 0x1p-100f)) return false;   // a score near the end of fp32's range is itself not exact
  float tot = 0.f;
  for (int r = 0; r < a.k; ++r) tot += __shfl_sync(0xffffffffu, sc, r);
  w = (a.renorm ? __fdiv_rn(sc, tot + 1e-20f) : sc) * a.scale;
  return true;
}

template <int R, bool SIG>
__global__ void __launch_bounds__(RG_WARPS * 32, R <= 8 ? 12 : R <= 16 ? 8 : 6) route_grouped_kernel(const RouteGroupedArgs a) {
  extern __shared__ double rg_sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, m = blockIdx.x * RG_WARPS + warp;
  griddep_wait();
  griddep_launch();
  if (m >= a.M) return;
  double* c = rg_sm + (size_t)warp * max(a.E, 32);
  const float* lr = a.logits + (size_t)m * a.ld;
  int id; float w;
  if (!route_grouped_row32<R, SIG>(a, lr, reinterpret_cast<float*>(c), lane, id, w)) {
    __syncwarp();
    route_grouped_row64(a, lr, c, lane, id, w);
  }
  if (lane < a.k) { a.ids[(size_t)m * a.k + lane] = id; a.w[(size_t)m * a.k + lane] = w; }
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
  HB_REQUIRE(ctx, hb_aligned(logits, 4) && hb_aligned(bias, 4) && hb_aligned(ids, 4) && hb_aligned(w, 4), HB_ERR_INVALID, "route_grouped_topk: pointers must be aligned to their elements");
  RouteGroupedArgs a{logits, ld, M, E, k, n_group, topk_group, group_top, score == HB_SCORE_SIGMOID, renorm, bias, scale, ids, w};
  auto pick = [&](auto sig) {
    constexpr bool S = decltype(sig)::value;
    return E <= 128 ? route_grouped_kernel<4, S> : E <= 256 ? route_grouped_kernel<8, S> : E <= 512 ? route_grouped_kernel<16, S> : route_grouped_kernel<32, S>;
  };
  auto fn = a.sigmoid ? pick(std::true_type{}) : pick(std::false_type{});
  return hb_launch(ctx, "route_grouped", !(ctx->flags & HB_FLAG_NO_PDL), fn, dim3((M - 1) / RG_WARPS + 1), dim3(RG_WARPS * 32),
                   (size_t)RG_WARPS * (E > 32 ? E : 32) * 8, reinterpret_cast<cudaStream_t>(stream), a);
}
