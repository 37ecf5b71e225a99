// The product of 8-bit rows and 8-bit weights with a scale per block of 128, on the 5th-generation tensor cores: one kernel for the dense
// product, for the gate/up pass of routed experts (SwiGLU and the quantisation of its result in the epilogue) and for their down pass.
//
//   acc[n, m] += (ws[n / 128, b] · xs[b, m]) · Σ_{k in block b} w[n, k]·x[m, k]          for every block b of 128 values of K
//
// A block's sum is one accumulator tile of tcgen05.mma kind::f8f6f4 (e4m3 × e4m3: exact products, fp32 sums) in tensor memory; the scales are fp32
// numbers of any value, which no MMA applies, so the epilogue warps read every block's sums back and add them, scaled, to sums of their own in registers.
// The weights are the A operand (128 rows a tile, two tiles an item), the rows of x the B operand (N = up to BN of them): a lane of tensor memory is
// a weight row, a column a row of x, so a call with few rows wastes no tensor-core columns, and what a thread ends up with is one output column
// n for many rows m — in the gate/up pass gate and up of the same value.
//
// Work: items (tile of rows × 256 weight rows) of ceil(K / 128) steps.  The list is cut into equal runs of steps, one a CTA, without regard to where an item
// ends.  A CTA that holds part of an item leaves its sums in the workspace; the last
// one to arrive (a counter an item) adds all parts in the order of the CTAs — the same order in every run — and finishes the item.  So a product
// with one row of x keeps all SMs streaming weights to the end.  Nobody waits for anybody.  What bounds it: HBM (one row of 139264 x 5120: 112 us, 6.35 TB/s; 32
// rows 123) behind some 7 us of start, join and end (17408 x 5120: 20 us).
//
// Per CTA (persistent, one per SM, 12 warps): warp 8 (one thread) loads the operand tiles by TMA under the 128-byte swizzle, warp 9 (one thread) issues the
// MMAs, warp 10 multiplies the step's scales, warps 0-7 read the sums back (a warp reaches the 32 lanes of its number mod 4; warps 0-3 take the first half
// of the columns, 4-7 the second) and end the items.  Two accumulator buffers: one fills while the other is read.  Every wait is bounded.
#pragma once
#include <type_traits>

#include "device_error.h"
#include "fp8_common.cuh"
#include "hb_kernels.h"
#include "tc_common.cuh"

namespace hb {

enum { F8_PLAIN = 0, F8_GU = 1, F8_DOWN = 2, F8_DOWN32 = 3 };   // the down pass of a bf16 and of an fp32 result

constexpr int F8_COUNTERS = F8_MAX_CTAS;               // items that are cut, at most: a CTA's last one
constexpr int F8_THREADS = 12 * 32, F8_W_TMA = 8, F8_W_MMA = 9, F8_W_SCALE = 10;
// Plan of a short list of pairs (at most F8_PLAN_PAIRS), worked out by every CTA that needs it for itself: a pair's slot is the number of pairs with a smaller
// expert plus the number of earlier ones with its own: the same for every CTA, whatever the order its threads run in, without a launch of its own.
constexpr int F8_PLAN_PAIRS = 1024;
struct F8Plan { const int32_t* ids; int P, E, bm; const uint8_t* const* tab; };   // bm: pairs of a tile, at most
// ids with a record, the others NONE, to shared memory (room for P rounded up to four); the caller synchronises behind it
__device__ __forceinline__ void f8_plan_load(const F8Plan& a, int* e_s, int threads) {
  for (int p = threadIdx.x; p < (a.P + 3) / 4 * 4; p += threads) {
    const int e = p < a.P ? __ldg(a.ids + p) : -1;
    e_s[p] = e >= 0 && e < a.E && __ldg(reinterpret_cast<const unsigned long long*>(a.tab) + e) != 0ull ? e : 0x7fffffff;
  }
}
// The slot of pair p, -1 if it contributes nothing.
__device__ __forceinline__ int f8_plan_at(const F8Plan& a, const int* e_s, int p) {
  const int e = e_s[p];
  int n = 0;
#pragma unroll 4
  for (int i = 0; i < (a.P + 3) / 4; ++i) {
    const int4 v = reinterpret_cast<const int4*>(e_s)[i];
    n += (v.x < e) + (v.y < e) + (v.z < e) + (v.w < e);
    if (4 * i + 4 <= p) n += (v.x == e) + (v.y == e) + (v.z == e) + (v.w == e);
    else n += (v.x == e && 4 * i < p) + (v.y == e && 4 * i + 1 < p) + (v.z == e && 4 * i + 2 < p);
  }
  return e == 0x7fffffff ? -1 : n;
}
// The tile list; tmp: 16-byte aligned room of F8_PLAN_TMP bytes that may be written over.  A run of pairs is cut into tiles of equal size.  Returns the number of
// tiles; the caller synchronises before the list is read.  slots: where pair p's slot goes (or nullptr).
constexpr int F8_PLAN_TMP = F8_PLAN_PAIRS * 8 + HB_MAX_EXPERTS * 4 + 256;
__device__ __forceinline__ int f8_plan_tiles(const F8Plan& a, uint8_t* tmp, TileRef* tiles, int threads, int* slots = nullptr) {
  if (a.P <= 32) {                                     // a token or a few: one warp, a pair a lane (a kernel's code comes from afar the first time: the less, the sooner)
    uint32_t starts = 0u;
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      int e = lane < a.P ? __ldg(a.ids + lane) : -1;
      if (e < 0 || e >= a.E || __ldg(reinterpret_cast<const unsigned long long*>(a.tab) + e) == 0ull) e = 0x7fffffff;
      int less = 0;
#pragma unroll 4
      for (int i = 0; i < 32; ++i) less += __shfl_sync(0xffffffffu, e, i) < e;
      const uint32_t same = __match_any_sync(0xffffffffu, e), front = same & ((1u << lane) - 1u);
      const int rank = __popc(front), run = __popc(same), slot = less + rank, nt = (run + a.bm - 1) / a.bm, tper = (run + nt - 1) / nt;
      const bool on = e != 0x7fffffff, start = on && rank % tper == 0;
      starts = __reduce_or_sync(0xffffffffu, start ? 1u << slot : 0u);
      if (start) tiles[__popc(starts & ((1u << slot) - 1u))] = TileRef{slot, min(tper, run - rank), e};
      if (slots && lane < a.P) slots[lane] = on ? slot : -1;
      if (lane == 0) *reinterpret_cast<int*>(tmp) = __popc(starts);
    }
    __syncthreads();
    return *reinterpret_cast<const int*>(tmp);
  }
  // Ranks by one warp that goes through the list 32 pairs at a time, counting as it goes; then the experts' starts by a scan over the counts.  (Counting for every
  // pair over the whole list, as f8_plan_at does for a few, took 30 us of 640 pairs in every CTA.)
  int *e_s = reinterpret_cast<int*>(tmp), *rank_s = e_s + F8_PLAN_PAIRS, *cnt = rank_s + F8_PLAN_PAIRS, *tot = cnt + HB_MAX_EXPERTS;
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5, nw = threads >> 5;
  f8_plan_load(a, e_s, threads);
  for (int e = t; e < a.E; e += threads) cnt[e] = 0;
  __syncthreads();
  if (wp == 0) {
    for (int p0 = 0; p0 < a.P; p0 += 32) {
      const int e = p0 + lane < a.P ? e_s[p0 + lane] : 0x7fffffff;
      const uint32_t same = __match_any_sync(0xffffffffu, e), front = same & ((1u << lane) - 1u);
      const int base = e != 0x7fffffff ? cnt[e] : 0;
      __syncwarp();
      if (p0 + lane < a.P) rank_s[p0 + lane] = base + __popc(front);
      if (e != 0x7fffffff && front == 0u) cnt[e] = base + __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
  // thread t: experts [t·per, (t + 1)·per)
  const int per = (a.E + threads - 1) / threads, e0 = min(t * per, a.E), e1 = min(e0 + per, a.E);
  int c = 0, n = 0;
  for (int e = e0; e < e1; ++e) { c += cnt[e]; n += (cnt[e] + a.bm - 1) / a.bm; }
  int ic = c, in = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int uc = __shfl_up_sync(0xffffffffu, ic, o), un = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) { ic += uc; in += un; }
  }
  if (lane == 31) { tot[wp] = ic; tot[16 + wp] = in; }
  __syncthreads();
  int total = 0;
  for (int w = 0; w < nw; ++w) { if (w < wp) { ic += tot[w]; in += tot[16 + w]; } total += tot[16 + w]; }
  int run0 = ic - c, tile = in - n;
  for (int e = e0; e < e1; ++e) {
    const int run = cnt[e], nt = (run + a.bm - 1) / a.bm, tper = nt > 0 ? (run + nt - 1) / nt : 0;
    for (int i = 0; i < nt; ++i) tiles[tile++] = TileRef{run0 + i * tper, min(tper, run - i * tper), e};
    cnt[e] = run0;                                     // from here on the run's first slot
    run0 += run;
  }
  __syncthreads();
  if (slots) for (int p = t; p < a.P; p += threads) slots[p] = e_s[p] != 0x7fffffff ? cnt[e_s[p]] + rank_s[p] : -1;
  return total;
}

constexpr int F8_STG_PITCH = 80, F8_STG_BYTES = 32 * F8_STG_PITCH;   // a warp's staging: 32 rows of 64 bytes (pitch: 16-byte accesses without bank conflicts)
constexpr int F8_REGS = 168, F8_REGS_SUM = 216, F8_REGS_REST = 72;   // a thread's at launch (hbk_fp8_setup checks it), then of the sums' and of the other warps
static_assert(8 * F8_REGS_SUM + 4 * F8_REGS_REST <= 12 * F8_REGS, "register split");
constexpr int F8_A_BYTES = 128 * 128;                  // a tile of weights: 128 rows × 128 values

template <int BN_>
struct F8Cfg {
  static constexpr int BN = BN_, CW = BN / 2;          // rows of x a tile may have; columns of tensor memory an epilogue warp reads of each weight tile, at a time
  static constexpr int B_BYTES = BN * 128, STAGE = 2 * F8_A_BYTES + B_BYTES;
  static constexpr int ST = 200 * 1024 / STAGE;        // ring of operand stages
  static constexpr int TMEM = BN <= 16 ? 64 : 4 * BN;  // two buffers of two tiles
  static constexpr int SMEM = 1024 + ST * STAGE + 4 * 2 * BN * 4 + 8 * CW * 4 + 512 + F8_PLAN_PAIRS * (int)sizeof(TileRef);   // (the tile list: GU)
  static_assert(F8_COUNTERS <= kErrCounterWords, "counters of the context");
  static_assert(ST < 8 && SMEM <= 227 * 1024 && TMEM <= 512 && STAGE % 1024 == 0, "shared memory, tensor memory, swizzle atoms");
};

struct F8Args {
  const TileRef* tiles; const int* n_tiles;            // GU / DOWN / DOWN32: tiles of slots; PLAIN: ceil(M / per) tiles of `per` rows
  F8Plan plan;                                         // GU with plan.P > 0: the tiles are worked out here
  int M, per, N, K, n_nt;                              // n_nt: items a tile has (GU: N / 128 with N = I, else ceil(N / 256))
  int split;                                           // fp8_pair.cuh, tiles of single CTAs: CTAs of a cluster, 1, 2 or 4
  const float* ws; const uint8_t* const* tab; uint64_t off_w, off_s0, off_s1; int row2;   // PLAIN: scales; else records, offsets of the codes and of the two tiles' scales, rows from the first tile's matrix to the second's (GU)
  uint8_t* maps;                                       // GU / DOWN / DOWN32: room for F8_MAPS tensor maps a CTA
  const float* xs; int lds;                            // scales of the rows
  float limit;
  __nv_bfloat16* yb; float* yf; int ldy;               // PLAIN: one of them; DOWN: yb; DOWN32: yf
  uint8_t* yq; float* ys; int ldys;                    // GU: codes [slot, I], scales [I / 128][ldys]
  float* part; unsigned int* count;                    // sums of cut items [CTA][2][BN][256]; arrivals, by the CTA of an item's first step (zero before and after)
  uint32_t room;                                       // of part, in sums: range checks of the debug build
  uint32_t* err;
};

// Tensor maps of expert records, made by the thread that loads through them: a record's address is known on the device only, and the map of a matrix
// is one map for all experts but for its address.  A CTA's slots go round; one is written again when F8_MAPS maps, of at least one stage each, have gone by, more
// than there are stages: what was loaded through it has been multiplied.
constexpr int F8_MAPS = 8;
// A record has to lie at a 16-byte boundary.  One that does not is read from the boundary in front of it, where no load faults, and reported (0x400000).
__device__ __forceinline__ const uint8_t* f8_rec(const uint8_t* const* tab, int expert) {
  return reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(tab[expert]) & ~(uintptr_t)15);
}
struct F8Maps {
  uint8_t* slots; uint32_t n; int last; uint8_t* to;    // last: the expert that the newest map is of
  __device__ __forceinline__ const void* make(const CUtensorMap& tpl, const uint8_t* const* tab, int expert, uint64_t off, uint32_t* err) {
    if (expert == last) return to;                       // a CTA stays with an expert for some items; making a map takes as long as a few steps
    last = expert;
    const uint8_t* addr = f8_rec(tab, expert) + off;
    if (reinterpret_cast<uintptr_t>(tab[expert]) & 15u) atomicOr(err, 0x400000u);
    to = slots + (size_t)(n++ % F8_MAPS) * sizeof(CUtensorMap);
    const uint4* from = reinterpret_cast<const uint4*>(&tpl);
#pragma unroll
    for (int j = 0; j < 8; ++j) reinterpret_cast<uint4*>(to)[j] = from[j];
    asm volatile("tensormap.replace.tile.global_address.global.b1024.b64 [%0], %1;" ::"l"(to), "l"(addr) : "memory");
    asm volatile("fence.proxy.tensormap::generic.release.gpu;" ::: "memory");
    tmap_acquire(to);
    return to;
  }
};

__device__ __forceinline__ void tma_prefetch_2d(const void* tmap, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(tmap), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// a += d·s, two values at a time
__device__ __forceinline__ void f8_fma2(float& a0, float& a1, uint32_t d0, uint32_t d1, float s0, float s1) {
  asm("{\n .reg .b64 a, d, s;\n mov.b64 a, {%0, %1};\n mov.b64 d, {%2, %3};\n mov.b64 s, {%4, %5};\n fma.rn.f32x2 a, d, s, a;\n mov.b64 {%0, %1}, a;\n}"
      : "+f"(a0), "+f"(a1) : "r"(d0), "r"(d1), "f"(s0), "f"(s1));
}
__device__ __forceinline__ float f8_swiglu(float g, float u, float limit) {
  if (limit > 0.f) { g = g > limit ? limit : g; u = u > limit ? limit : u < -limit ? -limit : u; }   // (NaN stays)
  return __fdividef(g, 1.f + expf(-g)) * u;                                    // (two steps; y is rounded to three bits next)
}
__device__ __forceinline__ uint4 f8_pack8(const float* v) {                     // eight values as bf16
  uint32_t p[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) { const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]); p[j] = *reinterpret_cast<const uint32_t*>(&b); }
  return make_uint4(p[0], p[1], p[2], p[3]);
}
// A warp's staged 32 rows × 64 bytes to memory, eight rows an instruction (a lane has a row: its own stores would touch 32 rows each).  to: the first
// row's place; bytes: how much of the 64 there is room for.
__device__ __forceinline__ void f8_flush(const uint8_t* stg, uint8_t* to, size_t ld, int rows, int bytes, int lane) {
  __syncwarp();
  const int c = (lane & 3) * 16;
  const uint32_t al = (uint32_t)(reinterpret_cast<uintptr_t>(to) | ld) & 15u;   // what all rows' places are aligned to: 0: 16 bytes
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 2);
    const uint4 v = *reinterpret_cast<const uint4*>(stg + r * F8_STG_PITCH + c);
    if (r >= rows) continue;
    uint8_t* p = to + (size_t)r * ld + c;
    if (al == 0 && c + 16 <= bytes) *reinterpret_cast<uint4*>(p) = v;
    else if ((al & 7u) == 0 && c + 16 <= bytes) {
      *reinterpret_cast<uint2*>(p) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(p + 8) = make_uint2(v.z, v.w);
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if ((al & 3u) == 0 && c + 4 * j + 4 <= bytes) *reinterpret_cast<uint32_t*>(p + 4 * j) = w[j];
        else {                                                                 // (a row of fp32 has room for whole words)
          if (c + 4 * j < bytes) *reinterpret_cast<uint16_t*>(p + 4 * j) = (uint16_t)(w[j] & 0xffffu);
          if (c + 4 * j + 2 < bytes) *reinterpret_cast<uint16_t*>(p + 4 * j + 2) = (uint16_t)(w[j] >> 16);
        }
      }
    }
  }
  __syncwarp();
}
template <int W>
__device__ __forceinline__ void f8_add(float* acc, const uint32_t (&d)[W], const float* s) {
#pragma unroll
  for (int c = 0; c < W; c += 4) {
    const float4 v = *reinterpret_cast<const float4*>(s + c);
    f8_fma2(acc[c], acc[c + 1], d[c], d[c + 1], v.x, v.y);
    f8_fma2(acc[c + 2], acc[c + 3], d[c + 2], d[c + 3], v.z, v.w);
  }
}
template <int W>
__device__ __forceinline__ void f8_add(float* acc, const uint32_t (&d)[W], float s) {
#pragma unroll
  for (int c = 0; c < W; c += 2) f8_fma2(acc[c], acc[c + 1], d[c], d[c + 1], s, s);
}
// The columns asked for before have arrived; the registers are named so that nothing that reads them is moved in front of it.
template <int W>
__device__ __forceinline__ void f8_landed(uint32_t (&r)[W], uint32_t (&p)[W]) {
  tc_wait_ld();
#pragma unroll
  for (int i = 0; i < W; i += 8) {
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
    asm volatile("" : "+r"(p[i]), "+r"(p[i + 1]), "+r"(p[i + 2]), "+r"(p[i + 3]), "+r"(p[i + 4]), "+r"(p[i + 5]), "+r"(p[i + 6]), "+r"(p[i + 7]));
  }
}
template <int W>
__device__ __forceinline__ void f8_ld(uint32_t taddr, uint32_t (&r)[W]) {
  if constexpr (W == 16) tc_ld16(taddr, r);
  else tc_ld8(taddr, r);
}

// Registers: with 16 rows a tile 128 a thread are enough and leave room on the SM for a block of the small kernel behind this one, which then starts without waiting
// for it to leave (16 rows over 512 experts: 106 us with 168, 103.5; one row of 5120 x 17408 behind its quantiser 26 and 25; with 32 rows a tile they spill, 24.4 and 27.6).
template <int BN, int MODE>
__global__ void __launch_bounds__(BN <= 16 ? 512 : F8_THREADS, 1) fp8_gemm_kernel(const __grid_constant__ F8Args a, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX) {
  using C = F8Cfg<BN>;
  extern __shared__ uint8_t f8_raw[];
  const uint32_t raw = smem_u32(f8_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* sm = f8_raw + (base - raw);
  // Scales of a step [step mod 4][2 tiles][BN]: a warp may still read those of a step whose sums it has taken out, while the next two's are written
  float* scl = reinterpret_cast<float*>(sm + C::ST * C::STAGE);
  uint32_t* amx = reinterpret_cast<uint32_t*>(scl + 8 * BN);                 // magnitudes of y: [2 halves][4 warps][CW]
  uint64_t* full = reinterpret_cast<uint64_t*>(amx + 8 * C::CW);             // [ST] the stage's operands have landed
  uint64_t* empty = full + C::ST;                                            // [ST] the MMAs that read them are done
  uint64_t* acc_full = empty + C::ST;                                        // [2] the buffer's sums and scales are there
  uint64_t* acc_empty = acc_full + 2;                                        // [2] the epilogue has read them
  uint64_t* mma_done = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile uint32_t* last = tmem_slot + 1;
  TileRef* tile_s = reinterpret_cast<TileRef*>(tmem_slot + 4);
  const int warp = warp_uniform(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::ST; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 2); mbar_init(&acc_empty[s], 8); }
    mbar_init(mma_done, 1);
    mbar_fence_init();
  }
  if (warp == F8_W_MMA) { tmem_alloc(tmem_slot, C::TMEM); tmem_relinquish(); }
  // What comes before griddep_wait runs beside the end of the kernel in front.  Routed: that one is this library's, and all that was there before it (routing,
  // table, records, for long lists and for the down pass the tiles) is complete, as it announced itself after its own wait; the tiles are found and the first
  // stages' weights loaded here.  Dense: the kernel in front is anybody's, and only sends weights on their way to L2.
  const bool own_plan = MODE == F8_GU && a.plan.P > 0;
  int n_tiles = 0;
  if (own_plan) {
    n_tiles = f8_plan_tiles(a.plan, sm, tile_s, F8_THREADS);
    fence_proxy_async_smem();                                                  // its scratch becomes operand stages
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int KB = f8_blocks(a.K);
  if (!own_plan) n_tiles = MODE == F8_PLAIN ? (a.M + a.per - 1) / a.per : *a.n_tiles;
  F8Sched sch;
  sch.init((uint32_t)n_tiles * a.n_nt, KB, gridDim.x, blockIdx.x, true, 0u);
  auto tile_of = [&](int ti) -> TileRef {
    if (own_plan) return tile_s[ti];
    if (MODE != F8_PLAIN) return a.tiles[ti];
    return TileRef{ti * a.per, min(a.per, a.M - ti * a.per), 0};
  };
  int item, kb0, kb1;

  if (warp >= 8) {
  if (warp == F8_W_TMA) {
    // ------------------------------------------------------------------------------------------------ operand tiles, one thread
    if (elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true, waited = false;
      F8Maps maps{a.maps + (size_t)blockIdx.x * F8_MAPS * sizeof(CUtensorMap), 0u, -1, nullptr};
      while (ok && sch.next(item, kb0, kb1)) {
        const int ti = item / a.n_nt, nt = item - ti * a.n_nt;
        const TileRef tl = tile_of(ti);
        const void* mw = MODE == F8_PLAIN ? &tmW : maps.make(tmW, a.tab, tl.expert, a.off_w, a.err);
        const int r0 = MODE == F8_GU ? nt * 128 : nt * 256, r1 = MODE == F8_GU ? r0 + a.row2 : r0 + 128;   // rows past the last read as zero codes
        auto weights = [&](uint32_t st, int kb) {
          mbar_expect_tx(&full[st], C::STAGE);
          tma_load_2d(base + st * C::STAGE, mw, kb * 128, r0, &full[st]);
          tma_load_2d(base + st * C::STAGE + F8_A_BYTES, mw, kb * 128, r1, &full[st]);
        };
        auto rows = [&](uint32_t st, int kb) { tma_load_2d(base + st * C::STAGE + 2 * F8_A_BYTES, &tmX, kb * 128, tl.slot0, &full[st]); };
        int kb = kb0;
        if (!waited) {
          const int n = min(kb1 - kb0, C::ST);
          for (int i = 0; i < n; ++i) {
            if (MODE != F8_PLAIN) weights(i, kb0 + i);
            else { tma_prefetch_2d(&tmW, (kb0 + i) * 128, r0); tma_prefetch_2d(&tmW, (kb0 + i) * 128, r1); }
          }
          griddep_wait();
          waited = true;
          if (MODE != F8_PLAIN) {
            for (int i = 0; i < n; ++i) rows(i, kb0 + i);
            kb += n;
            s = n == C::ST ? 0 : n; ph = n == C::ST ? 0 : 1;
          }
        }
        for (; kb < kb1; ++kb) {
          if (!(ok = mbar_wait(&empty[s], ph, a.err, kErrFp8Stage))) break;
          weights(s, kb);
          rows(s, kb);
          if (++s == C::ST) { s = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp == F8_W_MMA) {
    // ------------------------------------------------------------------------------------------------ MMA issue, one thread
    if (elect_one()) {
      uint32_t s = 0, ph = 0, it = 0;
      bool ok = true;
      while (ok && sch.next(item, kb0, kb1)) {
        const int rows = tile_of(item / a.n_nt).rows;
        // kind::f8f6f4: D fp32 (bit 4), A and B e4m3 (format 0 at bits 7 and 10), both K-major, N / 8 at bit 17, M / 16 at bit 24
        const uint32_t idesc = (1u << 4) | ((uint32_t)((rows + 15) >> 4) << 18) | ((128u >> 4) << 24);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t buf = it & 1u;
          if (!(ok = mbar_wait(&acc_empty[buf], ((it >> 1) & 1u) ^ 1u, a.err, kErrFp8AccFree))) break;
          if (!(ok = mbar_wait(&full[s], ph, a.err, kErrFp8Loads))) break;
          tc_fence_after();
          const uint32_t sb = base + s * C::STAGE, d = tmem + buf * (2 * BN);
          const uint64_t ad = tc_desc_sw128(sb), bd = tc_desc_sw128(sb + 2 * F8_A_BYTES);
#pragma unroll
          for (uint32_t u = 0; u < 2; ++u)
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)                                 // 32 values further along the swizzled rows
              tc_mma_f8(d + u * BN, ad + u * (F8_A_BYTES >> 4) + 2 * j, bd + 2 * j, idesc, j);
          tc_commit(&empty[s]);
          tc_commit(&acc_full[buf]);
          if (++s == C::ST) { s = 0; ph ^= 1u; }
        }
      }
      tc_commit(mma_done);                                                     // nothing is in flight when tensor memory is freed
      mbar_wait(mma_done, 0, a.err, kErrFp8Mma);
    }
  } else if (warp == F8_W_SCALE) {
    // ------------------------------------------------------------------------------------------------ scales of a step: weight block × row, a step ahead
    constexpr int NL = (BN + 31) / 32;
    griddep_wait();
    uint32_t it = 0;
    bool ok = true;
    while (ok && sch.next(item, kb0, kb1)) {
      const int ti = item / a.n_nt, nt = item - ti * a.n_nt;
      const TileRef tl = tile_of(ti);
      const float *w0, *w1;
      if (MODE == F8_PLAIN) { w0 = a.ws + (size_t)(2 * nt) * KB; w1 = nt * 256 + 128 < a.N ? w0 + KB : w0; }
      else {
        const uint8_t* rec = f8_rec(a.tab, tl.expert);
        const int b0 = MODE == F8_GU ? nt : 2 * nt, b1 = MODE == F8_GU ? nt : nt * 256 + 128 < a.N ? b0 + 1 : b0;
        w0 = reinterpret_cast<const float*>(rec + a.off_s0) + (size_t)b0 * KB;
        w1 = reinterpret_cast<const float*>(rec + a.off_s1) + (size_t)b1 * KB;
      }
      float nx[NL], n0, n1;
      auto fetch = [&](int kb) {
        n0 = __ldg(w0 + kb); n1 = __ldg(w1 + kb);
#pragma unroll
        for (int i = 0; i < NL; ++i) nx[i] = lane + 32 * i < tl.rows ? __ldcg(a.xs + (size_t)kb * a.lds + tl.slot0 + lane + 32 * i) : 0.f;
      };
      fetch(kb0);
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t buf = it & 1u;
        float x[NL]; const float s0 = n0, s1 = n1;
#pragma unroll
        for (int i = 0; i < NL; ++i) x[i] = nx[i];
        if (kb + 1 < kb1) fetch(kb + 1);
        ok = mbar_wait(&acc_empty[buf], ((it >> 1) & 1u) ^ 1u, a.err, kErrFp8ScaleFree);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        float* d = scl + (it & 3u) * (2 * BN);
#pragma unroll
        for (int i = 0; i < NL; ++i)
          if (BN >= 32 || lane < BN) { d[lane + 32 * i] = x[i] * s0; d[BN + lane + 32 * i] = x[i] * s1; }
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_full[buf]);
      }
    }
  }
  } else {
    griddep_wait();
    griddep_launch();
    // ------------------------------------------------------------------------------------------------ sums: warp (h, q) has lanes [32 q, 32 q + 32) and of each weight
    // tile's columns [h·CW, (h + 1)·CW): a lane is a weight row, a column a row of x with a scale of its own, read from shared memory by all lanes together
    const int h = warp >> 2, q = warp & 3, row = 32 * q + lane;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16) + h * C::CW;
    uint32_t it = 0;
    bool ok = true;
    while (sch.next(item, kb0, kb1)) {                                          // after a wait that gave up: on to the end without waits and results, but through every barrier
      const int ti = item / a.n_nt, nt = item - ti * a.n_nt;
      const TileRef tl = tile_of(ti);
      const int cols = min(max(tl.rows - h * C::CW, 0), C::CW);                // this warp's columns that hold rows of x
      const bool active = cols > 0;
      float acc[2][C::CW];
#pragma unroll
      for (int c = 0; c < C::CW; ++c) acc[0][c] = acc[1][c] = 0.f;
      // A wait for reads waits for all that are under way, so two go out together (one weight tile each), each as soon as the registers it writes have been
      // added up (one at a time, each behind the other's additions: 730 clocks a step of 256 columns)
      uint32_t ra[C::CW], rb[C::CW];
      auto arrived = [&](uint32_t n) {
        const bool o = mbar_wait(&acc_full[n & 1u], (n >> 1) & 1u, a.err, kErrFp8Acc);
        tc_fence_after();
        return (bool)__all_sync(0xffffffffu, o);
      };
      if ((ok = ok && arrived(it)) && active) { f8_ld<C::CW>(trow + (it & 1u) * (2 * BN), ra); f8_ld<C::CW>(trow + (it & 1u) * (2 * BN) + BN, rb); }
      for (int kb = kb0; kb < kb1 && ok; ++kb, ++it) {
        const uint32_t buf = it & 1u, nb = trow + (buf ^ 1u) * (2 * BN);
        const float* sb = scl + (it & 3u) * (2 * BN) + h * C::CW;
        if (active) {
          f8_landed<C::CW>(ra, rb);
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);                           // the buffer's sums are in registers
        if (active) f8_add<C::CW>(acc[0], ra, sb);
        const bool more = kb + 1 < kb1 && (ok = arrived(it + 1)) && active;
        if (more) f8_ld<C::CW>(nb, ra);
        if (active) f8_add<C::CW>(acc[1], rb, sb + BN);
        if (more) f8_ld<C::CW>(nb + BN, rb);
      }
      // ---- an item that other CTAs have parts of: leave the sums, the last one to arrive goes on with everybody's
      if (kb1 - kb0 < KB) {
        const uint32_t s0 = (uint32_t)item * (uint32_t)KB, c_first = sch.owner(s0), c_last = sch.owner(s0 + KB - 1);
        // a part: [column][tile][lane]; a CTA's first run is its part 0
        auto part_of = [&](uint32_t c, uint32_t st) { return a.part + ((size_t)c * 2 + (c == c_first && st != s0 ? 1 : 0)) * (256 * BN) + (size_t)h * C::CW * 256 + row; };
        float* mine = part_of(blockIdx.x, sch.start(blockIdx.x));
#pragma unroll
        for (int c = 0; c < C::CW; ++c)
          if (active && c < cols && HB_BOUND(a.err, (size_t)(mine - a.part) + c * 256 + 128 < a.room, 0x801u, mine - a.part)) {
            __stcg(mine + c * 256, acc[0][c]); __stcg(mine + c * 256 + 128, acc[1][c]);
          }
        named_bar_sync(1, 256);
        if (threadIdx.x == 0 && !ok) *last = 0u;
        else if (threadIdx.x == 0) {
          __threadfence();                                                     // everybody's sums are out before this CTA is counted
          const bool all = atomicAdd(a.count + c_first, 1u) == c_last - c_first;
          if (all) a.count[c_first] = 0u;                                         // zero again for the next launch
          __threadfence();
          *last = all;
        }
        named_bar_sync(1, 256);
        const bool mine_to_end = *last != 0u;
        named_bar_sync(1, 256);                                                // the flag has been read: the next item may write it
        if (!mine_to_end) continue;
#pragma unroll
        for (int c = 0; c < C::CW; ++c) acc[0][c] = acc[1][c] = 0.f;
        // parts and columns fetched together; a value's parts are added in order
        constexpr int NP = C::CW <= 8 ? 8 : 2, GC = C::CW <= 8 ? 4 : C::CW;
        const float* first = part_of(c_first, sch.start(c_first));
        const float* rest = part_of(c_first, s0);                              // the later CTAs' parts are their first ones: 2 · 256 · BN apart
        for (uint32_t cc = c_first; cc <= c_last; cc += NP) {
#pragma unroll
          for (int g = 0; g < C::CW; g += GC) {
            if (g >= cols) break;
            float t[NP][2][GC];
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              const float* p = cc + i == c_first ? first : rest + (size_t)(cc + i - c_first) * (2 * 256 * BN);
#pragma unroll
              for (int c = 0; c < GC; ++c) {
                const bool on = g + c < cols && cc + i <= c_last;
                t[i][0][c] = on ? __ldcg(p + (g + c) * 256) : 0.f; t[i][1][c] = on ? __ldcg(p + (g + c) * 256 + 128) : 0.f;
              }
            }
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
              for (int c = 0; c < GC; ++c) { acc[0][g + c] += t[i][0][c]; acc[1][g + c] += t[i][1][c]; }
          }
        }
      }
      // ---- the item's results
      if constexpr (MODE == F8_GU) {
        uint32_t* am = amx + (h * 4) * C::CW;
#pragma unroll
        for (int c = 0; c < C::CW; ++c) {
          if (c < cols) {
            acc[0][c] = f8_swiglu(acc[0][c], acc[1][c], a.limit);
            const uint32_t mx = __reduce_max_sync(0xffffffffu, f8_mag(acc[0][c]));
            if (lane == 0) am[q * C::CW + c] = mx;
          }
        }
        named_bar_sync(2 + h, 128);
#pragma unroll
        for (int c = 0; c < C::CW; ++c) {
          if (c < cols && ok) {
            F8Block blk;
            const float sc = blk.init(max(max(am[c], am[C::CW + c]), max(am[2 * C::CW + c], am[3 * C::CW + c])));
            const int slot = tl.slot0 + h * C::CW + c;
            a.yq[(size_t)slot * a.N + nt * 128 + row] = (uint8_t)blk.pair(acc[0][c], 0.f);
            if (row == 0) a.ys[(size_t)nt * a.ldys + slot] = sc;
          }
        }
        named_bar_sync(2 + h, 128);                                            // the magnitudes have been read
      } else {
        auto store = [&](auto* y, auto value) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int n = nt * 256 + u * 128 + row;
            if (n < a.N && ok) {
#pragma unroll
              for (int c = 0; c < C::CW; ++c)
                if (c < cols) y[(size_t)(tl.slot0 + h * C::CW + c) * a.ldy + n] = value(acc[u][c]);
            }
          }
        };
        if (MODE == F8_DOWN || (MODE == F8_PLAIN && a.yb)) store(a.yb, [](float v) { return __float2bfloat16(v); });
        else store(a.yf, [](float v) { return v; });
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == F8_W_MMA) { tc_fence_after(); tmem_dealloc(tmem, C::TMEM); }
}

}  // namespace hb
