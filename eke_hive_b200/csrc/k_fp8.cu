// 8-bit floats with a scale per block of 128: the quantisers of activations and weights, the product, the routed experts.
#include "fp8_pair.cuh"
#include "hb_kernels.h"

namespace hb {

// Rows: 16 lanes take a block of 128 values, 8 each.  Without destinations row m becomes row m of q / s.  With them (a routed layer's rows are quantised once
// and written into expert order) row m goes to the slots of its nd pairs, those that have one.
struct F8RowsArgs {
  const __nv_bfloat16* x; int ldx, M, K;
  const int* dest; int nd;                             // [M, nd], negative: none; nd == 0: no destinations
  uint8_t* q; int ldq; float* s; int lds;
};
// Block b of row m by LN lanes, 128 / LN values each; slot: of lane l < nd's pair, or -1.
template <int LN>
__device__ __forceinline__ void f8_quant_unit(const F8RowsArgs& a, int m, int b, int slot) {
  constexpr int V = F8_B / LN;
  const int l = threadIdx.x & (LN - 1), k = b * F8_B + l * V, sh = threadIdx.x & (32 - LN);
  const uint32_t group = (uint32_t)((1ull << LN) - 1ull) << sh;
  float v[V];
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = 0.f;
  if (k < a.K) {                                                               // K is a multiple of 16: a lane's values are inside or outside together
    const __nv_bfloat16* p = a.x + (size_t)m * a.ldx + k;
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < V / 8; ++i) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(p) + i);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[8 * i + 2 * j] = __uint_as_float(ww[j] << 16); v[8 * i + 2 * j + 1] = __uint_as_float(ww[j] & 0xffff0000u); }
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = __bfloat162float(p[j]);
    }
  }
  uint32_t mx = 0u;
#pragma unroll
  for (int j = 0; j < V; ++j) mx = max(mx, f8_mag(v[j]));
#pragma unroll
  for (int o = LN / 2; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(group, mx, o));
  F8Block blk;
  const float sc = blk.init(mx);
  uint32_t c[V / 4];
#pragma unroll
  for (int j = 0; j < V / 4; ++j) c[j] = blk.pair(v[4 * j], v[4 * j + 1]) | blk.pair(v[4 * j + 2], v[4 * j + 3]) << 16;
  auto put = [&](int to) {
    if (k >= a.K) return;
    uint8_t* d = a.q + (size_t)to * a.ldq + k;
    if constexpr (V == 8) *reinterpret_cast<uint2*>(d) = make_uint2(c[0], c[1]);
    else *reinterpret_cast<uint4*>(d) = make_uint4(c[0], c[1], c[2], c[3]);
  };
  if (a.nd == 0) {
    put(m);
    if (l == 0) a.s[(size_t)b * a.lds + m] = sc;
    return;
  }
  if (slot >= 0) a.s[(size_t)b * a.lds + slot] = sc;
  for (uint32_t on = (__ballot_sync(group, slot >= 0) >> sh) & (uint32_t)((1ull << LN) - 1ull); on; on &= on - 1u) put(__shfl_sync(group, slot, (__ffs(on) - 1) + sh));
}
// Eight lanes a block: what a lane does once for a block (the reciprocal, the scale) is some 40 instructions beside five a value, and their number is what
// bounds the kernel (4096 rows of 5120: 28 us with sixteen lanes a block and nine instructions a value, 24 with eight; two blocks a lane at a time need registers that
// halve the warps: 27).
__global__ void __launch_bounds__(256) fp8_quant_rows_kernel(const F8RowsArgs a) {
  griddep_wait();
  griddep_launch();
  const int nb = f8_blocks(a.K), l = threadIdx.x & 7;
  const uint32_t group = 0xffu << (threadIdx.x & 24);
  const long long total = (long long)a.M * nb;
  for (long long i = (long long)blockIdx.x * 32 + (threadIdx.x >> 3); i < total; i += (long long)gridDim.x * 32) {
    const int m = (int)(i / nb), b = (int)(i - (long long)m * nb);
    if (a.nd == 0) { f8_quant_unit<8>(a, m, b, -1); continue; }
    for (int d = 0; d < a.nd; d += 8) {                                        // (more than eight destinations: once more)
      const int slot = d + l < a.nd ? __ldg(a.dest + (size_t)m * a.nd + d + l) : -1;
      if (__any_sync(group, slot >= 0)) f8_quant_unit<8>(a, m, b, slot);       // a row nobody here wants is not read
    }
  }
}

// The front of a routed layer's call with a short list of pairs, in one launch: CTA 0 writes the plan down (the slots for the sum at the end, the tiles for the down
// pass; the gate/up pass finds them for itself), the others work out the slots of their rows and quantise.  (A plan kernel and the quantiser behind it took 19 of a
// one-row call's 75 us.)
struct F8PrepArgs { F8RowsArgs rows; F8Plan plan; int* pos_of; TileRef* tiles; int* n_tiles; };
__global__ void __launch_bounds__(256) fp8_prep_kernel(const F8PrepArgs a) {
  __shared__ __align__(16) uint8_t tmp[F8_PLAN_TMP];
  __shared__ int slots[512];
  const int t = threadIdx.x;
  griddep_wait();
  griddep_launch();
  if (blockIdx.x == 0) {
    const int n = f8_plan_tiles(a.plan, tmp, a.tiles, 256, a.pos_of);
    if (t == 0) *a.n_tiles = n;
    return;
  }
  // 16 blocks of 128 values a CTA
  int* e_s = reinterpret_cast<int*>(tmp);
  f8_plan_load(a.plan, e_s, 256);
  __syncthreads();
  const int nb = f8_blocks(a.rows.K), u0 = (blockIdx.x - 1) * 16, total = a.rows.M * nb, nd = a.rows.nd;
  const int m0 = u0 / nb, m1 = min(u0 + 15, total - 1) / nb;
  for (int i = t; i < (m1 - m0 + 1) * nd; i += 256) slots[i] = f8_plan_at(a.plan, e_s, m0 * nd + i);
  __syncthreads();
  const int u = u0 + (t >> 4), l16 = t & 15;
  if (u < total) {
    const int m = u / nb;
    for (int d = 0; d < nd; d += 16) {
      const int slot = d + l16 < nd ? slots[(m - m0) * nd + d + l16] : -1;
      if (__any_sync(0xffffu << (t & 16), slot >= 0)) f8_quant_unit<16>(a.rows, m, u - m * nb, slot);
    }
  }
}

// Weights: a CTA takes a block of 128 × 128, sixteen lanes a row of it, eight rows a thread: the block stays in registers between its largest magnitude and its
// codes, so memory is read once (17408 x 5120 fp32: 69-71 us, 6.3-6.5 TB/s).
template <class T>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const T* __restrict__ w, int N, int K, uint8_t* __restrict__ q, float* __restrict__ s) {
  __shared__ uint32_t red[8];
  const int nb = f8_blocks(K), bn = blockIdx.x / nb, bk = blockIdx.x - bn * nb;
  const int k = bk * F8_B + (threadIdx.x & 15) * 8, n0 = bn * F8_B + (threadIdx.x >> 4);
  float v[8][8];
  uint32_t mx = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + 16 * i;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    if (n < N && k < K) {
      const T* p = w + (size_t)n * K + k;
      if constexpr (sizeof(T) == 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p)), y = __ldg(reinterpret_cast<const float4*>(p) + 1);
        v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w; v[i][4] = y.x; v[i][5] = y.y; v[i][6] = y.z; v[i][7] = y.w;
      } else {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t xx[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[i][2 * j] = __uint_as_float(xx[j] << 16); v[i][2 * j + 1] = __uint_as_float(xx[j] & 0xffff0000u); }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = max(mx, f8_mag(v[i][j]));
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) mx = max(mx, red[i]);
  F8Block blk;
  const float sc = blk.init(mx);
  if (threadIdx.x == 0) s[blockIdx.x] = sc;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + 16 * i;
    if (n < N && k < K)
      *reinterpret_cast<uint2*>(q + (size_t)n * K + k) = make_uint2(blk.pair(v[i][0], v[i][1]) | blk.pair(v[i][2], v[i][3]) << 16, blk.pair(v[i][4], v[i][5]) | blk.pair(v[i][6], v[i][7]) << 16);
  }
}

// ---- the sum over a row's pairs: out[m] = Σ_k w[m,k]·part[slot of (m,k)], k in order (+ gate·shared[m]) ----------------------------------
// A warp takes 512 columns of a row (fp32 parts: 256), a lane twice 16 bytes of every pair's part.  Lane k looks up pair k; only pairs that have a slot are gone
// through, four parts fetched at a time: 8192 rows of 7168 with a bf16 pair each and shared rows 75 us, 4.7 TB/s (two at a time and more warps: 69, but ten pairs a
// row of 2048, 16 rows: 10.7 us instead of 9).  T, what the parts are held in: fp32 for an fp32 result; for one that is rounded to bf16 in the end bf16, which is off by 2^-8
// of a pair's own share at most and half the bytes (8192 rows of 7168 with a pair each: a whole layer of 32 held experts of 256 takes 677 us, with fp32 parts 734; of 1000
// rows of 4096 with eight pairs each 586, 620).
constexpr int F8_SUM_THREADS = 128;
template <class T>
struct F8SumArgs {
  const T* part; const int* pos_of; const float* w; int M, K, H; float* out;
  const __nv_bfloat16* shared; const float* lg; int ld, col; __nv_bfloat16* cout;
};
template <class T>
constexpr int F8_SUM_COLS = 2 * 32 * (16 / (int)sizeof(T));
template <class T>
__global__ void __launch_bounds__(F8_SUM_THREADS) fp8_sum_kernel(const F8SumArgs<T> a) {
  constexpr int WARPS = F8_SUM_THREADS / 32, V = 16 / (int)sizeof(T), COLS = F8_SUM_COLS<T>, HALF = COLS / 2;
  bool waited = false;                                                         // only the parts are of the kernel in front
  const int chunks = (a.H + COLS - 1) / COLS, lane = threadIdx.x & 31;
  const long long total = (long long)a.M * chunks;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (long long i = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); i < total; i += (long long)gridDim.x * WARPS) {
    const int m = (int)(i / chunks), n = (int)(i - (long long)m * chunks) * COLS + lane * V;
    const bool in[2] = {n < a.H, n + HALF < a.H};                              // H is a multiple of 128
    const size_t o = (size_t)m * a.H + n;
    const int slot = lane < a.K ? __ldg(a.pos_of + (size_t)m * a.K + lane) : -1;
    const float wk = lane < a.K ? __ldg(a.w + (size_t)m * a.K + lane) : 0.f;
    uint4 sv[2] = {zero, zero};
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) if (a.shared && in[h]) sv[h] = __ldg(reinterpret_cast<const uint4*>(a.shared + o + HALF * h));
    }
    const float gate = a.lg ? 1.f / (1.f + expf(-__ldg(a.lg + (size_t)m * a.ld + a.col))) : 1.f;
    if (!waited) { griddep_wait(); waited = true; }
    float acc[2][V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[0][j] = acc[1][j] = 0.f;
    auto add = [&](float (&to)[V], const uint4& v, float f) {
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) to[j] = fmaf(f, __uint_as_float(u[j]), to[j]);
        else { to[2 * j] = fmaf(f, __uint_as_float(u[j] << 16), to[2 * j]); to[2 * j + 1] = fmaf(f, __uint_as_float(u[j] & 0xffff0000u), to[2 * j + 1]); }
      }
    };
    for (uint32_t on = __ballot_sync(0xffffffffu, slot >= 0); on;) {
      uint4 v[4][2]; float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = on ? __ffs(on) - 1 : 0;
        const T* p = a.part + (size_t)__shfl_sync(0xffffffffu, slot, k) * a.H + n;
        f[j] = on ? __shfl_sync(0xffffffffu, wk, k) : 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) v[j][h] = on && in[h] ? __ldcs(reinterpret_cast<const uint4*>(p + HALF * h)) : zero;
        on &= on - 1u;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) { add(acc[0], v[j][0], f[j]); add(acc[1], v[j][1], f[j]); }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!in[h]) continue;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(a.out + o + HALF * h) = make_float4(acc[h][0], acc[h][1], acc[h][2], acc[h][3]);
      else {
        if (a.shared) add(acc[h], sv[h], gate);
        *reinterpret_cast<uint4*>(a.cout + o + HALF * h) = f8_pack8(acc[h]);
      }
    }
  }
}

}  // namespace hb

using namespace hb;

namespace {
using F8Kernel = void (*)(const F8Args, const CUtensorMap, const CUtensorMap);
struct F8Pick { F8Kernel fn; int smem; };
// rows: of a tile, at most (256: a pair's)
template <int MODE>
F8Pick f8_kernel(int rows) {
  switch (rows) {
    case 16: return {fp8_gemm_kernel<16, MODE>, F8Cfg<16>::SMEM};
    case 32: return {fp8_gemm_kernel<32, MODE>, F8Cfg<32>::SMEM};
    case F8S_ROWS: return {fp8_many_kernel<MODE, false>, F8PCfg<false>::SMEM};
    default: return {fp8_many_kernel<F8_PLAIN, true>, F8PCfg<true>::SMEM};
  }
}
F8Gpu f8_gpu(const hb_ctx* ctx) { return {ctx->sm_count, ctx->max_ctas, ctx->fp8_clusters}; }
template <int MODE>
int f8_launch(hb_ctx* ctx, const char* name, int rows, const F8Args& a, const CUtensorMap& w, const CUtensorMap& x, cudaStream_t st) {
  const F8Pick k = f8_kernel<MODE>(rows);
  const int cl = rows == F8P_ROWS ? 2 : rows == F8S_ROWS ? a.split : 1;
  return hb_launch_cluster(ctx, name, true, cl, k.fn, dim3(f8_grid(f8_gpu(ctx), rows, cl)), dim3(F8_THREADS), (size_t)k.smem, st, a, w, x);
}
// Pairs of a tile by what an expert gets on average: longer runs are cut into tiles, which read the expert's weights again, and a tile that is not full
// wastes its MMAs.  Gate/up + down of 512 experts of 2048 / 512: 20 pairs an expert 310 us with 32, 359 with 128 (39 pairs: 476, 375; 10 pairs: 294, and 293
// with 16).  Pairs of CTAs gained nothing here (32 experts of 7168 / 2048, 256 pairs an expert: 533 us with 128, 661 with 256, half of whose second tiles were
// empty; 8 experts of 4096 / 1536, 2048 pairs: 399, 439), so routed experts have no such form.
int f8_rows_for_pairs(long long P, int E) { return P <= 8ll * E ? 16 : P <= 24ll * E ? 32 : F8S_ROWS; }
// map of a byte matrix [n_rows][row_bytes], rows ld bytes apart, in boxes of 128 bytes × box_rows under the 128-byte swizzle; bytes and rows past the
// end read as zero codes
int f8_map(hb_ctx* ctx, CUtensorMap* m, const void* base, size_t row_bytes, size_t ld, size_t n_rows, int box_rows) {
  TcEncodeFn fn = tc_encode_fn();
  HB_REQUIRE(ctx, fn, HB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)n_rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {128u, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  HB_REQUIRE(ctx, r == CUDA_SUCCESS, HB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %zu rows of %zu bytes at %p", (int)r, n_rows, row_bytes, base);
  return HB_OK;
}

struct F8Ws {
  int* hist; int* n_slots; int* n_tiles; TileRef* tiles; int* perm; int* pos_of; uint8_t* xq; float* xs; uint8_t* yq; float* ys; void* part; float* cut; uint8_t* maps;
};
size_t f8_carve(void* ws, int M, int K, int E, int H, int I, F8Ws* w) {
  size_t off = 0;
  auto take = [&](size_t b) { void* r = ws ? static_cast<char*>(ws) + off : nullptr; off += hb_align256(b); return r; };
  const size_t P = (size_t)M * K;
  const int bn = f8_rows_for_pairs((long long)P, E);
  F8Ws t;
  t.hist = (int*)take(hbk_pf_plan_hist_bytes(E)); t.n_slots = (int*)take(4); t.n_tiles = (int*)take(4);
  t.tiles = (TileRef*)take((P / 16 + E) * sizeof(TileRef)); t.perm = (int*)take(P * 4); t.pos_of = (int*)take(P * 4);
  t.yq = (uint8_t*)take(P * I); t.ys = (float*)take(P * f8_blocks(I) * 4);
  // The down pass writes its results, of two or four bytes, over the rows that the gate/up pass was given (codes and scales, 1 + 1 / 32 bytes a value)
  const size_t rows = off;
  t.xq = (uint8_t*)take(P * H); t.xs = (float*)take(P * f8_blocks(H) * 4);
  off = rows;
  t.part = take(P * H * 4);
  t.cut = (float*)take(f8_part_bytes(bn));
  t.maps = (uint8_t*)take((size_t)2 * F8_MAX_CTAS * F8_MAPS * sizeof(CUtensorMap));   // of the gate/up pass and of the down pass
  if (w) *w = t;
  return off;
}
unsigned int* f8_counters(hb_ctx* ctx) { return reinterpret_cast<unsigned int*>(ctx->dev_err) + kErrCounters; }
int f8_rows(hb_ctx* ctx, const F8RowsArgs& a, cudaStream_t st) {
  const long long units = (long long)a.M * f8_blocks(a.K), ctas = (units + 31) / 32, cap = (long long)ctx->sm_count * 32;
  return hb_launch(ctx, "fp8_quant_rows", true, fp8_quant_rows_kernel, dim3((unsigned)(ctas < cap ? ctas : cap)), dim3(256), 0, st, a);
}
}  // namespace

int hbk_fp8_setup(hb_ctx* ctx) {
  for (int bn : {16, 32, F8S_ROWS, F8P_ROWS})
    for (const F8Pick& k : {f8_kernel<F8_PLAIN>(bn), f8_kernel<F8_GU>(bn), f8_kernel<F8_DOWN>(bn), f8_kernel<F8_DOWN32>(bn)}) {   // (256: the dense product alone)
      cudaFuncAttributes at;
      HB_CUDA(ctx, cudaFuncGetAttributes(&at, reinterpret_cast<const void*>(k.fn)));
      // a warp that asks for more registers than the block was launched with would wait for good
      HB_REQUIRE(ctx, bn < F8S_ROWS || at.numRegs >= F8_REGS, HB_ERR_CUDA, "fp8_gemm: built with %d registers a thread, its warps share out %d", at.numRegs, F8_REGS);
      HB_CUDA(ctx, cudaFuncSetAttribute(reinterpret_cast<const void*>(k.fn), cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem));
    }
  // clusters of four CTAs of the one-CTA form that are resident at once: where an SM group's number of SMs is not a multiple of four, SMs are left over
  const F8Pick k = f8_kernel<F8_PLAIN>(F8S_ROWS);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(4 * F8_MAX_CTAS); cfg.blockDim = dim3(F8_THREADS); cfg.dynamicSmemBytes = (size_t)k.smem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 4; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  HB_CUDA(ctx, cudaOccupancyMaxActiveClusters(&ctx->fp8_clusters, reinterpret_cast<const void*>(k.fn), &cfg));
  return HB_OK;
}

extern "C" {

int hb_fp8_quant_rows(hb_ctx* ctx, const void* x, int ldx, int M, int K, uint8_t* q, int ldq, float* s, int lds, void* stream) {
  if (!ctx) return HB_ERR_INVALID;
  if (M == 0) return HB_OK;
  HB_REQUIRE(ctx, x && q && s, HB_ERR_INVALID, "fp8_quant_rows: NULL argument");
  HB_REQUIRE(ctx, M > 0 && K > 0 && K % 16 == 0 && K <= 1 << 30, HB_ERR_UNSUPPORTED, "fp8_quant_rows: M=%d K=%d (K %% 16, K <= 2^30)", M, K);
  HB_REQUIRE(ctx, ldx >= K && ldq >= K && ldq % 16 == 0 && lds >= M, HB_ERR_INVALID, "fp8_quant_rows: ldx=%d ldq=%d (>= K=%d, ldq %% 16) lds=%d (>= M=%d)", ldx, ldq, K, lds, M);
  HB_REQUIRE(ctx, hb_aligned(x, 2) && hb_aligned(q, 16) && hb_aligned(s, 4), HB_ERR_INVALID, "fp8_quant_rows: q must be 16-byte aligned, x and s to their elements");
  F8RowsArgs a{};
  a.x = reinterpret_cast<const __nv_bfloat16*>(x); a.ldx = ldx; a.M = M; a.K = K; a.q = q; a.ldq = ldq; a.s = s; a.lds = lds;
  return f8_rows(ctx, a, reinterpret_cast<cudaStream_t>(stream));
}

int hb_fp8_quantize(hb_ctx* ctx, const void* w, int bf16, int N, int K, uint8_t* q, float* s, void* stream) {
  if (!ctx) return HB_ERR_INVALID;
  HB_REQUIRE(ctx, w && q && s, HB_ERR_INVALID, "fp8_quantize: NULL argument");
  HB_REQUIRE(ctx, N > 0 && N <= 1 << 30 && K > 0 && K % 16 == 0 && K <= 1 << 30, HB_ERR_UNSUPPORTED, "fp8_quantize: N=%d K=%d (K %% 16, both <= 2^30)", N, K);
  HB_REQUIRE(ctx, hb_aligned(w, 16) && hb_aligned(q, 16) && hb_aligned(s, 4), HB_ERR_INVALID, "fp8_quantize: w and q must be 16-byte aligned, s to its elements");
  const long long blocks = (long long)f8_blocks(N) * f8_blocks(K);
  HB_REQUIRE(ctx, blocks < (1ll << 31), HB_ERR_UNSUPPORTED, "fp8_quantize: N=%d K=%d", N, K);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (bf16) return hb_launch(ctx, "fp8_quantize", false, fp8_quantize_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), 0, st, reinterpret_cast<const __nv_bfloat16*>(w), N, K, q, s);
  return hb_launch(ctx, "fp8_quantize", false, fp8_quantize_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, reinterpret_cast<const float*>(w), N, K, q, s);
}

size_t hb_fp8_gemm_ws_bytes(int M, int N, int K) { return M > 0 && N > 0 && K > 0 ? f8_part_bytes(f8_most_rows(M)) : 0; }

int hb_fp8_gemm(hb_ctx* ctx, const hb_qmat* W, const uint8_t* xq, int ldq, const float* xs, int lds, int M, void* yb, float* yf, int ldy, void* ws, void* stream) {
  if (!ctx) return HB_ERR_INVALID;
  if (M == 0) return HB_OK;
  HB_REQUIRE(ctx, W && W->w && W->s && xq && xs && (!yb != !yf), HB_ERR_INVALID, "fp8_gemm: NULL argument, or not exactly one output");
  HB_REQUIRE(ctx, W->fmt == HB_FMT_FP8_B128 && W->N > 0 && W->K > 0 && W->K % 16 == 0 && M > 0, HB_ERR_UNSUPPORTED, "fp8_gemm: FP8_B128 matrix with K %% 16 == 0 wanted (fmt %d N=%d K=%d M=%d)",
             W->fmt, W->N, W->K, M);
  HB_REQUIRE(ctx, W->K <= 1 << 23 && W->N <= 1 << 30 && M <= 1 << 30, HB_ERR_UNSUPPORTED, "fp8_gemm: M=%d N=%d (<= 2^30) K=%d (<= 2^23)", M, W->N, W->K);
  HB_REQUIRE(ctx, ldq >= W->K && ldq % 16 == 0 && lds >= M && ldy >= W->N, HB_ERR_INVALID, "fp8_gemm: ldq=%d (>= K=%d, %% 16) lds=%d (>= M=%d) ldy=%d (>= N=%d)", ldq, W->K, lds, M, ldy, W->N);
  HB_REQUIRE(ctx, hb_aligned(W->w, 16) && hb_aligned(xq, 16) && hb_aligned(W->s, 4) && hb_aligned(xs, 4) && hb_aligned(yb, 2) && hb_aligned(yf, 4), HB_ERR_INVALID,
             "fp8_gemm: codes must be 16-byte aligned, scales and outputs to their elements");
  HB_REQUIRE(ctx, ws && hb_aligned(ws, 256), HB_ERR_WORKSPACE, "fp8_gemm: ws NULL or not 256-byte aligned");
  const F8Cut cut = f8_cut(f8_gpu(ctx), M, W->N, W->K);
  const int rows = cut.rows, nt = (M + rows - 1) / rows;
  F8Args a{};
  a.M = M; a.per = rows == F8P_ROWS ? rows : ((M + nt - 1) / nt + 15) & ~15; a.N = W->N; a.K = W->K; a.n_nt = (W->N + 255) / 256;
  HB_REQUIRE(ctx, (long long)nt * a.n_nt < (1ll << 31), HB_ERR_UNSUPPORTED, "fp8_gemm: M=%d N=%d", M, W->N);
  a.ws = reinterpret_cast<const float*>(W->s); a.xs = xs; a.lds = lds;
  a.yb = reinterpret_cast<__nv_bfloat16*>(yb); a.yf = yf; a.ldy = ldy; a.part = reinterpret_cast<float*>(ws); a.room = (uint32_t)(f8_part_bytes(f8_most_rows(M)) / 4); a.count = f8_counters(ctx); a.err = ctx->dev_err;
  CUtensorMap tw, tx;
  const bool many = rows >= F8S_ROWS;
  a.split = cut.split;
  int r;
  if ((r = f8_map(ctx, &tw, W->w, W->K, W->K, W->N, many ? 64 : 128)) || (r = f8_map(ctx, &tx, xq, W->K, ldq, M, many ? 128 : rows))) return r;
  return f8_launch<F8_PLAIN>(ctx, "fp8_gemm", rows, a, tw, tx, reinterpret_cast<cudaStream_t>(stream));
}

int hb_fp8_rec_layout_make(int H, int I, hb_fp8_rec_layout* L) {
  if (!L || H <= 0 || I <= 0 || (H % 128) || (I % 128) || H > 1 << 20 || I > 1 << 20) return HB_ERR_INVALID;
  const uint64_t w = (uint64_t)H * I, s = (uint64_t)(H / 128) * (I / 128) * 4;
  L->w1 = 0; L->w3 = w; L->w2 = 2 * w; L->s1 = 3 * w; L->s3 = L->s1 + s; L->s2 = L->s3 + s;
  L->total = (L->s2 + s + 4095) / 4096 * 4096;
  return HB_OK;
}

size_t hb_moe_fp8_ws_bytes(int M, int K, int E, int H, int I) {
  hb_fp8_rec_layout L;
  if (M < 1 || K < 1 || E < 1 || hb_fp8_rec_layout_make(H, I, &L) != HB_OK) return 0;
  return f8_carve(nullptr, M, K, E, H, I, nullptr);
}

int hb_moe_fp8(hb_ctx* ctx, const int32_t* ids, const float* w, int M, int K, const uint8_t* const* rec_tab, int li, int E, const void* x, int H, int I, float limit,
               float* out, const hb_pf_combine* cmb, void* ws, void* stream) {
  if (!ctx) return HB_ERR_INVALID;
  if (M == 0) return HB_OK;
  HB_REQUIRE(ctx, ids && w && rec_tab && x && (cmb ? cmb->out != nullptr : out != nullptr), HB_ERR_INVALID, "moe_fp8: NULL argument");
  hb_fp8_rec_layout L;
  HB_REQUIRE(ctx, hb_fp8_rec_layout_make(H, I, &L) == HB_OK && M > 0 && K >= 1 && K <= 32 && E >= 1 && E <= HB_MAX_EXPERTS && li >= 0 && (long long)M * K < (1ll << 30), HB_ERR_UNSUPPORTED,
             "moe_fp8: H=%d I=%d (multiples of 128 up to 2^20) M=%d K=%d (1..32, M·K < 2^30) E=%d (1..%d) li=%d", H, I, M, K, E, HB_MAX_EXPERTS, li);
  HB_REQUIRE(ctx, hb_aligned(x, 16) && hb_aligned(out, 16) && (!cmb || (hb_aligned(cmb->shared, 16) && hb_aligned(cmb->out, 16))), HB_ERR_INVALID,
             "moe_fp8: x, out, shared rows and combined output must be 16-byte aligned");
  HB_REQUIRE(ctx, hb_aligned(ids, 4) && hb_aligned(w, 4) && hb_aligned(rec_tab, 8) && (!cmb || (hb_aligned(cmb->lg, 4) && (!cmb->shared || !cmb->lg || (cmb->col >= 0 && cmb->col < cmb->ld)))), HB_ERR_INVALID,
             "moe_fp8: ids, w, rec_tab and lg must be aligned to their elements, col within lg's rows");
  HB_REQUIRE(ctx, ws && hb_aligned(ws, 256), HB_ERR_WORKSPACE, "moe_fp8: ws NULL or not 256-byte aligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uint8_t* const* tab = rec_tab + (size_t)li * E;
  F8Ws W;
  f8_carve(ws, M, K, E, H, I, &W);
  const int P = M * K, rows = f8_rows_for_pairs(P, E), box = rows < 128 ? rows : 128;
  int r;
  // maps of a record's matrices (gate and up lie one behind the other), to be given their addresses on the device; of the rows of x and y
  CUtensorMap tg, td, tx, ty;
  const int wbox = rows >= F8S_ROWS ? 64 : 128;
  if ((r = f8_map(ctx, &tg, W.xq, H, H, 2 * I, wbox)) || (r = f8_map(ctx, &td, W.xq, I, I, H, wbox))) return r;
  if ((r = f8_map(ctx, &tx, W.xq, H, H, P, box)) || (r = f8_map(ctx, &ty, W.yq, I, I, P, box))) return r;
  F8PrepArgs pr{};
  F8RowsArgs& q = pr.rows;
  q.x = reinterpret_cast<const __nv_bfloat16*>(x); q.ldx = H; q.M = M; q.K = H; q.dest = W.pos_of; q.nd = K; q.q = W.xq; q.ldq = H; q.s = W.xs; q.lds = P;
  const bool own_plan = P <= F8_PLAN_PAIRS && rows < F8S_ROWS;
  if (own_plan) {
    pr.plan = F8Plan{ids, P, E, rows, tab}; pr.pos_of = W.pos_of; pr.tiles = W.tiles; pr.n_tiles = W.n_tiles;
    if ((r = hb_launch(ctx, "fp8_prep", true, fp8_prep_kernel, dim3(1 + (unsigned)((M * f8_blocks(H) + 15) / 16)), dim3(256), 0, st, pr))) return r;
  } else {
    if ((r = hbk_pf_plan(ctx, hbk_plan{ids, P, E, tab, rows, W.hist, W.perm, W.pos_of, W.tiles, W.n_tiles, W.n_slots}, st))) return r;
    if ((r = f8_rows(ctx, q, st))) return r;
  }
  F8Args a{};
  a.tiles = W.tiles; a.n_tiles = W.n_tiles; a.tab = tab; a.limit = limit; a.part = W.cut; a.room = (uint32_t)(f8_part_bytes(rows) / 4); a.count = f8_counters(ctx); a.err = ctx->dev_err;
  a.N = I; a.K = H; a.n_nt = I / 128; a.off_w = L.w1; a.off_s0 = L.s1; a.off_s1 = L.s3; a.row2 = I; a.maps = W.maps;
  a.xs = W.xs; a.lds = P; a.yq = W.yq; a.ys = W.ys; a.ldys = P;
  if (own_plan) a.plan = pr.plan;
  a.split = 2;                                                                 // (all SMs are in reach of clusters of two)
  if ((r = f8_launch<F8_GU>(ctx, "fp8_gemm_gu", rows, a, tg, tx, st))) return r;
  a.N = H; a.K = I; a.n_nt = (H + 255) / 256; a.off_w = L.w2; a.off_s0 = a.off_s1 = L.s2; a.maps = W.maps + (size_t)F8_MAX_CTAS * F8_MAPS * sizeof(CUtensorMap);
  a.xs = W.ys; a.ldy = H;
  if (cmb) a.yb = reinterpret_cast<__nv_bfloat16*>(W.part); else a.yf = reinterpret_cast<float*>(W.part);
  if ((r = cmb ? f8_launch<F8_DOWN>(ctx, "fp8_gemm_down", rows, a, td, ty, st) : f8_launch<F8_DOWN32>(ctx, "fp8_gemm_down", rows, a, td, ty, st))) return r;
  auto sum = [&](auto su) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(su.part)>>;
    const long long sums = ((long long)M * ((H + F8_SUM_COLS<T> - 1) / F8_SUM_COLS<T>) + F8_SUM_THREADS / 32 - 1) / (F8_SUM_THREADS / 32), cap = (long long)ctx->sm_count * 16;
    return hb_launch(ctx, "fp8_sum", true, fp8_sum_kernel<T>, dim3((unsigned)(sums < cap ? sums : cap)), dim3(F8_SUM_THREADS), 0, st, su);
  };
  if (!cmb) return sum(F8SumArgs<float>{reinterpret_cast<const float*>(W.part), W.pos_of, w, M, K, H, out, nullptr, nullptr, 0, 0, nullptr});
  F8SumArgs<__nv_bfloat16> su{reinterpret_cast<const __nv_bfloat16*>(W.part), W.pos_of, w, M, K, H, nullptr, nullptr, nullptr, 0, 0, reinterpret_cast<__nv_bfloat16*>(cmb->out)};
  su.shared = reinterpret_cast<const __nv_bfloat16*>(cmb->shared);
  if (cmb->shared) { su.lg = cmb->lg; su.ld = cmb->ld; su.col = cmb->col; }
  return sum(su);
}

}  // extern "C"
