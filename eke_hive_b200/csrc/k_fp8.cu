// 8-bit floats with a scale per block of 128: the quantisers of activations and weights, the product, the routed experts.
#include <cuda_fp8.h>

#include "hb_common.cuh"
#include "hb_kernels.h"
#include "tc_common.cuh"

namespace hb {

constexpr int F8_B = 128;                              // values a scale covers
__host__ __device__ constexpr int f8_blocks(int n) { return (n + F8_B - 1) / F8_B; }

// ---- quantisation -------------------------------------------------------------------------------------------------------------------
// The largest magnitude of a block as the bits of a float: they order like the magnitudes, infinities and NaN last.  From it the scale that
// is stored (amax / 448) and the code of each value: e4m3(v · 448 / amax).  v · 448 of a bf16 value is exact in fp32; the quotient is worked out
// from the reciprocal with one residual step, which gives the correctly rounded one (Markstein, "Computation of elementary functions on the
// IBM RISC System/6000 processor", 1990), and exactly the quotient where fp32 holds it, so a tie between two codes is seen as one.
// Blocks of very small or very large values are brought to the middle of the range by a power of two first: nothing over- or underflows
// that could be more than a zero code.
struct F8Block {
  float f, d, r; bool live;                            // v·f is the value scaled, d = amax·f, r = 1 / d
  __device__ __forceinline__ float init(uint32_t bits) {   // returns the scale
    const float amax = __uint_as_float(bits);
    live = bits > 0u && bits < 0x7f800000u;
    f = amax < 0x1p-60f ? 0x1p64f : amax > 0x1p60f ? 0x1p-64f : 1.f;
    d = __fmul_rn(amax, f); r = live ? __frcp_rn(d) : 0.f;
    return bits < 0x7f800000u ? __fdiv_rn(amax, 448.f) : __int_as_float(0x7fc00000);
  }
  __device__ __forceinline__ float quotient(float v) const {
    const float t = __fmul_rn(__fmul_rn(v, f), 448.f), q = __fmul_rn(t, r);
    return copysignf(__fmaf_rn(__fmaf_rn(-q, d, t), r, q), t);
  }
  __device__ __forceinline__ uint32_t pair(float a, float b) const {   // codes of two values, the first in the low byte
    uint16_t o;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(o) : "f"(quotient(b)), "f"(quotient(a)));
    return live ? (uint32_t)o : 0u;
  }
};
__device__ __forceinline__ uint32_t f8_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Rows: 16 lanes take a block of 128 values, 8 each.  dest == nullptr: row m of q / s; else row m goes to slots dest[m·nd + j], j < nd, negative ones
// skipped (the rows of a routed layer are quantised once and written into expert order).  Source: bf16, or silu(g)·u of two fp32 matrices.
struct F8RowsArgs {
  const __nv_bfloat16* x; int ldx;
  const float* g; const float* u; float limit;         // x == nullptr: y = silu(g)·u, both [M,K]
  int M, K; const int* m_dev;                          // m_dev: rows there really are (device), at most M
  const int* dest; int nd;
  uint8_t* q; int ldq; float* s; int lds;
};
__global__ void __launch_bounds__(256) fp8_quant_rows_kernel(const F8RowsArgs a) {
  griddep_wait();
  const int nb = f8_blocks(a.K), l16 = threadIdx.x & 15;
  const uint32_t half = 0xffffu << (threadIdx.x & 16);
  const int M = a.m_dev ? min(a.M, *a.m_dev) : a.M;
  const long long total = (long long)M * nb;
  for (long long i = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); i < total; i += (long long)gridDim.x * 16) {
    const int m = (int)(i / nb), b = (int)(i - (long long)m * nb), k = b * F8_B + l16 * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (k < a.K) {                                                             // K is a multiple of 16: eight values are inside or outside together
      if (a.x) {
        const __nv_bfloat16* p = a.x + (size_t)m * a.ldx + k;
        if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
          const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(ww[j] << 16); v[2 * j + 1] = __uint_as_float(ww[j] & 0xffff0000u); }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __bfloat162float(p[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float gv = a.g[(size_t)m * a.K + k + j], uv = a.u[(size_t)m * a.K + k + j];
          if (a.limit > 0.f) { gv = fminf(gv, a.limit); uv = fminf(fmaxf(uv, -a.limit), a.limit); }
          v[j] = gv / (1.f + expf(-gv)) * uv;
        }
      }
    }
    uint32_t mx = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = max(mx, f8_mag(v[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(half, mx, o));
    F8Block blk;
    const float sc = blk.init(mx);
    const uint2 c = make_uint2(blk.pair(v[0], v[1]) | blk.pair(v[2], v[3]) << 16, blk.pair(v[4], v[5]) | blk.pair(v[6], v[7]) << 16);
    for (int j = 0; j < (a.dest ? a.nd : 1); ++j) {
      const int slot = a.dest ? a.dest[(size_t)m * a.nd + j] : m;
      if (slot < 0) continue;
      if (k < a.K) *reinterpret_cast<uint2*>(a.q + (size_t)slot * a.ldq + k) = c;
      if (l16 == 0) a.s[(size_t)b * a.lds + slot] = sc;
    }
  }
}

// Weights: a CTA takes a block of 128 × 128, sixteen lanes a row of it, eight rows a thread.
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

// ---- the product, simple form: 64 rows × 64 tokens a CTA, fp32 on the CUDA cores --------------------------------------------------------
struct F8GemmArgs {
  const uint8_t* w; const float* ws;                   // one matrix, or (tab) the expert's at these offsets
  const uint8_t* const* tab; uint64_t off_w, off_s;
  const TileRef* tiles; const int* n_tiles;            // tab: tiles of slots
  const uint8_t* xq; int ldq; const float* xs; int lds;
  int M, N, K;
  __nv_bfloat16* yb; float* yf; int ldy;
};
__global__ void __launch_bounds__(256) fp8_gemm_simple_kernel(const F8GemmArgs a) {
  __shared__ float xa[32][65], wa[32][65];
  TileRef t{(int)blockIdx.y * 64, min(64, a.M - (int)blockIdx.y * 64), 0};
  const uint8_t* w = a.w; const float* ws = a.ws;
  if (a.tab) {
    if ((int)blockIdx.y >= *a.n_tiles) return;
    t = a.tiles[blockIdx.y];
    w = a.tab[t.expert] + a.off_w; ws = reinterpret_cast<const float*>(a.tab[t.expert] + a.off_s);
  }
  const int n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, nb = f8_blocks(a.K);
  float acc[4][4] = {}, part[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += 32) {
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
      const int r = i >> 5, k = k0 + (i & 31);
      xa[i & 31][r] = r < t.rows && k < a.K ? e4m3_to_f32(a.xq[(size_t)(t.slot0 + r) * a.ldq + k]) : 0.f;
      wa[i & 31][r] = n0 + r < a.N && k < a.K ? e4m3_to_f32(w[(size_t)(n0 + r) * a.K + k]) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = fmaf(xa[k][ty * 4 + i], wa[k][tx + 16 * j], part[i][j]);
    __syncthreads();
    if ((k0 & 127) == 96 || k0 + 32 >= a.K) {
      const float sw = ws[(size_t)(n0 >> 7) * nb + (k0 >> 7)];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float sx = ty * 4 + i < t.rows ? a.xs[(size_t)(k0 >> 7) * a.lds + t.slot0 + ty * 4 + i] * sw : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) { acc[i][j] = fmaf(part[i][j], sx, acc[i][j]); part[i][j] = 0.f; }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = ty * 4 + i, n = n0 + tx + 16 * j;
      if (r >= t.rows || n >= a.N) continue;
      const size_t at = (size_t)(t.slot0 + r) * a.ldy + n;
      if (a.yb) a.yb[at] = __float2bfloat16(acc[i][j]);
      else a.yf[at] = acc[i][j];
    }
}

// ---- the sum over a row's pairs: out[m] = Σ_k w[m,k]·part[slot of (m,k)] (+ gate·shared[m]) --------------------------------------------
__global__ void __launch_bounds__(256) fp8_sum_kernel(const __nv_bfloat16* __restrict__ part, const int* __restrict__ pos_of, const float* __restrict__ w, int K, int H,
                                                      float* __restrict__ out, const __nv_bfloat16* __restrict__ shared, const float* __restrict__ lg, int ld, int col,
                                                      __nv_bfloat16* __restrict__ cout) {
  const int m = blockIdx.x;
  const float gate = lg ? 1.f / (1.f + expf(-lg[(size_t)m * ld + col])) : 1.f;
  for (int n = threadIdx.x; n < H; n += 256) {
    float acc = 0.f;
    for (int k = 0; k < K; ++k) {
      const int slot = pos_of[(size_t)m * K + k];
      if (slot >= 0) acc = fmaf(w[(size_t)m * K + k], __bfloat162float(part[(size_t)slot * H + n]), acc);
    }
    if (!cout) out[(size_t)m * H + n] = acc;
    else cout[(size_t)m * H + n] = __float2bfloat16(shared ? fmaf(gate, __bfloat162float(shared[(size_t)m * H + n]), acc) : acc);
  }
}

}  // namespace hb

using namespace hb;

namespace {
constexpr int F8_BM = 64;                              // tokens of a tile
struct F8Ws {
  int* hist; int* n_slots; int* n_tiles; TileRef* tiles; int* perm; int* pos_of; uint8_t* xq; float* xs; float* g; float* u; uint8_t* yq; float* ys; __nv_bfloat16* part;
};
size_t f8_carve(void* ws, int M, int K, int E, int H, int I, F8Ws* w) {
  size_t off = 0;
  auto take = [&](size_t b) { void* r = ws ? static_cast<char*>(ws) + off : nullptr; off += hb_align256(b); return r; };
  const size_t P = (size_t)M * K;
  F8Ws t;
  t.hist = (int*)take(hbk_pf_plan_hist_bytes(E)); t.n_slots = (int*)take(4); t.n_tiles = (int*)take(4);
  t.tiles = (TileRef*)take((P / F8_BM + E) * sizeof(TileRef)); t.perm = (int*)take(P * 4); t.pos_of = (int*)take(P * 4);
  t.xq = (uint8_t*)take(P * H); t.xs = (float*)take(P * f8_blocks(H) * 4);
  t.g = (float*)take(P * I * 4); t.u = (float*)take(P * I * 4);
  t.yq = (uint8_t*)take(P * I); t.ys = (float*)take(P * f8_blocks(I) * 4);
  t.part = (__nv_bfloat16*)take(P * H * 2);
  if (w) *w = t;
  return off;
}
int f8_rows(hb_ctx* ctx, const F8RowsArgs& a, cudaStream_t st) {
  const long long units = (long long)a.M * f8_blocks(a.K), ctas = (units + 15) / 16, cap = (long long)ctx->sm_count * 32;
  return hb_launch(ctx, "fp8_quant_rows", !(ctx->flags & HB_FLAG_NO_PDL), fp8_quant_rows_kernel, dim3((unsigned)(ctas < cap ? ctas : cap)), dim3(256), 0, st, a);
}
}  // namespace

extern "C" {

int hb_fp8_quant_rows(hb_ctx* ctx, const void* x, int ldx, int M, int K, uint8_t* q, int ldq, float* s, int lds, void* stream) {
  if (!ctx) return HB_ERR_INVALID;
  if (M == 0) return HB_OK;
  HB_REQUIRE(ctx, x && q && s, HB_ERR_INVALID, "fp8_quant_rows: NULL argument");
  HB_REQUIRE(ctx, M > 0 && K > 0 && K % 16 == 0, HB_ERR_UNSUPPORTED, "fp8_quant_rows: M=%d K=%d (K %% 16)", M, K);
  HB_REQUIRE(ctx, ldx >= K && ldq >= K && ldq % 16 == 0 && lds >= M, HB_ERR_INVALID, "fp8_quant_rows: ldx=%d ldq=%d (>= K=%d, ldq %% 16) lds=%d (>= M=%d)", ldx, ldq, K, lds, M);
  HB_REQUIRE(ctx, hb_aligned(x, 2) && hb_aligned(q, 16) && hb_aligned(s, 4), HB_ERR_INVALID, "fp8_quant_rows: q must be 16-byte aligned, x and s to their elements");
  F8RowsArgs a{};
  a.x = reinterpret_cast<const __nv_bfloat16*>(x); a.ldx = ldx; a.M = M; a.K = K; a.nd = 1; a.q = q; a.ldq = ldq; a.s = s; a.lds = lds;
  return f8_rows(ctx, a, reinterpret_cast<cudaStream_t>(stream));
}

int hb_fp8_quantize(hb_ctx* ctx, const void* w, int bf16, int N, int K, uint8_t* q, float* s, void* stream) {
  if (!ctx) return HB_ERR_INVALID;
  HB_REQUIRE(ctx, w && q && s, HB_ERR_INVALID, "fp8_quantize: NULL argument");
  HB_REQUIRE(ctx, N > 0 && K > 0 && K % 16 == 0, HB_ERR_UNSUPPORTED, "fp8_quantize: N=%d K=%d (K %% 16)", N, K);
  HB_REQUIRE(ctx, hb_aligned(w, 16) && hb_aligned(q, 16) && hb_aligned(s, 4), HB_ERR_INVALID, "fp8_quantize: w and q must be 16-byte aligned");
  const long long blocks = (long long)f8_blocks(N) * f8_blocks(K);
  HB_REQUIRE(ctx, blocks < (1ll << 31), HB_ERR_UNSUPPORTED, "fp8_quantize: N=%d K=%d", N, K);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (bf16) return hb_launch(ctx, "fp8_quantize", false, fp8_quantize_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), 0, st, reinterpret_cast<const __nv_bfloat16*>(w), N, K, q, s);
  return hb_launch(ctx, "fp8_quantize", false, fp8_quantize_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, reinterpret_cast<const float*>(w), N, K, q, s);
}

size_t hb_fp8_gemm_ws_bytes(int M, int N, int K) { return M > 0 && N > 0 && K > 0 ? 256 : 0; }

int hb_fp8_gemm(hb_ctx* ctx, const hb_qmat* W, const uint8_t* xq, int ldq, const float* xs, int lds, int M, void* yb, float* yf, int ldy, void* ws, void* stream) {
  if (!ctx) return HB_ERR_INVALID;
  if (M == 0) return HB_OK;
  HB_REQUIRE(ctx, W && W->w && W->s && xq && xs && (!yb != !yf), HB_ERR_INVALID, "fp8_gemm: NULL argument, or not exactly one output");
  HB_REQUIRE(ctx, W->fmt == HB_FMT_FP8_B128 && W->N > 0 && W->K > 0 && W->K % 16 == 0 && M > 0, HB_ERR_UNSUPPORTED, "fp8_gemm: FP8_B128 matrix with K %% 16 == 0 wanted (fmt %d N=%d K=%d M=%d)",
             W->fmt, W->N, W->K, M);
  HB_REQUIRE(ctx, ldq >= W->K && ldq % 16 == 0 && lds >= M && ldy >= W->N, HB_ERR_INVALID, "fp8_gemm: ldq=%d (>= K=%d, %% 16) lds=%d (>= M=%d) ldy=%d (>= N=%d)", ldq, W->K, lds, M, ldy, W->N);
  HB_REQUIRE(ctx, hb_aligned(W->w, 16) && hb_aligned(xq, 16) && hb_aligned(W->s, 4) && hb_aligned(xs, 4) && hb_aligned(yb, 2) && hb_aligned(yf, 4), HB_ERR_INVALID,
             "fp8_gemm: codes must be 16-byte aligned, scales and outputs to their elements");
  HB_REQUIRE(ctx, ws && hb_aligned(ws, 256), HB_ERR_WORKSPACE, "fp8_gemm: ws NULL or not 256-byte aligned");
  F8GemmArgs a{};
  a.w = W->w; a.ws = reinterpret_cast<const float*>(W->s); a.xq = xq; a.ldq = ldq; a.xs = xs; a.lds = lds; a.M = M; a.N = W->N; a.K = W->K;
  a.yb = reinterpret_cast<__nv_bfloat16*>(yb); a.yf = yf; a.ldy = ldy;
  return hb_launch(ctx, "fp8_gemm", false, fp8_gemm_simple_kernel, dim3((W->N + 63) / 64, (M + 63) / 64), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), a);
}

int hb_fp8_rec_layout_make(int H, int I, hb_fp8_rec_layout* L) {
  if (!L || H <= 0 || I <= 0 || (H % 128) || (I % 128)) return HB_ERR_INVALID;
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
             "moe_fp8: H=%d I=%d (multiples of 128) M=%d K=%d (1..32, M·K < 2^30) E=%d (1..%d) li=%d", H, I, M, K, E, HB_MAX_EXPERTS, li);
  HB_REQUIRE(ctx, hb_aligned(x, 16) && hb_aligned(out, 16) && (!cmb || (hb_aligned(cmb->shared, 16) && hb_aligned(cmb->out, 16))), HB_ERR_INVALID,
             "moe_fp8: x, out, shared rows and combined output must be 16-byte aligned");
  HB_REQUIRE(ctx, ws && hb_aligned(ws, 256), HB_ERR_WORKSPACE, "moe_fp8: ws NULL or not 256-byte aligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uint8_t* const* tab = rec_tab + (size_t)li * E;
  F8Ws W;
  f8_carve(ws, M, K, E, H, I, &W);
  const int P = M * K;
  int r;
  if ((r = hbk_pf_plan(ctx, hbk_plan{ids, P, E, tab, F8_BM, W.hist, W.perm, W.pos_of, W.tiles, W.n_tiles, W.n_slots}, st))) return r;
  F8RowsArgs q{};
  q.x = reinterpret_cast<const __nv_bfloat16*>(x); q.ldx = H; q.M = M; q.K = H; q.dest = W.pos_of; q.nd = K; q.q = W.xq; q.ldq = H; q.s = W.xs; q.lds = P;
  if ((r = f8_rows(ctx, q, st))) return r;
  const unsigned tiles = (unsigned)(P / F8_BM + (E < P ? E : P));
  F8GemmArgs a{};
  a.tab = tab; a.tiles = W.tiles; a.n_tiles = W.n_tiles; a.xq = W.xq; a.ldq = H; a.xs = W.xs; a.lds = P; a.N = I; a.K = H; a.ldy = I;
  a.off_w = L.w1; a.off_s = L.s1; a.yf = W.g;
  if ((r = hb_launch(ctx, "fp8_gemm_gate", false, fp8_gemm_simple_kernel, dim3((I + 63) / 64, tiles), dim3(256), 0, st, a))) return r;
  a.off_w = L.w3; a.off_s = L.s3; a.yf = W.u;
  if ((r = hb_launch(ctx, "fp8_gemm_up", false, fp8_gemm_simple_kernel, dim3((I + 63) / 64, tiles), dim3(256), 0, st, a))) return r;
  F8RowsArgs y{};
  y.g = W.g; y.u = W.u; y.limit = limit; y.M = P; y.m_dev = W.n_slots; y.K = I; y.nd = 1; y.q = W.yq; y.ldq = I; y.s = W.ys; y.lds = P;
  if ((r = f8_rows(ctx, y, st))) return r;
  a.off_w = L.w2; a.off_s = L.s2; a.yf = nullptr; a.yb = W.part; a.xq = W.yq; a.ldq = I; a.xs = W.ys; a.N = H; a.K = I; a.ldy = H;
  if ((r = hb_launch(ctx, "fp8_gemm_down", false, fp8_gemm_simple_kernel, dim3((H + 63) / 64, tiles), dim3(256), 0, st, a))) return r;
  return hb_launch(ctx, "fp8_sum", false, fp8_sum_kernel, dim3(M), dim3(256), 0, st, (const __nv_bfloat16*)W.part, (const int*)W.pos_of, w, K, H, out,
                   cmb ? reinterpret_cast<const __nv_bfloat16*>(cmb->shared) : (const __nv_bfloat16*)nullptr, cmb && cmb->shared ? cmb->lg : (const float*)nullptr, cmb ? cmb->ld : 0,
                   cmb ? cmb->col : 0, cmb ? reinterpret_cast<__nv_bfloat16*>(cmb->out) : (__nv_bfloat16*)nullptr);
}

}  // extern "C"
