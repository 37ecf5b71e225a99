// The product of fp8_gemm.cuh for many rows: two CTAs of a cluster work on one tile of 256 rows of x × 256 weight rows (tcgen05 cta_group::2), or one CTA on a
// tile of 128 rows.
//
// Rows of x are the A operand, 128 of them in each CTA's shared and tensor memory; the weight rows are the B operand, of which each CTA of a pair loads half
// and both read all: 32 KB of operands per CTA and step for 128 × 256 × 128 multiply-adds.  (One CTA alone needs 48 KB for them, which is 11.6 TB/s out of L2 at
// the rate it reaches: 4096 rows of 17408 x 5120 take 368 us with single CTAs, 338 with pairs.  That form is for runs of rows that would leave much of a
// pair's tile empty, and where there are few items.)  A lane of tensor memory is a row of x: the scale of a step is one number a thread, the row's times the
// weight block's.
//
// The 256 weight rows are two halves of 128, each with an accumulator of its own, double buffered (all of tensor memory), and its own warps: warps 0-3 read
// back half 0, warps 4-7 half 1, and while one half's MMAs run the other half is read.  Gate/up (single CTAs): a half is 64 gate rows and the 64 up rows that
// belong to them, so a thread has both for its row of x.
//
// Warp 8 (one thread) loads, warps 9 and 10 (one thread each, of a pair those of CTA 0) issue the MMAs, a half each, and announce finished buffers and free
// stages.  What bounds it: the read-back and scaling of every block's sums, 256 clocks of fused multiply-adds a step of 512 clocks of MMAs, behind waits and
// scales of their own: some 1000 clocks a step in all; large products run at the power limit's clock.
//
// Work is items as in fp8_gemm.cuh, in rounds of one item a CTA (or pair).  Of single CTAs, items that the last full round leaves over are split along K among
// the CTAs of a cluster, two or four, that add their sums up through each other's shared memory: 4 to 5 us.  Of pairs, they are cut and put together through the
// workspace as in fp8_gemm.cuh, each CTA with the parts of its own 128 rows, where 20 us of that are less than what it saves.
#pragma once
#include "fp8_gemm.cuh"

namespace hb {

constexpr int F8M_GROUP = 16;                          // tiles of rows that are gone through together
template <bool PAIR>
struct F8PCfg {
  static constexpr int CTAS = PAIR ? 2 : 1, ROWS = 128 * CTAS;
  static constexpr int XB = 128 * 128, HB = 128 * 128 / CTAS;   // a stage of one CTA: 128 rows of x, its rows of each half (64 or 128), 128 values each
  static constexpr int STAGE = XB + 2 * HB, ST = PAIR ? 6 : 4;
  static constexpr int STG = 8 * F8_STG_BYTES;
  static constexpr int SMEM = 1024 + ST * STAGE + STG + 2 * 128 * 4 + 512;
  using Sched = std::conditional_t<PAIR, F8Sched, F8Rounds>;
  static_assert(PAIR || ST * STAGE >= 2 * 128 * 128 * 4, "a split item's sums take the place of the operands");
  static_assert(ST < F8_MAPS && SMEM <= 227 * 1024, "map slots, shared memory");
};

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t mapa_u32(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// Arrival on a barrier of the pair.  No memory is handed over by it: what it orders are reads of tensor memory that have come back (tcgen05.wait::ld) and the
// MMAs that write there next; a release for the cluster, and acquires to match in every wait, cost 1000 clocks a step.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void tmem_alloc2(uint32_t* dst_smem, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// everything issued before is done: one arrival on the barrier at this place in both CTAs
__device__ __forceinline__ void tc_commit2(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tc_mma2_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// a box into this CTA's shared memory, its bytes counted on a barrier of the pair (an address in the cluster's window)
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* tmap, int c0, int c1, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(tmap), "r"(bar), "r"(c0), "r"(c1) : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void f8_mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR) tc_mma2_f8(d, ad, bd, idesc, accumulate);
  else tc_mma_f8(d, ad, bd, idesc, accumulate);
}
template <bool PAIR>
__device__ __forceinline__ void f8_commit(uint64_t* bar) {
  if constexpr (PAIR) tc_commit2(bar);
  else tc_commit(bar);
}

template <int MODE, bool PAIR>
__global__ void __launch_bounds__(F8_THREADS, 1) fp8_many_kernel(const __grid_constant__ F8Args a, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX) {
  using C = F8PCfg<PAIR>;
  extern __shared__ uint8_t f8p_raw[];
  const uint32_t raw = smem_u32(f8p_raw), base = (raw + 1023u) & ~1023u;       // the same offset in both CTAs
  uint8_t* sm = f8p_raw + (base - raw);
  uint32_t* amx = reinterpret_cast<uint32_t*>(sm + C::ST * C::STAGE + C::STG);   // magnitudes of y [2 halves][128 rows]
  uint64_t* full = reinterpret_cast<uint64_t*>(amx + 256);                     // [ST] CTA 0: both CTAs' operands of the stage have landed
  uint64_t* empty = full + C::ST;                                             // [ST] each CTA: the MMAs that read the stage are done
  uint64_t* acc_full = empty + C::ST;                                         // [2 halves][2 buffers] each CTA: its sums are there
  uint64_t* acc_empty = acc_full + 4;                                          // [2][2] CTA 0: both CTAs have read them
  uint64_t* mma_done = acc_empty + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile uint32_t* last = tmem_slot + 1;
  const int warp = warp_uniform(), lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;                            // of the pair
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::ST; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 2); }
    for (int s = 0; s < 4; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 4 * C::CTAS); }
    mbar_init(mma_done, 2);
    mbar_fence_init();
  }
  if (warp == F8_W_MMA) {
    if constexpr (PAIR) tmem_alloc2(tmem_slot, 512);
    else { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // before griddep_wait: as in fp8_gemm.cuh (the tiles come from the kernel in front of the one in front)
  const int KB = f8_blocks(a.K), n_tiles = MODE == F8_PLAIN ? (a.M + a.per - 1) / a.per : *a.n_tiles;
  typename C::Sched sch;
  sch.init((uint32_t)n_tiles * a.n_nt, KB, gridDim.x / C::CTAS, blockIdx.x / C::CTAS, false, PAIR ? F8P_SLACK : (uint32_t)a.split);
  auto tile_of = [&](int ti) -> TileRef {
    if (MODE != F8_PLAIN) return a.tiles[ti];
    return TileRef{ti * a.per, min(a.per, a.M - ti * a.per), 0};
  };
  // Item → tile of rows, 256 weight rows.  Dense: the row tiles (in groups of 16) go by faster, so that the CTAs of a round share weights as well as rows of x and
  // each comes from memory about once.  (Weights faster: 2048 rows of 17408 x 5120 read 577 MB, 203 us; this way 100 MB, all there is, 177.)
  auto place = [&](int item, int& ti, int& nt) {
    if (MODE != F8_PLAIN) { ti = item / a.n_nt; nt = item - ti * a.n_nt; return; }
    const int g = item / (F8M_GROUP * a.n_nt), r = item - g * (F8M_GROUP * a.n_nt), gs = min(F8M_GROUP, n_tiles - g * F8M_GROUP);
    nt = r / gs; ti = g * F8M_GROUP + r - nt * gs;
  };
  int item, kb0, kb1;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F8_REGS_REST));
    if (warp == F8_W_TMA) {
      // ---------------------------------------------------------------------------------------------- operand tiles, one thread of each CTA
      if (elect_one()) {
        uint32_t s = 0, ph = 1;
        bool ok = true, waited = false;
        F8Maps maps{a.maps + (size_t)blockIdx.x * F8_MAPS * sizeof(CUtensorMap), 0u, -1, nullptr};
        const uint32_t full0 = PAIR ? mapa_u32(smem_u32(full), 0) : 0u;
        while (ok && sch.next(item, kb0, kb1)) {
          int ti, nt;
          place(item, ti, nt);
          const TileRef tl = tile_of(ti);
          const void* mw = MODE == F8_PLAIN ? &tmW : maps.make(tmW, a.tab, tl.expert, a.off_w, a.err);
          // rows of each half, in boxes of 64: of a pair each CTA loads one, else both are this CTA's.  Rows past the last read as zero codes
          const int r0 = MODE == F8_GU ? nt * 128 : nt * 256, box = MODE == F8_GU ? a.row2 : 64, half = MODE == F8_GU ? 64 : 128;
          auto weights = [&](uint32_t st, int kb) {
            const uint32_t wb = base + st * C::STAGE + C::XB, bar = full0 + st * 8;
            if (rank == 0) mbar_expect_tx(&full[st], C::CTAS * C::STAGE);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if constexpr (PAIR) tma_load_2d_pair(wb + h * C::HB, mw, kb * 128, r0 + h * half + (int)rank * box, bar);
              else {
                tma_load_2d(wb + h * C::HB, mw, kb * 128, r0 + h * half, &full[st]);
                tma_load_2d(wb + h * C::HB + C::HB / 2, mw, kb * 128, r0 + h * half + box, &full[st]);
              }
            }
          };
          auto rows = [&](uint32_t st, int kb) {
            if constexpr (PAIR) tma_load_2d_pair(base + st * C::STAGE, &tmX, kb * 128, tl.slot0 + (int)rank * 128, full0 + st * 8);
            else tma_load_2d(base + st * C::STAGE, &tmX, kb * 128, tl.slot0, &full[st]);
          };
          int kb = kb0;
          if (!waited) {
            const int n = MODE == F8_PLAIN ? 0 : min(kb1 - kb0, C::ST);
            for (int i = 0; i < n; ++i) weights(i, kb0 + i);
            griddep_wait();
            waited = true;
            for (int i = 0; i < n; ++i) rows(i, kb0 + i);
            kb += n;
            s = n == C::ST ? 0 : n; ph = n == C::ST ? 0 : 1;
          }
          for (; kb < kb1; ++kb) {
            if (!(ok = mbar_wait(&empty[s], ph, a.err, kErrFp8Stage))) break;
            weights(s, kb);
            rows(s, kb);
            if (++s == C::ST) { s = 0; ph ^= 1u; }
          }
        }
        // free stages are announced to both CTAs of a pair: the last announcements arrive before either ends
        for (int n = 0; ok && n < C::ST; ++n) {
          ok = mbar_wait(&empty[s], ph, a.err, kErrFp8Stage);
          if (++s == C::ST) { s = 0; ph ^= 1u; }
        }
      }
    } else if ((warp == F8_W_MMA || warp == F8_W_MMA + 1) && rank == 0) {
      // ---------------------------------------------------------------------------------------------- MMA issue, one thread of CTA 0 for each half (one for both spent
      // 700 clocks a step on its waits and instructions)
      if (elect_one()) {
        const uint32_t h = warp - F8_W_MMA;
        uint32_t s = 0, ph = 0, it = 0;
        bool ok = true;
        // kind::f8f6f4: D fp32 (bit 4), A and B e4m3, both K-major, N / 8 = 16 at bit 17, M / 16 at bit 24
        constexpr uint32_t idesc = (1u << 4) | ((128u >> 3) << 17) | ((uint32_t)(C::ROWS >> 4) << 24);
        const uint64_t ad0 = tc_desc_sw128(base), bd0 = tc_desc_sw128(base + C::XB + h * C::HB);
        while (ok && sch.next(item, kb0, kb1)) {
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const uint32_t buf = it & 1u;
            if (!(ok = mbar_wait(&full[s], ph, a.err, kErrFp8Loads))) break;
            if (!(ok = mbar_wait(&acc_empty[h * 2 + buf], ((it >> 1) & 1u) ^ 1u, a.err, kErrFp8AccFree))) break;
            tc_fence_after();
            const uint64_t ad = ad0 + s * (uint32_t)(C::STAGE >> 4), bd = bd0 + s * (uint32_t)(C::STAGE >> 4);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)                                   // 32 values further along the swizzled rows
              f8_mma<PAIR>(tmem + buf * 256 + h * 128, ad + 2 * j, bd + 2 * j, idesc, j);
            f8_commit<PAIR>(&acc_full[h * 2 + buf]);
            f8_commit<PAIR>(&empty[s]);
            if (++s == C::ST) { s = 0; ph ^= 1u; }
          }
        }
        f8_commit<PAIR>(mma_done);                                                  // nothing is in flight when tensor memory is freed
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F8_REGS_SUM));
    griddep_wait();
    griddep_launch();
    // ------------------------------------------------------------------------------------------------ sums: warp (h, q) has rows [32 q, 32 q + 32) of half h, a row a lane
    const int h = warp >> 2, q = warp & 3, row = 32 * q + lane;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16) + h * 128;
    const uint32_t empty0 = PAIR ? mapa_u32(smem_u32(&acc_empty[h * 2]), 0) : 0u;
    uint32_t it = 0;
    bool ok = true;
    while (sch.next(item, kb0, kb1)) {                                          // after a wait that gave up: on to the end without waits and results, but through every barrier
      int ti, nt;
      place(item, ti, nt);
      const TileRef tl = tile_of(ti);
      const int rows = min(max(tl.rows - 128 * (int)rank, 0), 128);            // of this CTA
      const size_t slot0 = (size_t)tl.slot0 + 128 * rank;
      bool active = 32 * q < rows, valid = row < rows;
      // scales: of the row, of the weight blocks (gate/up: columns 0-63 gate, 64-127 up; else one block)
      const float *w0, *w1;
      if (MODE == F8_PLAIN) w0 = w1 = a.ws + (size_t)min(2 * nt + h, (a.N - 1) / 128) * KB;
      else {
        const uint8_t* rec = f8_rec(a.tab, tl.expert);
        const int b = MODE == F8_GU ? nt : min(2 * nt + h, (a.N - 1) / 128);
        w0 = reinterpret_cast<const float*>(rec + a.off_s0) + (size_t)b * KB;
        w1 = MODE == F8_GU ? reinterpret_cast<const float*>(rec + a.off_s1) + (size_t)b * KB : w0;
      }
      const float* xr = a.xs + slot0 + row;
      // three steps ahead: a scale comes from L2 in the time of two
      float x[3], s0[3], s1[3];
      auto fetch = [&](int kb, float& xv, float& v0, float& v1) {
        const bool on = kb < kb1;
        xv = on && valid ? __ldcg(xr + (size_t)kb * a.lds) : 0.f;
        v0 = on ? __ldg(w0 + kb) : 0.f;
        if (MODE == F8_GU) v1 = on ? __ldg(w1 + kb) : 0.f;
      };
#pragma unroll
      for (int i = 0; i < 3; ++i) fetch(kb0 + i, x[i], s0[i], s1[i]);
      float acc[128];
#pragma unroll
      for (int c = 0; c < 128; ++c) acc[c] = 0.f;
      uint32_t ra[32], rb[32];
      auto arrived = [&](uint32_t n) {
        const bool o = mbar_wait(&acc_full[h * 2 + (n & 1u)], (n >> 1) & 1u, a.err, kErrFp8Acc);
        tc_fence_after();
        return (bool)__all_sync(0xffffffffu, o);
      };
      if ((ok = ok && arrived(it)) && active) { tc_ld32(trow + (it & 1u) * 256, ra); tc_ld32(trow + (it & 1u) * 256 + 32, rb); }
      for (int kb = kb0; kb < kb1 && ok; ++kb, ++it) {
        const uint32_t buf = it & 1u, tb = trow + buf * 256;
        const float f0 = x[0] * s0[0], f1 = MODE == F8_GU ? x[0] * s1[0] : f0;
#pragma unroll
        for (int i = 0; i < 2; ++i) { x[i] = x[i + 1]; s0[i] = s0[i + 1]; if (MODE == F8_GU) s1[i] = s1[i + 1]; }
        fetch(kb + 3, x[2], s0[2], s1[2]);
        if (active) {
          f8_landed<32>(ra, rb);
          f8_add<32>(acc, ra, f0);
          tc_ld32(tb + 64, ra);
          f8_add<32>(acc + 32, rb, f0);
          tc_ld32(tb + 96, rb);
          f8_landed<32>(ra, rb);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {                                                       // the buffer's sums are in registers
          if constexpr (PAIR) mbar_arrive_cluster(empty0 + buf * 8);
          else mbar_arrive(&acc_empty[h * 2 + buf]);
        }
        if (active) f8_add<32>(acc + 64, ra, f1);
        const bool more = kb + 1 < kb1 && (ok = arrived(it + 1)) && active;
        const uint32_t nb = trow + (buf ^ 1u) * 256;
        if (more) tc_ld32(nb, ra);
        if (active) f8_add<32>(acc + 96, rb, f1);
        if (more) tc_ld32(nb + 32, rb);
      }
      if constexpr (!PAIR) {
        // ---- an item split among the cluster's CTAs (this one's last): the sums take the operands' place in shared memory, CTA r goes on with everybody's
        // of its part of the rows, added up in the order of the CTAs
        if (kb1 - kb0 < KB) {
          mbar_wait(mma_done, 0, a.err, kErrFp8Mma);                          // no MMA reads the operands any more
          float4* mine = reinterpret_cast<float4*>(sm) + h * 128 + row;        // [four columns][half][row]
          if (active) {
#pragma unroll
            for (int c = 0; c < 128; c += 4) mine[c * 64] = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
          }
          __syncwarp();
          cluster_sync_all();
          // all eight warps add up, four columns of a row at a time, and put the sum in the place of this CTA's own
          const int rs = 128 / (int)sch.split, r0 = (int)cluster_rank() * rs, lr = 31 - __clz(rs);
          if (r0 < rows) {
#pragma unroll 1
            for (int u0 = threadIdx.x; u0 < 64 * rs; u0 += 4 * 256) {          // [four columns][half][row], four under way at a time
              uint32_t at[4]; float4 v[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int u = u0 + 256 * i;
                at[i] = (uint32_t)(((u >> lr) << 7) + r0 + (u & (rs - 1))) * 16u; v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
              }
#pragma unroll 1
              for (uint32_t cc = 0; cc < sch.split; ++cc) {
                const uint32_t from = mapa_u32(base, cc);
                float4 t[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] = ld_cluster(from + at[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) { v[i].x += t[i].x; v[i].y += t[i].y; v[i].z += t[i].z; v[i].w += t[i].w; }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(sm + at[i]) = v[i];
            }
          }
          named_bar_sync(1, 256);
          active = active && 32 * q / rs == (int)cluster_rank(); valid = valid && active;
          if (active) {
#pragma unroll
            for (int c = 0; c < 128; c += 4) { const float4 v = mine[c * 64]; acc[c] = v.x; acc[c + 1] = v.y; acc[c + 2] = v.z; acc[c + 3] = v.w; }
          }
        }
      } else if (kb1 - kb0 < KB) {
        // ---- an item that other pairs have parts of: leave the sums, the last one to arrive goes on with everybody's
        const uint32_t st0 = (uint32_t)item * (uint32_t)KB, c_first = sch.owner(st0), c_last = sch.owner(st0 + KB - 1);
        // a part: [column][half][row]; a pair's first run is its part 0
        auto part_of = [&](uint32_t c, uint32_t st) { return a.part + ((size_t)(C::CTAS * c + rank) * 2 + (c == c_first && st != st0 ? 1 : 0)) * (256 * 128) + h * 128 + row; };
        float* mine = part_of(sch.me, sch.start(sch.me));
        if (active && HB_BOUND(a.err, (size_t)(mine - a.part) + 127 * 256 < a.room, 0x802u, mine - a.part)) {
#pragma unroll
          for (int c = 0; c < 128; ++c) __stcg(mine + c * 256, acc[c]);
        }
        named_bar_sync(1, 256);
        if (threadIdx.x == 0 && !ok) *last = 0u;
        else if (threadIdx.x == 0) {
          __threadfence();                                                     // everybody's sums are out before this CTA is counted
          unsigned int* count = a.count + C::CTAS * c_first + rank;
          const bool all = atomicAdd(count, 1u) == c_last - c_first;
          if (all) *count = 0u;                                                // zero again for the next launch
          __threadfence();
          *last = all;
        }
        named_bar_sync(1, 256);
        const bool mine_to_end = *last != 0u;
        named_bar_sync(1, 256);                                                // the flag has been read: the next item may write it
        if (!mine_to_end) continue;
#pragma unroll
        for (int c = 0; c < 128; ++c) acc[c] = 0.f;
        const float* first = part_of(c_first, sch.start(c_first));
        const float* rest = part_of(c_first, st0);                             // the later pairs' parts are their first ones
        if (active) {
          for (uint32_t cc = c_first; cc <= c_last; ++cc) {
            const float* p = cc == c_first ? first : rest + (size_t)(cc - c_first) * (C::CTAS * 2 * 256 * 128);
#pragma unroll
            for (int g = 0; g < 128; g += 64) {
              float t[64];
#pragma unroll
              for (int c = 0; c < 64; ++c) t[c] = __ldcg(p + (g + c) * 256);
#pragma unroll
              for (int c = 0; c < 64; ++c) acc[g + c] += t[c];
            }
          }
        }
      }
      // ---- the item's results
      if constexpr (MODE == F8_GU) {
        uint32_t mx = 0u;
        if (active) {
#pragma unroll
          for (int c = 0; c < 64; ++c) { acc[c] = f8_swiglu(acc[c], acc[64 + c], a.limit); mx = max(mx, f8_mag(acc[c])); }
        }
        amx[h * 128 + row] = mx;
        named_bar_sync(1, 256);
        F8Block blk;
        const float sc = blk.init(max(amx[row], amx[128 + row]));
        if (valid && ok) {
          uint8_t* to = a.yq + (slot0 + row) * a.N + nt * 128 + h * 64;
#pragma unroll
          for (int c = 0; c < 64; c += 16) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = blk.pair(acc[c + 4 * j], acc[c + 4 * j + 1]) | blk.pair(acc[c + 4 * j + 2], acc[c + 4 * j + 3]) << 16;
            *reinterpret_cast<uint4*>(to + c) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (h == 0) a.ys[(size_t)nt * a.ldys + slot0 + row] = sc;
        }
        named_bar_sync(1, 256);                                                // the magnitudes have been read
      } else if (active && ok) {
        uint8_t* stg = sm + C::ST * C::STAGE + (size_t)warp * F8_STG_BYTES;
        const int nrow = min(32, rows - 32 * q), n0 = nt * 256 + h * 128;
        const size_t row0 = slot0 + 32 * q;
        if (MODE == F8_DOWN || (MODE == F8_PLAIN && a.yb)) {
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stg + lane * F8_STG_PITCH + 16 * j) = f8_pack8(&acc[c + 8 * j]);
            f8_flush(stg, reinterpret_cast<uint8_t*>(a.yb + row0 * a.ldy + n0 + c), (size_t)a.ldy * 2, nrow, min(a.N - n0 - c, 32) * 2, lane);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 128; c += 16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(stg + lane * F8_STG_PITCH + 16 * j) = make_float4(acc[c + 4 * j], acc[c + 4 * j + 1], acc[c + 4 * j + 2], acc[c + 4 * j + 3]);
            f8_flush(stg, reinterpret_cast<uint8_t*>(a.yf + row0 * a.ldy + n0 + c), (size_t)a.ldy * 4, nrow, min(a.N - n0 - c, 16) * 4, lane);
          }
        }
      }
    }
  }
  __syncwarp();
  bool splits = false;
  if constexpr (!PAIR) splits = sch.splits();
  if (splits && warp >= 8) cluster_sync_all();                                 // the sums are in shared memory
  if (warp == F8_W_TMA) mbar_wait(mma_done, 0, a.err, kErrFp8Mma);            // in both CTAs: the last MMA has retired, and so has the announcement of it
  tc_fence_before();
  __syncthreads();
  if (PAIR || splits) cluster_sync_all();                                      // nobody reads this CTA's shared memory any more
  if (warp == F8_W_MMA) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc2(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

}  // namespace hb
