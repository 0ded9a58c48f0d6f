// Block-scaled e4m3 product on CTA pairs: C tile 256 x 256 per cluster of two CTAs, tcgen05.mma cta_group::2.
//
//   C[m][n] = sum_g sa[g][m] * sw[n / 128][g] * P_g[m][n] (+ bias[n]),   P_g = the group's 128 channels of A W^T
//
// As in gemm_f8_small.cu a group's P_g (four instructions of 32 channels, fp32 in tensor memory) is added, scaled, to
// running sums in fp32 registers. An epilogue thread owns one row of the tile and 128 of its columns - exactly the
// columns of one weight block, so that the scale of a group is ONE number per thread, sa * sw - and 128 running sums.
//
// What bounds it: a group's MMAs take 512 cycles; reading it out of tensor memory, 128 x 256 values per SM, and the
// multiply-adds (two columns per packed instruction) take about 250 each, beside the MMAs of the next group, for
// which there is a second accumulator of 256 columns. An accumulator goes round (MMAs done -> both epilogues -> leader), and
// a group takes 860 to 900 cycles, with no pipe near its limit: latency somewhere in that round, where is not
// measured. Messages between the two SMs are not all of it, since single CTAs, which send none, are no faster. Measured, back
// to back under the board's power cap: 17408 x 18432 x 6144 in 1.87 to 1.91 ms = 2.06 to 2.10 PFLOP/s at 1.46 GHz, 9.7 of
// 16.4 kflop per clock and SM (60 %); three launches from idle 2.39 PFLOP/s. With an epilogue that only hands accumulators
// back: 2.24; without its multiply-adds: 2.27. Not taken: three accumulators of 160 columns (2.48 against 1.96 ms:
// more bytes per multiply, and the issuing thread's four instructions and commit per group no longer hide), MMAs of
// 128 columns into four accumulators (+17 %: A is read twice from shared memory), single CTAs on 128 x 256 tiles (+10
// %, half as many more bytes), sixteen epilogue warps (+10 %).
//
// Roles per CTA (rank 0 of a pair = leader): warp 0 TMA producer (own 128 rows of A, own half of the 256 rows of W
// per group, bytes of both CTAs counted on the leader's barrier), warp 1 of the leader issues the MMAs, warps 2 and 3
// idle, warps 4..11 epilogue: four lane quarters x two halves of 128 columns; the first four warps hand them most of
// their registers. One commit per group says both that the stage may be refilled and that the accumulator may be
// read. 16-bit results are staged in shared memory as 128-byte-swizzled panels and stored by TMA while the next tile
// runs; fp32 results and unaligned outputs are turned there and stored row by row. Set-up overlaps the kernel before
// (programmatic stream serialization). All waits are bounded. No load uses multicast.
#include <cuda.h>

#include "gemm_common.cuh"

namespace h3b {
namespace {

using namespace gemm;

constexpr int kF8BN = 256;
constexpr int kF8Stage = kABytes + 128 * kBKBytes;  // 32 KB: this CTA's rows of A and its half of W
constexpr int kF8EpiWarps = 8;
constexpr int kF8Cols = kF8BN / (kF8EpiWarps / 4);  // columns per epilogue thread: 128, those of one weight block
constexpr int kF8Threads = 128 + 32 * kF8EpiWarps;
// Registers per thread after the split: 128 x 104 + 256 x 200 = 64512 = 384 x 168, what the launch was
// given. Neither side spills with these; 56 and 224 make the issuing warps spill and cost 6 % of the whole product.
constexpr int kF8RegsIssue = 104, kF8RegsEpi = 200;
constexpr int kF8OutWarp = 2 * kOutPanel;           // a warp's 32 rows x 128 two-byte columns
constexpr int kF8MailWarp = 32 * 128 * 4;           // a warp's 32 x 128 fp32 sums

// SPLIT 1: a pair has the whole of K, eight warps stage results. SPLIT 2: two pairs of a cluster have half of K each
// for ONE tile per cluster; four warps of each stage results and receive the other pair's sums.
template <int SPLIT> struct PairShape {
  static constexpr int kStages = SPLIT == 1 ? 5 : 4;
  static constexpr int kMailOff = kStages * kF8Stage;
  static constexpr int kOutOff = kMailOff + (SPLIT == 1 ? 0 : 4 * kF8MailWarp);
  static constexpr int kBarsOff = kOutOff + (SPLIT == 1 ? 8 : 4) * kF8OutWarp;
  static constexpr size_t kSmem = 1024 + kBarsOff + kBarrierBytes;
  static_assert(kSmem <= 232448, "ring, mail and staging share 227 KB");
};

// acc += p * s for 16 columns, two at a time
__device__ __forceinline__ void scale_add16(const uint32_t (&p)[16], float2 s2, float2 *acc) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    acc[j] = __ffma2_rn(make_float2(__uint_as_float(p[2 * j]), __uint_as_float(p[2 * j + 1])), s2, acc[j]);
}

// 32 columns of a warp's 32 rows, from (m, n) on, without TMA: turned in 4 KB of shared memory (piece p of row r sits at
// p ^ (r & 7)) so that a store instruction writes whole rows. A thread's own row, stored as it lies in registers, would
// touch 32 lines per instruction: 575 against 204 us at 4608 x 11520 x 3840.
__device__ __forceinline__ void store_chunk(const GemmF8Launch &g, float *buf, int lane, const float (&v)[32], int m, int n) {
  __syncwarp();  // the chunk before has been read
#pragma unroll
  for (int q = 0; q < 8; ++q)
    reinterpret_cast<float4 *>(buf)[lane * 8 + (q ^ (lane & 7))] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  __syncwarp();
  if (g.c_dtype == kDtypeF32 && n + 32 <= g.N && reinterpret_cast<uintptr_t>(g.c) % 16 == 0 && g.c_stride % 4 == 0) {
    const int q = lane & 7;
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // four rows per instruction
      const int r = 4 * i + (lane >> 3);
      const float4 x = reinterpret_cast<const float4 *>(buf)[r * 8 + (q ^ (r & 7))];
      float *dst = static_cast<float *>(g.c) + static_cast<size_t>(m + r) * g.c_stride + n + 4 * q;
      if (m + r < g.M) *reinterpret_cast<float4 *>(dst) = x;
    }
  } else if (n + lane < g.N) {
    const int rows = min(32, g.M - m);
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
      const float x = buf[(r * 8 + ((lane >> 2) ^ (r & 7))) * 4 + (lane & 3)];
      const size_t at = static_cast<size_t>(m + r) * g.c_stride + n + lane;
      if (g.c_dtype == kDtypeF32) static_cast<float *>(g.c)[at] = x;
      else if (g.c_dtype == kDtypeBf16) static_cast<__nv_bfloat16 *>(g.c)[at] = __float2bfloat16_rn(x);
      else static_cast<__half *>(g.c)[at] = __float2half_rn(x);
    }
  }
}

// STAGED: 16-bit results by TMA (g.map_c). A kernel of its own, because the other way out costs the main loop registers.
template <bool STAGED, int SPLIT>
__global__ void __cluster_dims__(2 * SPLIT, 1, 1) __launch_bounds__(kF8Threads, 1)
gemm_f8_pair_kernel(const __grid_constant__ GemmF8Launch g) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t *base_ptr = smem_raw + (base - raw_addr);
  // [ring][mail: 64 KB, split only][staging of results][barriers 256 B]
  using P = PairShape<SPLIT>;
  constexpr int stages = P::kStages;
  constexpr uint32_t bars_off = P::kBarsOff;
  const uint32_t bars = base + bars_off;
  auto full_bar = [&](int i) { return bars + 8u * i; };
  auto done_bar = [&](int i) { return bars + 64u + 8u * i; };
  auto acc_empty_bar = [&](int i) { return bars + 128u + 8u * i; };
  volatile uint32_t *tmem_holder = reinterpret_cast<volatile uint32_t *>(base_ptr + bars_off + 176);
  volatile int *cta_abort = reinterpret_cast<volatile int *>(base_ptr + bars_off + 180);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_cta_rank(), rank = cta & 1u;  // rank in the pair
  const int pair = SPLIT == 1 ? 0 : static_cast<int>(cta >> 1);
  const uint32_t leader_cta = cta & ~1u;
  const bool leader = rank == 0;
  const int n_tiles = (g.N + kF8BN - 1) / kF8BN;
  const int num_tiles = g.m_tiles * n_tiles;
  const int all_groups = (g.K + kBKBytes - 1) / kBKBytes;
  const int g_begin = all_groups * pair / SPLIT, groups = all_groups * (pair + 1) / SPLIT - g_begin;
  const int first_tile = cluster_id_x(), tile_step = SPLIT == 1 ? static_cast<int>(cluster_count_x()) : num_tiles;

  if (warp == 0 && lane == 0) {
    tma_prefetch_descriptor(&g.map_a);
    tma_prefetch_descriptor(&g.map_w);
    if (STAGED) tma_prefetch_descriptor(&g.map_c);
    for (int i = 0; i < stages; ++i) {
      mbar_init(full_bar(i), 1);  // the leader's producer arms it; bytes arrive from both CTAs
      mbar_init(done_bar(i), 1);  // one commit arrival per use
    }
    for (int i = 0; i < 2; ++i) mbar_init(acc_empty_bar(i), 2 * kF8EpiWarps);
    *cta_abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(const_cast<uint32_t *>(tmem_holder)), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  grid_dep_launch();
  grid_dep_wait();  // global memory is read and written from here on only

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kF8RegsIssue));
    if (warp == 0) {
      if (lane == 0) {
        RingPos pos;
        uint32_t filled = 0;  // stages filled so far, saturating at `stages` (for the wind-down)
        const uint32_t leader_full0 = map_to_cta(full_bar(0), leader_cta);
        bool ok = true;
        for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
          const TileCoord tc = tile_coord(tile, g.m_tiles, n_tiles, g.band);
          const int m0 = tc.m_blk * 256 + static_cast<int>(rank) * 128;
          const int n0 = tc.n_blk * kF8BN + static_cast<int>(rank) * 128;
          for (int kb = 0; kb < groups; ++kb) {
            const uint32_t s = pos.s;
            ok = mbar_wait(done_bar(s), pos.ph ^ 1u, cta_abort, g.status, kStatusProducerTimeout);
            if (!ok) break;
            if (leader) mbar_arrive_expect_tx(full_bar(s), 2u * kF8Stage);
            const uint32_t leader_full = leader_full0 + 8u * s;
            const uint32_t dst = base + s * kF8Stage;
            tma_load_2d_pair(dst, &g.map_a, leader_full, (g_begin + kb) * kBKBytes, m0);
            tma_load_2d_pair(dst + kABytes, &g.map_w, leader_full, (g_begin + kb) * kBKBytes, n0);
            pos.advance(stages);
            filled += filled < static_cast<uint32_t>(stages);
          }
        }
        if (*cta_abort && leader) {
          // wind-down after a timeout: the pair's copies into the last stages filled are counted on the leader's full
          // barriers; wait (bounded) for them so that neither CTA leaves with copies still landing in its shared memory
          for (uint32_t j = 0; j < filled; ++j) {
            pos.retreat(stages);
            int dummy_abort = 0;
            mbar_wait(full_bar(pos.s), pos.ph, &dummy_abort, g.status, kStatusDrainTimeout, kDrainLimitCycles);
          }
        }
      }
    } else if (warp == 1) {
      if (leader && lane == 0) {
        constexpr uint32_t idesc = umma_instr_desc(1, 0, 256, kF8BN);  // f32 accumulate, e4m3 x e4m3, M 256 over the pair
        const uint64_t ad0 = umma_smem_desc(base, 1024, 2);
        const uint64_t bd0 = umma_smem_desc(base + kABytes, 1024, 2);
        RingPos pos, buf;
        bool ok = true, issued = false;
        for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
          for (int kb = 0; kb < groups; ++kb) {
            const uint32_t s = pos.s;
            const bool full = mbar_test(full_bar(s), pos.ph), free = mbar_test(acc_empty_bar(buf.s), buf.ph ^ 1u);
            ok = full || mbar_wait(full_bar(s), pos.ph, cta_abort, g.status, kStatusMmaTimeout);
            if (!ok) break;
            ok = free || mbar_wait(acc_empty_bar(buf.s), buf.ph ^ 1u, cta_abort, g.status, kStatusMmaTimeout);
            if (!ok) break;
            tc_fence_after_sync();
            const uint64_t ad = ad0 + static_cast<uint64_t>(s * (kF8Stage >> 4));
            const uint64_t bd = bd0 + static_cast<uint64_t>(s * (kF8Stage >> 4));
            const uint32_t d = tmem_base + buf.s * kF8BN;
#pragma unroll
            for (int k = 0; k < kBKBytes / 32; ++k) umma_f8_pair(d, ad + 2u * k, bd + 2u * k, idesc, k ? 1u : 0u);
            umma_commit_pair(done_bar(s), static_cast<uint16_t>(3u << leader_cta));
            pos.advance(stages);
            buf.advance(2);
            issued = true;
          }
        }
        if (*cta_abort && issued) {
          // wind-down after a timeout: the last instructions issued must be done with both CTAs' shared and tensor memory
          // before either gives them up
          pos.retreat(stages);
          int dummy_abort = 0;
          mbar_wait(done_bar(pos.s), pos.ph, &dummy_abort, g.status, kStatusDrainTimeout, kDrainLimitCycles);
        }
      }
    }
    if (SPLIT > 1) {  // the barrier between the pairs' sums (see the epilogue)
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kF8RegsEpi));
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    const int row = quarter * 32 + lane;
    const int n_blocks = (g.N + 127) / 128;
    const uint32_t leader_acc_empty0 = map_to_cta(acc_empty_bar(0), leader_cta);
    RingPos pos;
    uint32_t buf = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
      const TileCoord tc = tile_coord(tile, g.m_tiles, n_tiles, g.band);
      const int m0 = tc.m_blk * 256 + static_cast<int>(rank) * 128, n0 = tc.n_blk * kF8BN + part * kF8Cols;
      const int m = m0 + row;
      // rows and columns past the end compute zeros (TMA fills their codes with them) and are not stored: any scale
      // will do
      const int m_s = min(m, g.M - 1), n_s = min(n0 / 128, n_blocks - 1);
      float2 acc[kF8Cols / 2];
#pragma unroll
      for (int j = 0; j < kF8Cols / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
      // the next group's scales are fetched while this group's are waited for and used
      float a_s = ld_f32(g.sa + static_cast<size_t>(g_begin) * g.sa_stride + m_s);
      float w_s = ld_f32(g.sw + static_cast<size_t>(n_s) * g.sw_stride + g_begin);
#pragma unroll 1
      for (int kb = 0; kb < groups; ++kb) {
        const float s = __fmul_rn(a_s, w_s);
        if (kb + 1 < groups) {
          a_s = ld_f32(g.sa + static_cast<size_t>(g_begin + kb + 1) * g.sa_stride + m_s);
          w_s = ld_f32(g.sw + static_cast<size_t>(n_s) * g.sw_stride + g_begin + kb + 1);
        }
        ok = mbar_wait(done_bar(pos.s), pos.ph, cta_abort, g.status, kStatusEpilogueTimeout);
        ok = __all_sync(0xFFFFFFFFu, ok);  // a warp gives up as a whole
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * kF8BN + part * kF8Cols;
        const float2 s2 = make_float2(s, s);
        // two register sets: the next 16 columns are on their way while these are added
        uint32_t p[2][16];
        tmem_ld_32x32b_x16(t_acc, p[0]);
#pragma unroll
        for (int c = 0; c < kF8Cols / 16; ++c) {
          tmem_ld_wait();
          if (c + 1 < kF8Cols / 16) tmem_ld_32x32b_x16(t_acc + (c + 1) * 16, p[(c + 1) & 1]);
          else {  // the warp's last values of the group are in registers: the leader may overwrite them
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(leader_acc_empty0 + 8u * buf);
          }
          scale_add16(p[c & 1], s2, acc + c * 8);
        }
        pos.advance(stages);
        buf ^= 1u;
      }
      if constexpr (SPLIT > 1) {
        // Each pair finishes one column half: the warps of the other half leave their sums with the same warp quarter
        // of the other pair's CTA with the same rows, 16 bytes per lane at [piece of four columns][lane]. A cluster
        // has one tile, so the two barriers of the cluster, here and at the end, are all it takes; a warp that gave
        // up meets them too.
        if (ok && part != pair) {
          const uint32_t dst = map_to_cta(base + P::kMailOff + quarter * kF8MailWarp + lane * 16, cta ^ 2u);
#pragma unroll
          for (int q = 0; q < kF8Cols / 4; ++q)
            st_cluster_v4(dst + q * 512, acc[2 * q].x, acc[2 * q].y, acc[2 * q + 1].x, acc[2 * q + 1].y);
        }
        cluster_arrive();
        cluster_wait();
        if (part != pair) break;
        if (ok) {
          const float4 *mail = reinterpret_cast<const float4 *>(base_ptr + P::kMailOff + quarter * kF8MailWarp) + lane;
#pragma unroll
          for (int q = 0; q < kF8Cols / 4; ++q) {
            const float4 x = mail[q * 32];
            acc[2 * q] = __fadd2_rn(acc[2 * q], make_float2(x.x, x.y));
            acc[2 * q + 1] = __fadd2_rn(acc[2 * q + 1], make_float2(x.z, x.w));
          }
        }
      }
      if (!ok) break;
      float bias[kF8Cols / 32];
#pragma unroll
      for (int j = 0; j < kF8Cols / 32; ++j) {
        const int n = n0 + j * 32 + lane;
        bias[j] = g.bias != nullptr && n < g.N ? ld_f32(g.bias + n) : 0.0f;
      }
      const int out_warp = SPLIT == 1 ? part * 4 + quarter : quarter;
      uint8_t *out_buf = base_ptr + P::kOutOff + out_warp * kF8OutWarp;
      const uint32_t out_addr = base + P::kOutOff + out_warp * kF8OutWarp;
      if constexpr (STAGED) {  // the panels of the tile before must have been read out of shared memory
        if (lane == 0) tma_store_wait_read();
        __syncwarp();
      }
#pragma unroll
      for (int c = 0; c < kF8Cols / 32; ++c) {
        float v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[2 * j] = acc[c * 16 + j].x;
          v[2 * j + 1] = acc[c * 16 + j].y;
        }
        if (g.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __fadd_rn(v[j], __shfl_sync(0xFFFFFFFFu, bias[c], j));
        }
        if constexpr (STAGED) {
          if (g.c_dtype == kDtypeBf16) stage_out32<__nv_bfloat16>(out_buf, c, lane, v);
          else stage_out32<__half>(out_buf, c, lane, v);
        } else {
          store_chunk(g, reinterpret_cast<float *>(out_buf), lane, v, m0 + quarter * 32, n0 + c * 32);
        }
      }
      if constexpr (STAGED) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          const int y = m0 + quarter * 32;
          if (y < g.M) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (n0 + i * 64 < g.N) tma_store_2d(&g.map_c, out_addr + i * kOutPanel, n0 + i * 64, y);
          }
          tma_store_commit();
        }
      }
    }
    if (STAGED && lane == 0) tma_store_wait_all();
    __syncwarp();
  }

  // Neither CTA may leave while the other can still read its shared memory, signal its barriers or write its TMEM.
  tc_fence_before_sync();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

template <int SPLIT>
cudaError_t configure(int *clusters) {
  constexpr int smem = static_cast<int>(PairShape<SPLIT>::kSmem);
  cudaError_t e = cudaFuncSetAttribute(gemm_f8_pair_kernel<true, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(gemm_f8_pair_kernel<false, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * SPLIT, 1, 1);
  cfg.blockDim = dim3(kF8Threads, 1, 1);
  cfg.dynamicSmemBytes = PairShape<SPLIT>::kSmem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2 * SPLIT; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(clusters, gemm_f8_pair_kernel<true, SPLIT>, &cfg);
}

template <int SPLIT>
cudaError_t launch(const GemmF8Launch &g, int clusters, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * SPLIT * clusters);  // the cluster shape is part of the kernel's declaration
  cfg.blockDim = dim3(kF8Threads);
  cfg.dynamicSmemBytes = PairShape<SPLIT>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g.overlap ? 1 : 0;
  return g.tma_store ? cudaLaunchKernelEx(&cfg, gemm_f8_pair_kernel<true, SPLIT>, g)
                     : cudaLaunchKernelEx(&cfg, gemm_f8_pair_kernel<false, SPLIT>, g);
}

}  // namespace

cudaError_t gemm_f8_pair_configure(int *pairs, int *twos) {
  *pairs = *twos = 0;
  const cudaError_t e = configure<1>(pairs);
  return e != cudaSuccess ? e : configure<2>(twos);
}

cudaError_t launch_gemm_f8_pair(const GemmF8Launch &g, int clusters, cudaStream_t stream) {
  return g.split == 1 ? launch<1>(g, clusters, stream) : launch<2>(g, clusters, stream);
}

}  // namespace h3b
