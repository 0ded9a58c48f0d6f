// Block-scaled e4m3 product for few rows: C[m][n] = sum_g sa[g][m] * sw[n / 128][g] * P_g[m][n] (+ bias[n]),
// P_g[m][n] = sum over the 128 channels of group g of A[m][k] * W[n][k].
//
// The tensor core multiplies codes and accumulates a group in fp32; the scales differ from group to group, so every
// group's P_g leaves tensor memory on its own and is added, scaled, to running sums that stay in fp32 registers:
// one fused multiply-add per output and group, no rounding to fewer bits before the end.
//
// Few rows mean that the weights are all the traffic. So the WEIGHTS take the wide side of the instruction: a tile is 128
// rows of W (MMA M = 128, one TMEM lane and one epilogue thread per output channel) by NT rows of A (MMA N = NT, 16
// to 128), and K is split over the CTAs of a cluster (1 to 8) until the GPU has enough copies in flight to draw the
// weights at full bandwidth. The parts meet in shared memory of the cluster: CTA r adds the S partial sums of its
// share of the rows in the order of their ranks, so that the result does not depend on who finished first.
//
// Roles: warp 0 TMA producer (W tile 16 KB and NT x 128 bytes of A per group), warp 1 MMA issuer, warps 2..5 epilogue.
// Out-of-range rows and channels are zero-filled by TMA. All waits are bounded. No load uses multicast.
#include <cuda.h>

#include "gemm_common.cuh"

namespace h3b {
namespace {

using namespace gemm;

constexpr int kWRows = 128;                     // weight rows per tile = MMA M = one scale block of W
constexpr int kWBytes = kWRows * kBKBytes;      // 16 KB
constexpr int kScaleSlots = 4;                  // groups whose activation scales are on their way
constexpr int kSmallBars = 256;

template <int NT> struct Small {
  static constexpr int kStage = kWBytes + NT * kBKBytes;
  static constexpr int kBufs = NT <= 64 ? 4 : 2;             // accumulators in tensor memory
  static constexpr int kCols = NT * kBufs;                   // 64, 128, 256, 256
  static constexpr int kScaleBytes = 4 * kScaleSlots * NT * 4;  // per epilogue warp
};

// fp32 value of the other CTA's shared memory
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void store_one(const GemmF8Launch &g, int m, int n, float v) {
  const size_t at = static_cast<size_t>(m) * g.c_stride + n;
  if (g.c_dtype == kDtypeBf16) static_cast<__nv_bfloat16 *>(g.c)[at] = __float2bfloat16_rn(v);
  else if (g.c_dtype == kDtypeF16) static_cast<__half *>(g.c)[at] = __float2half_rn(v);
  else static_cast<float *>(g.c)[at] = v;
}

template <int NT>
__global__ void __launch_bounds__(192, NT <= 16 ? 3 : NT <= 64 ? 2 : 1)
gemm_f8_small_kernel(const __grid_constant__ GemmF8Launch g, const int stages) {
  using S = Small<NT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t *base_ptr = smem_raw + (base - raw_addr);
  const uint32_t bars_off = stages * S::kStage;
  const uint32_t bars = base + bars_off;
  auto full_bar = [&](int i) { return bars + 8u * i; };
  auto empty_bar = [&](int i) { return bars + 64u + 8u * i; };
  auto acc_full_bar = [&](int i) { return bars + 128u + 8u * i; };
  auto acc_empty_bar = [&](int i) { return bars + 160u + 8u * i; };
  volatile uint32_t *tmem_holder = reinterpret_cast<volatile uint32_t *>(base_ptr + bars_off + 192);
  volatile int *cta_abort = reinterpret_cast<volatile int *>(base_ptr + bars_off + 196);
  const uint32_t scales_off = bars_off + kSmallBars;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = g.split;
  const int rank = split > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int tile = blockIdx.x / split;
  const int n_blk = tile / g.m_tiles, m_blk = tile % g.m_tiles;  // tiles of the same weights are neighbours
  const int n0 = n_blk * kWRows, m0 = m_blk * NT;
  const int groups = (g.K + kBKBytes - 1) / kBKBytes;
  const int g_begin = static_cast<int>(static_cast<long long>(groups) * rank / split);
  const int g_end = static_cast<int>(static_cast<long long>(groups) * (rank + 1) / split);

  if (warp == 0 && lane == 0) {
    tma_prefetch_descriptor(&g.map_a);
    tma_prefetch_descriptor(&g.map_w);
    for (int i = 0; i < stages; ++i) {
      mbar_init(full_bar(i), 1);
      mbar_init(empty_bar(i), 1);
    }
    for (int i = 0; i < S::kBufs; ++i) {
      mbar_init(acc_full_bar(i), 1);
      mbar_init(acc_empty_bar(i), 4);
    }
    *cta_abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_holder)), S::kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  grid_dep_launch();
  grid_dep_wait();  // global memory is read and written from here on only

  float acc[NT];  // epilogue threads: running sums of output channel n0 + row for NT rows of A
  if (warp == 0) {
    if (lane == 0) {
      RingPos pos;
      uint32_t filled = 0;
      for (int kb = g_begin; kb < g_end; ++kb) {
        const uint32_t s = pos.s;
        if (!mbar_wait(empty_bar(s), pos.ph ^ 1u, cta_abort, g.status, kStatusProducerTimeout)) break;
        mbar_arrive_expect_tx(full_bar(s), S::kStage);
        const uint32_t dst = base + s * S::kStage;
        tma_load_2d(dst, &g.map_w, full_bar(s), kb * kBKBytes, n0);
        tma_load_2d(dst + kWBytes, &g.map_a, full_bar(s), kb * kBKBytes, m0);
        pos.advance(stages);
        filled += filled < static_cast<uint32_t>(stages);
      }
      if (*cta_abort) {  // copies still in flight must land before this CTA's shared memory is given up
        for (uint32_t j = 0; j < filled; ++j) {
          pos.retreat(stages);
          int dummy_abort = 0;
          mbar_wait(full_bar(pos.s), pos.ph, &dummy_abort, g.status, kStatusDrainTimeout, kDrainLimitCycles);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_instr_desc(1, 0, kWRows, NT);  // f32 accumulate, e4m3 x e4m3
      const uint64_t wd0 = umma_smem_desc(base, 1024, 2);
      const uint64_t ad0 = umma_smem_desc(base + kWBytes, 1024, 2);
      RingPos pos, buf;
      for (int kb = g_begin; kb < g_end; ++kb) {
        if (!mbar_wait(acc_empty_bar(buf.s), buf.ph ^ 1u, cta_abort, g.status, kStatusMmaTimeout)) break;
        const uint32_t s = pos.s;
        if (!mbar_wait(full_bar(s), pos.ph, cta_abort, g.status, kStatusMmaTimeout)) break;
        tc_fence_after_sync();
        const uint64_t wd = wd0 + static_cast<uint64_t>(s * (S::kStage >> 4));
        const uint64_t ad = ad0 + static_cast<uint64_t>(s * (S::kStage >> 4));
        const uint32_t d = tmem_base + buf.s * NT;
#pragma unroll
        for (int k = 0; k < kBKBytes / 32; ++k) umma_f8(d, wd + 2u * k, ad + 2u * k, idesc, k ? 1u : 0u);
        umma_commit(empty_bar(s));
        umma_commit(acc_full_bar(buf.s));
        pos.advance(stages);
        buf.advance(S::kBufs);
      }
    }
  } else {
    const int quarter = warp & 3;
    float *my_scales = reinterpret_cast<float *>(base_ptr + scales_off) + (warp - 2) * kScaleSlots * NT;
    const uint32_t my_scales_addr = base + scales_off + (warp - 2) * kScaleSlots * NT * 4;
    const float *sw_row = g.sw + static_cast<size_t>(n_blk) * g.sw_stride;
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = 0.0f;
    // the activation scales of group kb on their way to this warp's slot; rows past the end read as 0
    auto fetch = [&](int kb) {
      if (kb < g_end) {
#pragma unroll
        for (int t = lane; t < NT; t += 32) {
          const bool ok = m0 + t < g.M;
          cp_async_4(my_scales_addr + ((kb & (kScaleSlots - 1)) * NT + t) * 4,
                     g.sa + static_cast<size_t>(kb) * g.sa_stride + (ok ? m0 + t : 0), ok);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kScaleSlots - 1; ++i) fetch(g_begin + i);
    float ws = __ldg(sw_row + g_begin);
    RingPos buf;
    for (int kb = g_begin; kb < g_end; ++kb) {
      __syncwarp();  // every lane is done with the slot that is filled next
      fetch(kb + kScaleSlots - 1);
      const float ws_next = kb + 1 < g_end ? __ldg(sw_row + kb + 1) : 0.0f;
      cp_async_wait<kScaleSlots - 1>();
      __syncwarp();
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(acc_full_bar(buf.s), buf.ph, cta_abort, g.status, kStatusEpilogueTimeout))) break;
      tc_fence_after_sync();
      const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf.s * NT;
      const float *s4 = my_scales + (kb & (kScaleSlots - 1)) * NT;
      constexpr int kChunk = NT < 32 ? 16 : 32;
#pragma unroll
      for (int c = 0; c < NT; c += kChunk) {
        uint32_t p[kChunk];
        if constexpr (kChunk == 16) tmem_ld_32x32b_x16(t_acc + c, p);
        else tmem_ld_32x32b_x32(t_acc + c, p);
        tmem_ld_wait();
        if (c + kChunk == NT) {  // the group's last values are in registers
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty_bar(buf.s));
        }
#pragma unroll
        for (int j = 0; j < kChunk; j += 4) {
          const float4 s = *reinterpret_cast<const float4 *>(s4 + c + j);
          acc[c + j] = __fmaf_rn(__uint_as_float(p[j]), __fmul_rn(s.x, ws), acc[c + j]);
          acc[c + j + 1] = __fmaf_rn(__uint_as_float(p[j + 1]), __fmul_rn(s.y, ws), acc[c + j + 1]);
          acc[c + j + 2] = __fmaf_rn(__uint_as_float(p[j + 2]), __fmul_rn(s.z, ws), acc[c + j + 2]);
          acc[c + j + 3] = __fmaf_rn(__uint_as_float(p[j + 3]), __fmul_rn(s.w, ws), acc[c + j + 3]);
        }
      }
      ws = ws_next;
      buf.advance(S::kBufs);
    }
    cp_async_wait<0>();
  }

  const int row = (warp & 3) * 32 + lane, n = n0 + row;  // epilogue threads: their output channel
  const float bias = warp >= 2 && g.bias != nullptr && n < g.N ? __ldg(g.bias + n) : 0.0f;
  if (split == 1) {
    if (warp >= 2 && n < g.N && !*cta_abort) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (m0 + t < g.M) store_one(g, m0 + t, n, __fadd_rn(acc[t], bias));
    }
  } else {
    // every copy has landed and every MMA has read it (the last group's accumulator has been waited for, by all four
    // epilogue warps before any of them can pass the barrier below), so the ring holds the partial sums: [row of A][128]
    float *part = reinterpret_cast<float *>(base_ptr);
    __syncthreads();
    if (warp >= 2) {
#pragma unroll
      for (int t = 0; t < NT; ++t) part[t * kWRows + row] = acc[t];
    }
    cluster_sync_all();
    if (warp >= 2 && n < g.N && !*cta_abort) {
      const int t_begin = NT * rank / split, t_end = NT * (rank + 1) / split;
      for (int t = t_begin; t < t_end && m0 + t < g.M; ++t) {
        float sum = 0.0f;
        for (int q = 0; q < split; ++q)
          sum = __fadd_rn(sum, ld_cluster_f32(map_to_cta(base + (t * kWRows + row) * 4, q)));
        store_one(g, m0 + t, n, __fadd_rn(sum, bias));
      }
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are still being read
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, S::kCols);
  }
}

template <int NT>
cudaError_t launch_nt(const GemmF8Launch &g, int stages, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const int n_tiles = (g.N + kWRows - 1) / kWRows;
  cfg.gridDim = dim3(static_cast<unsigned>(n_tiles) * g.m_tiles * g.split);
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = 1024 + static_cast<size_t>(stages) * Small<NT>::kStage + kSmallBars + Small<NT>::kScaleBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = g.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g.overlap ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, gemm_f8_small_kernel<NT>, g, stages);
}

}  // namespace

cudaError_t gemm_f8_small_configure() {
  cudaError_t e;
#define H3B_F8_CFG(NT)                                                                                                   \
  if ((e = cudaFuncSetAttribute(gemm_f8_small_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448)) != cudaSuccess) \
    return e;
  H3B_F8_CFG(16) H3B_F8_CFG(32) H3B_F8_CFG(64) H3B_F8_CFG(128)
#undef H3B_F8_CFG
  return cudaSuccess;
}

cudaError_t launch_gemm_f8_small(const GemmF8Launch &g, cudaStream_t stream) {
  // ring depth: three, two or one CTA per SM share its 227 KB
  switch (g.nt) {
    case 16: return launch_nt<16>(g, 4, stream);
    case 32: return launch_nt<32>(g, 5, stream);
    case 64: return launch_nt<64>(g, 4, stream);
    default: return launch_nt<128>(g, 6, stream);
  }
}

}  // namespace h3b
