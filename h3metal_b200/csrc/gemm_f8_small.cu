// Block-scaled e4m3 product for few rows: C[m][n] = sum_g sa[g][m] * sw[n / 128][g] * P_g[m][n] (+ bias[n]),
// P_g[m][n] = sum over the 128 channels of group g of A[m][k] * W[n][k].
//
// The tensor core multiplies codes and accumulates a group in fp32; the scales differ from group to group, so every
// group's P_g leaves tensor memory on its own and is added, scaled, to running sums that stay in fp32 registers: one
// fused multiply-add per output and group, no rounding to fewer bits before the end.
//
// Few rows mean that the weights are all the traffic. So the WEIGHTS take the wide side of the instruction: a tile is
// 128 rows of W (MMA M = 128, one TMEM lane and one epilogue thread per output channel) by NT rows of A (MMA N = NT,
// 16 to 128), and K is split over the CTAs of a cluster (2 to 8) until the GPU has enough copies in flight to draw
// the weights at full bandwidth. The parts meet in shared memory of the cluster: CTA r adds the S partial sums of its
// share of the rows in the order of their ranks, so that the result does not depend on who finished first.
//
// Roles: warp 0 TMA producer (W tile 16 KB and NT x 128 bytes of A per group), warp 1 MMA issuer, warps 2.. epilogue,
// four lane quarters x parts of up to 32 rows of A. Out-of-range rows and channels are zero-filled by TMA. All waits
// are bounded. No load uses multicast.
//
// What bounds it: HBM for few rows. In a chain of launches whose weights rotate through 354 MB, so that each comes from HBM
// (44.3 MB of DRAM reads per launch counted): 1 x 11520 x 3840 10.2 us = 4.3 TB/s, 16 x 3840 x 10240 10.3 us; with the
// weights of the launch before in L2 8.9 and 8.6 us. What is not the weights' way is the first tile's latency (1.3 us), the two
// cluster barriers and the exit. For 64 and more rows the one issuing thread: two barrier polls, four instructions and a
// commit take 600 to 850 cycles per group.
#include <cuda.h>

#include "gemm_common.cuh"

namespace h3b {
namespace {

using namespace gemm;

constexpr int kWRows = 128;                     // weight rows per tile = MMA M = one scale block of W
constexpr int kWBytes = kWRows * kBKBytes;      // 16 KB
constexpr int kSmallBars = 512;
constexpr int kSmallMaxStages = 12;
constexpr int kMaxSplit = 8;                    // CTAs of a cluster that share K
constexpr int kPrefetchGroups = 4;

template <int NT> struct Small {
  static constexpr int kStage = kWBytes + NT * kBKBytes;
  static constexpr int kEpiWarps = NT <= 32 ? 4 : NT / 8;    // four lane quarters x parts of up to 32 rows of A
  static constexpr int kRows = NT / (kEpiWarps / 4);         // rows of A (accumulator columns) per epilogue thread
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kBufs = 4;                            // accumulators in tensor memory, at most
  static constexpr int kCols = NT * kBufs;                   // 64 .. 512
  static constexpr int kScaleBytes = kEpiWarps * 2 * kRows * 4;  // two slots per epilogue warp
  static constexpr int kPerSm = NT <= 32 ? 3 : NT <= 64 ? 2 : 1; // CTAs an SM can hold (registers, tensor memory)
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
__global__ void __launch_bounds__(Small<NT>::kThreads, Small<NT>::kPerSm)
gemm_f8_small_kernel(const __grid_constant__ GemmF8Launch g, const int stages, const int bufs) {
  using S = Small<NT>;
  constexpr int kRows = S::kRows;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t *base_ptr = smem_raw + (base - raw_addr);
  const uint32_t bars_off = stages * S::kStage;
  const uint32_t bars = base + bars_off;
  auto full_bar = [&](int i) { return bars + 8u * i; };
  auto done_bar = [&](int i) { return bars + 128u + 8u * i; };
  auto acc_empty_bar = [&](int i) { return bars + 256u + 8u * i; };
  volatile uint32_t *tmem_holder = reinterpret_cast<volatile uint32_t *>(base_ptr + bars_off + 288);
  volatile int *cta_abort = reinterpret_cast<volatile int *>(base_ptr + bars_off + 292);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = g.split;
  const int rank = static_cast<int>(cluster_cta_rank());
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
      mbar_init(done_bar(i), 1);  // one commit per use: the stage may be refilled, the accumulator read
    }
    for (int i = 0; i < bufs; ++i) mbar_init(acc_empty_bar(i), S::kEpiWarps);
    *cta_abort = 0;
    fence_barrier_init();
  }
  if (warp == 2 && lane == 0) {
    // The weights' way from HBM into L2 may start while the kernel before still runs: 0.5 us on each of a chain of
    // products (1 x 11520 x 3840: 10.3 -> 9.7). Eight groups gain no more than four.
    const int ahead = min(g_end, g_begin + kPrefetchGroups);
    for (int kb = g_begin; kb < ahead; ++kb) tma_prefetch_2d(&g.map_w, kb * kBKBytes, n0);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_holder)), S::kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncwarp();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  grid_dep_launch();
  grid_dep_wait();  // global memory is read and written from here on only

  const int quarter = warp & 3, part = (warp - 2) >> 2;  // epilogue warps: TMEM lanes and rows of A
  const int row = quarter * 32 + lane, n = n0 + row;     // their output channel
  float acc[kRows];                                      // its running sums for rows m0 + part * kRows ..
  if (warp == 0) {
    if (lane == 0) {
      RingPos pos;
      uint32_t filled = 0;
      for (int kb = g_begin; kb < g_end; ++kb) {
        const uint32_t s = pos.s;
        if (!mbar_wait(done_bar(s), pos.ph ^ 1u, cta_abort, g.status, kStatusProducerTimeout)) break;
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
      bool issued = false;
      for (int kb = g_begin; kb < g_end; ++kb) {
        const uint32_t s = pos.s;
        // two polls in flight at once: a barrier's answer takes about 80 cycles, a third of the instructions' own issue
        const bool full = mbar_test(full_bar(s), pos.ph), free = mbar_test(acc_empty_bar(buf.s), buf.ph ^ 1u);
        if (!full && !mbar_wait(full_bar(s), pos.ph, cta_abort, g.status, kStatusMmaTimeout)) break;
        if (!free && !mbar_wait(acc_empty_bar(buf.s), buf.ph ^ 1u, cta_abort, g.status, kStatusMmaTimeout)) break;
        tc_fence_after_sync();
        const uint64_t wd = wd0 + static_cast<uint64_t>(s * (S::kStage >> 4));
        const uint64_t ad = ad0 + static_cast<uint64_t>(s * (S::kStage >> 4));
        const uint32_t d = tmem_base + buf.s * NT;
#pragma unroll
        for (int k = 0; k < kBKBytes / 32; ++k) umma_f8(d, wd + 2u * k, ad + 2u * k, idesc, k ? 1u : 0u);
        umma_commit(done_bar(s));
        pos.advance(stages);
        buf.advance(bufs);
        issued = true;
      }
      if (*cta_abort && issued) {  // instructions still in flight must finish before tensor memory is given up
        pos.retreat(stages);
        int dummy_abort = 0;
        mbar_wait(done_bar(pos.s), pos.ph, &dummy_abort, g.status, kStatusDrainTimeout, kDrainLimitCycles);
      }
    }
  } else {
    float *slots = reinterpret_cast<float *>(base_ptr + bars_off + kSmallBars) + (warp - 2) * 2 * kRows;
    const float *sw_p = g.sw + static_cast<size_t>(n_blk) * g.sw_stride;
    // Lane t of the warp fetches the scale of its t-th row of A two or four groups ahead; the product with the weight
    // block's scale goes through a slot of shared memory to all lanes. Rows past the end read another row's scale:
    // their sums are zeros (TMA fills their codes with them) and are not stored.
    const int t = part * kRows + lane;
    const float *sa_p = g.sa + (lane < kRows && m0 + t < g.M ? m0 + t : m0);
#pragma unroll
    for (int j = 0; j < kRows; ++j) acc[j] = 0.0f;
    // Unrolled over the fetches in flight, so that a scale stays in the register that its load wrote: moving it on would
    // wait for the load.
    constexpr int kAhead = kRows == 16 ? 4 : 2;  // even: consecutive groups alternate between the slots
    float a_s[kAhead], w_s[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool have = g_begin + u < g_end;
      a_s[u] = have ? ld_f32(sa_p + static_cast<size_t>(g_begin + u) * g.sa_stride) : 0.0f;
      w_s[u] = have ? ld_f32(sw_p + g_begin + u) : 0.0f;
    }
    RingPos pos, buf;
    bool ok = true;
    for (int kb0 = g_begin; ok && kb0 < g_end; kb0 += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int kb = kb0 + u;
        if (kb >= g_end) break;
        float *slot = slots + (u & 1) * kRows;
        if (lane < kRows) slot[lane] = __fmul_rn(a_s[u], w_s[u]);
        if (kb + kAhead < g_end) {
          a_s[u] = ld_f32(sa_p + static_cast<size_t>(kb + kAhead) * g.sa_stride);
          w_s[u] = ld_f32(sw_p + kb + kAhead);
        }
        __syncwarp();  // this slot is written, and every lane is done with the other one
        ok = mbar_wait(done_bar(pos.s), pos.ph, cta_abort, g.status, kStatusEpilogueTimeout);
        ok = __all_sync(0xFFFFFFFFu, ok);  // a warp gives up as a whole
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf.s * NT + part * kRows;
        uint32_t p[kRows];
        if constexpr (kRows == 16) tmem_ld_32x32b_x16(t_acc, p);
        else tmem_ld_32x32b_x32(t_acc, p);
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty_bar(buf.s));
#pragma unroll
        for (int j = 0; j < kRows; j += 4) {
          const float4 s = *reinterpret_cast<const float4 *>(slot + j);
          acc[j] = __fmaf_rn(__uint_as_float(p[j]), s.x, acc[j]);
          acc[j + 1] = __fmaf_rn(__uint_as_float(p[j + 1]), s.y, acc[j + 1]);
          acc[j + 2] = __fmaf_rn(__uint_as_float(p[j + 2]), s.z, acc[j + 2]);
          acc[j + 3] = __fmaf_rn(__uint_as_float(p[j + 3]), s.w, acc[j + 3]);
        }
        pos.advance(stages);
        buf.advance(bufs);
      }
    }
  }

  const float bias = warp >= 2 && g.bias != nullptr && n < g.N ? ld_f32(g.bias + n) : 0.0f;
  // Every copy has landed and every MMA has read it (the last group has been waited for by all epilogue warps before
  // any of them can pass the barrier below), so tensor memory can go and the ring holds the partial sums: [row of
  // A][128]
  float *sums = reinterpret_cast<float *>(base_ptr);
  tc_fence_before_sync();
  __syncwarp();  // warps 0 and 1 come from loops that lane 0 ran alone
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, S::kCols);
  }
  if (warp >= 2) {
#pragma unroll
    for (int j = 0; j < kRows; ++j) sums[(part * kRows + j) * kWRows + row] = acc[j];
  }
  cluster_sync_all();
  if (warp >= 2 && n < g.N && !*cta_abort) {
    // this CTA finishes the rows t = rank, rank + split, ..: its epilogue warps take them in turn
    const int rows_here = min(NT, g.M - m0);
    for (int t = rank + split * part; t < rows_here; t += split * (S::kEpiWarps / 4)) {
      float part_sum[kMaxSplit], sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kMaxSplit; ++q)
        part_sum[q] = q < split ? ld_cluster_f32(map_to_cta(base + (t * kWRows + row) * 4, q)) : 0.0f;
#pragma unroll
      for (int q = 0; q < kMaxSplit; ++q) sum = __fadd_rn(sum, part_sum[q]);
      store_one(g, m0 + t, n, __fadd_rn(sum, bias));
    }
  }
  cluster_sync_all();  // nobody leaves while its sums are still being read
}

template <int NT>
cudaError_t launch_nt(const GemmF8Launch &g, int sms, cudaStream_t stream) {
  using S = Small<NT>;
  cudaLaunchConfig_t cfg = {};
  const unsigned grid = static_cast<unsigned>((g.N + kWRows - 1) / kWRows) * g.m_tiles * g.split;
  // Ring depth: what is left of an SM's 228 KB for each of the CTAs that share it, and no more than there are groups.
  const int want = static_cast<int>((grid + sms - 1) / sms);
  // Room for a second CTA even where one per SM would do: a cluster lies inside a GPC, and clusters of eight CTAs that
  // take a whole SM each do not pack (24 x 2048 x 8192 in 8 parts, 128 CTAs: 13.5 us, with room for two CTAs to an SM 7.7).
  const int per_sm = want >= S::kPerSm ? S::kPerSm : want < 2 && S::kPerSm > 1 ? 2 : want;
  const int fixed = 1024 + kSmallBars + S::kScaleBytes;
  const int room = 233472 / per_sm - 1024;  // the runtime keeps 1 KB per CTA
  int stages = (room - fixed) / S::kStage;
  const int groups = ((g.K + kBKBytes - 1) / kBKBytes + g.split - 1) / g.split;
  if (stages > groups) stages = groups;
  if (stages > kSmallMaxStages) stages = kSmallMaxStages;
  const int for_sums = (NT * kWRows * 4 + S::kStage - 1) / S::kStage;  // the ring also holds the partial sums
  if (stages < for_sums) stages = for_sums;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(S::kThreads);
  // Never more CTAs on an SM than its 512 columns of tensor memory serve: a CTA that waits for columns while its
  // cluster waits for it could otherwise close a circle with another cluster.
  const size_t needed = fixed + static_cast<size_t>(stages) * S::kStage, least = 233472 / (512 / S::kCols + 1);
  cfg.dynamicSmemBytes = needed > least ? needed : least;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = g.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g.overlap ? 2 : 1;
  // A stage's barrier tells its uses apart by their parity alone. The epilogue, which waits on it too, must therefore
  // be less than a whole ring behind the MMAs, and it can be as many groups behind as there are accumulators.
  const int bufs = stages < S::kBufs ? stages : S::kBufs;
  return cudaLaunchKernelEx(&cfg, gemm_f8_small_kernel<NT>, g, stages, bufs);
}

}  // namespace

// Which kernel, and for few rows which tile height and how many CTAs share K. Times in nanoseconds, measured on B200
// as back-to-back launches. All follow
//   launch + (groups a CTA works through) * (time of a group),
// a group taking 0.5 us on 128-row tiles here, where every wave of CTAs starts anew, and 0.45 us on pairs; two pairs
// that share K pay 1.5 us to meet, and take one tile per cluster. M x N x K: here / a pair / two pairs, us: 256 x 3840
// x 3840: 15.2 / 17.4 / 13.8; 512 x 3840 x 10240: 42.4 / 37.8 / 26.8; 128 x 3840 x 3840: 10.4 / 17 / 13.6; 128 x 20480
// x 3840: 44.6 / 33.2; 512 x 20480 x 3840: 97 / 47. Over nine M of 1 to 640 and seven N x K the choice is within 2 % of
// the best; larger products were not swept.
bool gemm_f8_choose(GemmF8Launch &g, int sms, const F8Clusters &resident) {
  const long long groups = (g.K + kBKBytes - 1) / kBKBytes;
  const long long n_tiles = (static_cast<long long>(g.N) + kWRows - 1) / kWRows;
  g.nt = g.M <= 16 ? 16 : g.M <= 32 ? 32 : g.M <= 64 ? 64 : 128;
  g.m_tiles = (g.M - 1) / g.nt + 1;
  const long long tiles = n_tiles * g.m_tiles;
  // K is split two ways at least, and on while the parts still run side by side: 1 x 11520 x 3840 takes 11.6 / 10.3 /
  // 13.7 us with 2 / 4 / 8 parts (90 tiles, three CTAs to an SM), 16 x 3840 x 10240 18.6 / 12.3 / 10.7 (30 tiles).
  // 128-row tiles have an SM each, and what fits is a matter of whole clusters.
  const int per_sm = g.nt <= 32 ? 3 : g.nt <= 64 ? 2 : 1;
  g.split = 2;
  int room = 0;  // clusters of g.split that run side by side
  for (int i = 0; i < 3; ++i) {
    const int split = 2 << i;
    const int fits = per_sm == 1 ? resident.rows128[i] : sms * per_sm / split;
    if (i > 0 && (tiles >= sms || tiles > fits || split > groups)) break;
    g.split = split;
    room = fits;
  }
  const bool can_split = groups >= 2 && room > 0;
  if (can_split && g.nt < 128) return false;
  const long long waves = room > 0 ? (tiles + room - 1) / room : 0;
  const long long here = 2000 + waves * (4500 + (groups + g.split - 1) / g.split * 500);
  const long long pair_tiles = ((g.M - 1LL) / 256 + 1) * ((g.N - 1LL) / 256 + 1);
  const long long one = 5000 + (pair_tiles + resident.pairs - 1) / resident.pairs * groups * 450;
  const long long two = groups >= 4 && pair_tiles <= resident.twos ? 6500 + (groups + 1) / 2 * 450 : one;
  if (can_split && here <= one && here <= two) return false;
  g.split = two < one ? 2 : 1;
  return true;
}

cudaError_t gemm_f8_small_configure(int rows128[3]) {
  cudaError_t e;
#define H3B_F8_CFG(NT)                                                                                               \
  e = cudaFuncSetAttribute(gemm_f8_small_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);           \
  if (e != cudaSuccess) return e;
  H3B_F8_CFG(16) H3B_F8_CFG(32) H3B_F8_CFG(64) H3B_F8_CFG(128)
#undef H3B_F8_CFG
  for (int i = 0; i < 3; ++i) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 << i);
    cfg.blockDim = dim3(Small<128>::kThreads);
    cfg.dynamicSmemBytes = 232448;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2 << i; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if ((e = cudaOccupancyMaxActiveClusters(&rows128[i], gemm_f8_small_kernel<128>, &cfg)) != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_gemm_f8_small(const GemmF8Launch &g, int sms, cudaStream_t stream) {
  switch (g.nt) {
    case 16: return launch_nt<16>(g, sms, stream);
    case 32: return launch_nt<32>(g, sms, stream);
    case 64: return launch_nt<64>(g, sms, stream);
    default: return launch_nt<128>(g, sms, stream);
  }
}

}  // namespace h3b
