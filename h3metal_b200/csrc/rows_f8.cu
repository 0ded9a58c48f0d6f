// Rows as e4m3 codes with one fp32 scale per 128 channels: the producers of gemm_f8's activations.
//
//   rms_f8     h = x (+ y), rounded to x's type and kept;  v = h * rsqrt(mean(h^2) + eps) * w
//   quant_f8   v = x,  or  v = x[:, :D] * silu(x[:, D:2D])
//   both       s[g][m] = max(amax over the group |v| / 448, 2^-126), 1 where the group is all zero;  code = e4m3(v * (1 / s))
//
// 448 is the largest finite e4m3 value. The floor 2^-126 keeps 1 / s finite: groups whose largest magnitude is below
// 448 * 2^-126 lose their smallest codes instead of turning into 0 * inf. Codes are the nearest e4m3 value (ties to
// even) of v * (1 / s): two roundings of 2^-24 each away from v / s, which matters only to values within 2^-23 of the
// middle between two codes - to which both codes are equally near. A NaN keeps its own place (code 0x7F) and the group's scale comes from the
// other values; an infinity makes the scale infinite, and the group NaN when it is read back. Sums, statistics and
// scales are fp32. The stream h is rounded to x's type BEFORE it is normed, as if the addition had been a call of its
// own: what is normed is what the next layer adds to.
//
// A thread owns a piece of 16 channels (one 16-byte store of codes), eight neighbouring lanes a group of 128: the
// group's largest magnitude is three shuffles. Both kernels are bound by memory: 1 byte written per channel beside
// the 2 to 10 read and kept. Measured as a chain of launches over more than L2 holds (the measured copy rate is 6.55 TB/s):
// quant_f8 17408 x 16384 gated, 1.43 GB in 208 us = 6.9 TB/s (222 us called one by one from Python), 17408 x 6144 plain
// 52 us = 6.2 TB/s; rms_f8 17408 x 6144 with a bf16 stream and addend 118 us = 6.4 TB/s, with an fp32 stream 209 us = 5.6,
// 4608 x 3840 24 us = 5.2 (a tenth of it launch and first rows), bf16 without an addend 69 us = 4.7 and fp32 83 us = 6.5
// (the chain of a row's sum shows where there are few bytes). Where registers do not reach the row loop spills: two fp32
// inputs (172 bytes of spill stores; 17408 x 6144 258 us = 5.4 TB/s), and D of 8193 to 16384 with an addend, where 1024
// threads leave 64 each (192 to 356 bytes; 4096 x 16384: bf16 88 us = 5.4, fp32 stream 126 us = 5.9, both fp32 204 us = 4.3);
// beyond, rows of four pieces per thread without the next row on its way (4096 x 32768 bf16 228 us = 4.1).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "kernels.h"
#include "ptx.cuh"

namespace h3b {
namespace {

constexpr int kPiece = 16;    // channels per thread
constexpr int kGroup = 128;   // channels per scale
constexpr float kTop = 448.0f;
constexpr float kTiny = 1.17549435e-38f;  // 2^-126

// Sixteen consecutive values of type T as they lie in memory: two per 32-bit word, or one.
template <typename T>
struct Raw {
  static constexpr int kWords = kPiece * sizeof(T) / 4;
  uint32_t w[kWords];
  // The first n values at p (n >= 1); the others read as 0. align: 16-byte or 32-byte boundary of p, else any. A
  // piece of 16-bit values is ONE 32-byte access: with two of 16 bytes, each touches every second half of the warp's
  // cache lines.
  __device__ __forceinline__ void load(const T *p, int n, int align) {
    if (align >= 32 && n >= kPiece) {
#pragma unroll
      for (int q = 0; q < kWords / 8; ++q)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[8 * q]), "=r"(w[8 * q + 1]), "=r"(w[8 * q + 2]), "=r"(w[8 * q + 3]), "=r"(w[8 * q + 4]),
                       "=r"(w[8 * q + 5]), "=r"(w[8 * q + 6]), "=r"(w[8 * q + 7])
                     : "l"(reinterpret_cast<const uint32_t *>(p) + 8 * q)
                     : "memory");
    } else if (align >= 16 && n >= kPiece) {
#pragma unroll
      for (int q = 0; q < kWords / 4; ++q) {
        const uint4 u = reinterpret_cast<const uint4 *>(p)[q];
        w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        if (i >= n) continue;
        if constexpr (sizeof(T) == 4) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
        else w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[i]) << (16 * (i & 1));
      }
    }
  }
  __device__ __forceinline__ void store(T *p, int n, int align) const {
    if (align >= 32 && n >= kPiece) {
#pragma unroll
      for (int q = 0; q < kWords / 8; ++q)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t *>(p) + 8 * q),
                     "r"(w[8 * q]), "r"(w[8 * q + 1]), "r"(w[8 * q + 2]), "r"(w[8 * q + 3]), "r"(w[8 * q + 4]),
                     "r"(w[8 * q + 5]), "r"(w[8 * q + 6]), "r"(w[8 * q + 7])
                     : "memory");
    } else if (n >= kPiece) {
#pragma unroll
      for (int q = 0; q < kWords / 4; ++q)
        reinterpret_cast<uint4 *>(p)[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        if (i >= n) continue;
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t *>(p)[i] = w[i];
        else reinterpret_cast<uint16_t *>(p)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
      }
    }
  }
  // Values 2 i and 2 i + 1, exactly. All arithmetic below works on such pairs (packed fp32 instructions: half the
  // issue slots, each half rounded like the scalar operation): the kernels are otherwise bound by issue.
  __device__ __forceinline__ float2 get(int i) const {
    if constexpr (std::is_same<T, float>::value) {
      return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if constexpr (std::is_same<T, __half>::value) {
      __half2 h;
      memcpy(&h, &w[i], 4);
      return __half22float2(h);
    } else {
      return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
  }
  __device__ __forceinline__ void set(int i, float2 v) {
    if constexpr (std::is_same<T, float>::value) {
      w[2 * i] = __float_as_uint(v.x);
      w[2 * i + 1] = __float_as_uint(v.y);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(v.x, v.y);
      memcpy(&w[i], &h, 4);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
      memcpy(&w[i], &h, 4);
    }
  }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The scale of a group and the codes of this thread's piece. Called by the eight lanes of a group together; lanes past
// the end of the row pass zeros and n <= 0.
__device__ __forceinline__ void encode_piece(const float2 (&v)[kPiece / 2], int n, uint8_t *dst, float *scale, bool first) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kPiece / 2; ++i) top = fmaxf(top, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
#pragma unroll
  for (int s = 1; s < 8; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
  const float sc = top > 0.0f ? fmaxf(__fdiv_rn(top, kTop), kTiny) : 1.0f;
  const float rs = __fdiv_rn(1.0f, sc);
  if (first) *scale = sc;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(__fmul2_rn(v[2 * j], both(rs)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(__fmul2_rn(v[2 * j + 1], both(rs)), __NV_SATFINITE, __NV_E4M3);
    w[j] = lo | (hi << 16);
  }
  if (n >= kPiece) {
    *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      if (i < n) dst[i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
  }
}

// g / (1 + e^-g) for two gates, e^-g as 2^(-g log2 e). Relative error: the exponent's rounding, |g| * 2^-24 at most
// (|g| < 104; beyond, e^-g is 0 or infinite), ex2 2^-22, rcp 2^-23, the other four roundings 2^-24 each. The
// denominator is formed at a sixteenth, so that its reciprocal is never subnormal (ex2 and rcp flush those); the last
// product may be.
__device__ __forceinline__ float2 silu(float2 g) {
  const float2 h = __fmul2_rn(g, both(-1.44269504f));
  float2 e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(h.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(h.y));
  const float2 d = __ffma2_rn(e, both(0.0625f), both(0.0625f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  return __fmul2_rn(g, __fmul2_rn(r, both(0.0625f)));
}

// ---- quantiser: no statistics over the row. A CTA covers blockDim.y rows (or part of one row, gridDim.y parts) --------
struct QuantArgs {
  const void *x;
  uint8_t *out;
  float *sa;
  long long x_stride, out_stride, sa_stride;
  int M, D;
  int x_align, gate_align;  // boundaries on which the rows and their gates start: 32 or 16 bytes, or (gates) any
};

template <typename T, bool GATED>
__global__ void __launch_bounds__(256) quant_f8_kernel(const QuantArgs p) {
  grid_dep_launch();
  grid_dep_wait();
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  const long long m = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int n = m < p.M ? p.D - piece * kPiece : 0;  // values of this piece that exist
  float2 v[kPiece / 2];
  if (n > 0) {
    const T *row = static_cast<const T *>(p.x) + m * p.x_stride + piece * kPiece;
    Raw<T> x, g;
    x.load(row, n, p.x_align);
    if (GATED) g.load(row + p.D, n, p.gate_align);
#pragma unroll
    for (int i = 0; i < kPiece / 2; ++i) {
      v[i] = x.get(i);
      if (GATED) v[i] = __fmul2_rn(v[i], silu(g.get(i)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPiece / 2; ++i) v[i] = both(0.0f);
  }
  const int group = piece >> 3;
  encode_piece(v, n, p.out + m * p.out_stride + piece * kPiece, p.sa + group * p.sa_stride + m, n > 0 && (piece & 7) == 0);
}

// ---- norm: a CTA has a row at a time, C pieces per thread ---------------------------------------------------------
struct RmsArgs {
  const void *x, *y, *w;
  void *res;
  uint8_t *out;
  float *sa;
  long long x_stride, y_stride, res_stride, out_stride, sa_stride;
  int M, D, w_dtype, x_align, y_align, res_align, w_align;
  float eps;
};

struct None {};

template <typename T>
__device__ __forceinline__ void read_gain(float2 (&g)[kPiece / 2], const void *w, int at, int n, int align) {
  Raw<T> raw;
  raw.load(static_cast<const T *>(w) + at, n, align);
#pragma unroll
  for (int i = 0; i < kPiece / 2; ++i) g[i] = raw.get(i);
}

// blockDim.x threads have a row, blockDim.y rows go side by side. Where a thread has one piece, the row that comes
// next is on its way while the current one is normed (x and y in registers, as they lie in memory), and the gain
// stays in registers: read for every row, fp32 gains kept the L1 pipeline 73 % busy. Registers decide how many rows
// an SM holds: 80 keep two CTAs of 384 threads (17408 x 6144: 119 us; with the 87 the compiler takes unasked, one
// CTA, 168).
template <typename TX, typename TY, int C, int WARPS>
__global__ void __maxnreg__(WARPS == 32 ? 64 : C == 1 ? 80 : 128) rms_f8_kernel(const RmsArgs p) {
  __shared__ alignas(16) float part[2][WARPS];  // the warps' sums of squares, zeros for warps that do not exist
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool one_warp = blockDim.x == 32;
  constexpr bool kAdd = !std::is_same<TY, None>::value;
  using Y = std::conditional_t<kAdd, TY, TX>;
  Raw<TX> x;
  Raw<Y> y;
  auto fetch = [&](long long m, int c) {
    const int at = (threadIdx.x + c * blockDim.x) * kPiece, n = p.D - at;
    if (n <= 0 || m >= p.M) return;
    x.load(static_cast<const TX *>(p.x) + m * p.x_stride + at, n, p.x_align);
    if constexpr (kAdd) y.load(static_cast<const TY *>(p.y) + m * p.y_stride + at, n, p.y_align);
  };
  auto gain_of = [&](int c, float2 (&g)[kPiece / 2]) {
    const int at = (threadIdx.x + c * blockDim.x) * kPiece, n = p.D - at;
    if (n <= 0) return;
    if (p.w_dtype == kDtypeF32) read_gain<float>(g, p.w, at, n, p.w_align);
    else if (p.w_dtype == kDtypeBf16) read_gain<__nv_bfloat16>(g, p.w, at, n, p.w_align);
    else read_gain<__half>(g, p.w, at, n, p.w_align);
  };
  if (!one_warp) {
    for (int i = threadIdx.x; i < 2 * WARPS; i += blockDim.x) part[0][i] = 0.0f;  // blockDim.y is 1
    __syncthreads();
  }
  float2 gain[kPiece / 2] = {};
  const long long step = static_cast<long long>(gridDim.x) * blockDim.y;
  long long m = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if constexpr (C == 1) {
    fetch(m, 0);
    gain_of(0, gain);
  }
  // the same trips for all threads of a row; only rows that are alone in their CTA meet a barrier
  for (int turn = 0; m < p.M; m += step, turn ^= 1) {
    float2 v[C][kPiece / 2];
    float2 ss2 = both(0.0f);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = (threadIdx.x + c * blockDim.x) * kPiece, n = p.D - at;
      if constexpr (C > 1) fetch(m, c);
#pragma unroll
      for (int i = 0; i < kPiece / 2; ++i) v[c][i] = both(0.0f);
      if (n > 0) {
        if constexpr (kAdd) {
#pragma unroll
          for (int i = 0; i < kPiece / 2; ++i) x.set(i, __fadd2_rn(x.get(i), y.get(i)));
          x.store(static_cast<TX *>(p.res) + m * p.res_stride + at, n, p.res_align);
        }
#pragma unroll
        for (int i = 0; i < kPiece / 2; ++i) v[c][i] = x.get(i);
      }
#pragma unroll
      for (int i = 0; i < kPiece / 2; ++i) ss2 = __ffma2_rn(v[c][i], v[c][i], ss2);
    }
    if constexpr (C == 1) fetch(m + step, 0);
    float ss = __fadd_rn(ss2.x, ss2.y);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xFFFFFFFFu, ss, s));
    if (!one_warp) {  // two sets of partial sums: the next row's cannot meet a warp that still reads this row's
      if (lane == 0) part[turn][warp] = ss;
      __syncthreads();
      float2 sum = both(0.0f);
#pragma unroll
      for (int i = 0; i < WARPS / 4; ++i) {
        const float4 q = reinterpret_cast<const float4 *>(part[turn])[i];
        sum = __fadd2_rn(sum, __fadd2_rn(make_float2(q.x, q.y), make_float2(q.z, q.w)));
      }
      ss = __fadd_rn(sum.x, sum.y);
    }
    const float inv = __frsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(p.D)), p.eps));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int piece = threadIdx.x + c * blockDim.x, at = piece * kPiece, n = p.D - at;
      if constexpr (C > 1) gain_of(c, gain);
#pragma unroll
      for (int i = 0; i < kPiece / 2; ++i) v[c][i] = __fmul2_rn(__fmul2_rn(v[c][i], both(inv)), gain[i]);
      const int group = piece >> 3;
      encode_piece(v[c], n, p.out + m * p.out_stride + at, p.sa + group * p.sa_stride + m,
                   (piece & 7) == 0 && group * kGroup < p.D);
    }
  }
}

template <typename F, typename... Args>
cudaError_t launch(F *kernel, dim3 grid, dim3 threads, bool overlap, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = threads;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// 32, 16 or 1: the boundary on which every row of a tensor starts
int boundary(const void *p, long long row_bytes) {
  const unsigned long long bits = reinterpret_cast<uintptr_t>(p) | static_cast<unsigned long long>(row_bytes);
  return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 1;
}

// CTAs of this kernel that an SM holds at once, asked once per CTA size.
template <typename TX, typename TY, int C, int WARPS>
int rms_resident(unsigned threads) {
  static std::atomic<int> known[WARPS + 1];
  int n = known[threads / 32].load(std::memory_order_relaxed);
  if (n == 0) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, rms_f8_kernel<TX, TY, C, WARPS>,
                                                                        static_cast<int>(threads), 0);
    if (e != cudaSuccess || n < 1) n = 1;
    known[threads / 32].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <typename TX, typename TY, int C, int WARPS>
cudaError_t launch_rms_c(RmsArgs a, int pieces, int sms, bool overlap, cudaStream_t stream) {
  const unsigned tx = ((pieces + C - 1) / C + 31) / 32 * 32;
  const unsigned ty = tx == 32 ? 4 : 1;  // rows of up to 512 channels: a warp each, four to a CTA
  a.x_align = boundary(a.x, a.x_stride * sizeof(TX));
  a.w_align = boundary(a.w, 0);
  if constexpr (!std::is_same<TY, None>::value) {
    a.y_align = boundary(a.y, a.y_stride * sizeof(TY));
    a.res_align = boundary(a.res, a.res_stride * sizeof(TX));
  }
  const int resident = sms * rms_resident<TX, TY, C, WARPS>(tx * ty), wanted = (a.M - 1) / static_cast<int>(ty) + 1;
  return launch(rms_f8_kernel<TX, TY, C, WARPS>, dim3(wanted < resident ? wanted : resident), dim3(tx, ty), overlap, stream, a);
}

template <typename TX, typename TY>
cudaError_t launch_rms(const RmsArgs &a, int sms, bool overlap, cudaStream_t stream) {
  const int pieces = (a.D + kGroup - 1) / kGroup * (kGroup / kPiece);
  if (pieces <= 512) return launch_rms_c<TX, TY, 1, 16>(a, pieces, sms, overlap, stream);
  if (pieces <= 1024) return launch_rms_c<TX, TY, 1, 32>(a, pieces, sms, overlap, stream);
  return launch_rms_c<TX, TY, 4, 16>(a, pieces, sms, overlap, stream);
}

template <typename TX>
cudaError_t launch_rms_y(const RmsArgs &a, int y_dtype, int sms, bool overlap, cudaStream_t stream) {
  if (!a.y) return launch_rms<TX, None>(a, sms, overlap, stream);
  if (y_dtype == kDtypeF32) return launch_rms<TX, float>(a, sms, overlap, stream);
  if (y_dtype == kDtypeF16) return launch_rms<TX, __half>(a, sms, overlap, stream);
  return launch_rms<TX, __nv_bfloat16>(a, sms, overlap, stream);
}

template <typename T>
cudaError_t launch_quant(const QuantF8Launch &q, bool overlap, cudaStream_t stream) {
  QuantArgs a;
  a.x = q.x; a.out = static_cast<uint8_t *>(q.out); a.sa = q.sa;
  a.x_stride = q.x_stride; a.out_stride = q.out_stride; a.sa_stride = q.sa_stride; a.M = q.M; a.D = q.D;
  a.x_align = boundary(q.x, q.x_stride * sizeof(T));
  a.gate_align = boundary(static_cast<const T *>(q.x) + q.D, q.x_stride * sizeof(T));
  // About 256 threads: parts of a row of equal length, or several short rows. Whole warps, whole groups of eight lanes.
  const int pieces = (q.D + kGroup - 1) / kGroup * (kGroup / kPiece);
  const int parts = (pieces + 255) / 256;
  int tx = (pieces + parts - 1) / parts, ty = 1;
  if (tx <= 64) {
    tx = (tx + 7) / 8 * 8;
    ty = 256 / tx / 4 * 4;
  } else {
    tx = (tx + 31) / 32 * 32;
    ty = 256 / tx;
  }
  const dim3 grid((q.M - 1) / ty + 1, (pieces + tx - 1) / tx), threads(tx, ty);
  if (q.gated) return launch(quant_f8_kernel<T, true>, grid, threads, overlap, stream, a);
  return launch(quant_f8_kernel<T, false>, grid, threads, overlap, stream, a);
}

}  // namespace

cudaError_t launch_quant_f8(const QuantF8Launch &q, bool overlap, cudaStream_t stream) {
  if (q.x_dtype == kDtypeF32) return launch_quant<float>(q, overlap, stream);
  if (q.x_dtype == kDtypeF16) return launch_quant<__half>(q, overlap, stream);
  return launch_quant<__nv_bfloat16>(q, overlap, stream);
}

cudaError_t launch_rms_f8(const RmsF8Launch &r, int sms, bool overlap, cudaStream_t stream) {
  RmsArgs a;
  a.x = r.x; a.y = r.y; a.w = r.w; a.res = r.res; a.out = static_cast<uint8_t *>(r.out); a.sa = r.sa;
  a.x_stride = r.x_stride; a.y_stride = r.y_stride; a.res_stride = r.res_stride; a.out_stride = r.out_stride;
  a.sa_stride = r.sa_stride; a.M = r.M; a.D = r.D; a.w_dtype = r.w_dtype; a.eps = r.eps;
  if (r.x_dtype == kDtypeF32) return launch_rms_y<float>(a, r.y_dtype, sms, overlap, stream);
  if (r.x_dtype == kDtypeF16) return launch_rms_y<__half>(a, r.y_dtype, sms, overlap, stream);
  return launch_rms_y<__nv_bfloat16>(a, r.y_dtype, sms, overlap, stream);
}

}  // namespace h3b
