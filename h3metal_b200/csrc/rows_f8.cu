// Rows as e4m3 codes with one fp32 scale per 128 channels: the producers of gemm_f8's activations.
//
//   rms_f8     h = x (+ y), rounded to x's type and kept;  v = h * rsqrt(mean(h^2) + eps) * w
//   quant_f8   v = x,  or  v = x[:, :D] * silu(x[:, D:2D])
//   both       s[g][m] = max(amax over the group |v| / 448, 2^-126), 1 where the group is all zero;  code = e4m3(v / s)
//
// 448 is the largest finite e4m3 value. The floor 2^-126 keeps 1 / s finite: groups whose largest magnitude is below
// 448 * 2^-126 lose their smallest codes instead of turning into 0 * inf. Codes are the nearest e4m3 value (ties to
// even) of v * (1 / s); the reciprocal is one rounding away from a division, which matters only to values within 2^-23
// of the middle between two codes. A NaN keeps its own place (code 0x7F) and the group's scale comes from the other
// values; an infinity makes the scale infinite, and the group NaN when it is read back.
// Sums, statistics and scales are fp32. The stream h is rounded to x's type BEFORE it is normed, as if the addition had
// been a call of its own: what is normed is what the next layer adds to.
//
// A thread owns a piece of 16 channels (one 16-byte store of codes), eight neighbouring lanes a group of 128: the
// group's largest magnitude is three shuffles. Both kernels are bound by memory: 1 byte written per channel beside
// the 2 to 10 read and kept.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

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

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Sixteen consecutive values at p, of which the first n (>= 1) exist; the others read as 0. vec: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load_piece(const T *p, int n, bool vec, float (&v)[kPiece]) {
  if (vec && n >= kPiece) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < kPiece / kPer; ++q) {
      const uint4 raw = reinterpret_cast<const uint4 *>(p)[q];
      T e[kPer];
      memcpy(e, &raw, 16);
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[q * kPer + i] = to_f32(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store_piece(T *p, int n, const float (&v)[kPiece]) {
  if (n >= kPiece) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < kPiece / kPer; ++q) {
      T e[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) e[i] = from_f32<T>(v[q * kPer + i]);
      uint4 raw;
      memcpy(&raw, e, 16);
      reinterpret_cast<uint4 *>(p)[q] = raw;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}

// The scale of a group and the codes of this thread's piece. Called by the eight lanes of a group together; lanes past
// the end of the row pass zeros and n <= 0.
__device__ __forceinline__ void encode_piece(const float (&v)[kPiece], int n, uint8_t *dst, float *scale, bool first) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kPiece; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
  for (int s = 1; s < 8; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
  const float sc = top > 0.0f ? fmaxf(__fdiv_rn(top, kTop), kTiny) : 1.0f;
  const float rs = __fdiv_rn(1.0f, sc);
  if (first) *scale = sc;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(v[4 * j], rs), __fmul_rn(v[4 * j + 1], rs)),
                                                 __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(v[4 * j + 2], rs), __fmul_rn(v[4 * j + 3], rs)),
                                                 __NV_SATFINITE, __NV_E4M3);
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

// ---- quantiser: no statistics over the row, so a CTA simply takes the next 256 pieces -------------------------------
template <typename T, bool GATED>
__global__ void __launch_bounds__(256) quant_f8_kernel(const T *x, long long x_stride, uint8_t *out, long long out_stride,
                                                       float *sa, long long sa_stride, int M, int D, int per_row,
                                                       bool gate_vec) {
  grid_dep_launch();
  grid_dep_wait();
  // per_row: pieces of a row rounded up to whole groups, so that the lanes of a group stay together
  const long long start = static_cast<long long>(blockIdx.x) * 256;
  const long long m_first = start / per_row;
  const int at = static_cast<int>(start - m_first * per_row) + threadIdx.x;
  const long long m = m_first + at / per_row;
  const int piece = at % per_row;
  const bool have = m < M;
  const int n = have ? D - piece * kPiece : 0;  // values of this piece that exist
  float v[kPiece];
#pragma unroll
  for (int i = 0; i < kPiece; ++i) v[i] = 0.0f;
  if (n > 0) {
    const T *row = x + m * x_stride;
    load_piece(row + piece * kPiece, n, true, v);
    if (GATED) {
      float g[kPiece];
      load_piece(row + D + piece * kPiece, n, gate_vec, g);
#pragma unroll
      for (int i = 0; i < kPiece; ++i)
        v[i] = __fmul_rn(v[i], __fdividef(g[i], __fadd_rn(1.0f, expf(-g[i]))));
    }
  }
  const int group = piece >> 3;
  encode_piece(v, n, out + m * out_stride + piece * kPiece, sa + group * sa_stride + m, have && (piece & 7) == 0);
}

// ---- norm: one CTA per row, C pieces per thread --------------------------------------------------------------------
struct RmsArgs {
  const void *x, *y, *w;
  void *res;
  uint8_t *out;
  float *sa;
  long long x_stride, y_stride, res_stride, out_stride, sa_stride;
  int D, w_dtype;
  float eps;
};

struct None {};

__device__ __forceinline__ void load_gain(const RmsArgs &p, int at, int n, float (&w)[kPiece]) {
  if (p.w_dtype == kDtypeF32) load_piece(static_cast<const float *>(p.w) + at, n, true, w);
  else if (p.w_dtype == kDtypeBf16) load_piece(static_cast<const __nv_bfloat16 *>(p.w) + at, n, true, w);
  else load_piece(static_cast<const __half *>(p.w) + at, n, true, w);
}

template <typename TX, typename TY, int C>
__global__ void __launch_bounds__(512) rms_f8_kernel(const RmsArgs p) {
  __shared__ float part[16];
  grid_dep_launch();
  grid_dep_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const long long m = blockIdx.x;
  constexpr bool kAdd = !std::is_same<TY, None>::value;
  float v[C][kPiece];
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = (tid + c * blockDim.x) * kPiece, n = p.D - at;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) v[c][i] = 0.0f;
    if (n > 0) {
      load_piece(static_cast<const TX *>(p.x) + m * p.x_stride + at, n, true, v[c]);
      if constexpr (kAdd) {
        float y[kPiece];
        load_piece(static_cast<const TY *>(p.y) + m * p.y_stride + at, n, true, y);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) v[c][i] = to_f32(from_f32<TX>(__fadd_rn(v[c][i], y[i])));
        store_piece(static_cast<TX *>(p.res) + m * p.res_stride + at, n, v[c]);
      }
    }
#pragma unroll
    for (int i = 0; i < kPiece; ++i) ss = __fmaf_rn(v[c][i], v[c][i], ss);
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xFFFFFFFFu, ss, s));
  if (warps > 1) {
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    ss = part[0];
    for (int i = 1; i < warps; ++i) ss = __fadd_rn(ss, part[i]);
  }
  const float inv = __frsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(p.D)), p.eps));
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int piece = tid + c * blockDim.x, at = piece * kPiece, n = p.D - at;
    if (n > 0) {
      float w[kPiece];
      load_gain(p, at, n, w);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) v[c][i] = __fmul_rn(__fmul_rn(v[c][i], inv), w[i]);
    }
    const int group = piece >> 3;
    encode_piece(v[c], n, p.out + m * p.out_stride + at, p.sa + group * p.sa_stride + m,
                 (piece & 7) == 0 && group * kGroup < p.D);
  }
}

template <typename F, typename... Args>
cudaError_t launch(F *kernel, unsigned grid, unsigned threads, bool overlap, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename TX, typename TY>
cudaError_t launch_rms(const RmsArgs &a, int M, bool overlap, cudaStream_t stream) {
  const int pieces = (a.D + kGroup - 1) / kGroup * (kGroup / kPiece);
  const int c = pieces <= 512 ? 1 : pieces <= 1024 ? 2 : 4;
  const unsigned threads = ((pieces + c - 1) / c + 31) / 32 * 32;
  switch (c) {
    case 1: return launch(rms_f8_kernel<TX, TY, 1>, M, threads, overlap, stream, a);
    case 2: return launch(rms_f8_kernel<TX, TY, 2>, M, threads, overlap, stream, a);
    default: return launch(rms_f8_kernel<TX, TY, 4>, M, threads, overlap, stream, a);
  }
}

template <typename TX>
cudaError_t launch_rms_y(const RmsArgs &a, int y_dtype, int M, bool overlap, cudaStream_t stream) {
  if (!a.y) return launch_rms<TX, None>(a, M, overlap, stream);
  if (y_dtype == kDtypeF32) return launch_rms<TX, float>(a, M, overlap, stream);
  if (y_dtype == kDtypeF16) return launch_rms<TX, __half>(a, M, overlap, stream);
  return launch_rms<TX, __nv_bfloat16>(a, M, overlap, stream);
}

template <typename T>
cudaError_t launch_quant(const QuantF8Launch &q, bool overlap, cudaStream_t stream) {
  const int per_row = (q.D + kGroup - 1) / kGroup * (kGroup / kPiece);
  const long long blocks = (static_cast<long long>(q.M) * per_row + 255) / 256;
  if (blocks > 0x7FFFFFFFLL) return cudaErrorInvalidConfiguration;
  const bool gate_vec = (static_cast<long long>(q.D) * sizeof(T)) % 16 == 0;
  const T *x = static_cast<const T *>(q.x);
  uint8_t *out = static_cast<uint8_t *>(q.out);
  if (q.gated)
    return launch(quant_f8_kernel<T, true>, static_cast<unsigned>(blocks), 256, overlap, stream, x, q.x_stride, out,
                  q.out_stride, q.sa, q.sa_stride, q.M, q.D, per_row, gate_vec);
  return launch(quant_f8_kernel<T, false>, static_cast<unsigned>(blocks), 256, overlap, stream, x, q.x_stride, out,
                q.out_stride, q.sa, q.sa_stride, q.M, q.D, per_row, gate_vec);
}

}  // namespace

cudaError_t launch_quant_f8(const QuantF8Launch &q, bool overlap, cudaStream_t stream) {
  if (q.x_dtype == kDtypeF32) return launch_quant<float>(q, overlap, stream);
  if (q.x_dtype == kDtypeF16) return launch_quant<__half>(q, overlap, stream);
  return launch_quant<__nv_bfloat16>(q, overlap, stream);
}

cudaError_t launch_rms_f8(const RmsF8Launch &r, bool overlap, cudaStream_t stream) {
  RmsArgs a;
  a.x = r.x; a.y = r.y; a.w = r.w; a.res = r.res; a.out = static_cast<uint8_t *>(r.out); a.sa = r.sa;
  a.x_stride = r.x_stride; a.y_stride = r.y_stride; a.res_stride = r.res_stride; a.out_stride = r.out_stride;
  a.sa_stride = r.sa_stride; a.D = r.D; a.w_dtype = r.w_dtype; a.eps = r.eps;
  if (r.x_dtype == kDtypeF32) return launch_rms_y<float>(a, r.y_dtype, r.M, overlap, stream);
  if (r.x_dtype == kDtypeF16) return launch_rms_y<__half>(a, r.y_dtype, r.M, overlap, stream);
  return launch_rms_y<__nv_bfloat16>(a, r.y_dtype, r.M, overlap, stream);
}

}  // namespace h3b
