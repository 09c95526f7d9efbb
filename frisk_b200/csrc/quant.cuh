// Rows of 8-bit numbers with one fp32 scale each: what the 8-bit gemm plans take as A and B.
//
//   plain     v = x
//   rmsnorm   h = x + residual,  v = h * rsqrt(mean(h^2) + eps) * weight   (h also stored)
//   silu_mul  v = gate / (1 + exp(-gate)) * up
//   scale[r] = max(max |v[r, :]| / Q, 2^-126),  q[r, c] = round_to_nearest_even(v[r, c] / scale[r])
//
// with Q = 127 (int8), 448 (e4m3), 57344 (e5m2); everything in fp32 and one rounding into the stored
// type.  The factor rsqrt(..) is the same for a whole row, so it cancels in q: with g = h * weight
// and a = max |g|, q = round(g / (a / Q)) and scale = rsqrt(..) * (a / Q), and the sum of squares
// and the maximum come out of ONE pass over the row.
// The maximum is taken over the bit patterns of |g| as unsigned integers: the same order as the
// numbers', with infinity above them and NaN above infinity, so a row that holds either gets a scale
// of infinity or NaN (and every product with it is NaN) instead of losing it silently.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/frisk_b200.h"

namespace frisk_quant {

constexpr float kTinyScale = 1.17549435e-38f;   // 2^-126: 1 / scale is finite, q of a zero row is 0

struct Params {
  const void* x;
  const void* other;    // residual (rmsnorm) or the up matrix (silu_mul); nullptr: none
  const void* weight;   // rmsnorm; nullptr: ones
  void* sum_out;        // rmsnorm; nullptr: not stored
  void* q;
  float* scale;
  int64_t rows, cols;
  int64_t ldx, ldo, lds, ldq;
  float eps;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int QT>
__device__ __forceinline__ constexpr float q_max() {
  return QT == FRISK_DT_I8 ? 127.f : QT == FRISK_DT_E4M3 ? 448.f : 57344.f;
}
// One value of at most Q in magnitude (a little above it by rounding) into its 8 bits; NaN becomes 0
// in int8, which has none.
template <int QT>
__device__ __forceinline__ uint8_t encode8(float v) {
  if (QT == FRISK_DT_I8) return (uint8_t)(int8_t)max(-127, min(127, __float2int_rn(v)));
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, QT == FRISK_DT_E4M3 ? __NV_E4M3 : __NV_E5M2);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float silu_mul(float gate, float up) { return gate / (1.f + expf(-gate)) * up; }

// scale and the divisor of g from the row's sum of h^2 and maximum of |g| (as bits)
template <int KIND, int QT>
__device__ __forceinline__ void row_scale(float sum_sq, uint32_t max_bits, int64_t cols, float eps, float* scale,
                                          float* divisor) {
  const float d = __fdiv_rn(__uint_as_float(max_bits), q_max<QT>());
  if (KIND != FRISK_QUANT_RMSNORM) {
    *scale = *divisor = max_bits > 0x7f800000u ? d : fmaxf(d, kTinyScale);
    return;
  }
  // a sum of squares past the range of fp32 has no norm: NaN, not a scale of zero
  const float rstd = sum_sq < __uint_as_float(0x7f800000u)
                         ? __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(sum_sq, (float)cols) + eps))
                         : __uint_as_float(0x7fc00000u);
  const float s = rstd * d;
  // (a scale below 2^-126 is raised to it, and g's divisor with it; NaN fails the test and stays)
  *scale = s < kTinyScale ? kTinyScale : s;
  // (not to zero: g is zero or a few of fp32's smallest steps there)
  *divisor = s < kTinyScale ? fmaxf(__fdiv_rn(kTinyScale, rstd), __uint_as_float(1u)) : d;
}

// The plain form of the three kinds: a CTA per row, two passes over it, element by element.  Serves
// any type, pitch, alignment and width.
template <typename TIn, typename TW, int QT, int KIND>
__global__ void __launch_bounds__(256) quant_rows_generic_kernel(const Params p) {
  __shared__ float s_sum[8];
  __shared__ uint32_t s_max[8];
  const TW* w = static_cast<const TW*>(p.weight);
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const TIn* x = static_cast<const TIn*>(p.x) + r * p.ldx;
    const TIn* o = static_cast<const TIn*>(p.other);
    if (o) o += r * p.ldo;
    auto value = [&](int64_t c, float* h) {
      float v = to_float<TIn>(x[c]);
      if (KIND == FRISK_QUANT_SILU_MUL) return silu_mul(v, to_float<TIn>(o[c]));
      if (KIND == FRISK_QUANT_RMSNORM) {
        if (o) v += to_float<TIn>(o[c]);
        *h = v;
        if (w) v *= to_float<TW>(w[c]);
      }
      return v;
    };
    float sum = 0.f, h = 0.f;
    uint32_t mx = 0;
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) {
      mx = max(mx, abs_bits(value(c, &h)));
      if (KIND == FRISK_QUANT_RMSNORM) sum = fmaf(h, h, sum);
    }
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    mx = __reduce_max_sync(0xffffffffu, mx);
    if ((threadIdx.x & 31) == 0) {
      s_sum[threadIdx.x >> 5] = sum;
      s_max[threadIdx.x >> 5] = mx;
    }
    __syncthreads();
    sum = s_sum[0];
    mx = s_max[0];
    for (int i = 1; i < 8; ++i) {
      sum += s_sum[i];
      mx = max(mx, s_max[i]);
    }
    float scale, divisor;
    row_scale<KIND, QT>(sum, mx, p.cols, p.eps, &scale, &divisor);
    if (threadIdx.x == 0) p.scale[r] = scale;
    uint8_t* q = static_cast<uint8_t*>(p.q) + r * p.ldq;
    TIn* so = p.sum_out ? static_cast<TIn*>(p.sum_out) + r * p.lds : nullptr;
    // sum_out may be x or the residual: an element is written by the thread that has just read it
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) {
      q[c] = encode8<QT>(__fdiv_rn(value(c, &h), divisor));
      if (KIND == FRISK_QUANT_RMSNORM && so) so[c] = from_float<TIn>(h);
    }
    __syncthreads();   // the shared arrays are written again by the next row
  }
}

}  // namespace frisk_quant
