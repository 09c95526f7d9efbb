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
  int32_t q_type;
  int32_t warps_per_row, rows_per_cta;   // quant_rows_kernel
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

// The 8-bit type is a run-time value, the same for the whole grid: it decides a few instructions per
// group of elements, not worth three times the kernels.
__device__ __forceinline__ float q_max(int qt) {
  return qt == FRISK_DT_I8 ? 127.f : qt == FRISK_DT_E4M3 ? 448.f : 57344.f;
}
// Values of at most Q in magnitude (a little above it by rounding) into their 8 bits; NaN becomes 0
// in int8, which has none.
__device__ __forceinline__ uint8_t encode8(float v, int qt) {
  if (qt == FRISK_DT_I8) return (uint8_t)(int8_t)max(-127, min(127, __float2int_rn(v)));
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, qt == FRISK_DT_E4M3 ? __NV_E4M3 : __NV_E5M2);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Sum and maximum over a warp, in every lane.
template <int KIND>
__device__ __forceinline__ void warp_fold(float& sum, uint32_t& mx) {
  if (KIND == FRISK_QUANT_RMSNORM) {
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
}

__device__ __forceinline__ float silu_mul(float gate, float up) { return gate / (1.f + expf(-gate)) * up; }

// scale[r] and the divisor of g from the row's sum of h^2 and maximum of |g| (as bits).  Every thread
// of the row needs the divisor; the scale, with its root, only the one that stores it (`writer`).
template <int KIND>
__device__ __forceinline__ float row_divisor(float sum_sq, uint32_t max_bits, int64_t cols, float eps, int qt,
                                             bool writer, float* scale) {
  const float d = __fdiv_rn(__uint_as_float(max_bits), q_max(qt));
  if (KIND != FRISK_QUANT_RMSNORM) {
    const float s = max_bits > 0x7f800000u ? d : fmaxf(d, kTinyScale);
    if (writer) *scale = s;
    return s;
  }
  // (rsqrt(..) of a finite sum is above 1e-20: a divisor of 1e-18 needs no look at the scale)
  if (!writer && d >= 1e-18f) return d;
  // a sum of squares past the range of fp32 has no norm: NaN, not a scale of zero
  const float rstd = sum_sq < __uint_as_float(0x7f800000u)
                         ? __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(sum_sq, (float)cols) + eps))
                         : __uint_as_float(0x7fc00000u);
  const float s = rstd * d;
  // a scale below 2^-126 is raised to it, and g's divisor with it (not to zero: g is zero or a few
  // of fp32's smallest steps there); NaN fails the test and stays
  const bool tiny = s < kTinyScale;
  if (writer) *scale = tiny ? kTinyScale : s;
  return tiny ? fmaxf(__fdiv_rn(kTinyScale, rstd), __uint_as_float(1u)) : d;
}

// The plain form of the three kinds: a CTA per row, two passes over it, element by element.  Serves
// any type, pitch, alignment and width.
template <typename TIn, typename TW, int KIND>
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
    warp_fold<KIND>(sum, mx);
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
    const float divisor = row_divisor<KIND>(sum, mx, p.cols, p.eps, p.q_type, threadIdx.x == 0, p.scale + r);
    uint8_t* q = static_cast<uint8_t*>(p.q) + r * p.ldq;
    TIn* so = p.sum_out ? static_cast<TIn*>(p.sum_out) + r * p.lds : nullptr;
    // sum_out may be x or the residual: an element is written by the thread that has just read it
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) {
      q[c] = encode8(__fdiv_rn(value(c, &h), divisor), p.q_type);
      if (KIND == FRISK_QUANT_RMSNORM && so) so[c] = from_float<TIn>(h);
    }
    __syncthreads();   // the shared arrays are written again by the next row
  }
}

// ---- rows in registers -------------------------------------------------------------------------
// Eight neighbouring elements as they are stored: one or two 16-byte words.
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* p) {   // read once: past L1
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.w[i].x), "=r"(r.w[i].y), "=r"(r.w[i].z), "=r"(r.w[i].w)
                 : "l"(reinterpret_cast<const uint4*>(p) + i)
                 : "memory");
  return r;
}
template <typename T>
__device__ __forceinline__ Eight<T> load8_shared_by_rows(const T* p) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
// Two fp32 numbers in a register pair: the packed instructions do both for one issue slot, and it is
// issue slots that the gated kind would otherwise be bound by.
using f2 = uint64_t;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ f2 pack2(float v) { return pack2(v, v); }
__device__ __forceinline__ float lo2(f2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi2(f2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// max(|a|, |b|, m), NaN if one of them is
__device__ __forceinline__ float abs_max(f2 v, float m) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(lo2(v)), "f"(hi2(v)), "f"(m));
  return r;
}
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const Eight<T>& r, f2 (&f)[4]) {
  const T* e = reinterpret_cast<const T*>(r.w);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = pack2(to_float<T>(e[2 * j]), to_float<T>(e[2 * j + 1]));
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const f2 (&f)[4]) {
  Eight<T> r;
  T* e = reinterpret_cast<T*>(r.w);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    e[2 * j] = from_float<T>(lo2(f[j]));
    e[2 * j + 1] = from_float<T>(hi2(f[j]));
  }
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}
// Eight values into eight bytes.
__device__ __forceinline__ uint2 encode8x8(const f2 (&v)[4], int qt) {
  union {
    uint32_t u[2];
    uint16_t h[4];
  } r;
  if (qt == FRISK_DT_I8) {
    // (|v| rounds to 127 at most; NaN becomes 0)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t upper;
      asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(upper) : "r"(__float2int_rn(hi2(v[2 * j + 1]))), "r"(__float2int_rn(lo2(v[2 * j + 1]))), "r"(0));
      asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(r.u[j]) : "r"(__float2int_rn(hi2(v[2 * j]))), "r"(__float2int_rn(lo2(v[2 * j]))), "r"(upper));
    }
  } else if (qt == FRISK_DT_E4M3) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.h[j] = __nv_cvt_float2_to_fp8x2(make_float2(lo2(v[j]), hi2(v[j])), __NV_SATFINITE, __NV_E4M3);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.h[j] = __nv_cvt_float2_to_fp8x2(make_float2(lo2(v[j]), hi2(v[j])), __NV_SATFINITE, __NV_E5M2);
  }
  return make_uint2(r.u[0], r.u[1]);
}

// gate / (1 + exp(-gate)) * up for two elements.  With e = exp(-|gate|), which cannot overflow:
//   silu = gate * (gate < 0 ? e : 1) / (1 + e).
// e = 2^-(a log2(e)), a = |gate| (at most 200: e is 0 long before): the product is split into its
// rounded value t, for the hardware's 2^x, and the exact rest, which with log2(e)'s own rest enters
// to first order, 2^rest = 1 + rest ln 2.  The quotient is the reciprocal's, corrected by its remainder
// as in div_by.  Exponentials below 2^-126 (gates below -87) are zero.
__device__ __forceinline__ f2 silu_mul2(f2 gate, f2 up) {
  constexpr float kLog2e = 1.44269504f, kLog2eRest = (float)(1.4426950408889634074 - (double)1.44269504f);
  constexpr float kLn2 = 0.693147181f;
  const float g0 = lo2(gate), g1 = hi2(gate);
  const f2 a = pack2(fminf(fabsf(g0), 200.f), fminf(fabsf(g1), 200.f));
  const f2 t = mul2(a, pack2(kLog2e));
  f2 rest = fma2(a, pack2(-kLog2e), t);
  rest = mul2(fma2(a, pack2(-kLog2eRest), rest), pack2(kLn2));
  f2 e = pack2(ex2(-lo2(t)), ex2(-hi2(t)));
  e = fma2(e, rest, e);
  const f2 d = add2(e, pack2(1.f));
  const f2 minus_y = pack2(rcp(-lo2(d)), rcp(-hi2(d)));
  const f2 minus_n = mul2(gate, pack2(g0 < 0.f ? -lo2(e) : -1.f, g1 < 0.f ? -hi2(e) : -1.f));
  const f2 s = mul2(minus_n, minus_y);
  return mul2(fma2(fma2(s, d, minus_n), minus_y, s), up);
}

// v / d to nearest for many v and one d: with y the reciprocal of d to nearest and q = v y, the
// remainder v - q d is exact in one fused multiply-add, and q plus the remainder times y is the
// correctly rounded quotient (P. Markstein, IBM Journal of Research and Development 34(1), 1990) where
// nothing leaves the range of normal numbers: d is at least 1e-30 here and v at most Q d.  A divisor
// of infinity or NaN makes the values NaN, as the row's scale says.
__device__ __forceinline__ f2 div_by(f2 v, f2 minus_d, f2 y) {
  const f2 q = mul2(v, y);
  return fma2(fma2(q, minus_d, v), y, q);
}

// Whole rows in registers: `warps_per_row` warps share a row, every thread NV groups of eight elements
// of it, so the row is read once and the only pause is the fold of (sum, maximum) over the warps.
// For rows whose starts, in every buffer, allow 16-byte accesses (8 for q) and whose width is a
// multiple of eight.  CTAs of more than one row fold them side by side.
template <typename TIn, typename TW, int KIND, int NV>
__global__ void __launch_bounds__(1024) quant_rows_kernel(const Params p) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wpr = p.warps_per_row;
  const int slot = warp / wpr, warp_in_row = warp - slot * wpr;
  const int64_t r = (int64_t)blockIdx.x * p.rows_per_cta + slot;
  const bool live = r < p.rows;
  const int t = warp_in_row * 32 + lane, step = wpr * 32, groups = (int)(p.cols >> 3);
  const TIn* x = static_cast<const TIn*>(p.x) + r * p.ldx;
  const TIn* o = p.other ? static_cast<const TIn*>(p.other) + r * p.ldo : nullptr;
  const TW* w = static_cast<const TW*>(p.weight);
  TIn* so = p.sum_out ? static_cast<TIn*>(p.sum_out) + r * p.lds : nullptr;

  Eight<TIn> rx[NV], ro[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int gidx = t + i * step;
    if (live && gidx < groups) {
      rx[i] = load8(x + 8 * (int64_t)gidx);
      if (KIND != FRISK_QUANT_PLAIN && o) ro[i] = load8(o + 8 * (int64_t)gidx);
    }
  }
  f2 g[NV][4];
  f2 sums = 0;      // of squares, even and odd elements
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int gidx = t + i * step;
    if (live && gidx < groups) {
      unpack8(rx[i], g[i]);
      f2 u[4];
      if (KIND == FRISK_QUANT_SILU_MUL) {
        unpack8(ro[i], u);
#pragma unroll
        for (int j = 0; j < 4; ++j) g[i][j] = silu_mul2(g[i][j], u[j]);
      }
      if (KIND == FRISK_QUANT_RMSNORM) {
        if (o) {
          unpack8(ro[i], u);
#pragma unroll
          for (int j = 0; j < 4; ++j) g[i][j] = add2(g[i][j], u[j]);
          if (so) store8(so + 8 * (int64_t)gidx, g[i]);   // read above by this thread, if it is x or the residual
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) sums = fma2(g[i][j], g[i][j], sums);
        if (w) {
          f2 v[4];
          unpack8(load8_shared_by_rows(w + 8 * (int64_t)gidx), v);
#pragma unroll
          for (int j = 0; j < 4; ++j) g[i][j] = mul2(g[i][j], v[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) top = abs_max(g[i][j], top);
    }
  }
  float sum = lo2(sums) + hi2(sums);
  uint32_t mx = __float_as_uint(top);
  warp_fold<KIND>(sum, mx);
  if (wpr > 1) {
    if (lane == 0) {
      s_sum[warp] = sum;
      s_max[warp] = mx;
    }
    __syncthreads();
    sum = lane < wpr ? s_sum[slot * wpr + lane] : 0.f;
    mx = lane < wpr ? s_max[slot * wpr + lane] : 0u;
    warp_fold<KIND>(sum, mx);
  }
  if (!live) return;
  float d = row_divisor<KIND>(sum, mx, p.cols, p.eps, p.q_type, t == 0, p.scale + r);
  if (d < 1e-30f) {   // both up by the same power of two (exact), so that div_by stays in range
    d *= 0x1p96f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) g[i][j] = mul2(g[i][j], pack2(0x1p96f));
  }
  const f2 minus_d = pack2(-d), y = pack2(__frcp_rn(d));
  uint8_t* q = static_cast<uint8_t*>(p.q) + r * p.ldq;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int gidx = t + i * step;
    if (gidx < groups) {
#pragma unroll
      for (int j = 0; j < 4; ++j) g[i][j] = div_by(g[i][j], minus_d, y);
      *reinterpret_cast<uint2*>(q + 8 * (int64_t)gidx) = encode8x8(g[i], p.q_type);
    }
  }
}

}  // namespace frisk_quant
