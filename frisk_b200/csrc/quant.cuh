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
#include "ptx_sm100.cuh"

namespace frisk_quant {

constexpr float kTinyScale = 1.17549435e-38f;   // 2^-126: 1 / scale is finite, q of a zero row is 0
// A norm with mean(h^2) + eps below this, 1 / rms above 2^20: fp32 loses the squares of small h, and g =
// h * weight may be a few of its smallest steps although the row's scale is a regular number.  Such rows,
// possible only with an eps below it, are worked out in 64 bits (small_norm_row).  Above it a square that
// is lost changes the mean by less than 2^-109 of it, and a row whose scale is regular has a maximum of 2^10
// steps or more.
constexpr float kSmallNorm = 0x1p-40f;
// The kinds as template arguments: frisk_quant_kind, and the norm with an eps below kSmallNorm (in the
// ordinary norm's kernels the mere presence of small_norm_row cost 8 % of 8192 x 8192 bf16, 30 % of
// 1023 x 5001 f16).
constexpr int kNormAnyEps = FRISK_QUANT_SILU_MUL + 1;
constexpr bool is_norm(int kind) { return kind == FRISK_QUANT_RMSNORM || kind == kNormAnyEps; }

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
  int32_t stages;       // streamed rows: rows in the ring
  int32_t* status;      // streamed rows: where a wait that ran out is reported; nullptr: nowhere
  int64_t wait_cycles;  // ... and how long a wait may take
  int32_t late_sum;     // rmsnorm, rows in registers: sum_out is written when nothing of the row is needed any more
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
// A finite value of at most Q in magnitude (a little above it by rounding) into its 8 bits.
__device__ __forceinline__ uint8_t encode8(float v, int qt) {
  if (qt == FRISK_DT_I8) return (uint8_t)(int8_t)max(-127, min(127, __float2int_rn(v)));
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, qt == FRISK_DT_E4M3 ? __NV_E4M3 : __NV_E5M2);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Sum and maximum over a warp, in every lane.
template <int KIND>
__device__ __forceinline__ void warp_fold(float& sum, uint32_t& mx) {
  if (is_norm(KIND)) {
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
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

// gate / (1 + exp(-gate)) * up.  Gates from -kNearGate on leave every step in fp32's normal numbers: exp(87)
// is 6.1e37, and its reciprocal is above 2^-126.
constexpr float kNearGate = 87.f;
constexpr float kLog2e = 1.44269504f, kLog2eRest = (float)(1.4426950408889634074 - (double)1.44269504f), kLn2 = 0.693147181f;

// Below, 1 + exp(-gate) is exp(-gate) in fp32, past its range from -88.7 on, though the product with a
// large up is not: gate * (2^160 exp(gate)) * (2^-64 up) * 2^-96 rounds in the range of normal numbers until
// the last step.  2^160 exp(gate) is zero from about -198 on, where the product with the largest up is
// less than half of fp32's smallest number.
__device__ __forceinline__ float silu_mul(float gate, float up) {
  if (!(gate < -kNearGate)) return gate / (1.f + expf(-gate)) * up;
  const float a = fmaxf(gate, -200.f), t = a * kLog2e;
  const float rest = fmaf(a, kLog2eRest, fmaf(a, kLog2e, -t)) * kLn2;   // as in silu_mul2
  const float e = ex2(t + 160.f);                                       // (the sum is exact)
  return gate * fmaf(e, rest, e) * (up * 0x1p-64f) * 0x1p-96f;
}

// What a row's elements are multiplied by: q = round(v * up * (hi + lo)).  hi + lo is Q / max |v| as the
// sum of two fp32 numbers (to 2^-46), not the reciprocal of the stored scale, whose rounding would move
// every quotient of a row a little: an element exactly half way between two 8-bit numbers (half of the
// maximum is 63.5 in int8) has to stay there to be rounded to even.  hi = 0: q is zero.
struct Factor {
  float hi, lo, up;
};

// scale[r] and the factor of g from the row's sum of h^2 and maximum of |g| (as bits).  Every thread
// of the row needs the factor; the scale, with its root, only the one that stores it (`writer`).
template <int KIND>
__device__ __forceinline__ Factor row_factor(float sum_sq, uint32_t max_bits, int64_t cols, float eps, int qt,
                                             bool writer, float* scale) {
  const float top = __uint_as_float(max_bits), q = q_max(qt);
  // A norm's row of very small g: Q over its maximum would leave fp32, so the row is worked on 2^96 times
  // as large (exact).
  const bool low = is_norm(KIND) && top < 0x1p-100f;
  const float up = low ? 0x1p96f : 1.f, m = top * up;
  Factor f{__fdiv_rn(q, m), 0.f, up};
  f.lo = fmaf(-f.hi, m, q) * (qt == FRISK_DT_I8 ? 1.f / 127.f : qt == FRISK_DT_E4M3 ? 1.f / 448.f : 1.f / 57344.f) * f.hi;
  // zeros next to a scale that makes every product NaN; a sum of squares past the range of fp32 has no norm
  // and gets one as well
  const bool no_norm = is_norm(KIND) && !(sum_sq < __uint_as_float(0x7f800000u));
  if (max_bits >= 0x7f800000u || no_norm) f = {0.f, 0.f, 1.f};
  if (!is_norm(KIND)) {
    const bool tiny = top < q * kTinyScale;   // the scale is 2^-126, and the factor 2^126
    if (writer) *scale = tiny ? kTinyScale : __fdiv_rn(top, q);
    if (tiny) f = {0x1p126f, 0.f, 1.f};
    return f;
  }
  // (rsqrt(..) of a finite sum is above 1e-20: a maximum of 1e-12 needs no look at the scale)
  if (!writer && top >= 1e-12f) return f;
  const float mean = __fdiv_rn(sum_sq, (float)cols);
  float rstd = __fdiv_rn(1.f, __fsqrt_rn(mean + eps));
  if (rstd == 0.f) rstd = __fdiv_rn(0.5f, __fsqrt_rn(0.25f * mean + 0.25f * eps));   // the sum alone left fp32
  if (no_norm) rstd = __uint_as_float(0x7fc00000u);
  const float s = rstd * __fdiv_rn(m, q) * (low ? 0x1p-96f : 1.f);
  // a scale below 2^-126 is raised to it, and the factor goes with it; NaN fails the test and stays
  const bool tiny = s < kTinyScale;
  if (writer) *scale = tiny ? kTinyScale : s;
  if (tiny) f = {rstd * (low ? 0x1p30f : 0x1p126f), 0.f, up};
  return f;
}
// A product r = v * (hi + lo) that fp32's rounding may have put on a border between two 8-bit numbers: an
// odd number of at most 8 bits times a power of two, its lower 16 bits zero.  What the rounding took away
// decides then: at least 2^-32 of r where v Q / max |v| is not that border (a quotient of 24-bit numbers
// times Q), below 2^-45 where it is (hi + lo is good to 2^-46).  r goes to the neighbour on that side.
__device__ __forceinline__ bool maybe_border(float r) { return (__float_as_uint(r) & 0xffffu) == 0; }
__device__ __forceinline__ float off_border(float r, float v, float hi, float lo) {
  const float rest = fmaf(v, lo, fmaf(v, hi, -r));
  if (!maybe_border(r) || !(fabsf(rest) > fabsf(r) * 0x1p-40f) || !(fabsf(hi) > 0x1p-90f)) return r;   // (a smaller lo has too few bits)
  return __uint_as_float(__float_as_uint(r) + ((rest < 0.f) == (r < 0.f) ? 1u : 0xffffffffu));
}
// fp32 values as they are: q is the exact rounding.  (The other kinds' v carries roundings of its own; for
// 16-bit values no quotient that is not a border comes as near to one.)
template <typename TIn, int KIND>
constexpr bool kExactQ = sizeof(TIn) == 4 && KIND == FRISK_QUANT_PLAIN;
// v * up * (hi + lo), to 2^-24 of it: exact where that is an fp32 number.
template <bool kExact>
__device__ __forceinline__ float times(float v, Factor f) {
  if (f.hi == 0.f) return 0.f;
  v *= f.up;
  const float r = fmaf(v, f.hi, v * f.lo);
  return kExact ? off_border(r, v, f.hi, f.lo) : r;
}

// Every kernel here is a programmatic dependent launch: it may be scheduled while the kernel before it
// in the stream drains, waits here until that one's writes are visible, and lets the next one do the
// same.
__device__ __forceinline__ void after_the_kernel_before() {
  frisk::ptx::griddep_launch_dependents();
  frisk::ptx::griddep_wait();
}

// Whether a row's norm is one for small_norm_row (the same in every thread of the row).
__device__ __forceinline__ bool small_norm(float sum_sq, uint32_t max_bits, const Params& p) {
  return p.eps < kSmallNorm && max_bits < 0x7f800000u && __fdiv_rn(sum_sq, (float)p.cols) + p.eps < kSmallNorm;
}

// One row after a norm in 64 bits, by a CTA: h in fp32 like everywhere, its squares, their sum
// and h * weight in double (no range is left, the product is exact), q rounded from fp32.  Two passes over
// the row, element by element; the sum is stored in the second, by the thread that has read the element.
template <typename TIn, typename TW>
__device__ __noinline__ void small_norm_row(const Params& p, int64_t r) {
  __shared__ double s_sum[32], s_top[32];
  const TIn* x = static_cast<const TIn*>(p.x) + r * p.ldx;
  const TIn* o = p.other ? static_cast<const TIn*>(p.other) + r * p.ldo : nullptr;
  const TW* w = static_cast<const TW*>(p.weight);
  TIn* so = p.sum_out ? static_cast<TIn*>(p.sum_out) + r * p.lds : nullptr;
  auto value = [&](int64_t c, float* h) {
    *h = to_float<TIn>(x[c]);
    if (o) *h += to_float<TIn>(o[c]);
    return w ? (double)*h * (double)to_float<TW>(w[c]) : (double)*h;
  };
  double sum = 0., top = 0.;
  float h;
  for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
    top = fmax(top, fabs(value(c, &h)));
    sum += (double)h * h;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    top = fmax(top, __shfl_xor_sync(0xffffffffu, top, d));
  }
  __syncthreads();   // a row before this one may still be reading the shared arrays
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_top[threadIdx.x >> 5] = top;
  }
  __syncthreads();
  sum = top = 0.;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) {
    sum += s_sum[i];
    top = fmax(top, s_top[i]);
  }
  // (a row of zeros, which has no norm without eps: q = 0 and the least scale)
  const double rstd = top == 0. ? 0. : 1. / sqrt(sum / (double)p.cols + (double)p.eps);
  const double scale = top * rstd / q_max(p.q_type);
  const bool tiny = scale < kTinyScale;
  const double f = tiny ? rstd * 0x1p126 : q_max(p.q_type) / top;
  if (threadIdx.x == 0) p.scale[r] = tiny ? kTinyScale : (float)scale;
  uint8_t* q = static_cast<uint8_t*>(p.q) + r * p.ldq;
  for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
    q[c] = encode8((float)(value(c, &h) * f), p.q_type);
    if (so) so[c] = from_float<TIn>(h);
  }
}

// The plain form of the three kinds: a CTA per row, two passes over it, element by element.  Serves
// any type, pitch, alignment and width.
template <typename TIn, typename TW, int KIND>
__global__ void __launch_bounds__(256) quant_rows_generic_kernel(const Params p) {
  __shared__ float s_sum[8];
  __shared__ uint32_t s_max[8];
  const TW* w = static_cast<const TW*>(p.weight);
  after_the_kernel_before();
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const TIn* x = static_cast<const TIn*>(p.x) + r * p.ldx;
    const TIn* o = static_cast<const TIn*>(p.other);
    if (o) o += r * p.ldo;
    auto value = [&](int64_t c, float* h) {
      float v = to_float<TIn>(x[c]);
      if (KIND == FRISK_QUANT_SILU_MUL) return silu_mul(v, to_float<TIn>(o[c]));
      if (is_norm(KIND)) {
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
      if (is_norm(KIND)) sum = fmaf(h, h, sum);
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
    if constexpr (KIND == kNormAnyEps) {
      if (small_norm(sum, mx, p)) {
        small_norm_row<TIn, TW>(p, r);
        __syncthreads();
        continue;
      }
    }
    const Factor f = row_factor<KIND>(sum, mx, p.cols, p.eps, p.q_type, threadIdx.x == 0, p.scale + r);
    uint8_t* q = static_cast<uint8_t*>(p.q) + r * p.ldq;
    TIn* so = p.sum_out ? static_cast<TIn*>(p.sum_out) + r * p.lds : nullptr;
    // sum_out may be x or the residual: an element is written by the thread that has just read it
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) {
      const float v = value(c, &h);
      q[c] = encode8(times<kExactQ<TIn, KIND>>(v, f), p.q_type);
      if (is_norm(KIND) && so) so[c] = from_float<TIn>(h);
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
// min(a, b, m), NaN if one of them is, and max(a, b, m) of the numbers among them
__device__ __forceinline__ float min3(f2 v, float m) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(lo2(v)), "f"(hi2(v)), "f"(m));
  return r;
}
__device__ __forceinline__ float max3(f2 v, float m) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(lo2(v)), "f"(hi2(v)), "f"(m));
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const Eight<T>& r, f2 (&f)[4]) {
  const T* e = reinterpret_cast<const T*>(r.w);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = pack2(to_float<T>(e[2 * j]), to_float<T>(e[2 * j + 1]));
}
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const Eight<__nv_bfloat16>& r, f2 (&f)[4]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};   // a bf16 is the upper half of its fp32
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = pack2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
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
// A thread's NV groups of eight values into eight bytes each.
template <int NV>
__device__ __forceinline__ void encode_groups(const f2 (&v)[NV][4], int qt, uint2 (&out)[NV]) {
  if (qt == FRISK_DT_I8) {
    // v + 1.5 * 2^23 rounds v to the nearest integer, ties to even, and holds it in its low byte
    // (the conversion instruction shares its unit with the gate's 2^x and reciprocal)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t b[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f2 m = add2(v[i][j], pack2(12582912.f));
        b[2 * j] = __float_as_uint(lo2(m));
        b[2 * j + 1] = __float_as_uint(hi2(m));
      }
      uint32_t* o = &out[i].x;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        o[j] = __byte_perm(__byte_perm(b[4 * j], b[4 * j + 1], 0x0040), __byte_perm(b[4 * j + 2], b[4 * j + 3], 0x0040), 0x5410);
    }
    return;
  }
  auto floats = [&](__nv_fp8_interpretation_t kind) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __nv_cvt_float2_to_fp8x2(make_float2(lo2(v[i][j]), hi2(v[i][j])), __NV_SATFINITE, kind);
      out[i] = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
  };
  if (qt == FRISK_DT_E4M3) floats(__NV_E4M3);
  else floats(__NV_E5M2);
}

// gate / (1 + exp(-gate)) * up for two gates from -kNearGate to kLargeGate.  e = exp(-gate) = 2^-t, t = gate
// log2(e): the product is split into its rounded value, for the hardware's 2^x, and the exact rest, which
// with log2(e)'s own rest enters to first order, 2^rest = 1 + rest ln 2.  The quotient is the reciprocal's,
// corrected by its remainder, which is exact in one fused multiply-add (P. Markstein, IBM Journal of Research
// and Development 34(1), 1990).
constexpr float kLargeGate = 1e38f;   // t is finite
__device__ __forceinline__ f2 silu_mul2(f2 gate, f2 up) {
  const f2 t = mul2(gate, pack2(kLog2e));
  f2 rest = fma2(gate, pack2(-kLog2e), t);
  rest = mul2(fma2(gate, pack2(-kLog2eRest), rest), pack2(kLn2));
  f2 e = pack2(ex2(-lo2(t)), ex2(-hi2(t)));
  e = fma2(e, rest, e);
  const f2 minus_d = fma2(e, pack2(-1.f), pack2(-1.f));
  const f2 y = pack2(rcp(-lo2(minus_d)), rcp(-hi2(minus_d)));
  const f2 s = mul2(gate, y);
  return mul2(fma2(fma2(s, minus_d, gate), y, s), up);
}
// ... for any two: see silu_mul.
__device__ __forceinline__ f2 silu_mul2_any(f2 gate, f2 up) {
  const float g0 = lo2(gate), g1 = hi2(gate);
  const bool far0 = g0 < -kNearGate, far1 = g1 < -kNearGate;
  const f2 a = pack2(fminf(fmaxf(g0, -200.f), kNearGate), fminf(fmaxf(g1, -200.f), kNearGate));
  const f2 t = mul2(a, pack2(kLog2e));
  f2 rest = fma2(a, pack2(-kLog2e), t);
  rest = mul2(fma2(a, pack2(-kLog2eRest), rest), pack2(kLn2));
  f2 e = pack2(ex2(far0 ? lo2(t) + 160.f : -lo2(t)), ex2(far1 ? hi2(t) + 160.f : -hi2(t)));
  e = fma2(e, pack2(far0 ? -lo2(rest) : lo2(rest), far1 ? -hi2(rest) : hi2(rest)), e);
  const f2 minus_d = fma2(e, pack2(-1.f), pack2(-1.f));
  const f2 y = pack2(rcp(-lo2(minus_d)), rcp(-hi2(minus_d)));
  const f2 s = mul2(gate, y);
  const f2 near = mul2(fma2(fma2(s, minus_d, gate), y, s), up), large = mul2(gate, up);
  const f2 far = mul2(mul2(mul2(gate, e), mul2(up, pack2(0x1p-64f))), pack2(0x1p-96f));
  return pack2(far0 ? lo2(far) : g0 > kNearGate ? lo2(large) : lo2(near), far1 ? hi2(far) : g1 > kNearGate ? hi2(large) : hi2(near));
}

// Eight elements from storage to g, with the running sum of squares and maximum.  `weights(v)` fills v
// with the elements' weights, false if there are none; `store_sum(h)` stores h where that is wanted (x
// and the residual have been read: it may go to either).
template <typename TIn, int KIND, typename Weights, typename StoreSum>
__device__ __forceinline__ void group_values(const Eight<TIn>& x, const Eight<TIn>& other, bool has_other, Weights weights,
                                             StoreSum store_sum, f2 (&g)[4], f2& sums, float& top) {
  unpack8(x, g);
  f2 u[4];
  if (KIND == FRISK_QUANT_SILU_MUL) {
    unpack8(other, u);
    float least = 0.f, most = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      least = min3(g[j], least);
      most = max3(g[j], most);
    }
    if (least >= -kNearGate && most <= kLargeGate) {
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = silu_mul2(g[j], u[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = silu_mul2_any(g[j], u[j]);
    }
  }
  if (is_norm(KIND)) {
    if (has_other) {
      unpack8(other, u);
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = add2(g[j], u[j]);
      store_sum(g);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums = fma2(g[j], g[j], sums);
    f2 v[4];
    if (weights(v)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = mul2(g[j], v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) top = abs_max(g[j], top);
}

// g times the row's factor, in place.
template <bool kExact, int NV>
__device__ __forceinline__ void multiply(f2 (&g)[NV][4], Factor f) {
  if (f.up != 1.f || f.hi == 0.f) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) g[i][j] = f.hi == 0.f ? 0 : mul2(g[i][j], pack2(f.up));
  }
  const f2 hi = pack2(f.hi), lo = pack2(f.lo);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    f2 r[4];
    uint32_t low = 0xffffffffu;   // the least lower halves, of even and odd elements
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r[j] = fma2(g[i][j], hi, mul2(g[i][j], lo));
      if (kExact) low = __vminu2(low, __byte_perm(__float_as_uint(lo2(r[j])), __float_as_uint(hi2(r[j])), 0x5410));
    }
    if (kExact && ((low & 0xffffu) == 0 || (low & 0xffff0000u) == 0)) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[j] = pack2(off_border(lo2(r[j]), lo2(g[i][j]), f.hi, f.lo), off_border(hi2(r[j]), hi2(g[i][j]), f.hi, f.lo));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) g[i][j] = r[j];
  }
}

// Sum and maximum over the `wpr` warps of each of the CTA's rows, in every thread (a CTA barrier).
template <int KIND>
__device__ __forceinline__ void row_fold(float& sum, uint32_t& mx, float* s_sum, uint32_t* s_max, int warp, int lane,
                                         int slot, int wpr) {
  warp_fold<KIND>(sum, mx);
  if (wpr == 1) return;
  if (lane == 0) {
    s_sum[warp] = sum;
    s_max[warp] = mx;
  }
  __syncthreads();
  sum = lane < wpr ? s_sum[slot * wpr + lane] : 0.f;
  mx = lane < wpr ? s_max[slot * wpr + lane] : 0u;
  warp_fold<KIND>(sum, mx);
}

// Whole rows in registers: blockDim.x threads (whole warps) share a row, each with NV groups of eight
// elements of it, so the row is read once and the only pause is the fold of (sum, maximum) over the
// warps.
// For rows whose starts, in every buffer, allow 16-byte accesses (8 for q) and whose width is a
// multiple of eight.  CTAs of more than one row (blockDim.y) fold them side by side.
// kFull: every thread has all of its groups, of a row that exists (no bounds to test).
// Bound by memory where rows are many: 8192 x 8192 bf16 norm with residual 73 - 77 us (470 MB, 0.94 - 0.99
// of the copy rate; two passes element by element 168 us), fp32 as it is 50 us (336 MB, 1.0; 96 us).
// Few rows take one group per thread, since then the launch and the row's own latency are all there
// is: 1 x 4096 norm 1.8 us.
template <typename TIn, typename TW, int KIND, int NV, bool kFull>
__global__ void __launch_bounds__(1024) quant_rows_kernel(const Params p) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  // threadIdx.y: which of the CTA's rows (the same in a whole warp: the broadcast tells the compiler)
  const int t = threadIdx.x, step = blockDim.x, lane = t & 31, wpr = step >> 5;
  const int slot = __shfl_sync(0xffffffffu, threadIdx.y, 0), warp = slot * wpr + (t >> 5);
  const int64_t r = (int64_t)blockIdx.x * blockDim.y + slot;
  const bool live = kFull || r < p.rows;
  const int groups = (int)(p.cols >> 3);
  const TIn* x = static_cast<const TIn*>(p.x) + r * p.ldx;
  const TIn* o = p.other ? static_cast<const TIn*>(p.other) + r * p.ldo : nullptr;
  const TW* w = static_cast<const TW*>(p.weight);
  TIn* so = p.sum_out ? static_cast<TIn*>(p.sum_out) + r * p.lds : nullptr;

  after_the_kernel_before();
  Eight<TIn> rx[NV], ro[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int gidx = t + i * step;
    if (kFull || (live && gidx < groups)) {
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
    if (kFull || (live && gidx < groups))
      group_values<TIn, KIND>(
          rx[i], ro[i], o != nullptr,
          [&](f2 (&v)[4]) {
            if (w) unpack8(load8_shared_by_rows(w + 8 * gidx), v);
            return w != nullptr;
          },
          [&](const f2 (&h)[4]) {
            if (so && !(KIND == kNormAnyEps && p.late_sum)) store8(so + 8 * (int64_t)gidx, h);
          },
          g[i], sums, top);
  }
  float sum = lo2(sums) + hi2(sums);
  uint32_t mx = __float_as_uint(top);
  row_fold<KIND>(sum, mx, s_sum, s_max, warp, lane, slot, wpr);
  if (!live) return;
  if constexpr (KIND == kNormAnyEps) {
    if (small_norm(sum, mx, p)) return small_norm_row<TIn, TW>(p, r);   // (the CTA has one row)
  }
  multiply<kExactQ<TIn, KIND>, NV>(g, row_factor<KIND>(sum, mx, p.cols, p.eps, p.q_type, t == 0, p.scale + r));
  uint8_t* q = static_cast<uint8_t*>(p.q) + r * p.ldq;
  uint2 bytes[NV];
  encode_groups<NV>(g, p.q_type, bytes);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int gidx = t + i * step;
    if (kFull || gidx < groups) *reinterpret_cast<uint2*>(q + 8 * (int64_t)gidx) = bytes[i];
  }
  if (KIND == kNormAnyEps && p.late_sum) {
#pragma unroll 1
    for (int gidx = t; gidx < groups; gidx += step) {
      f2 h[4], u[4];
      unpack8(load8(x + 8 * (int64_t)gidx), h);
      unpack8(load8(o + 8 * (int64_t)gidx), u);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = add2(h[j], u[j]);
      store8(so + 8 * (int64_t)gidx, h);
    }
  }
}

// Rows wider than a CTA's registers hold, with the alignment of quant_rows_kernel: two passes over the
// row, the second one from L2, a group of eight per thread and step (2048 x 53248 bf16 as it is: 89 us,
// 273 element by element).  (h goes to sum_out in the second
// pass: the first one may not yet have read its place.)
template <typename TIn, typename TW, int KIND>
__global__ void __launch_bounds__(1024) quant_rows_wide_kernel(const Params p) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  const int t = threadIdx.x, lane = t & 31, groups = (int)(p.cols >> 3);
  const TW* w = static_cast<const TW*>(p.weight);
  after_the_kernel_before();
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const TIn* x = static_cast<const TIn*>(p.x) + r * p.ldx;
    const TIn* o = p.other ? static_cast<const TIn*>(p.other) + r * p.ldo : nullptr;
    TIn* so = p.sum_out ? static_cast<TIn*>(p.sum_out) + r * p.lds : nullptr;
    f2 g[1][4], sums = 0;
    float top = 0.f;
    auto values = [&](int64_t c, bool store, f2& sq, float& mx) {
      const Eight<TIn> ex = load8(x + c);
      Eight<TIn> eo = ex;
      if (KIND != FRISK_QUANT_PLAIN && o) eo = load8(o + c);
      group_values<TIn, KIND>(
          ex, eo, o != nullptr,
          [&](f2 (&v)[4]) {
            if (w) unpack8(load8_shared_by_rows(w + c), v);
            return w != nullptr;
          },
          [&](const f2 (&h)[4]) {
            if (store && so) store8(so + c, h);
          },
          g[0], sq, mx);
    };
#pragma unroll 2
    for (int i = t; i < groups; i += 1024) values(8 * (int64_t)i, false, sums, top);
    float sum = lo2(sums) + hi2(sums);
    uint32_t mx = __float_as_uint(top);
    row_fold<KIND>(sum, mx, s_sum, s_max, t >> 5, lane, 0, 32);
    if constexpr (KIND == kNormAnyEps) {
      if (small_norm(sum, mx, p)) {
        small_norm_row<TIn, TW>(p, r);
        __syncthreads();
        continue;
      }
    }
    const Factor f = row_factor<KIND>(sum, mx, p.cols, p.eps, p.q_type, t == 0, p.scale + r);
    uint8_t* q = static_cast<uint8_t*>(p.q) + r * p.ldq;
#pragma unroll 2
    for (int i = t; i < groups; i += 1024) {
      values(8 * (int64_t)i, true, sums, top);
      multiply<kExactQ<TIn, KIND>, 1>(g, f);
      uint2 bytes[1];
      encode_groups<1>(g, p.q_type, bytes);
      *reinterpret_cast<uint2*>(q + 8 * (int64_t)i) = bytes[0];
    }
    __syncthreads();   // the shared arrays are written again by the next row
  }
}

// ---- the same for rows at any alignment and width -----------------------------------------------
// What it takes is its instructions (35 per element, 52 when every element was accessed by itself): 1023 x
// 5001 f16 norm 8.9 us, 12.9 element by element; 2047 x 4095 bf16 out of rows of 6150 8.1 us (20).
// Memory is still touched in aligned words of 16 bytes (8 for q): a group that starts inside a word is
// shifted together from the words it lies in, and a stored word from the end of one lane's group and
// the start of the next one's.

// The words of v from byte `by` on (below 16): W of them, out of W + 4.
template <int W>
__device__ __forceinline__ void shift_words(uint32_t (&v)[W + 4], uint32_t by) {
#pragma unroll
  for (int i = 0; i < W + 2; ++i) v[i] = by & 8u ? v[i + 2] : v[i];
#pragma unroll
  for (int i = 0; i < W + 1; ++i) v[i] = by & 4u ? v[i + 1] : v[i];
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] = __funnelshift_r(v[i], v[i + 1], 8u * (by & 3u));
}

// Elements c .. c + 7 of a row; zeros past its end.  A group whose words reach out of the row is read
// element by element: what lies there may be no part of any buffer, or another row that is being
// replaced by its sum at that moment.
template <typename T>
struct Ragged {
  uint32_t w[2 * sizeof(T) + 4];
  uint32_t by;   // where the group starts in w
};
template <typename T>
__device__ __forceinline__ void load8_ragged(Ragged<T>& g, const T* row, int c, int cols) {
  constexpr int W = 2 * sizeof(T);   // 32-bit words of a group
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + c);
  g.by = (uint32_t)(at & 15u);
  const uint4* p = reinterpret_cast<const uint4*>(at - g.by);
  // (elements in front of the group in its first word, and behind it in the last one)
  const int before = (int)g.by / (int)sizeof(T), after = 16 / (int)sizeof(T) - before;
  if (c >= before && c + 8 + after <= cols) {
#pragma unroll
    for (int i = 0; i < W / 4 + 1; ++i) {
      asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(g.w[4 * i]), "=r"(g.w[4 * i + 1]), "=r"(g.w[4 * i + 2]), "=r"(g.w[4 * i + 3])
                   : "l"(p + i)
                   : "memory");
    }
    return;
  }
  g.by = 0;
  constexpr int kPer = 4 / (int)sizeof(T);   // elements of a word
#pragma unroll
  for (int i = 0; i < W; ++i) {
    uint32_t x = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (c + i * kPer + k < cols) {
        const T e = row[c + i * kPer + k];
        uint32_t bits;
        if constexpr (sizeof(T) == 2) bits = *reinterpret_cast<const uint16_t*>(&e);
        else bits = *reinterpret_cast<const uint32_t*>(&e);
        x |= bits << (16 * k);
      }
    }
    g.w[i] = x;
  }
}
template <typename T>
__device__ __forceinline__ Eight<T> take8(Ragged<T>& g) {
  constexpr int W = 2 * sizeof(T);
  shift_words<W>(g.w, g.by);
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < W / 4; ++i) r.w[i] = make_uint4(g.w[4 * i], g.w[4 * i + 1], g.w[4 * i + 2], g.w[4 * i + 3]);
  return r;
}

// A warp's 32 x NV neighbouring groups into a row: lane L's i-th group, w[i] (elements of ES bytes), is
// elements c0 + 8 (32 i + L) and on.  A lane stores the units (aligned words) that end in its group; the
// first of them begins in the group to the left.  What no unit covers -- the first group's start, the
// last one's end, the end of the row -- goes element by element, a group at a time.
template <int ES, int NV>
__device__ __forceinline__ void store_ragged(unsigned char* row, int c0, int cols, const uint32_t (&w)[NV][2 * ES], int lane) {
  constexpr int W = 2 * ES;                 // words of a group
  constexpr int U = W < 4 ? W : 4;          // words of a unit
  constexpr int EU = 4 * U / ES;            // elements of a unit
  const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(row) % (4 * U));   // groups are whole units long
  const int o = (int)off / ES;              // elements of the left group in a group's first unit
  uint32_t carry[U] = {};                   // lane 0: the end of lane 31's group before
  uint32_t need[NV];                        // elements of the group that no unit covers
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + 8 * (32 * i + lane);
    const int have = max(0, min(8, cols - c)), have_next = cols - (c + 8);
    uint32_t v[W + 4] = {};
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint32_t left = __shfl_sync(0xffffffffu, w[i][W - U + k], (lane + 31) & 31);
      v[k] = lane == 0 ? carry[k] : left;
      carry[k] = left;
    }
#pragma unroll
    for (int k = 0; k < W; ++k) v[U + k] = w[i][k];
    if (off == 0) {
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = w[i][k];
    } else {   // from byte 4 U - off on (1 .. 4 U - 1)
      shift_words<W>(v, 4 * U - off);
    }
    unsigned char* first = row + (int64_t)c * ES - off;
    uint32_t covered = 0;
#pragma unroll
    for (int u = 0; u < W / U; ++u) {
      if ((u > 0 || lane > 0 || i > 0 || o == 0) && (u + 1) * EU - o <= have) {
        if constexpr (U == 4) *reinterpret_cast<uint4*>(first + 16 * u) = make_uint4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
        else *reinterpret_cast<uint2*>(first) = make_uint2(v[0], v[1]);
        covered |= (((1u << EU) - 1u) << (u * EU)) >> o;
      }
    }
    // (the right group's first unit)
    if (o > 0 && (lane < 31 || i < NV - 1) && have_next >= EU - o) covered |= 0xffu << (8 - o);
    need[i] = ((1u << have) - 1u) & ~covered;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    uint32_t lanes = __ballot_sync(0xffffffffu, need[i] != 0);
    while (lanes) {
      const int src = __ffs(lanes) - 1;
      lanes &= lanes - 1;
      const uint32_t which = __shfl_sync(0xffffffffu, need[i], src);
      uint32_t x = 0;   // the word of the group with element `lane`
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const uint32_t y = __shfl_sync(0xffffffffu, w[i][k], src);
        if (lane * ES / 4 == k) x = y;
      }
      if (lane < 8 && (which >> lane & 1u)) {
        unsigned char* dst = row + (int64_t)(c0 + 8 * (32 * i + src) + lane) * ES;
        x >>= 8 * (lane * ES & 3);
        if constexpr (ES == 1) *dst = (uint8_t)x;
        else if constexpr (ES == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)x;
        else *reinterpret_cast<uint32_t*>(dst) = x;
      }
    }
  }
}

template <typename TIn, typename TW, int KIND, int NV>
__global__ void __launch_bounds__(1024) quant_rows_unaligned_kernel(const Params p) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  const int t = threadIdx.x, lane = t & 31, wpr = blockDim.x >> 5;
  const int slot = __shfl_sync(0xffffffffu, threadIdx.y, 0), warp_in_row = __shfl_sync(0xffffffffu, t >> 5, 0);
  const int64_t r = (int64_t)blockIdx.x * blockDim.y + slot;
  const bool live = r < p.rows;
  const int cols = live ? (int)p.cols : 0, c0 = warp_in_row * 256 * NV;   // the warp's first element
  const TW* w = static_cast<const TW*>(p.weight);
  const TIn* x = static_cast<const TIn*>(p.x) + r * p.ldx;
  const TIn* o = p.other ? static_cast<const TIn*>(p.other) + r * p.ldo : nullptr;
  const bool w_aligned = (reinterpret_cast<uintptr_t>(w) & 15) == 0;

  after_the_kernel_before();
  Ragged<TIn> rx[NV], ro[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + 8 * (32 * i + lane);
    load8_ragged(rx[i], x, c, cols);
    if (KIND != FRISK_QUANT_PLAIN && o) load8_ragged(ro[i], o, c, cols);
  }
  f2 g[NV][4];
  f2 sums = 0;
  float top = 0.f;
  uint32_t hw[NV][2 * sizeof(TIn)];   // h as stored
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    Eight<TIn> ex = take8(rx[i]), eo = ex;
    if (KIND != FRISK_QUANT_PLAIN && o) eo = take8(ro[i]);
    group_values<TIn, KIND>(
        ex, eo, o != nullptr,
        [&](f2 (&v)[4]) {
          const int c = c0 + 8 * (32 * i + lane);
          if (w && w_aligned && c + 8 <= cols) {
            unpack8(load8_shared_by_rows(w + c), v);
          } else if (w) {
            Ragged<TW> rw;
            load8_ragged(rw, w, c, cols);
            unpack8(take8(rw), v);
          }
          return w != nullptr;
        },
        [&](const f2 (&h)[4]) {
          Eight<TIn> e;
          store8(reinterpret_cast<TIn*>(e.w), h);
#pragma unroll
          for (int k = 0; k < (int)sizeof(TIn) / 2; ++k) {
            hw[i][4 * k] = e.w[k].x;
            hw[i][4 * k + 1] = e.w[k].y;
            hw[i][4 * k + 2] = e.w[k].z;
            hw[i][4 * k + 3] = e.w[k].w;
          }
        },
        g[i], sums, top);
  }
  auto store_sum = [&] {
    if (p.sum_out)
      store_ragged<sizeof(TIn), NV>(reinterpret_cast<unsigned char*>(static_cast<TIn*>(p.sum_out) + r * p.lds), c0, cols, hw, lane);
  };
  if (KIND == FRISK_QUANT_RMSNORM && p.sum_out) {
    // h may take the place of x or of the residual, and what this warp stores lies in words that the
    // row's other warps read: they have to have read them
    __syncthreads();
    store_sum();
  }
  float sum = lo2(sums) + hi2(sums);
  uint32_t mx = __float_as_uint(top);
  row_fold<KIND>(sum, mx, s_sum, s_max, slot * wpr + warp_in_row, lane, slot, wpr);
  if constexpr (KIND == kNormAnyEps) {
    if (small_norm(sum, mx, p)) return small_norm_row<TIn, TW>(p, r);   // (the CTA has one row)
    store_sum();   // (the row's reads are behind the fold)
  }
  if (!live) return;
  multiply<kExactQ<TIn, KIND>, NV>(g, row_factor<KIND>(sum, mx, p.cols, p.eps, p.q_type, t == 0, p.scale + r));
  uint2 bytes[NV];
  encode_groups<NV>(g, p.q_type, bytes);
  uint32_t qw[NV][2];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    qw[i][0] = bytes[i].x;
    qw[i][1] = bytes[i].y;
  }
  store_ragged<1, NV>(static_cast<unsigned char*>(p.q) + r * p.ldq, c0, cols, qw, lane);
}

// ---- many gated rows: streamed through shared memory ---------------------------------------------
// The gate costs enough arithmetic that rows in registers alternate between loading and computing
// (4096 x 16384 bf16: 59.5 us; streamed 55 - 57 us; the other kinds are faster in registers: norm 8192 x
// 8192 with residual 79 against 80 us, fp32 8192 x 8192 as it is 50 against 55).
// One CTA per SM walks the rows blockIdx.x, + gridDim.x, ...; bulk copies bring them into a ring of
// `stages` whole rows (both operands), several ahead of the arithmetic, so that the memory is read
// without a pause while rows are folded, scaled and stored.  The CTA is blockDim.y teams of
// blockDim.x threads; a team takes every blockDim.y-th row, so that one team's barrier is another's
// arithmetic.  The row's stage is refilled as soon as its team has read it into registers.
// Waits are bounded: a team whose copies do not arrive gives up, sets the status word and leaves NaN scales
// and zeros for its rows from there on; the CTA stays until the copies that were asked for have landed.
constexpr int kMaxRowStages = 16;
constexpr int64_t kRowWaitCycles = 1ll << 29;   // about 0.3 s
constexpr int64_t kPollCycles = 1ll << 22;      // a poll counts as this at most
constexpr int32_t kStatusRowsTimeout = 16;      // (the gemm kernels use the bits below)

__device__ __forceinline__ uint32_t load_tag(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store_tag(uint32_t addr, uint32_t v) {
  asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// Polls a phase of the barrier `bar` until it is over and `also()` holds, for `limit` cycles: cycles of polling,
// so that a CTA which did not run for a while (its context switched out) has not used its limit up, and with
// a last look after them.
template <typename Also>
__device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity, int64_t limit, Also also) {
  if (also() && frisk::ptx::mbar_test_wait(bar, parity)) return true;
  for (long long last = clock64(); limit > 0;) {
    if (also() && frisk::ptx::mbar_try_wait(bar, parity)) return true;
    const long long now = clock64();
    limit -= min((int64_t)(now - last), kPollCycles);
    last = now;
  }
  return also() && frisk::ptx::mbar_test_wait(bar, parity);
}
// Waits for row `row` of this CTA in the stage behind `bar`.  A phase's parity alone does not say
// which row it is: a team may be ahead of the one that has yet to read the stage's row before, and
// would take the phase before that for its own.  So the stage's tag, set when a row is asked for,
// comes first; from then on the barrier is in that row's phase or past it.
__device__ __forceinline__ bool wait_row(uint32_t bar, uint32_t parity, uint32_t tag, uint32_t row, int64_t limit) {
  return poll(bar, parity, limit, [&] { return load_tag(tag) == row; });
}
// Barrier of one team (hardware barrier 1 + team): true if any thread brings `bad`.
__device__ __forceinline__ bool team_barrier(int team, int threads, bool bad) {
  uint32_t any;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(any)
      : "r"(1 + team), "r"(threads), "r"((uint32_t)bad)
      : "memory");
  return any != 0;
}
template <typename T>
__device__ __forceinline__ Eight<T> load8_smem(uint32_t addr) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.w[i].x), "=r"(r.w[i].y), "=r"(r.w[i].z), "=r"(r.w[i].w)
                 : "r"(addr + 16 * i)
                 : "memory");
  return r;
}

template <typename TIn, int NV, bool kFull>
__global__ void __launch_bounds__(1024, 1) quant_gated_stream_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t bars[kMaxRowStages];
  __shared__ uint32_t tags[kMaxRowStages];   // which of the CTA's rows a stage was last asked for
  __shared__ uint32_t s_max[2][32], gave_up;
  const int t = threadIdx.x, step = blockDim.x, lane = t & 31, wpr = step >> 5;
  const int teams = blockDim.y, stages = p.stages;
  const int team = __shfl_sync(0xffffffffu, threadIdx.y, 0), warp = team * wpr + (t >> 5);
  const int groups = (int)(p.cols >> 3);
  const uint32_t bytes = (uint32_t)p.cols * (uint32_t)sizeof(TIn);   // of one operand's row
  const uint32_t stage_bytes = 2 * bytes;
  const uint32_t ring0 = frisk::ptx::smem_u32(ring), bar0 = frisk::ptx::smem_u32(bars);
  const uint32_t tag0 = frisk::ptx::smem_u32(tags);
  const int64_t n = (p.rows - blockIdx.x + gridDim.x - 1) / gridDim.x;   // rows of this CTA

  auto fetch = [&](int64_t j, int stage) {   // one thread: row j of this CTA into a stage
    const int64_t r = blockIdx.x + j * gridDim.x;
    const uint32_t dst = ring0 + stage * stage_bytes, bar = bar0 + 8 * stage;
    store_tag(tag0 + 4 * stage, (uint32_t)j);
    frisk::ptx::mbar_arrive_expect_tx(bar, stage_bytes);
    frisk::ptx::bulk_load(dst, static_cast<const TIn*>(p.x) + r * p.ldx, bytes, bar);
    frisk::ptx::bulk_load(dst + bytes, static_cast<const TIn*>(p.other) + r * p.ldo, bytes, bar);
  };
  if (threadIdx.x == 0 && threadIdx.y == 0) {
    for (int s = 0; s < stages; ++s) {
      frisk::ptx::mbar_init(bar0 + 8 * s, 1);
      tags[s] = 0xffffffffu;   // (n is below that: checked when launching)
    }
    gave_up = 0;
    frisk::ptx::fence_mbar_init();
  }
  after_the_kernel_before();
  if (threadIdx.x == 0 && threadIdx.y == 0) {
    for (int s = 0; s < stages && s < n; ++s) fetch(s, s);
  }
  __syncthreads();

  int stage = team;
  uint32_t phase = 0;
  int buf = 0;
  for (int64_t j = team; j < n; j += teams) {   // teams <= stages
    const int64_t r = blockIdx.x + j * gridDim.x;
    const bool ok = wait_row(bar0 + 8 * stage, phase, tag0 + 4 * stage, (uint32_t)j, p.wait_cycles);
    const uint32_t at = ring0 + stage * stage_bytes;
    f2 g[NV][4];
    f2 sums = 0;
    float top = 0.f;
    if (ok) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int gidx = t + i * step;
        if (kFull || gidx < groups) {
          const uint32_t e = at + (uint32_t)gidx * 8u * (uint32_t)sizeof(TIn);
          group_values<TIn, FRISK_QUANT_SILU_MUL>(load8_smem<TIn>(e), load8_smem<TIn>(e + bytes), true,
                                                  [](f2 (&)[4]) { return false; }, [](const f2 (&)[4]) {}, g[i], sums, top);
        }
      }
    }
    float sum = 0.f;   // (of the norm)
    uint32_t mx = __float_as_uint(top);
    warp_fold<FRISK_QUANT_SILU_MUL>(sum, mx);
    if (lane == 0) s_max[buf][warp] = mx;
    if (team_barrier(team, step, !ok)) {
      if (t == 0) {
        gave_up = 1;
        if (p.status) atomicOr(p.status, kStatusRowsTimeout);
      }
      for (; j < n; j += teams) {
        const int64_t left = blockIdx.x + j * gridDim.x;
        if (t == 0) p.scale[left] = __uint_as_float(0x7fc00000u);
        for (int gidx = t; gidx < groups; gidx += step)
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.q) + left * p.ldq + 8 * gidx) = make_uint2(0, 0);
      }
      break;
    }
    // every thread of the team has read the stage
    if (t == 0 && j + stages < n) fetch(j + stages, stage);
    mx = lane < wpr ? s_max[buf][team * wpr + lane] : 0u;
    warp_fold<FRISK_QUANT_SILU_MUL>(sum, mx);
    multiply<false, NV>(g, row_factor<FRISK_QUANT_SILU_MUL>(sum, mx, p.cols, p.eps, p.q_type, t == 0, p.scale + r));
    uint8_t* q = static_cast<uint8_t*>(p.q) + r * p.ldq;
    uint2 eight[NV];
    encode_groups<NV>(g, p.q_type, eight);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int gidx = t + i * step;
      if (kFull || gidx < groups) *reinterpret_cast<uint2*>(q + 8 * gidx) = eight[i];
    }
    buf ^= 1;
    stage += teams;
    if (stage >= stages) {
      stage -= stages;
      phase ^= 1u;
    }
  }
  __syncthreads();   // no more rows are asked for
  if (gave_up && threadIdx.x == 0 && threadIdx.y == 0) {   // the last row of every stage lands before the CTA leaves
    for (int s = 0; s < stages; ++s) {
      const uint32_t row = load_tag(tag0 + 4 * s);
      if (row == 0xffffffffu) continue;
      poll(bar0 + 8 * s, row / stages & 1u, kRowWaitCycles, [] { return true; });
    }
  }
}

}  // namespace frisk_quant
