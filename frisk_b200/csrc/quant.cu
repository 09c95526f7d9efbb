// Host side of the 8-bit row makers: argument checks, launches, and the C ABI entry points declared
// in include/frisk_b200.h.
#include "quant.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <string>

#include "../../include/frisk_b200.h"
#include "abi_internal.h"

namespace {

using frisk_quant::Params;

int in_bytes(int dt) { return dt == FRISK_DT_F32 ? 4 : (dt == FRISK_DT_F16 || dt == FRISK_DT_BF16) ? 2 : 0; }
bool is_8bit(int dt) { return dt == FRISK_DT_I8 || dt == FRISK_DT_E4M3 || dt == FRISK_DT_E5M2; }

int fail(int code, const char* text) {
  frisk_internal_set_error(text);
  return code;
}
int fail_cuda(cudaError_t e, const char* what) {
  frisk_internal_set_error((std::string(what) + ": " + cudaGetErrorString(e)).c_str());
  return FRISK_ERR_CUDA;
}

int check_desc(const frisk_quant_desc& d) {
  if (d.rows < 0 || d.cols <= 0) return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: rows must not be negative, cols must be positive");
  if (d.kind < FRISK_QUANT_PLAIN || d.kind > FRISK_QUANT_SILU_MUL) return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: unknown kind");
  if (!in_bytes(d.in_type)) return fail(FRISK_ERR_UNSUPPORTED, "quant: the input type must be f32, f16 or bf16");
  if (!is_8bit(d.q_type)) return fail(FRISK_ERR_UNSUPPORTED, "quant: the output type must be i8, e4m3 or e5m2");
  if (d.kind == FRISK_QUANT_RMSNORM) {
    if (d.weight_type != d.in_type && d.weight_type != FRISK_DT_F32)
      return fail(FRISK_ERR_UNSUPPORTED, "quant: the weight's type must be the input's or f32");
    if (!(d.eps >= 0.f) || std::isinf(d.eps)) return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: eps must be finite and not negative");
  }
  if (d.cols >= (1ll << 31)) return fail(FRISK_ERR_TOO_LARGE, "quant: 2^31 columns or more");
  // every offset in bytes has to fit 63 bits (the widest packed pitch is 2 * cols of four bytes)
  for (int64_t ld : {d.ldx, d.ldo, d.lds, d.ldq, 2 * d.cols})
    if (ld > 0 && (unsigned __int128)d.rows * (unsigned __int128)ld >= ((unsigned __int128)1 << 60))
      return fail(FRISK_ERR_TOO_LARGE, "quant: rows times a pitch is 2^60 or more");
  // (silu_mul with gate and up in one buffer needs 2 * cols; checked when the pointers are known)
  if ((d.ldx && d.ldx < d.cols) || (d.ldo && d.ldo < d.cols) || (d.lds && d.lds < d.cols) || (d.ldq && d.ldq < d.cols))
    return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: a pitch is shorter than a row");
  return FRISK_OK;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether every row of a buffer at `ptr` with row pitch `ld` (elements of `es` bytes) starts on a
// multiple of `to` bytes.  A buffer that is not there does.
bool rows_on(const void* ptr, int64_t ld, int es, int to) {
  return !ptr || (reinterpret_cast<uintptr_t>(ptr) % to == 0 && (ld * es) % to == 0);
}

constexpr int kMaxGroups = 4;   // groups of eight elements a thread holds at most
constexpr size_t kRingBytes = 226 * 1024;   // shared memory of a CTA for rows in flight, but for a little

// Opts a kernel into kRingBytes of shared memory, once per device.
template <typename TIn, bool kFull>
cudaError_t allow_ring(int device) {
  static bool done[64] = {};
  const bool tracked = device >= 0 && device < 64;
  if (tracked && __atomic_load_n(&done[device], __ATOMIC_ACQUIRE)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(frisk_quant::quant_gated_stream_kernel<TIn, kMaxGroups, kFull>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes);
  if (e == cudaSuccess && tracked) __atomic_store_n(&done[device], true, __ATOMIC_RELEASE);
  return e;
}

cudaError_t go(void (*kern)(const Params), int64_t ctas, dim3 threads, size_t smem, const Params& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename TIn, typename TW, int KIND>
cudaError_t launch(Params p, int device, int sms, cudaStream_t st) {
  const int es = sizeof(TIn);
  const bool aligned = p.cols % 8 == 0 && rows_on(p.x, p.ldx, es, 16) && rows_on(p.other, p.ldo, es, 16) &&
                       rows_on(p.sum_out, p.lds, es, 16) && rows_on(p.q, p.ldq, 1, 8) && rows_on(p.weight, 0, 1, 16);
  constexpr int64_t kMaxCtas = 0x7fffffff;
  if (aligned && p.cols > 8 * 1024 * kMaxGroups)   // more than registers hold
    return go(frisk_quant::quant_rows_wide_kernel<TIn, TW, KIND>, std::min(p.rows, kMaxCtas), dim3(1024), 0, p, st);
  if (p.cols > 8 * 1024 * kMaxGroups || p.rows > kMaxCtas) {   // ... or rows than a grid has CTAs
    return go(frisk_quant::quant_rows_generic_kernel<TIn, TW, KIND>, std::min(p.rows, kMaxCtas), dim3(256), 0, p, st);
  }
  // Rows that may have to be looked at again (small_norm_row): a CTA each, and a sum in place of x or of
  // the residual waits for that.
  constexpr bool small_norms = KIND == frisk_quant::kNormAnyEps;
  p.late_sum = small_norms && p.sum_out && (p.sum_out == p.x || p.sum_out == p.other);
  const int64_t groups = ceil_div(p.cols, 8);
  if constexpr (KIND == FRISK_QUANT_SILU_MUL) {
    // Streamed from two fillings of all SMs' rings on, 68 MB of input.  In registers -> streamed, us: bf16 of
    // 8192 columns 50 MB 12.6 -> 14.9, 67 MB 15.9 -> 17.3, 134 MB 29.5 -> 29.7, 268 MB 54.9 -> 54.3; of 16384
    // columns 50 MB 14.2 -> 16.1, 67 MB 17.3 -> 18.0, 134 MB 31.1 -> 30.1, 268 MB 59.5 -> 54.9; with one
    // team a CTA, 20480 columns, 34 MB 12.3 -> 12.8, 67 MB 22.9 -> 20.8, 268 MB 78.8 -> 64.7; fp32 of 8192 columns
    // 67 MB 24.1 -> 20.3, 268 MB 58.0 -> 47.3.
    const size_t row = 2 * (size_t)p.cols * es;
    const int stages = (int)std::min<size_t>(frisk_quant::kMaxRowStages, kRingBytes / row);
    const int wpr = (int)ceil_div(groups, 32 * kMaxGroups);
    if (aligned && wpr >= 4 && stages >= 2 && p.rows >= 4 * (int64_t)sms &&
        (size_t)p.rows * row >= 2 * kRingBytes * sms) {
      const int teams = std::min(32 / wpr, stages);
      p.stages = stages;
      const bool full = p.cols == 256ll * kMaxGroups * wpr;
      auto kern = full ? frisk_quant::quant_gated_stream_kernel<TIn, kMaxGroups, true>
                       : frisk_quant::quant_gated_stream_kernel<TIn, kMaxGroups, false>;
      if (const cudaError_t e = full ? allow_ring<TIn, true>(device) : allow_ring<TIn, false>(device)) return e;
      return go(kern, sms, dim3(32 * wpr, teams), stages * row, p, st);
    }
  }
  // Many rows: four groups a thread, for loads in flight (norms and gates of fp32 rows spill 80 - 210 bytes
  // with them); off the 16-byte grid two, but of 16-bit rows as they are (1023 x 5001 f16
  // norm with one, two, four: 15.5, 8.9, 11.1 us; 8192 x 4095 bf16 as it is 43.3, 35.8, 30.5).  Few rows: one, so
  // that a row is spread over as many threads as there are.
  const bool few = p.rows < 2 * (int64_t)sms;
  int nv = few ? 1 : aligned || (es == 2 && KIND == FRISK_QUANT_PLAIN) ? kMaxGroups : 2;
  while (ceil_div(groups, 32 * nv) > 32) nv *= 2;
  while (nv > 1 && 32 * (nv / 2) >= groups) nv /= 2;   // short rows: no more than a warp can use
  const int wpr = (int)ceil_div(groups, 32 * nv), rows_per_cta = small_norms ? 1 : std::max(1, 8 / wpr);
  const int64_t ctas = ceil_div(p.rows, rows_per_cta);
  const dim3 threads(32 * wpr, rows_per_cta);
  const bool full = p.cols == 256ll * nv * wpr && p.rows % rows_per_cta == 0;
  using namespace frisk_quant;
  void (*kern)(const Params);
  if (!aligned)
    kern = nv == 1   ? quant_rows_unaligned_kernel<TIn, TW, KIND, 1>
           : nv == 2 ? quant_rows_unaligned_kernel<TIn, TW, KIND, 2>
                     : quant_rows_unaligned_kernel<TIn, TW, KIND, 4>;
  else if (full && !small_norms)
    kern = nv == 1   ? quant_rows_kernel<TIn, TW, KIND, 1, true>
           : nv == 2 ? quant_rows_kernel<TIn, TW, KIND, 2, true>
                     : quant_rows_kernel<TIn, TW, KIND, 4, true>;
  else
    kern = nv == 1   ? quant_rows_kernel<TIn, TW, KIND, 1, false>
           : nv == 2 ? quant_rows_kernel<TIn, TW, KIND, 2, false>
                     : quant_rows_kernel<TIn, TW, KIND, 4, false>;
  return go(kern, ctas, threads, 0, p, st);
}

template <typename TIn>
cudaError_t launch_kind(const frisk_quant_desc& d, const Params& p, int device, int sms, cudaStream_t st) {
  switch (d.kind) {
    case FRISK_QUANT_PLAIN: return launch<TIn, TIn, FRISK_QUANT_PLAIN>(p, device, sms, st);
    case FRISK_QUANT_SILU_MUL: return launch<TIn, TIn, FRISK_QUANT_SILU_MUL>(p, device, sms, st);
    default: break;
  }
  if (d.eps < frisk_quant::kSmallNorm) {
    return d.weight_type == d.in_type ? launch<TIn, TIn, frisk_quant::kNormAnyEps>(p, device, sms, st)
                                      : launch<TIn, float, frisk_quant::kNormAnyEps>(p, device, sms, st);
  }
  return d.weight_type == d.in_type ? launch<TIn, TIn, FRISK_QUANT_RMSNORM>(p, device, sms, st)
                                    : launch<TIn, float, FRISK_QUANT_RMSNORM>(p, device, sms, st);
}

}  // namespace

std::atomic<int64_t> g_wait_cycles{frisk_quant::kRowWaitCycles};

extern "C" {

int64_t frisk_internal_quant_wait_cycles(int64_t cycles) { return g_wait_cycles.exchange(cycles); }

int frisk_b200_quant_run(const frisk_quant_desc* desc, const frisk_quant_args* args) {
  return frisk_b200_quant_run_status(desc, args, nullptr);
}

int frisk_b200_quant_run_status(const frisk_quant_desc* desc, const frisk_quant_args* args, int32_t* device_status) {
  if (!desc || !args) return FRISK_ERR_INVALID_ARGUMENT;
  const frisk_quant_desc& d = *desc;
  if (int rc = check_desc(d)) return rc;
  const bool norm = d.kind == FRISK_QUANT_RMSNORM, gated = d.kind == FRISK_QUANT_SILU_MUL;
  if ((!norm && (args->residual || args->weight || args->sum_out)) || (!gated && args->up))
    return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: an operand that this kind does not take was given");
  if (args->sum_out && !args->residual) return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: sum_out without a residual");
  Params p{};
  p.rows = d.rows;
  p.cols = d.cols;
  const bool halves = gated && !args->up;   // gate and up side by side in one buffer
  p.ldx = d.ldx ? d.ldx : (halves ? 2 : 1) * d.cols;
  if (halves && p.ldx < 2 * d.cols) return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: a pitch is shorter than gate and up together");
  p.ldo = halves ? p.ldx : d.ldo ? d.ldo : d.cols;
  p.lds = d.lds ? d.lds : d.cols;
  p.ldq = d.ldq ? d.ldq : d.cols;
  p.eps = d.eps;
  p.q_type = d.q_type;
  p.status = device_status;
  p.wait_cycles = g_wait_cycles.load(std::memory_order_relaxed);
  if (d.rows == 0) return FRISK_OK;
  if (!args->x || !args->q || !args->scale) return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: null x, q or scale");
  const int es = in_bytes(d.in_type), ws = in_bytes(norm ? d.weight_type : d.in_type);
  p.x = args->x;
  p.other = norm ? args->residual : halves ? static_cast<const char*>(args->x) + d.cols * es : args->up;
  p.weight = args->weight;
  p.sum_out = args->sum_out;
  p.q = args->q;
  p.scale = args->scale;
  auto off = [](const void* ptr, int a) { return reinterpret_cast<uintptr_t>(ptr) % (unsigned)a != 0; };
  if (off(p.x, es) || off(p.other, es) || off(p.weight, ws) || off(p.sum_out, es) || off(p.scale, 4) || off(p.status, 4))
    return fail(FRISK_ERR_MISALIGNED, "quant: a pointer is not aligned to its element size");
  // the sum may replace x or the residual, element for element
  if ((p.sum_out == p.x && p.sum_out && p.lds != p.ldx) || (p.sum_out == p.other && p.sum_out && p.lds != p.ldo))
    return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: sum_out in place of x or the residual needs the same pitch");
  // q and scale lie by themselves (the caller answers for partial overlaps)
  for (const void* b : {p.x, p.other, p.weight, (const void*)p.sum_out, (const void*)p.status})
    if (b == p.q || b == p.scale || p.q == p.scale)
      return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: q and scale must not be one of the other buffers");
  int prev = -1;
  cudaError_t e;
  if (d.device >= 0) {
    if ((e = cudaGetDevice(&prev)) != cudaSuccess) return fail_cuda(e, "cudaGetDevice");
    if (prev != d.device && (e = cudaSetDevice(d.device)) != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  }
  cudaStream_t st = static_cast<cudaStream_t>(args->stream);
  int dev = d.device, sms = 0;
  e = dev >= 0 ? cudaSuccess : cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) {
    switch (d.in_type) {
      case FRISK_DT_F32: e = launch_kind<float>(d, p, dev, sms, st); break;
      case FRISK_DT_F16: e = launch_kind<__half>(d, p, dev, sms, st); break;
      default: e = launch_kind<__nv_bfloat16>(d, p, dev, sms, st); break;
    }
  }
  if (prev >= 0 && prev != d.device) cudaSetDevice(prev);
  if (e != cudaSuccess) return fail_cuda(e, "quant kernel launch");
  return FRISK_OK;
}

int frisk_b200_quant_run_host(const frisk_quant_desc* desc, const frisk_quant_args* args) {
  if (!desc || !args) return FRISK_ERR_INVALID_ARGUMENT;
  frisk_quant_desc d = *desc;
  if (int rc = check_desc(d)) return rc;
  if (d.rows == 0) return FRISK_OK;
  if (!args->x || !args->q || !args->scale) return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: null x, q or scale");
  const bool norm = d.kind == FRISK_QUANT_RMSNORM, gated = d.kind == FRISK_QUANT_SILU_MUL;
  const int es = in_bytes(d.in_type);
  // only the elements of each row travel: a host buffer may end behind the last row's
  const int64_t xw = (gated && !args->up ? 2 : 1) * d.cols;
  if (d.ldx && d.ldx < xw) return fail(FRISK_ERR_INVALID_ARGUMENT, "quant: a pitch is shorter than gate and up together");
  struct Buf {
    void* dev;
    const void* in;   // host source, or nullptr
    void* out;        // host destination, or nullptr
    int64_t ld, width, rows;
    int es;
  };
  const void* other = norm ? args->residual : gated ? args->up : nullptr;
  enum { X, O, Wt, S, Q, Sc, St, N };
  int32_t status = 0;
  Buf b[N] = {
      {nullptr, args->x, nullptr, d.ldx ? d.ldx : xw, xw, d.rows, es},
      {nullptr, other, nullptr, d.ldo ? d.ldo : d.cols, d.cols, d.rows, es},
      {nullptr, norm ? args->weight : nullptr, nullptr, d.cols, d.cols, 1, norm ? in_bytes(d.weight_type) : es},
      {nullptr, nullptr, norm ? args->sum_out : nullptr, d.lds ? d.lds : d.cols, d.cols, d.rows, es},
      {nullptr, nullptr, args->q, d.ldq ? d.ldq : d.cols, d.cols, d.rows, 1},
      {nullptr, nullptr, args->scale, 1, 1, d.rows, 4},
      {nullptr, &status, &status, 1, 1, 1, 4},
  };
  int prev = -1;
  cudaError_t e = cudaSuccess;
  if (d.device >= 0) {
    if ((e = cudaGetDevice(&prev)) != cudaSuccess) return fail_cuda(e, "cudaGetDevice");
    if (prev != d.device && (e = cudaSetDevice(d.device)) != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  }
  cudaStream_t st = nullptr;
  e = cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking);
  for (Buf& u : b) {   // packed on the device
    if (e != cudaSuccess || (!u.in && !u.out)) continue;
    e = cudaMalloc(&u.dev, (size_t)u.rows * u.width * u.es);
    if (e == cudaSuccess && u.in)
      e = cudaMemcpy2DAsync(u.dev, u.width * u.es, u.in, u.ld * u.es, u.width * u.es, u.rows, cudaMemcpyHostToDevice, st);
  }
  int rc = FRISK_OK;
  if (e == cudaSuccess) {
    frisk_quant_args a = *args;
    a.x = b[X].dev;
    if (norm) a.residual = b[O].dev;
    if (gated) a.up = b[O].dev;
    if (norm) a.weight = b[Wt].dev;
    if (norm) a.sum_out = b[S].dev;
    a.q = b[Q].dev;
    a.scale = static_cast<float*>(b[Sc].dev);
    a.stream = st;
    d.ldx = d.ldo = d.lds = d.ldq = 0;
    d.device = -1;
    rc = frisk_b200_quant_run_status(&d, &a, static_cast<int32_t*>(b[St].dev));
    for (Buf& u : b)
      if (rc == FRISK_OK && e == cudaSuccess && u.out)
        e = cudaMemcpy2DAsync(u.out, u.ld * u.es, u.dev, u.width * u.es, u.width * u.es, u.rows, cudaMemcpyDeviceToHost, st);
  }
  if (st) {
    const cudaError_t e2 = cudaStreamSynchronize(st);
    if (e == cudaSuccess) e = e2;
  }
  if (e != cudaSuccess && rc == FRISK_OK) rc = fail_cuda(e, "frisk_b200_quant_run_host");
  if (status && rc == FRISK_OK) rc = fail(FRISK_ERR_DEVICE_TIMEOUT, "quant: a wait for rows ran out");
  for (Buf& u : b) cudaFree(u.dev);
  if (st) cudaStreamDestroy(st);
  if (prev >= 0 && prev != d.device) cudaSetDevice(prev);
  return rc;
}

}  // extern "C"
