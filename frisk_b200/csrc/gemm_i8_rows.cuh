// The integer gemm of a few tokens, C[m, n] = sum_k A[m, k] B[n, k] with M <= 16: bound by reading the
// weights once, so the kernel is a stream of 16-byte loads with just enough arithmetic behind it.
//
// A CTA owns 16 R rows of weights (output channels) and all of K, which its warps share in chunks of
// 128; the warps' 32-bit partial sums meet in shared memory (integers: any order, the same result).
// The products are mma.sync m16n8k32 with the weights as the 16-row operand and the tokens as the
// 8 columns.  The sum over k does not care which k an operand's slot holds as long as both operands
// agree, so a lane takes 16 neighbouring bytes of its rows -- one load -- for the slots of two MMAs
// instead of the 4-byte pieces that the instruction's layout names.
//
// Every lane brings its pieces into its own slots of shared memory with 16-byte asynchronous copies,
// up to four chunks of K ahead, and reads them back itself: bytes in flight without registers for
// them, and no barrier before the fold.
//
// Against the tensor-core few-row plan (TMA, tensor memory, clusters) this saves the set-up and the
// fold through the cluster, and its smaller shared memory lets the next launch start beside it
// (bf16 C, that plan -> this kernel, replayed from a graph): one token, N x K = 4096 x 4096 6.2 -> 3.5 us
// (from L2), 8192 x 8192 15.6 -> 12.9 us (5190 GB/s, 0.80 of the copy rate), 28672 x 4096 27.4 -> 20.7
// us, 1000 x 4096 4.8 -> 3.0 us; 16 tokens, 4096 x 4096 6.1 -> 4.6 us, 8192 x 8192 16.1 -> 15.4 us, 28672 x
// 4096 29.9 -> 25.3 us, but 8192 x 28672 40.7 -> 43.4 us and with 32 tokens slower throughout: every
// CTA reads all of its tokens' K from L2, traffic that the clusters share.
#pragma once
#include "gemm_tcgen05.cuh"   // cast_in / cast_out, ptx

namespace frisk {

constexpr int kI8RowsWarps = 8;
constexpr int kI8RowsMaxM = 16;

struct I8RowsParams {
  const int8_t* A;       // tokens [M, K], pitch lda
  const int8_t* B;       // weights [N, K], pitch ldb
  void* C;
  const float* scale_a;  // [M] or nullptr
  const float* scale_b;  // [N] or nullptr
  int64_t lda, ldb, ldc;
  int32_t M, N, K;
  int32_t clear_accum;
};

// Sixteen bytes of a row at k into shared memory, asynchronously; zeros past K (only what exists of
// the row is read).
template <bool kL1>
__device__ __forceinline__ void i8_fetch16(uint32_t dst, const int8_t* row, int k, int K, bool live) {
  const int left = live ? max(0, min(16, K - k)) : 0;
  if (kL1) asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(row + (left ? k : 0)), "r"(left) : "memory");
  else asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(row + (left ? k : 0)), "r"(left) : "memory");
}

__device__ __forceinline__ void mma_s8(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                       uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared memory of a CTA: every warp's ring, 16-byte pieces as [stage][piece][lane] (a lane reads back
// only what it fetched itself, so no barrier is needed and no bank is hit twice), then -- over the
// same bytes -- the warps' partial sums.
template <int R, int MT>
constexpr int i8_rows_pieces() { return 4 * R + 2 * MT; }   // of a lane and chunk: its rows and tokens, two 64-byte pieces each
template <int R, int MT, int S>
constexpr int i8_rows_smem() {
  constexpr int ring = kI8RowsWarps * S * i8_rows_pieces<R, MT>() * 512;
  constexpr int part = kI8RowsWarps * 8 * MT * (16 * R + 4) * 4;
  return ring > part ? ring : part;
}

// R: 16-row tiles of weights per CTA; MT: tiles of eight tokens; S: chunks in flight per warp.
template <typename TC, int R, int MT, int S>
__global__ void __launch_bounds__(32 * kI8RowsWarps) gemm_i8_rows_kernel(const I8RowsParams p) {
  constexpr int kRows = 16 * R, kTokens = 8 * MT, kPieces = i8_rows_pieces<R, MT>();
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, kq = (lane & 3) * 16;   // the lane's row in a tile's halves, its bytes of a 64-byte piece
  const int n0 = blockIdx.x * kRows;
  constexpr int kLines = 2 * R + MT;
  const int8_t* row[kLines];   // the lane's rows of weights and its tokens
  bool live[kLines];
#pragma unroll
  for (int r = 0; r < 2 * R; ++r) {
    const int n = n0 + 8 * r + g;
    live[r] = n < p.N;
    row[r] = p.B + (int64_t)(live[r] ? n : 0) * p.ldb;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    live[2 * R + t] = 8 * t + g < p.M;
    row[2 * R + t] = p.A + (int64_t)(live[2 * R + t] ? 8 * t + g : 0) * p.lda;
  }
  const uint32_t ring = ptx::smem_u32(smem) + (uint32_t)(warp * S * kPieces * 512 + lane * 16);
  auto fetch = [&](int k, int stage) {
    if (k < p.K) {
#pragma unroll
      for (int r = 0; r < kLines; ++r)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (r < 2 * R)
            i8_fetch16<false>(ring + (uint32_t)((stage * kPieces + 2 * r + s) * 512), row[r], k + 64 * s + kq, p.K, live[r]);
          else   // tokens through L1 where another CTA of the SM reads them too (16 x 8192 x 8192 15.5 -> 15.2 us)
            i8_fetch16<MT == 1 || S == 2>(ring + (uint32_t)((stage * kPieces + 2 * r + s) * 512), row[r], k + 64 * s + kq, p.K, live[r]);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");   // (empty past the end: the waits count groups)
  };
  constexpr int kStep = 128 * kI8RowsWarps;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(128 * warp + s * kStep, s);
  int32_t acc[R][MT][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][t][i] = 0;
  int stage = 0;
  for (int k = 128 * warp; k < p.K; k += kStep) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    uint4 v[kLines][2];
#pragma unroll
    for (int r = 0; r < kLines; ++r)
#pragma unroll
      for (int s = 0; s < 2; ++s) v[r][s] = ld_shared_v4(ring + (uint32_t)((stage * kPieces + 2 * r + s) * 512));
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const uint4 &lo = v[2 * r][s], &hi = v[2 * r + 1][s], &a = v[2 * R + t][s];
          mma_s8(acc[r][t], lo.x, hi.x, lo.y, hi.y, a.x, a.y);
          mma_s8(acc[r][t], lo.z, hi.z, lo.w, hi.w, a.z, a.w);
        }
    fetch(k + S * kStep, stage);   // this lane has read the stage: the MMAs above have their operands
    if (++stage == S) stage = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // every ring is done with: the sums go over them
  int32_t(*part)[kTokens][kRows + 4] = reinterpret_cast<int32_t(*)[kTokens][kRows + 4]>(smem);
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = 8 * t + 2 * (lane & 3), n = 16 * r + g;
      part[warp][m][n] = acc[r][t][0];
      part[warp][m + 1][n] = acc[r][t][1];
      part[warp][m][n + 8] = acc[r][t][2];
      part[warp][m + 1][n + 8] = acc[r][t][3];
    }
  __syncthreads();
  TC* C = static_cast<TC*>(p.C);
  for (int i = threadIdx.x; i < kRows * p.M; i += 32 * kI8RowsWarps) {
    const int m = i / kRows, n = i % kRows;
    if (n0 + n >= p.N) continue;
    int32_t sum = 0;
#pragma unroll
    for (int x = 0; x < kI8RowsWarps; ++x) sum += part[x][m][n];
    float v = __int2float_rn(sum);
    if (p.scale_a) v = v * __ldg(p.scale_a + m) * __ldg(p.scale_b + n0 + n);
    TC* dst = C + (int64_t)m * p.ldc + n0 + n;
    if (!p.clear_accum) v += cast_in<TC>(*dst);
    *dst = cast_out<TC>(v);
  }
}

}  // namespace frisk
