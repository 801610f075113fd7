// The bf16 product's 256 x 256 tile for groups of many rows (contract:
// product.hip; division of the work and LDS ring: product256.hpp).
//
// Bound by the card's power: 4096 x 4096 x 8192 takes 187 us (1.5 PFLOP/s), 144
// on zeros (of rows of 64 KiB 760 and 743: there it is memory); a large library
// product reaches 1.6 PFLOP/s.
//
// Four waves of 128 x 128 outputs (128 x 64 of a tile of 128 rows), the
// accumulators in AGPRs.  v_mfma_f32_16x16x32_bf16: the 32 x 32 one, with half
// as many instructions, is 10 % slower here (4096 x 16384 x 4096: 416 against
// 377 us).  A DMA issue holds a wave up for longer than one of these
// instructions lasts, so two of the four waves issue theirs three
// instructions later than the other two.
#include "kernels.hpp"
#include "product256.hpp"

namespace kiosk {
namespace {

using namespace ring256;

// Matrix instructions on AGPR accumulators (with the builtins the operands
// land in AGPRs and VGPRs spill).  Operands come from LDS reads, for which the
// compiler waits; the epilogue's first read of an accumulator waits in
// drain().
__device__ __forceinline__ void mfma(f32x4& acc, const i32x4& w,
                                     const i32x4& x) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0"
               : "+a"(acc) : "v"(w), "v"(x));
}
__device__ __forceinline__ void mfma_first(f32x4& acc, const i32x4& w,
                                           const i32x4& x) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0"
               : "=a"(acc) : "v"(w), "v"(x));
}

constexpr int kLate = 3;

// Lane l holds product row l & 15 and columns 4 (l >> 4) .. + 3 of a 16 x 16
// tile.  Lanes l and l ^ 16 exchange one tile's half of a tile pair, so that
// each stores eight columns (16 bytes) at once.
template <int EPI, int TN>
__device__ __forceinline__ void store_tile(const ProductArgs& p, const Work& w,
                                           int row0, int col0, int lane,
                                           const float* bias, float* piece,
                                           f32x4 (&acc)[8][TN]) {
  const int fr = lane & 15, g = lane >> 4;
  const bool odd = (g & 1) != 0;
  float4 bias4[TN];
  if constexpr (EPI != PRODUCT_NONE) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
      bias4[j] = *reinterpret_cast<const float4*>(bias + col0 + j * 16 +
                                                  g * 4);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = w.lo + row0 + i * 16 + fr;
    const bool in = row < w.hi;
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      const int base = w.n0 + col0 + j * 16;
      if (piece != nullptr) {
        if (in)
#pragma unroll
          for (int s = 0; s < 2; ++s)
            *reinterpret_cast<float4*>(piece + (row - w.lo) * BN + col0 +
                                       (j + s) * 16 + g * 4) =
                float4{acc[i][j + s][0], acc[i][j + s][1], acc[i][j + s][2],
                       acc[i][j + s][3]};
        continue;
      }
      uint32_t u[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float v[4] = {acc[i][j + s][0], acc[i][j + s][1], acc[i][j + s][2],
                      acc[i][j + s][3]};
        if constexpr (EPI != PRODUCT_NONE) add4(v, bias4[j + s]);
        if constexpr (EPI == PRODUCT_BIAS_GELU) gelu4(v);
        u[s][0] = pack2(v[0], v[1]);
        u[s][1] = pack2(v[2], v[3]);
      }
      const auto x0 = __builtin_amdgcn_permlane16_swap(u[0][0], u[1][0],
                                                       false, false);
      const auto x1 = __builtin_amdgcn_permlane16_swap(u[0][1], u[1][1],
                                                       false, false);
      const int col = odd ? base + 16 + (g - 1) * 4 : base + g * 4;
      if (in && col < p.n)
        *reinterpret_cast<uint4*>(p.c + static_cast<size_t>(row) * p.n + col) =
            uint4{x0[0], x1[0], x0[1], x1[1]};
    }
    // one row of tiles at a time bounds the AGPR -> VGPR copies
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int EPI, bool HALF>
__device__ __forceinline__ void run_tile(const ProductArgs& p, const Work& w,
                                         char* smem) {
  constexpr int TN = HALF ? 4 : 8;
  const Ring<HALF> ring(p, w, smem);
  const int wave = ring.wave, lane = ring.lane;
  const int row0 = HALF ? 0 : (wave >> 1) * 128;
  const int col0 = HALF ? wave * 64 : (wave & 1) * 128;
  const int steps = ring.steps;

  // fragment r of a half: r < TN -> b's rows 16 r + fr, else a's
  const int fr = lane & 15, g = lane >> 4;
  const int sw = (fr >> 1) & 7;
  int off_a[2], off_b[2];
#pragma unroll
  for (int hi = 0; hi < 2; ++hi) {
    const int chunk = ((hi * 4 + g) ^ sw) << 4;
    off_a[hi] = (row0 + fr) * 128 + chunk;
    off_b[hi] = (col0 + fr) * 128 + chunk;
  }
  auto read = [&](auto hh, int t, int r, i32x4 (&wb)[TN], i32x4 (&xa)[8]) {
    constexpr int kHi = decltype(hh)::value;
    if (r < TN)
      wb[r] = *reinterpret_cast<const i32x4*>(ring.unit(2 * t + 1) +
                                              off_b[kHi] + r * 2048);
    else
      xa[r - TN] = *reinterpret_cast<const i32x4*>(
          ring.unit(2 * t) + off_a[kHi] + (r - TN) * 2048);
  };

  // this thread's column's bias, on its way while the loop runs
  float bias = 0.0f;
  if constexpr (EPI != PRODUCT_NONE)
    bias = p.bias[static_cast<size_t>(w.e) * p.n +
                  min(w.n0 + static_cast<int>(threadIdx.x), p.n - 1)];

  f32x4 acc[8][TN];
  i32x4 wb0[TN], xa0[8], wb1[TN], xa1[8];
  constexpr int kA = Ring<HALF>::kPiecesA, kB = Ring<HALF>::kPiecesB;
  // half-step h = 2 t + odd
  auto half = [&](auto late, auto first, auto odd, int t,
                  const i32x4 (&wb)[TN], const i32x4 (&xa)[8],
                  i32x4 (&wb_next)[TN], i32x4 (&xa_next)[8]) {
    constexpr int kOff = decltype(late)::value;
    constexpr int kOdd = decltype(odd)::value;
    const int h = 2 * t + kOdd;
    __builtin_amdgcn_sched_barrier(0);
    // in flight: group h + 3 and, before it is needed, h + 2
    __builtin_amdgcn_s_waitcnt(wait_imm(kOdd ? kA : kA + kB));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    const int tn = kOdd ? t + 1 : t;
    // the DMA pieces of group h + 4 and the TN + 8 LDS reads spread over
    // the first three quarters: the last read has a quarter to return
    constexpr int kPieces = kOdd ? kB : kA;
    constexpr int kSpan = TN * 6;
    constexpr int kEvery = kSpan / kPieces;
    constexpr int kReadEvery = HALF ? 2 : 3;
#pragma unroll
    for (int u = 0; u < 8 * TN; ++u) {
      const int i = u / TN, j = u % TN;
      if constexpr (decltype(first)::value)
        mfma_first(acc[i][j], wb[j], xa[i]);
      else
        mfma(acc[i][j], wb[j], xa[i]);
      if (u >= kOff && (u - kOff) % kEvery == 0 && u - kOff < kSpan)
        ring.template dma<false>(h + 4, (u - kOff) / kEvery);
      if (u % kReadEvery == 1 && u / kReadEvery < TN + 8)
        read(Int<kOdd ? 0 : 1>(), tn, u / kReadEvery, wb_next, xa_next);
    }
  };
  ring.template start<false>();
  __builtin_amdgcn_s_waitcnt(wait_imm(kA + kB));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int r = 0; r < TN + 8; ++r) read(Int<0>(), 0, r, wb0, xa0);
  auto loop = [&](auto late) {
    half(late, Int<1>(), Int<0>(), 0, wb0, xa0, wb1, xa1);
    half(late, Int<0>(), Int<1>(), 0, wb1, xa1, wb0, xa0);
    for (int t = 1; t < steps; ++t) {
      half(late, Int<0>(), Int<0>(), t, wb0, xa0, wb1, xa1);
      half(late, Int<0>(), Int<1>(), t, wb1, xa1, wb0, xa0);
    }
  };
  if (wave >> 1)
    loop(Int<kLate>());
  else
    loop(Int<0>());
  // the tail's DMA lands before the workgroup's LDS is given up
  __builtin_amdgcn_s_waitcnt(wait_imm(0));
  drain();
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));

  // the bias goes round through LDS, once for all rows
  auto* shared = reinterpret_cast<float*>(smem);
  if constexpr (EPI != PRODUCT_NONE) {
    __syncthreads();
    shared[threadIdx.x] = bias;
    __syncthreads();
  }
  float* piece = w.piece < 0 ? nullptr
                             : p.partial + static_cast<size_t>(w.piece) *
                                               kPieceFloats;
  store_tile<EPI, TN>(p, w, row0, col0, lane, shared, piece, acc);
}

template <int EPI>
__global__ __launch_bounds__(kThreads, 1) void product256_bf16_kernel(
    ProductArgs p, int tiles_n, int grid) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Work w;
  if (!find_work(p, tiles_n, grid, &w)) return;
  if (w.half)
    run_tile<EPI, true>(p, w, smem);
  else
    run_tile<EPI, false>(p, w, smem);
}

template <int EPI>
hipError_t configure() {
  hipError_t err = hipFuncSetAttribute(
      reinterpret_cast<const void*>(&product256_bf16_kernel<EPI>),
      hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
  return err == hipSuccess ? prepare_kernel(&product256_bf16_kernel<EPI>)
                           : err;
}

}  // namespace

hipError_t product256_bf16_prepare() {
  hipError_t err = configure<PRODUCT_NONE>();
  if (err == hipSuccess) err = configure<PRODUCT_BIAS_GELU>();
  if (err == hipSuccess) err = configure<PRODUCT_BIAS>();
  return err;
}

hipError_t launch_product256_bf16(const ProductArgs& p, int tiles_n, int grid,
                                  long long blocks, hipStream_t stream) {
  auto launch = [&](auto kernel) {
    return launch_tiles(kernel, blocks, kThreads, kLdsBytes, stream, p, tiles_n,
                        grid);
  };
  switch (p.epilogue) {
    case PRODUCT_NONE:
      return launch(&product256_bf16_kernel<PRODUCT_NONE>);
    case PRODUCT_BIAS_GELU:
      return launch(&product256_bf16_kernel<PRODUCT_BIAS_GELU>);
    case PRODUCT_BIAS:
      return launch(&product256_bf16_kernel<PRODUCT_BIAS>);
    default:   // (the product with a residual is gemm's)
      return hipErrorInvalidValue;
  }
}

}  // namespace kiosk
