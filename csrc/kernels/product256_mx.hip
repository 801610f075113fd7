// The MXFP4 product's 256 x 256 tile for groups of many rows (contract:
// product.hip; division of the work and LDS ring: product256.hpp).
//
// Bound by the card's power and by its loads: 4096 x 4096 x 16384 takes 123 us
// (4.5 PFLOP/s; the clock falls to 1.8 GHz), with the same instructions on
// zeros 88 us, without LDS reads and loads in the loop 94.  Besides, a tile costs some 10 us that no other one's work covers (it has
// the CU's LDS to itself): the first loads and the stores.
//
// Four waves of 128 x 128 outputs (128 x 64 of a tile of 128 rows), the
// accumulators in AGPRs.  v_mfma_scale_f32_32x32x64_f8f6f4 on 16 bytes a lane:
// the same bytes move at the same rate as for bf16, the instruction does four
// times the operations.  Lane l holds row l & 31, bytes 32 ks + 16 (l >> 5) of
// the half-step.
//
// The scales go from memory to registers, four steps (32 bytes of a row) at a
// time and ahead: lane l loads 16 of row l & 31, those of the first or the
// last two steps.  A lane swap and byte permutations leave the four that this
// lane's blocks need in one register a step, the instruction picks one.  (Two
// steps a load are as many cache lines asked for as the operands themselves.)
#include "kernels.hpp"
#include "product256.hpp"

namespace kiosk {
namespace {

using namespace ring256;

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) unsigned scale4_t;

// Matrix instructions on AGPR accumulators (with the builtins the operands
// land in AGPRs and VGPRs spill).  Inline asm gets no wait states: operands
// come from LDS reads, for which the compiler waits; scales, which VALU
// instructions pack, are held to their place before a barrier (settle), for a
// matrix instruction needs two wait states behind them; the epilogue's first
// read of an accumulator waits in drain().  Byte `S` of both scale registers.
template <int S>
__device__ __forceinline__ void mfma_mx(f32x16& acc, const i32x4& w,
                                        const i32x4& x, int ws, int xs) {
  asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 "
               "op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4 blgp:4"
               : "+a"(acc)
               : "v"(w), "v"(x), "v"(ws), "v"(xs), "n"(S & 1), "n"(S >> 1));
}
__device__ __forceinline__ void mfma_mx_first(f32x16& acc, const i32x4& w,
                                              const i32x4& x, int ws,
                                              int xs) {
  asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, 0, %3, %4 "
               "op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
               : "=a"(acc)
               : "v"(w), "v"(x), "v"(ws), "v"(xs));
}

// No VALU instruction that makes these words is moved behind this point.
template <int N>
__device__ __forceinline__ void settle(int (&words)[N][4]) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(words[k][q]));
}

// Lane l holds product row l & 31 and columns 8 b + 4 (l >> 5) .. + 3 of a
// 32 x 32 tile.  Lanes l and l ^ 32 exchange one column group of a pair, so
// that each stores eight columns (16 bytes) at once.
template <int EPI, int TN>
__device__ __forceinline__ void store_tile(const ProductArgs& p, const Work& w,
                                           int row0, int col0, int lane,
                                           const float* bias, float* piece,
                                           f32x16 (&acc)[4][TN]) {
  const int fr = lane & 31, hk = lane >> 5;
  float4 bias4[TN][4];
  if constexpr (EPI != PRODUCT_NONE) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        bias4[j][b] = *reinterpret_cast<const float4*>(
            bias + col0 + j * 32 + b * 8 + hk * 4);
  }
  // a tile's residual is asked for a row of tiles ahead
  uint2 residual[TN][4];
  auto fetch = [&](int i, int j) {
    // (inside the product always: what is not stored may be any of it)
    const int row = min(w.lo + row0 + i * 32 + fr, w.hi - 1);
    const uint16_t* from = p.residual + static_cast<size_t>(row) * p.n;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      residual[j][b] = *reinterpret_cast<const uint2*>(
          from + min(w.n0 + col0 + j * 32 + b * 8 + hk * 4, p.n - 4));
  };
  if constexpr (EPI == PRODUCT_BIAS_RESIDUAL)
    if (piece == nullptr)
#pragma unroll
      for (int j = 0; j < TN; ++j) fetch(0, j);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = w.lo + row0 + i * 32 + fr;
    const bool in = row < w.hi;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
      for (int b = 0; b < 4; b += 2) {
        const int base = w.n0 + col0 + j * 32 + b * 8;
        if (piece != nullptr) {
          if (in)
#pragma unroll
            for (int s = 0; s < 2; ++s)
              *reinterpret_cast<float4*>(piece + (row - w.lo) * BN + col0 +
                                         j * 32 + (b + s) * 8 + hk * 4) =
                  float4{acc[i][j][4 * (b + s)], acc[i][j][4 * (b + s) + 1],
                         acc[i][j][4 * (b + s) + 2],
                         acc[i][j][4 * (b + s) + 3]};
          continue;
        }
        uint32_t u[2][2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float v[4] = {acc[i][j][4 * (b + s)], acc[i][j][4 * (b + s) + 1],
                        acc[i][j][4 * (b + s) + 2],
                        acc[i][j][4 * (b + s) + 3]};
          if constexpr (EPI != PRODUCT_NONE) add4(v, bias4[j][b + s]);
          if constexpr (EPI == PRODUCT_BIAS_GELU) gelu4(v);
          if constexpr (EPI == PRODUCT_BIAS_RESIDUAL)
            add_residual(v, residual[j][b + s]);
          u[s][0] = pack2(v[0], v[1]);
          u[s][1] = pack2(v[2], v[3]);
        }
        const auto x0 = __builtin_amdgcn_permlane32_swap(u[0][0], u[1][0],
                                                         false, false);
        const auto x1 = __builtin_amdgcn_permlane32_swap(u[0][1], u[1][1],
                                                         false, false);
        const int col = base + hk * 8;
        if (in && col < p.n)
          *reinterpret_cast<uint4*>(p.c + static_cast<size_t>(row) * p.n +
                                    col) =
              uint4{x0[0], x1[0], x0[1], x1[1]};
      }
      if constexpr (EPI == PRODUCT_BIAS_RESIDUAL)
        if (piece == nullptr && i < 3) fetch(i + 1, j);
    }
    // one row of tiles at a time bounds the AGPR -> VGPR copies
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int EPI, bool HALF, bool CUT>
__device__ __forceinline__ void run_tile(const ProductArgs& p, const Work& w,
                                         char* smem) {
  constexpr int TN = HALF ? 2 : 4;
  const Ring<HALF> ring(p, w, smem);
  const int wave = ring.wave, lane = ring.lane;
  const int row0 = HALF ? 0 : (wave >> 1) * 128;
  const int col0 = HALF ? wave * 64 : (wave & 1) * 128;
  const int steps = ring.steps;

  const int fr = lane & 31, hk = lane >> 5;
  const int sw = (fr >> 1) & 7;
  int off_a[2][2], off_b[2][2];      // [half][ks]
#pragma unroll
  for (int hi = 0; hi < 2; ++hi)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int chunk = ((hi * 4 + ks * 2 + hk) ^ sw) << 4;
      off_a[hi][ks] = (row0 + fr) * 128 + chunk;
      off_b[hi][ks] = (col0 + fr) * 128 + chunk;
    }
  // fragment r of a half: r < 2 TN -> b (ks r / TN, tile r % TN), else a
  constexpr int kReads = 2 * TN + 8;
  auto read = [&](auto hh, int t, int r, i32x4 (&wb)[2][TN],
                  i32x4 (&xa)[2][4]) {
    constexpr int kHi = decltype(hh)::value;
    if (r < 2 * TN) {
      const int ks = r / TN, idx = r % TN;
      wb[ks][idx] = *reinterpret_cast<const i32x4*>(
          ring.unit(2 * t + 1) + off_b[kHi][ks] + idx * 4096);
    } else {
      const int ks = (r - 2 * TN) >> 2, idx = r & 3;
      xa[ks][idx] = *reinterpret_cast<const i32x4*>(
          ring.unit(2 * t) + off_a[kHi][ks] + idx * 4096);
    }
  };

  // scales: rows of row_bytes / 16 bytes, 8 of them a step
  const unsigned scale_row = p.row_bytes / 16;
  const auto rsrc_sa = buffer(
      p.a_scales + static_cast<size_t>(ring.first_a) * scale_row,
      ring.rows_here * scale_row);
  const auto rsrc_sb = buffer(
      p.b_scales + static_cast<size_t>(w.e) * p.n * scale_row,
      p.n * scale_row);
  unsigned soff_a[4], soff_b[TN];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    soff_a[i] = ring.buffer_row(p, w, min(w.lo + row0 + i * 32 + fr,
                                          w.hi - 1)) * scale_row + hk * 16;
#pragma unroll
  for (int j = 0; j < TN; ++j)
    soff_b[j] = static_cast<unsigned>(min(w.n0 + col0 + j * 32 + fr,
                                          p.n - 1)) * scale_row + hk * 16;
  // (the last 32 bytes of a row may begin in it and end in the next; what
  // lies past the last row's end reads as zero: either scales nothing that is
  // used)
  const int last_q = (steps - 1) >> 2;
  auto load_sa = [&](int q, int i) -> scale4_t {
    return __builtin_amdgcn_raw_buffer_load_b128(
        rsrc_sa, soff_a[i], w.step0 * 8 + min(q, last_q) * 32, 0);
  };
  auto load_sb = [&](int q, int j) -> scale4_t {
    return __builtin_amdgcn_raw_buffer_load_b128(
        rsrc_sb, soff_b[j], w.step0 * 8 + min(q, last_q) * 32, 0);
  };
  // Of a step's two words (halves) lanes below 32 need bytes 0 and 2 each, the
  // others 1 and 3.  1 for the zeros of a half behind the rows' end (another
  // row's scale may be NaN).
  auto pack = [&](int q, const scale4_t& v, int (&out)[4]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const auto got = __builtin_amdgcn_permlane32_swap(
          __builtin_amdgcn_perm(v[2 * k + 1], v[2 * k], 0x06040200u),
          __builtin_amdgcn_perm(v[2 * k + 1], v[2 * k], 0x07050301u), false,
          false);
      out[k] = got[0];
      out[2 + k] = got[1];
    }
    if constexpr (CUT)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int keep = ring.cut && 4 * q + k >= steps - 1 ? 0xffff : -1;
        out[k] = (out[k] & keep) | (~keep & 0x7f7f0000);
      }
  };

  // this thread's column's bias, on its way while the loop runs
  float bias = 0.0f;
  if constexpr (EPI != PRODUCT_NONE)
    bias = p.bias[static_cast<size_t>(w.e) * p.n +
                  min(w.n0 + static_cast<int>(threadIdx.x), p.n - 1)];

  f32x16 acc[4][TN];
  i32x4 wb0[2][TN], xa0[2][4], wb1[2][TN], xa1[2][4];
  int ws[TN][4], xs[4][4], ws_next[TN][4], xs_next[4][4];
  scale4_t ta[4], tb[TN];
  constexpr int kA = Ring<HALF>::kPiecesA, kB = Ring<HALF>::kPiecesB;

  // half-step h = 2 t + odd; `quarter`: t's place in its four steps
  auto half = [&](auto first, auto odd, auto quarter, int t,
                  const i32x4 (&wb)[2][TN], const i32x4 (&xa)[2][4],
                  i32x4 (&wb_next)[2][TN], i32x4 (&xa_next)[2][4]) {
    constexpr bool kFirst = decltype(first)::value != 0;
    constexpr int kOdd = decltype(odd)::value;
    constexpr int kStep = decltype(quarter)::value;
    constexpr int kPlace = kStep * 2 + kOdd;
    const int h = 2 * t + kOdd;
    // in flight: group h + 3 and, before it is needed, h + 2; the scales of
    // a (4 loads, behind the DMA of place 0) and of b (TN, place 1)
    constexpr int kWait = kPlace == 0   ? kA + kB
                          : kPlace == 1 ? kA + 4
                          : kPlace == 2 ? kA + 4 + kB + TN
                          : kPlace == 3 ? TN + kA
                          : kOdd        ? kA
                                        : kA + kB;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(wait_imm(kWait));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    const int tn = kOdd ? t + 1 : t;
    // the pieces of group h + 4 and the LDS reads in the first three
    // quarters, the scales in the last
    constexpr int kAll = 8 * TN, kSpan = 6 * TN;
    constexpr int kPieces = kOdd ? kB : kA;
#pragma unroll
    for (int u = 0; u < kAll; ++u) {
      const int ks = u / (4 * TN), i = u / TN & 3, j = u % TN;
      if (kFirst && ks == 0)
        mfma_mx_first(acc[i][j], wb[ks][j], xa[ks][i], ws[j][kStep],
                      xs[i][kStep]);
      else if (ks == 0)
        mfma_mx<kOdd * 2>(acc[i][j], wb[ks][j], xa[ks][i], ws[j][kStep],
                          xs[i][kStep]);
      else
        mfma_mx<kOdd * 2 + 1>(acc[i][j], wb[ks][j], xa[ks][i],
                              ws[j][kStep], xs[i][kStep]);
      // item k of n falls to instruction k * kSpan / n
#pragma unroll
      for (int k = 0; k < kPieces; ++k)
        if (k * kSpan / kPieces + (kPieces * 2 < kSpan) == u)
          ring.template dma<CUT>(h + 4, k);
#pragma unroll
      for (int k = 0; k < kReads; ++k)
        if (k * kSpan / kReads == u)
          read(Int<kOdd ? 0 : 1>(), tn, k, wb_next, xa_next);
      const int q = (t >> 2) + 1;            // the next four steps
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (kSpan + k * (kAll - kSpan) / 4 != u) continue;
        if (kPlace == 0) ta[k] = load_sa(q, k);
        if (kPlace == 6) pack(q, ta[k], xs_next[k]);
        if (k < TN) {
          if (kPlace == 1) tb[k] = load_sb(q, k);
          if (kPlace == 7) pack(q, tb[k], ws_next[k]);
        }
      }
    }
    if constexpr (kPlace == 7) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int k = 0; k < 4; ++k) xs[k][q] = xs_next[k][q];
#pragma unroll
        for (int k = 0; k < TN; ++k) ws[k][q] = ws_next[k][q];
      }
      settle(xs);
      settle(ws);
    }
  };

#pragma unroll
  for (int k = 0; k < 4; ++k) ta[k] = load_sa(0, k);
#pragma unroll
  for (int k = 0; k < TN; ++k) tb[k] = load_sb(0, k);
  ring.template start<CUT>();
#pragma unroll
  for (int k = 0; k < 4; ++k) pack(0, ta[k], xs[k]);
#pragma unroll
  for (int k = 0; k < TN; ++k) pack(0, tb[k], ws[k]);
  settle(xs);
  settle(ws);
  __builtin_amdgcn_s_waitcnt(wait_imm(kA + kB));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int r = 0; r < kReads; ++r) read(Int<0>(), 0, r, wb0, xa0);
  auto step = [&](auto first, auto quarter, int t) {
    half(first, Int<0>(), quarter, t, wb0, xa0, wb1, xa1);
    half(Int<0>(), Int<1>(), quarter, t, wb1, xa1, wb0, xa0);
  };
  step(Int<1>(), Int<0>(), 0);
  for (int t = 1; t < steps; t += 4) {
    step(Int<0>(), Int<1>(), t);
    if (t + 1 >= steps) break;
    step(Int<0>(), Int<2>(), t + 1);
    if (t + 2 >= steps) break;
    step(Int<0>(), Int<3>(), t + 2);
    if (t + 3 >= steps) break;
    step(Int<0>(), Int<0>(), t + 3);
  }
  // the tail's DMA lands before the workgroup's LDS is given up
  __builtin_amdgcn_s_waitcnt(wait_imm(0));
  drain();
#pragma unroll
  for (int i = 0; i < 4; ++i)
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

// CUT: rows end in the middle of a step (asking for that costs the others
// 2 %: 4096 x 8192 x 8192 131 against 128 us)
template <int EPI, bool CUT>
__global__ __launch_bounds__(kThreads, 1) void product256_mx_kernel(
    ProductArgs p, int tiles_n, int grid) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Work w;
  if (!find_work(p, tiles_n, grid, &w)) return;
  if (w.half)
    run_tile<EPI, true, CUT>(p, w, smem);
  else
    run_tile<EPI, false, CUT>(p, w, smem);
}

template <int EPI, bool CUT>
hipError_t configure() {
  const auto kernel = &product256_mx_kernel<EPI, CUT>;
  hipError_t err = hipFuncSetAttribute(
      reinterpret_cast<const void*>(kernel),
      hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
  return err == hipSuccess ? prepare_kernel(kernel) : err;
}

template <bool CUT>
hipError_t configure_all() {
  hipError_t err = configure<PRODUCT_NONE, CUT>();
  if (err == hipSuccess) err = configure<PRODUCT_BIAS_GELU, CUT>();
  if (err == hipSuccess) err = configure<PRODUCT_BIAS, CUT>();
  if (err == hipSuccess) err = configure<PRODUCT_BIAS_RESIDUAL, CUT>();
  return err;
}

template <bool CUT>
hipError_t launch_cut(const ProductArgs& p, int tiles_n, int grid,
                      long long blocks, hipStream_t stream) {
  auto launch = [&](auto kernel) {
    return launch_tiles(kernel, blocks, kThreads, kLdsBytes, stream, p, tiles_n,
                        grid);
  };
  switch (p.epilogue) {
    case PRODUCT_NONE:
      return launch(&product256_mx_kernel<PRODUCT_NONE, CUT>);
    case PRODUCT_BIAS_GELU:
      return launch(&product256_mx_kernel<PRODUCT_BIAS_GELU, CUT>);
    case PRODUCT_BIAS:
      return launch(&product256_mx_kernel<PRODUCT_BIAS, CUT>);
    case PRODUCT_BIAS_RESIDUAL:
      return launch(&product256_mx_kernel<PRODUCT_BIAS_RESIDUAL, CUT>);
    default:
      return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t product256_mx_prepare() {
  const hipError_t err = configure_all<false>();
  return err == hipSuccess ? configure_all<true>() : err;
}

hipError_t launch_product256_mx(const ProductArgs& p, int tiles_n, int grid,
                                long long blocks, hipStream_t stream) {
  return p.row_bytes % 128 != 0
             ? launch_cut<true>(p, tiles_n, grid, blocks, stream)
             : launch_cut<false>(p, tiles_n, grid, blocks, stream);
}

}  // namespace kiosk
