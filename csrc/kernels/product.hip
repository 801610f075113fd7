// Products of row groups with their own weights:
//
//   c[i] = epi(a[rows[i]] . b[e]^T)     offsets[e] <= i < offsets[e + 1]
//
// for bf16 operands and for MXFP4 ones (v_mfma_scale_f32_16x16x128_f8f6f4,
// the scales applied by the matrix instruction), fp32 accumulation, one
// rounding to bf16 behind the epilogue.  A single group (offsets null) is the
// plain product.
#include "product.hpp"

#include "kernels.hpp"

namespace kiosk {
namespace {

// 128 x 128 tile, 4 waves of 64 x 64, for products that are a tile or two for
// each CU: bound by the latency of a launch, of the first loads and of a
// step's chain of loads, LDS reads and matrix instructions (512 x 512, bf16
// rows of 2 and 4 KiB: 17 and 25 us, 0.5 us a step; MXFP4 21 and 32).
//
// A ring of D LDS buffers of one 128-byte step each, filled by LDS-DMA D steps
// ahead; the wait for a step is counted, so later ones stay in flight.  A
// half-step's fragments are read under the matrix instructions of the half
// before.  Row r's 16-byte chunk c stands at chunk c ^ ((r >> 1) & 7), so the
// 16-lane groups of a ds_read_b128 meet 16 different bank slots.  Behind the
// operands of a step stand its MXFP4 scales, 8 bytes a row.
constexpr int BM = 128, BN = 128;
constexpr int kThreads = 256;
constexpr int kTileBytes = 128 * 128;
constexpr int kScaleBytes = 256 * 8;

template <int MODE>
constexpr int kStepBytes = 2 * kTileBytes + (MODE == kMx ? kScaleBytes : 0);
// loads of a wave and step
template <int MODE>
constexpr int kStepLoads = 8 + (MODE == kMx ? 2 : 0);

template <int MODE, int EPI, int D>
__global__ __launch_bounds__(kThreads, 4 / D) void product_tile_kernel(
    ProductArgs p, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int grid = tiles_m * tiles_n;
  if (static_cast<int>(blockIdx.x) >= grid) {
    zero_rest(p, blockIdx.x - grid, gridDim.x - grid);
    return;
  }
  Tiles<BM> tiles(p);
  const int real = min(tiles.total, tiles_m) * tiles_n;
  if (static_cast<int>(blockIdx.x) >= real) return;
  const int wg = xcd_remap(blockIdx.x, real);
  const RowTile tile = tiles.find(wg / tiles_n);
  const int n0 = (wg % tiles_n) * BN;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const size_t row_bytes = p.row_bytes;
  const uint8_t* b = p.b + static_cast<size_t>(tile.e) * p.n * row_bytes;

  // this lane's 4 rows of either operand (a wave moves 8 rows an issue)
  const uint8_t* pa[4];
  const uint8_t* pb[4];
  const int chunk = lane & 7;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (wave * 4 + i) * 8 + (lane >> 3);
    pa[i] = p.a + row_bytes * source_row(p, min(tile.lo + r, tile.hi - 1));
    pb[i] = b + row_bytes * min(n0 + r, p.n - 1);
  }
  // scales: half of a row's 8 bytes a lane, 32 rows an issue; rows 0 .. 127
  // are a's (waves 0 and 1), the others b's
  const uint8_t* ps[2];
  if constexpr (MODE == kMx) {
    const size_t scale_bytes = p.row_bytes / 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (wave & 1) * 64 + i * 32 + (lane >> 1);
      const size_t row_a = source_row(p, min(tile.lo + r, tile.hi - 1));
      const size_t row_b = static_cast<size_t>(tile.e) * p.n +
                           min(n0 + r, p.n - 1);
      ps[i] = wave < 2 ? p.a_scales + scale_bytes * row_a
                       : p.b_scales + scale_bytes * row_b;
    }
  }
  const int chunks = p.row_bytes / 16, halves = p.row_bytes / 64;
  const int steps = (halves + 1) / 2;
  // (behind the last step it is loaded again: the same count to wait for)
  auto stage = [&](int step) {
    const int t = min(step, steps - 1);
    char* lds = smem + step % D * kStepBytes<MODE>;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (wave * 4 + i) * 8 + (lane >> 3);
      // a row may end inside the step: its second half is then read as the
      // first again, and not used
      int c = t * 8 + (chunk ^ ((r >> 1) & 7));
      c = c < chunks ? c : c - 4;
      glds16(pa[i] + c * 16, lds + (wave * 4 + i) * 1024);
      glds16(pb[i] + c * 16, lds + kTileBytes + (wave * 4 + i) * 1024);
    }
    if constexpr (MODE == kMx)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        __builtin_amdgcn_global_load_lds(
            (gbl_void_t*)(ps[i] + min(2 * t + (lane & 1), halves - 1) * 4),
            (lds_void_t*)(lds + 2 * kTileBytes + (wave * 2 + i) * 256), 4, 0,
            0);
  };
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // half a step's fragments (and MXFP4 scales) of one wave
  struct Half {
    i32x4 x[4], w[4];
    int xs[4], ws[4];
  };
  auto read = [&](int t, int half, Half& f) {
    const char* cur = smem + t % D * kStepBytes<MODE>;
    const auto* scale = reinterpret_cast<const uint8_t*>(
        cur + 2 * kTileBytes + half * 4 + (lane >> 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 16 + (lane & 15);
      const int off = r * 128 +
                      (((half * 4 + (lane >> 4)) ^ ((r >> 1) & 7)) << 4);
      f.x[i] = *reinterpret_cast<const i32x4*>(cur + wm * 64 * 128 + off);
      f.w[i] = *reinterpret_cast<const i32x4*>(cur + kTileBytes +
                                               wn * 64 * 128 + off);
      f.xs[i] = MODE == kMx ? scale[(wm * 64 + r) * 8] : 0;
      f.ws[i] = MODE == kMx ? scale[(128 + wn * 64 + r) * 8] : 0;
    }
  };
  auto multiply = [&](const Half& f) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        mma<MODE>(acc[i][j], f.w[j], f.x[i], f.ws[j], f.xs[i]);
  };
  // every wave's loads of all steps but the last `later` have landed, and
  // every wave has what it asked LDS for
  auto meet = [&](auto later) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)"
                 :: "n"(decltype(later)::value * kStepLoads<MODE>)
                 : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

#pragma unroll
  for (int t = 0; t < D; ++t) stage(t);
  Half first, second;
  meet(std::integral_constant<int, D - 1>());
  read(0, 0, first);
  for (int t = 0; t < steps; ++t) {
    read(t, 1, second);
    multiply(first);
    // step t + 1 has landed; step t is in registers, step t + D takes its
    // buffer
    meet(std::integral_constant<int, D - 2>());
    stage(t + D);
    read(t + 1, 0, first);      // (behind the last step: not used)
    if (2 * t + 1 < halves) multiply(second);
  }
  // the last loads land before the workgroup's LDS is given up
  wait_vmcnt0();

#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = tile.lo + wm * 64 + i * 16 + (lane & 15);
    if (row >= tile.hi) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = n0 + wn * 64 + j * 16 + (lane >> 4) * 4;
      if (col >= p.n) continue;
      float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      epilogue4<EPI>(p, tile.e, row, col, v);
      *reinterpret_cast<uint2*>(p.c + static_cast<size_t>(row) * p.n + col) =
          uint2{pack2(v[0], v[1]), pack2(v[2], v[3])};
    }
  }
}

template <int MODE, int EPI, int D>
hipError_t configure_depth() {
  const auto kernel = &product_tile_kernel<MODE, EPI, D>;
  const hipError_t err = hipFuncSetAttribute(
      reinterpret_cast<const void*>(kernel),
      hipFuncAttributeMaxDynamicSharedMemorySize, D * kStepBytes<MODE>);
  return err == hipSuccess ? prepare_kernel(kernel) : err;
}

template <int MODE, int EPI>
hipError_t configure() {
  const hipError_t err = configure_depth<MODE, EPI, 2>();
  return err == hipSuccess ? configure_depth<MODE, EPI, 4>() : err;
}

template <int MODE>
hipError_t configure_mode() {
  hipError_t err = configure<MODE, PRODUCT_NONE>();
  if (err == hipSuccess) err = configure<MODE, PRODUCT_BIAS_GELU>();
  if constexpr (MODE == kMx)
    if (err == hipSuccess) err = configure<MODE, PRODUCT_BIAS_RESIDUAL>();
  if (err == hipSuccess) err = configure<MODE, PRODUCT_BIAS>();
  return err;
}

long long tiles128(const ProductArgs& p) {
  return static_cast<long long>(most_tiles(p.rows_c, p.experts, BM)) *
         ((p.n + BN - 1) / BN);
}

template <int MODE, int EPI>
hipError_t launch_epilogue(const ProductArgs& p, hipStream_t stream) {
  const int tiles_m = most_tiles(p.rows_c, p.experts, BM);
  const int tiles_n = (p.n + BN - 1) / BN;
  const long long blocks = tiles128(p) + (p.zero_rest ? kZeroBlocks : 0);
  // a tile for each CU: deep; two of them there hide each other's waits
  return tiles128(p) <= p.cus
             ? launch_tiles(&product_tile_kernel<MODE, EPI, 4>, blocks,
                            kThreads, 4 * kStepBytes<MODE>, stream, p, tiles_m,
                            tiles_n)
             : launch_tiles(&product_tile_kernel<MODE, EPI, 2>, blocks,
                            kThreads, 2 * kStepBytes<MODE>, stream, p, tiles_m,
                            tiles_n);
}

template <int MODE>
hipError_t launch_mode(const ProductArgs& p, hipStream_t stream) {
  switch (p.epilogue) {
    case PRODUCT_NONE:
      return launch_epilogue<MODE, PRODUCT_NONE>(p, stream);
    case PRODUCT_BIAS_GELU:
      return launch_epilogue<MODE, PRODUCT_BIAS_GELU>(p, stream);
    case PRODUCT_BIAS:
      return launch_epilogue<MODE, PRODUCT_BIAS>(p, stream);
    case PRODUCT_BIAS_RESIDUAL:
      if constexpr (MODE == kMx)
        return launch_epilogue<MODE, PRODUCT_BIAS_RESIDUAL>(p, stream);
    default:
      return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t experts_prepare() {
  static std::atomic<unsigned long long> done{0};
  return prepare_per_device(done, [] {
    hipError_t err = configure_mode<kBf16>();
    if (err == hipSuccess) err = configure_mode<kMx>();
    if (err == hipSuccess) err = product256_prepare();
    return err;
  });
}

namespace {

enum Variant { kRows, kTile, k256 };

// Small groups read their weights once, straight to registers, larger ones go
// to the 256 x 256 tiles (64 rows against bf16 4096 x 16384: 90 us from
// registers, 50 in tiles).  Where they part depends on how many tiles there
// are, one a group and 256 columns: fewer than CUs, 32 rows a group on average
// (16 experts of 2048 columns, 320 rows: 75 us from registers, 87 in tiles);
// at least as many, 16 (16 of 4096 columns, 300 rows: 197 and 168; 8 of 8192,
// 104 rows: 112 and 130); two rounds of them, 12 (64 of 2048 columns, 1024
// rows: 72 and 61; 32 of 4096, 320 rows: 68 and 70).
//
// The 128 x 128 tiles cost some 4 us less each and are four times as many, but
// each operand passes through LDS twice as often: they are better where two of
// them on each CU are all there is and rows are up to 2 KiB (2048 x 1024 x
// 1024: 29 us in large tiles, 18 in these; MXFP4 2048 x 1024 x 4096 31 and 22),
// or 4 KiB and there are enough of them to rival the large tiles' slices (bf16
// 2048 x 1024 x 2048: 35 and 27; 512 x 512 x 2048: 24 and 25; MXFP4 1024 x 4096
// x 8192: 46 and 39; 1024 x 1024 x 8192 in four groups: 30 and 35).  Of very
// short rows in groups up to 128 rows the large ones, halved, are ahead (eight
// groups of 75 rows, 128 -> 2048: 9.0 and 9.8).  Besides they take operands
// beyond 32-bit offsets.
bool small_tiles(const ProductArgs& p) {
  const long long tiles = tiles128(p);
  if (tiles > 2ll * p.cus || p.row_bytes > 4096) return false;
  if (p.row_bytes > 2048)
    return tiles >= (p.a_scales != nullptr ? p.cus : p.cus / 4);
  return p.row_bytes > 1024 || p.rows_c > 128ll * p.experts;
}

Variant pick(const ProductArgs& p) {
  const long long tiles = p.experts * ((p.n + 255ll) / 256);
  const int few = tiles >= 2ll * p.cus ? 12 : tiles >= p.cus ? 16 : 32;
  if (p.rows_c <= few * static_cast<long long>(p.experts)) return kRows;
  if (product256_ok(p)) return small_tiles(p) ? kTile : k256;
  return p.rows_c <= 64ll * p.experts ? kRows : kTile;
}

}  // namespace

size_t product_workspace(const ProductArgs& p) {
  if (p.rows_c <= 0 || p.experts < 1) return 0;
  return pick(p) == k256 ? product256_workspace(p) : 0;
}

const char* product_kernel(const ProductArgs& p) {
  const Variant v = pick(p);
  return v == kRows ? "rows" : v == kTile ? "tile128" : "tile256";
}

hipError_t launch_product(const ProductArgs& p, hipStream_t stream) {
  // (an empty tensor has no address: nothing below holds for it)
  if (p.rows_c == 0) return hipSuccess;
  if (p.rows_c < 0 || p.rows_a < 1 || p.experts < 1 ||
      p.experts > kProductMaxExperts || p.n < 16 ||
      p.n % 16 != 0 || p.row_bytes < 64 || p.row_bytes % 64 != 0 ||
      (p.offsets == nullptr && p.experts != 1) ||
      (p.a_scales == nullptr) != (p.b_scales == nullptr) ||
      (p.epilogue != PRODUCT_NONE && p.bias == nullptr) ||
      // (the bf16 product with a residual is gemm's)
      (p.epilogue == PRODUCT_BIAS_RESIDUAL &&
       (p.residual == nullptr || p.a_scales == nullptr)))
    return hipErrorInvalidValue;
  switch (pick(p)) {
    case kRows:
      return launch_product_rows(p, stream);
    case k256:
      return launch_product256(p, stream);
    default:
      break;
  }
  return p.a_scales != nullptr ? launch_mode<kMx>(p, stream)
                               : launch_mode<kBf16>(p, stream);
}

}  // namespace kiosk
