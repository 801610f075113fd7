// The product for groups of few rows (contract: product.hip): what is read
// is the weights, once, and their rate is the bound (two experts of bf16 4096
// -> 16384, one row each: 52 us, 5.2 TB/s; 31 of MXFP4 4096 -> 4096, 128 rows:
// 55 us, 5.0 TB/s; a plain read of 1 GiB: 6.1 TB/s).
//
// A workgroup of W waves owns NF x 16 columns of one row tile (MF x 16 rows).
// The waves deal the 256-byte pieces of the weight rows out among themselves,
// so all of them stream all the time, and add their partial tiles in LDS at
// the end, in the order of the waves.  Weights and activations go from memory
// straight to registers: no element is used by two waves.
//
// The 16 x 16 instructions want 16 bytes of 4 lane groups g for each row; any
// order along the inner dimension will do if both operands keep it.  Here the
// groups' bytes follow each other: instruction q of a 256-byte piece takes
// bytes 64 q + 16 g, so that a load covers 64 bytes of a row in one go (with
// 64 bytes for each lane eight experts of 16 rows each, MXFP4 4096 -> 14336,
// take 57 instead of 53 us, bf16 4096 -> 4096 61 instead of 59).
//
// MXFP4 scales are a 17th of the bytes, but a word for each lane and piece is
// as many memory transactions as a quarter of the weights (33 experts of 4096
// rows of 2 KiB: 71 us, 54 without the scales).  So a wave takes four pieces
// in a row: lane group g loads the 16 scale bytes of piece g of the four, and
// a transposition in registers leaves every lane its four bytes of each piece
// in a word, whose byte the instruction picks.
#include "kernels.hpp"
#include "product.hpp"

namespace kiosk {
namespace {

template <int B>
__device__ __forceinline__ void mma_piece(f32x4& acc, const i32x4& w,
                                          const i32x4& x, int ws, int xs,
                                          std::integral_constant<int, kMx>) {
  const i32x8 w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0};
  const i32x8 x8 = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc, 4, 4, B,
                                                         ws, B, xs);
}
template <int B>
__device__ __forceinline__ void mma_piece(f32x4& acc, const i32x4& w,
                                          const i32x4& x, int, int,
                                          std::integral_constant<int, kBf16>) {
  mma<kBf16>(acc, w, x, 0, 0);
}

// One row fragment (16 rows) of a 256-byte piece: a lane's 4 x 16 bytes.
struct Frag {
  i32x4 v[4];
};

__device__ __forceinline__ void load(Frag& f, const uint8_t* p) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f.v[i] = *reinterpret_cast<const i32x4*>(p + i * 64);
}

// The scales of a row fragment's four pieces: lane group g's 16 bytes are
// those of piece g; turned over, byte q of word u is what its instruction q of
// piece u needs (byte 4 q + g of that piece).
struct Scales {
  typedef int words_t __attribute__((ext_vector_type(4), aligned(4)));
  int v[4];

  __device__ __forceinline__ void load(const uint8_t* p) {
    const words_t w = *reinterpret_cast<const words_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = w[i];
  }
  __device__ __forceinline__ void turn() {
    // within the lane: word g takes byte g of all four
    auto perm = [](int hi, int lo, unsigned sel) {
      return static_cast<int>(__builtin_amdgcn_perm(hi, lo, sel));
    };
    const int lo01 = perm(v[1], v[0], 0x05010400);
    const int hi01 = perm(v[1], v[0], 0x07030602);
    const int lo23 = perm(v[3], v[2], 0x05010400);
    const int hi23 = perm(v[3], v[2], 0x07030602);
    v[0] = perm(lo23, lo01, 0x05040100);
    v[1] = perm(lo23, lo01, 0x07060302);
    v[2] = perm(hi23, hi01, 0x05040100);
    v[3] = perm(hi23, hi01, 0x07060302);
    // word u of group g <- word g of group u
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto s = __builtin_amdgcn_permlane32_swap(v[i], v[i + 2], false,
                                                      false);
      v[i] = s[0];
      v[i + 2] = s[1];
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const auto s = __builtin_amdgcn_permlane16_swap(v[i], v[i + 1], false,
                                                      false);
      v[i] = s[0];
      v[i + 1] = s[1];
    }
  }
};

template <int MODE, int EPI, int MF, int NF, int W>
__global__ __launch_bounds__(64 * W) void product_rows_kernel(
    ProductArgs p, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int BM = MF * 16, BN = NF * 16;
  const int grid = tiles_m * tiles_n;
  if (static_cast<int>(blockIdx.x) >= grid) {
    zero_rest(p, blockIdx.x - grid, gridDim.x - grid);
    return;
  }
  Tiles<BM> tiles(p);
  const int rows_m = min(tiles.total, tiles_m);
  const int real = rows_m * tiles_n;
  if (static_cast<int>(blockIdx.x) >= real) return;
  // Expert after expert; consecutive workgroups (which go to the XCDs in
  // turn) take consecutive columns, so that all XCDs read one stretch of the
  // weights (a stretch for each XCD has them meet in the same memory
  // channels: 54 instead of 44 us for 256 MiB).  A column's other row tiles
  // follow 8 workgroups behind, on the same XCD, and find it in its L2.
  const GroupTiles group = tiles.group(blockIdx.x / tiles_n);
  const int local = blockIdx.x - group.first * tiles_n;
  const int eight = local / (8 * group.count);
  const int in_eight = local - eight * 8 * group.count;
  const int width = min(8, tiles_n - eight * 8);
  const int first = group.lo + in_eight / width * BM;
  const RowTile tile{group.e, first, min(first + BM, group.hi)};
  const int n0 = (eight * 8 + in_eight % width) * BN;

  // (asked for before the weights, used behind them)
  int source[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
    source[i] = source_row(p, min(tile.lo + i * 16 + (threadIdx.x & 15),
                                  tile.hi - 1));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, g = lane >> 4;
  const size_t row_bytes = p.row_bytes, scale_row = p.row_bytes / 16;
  const uint8_t* pw[NF];
  const uint8_t* sw[NF];
  const uint8_t* px[MF];
  const uint8_t* sx[MF];
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const size_t row = static_cast<size_t>(tile.e) * p.n +
                       min(n0 + j * 16 + fr, p.n - 1);
    pw[j] = p.b + row * row_bytes + g * 16;
    sw[j] = p.b_scales + row * scale_row;
  }

  f32x4 acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // A weight fragment is refilled as soon as it is used.  Loads return in the
  // order they are asked for: a piece's activations go ahead of its weights,
  // into a second buffer while the first is in use.
  Frag fw[NF], fx[2][MF];
  Scales kw[NF], kx[MF];        // of the pieces in use, turned over
  auto fetch_w = [&](int j, int s) { load(fw[j], pw[j] + s * 256); };
  auto fetch_x = [&](int x, int s) {
#pragma unroll
    for (int i = 0; i < MF; ++i) load(fx[x][i], px[i] + s * 256);
  };
  auto use = [&](int j, int x, int u) {
    constexpr std::integral_constant<int, MODE> mode{};
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const Frag &w = fw[j], &a = fx[x][i];
      const int ws = MODE == kMx ? kw[j].v[u] : 0;
      const int xs = MODE == kMx ? kx[i].v[u] : 0;
      mma_piece<0>(acc[i][j], w.v[0], a.v[0], ws, xs, mode);
      mma_piece<1>(acc[i][j], w.v[1], a.v[1], ws, xs, mode);
      mma_piece<2>(acc[i][j], w.v[2], a.v[2], ws, xs, mode);
      mma_piece<3>(acc[i][j], w.v[3], a.v[3], ws, xs, mode);
    }
  };
  const int pieces = p.row_bytes / 256;
  // G pieces in a row go to a wave; those past the last are fetched as the
  // last again and not used
  constexpr int G = MODE == kMx ? 4 : 1;
  const int turns = (pieces + G - 1) / G;
  const int own = wave < turns ? (turns - wave + W - 1) / W : 0;
  const int mine = own * G - (own > 0 && (turns - 1) % W == wave
                                  ? turns * G - pieces : 0);
  auto piece = [&](int q) {
    return min((wave + q / G * W) * G + q % G, pieces - 1);
  };
  auto address_x = [&] {
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const size_t row = source[i];
      px[i] = p.a + row * row_bytes + g * 16;
      sx[i] = p.a_scales + row * scale_row;
    }
  };
  Scales kw_next[NF], kx_next[MF];
  auto fetch_kw = [&](int q) {
#pragma unroll
    for (int j = 0; j < NF; ++j) kw_next[j].load(sw[j] + piece(q + g) * 16);
  };
  auto fetch_kx = [&](int q) {
#pragma unroll
    for (int i = 0; i < MF; ++i) kx_next[i].load(sx[i] + piece(q + g) * 16);
  };
  if (mine > 0) {
    if constexpr (MODE == kMx) fetch_kw(0);
#pragma unroll
    for (int j = 0; j < NF; ++j) fetch_w(j, piece(0));
    address_x();
    if constexpr (MODE == kMx) fetch_kx(0);
    fetch_x(0, piece(0));
    constexpr int U = MODE == kMx ? 4 : 2;
    for (int q = 0; q < mine; q += U) {
      if constexpr (MODE == kMx) {
#pragma unroll
        for (int j = 0; j < NF; ++j) (kw[j] = kw_next[j]).turn();
#pragma unroll
        for (int i = 0; i < MF; ++i) (kx[i] = kx_next[i]).turn();
        fetch_kw(q + U);
        fetch_kx(q + U);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (q + u >= mine) break;
        fetch_x((u + 1) & 1, piece(q + u + 1));
#pragma unroll
        for (int j = 0; j < NF; ++j) {
          use(j, u & 1, u);
          fetch_w(j, piece(q + u + 1));
        }
      }
    }
  }
  // a row's last 64, 128 or 192 bytes: the wave whose turn it is
  const int rest = p.row_bytes - pieces * 256;
  if (rest != 0 && wave == turns % W) {
    auto load_rest = [&](Frag& f, const uint8_t* at) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        f.v[q] = q * 64 < rest ? *reinterpret_cast<const i32x4*>(
                                     at + pieces * 256 + q * 64)
                               : i32x4{0, 0, 0, 0};
    };
    auto scale_rest = [&](const uint8_t* at) {
      unsigned word = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        word |= (q * 64 < rest ? at[pieces * 16 + q * 4 + g] : 0x7fu)
                << (8 * q);
      return static_cast<int>(word);
    };
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      load_rest(fw[j], pw[j]);
      if constexpr (MODE == kMx) kw[j].v[0] = scale_rest(sw[j]);
    }
    address_x();
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      load_rest(fx[0][i], px[i]);
      if constexpr (MODE == kMx) kx[i].v[0] = scale_rest(sx[i]);
    }
#pragma unroll
    for (int j = 0; j < NF; ++j) use(j, 0, 0);
  }

  // the partial tiles meet in LDS: [wave][tile of 16 x 16][lane] float4
  constexpr int kTiles = MF * NF;
  auto* part = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j)
      part[(wave * kTiles + i * NF + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int q = threadIdx.x; q < kTiles * 64; q += 64 * W) {
    f32x4 sum = part[q];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += part[w * kTiles * 64 + q];
    const int l = q & 63, t = q >> 6;
    const int row = tile.lo + (t / NF) * 16 + (l & 15);
    const int col = n0 + (t % NF) * 16 + (l >> 4) * 4;
    if (row < tile.hi && col < p.n) {
      float v[4] = {sum[0], sum[1], sum[2], sum[3]};
      epilogue4<EPI>(p, tile.e, row, col, v);
      *reinterpret_cast<uint2*>(p.c + static_cast<size_t>(row) * p.n + col) =
          uint2{pack2(v[0], v[1]), pack2(v[2], v[3])};
    }
  }
}

template <int MODE, int EPI, int MF, int NF, int W>
hipError_t launch(const ProductArgs& p, hipStream_t stream) {
  const int tiles_m = most_tiles(p.rows_c, p.experts, MF * 16);
  const int tiles_n = (p.n + NF * 16 - 1) / (NF * 16);
  const long long blocks = static_cast<long long>(tiles_m) * tiles_n +
                           (p.zero_rest ? kZeroBlocks : 0);
  constexpr int lds = W * MF * NF * 64 * 16;
  static_assert(lds <= 65536, "more LDS than a launch may ask for");
  return launch_tiles(&product_rows_kernel<MODE, EPI, MF, NF, W>, blocks,
                      64 * W, lds, stream, p, tiles_m, tiles_n);
}

// fragments of 16 columns over all row tiles of MF fragments
long long columns_of(const ProductArgs& p, int mf) {
  return static_cast<long long>(most_tiles(p.rows_c, p.experts, mf * 16)) *
         (p.n / 16);
}
bool short_rows(const ProductArgs& p) { return p.row_bytes <= 2048; }

// Shapes by measurement (us; bf16 weights with rows of 8 KiB, MXFP4 of 2):
//  * MF: so that most groups are one row tile, whose weights are read once.
//    Groups are uneven, so 32 rows from a mean of 8 on (16 experts of 2048
//    columns, 128 rows: 55 against 66 with 16; 8 of MXFP4, rows of 8 KiB: 36
//    against 50; even groups of 16: 59 against 58).  Short rows come out of
//    the cache the second time (320 rows over 32 experts: 67 against 63), and
//    of few columns none may wait for another (13 experts of 208 columns, 170
//    rows: 18 against 14).
//  * columns that do not fill the chip with 64 of them a workgroup: 16, and 4
//    waves along the row (one row against 4096 MXFP4 rows of 8 KiB: 9.0
//    against 13.6 with 32, 9.3 with 8 waves).
//  * columns that do and up to four rows a group: the activations cost
//    little, so 16 columns too (two experts of 16384 columns, one row each:
//    52 against 54 with 32 columns and 8 waves; four of 4096: 29 against
//    34).  Short rows leave nothing to split: 32 columns and 2 waves (33
//    experts: 62 against 69 with 16 columns and 4 waves).
//  * more rows: 64 columns share the activations (eight experts of 4096
//    columns, 16 rows each: 61 against 71 with 32 columns and 8 waves, 79
//    with 16 columns).  Short rows of many columns want one wave, without
//    the sum over the waves (eight experts of 14336 columns, 16 rows each:
//    57 against 65 with 4 waves, bf16 52 against 60; with 32 rows 64 against
//    77; a single one of 28672 columns: 17 against 16).
template <int MODE, int EPI, int MF>
hipError_t launch_rows(const ProductArgs& p, int rows, hipStream_t stream) {
  const long long columns = columns_of(p, MF);
  const bool is_short = short_rows(p);
  if (columns < 1024) return launch<MODE, EPI, MF, 1, 4>(p, stream);
  if constexpr (MF == 1)
    if (rows <= 4)
      return is_short ? launch<MODE, EPI, 1, 2, 2>(p, stream)
                      : launch<MODE, EPI, 1, 1, 4>(p, stream);
  return is_short && columns >= 4096 ? launch<MODE, EPI, MF, 4, 1>(p, stream)
                                     : launch<MODE, EPI, MF, 4, 4>(p, stream);
}

template <int MODE, int EPI>
hipError_t launch_shape(const ProductArgs& p, hipStream_t stream) {
  const int rows = (p.rows_c + p.experts - 1) / p.experts;
  const int one =
      p.experts == 1 || short_rows(p) || columns_of(p, 2) < 512 ? 16 : 7;
  return rows <= one  ? launch_rows<MODE, EPI, 1>(p, rows, stream)
         : rows <= 32 ? launch_rows<MODE, EPI, 2>(p, rows, stream)
                      : launch_rows<MODE, EPI, 4>(p, rows, stream);
}

template <int MODE>
hipError_t launch_mode(const ProductArgs& p, hipStream_t stream) {
  switch (p.epilogue) {
    case PRODUCT_NONE:
      return launch_shape<MODE, PRODUCT_NONE>(p, stream);
    case PRODUCT_BIAS_GELU:
      return launch_shape<MODE, PRODUCT_BIAS_GELU>(p, stream);
    case PRODUCT_BIAS:
      return launch_shape<MODE, PRODUCT_BIAS>(p, stream);
    case PRODUCT_BIAS_RESIDUAL:
      if constexpr (MODE == kMx)
        return launch_shape<MODE, PRODUCT_BIAS_RESIDUAL>(p, stream);
    default:
      return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_product_rows(const ProductArgs& p, hipStream_t stream) {
  return p.a_scales != nullptr ? launch_mode<kMx>(p, stream)
                               : launch_mode<kBf16>(p, stream);
}

}  // namespace kiosk
