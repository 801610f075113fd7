// What the product kernels share: the two operand formats, the search for a
// tile's expert, the epilogue.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "experts.hpp"
#include "launch.hpp"

namespace kiosk {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;

// Rows are walked in steps of 128 bytes, two halves of 64: a half is one
// matrix instruction deep (32 bf16 or 128 MXFP4 elements), lane group
// g = lane >> 4 holds its bytes 16 g .. 16 g + 15 of row lane & 15.  For
// MXFP4 these are the 32 elements of one scale.
enum { kBf16 = 0, kMx = 1 };

// 16x16 tile += A(16 rows) . B(16 rows)^T over one half.  Operands are
// given as (weight rows, activation rows): lane l then holds activation row
// l & 15 and the weight rows 4 (l >> 4) .. + 3, four consecutive columns of
// the product.
template <int MODE>
__device__ __forceinline__ void mma(f32x4& acc, const i32x4& w,
                                    const i32x4& x, int ws, int xs) {
  if constexpr (MODE == kBf16) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0,
        0, 0);
  } else {
    const i32x8 w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0};
    const i32x8 x8 = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    // formats 4: e2m1 for both operands; scale byte 0 of each lane
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc, 4, 4,
                                                           0, ws, 0, xs);
  }
}

// A tile of `BM` product rows: rows [lo, hi) of expert `e` (hi - lo <= BM).
struct RowTile {
  int e, lo, hi;
};

// An expert's tiles: rows [lo, hi), `count` of them, the first is tile
// `first` of all.
struct GroupTiles {
  int e, lo, hi, first, count;
};

// The rows of expert e, whatever the offsets hold: inside [0, rows).
__device__ __forceinline__ void group_bounds(const ProductArgs& p, int e,
                                             int& lo, int& hi) {
  lo = min(max(p.offsets[e], 0), p.rows_c);
  hi = min(max(p.offsets[e + 1], lo), p.rows_c);
}

// Inclusive sum over the lanes of a wave, in the VALU (row shifts, then the
// rows' last lanes carried on): no LDS round trips.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);
  return v;
}

// The tiles of BM rows that the groups make, and where they lie.  The host
// knows the number of rows, not their groups: it launches for the most tiles
// they can make, and every workgroup counts the real ones.  A wave looks at
// 64 groups at a time: lane l counts group base + l's tiles, a scan over the
// lanes finds the one that holds a tile.
template <int BM>
struct Tiles {
  const ProductArgs& p;
  int lane, total;
  // this lane's group of the first 64
  int lo = 0, hi = 0, own = 0, incl = 0;

  __device__ __forceinline__ void look(int base) {
    const int e = base + lane;
    lo = hi = 0;
    if (e < p.experts) group_bounds(p, e, lo, hi);
    own = (hi - lo + BM - 1) / BM;
    incl = wave_scan(own);
  }

  __device__ __forceinline__ explicit Tiles(const ProductArgs& args)
      : p(args), lane(threadIdx.x & (kWave - 1)) {
    if (p.offsets == nullptr) {
      total = (p.rows_c + BM - 1) / BM;
      return;
    }
    total = 0;
    for (int base = 0; base < p.experts; base += kWave) {
      look(base);
      // (groups of a wrong plan may overlap: no sum leaves 32 bits)
      total = min(total + __builtin_amdgcn_readlane(incl, kWave - 1), 1 << 30);
    }
  }

  // the group that holds tile `index` < total
  __device__ __forceinline__ GroupTiles group(int index) {
    if (p.offsets == nullptr) return GroupTiles{0, 0, p.rows_c, 0, total};
    int before = 0;
    for (int base = 0;; base += kWave) {
      if (p.experts > kWave) look(base);
      const unsigned long long past = __ballot(before + incl > index);
      if (past != 0) {
        const int l = __builtin_ctzll(past);
        return GroupTiles{base + l, __builtin_amdgcn_readlane(lo, l),
                          __builtin_amdgcn_readlane(hi, l),
                          before + __builtin_amdgcn_readlane(incl - own, l),
                          __builtin_amdgcn_readlane(own, l)};
      }
      before += __builtin_amdgcn_readlane(incl, kWave - 1);
    }
  }
  __device__ __forceinline__ RowTile find(int index) {
    const GroupTiles g = group(index);
    const int first = g.lo + (index - g.first) * BM;
    return RowTile{g.e, first, min(first + BM, g.hi)};
  }
};

// Row of `a` that product row `i` reads.  An index outside `a` is brought
// inside: no index makes the kernel read past the tensor.
// (A load either way, without a gather one of the weights: a branch around it
// would have the compiler wait for every load in flight where it ends.)
__device__ __forceinline__ int source_row(const ProductArgs& p, int i) {
  const int* at = p.rows != nullptr ? p.rows + i
                                    : reinterpret_cast<const int*>(p.b);
  const int got = *at;
  const int r = p.rows != nullptr ? got : i;
  return min(max(r, 0), p.rows_a - 1);
}

__device__ __forceinline__ void add4(float (&v)[4], const float4& b) {
  v[0] += b.x; v[1] += b.y; v[2] += b.z; v[3] += b.w;
}

__device__ __forceinline__ void gelu4(float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = gelu_tanh(v[i]);
}

__device__ __forceinline__ void add_residual(float (&v)[4], const uint2& r) {
  add4(v, float4{bf16_to_f32(r.x & 0xffff), bf16_to_f32(r.x >> 16),
                 bf16_to_f32(r.y & 0xffff), bf16_to_f32(r.y >> 16)});
}

// v = columns col .. col + 3 of product row `row`, inside the product
template <int EPI>
__device__ __forceinline__ void epilogue4(const ProductArgs& p, int e, int row,
                                          int col, float (&v)[4]) {
  if constexpr (EPI != PRODUCT_NONE)
    add4(v, *reinterpret_cast<const float4*>(
                p.bias + static_cast<size_t>(e) * p.n + col));
  if constexpr (EPI == PRODUCT_BIAS_GELU) gelu4(v);
  if constexpr (EPI == PRODUCT_BIAS_RESIDUAL)
    add_residual(v, *reinterpret_cast<const uint2*>(
                        p.residual + static_cast<size_t>(row) * p.n + col));
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return f32_to_bf16(lo) | (static_cast<uint32_t>(f32_to_bf16(hi)) << 16);
}

// Workgroup `index` of `count` zeroes its share of the rows that no group
// holds: those before the first offset and behind the last.
__device__ __forceinline__ void zero_rest(const ProductArgs& p, int index,
                                          int count) {
  const int first = min(max(p.offsets[0], 0), p.rows_c);
  const int last = min(max(p.offsets[p.experts], first), p.rows_c);
  const size_t head = static_cast<size_t>(first) * p.n;
  const size_t tail = static_cast<size_t>(last) * p.n;
  const size_t end = static_cast<size_t>(p.rows_c) * p.n;
  const size_t step = static_cast<size_t>(count) * blockDim.x * 8;
  const size_t at = (static_cast<size_t>(index) * blockDim.x + threadIdx.x) * 8;
  // n is a multiple of 16, so both spans are of whole 16-byte pieces
  for (size_t i = at; i < head; i += step)
    *reinterpret_cast<uint4*>(p.c + i) = uint4{0, 0, 0, 0};
  for (size_t i = tail + at; i < end; i += step)
    *reinterpret_cast<uint4*>(p.c + i) = uint4{0, 0, 0, 0};
}
constexpr int kZeroBlocks = 64;

// The most row tiles of `bm` that `rows` rows in `experts` groups can make.
__host__ __device__ inline int most_tiles(int rows, int experts, int bm) {
  return experts <= 1 ? (rows + bm - 1) / bm
                      : rows / bm + (experts < rows ? experts : rows);
}

// Launches the first kernel of a product, if its grid is within bounds: fewer
// than 2^32 threads.
template <typename Kernel, typename... Args>
hipError_t launch_tiles(Kernel kernel, long long blocks, int threads,
                        unsigned lds, hipStream_t stream,
                        const ProductArgs& p, Args... args) {
  if (blocks > 0xffffffffll / threads) return hipErrorInvalidConfiguration;
  if (p.dry) return hipSuccess;
  return launch_kernel(kernel, dim3(static_cast<unsigned>(blocks)),
                       dim3(threads), lds, stream, p, args...);
}

// product256.hip
bool product256_ok(const ProductArgs& p);
size_t product256_workspace(const ProductArgs& p);
hipError_t product256_prepare();
hipError_t launch_product256(const ProductArgs& p, hipStream_t stream);
// product256_bf16.hip, product256_mx.hip
hipError_t product256_bf16_prepare();
hipError_t product256_mx_prepare();
hipError_t launch_product256_bf16(const ProductArgs& p, int tiles_n, int grid,
                                  long long blocks, hipStream_t stream);
hipError_t launch_product256_mx(const ProductArgs& p, int tiles_n, int grid,
                                long long blocks, hipStream_t stream);
// product_rows.hip
hipError_t launch_product_rows(const ProductArgs& p, hipStream_t stream);

}  // namespace kiosk
