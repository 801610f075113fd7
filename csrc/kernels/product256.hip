// Host side of the 256 x 256 tile products, and the sum over their slices.
#include "kernels.hpp"
#include "product256.hpp"

namespace kiosk {
namespace {

using namespace ring256;

template <int EPI>
hipError_t join(const ProductArgs& p, int tiles_n, int pieces,
                hipStream_t stream) {
  // (each workgroup finds its tiles anew: four workgroups a tile will do)
  return launch_kernel(&product256_join_kernel<EPI>, dim3(pieces * 4),
                       dim3(kThreads), 0, stream, p, tiles_n);
}

int columns(const ProductArgs& p) { return (p.n + BN - 1) / BN; }

// The most partial tiles the slices can make; 0: nothing is sliced.
int most_pieces(const ProductArgs& p) {
  const int steps = (p.row_bytes + 127) / 128, tiles_n = columns(p);
  if (steps < kMinFew) return 0;
  if (p.offsets == nullptr) {
    Shares s{};
    const int over = p.rows_c & (BM - 1);
    s.full = p.rows_c / BM + (over > BM / 2);
    s.half = over > 0 && over <= BM / 2;
    s.divide(tiles_n, steps, p.cus, p.cus);
    return s.rest * s.slices;
  }
  // eight rounds and more: the last one's idle time is not worth it
  const long long least =
      static_cast<long long>(p.rows_c / BM) * tiles_n;
  if (least >= 8ll * p.cus || (steps < kMinSteps && least * 4 > p.cus))
    return 0;
  const long long most =
      static_cast<long long>(most_tiles(p.rows_c, p.experts, BM)) * tiles_n *
      kMaxSlices;
  return static_cast<int>(most < p.cus ? most : p.cus);
}

}  // namespace

// 32-bit offsets reach an expert's weights and, with a gather, all of a.
bool product256_ok(const ProductArgs& p) {
  constexpr unsigned long long reach = 0xffffff00ull;
  const unsigned long long bytes = p.row_bytes;
  const unsigned long long rows = p.rows == nullptr ? BM : p.rows_a;
  return (p.a_scales != nullptr || p.row_bytes % 128 == 0) &&
         p.n * bytes < reach && rows * bytes < reach;
}

size_t product256_workspace(const ProductArgs& p) {
  return static_cast<size_t>(most_pieces(p)) * kPieceFloats * sizeof(float);
}

hipError_t product256_prepare() {
  hipError_t err = product256_bf16_prepare();
  if (err == hipSuccess) err = product256_mx_prepare();
  if (err == hipSuccess)
    err = prepare_kernel(&product256_join_kernel<PRODUCT_NONE>);
  if (err == hipSuccess)
    err = prepare_kernel(&product256_join_kernel<PRODUCT_BIAS_GELU>);
  if (err == hipSuccess)
    err = prepare_kernel(&product256_join_kernel<PRODUCT_BIAS_RESIDUAL>);
  if (err == hipSuccess)
    err = prepare_kernel(&product256_join_kernel<PRODUCT_BIAS>);
  return err;
}

hipError_t launch_product256(const ProductArgs& args, hipStream_t stream) {
  ProductArgs p = args;
  const int pieces = p.partial != nullptr ? most_pieces(p) : 0;
  p.pieces = pieces;
  const int tiles_n = columns(p);
  const long long grid =
      static_cast<long long>(most_tiles(p.rows_c, p.experts, BM)) * tiles_n +
      pieces;
  const long long blocks = grid + (p.zero_rest ? kZeroBlocks : 0);
  // (`grid` fits 32 bits where `blocks` is launched)
  const hipError_t err =
      (p.a_scales != nullptr ? launch_product256_mx : launch_product256_bf16)(
          p, tiles_n, static_cast<int>(grid), blocks, stream);
  if (err != hipSuccess || pieces == 0 || p.dry) return err;
  switch (p.epilogue) {
    case PRODUCT_BIAS_GELU:
      return join<PRODUCT_BIAS_GELU>(p, tiles_n, pieces, stream);
    case PRODUCT_BIAS_RESIDUAL:
      return join<PRODUCT_BIAS_RESIDUAL>(p, tiles_n, pieces, stream);
    case PRODUCT_BIAS:
      return join<PRODUCT_BIAS>(p, tiles_n, pieces, stream);
    default:
      return join<PRODUCT_NONE>(p, tiles_n, pieces, stream);
  }
}

}  // namespace kiosk
