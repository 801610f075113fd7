// Host-side launchers of the expert-MLP operators: the router and its plan,
// products grouped by expert (bf16 or MXFP4), the weighted sum behind them,
// and the MXFP4 codec.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace kiosk {

// Router.  logits [tokens, experts] (fp32, or bf16 when `bf16`).  Limits:
// experts <= kRouteMaxExperts, k <= min(experts, kRouteMaxK).
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;
struct RouteArgs {
  const void* logits;
  int bf16;
  int tokens, experts, k;
  int renormalize;
  int* chosen;        // [tokens, k]
  float* weights;     // [tokens, k]
  int* row_tokens;    // [tokens * k]
  int* positions;     // [tokens, k]
  int* offsets;       // [experts + 1]
  int* counts;        // [route_count_words(tokens, experts)] scratch
};
size_t route_count_words(int tokens, int experts);
hipError_t launch_route(const RouteArgs& args, hipStream_t stream);

// out[t] = residual[t] + sum_j weights[t, j] * y[positions[t, j]]; width a
// multiple of 8.  A position outside [0, rows) adds nothing.
hipError_t launch_combine(const uint16_t* y, const int* positions,
                          const float* weights, const uint16_t* residual,
                          uint16_t* out, int tokens, int k, int rows,
                          int width, hipStream_t stream);

// MXFP4: blocks of 32 elements (n a multiple of 32), codes n / 2 bytes (low
// nibble first), scales n / 32 bytes (E8M0).  `x`/`out` bf16 or fp32.
hipError_t launch_mxfp4_quantize(const void* x, int bf16, uint8_t* codes,
                                 uint8_t* scales, size_t n,
                                 hipStream_t stream);
hipError_t launch_mxfp4_dequantize(const uint8_t* codes,
                                   const uint8_t* scales, void* out, int bf16,
                                   size_t n, hipStream_t stream);

constexpr int kProductMaxExperts = 65536;
enum ProductEpilogue {
  PRODUCT_NONE = 0,
  PRODUCT_BIAS_GELU = 1,
  PRODUCT_BIAS_RESIDUAL = 2,
  PRODUCT_BIAS = 3,
};

// c[i] = epi(a[rows[i]] . b[e]^T), offsets[e] <= i < offsets[e + 1].
// Operands are rows of `row_bytes` (a multiple of 64): bf16 (scales null) or
// MXFP4 codes with their scale rows of row_bytes / 16 bytes.
struct ProductArgs {
  const uint8_t* a;
  const uint8_t* a_scales;
  const uint8_t* b;
  const uint8_t* b_scales;
  uint16_t* c;
  const float* bias;          // [experts, n]
  const uint16_t* residual;   // [rows_c, n], MXFP4 only
  const int* offsets;         // [experts + 1], null: one group of all rows
  const int* rows;            // [rows_c] gather, null: row i of a
  int rows_a, rows_c, n, row_bytes, experts;
  int epilogue;
  int zero_rest;              // zero the rows that belong to no group
  int cus;                    // compute units of the device
  float* partial;             // workspace (product_workspace bytes) or null
  int pieces;                 // partial tiles that it holds (set by launch)
  bool dry;                   // check the sizes, launch nothing
};
// Bytes of fp32 workspace that speed the product up (0: none is used).  Only
// the sizes, `cus` and whether scales, offsets and rows are null matter.
size_t product_workspace(const ProductArgs& args);
// The kernel that such a product runs on: "rows", "tile128" or "tile256".
const char* product_kernel(const ProductArgs& args);
// hipErrorInvalidConfiguration: more tiles than one launch takes.
hipError_t launch_product(const ProductArgs& args, hipStream_t stream);
hipError_t experts_prepare();   // load the code objects, raise LDS limits

}  // namespace kiosk
