#include "bind_experts.hpp"

#include "../kernels/experts.hpp"
#include "engine.hpp"

namespace py = pybind11;

namespace kiosk {
namespace {

typedef unsigned long long addr_t;

template <typename T>
T* ptr(addr_t p) {
  return reinterpret_cast<T*>(static_cast<uintptr_t>(p));
}

hipStream_t stream_of(addr_t s) {
  return reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(s));
}

// A product's sizes without its operands; `grouped`, `gather`: offsets and
// rows are given.
ProductArgs product_sizes(bool mx, bool grouped, bool gather, int rows_a,
                          int rows_c, int n, int row_bytes, int experts,
                          int cus) {
  static const uint8_t some = 0;
  static const int one = 0;
  ProductArgs p{};
  p.a_scales = p.b_scales = mx ? &some : nullptr;
  p.offsets = grouped ? &one : nullptr;
  p.rows = gather ? &one : nullptr;
  p.rows_a = rows_a;
  p.rows_c = rows_c;
  p.n = n;
  p.row_bytes = row_bytes;
  p.experts = experts;
  p.cus = cus;
  return p;
}

}  // namespace

void bind_experts(py::module_& m) {
  m.attr("route_max_experts") = kRouteMaxExperts;
  m.attr("route_max_k") = kRouteMaxK;
  m.attr("product_max_experts") = kProductMaxExperts;
  m.def("route_count_words", &route_count_words, py::arg("tokens"),
        py::arg("experts"));
  m.def(
      "route",
      [](addr_t logits, bool bf16, int tokens, int experts, int k,
         bool renormalize, addr_t chosen, addr_t weights, addr_t row_tokens,
         addr_t positions, addr_t offsets, addr_t counts, addr_t stream) {
        RouteArgs a;
        a.logits = ptr<const void>(logits);
        a.bf16 = bf16;
        a.tokens = tokens;
        a.experts = experts;
        a.k = k;
        a.renormalize = renormalize;
        a.chosen = ptr<int>(chosen);
        a.weights = ptr<float>(weights);
        a.row_tokens = ptr<int>(row_tokens);
        a.positions = ptr<int>(positions);
        a.offsets = ptr<int>(offsets);
        a.counts = ptr<int>(counts);
        check_hip(launch_route(a, stream_of(stream)), "route");
      },
      py::arg("logits"), py::arg("bf16"), py::arg("tokens"),
      py::arg("experts"), py::arg("k"), py::arg("renormalize"),
      py::arg("chosen"), py::arg("weights"), py::arg("row_tokens"),
      py::arg("positions"), py::arg("offsets"), py::arg("counts"),
      py::arg("stream"), py::call_guard<py::gil_scoped_release>());
  m.def(
      "combine",
      [](addr_t y, addr_t positions, addr_t weights, addr_t residual,
         addr_t out, int tokens, int k, int rows, int width, addr_t stream) {
        check_hip(launch_combine(ptr<const uint16_t>(y),
                                 ptr<const int>(positions),
                                 ptr<const float>(weights),
                                 ptr<const uint16_t>(residual),
                                 ptr<uint16_t>(out), tokens, k, rows, width,
                                 stream_of(stream)),
                  "combine");
      },
      py::arg("y"), py::arg("positions"), py::arg("weights"),
      py::arg("residual"), py::arg("out"), py::arg("tokens"), py::arg("k"),
      py::arg("rows"), py::arg("width"), py::arg("stream"),
      py::call_guard<py::gil_scoped_release>());
  m.def(
      "mxfp4_quantize",
      [](addr_t x, bool bf16, addr_t codes, addr_t scales, size_t n,
         addr_t stream) {
        check_hip(launch_mxfp4_quantize(ptr<const void>(x), bf16,
                                        ptr<uint8_t>(codes),
                                        ptr<uint8_t>(scales), n,
                                        stream_of(stream)),
                  "mxfp4_quantize");
      },
      py::arg("x"), py::arg("bf16"), py::arg("codes"), py::arg("scales"),
      py::arg("n"), py::arg("stream"),
      py::call_guard<py::gil_scoped_release>());
  m.def(
      "mxfp4_dequantize",
      [](addr_t codes, addr_t scales, addr_t out, bool bf16, size_t n,
         addr_t stream) {
        check_hip(launch_mxfp4_dequantize(ptr<const uint8_t>(codes),
                                          ptr<const uint8_t>(scales),
                                          ptr<void>(out), bf16, n,
                                          stream_of(stream)),
                  "mxfp4_dequantize");
      },
      py::arg("codes"), py::arg("scales"), py::arg("out"), py::arg("bf16"),
      py::arg("n"), py::arg("stream"),
      py::call_guard<py::gil_scoped_release>());
  // bytes of workspace for such a product, and the kernel that it runs on
  m.def("product_workspace", [](bool mx, bool grouped, bool gather, int rows_a,
                                int rows_c, int n, int row_bytes, int experts,
                                int cus) {
    return product_workspace(product_sizes(mx, grouped, gather, rows_a, rows_c,
                                           n, row_bytes, experts, cus));
  });
  m.def("product_kernel", [](bool mx, bool grouped, bool gather, int rows_a,
                             int rows_c, int n, int row_bytes, int experts,
                             int cus) {
    return product_kernel(product_sizes(mx, grouped, gather, rows_a, rows_c, n,
                                        row_bytes, experts, cus));
  });
  m.def(
      "product",
      [](addr_t a, addr_t a_scales, addr_t b, addr_t b_scales, addr_t c,
         addr_t bias, addr_t residual, addr_t offsets, addr_t rows,
         int rows_a, int rows_c, int n, int row_bytes, int experts,
         int epilogue, bool zero_rest, int cus, addr_t partial,
         addr_t stream) {
        ProductArgs p{};
        p.cus = cus;
        p.partial = ptr<float>(partial);
        p.a = ptr<const uint8_t>(a);
        p.a_scales = ptr<const uint8_t>(a_scales);
        p.b = ptr<const uint8_t>(b);
        p.b_scales = ptr<const uint8_t>(b_scales);
        p.c = ptr<uint16_t>(c);
        p.bias = ptr<const float>(bias);
        p.residual = ptr<const uint16_t>(residual);
        p.offsets = ptr<const int>(offsets);
        p.rows = ptr<const int>(rows);
        p.rows_a = rows_a;
        p.rows_c = rows_c;
        p.n = n;
        p.row_bytes = row_bytes;
        p.experts = experts;
        p.epilogue = epilogue;
        p.zero_rest = zero_rest;
        p.dry = true;
        if (launch_product(p, nullptr) == hipErrorInvalidConfiguration)
          throw py::value_error(
              "a product of so many experts and columns has more tiles than "
              "one launch takes (2^32 threads): split the columns");
        p.dry = false;
        check_hip(experts_prepare(), "experts_prepare");
        check_hip(launch_product(p, stream_of(stream)), "product");
      },
      py::arg("a"), py::arg("a_scales"), py::arg("b"), py::arg("b_scales"),
      py::arg("c"), py::arg("bias"), py::arg("residual"), py::arg("offsets"),
      py::arg("rows"), py::arg("rows_a"), py::arg("rows_c"), py::arg("n"),
      py::arg("row_bytes"), py::arg("experts"), py::arg("epilogue"),
      py::arg("zero_rest"), py::arg("cus"), py::arg("partial"),
      py::arg("stream"),
      py::call_guard<py::gil_scoped_release>());
}

}  // namespace kiosk
