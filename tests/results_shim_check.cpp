// CPU check of include/b200q.hpp: results that are not as large as what the microscaled and grouped functions would write must be
// rejected on the host before any CUDA call.  Prints SHIM-OK on success.
#include <cstdio>
#include <cstring>

#include "b200q.hpp"

using namespace b200q;

static ArrayView view(Dtype t, std::vector<int64_t> shape) {
  ArrayView a;
  a.data = reinterpret_cast<void*>(0x1000);
  a.dtype = t;
  a.shape = std::move(shape);
  return a;
}
template <class F>
static int refused(const char* what, const char* needle, F f) {
  try {
    f();
  } catch (const std::exception& e) {
    if (std::strstr(e.what(), needle)) return 0;
    std::printf("%s: wrong message: %s\n", what, e.what());
    return 1;
  }
  std::printf("%s: not rejected\n", what);
  return 1;
}

int main() {
  const auto bf = Dtype::bfloat16;
  auto x = view(bf, {6, 64}), wq = view(Dtype::uint32, {5, 8}), s = view(Dtype::uint8, {5, 2}), w = view(bf, {2, 5, 64});
  auto stack = view(Dtype::uint32, {2, 5, 8}), ss = view(Dtype::uint8, {2, 5, 2}), n = view(Dtype::int64, {2});
  const Workspace none{};
  int bad = 0;
  bad += refused("more rows than codes", "does not match the packed matrix", [&] { quantize(view(bf, {6, 64}), wq, s, Fp4::mxfp4); });
  bad += refused("wider than the codes", "does not match the packed matrix", [&] { quantize(view(bf, {5, 128}), wq, s, Fp4::mxfp4); });
  bad += refused("a vector", "does not match the packed matrix", [&] { quantize(view(bf, {64}), wq, s, Fp4::mxfp4); });
  bad += refused("no dimensions", "does not match the packed matrix", [&] { quantize(view(bf, {}), wq, s, Fp4::mxfp4); });
  bad += refused("a stack as a matrix", "does not match the packed matrix", [&] { quantize(view(bf, {10, 64}), stack, ss, Fp4::mxfp4); });
  for (auto shape : {std::vector<int64_t>{5, 32}, {4, 64}, {}}) {
    auto small = view(bf, shape);
    bad += refused("dequantize", "elements", [&] { dequantize(wq, s, small, Fp4::mxfp4); });
    bad += refused("qqmm", "elements", [&] { qqmm(x, wq, s, small, none, Fp4::mxfp4); });
    bad += refused("grouped_qqmm", "elements", [&] { grouped_qqmm(x, stack, ss, n, small, none, Fp4::mxfp4); });
    bad += refused("grouped_mm", "elements", [&] { grouped_mm(x, w, n, small, none); });
    bad += refused("grouped_mm_dw", "elements", [&] { grouped_mm_dw(view(bf, {6, 5}), x, n, small, none); });
  }
  auto f = view(Dtype::float32, {6, 5}), h = view(Dtype::float16, {2, 5, 64});
  bad += refused("another type", "dtype of the result", [&] { qqmm(x, wq, s, f, none, Fp4::mxfp4); });
  bad += refused("another type, experts", "dtype of the result", [&] { grouped_qqmm(x, stack, ss, n, f, none, Fp4::mxfp4); });
  bad += refused("another type, 16 bits", "dtype of the result", [&] { grouped_mm(x, w, n, f, none); });
  bad += refused("another type, gradient", "dtype of the result", [&] { grouped_mm_dw(view(bf, {6, 5}), x, n, h, none); });
  // what fits goes on to the library
  auto y = view(bf, {6, 5}), flat = view(bf, {30});
  bad += refused("as large", "workspace", [&] { qqmm(x, wq, s, y, none, Fp4::mxfp4); });
  bad += refused("as large, of another shape", "workspace", [&] { qqmm(x, wq, s, flat, none, Fp4::mxfp4); });
  if (bad == 0) std::printf("SHIM-OK\n");
  return bad;
}
