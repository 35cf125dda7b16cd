// CPU check of the microscaled and grouped functions of include/b200q.hpp: every case must be rejected on the host before any CUDA
// call.  Prints SHIM-OK on success.
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
  auto x = view(bf, {6, 64}), wq = view(Dtype::uint32, {5, 8}), s = view(Dtype::uint8, {5, 2}), y = view(bf, {6, 5}), w = view(bf, {2, 5, 64});
  auto stack = view(Dtype::uint32, {2, 5, 8}), ss = view(Dtype::uint8, {2, 5, 2}), n = view(Dtype::int64, {2});
  auto one = view(Dtype::float32, {1}), dw = view(bf, {2, 5, 64});
  const Workspace none{};
  int bad = 0;
  bad += refused("integer input", "Only real floating", [&] { quantize(wq, wq, s, Fp4::mxfp4); });
  bad += refused("scales of another group size", "incompatible", [&] { quantize(view(bf, {5, 64}), wq, s, Fp4::nvfp4); });
  bad += refused("global scale with mxfp4", "belongs to nvfp4", [&] { quantize(view(bf, {5, 64}), wq, s, Fp4::mxfp4, one); });
  bad += refused("scales' type", "uint8", [&] { dequantize(wq, view(Dtype::float32, {5, 2}), y, Fp4::mxfp4); });
  bad += refused("output type", "unsupported dtype", [&] { auto o = view(Dtype::uint32, {5, 64}); dequantize(wq, s, o, Fp4::mxfp4); });
  bad += refused("widths", "does not match", [&] { qqmm(view(bf, {6, 32}), wq, s, y, none, Fp4::mxfp4); });
  bad += refused("no workspace", "workspace", [&] { qqmm(x, wq, s, y, none, Fp4::mxfp4); });
  bad += refused("sizes' type", "integral group size", [&] { grouped_qqmm(x, stack, ss, view(Dtype::float32, {2}), y, none, Fp4::mxfp4); });
  bad += refused("number of sizes", "integral group size", [&] { grouped_qqmm(x, stack, ss, view(Dtype::int64, {3}), y, none, Fp4::mxfp4); });
  bad += refused("no workspace for experts", "workspace", [&] { grouped_qqmm(x, stack, ss, n, y, none, Fp4::mxfp4); });
  bad += refused("the other layout", "does not match", [&] { grouped_mm(x, w, n, y, none, false); });
  bad += refused("float32", "unsupported dtype", [&] { grouped_mm(view(Dtype::float32, {6, 64}), view(Dtype::float32, {2, 5, 64}), n, y, none); });
  bad += refused("no workspace for 16 bits", "workspace", [&] { grouped_mm(x, w, n, y, none); });
  bad += refused("rows of dy and x", "as many rows", [&] { grouped_mm_dw(view(bf, {5, 5}), x, n, dw, none); });
  bad += refused("no workspace for the gradient", "workspace", [&] { grouped_mm_dw(view(bf, {6, 5}), x, n, dw, none); });
  if (bad == 0) std::printf("SHIM-OK\n");
  return bad;
}
