// CPU check of the routing and adapter functions of include/b200q.hpp: every case must be rejected on the host before any CUDA call.  Prints SHIM-OK on success.
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
  const auto bf = Dtype::bfloat16, f32 = Dtype::float32, i32 = Dtype::int32;
  const Workspace none{}, some{reinterpret_cast<void*>(0x1000), 1 << 20};
  auto routing = [&](int64_t T) { return Routing{view(f32, {T, 2}), view(i32, {T, 2}), view(i32, {8}), view(i32, {T, 2}), view(i32, {2 * T})}; };
  Routing r = routing(6);
  auto x = view(bf, {6, 16}), y = view(bf, {12, 16}), o = view(bf, {6, 16});
  int bad = 0;
  bad += refused("integer logits", "do not match", [&] { route_experts(view(i32, {6, 8}), r, some); });
  bad += refused("number of tokens", "do not match", [&] { route_experts(view(f32, {5, 8}), r, some); });
  bad += refused("number of experts", "does not have 9", [&] { route_experts(view(f32, {6, 9}), r, some); });
  bad += refused("weights' type", "unsupported dtype", [&] { Routing q = routing(6); q.weights = view(bf, {6, 2}); route_experts(view(f32, {6, 8}), q, some); });
  bad += refused("bias", "does not have 8", [&] { RouteOptions p; p.bias = view(f32, {7}); route_experts(view(f32, {6, 8}), r, some, p); });
  bad += refused("groups", "groups of 8 experts", [&] { RouteOptions p; p.groups = 3; route_experts(view(f32, {6, 8}), r, some, p); });
  bad += refused("no workspace", "workspace", [&] { Routing q = routing(4096); route_experts(view(f32, {4096, 8}), q, none); });
  bad += refused("gradient's shape", "does not have", [&] { auto d = view(f32, {6, 7}); route_dlogits(view(f32, {6, 2}), view(f32, {6, 8}), r.experts, d); });
  bad += refused("rows of x", "for every token", [&] { dispatch_rows(view(bf, {5, 16}), r, y); });
  bad += refused("places' type", "one entry per pair", [&] { Routing q = routing(6); q.places = view(Dtype::int64, {6, 2}); dispatch_rows(x, q, y); });
  bad += refused("rows of the result", "does not have", [&] { dispatch_rows(x, r, o); });
  bad += refused("type", "unsupported dtype", [&] { auto u = view(i32, {12, 16}); dispatch_rows(view(i32, {6, 16}), r, u); });
  bad += refused("rows of y", "for every pair", [&] { combine_rows(x, r, o); });
  bad += refused("width of the result", "does not have", [&] { auto u = view(bf, {6, 15}); combine_rows(y, r, u); });
  bad += refused("gradient of the result", "does not match", [&] { ArrayView no; combine_rows_grad(view(bf, {6, 15}), y, r, no, no); });
  RowGroups g{view(i32, {3}), view(i32, {4}), view(i32, {6}), view(i32, {b200q_group_rows_tiles(6, 3), 4})};
  auto a = view(bf, {3, 4, 16}), b = view(bf, {3, 32, 4}), base = view(bf, {6, 32});
  bad += refused("ids' type", "int32 or int64", [&] { group_rows(view(f32, {6}), 3, g, some); });
  bad += refused("number of ids", "does not have", [&] { group_rows(view(i32, {7}), 3, g, some); });
  bad += refused("no workspace for groups", "workspace", [&] {
    RowGroups q{view(i32, {3}), view(i32, {4}), view(i32, {5000}), view(i32, {b200q_group_rows_tiles(5000, 3), 4})};
    group_rows(view(i32, {5000}), 3, q, none);
  });
  bad += refused("width of x", "do not match", [&] { add_adapters(base, view(bf, {6, 15}), a, b, g, some, base); });
  bad += refused("types", "one type", [&] { add_adapters(base, view(Dtype::float16, {6, 16}), a, b, g, some, base); });
  bad += refused("float32", "unsupported dtype", [&] {
    auto u = view(f32, {6, 32});
    add_adapters(u, view(f32, {6, 16}), view(f32, {3, 4, 16}), view(f32, {3, 32, 4}), g, some, u);
  });
  bad += refused("groups of other rows", "does not have", [&] { add_adapters(view(bf, {5, 32}), view(bf, {5, 16}), a, b, g, some, base); });
  bad += refused("scales", "does not have 3", [&] { add_adapters(base, x, a, b, g, some, base, view(f32, {2})); });
  bad += refused("inner products", "too small", [&] { add_adapters(base, x, a, b, g, none, base); });
  bad += refused("gradient's shape", "does not have", [&] { ArrayView no; auto d = view(bf, {6, 15}); add_adapters_grad(base, x, a, b, g, some, some, d, no, no); });
  bad += refused("scratch of the gradient", "too small", [&] { ArrayView no; auto d = view(bf, {6, 16}); add_adapters_grad(base, x, a, b, g, some, none, d, no, no); });
  if (bad == 0) std::printf("SHIM-OK\n");
  return bad;
}
