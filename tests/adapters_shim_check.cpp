// CPU check of add_adapters_grad of include/b200q.hpp: which gradients need the forward pass's inner products.  Widths of zero: what is accepted launches nothing.  Prints
// SHIM-OK on success.
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

int main() {
  const auto bf = Dtype::bfloat16, i32 = Dtype::int32;
  const Workspace none{}, some{reinterpret_cast<void*>(0x1000), 1 << 20};
  const RowGroups g{view(i32, {3}), view(i32, {4}), view(i32, {6}), view(i32, {b200q_group_rows_tiles(6, 3), 4})};
  const auto a = view(bf, {3, 4, 0}), b = view(bf, {3, 0, 4}), x = view(bf, {6, 0}), dy = view(bf, {6, 0});
  int bad = 0;
  auto call = [&](const char* what, bool ok, const Workspace& h, const Workspace& s, bool for_x, bool for_a, bool for_b) {
    ArrayView dx = for_x ? view(bf, {6, 0}) : ArrayView{}, da = for_a ? view(bf, {3, 4, 0}) : ArrayView{}, db = for_b ? view(bf, {3, 0, 4}) : ArrayView{};
    bool accepted = true;
    try {
      add_adapters_grad(dy, x, a, b, g, h, s, dx, da, db);
    } catch (const std::exception& e) {
      accepted = false;
      if (!std::strstr(e.what(), "too small")) { std::printf("%s: %s\n", what, e.what()); ++bad; }
    }
    if (accepted != ok) { std::printf("%s: %s\n", what, accepted ? "accepted" : "refused"); ++bad; }
  };
  call("all", true, some, some, true, true, true);
  call("x alone, without inner products", true, none, some, true, false, false);
  call("a alone, without inner products", true, none, some, false, true, false);
  call("x and a, without inner products", true, none, some, true, true, false);
  call("b alone, without scratch", true, some, none, false, false, true);
  call("b without inner products", false, none, some, false, false, true);
  call("x without scratch", false, some, none, true, false, false);
  call("a without scratch", false, some, none, false, true, false);
  if (bad == 0) std::printf("SHIM-OK\n");
  return bad;
}
