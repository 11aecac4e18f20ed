// Descriptors that the device layer of the layer products has to refuse, given to both of its entry points (clblast_amd/csrc/device/
// launch_layer.hip, in the built library): no size, group number or grouping may end the process or reach a launch, and a
// call that is refused asks for no workspace. Compiled, linked with the library and run by tests/test_layer_limits_cpu.py.
#include <cstdio>
#include <initializer_list>

#include "clbh_device.h"

namespace {
int violations = 0, cases = 0;
alignas(256) char memory[4096];

clbh_layer_desc Good(const int grouping) {
  clbh_layer_desc d{};
  d.type = CLBH_TYPE_BF16;
  d.tile_variant = -1;
  d.m = d.n = d.k = 8;
  d.alpha = 1.0f;
  d.a = d.b = d.c = memory;
  d.a_ld = d.b_ld = d.c_ld = 8;
  d.b_kcontig = grouping == CLBH_GROUPS_BY_ROWS;
  d.a_stride = d.c_stride = 64;
  d.activation = 161;
  d.grouping = grouping;
  d.groups = 2;
  d.offsets = reinterpret_cast<const long long*>(memory);
  return d;
}

void Refused(const char* what, const clbh_layer_desc& d) {
  ++cases;
  std::printf("%s\n", what);
  std::fflush(stdout);  // (a process that ends here has named its case)
  const size_t bytes = clbh_layer_workspace_bytes(&d);
  if (bytes != 0) { ++violations; std::printf("VIOLATION %s: workspace of %zu bytes\n", what, bytes); }
  if (clbh_layer_launch(&d, nullptr) == 0) { ++violations; std::printf("VIOLATION %s: launched\n", what); }
}
}  // namespace

int main() {
  ++cases;
  if (clbh_layer_workspace_bytes(nullptr) != 0 || clbh_layer_launch(nullptr, nullptr) == 0) { ++violations; }
  for (const int grouping : {CLBH_GROUPS_NONE, CLBH_GROUPS_BY_ROWS, CLBH_GROUPS_BY_DEPTH}) {
    for (const int size : {0, -1, -2147483647 - 1, 2147483647, 2147483647 - 1022}) {
      auto d = Good(grouping);
      d.m = size;
      Refused("m", d);
      d = Good(grouping);
      d.n = size;
      Refused("n", d);
      d = Good(grouping);
      d.k = size;
      Refused("k", d);
    }
    for (const int type : {0, 15, 64, -1}) {
      auto d = Good(grouping);
      d.type = type;
      Refused("type", d);
    }
    if (grouping == CLBH_GROUPS_NONE) { continue; }
    for (const int groups : {0, -1, -2147483647 - 1, 65537, 2147483647}) {
      auto d = Good(grouping);
      d.groups = groups;
      Refused("groups", d);
      d.upstream = memory;
      d.upstream_ld = 8;
      d.gradient = 1;
      Refused("groups of an elementwise call", d);
    }
    auto d = Good(grouping);
    (grouping == CLBH_GROUPS_BY_ROWS ? d.n : d.k) = 1 << 26;
    Refused("rows of a grouped call", d);
  }
  for (const int type : {CLBH_TYPE_FP16, CLBH_TYPE_FP32}) {  // lines that no 32-bit offset reaches
    auto d = Good(CLBH_GROUPS_NONE);
    d.type = type;
    d.k = (type == CLBH_TYPE_FP32 ? 1 << 26 : 1 << 27) + (1 << 24);
    d.m = 16;
    d.a_kcontig = 1;
    d.a_ld = d.k;
    Refused("k-contiguous lines", d);
    d = Good(CLBH_GROUPS_NONE);
    d.type = type;
    d.n = type == CLBH_TYPE_FP32 ? 160000000 : 320000000;
    d.k = 1;
    d.b_ld = d.n;
    Refused("lines of rows", d);
  }
  for (const int grouping : {-1, 3, 2147483647}) { Refused("grouping", Good(grouping)); }
  std::printf("cases %d violations %d\n", cases, violations);
  return violations == 0 ? 0 : 1;
}
