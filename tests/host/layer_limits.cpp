// Host-only checks of the plan of the layer products (clblast_amd/csrc/device/layer_plans.hpp) at the largest sizes: no grid
// dimension of 2^32 threads, every work-group of a grid in one slice.
// Compiled and run by tests/test_layer_limits_cpu.py.
#include <cstdio>
#include <initializer_list>

#include "clbh_device.h"
#include "device/layer_plans.hpp"

namespace {
long long violations = 0, cases = 0;
void Violation(const char* what, const long long value) {
  if (++violations <= 20) { std::printf("VIOLATION %s: %lld\n", what, value); }
}

void CheckSlices() {
  for (const int threads : {256, 512, 1024}) {
    const long long most = (1ll << 31) / threads;
    for (const long long blocks : {1ll, 7ll, most - 1, most, most + 1, 3 * most - 5, 0x7fffffffll}) {
      ++cases;
      long long next = 0;
      const int status = clbh::LayerSlices(blocks, threads, [&](const int first, const unsigned count) {
        if (first != next || first % 8 != 0) { Violation("slices one behind the other", first); }
        if (count == 0 || static_cast<long long>(count) * threads >= 1ll << 32) { Violation("threads of a slice", count); }
        next += count;
        return 0;
      });
      if (status != 0 || next != blocks) { Violation("the slices make up the grid", next); }
    }
    int calls = 0;
    if (clbh::LayerSlices(2 * most, threads, [&](int, unsigned) { ++calls; return 7; }) != 7 || calls != 1) { Violation("an error ends the launches", calls); }
  }
}
}  // namespace

int main() {
  CheckSlices();
  std::printf("cases %lld violations %lld\n", cases, violations);
  return violations == 0 ? 0 : 1;
}
