// Host-only checks of the plan of the layer products (clblast_amd/csrc/device/layer_plans.hpp) at the largest sizes: no grid
// dimension of 2^32 threads, every work-group of a grid in one slice, the work-groups' rows and the K ranges make up the
// sizes up to the largest ones, lines that are too far apart for 32-bit offsets are told from those that are not.
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

void CheckLargest() {
  char* const place = reinterpret_cast<char*>(4096);
  constexpr int kMost = static_cast<int>(CLBH_LAYER_MAX_SIZE);
  for (const int type : {CLBH_TYPE_FP16, CLBH_TYPE_FP32, CLBH_TYPE_BF16})
  for (const int large : {kMost, kMost - 1, kMost - 4097, kMost - 9000, 1 << 30, (1 << 30) + 1})
  for (const int small : {1, 2, 8, 9, 17, 64}) {
    ++cases;
    clbh_layer_desc d{};
    d.type = type;
    d.tile_variant = -1;
    d.m = small; d.n = large; d.k = 1;
    d.gradient = 1;
    d.activation = 161;
    d.upstream = d.c = d.bias_gradient = place;
    d.upstream_ld = d.c_ld = small;
    const auto rows = clbh::PlanLayer(d, 256);  // elementwise, many rows
    if (rows.rows_chunk < 1 || rows.rows_chunks * rows.rows_chunk < large || (rows.rows_chunks - 1) * rows.rows_chunk >= large) { Violation("chunks of rows", rows.rows_chunks); }
    if (rows.workspace_bytes < sizeof(float) * rows.rows_chunks * small || rows.workspace_bytes > sizeof(float) * rows.rows_chunks * small + 256) { Violation("workspace of the sums", static_cast<long long>(rows.workspace_bytes)); }
    d.upstream = nullptr;
    d.gradient = 0;
    d.bias_gradient = nullptr;
    d.a = d.b = place;
    for (const bool deep : {false, true}) {  // products of many rows, and of a long depth
      d.n = deep ? small : large;
      d.k = deep ? large : small;
      d.a_kcontig = d.b_kcontig = 1;
      d.a_ld = d.b_ld = d.k;
      for (const int split : {0, 2, 3, 7, 32}) {
        d.split_k = split;
        const auto plan = clbh::PlanLayer(d, 256);
        if (plan.tiles_n * plan.tile.tile_n < d.n || (plan.tiles_n - 1) * plan.tile.tile_n >= d.n) { Violation("tiles along the rows", plan.tiles_n); }
        if (plan.splits < 1 || (split > 1 && deep && plan.splits != split)) { Violation("K ranges", plan.splits); }
        if (plan.splits > 1 && (static_cast<long long>(plan.chunk) * plan.splits < d.k || static_cast<long long>(plan.chunk) * (plan.splits - 1) >= d.k)) { Violation("length of the K ranges", plan.chunk); }
      }
    }
  }
}

// The offsets of a piece's lines as the loads take them, unsigned and in 32 bits: of every line that counts it is the true one
void CheckReach() {
  for (const int type : {CLBH_TYPE_FP16, CLBH_TYPE_FP32, CLBH_TYPE_BF16})
  for (const bool k_contiguous : {false, true})
  for (const long long lines : {1ll, 2ll, 3ll, 8ll, 9ll, 16ll, 17ll, 1000ll}) {
    const long long size = type == CLBH_TYPE_FP32 ? 4 : 2;
    const auto wraps = [&](const long long ld) {
      for (long long line = 0; line < (k_contiguous ? 16 : 8); ++line) {
        if (k_contiguous && line >= lines) { break; }  // (what a row that does not exist fetches is not stored)
        const long long last = line * ld * size + 511;
        if (static_cast<long long>(static_cast<unsigned>(last)) != last) { return true; }
      }
      return false;
    };
    for (long long ld = 8; ld < 1ll << 33; ld = ld * 5 / 4 / 8 * 8 + 8) {
      ++cases;
      if (clbh::LayerLinesReachable(k_contiguous, lines, ld, type) == wraps(ld)) { Violation("lines within reach", ld); }
    }
  }
  for (const long long length : {1ll, 8ll, 9ll, 16ll, 2147482624ll}) {
    if (clbh::LayerCopyLd(length) < length || clbh::LayerCopyLd(length) % 8 != 0) { Violation("leading dimension of a copy", length); }
  }
}
}  // namespace

int main() {
  CheckReach();
  CheckSlices();
  CheckLargest();
  std::printf("cases %lld violations %lld\n", cases, violations);
  return violations == 0 ? 0 : 1;
}
