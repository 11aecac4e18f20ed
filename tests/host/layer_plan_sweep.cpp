// Host-only sweep of the plan of the layer products (clblast_amd/csrc/device/layer_plans.hpp, compiled next to this file by
// tests/test_layers_cpu.py): the tiles cover the result, the K ranges cover the depth once in whole slabs, group tiles never
// outnumber the work-groups, and the pieces of the workspace neither overlap nor leave it.
#include <cstdio>
#include <initializer_list>
#include <vector>

#include "clbh_device.h"
#include "device/layer_plans.hpp"

namespace {
long long violations = 0, cases = 0;
void Violation(const char* what, const clbh_layer_desc& d) {
  ++violations;
  std::printf("VIOLATION %s: type %d m %d n %d k %d grouping %d groups %d variant %d split %d\n", what, d.type, d.m, d.n, d.k, d.grouping,
              d.groups, d.tile_variant, d.split_k);
}
unsigned long long state = 12345;
long long Random(const long long below) {
  state = state * 6364136223846793005ull + 1442695040888963407ull;
  return static_cast<long long>((state >> 33) % static_cast<unsigned long long>(below));
}

void Check(const clbh_layer_desc& d, const int units) {
  ++cases;
  const auto plan = clbh::PlanLayer(d, units);
  const bool by_rows = d.grouping == CLBH_GROUPS_BY_ROWS;
  const size_t size = d.type == CLBH_TYPE_FP32 ? 4 : 2;
  std::vector<std::pair<size_t, size_t>> pieces;
  if (d.upstream == nullptr) {
    if (!clbh::LayerTileExists(d.type, plan.tile)) { Violation("no such tile", d); }
    if (plan.tiles_m * plan.tile.tile_m < d.m || (plan.tiles_m - 1) * plan.tile.tile_m >= d.m) { Violation("tiles along the features", d); }
    if (!by_rows && (plan.tiles_n * plan.tile.tile_n < d.n || (plan.tiles_n - 1) * plan.tile.tile_n >= d.n)) { Violation("tiles along the rows", d); }
    if (plan.splits < 1 || (plan.splits > 1 && d.grouping != CLBH_GROUPS_NONE)) { Violation("K ranges of a grouped call", d); }
    if (plan.splits > 1) {
      if (plan.chunk % 64 != 0 || static_cast<long long>(plan.chunk) * plan.splits < d.k || static_cast<long long>(plan.chunk) * (plan.splits - 1) >= d.k) { Violation("K ranges", d); }
      pieces.emplace_back(0, size_t{4} * plan.splits * d.n * d.m);
    }
    if (plan.a_copy_ld > 0) {
      if (plan.a_copy_ld % 8 != 0 || plan.a_copy_ld < (d.a_kcontig ? d.k : d.m)) { Violation("copy of a", d); }
      pieces.emplace_back(plan.a_copy_offset, size * plan.a_copy_ld * (d.a_kcontig ? d.m : d.k) * (by_rows ? d.groups : 1));
    }
    if (plan.b_copy_ld > 0) {
      if (plan.b_copy_ld % 8 != 0 || plan.b_copy_ld < (d.b_kcontig ? d.k : d.n)) { Violation("copy of b", d); }
      pieces.emplace_back(plan.b_copy_offset, size * plan.b_copy_ld * (d.b_kcontig ? d.n : d.k));
    }
    const bool fit_a = clbh::LayerOperandFits(d.a, d.a_ld, by_rows ? d.a_stride : 0, d.type), fit_b = clbh::LayerOperandFits(d.b, d.b_ld, 0, d.type);
    if (fit_a == (plan.a_copy_ld > 0) || fit_b == (plan.b_copy_ld > 0)) { Violation("which operands are copied", d); }
  }
  const bool elementwise = d.upstream != nullptr || plan.splits > 1;
  if (elementwise && (plan.rows_chunk < 1 || (!by_rows && plan.rows_chunks * plan.rows_chunk < d.n))) { Violation("chunks of rows", d); }
  if (d.bias_gradient != nullptr) {
    pieces.emplace_back(plan.sums_offset, size_t{4} * d.m * (elementwise ? plan.rows_chunks : plan.tiles_n));
  }
  for (size_t i = 0; i < pieces.size(); ++i) {
    if (pieces[i].first % 256 != 0 || pieces[i].first + pieces[i].second > plan.workspace_bytes) { Violation("a piece leaves the workspace", d); }
    for (size_t j = 0; j < i; ++j) {
      if (pieces[i].first < pieces[j].first + pieces[j].second && pieces[j].first < pieces[i].first + pieces[i].second) { Violation("pieces overlap", d); }
    }
  }
  if (by_rows) {  // groups of any sizes within the rows
    for (int attempt = 0; attempt < 4; ++attempt) {
      long long left = d.n, tiles = 0, chunks = 0;
      for (int g = 0; g < d.groups; ++g) {
        long long rows = attempt == 0 ? left / (d.groups - g) : attempt == 1 ? std::min<long long>(left, 1) : Random(left + 1);
        if (attempt == 3 && g == d.groups - 1) { rows = left; }
        left -= rows;
        if (d.upstream == nullptr) { tiles += (rows + plan.tile.tile_n - 1) / plan.tile.tile_n; }
        chunks += (rows + plan.rows_chunk - 1) / plan.rows_chunk;
      }
      if (d.upstream == nullptr && tiles > plan.tiles_n) { Violation("more tiles than work-groups", d); }
      if (chunks > plan.rows_chunks) { Violation("more chunks than work-groups", d); }
    }
  }
}
}  // namespace

int main() {
  char* const place = reinterpret_cast<char*>(4096);
  for (const int type : {CLBH_TYPE_FP16, CLBH_TYPE_FP32, CLBH_TYPE_BF16})
  for (const int m : {1, 3, 64, 65, 130, 1000, 1001, 4096, 8192, 40000})
  for (const int n : {1, 2, 17, 64, 129, 777, 4096, 16384, 100001})
  for (const int k : {1, 15, 64, 100, 513, 1023, 4096, 65536})
  for (int form = 0; form < 7; ++form)
  for (const int units : {8, 256, 304}) {
    if (static_cast<double>(m) * n > 1e9) { continue; }
    clbh_layer_desc d{};
    d.type = type;
    d.tile_variant = (form == 6) ? static_cast<int>(Random(7)) - 1 : -1;
    d.split_k = (form == 6) ? static_cast<int>(Random(20)) : 0;
    d.m = m; d.n = n; d.k = k;
    d.a_kcontig = Random(2); d.b_kcontig = Random(2);
    d.a = place + 2 * Random(3) * (type == CLBH_TYPE_FP32 ? 2 : 1); d.b = place; d.c = place;
    d.a_ld = (d.a_kcontig ? k : m) + Random(4); d.b_ld = (d.b_kcontig ? k : n) + Random(4); d.c_ld = m;
    if (Random(20) == 0) { d.b_ld += 1 << 22; }
    d.activation = 161;
    if (form == 1 || form == 2 || form == 6) { d.gradient = 1; d.bias_gradient = place; d.pre = place; d.pre_ld = m; }
    if (form == 2) { d.upstream = place; d.upstream_ld = m; d.groups = 1 + Random(70); d.grouping = Random(2) ? CLBH_GROUPS_BY_ROWS : CLBH_GROUPS_NONE; }
    if (form == 3 || form == 4) { d.grouping = CLBH_GROUPS_BY_ROWS; d.groups = 1 + Random(form == 3 ? 8 : 200); d.b_kcontig = 1; d.b_ld = k; d.a_stride = d.a_ld * (d.a_kcontig ? m : k); }
    if (form == 5) { d.grouping = CLBH_GROUPS_BY_DEPTH; d.groups = 1 + Random(100); d.a_kcontig = d.b_kcontig = 0; d.a_ld = m; d.b_ld = n; }
    Check(d, units);
  }
  std::printf("cases %lld violations %lld\n", cases, violations);
  return violations == 0 ? 0 : 1;
}
