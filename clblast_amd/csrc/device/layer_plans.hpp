// =================================================================================================
// Launch geometry of the layer products (kernels/layer_gemm.hpp, kernels/layer_rows.hpp): which tile, how many K ranges,
// how much workspace. Depends on nothing but the descriptor and the number of compute units and is free of HIP, so that a
// host-only test can sweep it (tests/host/layer_plan_sweep.cpp).
// =================================================================================================
#ifndef CLBLAST_HIP_DEVICE_LAYER_PLANS_HPP_
#define CLBLAST_HIP_DEVICE_LAYER_PLANS_HPP_

#include <algorithm>
#include <climits>
#include <cstddef>

#include "clbh_device.h"

namespace clbh {

// Tiles (features x rows), and what a work-group of one costs: ns per unit of k while it has a compute unit to itself
// (`alone`), its share when the compute unit is full of them (`full`), and the us that its start and epilogue keep
// the compute unit from other work (`fixed`). Fitted on an MI355X to forced tiles at 256 .. 8192 x 4096 x 4096 and 8192^2 x 1024; a
// tile that is alone on half of the compute units runs faster than one on all of them (the 16-bit products run against the
// power limit), which the smallest tiles' k-walk, bound by latency, does not show. The last one is the 64 x 64 tile whose depth two
// sets of wavefronts share. On 40 random shapes the choice is 1.2 % behind the best of all forced ones, 17 % at worst.
struct LayerTile {
  int variant, tile_m, tile_n, per_cu;
  double alone_16, full_16, fixed_16, alone_32, full_32, fixed_32;
};
constexpr LayerTile kLayerTiles[] = {
    {0, 128, 128, 2, 7.3, 9.3, 0.4, 61.6, 58.0, 2.0}, {1, 256, 256, 1, 17.0, 25.4, 4.5, 0.0, 0.0, 0.0},
    {2, 256, 128, 2, 15.0, 15.2, 1.5, 0.0, 0.0, 0.0}, {3, 64, 64, 4, 4.1, 3.7, 0.2, 16.8, 14.6, 0.3},
    {4, 128, 32, 4, 0.0, 0.0, 0.0, 18.5, 16.0, 0.3},
    {5, 64, 64, 2, 3.6, 4.0, 0.3, 15.8, 14.6, 0.5},
};
constexpr int kLayerTileCount = sizeof(kLayerTiles) / sizeof(kLayerTiles[0]);

struct LayerPlan {
  LayerTile tile;
  long long tiles_m, tiles_n;  // tiles_n: for groups by rows the most there can be
  int splits, chunk;           // K ranges (1: none)
  int rows_lane_shift;         // elementwise kernel: 2^ of it lanes per row
  int rows_chunk;              // rows per work-group of the elementwise kernel
  long long rows_chunks;       // work-groups of it along the rows (the most there can be)
  // operands that the kernel cannot fetch as they are and that are copied first (0: not), with the copy's leading dimension
  long long a_copy_ld, b_copy_ld;
  // the workspace: sums of K ranges, sums for the bias gradient, copies of a and b
  size_t sums_offset, a_copy_offset, b_copy_offset, workspace_bytes;
};

// 16-bit operands are fetched in dwords: their lines (and the groups' matrices) have to start at dwords. The lines of a slab
// are reached by 32-bit byte offsets.
inline bool LayerOperandFits(const void* pointer, const long long ld, const long long stride, const int type) {
  if (ld >= CLBH_LAYER_MAX_LD) { return false; }
  return type == CLBH_TYPE_FP32 || (reinterpret_cast<unsigned long long>(pointer) % 4 == 0 && ld % 2 == 0 && stride % 2 == 0);
}

// The leading dimension of an operand's copy
inline long long LayerCopyLd(const long long length) { return (length + 7) / 8 * 8; }

// A slab's pieces reach their lines - sixteen rows or features of a k-contiguous operand, up to eight depths of another - by
// unsigned 32-bit byte offsets. Where these do not suffice for a copy without padding either, there is no launch for the operand. Rows
// and features that do not exist may wrap: what they fetch lies inside the operand and is not stored. Depths may not, they have
// to read as zero.
inline bool LayerLinesReachable(const bool k_contiguous, const long long lines, const long long ld, const int type) {
  const long long last = (k_contiguous ? std::min(lines, 16ll) : 8) - 1, size = (type == CLBH_TYPE_FP32) ? 4 : 2;
  return last * ld * size + 512 <= 1ll << 32;
}
inline bool LayerOperandsReachable(const clbh_layer_desc& d) {
  if (d.upstream != nullptr) { return true; }
  const auto reachable = [&](const int k_contiguous, const long long across) {
    const long long length = k_contiguous ? d.k : across, lines = k_contiguous ? across : d.k;
    return LayerLinesReachable(k_contiguous != 0, lines, LayerCopyLd(length), d.type);
  };
  return reachable(d.a_kcontig, d.m) && reachable(d.b_kcontig, d.n);
}

// Most tiles of `tile` rows that `groups` ranges within `rows` rows can be cut into: every group can add one that is not full
inline long long MostGroupTiles(const long long rows, const long long groups, const long long tile) {
  return std::min(rows, (rows + groups * (tile - 1)) / tile);
}

inline bool LayerTileExists(const int type, const LayerTile& tile) {
  return (type == CLBH_TYPE_FP32) ? tile.full_32 > 0.0 : tile.full_16 > 0.0;
}

// Rows per work-group of the elementwise kernel: as few as give about 2048 work-groups, at least 8 (two per wavefront), at
// most 128, times the rows that a wavefront takes side by side
inline int LayerRowsChunk(const long long rows, const long long column_blocks, const int lane_shift) {
  int chunk = 8 * (64 >> lane_shift);
  const int most = 16 * chunk;
  while (chunk < most && rows * column_blocks > 2048ll * chunk) { chunk *= 2; }
  return chunk;
}
// A row of a narrow matrix is the work of 2^shift lanes, a wavefront takes 64 of them side by side
inline int LayerRowsLaneShift(const long long features, const int vector) {
  int shift = 0;
  while (shift < 6 && (static_cast<long long>(vector) << shift) < features) { ++shift; }
  return shift;
}

inline int LayerVector(const int type) { return type == CLBH_TYPE_FP32 ? 4 : 8; }

// Estimated time in us of so many work-groups of a tile that each walk k: rounds of as many as stay resident, the last one with
// what is left; no round is over before its first loads and its stores have had their latencies. (bf16: 256 x 4096 x 4096 on
// 64 x 64 22 estimated, 21 measured; 8192 x 8192 x 1024 on 256 x 256 125 and 121; 1024 x 4096 x 4096 on 128 x 128 35 and 40.)
inline double LayerCost(const LayerTile& t, const bool wide, const double work_groups, const double k, const int units) {
  const double alone = (wide ? t.alone_32 : t.alone_16) * k * 1e-3, full = (wide ? t.full_32 : t.full_16) * k * 1e-3;
  const double fixed = wide ? t.fixed_32 : t.fixed_16, latency = 2.5;
  const double slots = static_cast<double>(units) * t.per_cu;
  const double rounds = static_cast<double>(static_cast<long long>(work_groups / slots));
  double cost = 2.5 + rounds * std::max(t.per_cu * (full + fixed), alone + latency);
  const double left = (work_groups - rounds * slots) / units;  // work-groups per compute unit in the last round
  if (left > 0.0) {
    const double together = static_cast<double>(static_cast<long long>(left + 0.999));
    cost += std::max((t.per_cu == 1 ? left : together) * full + together * fixed, alone + latency);
  }
  return cost;
}

// Tile and K ranges by that estimate; ranges pay for the sums' way through memory and the second kernel. Measured with two
// kernels against one: 64 x 1024 x 1024 10.9 / 13.2 us, 64 x 4096 x 4096 33 / 17, 1 x 8192 x 4096 33 / 15.4.
inline void ChooseLayerTile(const clbh_layer_desc& d, const int units, int& variant, int& ranges) {
  const bool wide = d.type == CLBH_TYPE_FP32;
  const bool by_rows = d.grouping == CLBH_GROUPS_BY_ROWS, by_depth = d.grouping == CLBH_GROUPS_BY_DEPTH;
  double best = 0.0;
  for (const auto& t : kLayerTiles) {
    if (!LayerTileExists(d.type, t)) { continue; }
    const double along_m = static_cast<double>((d.m + t.tile_m - 1) / t.tile_m);
    // (of groups the host knows the number alone: even ones are assumed)
    const double rows = by_rows ? static_cast<double>((d.n + d.groups - 1) / d.groups) : static_cast<double>(d.n);
    const double along_n = static_cast<double>(static_cast<long long>((rows + t.tile_n - 1) / t.tile_n)) * (by_rows ? std::min(d.groups, d.n) : 1);
    // (of groups by depth every XCD has an eighth of each group's tiles)
    const double tiles = along_m * along_n;
    const double groups = by_depth ? static_cast<double>(static_cast<long long>((tiles + 7.0) / 8.0)) * 8.0 * d.groups : tiles;
    const double k = by_depth ? std::max(1.0, static_cast<double>(d.k) / d.groups) : static_cast<double>(d.k);
    for (int s = 1; s <= 32; s = (s < 4) ? s + 1 : s + s / 2) {
      if (s > 1 && (d.grouping != CLBH_GROUPS_NONE || d.k < 256 * s)) { break; }
      const double sums = static_cast<double>(s) * d.m * d.n;
      if (s > 1 && sums * 4.0 > 64e6) { break; }
      const double cost = LayerCost(t, wide, groups * s, k / s, units) + ((s > 1) ? 5.0 + sums * 8.0 / 4e6 : 0.0);
      if (best == 0.0 || cost < best) { best = cost; variant = t.variant; ranges = s; }
    }
  }
}

// A grid dimension takes less than 2^32 threads. A longer one - 2^30 rows of one feature, in tiles of 64 - goes out in slices of
// 2^31 threads (a multiple of eight work-groups, so that these still meet the XCDs in turn): launch(first work-group, how many)
// is called for each and returns 0, or an error that ends it.
template <typename Launch>
int LayerSlices(const long long blocks, const int threads, Launch&& launch) {
  const long long most = (1ll << 31) / threads;
  for (long long first = 0; first < blocks; first += most) {
    const int status = launch(static_cast<int>(first), static_cast<unsigned>(std::min(most, blocks - first)));
    if (status != 0) { return status; }
  }
  return 0;
}

inline LayerPlan PlanLayer(const clbh_layer_desc& d, const int units) {
  auto plan = LayerPlan{};
  plan.splits = 1;
  const auto take = [&](const size_t bytes) {  // a piece of the workspace
    const size_t offset = plan.workspace_bytes;
    plan.workspace_bytes += (bytes + 255) / 256 * 256;
    return offset;
  };
  if (d.upstream == nullptr) {
    int variant = 0, wanted = 1;
    ChooseLayerTile(d, units, variant, wanted);
    if (d.tile_variant >= 0 && d.tile_variant < kLayerTileCount && LayerTileExists(d.type, kLayerTiles[d.tile_variant])) { variant = d.tile_variant; }
    plan.tile = kLayerTiles[variant];
    plan.tiles_m = (d.m + plan.tile.tile_m - 1) / plan.tile.tile_m;
    plan.tiles_n = (d.grouping == CLBH_GROUPS_BY_ROWS) ? MostGroupTiles(d.n, d.groups, plan.tile.tile_n) : (d.n + plan.tile.tile_n - 1) / plan.tile.tile_n;
    if (variant == d.tile_variant && d.split_k == 0) { wanted = 1; }  // a tile that is forced alone
    if (d.split_k > 0) { wanted = d.split_k; }
    if (d.grouping == CLBH_GROUPS_NONE && wanted > 1) {
      const int chunk = static_cast<int>(((static_cast<long long>(d.k) + wanted - 1) / wanted + 63) / 64 * 64);
      const int splits = static_cast<int>((static_cast<long long>(d.k) + chunk - 1) / chunk);
      if (splits > 1 && splits <= 65535) {
        plan.splits = splits;
        plan.chunk = chunk;
        take(sizeof(float) * static_cast<size_t>(splits) * static_cast<size_t>(d.n) * static_cast<size_t>(d.m));
      }
    }
  }
  const int vector = (d.upstream != nullptr) ? LayerVector(d.type) : 4;
  const long long per_block = 64ll * vector, column_blocks = (d.m + per_block - 1) / per_block;
  plan.rows_lane_shift = LayerRowsLaneShift(d.m, vector);
  plan.rows_chunk = LayerRowsChunk(d.n, column_blocks, plan.rows_lane_shift);
  plan.rows_chunks = (d.grouping == CLBH_GROUPS_BY_ROWS) ? MostGroupTiles(d.n, d.groups, plan.rows_chunk) : (static_cast<long long>(d.n) + plan.rows_chunk - 1) / plan.rows_chunk;
  if (d.bias_gradient != nullptr) {
    const long long rows_of_sums = (d.upstream != nullptr || plan.splits > 1) ? plan.rows_chunks : plan.tiles_n;
    plan.sums_offset = take(sizeof(float) * static_cast<size_t>(rows_of_sums) * static_cast<size_t>(d.m));
  }
  if (d.upstream == nullptr) {
    const size_t size = (d.type == CLBH_TYPE_FP32) ? 4 : 2;
    const bool by_rows = d.grouping == CLBH_GROUPS_BY_ROWS;
    if (!LayerOperandFits(d.a, d.a_ld, by_rows ? d.a_stride : 0, d.type)) {
      plan.a_copy_ld = LayerCopyLd(d.a_kcontig ? d.k : d.m);
      plan.a_copy_offset = take(size * static_cast<size_t>(plan.a_copy_ld) * static_cast<size_t>(d.a_kcontig ? d.m : d.k) * static_cast<size_t>((by_rows && d.a_stride != 0) ? d.groups : 1));
    }
    if (!LayerOperandFits(d.b, d.b_ld, 0, d.type)) {
      plan.b_copy_ld = LayerCopyLd(d.b_kcontig ? d.k : d.n);
      plan.b_copy_offset = take(size * static_cast<size_t>(plan.b_copy_ld) * static_cast<size_t>(d.b_kcontig ? d.n : d.k));
    }
  }
  return plan;
}

}  // namespace clbh

#endif  // CLBLAST_HIP_DEVICE_LAYER_PLANS_HPP_
