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

// Tiles (features x rows): number, extents, work-groups that share a compute unit
struct LayerTile {
  int variant, tile_m, tile_n, per_cu;
};
constexpr LayerTile kLayerTiles[] = {
    {0, 128, 128, 2}, {1, 256, 256, 1}, {2, 256, 128, 2}, {3, 64, 64, 4}, {4, 128, 32, 4},
};
constexpr int kLayerTileCount = sizeof(kLayerTiles) / sizeof(kLayerTiles[0]);

struct LayerPlan {
  LayerTile tile;
  long long tiles_m, tiles_n;  // tiles_n: for groups by rows the most there can be
  int splits, chunk;           // K ranges (1: none)
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

// Most tiles of `tile` rows that `groups` ranges within `rows` rows can be cut into: every group can add one that is not full
inline long long MostGroupTiles(const long long rows, const long long groups, const long long tile) {
  return std::min(rows, (rows + groups * (tile - 1)) / tile);
}

inline bool LayerTileExists(const int type, const LayerTile& tile) {
  return type != CLBH_TYPE_FP32 || tile.variant != 1;
}

// Rows per work-group of the elementwise kernel: as few as give about 2048 work-groups, at least 8 (two per wavefront), at
// most 128
inline int LayerRowsChunk(const long long rows, const long long column_blocks) {
  int chunk = 8;
  while (chunk < 128 && rows * column_blocks > 2048ll * chunk) { chunk *= 2; }
  return chunk;
}

inline int LayerVector(const int type) { return type == CLBH_TYPE_FP32 ? 4 : 8; }

inline LayerPlan PlanLayer(const clbh_layer_desc& d, const int units) {
  auto plan = LayerPlan{};
  plan.splits = 1;
  const auto take = [&](const size_t bytes) {  // a piece of the workspace
    const size_t offset = plan.workspace_bytes;
    plan.workspace_bytes += (bytes + 255) / 256 * 256;
    return offset;
  };
  if (d.upstream == nullptr) {
    const auto count = [&](const LayerTile& t) {
      const long long along_m = (d.m + t.tile_m - 1) / t.tile_m;
      const long long along_n = (d.grouping == CLBH_GROUPS_BY_ROWS) ? MostGroupTiles(d.n, d.groups, t.tile_n) : (d.n + t.tile_n - 1) / t.tile_n;
      return along_m * along_n * ((d.grouping == CLBH_GROUPS_BY_DEPTH) ? d.groups : 1);
    };
    int variant = 0;
    const long long rows_per_group = (d.grouping == CLBH_GROUPS_BY_ROWS) ? (d.n + d.groups - 1) / d.groups : d.n;
    if (rows_per_group <= 32) { variant = 4; }
    else if (count(kLayerTiles[0]) < 2ll * units) { variant = 3; }
    else { variant = (count(kLayerTiles[2]) >= 2ll * units) ? 2 : 0; }
    if (d.tile_variant >= 0 && d.tile_variant < kLayerTileCount && LayerTileExists(d.type, kLayerTiles[d.tile_variant])) { variant = d.tile_variant; }
    plan.tile = kLayerTiles[variant];
    plan.tiles_m = (d.m + plan.tile.tile_m - 1) / plan.tile.tile_m;
    plan.tiles_n = (d.grouping == CLBH_GROUPS_BY_ROWS) ? MostGroupTiles(d.n, d.groups, plan.tile.tile_n) : (d.n + plan.tile.tile_n - 1) / plan.tile.tile_n;
    int wanted = 1;
    const long long tiles = plan.tiles_m * plan.tiles_n, slots = static_cast<long long>(units) * plan.tile.per_cu;
    if (2 * tiles <= slots && d.k >= 512) { wanted = static_cast<int>(std::min<long long>({slots / tiles, d.k / 256, 16})); }
    if (d.split_k > 0) { wanted = d.split_k; }
    if (d.grouping == CLBH_GROUPS_NONE && wanted > 1) {
      const int chunk = static_cast<int>(((static_cast<long long>(d.k) + wanted - 1) / wanted + 63) / 64 * 64);
      const int splits = (d.k + chunk - 1) / chunk;
      if (splits > 1 && splits <= 65535) {
        plan.splits = splits;
        plan.chunk = chunk;
        take(sizeof(float) * static_cast<size_t>(splits) * static_cast<size_t>(d.n) * static_cast<size_t>(d.m));
      }
    }
  }
  const long long per_block = 64ll * ((d.upstream != nullptr) ? LayerVector(d.type) : 4), column_blocks = (d.m + per_block - 1) / per_block;
  plan.rows_chunk = LayerRowsChunk(d.n, column_blocks);
  plan.rows_chunks = (d.grouping == CLBH_GROUPS_BY_ROWS) ? MostGroupTiles(d.n, d.groups, plan.rows_chunk) : (d.n + plan.rows_chunk - 1) / plan.rows_chunk;
  if (d.bias_gradient != nullptr) {
    const long long rows_of_sums = (d.upstream != nullptr || plan.splits > 1) ? plan.rows_chunks : plan.tiles_n;
    plan.sums_offset = take(sizeof(float) * static_cast<size_t>(rows_of_sums) * static_cast<size_t>(d.m));
  }
  if (d.upstream == nullptr) {
    const size_t size = (d.type == CLBH_TYPE_FP32) ? 4 : 2;
    const bool by_rows = d.grouping == CLBH_GROUPS_BY_ROWS;
    if (!LayerOperandFits(d.a, d.a_ld, by_rows ? d.a_stride : 0, d.type)) {
      plan.a_copy_ld = ((d.a_kcontig ? d.k : d.m) + 7ll) / 8 * 8;
      plan.a_copy_offset = take(size * static_cast<size_t>(plan.a_copy_ld) * static_cast<size_t>(d.a_kcontig ? d.m : d.k) * static_cast<size_t>(by_rows ? d.groups : 1));
    }
    if (!LayerOperandFits(d.b, d.b_ld, 0, d.type)) {
      plan.b_copy_ld = ((d.b_kcontig ? d.k : d.n) + 7ll) / 8 * 8;
      plan.b_copy_offset = take(size * static_cast<size_t>(plan.b_copy_ld) * static_cast<size_t>(d.b_kcontig ? d.n : d.k));
    }
  }
  return plan;
}

}  // namespace clbh

#endif  // CLBLAST_HIP_DEVICE_LAYER_PLANS_HPP_
