// =================================================================================================
// Instances and launches of the layer products for one storage type (see clbh_layer_desc).
// =================================================================================================
#ifndef CLBLAST_HIP_DEVICE_LAUNCH_LAYER_HPP_
#define CLBLAST_HIP_DEVICE_LAUNCH_LAYER_HPP_

#include <hip/hip_runtime.h>

#include <climits>

#include "clbh_device.h"
#include "device/layer_plans.hpp"
#include "kernels/layer_gemm.hpp"
#include "kernels/layer_rows.hpp"

namespace clbh {

int LaunchLayerF16(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream);
int LaunchLayerBF16(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream);
int LaunchLayerF32(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream);

inline LayerArgs MakeLayerArgs(const clbh_layer_desc& d, const LayerPlan& plan) {
  LayerArgs p{};
  p.a = d.a;
  p.b = d.b;
  p.c = d.c;
  p.a_ld = d.a_ld;
  p.b_ld = d.b_ld;
  p.c_ld = d.c_ld;
  p.a_stride = d.a_stride;
  p.c_stride = d.c_stride;
  p.m = d.m;
  p.n = d.n;
  p.k = d.k;
  p.alpha = d.alpha;
  p.beta = d.beta;
  p.bias = d.bias;
  p.bias_stride = d.bias_stride;
  p.pre = d.pre;
  p.pre_ld = d.pre_ld;
  p.residual = d.residual;
  p.residual_ld = d.residual_ld;
  p.activation = d.activation;
  p.gradient = d.gradient;
  p.grouping = d.grouping;
  p.groups = d.groups;
  p.offsets = d.offsets;
  if (plan.splits > 1) {
    p.split_chunk = plan.chunk;
    p.partials = static_cast<float*>(d.workspace);
  }
  if (d.bias_gradient != nullptr) {
    p.bias_partials = reinterpret_cast<float*>(static_cast<char*>(d.workspace) + plan.sums_offset);
  }
  return p;
}

template <typename Config, bool A_KC, bool B_KC>
int LaunchLayerTile(const clbh_layer_desc& d, const LayerPlan& plan, const LayerArgs& args, hipStream_t stream) {
  if (Config::TILE_M != plan.tile.tile_m || Config::TILE_N != plan.tile.tile_n) { return hipErrorInvalidValue; }
  // (groups by depth: every XCD takes an eighth of each group's tiles)
  const long long blocks = (d.grouping == CLBH_GROUPS_BY_DEPTH) ? d.groups * ((plan.tiles_m * plan.tiles_n + 7) / 8 * 8) : plan.tiles_m * plan.tiles_n;
  if (blocks > INT_MAX) { return hipErrorInvalidConfiguration; }
  auto kernel = LayerGemmKernel<Config, A_KC, B_KC>;
  constexpr int lds_bytes = Config::LDS_BYTES;
  if (lds_bytes > 48 * 1024) {
    static const hipError_t attribute_status =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes);
    if (attribute_status != hipSuccess) { return static_cast<int>(attribute_status); }
  }
  return LayerSlices(blocks, Config::THREADS, [&](const int first, const unsigned count) {
    kernel<<<dim3(count, static_cast<unsigned>(plan.splits)), dim3(Config::THREADS), lds_bytes, stream>>>(
        args, static_cast<int>(plan.tiles_m), static_cast<int>(plan.tiles_n), first);
    return static_cast<int>(hipGetLastError());
  });
}

template <typename Config>
int LaunchLayerConfig(const clbh_layer_desc& d, const LayerPlan& plan, const LayerArgs& args, hipStream_t stream) {
  switch ((d.a_kcontig ? 2 : 0) | (d.b_kcontig ? 1 : 0)) {
    case 0: return LaunchLayerTile<Config, false, false>(d, plan, args, stream);
    case 1: return LaunchLayerTile<Config, false, true>(d, plan, args, stream);
    case 2: return LaunchLayerTile<Config, true, false>(d, plan, args, stream);
    default: return LaunchLayerTile<Config, true, true>(d, plan, args, stream);
  }
}

// Rings of LDS buffers: as deep as the work-groups that share a compute unit leave room for. 16 bits (512 x 4096 x 4096 on 128 x 128,
// 256 x 4096 x 4096 on 64 x 64, one work-group per compute unit): ring of three 45 and 32 us, four 36 and 23, five 36 and
// 21, six - one work-group less fits - 45 and 20. The fp32 walk is bound by its products: 254 and 81 us with any of them.
template <typename T>
int LaunchLayerProduct(const clbh_layer_desc& d, const LayerPlan& plan, const LayerArgs& args, hipStream_t stream) {
  constexpr bool HALF = sizeof(T) == 2;
  switch (plan.tile.variant) {
    case 1:
      if constexpr (HALF) { return LaunchLayerConfig<LayerConfig<T, 2, 4, 4, 2, 2>>(d, plan, args, stream); }
      else { return hipErrorInvalidValue; }
    case 2:
      if constexpr (HALF) { return LaunchLayerConfig<LayerConfig<T, 2, 2, 4, 2, 2>>(d, plan, args, stream); }
      else { return hipErrorInvalidValue; }
    case 3: return LaunchLayerConfig<LayerConfig<T, 2, 2, 1, 1, 4, HALF ? 5 : 3>>(d, plan, args, stream);
    case 4:
      if constexpr (!HALF) { return LaunchLayerConfig<LayerConfig<T, 4, 1, 1, 1, 4>>(d, plan, args, stream); }
      else { return hipErrorInvalidValue; }
    case 5: return LaunchLayerConfig<LayerConfig<T, 2, 2, 1, 1, 4, HALF ? 5 : 3, 2>>(d, plan, args, stream);
    default: return LaunchLayerConfig<LayerConfig<T, 2, 2, 2, 2, 2, HALF ? 4 : 3>>(d, plan, args, stream);
  }
}

template <typename T, int V, bool UPSTREAM>
int LaunchLayerRowsOf(const clbh_layer_desc& d, const LayerPlan& plan, const LayerArgs& args, hipStream_t stream) {
  LayerRowsArgs q{};
  q.layer = args;
  q.upstream = d.upstream;
  q.upstream_ld = d.upstream_ld;
  q.ranges = (d.upstream != nullptr) ? 1 : plan.splits;
  q.chunk = plan.rows_chunk;
  q.row_blocks = static_cast<int>(plan.rows_chunks);
  q.lane_shift = plan.rows_lane_shift;
  const long long column_blocks = (static_cast<long long>(d.m) + 64 * V - 1) / (64 * V);
  // (in one grid: a work-group has room for 32768 values at least, of which half exist, so that 2^32 threads would have 2^38)
  if (column_blocks * plan.rows_chunks >= (1ll << 32) / kLayerRowsThreads) { return hipErrorInvalidConfiguration; }
  q.column_blocks = static_cast<int>(column_blocks);
  const auto kernel = (plan.rows_lane_shift < 6) ? LayerRowsKernel<T, V, UPSTREAM, true> : LayerRowsKernel<T, V, UPSTREAM, false>;
  kernel<<<dim3(static_cast<unsigned>(column_blocks * plan.rows_chunks)), dim3(kLayerRowsThreads), 0, stream>>>(q);
  return static_cast<int>(hipGetLastError());
}

// Copies the operands that do not fit (LayerOperandFits) into the workspace, in one launch, and puts the copies in their place
template <typename T>
int AlignLayerOperands(const clbh_layer_desc& d, const LayerPlan& plan, LayerArgs& args, hipStream_t stream) {
  LayerAlignArgs q{};
  long long blocks[2] = {0, 0};
  const auto describe = [&](const int index, const void* from, const long long ld, const long long stride, const long long new_ld,
                            const size_t offset, const int length, const int lines, const int matrices) {
    auto& o = q.operand[index];
    o.from = from;
    o.to = static_cast<char*>(d.workspace) + offset;
    o.ld = ld;
    o.stride = stride;
    o.new_ld = new_ld;
    o.length = length;
    o.lines = lines;
    o.matrices = matrices;
    while (o.lane_shift < 6 && (16ll / static_cast<long long>(sizeof(T)) << o.lane_shift) < length) { ++o.lane_shift; }
    const long long lines_per_block = kLayerRowsThreads >> o.lane_shift;
    blocks[index] = (static_cast<long long>(lines) * matrices + lines_per_block - 1) / lines_per_block;
  };
  const bool by_rows = d.grouping == CLBH_GROUPS_BY_ROWS;
  if (plan.a_copy_ld > 0) {
    const int lines = d.a_kcontig ? d.m : d.k;
    describe(0, d.a, d.a_ld, by_rows ? d.a_stride : 0, plan.a_copy_ld, plan.a_copy_offset, d.a_kcontig ? d.k : d.m, lines,
             (by_rows && d.a_stride != 0) ? d.groups : 1);
    args.a = q.operand[0].to;
    args.a_ld = plan.a_copy_ld;
    args.a_stride = (d.a_stride != 0) ? plan.a_copy_ld * lines : 0;
  }
  if (plan.b_copy_ld > 0) {
    describe(1, d.b, d.b_ld, 0, plan.b_copy_ld, plan.b_copy_offset, d.b_kcontig ? d.k : d.n, d.b_kcontig ? d.n : d.k, 1);
    args.b = q.operand[1].to;
    args.b_ld = plan.b_copy_ld;
  }
  if (blocks[0] + blocks[1] == 0) { return 0; }
  if (blocks[0] + blocks[1] > INT_MAX) { return hipErrorInvalidConfiguration; }
  q.blocks_of_first = static_cast<int>(blocks[0]);
  return LayerSlices(blocks[0] + blocks[1], kLayerRowsThreads, [&](const int first, const unsigned count) {
    LayerAlignKernel<T><<<dim3(count), dim3(kLayerRowsThreads), 0, stream>>>(q, first);
    return static_cast<int>(hipGetLastError());
  });
}

template <typename T>
int LaunchLayerTyped(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream) {
  auto args = MakeLayerArgs(d, plan);
  const bool elementwise = d.upstream != nullptr || plan.splits > 1;
  if (d.upstream == nullptr) {
    int status = AlignLayerOperands<T>(d, plan, args, stream);
    if (status == 0) { status = LaunchLayerProduct<T>(d, plan, args, stream); }
    if (status != 0) { return status; }
  }
  if (elementwise) {
    // (of the fp32 sums of K ranges a lane takes four, 16 bytes)
    const int status = (d.upstream != nullptr) ? LaunchLayerRowsOf<T, 16 / sizeof(T), true>(d, plan, args, stream) : LaunchLayerRowsOf<T, 4, false>(d, plan, args, stream);
    if (status != 0) { return status; }
  }
  if (d.bias_gradient != nullptr) {
    const long long rows_of_sums = elementwise ? plan.rows_chunks : plan.tiles_n;
    const bool grouped = d.grouping == CLBH_GROUPS_BY_ROWS;
    const int groups = grouped ? d.groups : 1;
    const bool many = rows_of_sums >= 64ll * groups;  // sums per group
    const auto kernel = many ? LayerColumnSumsKernel<T, 16> : LayerColumnSumsKernel<T, 4>;
    const int threads = many ? 1024 : 256;
    return LayerSlices((static_cast<long long>(d.m) + 63) / 64, threads, [&](const int first, const unsigned count) {
      kernel<<<dim3(count, static_cast<unsigned>(groups < 65535 ? groups : 65535)), dim3(threads), 0, stream>>>(
          args.bias_partials, static_cast<int>(rows_of_sums), d.m, grouped ? d.offsets : nullptr, groups, d.n,
          elementwise ? plan.rows_chunk : plan.tile.tile_n, static_cast<T*>(d.bias_gradient), static_cast<long long>(d.m), first);
      return static_cast<int>(hipGetLastError());
    });
  }
  return 0;
}

}  // namespace clbh

#endif  // CLBLAST_HIP_DEVICE_LAUNCH_LAYER_HPP_
