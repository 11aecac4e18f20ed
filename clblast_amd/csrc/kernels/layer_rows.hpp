// =================================================================================================
// The elementwise work of a layer without a product of its own, and column sums:
//   * LayerRowsKernel: the epilogue of kernels/layer_gemm.hpp on sums that are already there - the fp32 sums of a product
//     whose K range was split over several work-groups (added up here in the order of the ranges), or, for the gradient of
//     an activation, a matrix of the caller's. One pass over memory; bound by it: GELU's gradient of 8192 x 8192 bf16 in
//     72 us, 5.6 TB/s, the rate of a large copy; with the bias's gradient, whose sums take a second launch, 78 (with one row in flight per wavefront 94, with four 231 - the compiler then spills -
//     with the matrices kept in the caches 87, with one register more than the 64 that eight wavefronts per SIMD leave 88).
//   * LayerAlignKernel: copies of operands whose lines do not start at dwords, for the tiled kernel's loads.
//   * LayerColumnSumsKernel: the second half of a bias gradient, which adds up the sums that the work-groups of either
//     kernel left for their tiles of rows, in the order of the tiles: the result does not depend on timing.
// =================================================================================================
#ifndef CLBLAST_HIP_KERNELS_LAYER_ROWS_HPP_
#define CLBLAST_HIP_KERNELS_LAYER_ROWS_HPP_

#include "kernels/layer_gemm.hpp"

namespace clbh {

constexpr int kLayerRowsThreads = 256;

struct LayerRowsArgs {
  LayerArgs layer;       // c (nullptr: only the column sums are wanted), pre, residual, bias, alpha, beta, groups, ...
  const void* upstream;  // of the storage type, or nullptr: the fp32 sums at layer.partials
  long long upstream_ld;
  int ranges;            // K ranges at layer.partials
  int chunk;             // rows per work-group
  int row_blocks;        // work-groups along the rows where there are no groups
  int lane_shift;        // 2^lane_shift lanes per row, a wavefront takes 64 >> lane_shift rows side by side
  int column_blocks;     // work-groups side by side; the grid's only dimension counts them first
};

// Work-group: 64 pieces of V features (lanes; fewer of a narrow matrix, several rows side by side then) times `chunk` rows; the work-groups
// of a group (of the matrix) take its rows in turn, so that what is in flight at a time lies together (8192 x 8192 75 -> 72 us,
// 8192 x 11008 115 -> 107; with its bias gradient 119 -> 111). bias_partials: one row of m sums for every work-group, numbered through
// the groups. UPSTREAM: the caller's matrix takes the place of the sums. NARROW: a row is the work of less than 64 lanes (65536 x 64 with all lanes on one row: 28 us, 9 like this;
// 8192 x 8192 with row numbers in vector registers: 87 us, 74 with scalar ones).
template <typename T, int V, bool UPSTREAM, bool NARROW>
__global__ __launch_bounds__(kLayerRowsThreads, UPSTREAM ? 8 : 4) void LayerRowsKernel(const LayerRowsArgs q) {
  constexpr bool FAST = sizeof(T) == 2;
  constexpr int WAVES = kLayerRowsThreads / 64, FLIGHT = UPSTREAM ? 2 : 1;  // rows of a wavefront in flight together
  constexpr int RANGES = 8;                                                // K ranges in flight together
  const LayerArgs& p = q.layer;
  __shared__ float wave_sums[WAVES][64 * V];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int column_block = blockIdx.x % q.column_blocks;
  const int lane_shift = NARROW ? q.lane_shift : 6;
  const int lanes = 1 << lane_shift, beside = 64 >> lane_shift;  // (less than 64 lanes: one column block)
  const int col = (column_block * 64 + (lane & (lanes - 1))) * V;
  const int inside = p.m - col;  // features from this lane's first one on

  const int sums_row = blockIdx.x / q.column_blocks;
  constexpr unsigned PASS = WAVES * FLIGHT;  // (times `beside`: the rows that a work-group takes together)
  unsigned first, end, stride = PASS * beside;
  if (p.grouping == kLayerGroupedRows) {
    int group = 0, before = 0, begin = 0, last = 0;
    if (!FindGroupTile(p.offsets, p.groups, p.n, q.chunk, lane, [&](int) { return sums_row; }, group, before, begin, last)) { return; }
    first = begin + (sums_row - before) * stride;
    end = last;
    stride *= (last - begin + q.chunk - 1) / q.chunk;
  } else {
    first = sums_row * stride;
    end = p.n;
    stride *= q.row_blocks;  // (at most the rows and a chunk: what is added up stays below 2^32)
  }

  float bias[V], sums[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sums[e] = 0.0f;
    bias[e] = (!UPSTREAM && p.bias != nullptr && e < inside) ? static_cast<float>(static_cast<const T*>(p.bias)[col + e]) : 0.0f;
  }
  const T* other = p.gradient ? static_cast<const T*>(p.pre) : ((p.beta != 0.0f) ? static_cast<const T*>(p.residual) : nullptr);
  const long long other_ld = p.gradient ? p.pre_ld : p.residual_ld;

  if (inside > 0) {
    for (unsigned row0 = first + wave * beside + (NARROW ? lane >> lane_shift : 0); row0 < end; row0 += stride) {
      // (as they are in memory until their row's turn: half the registers of their values for 16 bits)
      typename LayerPiece<T, V>::Raw upstream[FLIGHT], old[FLIGHT];
      float z[V];
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) {
        const long long row = min(row0 + WAVES * beside * u, end - 1);  // (a row beyond the end: the last one again, not used)
#pragma unroll
        for (int e = 0; e < V; ++e) { old[u][e] = T(0.0f); }
        if constexpr (UPSTREAM) { upstream[u] = LayerPiece<T, V>::template LoadRaw<true>(static_cast<const T*>(q.upstream) + row * q.upstream_ld + col, inside); }
        if (other != nullptr) { old[u] = LayerPiece<T, V>::template LoadRaw<UPSTREAM>(other + row * other_ld + col, inside); }
      }
      if constexpr (!UPSTREAM) {
#pragma unroll
        for (int e = 0; e < V; ++e) { z[e] = 0.0f; }
        const float* from = p.partials + static_cast<long long>(row0) * p.m + col;
        const long long slab = static_cast<long long>(p.n) * p.m;
        for (int range = 0; range < q.ranges; range += RANGES) {
          float more[RANGES][V];
#pragma unroll
          for (int r = 0; r < RANGES; ++r) {
#pragma unroll
            for (int e = 0; e < V; ++e) { more[r][e] = 0.0f; }
            if (range + r < q.ranges) { LayerPiece<float, V>::Load(from + (range + r) * slab, inside, more[r]); }
          }
#pragma unroll
          for (int r = 0; r < RANGES; ++r) {
#pragma unroll
            for (int e = 0; e < V; ++e) { z[e] += more[r][e]; }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) {
        const long long row = row0 + WAVES * beside * u;
        if (row < end) {
          float now[V], y[V];
          LayerPiece<T, V>::Values(old[u], now);
          if constexpr (UPSTREAM) { LayerPiece<T, V>::Values(upstream[u], z); }
          if constexpr (!UPSTREAM) {
#pragma unroll
            for (int e = 0; e < V; ++e) { z[e] = __builtin_fmaf(p.alpha, z[e], bias[e]); }
          }
          LayerValues<FAST, true>(p, z, now, y);
#pragma unroll
          for (int e = 0; e < V; ++e) { sums[e] += y[e]; }
          if (p.c != nullptr) { LayerPiece<T, V>::Store(static_cast<T*>(p.c) + row * p.c_ld + col, inside, y); }
          if (!UPSTREAM && p.pre != nullptr && !p.gradient) { LayerPiece<T, V>::Store(static_cast<T*>(p.pre) + row * p.pre_ld + col, inside, z); }
        }
      }
    }
  }
  if (p.bias_partials != nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      for (int step = lanes; NARROW && step < 64; step *= 2) { sums[e] += __shfl_xor(sums[e], step, 64); }  // (rows side by side)
      if (lane < lanes) { wave_sums[wave][lane * V + e] = sums[e]; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < lanes * V; i += kLayerRowsThreads) {
      const int feature = column_block * 64 * V + i;
      if (feature < p.m) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) { sum += wave_sums[w][i]; }
        p.bias_partials[static_cast<long long>(sums_row) * p.m + feature] = sum;
      }
    }
  }
}

// One operand to copy: `matrices` matrices of `lines` lines of `length` elements, ld and stride apart, to lines of new_ld
// elements, one matrix behind the other. lane_shift: a line takes 2^lane_shift lanes, a piece of 16 bytes each and in turn.
struct LayerAlignOperand {
  const void* from;
  void* to;
  long long ld, stride, new_ld;
  int length, lines, matrices, lane_shift;
};
struct LayerAlignArgs {
  LayerAlignOperand operand[2];
  int blocks_of_first;  // the work-groups from this one on copy the second operand
};
template <typename T>
__global__ __launch_bounds__(kLayerRowsThreads) void LayerAlignKernel(const LayerAlignArgs q, const int first_block) {
  constexpr int V = 16 / sizeof(T);
  typedef T Loose __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  typedef T Tight __attribute__((ext_vector_type(V)));
  const int grid_block = first_block + static_cast<int>(blockIdx.x);  // (first_block: of this slice of the grid)
  const bool second = grid_block >= q.blocks_of_first;
  const LayerAlignOperand& o = q.operand[second ? 1 : 0];
  const long long block = second ? grid_block - q.blocks_of_first : grid_block;
  const long long line = ((block * kLayerRowsThreads + threadIdx.x) >> o.lane_shift);
  if (line >= static_cast<long long>(o.lines) * o.matrices) { return; }
  const int matrix = static_cast<int>(line / o.lines), in_matrix = static_cast<int>(line - static_cast<long long>(matrix) * o.lines);
  const T* from = static_cast<const T*>(o.from) + matrix * o.stride + in_matrix * o.ld;
  T* to = static_cast<T*>(o.to) + line * o.new_ld;
  const int lanes = 1 << o.lane_shift;
  for (int at = (threadIdx.x & (lanes - 1)) * V; at < o.length; at += lanes * V) {
    Tight piece;
    if (at + V <= o.length) { piece = __builtin_bit_cast(Tight, *reinterpret_cast<const Loose*>(from + at)); }
    else {
#pragma unroll
      for (int e = 0; e < V; ++e) { piece[e] = (at + e < o.length) ? from[at + e] : T(0.0f); }
    }
    *reinterpret_cast<Tight*>(to + at) = piece;
  }
}

// out[group * out_stride + i] = the sum of the group's rows of `partials` (m values each): with offsets the tiles of `tile`
// rows that the groups are cut into, numbered through from group 0 on; without, all `rows_of_sums` rows. Zero for a
// group without a tile. grid: (ceil(m / 64), from `first_block` on, groups); each of the WAVES wavefronts takes every WAVES-th row.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void LayerColumnSumsKernel(const float* __restrict__ partials, const int rows_of_sums,
                                                                           const int m, const long long* __restrict__ offsets,
                                                                           const int groups, const int rows, const int tile,
                                                                           T* __restrict__ out, const long long out_stride,
                                                                           const int first_block) {
  __shared__ float wave_sums[WAVES][64];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  for (int group = blockIdx.y; group < groups; group += gridDim.y) {
    int first = 0, count = rows_of_sums;
    if (offsets != nullptr) {  // tiles of the groups in front of this one, and of this one
      int before = 0;
      for (int g = lane; g < group; g += 64) {
        const long long from = offsets[g], to = offsets[g + 1];
        const int begin = static_cast<int>(from < 0 ? 0 : (from > rows ? rows : from));
        const int size = static_cast<int>(to < begin ? 0 : (to > rows ? rows : to) - begin);
        before = min(before + (size + tile - 1) / tile, rows_of_sums);  // (groups that overlap can have any number of tiles)
      }
#pragma unroll
      for (int step = 32; step >= 1; step /= 2) { before += __shfl_xor(before, step, 64); }
      int begin, end;
      GroupRange(offsets, group, rows, begin, end);
      first = min(before, rows_of_sums);
      count = min((end - begin + tile - 1) / tile, rows_of_sums - first);
    }
    const int feature = (first_block + static_cast<int>(blockIdx.x)) * 64 + lane;
    float sum = 0.0f;
    if (feature < m) {
      const float* from = partials + static_cast<long long>(first) * m + feature;
#pragma unroll 8
      for (int t = wave; t < count; t += WAVES) { sum += from[static_cast<long long>(t) * m]; }
    }
    wave_sums[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && feature < m) {
#pragma unroll
      for (int w = 1; w < WAVES; ++w) { sum += wave_sums[w][lane]; }
      out[group * out_stride + feature] = static_cast<T>(sum);
    }
    __syncthreads();
  }
}

}  // namespace clbh

#endif  // CLBLAST_HIP_KERNELS_LAYER_ROWS_HPP_
