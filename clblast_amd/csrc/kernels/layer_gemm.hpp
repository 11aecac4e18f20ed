// =================================================================================================
// Products of a network's layers for gfx950: fp32, fp16 and bf16, sums in fp32, with the layer's elementwise work in the
// epilogue and, where the rows belong to groups (experts), every group multiplied by its own matrix in the same launch.
//
// Canonical problem (the caller's row-major matrices read as column-major ones): C(i, j) for i < m features - contiguous in
// C - and j < n rows,
//   S(i, j) = sum_p A(i, p) B(p, j)         A: the weights, B: the rows the layer is applied to
//   forward:   Z = alpha S + bias(i)        C = act(Z) + beta R(i, j)        (Z stored too where `pre` is set)
//   gradient:  C = alpha S act'(Z(i, j))    Z read from `pre`; sums of C over the tile's rows go to `bias_partials`
// Groups by rows:  group g owns the rows offsets[g] .. offsets[g + 1] - 1 of B, C and pre, and has its own A and bias.
// Groups by depth: group g owns that range of p in A and B, and has its own C: the gradients of the groups' weights.
// The offsets lie in device memory; they are clamped to the rows that exist, so no offset leads outside a matrix.
//
// Structure: a work-group owns a TILE_M x TILE_N tile, K is walked in slabs of 64 bytes per line (32 halfs, 16 floats) in a
// ring of three to five LDS buffers. Both types share the byte layout of a slab, the direct global -> LDS requests (16 bytes per lane, range-checked
// by the buffer resource), the one barrier per slab and the order of products: the wavefront's blocks form four quadrants
// whose missing fragments are read under the products of the quadrant before. What differs is the instruction: 16 bits
// v_mfma_f32_16x16x32_{f16,bf16}, a slab is one instruction deep, and x-contiguous operands are read with the transposing LDS
// read; fp32 v_mfma_f32_32x32x2_f32 (16x16x4 on the smallest tile), where lane half h feeds the depths 4h + s and
// 8 + 4h + s (s = 0..3) in both operands, so that a k-contiguous operand is read in 16-byte pieces and an
// x-contiguous one value by value, neither of them transposed.
//
// Epilogue: half of its rows at a time, a wavefront writes its sums to LDS in fp32 as [row][feature] and reads them back with
// consecutive lanes along the features, so that bias, residual, Z and C all move in 16-byte pieces of whole lines, and a
// lane keeps the same features for the whole tile (its bias values and its part of the bias gradient stay in registers).
// Only the final value is rounded.
//
// What bounds it (bf16 and fp32, with the host's time per call where that is part of it): 8192 x 8192 x 4096 with bias, GELU and
// stored Z 471 us, 1.17 PFLOP/s of the 1.29 that a large library product reaches here - the matrix pipe, and 4 us per
// round of tiles for an epilogue under which nothing multiplies (a persistent form that loads the next tile under it held
// both tiles' registers and was slower, 482 us). fp32 1024 x 1024 x 4096 74 us, 116 of 154 TFLOP/s: the matrix pipe is busy for 76 %
// of the cycles, the rest is a barrier per slab of 64 products of a block. Products of few rows: the weights' way from
// memory, 128 rows over 64 experts of 2048 x 1024 in bf16 41 us for the 205 MB of the experts that have rows. Small ones: the latency of a slab, about 0.15 us, times their number.
//
// Teams: few tiles of a long depth leave one work-group to a compute unit, whose four wavefronts wait for each slab. Two sets of
// wavefronts with half the depth each, in one work-group, halve the number of slabs without a second kernel: 512 x 512 x 4096
// in bf16 20.8 -> 18.9 us, 300 x 1000 x 512 in fp32 16.2 -> 14.1, 777 x 1001 x 1024 25.7 -> 22.3. With four tiles of 64 x 64
// per compute unit the single set is ahead: 1024 x 4096 x 1024 in bf16 19.8 against 21.6.
// =================================================================================================
#ifndef CLBLAST_HIP_KERNELS_LAYER_GEMM_HPP_
#define CLBLAST_HIP_KERNELS_LAYER_GEMM_HPP_

#include <type_traits>

#include "kernels/activations.hpp"
#include "kernels/gemm_direct_f16.hpp"
#include "kernels/gemm_mfma.hpp"
#include "kernels/layer_requests.hpp"

namespace clbh {

constexpr int kLayerPlain = 0, kLayerGroupedRows = 1, kLayerGroupedDepth = 2;

struct LayerArgs {
  const void* a;
  const void* b;
  void* c;
  long long a_ld, b_ld, c_ld;
  long long a_stride, c_stride;  // from one group's A (groups by rows) or C (groups by depth) to the next one's
  int m, n, k;                   // n: all rows there are; k: the depth, for groups by depth all of it
  float alpha, beta;
  const void* bias;  // or nullptr
  long long bias_stride;
  void* pre;  // Z: written (forward, or nullptr), read (gradient)
  long long pre_ld;
  const void* residual;  // not read when beta == 0
  long long residual_ld;
  int activation;
  int gradient;
  int grouping;  // kLayerPlain, ...
  int groups;
  const long long* offsets;  // groups + 1 values
  float* bias_partials;      // [tile of rows][m], or nullptr
  // K ranges of one plain product: range s goes to partials + s * n * m as fp32 sums, a second kernel finishes
  int split_chunk;
  float* partials;
};

// ---- group lookup ------------------------------------------------------------------------------------------------------

// The rows of group g, inside 0 .. rows whatever the offsets say
__device__ __forceinline__ void GroupRange(const long long* offsets, const int g, const int rows, int& begin, int& end) {
  const long long first = UniformRead(offsets + g), last = UniformRead(offsets + g + 1);
  begin = static_cast<int>(first < 0 ? 0 : (first > rows ? rows : first));
  end = static_cast<int>(last < begin ? begin : (last > rows ? rows : last));
}

// No group of a valid call has more tiles than this: grouped calls have less than 2^26 rows, a tile has at least 8. Offsets
// that are out of order can make the groups overlap; the numbers of tiles still fit 32 bits then.
constexpr int kLayerMostGroupTiles = 1 << 23;

// Every group's rows are cut into tiles of `tile` rows, numbered through from group 0 on. Sums up all tiles and finds the
// group that owns tile `wanted` (a function of that sum): 64 groups at a time, one per lane, and a scan over the lanes.
// wanted_of(total) returns the tile's number, or a negative one where this work-group has none. Uniform results;
// returns false without a tile. `before`: tiles of the groups in front of the one found.
template <typename Wanted>
__device__ __forceinline__ bool FindGroupTile(const long long* __restrict__ offsets, const int groups, const int rows,
                                              const int tile, const int lane, Wanted wanted_of, int& group, int& before,
                                              int& begin, int& end) {
  // `first`: the lane's first row, `count`: rows, `tiles`: up to and including the lane's group
  int first = 0, count = 0, tiles = 0;
  const auto load = [&](const int base) {
    const int g = base + lane;
    first = 0;
    count = 0;
    if (g < groups) {
      const long long from = offsets[g], to = offsets[g + 1];
      first = static_cast<int>(from < 0 ? 0 : (from > rows ? rows : from));
      count = static_cast<int>(to < first ? 0 : (to > rows ? rows : to) - first);
    }
    tiles = min((count + tile - 1) / tile, kLayerMostGroupTiles);
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const int other = __shfl_up(tiles, step, 64);
      if (lane >= step) { tiles += other; }
    }
  };
  int total = 0;
  for (int base = 0; base < groups; base += 64) {
    load(base);
    total = min(total + __builtin_amdgcn_readlane(tiles, 63), 128 * kLayerMostGroupTiles);
  }
  const int wanted = wanted_of(total);
  if (wanted < 0 || wanted >= total) { return false; }
  int passed = 0;
  for (int base = 0; base < groups; base += 64) {
    if (groups > 64) { load(base); }
    const int here = __builtin_amdgcn_readlane(tiles, 63);
    if (wanted < passed + here) {
      const unsigned long long reached = __ballot(passed + tiles > wanted);
      const int owner = __builtin_ctzll(reached);
      group = base + owner;
      begin = __builtin_amdgcn_readlane(first, owner);
      end = begin + __builtin_amdgcn_readlane(count, owner);
      before = passed + ((owner > 0) ? __builtin_amdgcn_readlane(tiles, (owner > 0) ? owner - 1 : 0) : 0);
      return true;
    }
    passed += here;
  }
  return false;
}

// The group with the rank-th largest range (of equal ones the first comes first), where it begins and how long it is; for up to
// 64 groups, one per lane. Group number `rank` beyond.
__device__ __forceinline__ void GroupOfRank(const long long* __restrict__ offsets, const int groups, const int rows, const int rank,
                                            const int lane, int& group, int& begin, int& length) {
  if (groups > 64) {
    group = rank;
    int end;
    GroupRange(offsets, group, rows, begin, end);
    length = end - begin;
    return;
  }
  int first = 0, count = -1;
  if (lane < groups) {
    const long long from = offsets[lane], to = offsets[lane + 1];
    first = static_cast<int>(from < 0 ? 0 : (from > rows ? rows : from));
    count = static_cast<int>(to < first ? 0 : (to > rows ? rows : to) - first);
  }
  int above = 0;
  for (int g = 0; g < groups; ++g) {
    const int other = __builtin_amdgcn_readlane(count, g);
    above += (other > count || (other == count && g < lane)) ? 1 : 0;
  }
  group = __builtin_ctzll(__ballot(lane < groups && above == rank));
  begin = __builtin_amdgcn_readlane(first, group);
  length = __builtin_amdgcn_readlane(count, group);
}

// ---- types and configurations ------------------------------------------------------------------------------------------

typedef short short8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bfloat8_t __attribute__((ext_vector_type(8)));
typedef float layer_float4_t __attribute__((ext_vector_type(4)));
typedef float layer_float8_t __attribute__((ext_vector_type(8)));

// WM x WN wavefronts, each owning (32 FM) x (32 FN) of the tile; BLOCK: extent of the matrix instruction's block.
// TEAMS = 2: two such sets of wavefronts with a ring each, of which the second takes the second half of the depth.
template <typename T_, int WM_, int WN_, int FM_, int FN_, int MIN_WAVES_, int STAGES_ = 3, int TEAMS_ = 1>
struct LayerConfig {
  using T = T_;
  static constexpr int WM = WM_, WN = WN_, FM = FM_, FN = FN_, MIN_WAVES = MIN_WAVES_;
  static constexpr int TEAMS = TEAMS_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES * TEAMS;  // WAVES: of a team
  static constexpr int TILE_M = WM * FM * 32, TILE_N = WN * FN * 32;
  static constexpr int TILE_K = 64 / sizeof(T);
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr int BLOCK = (sizeof(T) == 4 && FM % 2 == 0 && FN % 2 == 0) ? 32 : 16;
  static constexpr int BM = 32 * FM / BLOCK, BN = 32 * FN / BLOCK;  // the wavefront's blocks
  static constexpr int STAGES = STAGES_;  // LDS slab buffers: slab + STAGES - 1 is requested under the products of a slab
  static constexpr int PIECES_A = TILE_M / 16, PIECES_B = TILE_N / 16;  // 1 KiB pieces of a slab
  static constexpr int ROUNDS = (PIECES_A + PIECES_B + WAVES - 1) / WAVES;
  static constexpr bool DUMMY = (PIECES_A + PIECES_B) % WAVES != 0;
  static constexpr int A_BYTES = PIECES_A * 1024, B_BYTES = PIECES_B * 1024;
  static constexpr int RING_BYTES = STAGES * (A_BYTES + B_BYTES) + (DUMMY ? 1024 : 0);
  static constexpr int WAVE_M = 32 * FM, WAVE_N = 32 * FN;
  static constexpr int PITCH = WAVE_M + 4;  // floats of a row of the epilogue's staging tile
  static constexpr int HALF_N = WAVE_N / 2;  // rows that a wavefront stages at a time
  static constexpr int STAGE_BYTES = HALF_N * PITCH * 4;
  static constexpr int EPILOGUE_BYTES = TEAMS * WAVES * STAGE_BYTES;
  static constexpr int SUM_BYTES = TEAMS * WN * TILE_M * 4;  // the wavefronts' parts of the bias gradient
  static constexpr int EXCHANGE_FLOATS = (TEAMS == 2) ? WAVE_M * HALF_N : 0;  // sums that a wavefront hands to the other team
  static constexpr int TAIL_BYTES = EPILOGUE_BYTES + SUM_BYTES + TEAMS * WAVES * EXCHANGE_FLOATS * 4;
  static constexpr int LDS_BYTES = (TEAMS * RING_BYTES > TAIL_BYTES) ? TEAMS * RING_BYTES : TAIL_BYTES;
  static_assert(TEAMS == 1 || TEAMS == 2, "each team finishes one half of the rows");
  static_assert(BM % 2 == 0 && BN % 2 == 0 && BM >= BN, "the quadrants are halves of the blocks, walked along m");
};

template <typename Config> struct LayerMath;

// Fragment reads and products of a slab, per type. Offsets are in bytes from the start of the operand's stage.
template <typename Config>
struct LayerMath16 {
  using Frag = short8_t;
  typedef float Acc __attribute__((ext_vector_type(4)));
  template <int W, bool KC>
  static __device__ __forceinline__ int Offset(const int lane, const int x0) { return 2 * HFragmentOffset<W, KC>(lane, x0); }
  template <int W, bool KC>
  static __device__ __forceinline__ Frag Read(const char* stage, const int offset) {
    return __builtin_bit_cast(Frag, HFragment<W, KC>(reinterpret_cast<const _Float16*>(stage + offset), 0));
  }
  static __device__ __forceinline__ Acc Multiply(const Frag a, const Frag b, const Acc acc) {
    if constexpr (std::is_same<typename Config::T, __bf16>::value) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfloat8_t, a), __builtin_bit_cast(bfloat8_t, b), acc, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), acc, 0, 0, 0);
    }
  }
};

template <typename Config, int BLOCK> struct LayerMath32;
template <typename Config>
struct LayerMath32<Config, 32> {
  using Frag = layer_float8_t;
  using Acc = float16_t;
  template <int W, bool KC>
  static __device__ __forceinline__ int Offset(const int lane, const int x0) {
    const int x = x0 + lane % 32, h = lane / 32;
    return KC ? x * 64 : (4 * h * W + x) * 4;
  }
  template <int W, bool KC>
  static __device__ __forceinline__ Frag Read(const char* stage, const int offset, const int lane) {
    Frag out;
    if constexpr (KC) {
      // (offset is a multiple of 64 bytes: the row; its swizzle comes from the row's number)
      const int h = lane / 32, swizzle = (offset >> 8) & 3;
      const layer_float4_t low = *reinterpret_cast<const layer_float4_t*>(stage + offset + 16 * (h ^ swizzle));
      const layer_float4_t high = *reinterpret_cast<const layer_float4_t*>(stage + offset + 16 * ((2 + h) ^ swizzle));
#pragma unroll
      for (int s = 0; s < 4; ++s) { out[s] = low[s]; out[4 + s] = high[s]; }
    } else {
      const float* from = reinterpret_cast<const float*>(stage + offset);
#pragma unroll
      for (int s = 0; s < 4; ++s) { out[s] = from[s * W]; out[4 + s] = from[(8 + s) * W]; }
    }
    return out;
  }
  static constexpr int STEPS = 8;  // instructions per block and slab
  static __device__ __forceinline__ Acc Step(const Frag a, const Frag b, const Acc acc, const int s) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], acc, 0, 0, 0);
  }
};
template <typename Config>
struct LayerMath32<Config, 16> {
  using Frag = layer_float4_t;
  typedef float Acc __attribute__((ext_vector_type(4)));
  template <int W, bool KC>
  static __device__ __forceinline__ int Offset(const int lane, const int x0) {
    const int x = x0 + lane % 16, g = lane / 16;
    return KC ? x * 64 + 16 * (g ^ ((x >> 2) & 3)) : (4 * g * W + x) * 4;
  }
  template <int W, bool KC>
  static __device__ __forceinline__ Frag Read(const char* stage, const int offset, const int) {
    if constexpr (KC) { return *reinterpret_cast<const Frag*>(stage + offset); }
    Frag out;
    const float* from = reinterpret_cast<const float*>(stage + offset);
#pragma unroll
    for (int s = 0; s < 4; ++s) { out[s] = from[s * W]; }
    return out;
  }
  static constexpr int STEPS = 4;
  static __device__ __forceinline__ Acc Step(const Frag a, const Frag b, const Acc acc, const int s) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], acc, 0, 0, 0);
  }
};

template <typename Config, bool WIDE = (sizeof(typename Config::T) == 4)> struct LayerMathOf { using type = LayerMath16<Config>; };
template <typename Config> struct LayerMathOf<Config, true> { using type = LayerMath32<Config, Config::BLOCK>; };

// ---- slab movement -----------------------------------------------------------------------------------------------------

// Byte offset of a lane's 16 bytes from the first line of a 1 KiB piece. KC: 16 lines x of 64 bytes, the chunk swizzled
// by (x >> 2) & 3; else lines k of W elements (16 bits: swizzled for the transposing read, fp32: in order).
template <typename T, int W, bool KC>
__device__ __forceinline__ int LayerPieceLaneBytes(const long long ld, const int piece, const int lane) {
  constexpr int LINES = LayerPieceLines(KC, W, sizeof(T)), CHUNKS = 64 / LINES;
  static_assert(LINES >= 1, "a piece holds whole lines");
  const int line = lane / CHUNKS, position = lane % CHUNKS;
  int chunk = position;
  if constexpr (KC) { chunk = position ^ ((line >> 2) & 3); }
  else if constexpr (sizeof(T) == 2) { chunk = position ^ HSwizzle<W>(LINES * piece + line); }
  return static_cast<int>(static_cast<unsigned>(line * ld * static_cast<long long>(sizeof(T)) + 16 * chunk));  // (the load takes it as unsigned)
}

template <bool RANGE, typename Tag>
__device__ __forceinline__ void LayerRequestPiece(const char* source, const char* valid_end, char* destination, const int lane_bytes) {
  typedef __attribute__((address_space(3))) void* LdsPtr;
  const int records = RANGE ? HRecordsUpTo(source, valid_end) : -1;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(source), 0, records, kRawBufferFlags),
                                           (LdsPtr)(destination), 16, lane_bytes, 0, 0, 0);
}

// Zeroes the values k >= k_valid of a k-contiguous piece that this wavefront requested itself
template <typename T>
__device__ __forceinline__ void LayerZeroTail(char* stage, const int piece, const int lane, const int k_valid) {
  constexpr int VEC = 16 / sizeof(T);
  const int line = lane / 4, chunk = (lane % 4) ^ ((line >> 2) & 3);
  T* cell = reinterpret_cast<T*>(stage + piece * 1024 + lane * 16);
  if (VEC * chunk + VEC - 1 >= k_valid) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) { if (VEC * chunk + e >= k_valid) { cell[e] = T(0); } }
  }
}

// ---- epilogue ----------------------------------------------------------------------------------------------------------

// V values through the layer's elementwise work: z is alpha times the sum (+ bias), `other` the residual (forward) or Z
// (gradient). The choices are the launch's; they stand outside the loops over the values.
// OTHER: there is such a value (without one a gradient has no activation to go through)
template <bool FAST, int ACTIVATION, bool OTHER, int V>
__device__ __forceinline__ void LayerValuesOf(const LayerArgs& p, const float (&z)[V], const float (&other)[V], float (&y)[V]) {
  if (OTHER && p.gradient) {
#pragma unroll
    for (int e = 0; e < V; ++e) { y[e] = z[e] * ActivationSlope<FAST>(ACTIVATION, other[e]); }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) { y[e] = Activate<FAST>(ACTIVATION, z[e]); }
    if (OTHER && p.beta != 0.0f) {
#pragma unroll
      for (int e = 0; e < V; ++e) { y[e] = __builtin_fmaf(p.beta, other[e], y[e]); }
    }
  }
}
template <bool FAST, bool OTHER, int V>
__device__ __forceinline__ void LayerValues(const LayerArgs& p, const float (&z)[V], const float (&other)[V], float (&y)[V]) {
  switch (p.activation) {
    case kActivationRelu: LayerValuesOf<FAST, kActivationRelu, OTHER>(p, z, other, y); break;
    case kActivationGelu: LayerValuesOf<FAST, kActivationGelu, OTHER>(p, z, other, y); break;
    case kActivationGeluTanh: LayerValuesOf<FAST, kActivationGeluTanh, OTHER>(p, z, other, y); break;
    case kActivationSilu: LayerValuesOf<FAST, kActivationSilu, OTHER>(p, z, other, y); break;
    default: LayerValuesOf<FAST, kActivationNone, OTHER>(p, z, other, y); break;
  }
}

// A global address that is the same in all lanes, in scalar registers whatever the compiler thinks of how it came about
typedef __attribute__((address_space(1))) char* GlobalBytes;
__device__ __forceinline__ GlobalBytes UniformAddress(const void* pointer) {
  const unsigned long long address = reinterpret_cast<unsigned long long>(pointer);
  const unsigned long long low = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(address)));
  const unsigned long long high = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(address >> 32)));
  return (GlobalBytes)((high << 32) | low);
}

// V consecutive values of a row, of which the first `inside` exist, as one access at whatever address the row starts (the
// hardware splits one that is not aligned). Results are stored past the caches' keeping: they are not read again here and would push
// out the operands that neighbouring tiles share (8192 x 8192 x 1024 142 -> 121 us, x 4096 with GELU and Z 476 -> 462 us);
// so does a residual, read once (what it adds to the former: 45 -> 31 us).
template <typename T, int V>
struct LayerPiece {
  typedef T Piece __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  typedef T Raw __attribute__((ext_vector_type(V)));  // as it is in memory: half the registers of its values for 16 bits
  static __device__ __forceinline__ void Values(const Raw raw, float (&values)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) { const T value = raw[e]; values[e] = static_cast<float>(value); }
  }
  // at a uniform address and a lane's byte offset from there (the access carries both, no address is computed)
  typedef __attribute__((address_space(1))) Piece* GlobalPiece;
  static __device__ __forceinline__ Raw LoadAt(const GlobalBytes base, const unsigned offset) { return __builtin_nontemporal_load((GlobalPiece)(base + offset)); }
  static __device__ __forceinline__ void StoreAt(const GlobalBytes base, const unsigned offset, const float (&values)[V]) {
    Piece piece;
#pragma unroll
    for (int e = 0; e < V; ++e) { piece[e] = static_cast<T>(values[e]); }
    __builtin_nontemporal_store(piece, (GlobalPiece)(base + offset));
  }
  static __device__ __forceinline__ void Load(const T* from, const int inside, float (&values)[V]) {
    if (inside >= V) {
      const Piece piece = *reinterpret_cast<const Piece*>(from);
#pragma unroll
      for (int e = 0; e < V; ++e) { const T value = piece[e]; values[e] = static_cast<float>(value); }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) { values[e] = (e < inside) ? static_cast<float>(from[e]) : 0.0f; }
    }
  }
  // the same without the conversion, zeros behind `inside`. STREAM: what nobody reads a second time
  template <bool STREAM>
  static __device__ __forceinline__ Raw LoadRaw(const T* from, const int inside) {
    if (inside >= V) {
      if constexpr (STREAM) { return __builtin_bit_cast(Raw, __builtin_nontemporal_load(reinterpret_cast<const Piece*>(from))); }
      else { return __builtin_bit_cast(Raw, *reinterpret_cast<const Piece*>(from)); }
    }
    Raw raw;
#pragma unroll
    for (int e = 0; e < V; ++e) { raw[e] = (e < inside) ? from[e] : T(0.0f); }
    return raw;
  }
  static __device__ __forceinline__ void Store(T* to, const int inside, const float (&values)[V]) {
    if (inside >= V) {
      Piece piece;
#pragma unroll
      for (int e = 0; e < V; ++e) { piece[e] = static_cast<T>(values[e]); }
      __builtin_nontemporal_store(piece, reinterpret_cast<Piece*>(to));
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) { if (e < inside) { to[e] = static_cast<T>(values[e]); } }
    }
  }
};

// Moves staged rows of a wavefront through the epilogue, lanes along the features in pieces of V values. The loops over the
// rows are not unrolled (their bodies hold every activation).
template <typename Config>
struct LayerRows {
  using T = typename Config::T;
  static constexpr int V = Config::VEC;
  using Piece = LayerPiece<T, V>;
  static constexpr bool FAST = sizeof(T) == 2;
  static constexpr int ROW_LANES = Config::WAVE_M / V;  // pieces of a row, one per lane
  static constexpr int ROWS = 64 / ROW_LANES;           // rows per pass
  static constexpr int PASSES = Config::HALF_N / ROWS;
  static_assert(ROW_LANES <= 64, "a row is at most one piece per lane");
  float bias[V], sums[V];

  __device__ __forceinline__ void Begin(const T* bias_from, const int lane, const int inside) {
    const int col = V * (lane % ROW_LANES);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sums[e] = 0.0f;
      bias[e] = 0.0f;
    }
    if (bias_from != nullptr) { Piece::Load(bias_from + col, inside - col, bias); }
  }

  // stage: the wavefront's staging tile of HALF_N rows, of which `rows` exist, each with `inside` features; c, pre, other: at
  // the first of them
  __device__ __forceinline__ void Run(const LayerArgs& p, const float* stage, T* c, T* pre, const T* other, const long long other_ld,
                                      const int lane, const int rows, const int inside) {
    T* z_out = p.gradient ? nullptr : pre;
    // (a lane's offset within a pass, up to 16 rows, in 32 bits)
    const bool small = p.c_ld < (1 << 25) && (z_out == nullptr || p.pre_ld < (1 << 25)) && (other == nullptr || other_ld < (1 << 25));
    if (rows >= Config::HALF_N && inside >= Config::WAVE_M && small) {
      if (other != nullptr) { Whole<true>(p, stage, c, z_out, other, other_ld, lane); }
      else { Whole<false>(p, stage, c, z_out, other, other_ld, lane); }
    } else {
      Partial(p, stage, c, z_out, other, other_ld, lane, rows, inside);
    }
  }

  static constexpr int FOURS = V / 4;
  static __device__ __forceinline__ void Fetch(const float* from, layer_float4_t (&staged)[FOURS]) {
#pragma unroll
    for (int q = 0; q < FOURS; ++q) { staged[q] = *reinterpret_cast<const layer_float4_t*>(from + 4 * q); }
  }
  __device__ __forceinline__ void Scale(const LayerArgs& p, const layer_float4_t (&staged)[FOURS], float (&z)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) { z[e] = __builtin_fmaf(p.alpha, staged[e / 4][e % 4], bias[e]); }
  }

  // All rows and features exist. Nothing but the values is left to the vector unit: addresses advance as scalars. (With them
  // and the tests for partial pieces in vector registers the pass took 4.6 of a 256 x 256 tile's 12 us.)
  template <bool OTHER>
  __device__ __forceinline__ void Whole(const LayerArgs& p, const float* stage, T* c, T* z_out, const T* other, const long long other_ld,
                                        const int lane) {
    constexpr int AHEAD = PASSES < 4 ? PASSES : 4;  // passes that `other` is asked for in advance
    constexpr unsigned SIZE = sizeof(T);
    const int row0 = lane / ROW_LANES, col = V * (lane % ROW_LANES);
    const auto offset = [&](const long long ld) { return (static_cast<unsigned>(row0) * static_cast<unsigned>(ld) + col) * SIZE; };
    GlobalBytes c_base = UniformAddress(c);
    GlobalBytes z_base = UniformAddress(z_out);
    GlobalBytes other_base = UniformAddress(other);
    const unsigned c_offset = offset(p.c_ld), z_offset = offset(p.pre_ld), other_offset = offset(other_ld);
    const long long c_step = ROWS * p.c_ld * SIZE, z_step = ROWS * p.pre_ld * SIZE, other_step = ROWS * other_ld * SIZE;
    typename Piece::Raw old[AHEAD];
    if constexpr (OTHER) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        old[u] = Piece::LoadAt(other_base, other_offset);
        other_base += other_step;
      }
    }
    const float* from = stage + row0 * Config::PITCH + col;
    layer_float4_t staged[FOURS];
    Fetch(from, staged);
#pragma unroll 1
    for (int pass = 0; pass < PASSES; ++pass) {
      float now[V], z[V], y[V];
      Scale(p, staged, z);
      if (pass + 1 < PASSES) { from += ROWS * Config::PITCH; }
      Fetch(from, staged);  // (of the next pass: its latency under this one's arithmetic)
      if constexpr (OTHER) {
        Piece::Values(old[0], now);
#pragma unroll
        for (int u = 0; u + 1 < AHEAD; ++u) { old[u] = old[u + 1]; }
        if (pass + AHEAD < PASSES) { old[AHEAD - 1] = Piece::LoadAt(other_base, other_offset); }
        other_base += other_step;
      }
      LayerValues<FAST, OTHER>(p, z, now, y);
      if (p.bias_partials != nullptr) {
#pragma unroll
        for (int e = 0; e < V; ++e) { sums[e] += y[e]; }
      }
      Piece::StoreAt(c_base, c_offset, y);
      c_base += c_step;
      if (z_out != nullptr) {
        Piece::StoreAt(z_base, z_offset, z);
        z_base += z_step;
      }
    }
  }

  // A tile at the edge of the matrix or of a group
  __device__ __forceinline__ void Partial(const LayerArgs& p, const float* stage, T* c, T* z_out, const T* other, const long long other_ld,
                                          const int lane, const int rows, const int inside) {
    const int row0 = lane / ROW_LANES, col = V * (lane % ROW_LANES);
    const auto inside_of = [&](const int row) { return (row < rows) ? inside - col : 0; };
    float next[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { next[e] = 0.0f; }
    if (other != nullptr) { Piece::Load(other + row0 * other_ld + col, inside_of(row0), next); }
#pragma unroll 1
    for (int pass = 0; pass < PASSES; ++pass) {
      const int row = row0 + pass * ROWS, here = inside_of(row);
      float now[V], z[V], y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) { now[e] = next[e]; }
      if (other != nullptr && pass + 1 < PASSES) { Piece::Load(other + (row + ROWS) * other_ld + col, inside_of(row + ROWS), next); }
      layer_float4_t staged[FOURS];
      Fetch(stage + row * Config::PITCH + col, staged);
      Scale(p, staged, z);
      LayerValues<FAST, true>(p, z, now, y);
      if (here > 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) { sums[e] += y[e]; }
      }
      Piece::Store(c + row * p.c_ld + col, here, y);
      if (z_out != nullptr) { Piece::Store(z_out + row * p.pre_ld + col, here, z); }
    }
  }

  // The wavefront's sums over its rows to `to` (LDS, WAVE_M values): lanes with the same features are added up first
  __device__ __forceinline__ void StoreSums(float* to, const int lane) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float sum = sums[e];
#pragma unroll
      for (int step = ROW_LANES; step < 64; step *= 2) { sum += __shfl_xor(sum, step, 64); }
      if (lane < ROW_LANES) { to[V * lane + e] = sum; }
    }
  }
};

// ---- the kernel --------------------------------------------------------------------------------------------------------

template <typename Config, bool A_KC, bool B_KC>
__global__ __launch_bounds__(Config::THREADS, Config::MIN_WAVES) void LayerGemmKernel(const LayerArgs p, const int tiles_m,
                                                                                     const int tiles_n, const int first_block) {
  using T = typename Config::T;
  using Math = typename LayerMathOf<Config>::type;
  using Frag = typename Math::Frag;
  using Acc = typename Math::Acc;
  constexpr int TILE_M = Config::TILE_M, TILE_N = Config::TILE_N, TILE_K = Config::TILE_K, BLOCK = Config::BLOCK;
  constexpr int BM = Config::BM, BN = Config::BN, HM = BM / 2, HN = BN / 2;
  constexpr int TEAMS = Config::TEAMS, WAVES = Config::WAVES, ROUNDS = Config::ROUNDS, STAGES = Config::STAGES, AHEAD = STAGES - 1;
  static_assert(AHEAD >= 2 && AHEAD <= 5 && AHEAD * ROUNDS < 64, "the waits below");
  using KernelTag = std::tuple<Config, std::integral_constant<int, (A_KC ? 2 : 0) | (B_KC ? 1 : 0)>>;

  extern __shared__ __align__(16) unsigned char lds_raw[];
  const int tid = threadIdx.x, lane = tid % 64;
  const int any_wave = __builtin_amdgcn_readfirstlane(tid / 64);  // of both teams
  const int wave = any_wave % WAVES, team = (TEAMS == 1) ? 0 : any_wave / WAVES;
  char* a_ring = reinterpret_cast<char*>(lds_raw) + team * Config::RING_BYTES;
  char* b_ring = a_ring + STAGES * Config::A_BYTES;
  char* scratch_piece = b_ring + STAGES * Config::B_BYTES;

  const int wave_m = wave % Config::WM, wave_n = wave / Config::WM;
  const unsigned block = first_block + blockIdx.x;  // (first_block: of this slice of the grid)

  // ---- which tile, of which group
  int tile_m, tile_n, group = 0;
  int rows = p.n, depth = p.k, first = 0;  // the group's rows or depths, and where they begin
  int sums_row;                            // the tile's row of bias_partials
  if (p.grouping == kLayerGroupedRows) {
    int before = 0, end = 0, index = 0;
    const bool found = FindGroupTile(p.offsets, p.groups, p.n, TILE_N, lane, [&](const int total) {
      const long long all = static_cast<long long>(total) * tiles_m;
      if (static_cast<long long>(block) >= all || all > 0x7fffffff) { return -1; }
      index = XcdContiguousIndex(block, total * tiles_m);
      return index / tiles_m;
    }, group, before, first, end);
    if (!found) { return; }
    rows = end - first;
    // inside a group: eight tile rows of features at a time, so that the tiles in flight on an XCD share panels
    const int group_tiles = (rows + TILE_N - 1) / TILE_N;
    const int local = index - before * tiles_m;
    const int walk = local / (8 * group_tiles), height = min(tiles_m - 8 * walk, 8);
    tile_m = 8 * walk + (local - walk * 8 * group_tiles) % height;
    tile_n = (local - walk * 8 * group_tiles) / height;
    sums_row = before + tile_n;
  } else if (p.grouping == kLayerGroupedDepth) {
    // The depths differ from group to group: every XCD (work-groups are dealt to the eight in turn) takes an eighth of every
    // group's tiles, a contiguous one, and the groups come in the order of their depths, the deepest first.
    const int share = (tiles_m * tiles_n + kNumXcd - 1) / kNumXcd;
    const int local = static_cast<int>(block / kNumXcd) % share + static_cast<int>(block % kNumXcd) * share;
    if (local >= tiles_m * tiles_n) { return; }
    GroupOfRank(p.offsets, p.groups, p.k, block / kNumXcd / share, lane, group, first, depth);
    const int walk = local / (8 * tiles_n), height = min(tiles_m - 8 * walk, 8);
    tile_m = 8 * walk + (local - walk * 8 * tiles_n) % height;
    tile_n = (local - walk * 8 * tiles_n) / height;
    sums_row = tile_n;
  } else {
    TileOfBlock<(TILE_M >= 2 * TILE_N) ? 4 : 8>(block, tiles_m * tiles_n, tiles_m, tiles_n, tile_m, tile_n);
    sums_row = tile_n;
    if (p.split_chunk > 0) {
      first = blockIdx.y * p.split_chunk;
      depth = min(p.split_chunk, p.k - first);
    }
  }
  const int m0 = tile_m * TILE_M, n0 = tile_n * TILE_N;
  const T* a = static_cast<const T*>(p.a);
  const T* b = static_cast<const T*>(p.b);
  if (p.grouping == kLayerGroupedRows) {
    a += group * p.a_stride;
    b += first * (B_KC ? p.b_ld : 1);
  } else {  // (first is 0 but for K ranges and groups by depth)
    a += first * (A_KC ? 1 : p.a_ld);
    b += first * (B_KC ? 1 : p.b_ld);
  }

  Acc acc[BM][BN];
#pragma unroll
  for (int i = 0; i < BM; ++i) {
#pragma unroll
    for (int j = 0; j < BN; ++j) { acc[i][j] = Acc(0.0f); }
  }

  // Slabs of either team (both walk as many, they share the barriers; what lies behind the depth is zero)
  const int slabs = LayerTeamSlabs(depth, TILE_K, TEAMS);
  const bool whole_slabs = depth % (TEAMS * TILE_K) == 0;
  // behind the last element of the operand, taken before the teams part: the same for both
  const char* a_end = reinterpret_cast<const char*>(a + LayerOperandElements(A_KC, p.m, depth, p.a_ld));
  const char* b_end = reinterpret_cast<const char*>(b + LayerOperandElements(B_KC, rows, depth, p.b_ld));
  if (TEAMS == 2) {
    const int before = LayerTeamStart(depth, TILE_K, TEAMS, team);
    a += before * (A_KC ? 1 : p.a_ld);
    b += before * (B_KC ? 1 : p.b_ld);
    depth = LayerTeamDepth(depth, TILE_K, TEAMS, team);
  }
  const int k_tail = depth % TILE_K;
  if (slabs > 0) {
    int a_offset[BM], b_offset[BN];
#pragma unroll
    for (int q = 0; q < BM; ++q) { a_offset[q] = Math::template Offset<TILE_M, A_KC>(lane, (wave_m * BM + q) * BLOCK); }
#pragma unroll
    for (int q = 0; q < BN; ++q) { b_offset[q] = Math::template Offset<TILE_N, B_KC>(lane, (wave_n * BN + q) * BLOCK); }
    const auto read_a = [&](const char* stage, const int q) {
      if constexpr (sizeof(T) == 4) { return Math::template Read<TILE_M, A_KC>(stage, a_offset[q], lane); }
      else { return Math::template Read<TILE_M, A_KC>(stage, a_offset[q]); }
    };
    const auto read_b = [&](const char* stage, const int q) {
      if constexpr (sizeof(T) == 4) { return Math::template Read<TILE_N, B_KC>(stage, b_offset[q], lane); }
      else { return Math::template Read<TILE_N, B_KC>(stage, b_offset[q]); }
    };

    constexpr long long SIZE = sizeof(T);
    const char* a_tile = reinterpret_cast<const char*>(a + (A_KC ? m0 * p.a_ld : static_cast<long long>(m0)));
    const char* b_tile = reinterpret_cast<const char*>(b + (B_KC ? n0 * p.b_ld : static_cast<long long>(n0)));

    auto walk = [&](auto range_tag) {
      constexpr bool RANGE = decltype(range_tag)::value;
      const char* a_request = a_tile;  // first line of the slab to be requested next
      const char* b_request = b_tile;
      const long long a_step = A_KC ? 64 : TILE_K * p.a_ld * SIZE;
      const long long b_step = B_KC ? 64 : TILE_K * p.b_ld * SIZE;
      constexpr int A_LINES = LayerPieceLines(A_KC, TILE_M, SIZE), B_LINES = LayerPieceLines(B_KC, TILE_N, SIZE);
      const auto is_a = [&](const int round, const int piece) {
        return (Config::PIECES_A % WAVES == 0) ? (round < Config::PIECES_A / WAVES) : (piece < Config::PIECES_A);
      };
      long long piece_start[ROUNDS];
      int piece_lane_bytes[ROUNDS], piece_place[ROUNDS];
#pragma unroll
      for (int round = 0; round < ROUNDS; ++round) {
        const int piece = wave + WAVES * round;
        if (is_a(round, piece)) {
          piece_start[round] = static_cast<long long>(A_LINES * piece) * p.a_ld * SIZE;
          piece_lane_bytes[round] = LayerPieceLaneBytes<T, TILE_M, A_KC>(p.a_ld, piece, lane);
          piece_place[round] = piece * 1024;
        } else {
          const int b_piece = piece - Config::PIECES_A;
          piece_start[round] = static_cast<long long>(B_LINES * b_piece) * p.b_ld * SIZE;
          piece_lane_bytes[round] = LayerPieceLaneBytes<T, TILE_N, B_KC>(p.b_ld, b_piece, lane);
          piece_place[round] = b_piece * 1024;
        }
      }
      const auto request = [&](const int round, const int buffer) {
        const int piece = wave + WAVES * round;
        if (is_a(round, piece)) {
          char* place = a_ring + buffer * Config::A_BYTES + piece_place[round];
          LayerRequestPiece<RANGE, KernelTag>(a_request + piece_start[round], a_end, place, piece_lane_bytes[round]);
        } else if (!Config::DUMMY || piece < Config::PIECES_A + Config::PIECES_B) {
          char* place = b_ring + buffer * Config::B_BYTES + piece_place[round];
          LayerRequestPiece<RANGE, KernelTag>(b_request + piece_start[round], b_end, place, piece_lane_bytes[round]);
        } else {
          // keeps the number of requests in flight equal in all wavefronts (the waits count them): moves nothing
          LayerRequestPiece<true, KernelTag>(a_tile, a_tile, scratch_piece, lane * 16);
        }
      };
      // (one team: called for the last slab alone)
      const auto zero_tail = [&](const int buffer, const int of_slab) {
        if (!RANGE || !(A_KC || B_KC)) { return; }
        const int k_valid = (TEAMS == 1) ? k_tail : max(0, min(TILE_K, depth - of_slab * TILE_K));
        if (k_valid == ((TEAMS == 1) ? 0 : TILE_K)) { return; }
#pragma unroll
        for (int round = 0; round < ROUNDS; ++round) {
          const int piece = wave + WAVES * round;
          if (piece < Config::PIECES_A) {
            if (A_KC) { LayerZeroTail<T>(a_ring + buffer * Config::A_BYTES, piece, lane, k_valid); }
          } else if (piece < Config::PIECES_A + Config::PIECES_B) {
            if (B_KC) { LayerZeroTail<T>(b_ring + buffer * Config::B_BYTES, piece - Config::PIECES_A, lane, k_valid); }
          }
        }
      };

      const int first_slabs = min(slabs, AHEAD);
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        if (s < first_slabs) {
#pragma unroll
          for (int round = 0; round < ROUNDS; ++round) { request(round, s); }
          a_request += a_step;
          b_request += b_step;
        }
      }
      if (first_slabs == 1) { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
      else if (first_slabs == 2) { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ROUNDS) : "memory"); }
      else if (first_slabs == 3) { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * ROUNDS) : "memory"); }
      else if (first_slabs == 4) { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * ROUNDS) : "memory"); }
      else { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * ROUNDS) : "memory"); }
      if (TEAMS == 2 || slabs == 1) { zero_tail(0, 0); }
      __syncthreads();
      // 16 bits: halves of the fragments of one slab; fp32: all fragments of two slabs
      constexpr bool WIDE = sizeof(T) == 4;
      Frag a_frag[2][WIDE ? BM : HM], b_frag[2][WIDE ? BN : HN];
#pragma unroll
      for (int q = 0; q < (WIDE ? BM : HM); ++q) { a_frag[0][q] = read_a(a_ring, q); }
#pragma unroll
      for (int q = 0; q < (WIDE ? BN : HN); ++q) { b_frag[0][q] = read_b(b_ring, q); }
      int cur = 0, slab = 0;
      // One slab; LATER: how many follow it, capped at AHEAD. Slab + AHEAD is requested under the first two quadrants, into the
      // buffer whose reads everybody had waited for at the previous barrier.
      constexpr int PER_SLOT = (ROUNDS + 2 * HM - 1) / (2 * HM);
      const auto slab_body = [&](auto later_tag, auto parity_tag) {
        constexpr int LATER = decltype(later_tag)::value;
        constexpr int PARITY = decltype(parity_tag)::value;  // fp32: which set of fragments holds the slab
        constexpr bool LOAD = LATER == AHEAD;
        const int nxt = (cur == STAGES - 1) ? 0 : cur + 1, prv = (cur == 0) ? STAGES - 1 : cur - 1;
        const char* a_cur = a_ring + cur * Config::A_BYTES;
        const char* b_cur = b_ring + cur * Config::B_BYTES;
        const char* a_nxt = a_ring + nxt * Config::A_BYTES;
        const char* b_nxt = b_ring + nxt * Config::B_BYTES;
        const auto next_slab_in_place = [&]() {
          // slab + 1 must have landed for everybody; the requests for the slabs behind it may stay in flight
          constexpr int IN_FLIGHT = (LATER >= 2) ? (LATER - 1) * ROUNDS : 0;
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(IN_FLIGHT) : "memory");
          if (LATER == 1 || (TEAMS == 2 && LATER > 1)) { zero_tail(nxt, slab + 1); }  // (LATER == 1: slab + 1 is the last one)
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        };
        if constexpr (WIDE) {
          // fp32: all blocks between two products into the same registers (block by block the 16x16x4 form of 64 x 64 tiles
          // loses a tenth); requests under the first half of the slab's steps, the next slab's fragments read under the second
          constexpr int STEPS = Math::STEPS, PER_STEP = (ROUNDS + STEPS / 2 - 1) / (STEPS / 2);
#pragma unroll
          for (int step = 0; step < STEPS; ++step) {
            if (step == STEPS / 2) {
              next_slab_in_place();
#pragma unroll
              for (int q = 0; q < BM; ++q) { a_frag[1 - PARITY][q] = read_a(a_nxt, q); }
#pragma unroll
              for (int q = 0; q < BN; ++q) { b_frag[1 - PARITY][q] = read_b(b_nxt, q); }
            }
#pragma unroll
            for (int i = 0; i < BM; ++i) {
#pragma unroll
              for (int j = 0; j < BN; ++j) { acc[i][j] = Math::Step(a_frag[PARITY][i], b_frag[PARITY][j], acc[i][j], step); }
            }
            if (LOAD && step < STEPS / 2) {
#pragma unroll
              for (int u = 0; u < PER_STEP; ++u) {
                const int round = step * PER_STEP + u;
                if (round < ROUNDS) { request(round, prv); }
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
#pragma unroll
        for (int quadrant = 0; quadrant < 4; ++quadrant) {
          const int ha = quadrant / 2, hb = quadrant % 2;
#pragma unroll
          for (int q = 0; q < HM; ++q) {
            if (quadrant == 0 || quadrant == 3) {
              if (q < HN) {
                if (quadrant == 0) { b_frag[1][q] = read_b(b_cur, HN + q); }
                else { b_frag[0][q] = read_b(b_nxt, q); }
              }
            } else if (quadrant == 1) {
              a_frag[1][q] = read_a(a_cur, HM + q);
            } else {
              a_frag[0][q] = read_a(a_nxt, q);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < HN; ++j) {
              acc[ha * HM + q][hb * HN + j] = Math::Multiply(a_frag[ha][q], b_frag[hb][j], acc[ha * HM + q][hb * HN + j]);
            }
            if (LOAD && quadrant < 2) {
#pragma unroll
              for (int u = 0; u < PER_SLOT; ++u) {
                const int round = (quadrant * HM + q) * PER_SLOT + u;
                if (round < ROUNDS) { request(round, prv); }
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if (quadrant == 1) { next_slab_in_place(); }
        }
        }
        cur = nxt;
        if (LOAD) {
          a_request += a_step;
          b_request += b_step;
        }
      };
      using Even = std::integral_constant<int, 0>;
      using Odd = std::integral_constant<int, WIDE ? 1 : 0>;
      using Steady = std::integral_constant<int, AHEAD>;
      using Last = std::integral_constant<int, AHEAD - 1>;
      if constexpr (WIDE) {
        // the last slabs, from the one that LATER others follow on; the sets of fragments take turns
        const auto last_slabs = [&](auto self, auto later_tag, auto parity_tag) {
          constexpr int LATER = decltype(later_tag)::value, PARITY = decltype(parity_tag)::value;
          if (slab + LATER < slabs) {
            slab_body(later_tag, parity_tag);
            ++slab;
            if constexpr (LATER > 0) { self(self, std::integral_constant<int, LATER - 1>{}, std::integral_constant<int, 1 - PARITY>{}); }
          } else {
            if constexpr (LATER > 0) { self(self, std::integral_constant<int, LATER - 1>{}, parity_tag); }
          }
        };
        while (slab + AHEAD + 1 < slabs) {
          slab_body(Steady{}, Even{});
          ++slab;
          slab_body(Steady{}, Odd{});
          ++slab;
        }
        if (slab + AHEAD < slabs) {
          slab_body(Steady{}, Even{});
          ++slab;
          last_slabs(last_slabs, Last{}, Odd{});
        } else {
          last_slabs(last_slabs, Last{}, Even{});
        }
      } else {
        const auto last_slabs = [&](auto self, auto later_tag) {
          constexpr int LATER = decltype(later_tag)::value;
          if (slab + LATER < slabs) {
            slab_body(later_tag, Even{});
            ++slab;
          }
          if constexpr (LATER > 0) { self(self, std::integral_constant<int, LATER - 1>{}); }
        };
        for (; slab + AHEAD < slabs; ++slab) { slab_body(Steady{}, Even{}); }
        last_slabs(last_slabs, Last{});
      }
    };
    if (m0 + TILE_M <= p.m && n0 + TILE_N <= rows && whole_slabs) { walk(std::false_type{}); }
    else { walk(std::true_type{}); }
  }

  // ---- teams: each keeps one half of the rows and adds what the other one has of it
  if constexpr (TEAMS == 2) {
    float* exchange = reinterpret_cast<float*>(lds_raw + Config::EPILOGUE_BYTES + Config::SUM_BYTES);
    float* given = exchange + (any_wave * Config::EXCHANGE_FLOATS + lane * 4);
    const float* taken = exchange + ((wave + (1 - team) * WAVES) * Config::EXCHANGE_FLOATS + lane * 4);
    constexpr int FOURS = sizeof(Acc) / 16;
    __syncthreads();  // every wavefront is done with the slab buffers
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half != team) {
#pragma unroll
        for (int i = 0; i < BM * HN * FOURS; ++i) {
          layer_float4_t run;
#pragma unroll
          for (int e = 0; e < 4; ++e) { run[e] = acc[i / FOURS % BM][half * HN + i / FOURS / BM][i % FOURS * 4 + e]; }
          *reinterpret_cast<layer_float4_t*>(given + i * 256) = run;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == team) {
#pragma unroll
        for (int i = 0; i < BM * HN * FOURS; ++i) {
          const layer_float4_t run = *reinterpret_cast<const layer_float4_t*>(taken + i * 256);
#pragma unroll
          for (int e = 0; e < 4; ++e) { acc[i / FOURS % BM][half * HN + i / FOURS / BM][i % FOURS * 4 + e] += run[e]; }
        }
      }
    }
  }

  // ---- K ranges: the sums as they are
  if (p.split_chunk > 0) {
    float* partial = p.partials + static_cast<long long>(blockIdx.y) * p.n * p.m;
#pragma unroll
    for (int j = 0; j < BN; ++j) {
      if (TEAMS == 2 && j / HN != team) { continue; }
      const int row = n0 + (wave_n * BN + j) * BLOCK + lane % BLOCK;
#pragma unroll
      for (int i = 0; i < BM; ++i) {
#pragma unroll
        for (int r = 0; r < static_cast<int>(sizeof(Acc) / 16); ++r) {
          const int col = m0 + (wave_m * BM + i) * BLOCK + (BLOCK == 32 ? 8 * r + 4 * (lane / 32) : 4 * (lane / 16));
          float* to = partial + static_cast<long long>(row) * p.m + col;
          if (row < p.n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) { if (col + e < p.m) { to[e] = acc[i][j][4 * r + e]; } }
          }
        }
      }
    }
    return;
  }

  // ---- epilogue
  if (TEAMS == 1) { __syncthreads(); }  // every wavefront is done with the slab buffers
  int late_lane = lane;  // (opaque, so that what the epilogue derives from it does not occupy registers during the walk)
  asm volatile("" : "+v"(late_lane));
  float* stage = reinterpret_cast<float*>(lds_raw + any_wave * Config::STAGE_BYTES);
  float* tile_sums = reinterpret_cast<float*>(lds_raw + Config::EPILOGUE_BYTES);
  const int wave_m0 = m0 + wave_m * Config::WAVE_M;
  const int inside = p.m - wave_m0;
  const long long first_row = (p.grouping == kLayerGroupedRows) ? first : 0;
  T* c = static_cast<T*>(p.c) + first_row * p.c_ld + ((p.grouping == kLayerGroupedDepth) ? group * p.c_stride : 0) + wave_m0;
  T* pre = (p.pre == nullptr) ? nullptr : static_cast<T*>(p.pre) + first_row * p.pre_ld + wave_m0;
  const T* other = nullptr;
  long long other_ld = 0;
  if (p.gradient) {
    other = pre;
    other_ld = p.pre_ld;
  } else if (p.beta != 0.0f) {
    // (of groups by depth the residual is C itself, in place)
    other = static_cast<const T*>(p.residual) + first_row * p.residual_ld +
            ((p.grouping == kLayerGroupedDepth) ? group * p.c_stride : 0) + wave_m0;
    other_ld = p.residual_ld;
  }
  const T* bias = (p.bias == nullptr) ? nullptr : static_cast<const T*>(p.bias) + group * p.bias_stride + wave_m0;
  const auto wave_fence = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  if (inside > 0) {
    LayerRows<Config> rows_of;
    rows_of.Begin(bias, late_lane, inside);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (TEAMS == 2 && half != team) { continue; }
#pragma unroll
      for (int j = 0; j < HN; ++j) {
#pragma unroll
        for (int i = 0; i < BM; ++i) {
#pragma unroll
          for (int r = 0; r < static_cast<int>(sizeof(Acc) / 16); ++r) {
            const int col = i * BLOCK + (BLOCK == 32 ? 8 * r + 4 * (late_lane / 32) : 4 * (late_lane / 16));
            layer_float4_t run;
#pragma unroll
            for (int e = 0; e < 4; ++e) { run[e] = acc[i][half * HN + j][4 * r + e]; }
            *reinterpret_cast<layer_float4_t*>(&stage[(j * BLOCK + late_lane % BLOCK) * Config::PITCH + col]) = run;
          }
        }
      }
      wave_fence();
      const int n_block = n0 + wave_n * Config::WAVE_N + half * Config::HALF_N;
      if (n_block < rows) {
        rows_of.Run(p, stage, c + n_block * p.c_ld, (pre == nullptr) ? nullptr : pre + n_block * p.pre_ld,
                    (other == nullptr) ? nullptr : other + n_block * other_ld, other_ld, late_lane, rows - n_block, inside);
      }
      wave_fence();
    }
    if (p.bias_partials != nullptr) { rows_of.StoreSums(tile_sums + (team * Config::WN + wave_n) * TILE_M + wave_m * Config::WAVE_M, late_lane); }
  }
  if (p.bias_partials != nullptr) {
    __syncthreads();
    for (int i = tid; i < TILE_M && m0 + i < p.m; i += Config::THREADS) {
      float sum = tile_sums[i];
#pragma unroll
      for (int w = 1; w < TEAMS * Config::WN; ++w) { sum += tile_sums[w * TILE_M + i]; }
      p.bias_partials[static_cast<long long>(sums_row) * p.m + m0 + i] = sum;
    }
  }
}

}  // namespace clbh

#endif  // CLBLAST_HIP_KERNELS_LAYER_GEMM_HPP_
