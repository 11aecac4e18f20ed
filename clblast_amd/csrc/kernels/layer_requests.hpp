// =================================================================================================
// Which part of the depth a team of wavefronts walks in kernels/layer_gemm.hpp, and how far an operand reaches: what the
// ranges of its requests follow from. Free of HIP, so that a host-only test can replay every request of a tile and
// check that none leaves its operand (tests/host/layer_requests.cpp).
// =================================================================================================
#ifndef CLBLAST_HIP_KERNELS_LAYER_REQUESTS_HPP_
#define CLBLAST_HIP_KERNELS_LAYER_REQUESTS_HPP_

namespace clbh {

// Slabs that each of `teams` teams walks: all of them as many, what lies behind the depth is zero
constexpr int LayerTeamSlabs(const int depth, const int tile_k, const int teams) {
  return ((depth + tile_k - 1) / tile_k + teams - 1) / teams;
}

// Where a team's first slab begins. Behind the depth for the second team of a depth that fits one slab.
constexpr int LayerTeamStart(const int depth, const int tile_k, const int teams, const int team) {
  return team * LayerTeamSlabs(depth, tile_k, teams) * tile_k;
}

// How much of the depth is the team's
constexpr int LayerTeamDepth(const int depth, const int tile_k, const int teams, const int team) {
  const int left = depth - LayerTeamStart(depth, tile_k, teams, team), most = LayerTeamSlabs(depth, tile_k, teams) * tile_k;
  return (left < 0) ? 0 : (left > most ? most : left);
}

// Elements from an operand's first one to behind its last: `across` features or rows, and the WHOLE depth - of the product, the
// group or the K range. The end of a team's own part will not do: that part may begin behind the depth (see above), and lines
// that are short would be asked for beyond the operand.
constexpr long long LayerOperandElements(const bool k_contiguous, const int across, const int depth, const long long ld) {
  return k_contiguous ? (across - 1) * ld + depth : (depth - 1) * ld + across;
}

// Lines of a 1 KiB piece of a slab: k-contiguous lines hold 64 bytes, the others a tile's whole width
constexpr int LayerPieceLines(const bool k_contiguous, const int tile_width, const int element) {
  return k_contiguous ? 16 : 1024 / (tile_width * element);
}

}  // namespace clbh

#endif  // CLBLAST_HIP_KERNELS_LAYER_REQUESTS_HPP_
