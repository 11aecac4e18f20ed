// Host-only replay of the requests with which the tiled kernel of the layer products (clblast_amd/csrc/kernels/layer_gemm.hpp)
// fetches an operand, over the functions that it takes its ranges from (kernels/layer_requests.hpp): both layouts, both
// sizes of elements, one and two teams of wavefronts, tight and padded lines. Whatever passes the range check lies inside the operand
// (to whole dwords: the check works per dword), and every element that enters a product is fetched, by the team that walks it.
// Compiled and run by tests/test_layer_limits_cpu.py.
#include <algorithm>
#include <cstdio>
#include <initializer_list>
#include <vector>

#include "kernels/layer_requests.hpp"

namespace {
long long violations = 0, cases = 0, requests = 0;

struct Case { int element, tile, teams, across, depth; bool kc; long long ld; };

void Violation(const char* what, const Case& c, const int team) {
  if (++violations <= 20) {
    std::printf("VIOLATION %s: element %d tile %d team %d of %d across %d depth %d %s ld %lld\n", what, c.element, c.tile, team, c.teams,
                c.across, c.depth, c.kc ? "k-contiguous" : "x-contiguous", c.ld);
  }
}

// The kernel's HRecordsUpTo: bytes between two places, in whole dwords, as an unsigned 32-bit number
long long Records(const long long from, const long long end) {
  const long long bytes = (end - from + 3) & ~3ll;
  return bytes < 0 ? 0 : std::min(bytes, 0xffffffffll);
}

void Check(const Case& c) {
  ++cases;
  const int tile_k = 64 / c.element, pieces = c.tile / 16, lines = clbh::LayerPieceLines(c.kc, c.tile, c.element), chunks = 64 / lines;
  const long long elements = c.kc ? (c.across - 1) * c.ld + c.depth : (c.depth - 1) * c.ld + c.across;  // (the operand, by its layout)
  const long long reach = (elements * c.element + 3) / 4 * 4;
  const long long end = clbh::LayerOperandElements(c.kc, c.across, c.depth, c.ld) * c.element;
  const int slabs = clbh::LayerTeamSlabs(c.depth, tile_k, c.teams);
  int walked = 0;
  for (int team = 0; team < c.teams; ++team) {
    const int start = clbh::LayerTeamStart(c.depth, tile_k, c.teams, team), mine = clbh::LayerTeamDepth(c.depth, tile_k, c.teams, team);
    if (mine > 0 && start != walked) { Violation("the teams' parts are not one behind the other", c, team); }
    walked += mine;
    for (int x0 = 0; x0 < c.across; x0 += c.tile) {
      std::vector<char> fetched(static_cast<size_t>(c.tile) * tile_k);
      const bool whole = x0 + c.tile <= c.across && c.depth % (c.teams * tile_k) == 0;  // (then nothing is range-checked)
      for (int slab = 0; slab < slabs; ++slab) {
        std::fill(fetched.begin(), fetched.end(), 0);
        const long long k0 = start + static_cast<long long>(slab) * tile_k;
        const long long tile_at = (c.kc ? x0 * c.ld + k0 : k0 * c.ld + x0) * c.element;
        for (int piece = 0; piece < pieces; ++piece) {
          const long long source = tile_at + static_cast<long long>(lines) * piece * c.ld * c.element;
          const long long records = whole ? 0xffffffffll : Records(source, end);
          for (int line = 0; line < lines; ++line) {
            for (int chunk = 0; chunk < chunks; ++chunk) {
              for (int dword = 0; dword < 4; ++dword) {
                const long long offset = line * c.ld * c.element + 16 * chunk + 4 * dword;
                if (offset + 4 > records) { continue; }
                ++requests;
                if (source + offset < 0 || source + offset + 4 > reach) { Violation("a request leaves the operand", c, team); return; }
                for (int part = 0; part < 4 / c.element; ++part) {
                  const int along = (16 * chunk + 4 * dword) / c.element + part, across = lines * piece + line;
                  fetched[c.kc ? static_cast<size_t>(across) * tile_k + along : static_cast<size_t>(along) * tile_k + across] = 1;
                }
              }
            }
          }
        }
        for (int x = 0; x < c.tile && x0 + x < c.across; ++x) {
          for (int k = 0; k < tile_k && slab * tile_k + k < mine; ++k) {
            if (!fetched[static_cast<size_t>(x) * tile_k + k]) { Violation("an element is not fetched", c, team); return; }
          }
        }
      }
    }
  }
  if (walked != c.depth) { Violation("the teams do not walk the depth", c, 0); }
}
}  // namespace

int main() {
  for (const int element : {2, 4})
  for (const int teams : {1, 2})
  for (const int tile : {32, 64, 128, 256}) {
    if (teams == 2 && tile != 64) { continue; }  // (the one tile that has two)
    for (const int across : {1, 2, 15, 17, 63, 64, 65, 130, 256})
    for (int depth = 1; depth <= 200; depth += (depth < 34 || depth % 32 > 28 || depth % 32 < 3) ? 1 : 9)
    for (const bool kc : {false, true}) {
      const long long line = kc ? depth : across;
      for (const long long pad : {0ll, 1ll, 2ll, 31ll, 66ll}) {
        // (16-bit operands whose lines do not start at dwords are copied first, to lines of a multiple of eight elements)
        Check({element, tile, teams, across, depth, kc, (element == 2 && (line + pad) % 2 != 0) ? (line + 7) / 8 * 8 : line + pad});
      }
    }
  }
  std::printf("cases %lld requests %lld violations %lld\n", cases, requests, violations);
  return violations == 0 ? 0 : 1;
}
