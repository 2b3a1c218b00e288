// attention_tile_d64.cu — attention_tile.cuh at head_dim 64.
#include "attention_tile.cuh"

namespace rb {
namespace tile {
int launch_d64(const CUtensorMap* tm, const TileParams& p, unsigned grid, int ranks, cudaStream_t st) {
  return ranks > 1 ? launch_types<64, true>(tm, p, grid, ranks, st) : launch_types<64, false>(tm, p, grid, 1, st);
}
}  // namespace tile
}  // namespace rb
