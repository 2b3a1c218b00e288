// attention_tile_d80.cu — attention_tile.cuh at head_dim 72, staged as 80
// columns (packed sequences only).
#include "attention_tile.cuh"

namespace rb {
namespace tile {
int launch_d80(const CUtensorMap* tm, const TileParams& p, unsigned grid, int ranks, cudaStream_t st) {
  return ranks > 1 ? launch_types<80, true>(tm, p, grid, ranks, st) : launch_types<80, false>(tm, p, grid, 1, st);
}
}  // namespace tile
}  // namespace rb
