// attention_tile_d128.cu — attention_tile.cuh at head_dim 128.
#include "attention_tile.cuh"

namespace rb {
namespace tile {
int launch_d128(const CUtensorMap* tm, const TileParams& p, unsigned grid, int ranks, cudaStream_t st) {
  return ranks > 1 ? launch_types<128, true>(tm, p, grid, ranks, st) : launch_types<128, false>(tm, p, grid, 1, st);
}
}  // namespace tile
}  // namespace rb
