// attention_tile_d64.cu — attention_tile.cuh at head_dim 64.
#include "attention_tile.cuh"

namespace rb {
namespace tile {
int launch_d64(const CUtensorMap* tm, const TileParams& p, const Work& w, cudaStream_t st) {
  return launch_types<64>(tm, p, w, st);
}
}  // namespace tile
}  // namespace rb
