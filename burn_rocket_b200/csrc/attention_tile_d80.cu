// attention_tile_d80.cu — attention_tile.cuh at head_dim 72, staged as 80
// columns (packed sequences only).
#include "attention_tile.cuh"

namespace rb {
namespace tile {
int launch_d80(const CUtensorMap* tm, const TileParams& p, const Work& w, cudaStream_t st) {
  return launch_types<80>(tm, p, w, st);
}
}  // namespace tile
}  // namespace rb
