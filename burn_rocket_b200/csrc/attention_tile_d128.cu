// attention_tile_d128.cu — attention_tile.cuh at head_dim 128.
#include "attention_tile.cuh"

namespace rb {
namespace tile {
int launch_d128(const CUtensorMap* tm, const TileParams& p, const Work& w, cudaStream_t st) {
  return launch_types<128>(tm, p, w, st);
}
}  // namespace tile
}  // namespace rb
