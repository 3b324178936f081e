// csrc/tile_attention.h for float queries over a float cache, on the float matrix instruction.
#include "tile_attention.h"

namespace st {
int tile_attention_f32(const StTileAttention& p, hipStream_t stream) { return launch_tiles_by_head<float, float, 1>(p, stream); }
}  // namespace st
