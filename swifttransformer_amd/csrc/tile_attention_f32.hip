// The float instances of csrc/tile_attention.h: both products on the float matrix instruction.
#include "tile_attention.h"

namespace st {
int tile_attention_f32(const StTileAttention& p, hipStream_t stream) { return launch_tiles_by_head<float, 2>(p, stream); }
}  // namespace st
