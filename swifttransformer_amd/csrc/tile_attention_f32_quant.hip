// csrc/tile_attention.h for float queries over the 8-bit cache, on the float matrix instruction.
#include "tile_attention.h"

namespace st {
int tile_attention_f32_quant(const StTileAttention& p, hipStream_t stream) { return launch_tiles_by_head<float, e4m3_t, 1>(p, stream); }
}  // namespace st
