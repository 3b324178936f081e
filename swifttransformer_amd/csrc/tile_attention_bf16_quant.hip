// csrc/tile_attention.h for bfloat16 queries over the 8-bit cache.
#include "tile_attention.h"

namespace st {
int tile_attention_bf16_quant(const StTileAttention& p, hipStream_t stream) { return launch_tiles_by_head<bf16_t, e4m3_t, 2>(p, stream); }
}  // namespace st
