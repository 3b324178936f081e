// csrc/tile_attention.h for bfloat16 queries over a bfloat16 cache, and its C entry.
#include "tile_attention.h"

namespace st {
int tile_attention_bf16(const StTileAttention& p, hipStream_t stream) { return launch_tiles_by_head<bf16_t, bf16_t, 2>(p, stream); }
}  // namespace st

using namespace st;

extern "C" int st_tile_attention(const StTileAttention* args, hipStream_t stream) {
    ST_CHECK(args, "attention: null arguments");
    const StTileAttention& p = *args;
    ST_CHECK(p.num_rows >= 0 && p.num_entries >= 0 && p.num_tiles >= 0 && p.num_groups >= 0 && p.num_shared >= 0 && p.heads > 0 && p.kv_heads > 0 &&
             p.page_size > 0 && p.max_pages > 0 && p.num_pages > 0 && p.num_items > 0, "attention: bad sizes");
    ST_CHECK(p.heads % p.kv_heads == 0, "attention: %d query heads do not divide into %d key heads", p.heads, p.kv_heads);
    ST_CHECK(p.head_dim > 0 && p.head_dim % 16 == 0 && p.head_dim <= 256, "attention: head_dim %d is no multiple of 16 up to 256", p.head_dim);
    // (keys are counted by ints, up to two rounds of the waves' blocks, 128 keys each, past the last one)
    ST_CHECK((int64_t)p.max_pages * p.page_size <= 0x7fffffff - 512, "attention: a block table of close to 2^31 positions or more");
    ST_CHECK(p.dtype == kF32 || p.dtype == kBF16, "attention: unknown dtype %d", p.dtype);
    ST_CHECK(p.cache_dtype == p.dtype || p.cache_dtype == 2, "attention: a cache of type %d under queries of type %d", p.cache_dtype, p.dtype);
    const int elem = p.cache_dtype == 2 ? 1 : p.dtype == kF32 ? 4 : 2;
    ST_CHECK(p.page_stride >= (int64_t)p.kv_heads * p.page_size * p.head_dim && p.page_stride * elem % 16 == 0 && p.page_stride < 0x7fffffff,
             "attention: page stride %lld is smaller than a page, unaligned or too large", (long long)p.page_stride);
    ST_CHECK(p.cache_dtype != 2 || (p.k_exp && p.v_exp && p.exp_stride >= (int64_t)p.kv_heads * p.page_size), "attention: an 8-bit cache needs its exponents");
    ST_CHECK(p.cache_dtype == 2 || p.num_groups > 0, "attention: single tokens and tiles over a cache of the queries' type have kernels of their own");
    ST_CHECK(p.num_groups == 0 ? !p.row_start : p.row_start && p.shared_rows && p.num_shared > 0 && p.group_off && p.num_tiles == 0 && !p.row_ids,
             "attention: shared prefixes need their lists, and rows that start behind one need the prefixes");
    ST_CHECK(p.num_tiles == 0 || (p.tile_rows > 0 && p.tile_rows <= 65536 && p.tile_item && p.tile_q0 && p.item_tok_off && p.item_start && p.item_len),
             "attention: tiles need their lists");
    ST_CHECK(p.own_waves == 4 || (p.own_waves == 1 && p.num_tiles == 0), "attention: %d waves a row (4, or 1 without tiles)", p.own_waves);
    ST_CHECK(p.own_splits >= 1 && (p.num_groups == 0 ? p.shared_splits == 0 : p.shared_splits >= 1) && p.slots == p.own_splits + p.shared_splits && p.slots <= 64,
             "attention: %d and %d splits of the keys in %d places (at most 64)", p.own_splits, p.shared_splits, p.slots);
    if (p.num_rows == 0 || (p.num_entries == 0 && p.num_tiles == 0)) return 0;
    ST_CHECK(p.out && p.q && (p.slots == 1 || (p.part_o && p.part_ml)), "attention: null operand");
    ST_CHECK(((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k_cache) | reinterpret_cast<uintptr_t>(p.v_cache) |
               reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.part_o)) & 15) == 0 && p.q_stride * (p.dtype == kF32 ? 4 : 2) % 16 == 0,
             "attention: queries, their rows, caches and results must be 16-byte aligned");
    if (p.cache_dtype == 2) return p.dtype == kBF16 ? tile_attention_bf16_quant(p, stream) : tile_attention_f32_quant(p, stream);
    return p.dtype == kBF16 ? tile_attention_bf16(p, stream) : tile_attention_f32(p, stream);
}
