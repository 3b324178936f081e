// Keys and values into the 8-bit paged cache, and entries of it back into the storage type (csrc/small_float.h has the format).
//
// What bounds both: memory.  A token's head is read once, its largest magnitude found by moves between the lanes that hold it, and written
// once.  A lane holds eight elements of a key and of a value: 16 bytes each of bfloat16 (two loads of 16 in float), 8 bytes in e4m3.  2,047 tokens of 40
// heads of 128: written in 16 us and read back in 13, 126 MB at 4.3 TB/s (17 and 16 with a thread for either, and 64-bit indices).
#include "api.h"
#include "small_float.h"

namespace st {

template <typename T> __device__ inline void load8(const T* p, float* x);
template <> __device__ inline void load8<bf16_t>(const bf16_t* p, float* x) { Elem<bf16_t>::load_vec(p, x); }
template <> __device__ inline void load8<float>(const float* p, float* x) {
    Elem<float>::load_vec(p, x);
    Elem<float>::load_vec(p + 4, x + 4);
}

// eight elements in e4m3, the group's exponent e: LG lanes hold a head between them
template <int LG> __device__ inline uint2 quantise8(const float* x, int& e) {
    uint32_t big = 0;                                                          // largest finite magnitude: its bits order as it does
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
        big = max(big, u < 0x7f800000u ? u : 0u);
    }
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o, 64));
    e = unit_exponent(big);
    const float inverse = __uint_as_float((uint32_t)(254 - e) << 23);          // 2^(127 - e)
    return make_uint2(pack_e4m3x4(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse),
                      pack_e4m3x4(x[4] * inverse, x[5] * inverse, x[6] * inverse, x[7] * inverse));
}

template <typename T> __device__ inline void restore8(uint2 v, uint32_t e, T* out) {
    const float unit_of = __uint_as_float(e << 23);
    const float2v a = e4m3x2_to_floats<false>(v.x), b = e4m3x2_to_floats<true>(v.x), c = e4m3x2_to_floats<false>(v.y), f = e4m3x2_to_floats<true>(v.y);
    float x[8] = {a.x, a.y, b.x, b.y, c.x, c.y, f.x, f.y};
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= unit_of;
    Elem<T>::store_vec(out, x);
    if (sizeof(T) == 4) Elem<T>::store_vec(out + 4, x + 4);
}

// The token's page, -1 where it has no item or position or the page is none of the pool's; its row there
__device__ inline int page_of(int item, int pos, const int* block_table, int num_items, int max_pages, int page_size, int num_pages, int& row) {
    row = 0;
    if (item < 0 || item >= num_items || pos < 0) return -1;
    const int pi = pos / page_size;
    row = pos - pi * page_size;
    if (pi >= max_pages) return -1;
    const int page = block_table[(int64_t)item * max_pages + pi];
    return page < num_pages ? page : -1;
}

// LG lanes share a token's head (LG * 8 >= head_dim), its keys and its values: one look at the table for both, both sources' loads under
// way during it.  A token that page_of has no page for is left out.
template <typename T, int LG>
__global__ __launch_bounds__(256) void quant_write_kernel(
    uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, int64_t page_stride, uint8_t* __restrict__ k_exp, uint8_t* __restrict__ v_exp,
    int64_t exp_stride, const T* __restrict__ k_src, const T* __restrict__ v_src, int64_t src_stride, const int* __restrict__ token_item,
    const int* __restrict__ positions, const int* __restrict__ block_table, int num_items, int max_pages, int page_size, int num_pages,
    int num_tokens, int num_kv_heads, int head_dim) {
    const uint32_t unit = (blockIdx.x * 256u + threadIdx.x) / LG, t = unit / (uint32_t)num_kv_heads;         // unit: token * heads + head
    const int d = (threadIdx.x % LG) * 8, h = (int)(unit - t * (uint32_t)num_kv_heads);
    if (t >= (uint32_t)num_tokens) return;                                     // (all lanes of a group alike)
    const bool here = d < head_dim;
    const int64_t from = (int64_t)t * src_stride + h * head_dim + (here ? d : 0);
    const int item = token_item[t], pos = positions[t];
    float k[8], v[8];
    load8<T>(k_src + from, k);
    load8<T>(v_src + from, v);
    int row, ke, ve;
    const int page = page_of(item, pos, block_table, num_items, max_pages, page_size, num_pages, row);
    if (page < 0) return;
    const uint2 kq = quantise8<LG>(k, ke), vq = quantise8<LG>(v, ve);
    const int64_t at = (int64_t)page * page_stride + ((int64_t)h * page_size + row) * head_dim + d;
    if (here) {
        *reinterpret_cast<uint2*>(k_cache + at) = kq;
        *reinterpret_cast<uint2*>(v_cache + at) = vq;
    }
    if (d == 0) {
        const int64_t to = (int64_t)page * exp_stride + (int64_t)h * page_size + row;
        k_exp[to] = (uint8_t)ke;
        v_exp[to] = (uint8_t)ve;
    }
}

// the entries of tokens, back in the storage type: [tokens, heads * head_dim]; zeros for a token that quant_write_kernel would leave out
template <typename T>
__global__ __launch_bounds__(256) void quant_read_kernel(
    T* __restrict__ k_out, T* __restrict__ v_out, const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, int64_t page_stride,
    const uint8_t* __restrict__ k_exp, const uint8_t* __restrict__ v_exp, int64_t exp_stride, const int* __restrict__ token_item,
    const int* __restrict__ positions, const int* __restrict__ block_table, int num_items, int max_pages, int page_size, int num_pages,
    int num_tokens, int num_kv_heads, int head_dim) {
    const uint32_t per = (uint32_t)head_dim / 8u, i = blockIdx.x * 256u + threadIdx.x, unit = i / per, t = unit / (uint32_t)num_kv_heads;
    if (t >= (uint32_t)num_tokens) return;
    const int d = (int)(i - unit * per) * 8, h = (int)(unit - t * (uint32_t)num_kv_heads);
    int row;
    const int page = page_of(token_item[t], positions[t], block_table, num_items, max_pages, page_size, num_pages, row);
    uint2 k = make_uint2(0, 0), v = make_uint2(0, 0);
    uint32_t ke = 127, ve = 127;
    if (page >= 0) {
        const int64_t entry = (int64_t)h * page_size + row, at = (int64_t)page * page_stride + entry * head_dim + d, e = (int64_t)page * exp_stride + entry;
        k = *reinterpret_cast<const uint2*>(k_cache + at);
        v = *reinterpret_cast<const uint2*>(v_cache + at);
        ke = k_exp[e];
        ve = v_exp[e];
    }
    const int64_t to = (int64_t)unit * head_dim + d;
    restore8<T>(k, ke, k_out + to);
    restore8<T>(v, ve, v_out + to);
}

static int check_quant(const char* what, int num_tokens, int num_items, int max_pages, int page_size, int num_pages, int num_kv_heads, int head_dim,
                       int64_t page_stride, int64_t exp_stride, int dtype) {
    ST_CHECK(num_tokens >= 0 && num_items > 0 && max_pages > 0 && page_size > 0 && num_pages > 0 && num_kv_heads > 0, "%s: bad sizes", what);
    ST_CHECK(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 256, "%s: head_dim %d is no multiple of 16 up to 256", what, head_dim);
    ST_CHECK(page_stride >= (int64_t)num_kv_heads * page_size * head_dim && page_stride % 16 == 0,
             "%s: page stride %lld is smaller than a page or no multiple of 16", what, (long long)page_stride);
    ST_CHECK(exp_stride >= (int64_t)num_kv_heads * page_size, "%s: a page's exponents overlap the next page's", what);
    ST_CHECK(dtype == kF32 || dtype == kBF16, "%s: unknown dtype %d", what, dtype);
    // (a thread's index has 32 bits; up to 32 threads hold 144 elements)
    ST_CHECK((int64_t)num_tokens * num_kv_heads * head_dim <= (int64_t)1 << 33, "%s: too many tokens at once", what);
    return 0;
}

template <typename T>
static int launch_quant_write(void* k_cache, void* v_cache, int64_t page_stride, void* k_exp, void* v_exp, int64_t exp_stride, const void* k_src,
                              const void* v_src, int64_t src_stride, const int* token_item, const int* positions, const int* block_table,
                              int num_items, int max_pages, int page_size, int num_pages, int num_tokens, int num_kv_heads, int head_dim,
                              hipStream_t stream) {
    int lg = 2;
    while (lg * 8 < head_dim) lg <<= 1;
    const int64_t groups = (int64_t)num_tokens * num_kv_heads;
    const dim3 grid((unsigned)((groups * lg + 255) / 256));
#define ST_QW(L) quant_write_kernel<T, L><<<grid, 256, 0, stream>>>((uint8_t*)k_cache, (uint8_t*)v_cache, page_stride, (uint8_t*)k_exp, (uint8_t*)v_exp, \
        exp_stride, (const T*)k_src, (const T*)v_src, src_stride, token_item, positions, block_table, num_items, max_pages, page_size, num_pages, \
        num_tokens, num_kv_heads, head_dim)
    switch (lg) {
        case 2: ST_QW(2); break;
        case 4: ST_QW(4); break;
        case 8: ST_QW(8); break;
        case 16: ST_QW(16); break;
        default: ST_QW(32); break;
    }
#undef ST_QW
    ST_LAUNCH_CHECK("quant_kv_write");
    return 0;
}

}  // namespace st

using namespace st;

extern "C" int st_quant_kv_write(void* k_cache, void* v_cache, int64_t page_stride, void* k_exp, void* v_exp, int64_t exp_stride, const void* k_src,
                                 const void* v_src, int64_t src_stride, const int* token_item, const int* positions, const int* block_table,
                                 int num_items, int max_pages, int page_size, int num_pages, int num_tokens, int num_kv_heads, int head_dim, int dtype,
                                 hipStream_t stream) {
    if (check_quant("quant_kv_write", num_tokens, num_items, max_pages, page_size, num_pages, num_kv_heads, head_dim, page_stride, exp_stride, dtype)) return 1;
    const int per16 = dtype == kF32 ? 4 : 8;
    ST_CHECK(src_stride % per16 == 0 && ((reinterpret_cast<uintptr_t>(k_src) | reinterpret_cast<uintptr_t>(v_src) |
             reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0,
             "quant_kv_write: sources and caches must be 16-byte aligned, rows of the sources too");
    if (num_tokens == 0) return 0;
    return (dtype == kF32 ? launch_quant_write<float> : launch_quant_write<bf16_t>)(
        k_cache, v_cache, page_stride, k_exp, v_exp, exp_stride, k_src, v_src, src_stride, token_item, positions, block_table, num_items, max_pages,
        page_size, num_pages, num_tokens, num_kv_heads, head_dim, stream);
}

extern "C" int st_quant_kv_read(void* k_out, void* v_out, const void* k_cache, const void* v_cache, int64_t page_stride, const void* k_exp,
                                const void* v_exp, int64_t exp_stride, const int* token_item, const int* positions, const int* block_table,
                                int num_items, int max_pages, int page_size, int num_pages, int num_tokens, int num_kv_heads, int head_dim, int dtype,
                                hipStream_t stream) {
    if (check_quant("quant_kv_read", num_tokens, num_items, max_pages, page_size, num_pages, num_kv_heads, head_dim, page_stride, exp_stride, dtype)) return 1;
    ST_CHECK(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out) | reinterpret_cast<uintptr_t>(k_cache) |
               reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0, "quant_kv_read: caches and results must be 16-byte aligned");
    if (num_tokens == 0) return 0;
    const dim3 grid((unsigned)(((int64_t)num_tokens * num_kv_heads * (head_dim / 8) + 255) / 256));
    if (dtype == kF32)
        quant_read_kernel<float><<<grid, 256, 0, stream>>>((float*)k_out, (float*)v_out, (const uint8_t*)k_cache, (const uint8_t*)v_cache, page_stride,
            (const uint8_t*)k_exp, (const uint8_t*)v_exp, exp_stride, token_item, positions, block_table, num_items, max_pages, page_size, num_pages,
            num_tokens, num_kv_heads, head_dim);
    else
        quant_read_kernel<bf16_t><<<grid, 256, 0, stream>>>((bf16_t*)k_out, (bf16_t*)v_out, (const uint8_t*)k_cache, (const uint8_t*)v_cache, page_stride,
            (const uint8_t*)k_exp, (const uint8_t*)v_exp, exp_stride, token_item, positions, block_table, num_items, max_pages, page_size, num_pages,
            num_tokens, num_kv_heads, head_dim);
    ST_LAUNCH_CHECK("quant_kv_read");
    return 0;
}
