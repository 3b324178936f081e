// Keys and values into the 8-bit paged cache, and entries of it back into the storage type (csrc/small_float.h has the format).
//
// What bounds both: memory.  A token's head is read once, its largest magnitude found by moves between the lanes that hold it, and written
// once.  A lane holds eight elements: 16 bytes of bfloat16 (two loads of 16 in float), 8 bytes in e4m3.
#include "api.h"
#include "small_float.h"

namespace st {

template <typename T> __device__ inline void load8(const T* p, float* x);
template <> __device__ inline void load8<bf16_t>(const bf16_t* p, float* x) { Elem<bf16_t>::load_vec(p, x); }
template <> __device__ inline void load8<float>(const float* p, float* x) {
    Elem<float>::load_vec(p, x);
    Elem<float>::load_vec(p + 4, x + 4);
}

// LG lanes share a token's head (LG * 8 >= head_dim); blockIdx.y: keys or values.  A token whose page is none of the pool's, or that
// has no item or position, is left out.
template <typename T, int LG>
__global__ __launch_bounds__(256) void quant_write_kernel(
    uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, int64_t page_stride, uint8_t* __restrict__ k_exp, uint8_t* __restrict__ v_exp,
    int64_t exp_stride, const T* __restrict__ k_src, const T* __restrict__ v_src, int64_t src_stride, const int* __restrict__ token_item,
    const int* __restrict__ positions, const int* __restrict__ block_table, int num_items, int max_pages, int page_size, int num_pages,
    int num_tokens, int num_kv_heads, int head_dim) {
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LG;        // token * heads + head
    const int d = (threadIdx.x % LG) * 8;
    const int64_t t = unit / num_kv_heads;
    const int h = (int)(unit - t * num_kv_heads);
    if (t >= num_tokens) return;                                               // (all lanes of a group alike)
    const int item = token_item[t], pos = positions[t];
    if (item < 0 || item >= num_items || pos < 0) return;
    const int pi = pos / page_size, row = pos - pi * page_size;
    if (pi >= max_pages) return;
    const int page = block_table[(int64_t)item * max_pages + pi];
    if (page < 0 || page >= num_pages) return;
    const bool here = d < head_dim;
    float x[8];
    load8<T>((blockIdx.y ? v_src : k_src) + t * src_stride + (int64_t)h * head_dim + (here ? d : 0), x);
    uint32_t big = 0;                                                          // largest finite magnitude: its bits order as it does
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
        big = max(big, u < 0x7f800000u ? u : 0u);
    }
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o, 64));
    const int e = unit_exponent(big);
    const float inverse = __uint_as_float((uint32_t)(254 - e) << 23);          // 2^(127 - e)
    if (here) {
        uint2 out;
        out.x = pack_e4m3x4(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse);
        out.y = pack_e4m3x4(x[4] * inverse, x[5] * inverse, x[6] * inverse, x[7] * inverse);
        *reinterpret_cast<uint2*>((blockIdx.y ? v_cache : k_cache) + (int64_t)page * page_stride + ((int64_t)h * page_size + row) * head_dim + d) = out;
    }
    if (d == 0) (blockIdx.y ? v_exp : k_exp)[(int64_t)page * exp_stride + (int64_t)h * page_size + row] = (uint8_t)e;
}

// the entries of tokens, back in the storage type: [tokens, heads * head_dim]; zeros for a token that quant_write_kernel would leave out
template <typename T>
__global__ __launch_bounds__(256) void quant_read_kernel(
    T* __restrict__ k_out, T* __restrict__ v_out, const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, int64_t page_stride,
    const uint8_t* __restrict__ k_exp, const uint8_t* __restrict__ v_exp, int64_t exp_stride, const int* __restrict__ token_item,
    const int* __restrict__ positions, const int* __restrict__ block_table, int num_items, int max_pages, int page_size, int num_pages,
    int num_tokens, int num_kv_heads, int head_dim) {
    const int per = head_dim / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t unit = i / per, t = unit / num_kv_heads;
    if (t >= num_tokens) return;
    const int d = (int)(i - unit * per) * 8, h = (int)(unit - t * num_kv_heads);
    const int item = token_item[t], pos = positions[t];
    int page = -1, row = 0;
    if (item >= 0 && item < num_items && pos >= 0) {
        const int pi = pos / page_size;
        row = pos - pi * page_size;
        if (pi < max_pages) page = block_table[(int64_t)item * max_pages + pi];
    }
    uint2 v = make_uint2(0, 0);
    float unit_of = 1.f;
    if (page >= 0 && page < num_pages) {
        v = *reinterpret_cast<const uint2*>((blockIdx.y ? v_cache : k_cache) + (int64_t)page * page_stride + ((int64_t)h * page_size + row) * head_dim + d);
        unit_of = __uint_as_float((uint32_t)(blockIdx.y ? v_exp : k_exp)[(int64_t)page * exp_stride + (int64_t)h * page_size + row] << 23);
    }
    float x[8];
    const float2v a = e4m3x2_to_floats<false>(v.x), b = e4m3x2_to_floats<true>(v.x), c = e4m3x2_to_floats<false>(v.y), f = e4m3x2_to_floats<true>(v.y);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = f.x; x[7] = f.y;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= unit_of;
    T* out = (blockIdx.y ? v_out : k_out) + unit * head_dim + d;
    Elem<T>::store_vec(out, x);
    if (sizeof(T) == 4) Elem<T>::store_vec(out + 4, x + 4);
}

static int check_quant(const char* what, int num_tokens, int num_items, int max_pages, int page_size, int num_pages, int num_kv_heads, int head_dim,
                       int64_t page_stride, int64_t exp_stride, int dtype) {
    ST_CHECK(num_tokens >= 0 && num_items > 0 && max_pages > 0 && page_size > 0 && num_pages > 0 && num_kv_heads > 0, "%s: bad sizes", what);
    ST_CHECK(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 256, "%s: head_dim %d is no multiple of 16 up to 256", what, head_dim);
    ST_CHECK(page_stride >= (int64_t)num_kv_heads * page_size * head_dim && page_stride % 16 == 0,
             "%s: page stride %lld is smaller than a page or no multiple of 16", what, (long long)page_stride);
    ST_CHECK(exp_stride >= (int64_t)num_kv_heads * page_size, "%s: a page's exponents overlap the next page's", what);
    ST_CHECK(dtype == kF32 || dtype == kBF16, "%s: unknown dtype %d", what, dtype);
    // (elements, over which a thread's index runs)
    ST_CHECK((int64_t)num_tokens * num_kv_heads * head_dim <= (int64_t)1 << 36, "%s: too many tokens at once", what);
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
    const dim3 grid((unsigned)((groups * lg + 255) / 256), 2);
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
    const dim3 grid((unsigned)(((int64_t)num_tokens * num_kv_heads * (head_dim / 8) + 255) / 256), 2);
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
