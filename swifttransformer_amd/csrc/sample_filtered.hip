// A token for each row of float logits: temperature, then the k largest, of those the fewest that hold a share p of the weight, of those the
// ones with a share of the largest's weight, then the place of a given random number among them in the order of their indices.
//
//   w_i = e^((x_i - max) / temperature), in fixed point: units of 2^-44 of the largest.  Sums of such weights are whole numbers: they are
//   exact, so no result depends on the order in which lanes and atomics form them, and a border between two tokens lies
//   where 64-bit arithmetic puts it (to 2^-45 of the largest weight a token).
//   order: by value, the lower index first among equals.  kept: a beginning of that order (top k, then top p), then w_i >= min_p.
//   token: the first index, upwards, at which the kept weights' sum exceeds u times all of it.
//
// A workgroup a row.  Where the order is to be cut (after k tokens; where the sum reaches its share) a histogram over 2,048 steps of the
// value finds the step that holds the border; what lies in that step, if it is little, is ranked in LDS, else the step is divided
// again, by the values' bits, until it is little or one value.
#include "api.h"
#include "common.h"

namespace st {

constexpr int kBins = 2048, kFew = 512, kPlaces = 2048;
constexpr double kOne = 17592186044416.0;             // 2^44
constexpr float kSpan = 31.25f;                       // e^-31.25 of the largest is less than half a unit

// the beginning of a row's order: all that lie before (value, index), and that one
struct Cut { float v; int i; };
__device__ inline bool within(const Cut& c, float x, int i) { return x > c.v || (x == c.v && i <= c.i); }

// bits that order as the values do
__device__ inline uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Shared {
    uint64_t weight[kBins];                           // of a histogram's steps; sums of places
    uint32_t count[kBins];
    uint64_t wave_sum[16];
    float cand_x[kFew];
    int cand_i[kFew];
    uint64_t cand_w[kFew];
    uint64_t before, total;
    uint32_t bin, bin_count, key_low, key_high, n;
    Cut cut;
    float top[16];
    int top_i[16];
};

struct Row {
    const float* p;
    int vocab;
    float top, span;                                  // largest value; how far below it weights are not zero
    double temperature;
    __device__ float at(int i) const {
        const float x = p[i];
        return x != x ? -INFINITY : x;                // a NaN logit is never chosen
    }
    __device__ bool active(float x) const { return x == top || (x > -INFINITY && top - x <= span); }
    __device__ uint64_t weight(float x) const {
        if (x == top) return (uint64_t)1 << 44;
        return (uint64_t)(exp(((double)x - (double)top) / temperature) * kOne + 0.5);
    }
};

// sum over the threads up to and with one's own, and over all, of 64-bit numbers (1,024 threads)
__device__ inline uint64_t block_scan(uint64_t v, Shared& s, uint64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t a = (uint64_t)__shfl_up((unsigned long long)v, o, 64);
        if (lane >= o) v += a;
    }
    __syncthreads();
    if (lane == 63) s.wave_sum[wave] = v;
    __syncthreads();
    total = 0;
    uint64_t before = 0;
    for (int w = 0; w < 16; ++w) {
        if (w < wave) before += s.wave_sum[w];
        total += s.wave_sum[w];
    }
    return before + v;
}

// The place (of kPlaces, in s.weight) in which the running sum first reaches `target` (1 .. total): s.bin, and s.before, the sum
// before it.
__device__ inline void find_place(Shared& s, uint64_t own0, uint64_t upto, uint64_t own1, uint64_t target) {
    // this thread has places 2t and 2t + 1; upto: with both
    const uint64_t before = upto - own0 - own1;
    if (before < target && before + own0 >= target) {
        s.bin = 2 * threadIdx.x;
        s.before = before;
    } else if (before + own0 < target && upto >= target) {
        s.bin = 2 * threadIdx.x + 1;
        s.before = before + own0;
    }
    __syncthreads();
}

// Places in index order: [place * size, (place + 1) * size)
__device__ inline int place_size(int vocab) { return 256 * ((vocab + 256 * kPlaces - 1) / (256 * kPlaces)); }

// The index, upwards, at which the running sum of measure(x, i) first reaches target(total); a wave a place
template <typename F, typename G>
__device__ int index_reaching(const Row& row, Shared& s, F measure, G target_of) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, size = place_size(row.vocab);
    const int places = (row.vocab + size - 1) / size;
    __syncthreads();
    for (int pl = threadIdx.x; pl < kPlaces; pl += 1024)
        if (pl >= places) s.weight[pl] = 0;
    for (int pl = wave; pl < places; pl += 16) {
        uint64_t sum = 0;
        for (int j = 0; j < size; j += 64) {
            const int i = pl * size + j + lane;
            if (i < row.vocab) sum += measure(row.at(i), i);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += (uint64_t)__shfl_xor((unsigned long long)sum, o, 64);
        if (lane == 0) s.weight[pl] = sum;
    }
    __syncthreads();
    const uint64_t a = s.weight[2 * threadIdx.x], b = s.weight[2 * threadIdx.x + 1];
    uint64_t total;
    const uint64_t upto = block_scan(a + b, s, total);
    const uint64_t target = target_of(total);
    find_place(s, a, upto, b, target);
    if (wave == 0) {
        uint64_t before = s.before;
        for (int j = 0; j < size; j += 64) {
            const int i = s.bin * size + j + lane;
            uint64_t v = i < row.vocab ? measure(row.at(i), i) : 0;
            const uint64_t own = v;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint64_t up = (uint64_t)__shfl_up((unsigned long long)v, o, 64);
                if (lane >= o) v += up;
            }
            if (before + v >= target && before + v - own < target) s.cut.i = i;
            before += (uint64_t)__shfl((unsigned long long)v, 63, 64);
        }
    }
    __syncthreads();
    return s.cut.i;
}

// Cuts the order where `cut` leaves it at the place where the measure (a token counts one, or its weight) first reaches k, or the
// share p of all that is there.
template <bool COUNT>
__device__ void cut_order(const Row& row, Shared& s, Cut& cut, uint64_t k, double p) {
    const auto measure = [&](float x) { return COUNT ? (uint64_t)1 : row.weight(x); };
    const float scale = fminf((float)kBins / row.span, 3.0e38f);
    uint64_t base = 0, target = 0;
    bool first = true;
    uint32_t low = 0, high = 0xffffffffu;
    const auto step_of = [&](float x) {
        if (first) return (int)fminf((row.top == x ? 0.f : row.top - x) * scale, (float)(kBins - 1));
        return (int)((uint64_t)(high - ordered(x)) * kBins / ((uint64_t)(high - low) + 1));
    };
    const auto in_zone = [&](float x, int i) {
        if (!row.active(x) || !within(cut, x, i)) return false;
        const uint32_t key = ordered(x);
        return first || (key >= low && key <= high);
    };
    for (;;) {
        __syncthreads();
        for (int b = threadIdx.x; b < kBins; b += 1024) {
            s.weight[b] = 0;
            s.count[b] = 0;
        }
        if (threadIdx.x == 0) {
            s.key_low = 0xffffffffu;
            s.key_high = 0;
            s.n = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < row.vocab; i += 1024) {
            const float x = row.at(i);
            if (!in_zone(x, i)) continue;
            const int b = step_of(x);
            atomicAdd(&s.count[b], 1u);
            if (!COUNT) atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)row.weight(x));
        }
        __syncthreads();
        const int b0 = 2 * threadIdx.x;
        const uint64_t m0 = COUNT ? s.count[b0] : s.weight[b0], m1 = COUNT ? s.count[b0 + 1] : s.weight[b0 + 1];
        uint64_t total;
        const uint64_t upto = block_scan(m0 + m1, s, total);
        if (first) {
            if (COUNT) {
                if (total <= k) return;               // (what is further down has no weight)
                target = k;
            } else {
                const double share = ceil(p * (double)total);
                target = share < 1.0 ? 1 : share >= (double)total ? total : (uint64_t)share;
            }
        }
        find_place(s, m0, upto, m1, target - base);
        const int bin = s.bin;
        base += s.before;
        if (s.count[bin] <= kFew) {
            for (int i = threadIdx.x; i < row.vocab; i += 1024) {
                const float x = row.at(i);
                if (!in_zone(x, i) || step_of(x) != bin) continue;
                const uint32_t at = atomicAdd(&s.n, 1u);
                s.cand_x[at] = x;
                s.cand_i[at] = i;
                s.cand_w[at] = measure(x);
            }
            __syncthreads();
            const int n = (int)s.n;
            if ((int)threadIdx.x < n) {
                const float x = s.cand_x[threadIdx.x];
                const int i = s.cand_i[threadIdx.x];
                uint64_t ahead = base;
                for (int j = 0; j < n; ++j)
                    if (s.cand_x[j] > x || (s.cand_x[j] == x && s.cand_i[j] < i)) ahead += s.cand_w[j];
                if (ahead < target && ahead + s.cand_w[threadIdx.x] >= target) s.cut = Cut{x, i};
            }
            __syncthreads();
            cut = s.cut;
            return;
        }
        for (int i = threadIdx.x; i < row.vocab; i += 1024) {
            const float x = row.at(i);
            if (!in_zone(x, i) || step_of(x) != bin) continue;
            atomicMin(&s.key_low, ordered(x));
            atomicMax(&s.key_high, ordered(x));
        }
        __syncthreads();
        low = s.key_low;
        high = s.key_high;
        first = false;
        if (low == high) break;
    }
    // equals: the lower indices of them
    const float v = __uint_as_float(low & 0x80000000u ? low & 0x7fffffffu : ~low);
    const uint64_t each = measure(v), wanted = (target - base + each - 1) / each;
    const Cut from = cut;
    const int i = index_reaching(row, s, [&](float x, int j) { return (uint64_t)(x == v && within(from, x, j)); }, [&](uint64_t) { return wanted; });
    cut = Cut{v, i};
}

__global__ __launch_bounds__(1024) void sample_filtered_kernel(int* __restrict__ out, const float* __restrict__ logits, int64_t row_stride, int vocab,
                                                               const float* __restrict__ uniforms, const float* __restrict__ temperature,
                                                               const int* __restrict__ top_k, const float* __restrict__ top_p,
                                                               const float* __restrict__ min_p) {
    __shared__ Shared s;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Row row;
    row.p = logits + r * row_stride;
    row.vocab = vocab;
    float best = -INFINITY;
    int best_i = 0x7fffffff;
    for (int i = threadIdx.x; i < vocab; i += 1024) {
        const float x = row.at(i);
        if (x > best || (x == best && i < best_i)) { best = x; best_i = i; }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float x = __shfl_xor(best, o, 64);
        const int i = __shfl_xor(best_i, o, 64);
        if (x > best || (x == best && i < best_i)) { best = x; best_i = i; }
    }
    if (lane == 0) { s.top[wave] = best; s.top_i[wave] = best_i; }
    __syncthreads();
    for (int w = 0; w < 16; ++w)
        if (s.top[w] > best || (s.top[w] == best && s.top_i[w] < best_i)) { best = s.top[w]; best_i = s.top_i[w]; }
    const float t = temperature[r];
    const int k = top_k ? top_k[r] : 0;
    const float p = top_p ? top_p[r] : 1.f;
    if (!(t > 0.f) || k == 1 || !(p > 0.f) || best == -INFINITY) {
        if (threadIdx.x == 0) out[r] = best_i;
        return;
    }
    row.top = best;
    row.temperature = (double)t;
    row.span = best < INFINITY ? kSpan * t : -1.f;   // (beside an infinity nothing else has weight)
    Cut cut{-INFINITY, vocab};
    if (k > 0 && k < vocab) cut_order<true>(row, s, cut, (uint64_t)k, 0.0);
    if (p < 1.f) cut_order<false>(row, s, cut, 0, (double)p);
    const double least = min_p ? (double)fminf(min_p[r], 1.f) * kOne : 0.0;
    const float u = uniforms[r];
    const int token = index_reaching(row, s, [&](float x, int i) {
        if (!row.active(x) || !within(cut, x, i)) return (uint64_t)0;
        const uint64_t w = row.weight(x);
        return (double)w >= least ? w : 0;
    }, [&](uint64_t total) {
        const double at = (double)u * (double)total;
        const uint64_t below = at > 0.0 ? (at < (double)total ? (uint64_t)at : total - 1) : 0;      // (a u that is none of [0, 1) is drawn to its end)
        return min(below, total - 1) + 1;
    });
    if (threadIdx.x == 0) out[r] = token;
}

}  // namespace st

using namespace st;

extern "C" int st_sample_filtered(int* out, const float* logits, int64_t row_stride, int num_rows, int vocab, const float* uniforms,
                                  const float* temperature, const int* top_k, const float* top_p, const float* min_p, hipStream_t stream) {
    ST_CHECK(num_rows >= 0 && vocab > 0 && row_stride >= vocab, "sample_filtered: bad sizes rows=%d vocab=%d", num_rows, vocab);
    ST_CHECK(vocab <= 1 << 18, "sample_filtered: %d logits a row (at most %d: sums of weights are 64-bit numbers)", vocab, 1 << 18);
    if (num_rows == 0) return 0;
    ST_CHECK(out && logits && uniforms && temperature, "sample_filtered: null operand");
    sample_filtered_kernel<<<num_rows, 1024, 0, stream>>>(out, logits, row_stride, vocab, uniforms, temperature, top_k, top_p, min_p);
    ST_LAUNCH_CHECK("sample_filtered");
    return 0;
}
