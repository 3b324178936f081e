// A token for each row of float logits: temperature, then the k largest, of those the fewest that hold a share p of the weight, of those the
// ones with a share of the largest's weight, then the place of a given random number among them in the order of their indices.
//
//   w_i = e^((x_i - max) / temperature), in fixed point: units of 2^-44 of the largest.  Sums of such weights are whole numbers: they are
//   exact, so no result depends on the order in which lanes and atomics form them, and a border between two tokens lies
//   where 64-bit arithmetic puts it (to 2^-44 of the largest weight a token).
//   order: by value, the lower index first among equals.  kept: a beginning of that order (top k, then top p), then w_i >= min_p.
//   token: the first index, upwards, at which the kept weights' sum exceeds u times all of it.
//
// A workgroup a row.  A pass goes over the row in memory (in the L2 from the second on), each wave over a stretch of its own, so that sums over
// waves are sums over stretches of indices.
//   top k    the k-th largest of the threads' largest is no larger than the k-th largest of all: a histogram of those 1,024 gives a line
//            above which little more than k logits lie.  They go to a list in LDS, and what is left to do is done there.
//   top p    (and a top k above 512) weights (or ones) are summed by 2,048 steps of the value.  The step that holds the border is known
//            then, and from the steps' weights how many there are up to it; if they are few they go to the list, else the pass that sums
//            weights for the draw leaves out that step and gathers its keys (value, then index), which are divided in LDS until one is
//            left.  A step with more than 4,096 in it (a row of few values) is divided by passes over the row (cut_order).
//   draw     in the list; or, where many are kept, by sums over the waves' stretches, over lines of 64 of one, over a line.
//
// What bounds it: the passes' instructions, not memory: a weight and its sum are 23 to 33 of them, most on doubles.  A row of 50,272 alone: 16 us by top k 50 with all
// other filters, 20 by temperature alone (the largest, weights, draw), 45 by top p of a flat row (weights twice, and the border's keys).  256 rows of
// 128,007 by top p, flat: 115 us, where reading them once takes 27.  Passes read the row again from the L2: held in registers it was slower, since the
// unrolled code waits for its own instructions (the largest of 64 rows 35 us, 10 this way).
#include "api.h"
#include "common.h"

#include <type_traits>

namespace st {

constexpr int kBins = 2048, kFew = 512, kNear = 4096, kPlaces = 2048;
constexpr int kUnit = 44;                             // a weight of one is 2^kUnit
constexpr float kSpan = 31.25f;                       // e^-31.25 of the largest is less than half a unit

// the beginning of a row's order: all that lie before (value, index), and that one
struct Cut { float v; int i; };
__device__ inline bool within(const Cut& c, float x, int i) { return (x > c.v) | ((x == c.v) & (i <= c.i)); }     // (no branches)

// the larger, of a number and any NaN the number (the hardware's maximum makes a NaN of a signalling one, fmaxf has the compiler quiet both first)
__device__ inline float max_of(float a, float x) { return x > a ? x : a; }

// bits that order as the values do
__device__ inline uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Shared {
    uint64_t weight[kBins];                           // of a histogram's steps; sums of places
    uint32_t count[kBins];
    uint64_t wave_sum[16], stretch[16];
    float estimate[16];
    uint64_t key[kFew], sorted[kFew];                 // the list: (value's bits, index's complement); weights in an order
    int rank[kFew];
    uint64_t near_key[kNear];                         // keys of the step that holds a border
    uint64_t before;
    uint32_t bin, key_low, key_high, n, near;
    Cut cut;
    float top[16];
    int top_i[16];
};

// 2^t for t <= 0 in units of 2^-44, a whole number: 2^r, |r| <= 1/2, by a polynomial (fitted for the least largest relative error, 2^-45.9), times
// 2^n by the exponent.
// (Nearest whole numbers by adding 1.5 * 2^52, whose low bits they then are, powers by the exponent's bits: conversions, rounding and scaling
// instructions of doubles take four times as long as sums and products.  t far below -46 gives anything.)
struct Powers {
    double c[10];
    __device__ __forceinline__ void set() {
        const double k[10] = {1.0000000000000142, 0.6931471805598745, 0.24022650695649087, 0.05550410866861358, 0.009618129192178193,
                              0.0013333557629088744, 0.0001540343485947064, 1.525297804248623e-05, 1.3259425750445644e-06, 1.0151654016088282e-07};
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            c[i] = k[i];
            asm("" : "+s"(c[i]));                     // (in scalar registers: as literals each costs two moves a use)
        }
    }
    __device__ __forceinline__ double weight(double t) const {
        constexpr double kRound = 6755399441055744.0;
        const double v = t + kRound, r = t - (v - kRound);
        const int n = (int)(uint32_t)__double_as_longlong(v);
        double y = fma(c[9], r, c[8]);
#pragma unroll
        for (int i = 7; i >= 0; --i) y = fma(y, r, c[i]);
        const uint64_t bits = (uint64_t)__double_as_longlong(y);
        const uint32_t high = (uint32_t)(bits >> 32) + ((uint32_t)(n + kUnit) << 20);
        return (__longlong_as_double((long long)((uint64_t)high << 32 | (uint32_t)bits)) + kRound) - kRound;
    }
};
// a whole number below 2^52 that a double holds (a weight; sums of 256 may be 2^52)
__device__ inline uint64_t whole(double w) { return (uint64_t)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull; }

struct Row {
    const float* p;
    int vocab, lines;                                 // lines of 64 logits a wave's stretch has
    float top, low;                                   // largest value; below `low` weights are zero
    float scale;                                      // steps of a histogram in one of the value
    double from, rate;                                // weights are 2^((value - from) rate)
    Powers powers;
    __device__ inline float at(int i) const { return p[i]; }      // (a NaN is within no cut)
    __device__ inline double weight_of(float x) const { return powers.weight(((double)x - from) * rate); }       // of a finite one
    __device__ inline double weight_whole(float x) const {      // of one from `low` on (an infinity counts as the largest number, of a row whose rate is 0)
        float y;
        asm("v_min_f32 %0, %1, %2" : "=v"(y) : "v"(3.4028234663852886e38f), "v"(x));      // (without the quieting of NaN that fminf asks for)
        return weight_of(y);
    }
    __device__ inline uint64_t weight(float x) const { return whole(weight_whole(x)); }
    __device__ inline int step(float x) const { return (int)fminf(x == top ? 0.f : (top - x) * scale, (float)(kBins - 1)); }

    // f(values, index of the first) for all of the row, U values at a time, 64 indices apart, every wave over its own stretch; -infinity
    // where there is nothing (and NaN where that is there).  The next U are on their way while U are used.
    template <int U, typename F> __device__ __forceinline__ void each(F f) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        const int first = wave * lines * 64, stop = min(lines * 64, vocab - first);
        if (stop <= 0) return;
        const float* q = p + first;
        float next[U];
        const auto load = [&](int j) {
            if (j + 64 * U <= stop) {
                const float* at = q + (uint32_t)(j + lane);
#pragma unroll
                for (int u = 0; u < U; ++u) next[u] = at[64 * u];
            } else if (j < stop) {
#pragma unroll
                for (int u = 0; u < U; ++u) next[u] = q[(uint32_t)min(j + 64 * u + lane, stop - 1)];
            }
        };
        load(0);
        for (int j = 0; j < stop; j += 64 * U) {
            float x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = next[u];
            if (j + 64 * U > stop) {
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = j + 64 * u + lane < stop ? x[u] : -INFINITY;
            }
            load(j + 64 * U);
            __builtin_amdgcn_sched_barrier(0);
            f(x, first + j + lane);
        }
    }
};

// what the lanes up to and with one's own hold together: within 16 by shifts, then the rows' ends to the rows behind
__device__ inline uint64_t wave_scan64(uint64_t v) {
    const auto turn = [&](auto ctrl, auto rows, auto bound) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, decltype(ctrl)::value, decltype(rows)::value, 0xF, decltype(bound)::value);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xF, decltype(bound)::value);
        v += (uint64_t)hi << 32 | lo;
    };
    using std::integral_constant;
    turn(integral_constant<int, 0x111>(), integral_constant<int, 0xF>(), std::true_type());
    turn(integral_constant<int, 0x112>(), integral_constant<int, 0xF>(), std::true_type());
    turn(integral_constant<int, 0x114>(), integral_constant<int, 0xF>(), std::true_type());
    turn(integral_constant<int, 0x118>(), integral_constant<int, 0xF>(), std::true_type());
    turn(integral_constant<int, 0x142>(), integral_constant<int, 0xA>(), std::false_type());
    turn(integral_constant<int, 0x143>(), integral_constant<int, 0xC>(), std::false_type());
    return v;
}

// sum over the threads up to and with one's own, and over all, of 64-bit numbers (1,024 threads)
__device__ inline uint64_t block_scan(uint64_t v, Shared& s, uint64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan64(v);
    __syncthreads();
    if (lane == 63) s.wave_sum[wave] = v;
    __syncthreads();
    total = 0;
    uint64_t before = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const uint64_t x = s.wave_sum[w];
        before += w < wave ? x : 0;
        total += x;
    }
    return before + v;
}

// sum over a wave's lanes, which are all there
__device__ inline uint64_t wave_sum64(uint64_t v) {
    const auto turn = [&](auto o) {
        uint32_t la, lb, ha, hb;
        pair_across<decltype(o)::value>((uint32_t)v, la, lb);
        pair_across<decltype(o)::value>((uint32_t)(v >> 32), ha, hb);
        v = ((uint64_t)ha << 32 | la) + ((uint64_t)hb << 32 | lb);
    };
    turn(std::integral_constant<int, 32>());
    turn(std::integral_constant<int, 16>());
    turn(std::integral_constant<int, 8>());
    turn(std::integral_constant<int, 4>());
    turn(std::integral_constant<int, 2>());
    turn(std::integral_constant<int, 1>());
    return v;
}

// the sum at which u draws: the first whole number above u times all (a u that is none of [0, 1) draws an end)
__device__ inline uint64_t drawn_at(float u, uint64_t total) {
    const double at = (double)u * (double)total;
    const uint64_t below = at > 0.0 ? (at < (double)total ? (uint64_t)at : total - 1) : 0;
    return min(below, total - 1) + 1;
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
__device__ __forceinline__ int index_reaching(const Row& row, Shared& s, F measure, G target_of) {
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
        sum = wave_sum64(sum);
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
            const uint64_t own = i < row.vocab ? measure(row.at(i), i) : 0, v = wave_scan64(own);
            if (before + v >= target && before + v - own < target) s.cut.i = i;
            before += (uint64_t)__shfl((unsigned long long)v, 63, 64);
        }
    }
    __syncthreads();
    return s.cut.i;
}

__device__ inline uint64_t key_of(float x, int i) { return (uint64_t)ordered(x) << 32 | (uint32_t)~(uint32_t)i; }
__device__ inline float value_of(uint64_t key) {
    const uint32_t v = (uint32_t)(key >> 32);
    return __uint_as_float(v & 0x80000000u ? v & 0x7fffffffu : ~v);
}

// Of the n keys in s.near_key, downwards, the one at which `base` and the sum of the measure (ones, or weights) reach `target`: the range of keys
// is divided into up to 2,048 parts, then the part that holds it, until that holds one key.
template <bool COUNT>
__device__ __forceinline__ Cut cut_near(const Row& row, Shared& s, int n, uint64_t base, uint64_t target) {
    uint64_t high = ~(uint64_t)0, low = 0;            // the part, both ends in it
    {
        uint64_t a = 0, b = ~(uint64_t)0;
        for (int j = threadIdx.x; j < n; j += 1024) {
            a = max(a, s.near_key[j]);
            b = min(b, s.near_key[j]);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            a = max(a, (uint64_t)__shfl_xor((unsigned long long)a, o, 64));
            b = min(b, (uint64_t)__shfl_xor((unsigned long long)b, o, 64));
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            s.sorted[threadIdx.x >> 6] = a;
            s.sorted[16 + (threadIdx.x >> 6)] = b;
        }
        __syncthreads();
        high = s.sorted[0];
        low = s.sorted[16];
        for (int w = 1; w < 16; ++w) {
            high = max(high, s.sorted[w]);
            low = min(low, s.sorted[16 + w]);
        }
    }
    for (int round = 0; round < 6; ++round) {         // (each leaves 2^-11 of the 64 bits at most)
        const uint64_t range = high - low;
        const int shift = range < kBins ? 0 : 64 - __builtin_clzll(range) - 11;      // range >> shift < 2,048
        __syncthreads();
        for (int b = threadIdx.x; b < kBins; b += 1024) {
            s.weight[b] = 0;
            s.count[b] = 0;
        }
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += 1024) {
            const uint64_t key = s.near_key[j];
            if (key > high || key < low) continue;
            const int b = (int)((high - key) >> shift);
            atomicAdd(&s.count[b], 1u);
            atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)(COUNT ? 1 : row.weight(value_of(key))));
        }
        __syncthreads();
        const uint64_t m0 = s.weight[2 * threadIdx.x], m1 = s.weight[2 * threadIdx.x + 1];
        uint64_t total;
        const uint64_t upto = block_scan(m0 + m1, s, total);
        find_place(s, m0, upto, m1, target - base);
        const uint64_t bin = s.bin;
        base += s.before;
        high -= bin << shift;
        const uint64_t last = high - ((((uint64_t)1 << shift) - 1));
        low = shift == 0 ? high : last > high ? low : max(low, last);
        if (s.count[bin] == 1) break;
    }
    for (int j = threadIdx.x; j < n; j += 1024) {
        const uint64_t key = s.near_key[j];
        if (key <= high && key >= low) s.cut = Cut{value_of(key), (int)~(uint32_t)key};
    }
    __syncthreads();
    return s.cut;
}

// Cuts the order where `cut` leaves it at the place where the measure (a token counts one, or its weight) first reaches k, or the
// share p of all that is there.
template <bool COUNT>
__device__ __forceinline__ void cut_order(const Row& row, Shared& s, Cut& cut, uint64_t k, double p) {
    const auto measure = [&](float x) { return COUNT ? (uint64_t)1 : row.weight(x); };
    uint64_t base = 0, target = 0;
    bool first = true;
    uint32_t low = 0, high = 0xffffffffu;
    const auto step_of = [&](float x) {
        if (first) return row.step(x);
        return (int)((uint64_t)(high - ordered(x)) * kBins / ((uint64_t)(high - low) + 1));
    };
    const auto in_zone = [&](float x, int i) {
        if (!within(cut, x, i)) return false;
        const uint32_t key = ordered(x);
        return first || (key >= low && key <= high);
    };
    for (int round = 0; round < 8; ++round) {         // (the first by steps, then 2^-11 of a value's 32 bits each)
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
        if (s.count[bin] <= kNear) {
            for (int i = threadIdx.x; i < row.vocab; i += 1024) {
                const float x = row.at(i);
                if (!in_zone(x, i) || step_of(x) != bin) continue;
                s.near_key[atomicAdd(&s.n, 1u)] = key_of(x, i);
            }
            __syncthreads();
            cut = cut_near<COUNT>(row, s, (int)s.n, base, target);
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

// s.rank[c] = how many of the list's n numbers in `keys` are above (ABOVE) or below that of place c: several threads a place
template <bool ABOVE>
__device__ __forceinline__ void count_others(Shared& s, const uint64_t* keys, int n) {
    const int t = threadIdx.x;
    int places = 64;
    while (places < n) places <<= 1;                  // (a power of two, so that a wave's lanes are places that follow each other)
    const int c = t & (places - 1), turn = t / places, turns = 1024 / places;
    if (t < kFew) s.rank[t] = 0;
    __syncthreads();
    const uint64_t key = keys[c < n ? c : 0];
    int found = 0;
    int j = turn;
    for (; j + 3 * turns < n; j += 4 * turns) {
        uint64_t other[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) other[v] = keys[j + v * turns];
#pragma unroll
        for (int v = 0; v < 4; ++v) found += ABOVE ? other[v] > key : other[v] < key;
    }
    for (; j < n; j += turns) found += ABOVE ? keys[j] > key : keys[j] < key;
    if (c < n && found) atomicAdd(&s.rank[c], found);
    __syncthreads();
}

// The list's tokens (s.key; n of them, at most kFew) in order: the first `most`, of those the fewest that reach `share` (a
// number of units, or by p of their own sum where that is 0), of those with `least`; the one that u draws.
__device__ __forceinline__ int draw_from_list(const Row& row, Shared& s, int n, int most, double p, uint64_t share, double least, float u) {
    const int t = threadIdx.x;
    const bool in = t < n;
    const uint64_t key = in ? s.key[t] : 0;
    const uint32_t index = ~(uint32_t)key;
    const uint64_t w = in ? row.weight(value_of(key)) : 0;
    count_others<true>(s, s.key, n);
    const int rank = in ? s.rank[t] : 0;
    if (in) s.sorted[rank] = rank < most ? w : 0;
    __syncthreads();
    const uint64_t mine = in ? s.sorted[t] : 0;
    uint64_t total;
    const uint64_t upto = block_scan(mine, s, total);
    if (share == 0) {
        const double part = ceil(p * (double)total);
        share = part < 1.0 ? 1 : part >= (double)total ? total : (uint64_t)part;
    }
    // (weights are not zero where the running sum first reaches the share: the rank of that token)
    if (in && upto >= share && upto - mine < share) s.bin = t;
    __syncthreads();
    const bool kept = in && rank <= (int)s.bin && rank < most && w > 0 && (double)w >= least;
    if (in) s.key[t] = kept ? index : 0xffffffffu;
    count_others<false>(s, s.key, n);                  // (its first barrier: the keys are there)
    if (in) s.sorted[t] = 0;
    __syncthreads();
    const int place = in ? s.rank[t] : 0;
    if (kept) s.sorted[place] = w;
    __syncthreads();
    const uint64_t own = in ? s.sorted[t] : 0;
    const uint64_t sum = block_scan(own, s, total);
    const uint64_t target = drawn_at(u, total);
    if (own > 0 && sum >= target && sum - own < target) s.bin = t;
    __syncthreads();
    if (kept && place == (int)s.bin) s.cut.i = (int)index;
    __syncthreads();
    return s.cut.i;
}

// s.stretch: the waves' stretches' sums of the weights within the cut, of those with `least`
__device__ __forceinline__ void sum_stretches(const Row& row, Shared& s, const Cut cut, double least) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum = 0.0;                                 // (of at most 256 weights: exact in 53 bits)
    const auto add = [&](auto plain) {
        row.each<8>([&](const float* x, int i) {
            bool in = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) in |= x[j] >= cut.v;
            if (!__any(in)) return;
            double w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (decltype(plain)::value) {
                    w[j] = row.weight_of(max_of(cut.v, x[j]));
                } else {
                    w[j] = row.weight_whole(x[j]);
                    w[j] = within(cut, x[j], i + 64 * j) & (w[j] >= least) ? w[j] : 0.0;
                }
            }
            sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        });
    };
    // (nothing but the value to be above where weights begin, which has none itself and stands for all below it, unless it is so far down that
    // its power is no number: 23 instructions a logit in the place of 33)
    if (cut.i < 0 && least == 0.0 && row.rate > 0.0 && ((double)cut.v - row.from) * row.rate > -1000.0) add(std::true_type());
    else add(std::false_type());
    const uint64_t stretch = wave_sum64((uint64_t)sum);
    if (lane == 0) s.stretch[wave] = stretch;
    __syncthreads();
}

// The token that u draws of all within the cut that weigh at least so much, from s.stretch.
__device__ __forceinline__ int draw_from_row(const Row& row, Shared& s, const Cut cut, double least, float u) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const auto weigh = [&](float x, int i) {
        const double w = row.weight_whole(x);
        return within(cut, x, i) & (w >= least) ? w : 0.0;
    };
    uint64_t total = 0;
    for (int w = 0; w < 16; ++w) total += s.stretch[w];
    const uint64_t target = drawn_at(u, total);
    uint64_t before = 0;
    int at = 0;
    for (; at < 15 && before + s.stretch[at] < target; ++at) before += s.stretch[at];
    // the stretch's lines, a wave every sixteenth
    const int first = at * row.lines * 64;
    for (int j = wave; j < row.lines; j += 64) {
        float x[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) x[v] = row.at(min(first + (j + 16 * v) * 64 + lane, row.vocab - 1));
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int i = first + (j + 16 * v) * 64 + lane;
            const uint64_t line = wave_sum64(j + 16 * v < row.lines && i < row.vocab ? whole(weigh(x[v], i)) : 0);
            if (lane == 0 && j + 16 * v < row.lines) s.weight[j + 16 * v] = line;
        }
    }
    __syncthreads();
    const uint64_t mine = (int)threadIdx.x < row.lines ? s.weight[threadIdx.x] : 0;       // (at most 256 lines)
    const uint64_t upto = before + block_scan(mine, s, total);
    if (upto >= target && upto - mine < target) {
        s.bin = threadIdx.x;
        s.before = upto - mine;
    }
    __syncthreads();
    if (wave == 0) {
        const int i = first + (int)s.bin * 64 + lane;
        const uint64_t own = i < row.vocab ? whole(weigh(row.at(min(i, row.vocab - 1)), i)) : 0;
        const uint64_t v = wave_scan64(own) + s.before;
        if (v >= target && v - own < target) s.cut.i = i;
    }
    __syncthreads();
    return s.cut.i;
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
    const float t = temperature[r], u = uniforms[r];
    const int k = top_k ? top_k[r] : 0;
    const float p = top_p ? top_p[r] : 1.f;
    const float min_share = min_p ? min_p[r] : 0.f;
    row.lines = (vocab + 1023) / 1024;
    float own = -INFINITY;                            // this thread's largest, the first of those
    int own_i = 0x7fffffff;
    row.each<16>([&](const float* x, int i) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            own_i = x[j] > own ? i + 64 * j : own_i;
            own = max_of(own, x[j]);
        }
    });
    const float mine = wave_max(own);
    if (lane == 0) s.top[wave] = mine;
    for (int b = threadIdx.x; b < kBins; b += 1024) {
        s.weight[b] = 0;
        s.count[b] = 0;
    }
    if (threadIdx.x == 0) {
        s.n = s.near = s.bin = 0;                         // (a place is always found; were one not, no index would be whatever lay here)
        s.before = 0;
        s.cut = Cut{0.f, 0};
    }
    __syncthreads();
    float best = s.top[0];
    for (int w = 1; w < 16; ++w) best = max_of(best, s.top[w]);
    if (!(t > 0.f) || k == 1 || !(p > 0.f) || best == -INFINITY) {
        int at = own == best ? own_i : 0x7fffffff;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
        if (lane == 0) s.top_i[wave] = at;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 16; ++w) at = min(at, s.top_i[w]);
            out[r] = at == 0x7fffffff ? 0 : at;       // (nothing but -infinity and NaN)
        }
        return;
    }
    row.powers.set();
    row.top = best;
    // (beside an infinity nothing else has weight)
    row.rate = best < INFINITY ? 1.4426950408889634 / (double)t : 0.0;
    row.from = best < INFINITY ? (double)best : 0.0;
    row.low = best < INFINITY ? fmaxf(best - kSpan * t, -3.4028234663852886e38f) : best;
    row.scale = (float)fmin((double)kBins / ((double)kSpan * (double)t), 3.0e38);      // (not zero but for an infinite temperature)
    const double least = min_share > 0.f ? (double)fminf(min_share, 1.f) * 17592186044416.0 : 0.0;
    // a wave's lanes that ask for it get places one behind the other (the counter's old value and up)
    const auto places = [&](uint32_t* counter, uint64_t all) {
        const int leader = __ffsll((unsigned long long)all) - 1;
        uint32_t at = 0;
        if (lane == leader) at = atomicAdd(counter, (uint32_t)__popcll(all));
        at = __builtin_amdgcn_readlane(at, leader);
        return at + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
    };
    bool full = false;                                // (of the wave: the list has no room)
    const auto list = [&](float x, int i, bool wanted) {
        const uint64_t all = __ballot(wanted);
        if (all == 0 || full) return;
        const uint32_t at = places(&s.n, all);
        if (wanted && at < kFew) s.key[at] = key_of(x, i);
        full = __any(wanted && at >= kFew);
    };
    const auto near = [&](float x, int i, bool wanted) {
        const uint64_t all = __ballot(wanted);
        if (all == 0) return;
        const uint32_t at = places(&s.near, all);
        if (wanted && at < kNear) s.near_key[at] = key_of(x, i);
    };
    // a value that all of the steps up to this one are above: a little below the step's end
    const auto below_step = [&](int step) {
        return step >= kBins - 1 ? row.low : fmaxf(best - (float)(step + 1) / row.scale * 1.00001f - fabsf(best) * 1e-6f, row.low);
    };
    // all from `low` on; with a least share of the largest weight, all from a little below the value that has it
    const auto above = [](float v) { return Cut{v > 0.f ? __uint_as_float(__float_as_uint(v) - 1) : v == 0.f ? -1e-45f : __uint_as_float(__float_as_uint(v) + 1), -1}; };
    Cut cut = above(row.low);
    if (k > 0 && k < vocab) {
        if (k <= kFew) {
            if (own >= row.low) atomicAdd(&s.count[row.step(own)], 1u);
            __syncthreads();
            const uint32_t a = s.count[2 * threadIdx.x], b = s.count[2 * threadIdx.x + 1];
            uint64_t total;
            const uint64_t upto = block_scan(a + b, s, total);
            find_place(s, a, upto, b, min((uint64_t)k, total));
            // (fewer threads than k hold anything: all of it)
            const float line = total < (uint64_t)k ? row.low : below_step((int)s.bin);
            row.each<16>([&](const float* x, int i) {
                bool any = false;
#pragma unroll
                for (int j = 0; j < 16; ++j) any |= x[j] >= line;
                if (!__any(any)) return;
#pragma unroll
                for (int j = 0; j < 16; ++j) list(x[j], i + 64 * j, x[j] >= line);
            });
            __syncthreads();
            const int n = (int)s.n;
            if (n <= kFew) {
                const int token = draw_from_list(row, s, n, k, (double)p < 1.0 ? (double)p : 1.0, 0, least, u);
                if (threadIdx.x == 0) out[r] = token;
                return;
            }
        }
        __syncthreads();
        for (int b = threadIdx.x; b < kBins; b += 1024) s.count[b] = 0;
        if (threadIdx.x == 0) s.n = 0;
        full = false;
        __syncthreads();
        row.each<8>([&](const float* x, int) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (x[j] >= row.low) atomicAdd(&s.count[row.step(x[j])], 1u);
        });
        __syncthreads();
        const uint32_t a = s.count[2 * threadIdx.x], b = s.count[2 * threadIdx.x + 1];
        uint64_t total;
        const uint64_t upto = block_scan(a + b, s, total);
        if (total > (uint64_t)k) {                    // (what is further down has no weight)
            find_place(s, a, upto, b, (uint64_t)k);
            const int bin = (int)s.bin;
            const uint64_t base = s.before;
            if (s.count[bin] <= kNear) {
                row.each<8>([&](const float* x, int i) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) near(x[j], i + 64 * j, (x[j] >= row.low) & (row.step(x[j]) == bin));
                });
                __syncthreads();
                cut = cut_near<true>(row, s, (int)s.near, base, (uint64_t)k);
            } else {
                cut_order<true>(row, s, cut, (uint64_t)k, 0.0);
            }
            __syncthreads();
            for (int b = threadIdx.x; b < kBins; b += 1024) s.weight[b] = 0;
            if (threadIdx.x == 0) s.n = s.near = 0;
        }
        __syncthreads();
    }
    if (p < 1.f) {
        const auto add = [&](auto plain) {
            row.each<8>([&](const float* x, int i) {
                bool any = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) any |= x[j] >= cut.v;
                if (!__any(any)) return;
                uint64_t w[8];
                int at[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = row.weight(x[j]);
                    at[j] = row.step(x[j]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (decltype(plain)::value ? x[j] > cut.v : within(cut, x[j], i + 64 * j))
                        atomicAdd((unsigned long long*)&s.weight[at[j]], (unsigned long long)w[j]);
            });
        };
        if (cut.i < 0) add(std::true_type());
        else add(std::false_type());
        __syncthreads();
        const uint64_t a = s.weight[2 * threadIdx.x], b = s.weight[2 * threadIdx.x + 1];
        uint64_t total;
        const uint64_t upto = block_scan(a + b, s, total);
        const double part = ceil((double)p * (double)total);
        const uint64_t share = part < 1.0 ? 1 : part >= (double)total ? total : (uint64_t)part;
        find_place(s, a, upto, b, share);
        const int bin = (int)s.bin;
        const uint64_t base = s.before;
        // (all that are kept, and perhaps a few more, are not below `line`, and those of the border's step not above `end`)
        // (differences that are no float any more lie in the last step: all of the row is close to it then)
        const float down = (float)bin / row.scale * 0.99999f;
        const float line = below_step(bin), end = bin == 0 || !(down < 3.0e38f) ? best : best - down + fabsf(best) * 1e-6f;
        // how many there are up to the border: a step's weight over that of its upper end, too few by a step's width (1.5 %) at most
        const float one = 5.684341886080802e-14f;     // 2^-44
        const float falls = (float)row.rate / row.scale;
        const auto tokens = [&](int step, uint64_t w) { return step <= bin ? (float)w * one * __builtin_amdgcn_exp2f((float)step * falls) : 0.f; };
        const float some = wave_sum(tokens(2 * threadIdx.x, a) + tokens(2 * threadIdx.x + 1, b));
        __syncthreads();
        if (lane == 0) s.estimate[wave] = some;
        __syncthreads();
        float about = 0.f;
        for (int w = 0; w < 16; ++w) about += s.estimate[w];
        if (!(about > (float)kFew)) {
            row.each<16>([&](const float* x, int i) {
                bool any = false;
#pragma unroll
                for (int j = 0; j < 16; ++j) any |= x[j] >= line;
                if (!__any(any)) return;
#pragma unroll
                for (int j = 0; j < 16; ++j) list(x[j], i + 64 * j, (x[j] >= line) & within(cut, x[j], i + 64 * j));
            });
            __syncthreads();
            const int n = (int)s.n;
            if (n <= kFew) {
                const int token = draw_from_list(row, s, n, n, 1.0, share, least, u);
                if (threadIdx.x == 0) out[r] = token;
                return;
            }
        }
        // many: the sums over the stretches of all up to the border's step, and the keys of that step, in one pass
        double sum = 0.0;
        const auto gather = [&](auto plain) {
            row.each<8>([&](const float* x, int i) {
                uint32_t close = 0;
                bool any = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    close |= (x[j] >= line) & (x[j] <= end) ? 1u << j : 0u;
                    any |= x[j] >= line;
                }
                if (!__any(any)) return;
                double w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = row.weight_whole(x[j]);
                    if constexpr (decltype(plain)::value) w[j] = x[j] > end ? w[j] : 0.0;
                    else w[j] = (x[j] > end) & within(cut, x[j], i + 64 * j) & (w[j] >= least) ? w[j] : 0.0;
                }
                sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                // those close to the step: a lane's one by one (few lanes have any, hardly one has two)
                while (__any(close != 0)) {
                    const int j = __ffs((int)close) - 1;
                    float y = -INFINITY;
#pragma unroll
                    for (int v = 0; v < 8; ++v) y = j == v ? x[v] : y;
                    const int at = row.step(y);
                    const bool in = close != 0 && within(cut, y, i + 64 * j);
                    near(y, i + 64 * j, in & (at == bin));
                    if (in && at < bin) {
                        const double own = row.weight_whole(y);
                        sum += own >= least ? own : 0.0;
                    }
                    close &= close - 1;
                }
            });
        };
        if (cut.i < 0 && least == 0.0) gather(std::true_type());
        else gather(std::false_type());
        const uint64_t stretch = wave_sum64((uint64_t)sum);
        if (lane == 0) s.stretch[wave] = stretch;
        __syncthreads();
        if (s.near <= kNear) {
            const int n = (int)s.near;
            cut = cut_near<false>(row, s, n, base, share);
            for (int j = threadIdx.x; j < n; j += 1024) {
                const uint64_t key = s.near_key[j];
                const int i = (int)~(uint32_t)key;
                const uint64_t w = row.weight(value_of(key));
                if (within(cut, value_of(key), i) && (double)w >= least)
                    atomicAdd((unsigned long long*)&s.stretch[(i >> 6) / row.lines], (unsigned long long)w);
            }
            __syncthreads();
            const int token = draw_from_row(row, s, cut, least, u);
            if (threadIdx.x == 0) out[r] = token;
            return;
        }
        cut_order<false>(row, s, cut, 0, (double)p);
        __syncthreads();
    }
    if (least > 0.0) {
        const Cut c = above(fmaxf(best + t * logf(fminf(min_share, 1.f)) * 1.0001f - 1e-4f * t, row.low));
        if (best < INFINITY && c.v > cut.v) cut = c;
    }
    sum_stretches(row, s, cut, least);
    const int token = draw_from_row(row, s, cut, least, u);
    if (threadIdx.x == 0) out[r] = token;
}

}  // namespace st

using namespace st;

extern "C" int st_sample_filtered(int* out, const float* logits, int64_t row_stride, int num_rows, int vocab, const float* uniforms,
                                  const float* temperature, const int* top_k, const float* top_p, const float* min_p, hipStream_t stream) {
    ST_CHECK(num_rows >= 0 && vocab > 0 && row_stride >= vocab, "sample_filtered: bad sizes rows=%d vocab=%d", num_rows, vocab);
    ST_CHECK(vocab <= 1 << 18, "sample_filtered: %d logits a row (at most %d: sums of weights are 64-bit numbers)", vocab, 1 << 18);
    ST_CHECK(num_rows < 1 << 22, "sample_filtered: %d rows at once", num_rows);        // (a launch has less than 2^32 threads)
    if (num_rows == 0) return 0;
    ST_CHECK(out && logits && uniforms && temperature, "sample_filtered: null operand");
    sample_filtered_kernel<<<num_rows, 1024, 0, stream>>>(out, logits, row_stride, vocab, uniforms, temperature, top_k, top_p, min_p);
    ST_LAUNCH_CHECK("sample_filtered");
    return 0;
}
