// Attention of any query rows that read the same keys, on the matrix cores: the kernel behind attention over the 8-bit cache
// (single tokens, portions of prompts) and attention over shared prefixes.
//
// A workgroup takes one key head, up to 16 * RT query rows and a share of the keys.  Query rows are (token, query head of the key head's
// group) pairs: the heads of one token, of the tokens of a prompt's portion, or of all tokens whose requests begin with the same pages.
// A key is then read once for all of them.  Its four waves take blocks of 32 keys in turn, each with a running maximum, normaliser and
// sum of its own (an online softmax in float), and meet in LDS at the end; several workgroups that share a row's keys leave
// sums, maxima and normalisers, which a second kernel joins.
//
//   S^T = K Q^T      a lane's scores belong to one query row: l % 16.  Keys come from memory as the operand, eight dims a lane.
//   O^T += V^T P^T   P^T is the scores' registers as they are.  V goes through LDS, a wave's block in its own part (no barrier), and
//                    comes back transposed.
//
// Keys and values in 8 bits (csrc/small_float.h) become bfloat16 (exact) or float on their way into the product; a key's power of two is part of
// its conversion (float: it multiplies its scores), a value's multiplies its probability, all without rounding.  Probabilities are rounded to
// bfloat16 for the second product (at most 2^-8 of each, as the queries and keys that they come from are), or stay float in the float
// instances; maxima, sums and normalisers are float.
//
// What bounds it, and what was measured for it (bfloat16 over the 8-bit cache; a large copy reaches 4.9 TB/s, a large product 1,220 TFLOP/s):
//   single tokens    the cache's bytes: 64 rows of up to 1,000 keys, 8 key heads of 128: 133 MB in 29 us, 4.6 TB/s; 64 of 4,000: 4.6 TB/s.
//   tiles, prefixes  instructions: a block of 32 keys for 32 rows of 128 dims is 32 matrix instructions (16 cycles each, 512) and about 355 others (four each,
//                    1,420), most of them conversions and the softmax (counted over a portion of 512 rows: 0.66 and 7.4 million).  200 rows in
//                    groups of 67 behind 6,000 keys: 70 to 76 us, of which the SIMDs issue for half.  So 32 rows a wave (16: 98 us; 64, which leave a
//                    wave a SIMD: 97 where 32 took 72), powers of two in conversions (77 -> 72 with the scale in the exponent's product, which
//                    scores of any size have undone, 1 %), and two products' dims by one load (91 -> 76; the 64 rows above 35 -> 30).
//   few short rows   the way from the lists to the first key, five dependent reads, and the join: 4 to 5 us of each workgroup.
#pragma once

#include "api.h"
#include "small_float.h"

#include <type_traits>

namespace st {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef int int2v __attribute__((ext_vector_type(2)));

#define ST_LDS_PTR(T, p) ((__attribute__((address_space(3))) T*)(p))

// ---- eight elements a lane: as they lie in memory, and as an operand
template <typename TC> struct Raw8;
template <> struct Raw8<bf16_t> { uint4 a; };
template <> struct Raw8<e4m3_t> { uint2 a; };
template <> struct Raw8<float> { uint4 a, b; };

template <typename TC> __device__ inline Raw8<TC> raw8(const TC* p) { return *reinterpret_cast<const Raw8<TC>*>(p); }
template <typename TC> __device__ inline void clear(Raw8<TC>& r) { r = Raw8<TC>{}; }

__device__ inline void flip(Raw8<bf16_t>& r) { r.a.x ^= 0x80008000u; r.a.y ^= 0x80008000u; r.a.z ^= 0x80008000u; r.a.w ^= 0x80008000u; }
__device__ inline void flip(Raw8<float>& r) {
    r.a.x ^= 0x80000000u; r.a.y ^= 0x80000000u; r.a.z ^= 0x80000000u; r.a.w ^= 0x80000000u;
    r.b.x ^= 0x80000000u; r.b.y ^= 0x80000000u; r.b.z ^= 0x80000000u; r.b.w ^= 0x80000000u;
}

template <typename TQ> struct Op8;
template <> struct Op8<bf16_t> { bf16x8 v; };
template <> struct Op8<float> { float v[8]; };

__device__ inline void to_op(const Raw8<bf16_t>& r, Op8<bf16_t>& o) { o.v = __builtin_bit_cast(bf16x8, r.a); }
__device__ inline void to_op(const Raw8<float>& r, Op8<float>& o) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = __uint_as_float(w[i]);
}
__device__ inline void to_op(const Raw8<e4m3_t>& r, Op8<bf16_t>& o, float unit = 1.f) {      // times a power of two
    o.v = __builtin_bit_cast(bf16x8, make_uint4(e4m3x2_to_bf16x2<false>(r.a.x, unit), e4m3x2_to_bf16x2<true>(r.a.x, unit),
                                                e4m3x2_to_bf16x2<false>(r.a.y, unit), e4m3x2_to_bf16x2<true>(r.a.y, unit)));
}
__device__ inline void to_op(const Raw8<e4m3_t>& r, Op8<float>& o) {
    const float2v a = e4m3x2_to_floats<false>(r.a.x), b = e4m3x2_to_floats<true>(r.a.x);
    const float2v c = e4m3x2_to_floats<false>(r.a.y), d = e4m3x2_to_floats<true>(r.a.y);
    o.v[0] = a.x; o.v[1] = a.y; o.v[2] = b.x; o.v[3] = b.y; o.v[4] = c.x; o.v[5] = c.y; o.v[6] = d.x; o.v[7] = d.y;
}
__device__ inline floatx4 mma8(const Op8<bf16_t>& a, const Op8<bf16_t>& b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ inline floatx4 mma8(const Op8<float>& a, const Op8<float>& b, floatx4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}
// for scores: in float 16 products a chain (one chain over all of a head's dims is two to four times as far off, and an exponent shows it)
__device__ inline floatx4 scores8(const Op8<bf16_t>& a, const Op8<bf16_t>& b, floatx4 c) { return mma8(a, b, c); }
__device__ inline floatx4 scores8(const Op8<float>& a, const Op8<float>& b, floatx4 c) {
    floatx4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], x, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[4 + i], b.v[4 + i], y, 0, 0, 0);
    }
    return c + (x + y);
}
__device__ inline void weights_to_op(const float* p, Op8<bf16_t>& o) {
    o.v = __builtin_bit_cast(bf16x8, make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])));
}
__device__ inline void weights_to_op(const float* p, Op8<float>& o) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = p[i];
}

// ---- a wave's block of 16 NU values in LDS: rows of kPitch bytes, and an operand of V^T from 32 of them: dim 16 * dt + l % 16, keys 4g .. 4g+3 and
// 16 + 4g .. 16 + 4g+3 (g = l / 16), the keys of the scores that the lane holds
template <typename TC, int HDP, int NU> struct Values {
    // (a pitch that keeps the rows of a transposing read on different banks)
    static constexpr int kPitch = 32 * HDP * (int)sizeof(TC) + (sizeof(TC) == 2 ? 32 : 16);
    static constexpr int kBytes = 16 * NU * kPitch;
};
template <int HDP> __device__ inline void value_op(const char* block, int dt, int g, int r16, bf16_t, Op8<bf16_t>& o) {
    constexpr int P = Values<bf16_t, HDP, 2>::kPitch;
    const char* at = block + (4 * g + (r16 >> 2)) * P + 32 * dt + 8 * (r16 & 3);
    const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(ST_LDS_PTR(short4v, at)));
    const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(ST_LDS_PTR(short4v, at + 16 * P)));
    o.v = __builtin_bit_cast(bf16x8, make_uint4(x.x, x.y, y.x, y.y));
}
template <int HDP> __device__ inline Raw8<e4m3_t> value_raw(const char* block, int dt, int g, int r16) {
    constexpr int P = Values<e4m3_t, HDP, 2>::kPitch;
    const int k = r16 >> 1;
    const char* at = block + ((k < 4 ? 4 * g + k : 12 + 4 * g + k)) * P + 16 * dt + 8 * (r16 & 1);
    Raw8<e4m3_t> r;
    r.a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(ST_LDS_PTR(int2v, at)));
    return r;
}
template <int HDP> __device__ inline void value_op(const char* block, int dt, int g, int r16, float, Op8<float>& o) {
    constexpr int P = Values<float, HDP, 2>::kPitch;
    const char* at = block + 4 * g * P + 4 * (16 * dt + r16);
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = *reinterpret_cast<const float*>(at + ((i & 3) + 16 * (i >> 2)) * P);
}

// the bits of a register of values' elements that are infinite or NaN, all of them set
__device__ inline uint32_t not_finite(uint32_t w, bf16_t) { return ((((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu; }
__device__ inline uint32_t not_finite(uint32_t w, float) { return (w & 0x7f800000u) == 0x7f800000u ? ~0u : 0u; }
__device__ inline uint32_t not_finite(uint32_t w, e4m3_t) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu; }
// four elements from memory as floats
__device__ inline floatx4 four(const bf16_t* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return floatx4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)};
}
__device__ inline floatx4 four(const float* p) { return *reinterpret_cast<const floatx4*>(p); }
__device__ inline floatx4 four(const e4m3_t* p) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    const float2v a = e4m3x2_to_floats<false>(w), b = e4m3x2_to_floats<true>(w);
    return floatx4{a.x, a.y, b.x, b.y};
}

// what has been written to LDS by the lanes of a wave is read by others of it: LDS takes a wave's accesses in order, the compiler must too
__device__ inline void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// subtiles of 16 dims that the waves' results are joined by at a time: so many that each thread has a quad of a row's dims
template <int RT> constexpr int turn_subtiles() { return 4 / RT; }

// Subtiles of 16 keys a block, and whether two blocks are held, one on its way while the other is used: where two waves a SIMD keep their
// registers.  (Else one, asked for when its registers are free: 40 float rows of 80 dims behind a prefix 39 us with two and a wave a SIMD, 31 with one.)
template <typename TQ, typename TC, int HDP, int RT> struct Shape {
    static constexpr int NU = 2;
    static constexpr int NV = (2 * HDP * (int)sizeof(TC) + 3) / 4;             // 16-byte chunks of a value that a lane moves (four lanes a value)
    static constexpr int kBlock = NU * (HDP * (int)sizeof(Raw8<TC>) / 4 + 4 * NV);
    static constexpr bool kTwo = 2 * kBlock + RT * (HDP * (int)sizeof(Op8<TQ>) / 4 + 8 * HDP + 8 * NU) <= 200;
};

// Waves a SIMD that the registers have to leave room for: two, but where float operands (or, over the storage type, heads of more than 128 dims) fill
// them; four for the smallest instance with groups, which is a register or two above that if it may be.
template <typename TQ, typename TC, int HDP, int RTS, bool WHOLE> constexpr int simd_waves() {
    constexpr bool quant = sizeof(TC) == 1, bf16 = sizeof(TQ) == 2;
    if (quant && bf16 && HDP == 2 && RTS == 1 && WHOLE) return 4;
    return HDP <= (quant ? (bf16 ? 8 : 4) : (bf16 ? 4 : 3)) ? 2 : 1;
}

constexpr float kFloor = -3.4028234663852886e38f;      // a running maximum before the first key

// Scores in units of log2 are products times sl > 0, so that their maximum is that of the products: the scale's sign goes to the queries, and with a
// scale of nothing they are nothing.
__device__ inline float log2_scale(float scale) {
    const float s = fabsf(scale) * 1.44269504088896340736f;
    return s == 0.f ? 1.f : s;
}
// Maxima are those of products, and what is scaled is a difference of two: 2^24 in units of log2 and more, a rounded maximum in those units would be off by
// more than the weights' range (scores of 10^9 and more came out as nothing or NaN; one instruction a score, 1 % of a portion's time).
__device__ inline float weight_of(float score, float top, float sl) { return __builtin_amdgcn_exp2f((score - top) * sl); }

// What a workgroup works on: rows [first, first + count) of the flat list (token j, query head) = (f / group, f % group).
struct TileWork {
    int item;              // whose block table
    int first, count;      // flat rows
    int lo;                // first key
    int kind;              // 0 one token, 1 consecutive rows of an item, 2 a list of rows over a prefix
    int base;              // the token; the item's first batch row; the list's first place
    int start;             // kinds 0 and 1: position of the first row's token
    int slot, splits, split;
    int waves;             // 4 share the keys, or 1 has them alone (the others work on other rows)
};

// flat row j's token and how many keys it sees; -1 where there is none
__device__ inline int row_token(const StTileAttention& p, const TileWork& w, int j, int& sees) {
    const int t = w.kind == 2 ? p.shared_rows[w.base + j] : w.base + j;
    sees = 0;
    if (t < 0 || t >= p.num_rows) return -1;
    if (w.kind == 2) {
        const int item = p.token_item[t], pos = p.positions[t], start = p.row_start[t];
        if ((uint32_t)item < (uint32_t)p.num_items) sees = min(pos + 1, start);      // (else a padding row)
    } else {
        sees = w.start + j + 1;
    }
    return t;
}

// the largest (or least) over a row of 16 lanes, to all of them
template <bool MAX>
__device__ inline int row16(int x) {
    const auto turn = [&](auto ctrl) {
        const int y = __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xF, 0xF, false);
        x = MAX ? max(x, y) : min(x, y);
    };
    turn(std::integral_constant<int, 0x128>());
    turn(std::integral_constant<int, 0x124>());
    turn(std::integral_constant<int, 0x122>());
    turn(std::integral_constant<int, 0x121>());
    return x;
}

template <typename TQ, typename TC, int HDP, int RT, bool WHOLE>
__device__ inline void tile_work(const StTileAttention& p, const TileWork& w, int kvh, char* lds) {
    constexpr int DT = 2 * HDP, R = 16 * RT;
    constexpr bool QUANT = sizeof(TC) == 1;
    constexpr int ES = sizeof(TC);
    // A key's power of two goes into its conversion to bfloat16 (at no cost, and exact but for what is below 2^-126), into its scores where it becomes float.
    constexpr bool SCALED = QUANT && sizeof(TQ) == 2;
    using S = Shape<TQ, TC, HDP, RT>;
    constexpr int NU = S::NU, NV = S::NV, KEYS = 16 * NU, NF = NU / 2;
    constexpr int VB = Values<TC, HDP, NU>::kBytes;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    const int STEP = w.waves * KEYS;                        // keys between a wave's blocks
    const int G = p.heads / p.kv_heads, hd = p.head_dim, ps = p.page_size;
    float* s_m = reinterpret_cast<float*>(lds);             // [4][R] the waves' maxima
    float* s_l = s_m + 4 * R;                               // [4][R] and normalisers
    int* s_t = reinterpret_cast<int*>(s_l + 4 * R);         // [R] the rows' tokens
    int* s_sees = s_t + R;                                  // [R] and how many keys they see
    int* s_wild = s_sees + R;                               // [4] whether the waves left out values that are not finite
    float* s_unit = s_l + 6 * R + 4 + wave * 2 * KEYS;      // the powers of two of a wave's keys, then values
    char* s_big = reinterpret_cast<char*>(s_l + 6 * R + 4 + (QUANT ? 8 * KEYS : 0));
    char* s_v = s_big + wave * VB;                          // [4][KEYS values], at the end the waves' sums

    // The first of the eight dims that a lane has in product s.  In 8 bits two products' dims lie behind each other, so that a load brings both
    // (a dot product takes its dims in any order).
    constexpr bool PAIRS = QUANT && HDP % 2 == 0;
    const auto dim_of = [&](int s) { return PAIRS ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; };

    const float sl = log2_scale(p.scale);
    const bool no_scale = fabsf(p.scale) * 1.44269504088896340736f == 0.f;

    // ---- query rows
    Op8<TQ> qf[RT][HDP];
    int lim[RT], most = 0, least = 0x7fffffff;
    const int last_key = p.max_pages * ps;                  // (the host has checked that this is an int)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int f = w.first + 16 * rt + r16;
        int t = -1, sees = 0, head = 0;
        if (f < w.count) {
            const int j = f / G;
            head = f - j * G;
            t = row_token(p, w, j, sees);
        }
        sees = min(max(sees, 0), last_key);
        const TQ* row = (const TQ*)p.q + (int64_t)max(t, 0) * p.q_stride + (int64_t)(kvh * G + head) * hd;
#pragma unroll
        for (int s = 0; s < HDP; ++s) {
            const int d = dim_of(s);
            Raw8<TQ> r = raw8(row + (d < hd ? d : 0));
            if (t < 0 || d >= hd || no_scale) clear(r);
            if (p.scale < 0.f) flip(r);
            to_op(r, qf[rt][s]);
        }
        if (wave == 0 && g == 0) {                          // (read only where the waves share their rows)
            s_t[16 * rt + r16] = t;
            s_sees[16 * rt + r16] = sees;
        }
        most = max(most, sees);
        lim[rt] = sees == 0 ? 0x7fffffff : sees;            // (a row that is none, or sees none, takes whatever comes)
        least = min(least, lim[rt]);
    }
    most = __builtin_amdgcn_readfirstlane(row16<true>(most));
    least = __builtin_amdgcn_readfirstlane(row16<false>(least));

    // ---- keys of this workgroup: [kb0, ke), from a multiple of 16 on (keys before w.lo are masked)
    const int lo = w.lo & ~15, len = max(most - lo, 0);
    const int blocks = (len + KEYS - 1) / KEYS, share = (blocks + w.splits - 1) / w.splits * KEYS;
    const int64_t from = (int64_t)lo + (int64_t)w.split * share;
    const int kb0 = w.lo < most ? (int)min(from, (int64_t)most) : 0, ke = w.lo < most ? (int)min(from + share, (int64_t)most) : 0;

    // Pages.  WHOLE: 16 divides the page size, so 16 keys lie in one page; its number comes by a scalar load, and what a lane adds to its
    // address never changes (but past the last key, which stands for those behind it).  Else every lane looks up its own keys.  Page
    // numbers are asked for a block ahead of the entries, and before them: loads come back in order, and what is behind the entries of a
    // block could not be used before all of them are there.  Nothing touches an entry between its load and its use, which would be a wait.
    const bool shifts = (ps & (ps - 1)) == 0;
    const int page_bits = 31 - __builtin_clz(ps);
    const int* bt = p.block_table + (int64_t)w.item * p.max_pages;
    typedef const __attribute__((address_space(4))) int* scalar_ints;
    const auto page_of = [&](int key) { return shifts ? key >> page_bits : key / ps; };
    struct Places {
        int page[NU], row[NU];                              // WHOLE: of 16 keys each, the page and the row of the first
        int kp[NU], kr[NU], vp[NU], vr[NU], ep[NF], er[NF]; // else of each lane's keys
    };
    const auto look_up_block = [&](int kb) {
        Places q;
        if constexpr (WHOLE) {
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int key = __builtin_amdgcn_readfirstlane(min(kb + 16 * u, ke - 1)), pi = page_of(key);
                q.page[u] = *(scalar_ints)(uintptr_t)(bt + pi);
                q.row[u] = key - pi * ps;
            }
        } else {
            const auto look_up = [&](int key, int& page, int& row) {
                key = min(key, ke - 1);
                const int pi = page_of(key);
                page = bt[pi];
                row = key - pi * ps;
            };
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                look_up(kb + 16 * u + r16, q.kp[u], q.kr[u]);
                look_up(kb + 16 * u + (lane >> 2), q.vp[u], q.vr[u]);
            }
            if (QUANT)
#pragma unroll
                for (int f = 0; f < NF; ++f) look_up(kb + (64 * f + lane) % KEYS, q.ep[f], q.er[f]);
        }
        return q;
    };
    struct Block {
        Raw8<TC> kr[NU][HDP];
        uint4 vr[NU][NV];
        // exponents of the powers of two.  WHOLE: of the values of the four keys that a lane has scores of in each 16, and of those four keys
        // or (SCALED) the key that it loads; else lane l's number f is that of key 64 f + l, values behind keys
        uint32_t field[WHOLE ? 2 * NU : NF];
        uint64_t bad;                                       // keys whose page is none of the pool's
    };
    const int head_off = kvh * ps * hd;
    const bool outside = hd < 32 * HDP;                     // some lanes hold dims that the head does not have
    uint32_t k_dims[HDP], v_bytes[NV];                      // what a lane adds for its dims (those outside: the row's start)
#pragma unroll
    for (int s = 0; s < HDP; ++s) k_dims[s] = dim_of(s) < hd ? dim_of(s) : 0;
#pragma unroll
    for (int c = 0; c < NV; ++c) v_bytes[c] = 16 * (4 * c + (lane & 3)) < hd * ES ? 16 * (4 * c + (lane & 3)) : 0;
    const auto load_keys = [&](Block& b, int u, const TC* at, uint32_t off) {
        if constexpr (PAIRS) {
#pragma unroll
            for (int s = 0; s < HDP; s += 2) {
                const uint4 both = *reinterpret_cast<const uint4*>(at + (off + k_dims[s]));
                b.kr[u][s].a = make_uint2(both.x, both.y);
                b.kr[u][s + 1].a = make_uint2(both.z, both.w);
            }
        } else {
#pragma unroll
            for (int s = 0; s < HDP; ++s) b.kr[u][s] = raw8(at + (off + k_dims[s]));
        }
    };
    const auto load_values = [&](Block& b, int u, const TC* at, uint32_t off) {
#pragma unroll
        for (int c = 0; c < NV; ++c) b.vr[u][c] = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(at) + (off * ES + v_bytes[c]));
    };
    const auto issue = [&](Block& b, const Places& q, int kb) {
        b.bad = 0;
        if constexpr (WHOLE) {
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const bool none = (uint32_t)q.page[u] >= (uint32_t)p.num_pages;
                const int64_t at = (int64_t)(none ? 0 : q.page[u]) * p.page_stride + head_off + q.row[u] * hd;
                const int left = max(ke - 1 - (kb + 16 * u), 0);         // rows behind the first that exist
                load_keys(b, u, (const TC*)p.k_cache + at, (uint32_t)(min(r16, left) * hd));
                load_values(b, u, (const TC*)p.v_cache + at, (uint32_t)(min(lane >> 2, left) * hd));
                if (none) b.bad |= (uint64_t)0xffffu << (16 * u);
            }
            if (QUANT) {
#pragma unroll
                for (int u = 0; u < NU; ++u) {
                    const uint64_t at = (uint64_t)((uint32_t)q.page[u] < (uint32_t)p.num_pages ? (uint32_t)q.page[u] : 0u) * (uint64_t)p.exp_stride +
                                        (uint64_t)(kvh * ps + (q.row[u] & ~15));
                    b.field[2 * u] = SCALED ? p.k_exp[at + r16] : *reinterpret_cast<const uint32_t*>(p.k_exp + at + 4 * g);
                    b.field[2 * u + 1] = *reinterpret_cast<const uint32_t*>(p.v_exp + at + 4 * g);
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const bool none = (uint32_t)q.kp[u] >= (uint32_t)p.num_pages, vnone = (uint32_t)q.vp[u] >= (uint32_t)p.num_pages;
                b.bad |= (__ballot(none) & 0xffffu) << (16 * u);
                load_keys(b, u, (const TC*)p.k_cache + (uint64_t)(none ? 0u : (uint32_t)q.kp[u]) * (uint64_t)p.page_stride + head_off, (uint32_t)(q.kr[u] * hd));
                load_values(b, u, (const TC*)p.v_cache + (uint64_t)(vnone ? 0u : (uint32_t)q.vp[u]) * (uint64_t)p.page_stride + head_off, (uint32_t)(q.vr[u] * hd));
            }
            if (QUANT) {
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const uint32_t page = (uint32_t)q.ep[f] < (uint32_t)p.num_pages ? (uint32_t)q.ep[f] : 0u;
                    b.field[f] = (64 * f + lane < KEYS ? p.k_exp : p.v_exp)[(uint64_t)page * (uint64_t)p.exp_stride + kvh * ps + q.er[f]];
                }
            }
        }
    };

    float m[RT], l[RT];
    floatx4 acc[RT][DT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = kFloor;
        l[rt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    // A value that is not finite is not to reach the rows that do not see its key, not even by a product with nothing: in blocks with keys that some
    // rows see and some do not (a wave's rows alone have none) such elements are cleared, and given to the rows that see them at the end.
    bool wild = false;

    // a block in registers -> maximum, normaliser and sums; `then` is called once its registers are free
    // (What the compiler knows of a product's result and of loads under way ends at a branch: two remain between the products, the mask of a
    // block that has keys to leave out, and the sums' turn to a new maximum, which most blocks of a long row do without.)
    const auto consume = [&](Block& b, int kb, auto then) {
        const uint64_t none = b.bad;
        const bool whole = kb >= w.lo && kb + KEYS <= min(ke, least) && none == 0;
        if (!whole) {
            const auto out = [&](int in) { return (kb + in >= ke) | (kb + in < w.lo) | (bool)((none >> in) & 1); };
            const uint32_t mixed = least < min(ke, kb + KEYS) ? ~0u : 0u;      // (keys that some rows see and some do not)
            uint32_t odd = 0;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const uint32_t none_of = out(16 * u + (lane >> 2)) ? ~0u : 0u;
#pragma unroll
                for (int c = 0; c < NV; ++c) {
                    uint4& v = b.vr[u][c];
                    const auto clear = [&](uint32_t& x) {
                        const uint32_t n = not_finite(x, TC{}) & mixed;
                        odd |= n;
                        x &= ~(n | none_of);
                    };
                    clear(v.x); clear(v.y); clear(v.z); clear(v.w);
                    asm volatile("" : "+v"(odd));           // (chunk by chunk: all at once take a register each)
                }
            }
            wild |= __any(odd != 0);
            if constexpr (!WHOLE)
#pragma unroll
                for (int f = 0; f < NF; ++f)
                    if (out((64 * f + lane) % KEYS)) b.field[f] = 127;
        }
        wave_fence();                                       // (the block before has been read)
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const int at = 16 * (4 * c + (lane & 3));
                if (64 * NV <= 32 * HDP * ES || at < 32 * HDP * ES)
                    *reinterpret_cast<uint4*>(s_v + (16 * u + (lane >> 2)) * Values<TC, HDP, NU>::kPitch + at) = b.vr[u][c];
            }
        if (QUANT && !WHOLE)
#pragma unroll
            for (int f = 0; f < NF; ++f) s_unit[64 * f + lane] = __uint_as_float(b.field[f] << 23);
        wave_fence();
        float k_unit[NU];
        if constexpr (SCALED)
#pragma unroll
            for (int u = 0; u < NU; ++u) k_unit[u] = WHOLE ? __uint_as_float(b.field[2 * u] << 23) : s_unit[16 * u + r16];
        floatx4 sc[RT][NU];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int u = 0; u < NU; ++u) sc[rt][u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < HDP; ++s)
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                Op8<TQ> a;
                // (dims outside: nothing times a dim of the same key, which may be infinite but in 8 bits)
                if (!QUANT && outside && dim_of(s) >= hd) clear(b.kr[u][s]);
                if constexpr (SCALED) to_op(b.kr[u][s], a, k_unit[u]);
                else to_op(b.kr[u][s], a);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sc[rt][u] = scores8(a, qf[rt][s], sc[rt][u]);
            }
        // (8-bit values: asked for before the softmax that their trip from LDS takes as long as, where registers are left for them)
        constexpr bool EARLY = QUANT && HDP <= 4;
        Raw8<e4m3_t> vraw[EARLY ? DT : 1][NF];
        if constexpr (EARLY)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int f = 0; f < NF; ++f) vraw[dt][f] = value_raw<HDP>(s_v + 32 * f * Values<TC, HDP, NU>::kPitch, dt, g, r16);
        floatx4 ku[NU], vu[NU];                             // powers of two
        if (QUANT) {
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                if constexpr (WHOLE) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (!SCALED) ku[u][r] = __uint_as_float(((b.field[2 * u] >> (8 * r)) & 0xffu) << 23);
                        vu[u][r] = __uint_as_float(((b.field[2 * u + 1] >> (8 * r)) & 0xffu) << 23);
                    }
                } else {
                    if (!SCALED) ku[u] = *reinterpret_cast<const floatx4*>(s_unit + 16 * u + 4 * g);
                    vu[u] = *reinterpret_cast<const floatx4*>(s_unit + KEYS + 16 * u + 4 * g);
                }
            }
        }
        then();                                             // (the block's registers are free)
        float x[RT][4 * NU];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 4 * NU; ++i) x[rt][i] = QUANT && !SCALED ? sc[rt][i >> 2][i & 3] * ku[i >> 2][i & 3] : sc[rt][i >> 2][i & 3];
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4 * NU; ++i) {
                const int in = 16 * (i >> 2) + 4 * g + (i & 3), key = kb + in;
                const bool out = (key >= ke) | (key < w.lo) | ((none >> in) & 1);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if (out | (key >= lim[rt])) x[rt][i] = -INFINITY;
                if (QUANT && out) vu[i >> 2][i & 3] = 1.f;  // (nothing times whatever lies there)
            }
        }
        Op8<TQ> pf[RT][NF];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float top = max_raw(x[rt][0], x[rt][1]);
#pragma unroll
            for (int i = 2; i < 4 * NU; i += 2) top = max3_raw(top, x[rt][i], x[rt][i + 1]);
            top = rows4_max(top);
            const float mn = max_raw(m[rt], top);
            if (__any(mn > m[rt])) {
                const float alpha = weight_of(m[rt], mn, sl);
                l[rt] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[rt][dt] *= alpha;
                m[rt] = mn;
            }
#pragma unroll
            for (int i = 0; i < 4 * NU; ++i) {
                x[rt][i] = weight_of(x[rt][i], mn, sl);
                l[rt] += x[rt][i];
                if (QUANT) x[rt][i] *= vu[i >> 2][i & 3];
            }
#pragma unroll
            for (int f = 0; f < NF; ++f) weights_to_op(x[rt] + 8 * f, pf[rt][f]);
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {                   // (dims that the head does not have: never stored)
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                Op8<TQ> v;
                if constexpr (EARLY) to_op(vraw[dt][f], v);
                else if constexpr (QUANT) to_op(value_raw<HDP>(s_v + 32 * f * Values<TC, HDP, NU>::kPitch, dt, g, r16), v);
                else value_op<HDP>(s_v + 32 * f * Values<TC, HDP, NU>::kPitch, dt, g, r16, TC{}, v);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt][dt] = mma8(v, pf[rt][f], acc[rt][dt]);
            }
        }
    };
    int kb = kb0 + (w.waves == 1 ? 0 : KEYS * wave);
    constexpr bool AHEAD = WHOLE || HDP <= 4;               // (a lane's own places take registers that the longest heads have not left)
    Places next;
    const auto ahead = [&](Block& b, int at) {              // asks for the block at `at`, whose pages are known, and for the pages of the one behind
        const Places now = AHEAD ? next : look_up_block(at);       // (whether or not there is one: what is asked for twice is the last key)
        if (AHEAD) next = look_up_block(at + STEP);
        issue(b, now, at);
    };
    Block one;
    if (kb < ke) {
        if (AHEAD) next = look_up_block(kb);
        ahead(one, kb);
        if constexpr (S::kTwo) {
            Block two;
            for (;;) {
                ahead(two, kb + STEP);
                __builtin_amdgcn_sched_barrier(0);
                consume(one, kb, [] {});
                __builtin_amdgcn_sched_barrier(0);
                if ((kb += STEP) >= ke) break;
                ahead(one, kb + STEP);
                __builtin_amdgcn_sched_barrier(0);
                consume(two, kb, [] {});
                __builtin_amdgcn_sched_barrier(0);
                if ((kb += STEP) >= ke) break;
            }
        } else {
            for (; kb < ke; kb += STEP) consume(one, kb, [&] { ahead(one, kb + STEP); });
        }
    }

    const int place = (w.kind == 2 ? p.own_splits : 0) + w.split;      // of the row's partial results
    if (RT == 1 && w.waves == 1) {                          // nothing to join: from the registers
        const float sum = rows4_sum(l[0]), inverse = sum == 0.f ? 0.f : 1.f / sum;
        const int f = w.first + r16, t = w.base + f / G, head = kvh * G + f - f / G * G;
        if (f < w.count) {                                  // (kind 0: one token, which is there)
            const int64_t at = (int64_t)(w.slot >= 0 ? w.slot : t) * p.heads + head;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const int d = 16 * dt + 4 * g;
                if (16 * dt >= hd) break;
                const float by = p.slots == 1 ? inverse : 1.f;
                const float res[4] = {acc[0][dt][0] * by, acc[0][dt][1] * by, acc[0][dt][2] * by, acc[0][dt][3] * by};
                if (p.slots == 1) Elem<TQ>::store4((TQ*)p.out + ((int64_t)t * p.heads + head) * hd + d, res);
                else Elem<float>::store4(p.part_o + (at * p.slots + place) * hd + d, res);
            }
            if (p.slots > 1 && g == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * (at * p.slots + place)) = make_float2(m[0], sum);
        }
        return;
    }

    // ---- the waves' results, joined
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = rows4_sum(l[rt]);
        if (g == 0) {
            s_m[wave * R + 16 * rt + r16] = m[rt];
            s_l[wave * R + 16 * rt + r16] = l[rt];
        }
    }
    if (lane == 0) s_wild[wave] = wild;
    __syncthreads();                                        // (and all blocks of values have been read)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float top = kFloor;
#pragma unroll
        for (int v = 0; v < 4; ++v) top = max_raw(top, s_m[v * R + 16 * rt + r16]);
        const float own = weight_of(m[rt], top, sl);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[rt][dt] *= own;
    }
    // a thread's row and four of its dims, in turns over the subtiles of the head
    constexpr int DC = turn_subtiles<RT>(), JP = 16 * DC + 4;       // subtiles a turn, floats between its rows in LDS
    float* s_o = reinterpret_cast<float*>(s_big);           // [4][R][JP]
    constexpr int TPR = 256 / R;                            // threads a row, a quad of dims each
    const int row = tid / TPR, quad = tid % TPR;
    const int f = w.first + row, t = s_t[row], head = kvh * G + f - f / G * G;
    float top = kFloor, sum = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) top = max_raw(top, s_m[v * R + row]);
#pragma unroll
    for (int v = 0; v < 4; ++v) sum += s_l[v * R + row] * weight_of(s_m[v * R + row], top, sl);
    const bool any = s_sees[row] > 0;                       // (else zeros, and what its lanes hold is not looked at)
    if (!any) {
        top = kFloor;
        sum = 0.f;
    }
    // (a sum that is no number belongs to the result)
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t out_row = (int64_t)(w.slot >= 0 ? w.slot : t) * p.heads + head;
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += DC) {
        if (16 * d0 >= hd) break;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int c = 0; c < DC; ++c)
                if (16 * rt + r16 + w.first < w.count && 16 * (d0 + c) < hd)
                    *reinterpret_cast<floatx4*>(s_o + (wave * R + 16 * rt + r16) * JP + 16 * c + 4 * g) = acc[rt][d0 + c];
        __syncthreads();
        const int d = 16 * d0 + 4 * quad;
        if (t >= 0 && d < hd) {
            floatx4 o = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < 4; ++v) o += *reinterpret_cast<const floatx4*>(s_o + (v * R + row) * JP + 4 * quad);
            if (s_wild[0] | s_wild[1] | s_wild[2] | s_wild[3]) {
                // (they were left out from the first block on in which a row sees less than others)
                const int seen = min(s_sees[row], ke);
                for (int key = max(kb0 + max(least - kb0, 0) / KEYS * KEYS, w.lo); key < seen; ++key) {
                    const int pi = page_of(key), page = bt[pi];
                    if ((uint32_t)page >= (uint32_t)p.num_pages) continue;
                    const floatx4 x = four((const TC*)p.v_cache + (int64_t)page * p.page_stride + head_off + (key - pi * ps) * hd + d);
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] += fabsf(x[r]) < INFINITY ? 0.f : x[r];
                }
            }
            if (!any) o = floatx4{0.f, 0.f, 0.f, 0.f};
            const float by = p.slots == 1 ? inverse : 1.f;
            const float res[4] = {o[0] * by, o[1] * by, o[2] * by, o[3] * by};
            if (p.slots == 1)
                Elem<TQ>::store4((TQ*)p.out + ((int64_t)t * p.heads + head) * hd + d, res);
            else
                Elem<float>::store4(p.part_o + (out_row * p.slots + place) * hd + d, res);
        }
        if (d0 + DC < DT) __syncthreads();
    }
    if (t >= 0 && p.slots > 1 && quad == 0)
        *reinterpret_cast<float2*>(p.part_ml + 2 * (out_row * p.slots + place)) = make_float2(top, sum);
}

// LDS of a workgroup
template <typename TQ, typename TC, int HDP, int RT>
constexpr int tile_lds() {
    constexpr int kTurn = 4 * 16 * RT * (16 * turn_subtiles<RT>() + 4) * 4;
    constexpr int NU = Shape<TQ, TC, HDP, RT>::NU;
    return (10 * 16 * RT + 4 + (sizeof(TC) == 1 ? 8 * 16 * NU : 0)) * 4 +
           (4 * Values<TC, HDP, NU>::kBytes > kTurn ? 4 * Values<TC, HDP, NU>::kBytes : kTurn);
}

// Workgroups: key head fastest (a head's workgroups share its keys and, dealt out in turn, an XCD's L2), then splits, then
// entries: shared prefixes first (kind 2, RTS subtiles of rows), then single tokens or tiles (RT).
template <typename TQ, typename TC, int HDP, int RT, int RTS, bool WHOLE>
__global__ __launch_bounds__(256, (simd_waves<TQ, TC, HDP, RTS, WHOLE>())) void tile_attention_kernel(const StTileAttention p) {
    extern __shared__ uint4 dyn[];
    char* lds = reinterpret_cast<char*>(dyn);
    const int G = p.heads / p.kv_heads;
    const int kvh = blockIdx.x % p.kv_heads;
    int y = blockIdx.x / p.kv_heads;
    TileWork w;
    w.start = w.lo = 0;
    w.slot = -1;
    w.waves = 4;
    if constexpr (RTS > 0) {
        if (y < p.shared_entries * p.shared_splits) {
            int e = y / p.shared_splits;
            w.split = y - e * p.shared_splits;
            w.splits = p.shared_splits;
            w.kind = 2;
            // the group that entry e belongs to: groups take ceil(rows * G / (16 RTS)) entries each, one behind the other
            constexpr int R = 16 * RTS;
            int found = -1, off = 0, n = 0;
            for (int base = 0; base < p.num_groups && found < 0; base += 64) {
                const int i = base + (int)(threadIdx.x & 63);
                int a = 0, b = 0;
                if (i < p.num_groups) {
                    a = min(max(p.group_off[i], 0), p.num_shared);
                    b = min(max(p.group_off[i + 1], a), p.num_shared);
                }
                const int mine = ((b - a) * G + R - 1) / R;
                const int upto = wave_scan(mine);
                const uint64_t in = __ballot(e < upto);
                if (in) {
                    const int at = __ffsll((unsigned long long)in) - 1;
                    found = base + at;
                    off = __shfl(a, at, 64);
                    n = __shfl(b, at, 64) - off;
                    e -= __shfl(upto - mine, at, 64);
                } else {
                    e -= __shfl(upto, 63, 64);
                }
            }
            if (found < 0) return;
            w.base = __builtin_amdgcn_readfirstlane(off);
            w.first = __builtin_amdgcn_readfirstlane(e) * R;
            w.count = __builtin_amdgcn_readfirstlane(n) * G;
            // the block table: that of the first of the group's rows that has a request
            uint64_t there = 0;
            int item = -1;
            for (int base = 0; base < n && !there; base += 64) {
                const int i = base + (int)(threadIdx.x & 63);
                const int t = i < n ? p.shared_rows[w.base + i] : -1;
                item = t >= 0 && t < p.num_rows ? p.token_item[t] : -1;
                there = __ballot((uint32_t)item < (uint32_t)p.num_items);
            }
            if (!there) w.lo = 0x7fffffff;                 // none: no key is seen
            w.item = there ? __builtin_amdgcn_readfirstlane(__shfl(item, __ffsll((unsigned long long)there) - 1, 64)) : 0;
            tile_work<TQ, TC, HDP, (RTS > 0 ? RTS : 1), WHOLE>(p, w, kvh, lds);
            return;
        }
        y -= p.shared_entries * p.shared_splits;
    }
    if (p.own_waves == 1) {                                 // a wave each
        w.waves = 1;
        y = 4 * y + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (y >= p.num_entries * ((G + 16 * RT - 1) / (16 * RT)) * p.own_splits) return;
    }
    const int entry = y / p.own_splits;
    w.split = y - entry * p.own_splits;
    w.splits = p.own_splits;
    constexpr int R = 16 * RT;
    if (p.num_tiles > 0) {
        const int chunks = (p.tile_rows * G + R - 1) / R;
        const int tile = entry / chunks;
        const int item = p.tile_item[tile], q0 = p.tile_q0[tile];
        if (item < 0 || item >= p.num_items) return;
        w.kind = 1;
        w.item = item;
        w.base = p.item_tok_off[item] + q0;
        w.start = p.item_start[item] + q0;
        w.first = (entry - tile * chunks) * R;
        w.count = min(p.tile_rows, p.item_len[item] - q0) * G;
        if (w.first >= w.count) return;
    } else {
        const int chunks = (G + R - 1) / R;
        const int ri = entry / chunks;
        int t = ri;
        if (p.row_ids) {
            t = p.row_ids[ri];
            if (t < 0 || t >= p.num_rows) return;
            w.slot = ri;
        }
        w.kind = 0;
        w.base = t;
        w.first = (entry - ri * chunks) * R;
        w.count = G;
        // (asked for together, by the scalar unit)
        w.item = __builtin_amdgcn_readfirstlane(p.token_item[t]);
        w.start = __builtin_amdgcn_readfirstlane(p.positions[t]);
        if (RTS > 0) w.lo = max(__builtin_amdgcn_readfirstlane(p.row_start[t]), 0);
        if ((uint32_t)w.item >= (uint32_t)p.num_items) {                   // a padding row sees no key
            w.item = 0;
            w.start = -1;
        }
    }
    tile_work<TQ, TC, HDP, RT, WHOLE>(p, w, kvh, lds);
}

// out[row, :] = sum_s w_s part_o[row, s, :] / sum_s w_s l_s, w_s = e^(m_s - max m): one wave a row and head.  (Maxima and normalisers, not the
// logarithms of their product: those round by 2^-24 of themselves, which at scores of 16 is 2^-20 of a weight.)
template <typename TQ>
__global__ __launch_bounds__(256) void tile_merge_kernel(const StTileAttention p, int rows) {
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, hd = p.head_dim;
    if (i >= (int64_t)rows * p.heads) return;
    int64_t ri = i / p.heads;
    const int64_t head = i - ri * p.heads;
    int64_t t = ri;
    if (p.num_tiles > 0) {
        const int tile = (int)(ri / p.tile_rows), j = (int)(ri - (int64_t)tile * p.tile_rows), item = p.tile_item[tile];
        if (item < 0 || item >= p.num_items || p.tile_q0[tile] + j >= p.item_len[item]) return;
        t = ri = p.item_tok_off[item] + p.tile_q0[tile] + j;
    } else if (p.row_ids) {
        t = p.row_ids[ri];
    }
    if (t < 0 || t >= p.num_rows) return;
    const int64_t at = (ri * p.heads + head) * p.slots;
    const float* parts = p.part_o + at * hd;
    float2 ml = lane < p.slots ? *reinterpret_cast<const float2*>(p.part_ml + 2 * (at + lane)) : make_float2(kFloor, 0.f);
    int slots = p.slots;
    if (p.row_start) {
        // Nothing has written the prefix's parts of a row that no group lists, or that has no prefix.  (Its place in the lists is looked for in 256 places at a time,
        // the first of them asked for with all the rest: a row's own loads are one trip to memory.)
        const int n = p.num_shared, begin = p.group_off[0], end = p.group_off[p.num_groups], start = p.row_start[t];
        int there[4];
        const auto ask = [&](int base) {
#pragma unroll
            for (int k = 0; k < 4; ++k) there[k] = p.shared_rows[min(base + 64 * k + lane, n - 1)];
        };
        ask(0);
        bool listed = false;
        for (int base = 0;; ask(base)) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int place = base + 64 * k + lane;
                listed |= there[k] == t && place >= begin && place < min(end, n);
            }
            listed = __any(listed);
            if (listed || start <= 0 || (base += 256) >= n) break;
        }
        if (!listed || start <= 0) slots = p.own_splits;
        if (lane >= slots) ml = make_float2(kFloor, 0.f);
    }
    const float weight = weight_of(ml.x, wave_max(ml.x), log2_scale(p.scale));
    const uint64_t held = __ballot(ml.y != 0.f);            // (parts without a key)
    const float sum = wave_sum(ml.y * weight);
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    for (int d = lane; d < hd; d += 64) {
        float o = 0.f;
        for (int s = 0; s < slots; ++s)
            // (read from the lane whether or not it has a dim in this turn: a shuffle gives nothing for lanes that are switched off)
            if ((held >> s) & 1) o += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), s)) * parts[(int64_t)s * hd + d];
        Elem<TQ>::store((TQ*)p.out + (t * p.heads + head) * hd + d, o * inverse);
    }
}

// The instances of a query type: for heads of up to 64, 96, 128 and 256 dims; rows in subtiles of 16: one for single tokens (a
// group's heads), MAX for tiles and long lists of rows.
template <typename TQ, typename TC, int HDP, int RT, int RTS, bool WHOLE>
int launch_tiles(const StTileAttention& p, hipStream_t stream) {
    constexpr int lds1 = tile_lds<TQ, TC, HDP, RT>(), lds2 = RTS > 0 ? tile_lds<TQ, TC, HDP, (RTS > 0 ? RTS : 1)>() : 0;
    const int G = p.heads / p.kv_heads;
    const int chunks = ((p.num_tiles > 0 ? p.tile_rows : 1) * G + 16 * RT - 1) / (16 * RT);
    const int64_t entries = (int64_t)(p.num_tiles > 0 ? p.num_tiles : p.num_entries) * chunks;
    StTileAttention q = p;
    q.shared_entries = RTS > 0 ? (int)((int64_t)p.num_shared * G / (16 * (RTS > 0 ? RTS : 1))) + p.num_groups : 0;
    const int64_t own = p.own_waves == 1 ? (entries * p.own_splits + 3) / 4 : entries * p.own_splits;
    const int64_t groups = (own + (int64_t)q.shared_entries * p.shared_splits) * p.kv_heads;
    const int64_t rows = p.num_tiles > 0 ? (int64_t)p.num_tiles * p.tile_rows : p.num_entries;
    // (a launch has less than 2^32 threads)
    ST_CHECK(entries * p.own_splits < ((int64_t)1 << 31) && groups < ((int64_t)1 << 24) && rows < ((int64_t)1 << 31) &&
             (p.slots == 1 || rows * p.heads <= ((int64_t)1 << 25)), "attention: too many rows at once");
    if (groups == 0) return 0;
    constexpr int lds = lds1 > lds2 ? lds1 : lds2;
    if constexpr (lds > 64 * 1024)
        ST_CHECK(hipFuncSetAttribute((const void*)tile_attention_kernel<TQ, TC, HDP, RT, RTS, WHOLE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess,
                 "attention: %d bytes of LDS refused", lds);
    tile_attention_kernel<TQ, TC, HDP, RT, RTS, WHOLE><<<(unsigned)groups, 256, lds, stream>>>(q);
    ST_LAUNCH_CHECK("tile_attention");
    if (p.slots > 1) {
        tile_merge_kernel<TQ><<<(unsigned)((rows * p.heads + 3) / 4), 256, 0, stream>>>(q, (int)rows);
        ST_LAUNCH_CHECK("tile_merge");
    }
    return 0;
}

// (Pages that 16 does not divide, or exponents that do not lie at multiples of four, go by subtiles of 16 rows only.)
template <typename TQ, typename TC, int HDP, int MAX>
int launch_tiles_of(const StTileAttention& p, hipStream_t stream) {
    const bool whole = p.page_size % 16 == 0 &&
                       (sizeof(TC) > 1 || ((reinterpret_cast<uintptr_t>(p.k_exp) | reinterpret_cast<uintptr_t>(p.v_exp) | (uintptr_t)p.exp_stride) & 3) == 0);
    // (rows go by MAX subtiles where a group's, or a tile's, fill more than one: 200 rows in three groups 76 us, 98 by one; 512 of a prompt behind 1,024 31, 39 by one)
    const bool many = (int64_t)p.num_shared * (p.heads / p.kv_heads) > 16 * (int64_t)p.num_groups;
    if (p.num_groups > 0) {
        if (!whole) return launch_tiles<TQ, TC, HDP, 1, 1, false>(p, stream);
        return many ? launch_tiles<TQ, TC, HDP, 1, MAX, true>(p, stream) : launch_tiles<TQ, TC, HDP, 1, 1, true>(p, stream);
    }
    if constexpr (sizeof(TC) == 1) {
        if (!whole) return launch_tiles<TQ, TC, HDP, 1, 0, false>(p, stream);
        return p.num_tiles > 0 ? launch_tiles<TQ, TC, HDP, MAX, 0, true>(p, stream) : launch_tiles<TQ, TC, HDP, 1, 0, true>(p, stream);
    }
    ST_CHECK(false, "attention: a cache of the queries' type goes by groups");
    return 0;
}

template <typename TQ, typename TC, int MAX>
int launch_tiles_by_head(const StTileAttention& p, hipStream_t stream) {
    if (p.head_dim <= 64) return launch_tiles_of<TQ, TC, 2, MAX>(p, stream);
    if (p.head_dim <= 96) return launch_tiles_of<TQ, TC, 3, MAX>(p, stream);
    if (p.head_dim <= 128) return launch_tiles_of<TQ, TC, 4, MAX>(p, stream);
    return launch_tiles_of<TQ, TC, 8, (MAX > 1 ? MAX / 2 : 1)>(p, stream);
}

// the sources that hold them: by the queries' type and the cache's
int tile_attention_bf16(const StTileAttention& p, hipStream_t stream);
int tile_attention_bf16_quant(const StTileAttention& p, hipStream_t stream);
int tile_attention_f32(const StTileAttention& p, hipStream_t stream);
int tile_attention_f32_quant(const StTileAttention& p, hipStream_t stream);

}  // namespace st
