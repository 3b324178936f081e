// The cache's 8-bit entries: e4m3 (four exponent bits, three of fraction, no infinities, all ones is NaN) times a power of two that the
// elements of a token's head share.  The power is kept as a float's exponent field: 2^(e - 127), e from 1 to 254, so that its bits
// are e << 23.  It is the smallest with which the largest element is at most 448, the largest finite e4m3: multiplying by it
// or its inverse rounds nothing, the one rounding is that to e4m3 (to nearest even, at most 2^-4 of an element down to 2^-15 of the
// largest, 2^-10 of the unit 2^(e - 127) below).
#pragma once

#include "common.h"

namespace st {

struct e4m3_t { uint8_t bits; };

// exponent field for the largest finite magnitude of a vector (its bits, sign cleared); 448 = 1.75 * 2^8
__host__ __device__ inline int unit_exponent(uint32_t largest) {
    if (largest == 0) return 127;
    const int e = (int)(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u);
    return e < 1 ? 1 : e;
}

// four floats -> four e4m3 in a register (hardware convert, to nearest even; magnitudes above 464 and NaN give NaN)
__device__ inline uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
    return (uint32_t)v;
}
typedef float float2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
// the upper or lower two of four e4m3 as floats
template <bool UPPER>
__device__ inline float2v e4m3x2_to_floats(uint32_t v) { return __builtin_amdgcn_cvt_pk_f32_fp8((int)v, UPPER); }
// as two bfloat16 in a register, times `unit` (a power of two): exact within bfloat16's range
template <bool UPPER>
__device__ inline uint32_t e4m3x2_to_bf16x2(uint32_t v, float unit) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, unit, UPPER));
}

}  // namespace st
