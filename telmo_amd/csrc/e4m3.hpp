// Values in eight bits (e4m3: sign, four bits of exponent, three of mantissa; up to 448, no infinities, NaN 0x7f and 0xff)
// and the power of two that a group of them shares.
//
// A group's exponent e is the least one with |x| <= 448 2^e for its finite values, from E4M3_LOWEST on, and each value is
// x 2^-e rounded to nearest, ties to even; what is not finite is NaN. A power of two costs a floating format nothing in
// relative precision (half a step, 2^-4), scales exactly, and leaves each value exact in bf16.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tg {

struct e4m3 {
    uint8_t bits;
};

constexpr int E4M3_LOWEST = -100;

// 2^e for the exponents that groups have; below -126 2^-126.
__host__ __device__ __forceinline__ float two_to(int e) {
    const uint32_t bits = (uint32_t)((e < -126 ? -126 : e) + 127) << 23;
    return __builtin_bit_cast(float, bits);
}

// The exponent of a group whose largest finite |x| has these bits: with x = m 2^b, m in [1, 2), 448 = 1.75 2^8. Values
// that f32 holds as subnormal lie far below the lowest exponent.
__host__ __device__ __forceinline__ int e4m3_exponent(uint32_t top) {
    const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffff) > 0x600000 ? 1 : 0);
    return e < E4M3_LOWEST ? E4M3_LOWEST : e;
}

// |x| as bits, 0 where it is not finite: what a group's largest is taken over.
__device__ __forceinline__ uint32_t e4m3_size(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

__device__ __forceinline__ float e4m3_to_f32(e4m3 x) { return __builtin_amdgcn_cvt_f32_fp8((int)x.bits, 0); }

// Four values under 2^-e (`down`), packed. An infinity becomes NaN before it is rounded: the conversion would take it for
// the largest value. f32's largest values round to 240 2^120 at most: 256 2^120 would have no f32.
__device__ __forceinline__ float e4m3_input(float x, float down) {
    const float y = __builtin_amdgcn_fmed3f(x, -0x1.ep127f, 0x1.ep127f);
    return x - x == 0.0f ? y * down : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t e4m3_pack(float a, float b, float c, float d, float down) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_input(a, down), e4m3_input(b, down), 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_input(c, down), e4m3_input(d, down), r, true);
    return (uint32_t)r;
}

// The two bf16 values of a word's lower (upper) half, times 2^e (`up`): exact.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <bool UPPER>
__device__ __forceinline__ uint32_t e4m3_widen(uint32_t word, float up) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, up, UPPER));
}

}  // namespace tg
