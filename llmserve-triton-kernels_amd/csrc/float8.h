// 8-bit floating point (e4m3: 4 bits of exponent, 3 behind the leading one, largest 448, one NaN a sign) with a power of two as scale
// for each block of 128: a value stands for e4m3 * 2^s.  A scale is stored as s + 127 in a byte (255: NaN), which is how the matrix
// instructions of gfx950 take it, so they apply it themselves and sums run over all of K in 32 bits.
//
// s is the smallest integer >= -126 for which nothing in the block is beyond 448 * 2^s.  Multiplying by 2^-s is exact (but for 32-bit
// numbers that it takes below 2^-126, which are far below half of e4m3's smallest step), so a value is rounded once, by the conversion.
// A block that holds a NaN or an infinity has the scale NaN and NaN as values: what is multiplied with it is NaN.
#pragma once

#include "common.h"

#include <utility>

#define F8_BLOCK 128

typedef __attribute__((ext_vector_type(4))) uint32_t f8_u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t f8_u32x2;
// The same at the address of a number of 2 or 4 bytes.  The memory takes any; asked for as if they began on 16 the compiler may use what that implies.
typedef f8_u32x4 __attribute__((aligned(2))) f8_u32x4_at2;
typedef f8_u32x4 __attribute__((aligned(4))) f8_u32x4_at4;
typedef f8_u32x2 __attribute__((aligned(2))) f8_u32x2_at2;

// The scale of a block as a byte, from the bits of its largest magnitude (NaN and infinity have the largest bits).
// 448 = 1.75 * 2^8: of the magnitudes with one exponent those up to 1.75 times the power of two need 8 less than it, the others 7 less.
__device__ __forceinline__ uint32_t f8_scale_byte(uint32_t most_bits) {
    const int exponent = (int)(most_bits >> 23);
    const int byte = exponent - 8 + ((most_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return exponent == 255 ? 255u : (uint32_t)max(byte, 1);
}

// 2^-s of a scale byte; NaN for the byte of a NaN.
__device__ __forceinline__ float f8_inverse(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : (254u - byte) << 23); }

// Four numbers, already multiplied by 2^-s, to e4m3, the first in the lowest byte.
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
#else
    return 0;
#endif
}

// The largest of a number of the 16 lanes of a row (lanes 16 i .. 16 i + 15), for all of them.
__device__ __forceinline__ uint32_t f8_max16(uint32_t v) {
#if defined(__HIP_DEVICE_COMPILE__)
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // (rotated by 8, 4, 2 and 1 lanes)
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
#endif
    return v;
}

typedef __attribute__((ext_vector_type(8))) __bf16 f8_bf16x8;

// 8 values with their scale as bfloat16 numbers, exactly (3 bits behind the leading one, and bfloat16 has 32-bit's exponents).
__device__ __forceinline__ f8_bf16x8 f8_numbers(uint32_t lo, uint32_t hi, float scale) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
#if defined(__HIP_DEVICE_COMPILE__)
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return (f8_bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#else
    return (f8_bf16x8){};
#endif
}

// 2^s of a scale byte as a number; NaN for the byte of a NaN.
__device__ __forceinline__ float f8_scale(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23); }

__device__ __forceinline__ uint32_t f8_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// x / (1 + exp(-x)) of a 32-bit number, by the steps that common.h has for bfloat16 ones: the hardware's exp2 and reciprocal with one Newton step (an expf
// and a division are some 35 instructions, these 9).  The exponent x log2(e) is rounded once, at its size, so the result is some 2 units of 2^-24 off for x
// above 0, 9 down to -10, 30 down to -30 and 65 down to -88, where it is 2^-121: at most 4e-6 of it, beside the 2^-4 or 2^-8 of what it is rounded to
// behind.  Numerator and denominator are a quarter of what they stand for, and bounded, so that no reciprocal is a denormal number; x
// below -89 gives -0, NaN and -infinity NaN, as the formula does.
__device__ __forceinline__ float f8_silu(float x) { return silu_of_bf16(x); }

// gated units, in 32 bits: 0 SiLU, 1 clamped, 3 gelu (the numbers of the product kernels).  A NaN stays one, so it is no fminf that clamps.
__device__ __forceinline__ float f8_unit(float gate, float up, int unit, float limit) {
    if (unit == 1) {
        const float g = gate > limit ? limit : gate, u = up > limit ? limit : up < -limit ? -limit : up;
        return g / (1.f + expf(-1.702f * g)) * (u + 1.f);
    }
    if (unit == 3) return gelu_tanh(gate) * up;
    return f8_silu(gate) * up;
}

// f(Number<0>()), ..., f(Number<N - 1>()): a loop whose places the compiler knows from the start.
template <typename F, int... I>
__device__ __forceinline__ void f8_each(F&& f, std::integer_sequence<int, I...>) {
    (f(Number<I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void f8_for(F&& f) {
    f8_each(f, std::make_integer_sequence<int, N>());
}

// Raises how much of LDS a kernel may ask for, once on each device (`set`: the kernel's own, of 64).
static inline int f8_raise_lds(const void* kernel, int bytes, bool* set) {
    int dev = 0;
    LLMS_HIP_CHECK(hipGetDevice(&dev));
    if (dev < 64 && set[dev]) return 0;
    LLMS_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev < 64) set[dev] = true;
    return 0;
}
