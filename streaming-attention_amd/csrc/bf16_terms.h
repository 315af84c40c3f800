// Values as bf16 MFMA operands: three bf16 terms of an fp32 one, one of an 8-bit
// cache's.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sa {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTerms = 3;   // |x - sum of the terms| <= 2^-27 |x|

// t_0 = rne(x), t_i = rne(x - t_0 - ... - t_{i-1}) of 8 values (each
// difference is exact in fp32).
__device__ __forceinline__ void split_terms(f32x4_t a, f32x4_t b, bf16x8_t (&t)[kTerms]) {
    f32x2_t v[4] = {{a[0], a[1]}, {a[2], a[3]}, {b[0], b[1]}, {b[2], b[3]}};
#pragma unroll
    for (int i = 0; i < kTerms; ++i) {
        u32x4_t packed;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t bits = __builtin_bit_cast(uint32_t, __builtin_convertvector(v[e], bf16x2_t));
            packed[e] = bits;
            v[e] -= f32x2_t{__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u)};
        }
        t[i] = __builtin_bit_cast(bf16x8_t, packed);
    }
}

// Eight codes in e4m3, times a power of two: exact.
__device__ __forceinline__ bf16x8_t codes_bf16x8(uint32_t lo, uint32_t hi, float scale) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return __builtin_bit_cast(bf16x8_t, u32x4_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                                                __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)});
}
// The scale that a byte of an 8-bit cache stands for.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Four values, rounded to bf16 where p is of that.
__device__ __forceinline__ void store4(float* p, f32x4_t v) { *reinterpret_cast<f32x4_t*>(p) = v; }
__device__ __forceinline__ void store4(uint16_t* p, f32x4_t v) {
    const bf16x2_t lo = __builtin_convertvector(f32x2_t{v[0], v[1]}, bf16x2_t);
    const bf16x2_t hi = __builtin_convertvector(f32x2_t{v[2], v[3]}, bf16x2_t);
    *reinterpret_cast<uint2*>(p) = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

}  // namespace sa
