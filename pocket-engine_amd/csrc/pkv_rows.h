// Element types of the kernels that take rows of bf16 or fp16: two elements to
// a 32-bit word, conversions round to nearest even, sums and products in f32.
#pragma once
#include "pkv_common.h"

namespace pkv {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Bf16 {
    static constexpr uint32_t EXP = 0x7f807f80u, MANT = 0x007f007fu;  // exponent and mantissa bits of a pair
    static constexpr uint32_t ONE = 0x3f803f80u;                      // (1, 1)
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack2_hw(a, b); }
    static __device__ __forceinline__ float lo(uint32_t u) { return bf_lo(u); }
    static __device__ __forceinline__ float hi(uint32_t u) { return bf_hi(u); }
    static __device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float dot(uint32_t a, uint32_t b, float c) { return dot2(a, b, c); }
};
struct Fp16 {
    static constexpr uint32_t EXP = 0x7c007c00u, MANT = 0x03ff03ffu;
    static constexpr uint32_t ONE = 0x3c003c00u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {  // round to nearest even
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
    }
    static __device__ __forceinline__ float lo(uint32_t u) { return (float)__builtin_bit_cast(f16x2, u).x; }
    static __device__ __forceinline__ float hi(uint32_t u) { return (float)__builtin_bit_cast(f16x2, u).y; }
    static __device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                      0);
    }
    static __device__ __forceinline__ float dot(uint32_t a, uint32_t b, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b), c, false);
    }
};

}  // namespace pkv
