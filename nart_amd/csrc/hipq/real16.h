// 16-bit floats in the kernels of the language-model operators: conversions and matrix instructions, by type.  gfx950 only.
#pragma once

#include "common.h"

namespace hipq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

static inline bool is_real16(int type) { return type == HIPQ_REAL_F16 || type == HIPQ_REAL_BF16; }

template <int TYPE>
struct Real16;

template <>
struct Real16<HIPQ_REAL_BF16> {
    __device__ static __forceinline__ float low(uint32_t pair) { return __builtin_bit_cast(float, pair << 16); }
    __device__ static __forceinline__ float high(uint32_t pair) { return __builtin_bit_cast(float, pair & 0xffff0000u); }
    // nearest even, a in the low half
    __device__ static __forceinline__ uint32_t pack(float a, float b)
    {
        const bf16x2 v = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    // of numbers that the type holds
    __device__ static __forceinline__ uint32_t pack_exact(float a, float b) { return pack(a, b); }
    // 16 x 16 products over k = 32: a lane holds row (a) or column (b) lane % 16, k = 8 (lane / 16) + 0..7; of the result column
    // lane % 16, rows 4 (lane / 16) + 0..3
    __device__ static __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};

template <>
struct Real16<HIPQ_REAL_F16> {
    __device__ static __forceinline__ float low(uint32_t pair) { return (float)__builtin_bit_cast(f16x2, pair)[0]; }
    __device__ static __forceinline__ float high(uint32_t pair) { return (float)__builtin_bit_cast(f16x2, pair)[1]; }
    __device__ static __forceinline__ uint32_t pack(float a, float b)
    {
        const f16x2 v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    // one instruction, which rounds to zero, instead of three
    __device__ static __forceinline__ uint32_t pack_exact(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b)); }
    __device__ static __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// 2^v in one instruction (1 unit in the last place; results under 2^-126 are 0)
__device__ static __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

} // namespace hipq
