// The matrix instructions that the sequence operators use, by the operands' type.
#pragma once

#include "seq.h"

namespace glif {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// One matrix instruction's operands from a row-major LDS row of 32 k's: 16-bit types take 8 consecutive k's a lane.
template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    typedef bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<f16> {
    typedef f16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
// float32: lane l holds four consecutive k's, element i of every lane makes one 16x16x4 product (the order of the k's in
// a sum is free, as long as both operands have it)
template <>
struct Mma<f32> {
    typedef f32 frag __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

}  // namespace glif
