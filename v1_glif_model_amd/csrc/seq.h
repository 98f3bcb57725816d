// Shared pieces of the sequence operators (layer norm, dropout, linear, short convolution, state space scan): the
// activation types, vectors of them, and sums over lanes.
#pragma once

#include "glif_internal.h"

namespace glif {

using f32 = float;
using bf16 = __bf16;
using f16 = _Float16;

// V elements of T at once.  The alignment is the element's: rows of odd lengths start anywhere, and gfx950 loads and
// stores dwords at any address (the ABI's unaligned access mode).
template <typename T, int V>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <typename T, int V>
using Vec = typename VecOf<T, V>::type;

// Results of more bytes than this go past the caches: these would not hold them for their reader anyway, and keep what the
// kernel itself reads again.
constexpr int64_t kPastCaches = int64_t(96) << 20;

// Blocks of `threads` that one launch can have: its threads are counted in 32 bits.
constexpr int64_t blocks_at_once(int threads) { return (int64_t(1) << 31) / threads; }

template <typename T>
constexpr int kVecBytes16 = 16 / static_cast<int>(sizeof(T));   // elements in a 16-byte access

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return static_cast<T>(v);   // to nearest even
}

inline bool known_dtype(int32_t dt) { return dt == GLIF_F32 || dt == GLIF_BF16 || dt == GLIF_F16; }
inline size_t dtype_size(int32_t dt) { return dt == GLIF_F32 ? 4 : 2; }

// Parameters (weights of a norm, taps, biases) are float32 or of the activations' type; they are few, so their type is
// read at run time.
__device__ __forceinline__ float load_param(const void *p, int32_t dt, int64_t i) {
    if (dt == GLIF_F32) return static_cast<const float *>(p)[i];
    if (dt == GLIF_BF16) return to_f32(static_cast<const bf16 *>(p)[i]);
    return to_f32(static_cast<const f16 *>(p)[i]);
}
__device__ __forceinline__ void store_param(void *p, int32_t dt, int64_t i, float v) {
    if (dt == GLIF_F32) static_cast<float *>(p)[i] = v;
    else if (dt == GLIF_BF16) static_cast<bf16 *>(p)[i] = from_f32<bf16>(v);
    else static_cast<f16 *>(p)[i] = from_f32<f16>(v);
}

// Sum over the wave, in every lane (a fixed tree: reproducible).
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) v += __shfl_xor(v, m, kWave);
    return v;
}

// sigmoid by the hardware's exponential and reciprocal (each within an ulp; a division in full takes ten instructions):
// exp(-x) overflows to infinity for x < -88, where the reciprocal is the right 0.
__device__ __forceinline__ float sigmoid_f(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// The call's launcher by activation type: FN<T>(args...).
#define GLIF_BY_DTYPE(dt, FN, ...)                        \
    ((dt) == GLIF_F32    ? FN<f32>(__VA_ARGS__)           \
     : (dt) == GLIF_BF16 ? FN<bf16>(__VA_ARGS__)          \
                         : FN<f16>(__VA_ARGS__))

}  // namespace glif
