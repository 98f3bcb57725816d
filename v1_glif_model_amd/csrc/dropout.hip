// Dropout whose mask is never stored: element i is kept where the float32 uniform u of word offset + i of the Philox
// stream `seed` (philox.h) is >= p, and then scaled by 1 / (1 - p):
//   y[i] = (u(seed, offset + i) >= p ? x[i] * scale : 0) + residual[i]
// The gradient is the same function of dy, without a residual.  A dropped element is 0 whatever x holds.
//
// Bound by memory where a residual or float32 is read, by the generator (10 rounds of two 32 x 32 products for 4 elements)
// where only 16 bits come in and go out: 65.5M bfloat16 elements 67 us with a residual (5.8 TB/s), 60 without; float32 89 us.
#include <cmath>

#include "philox.h"
#include "seq.h"

namespace glif {
namespace {

struct DropArgs {
    const void *x, *residual;
    void *y;
    int64_t n;
    uint64_t seed, offset;
    uint32_t drop;     // dropped where the word's upper 24 bits are below it
    float scale;
};

// A thread takes the elements of 16 bytes' worth of the stream's words (two blocks of the generator for 16-bit types, one
// for float32), so that no block is made twice; x starts anywhere among them.  u = (word >> 8) 2^-24 < p is decided on
// whole numbers.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_dropout(DropArgs a) {
    constexpr int V = kVecBytes16<T>;
    typedef Vec<T, V> vec;
    const T *x = static_cast<const T *>(a.x), *res = static_cast<const T *>(a.residual);
    T *y = static_cast<T *>(a.y);
    const int64_t shift = static_cast<int64_t>(a.offset % V), groups = (a.n + shift + V - 1) / V;
    const uint64_t first = a.offset / V;
    for (int64_t g = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; g < groups; g += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t i = g * V - shift;
        const bool whole = i >= 0 && i + V <= a.n;
        vec v = {}, q = {};
        if (whole) {
            v = *reinterpret_cast<const vec *>(x + i);
            if (res) q = *reinterpret_cast<const vec *>(res + i);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (i + e >= 0 && i + e < a.n) {
                    v[e] = x[i + e];
                    if (res) q[e] = res[i + e];
                }
        }
        uint32_t w[V / 4][4];
#pragma unroll
        for (int b = 0; b < V / 4; ++b) philox_block(a.seed, (first + static_cast<uint64_t>(g)) * (V / 4) + b, w[b]);
        vec o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float f = w[e / 4][e % 4] >> 8 < a.drop ? 0.0f : to_f32(static_cast<T>(v[e])) * a.scale;
            if (res) f += to_f32(static_cast<T>(q[e]));
            o[e] = from_f32<T>(f);
        }
        if (whole) {
            *reinterpret_cast<vec *>(y + i) = o;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (i + e >= 0 && i + e < a.n) y[i + e] = o[e];
        }
    }
}

template <typename T>
void run_dropout(const DropArgs &a, hipStream_t s) {
    constexpr int V = kVecBytes16<T>;
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((a.n + V - 1) / V / kBlock + 1, 32768));
    hipLaunchKernelGGL(k_dropout<T>, dim3(blocks), dim3(kBlock), 0, s, a);
}

}  // namespace
}  // namespace glif

using namespace glif;

extern "C" int glif_dropout(const void *x, const void *residual, int32_t dtype, int64_t n, double p, uint64_t seed,
                            uint64_t offset, void *y, void *stream) {
    if (n < 0 || !known_dtype(dtype)) return fail(GLIF_EINVAL, "dropout: n must be >= 0 and the type one of glif_dtype");
    if (!(p >= 0.0 && p <= 1.0)) return fail(GLIF_EINVAL, "dropout: p must be in [0, 1]");
    if (n == 0) return GLIF_OK;
    if (!x || !y) return fail(GLIF_EINVAL, "NULL argument");
    // u < p, u = (word >> 8) 2^-24 and p in float32: word >> 8 < ceil(p 2^24)
    DropArgs a{x, residual, y, n, seed, offset, static_cast<uint32_t>(std::ceil(static_cast<double>(static_cast<float>(p)) * 16777216.0)),
               p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.0f};
    GLIF_BY_DTYPE(dtype, run_dropout, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}
