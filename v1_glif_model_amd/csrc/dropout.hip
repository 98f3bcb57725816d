// Dropout whose mask is never stored: element i is kept where the float32 uniform u of word offset + i of the Philox
// stream `seed` (philox.h) is >= p, and then scaled by 1 / (1 - p):
//   y[i] = (u(seed, offset + i) >= p ? x[i] * scale : 0) + residual[i]
// The gradient is the same function of dy, without a residual.  A dropped element is 0 whatever x holds.
#include "philox.h"
#include "seq.h"

namespace glif {
namespace {

struct DropArgs {
    const void *x, *residual;
    void *y;
    int64_t n;
    uint64_t seed, offset;
    float p, scale;
};

template <typename T>
__global__ void __launch_bounds__(kBlock) k_dropout(DropArgs a) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < a.n; i += stride) {
        const bool keep = philox_uniform(a.seed, a.offset + static_cast<uint64_t>(i)) >= a.p;
        float v = keep ? to_f32(static_cast<const T *>(a.x)[i]) * a.scale : 0.0f;
        if (a.residual) v += to_f32(static_cast<const T *>(a.residual)[i]);
        static_cast<T *>(a.y)[i] = from_f32<T>(v);
    }
}

template <typename T>
void run_dropout(const DropArgs &a, hipStream_t s) {
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((a.n + kBlock - 1) / kBlock, 8192));
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
    DropArgs a{x, residual, y, n, seed, offset, static_cast<float>(p), p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.0f};
    if (p == 1.0) a.p = 2.0f;   // above every uniform
    GLIF_BY_DTYPE(dtype, run_dropout, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}
