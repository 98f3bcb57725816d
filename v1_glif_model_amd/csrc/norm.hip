// Layer norm over the last axis, forward and backward.  Per row of D elements:
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  xh = (x - mean) rstd
//   y = xh w + b
//   dx = rstd (dyw - mean(dyw) - xh mean(dyw xh)),  dyw = dy w;   dw = sum_rows dy xh,  db = sum_rows dy
// The backward takes the statistics from x itself, so the forward leaves nothing behind.  All sums are float32 in a
// fixed order; y and dx are rounded once.
#include "seq.h"

namespace glif {

namespace {

constexpr int kParts = 256;   // row chunks of the parameter gradients, at most

struct NormArgs {
    const void *x, *dy, *weight, *bias;
    void *y, *dx, *dweight, *dbias;
    int64_t rows, D, x_stride, dy_stride;
    int32_t pdt;
    float eps;
    float2 *stat;      // [rows] mean, rstd (backward)
    float *part;       // [2][parts][D]
    int32_t parts;
};

__device__ inline float block_sum(float v, float *red) {
    v = wave_sum(v);
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < static_cast<int>(blockDim.x) / kWave; ++i) s += red[i];
    __syncthreads();
    return s;
}

template <typename T>
__device__ inline float2 row_stats(const T *x, int64_t D, float eps, float *red) {
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < D; i += blockDim.x) s += to_f32(x[i]);
    const float mean = block_sum(s, red) / static_cast<float>(D);
    float q = 0.0f;
    for (int64_t i = threadIdx.x; i < D; i += blockDim.x) {
        const float d = to_f32(x[i]) - mean;
        q = fmaf(d, d, q);
    }
    return make_float2(mean, 1.0f / sqrtf(block_sum(q, red) / static_cast<float>(D) + eps));
}

template <typename T>
__global__ void __launch_bounds__(kBlock) k_norm_fwd(NormArgs a) {
    __shared__ float red[kBlock / kWave];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
        T *y = static_cast<T *>(a.y) + r * a.D;
        const float2 st = row_stats(x, a.D, a.eps, red);
        for (int64_t i = threadIdx.x; i < a.D; i += blockDim.x) {
            const float w = a.weight ? load_param(a.weight, a.pdt, i) : 1.0f;
            const float b = a.bias ? load_param(a.bias, a.pdt, i) : 0.0f;
            y[i] = from_f32<T>(fmaf((to_f32(x[i]) - st.x) * st.y, w, b));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kBlock) k_norm_dx(NormArgs a) {
    __shared__ float red[kBlock / kWave];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride, *dy = static_cast<const T *>(a.dy) + r * a.dy_stride;
        const float2 st = row_stats(x, a.D, a.eps, red);
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t i = threadIdx.x; i < a.D; i += blockDim.x) {
            const float g = to_f32(dy[i]) * (a.weight ? load_param(a.weight, a.pdt, i) : 1.0f);
            s1 += g;
            s2 = fmaf(g, (to_f32(x[i]) - st.x) * st.y, s2);
        }
        s1 = block_sum(s1, red) / static_cast<float>(a.D);
        s2 = block_sum(s2, red) / static_cast<float>(a.D);
        if (threadIdx.x == 0) a.stat[r] = st;
        if (!a.dx) continue;
        T *dx = static_cast<T *>(a.dx) + r * a.D;
        for (int64_t i = threadIdx.x; i < a.D; i += blockDim.x) {
            const float g = to_f32(dy[i]) * (a.weight ? load_param(a.weight, a.pdt, i) : 1.0f);
            dx[i] = from_f32<T>(st.y * (g - s1 - (to_f32(x[i]) - st.x) * st.y * s2));
        }
    }
}

// A thread per column over one chunk of rows.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_norm_dparam(NormArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (i >= a.D) return;
    const int64_t r0 = a.rows * blockIdx.y / a.parts, r1 = a.rows * (blockIdx.y + 1) / a.parts;
    float dw = 0.0f, db = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float2 st = a.stat[r];
        const float g = to_f32(static_cast<const T *>(a.dy)[r * a.dy_stride + i]);
        dw = fmaf(g, (to_f32(static_cast<const T *>(a.x)[r * a.x_stride + i]) - st.x) * st.y, dw);
        db += g;
    }
    a.part[static_cast<int64_t>(blockIdx.y) * a.D + i] = dw;
    a.part[static_cast<int64_t>(a.parts + blockIdx.y) * a.D + i] = db;
}

__global__ void __launch_bounds__(kBlock) k_norm_join(NormArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (i >= a.D) return;
    float dw = 0.0f, db = 0.0f;
    for (int p = 0; p < a.parts; ++p) {
        dw += a.part[static_cast<int64_t>(p) * a.D + i];
        db += a.part[static_cast<int64_t>(a.parts + p) * a.D + i];
    }
    if (a.dweight) store_param(a.dweight, a.pdt, i, dw);
    if (a.dbias) store_param(a.dbias, a.pdt, i, db);
}

int parts_for(int64_t rows) { return static_cast<int>(std::min<int64_t>(std::max<int64_t>(rows / 16, 1), kParts)); }

void carve(Carver &c, NormArgs &a, bool param) {
    a.parts = parts_for(a.rows);
    a.stat = c.take<float2>(static_cast<size_t>(a.rows));
    if (param) a.part = c.take<float>(static_cast<size_t>(2 * a.parts * a.D));
}

dim3 row_grid(int64_t rows) { return dim3(static_cast<unsigned>(std::min<int64_t>(rows, 1 << 20))); }

template <typename T>
void run_fwd(const NormArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(k_norm_fwd<T>, row_grid(a.rows), dim3(kBlock), 0, s, a);
}

template <typename T>
void run_bwd(const NormArgs &a, hipStream_t s) {
    const unsigned cols = static_cast<unsigned>(ceil_div(a.D, kBlock));
    if (a.rows) hipLaunchKernelGGL(k_norm_dx<T>, row_grid(a.rows), dim3(kBlock), 0, s, a);
    if (!a.dweight && !a.dbias) return;
    hipLaunchKernelGGL(k_norm_dparam<T>, dim3(cols, static_cast<unsigned>(a.parts)), dim3(kBlock), 0, s, a);
    hipLaunchKernelGGL(k_norm_join, dim3(cols), dim3(kBlock), 0, s, a);
}

int check_norm(int64_t rows, int64_t D, int32_t dtype, int32_t pdt, float eps) {
    if (rows < 0 || D < 1 || D >= (int64_t(1) << 31) || rows >= (int64_t(1) << 40))
        return fail(GLIF_EINVAL, "layer norm: rows must be >= 0 and 1 <= D < 2^31");
    if (!known_dtype(dtype) || (pdt != GLIF_F32 && pdt != dtype))
        return fail(GLIF_EINVAL, "layer norm: parameters are float32 or of x's type");
    if (!(eps >= 0.0f)) return fail(GLIF_EINVAL, "layer norm: eps must be >= 0");
    return GLIF_OK;
}

}  // namespace
}  // namespace glif

using namespace glif;

extern "C" {

int glif_layer_norm_fwd(const void *x, int64_t x_stride, const void *weight, const void *bias, int32_t dtype,
                        int32_t param_dtype, int64_t rows, int64_t D, float eps, void *y, void *stream) {
    if (int rc = check_norm(rows, D, dtype, param_dtype, eps)) return rc;
    if (rows == 0) return GLIF_OK;
    if (!x || !y) return fail(GLIF_EINVAL, "NULL argument");
    NormArgs a{};
    a.x = x, a.weight = weight, a.bias = bias, a.y = y;
    a.rows = rows, a.D = D, a.x_stride = x_stride, a.pdt = param_dtype, a.eps = eps;
    GLIF_BY_DTYPE(dtype, run_fwd, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

size_t glif_layer_norm_bwd_workspace(int64_t rows, int64_t D, int32_t want_params) {
    if (rows < 0 || D < 1) return 0;
    NormArgs a{};
    a.rows = rows, a.D = D;
    Carver c(nullptr, 0);
    carve(c, a, want_params != 0);
    return c.mark();
}

int glif_layer_norm_bwd(const void *dy, int64_t dy_stride, const void *x, int64_t x_stride, const void *weight,
                        int32_t dtype, int32_t param_dtype, int64_t rows, int64_t D, float eps, void *dx, void *dweight,
                        void *dbias, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_norm(rows, D, dtype, param_dtype, eps)) return rc;
    if (!dx && !dweight && !dbias) return GLIF_OK;
    if (rows && (!x || !dy)) return fail(GLIF_EINVAL, "NULL argument");
    NormArgs a{};
    a.x = x, a.dy = dy, a.weight = weight, a.dx = dx, a.dweight = dweight, a.dbias = dbias;
    a.rows = rows, a.D = D, a.x_stride = x_stride, a.dy_stride = dy_stride, a.pdt = param_dtype, a.eps = eps;
    Carver c(ws, ws_bytes);
    carve(c, a, dweight || dbias);
    if (!c.ok() || !ws) return fail(GLIF_ENOMEM, "layer norm: workspace too small");
    GLIF_BY_DTYPE(dtype, run_bwd, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
