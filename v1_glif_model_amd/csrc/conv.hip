// Short causal convolution along time, one filter of W taps per channel, forward, backward and single tick:
//   pre[t] = b + sum_k w[k] x[t - (W - 1) + k],   y[t] = act(pre[t]),   t < len
// Ticks before 0 are the state [B][W - 1][D] (zeros without one), and the state that is handed on holds the last W - 1
// inputs before `len`.  Ticks from `len` on are not read, their y is 0 and they take no part in any gradient:
//   dp[t] = dy[t] act'(pre[t]),   dx[t] = sum_k w[k] dp[t + (W - 1) - k] (+ the state's gradient where x[t] is in it)
//   dw[k] = sum_{t, b} dp[t] x[t - (W - 1) + k],   db = sum_{t, b} dp[t]
// Sequences are [T][B][D], channels next to each other: a thread owns a channel and walks a segment of ticks with its
// taps and its window of inputs in registers.
#include "seq.h"

namespace glif {
namespace {

constexpr int kMaxTaps = 8;
constexpr int kSeg = 32;   // ticks of a thread's segment

struct ConvArgs {
    const void *x, *weight, *bias, *state, *dy, *dlast;
    void *y, *last, *dx, *dweight, *dbias, *dstate;
    const int32_t *lengths;
    int64_t x_st, x_sb, dy_st, dy_sb;   // strides of tick and batch entry
    int32_t T, B, D, segs, pdt, silu;
    float *part;                        // [segs * B][W + 1][D]
};

__device__ __forceinline__ int length_of(const int32_t *lengths, int b, int T) {
    return lengths ? min(max(lengths[b], 0), T) : T;
}

// x at tick t, which may lie in the state
template <typename T, int W>
__device__ __forceinline__ float x_at(const ConvArgs &a, int t, int b, int d) {
    if (t >= 0) return to_f32(static_cast<const T *>(a.x)[t * a.x_st + b * a.x_sb + d]);
    return a.state ? to_f32(static_cast<const T *>(a.state)[(static_cast<int64_t>(b) * (W - 1) + (W - 1 + t)) * a.D + d]) : 0.0f;
}

template <typename T, int W>
__global__ void __launch_bounds__(kBlock) k_conv_fwd(ConvArgs a) {
    const int d = blockIdx.x * kBlock + threadIdx.x, b = blockIdx.z;
    if (d >= a.D) return;
    const int t0 = blockIdx.y * kSeg, t1 = min(t0 + kSeg, a.T), len = length_of(a.lengths, b, a.T);
    float w[W], win[W];
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = load_param(a.weight, a.pdt, static_cast<int64_t>(d) * W + k);
    const float bias = a.bias ? load_param(a.bias, a.pdt, d) : 0.0f;
    if (t0 < len) {
#pragma unroll
        for (int k = 1; k < W; ++k) win[k] = x_at<T, W>(a, t0 - W + k, b, d);
    }
    for (int t = t0; t < t1; ++t) {
        float y = 0.0f;
        if (t < len) {
#pragma unroll
            for (int k = 1; k < W; ++k) win[k - 1] = win[k];
            win[W - 1] = x_at<T, W>(a, t, b, d);
            y = bias;
#pragma unroll
            for (int k = 0; k < W; ++k) y = fmaf(w[k], win[k], y);
            if (a.silu) y *= sigmoid_f(y);
        }
        static_cast<T *>(a.y)[(static_cast<int64_t>(t) * a.B + b) * a.D + d] = from_f32<T>(y);
    }
    if (a.last && blockIdx.y == 0)
        for (int j = 0; j < W - 1; ++j)
            static_cast<T *>(a.last)[(static_cast<int64_t>(b) * (W - 1) + j) * a.D + d] =
                from_f32<T>(x_at<T, W>(a, len - (W - 1) + j, b, d));
}

template <typename T, int W>
__global__ void __launch_bounds__(kBlock) k_conv_bwd(ConvArgs a) {
    const int d = blockIdx.x * kBlock + threadIdx.x, b = blockIdx.z;
    if (d >= a.D) return;
    const int t0 = blockIdx.y * kSeg, t1 = min(t0 + kSeg, a.T), len = length_of(a.lengths, b, a.T);
    float w[W], win[W], dp[W], dw[W], db = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
        w[k] = load_param(a.weight, a.pdt, static_cast<int64_t>(d) * W + k);
        win[k] = dp[k] = dw[k] = 0.0f;
    }
    const float bias = a.bias ? load_param(a.bias, a.pdt, d) : 0.0f;
    if (t0 < len) {
#pragma unroll
        for (int k = 1; k < W; ++k) win[k] = x_at<T, W>(a, t0 - W + k, b, d);
    }
    const int first = blockIdx.y == 0 ? -(W - 1) : t0;   // the first tick whose gradient this segment writes
    for (int t = t0; t < t1 + W - 1; ++t) {
#pragma unroll
        for (int k = 1; k < W; ++k) dp[W - k] = dp[W - k - 1];   // dp[k] is that of tick t - k
        dp[0] = 0.0f;
        if (t < len) {
#pragma unroll
            for (int k = 1; k < W; ++k) win[k - 1] = win[k];
            win[W - 1] = x_at<T, W>(a, t, b, d);
            float g = to_f32(static_cast<const T *>(a.dy)[t * a.dy_st + b * a.dy_sb + d]);
            if (a.silu) {
                float pre = bias;
#pragma unroll
                for (int k = 0; k < W; ++k) pre = fmaf(w[k], win[k], pre);
                const float q = sigmoid_f(pre);
                g *= q * fmaf(pre, 1.0f - q, 1.0f);
            }
            dp[0] = g;
            if (t < t1) {
                db += g;
#pragma unroll
                for (int k = 0; k < W; ++k) dw[k] = fmaf(g, win[k], dw[k]);
            }
        }
        const int at = t - (W - 1);
        if (at < first) continue;
        float g = 0.0f;
        if (at < len) {
#pragma unroll
            for (int k = 0; k < W; ++k) g = fmaf(w[k], dp[k], g);
            const int j = at - (len - (W - 1));
            if (a.dlast && j >= 0) g += to_f32(static_cast<const T *>(a.dlast)[(static_cast<int64_t>(b) * (W - 1) + j) * a.D + d]);
        }
        if (at >= 0) {
            if (a.dx) static_cast<T *>(a.dx)[(static_cast<int64_t>(at) * a.B + b) * a.D + d] = from_f32<T>(g);
        } else if (a.dstate) {
            static_cast<T *>(a.dstate)[(static_cast<int64_t>(b) * (W - 1) + (W - 1 + at)) * a.D + d] = from_f32<T>(g);
        }
    }
    if (!a.part) return;
    float *part = a.part + static_cast<int64_t>(blockIdx.y * a.B + b) * (W + 1) * a.D + d;
#pragma unroll
    for (int k = 0; k < W; ++k) part[static_cast<int64_t>(k) * a.D] = dw[k];
    part[static_cast<int64_t>(W) * a.D] = db;
}

// dw and db: the segments' sums, added in order.
__global__ void __launch_bounds__(kBlock) k_conv_join(ConvArgs a, int W) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x, n = static_cast<int64_t>(W + 1) * a.D;
    if (i >= n) return;
    float s = 0.0f;
    for (int p = 0; p < a.segs * a.B; ++p) s += a.part[p * n + i];
    const int64_t k = i / a.D, d = i - k * a.D;
    if (k < W) {
        if (a.dweight) store_param(a.dweight, a.pdt, d * W + k, s);
    } else if (a.dbias) {
        store_param(a.dbias, a.pdt, d, s);
    }
}

// One tick: y from the state and x, and the state moved on by x.
template <typename T, int W>
__global__ void __launch_bounds__(kBlock) k_conv_step(ConvArgs a) {
    const int d = blockIdx.x * kBlock + threadIdx.x, b = blockIdx.y;
    if (d >= a.D) return;
    T *st = static_cast<T *>(a.last) + static_cast<int64_t>(b) * (W - 1) * a.D + d;
    T win[W];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) win[k] = st[static_cast<int64_t>(k) * a.D];
    win[W - 1] = static_cast<const T *>(a.x)[b * a.x_sb + d];
    float y = a.bias ? load_param(a.bias, a.pdt, d) : 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) y = fmaf(load_param(a.weight, a.pdt, static_cast<int64_t>(d) * W + k), to_f32(win[k]), y);
    if (a.silu) y *= sigmoid_f(y);
    static_cast<T *>(a.y)[static_cast<int64_t>(b) * a.D + d] = from_f32<T>(y);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) st[static_cast<int64_t>(k) * a.D] = win[k + 1];
}

enum Pass { kFwd, kBwd, kStep };

template <typename T, int W>
void launch(const ConvArgs &a, Pass pass, hipStream_t s) {
    const unsigned cols = static_cast<unsigned>(ceil_div(a.D, kBlock));
    const dim3 grid(cols, static_cast<unsigned>(a.segs), static_cast<unsigned>(a.B));
    if (pass == kStep) {
        hipLaunchKernelGGL((k_conv_step<T, W>), dim3(cols, static_cast<unsigned>(a.B)), dim3(kBlock), 0, s, a);
    } else if (pass == kFwd) {
        hipLaunchKernelGGL((k_conv_fwd<T, W>), grid, dim3(kBlock), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_conv_bwd<T, W>), grid, dim3(kBlock), 0, s, a);
        if (a.part)
            hipLaunchKernelGGL(k_conv_join, dim3(static_cast<unsigned>(ceil_div(static_cast<int64_t>(W + 1) * a.D, kBlock))),
                               dim3(kBlock), 0, s, a, W);
    }
}

template <typename T>
void by_taps(const ConvArgs &a, int W, Pass pass, hipStream_t s) {
    switch (W) {
        case 1: return launch<T, 1>(a, pass, s);
        case 2: return launch<T, 2>(a, pass, s);
        case 3: return launch<T, 3>(a, pass, s);
        case 4: return launch<T, 4>(a, pass, s);
        case 5: return launch<T, 5>(a, pass, s);
        case 6: return launch<T, 6>(a, pass, s);
        case 7: return launch<T, 7>(a, pass, s);
        default: return launch<T, 8>(a, pass, s);
    }
}

int check_conv(int32_t dtype, int32_t pdt, int32_t T, int32_t B, int32_t D, int32_t W) {
    if (!known_dtype(dtype) || (pdt != GLIF_F32 && pdt != dtype))
        return fail(GLIF_EINVAL, "short convolution: parameters are float32 or of x's type");
    if (T < 0 || B < 0 || B > 65535 || D < 1 || T > (1 << 20)) return fail(GLIF_EINVAL, "short convolution: T in [0, 2^20], B in [0, 65535], D >= 1");
    if (W < 1 || W > kMaxTaps) return fail(GLIF_EINVAL, "short convolution: 1 to 8 taps");
    return GLIF_OK;
}

int segs_for(int32_t T) { return std::max(1, ceil_div(T, kSeg)); }

}  // namespace
}  // namespace glif

using namespace glif;

extern "C" {

int glif_short_conv_fwd(const void *x, int64_t x_stride_t, int64_t x_stride_b, const void *weight, const void *bias,
                        const void *state, const int32_t *lengths, int32_t dtype, int32_t param_dtype, int32_t T, int32_t B,
                        int32_t D, int32_t W, int32_t silu, void *y, void *last, void *stream) {
    if (int rc = check_conv(dtype, param_dtype, T, B, D, W)) return rc;
    if (B == 0) return GLIF_OK;
    if (!weight || (T && (!x || !y))) return fail(GLIF_EINVAL, "NULL argument");
    ConvArgs a{};
    a.x = x, a.weight = weight, a.bias = bias, a.state = state, a.lengths = lengths, a.y = y, a.last = W > 1 ? last : nullptr;
    a.x_st = x_stride_t, a.x_sb = x_stride_b, a.T = T, a.B = B, a.D = D, a.segs = segs_for(T), a.pdt = param_dtype, a.silu = silu;
    GLIF_BY_DTYPE(dtype, by_taps, a, W, kFwd, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

size_t glif_short_conv_bwd_workspace(int32_t T, int32_t B, int32_t D, int32_t W) {
    if (T < 0 || B < 0 || D < 1 || W < 1) return 0;
    return static_cast<size_t>(segs_for(T)) * B * (W + 1) * D * sizeof(float) + 256;
}

int glif_short_conv_bwd(const void *dy, int64_t dy_stride_t, int64_t dy_stride_b, const void *dlast, const void *x,
                        int64_t x_stride_t, int64_t x_stride_b, const void *weight, const void *bias, const void *state,
                        const int32_t *lengths, int32_t dtype, int32_t param_dtype, int32_t T, int32_t B, int32_t D,
                        int32_t W, int32_t silu, void *dx, void *dweight, void *dbias, void *dstate, void *ws,
                        size_t ws_bytes, void *stream) {
    if (int rc = check_conv(dtype, param_dtype, T, B, D, W)) return rc;
    if (!weight || (T && B && (!x || !dy))) return fail(GLIF_EINVAL, "NULL argument");
    ConvArgs a{};
    a.x = x, a.weight = weight, a.bias = bias, a.state = state, a.lengths = lengths, a.dy = dy, a.dlast = dlast;
    a.dx = dx, a.dweight = dweight, a.dbias = dbias, a.dstate = W > 1 ? dstate : nullptr;
    a.x_st = x_stride_t, a.x_sb = x_stride_b, a.dy_st = dy_stride_t, a.dy_sb = dy_stride_b;
    a.T = T, a.B = B, a.D = D, a.segs = segs_for(T), a.pdt = param_dtype, a.silu = silu;
    if (dweight || dbias) {
        Carver c(ws, ws_bytes);
        a.part = c.take<float>(static_cast<size_t>(a.segs) * B * (W + 1) * D);
        if (!ws || !c.ok()) return fail(GLIF_ENOMEM, "short convolution: workspace too small");
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (B == 0) {
        if (a.part)
            hipLaunchKernelGGL(k_conv_join, dim3(static_cast<unsigned>(ceil_div(static_cast<int64_t>(W + 1) * D, kBlock))),
                               dim3(kBlock), 0, s, a, W);
    } else {
        GLIF_BY_DTYPE(dtype, by_taps, a, W, kBwd, s);
    }
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

int glif_short_conv_step(const void *x, int64_t x_stride_b, void *state, const void *weight, const void *bias, int32_t dtype,
                         int32_t param_dtype, int32_t B, int32_t D, int32_t W, int32_t silu, void *y, void *stream) {
    if (int rc = check_conv(dtype, param_dtype, 1, B, D, W)) return rc;
    if (B == 0) return GLIF_OK;
    if (!x || !weight || !y || (W > 1 && !state)) return fail(GLIF_EINVAL, "NULL argument");
    ConvArgs a{};
    a.x = x, a.weight = weight, a.bias = bias, a.last = state, a.y = y;
    a.x_sb = x_stride_b, a.T = 1, a.B = B, a.D = D, a.segs = 1, a.pdt = param_dtype, a.silu = silu;
    GLIF_BY_DTYPE(dtype, by_taps, a, W, kStep, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
