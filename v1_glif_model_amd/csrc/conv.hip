// Short causal convolution along time, one filter of W taps per channel, forward, backward and single tick:
//   pre[t] = b + sum_k w[k] x[t - (W - 1) + k],   y[t] = act(pre[t]),   t < len
// Ticks before 0 are the state [B][W - 1][D] (zeros without one), and the state that is handed on holds the last W - 1
// inputs before `len`.  Ticks from `len` on are not read, their y is 0 and they take no part in any gradient:
//   dp[t] = dy[t] act'(pre[t]),   dx[t] = sum_k w[k] dp[t + (W - 1) - k] (+ the state's gradient where x[t] is in it)
//   dw[k] = sum_{t, b} dp[t] x[t - (W - 1) + k],   db = sum_{t, b} dp[t]
// Sequences are [T][B][D], channels next to each other.  A thread owns a few neighbouring channels and walks a segment of ticks,
// four at a time with the next four on their way, its taps and its window of inputs in registers; a block is C such threads
// side by side by 256 / C segments, whose sums of dw and db it adds up.  Bound by memory: x in and y out, x and dy in and dx
// out.  The last W - 1 ticks' inputs of the segment before are read again, from cache.
#include "seq.h"

namespace glif {
namespace {

constexpr int kMaxTaps = 8;
constexpr int kAhead = 4;   // ticks at a time

struct ConvArgs {
    const void *x, *weight, *bias, *state, *dy, *dlast;
    void *y, *last, *dx, *dweight, *dbias, *dstate;
    const int32_t *lengths;
    int64_t x_st, x_sb, dy_st, dy_sb;   // strides of tick and batch entry
    int32_t T, B, D, W, pdt, silu;
    int32_t C, seg, segs;               // threads side by side (a power of 2), ticks of a segment, segments
    int32_t parts;
    float *part;                        // [parts][W + 1][D]
};

__device__ __forceinline__ int length_of(const int32_t *lengths, int b, int T) {
    return lengths ? min(max(lengths[b], 0), T) : T;
}

// The channels of a thread: V from c on, `have` of which exist.
template <typename T, int V>
struct Chan {
    typedef Vec<T, V> vec;
    int c, have, seg;
    __device__ __forceinline__ Chan(const ConvArgs &a) {
        c = (blockIdx.x * a.C + threadIdx.x % a.C) * V;
        have = min(V, a.D - c);
        seg = blockIdx.y * (kBlock / a.C) + threadIdx.x / a.C;
    }
    __device__ __forceinline__ vec load(const T *p) const {
        if (have == V) return *reinterpret_cast<const vec *>(p + c);
        vec v = {};
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < have) v[e] = p[c + e];
        return v;
    }
    __device__ __forceinline__ void store(T *p, const float (&f)[V]) const {
        vec v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = from_f32<T>(f[e]);
        if (have == V) {
            *reinterpret_cast<vec *>(p + c) = v;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < have) p[c + e] = v[e];
        }
    }
    template <int W>
    __device__ __forceinline__ void taps(float (&w)[W][V], float (&bias)[V], const ConvArgs &a) const {
        if (a.pdt == GLIF_F32 && have == V) {
            const Vec<float, 4> *p = reinterpret_cast<const Vec<float, 4> *>(static_cast<const float *>(a.weight) + static_cast<int64_t>(c) * W);
            float flat[V * W];
#pragma unroll
            for (int i = 0; i < V * W / 4; ++i) {
                const Vec<float, 4> q = p[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) flat[4 * i + j] = q[j];
            }
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int k = 0; k < W; ++k) w[k][e] = flat[e * W + k];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int k = 0; k < W; ++k) w[k][e] = e < have ? load_param(a.weight, a.pdt, static_cast<int64_t>(c + e) * W + k) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) bias[e] = a.bias && e < have ? load_param(a.bias, a.pdt, c + e) : 0.0f;
    }
};

// x at tick t, which may lie in the state
template <typename T, int V, int W>
__device__ __forceinline__ Vec<T, V> x_at(const ConvArgs &a, const Chan<T, V> &me, int t, int b) {
    if (t >= 0) return me.load(static_cast<const T *>(a.x) + t * a.x_st + b * a.x_sb);
    if (a.state) return me.load(static_cast<const T *>(a.state) + (static_cast<int64_t>(b) * (W - 1) + (W - 1 + t)) * a.D);
    return {};
}

// W - 1 ticks before the segment, then kAhead of it at a time
template <typename T, int V, int W>
struct Window {
    float x[W - 1 + kAhead][V];
    __device__ __forceinline__ void set(int i, Vec<T, V> v) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = to_f32(static_cast<T>(v[e]));
    }
    __device__ __forceinline__ void move() {
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) x[i][e] = x[i + kAhead][e];
    }
};

// 500 x 32 x 2048 bfloat16, 4 taps, with SiLU: 29 us, 4.5 TB/s.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kBlock) k_conv_fwd(ConvArgs a) {
    typedef Vec<T, V> vec;
    const Chan<T, V> me(a);
    if (me.have <= 0 || me.seg >= a.segs) return;
    const int b = blockIdx.z, t0 = me.seg * a.seg, t1 = min(t0 + a.seg, a.T), len = length_of(a.lengths, b, a.T), end = min(t1, len);
    float w[W][V], bias[V];
    me.template taps<W>(w, bias, a);
    const T *x = static_cast<const T *>(a.x) + b * a.x_sb;
    T *y = static_cast<T *>(a.y) + static_cast<int64_t>(b) * a.D;
    const int64_t y_st = static_cast<int64_t>(a.B) * a.D;
    Window<T, V, W> win;
    vec next[kAhead];
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) next[i] = t + i < end ? me.load(x + (t + i) * a.x_st) : vec{};
    };
    if (t0 < end) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) win.set(k, x_at<T, V, W>(a, me, t0 - (W - 1) + k, b));
        fetch(t0);
    }
    for (int t = t0; t < end; t += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) win.set(W - 1 + i, next[i]);
        fetch(t + kAhead);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (t + i >= end) continue;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                o[e] = bias[e];
#pragma unroll
                for (int k = 0; k < W; ++k) o[e] = fmaf(w[k][e], win.x[i + k][e], o[e]);
                if (a.silu) o[e] *= sigmoid_f(o[e]);
            }
            me.store(y + (t + i) * y_st, o);
        }
        win.move();
    }
    const float zero[V] = {};
    for (int t = max(t0, end); t < t1; ++t) me.store(y + t * y_st, zero);
    if (a.last && me.seg == 0)
        for (int j = 0; j < W - 1; ++j) {
            const vec v = x_at<T, V, W>(a, me, len - (W - 1) + j, b);
            float f[V];
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = to_f32(static_cast<T>(v[e]));
            me.store(static_cast<T *>(a.last) + (static_cast<int64_t>(b) * (W - 1) + j) * a.D, f);
        }
}

// pre is made again from x rather than kept by the forward: x is read anyway.  The same size: 54 us, 3.7 TB/s (eight channels a
// thread, whose sums leave half as many waves a SIMD, 104).  Ticks behind a length are not read but computed as zeros: trials of
// half that length take as long.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kBlock) k_conv_bwd(ConvArgs a) {
    typedef Vec<T, V> vec;
    __shared__ float sum[kBlock * V];
    const Chan<T, V> me(a);
    const bool on = me.have > 0 && me.seg < a.segs;
    const int b = blockIdx.z, t0 = me.seg * a.seg, t1 = min(t0 + a.seg, a.T), len = length_of(a.lengths, b, a.T);
    float dw[W][V] = {}, db[V] = {};
    if (on) {
        float w[W][V], bias[V];
        me.template taps<W>(w, bias, a);
        const T *x = static_cast<const T *>(a.x) + b * a.x_sb, *dy = static_cast<const T *>(a.dy) + b * a.dy_sb;
        T *dx = a.dx ? static_cast<T *>(a.dx) + static_cast<int64_t>(b) * a.D : nullptr;
        const int64_t dx_st = static_cast<int64_t>(a.B) * a.D;
        const int end = min(t1 + W - 1, len), first = me.seg == 0 ? -(W - 1) : t0;   // the first tick whose gradient this segment writes
        Window<T, V, W> win;
        float dp[W - 1 + kAhead][V] = {};   // dp[W - 1 + i] of tick t + i
        vec next_x[kAhead], next_g[kAhead];
        auto fetch = [&](int t) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                next_x[i] = next_g[i] = vec{};
                if (t + i < end) next_x[i] = me.load(x + (t + i) * a.x_st), next_g[i] = me.load(dy + (t + i) * a.dy_st);
            }
        };
#pragma unroll
        for (int k = 0; k < W - 1; ++k) win.set(k, t0 < len ? x_at<T, V, W>(a, me, t0 - (W - 1) + k, b) : vec{});
        fetch(t0);
        for (int t = t0; t < t1 + W - 1; t += kAhead) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                win.set(W - 1 + i, next_x[i]);
#pragma unroll
                for (int e = 0; e < V; ++e) dp[W - 1 + i][e] = to_f32(static_cast<T>(next_g[i][e]));   // 0 past the end
            }
            fetch(t + kAhead);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const bool mine = t + i < t1;
                float g[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (a.silu) {
                        float pre = bias[e];
#pragma unroll
                        for (int k = 0; k < W; ++k) pre = fmaf(w[k][e], win.x[i + k][e], pre);
                        const float q = sigmoid_f(pre);
                        dp[W - 1 + i][e] *= q * fmaf(pre, 1.0f - q, 1.0f);
                    }
                    const float d = mine ? dp[W - 1 + i][e] : 0.0f;
                    db[e] += d;
#pragma unroll
                    for (int k = 0; k < W; ++k) dw[k][e] = fmaf(d, win.x[i + k][e], dw[k][e]);
                    g[e] = 0.0f;
#pragma unroll
                    for (int k = 0; k < W; ++k) g[e] = fmaf(w[k][e], dp[W - 1 + i - k][e], g[e]);
                }
                const int at = t + i - (W - 1);
                if (at < first || at >= t1) continue;
                const int j = at - (len - (W - 1));
                if (a.dlast && j >= 0 && at < len) {
                    const vec q = me.load(static_cast<const T *>(a.dlast) + (static_cast<int64_t>(b) * (W - 1) + j) * a.D);
#pragma unroll
                    for (int e = 0; e < V; ++e) g[e] += to_f32(static_cast<T>(q[e]));
                }
                if (at >= len) {
#pragma unroll
                    for (int e = 0; e < V; ++e) g[e] = 0.0f;
                }
                if (at >= 0) {
                    if (dx) me.store(dx + at * dx_st, g);
                } else if (a.dstate) {
                    me.store(static_cast<T *>(a.dstate) + (static_cast<int64_t>(b) * (W - 1) + (W - 1 + at)) * a.D, g);
                }
            }
            win.move();
#pragma unroll
            for (int i = 0; i < W - 1; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) dp[i][e] = dp[i + kAhead][e];
        }
    }
    if (!a.part) return;
    // the block's segments, in order
    float *part = a.part + static_cast<int64_t>(blockIdx.z * gridDim.y + blockIdx.y) * (W + 1) * a.D + static_cast<int64_t>(blockIdx.x) * a.C * V;
    const int cols = min(a.C * V, a.D - static_cast<int>(blockIdx.x) * a.C * V), row = a.C * V;
#pragma unroll
    for (int k = 0; k <= W; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) sum[threadIdx.x * V + e] = k < W ? dw[k < W ? k : 0][e] : db[e];
        __syncthreads();
        for (int q = threadIdx.x; q < cols; q += kBlock) {
            float v = 0.0f;
            for (int s = 0; s < kBlock / a.C; ++s) v += sum[s * row + q];
            part[static_cast<int64_t>(k) * a.D + q] = v;
        }
    }
}

// dw and db: the parts' sums from i0 on, 32 columns by 8 threads each, which take the parts in turn.
__global__ void __launch_bounds__(kBlock) k_conv_join(ConvArgs a, int64_t i0) {
    __shared__ float sum[8][32];
    const int col = threadIdx.x % 32, lot = threadIdx.x / 32;
    const int64_t n = static_cast<int64_t>(a.W + 1) * a.D, i = i0 + static_cast<int64_t>(blockIdx.x) * 32 + col;
    float s = 0.0f;
    if (i < n) {
#pragma unroll 4
        for (int p = lot; p < a.parts; p += 8) s += a.part[p * n + i];
    }
    sum[lot][col] = s;
    __syncthreads();
    if (lot || i >= n) return;
    s = 0.0f;
#pragma unroll
    for (int l = 0; l < 8; ++l) s += sum[l][col];
    const int64_t k = i / a.D, d = i - k * a.D;
    if (k < a.W) {
        if (a.dweight) store_param(a.dweight, a.pdt, d * a.W + k, s);
    } else if (a.dbias) {
        store_param(a.dbias, a.pdt, d, s);
    }
}

// One tick: y from the state and x, and the state moved on by x.  32 x 2048 bfloat16 4.8 us, a launch.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kBlock) k_conv_step(ConvArgs a) {
    typedef Vec<T, V> vec;
    const Chan<T, V> me(a);
    const int b = blockIdx.z * (kBlock / a.C) + threadIdx.x / a.C;
    if (me.have <= 0 || b >= a.B) return;
    T *st = static_cast<T *>(a.last) + static_cast<int64_t>(b) * (W - 1) * a.D;
    float w[W][V], o[V];
    vec win[W];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) win[k] = me.load(st + static_cast<int64_t>(k) * a.D);
    win[W - 1] = me.load(static_cast<const T *>(a.x) + b * a.x_sb);
    me.template taps<W>(w, o, a);
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(w[k][e], to_f32(static_cast<T>(win[k][e])), o[e]);
    if (a.silu)
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] *= sigmoid_f(o[e]);
    me.store(static_cast<T *>(a.y) + static_cast<int64_t>(b) * a.D, o);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        float f[V];
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = to_f32(static_cast<T>(win[k + 1][e]));
        me.store(st + static_cast<int64_t>(k) * a.D, f);
    }
}

enum Pass { kFwd, kBwd, kStep };

// Threads side by side: as many as there are pieces of v channels, up to a wave (forward 16 bytes; backward 4 channels: with
// the 8 of a 16-bit type its windows and sums take the registers of half the waves, 500 x 32 x 2048 x 4 104 us for 57).
// Segments of 64 ticks, or of 32 or 16 where that gives fewer than 2048 waves.
void shape(ConvArgs &a, int v) {
    const int across = ceil_div(a.D, v);
    a.C = 1;
    while (a.C < across && a.C < kWave) a.C *= 2;
    a.seg = 64;
    while (a.seg > 16 && static_cast<int64_t>(ceil_div(across, a.C)) * a.C * a.B * ceil_div(a.T, a.seg) < 2048 * kWave) a.seg /= 2;
    a.segs = std::max(1, ceil_div(a.T, a.seg));
    a.parts = a.B * ceil_div(a.segs, kBlock / a.C);
}

void join(const ConvArgs &a, hipStream_t s) {
    constexpr int64_t kMost = blocks_at_once(kBlock) * 32;
    const int64_t n = static_cast<int64_t>(a.W + 1) * a.D;
    for (int64_t i = 0; a.part && i < n; i += kMost)
        hipLaunchKernelGGL(k_conv_join, dim3(static_cast<unsigned>(ceil_div(std::min(kMost, n - i), 32))), dim3(kBlock), 0, s, a, i);
}

template <typename T, int W>
void launch(const ConvArgs &a, Pass pass, hipStream_t s) {
    constexpr int V = kVecBytes16<T>, VB = 4;
    const unsigned cols = static_cast<unsigned>(ceil_div(ceil_div(a.D, pass == kBwd ? VB : V), a.C)), deep = kBlock / a.C;
    const dim3 grid(cols, (a.segs + deep - 1) / deep, static_cast<unsigned>(a.B));
    if (pass == kStep) hipLaunchKernelGGL((k_conv_step<T, V, W>), dim3(cols, 1, (a.B + deep - 1) / deep), dim3(kBlock), 0, s, a);
    else if (pass == kFwd) hipLaunchKernelGGL((k_conv_fwd<T, V, W>), grid, dim3(kBlock), 0, s, a);
    else hipLaunchKernelGGL((k_conv_bwd<T, VB, W>), grid, dim3(kBlock), 0, s, a);
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
    a.x_st = x_stride_t, a.x_sb = x_stride_b, a.T = T, a.B = B, a.D = D, a.W = W, a.pdt = param_dtype, a.silu = silu;
    shape(a, 16 / static_cast<int>(dtype_size(dtype)));
    GLIF_BY_DTYPE(dtype, by_taps, a, W, kFwd, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

size_t glif_short_conv_bwd_workspace(int32_t dtype, int32_t T, int32_t B, int32_t D, int32_t W) {
    if (check_conv(dtype, dtype, T, B, D, W)) return 0;
    ConvArgs a{};
    a.T = T, a.B = B, a.D = D;
    shape(a, 4);
    return static_cast<size_t>(a.parts) * (W + 1) * D * sizeof(float) + 256;
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
    a.T = T, a.B = B, a.D = D, a.W = W, a.pdt = param_dtype, a.silu = silu;
    shape(a, 4);
    if (dweight || dbias) {
        Carver c(ws, ws_bytes);
        a.part = c.take<float>(static_cast<size_t>(a.parts) * (W + 1) * D);
        if (!ws || !c.ok()) return fail(GLIF_ENOMEM, "short convolution: workspace too small");
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (B) GLIF_BY_DTYPE(dtype, by_taps, a, W, kBwd, s);
    join(a, s);
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
    a.x_sb = x_stride_b, a.T = 1, a.B = B, a.D = D, a.W = W, a.pdt = param_dtype, a.silu = silu;
    shape(a, 16 / static_cast<int>(dtype_size(dtype)));
    GLIF_BY_DTYPE(dtype, by_taps, a, W, kStep, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
