// Linear map with bias, activation and residual in its epilogue, and its backward:
//   pre = x W^T + bias,  y = act(pre) + residual
//   dp = dy act'(pre),  dx = dp W,  dW = dp^T x,  db = sum of dp's rows
// All three products run on the matrix cores with float32 accumulators (16-bit types 16x16x32, float32 16x16x4).
#include "seq.h"

namespace glif {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// C[m][n] = sum_k P(m, k) Q(n, k), P(m, k) = p[m * p_m + k * p_k], one of the two strides 1; likewise Q.
struct GemmArgs {
    const void *p, *q;
    int64_t p_m, p_k, q_n, q_k;
    int64_t M, N, K;
    void *c, *pre;             // [M][N]
    const void *bias, *residual;
    int64_t ldr;
    int32_t bias_dt, act;
};

__device__ __forceinline__ float act_of(float p, int act) {
    switch (act) {
        case GLIF_ACT_RELU: return fmaxf(p, 0.0f);
        case GLIF_ACT_GELU: return 0.5f * p * (1.0f + erff(p * 0.70710678118654752f));
        case GLIF_ACT_SILU: return p * sigmoid_f(p);
        default: return p;
    }
}

__device__ __forceinline__ float slope_of(float p, int act) {
    switch (act) {
        case GLIF_ACT_RELU: return p > 0.0f ? 1.0f : 0.0f;
        case GLIF_ACT_GELU:
            return fmaf(p * 0.39894228040143268f, expf(-0.5f * p * p), 0.5f * (1.0f + erff(p * 0.70710678118654752f)));
        case GLIF_ACT_SILU: {
            const float q = sigmoid_f(p);
            return q * fmaf(p, 1.0f - q, 1.0f);
        }
        default: return 1.0f;
    }
}

constexpr int kTile = 64;

// One matrix instruction's operands from a row-major LDS row of 32 k's: 16-bit types take 8 consecutive k's a lane.
template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    static constexpr int kLane = 8;
    typedef bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<f16> {
    static constexpr int kLane = 8;
    typedef f16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
// float32: lane l holds four consecutive k's, element i of every lane makes one 16x16x4 product (the order of the k's in
// a sum is free, as long as both operands have it)
template <>
struct Mma<f32> {
    static constexpr int kLane = 4;
    typedef f32 frag __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// 64 x 64 of C by four waves of 32 x 32; k in steps of one matrix instruction.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_gemm(GemmArgs a) {
    using M = Mma<T>;
    constexpr int KS = 4 * M::kLane, LD = KS + 16 / static_cast<int>(sizeof(T));
    __shared__ __attribute__((aligned(16))) T sp[kTile][LD], sq[kTile][LD];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, r16 = lane % 16, kq = lane / 16 * M::kLane;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile, n0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int wm = wave / 2 * 32, wn = wave % 2 * 32;
    f32x4 acc[2][2] = {};
    const T *p = static_cast<const T *>(a.p), *q = static_cast<const T *>(a.q);
    for (int64_t k0 = 0; k0 < a.K; k0 += KS) {
        for (int i = threadIdx.x; i < kTile * KS; i += kBlock) {
            int r = a.p_k == 1 ? i / KS : i % kTile, k = a.p_k == 1 ? i % KS : i / kTile;
            sp[r][k] = m0 + r < a.M && k0 + k < a.K ? p[(m0 + r) * a.p_m + (k0 + k) * a.p_k] : T(0.0f);
            r = a.q_k == 1 ? i / KS : i % kTile, k = a.q_k == 1 ? i % KS : i / kTile;
            sq[r][k] = n0 + r < a.N && k0 + k < a.K ? q[(n0 + r) * a.q_n + (k0 + k) * a.q_k] : T(0.0f);
        }
        __syncthreads();
        typename M::frag fp[2], fq[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fp[i] = *reinterpret_cast<const typename M::frag *>(&sp[wm + 16 * i + r16][kq]);
            fq[i] = *reinterpret_cast<const typename M::frag *>(&sq[wn + 16 * i + r16][kq]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = M::run(fq[j], fp[i], acc[i][j]);   // rows of the result: n
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t m = m0 + wm + 16 * i + r16, n = n0 + wn + 16 * j + lane / 16 * 4 + e;
                if (m >= a.M || n >= a.N) continue;
                float v = acc[i][j][e];
                if (a.bias) v += load_param(a.bias, a.bias_dt, n);
                if (a.pre) static_cast<T *>(a.pre)[m * a.N + n] = from_f32<T>(v);
                v = act_of(v, a.act);
                if (a.residual) v += to_f32(static_cast<const T *>(a.residual)[m * a.ldr + n]);
                static_cast<T *>(a.c)[m * a.N + n] = from_f32<T>(v);
            }
}

struct SlopeArgs {
    const void *dy, *pre;
    int64_t lddy, M, N;
    void *dp;            // [M][N] or NULL
    float *part;         // [parts][N] or NULL
    int32_t act, parts;
};

// dp = dy act'(pre), rounded to the activations' type for the products, and the column sums of the unrounded values over a
// chunk of rows.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_slope(SlopeArgs a) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (n >= a.N) return;
    const int64_t r0 = a.M * blockIdx.y / a.parts, r1 = a.M * (blockIdx.y + 1) / a.parts;
    float s = 0.0f;
    for (int64_t m = r0; m < r1; ++m) {
        float g = to_f32(static_cast<const T *>(a.dy)[m * a.lddy + n]);
        if (a.act != GLIF_ACT_NONE) g *= slope_of(to_f32(static_cast<const T *>(a.pre)[m * a.N + n]), a.act);
        if (a.dp) static_cast<T *>(a.dp)[m * a.N + n] = from_f32<T>(g);
        s += g;
    }
    if (a.part) a.part[static_cast<int64_t>(blockIdx.y) * a.N + n] = s;
}

__global__ void __launch_bounds__(kBlock) k_bias_join(const float *part, int parts, int64_t N, void *dbias, int32_t dt) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (n >= N) return;
    float s = 0.0f;
    for (int p = 0; p < parts; ++p) s += part[p * N + n];
    store_param(dbias, dt, n, s);
}

template <typename T>
void run_gemm(const GemmArgs &a, hipStream_t s) {
    if (a.M == 0 || a.N == 0) return;
    hipLaunchKernelGGL(k_gemm<T>, dim3(static_cast<unsigned>(ceil_div(a.N, kTile)), static_cast<unsigned>(ceil_div(a.M, kTile))),
                       dim3(kBlock), 0, s, a);
}

template <typename T>
void run_slope(const SlopeArgs &a, hipStream_t s) {
    if (a.N == 0) return;
    hipLaunchKernelGGL(k_slope<T>, dim3(static_cast<unsigned>(ceil_div(a.N, kBlock)), static_cast<unsigned>(a.parts)),
                       dim3(kBlock), 0, s, a);
}

int row_parts(int64_t M) { return static_cast<int>(std::min<int64_t>(std::max<int64_t>(M / 16, 1), 256)); }

int check_linear(int32_t dtype, int32_t bias_dtype, int64_t M, int64_t N, int64_t K, int32_t act) {
    if (!known_dtype(dtype) || (bias_dtype != GLIF_F32 && bias_dtype != dtype))
        return fail(GLIF_EINVAL, "linear: the bias is float32 or of x's type");
    if (M < 0 || N < 0 || K < 0 || M > (1 << 21) || N > (1 << 21) || K > (1 << 24))
        return fail(GLIF_EINVAL, "linear: M and N in [0, 2^21], K in [0, 2^24]");
    if (act < GLIF_ACT_NONE || act > GLIF_ACT_SILU) return fail(GLIF_EINVAL, "linear: unknown activation");
    return GLIF_OK;
}

struct Back {
    void *dp;
    float *part;
    int32_t parts;
};

void carve(Carver &c, Back &b, int32_t dtype, int64_t M, int64_t N, int32_t act) {
    b.parts = row_parts(M);
    b.part = c.take<float>(static_cast<size_t>(b.parts * N));
    b.dp = act != GLIF_ACT_NONE ? c.take<char>(static_cast<size_t>(M * N) * dtype_size(dtype)) : nullptr;
}

}  // namespace
}  // namespace glif

using namespace glif;

extern "C" {

size_t glif_linear_fwd_workspace(int32_t dtype, int64_t M, int64_t N, int64_t K) {
    (void)dtype, (void)M, (void)N, (void)K;
    return 0;
}

int glif_linear_fwd(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, const void *residual,
                    int64_t ldr, int32_t dtype, int32_t bias_dtype, int64_t M, int64_t N, int64_t K, int32_t activation,
                    void *y, void *pre, void *ws, size_t ws_bytes, void *stream) {
    (void)ws, (void)ws_bytes;
    if (int rc = check_linear(dtype, bias_dtype, M, N, K, activation)) return rc;
    if (M == 0 || N == 0) return GLIF_OK;
    if (!y || (K && (!x || !weight))) return fail(GLIF_EINVAL, "NULL argument");
    GemmArgs a{};
    a.p = x, a.p_m = ldx, a.p_k = 1, a.q = weight, a.q_n = ldw, a.q_k = 1, a.M = M, a.N = N, a.K = K;
    a.c = y, a.pre = pre, a.bias = bias, a.residual = residual, a.ldr = ldr, a.bias_dt = bias_dtype, a.act = activation;
    GLIF_BY_DTYPE(dtype, run_gemm, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

size_t glif_linear_bwd_workspace(int32_t dtype, int64_t M, int64_t N, int64_t K, int32_t activation) {
    if (check_linear(dtype, dtype, M, N, K, activation)) return 0;
    Carver c(nullptr, 0);
    Back b{};
    carve(c, b, dtype, M, N, activation);
    return c.mark();
}

int glif_linear_bwd(const void *dy, int64_t lddy, const void *pre, const void *x, int64_t ldx, const void *weight,
                    int64_t ldw, int32_t dtype, int32_t bias_dtype, int64_t M, int64_t N, int64_t K, int32_t activation,
                    void *dx, void *dweight, void *dbias, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_linear(dtype, bias_dtype, M, N, K, activation)) return rc;
    const bool some = M && N;
    if (some && (!dy || (activation != GLIF_ACT_NONE && !pre) || (dx && K && !weight) || (dweight && K && !x)))
        return fail(GLIF_EINVAL, "NULL argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    Back b{};
    Carver c(ws, ws_bytes);
    carve(c, b, dtype, M, N, activation);
    if (!c.ok() || (c.off && !ws)) return fail(GLIF_ENOMEM, "linear: workspace too small");
    const void *dp = dy;
    int64_t lddp = lddy;
    if (activation != GLIF_ACT_NONE || dbias) {
        SlopeArgs a{dy, pre, lddy, M, N, b.dp, dbias ? b.part : nullptr, activation, b.parts};
        GLIF_BY_DTYPE(dtype, run_slope, a, s);
        if (b.dp) dp = b.dp, lddp = N;
        if (dbias && N)
            hipLaunchKernelGGL(k_bias_join, dim3(static_cast<unsigned>(ceil_div(N, kBlock))), dim3(kBlock), 0, s, b.part, b.parts,
                               N, dbias, bias_dtype);
    }
    if (dx) {
        GemmArgs a{};
        a.p = dp, a.p_m = lddp, a.p_k = 1, a.q = weight, a.q_n = 1, a.q_k = ldw, a.M = M, a.N = K, a.K = N, a.c = dx;
        GLIF_BY_DTYPE(dtype, run_gemm, a, s);
    }
    if (dweight) {
        GemmArgs a{};
        a.p = dp, a.p_m = 1, a.p_k = lddp, a.q = x, a.q_n = 1, a.q_k = ldx, a.M = N, a.N = K, a.K = M, a.c = dweight;
        GLIF_BY_DTYPE(dtype, run_gemm, a, s);
    }
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
