// Fused ExponentiatedAdam step + SignedConstraint (v1_model_utils/optimizers.py:268-376,
// dense branch :354-376, models.py:419-427): one streaming pass over a weight vector; and AdamW over many tensors at once.
#include <cmath>

#include "mma.h"
#include "philox.h"

namespace glif {

// Per element, in TF's operation order (fp32, separate roundings):
//   m += (g - m) * (1 - beta_1);   v += (g * g - v) * (1 - beta_2)
//   vhat = max(vhat, v) (AMSGrad);  u = vhat or v
//   s = sign(w) with sign(0) = +1;  w = w * exp(((-alpha) * (m / (sqrt(u) + eps))) * s)
//   positive: w = positive ? relu(w) : -relu(-w)   (the variable's constraint, applied
//   by Keras after the update)
__global__ void __launch_bounds__(kBlock)
    k_exp_adam(float *__restrict__ w, float *__restrict__ m, float *__restrict__ v, float *__restrict__ vhat,
               const float *__restrict__ g, const uint8_t *__restrict__ positive, int64_t n, float alpha,
               float one_m_b1, float one_m_b2, float eps) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += stride) {
        const float gi = g[i];
        float mi = m[i], vi = v[i];
        mi = mi + (gi - mi) * one_m_b1;
        vi = vi + (gi * gi - vi) * one_m_b2;
        m[i] = mi;
        v[i] = vi;
        float u = vi;
        if (vhat) {
            u = fmaxf(vhat[i], vi);
            vhat[i] = u;
        }
        const float ag = mi / (sqrtf(u) + eps);
        const float wi = w[i];
        const float s = wi > 0.0f ? 1.0f : (wi < 0.0f ? -1.0f : 1.0f);
        float wn = wi * expf((-alpha * ag) * s);
        if (positive) wn = positive[i] ? fmaxf(wn, 0.0f) : -fmaxf(-wn, 0.0f);
        w[i] = wn;
    }
}

// ---- AdamW ------------------------------------------------------------------------------------------------------------
// With t the step that is taken:
//   m = beta_1 m + (1 - beta_1) g,   v = beta_2 v + (1 - beta_2) g^2
//   p = (1 - lr decay) p - lr / (1 - beta_1^t) * m / (sqrt(v) / sqrt(1 - beta_2^t) + eps)
// m and v are float32, or 8 bits with a float32 scale s (the largest magnitude) for each block of 256:
//   m = s (c / 127) |c / 127|,   v = s (c / 255)^4
// (squares and fourth powers give small values beside large ones the steps that a root would: about 1.6 % at the top, and
// a second moment of 1e-9 of its block's largest is not lost).  A code is the one below or above the value, by a random number, so that
// its mean is the value: moments that move by less than a code's step each time still move.  What is not 0 of v does not
// become 0, as the step divides by its root.  The random numbers of element i of all variables' blocks are the two halves of word
// (t - 1) P + i of the Philox stream `seed`, P the elements of all blocks.
//
// Bound by memory: 36M float32 elements of 20 tensors, 997 MB, 195 us (5.1 TB/s), with moments of 8 bits, 572 MB, 139 us (the
// random numbers, roots and codes are some 100 operations an element); results past the caches gained nothing.
constexpr int kUnit = 256;          // elements that a wave takes at once, and that share a scale
constexpr int kUnitsPerBlock = 16;  // that a block takes at once
constexpr int kMostTensors = 64;    // of a launch
// Four blocks a compute unit, which go through the units in turn: each ends with an addition to one word, which come one after
// the other (36M float32 elements 197 us; by 2048 blocks 207, by one for every 16 units 828).
constexpr unsigned kMostBlocks = 1024;

// One of a launch's tensors.  Its words are of 32 bits and more: arrays of bytes beside those of pointers, under one index, were
// read with an index in the scalar loads' base whose last two bits those do not add (the loads fell between two pointers).
struct AdamwTensor {
    void *var;
    const void *grad;
    int64_t n;
    int64_t home;             // the first unit of its state
    uint32_t before, after;   // units of the launch's tensors before it, and with it
    int32_t var_dt, grad_dt;
};

struct AdamwArgs {
    AdamwTensor of[kMostTensors];
    int32_t tensors;
    void *first, *second;
    float *first_scale, *second_scale;   // 8 bits: one a unit
    int64_t *iterations;                 // steps done, and the blocks that have ended (0 between launches)
    int64_t total;                       // elements of all units
    double log_beta_1, log_beta_2;
    float beta_1, beta_2, one_m_b1, one_m_b2, lr, eps, decay;   // decay: lr times the weights'
    uint64_t seed;
    int32_t last;                        // this launch ends the step
};

__device__ __forceinline__ f32x4 load_4(const void *p, int dt, int64_t i, int have) {
    f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
    if (have == 4) {
        if (dt == GLIF_F32) return *reinterpret_cast<const Vec<f32, 4> *>(static_cast<const f32 *>(p) + i);
        if (dt == GLIF_BF16) return __builtin_convertvector(*reinterpret_cast<const Vec<bf16, 4> *>(static_cast<const bf16 *>(p) + i), f32x4);
        return __builtin_convertvector(*reinterpret_cast<const Vec<f16, 4> *>(static_cast<const f16 *>(p) + i), f32x4);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < have) r[e] = load_param(p, dt, i + e);
    return r;
}

__device__ __forceinline__ void store_4(void *p, int dt, int64_t i, int have, f32x4 v) {
    if (have == 4) {
        if (dt == GLIF_F32) *reinterpret_cast<Vec<f32, 4> *>(static_cast<f32 *>(p) + i) = v;
        else if (dt == GLIF_BF16) *reinterpret_cast<Vec<bf16, 4> *>(static_cast<bf16 *>(p) + i) = __builtin_convertvector(v, Vec<bf16, 4>);
        else *reinterpret_cast<Vec<f16, 4> *>(static_cast<f16 *>(p) + i) = __builtin_convertvector(v, Vec<f16, 4>);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < have) store_param(p, dt, i + e, v[e]);
}

template <bool SECOND>
__device__ __forceinline__ float level(float code) {
    const float r = code * (SECOND ? 1.0f / 255.0f : 1.0f / 127.0f);
    return SECOND ? (r * r) * (r * r) : r * fabsf(r);
}

template <bool SECOND>
__device__ __forceinline__ f32x4 decode_4(uint32_t codes, float scale) {
    f32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint8_t c = static_cast<uint8_t>(codes >> (8 * e));
        r[e] = level<SECOND>(SECOND ? static_cast<float>(c) : static_cast<float>(static_cast<int8_t>(c))) * scale;
    }
    return r;
}

// The unit's largest magnitude as a float; NaN where there is one (the bits of magnitudes are in their order).
__device__ __forceinline__ float unit_most(f32x4 x) {
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d, kWave)));
    return __uint_as_float(most);
}

// Codes of four values by their halves of random words.  A root that is off by its last bit may take the code beside the
// right one, from which the comparison still finds the one above or below.  A scale that is not finite makes the whole unit so
// (0 * infinity); one below the normal numbers leaves 0.
template <bool SECOND>
__device__ __forceinline__ uint32_t encode_4(f32x4 x, float most, const uint32_t (&word)[4]) {
    constexpr float kTop = SECOND ? 255.0f : 127.0f;
    if (!(most >= 1.17549435e-38f && most < __builtin_inff())) return 0u;
    const float inv = 1.0f / most;
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float part = fabsf(x[e]) * inv;
        const float root = SECOND ? __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(part)) : __builtin_amdgcn_sqrtf(part);
        const float below = fminf(floorf(root * kTop), kTop - 1.0f);
        const float a = level<SECOND>(below), b = level<SECOND>(below + 1.0f);
        const float u = static_cast<float>(SECOND ? word[e] >> 16 : word[e] & 0xffffu);
        int c = static_cast<int>(below) + (u * (b - a) < (part - a) * 65536.0f ? 1 : 0);
        if (SECOND && x[e] > 0.0f) c = max(c, 1);
        if (!SECOND && x[e] < 0.0f) c = -c;
        codes |= (static_cast<uint32_t>(c) & 0xffu) << (8 * e);
    }
    return codes;
}

// What a lane holds of a unit: four neighbours of everything.
template <int BITS>
struct Quad {
    f32x4 p, g, m, v;
    uint32_t mc, vc;
    float ms, vs;
    int64_t at;   // of the moments

    __device__ __forceinline__ void moments(const AdamwArgs &a, int64_t home, int lane) {
        at = home * kUnit + lane * 4;
        if (BITS == 8) {
            mc = *reinterpret_cast<const uint32_t *>(static_cast<const int8_t *>(a.first) + at), ms = a.first_scale[home];
            vc = *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.second) + at), vs = a.second_scale[home];
        } else {
            m = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.first) + at);
            v = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.second) + at);
        }
    }
    __device__ __forceinline__ void step(const AdamwArgs &a, float size, float root) {
        if (BITS == 8) m = decode_4<false>(mc, ms), v = decode_4<true>(vc, vs);
        m = m * a.beta_1 + g * a.one_m_b1;
        v = v * a.beta_2 + (g * g) * a.one_m_b2;
        // The decay joins the update before anything is rounded to p's digits: of 1 - decay, float32 keeps nothing of a decay below 3e-8.
        // (An infinite p stays: what is taken off it is finite.)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float update = size * (m[e] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[e]) * root + a.eps));
            p[e] -= __builtin_fmaf(a.decay, __builtin_amdgcn_fmed3f(p[e], -3.40282347e38f, 3.40282347e38f), update);
        }
    }
    __device__ __forceinline__ void put(const AdamwArgs &a, int64_t home, int lane, int64_t t) const {
        if (BITS == 8) {
            uint32_t word[4];
            philox_block(a.seed, (static_cast<uint64_t>(t - 1) * static_cast<uint64_t>(a.total) + static_cast<uint64_t>(at)) >> 2, word);
            const float mm = unit_most(m), vm = unit_most(v);
            *reinterpret_cast<uint32_t *>(static_cast<int8_t *>(a.first) + at) = encode_4<false>(m, mm, word);
            *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a.second) + at) = encode_4<true>(v, vm, word);
            if (lane == 0) a.first_scale[home] = mm, a.second_scale[home] = vm;
        } else {
            *reinterpret_cast<f32x4 *>(static_cast<float *>(a.first) + at) = m;
            *reinterpret_cast<f32x4 *>(static_cast<float *>(a.second) + at) = v;
        }
    }
};

// A block's units all within one tensor whose variable and gradient are of type T: each wave's, N at a time.
template <int BITS, typename T, int N>
__device__ __forceinline__ void adamw_whole(const AdamwArgs &a, int i, int64_t first, float size, float root, int64_t t, int wave, int lane) {
    constexpr int kMine = kUnitsPerBlock / (kBlock / kWave);
    typedef Vec<T, 4> vec;
    T *p = static_cast<T *>(a.of[i].var) + lane * 4;
    const T *g = static_cast<const T *>(a.of[i].grad) + lane * 4;
    const int64_t home = a.of[i].home;
#pragma unroll 1
    for (int u = 0; u < kMine; u += N) {
        Quad<BITS> q[N];
        vec pv[N], gv[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t unit = first + wave * kMine + u + k;
            gv[k] = *reinterpret_cast<const vec *>(g + unit * kUnit);
            pv[k] = *reinterpret_cast<const vec *>(p + unit * kUnit);
            q[k].moments(a, home + unit, lane);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t unit = first + wave * kMine + u + k;
            q[k].p = __builtin_convertvector(pv[k], f32x4), q[k].g = __builtin_convertvector(gv[k], f32x4);
            q[k].step(a, size, root);
            const vec o = __builtin_convertvector(q[k].p, vec);
            *reinterpret_cast<vec *>(p + unit * kUnit) = o;
            q[k].put(a, home + unit, lane, t);
        }
    }
}

template <int BITS>
__global__ void __launch_bounds__(kBlock) k_adamw(AdamwArgs a) {
    constexpr int kAtOnce = 2;   // units a wave has under way (four: no faster)
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t t = *static_cast<volatile int64_t *>(a.iterations) + 1;
    const double td = static_cast<double>(t);
    // 1 - beta^t without the cancellation of a beta near 1
    const float size = static_cast<float>(static_cast<double>(a.lr) / -expm1(td * a.log_beta_1));
    const float root = static_cast<float>(1.0 / sqrt(-expm1(td * a.log_beta_2)));
    const uint32_t units = a.of[a.tensors - 1].after;
    for (uint64_t base = static_cast<uint64_t>(blockIdx.x) * kUnitsPerBlock; base < units; base += static_cast<uint64_t>(gridDim.x) * kUnitsPerBlock) {
        int i = 0;   // the tensor that holds unit `base`
#pragma unroll
        for (int s = kMostTensors / 2; s > 0; s >>= 1)
            if (i + s < a.tensors && a.of[i + s].before <= base) i += s;
        const int64_t first = static_cast<int64_t>(base - a.of[i].before);
        if ((first + kUnitsPerBlock) * kUnit <= a.of[i].n && a.of[i].var_dt == a.of[i].grad_dt) {
            const int32_t dt = a.of[i].var_dt;
            if (dt == GLIF_F32) adamw_whole<BITS, f32, kAtOnce>(a, i, first, size, root, t, wave, lane);
            else if (dt == GLIF_BF16) adamw_whole<BITS, bf16, kAtOnce>(a, i, first, size, root, t, wave, lane);
            else adamw_whole<BITS, f16, kAtOnce>(a, i, first, size, root, t, wave, lane);
            continue;
        }
        for (uint64_t unit = base + wave; unit < min(base + kUnitsPerBlock, static_cast<uint64_t>(units)); unit += kBlock / kWave) {
            while (a.of[i].after <= unit) ++i;
            const AdamwTensor &of = a.of[i];
            const int64_t in = static_cast<int64_t>(unit - of.before), at = in * kUnit + lane * 4, home = of.home + in;
            const int have = static_cast<int>(max(static_cast<int64_t>(0), min(of.n - at, static_cast<int64_t>(4))));
            Quad<BITS> q;
            q.g = load_4(of.grad, of.grad_dt, at, have);
            q.p = load_4(of.var, of.var_dt, at, have);
            q.moments(a, home, lane);
            q.step(a, size, root);
            store_4(of.var, of.var_dt, at, have, q.p);
            q.put(a, home, lane, t);
        }
    }
    if (!a.last) return;
    // The block that ends last counts the step: everybody has used the count by then.  Nothing else is passed on, so no block
    // waits for its results to be seen by others (with a fence each block's end cost 0.1 us, one after the other).
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned long long *ended = reinterpret_cast<unsigned long long *>(a.iterations + 1);
        if (atomicAdd(ended, 1ull) == gridDim.x - 1) {
            *ended = 0;
            *a.iterations = t;
        }
    }
}

// The values that 8-bit codes stand for.
template <bool SECOND>
__global__ void __launch_bounds__(kBlock) k_adamw_values(const uint8_t *codes, const float *scale, int64_t units, float *out) {
    const int lane = threadIdx.x % kWave;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave; u < units; u += static_cast<int64_t>(gridDim.x) * (kBlock / kWave)) {
        const int64_t at = u * kUnit + lane * 4;
        *reinterpret_cast<f32x4 *>(out + at) = decode_4<SECOND>(*reinterpret_cast<const uint32_t *>(codes + at), scale[u]);
    }
}

}  // namespace glif

using namespace glif;

extern "C" int glif_exp_adam(float *w, float *m, float *v, float *vhat, const float *g, const uint8_t *positive,
                             int64_t n, float alpha, float beta_1, float beta_2, float epsilon, void *stream) {
    if (n < 0) return fail(GLIF_EINVAL, "n must be >= 0");
    if (n == 0) return GLIF_OK;
    if (!w || !m || !v || !g) return fail(GLIF_EINVAL, "NULL argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t blocks = std::min<int64_t>((n + kBlock - 1) / kBlock, 8192);
    hipLaunchKernelGGL(k_exp_adam, dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0, s, w, m, v, vhat, g,
                       positive, n, alpha, 1.0f - beta_1, 1.0f - beta_2, epsilon);
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

extern "C" int glif_adamw(int32_t n_vars, void *const *vars, const int32_t *var_dtypes, const void *const *grads,
                          const int32_t *grad_dtypes, const int64_t *sizes, int32_t state_bits, void *first, void *second,
                          float *first_scale, float *second_scale, int64_t *iterations, double learning_rate, double beta_1,
                          double beta_2, double epsilon, double weight_decay, uint64_t seed, void *stream) {
    if (n_vars < 0 || (state_bits != 8 && state_bits != 32)) return fail(GLIF_EINVAL, "adamw: n_vars must be >= 0 and state_bits 8 or 32");
    if (!(beta_1 >= 0.0 && beta_1 < 1.0 && beta_2 >= 0.0 && beta_2 < 1.0)) return fail(GLIF_EINVAL, "adamw: the betas must be in [0, 1)");
    // What v keeps of gradients below some 1e-19 is 0 (their squares are below float32's normal numbers): beside an epsilon of 1e-12
    // their roots are nothing.
    if (!(epsilon >= 1e-12 && std::isfinite(epsilon) && weight_decay >= 0.0))
        return fail(GLIF_EINVAL, "adamw: epsilon must be finite and at least 1e-12, weight_decay >= 0");
    if (n_vars == 0) return GLIF_OK;
    if (!vars || !var_dtypes || !grads || !grad_dtypes || !sizes) return fail(GLIF_EINVAL, "NULL argument");
    int64_t total = 0, given = 0;
    for (int32_t i = 0; i < n_vars; ++i) {
        if (sizes[i] < 0 || sizes[i] > (int64_t(1) << 36)) return fail(GLIF_EINVAL, "adamw: sizes must be in [0, 2^36]");
        total += (sizes[i] + kUnit - 1) / kUnit;
        if (!grads[i] || sizes[i] == 0) continue;
        if (!vars[i]) return fail(GLIF_EINVAL, "NULL argument");
        if (!known_dtype(var_dtypes[i]) || (grad_dtypes[i] != GLIF_F32 && grad_dtypes[i] != var_dtypes[i]))
            return fail(GLIF_EINVAL, "adamw: a gradient is float32 or of its variable's type");
        ++given;
    }
    if (given == 0) return GLIF_OK;
    if (!first || !second || !iterations || (state_bits == 8 && (!first_scale || !second_scale))) return fail(GLIF_EINVAL, "NULL argument");
    if (reinterpret_cast<uintptr_t>(first) % 16 || reinterpret_cast<uintptr_t>(second) % 16)
        return fail(GLIF_EINVAL, "adamw: the moments must lie on 16 bytes");
    AdamwArgs a{};
    a.first = first, a.second = second, a.first_scale = first_scale, a.second_scale = second_scale, a.iterations = iterations;
    a.total = total * kUnit;
    // log(0) is -infinity, and expm1 of it -1: no correction
    a.log_beta_1 = std::log(beta_1), a.log_beta_2 = std::log(beta_2);
    a.beta_1 = static_cast<float>(beta_1), a.beta_2 = static_cast<float>(beta_2);
    a.one_m_b1 = static_cast<float>(1.0 - beta_1), a.one_m_b2 = static_cast<float>(1.0 - beta_2);
    a.lr = static_cast<float>(learning_rate), a.eps = static_cast<float>(epsilon);
    a.decay = static_cast<float>(learning_rate * weight_decay), a.seed = seed;
    hipStream_t s = static_cast<hipStream_t>(stream);
    int64_t home = 0;
    for (int32_t i = 0; i < n_vars; ++i) {
        const int64_t units = (sizes[i] + kUnit - 1) / kUnit;
        if (grads[i] && units) {
            const uint32_t before = a.tensors ? a.of[a.tensors - 1].after : 0u, after = before + static_cast<uint32_t>(units);
            a.of[a.tensors++] = AdamwTensor{vars[i], grads[i], sizes[i], home, before, after, var_dtypes[i], grad_dtypes[i]};
            --given;
            // units of a launch are counted in 32 bits: 2^28 of the largest size allowed fit eight times
            const bool full = a.tensors == kMostTensors || after >= 7u << 28;
            a.last = given == 0;
            if (full || a.last) {
                const unsigned blocks = std::min<unsigned>((after + kUnitsPerBlock - 1) / kUnitsPerBlock, kMostBlocks);
                if (state_bits == 8) hipLaunchKernelGGL(k_adamw<8>, dim3(blocks), dim3(kBlock), 0, s, a);
                else hipLaunchKernelGGL(k_adamw<32>, dim3(blocks), dim3(kBlock), 0, s, a);
                a.tensors = 0;
            }
        }
        home += units;
    }
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

extern "C" int glif_adamw_values(const void *first, const float *first_scale, const void *second, const float *second_scale,
                                 int64_t n, float *first_out, float *second_out, void *stream) {
    if (n < 0 || n % kUnit) return fail(GLIF_EINVAL, "adamw: n must be a multiple of 256");
    if (n == 0) return GLIF_OK;
    if (!first || !first_scale || !second || !second_scale || !first_out || !second_out) return fail(GLIF_EINVAL, "NULL argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((n / kUnit + 3) / 4, 8192)));
    hipLaunchKernelGGL(k_adamw_values<false>, grid, dim3(kBlock), 0, s, static_cast<const uint8_t *>(first), first_scale, n / kUnit, first_out);
    hipLaunchKernelGGL(k_adamw_values<true>, grid, dim3(kBlock), 0, s, static_cast<const uint8_t *>(second), second_scale, n / kUnit, second_out);
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}
