// Selective state space scan.  Per batch entry, channel d (of group g) and state n:
//   s = softplus(delta + bias),  a = exp(s A),  h[t] = a h[t - 1] + s B[t] u[t]
//   y1[t] = sum_n C[t] h[t] + D u[t],  y = y1 silu(z)
// and backward, with gh = dL/dh running from the last tick to the first:
//   dy1 = dy silu(z),  dz = dy y1 silu'(z),  gh[t] = dy1 C[t] + a[t + 1] gh[t + 1]
//   dC = sum_d dy1 h,  dB = sum_d gh s u,  du = D dy1 + s sum_n gh B
//   ds = sum_n gh (A a h[t - 1] + B u),  ddelta = ds softplus',  dA = sum gh a h[t - 1] s
// A channel's states are spread over kSpl lanes, four each, so that a wave has channels x states in registers whatever N.
// States past N are zeros that stay zeros.
#include "seq.h"

namespace glif {
namespace {

constexpr int kQ = 4;        // states of a lane
constexpr int kKeep = 16;    // ticks between kept states
constexpr float kLog2e = 1.4426950408889634f;

struct ScanArgs {
    glif_scan s;
    glif_scan_grad g;
    void *y;
    float *last;
    float *keep;             // [ceil(T / kKeep)][B][D][NP]
    int32_t np, tiles;       // states padded to the lanes; channel tiles of a group
    float *part_bc;          // [G * tiles][T][B][2][NP]
    float *part_a;           // [B][D][NP]
    float *part_d;           // [B][2][D]
};

// log(1 + exp(x)) = max(x, 0) + log(1 + e), e = exp(-|x|): with r = e / (2 + e) <= 1/3, log(1 + e) = 2 atanh(r), whose
// series to r^13 is good to 2e-8 of its value.  slope = sigmoid(x).
__device__ __forceinline__ float softplus_f(float x, float &slope) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
    const float r = e / (2.0f + e), r2 = r * r;
    float p = 1.0f / 13.0f;
    p = fmaf(p, r2, 1.0f / 11.0f);
    p = fmaf(p, r2, 1.0f / 9.0f);
    p = fmaf(p, r2, 1.0f / 7.0f);
    p = fmaf(p, r2, 1.0f / 5.0f);
    p = fmaf(p, r2, 1.0f / 3.0f);
    p = fmaf(p, r2, 1.0f);
    const float q = 1.0f / (1.0f + e);
    slope = x >= 0.0f ? q : e * q;
    return fmaxf(x, 0.0f) + 2.0f * r * p;
}

// sum over the SPL lanes of a channel
template <int SPL>
__device__ __forceinline__ float channel_sum(float v) {
#pragma unroll
    for (int m = 1; m < SPL; m <<= 1) v += __shfl_xor(v, m, kWave);
    return v;
}

// What a lane is: its channel and the first of its states.
template <int SPL>
struct Lane {
    static constexpr int kChan = kWave / SPL;   // channels of a wave
    int b, g, d, n0, tile;
    bool on;
    __device__ Lane(const ScanArgs &a) {
        const int wave = blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave, lane = threadIdx.x % kWave;
        const int per = a.s.n_channels / a.s.n_groups;
        b = blockIdx.y;
        tile = wave;
        g = wave / a.tiles;
        const int c = (wave - g * a.tiles) * kChan + lane / SPL;
        on = g < a.s.n_groups && c < per;
        d = on ? g * per + c : 0;
        if (g >= a.s.n_groups) g = 0;
        n0 = (lane % SPL) * kQ;
    }
};

template <typename T>
__device__ __forceinline__ void load_q(float (&v)[kQ], const void *p, int64_t at, int n0, int N) {
#pragma unroll
    for (int j = 0; j < kQ; ++j) v[j] = n0 + j < N ? to_f32(static_cast<const T *>(p)[at + n0 + j]) : 0.0f;
}

__device__ __forceinline__ int scan_length(const glif_scan &s, int b) {
    return s.lengths ? min(max(s.lengths[b], 0), s.n_ticks) : s.n_ticks;
}

// The inputs of one tick of a lane's channel.
struct Tick {
    float u, step, slope, z, sig;
    float B[kQ], C[kQ];
};

template <typename T>
__device__ __forceinline__ void load_tick(Tick &k, const glif_scan &s, int t, int b, int g, int d, int n0, float bias) {
    k.u = to_f32(static_cast<const T *>(s.u)[t * s.u_st + b * s.u_sb + d]);
    const float raw = to_f32(static_cast<const T *>(s.delta)[t * s.delta_st + b * s.delta_sb + d]) + bias;
    k.step = raw, k.slope = 1.0f;
    if (s.softplus) k.step = softplus_f(raw, k.slope);
    k.z = k.sig = 0.0f;
    if (s.z) {
        k.z = to_f32(static_cast<const T *>(s.z)[t * s.z_st + b * s.z_sb + d]);
        k.sig = sigmoid_f(k.z);
    }
    load_q<T>(k.B, s.B, t * s.B_st + b * s.B_sb + static_cast<int64_t>(g) * s.n_state, n0, s.n_state);
    load_q<T>(k.C, s.C, t * s.C_st + b * s.C_sb + static_cast<int64_t>(g) * s.n_state, n0, s.n_state);
}

template <typename T, int SPL>
__global__ void __launch_bounds__(kBlock) k_scan_fwd(ScanArgs a) {
    const glif_scan &s = a.s;
    const Lane<SPL> me(a);
    const int N = s.n_state, len = scan_length(s, me.b);
    const int64_t chan = static_cast<int64_t>(me.b) * s.n_channels + me.d;
    float A[kQ], h[kQ];
    load_q<f32>(A, s.A, static_cast<int64_t>(me.d) * N, me.n0, N);
#pragma unroll
    for (int j = 0; j < kQ; ++j) A[j] *= kLog2e, h[j] = 0.0f;
    if (s.state) load_q<f32>(h, s.state, chan * N, me.n0, N);
    const float skip = s.D ? s.D[me.d] : 0.0f, bias = s.delta_bias ? s.delta_bias[me.d] : 0.0f;
    for (int t = 0; t < s.n_ticks; ++t) {
        if (a.keep && t % kKeep == 0 && me.on) {
            const int64_t row = static_cast<int64_t>(t / kKeep) * s.n_batch * s.n_channels + chan;
            *reinterpret_cast<float4 *>(a.keep + row * a.np + me.n0) = make_float4(h[0], h[1], h[2], h[3]);
        }
        float y = 0.0f;
        if (t < len) {
            Tick k;
            load_tick<T>(k, s, t, me.b, me.g, me.d, me.n0, bias);
            const float su = k.step * k.u;
#pragma unroll
            for (int j = 0; j < kQ; ++j) {
                h[j] = fmaf(__builtin_amdgcn_exp2f(k.step * A[j]), h[j], su * k.B[j]);
                y = fmaf(k.C[j], h[j], y);
            }
            y = fmaf(skip, k.u, channel_sum<SPL>(y));
            if (s.z) y *= k.z * k.sig;
        }
        if (me.on && me.n0 == 0)
            static_cast<T *>(a.y)[(static_cast<int64_t>(t) * s.n_batch + me.b) * s.n_channels + me.d] = from_f32<T>(y);
    }
    if (a.last && me.on)
#pragma unroll
        for (int j = 0; j < kQ; ++j)
            if (me.n0 + j < N) a.last[chan * N + me.n0 + j] = h[j];
}

template <typename T, int SPL>
__global__ void __launch_bounds__(kBlock) k_scan_bwd(ScanArgs a) {
    const glif_scan &s = a.s;
    const glif_scan_grad &gr = a.g;
    const Lane<SPL> me(a);
    const int N = s.n_state, len = scan_length(s, me.b), lane = threadIdx.x % kWave;
    const bool tile_on = me.tile < s.n_groups * a.tiles;
    const int64_t chan = static_cast<int64_t>(me.b) * s.n_channels + me.d;
    float A[kQ], gh[kQ], dA[kQ];
    load_q<f32>(A, s.A, static_cast<int64_t>(me.d) * N, me.n0, N);
#pragma unroll
    for (int j = 0; j < kQ; ++j) gh[j] = dA[j] = 0.0f;
    if (gr.dlast) load_q<f32>(gh, gr.dlast, chan * N, me.n0, N);
    const float skip = s.D ? s.D[me.d] : 0.0f, bias = s.delta_bias ? s.delta_bias[me.d] : 0.0f;
    float dskip = 0.0f, dbias = 0.0f;
    for (int k0 = s.n_ticks > 0 ? (s.n_ticks - 1) / kKeep * kKeep : -1; k0 >= 0; k0 -= kKeep) {
        float hp[kKeep][kQ];    // the states before each tick
        const int64_t row = static_cast<int64_t>(k0 / kKeep) * s.n_batch * s.n_channels + chan;
        const float4 h0 = *reinterpret_cast<const float4 *>(a.keep + row * a.np + me.n0);
        hp[0][0] = h0.x, hp[0][1] = h0.y, hp[0][2] = h0.z, hp[0][3] = h0.w;
#pragma unroll
        for (int i = 0; i + 1 < kKeep; ++i) {
#pragma unroll
            for (int j = 0; j < kQ; ++j) hp[i + 1][j] = hp[i][j];
            if (k0 + i < len) {
                Tick k;
                load_tick<T>(k, s, k0 + i, me.b, me.g, me.d, me.n0, bias);
                const float su = k.step * k.u;
#pragma unroll
                for (int j = 0; j < kQ; ++j)
                    hp[i + 1][j] = fmaf(__builtin_amdgcn_exp2f(k.step * A[j] * kLog2e), hp[i][j], su * k.B[j]);
            }
        }
#pragma unroll
        for (int i = kKeep - 1; i >= 0; --i) {
            const int t = k0 + i;
            if (t >= s.n_ticks) continue;
            float dB[kQ], dC[kQ], du = 0.0f, draw = 0.0f, dz = 0.0f;
#pragma unroll
            for (int j = 0; j < kQ; ++j) dB[j] = dC[j] = 0.0f;
            if (t < len) {
                Tick k;
                load_tick<T>(k, s, t, me.b, me.g, me.d, me.n0, bias);
                const float dy = me.on ? to_f32(static_cast<const T *>(gr.dy)[t * gr.dy_st + me.b * gr.dy_sb + me.d]) : 0.0f;
                const float dy1 = s.z ? dy * (k.z * k.sig) : dy, su = k.step * k.u;
                float y1 = 0.0f, gB = 0.0f, thA = 0.0f;
#pragma unroll
                for (int j = 0; j < kQ; ++j) {
                    const float dec = __builtin_amdgcn_exp2f(k.step * A[j] * kLog2e);
                    const float h = fmaf(dec, hp[i][j], su * k.B[j]);
                    y1 = fmaf(k.C[j], h, y1);
                    gh[j] = fmaf(dy1, k.C[j], gh[j]);
                    dC[j] = me.on ? dy1 * h : 0.0f;
                    dB[j] = me.on ? gh[j] * su : 0.0f;
                    gB = fmaf(gh[j], k.B[j], gB);
                    gh[j] *= dec;
                    const float th = gh[j] * hp[i][j];
                    thA = fmaf(th, A[j], thA);
                    dA[j] = fmaf(th, k.step, dA[j]);
                }
                y1 = fmaf(skip, k.u, channel_sum<SPL>(y1));
                gB = channel_sum<SPL>(gB);
                thA = channel_sum<SPL>(thA);
                du = fmaf(skip, dy1, k.step * gB);
                draw = fmaf(k.u, gB, thA) * k.slope;
                dz = dy * y1 * (k.sig * fmaf(k.z, 1.0f - k.sig, 1.0f));
                dskip = fmaf(dy1, k.u, dskip);
                dbias += draw;
            }
            const int64_t at = (static_cast<int64_t>(t) * s.n_batch + me.b) * s.n_channels + me.d;
            if (me.on && me.n0 == 0) {
                if (gr.du) static_cast<T *>(gr.du)[at] = from_f32<T>(du);
                if (gr.ddelta) static_cast<T *>(gr.ddelta)[at] = from_f32<T>(draw);
                if (gr.dz) static_cast<T *>(gr.dz)[at] = from_f32<T>(dz);
            }
            if (a.part_bc) {
#pragma unroll
                for (int j = 0; j < kQ; ++j)
                    for (int m = SPL; m < kWave; m <<= 1) {
                        dB[j] += __shfl_xor(dB[j], m, kWave);
                        dC[j] += __shfl_xor(dC[j], m, kWave);
                    }
                if (tile_on && lane < SPL) {
                    float *p = a.part_bc + ((static_cast<int64_t>(me.tile) * s.n_ticks + t) * s.n_batch + me.b) * 2 * a.np + me.n0;
                    *reinterpret_cast<float4 *>(p) = make_float4(dB[0], dB[1], dB[2], dB[3]);
                    *reinterpret_cast<float4 *>(p + a.np) = make_float4(dC[0], dC[1], dC[2], dC[3]);
                }
            }
        }
    }
    if (!me.on) return;
    *reinterpret_cast<float4 *>(a.part_a + chan * a.np + me.n0) = make_float4(dA[0], dA[1], dA[2], dA[3]);
    if (me.n0 == 0) {
        a.part_d[(static_cast<int64_t>(me.b) * 2 + 0) * s.n_channels + me.d] = dskip;
        a.part_d[(static_cast<int64_t>(me.b) * 2 + 1) * s.n_channels + me.d] = dbias;
    }
    if (gr.dstate)
#pragma unroll
        for (int j = 0; j < kQ; ++j)
            if (me.n0 + j < N) gr.dstate[chan * N + me.n0 + j] = gh[j];
}

// dB, dC: the tiles of a group, in order.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_scan_join_bc(ScanArgs a) {
    const glif_scan &s = a.s;
    const int64_t n = static_cast<int64_t>(s.n_ticks) * s.n_batch * s.n_groups * s.n_state;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (i >= n) return;
    const int64_t tb = i / (s.n_groups * s.n_state);
    const int gn = static_cast<int>(i - tb * (s.n_groups * s.n_state)), g = gn / s.n_state, st = gn - g * s.n_state;
    const int64_t tbs = static_cast<int64_t>(s.n_ticks) * s.n_batch;
    float dB = 0.0f, dC = 0.0f;
    for (int k = 0; k < a.tiles; ++k) {
        const float *p = a.part_bc + ((static_cast<int64_t>(g) * a.tiles + k) * tbs + tb) * 2 * a.np + st;
        dB += p[0];
        dC += p[a.np];
    }
    if (a.g.dB) static_cast<T *>(a.g.dB)[i] = from_f32<T>(dB);
    if (a.g.dC) static_cast<T *>(a.g.dC)[i] = from_f32<T>(dC);
}

// dA, dD, ddelta_bias: the batch entries, in order.
__global__ void __launch_bounds__(kBlock) k_scan_join_param(ScanArgs a) {
    const glif_scan &s = a.s;
    const int64_t n = static_cast<int64_t>(s.n_channels) * a.np, i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (i >= n) return;
    const int d = static_cast<int>(i / a.np), st = static_cast<int>(i - static_cast<int64_t>(d) * a.np);
    if (a.g.dA && st < s.n_state) {
        float v = 0.0f;
        for (int b = 0; b < s.n_batch; ++b) v += a.part_a[b * n + i];
        a.g.dA[static_cast<int64_t>(d) * s.n_state + st] = v;
    }
    if (st == 0) {
        float dD = 0.0f, db = 0.0f;
        for (int b = 0; b < s.n_batch; ++b) {
            dD += a.part_d[(static_cast<int64_t>(b) * 2 + 0) * s.n_channels + d];
            db += a.part_d[(static_cast<int64_t>(b) * 2 + 1) * s.n_channels + d];
        }
        if (a.g.dD) a.g.dD[d] = dD;
        if (a.g.ddelta_bias) a.g.ddelta_bias[d] = db;
    }
}

int lanes_for(int32_t N) {
    int l = 1;
    while (l * kQ < N) l *= 2;
    return l;
}

void shape(ScanArgs &a) {
    const int spl = lanes_for(a.s.n_state), chan = kWave / spl;
    a.np = spl * kQ;
    a.tiles = ceil_div(a.s.n_channels / a.s.n_groups, chan);
}

template <typename T, int SPL>
void launch(const ScanArgs &a, bool back, hipStream_t st) {
    const int waves = a.s.n_groups * a.tiles;
    const dim3 grid(static_cast<unsigned>(ceil_div(waves, kBlock / kWave)), static_cast<unsigned>(a.s.n_batch));
    if (back) hipLaunchKernelGGL((k_scan_bwd<T, SPL>), grid, dim3(kBlock), 0, st, a);
    else hipLaunchKernelGGL((k_scan_fwd<T, SPL>), grid, dim3(kBlock), 0, st, a);
}

template <typename T>
void by_lanes(const ScanArgs &a, bool back, hipStream_t st) {
    switch (a.np / kQ) {
        case 1: return launch<T, 1>(a, back, st);
        case 2: return launch<T, 2>(a, back, st);
        case 4: return launch<T, 4>(a, back, st);
        case 8: return launch<T, 8>(a, back, st);
        default: return launch<T, 16>(a, back, st);
    }
}

template <typename T>
void run_bwd(const ScanArgs &a, hipStream_t st) {
    const int64_t bc = static_cast<int64_t>(a.s.n_ticks) * a.s.n_batch * a.s.n_groups * a.s.n_state;
    if (a.s.n_batch) by_lanes<T>(a, true, st);
    if (a.part_bc && bc)
        hipLaunchKernelGGL(k_scan_join_bc<T>, dim3(static_cast<unsigned>(ceil_div(bc, kBlock))), dim3(kBlock), 0, st, a);
    if (a.g.dA || a.g.dD || a.g.ddelta_bias)
        hipLaunchKernelGGL(k_scan_join_param, dim3(static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.s.n_channels) * a.np, kBlock))),
                           dim3(kBlock), 0, st, a);
}

int check_scan(const glif_scan *s) {
    if (!s) return fail(GLIF_EINVAL, "NULL argument");
    if (!known_dtype(s->dtype)) return fail(GLIF_EINVAL, "state space: unknown type");
    if (s->n_ticks < 0 || s->n_ticks > (1 << 20) || s->n_batch < 0 || s->n_batch > 65535 || s->n_channels < 1 ||
        s->n_channels > (1 << 24))
        return fail(GLIF_EINVAL, "state space: ticks in [0, 2^20], batch in [0, 65535], channels in [1, 2^24]");
    if (s->n_groups < 1 || s->n_channels % s->n_groups) return fail(GLIF_EINVAL, "state space: the groups must divide the channels");
    if (s->n_state < 1 || s->n_state > 64) return fail(GLIF_EINVAL, "state space: 1 to 64 states");
    return GLIF_OK;
}

bool have_inputs(const glif_scan *s) {
    return s->A && (s->n_ticks == 0 || s->n_batch == 0 || (s->u && s->delta && s->B && s->C));
}

void carve(Carver &c, ScanArgs &a) {
    const size_t rows = static_cast<size_t>(a.s.n_batch) * a.s.n_channels;
    a.part_a = c.take<float>(rows * a.np);
    a.part_d = c.take<float>(rows * 2);
    a.part_bc = c.take<float>(static_cast<size_t>(a.s.n_groups) * a.tiles * a.s.n_ticks * a.s.n_batch * 2 * a.np);
}

}  // namespace
}  // namespace glif

using namespace glif;

extern "C" {

size_t glif_scan_keep_bytes(const glif_scan *s) {
    if (check_scan(s)) return 0;
    return static_cast<size_t>(ceil_div(s->n_ticks, kKeep)) * s->n_batch * s->n_channels * lanes_for(s->n_state) * kQ * sizeof(float);
}

size_t glif_scan_fwd_workspace(const glif_scan *s) { return check_scan(s) ? 0 : 0; }

int glif_scan_fwd(const glif_scan *s, void *y, float *last, void *keep, void *ws, size_t ws_bytes, void *stream) {
    (void)ws, (void)ws_bytes;
    if (int rc = check_scan(s)) return rc;
    if (s->n_batch == 0) return GLIF_OK;
    if (!have_inputs(s) || (s->n_ticks && !y)) return fail(GLIF_EINVAL, "NULL argument");
    ScanArgs a{};
    a.s = *s, a.y = y, a.last = last, a.keep = static_cast<float *>(keep);
    shape(a);
    GLIF_BY_DTYPE(s->dtype, by_lanes, a, false, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

size_t glif_scan_bwd_workspace(const glif_scan *s) {
    if (check_scan(s)) return 0;
    ScanArgs a{};
    a.s = *s;
    shape(a);
    Carver c(nullptr, 0);
    carve(c, a);
    return c.mark();
}

int glif_scan_bwd(const glif_scan *s, const glif_scan_grad *g, const void *keep, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_scan(s)) return rc;
    if (!g || !have_inputs(s) || (s->n_ticks && s->n_batch && (!g->dy || !keep))) return fail(GLIF_EINVAL, "NULL argument");
    ScanArgs a{};
    a.s = *s, a.g = *g, a.keep = static_cast<float *>(const_cast<void *>(keep));
    shape(a);
    Carver c(ws, ws_bytes);
    carve(c, a);
    if (!ws || !c.ok()) return fail(GLIF_ENOMEM, "state space: workspace too small");
    if (!g->dB && !g->dC) a.part_bc = nullptr;
    GLIF_BY_DTYPE(s->dtype, run_bwd, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

int glif_scan_step(const glif_scan *s, void *y, float *state, void *stream) {
    if (int rc = check_scan(s)) return rc;
    if (s->n_batch == 0) return GLIF_OK;
    if (s->n_ticks != 1 || !have_inputs(s) || !y || !state) return fail(GLIF_EINVAL, "state space: a step is one tick, with its state");
    ScanArgs a{};
    a.s = *s, a.y = y, a.last = state;
    a.s.state = state, a.s.lengths = nullptr;
    shape(a);
    GLIF_BY_DTYPE(s->dtype, by_lanes, a, false, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
