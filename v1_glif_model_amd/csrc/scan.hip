// Selective state space scan.  Per batch entry, channel d (of group g) and state n:
//   s = softplus(delta + bias),  a = exp(s A),  h[t] = a h[t - 1] + s B[t] u[t]
//   y1[t] = sum_n C[t] h[t] + D u[t],  y = y1 silu(z)
// and backward, with gh = dL/dh running from the last tick to the first:
//   dy1 = dy silu(z),  dz = dy y1 silu'(z),  gh[t] = dy1 C[t] + a[t + 1] gh[t + 1]
//   dC = sum_d dy1 h,  dB = sum_d gh s u,  du = D dy1 + s sum_n gh B
//   ds = sum_n gh (A a h[t - 1] + B u),  ddelta = ds softplus',  dA = sum gh a h[t - 1] s
// A channel's states are spread over SPL lanes, four each (states past N are zeros that stay zeros), so that a wave holds
// 64 / SPL channels and the four waves of a block four such tiles of one group.  A block walks its ticks in chunks:
//   - the chunk's B and C come to LDS once for all the block's channels, ticks past a length as zeros;
//   - what a tick needs per channel (softplus, the gate) is computed by one of the channel's lanes for SPL ticks in turn,
//     which the others get by lane broadcasts; sums over a channel's lanes come out at the tick's lane (reduce-scatter);
//   - a tick past the length has step, u and dy 0: decay 1, no contribution, and its outputs are 0.
// Few channels do not fill the chip: time is then split into segments.  A first pass takes each segment's end state from
// zero and its sum of steps (its decay is exp(A sum)), a join runs over the segments, a second pass goes from the right
// states; the backward does the same from the other side.
//
// Bound by instruction issue: per state and tick an exponential (a quarter of the rate of the rest) and four products and
// sums forward, some 24 operations backward; what a channel needs per tick adds about a third (vector units busy 85 to 98
// percent of the time).  Memory would allow 27 us for 16.4M channels' ticks forward and 55 backward.  Ticks behind a length are
// issued like live ones: over trials of half the ticks, half of that issue is for none.
#include <cfloat>
#include <cmath>

#include "seq.h"

namespace glif {
namespace {

constexpr int kQ = 4;        // states of a lane
constexpr int kWaves = kBlock / kWave;
constexpr float kLog2e = 1.4426950408889634f;

// ticks of a chunk, and between the states that are kept for the backward: four per lane of a channel, at most 16
constexpr int chunk_of(int spl) { return spl >= 4 ? 16 : 4 * spl; }

struct ScanArgs {
    glif_scan s;
    glif_scan_grad g;
    void *y;
    float *last;
    float *keep;             // [ceil(T / chunk)][B][D][NP] states before each chunk
    int32_t np, blocks;      // states padded to the lanes; blocks of a group's channels
    int32_t segs, seg;       // segments of time, ticks of one (whole chunks)
    float *seg_state;        // [segs][B][D][NP] a segment's end, then what comes into it (adjoints: from behind)
    float *seg_step;         // [segs][B][D] sums of steps
    float *part_bc;          // [G * blocks][T][B][2][NP]
    float *part_a;           // [segs][B][D][NP]
    float *part_d;           // [segs][B][2][D]
};

// log(1 + exp(x)) = max(x, 0) + log(1 + e), e = exp(-|x|): with r = e / (2 + e) <= 1/3, log(1 + e) = 2 atanh(r), whose
// series to r^13 is good to 2e-8 of its value.  slope = sigmoid(x).
__device__ __forceinline__ float softplus_f(float x, float &slope) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
    const float r = e * __builtin_amdgcn_rcpf(2.0f + e), r2 = r * r;
    float p = 1.0f / 13.0f;
    p = fmaf(p, r2, 1.0f / 11.0f);
    p = fmaf(p, r2, 1.0f / 9.0f);
    p = fmaf(p, r2, 1.0f / 7.0f);
    p = fmaf(p, r2, 1.0f / 5.0f);
    p = fmaf(p, r2, 1.0f / 3.0f);
    p = fmaf(p, r2, 1.0f);
    const float q = __builtin_amdgcn_rcpf(1.0f + e);
    slope = x >= 0.0f ? q : e * q;
    return fmaxf(x, 0.0f) + 2.0f * r * p;
}

// ---- lanes ----------------------------------------------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// v of lane i of the channel's SPL
template <int SPL>
__device__ __forceinline__ float bcast(float v, int i) {
    if constexpr (SPL == 1) return v;
    else if constexpr (SPL == 2) return i ? dpp<0xF5>(v) : dpp<0xA0>(v);
    else if constexpr (SPL == 4) return i == 0 ? dpp<0x00>(v) : i == 1 ? dpp<0x55>(v) : i == 2 ? dpp<0xAA>(v) : dpp<0xFF>(v);
    else return __shfl(v, i, SPL);
}

template <int X>
__device__ __forceinline__ float lane_xor(float v) {
    if constexpr (X == 1) return dpp<0xB1>(v);
    else if constexpr (X == 2) return dpp<0x4E>(v);
    else return __shfl_xor(v, X, kWave);
}

// Sum over the channel's SPL lanes of v[i], to lane i.
template <int SPL>
__device__ __forceinline__ float to_lane(float (&v)[SPL], int me) {
    if constexpr (SPL == 1) {
        return v[0];
    } else {
        float h[SPL / 2];
        const bool odd = me & 1;
#pragma unroll
        for (int i = 0; i < SPL / 2; ++i) {
            const float keep = odd ? v[2 * i + 1] : v[2 * i], send = odd ? v[2 * i] : v[2 * i + 1];
            h[i] = keep + lane_xor<1>(send);
        }
        if constexpr (SPL == 2) {
            return h[0];
        } else {
            float q[SPL / 4];
            const bool two = me & 2;
#pragma unroll
            for (int i = 0; i < SPL / 4; ++i) {
                const float keep = two ? h[2 * i + 1] : h[2 * i], send = two ? h[2 * i] : h[2 * i + 1];
                q[i] = keep + lane_xor<2>(send);
            }
            if constexpr (SPL == 4) {
                return q[0];
            } else if constexpr (SPL == 8) {
                return (me & 4 ? q[1] : q[0]) + lane_xor<4>(me & 4 ? q[0] : q[1]);
            } else {
                const float r0 = (me & 4 ? q[1] : q[0]) + lane_xor<4>(me & 4 ? q[0] : q[1]);
                const float r1 = (me & 4 ? q[3] : q[2]) + lane_xor<4>(me & 4 ? q[2] : q[3]);
                return (me & 8 ? r1 : r0) + lane_xor<8>(me & 8 ? r0 : r1);
            }
        }
    }
}

// Sums over the wave's channels of a lane's dB[4] and dC[4]: lane l ends with two of them, x[k] that of state 2 (l >> 4 & 1) +
// k of its four, of dB in the lower and of dC in the upper half of the wave.  The swaps bring both halves (both 16s) of two
// values side by side, so that one sum serves two values.
template <int SPL>
__device__ __forceinline__ void channels_sum(const float (&dB)[kQ], const float (&dC)[kQ], float (&x)[2]) {
#ifdef __HIP_DEVICE_COMPILE__
    float w[kQ];
#pragma unroll
    for (int j = 0; j < kQ; ++j) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, dB[j]), __builtin_bit_cast(unsigned, dC[j]), false, false);
        w[j] = __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, w[k]), __builtin_bit_cast(unsigned, w[k + 2]), false, false);
        float v = __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
        if constexpr (SPL <= 8) v += dpp<0x128>(v);   // rotations of the 16 lanes by 8, 4, 2, 1
        if constexpr (SPL <= 4) v += dpp<0x124>(v);
        if constexpr (SPL <= 2) v += dpp<0x122>(v);
        if constexpr (SPL <= 1) v += dpp<0x121>(v);
        x[k] = v;
    }
#endif
}

// What a lane is: its channel and the first of its states.
template <int SPL>
struct Lane {
    static constexpr int kChan = kWave / SPL;   // channels of a wave
    int b, g, d, s, n0;
    bool on;
    __device__ Lane(const ScanArgs &a) {
        const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, per = a.s.n_channels / a.s.n_groups;
        b = blockIdx.y;
        g = blockIdx.x / a.blocks;
        const int c = ((blockIdx.x - g * a.blocks) * kWaves + wave) * kChan + lane / SPL;
        on = c < per;
        d = g * per + min(c, per - 1);
        s = lane % SPL;
        n0 = s * kQ;
    }
};

__device__ __forceinline__ int scan_length(const glif_scan &s, int b) {
    return s.lengths ? min(max(s.lengths[b], 0), s.n_ticks) : s.n_ticks;
}

// A for powers of 2.  A rate of -infinity (a decay of 0 over any step) is the largest there is: times the step of a tick behind
// a length, 0, it is a decay of 1.
__device__ __forceinline__ float rate_of(float A) {
    const float v = A * kLog2e;
    return v == -INFINITY ? -FLT_MAX : v;
}

__device__ __forceinline__ void load_q(float (&v)[kQ], const float *p, int64_t at, int n0, int N) {
#pragma unroll
    for (int j = 0; j < kQ; ++j) v[j] = n0 + j < N ? p[at + n0 + j] : 0.0f;
}
__device__ __forceinline__ void load_4(float (&v)[kQ], const float *p) {
    const float4 q = *reinterpret_cast<const float4 *>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
}
__device__ __forceinline__ void store_4(float *p, const float (&v)[kQ]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// A chunk's B or C on its way to LDS: this thread's values.
template <typename T, int SPL>
struct Maps {
    static constexpr int kCh = chunk_of(SPL), kNp = SPL * kQ, kAll = kCh * kNp, kN = (kAll + kBlock - 1) / kBlock;
    T v[kN];
    __device__ __forceinline__ void load(const void *p, int64_t st, int64_t at, int t0, int len, int N) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int q = threadIdx.x + i * kBlock, t = t0 + q / kNp, n = q % kNp;
            v[i] = (kAll % kBlock == 0 || q < kAll) && n < N && t < len ? static_cast<const T *>(p)[t * st + at + n] : T(0.0f);
        }
    }
    __device__ __forceinline__ void store(float *lds) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int q = threadIdx.x + i * kBlock;
            if (kAll % kBlock == 0 || q < kAll) lds[q] = to_f32(v[i]);
        }
    }
};

// A channel's values of a chunk on their way: this lane's ticks t0 + e SPL + s.  Ticks past the length and lanes without a
// channel have 0.
template <typename T, int SPL>
struct Own {
    static constexpr int kE = chunk_of(SPL) / SPL;
    T v[kE];
    __device__ __forceinline__ void load(const void *p, int64_t st, int64_t at, int t0, int len, const Lane<SPL> &me) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            const int t = t0 + e * SPL + me.s;
            v[e] = me.on && t < len ? static_cast<const T *>(p)[t * st + at + me.d] : T(0.0f);
        }
    }
};

// step and its slope at a tick of raw delta; 0 past the length
__device__ __forceinline__ float step_of(float raw, bool softplus, bool live, float &slope) {
    float v = raw;
    slope = 1.0f;
    if (softplus) v = softplus_f(raw, slope);
    return live ? v : 0.0f;
}

// ---- forward ----------------------------------------------------------------------------------------------------------------
// ENDS: the first pass over segments, which leaves the segment's end state from zero and its sum of steps.  500 x 32 x 1024 x 16
// bfloat16 108 us; one recording, 8000 x 1 x 2048 x 16, which segments make possible, 66 for the ends and 95.
template <typename T, int SPL, bool ENDS>
__global__ void __launch_bounds__(kBlock) k_scan_fwd(ScanArgs a) {
    constexpr int kCh = chunk_of(SPL), kNp = SPL * kQ, kE = kCh / SPL;
    __shared__ __attribute__((aligned(16))) float sB[2][kCh * kNp], sC[2][kCh * kNp];
    const glif_scan &s = a.s;
    const Lane<SPL> me(a);
    const int N = s.n_state, len = scan_length(s, me.b), t0 = blockIdx.z * a.seg, t1 = min(t0 + a.seg, s.n_ticks);
    const int64_t chan = static_cast<int64_t>(me.b) * s.n_channels + me.d;
    const int64_t row = (static_cast<int64_t>(blockIdx.z) * s.n_batch) * s.n_channels + chan;   // of the segment
    const int64_t map_b = me.b * s.B_sb + static_cast<int64_t>(me.g) * N, map_c = me.b * s.C_sb + static_cast<int64_t>(me.g) * N;
    float A[kQ], h[kQ] = {}, steps = 0.0f;
    load_q(A, s.A, static_cast<int64_t>(me.d) * N, me.n0, N);
#pragma unroll
    for (int j = 0; j < kQ; ++j) A[j] = rate_of(A[j]);
    if (!ENDS) {
        if (a.segs > 1) load_4(h, a.seg_state + row * kNp + me.n0);
        else if (s.state) load_q(h, s.state, chan * N, me.n0, N);
    }
    const float skip = s.D ? s.D[me.d] : 0.0f, bias = s.delta_bias ? s.delta_bias[me.d] : 0.0f;
    Maps<T, SPL> mB, mC;
    Own<T, SPL> u, delta, z;
    auto fetch = [&](int c0) {
        mB.load(s.B, s.B_st, map_b, c0, len, N);
        u.load(s.u, s.u_st, me.b * s.u_sb, c0, len, me);
        delta.load(s.delta, s.delta_st, me.b * s.delta_sb, c0, len, me);
        if (!ENDS) {
            mC.load(s.C, s.C_st, map_c, c0, len, N);
            if (s.z) z.load(s.z, s.z_st, me.b * s.z_sb, c0, len, me);
        }
    };
    fetch(t0);
    for (int c0 = t0, p = 0; c0 < t1; c0 += kCh, p ^= 1) {
        mB.store(sB[p]);
        if (!ENDS) mC.store(sC[p]);
        float own_step[kE], own_u[kE], own_su[kE], gate[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            float slope;
            own_u[e] = to_f32(u.v[e]);
            own_step[e] = step_of(to_f32(delta.v[e]) + bias, s.softplus, c0 + e * SPL + me.s < len, slope);
            own_su[e] = own_step[e] * own_u[e];
            gate[e] = 1.0f;
            if (!ENDS && s.z) {
                const float q = to_f32(z.v[e]);
                gate[e] = q * sigmoid_f(q);
            }
            if (ENDS) steps += own_step[e];
        }
        __syncthreads();
        fetch(c0 + kCh);
        if (!ENDS && a.keep && me.on)
            store_4(a.keep + (static_cast<int64_t>(c0 / kCh) * s.n_batch * s.n_channels + chan) * kNp + me.n0, h);
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            float y[SPL];
#pragma unroll
            for (int i = 0; i < SPL; ++i) {
                const float step = bcast<SPL>(own_step[e], i), su = bcast<SPL>(own_su[e], i);
                float B[kQ], C[kQ];
                load_4(B, sB[p] + (e * SPL + i) * kNp + me.n0);
                if (!ENDS) load_4(C, sC[p] + (e * SPL + i) * kNp + me.n0);
                y[i] = 0.0f;
#pragma unroll
                for (int j = 0; j < kQ; ++j) {
                    h[j] = fmaf(__builtin_amdgcn_exp2f(step * A[j]), h[j], su * B[j]);
                    if (!ENDS) y[i] = fmaf(C[j], h[j], y[i]);
                }
            }
            if (!ENDS) {
                const int t = c0 + e * SPL + me.s;
                const float sum = to_lane<SPL>(y, me.s);
                if (me.on && t < s.n_ticks)
                    static_cast<T *>(a.y)[(static_cast<int64_t>(t) * s.n_batch + me.b) * s.n_channels + me.d] =
                        from_f32<T>(t < len ? fmaf(skip, own_u[e], sum) * gate[e] : 0.0f);
            }
        }
    }
    if (!me.on) return;
    if (ENDS) {
        store_4(a.seg_state + row * kNp + me.n0, h);
#pragma unroll
        for (int m = 1; m < SPL; m <<= 1) steps += __shfl_xor(steps, m, kWave);
        if (me.s == 0) a.seg_step[row] = steps;
    } else if (a.last && blockIdx.z == static_cast<unsigned>(a.segs) - 1) {
#pragma unroll
        for (int j = 0; j < kQ; ++j)
            if (me.n0 + j < N) a.last[chan * N + me.n0 + j] = h[j];
    }
}

// What comes into each segment: forward h[s + 1] = exp(A steps[s]) h[s] + end[s] from the given state, backward the same
// from the last segment to the first.  seg_state goes from the segments' own ends to that, in place.
template <bool BACK>
__global__ void __launch_bounds__(kBlock) k_scan_join(ScanArgs a) {
    const glif_scan &s = a.s;
    const int64_t n = static_cast<int64_t>(s.n_batch) * s.n_channels * a.np;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t chan = i / a.np;
        const int st = static_cast<int>(i - chan * a.np), d = static_cast<int>(chan % s.n_channels);
        const bool real = st < s.n_state;
        const float A = real ? rate_of(s.A[static_cast<int64_t>(d) * s.n_state + st]) : 0.0f;
        const float *from = BACK ? a.g.dlast : s.state;
        float h = from && real ? from[chan * s.n_state + st] : 0.0f;
        constexpr int kAhead = 8;
        for (int k0 = 0; k0 < a.segs; k0 += kAhead) {
            float end[kAhead], steps[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (k0 + u >= a.segs) continue;
                const int k = BACK ? a.segs - 1 - k0 - u : k0 + u;
                end[u] = a.seg_state[k * n + i];
                steps[u] = a.seg_step[k * (n / a.np) + chan];
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (k0 + u >= a.segs) continue;
                const int k = BACK ? a.segs - 1 - k0 - u : k0 + u;
                a.seg_state[k * n + i] = h;
                // In two halves: growth past float32 over a segment may still meet a state small enough, and 0 stays 0.
                const float half = __builtin_amdgcn_exp2f(0.5f * A * steps[u]);
                h = h == 0.0f ? end[u] : fmaf(half, half * h, end[u]);
            }
        }
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------
// ENDS: the first pass over segments, which leaves what a segment hands to the one before it, and its sum of steps.  Else a
// chunk's states are run again from the kept one, and then the chunk backwards; its decays are taken again, too (kept in
// registers they leave one wave a SIMD: 500 x 32 x 1024 x 16 training 522 us, taken again 402, of which 284 are this kernel).
template <typename T, int SPL, bool ENDS>
__global__ void __launch_bounds__(kBlock) k_scan_bwd(ScanArgs a) {
    constexpr int kCh = chunk_of(SPL), kNp = SPL * kQ, kE = kCh / SPL;
    __shared__ __attribute__((aligned(16))) float sB[2][kCh * kNp], sC[2][kCh * kNp], sums[kWaves][kCh][2 * kNp];
    const glif_scan &s = a.s;
    const glif_scan_grad &gr = a.g;
    const Lane<SPL> me(a);
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int N = s.n_state, len = scan_length(s, me.b), t0 = blockIdx.z * a.seg, t1 = min(t0 + a.seg, s.n_ticks);
    const int64_t chan = static_cast<int64_t>(me.b) * s.n_channels + me.d;
    const int64_t row = (static_cast<int64_t>(blockIdx.z) * s.n_batch) * s.n_channels + chan;
    const int64_t map_b = me.b * s.B_sb + static_cast<int64_t>(me.g) * N, map_c = me.b * s.C_sb + static_cast<int64_t>(me.g) * N;
    float A[kQ], gh[kQ] = {}, dA[kQ] = {}, steps = 0.0f, dskip = 0.0f, dbias = 0.0f;
    // a lane without a channel adds its zeros to the channels' sums: its decay is 1, as another channel's might be infinite
    load_q(A, s.A, static_cast<int64_t>(me.d) * N, me.n0, me.on ? N : 0);
#pragma unroll
    for (int j = 0; j < kQ; ++j) A[j] = rate_of(A[j]);
    if (!ENDS && me.on) {
        if (a.segs > 1) load_4(gh, a.seg_state + row * kNp + me.n0);
        else if (gr.dlast) load_q(gh, gr.dlast, chan * N, me.n0, N);
    }
    const float skip = s.D ? s.D[me.d] : 0.0f, bias = s.delta_bias ? s.delta_bias[me.d] : 0.0f;
    Maps<T, SPL> mB, mC;
    Own<T, SPL> u, delta, z, dy;
    auto fetch = [&](int c0) {
        const int to = c0 >= t0 ? len : c0;   // nothing before the segment
        mC.load(s.C, s.C_st, map_c, c0, to, N);
        delta.load(s.delta, s.delta_st, me.b * s.delta_sb, c0, to, me);
        dy.load(gr.dy, gr.dy_st, me.b * gr.dy_sb, c0, to, me);
        if (s.z) z.load(s.z, s.z_st, me.b * s.z_sb, c0, to, me);
        if (!ENDS) {
            mB.load(s.B, s.B_st, map_b, c0, to, N);
            u.load(s.u, s.u_st, me.b * s.u_sb, c0, to, me);
        }
    };
    const int first = (t1 - 1 - t0) / kCh * kCh + t0;
    fetch(first);
    for (int c0 = first, p = 0; c0 >= t0; c0 -= kCh, p ^= 1) {
        mC.store(sC[p]);
        if (!ENDS) mB.store(sB[p]);
        float own_step[kE], own_u[kE], own_su[kE], own_dy1[kE], slope[kE], dgate[kE];   // dgate: dy silu'(z)
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            own_step[e] = step_of(to_f32(delta.v[e]) + bias, s.softplus, c0 + e * SPL + me.s < len, slope[e]);
            const float g = to_f32(dy.v[e]);
            own_dy1[e] = g, dgate[e] = 0.0f, own_u[e] = 0.0f;
            if (s.z) {
                const float q = to_f32(z.v[e]), sig = sigmoid_f(q);
                own_dy1[e] = g * (q * sig);
                dgate[e] = g * (sig * fmaf(q, 1.0f - sig, 1.0f));
            }
            if (ENDS) steps += own_step[e];
            else own_u[e] = to_f32(u.v[e]);
            own_su[e] = own_step[e] * own_u[e];
        }
        __syncthreads();
        fetch(c0 - kCh);
        if constexpr (ENDS) {
#pragma unroll
            for (int e = kE - 1; e >= 0; --e)
#pragma unroll
                for (int i = SPL - 1; i >= 0; --i) {
                    const float step = bcast<SPL>(own_step[e], i), dy1 = bcast<SPL>(own_dy1[e], i);
                    float C[kQ];
                    load_4(C, sC[p] + (e * SPL + i) * kNp + me.n0);
#pragma unroll
                    for (int j = 0; j < kQ; ++j) gh[j] = fmaf(dy1, C[j], gh[j]) * __builtin_amdgcn_exp2f(step * A[j]);
                }
        } else {
            float hs[kCh + 1][kQ];   // the states before each tick, and after the last
            if (me.on) load_4(hs[0], a.keep + (static_cast<int64_t>(c0 / kCh) * s.n_batch * s.n_channels + chan) * kNp + me.n0);
            else hs[0][0] = hs[0][1] = hs[0][2] = hs[0][3] = 0.0f;
#pragma unroll
            for (int e = 0; e < kE; ++e)
#pragma unroll
                for (int i = 0; i < SPL; ++i) {
                    const int k = e * SPL + i;
                    const float step = bcast<SPL>(own_step[e], i), su = bcast<SPL>(own_su[e], i);
                    float B[kQ];
                    load_4(B, sB[p] + k * kNp + me.n0);
#pragma unroll
                    for (int j = 0; j < kQ; ++j) {
                        hs[k + 1][j] = fmaf(__builtin_amdgcn_exp2f(step * A[j]), hs[k][j], su * B[j]);
                    }
                }
#pragma unroll
            for (int e = kE - 1; e >= 0; --e) {
                float y1[SPL], gB[SPL], thA[SPL];
#pragma unroll
                for (int i = SPL - 1; i >= 0; --i) {
                    const int k = e * SPL + i;
                    const float step = bcast<SPL>(own_step[e], i), su = bcast<SPL>(own_su[e], i), dy1 = bcast<SPL>(own_dy1[e], i);
                    float B[kQ], C[kQ], dB[kQ], dC[kQ];
                    load_4(B, sB[p] + k * kNp + me.n0);
                    load_4(C, sC[p] + k * kNp + me.n0);
                    y1[i] = gB[i] = thA[i] = 0.0f;
#pragma unroll
                    for (int j = 0; j < kQ; ++j) {
                        y1[i] = fmaf(C[j], hs[k + 1][j], y1[i]);
                        gh[j] = fmaf(dy1, C[j], gh[j]);
                        dC[j] = dy1 * hs[k + 1][j];
                        dB[j] = gh[j] * su;
                        gB[i] = fmaf(gh[j], B[j], gB[i]);
                        gh[j] *= __builtin_amdgcn_exp2f(step * A[j]);
                        const float th = gh[j] * hs[k][j];
                        thA[i] = fmaf(th, A[j], thA[i]);
                        dA[j] = fmaf(th, step, dA[j]);
                    }
                    if (a.part_bc) {
                        float x[2];
                        channels_sum<SPL>(dB, dC, x);
                        if (lane % 16 < SPL)
                            *reinterpret_cast<float2 *>(&sums[wave][k][(lane >> 5) * kNp + me.n0 + (lane >> 4 & 1) * 2]) = make_float2(x[0], x[1]);
                    }
                }
                // A carries log2(e)
                const float sy = to_lane<SPL>(y1, me.s), sB_ = to_lane<SPL>(gB, me.s), sA = to_lane<SPL>(thA, me.s) * 0.69314718055994531f;
                const int t = c0 + e * SPL + me.s;
                const float draw = t < len ? fmaf(own_u[e], sB_, sA) * slope[e] : 0.0f;
                dskip = fmaf(own_dy1[e], own_u[e], dskip);
                dbias += draw;
                if (me.on && t < s.n_ticks) {
                    const int64_t at = (static_cast<int64_t>(t) * s.n_batch + me.b) * s.n_channels + me.d;
                    if (gr.du) static_cast<T *>(gr.du)[at] = from_f32<T>(t < len ? fmaf(skip, own_dy1[e], own_step[e] * sB_) : 0.0f);
                    if (gr.ddelta) static_cast<T *>(gr.ddelta)[at] = from_f32<T>(draw);
                    if (gr.dz) static_cast<T *>(gr.dz)[at] = from_f32<T>(t < len ? dgate[e] * fmaf(skip, own_u[e], sy) : 0.0f);
                }
            }
            if (a.part_bc) {
                __syncthreads();
                for (int q = threadIdx.x; q < kCh * 2 * kNp; q += kBlock) {
                    const int k = q / (2 * kNp), v = q % (2 * kNp);
                    if (c0 + k >= s.n_ticks) break;
                    float sum = sums[0][k][v];
#pragma unroll
                    for (int w = 1; w < kWaves; ++w) sum += sums[w][k][v];
                    a.part_bc[((static_cast<int64_t>(blockIdx.x) * s.n_ticks + c0 + k) * s.n_batch + me.b) * 2 * kNp + v] = sum;
                }
            }
        }
    }
    if constexpr (ENDS) {
        if (!me.on) return;
        store_4(a.seg_state + row * kNp + me.n0, gh);
#pragma unroll
        for (int m = 1; m < SPL; m <<= 1) steps += __shfl_xor(steps, m, kWave);
        if (me.s == 0) a.seg_step[row] = steps;
    } else {
#pragma unroll
        for (int m = 1; m < SPL; m <<= 1) {
            dskip += __shfl_xor(dskip, m, kWave);
            dbias += __shfl_xor(dbias, m, kWave);
        }
        if (!me.on) return;
        store_4(a.part_a + row * kNp + me.n0, dA);
        if (me.s == 0) {
            const int64_t at = (static_cast<int64_t>(blockIdx.z) * s.n_batch + me.b) * 2 * s.n_channels + me.d;
            a.part_d[at] = dskip;
            a.part_d[at + s.n_channels] = dbias;
        }
        if (gr.dstate && blockIdx.z == 0)
#pragma unroll
            for (int j = 0; j < kQ; ++j)
                if (me.n0 + j < N) gr.dstate[chan * N + me.n0 + j] = gh[j];
    }
}

// No ticks: the adjoint of the last state is that of the first.
__global__ void __launch_bounds__(kBlock) k_scan_through(const float *dlast, float *dstate, int64_t n) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kBlock)
        dstate[i] = dlast ? dlast[i] : 0.0f;
}

// dB, dC: the blocks of a group, in order.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_scan_join_bc(ScanArgs a) {
    const glif_scan &s = a.s;
    const int64_t tbs = static_cast<int64_t>(s.n_ticks) * s.n_batch, gn = static_cast<int64_t>(s.n_groups) * s.n_state, n = tbs * gn;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t tb = i / gn;
        const int g = static_cast<int>(i - tb * gn) / s.n_state, st = static_cast<int>(i - tb * gn) % s.n_state;
        float dB = 0.0f, dC = 0.0f;
        for (int k = 0; k < a.blocks; ++k) {
            const float *p = a.part_bc + ((static_cast<int64_t>(g) * a.blocks + k) * tbs + tb) * 2 * a.np + st;
            dB += p[0];
            dC += p[a.np];
        }
        if (a.g.dB) static_cast<T *>(a.g.dB)[i] = from_f32<T>(dB);
        if (a.g.dC) static_cast<T *>(a.g.dC)[i] = from_f32<T>(dC);
    }
}

// dA, dD, ddelta_bias: the segments' and batch entries' sums, in order.
__global__ void __launch_bounds__(kBlock) k_scan_join_param(ScanArgs a) {
    const glif_scan &s = a.s;
    const int64_t n = static_cast<int64_t>(s.n_channels) * a.np, i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (i >= n) return;
    const int d = static_cast<int>(i / a.np), st = static_cast<int>(i - static_cast<int64_t>(d) * a.np), rows = a.segs * s.n_batch;
    if (a.g.dA && st < s.n_state) {
        float v = 0.0f;
#pragma unroll 4
        for (int r = 0; r < rows; ++r) v += a.part_a[r * n + i];
        a.g.dA[static_cast<int64_t>(d) * s.n_state + st] = v;
    }
    if (st == 0) {
        float dD = 0.0f, db = 0.0f;
#pragma unroll 4
        for (int r = 0; r < rows; ++r) {
            dD += a.part_d[static_cast<int64_t>(r) * 2 * s.n_channels + d];
            db += a.part_d[(static_cast<int64_t>(r) * 2 + 1) * s.n_channels + d];
        }
        if (a.g.dD) a.g.dD[d] = dD;
        if (a.g.ddelta_bias) a.g.ddelta_bias[d] = db;
    }
}

// ---- one tick ---------------------------------------------------------------------------------------------------------------
// A lane's four states in 16 bytes.  Bound by the launch, then by the state's way in and out: 32 x 2048 x 16 4.4 us, 8.4 MB.
template <typename T, int SPL>
__global__ void __launch_bounds__(kBlock) k_scan_step(ScanArgs a) {
    const glif_scan &s = a.s;
    const Lane<SPL> me(a);
    if (!me.on) return;
    const int N = s.n_state, n0 = me.n0;
    const int64_t chan = static_cast<int64_t>(me.b) * s.n_channels + me.d, map = static_cast<int64_t>(me.g) * N + n0;
    const T *Bp = static_cast<const T *>(s.B) + me.b * s.B_sb + map, *Cp = static_cast<const T *>(s.C) + me.b * s.C_sb + map;
    float *hp = a.last + chan * N + n0;
    const float *Ap = s.A + static_cast<int64_t>(me.d) * N + n0;
    typedef Vec<float, kQ> fvec;
    typedef Vec<T, kQ> tvec;
    fvec A = {}, h = {};
    tvec B = {}, C = {};
    const bool whole = n0 + kQ <= N;
    if (whole) {
        A = *reinterpret_cast<const fvec *>(Ap), h = *reinterpret_cast<const fvec *>(hp);
        B = *reinterpret_cast<const tvec *>(Bp), C = *reinterpret_cast<const tvec *>(Cp);
    } else {
#pragma unroll
        for (int j = 0; j < kQ; ++j)
            if (n0 + j < N) A[j] = Ap[j], h[j] = hp[j], B[j] = Bp[j], C[j] = Cp[j];
    }
    const float u = to_f32(static_cast<const T *>(s.u)[me.b * s.u_sb + me.d]);
    const float raw = to_f32(static_cast<const T *>(s.delta)[me.b * s.delta_sb + me.d]) + (s.delta_bias ? s.delta_bias[me.d] : 0.0f);
    const float q = s.z ? to_f32(static_cast<const T *>(s.z)[me.b * s.z_sb + me.d]) : 0.0f, skip = s.D ? s.D[me.d] : 0.0f;
    float slope, y = 0.0f;
    const float step = step_of(raw, s.softplus, true, slope), su = step * u;
#pragma unroll
    for (int j = 0; j < kQ; ++j) {
        h[j] = fmaf(__builtin_amdgcn_exp2f(step * (A[j] * kLog2e)), h[j], su * to_f32(static_cast<T>(B[j])));
        y = fmaf(to_f32(static_cast<T>(C[j])), h[j], y);
    }
    if (whole) {
        *reinterpret_cast<fvec *>(hp) = h;
    } else {
#pragma unroll
        for (int j = 0; j < kQ; ++j)
            if (n0 + j < N) hp[j] = h[j];
    }
#pragma unroll
    for (int m = 1; m < SPL; m <<= 1) y += __shfl_xor(y, m, kWave);
    if (me.s != 0) return;
    y = fmaf(skip, u, y);
    if (s.z) y *= q * sigmoid_f(q);
    static_cast<T *>(a.y)[chan] = from_f32<T>(y);
}

int lanes_for(int32_t N) {
    int l = 1;
    while (l * kQ < N) l *= 2;
    return l;
}

// Blocks and segments.  Time is split where the channels give fewer than 2 waves a SIMD, into segments of at least 64 ticks
// until there are about 4.
void shape(ScanArgs &a) {
    const int spl = lanes_for(a.s.n_state), chan = kWave / spl, chunk = chunk_of(spl);
    a.np = spl * kQ;
    a.blocks = ceil_div(a.s.n_channels / a.s.n_groups, chan * kWaves);
    const int64_t waves = static_cast<int64_t>(a.blocks) * a.s.n_groups * kWaves * std::max(a.s.n_batch, 1);
    int64_t segs = waves >= 2048 ? 1 : std::max<int64_t>(1, std::min<int64_t>(4096 / waves, a.s.n_ticks / 64));
    a.seg = std::max(ceil_div(ceil_div(a.s.n_ticks, segs), chunk) * chunk, chunk);
    a.segs = std::max(1, ceil_div(a.s.n_ticks, a.seg));
}

enum Pass { kEnds, kMain, kStep };

template <typename T, int SPL>
void launch(const ScanArgs &a, bool back, Pass pass, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(a.s.n_groups * a.blocks), static_cast<unsigned>(a.s.n_batch), static_cast<unsigned>(a.segs));
    if (pass == kStep) hipLaunchKernelGGL((k_scan_step<T, SPL>), grid, dim3(kBlock), 0, st, a);
    else if (back && pass == kEnds) hipLaunchKernelGGL((k_scan_bwd<T, SPL, true>), grid, dim3(kBlock), 0, st, a);
    else if (back) hipLaunchKernelGGL((k_scan_bwd<T, SPL, false>), grid, dim3(kBlock), 0, st, a);
    else if (pass == kEnds) hipLaunchKernelGGL((k_scan_fwd<T, SPL, true>), grid, dim3(kBlock), 0, st, a);
    else hipLaunchKernelGGL((k_scan_fwd<T, SPL, false>), grid, dim3(kBlock), 0, st, a);
}

template <typename T>
void by_lanes(const ScanArgs &a, bool back, Pass pass, hipStream_t st) {
    switch (a.np / kQ) {
        case 1: return launch<T, 1>(a, back, pass, st);
        case 2: return launch<T, 2>(a, back, pass, st);
        case 4: return launch<T, 4>(a, back, pass, st);
        case 8: return launch<T, 8>(a, back, pass, st);
        default: return launch<T, 16>(a, back, pass, st);
    }
}

dim3 flat_grid(int64_t n) { return dim3(static_cast<unsigned>(std::min<int64_t>((n + kBlock - 1) / kBlock, 16384))); }

// both passes of one direction
template <typename T>
void run(const ScanArgs &a, bool back, hipStream_t st) {
    if (a.segs > 1) {
        const int64_t n = static_cast<int64_t>(a.s.n_batch) * a.s.n_channels * a.np;
        by_lanes<T>(a, back, kEnds, st);
        if (back) hipLaunchKernelGGL(k_scan_join<true>, flat_grid(n), dim3(kBlock), 0, st, a);
        else hipLaunchKernelGGL(k_scan_join<false>, flat_grid(n), dim3(kBlock), 0, st, a);
    }
    by_lanes<T>(a, back, kMain, st);
}

template <typename T>
void run_step(const ScanArgs &a, hipStream_t st) { by_lanes<T>(a, false, kStep, st); }

template <typename T>
void run_bwd(const ScanArgs &a, hipStream_t st) {
    const int64_t bc = static_cast<int64_t>(a.s.n_ticks) * a.s.n_batch * a.s.n_groups * a.s.n_state;
    if (a.s.n_batch && a.s.n_ticks) run<T>(a, true, st);
    if (a.part_bc && bc) hipLaunchKernelGGL(k_scan_join_bc<T>, flat_grid(bc), dim3(kBlock), 0, st, a);
    if (a.g.dA || a.g.dD || a.g.ddelta_bias) {
        ScanArgs none = a;
        if (!a.s.n_batch || !a.s.n_ticks) none.segs = 0;
        hipLaunchKernelGGL(k_scan_join_param, dim3(static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.s.n_channels) * a.np, kBlock))),
                           dim3(kBlock), 0, st, none);
    }
    const int64_t rows = static_cast<int64_t>(a.s.n_batch) * a.s.n_channels * a.s.n_state;
    if (!a.s.n_ticks && rows && a.g.dstate)
        hipLaunchKernelGGL(k_scan_through, flat_grid(rows), dim3(kBlock), 0, st, a.g.dlast, a.g.dstate, rows);
}

int check_scan(const glif_scan *s) {
    if (!s) return fail(GLIF_EINVAL, "NULL argument");
    if (!known_dtype(s->dtype)) return fail(GLIF_EINVAL, "state space: unknown type");
    if (s->n_ticks < 0 || s->n_ticks > (1 << 20) || s->n_batch < 0 || s->n_batch > 65535 || s->n_channels < 1 ||
        s->n_channels > (1 << 24))
        return fail(GLIF_EINVAL, "state space: ticks in [0, 2^20], batch in [0, 65535], channels in [1, 2^24]");
    if (s->n_groups < 1 || s->n_channels % s->n_groups) return fail(GLIF_EINVAL, "state space: the groups must divide the channels");
    // a launch counts its threads in 32 bits, and a group has a block of them at least
    if (s->n_groups >= (1 << 24)) return fail(GLIF_EINVAL, "state space: fewer than 2^24 groups");
    if (s->n_state < 1 || s->n_state > 64) return fail(GLIF_EINVAL, "state space: 1 to 64 states");
    return GLIF_OK;
}

bool have_inputs(const glif_scan *s) {
    return s->A && (s->n_ticks == 0 || s->n_batch == 0 || (s->u && s->delta && s->B && s->C));
}

void carve_segs(Carver &c, ScanArgs &a) {
    const size_t rows = static_cast<size_t>(a.segs) * a.s.n_batch * a.s.n_channels;
    if (a.segs > 1) {
        a.seg_state = c.take<float>(rows * a.np);
        a.seg_step = c.take<float>(rows);
    }
}

void carve(Carver &c, ScanArgs &a) {
    const size_t rows = static_cast<size_t>(a.segs) * a.s.n_batch * a.s.n_channels;
    carve_segs(c, a);
    a.part_a = c.take<float>(rows * a.np);
    a.part_d = c.take<float>(rows * 2);
    a.part_bc = c.take<float>(static_cast<size_t>(a.s.n_groups) * a.blocks * a.s.n_ticks * a.s.n_batch * 2 * a.np);
}

}  // namespace
}  // namespace glif

using namespace glif;

extern "C" {

size_t glif_scan_keep_bytes(const glif_scan *s) {
    if (check_scan(s)) return 0;
    const int spl = lanes_for(s->n_state);
    return static_cast<size_t>(ceil_div(s->n_ticks, chunk_of(spl))) * s->n_batch * s->n_channels * spl * kQ * sizeof(float);
}

size_t glif_scan_fwd_workspace(const glif_scan *s) {
    if (check_scan(s)) return 0;
    ScanArgs a{};
    a.s = *s;
    shape(a);
    Carver c(nullptr, 0);
    carve_segs(c, a);
    return c.off;
}

int glif_scan_fwd(const glif_scan *s, void *y, float *last, void *keep, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_scan(s)) return rc;
    if (s->n_batch == 0) return GLIF_OK;
    if (!have_inputs(s) || (s->n_ticks && !y)) return fail(GLIF_EINVAL, "NULL argument");
    ScanArgs a{};
    a.s = *s, a.y = y, a.last = last, a.keep = static_cast<float *>(keep);
    shape(a);
    Carver c(ws, ws_bytes);
    carve_segs(c, a);
    if (!c.ok() || (c.off && !ws)) return fail(GLIF_ENOMEM, "state space: workspace too small");
    GLIF_BY_DTYPE(s->dtype, run, a, false, static_cast<hipStream_t>(stream));
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
    if (!c.ok() || (c.off && !ws)) return fail(GLIF_ENOMEM, "state space: workspace too small");
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
    shape(a);
    a.segs = 1;
    GLIF_BY_DTYPE(s->dtype, run_step, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
