// Linear attention with a decay for each head, its backward, and its form for single ticks:
//   S[t] = lam S[t-1] + k[t] v[t]^T,   y[t] = scale q[t] S[t],   lam = exp(log_decay[h]),   S [K][V] float32
//
// Everything but the step is one function of three sequences, F(a, b, c; X): over the ticks of a chunk, counted from 0,
//   out_i = sum over j <= i of lam^(i-j) (a_i . b_j) c_j  +  lam^(i+lead) a_i X
//   X    <- lam^n X + sum over j of lam^(n-lead-j) b_j c_j^T                        (n ticks in the chunk)
//   y  = scale F(q, k, v; S0)                    lead 1
//   dq = scale F(dy, v, k; S0^T)                 lead 1
//   dk = F(v, dy, scale q; dS^T)                 lead 0, time backwards: the gradient of the last state comes undecayed to the
//   dv = F(k, scale q, dy; dS)                   last tick, and what is left behind the first is dS0
// No power is of a negative exponent, so no decay, 0 among them, can overflow.
//
// Bound by latency within a chunk: 500 x 32 ticks of 8 heads of 128, bfloat16, trials of any length, 43 us forward (a block
// of eight waves alone on its compute unit; 10.0k cycles a chunk of 64 ticks, of which the matrix instructions are 3.2k), 85 us for
// the backward's three passes; of 32 heads, all ticks, 194 us (2.7 TB/s) and 525 (3.0 TB/s, 9 sequences read and 3 written).
// In float32 (its products at 1/16 of the rate) 290 x 18 ticks of 4 heads of 128 and 64 56 us.
#include <type_traits>

#include "mma.h"

namespace glif {
namespace {

struct AttSeq {
    const void *p;
    int64_t st, sb, sh;   // strides of ticks, batch entries and heads
    int32_t share, d;     // heads of the attention that share one of it; channels
};

struct AttPass {
    AttSeq a, b, c;
    void *out;                     // [T][B][H][c.d], or NULL
    int32_t wide;                  // out is float32, to be added up over shared heads
    int32_t back, lead;
    float out_scale, in_scale;
    const float *x;                // the state before the first tick, or NULL: strides of (segment, entry and head, b's and c's channels)
    int64_t x_seg, x_bh, x_b, x_c;
    float *x_out;                  // the state after the last, likewise, or NULL
};

struct AttArgs {
    AttPass pass[3];
    int32_t passes;
    const float *log_decay;
    const int32_t *lengths;
    int32_t T, B, H, segments, seg_ticks;
};

// lam = exp(log_decay) to whole powers n >= 0: 1 for n = 0 whatever the decay is.  What is below the normal numbers is the least of
// them, as long as lam itself is not: 1e-38 of a state is nothing, and an infinite one stays infinite, as it does tick by tick.
struct Decay {
    float rate, least;   // logarithms to base 2
    __device__ __forceinline__ explicit Decay(float log_decay)
        : rate(log_decay * 1.4426950408889634f), least(rate >= -126.0f ? -126.0f : rate) {}
    __device__ __forceinline__ float power(int n) const {
        return n == 0 ? 1.0f : __builtin_amdgcn_exp2f(fmaxf(rate * static_cast<float>(n), least));
    }
};

__device__ __forceinline__ int live_ticks(const int32_t *lengths, int b, int T) { return lengths ? min(max(lengths[b], 0), T) : T; }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

#ifdef __HIP_DEVICE_COMPILE__   // the host's pass does not know the builtins
// 16-bit products of bfloat16, and float32 ones for float32 and for float16: states and scores of float16 sequences do not
// stay within its range.
template <typename T>
struct Form {
    using C = float;
    static constexpr int kTicks = 32, kStep = 16, kPer = 4;   // ticks of a chunk, terms of a matrix product, those of a lane
};
template <>
struct Form<bf16> {
    using C = bf16;
    static constexpr int kTicks = 64, kStep = 32, kPer = 8;
};

// Rows of W values in LDS.  16-bit ones are read by 16 rows of the same 16 bytes, and, turned, by four rows of 8 bytes from each
// of four neighbouring 16: the 16-byte pieces of a row are permuted so that either goes to all banks.  float32 rows are 16 bytes
// apart for the first, and their columns lie apart anyway.
template <typename C, int W>
struct Rows {
    static constexpr bool kTurned = sizeof(C) == 2;
    static constexpr int kSize = static_cast<int>(sizeof(C)), kBytes = W * kSize + (kTurned ? 0 : 16);
    static __device__ __forceinline__ int key(int row) {
        return !kTurned ? 0 : W == 128 ? (row & 3) << 2 | (row >> 2 & 3) : W == 64 ? (row & 2) << 1 | (row >> 2 & 3) : row >> 2 & 3;
    }
    // of value i of a row
    static __device__ __forceinline__ int at(int row, int i) {
        const int byte = i * kSize;
        return row * kBytes + ((byte >> 4 ^ key(row)) << 4 | (byte & 15));
    }
    // Operands: lane l holds row l % 16 and the 16 bytes' terms from the (l / 16)th on.
    static __device__ __forceinline__ typename Mma<C>::frag rows(const char *lds, int row0, int k0, int lane) {
        return *reinterpret_cast<const typename Mma<C>::frag *>(lds + at(row0 + lane % 16, k0 + lane / 16 * (16 / kSize)));
    }
    // Columns as rows, rows k0, .. as terms.  Four columns from each of c0, c0 + GAP, c0 + 2 GAP and c0 + 3 GAP.
    template <int GAP>
    static __device__ __forceinline__ typename Mma<C>::frag columns(const char *lds, int c0, int k0, int lane) {
        const int r16 = lane % 16, kq = lane / 16;
        if constexpr (kTurned) {
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s4 *l4;
            const int row = k0 + 8 * kq + (r16 >> 2), col = c0 + (r16 & 3) * GAP;
            const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l4)(lds + at(row, col)));
            const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l4)(lds + at(row + 4, col)));
            return __builtin_bit_cast(typename Mma<C>::frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            static_assert(GAP == 4, "columns in order");
            typename Mma<C>::frag v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const C *>(lds + at(k0 + 4 * kq + e, c0 + r16));
            return v;
        }
    }
};

// kTicks x W of a sequence from memory to rows of LDS, in two steps: thread by thread the same 16 bytes of rows kRows apart, so
// that of a whole chunk of whole rows one address and nothing else is a lane's.  No load waits for a condition: ticks and
// channels that are not there repeat others, and are put away as zeros (channels never: init() clears them).
// WHOLE: all W channels are there.
template <typename T, int W, int NT, bool WHOLE>
struct Tile {
    using F = Form<T>;
    using C = typename F::C;
    static constexpr int kSize = static_cast<int>(sizeof(T)), kV = kVecBytes16<T>;
    using R = Rows<C, W>;
    static constexpr int kBytes = F::kTicks * R::kBytes, kAcross = W / kV, kRows = NT / kAcross, kN = (F::kTicks + kRows - 1) / kRows;
    static_assert(NT % kAcross == 0, "a thread keeps to its channels");
    typedef Vec<T, kV> vec;
    vec r[kN];
    const char *base;     // of the sequence's channels
    int64_t step;         // bytes from a tick to the next, in their order
    int row, at;          // the thread's first row and channel
    int d;                // channels
    uint32_t off;         // its first bytes in a whole chunk, from the lowest tick

    static __device__ __forceinline__ int least(int a, int b) { return a < b ? a : b; }
    // the first channel that is read: the last piece is moved back to end with them
    __device__ __forceinline__ int from() const { return WHOLE ? at : d < kV ? 0 : least(at, d - kV); }

    __device__ __forceinline__ void init(char *lds, const T *p, int64_t st, bool back, int channels) {
        base = reinterpret_cast<const char *>(p), step = back ? -st * kSize : st * kSize, d = channels;
        row = threadIdx.x / kAcross, at = threadIdx.x % kAcross * kV;
        const int first = least(row, F::kTicks - 1);
        off = static_cast<uint32_t>(back ? F::kTicks - 1 - first : first) * static_cast<uint32_t>(st * kSize) + static_cast<uint32_t>(from() * kSize);
        for (int u = threadIdx.x; u < kBytes / 4; u += NT) reinterpret_cast<uint32_t *>(lds)[u] = 0u;
    }
    // n ticks, the first of them `first`
    __device__ __forceinline__ void load(int64_t first, int n) {
        const bool back = step < 0;
        const int64_t apart = back ? -step : step;
        const char *low = base + (back ? first - (n - 1) : first) * apart;
        if (n == F::kTicks && (WHOLE || d >= kV)) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                r[i] = *reinterpret_cast<const vec *>(low + i * kRows * step + off);
            }
            return;
        }
        int mine = row;
        asm volatile("" : "+v"(mine));   // what follows is for the few other chunks: it must not take registers of the loop
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int at_row = least(mine + i * kRows, n - 1);
            const char *q = low + (static_cast<uint32_t>(back ? n - 1 - at_row : at_row) * static_cast<uint32_t>(apart) + static_cast<uint32_t>(from() * kSize));
            if (WHOLE || d >= kV) {
                r[i] = *reinterpret_cast<const vec *>(q);
            } else {
#pragma unroll
                for (int e = 0; e < kV; ++e) r[i][e] = e < d ? reinterpret_cast<const T *>(q)[least(e, d - 1)] : T(0.0f);
            }
        }
    }
    __device__ __forceinline__ void store(char *lds, int n) const {
        constexpr int kE = 16 / static_cast<int>(sizeof(C));
        typedef C out __attribute__((ext_vector_type(16 / sizeof(C))));
        if (n == F::kTicks && (WHOLE || d == W)) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                if (kN * kRows > F::kTicks && row + i * kRows >= F::kTicks) break;
#pragma unroll
                for (int s = 0; s < kV / kE; ++s) {
                    out o;
#pragma unroll
                    for (int e = 0; e < kE; ++e) o[e] = static_cast<C>(r[i][s * kE + e]);
                    *reinterpret_cast<out *>(lds + R::at(row + i * kRows, at + s * kE)) = o;
                }
            }
            return;
        }
        int mine = row;
        asm volatile("" : "+v"(mine));
        // the piece that was moved back moves on again; behind the channels are zeros
        const int bits = WHOLE ? 0 : least(at - from(), kV) * kSize * 8;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int to_row = mine + i * kRows;
            if (kN * kRows > F::kTicks && to_row >= F::kTicks) break;
            u64x2 w = __builtin_bit_cast(u64x2, r[i]);
            if (bits >= 128 || to_row >= n) {
                w = u64x2{0, 0};
            } else if constexpr (!WHOLE) {
                if (bits >= 64) w = u64x2{w[1] >> (bits - 64), 0};
                else if (bits > 0) w = u64x2{w[0] >> bits | w[1] << (64 - bits), w[1] >> bits};
            }
            const vec v = __builtin_bit_cast(vec, w);
#pragma unroll
            for (int s = 0; s < kV / kE; ++s) {
                out o;
#pragma unroll
                for (int e = 0; e < kE; ++e) o[e] = static_cast<C>(v[s * kE + e]);
                *reinterpret_cast<out *>(lds + R::at(to_row, at + s * kE)) = o;
            }
        }
    }
};

// Two bfloat16 in 32 bits.
__device__ __forceinline__ float low_half(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ uint32_t larger_halves(uint32_t a, uint32_t b) {
    typedef uint16_t pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair, a), __builtin_bit_cast(pair, b)));
}
__device__ __forceinline__ uint32_t two_halves(float lo, float hi) {   // to nearest even, one instruction (from conversions of both it made two)
    uint32_t w;
    asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(w) : "v"(lo), "v"(hi));
    return w;
}
// Scores and states that are multiplied as bfloat16: four as two values each, 16 bits together, which leaves outputs at their last
// rounding (500 x 32 ticks of 8 heads of 128 forward 42.9 us, backward 84.8; states as one value,
// 40.2 and 70.4, put as much error again into outputs that come from before their chunk, and far more where their terms cancel).
// What is left of an infinity, NaN by the difference, is made finite (what is left of a finite value is within it).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void two_parts(f32x4 v, u32x2 &first, u32x2 &rest) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float lo = v[2 * e], hi = v[2 * e + 1];
        first[e] = two_halves(lo, hi);
        rest[e] = two_halves(fmaxf(lo - low_half(first[e]), -1e36f), fmaxf(hi - high_half(first[e]), -1e36f));
    }
}
// Likewise eight of a state, as two operands.
__device__ __forceinline__ void two_parts(f32x4 v, f32x4 w, Mma<bf16>::frag (&parts)[2]) {
    u32x2 first[2], rest[2];
    two_parts(v, first[0], rest[0]);
    two_parts(w, first[1], rest[1]);
    parts[0] = __builtin_bit_cast(Mma<bf16>::frag, __builtin_shufflevector(first[0], first[1], 0, 1, 2, 3));
    parts[1] = __builtin_bit_cast(Mma<bf16>::frag, __builtin_shufflevector(rest[0], rest[1], 0, 1, 2, 3));
}

// The state's first row (b's channel) of the four that a lane holds in x[i].
template <int PER>
__device__ __forceinline__ int state_row(int i, int kq) { return PER == 8 ? 32 * (i / 2) + 8 * kq + 4 * (i % 2) : 16 * i + 4 * kq; }

// Whether some value of the wave's operands is not finite.
template <int N>
__device__ __forceinline__ bool any_odd(const Mma<bf16>::frag (&f)[N]) {
    uint32_t most = 0;
#pragma unroll
    for (int s = 0; s < N; ++s) {
        const u32x4 w = __builtin_bit_cast(u32x4, f[s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) most = larger_halves(most, w[e] & 0x7fff7fffu);
    }
    return __builtin_amdgcn_ballot_w64((most & 0xffffu) >= 0x7f80u || most >> 16 >= 0x7f80u) != 0;
}
template <int N>
__device__ __forceinline__ bool any_odd(const f32x4 (&f)[N]) {
    uint32_t most = 0;
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max(most, __float_as_uint(f[s][e]) & 0x7fffffffu);   // (a bit cast of an element takes the first)
    return __builtin_amdgcn_ballot_w64(most >= 0x7f800000u) != 0;
}

__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}
// A chunk's values times their weights, which the float32 state adds up: what a matrix instruction multiplies is not float32, so they
// are three bfloat16 values, 24 bits together.  odd: of one that is not finite the first is all (the difference would be NaN).
template <typename W>
__device__ __forceinline__ void three_parts(Mma<bf16>::frag c, W weight, bool odd, Mma<bf16>::frag (&parts)[3]) {
    const u32x4 two = __builtin_bit_cast(u32x4, c);
    u32x4 got[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float lo = low_half(two[e]) * weight(2 * e), hi = high_half(two[e]) * weight(2 * e + 1);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            got[q][e] = two_halves(lo, hi);
            lo -= low_half(got[q][e]), hi -= high_half(got[q][e]);
        }
    }
    if (odd)
#pragma unroll
        for (int q = 1; q < 3; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) got[q][e] = finite_halves(got[q][e]);
#pragma unroll
    for (int q = 0; q < 3; ++q) parts[q] = __builtin_bit_cast(Mma<bf16>::frag, got[q]);
}

// Answers to a chunk whose c is not finite in a wave's channels: tick by tick, as the definition has it, since a later tick's c
// would be multiplied by an earlier one's 0, and an infinite one, in scores of several values and with b's zeros from channel d on, by
// numbers of both signs and 0.  put(i, sum) takes tick i's answers, before their scale, of the lanes with kq = 0.
template <typename C, typename RD, typename RC, int PER, bool WHOLE, int XT, typename Put>
__device__ __forceinline__ void by_ticks(const char *ta, const char *tb, const char *tc, int n, int d, int wc, int lane, Decay decay,
                                         int lead, float in_scale, f32x4 (&x)[XT], Put put) {
    typedef C four __attribute__((ext_vector_type(4)));
    const float before = decay.power(lead), after = decay.power(1 - lead);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        asm volatile("" : "+v"(lane));   // this way is rare: its addresses and rows take no registers of the other
        const int r16 = lane % 16, kq = lane / 16;
        const float c = static_cast<float>(*reinterpret_cast<const C *>(tc + RC::at(i, wc + r16))) * in_scale;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < XT; ++k) {
            const int row = state_row<PER>(k, kq), at = RD::at(i, row);
            const four fb = *reinterpret_cast<const four *>(tb + at), fa = *reinterpret_cast<const four *>(ta + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float z = WHOLE || row + e < d ? x[k][e] * before + static_cast<float>(fb[e]) * c : 0.0f;
                sum += static_cast<float>(fa[e]) * z;
                x[k][e] = z * after;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        sum += __shfl_xor(sum, 16, kWave);
        sum += __shfl_xor(sum, 32, kWave);
        if (kq == 0) put(i, sum);
    }
}
#endif

// A block takes one pass of one entry and head, 16 of c's channels a wave, and one segment of the ticks, chunk by chunk; each wave keeps the
// state of its channels in registers, as a matrix product's result and the next one's operand (which of b's channels a row of it
// is, is chosen so that a lane's values are kPer neighbours).  STATES: no outputs, only the state that the segment adds to
// nothing.
// WHOLE: all heads have D channels in b and 16 NW in c, and outputs are of type T.
// Two blocks of float16 heads of 128 share a unit by 128 registers a wave (16 to 48 bytes spilled by the way of single ticks; 500 x 32
// ticks of 8 heads with gradients 377 us, one block 398; float32 ones lose by it, 450 against 415).
template <typename T, int D, int NW, bool STATES, bool WHOLE>
__global__ void __launch_bounds__(NW *kWave, D == 32 || (std::is_same_v<T, f16> && NW == 8) ? 4 : 2) k_attention(AttArgs args) {
#ifdef __HIP_DEVICE_COMPILE__
    using F = Form<T>;
    using C = typename F::C;
    using M = Mma<C>;
    typedef typename M::frag frag;
    constexpr int kTicks = F::kTicks, kStep = F::kStep, kPer = F::kPer, TI = kTicks / 16, KT = kTicks / kStep, KD = D / kStep;
    constexpr int NT = NW * kWave, W = NW * 16, XT = D / 16, GAP = kPer == 8 ? 8 : 4, kSize = static_cast<int>(sizeof(C));
    constexpr int kHalves = kSize == 2 ? 2 : 1;   // parts of a score, and of a state
    using TD = Tile<T, D, NT, WHOLE>;
    using TC = Tile<T, W, NT, WHOLE>;
    using RD = Rows<C, D>;
    using RC = Rows<C, W>;
    using RP = Rows<C, kTicks>;
    __shared__ __attribute__((aligned(16))) char lds_a[STATES ? 16 : TD::kBytes];
    __shared__ __attribute__((aligned(16))) char lds_b[TD::kBytes];
    __shared__ __attribute__((aligned(16))) char lds_c[TC::kBytes];
    __shared__ __attribute__((aligned(16))) char lds_p[kHalves][STATES ? 16 : kTicks * RP::kBytes];
    __shared__ __attribute__((aligned(32))) float weight[kTicks];   // of tick j in the state after the chunk
    __shared__ float apart[STATES ? 1 : kTicks + 16], across[STATES ? 1 : kTicks];   // decays of scores by distance, backwards; of the state by tick

    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r16 = lane % 16, kq = lane / 16;
    // The blocks that read the same sequences are on one XCD (block id mod 8), after each other.
    const int passes = args.passes, slot = static_cast<int>(blockIdx.x >> 3);
    const int64_t group = static_cast<int64_t>(slot / passes) * 8 + (blockIdx.x & 7);
    if (group >= static_cast<int64_t>(args.B) * args.H * args.segments) return;
    const AttPass &pass = args.pass[slot % passes];
    const int seg = static_cast<int>(group % args.segments);
    const int bh = static_cast<int>(group / args.segments), b = bh / args.H, h = bh % args.H;
    const int dc = WHOLE ? W : pass.c.d, db = WHOLE ? D : pass.b.d;
    const int len = live_ticks(args.lengths, b, args.T), seg_first = seg * args.seg_ticks, seg_end = min(args.T, seg_first + args.seg_ticks);
    const int begin = min(seg_first, len), end = min(seg_end, len);
    const Decay decay(args.log_decay[h]);
    const int wc = wave * 16;            // the wave's first channel
    const bool active = wc < dc, back = pass.back, wide = !WHOLE && pass.wide;
    const int lead = pass.lead;
    const float in_scale = pass.in_scale, out_scale = pass.out_scale;
    const int64_t out_st = static_cast<int64_t>(args.B) * args.H * dc;
    void *const out = pass.out;
    const int64_t out_lane = static_cast<int64_t>(bh) * dc + wc + 4 * kq;   // of the four channels that the lane writes
    const int have = dc - wc - 4 * kq;                                      // those that are there

    TD ra, rb;
    TC rc;
    if (!STATES) ra.init(lds_a, static_cast<const T *>(pass.a.p) + b * pass.a.sb + h / pass.a.share * pass.a.sh, pass.a.st, back, db);
    rb.init(lds_b, static_cast<const T *>(pass.b.p) + b * pass.b.sb + h / pass.b.share * pass.b.sh, pass.b.st, back, db);
    rc.init(lds_c, static_cast<const T *>(pass.c.p) + b * pass.c.sb + h / pass.c.share * pass.c.sh, pass.c.st, back, dc);
    auto fetch = [&](int at, int n) {
        const int64_t first = back ? len - 1 - at : at;
        if (!STATES) ra.load(first, n);
        rb.load(first, n);
        rc.load(first, n);
    };
    if (begin < end) fetch(begin, min(end - begin, kTicks));

    // state: x[i][r] is of b's channel row(i) + r and c's channel wc + r16
    auto row = [&](int i) { return state_row<kPer>(i, kq); };
    f32x4 x[XT] = {};
    if (!STATES && pass.x && active) {
        const int64_t x_b = pass.x_b;
        const float *from = pass.x + seg * pass.x_seg + bh * pass.x_bh + min(wc + r16, dc - 1) * pass.x_c;
#pragma unroll
        for (int i = 0; i < XT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[i][r] = from[min(row(i) + r, db - 1) * x_b];
#pragma unroll
        for (int i = 0; i < XT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row(i) + r >= db || wc + r16 >= dc) x[i][r] = 0.0f;
    }

    if (!STATES) {   // scores above the diagonal tiles are 0, and stay so
        for (int u = threadIdx.x; u < kHalves * kTicks * RP::kBytes / 4; u += NT) reinterpret_cast<uint32_t *>(lds_p)[u] = 0u;
    }
    if (!STATES && threadIdx.x < kTicks) {
        const int i = threadIdx.x;
        apart[kTicks - 1 - i] = decay.power(i) * in_scale * out_scale;
        across[i] = decay.power(i + lead) * out_scale;
    }

    int weighed = 0;
    for (int at = begin; at < end;) {
        const int n = min(end - at, kTicks);
        int l = lane;
        asm volatile("" : "+v"(l));   // addresses are made again for every chunk rather than kept, which would take more registers than there are
        __syncthreads();   // the last chunk's tiles have been read
        if (!STATES) ra.store(lds_a, n);
        rb.store(lds_b, n);
        rc.store(lds_c, n);
        if (n != weighed) {
            if (threadIdx.x < kTicks) {
                const int j = threadIdx.x;
                weight[j] = j < n ? decay.power(n - lead - j) * in_scale : 0.0f;
            }
            weighed = n;
        }
        __syncthreads();
        const int here = at;
        at += n;
        if (at < end) fetch(at, min(end - at, kTicks));
        if (!STATES) {
            // scores: rows j, columns i
            constexpr int kTiles = TI * (TI + 1) / 2, kMost = (kTiles + NW - 1) / NW;
            auto scores = [&](auto count) {   // of the wave's tiles wave, wave + NW, ..: their products are taken together
                constexpr int N = decltype(count)::value;
                int it[N], jt[N];
                f32x4 s[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int u = wave + i * NW;
                    it[i] = u < 1 ? 0 : u < 3 ? 1 : u < 6 ? 2 : 3, jt[i] = u - it[i] * (it[i] + 1) / 2;
                    s[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
                for (int k = 0; k < KD; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        s[i] = M::run(RD::rows(lds_b, 16 * jt[i], k * kStep, l), RD::rows(lds_a, 16 * it[i], k * kStep, l), s[i]);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float *by = apart + kTicks - 1 - 16 * (it[i] - jt[i]) - r16 + 4 * kq;   // (past its end in scores that are masked)
                    f32x4 o;
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = it[i] > jt[i] || 4 * kq + r <= r16 ? s[i][r] * by[r] : 0.0f;
                    const int to = RP::at(16 * it[i] + r16, 16 * jt[i] + 4 * kq);
                    if constexpr (kHalves == 2) {
                        u32x2 first, rest;
                        two_parts(o, first, rest);
                        *reinterpret_cast<u32x2 *>(lds_p[0] + to) = first, *reinterpret_cast<u32x2 *>(lds_p[1] + to) = rest;
                    } else {
                        *reinterpret_cast<f32x4 *>(lds_p[0] + to) = o;
                    }
                }
            };
            if (wave < kTiles - (kMost - 1) * NW) scores(std::integral_constant<int, kMost>{});
            else if constexpr (kMost > 1) scores(std::integral_constant<int, kMost - 1>{});
            __syncthreads();
        }
        if (!active) continue;
        frag fc[KT];
#pragma unroll
        for (int s = 0; s < KT; ++s) fc[s] = RC::template columns<4>(lds_c, wave * 16, s * kStep, l);
        const bool odd = (!STATES || kSize == 2) && any_odd(fc);
        if (!STATES && odd) {
            by_ticks<C, RD, RC, kPer, WHOLE>(lds_a, lds_b, lds_c, n, db, wc, l, decay, lead, in_scale, x, [&](int i, float sum) {
                if (!out || wc + r16 >= dc) return;
                const int64_t to = (back ? len - 1 - here - i : here + i) * out_st + static_cast<int64_t>(bh) * dc + wc + r16;
                if (wide) static_cast<float *>(out)[to] = sum * out_scale;
                else static_cast<T *>(out)[to] = from_f32<T>(sum * out_scale);
            });
            continue;
        }
        if (!STATES && out) {
            // rows c's channels, columns i
            f32x4 o[TI] = {};
#pragma unroll
            for (int k = 0; k < KD; ++k) {
                frag fx[kHalves];
                if constexpr (kHalves == 2) two_parts(x[2 * k], x[2 * k + 1], fx);
                else fx[0] = x[k];
#pragma unroll
                for (int it = 0; it < TI; ++it) {
                    const frag fa = RD::rows(lds_a, 16 * it, k * kStep, l);
#pragma unroll
                    for (int q = 0; q < kHalves; ++q) o[it] = M::run(fx[q], fa, o[it]);
                }
            }
#pragma unroll
            for (int it = 0; it < TI; ++it) o[it] *= across[16 * it + (l & 15)];
#pragma unroll
            for (int s = 0; s < KT; ++s)
#pragma unroll
                for (int it = 0; it < TI; ++it)
#pragma unroll
                    for (int q = 0; q < kHalves; ++q)
                        if (s * kStep <= 16 * it + 15) o[it] = M::run(fc[s], RP::rows(lds_p[q], 16 * it, s * kStep, l), o[it]);
            const int64_t by_tick = back ? -out_st : out_st;
            const int64_t to = (back ? len - 1 - here : here) * out_st + out_lane + r16 * by_tick;
            if (n == kTicks && (WHOLE || (dc - wc >= 16 && !wide))) {
                T *q = static_cast<T *>(out) + to;
#pragma unroll
                for (int it = 0; it < TI; ++it) *reinterpret_cast<Vec<T, 4> *>(q + 16 * it * by_tick) = __builtin_convertvector(o[it], Vec<T, 4>);
            } else {
#pragma unroll
                for (int it = 0; it < TI; ++it) {
                    if (16 * it + r16 >= n) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (!WHOLE && e >= have) continue;
                        if (wide) static_cast<float *>(out)[to + 16 * it * by_tick + e] = o[it][e];
                        else static_cast<T *>(out)[to + 16 * it * by_tick + e] = from_f32<T>(o[it][e]);
                    }
                }
            }
        }
        const float f = decay.power(n);
#pragma unroll
        for (int i = 0; i < XT; ++i) x[i] *= f;
        constexpr int kParts = kSize == 2 ? 3 : 1;
#pragma unroll
        for (int s = 0; s < KT; ++s) {
            frag part[kParts];
            typedef float many __attribute__((ext_vector_type(kPer)));
            const many w = *reinterpret_cast<const many *>(weight + s * kStep + kq * kPer);
            if constexpr (kSize == 2) three_parts(fc[s], [&](int e) { return w[e]; }, STATES && odd, part);
            else part[0] = fc[s] * w;
#pragma unroll
            for (int i = 0; i < XT; ++i) {
                const frag fb = RD::template columns<GAP>(lds_b, kPer == 8 ? 32 * (i / 2) + 4 * (i % 2) : 16 * i, s * kStep, l);
#pragma unroll
                for (int q = 0; q < kParts; ++q) x[i] = M::run(fb, part[q], x[i]);
            }
        }
    }
    // Ticks behind the length are 0.
    if (!STATES && out) {
        const int t0 = max(len, seg_first);
        for (int u = threadIdx.x; u < (seg_end - t0) * dc; u += NT) {
            const int64_t to = (t0 + u / dc) * out_st + static_cast<int64_t>(bh) * dc + u % dc;
            if (wide) static_cast<float *>(out)[to] = 0.0f;
            else static_cast<T *>(out)[to] = T(0.0f);
        }
    }
    if (pass.x_out && active && wc + r16 < dc) {
        const int64_t x_b = pass.x_b;
        float *to = pass.x_out + seg * pass.x_seg + bh * pass.x_bh + (wc + r16) * pass.x_c;
#pragma unroll
        for (int i = 0; i < XT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row(i) + r < db) to[(row(i) + r) * x_b] = x[i][r];
    }
#endif
}

// The same for bfloat16 heads of D = 16 NW channels in all three sequences, on 16 bytes, of which the tiles go to LDS without
// registers, a chunk ahead: two of each, and two barriers a chunk.
template <int D, int NW, int TICKS, bool STATES>
__global__ void __launch_bounds__(NW *kWave, NW == 8 && TICKS == 32 ? 4 : 2) k_attention_direct(AttArgs args) {
#ifdef __HIP_DEVICE_COMPILE__
    using M = Mma<bf16>;
    typedef M::frag frag;
    using R = Rows<bf16, D>;
    using RP = Rows<bf16, TICKS>;
    constexpr int kTicks = TICKS, TI = TICKS / 16, KT = TICKS / 32, KD = D / 32, XT = D / 16, NT = NW * kWave, kTile = kTicks * R::kBytes;
    constexpr int kLoad = 16 * kWave, kN = kTile / kLoad / NW, kAcross = R::kBytes / 16;   // bytes of a wave's load, a wave's loads, lanes of a row
    static_assert(D == 16 * NW && kN * kLoad * NW == kTile, "the tiles divide among the waves");
    // two of each, by names of their own: reads of the one must not wait for loads to the other
    __shared__ __attribute__((aligned(1024))) char a0[STATES ? 16 : kTile], a1[STATES ? 16 : kTile];
    __shared__ __attribute__((aligned(1024))) char b0[kTile], b1[kTile], c0[kTile], c1[kTile];
    __shared__ __attribute__((aligned(16))) char lds_p[2][STATES ? 16 : kTicks * RP::kBytes];   // the scores' two parts
    __shared__ f32x4 weight[kTicks / 4];
    __shared__ float apart[STATES ? 1 : kTicks + 16], across[STATES ? 1 : kTicks];

    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r16 = lane % 16, kq = lane / 16;
    const int passes = args.passes, slot = static_cast<int>(blockIdx.x >> 3);
    const int64_t group = static_cast<int64_t>(slot / passes) * 8 + (blockIdx.x & 7);
    if (group >= static_cast<int64_t>(args.B) * args.H * args.segments) return;
    const AttPass &pass = args.pass[slot % passes];
    const int seg = static_cast<int>(group % args.segments);
    const int bh = static_cast<int>(group / args.segments), b = bh / args.H, h = bh % args.H;
    const int len = live_ticks(args.lengths, b, args.T), seg_first = seg * args.seg_ticks, seg_end = min(args.T, seg_first + args.seg_ticks);
    const int begin = min(seg_first, len), end = min(seg_end, len);
    const Decay decay(args.log_decay[h]);
    const int wc = wave * 16, lead = pass.lead;
    const bool back = pass.back;
    const float in_scale = pass.in_scale, out_scale = pass.out_scale;
    const int64_t out_st = static_cast<int64_t>(args.B) * args.H * D;
    bf16 *const out = static_cast<bf16 *>(pass.out);
    const int64_t out_lane = static_cast<int64_t>(bh) * D + wc + 4 * kq;

    const bf16 *const pa = static_cast<const bf16 *>(pass.a.p) + b * pass.a.sb + h / pass.a.share * pass.a.sh;
    const bf16 *const pb = static_cast<const bf16 *>(pass.b.p) + b * pass.b.sb + h / pass.b.share * pass.b.sh;
    const bf16 *const pc = static_cast<const bf16 *>(pass.c.p) + b * pass.c.sb + h / pass.c.share * pass.c.sh;
    const int64_t a_st = pass.a.st, b_st = pass.b.st, c_st = pass.c.st;
    // n ticks from `at` on to a tile: what lands at a lane's place is the piece that belongs there by the rows' permutation;
    // rows past the n repeat the last
    auto bring = [&](const bf16 *p, int64_t st, int at, int n, char *to) {
        typedef __attribute__((address_space(3))) void *lptr;
        const bf16 *low = p + (back ? len - at - n : at) * st;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16 *>(low), 0, -1, 0x00020000);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int inst = wave * kN + i, row = inst * (kWave / kAcross) + lane / kAcross, piece = lane % kAcross ^ R::key(row), have = min(row, n - 1);
            const uint32_t off = static_cast<uint32_t>(back ? n - 1 - have : have) * static_cast<uint32_t>(st * 2) + static_cast<uint32_t>(piece * 16);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lptr)(to + inst * kLoad), 16, off, 0, 0, 0);
        }
    };
    auto fetch = [&](int at, int n, char *ta, char *tb, char *tc) {
        if (!STATES) bring(pa, a_st, at, n, ta);
        bring(pb, b_st, at, n, tb);
        bring(pc, c_st, at, n, tc);
    };
    if (begin < end) fetch(begin, min(end - begin, kTicks), a0, b0, c0);

    // state: x[i][r] is of b's channel row(i) + r and c's channel wc + r16
    auto row = [&](int i) { return state_row<8>(i, kq); };
    f32x4 x[XT] = {};
    if (!STATES && pass.x) {
        const int64_t x_b = pass.x_b;
        const float *from = pass.x + seg * pass.x_seg + bh * pass.x_bh + (wc + r16) * pass.x_c;
        if (x_b == 1) {
#pragma unroll
            for (int i = 0; i < XT; ++i) x[i] = *reinterpret_cast<const Vec<f32, 4> *>(from + row(i));
        } else {
#pragma unroll
            for (int i = 0; i < XT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[i][r] = from[(row(i) + r) * x_b];
        }
    }
    if (!STATES) {   // scores above the diagonal tiles are 0, and stay so
        for (int u = threadIdx.x; u < 2 * kTicks * RP::kBytes / 4; u += NT) reinterpret_cast<uint32_t *>(lds_p)[u] = 0u;
        if (threadIdx.x < kTicks) {
            const int i = threadIdx.x;
            apart[kTicks - 1 - i] = decay.power(i) * in_scale * out_scale;
            across[i] = decay.power(i + lead) * out_scale;
        }
    }

    // What has to be there before a chunk is gone through: its tiles, without what is behind its n ticks, its weights and
    // scores.
    auto ready = [&](int n, char *ta, char *tb, char *tc) {
        int l = lane, tid = threadIdx.x;
        if (TICKS == 32) asm volatile("" : "+v"(l), "+v"(tid));   // addresses are made again for every chunk: kept, they take more registers than two blocks have
        const int r16 = l % 16, kq = l / 16;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (n < kTicks) {
            for (int u = tid; u < (kTicks - n) * R::kBytes / 4; u += NT) {
                const int at = n * R::kBytes + u * 4;
                if (!STATES) *reinterpret_cast<uint32_t *>(ta + at) = 0u;
                *reinterpret_cast<uint32_t *>(tb + at) = 0u;
                *reinterpret_cast<uint32_t *>(tc + at) = 0u;
            }
            __syncthreads();
        }
        if (tid < kTicks) {
            const int j = tid;
            weight[j / 4][j % 4] = j < n ? decay.power(n - lead - j) * in_scale : 0.0f;
        }
        if (!STATES) {
            constexpr int kTiles = TI * (TI + 1) / 2, kMost = (kTiles + NW - 1) / NW;
            auto scores = [&](auto count) {   // of the wave's tiles wave, wave + NW, ..: their products are taken together
                constexpr int N = decltype(count)::value;
                int it[N], jt[N];
                f32x4 s[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int u = wave + i * NW;
                    it[i] = u < 1 ? 0 : u < 3 ? 1 : u < 6 ? 2 : 3, jt[i] = u - it[i] * (it[i] + 1) / 2;
                    s[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
                for (int k = 0; k < KD; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) s[i] = M::run(R::rows(tb, 16 * jt[i], k * 32, l), R::rows(ta, 16 * it[i], k * 32, l), s[i]);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float *by = apart + kTicks - 1 - 16 * (it[i] - jt[i]) - r16 + 4 * kq;   // (past its end in scores that are masked)
                    f32x4 o;
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = it[i] > jt[i] || 4 * kq + r <= r16 ? s[i][r] * by[r] : 0.0f;
                    u32x2 first, rest;
                    two_parts(o, first, rest);
                    const int to = RP::at(16 * it[i] + r16, 16 * jt[i] + 4 * kq);
                    *reinterpret_cast<u32x2 *>(lds_p[0] + to) = first, *reinterpret_cast<u32x2 *>(lds_p[1] + to) = rest;
                }
            };
            if (wave < kTiles - (kMost - 1) * NW) scores(std::integral_constant<int, kMost>{});
            else if constexpr (kMost > 1) scores(std::integral_constant<int, kMost - 1>{});
        }
        __syncthreads();
    };

    int at = begin;
    auto chunk = [&](const char *ta, const char *tb, const char *tc, char *na, char *nb, char *nc) {   // and the next one's tiles
        const int n = min(end - at, kTicks), here = at;
        int l = lane;
        if (TICKS == 32) asm volatile("" : "+v"(l));
        const int r16 = l % 16, kq = l / 16;
        at += n;
        if (at < end) fetch(at, min(end - at, kTicks), na, nb, nc);
        frag fc[KT];
#pragma unroll
        for (int s = 0; s < KT; ++s) fc[s] = R::template columns<4>(tc, wc, s * 32, l);
        const bool odd = any_odd(fc);
        if (!STATES && odd) {
            by_ticks<bf16, R, R, 8, true>(ta, tb, tc, n, D, wc, l, decay, lead, in_scale, x, [&](int i, float sum) {
                const int64_t to = (back ? len - 1 - here - i : here + i) * out_st + static_cast<int64_t>(bh) * D + wc + r16;
                if (out) out[to] = static_cast<bf16>(sum * out_scale);
            });
        } else {
            if (!STATES && out) {
                // rows c's channels, columns i
                f32x4 o[TI] = {};
#pragma unroll
                for (int k = 0; k < KD; ++k) {
                    frag fx[2];
                    two_parts(x[2 * k], x[2 * k + 1], fx);
#pragma unroll
                    for (int it = 0; it < TI; ++it) {
                        const frag fa = R::rows(ta, 16 * it, k * 32, l);
#pragma unroll
                        for (int q = 0; q < 2; ++q) o[it] = M::run(fx[q], fa, o[it]);
                    }
                }
#pragma unroll
                for (int it = 0; it < TI; ++it) o[it] *= across[16 * it + r16];
#pragma unroll
                for (int s = 0; s < KT; ++s)
#pragma unroll
                    for (int it = 0; it < TI; ++it)
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            if (s * 32 <= 16 * it + 15) o[it] = M::run(fc[s], RP::rows(lds_p[q], 16 * it, s * 32, l), o[it]);
                const int64_t by_tick = back ? -out_st : out_st;
                bf16 *to = out + (back ? len - 1 - here : here) * out_st + out_lane + r16 * by_tick;
#pragma unroll
                for (int it = 0; it < TI; ++it)
                    if (16 * it + r16 < n) *reinterpret_cast<Vec<bf16, 4> *>(to + 16 * it * by_tick) = __builtin_convertvector(o[it], Vec<bf16, 4>);
            }
            const float f = decay.power(n);
#pragma unroll
            for (int i = 0; i < XT; ++i) x[i] *= f;
#pragma unroll
            for (int s = 0; s < KT; ++s) {
                const f32x4 w4[2] = {weight[s * 8 + kq * 2], weight[s * 8 + kq * 2 + 1]};
                frag part[3];
                three_parts(fc[s], [&](int e) { return w4[e / 4][e % 4]; }, STATES && odd, part);
#pragma unroll
                for (int i = 0; i < XT; ++i) {
                    const frag fb = R::template columns<8>(tb, 32 * (i / 2) + 4 * (i % 2), s * 32, l);
#pragma unroll
                    for (int q = 0; q < 3; ++q) x[i] = M::run(fb, part[q], x[i]);
                }
            }
        }
        if (at < end) ready(min(end - at, kTicks), na, nb, nc);
    };
    if (begin < end) ready(min(end - begin, kTicks), a0, b0, c0);
    while (at < end) {
        chunk(a0, b0, c0, a1, b1, c1);
        if (at < end) chunk(a1, b1, c1, a0, b0, c0);
    }
    // Ticks behind the length are 0.
    if (!STATES && out) {
        const int t0 = max(len, seg_first);
        typedef bf16 many __attribute__((ext_vector_type(8)));
        for (int u = threadIdx.x; u < (seg_end - t0) * (D / 8); u += NT)
            *reinterpret_cast<many *>(out + (t0 + u / (D / 8)) * out_st + static_cast<int64_t>(bh) * D + u % (D / 8) * 8) = many{};
    }
    if (pass.x_out) {
        const int64_t x_b = pass.x_b;
        float *to = pass.x_out + seg * pass.x_seg + bh * pass.x_bh + (wc + r16) * pass.x_c;
#pragma unroll
        for (int i = 0; i < XT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) to[(row(i) + r) * x_b] = x[i][r];
    }
#endif
}

struct JoinArgs {
    float *states;          // [segments][B H][n]: what each segment adds; becomes the state before each
    const float *x;         // [B H][n] before the first, or NULL
    float *x_out;           // after the last, or NULL
    const float *log_decay;
    const int32_t *lengths;
    int32_t T, H, segments, seg_ticks;
    int64_t bh, n;
};

__global__ void __launch_bounds__(kBlock) k_attention_join(JoinArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (i >= a.bh * a.n) return;
    const int bh = static_cast<int>(i / a.n), len = live_ticks(a.lengths, bh / a.H, a.T);
    const Decay decay(a.log_decay[bh % a.H]);
    float x = a.x ? a.x[i] : 0.0f;
    const int64_t apart = a.bh * a.n;
    constexpr int kAhead = 8;   // loads under way
    for (int s0 = 0; s0 < a.segments; s0 += kAhead) {
        float more[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) more[k] = a.states[min(s0 + k, a.segments - 1) * apart + i];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int s = s0 + k, ticks = min(max(len - s * a.seg_ticks, 0), a.seg_ticks);
            if (s >= a.segments) break;
            a.states[s * apart + i] = x;
            if (ticks) x = x * decay.power(ticks) + more[k];
        }
    }
    if (a.x_out) a.x_out[i] = x;
}

// out[row][g][d] = the sum of in[row][g share + i][d] over i, in their order
template <typename T>
__global__ void __launch_bounds__(kBlock) k_attention_share(const float *in, int64_t rows, int groups, int share, int d, T *out) {
    const int64_t n = rows * groups * d;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kBlock) {
        const float *p = in + i / d * share * d + i % d;
        float s = 0.0f;
        for (int k = 0; k < share; ++k) s += p[static_cast<int64_t>(k) * d];
        out[i] = from_f32<T>(s);
    }
}

template <typename T, int D, int NW, bool WHOLE>
void run_pass(const AttArgs &a, bool states, hipStream_t s) {
    const int64_t groups = (static_cast<int64_t>(a.B) * a.H * a.segments + 7) / 8 * 8;
    const dim3 grid(static_cast<unsigned>(groups * a.passes)), block(NW * kWave);
    if (states) hipLaunchKernelGGL((k_attention<T, D, NW, true, WHOLE>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_attention<T, D, NW, false, WHOLE>), grid, block, 0, s, a);
}

// Chunks of 64 ticks are the faster for blocks that are alone on their compute unit, of 32 leave room for others (500 x 32 ticks
// of 8 heads of 128, trials of any length, 256 blocks forward, 43 us and 52, 768 backward, 96 and 85; of 16 heads of 64, 512 and 1536
// blocks, 34 and 36, 74 and 57).
template <int D, int NW>
void run_direct(const AttArgs &a, bool states, hipStream_t s) {
    const int64_t groups = (static_cast<int64_t>(a.B) * a.H * a.segments + 7) / 8 * 8;
    const dim3 grid(static_cast<unsigned>(groups * a.passes)), block(NW * kWave);
    const bool few = groups * a.passes <= (NW == 8 ? 256 : 512);
    if (states) {   // (of 128 channels at most 256 blocks: cut())
        if constexpr (NW == 4)
            if (!few) {
                hipLaunchKernelGGL((k_attention_direct<D, NW, 32, true>), grid, block, 0, s, a);
                return;
            }
        hipLaunchKernelGGL((k_attention_direct<D, NW, 64, true>), grid, block, 0, s, a);
    } else {
        if (few) hipLaunchKernelGGL((k_attention_direct<D, NW, 64, false>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_attention_direct<D, NW, 32, false>), grid, block, 0, s, a);
    }
}

// Whether all of a sequence's heads begin on 16 bytes.
bool on_16(const AttSeq &q) { return reinterpret_cast<uintptr_t>(q.p) % 16 == 0 && (q.st | q.sb | q.sh) % 8 == 0; }

template <typename T>
void run_passes(const AttArgs &a, bool states, hipStream_t s) {
    int da = 0, dc = 0;
    bool whole = true, direct = std::is_same_v<T, bf16>;
    for (int i = 0; i < a.passes; ++i) {
        const AttPass &p = a.pass[i];
        da = std::max(da, p.b.d), dc = std::max(dc, p.c.d);
        whole = whole && p.b.d == p.c.d && p.c.d == a.pass[0].c.d && !p.wide;
        direct = direct && on_16(p.a) && on_16(p.b) && on_16(p.c) && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    }
    if (direct && whole && dc == 64) {
        run_direct<64, 4>(a, states, s);
    } else if (direct && whole && dc == 128) {
        run_direct<128, 8>(a, states, s);
    } else if (whole && dc == 64) {
        run_pass<T, 64, 4, true>(a, states, s);
    } else if (whole && dc == 128) {
        run_pass<T, 128, 8, true>(a, states, s);
    } else if (dc <= 64) {
        if (da <= 32) run_pass<T, 32, 4, false>(a, states, s);
        else if (da <= 64) run_pass<T, 64, 4, false>(a, states, s);
        else run_pass<T, 128, 4, false>(a, states, s);
    } else {
        if (da <= 32) run_pass<T, 32, 8, false>(a, states, s);
        else if (da <= 64) run_pass<T, 64, 8, false>(a, states, s);
        else run_pass<T, 128, 8, false>(a, states, s);
    }
}

template <typename T>
void run_share(const float *in, int64_t rows, int groups, int share, int d, void *out, hipStream_t s) {
    const int64_t n = rows * groups * d;
    if (n == 0) return;
    hipLaunchKernelGGL(k_attention_share<T>, dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(n, kBlock), 16384))), dim3(kBlock), 0, s,
                       in, rows, groups, share, d, static_cast<T *>(out));
}

// One tick, bound by the state's way to the registers and back (32 entries of 8 heads of 64 x 64, 8.4 MB, 4.6 us of which a launch
// is 4): a block takes 32 of v's channels of an entry and head, 8 lanes by 32 lots of k's channels.
struct StepArgs {
    const void *q, *k, *v;
    int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh;
    const float *log_decay;
    float *state;
    void *y;
    int32_t H, share, K, V, tiles;
    float scale;
};

template <typename T>
__global__ void __launch_bounds__(kBlock) k_attention_step(StepArgs a) {
    __shared__ float sums[kBlock / kWave][32];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int tile = blockIdx.x % a.tiles, bh = blockIdx.x / a.tiles, b = bh / a.H, h = bh % a.H;
    const int c = tile * 32 + threadIdx.x % 8 * 4, have = a.V - c;
    const T *q = static_cast<const T *>(a.q) + b * a.q_sb + h * a.q_sh;
    const T *k = static_cast<const T *>(a.k) + b * a.k_sb + h / a.share * a.k_sh;
    const T *v = static_cast<const T *>(a.v) + b * a.v_sb + h / a.share * a.v_sh;
    const float lam = Decay(a.log_decay[h]).power(1);
    float *state = a.state + static_cast<int64_t>(bh) * a.K * a.V + c;
    f32x4 vv = {0.0f, 0.0f, 0.0f, 0.0f}, sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < have) vv[e] = to_f32(v[c + e]);
#pragma unroll 4
    for (int d = threadIdx.x / 8; d < a.K; d += 32) {
        const float kd = to_f32(k[d]), qd = to_f32(q[d]);
        float *p = state + static_cast<int64_t>(d) * a.V;
        if (have >= 4) {
            const f32x4 x = *reinterpret_cast<const Vec<f32, 4> *>(p) * lam + vv * kd;
            *reinterpret_cast<Vec<f32, 4> *>(p) = x;
            sum += x * qd;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < have) {
                    const float x = p[e] * lam + vv[e] * kd;
                    p[e] = x;
                    sum[e] += x * qd;
                }
        }
    }
#pragma unroll
    for (int m = 8; m < kWave; m <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], m, kWave);
    if (lane < 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[wave][lane * 4 + e] = sum[e];
    __syncthreads();
    const int ch = tile * 32 + threadIdx.x;
    if (threadIdx.x >= 32 || ch >= a.V) return;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kBlock / kWave; ++w) s += sums[w][threadIdx.x];
    static_cast<T *>(a.y)[static_cast<int64_t>(bh) * a.V + ch] = from_f32<T>(s * a.scale);
}

template <typename T>
void run_step(const StepArgs &a, int64_t blocks, hipStream_t s) {
    hipLaunchKernelGGL(k_attention_step<T>, dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0, s, a);
}

int check_attention(const glif_attention *a, bool step) {
    if (!a) return fail(GLIF_EINVAL, "NULL argument");
    if (!known_dtype(a->dtype)) return fail(GLIF_EINVAL, "attention: unknown type");
    if (a->n_ticks < 0 || a->n_ticks > (1 << 20) || a->n_batch < 0 || a->n_batch > 65535 || a->n_heads < 0 || a->n_heads > 4096)
        return fail(GLIF_EINVAL, "attention: at most 2^20 ticks, a batch of 65535 and 4096 heads");
    const int64_t most = std::max({a->q_st, a->k_st, a->v_st}), least = std::min({a->q_st, a->k_st, a->v_st});
    if (!step && (most >= (1 << 24) || least < 0)) return fail(GLIF_EINVAL, "attention: strides of ticks must be in [0, 2^24)");
    if (!step && a->n_ticks > 1 && static_cast<int64_t>(a->n_batch) * a->n_heads * std::max(a->d_value, 0) >= (1 << 24))
        return fail(GLIF_EINVAL, "attention: a tick of y must have fewer than 2^24 elements");
    if (a->n_groups < 1 || a->n_heads % a->n_groups) return fail(GLIF_EINVAL, "attention: n_groups must divide n_heads");
    if (a->d_key < 1 || a->d_key > 128 || a->d_value < 1 || a->d_value > 128)
        return fail(GLIF_EINVAL, "attention: keys and values have 1 to 128 channels");
    if (static_cast<int64_t>(a->n_batch) * a->n_heads > (1 << 20))
        return fail(GLIF_EINVAL, "attention: at most 2^20 heads in a batch");
    const bool some = static_cast<int64_t>(a->n_batch) * a->n_heads != 0;
    if (some && (!a->log_decay || ((step || a->n_ticks) && (!a->q || !a->k || !a->v)))) return fail(GLIF_EINVAL, "NULL argument");
    return GLIF_OK;
}

// Ticks in segments where there are too few blocks for the chip: a first launch gives the state that each segment adds,
// a second joins them, and then all segments go at once.  The first reads two of three sequences again and takes more than
// half as long, so that two segments lose (500 x 16 ticks of 8 heads of 128 in two 59 us, in one 43; 8000 x 16 of 24 heads of 64 615 and
// 496), but for thousands of ticks of 128-channel heads (8000 x 12 of 8 438 and 524).  As many segments as blocks are there at once,
// one a compute unit where heads have more than 64 channels, three where not (8000 ticks of 16 heads of 128 in 25 segments, two rounds of
// blocks, 86 us, in 16 75), and none of fewer than four chunks.
void cut(AttArgs &a, int64_t blocks, int ticks, const glif_attention *s) {
    a.segments = 1, a.seg_ticks = std::max((a.T + ticks - 1) / ticks, 1) * ticks;
    const int64_t slots = std::max(s->d_key, s->d_value) > 64 ? 256 : 768;
    const int64_t chunks = (a.T + ticks - 1) / ticks, want = blocks ? std::min<int64_t>(slots / blocks, chunks / 4) : 0;
    if (want < 3) return;
    a.seg_ticks = static_cast<int>((chunks + want - 1) / want) * ticks;
    a.segments = (a.T + a.seg_ticks - 1) / a.seg_ticks;
}

int chunk_ticks(int32_t dtype) { return dtype == GLIF_BF16 ? 64 : 32; }

AttArgs common(const glif_attention *s) {
    AttArgs a{};
    a.log_decay = s->log_decay, a.lengths = s->lengths, a.T = s->n_ticks, a.B = s->n_batch, a.H = s->n_heads;
    return a;
}

AttArgs forward_args(const glif_attention *s) {
    AttArgs a = common(s);
    cut(a, static_cast<int64_t>(a.B) * a.H, chunk_ticks(s->dtype), s);
    return a;
}

AttArgs backward_args(const glif_attention *s) {
    AttArgs a = common(s);
    cut(a, static_cast<int64_t>(a.B) * a.H * 3, chunk_ticks(s->dtype), s);
    return a;
}

size_t state_floats(const AttArgs &a, const glif_attention *s) {
    return a.segments > 1 ? static_cast<size_t>(a.segments) * a.B * a.H * s->d_key * s->d_value : 0;
}

struct AttBack {
    float *forward, *backward;   // states of the segments, each way
    float *dk, *dv;              // of every head, where heads share theirs
};

void carve(Carver &c, AttBack &b, const AttArgs &a, const glif_attention *s) {
    if (const size_t n = state_floats(a, s)) b.forward = c.take<float>(n), b.backward = c.take<float>(n);
    if (s->n_groups < s->n_heads) {
        const size_t rows = static_cast<size_t>(a.T) * a.B * a.H;
        b.dk = c.take<float>(rows * s->d_key), b.dv = c.take<float>(rows * s->d_value);
    }
}

// The states before every segment, [segments][B H][d_key][d_value].
void segment_states(const AttArgs &of, const AttSeq &b, const AttSeq &c, bool back, float in_scale, const float *x, float *x_out, float *states,
                    int32_t dtype, hipStream_t s) {
    AttArgs a = of;
    const int64_t n = static_cast<int64_t>(b.d) * c.d, bh = static_cast<int64_t>(a.B) * a.H;
    AttPass &p = a.pass[0];
    a.passes = 1;
    p = AttPass{};
    p.a = p.b = b, p.c = c, p.back = back, p.lead = back ? 0 : 1, p.in_scale = in_scale;
    p.x_out = states, p.x_seg = bh * n, p.x_bh = n, p.x_b = c.d, p.x_c = 1;
    GLIF_BY_DTYPE(dtype, run_passes, a, true, s);
    const JoinArgs j{states, x, x_out, a.log_decay, a.lengths, a.T, a.H, a.segments, a.seg_ticks, bh, n};
    hipLaunchKernelGGL(k_attention_join, dim3(static_cast<unsigned>(ceil_div(bh * n, kBlock))), dim3(kBlock), 0, s, j);
}

}  // namespace
}  // namespace glif

using namespace glif;

extern "C" {

size_t glif_attention_fwd_workspace(const glif_attention *s) {
    if (check_attention(s, false)) return 0;
    const AttArgs a = forward_args(s);
    Carver c(nullptr, 0);
    if (const size_t n = state_floats(a, s)) c.take<float>(n);
    return c.off;
}

int glif_attention_fwd(const glif_attention *s, void *y, float *last, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_attention(s, false)) return rc;
    AttArgs a = forward_args(s);
    if (static_cast<int64_t>(a.B) * a.H == 0) return GLIF_OK;
    if (a.T && !y) return fail(GLIF_EINVAL, "NULL argument");
    Carver c(ws, ws_bytes);
    const size_t n = state_floats(a, s);
    float *states = n ? c.take<float>(n) : nullptr;
    if (!c.ok() || (n && !ws)) return fail(GLIF_ENOMEM, "attention: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int32_t share = s->n_heads / s->n_groups;
    const AttSeq q{s->q, s->q_st, s->q_sb, s->q_sh, 1, s->d_key}, k{s->k, s->k_st, s->k_sb, s->k_sh, share, s->d_key};
    const AttSeq v{s->v, s->v_st, s->v_sb, s->v_sh, share, s->d_value};
    if (n) segment_states(a, k, v, false, 1.0f, s->state, last, states, s->dtype, st);
    AttPass &p = a.pass[0];
    a.passes = 1;
    p.a = q, p.b = k, p.c = v, p.out = y, p.lead = 1, p.out_scale = s->scale, p.in_scale = 1.0f;
    const int64_t each = static_cast<int64_t>(s->d_key) * s->d_value;
    p.x = n ? states : s->state, p.x_seg = n ? each * a.B * a.H : 0, p.x_bh = each, p.x_b = s->d_value, p.x_c = 1;
    p.x_out = n ? nullptr : last;
    GLIF_BY_DTYPE(s->dtype, run_passes, a, false, st);
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

size_t glif_attention_bwd_workspace(const glif_attention *s) {
    if (check_attention(s, false)) return 0;
    const AttArgs a = backward_args(s);
    Carver c(nullptr, 0);
    AttBack b{};
    carve(c, b, a, s);
    return c.off;
}

int glif_attention_bwd(const glif_attention *s, const glif_attention_grad *g, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_attention(s, false)) return rc;
    if (!g) return fail(GLIF_EINVAL, "NULL argument");
    AttArgs a = backward_args(s);
    if (static_cast<int64_t>(a.B) * a.H == 0) return GLIF_OK;
    if (a.T && !g->dy) return fail(GLIF_EINVAL, "NULL argument");
    if (g->dy_st < 0 || g->dy_st >= (1 << 24)) return fail(GLIF_EINVAL, "attention: strides of ticks must be in [0, 2^24)");
    Carver c(ws, ws_bytes);
    AttBack w{};
    carve(c, w, a, s);
    if (!c.ok() || (c.off && !ws)) return fail(GLIF_ENOMEM, "attention: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int32_t share = s->n_heads / s->n_groups;
    const bool shared = share > 1, cut = a.segments > 1;
    const AttSeq q{s->q, s->q_st, s->q_sb, s->q_sh, 1, s->d_key}, k{s->k, s->k_st, s->k_sb, s->k_sh, share, s->d_key};
    const AttSeq v{s->v, s->v_st, s->v_sb, s->v_sh, share, s->d_value}, dy{g->dy, g->dy_st, g->dy_sb, g->dy_sh, 1, s->d_value};
    const int64_t each = static_cast<int64_t>(s->d_key) * s->d_value, seg = cut ? each * a.B * a.H : 0;
    const bool back = g->dk || g->dv || g->dstate;
    if (cut && g->dq) segment_states(a, k, v, false, 1.0f, s->state, nullptr, w.forward, s->dtype, st);
    if (cut && back) segment_states(a, q, dy, true, s->scale, g->dlast, g->dstate, w.backward, s->dtype, st);
    if (g->dq) {
        AttPass &p = a.pass[a.passes++];
        p.a = dy, p.b = v, p.c = k, p.out = g->dq, p.lead = 1, p.out_scale = s->scale, p.in_scale = 1.0f;
        p.x = cut ? w.forward : s->state, p.x_seg = seg, p.x_bh = each, p.x_b = 1, p.x_c = s->d_value;
    }
    if (g->dk) {
        AttPass &p = a.pass[a.passes++];
        p.a = v, p.b = dy, p.c = q, p.out = shared ? w.dk : g->dk, p.wide = shared, p.back = 1, p.out_scale = 1.0f, p.in_scale = s->scale;
        p.x = cut ? w.backward : g->dlast, p.x_seg = seg, p.x_bh = each, p.x_b = 1, p.x_c = s->d_value;
    }
    if (g->dv || (g->dstate && !cut)) {
        AttPass &p = a.pass[a.passes++];
        p.a = k, p.b = q, p.c = dy, p.out = !g->dv ? nullptr : shared ? w.dv : g->dv, p.wide = shared, p.back = 1, p.out_scale = 1.0f;
        p.in_scale = s->scale;
        p.x = cut ? w.backward : g->dlast, p.x_seg = seg, p.x_bh = each, p.x_b = s->d_value, p.x_c = 1;
        p.x_out = cut ? nullptr : g->dstate;
    }
    if (a.passes) GLIF_BY_DTYPE(s->dtype, run_passes, a, false, st);
    if (shared) {
        const int64_t rows = static_cast<int64_t>(a.T) * a.B;
        if (g->dk) GLIF_BY_DTYPE(s->dtype, run_share, w.dk, rows, s->n_groups, share, s->d_key, g->dk, st);
        if (g->dv) GLIF_BY_DTYPE(s->dtype, run_share, w.dv, rows, s->n_groups, share, s->d_value, g->dv, st);
    }
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

int glif_attention_step(const glif_attention *s, void *y, float *state, void *stream) {
    if (int rc = check_attention(s, true)) return rc;
    const int64_t bh = static_cast<int64_t>(s->n_batch) * s->n_heads;
    if (bh == 0) return GLIF_OK;
    if (!y || !state) return fail(GLIF_EINVAL, "NULL argument");
    const int tiles = (s->d_value + 31) / 32;
    const StepArgs a{s->q, s->k, s->v, s->q_sb, s->q_sh, s->k_sb, s->k_sh, s->v_sb, s->v_sh, s->log_decay, state, y,
                     s->n_heads, s->n_heads / s->n_groups, s->d_key, s->d_value, tiles, s->scale};
    GLIF_BY_DTYPE(s->dtype, run_step, a, bh * tiles, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
