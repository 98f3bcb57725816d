// Layer norm over the last axis, forward and backward.  Per row of D elements:
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  xh = (x - mean) rstd
//   y = xh w + b
//   dx = rstd (dyw - mean(dyw) - xh mean(dyw xh)),  dyw = dy w;   dw = sum_rows dy xh,  db = sum_rows dy
// The backward takes the statistics from x itself, so the forward leaves nothing behind.  All sums are float32 in a
// fixed order; y and dx are rounded once.
//
// Bound by memory: x in and y out, or x and dy in and dx out.  A row is read once, in 16-byte pieces, into the registers of
// the L threads that share it (8 of a wave up to a block of 1024), and its mean, variance and results are taken from there.
// In the backward the same threads keep the columns' sums over the rows they go through, as long as those fit beside the
// row (16000 x 1024 bfloat16 forward 14 us, 4.7 TB/s, backward 37; 16000 x 4096 40 and 124).  Wider rows are gone through
// twice: once for their statistics, once, by columns, for dx and the columns' sums, in turns over parts of the rows that the
// last-level cache still holds.
#include "seq.h"
namespace glif {

namespace {

struct NormArgs {
    const void *x, *dy, *weight, *bias;
    void *y, *dx, *dweight, *dbias;
    int64_t rows, D, x_stride, dy_stride;
    int32_t pdt;
    float eps;
    float4 *stat;      // [rows] mean, rstd, mean(dyw), mean(dyw xh) (backward of wide rows)
    float *part;       // [parts][2][D] sums of dw and db
    int32_t parts;
    int32_t past;      // results go past the caches: they are larger than these
};

// ---- the threads of a row -----------------------------------------------------------------------------------------------
// L threads: a part of a wave, or the whole block.  Sum over them, in all of them.
template <int L>
__device__ __forceinline__ float row_sum(float v, float *red) {
    if constexpr (L <= kWave) {
#pragma unroll
        for (int m = 1; m < L; m <<= 1) v += __shfl_xor(v, m, kWave);
        return v;
    } else {
        constexpr int kW = L / kWave;
        v = wave_sum(v);
        __syncthreads();   // the last sum's readers are done
        if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
        __syncthreads();
        float s = red[threadIdx.x % kW];
#pragma unroll
        for (int m = 1; m < kW; m <<= 1) s += __shfl_xor(s, m, kWave);
        return s;
    }
}
// two at once
template <int L>
__device__ __forceinline__ float2 row_sum2(float a, float b, float *red) {
    if constexpr (L <= kWave) {
        return make_float2(row_sum<L>(a, red), row_sum<L>(b, red));
    } else {
        constexpr int kW = L / kWave;
        a = wave_sum(a), b = wave_sum(b);
        __syncthreads();
        if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = a, red[kW + threadIdx.x / kWave] = b;
        __syncthreads();
        float s = red[threadIdx.x % kW], t = red[kW + threadIdx.x % kW];
#pragma unroll
        for (int m = 1; m < kW; m <<= 1) s += __shfl_xor(s, m, kWave), t += __shfl_xor(t, m, kWave);
        return make_float2(s, t);
    }
}

// 16 bytes of a row from column c on, zeros past its end.  Whole words throughout: a piece put together from its elements would
// live in a register for each of them.  (Here and below a whole piece is one with c <= D - V: c + V passes 31 bits in the last
// piece of the longest rows.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ u32x4 piece(const T *p, int c, int D) {
    constexpr int V = kVecBytes16<T>;
    u32x4 q = {};
    if (c <= D - V) {
        q = __builtin_bit_cast(u32x4, *reinterpret_cast<const Vec<T, V> *>(p + c));
    } else if (c < D) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (c + e >= D) continue;
            if constexpr (sizeof(T) == 4) q[e] = __builtin_bit_cast(uint32_t, p[c + e]);
            else q[e / 2] |= static_cast<uint32_t>(__builtin_bit_cast(uint16_t, p[c + e])) << (e % 2 * 16);
        }
    }
    return q;
}

// A row in the registers of L threads, R pieces of V elements each; piece i of thread t starts at (i L + t) V.
template <typename T, int L, int R>
struct Row {
    static constexpr int V = kVecBytes16<T>, kR = R;
    typedef Vec<T, V> vec;
    u32x4 r[R];
    static __device__ __forceinline__ int at(int i) { return (i * L + static_cast<int>(threadIdx.x) % L) * V; }
    __device__ __forceinline__ void load(int i, const T *p, int D) { r[i] = piece<T>(p, at(i), D); }
    __device__ __forceinline__ void load(const T *p, int D) {
#pragma unroll
        for (int i = 0; i < R; ++i) load(i, p, D);
    }
    __device__ __forceinline__ float get(int i, int e) const { return to_f32(static_cast<T>(__builtin_bit_cast(vec, r[i])[e])); }
    // Between the passes over a long row: its float32 values are made again rather than kept in twice the registers.
    __device__ __forceinline__ void again() {
        if constexpr (R > 2 && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < R; ++i) asm volatile("" : "+v"(r[i]));
        }
    }
    template <bool PAST = false>
    static __device__ __forceinline__ void put(T *p, int c, int D, const float (&v)[V]) {
        if (c <= D - V) {
            vec o;
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = from_f32<T>(v[e]);
            if constexpr (PAST) __builtin_nontemporal_store(o, reinterpret_cast<vec *>(p + c));
            else *reinterpret_cast<vec *>(p + c) = o;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e < D) p[c + e] = from_f32<T>(v[e]);
        }
    }
    __device__ __forceinline__ float2 stats(int D, float eps, float *red) {
        float s = 0.0f;   // pieces past the row are zeros
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) s += get(i, e);
        const float mean = row_sum<L>(s, red) / static_cast<float>(D);
        again();
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = get(i, e) - mean;
                q = at(i) + e < D ? fmaf(d, d, q) : q;
            }
        return make_float2(mean, 1.0f / sqrtf(row_sum<L>(q, red) / static_cast<float>(D) + eps));
    }
};

// V parameters from column c on; `other` past the row and where there are none.
template <int V>
__device__ __forceinline__ void params(float (&v)[V], const void *p, int32_t dt, int c, int D, float other) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = other;
    } else if (dt == GLIF_F32 && c <= D - V) {
        const Vec<float, 4> *q = reinterpret_cast<const Vec<float, 4> *>(static_cast<const float *>(p) + c);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = q[e / 4][e % 4];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = c + e < D ? load_param(p, dt, c + e) : other;
    }
}

// V sums to the columns from c on of a part (more: added to what it holds), in pieces of 16 bytes.
template <int V>
__device__ __forceinline__ void flush(float *part, int c, int D, const float (&v)[V], bool more) {
    typedef Vec<float, 4> f4;
    if (c <= D - V) {
#pragma unroll
        for (int h = 0; h < V; h += 4) {
            f4 o = {v[h], v[h + 1], v[h + 2], v[h + 3]};
            if (more) o += *reinterpret_cast<const f4 *>(part + c + h);
            *reinterpret_cast<f4 *>(part + c + h) = o;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (c + e < D) part[c + e] = more ? part[c + e] + v[e] : v[e];
    }
}

// ---- rows in registers ----------------------------------------------------------------------------------------------------
template <typename T, int L, int R>
__global__ void __launch_bounds__(L > kBlock ? L : kBlock, L > kBlock ? 8 : 1) k_norm_fwd(NormArgs a) {
    constexpr int V = Row<T, L, R>::V, kRows = L > kBlock ? 1 : kBlock / L;
    __shared__ float red[32];
    const int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / L;
    if (r >= a.rows) return;
    const int D = static_cast<int>(a.D);
    Row<T, L, R> x;
    x.load(static_cast<const T *>(a.x) + r * a.x_stride, D);
    const float2 st = x.stats(D, a.eps, red);
    x.again();
    T *y = static_cast<T *>(a.y) + r * a.D;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int c = x.at(i);
        if (c >= D) continue;
        float w[V], b[V], o[V];
        params<V>(w, a.weight, a.pdt, c, D, 1.0f);
        params<V>(b, a.bias, a.pdt, c, D, 0.0f);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf((x.get(i, e) - st.x) * st.y, w[e], b[e]);
        x.put(y, c, D, o);
    }
}

// dx, and the columns' sums over the block's rows.
template <typename T, int L, int R>
__global__ void __launch_bounds__(kBlock) k_norm_bwd(NormArgs a) {
    constexpr int V = Row<T, L, R>::V, kRows = kBlock / L;
    __shared__ float red[2 * kBlock / kWave];
    float dw[R][V] = {}, db[R][V] = {};
    const int D = static_cast<int>(a.D);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / L;
    constexpr bool kNext = R <= 2;   // the next row is on its way while this one is worked on
    Row<T, L, R> next_x, next_dy;
    if (kNext && first < a.rows) {
        next_x.load(static_cast<const T *>(a.x) + first * a.x_stride, D);
        next_dy.load(static_cast<const T *>(a.dy) + first * a.dy_stride, D);
    }
    for (int64_t r = first; r < a.rows; r += step) {
        // the weights are read again for every row: kept, they would take the registers that other waves live in
        const void *weight = a.weight;
        asm volatile("" : "+s"(weight));
        Row<T, L, R> x, dy;
        if constexpr (kNext) {
            x = next_x, dy = next_dy;
            if (r + step < a.rows) {
                next_x.load(static_cast<const T *>(a.x) + (r + step) * a.x_stride, D);
                next_dy.load(static_cast<const T *>(a.dy) + (r + step) * a.dy_stride, D);
            }
        } else {
            x.load(static_cast<const T *>(a.x) + r * a.x_stride, D);
            dy.load(static_cast<const T *>(a.dy) + r * a.dy_stride, D);
        }
        const float2 st = x.stats(D, a.eps, red);
        x.again();
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = x.at(i);
            if (c >= D) continue;
            float w[V];
                params<V>(w, weight, a.pdt, c, D, 1.0f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float g = dy.get(i, e), xh = (x.get(i, e) - st.x) * st.y;   // past the row g is 0
                s1 = fmaf(g, w[e], s1);
                s2 = fmaf(g * w[e], xh, s2);
                dw[i][e] = fmaf(g, xh, dw[i][e]), db[i][e] += g;
            }
        }
        const float2 s = row_sum2<L>(s1, s2, red);
        const float m1 = s.x / static_cast<float>(D), m2 = s.y / static_cast<float>(D);
        if (!a.dx) continue;
        T *dx = static_cast<T *>(a.dx) + r * a.D;
        asm volatile("" : "+s"(weight));
        x.again(), dy.again();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = x.at(i);
            if (c >= D) continue;
            float w[V], o[V];
                params<V>(w, weight, a.pdt, c, D, 1.0f);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = st.y * (dy.get(i, e) * w[e] - m1 - (x.get(i, e) - st.x) * st.y * m2);
            x.put(dx, c, D, o);
        }
    }
    if (!a.part) return;
    float *part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.D;
    if constexpr (L >= kBlock) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            flush(part, Row<T, L, R>::at(i), D, dw[i], false), flush(part + a.D, Row<T, L, R>::at(i), D, db[i], false);
    } else {
        // the block's rows side by side: their threads' sums one piece after the other through LDS
        constexpr int kCols = L * V;
        __shared__ float sum[2][kBlock / L][kCols];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sum[0][threadIdx.x / L][(threadIdx.x % L) * V + e] = dw[i][e];
                sum[1][threadIdx.x / L][(threadIdx.x % L) * V + e] = db[i][e];
            }
            __syncthreads();
            for (int q = threadIdx.x; q < 2 * kCols; q += kBlock) {
                const int k = q / kCols, c = q % kCols;
                float v = 0.0f;
#pragma unroll
                for (int row = 0; row < kBlock / L; ++row) v += sum[k][row][c];
                if (i * kCols + c < a.D) part[k * a.D + i * kCols + c] = v;
            }
        }
    }
}

// ---- wide rows --------------------------------------------------------------------------------------------------------------
// A block's threads go through a row in pieces and through it again for the results; a compute unit holds several such
// rows, and the second time comes from cache.
constexpr int kWide = 512, kLong = 1024, kLongR = 9, kLongFrom = 6144;

// Count, mean and sum of squared differences from it, of the elements seen.  A thread takes them from its own first element
// on, so that a mean far from zero costs no digits, and piece by piece about each piece's own mean, so that a first element far
// from the others costs none either (one sum of squares about it lost 4e-4 of the variance where it was the row's only one).
struct Moments {
    float n, mean, m2;
    template <int V>
    __device__ __forceinline__ void add(const float (&d)[V], int have) {   // d: 0 from `have` on
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) s += d[e];
        const float h = static_cast<float>(have), its = s / h;
#pragma unroll
        for (int e = 0; e < V; ++e) q = e < have ? fmaf(d[e] - its, d[e] - its, q) : q;
        const float before = n, far = its - mean;
        n += h;
        const float share = h * __builtin_amdgcn_rcpf(n);
        m2 += fmaf(far * far, before * share, q);
        mean = fmaf(far, share, mean);
    }
};
__device__ __forceinline__ Moments both(Moments a, Moments b) {
    const float n = a.n + b.n, d = b.mean - a.mean, share = n > 0.0f ? b.n / n : 0.0f;
    return {n, fmaf(d, share, a.mean), a.m2 + b.m2 + d * d * a.n * share};
}
template <int L>
__device__ __forceinline__ Moments all_moments(Moments v, Moments *red) {
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) v = both(v, {__shfl_xor(v.n, m, kWave), __shfl_xor(v.mean, m, kWave), __shfl_xor(v.m2, m, kWave)});
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < L / kWave; ++w) v = both(v, red[w]);   // in order, the same in all threads
    return v;
}

// f(column, count, values...) for every piece of this thread
template <typename T, typename F>
__device__ __forceinline__ void pieces(const T *p, int D, F f) {
    constexpr int V = kVecBytes16<T>;
    typedef Vec<T, V> vec;
    const int whole = D / V;
#pragma unroll 4
    for (int i = threadIdx.x; i < whole; i += kWide) f(i * V, V, *reinterpret_cast<const vec *>(p + i * V));
    if (D % V && static_cast<int>(threadIdx.x) == whole % kWide) {
        vec v = {};
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (whole * V + e < D) v[e] = p[whole * V + e];
        f(whole * V, D - whole * V, v);
    }
}
template <typename T, typename F>
__device__ __forceinline__ void pieces2(const T *p, const T *q, int D, F f) {
    constexpr int V = kVecBytes16<T>;
    typedef Vec<T, V> vec;
    const int whole = D / V;
#pragma unroll 2
    for (int i = threadIdx.x; i < whole; i += kWide)
        f(i * V, V, *reinterpret_cast<const vec *>(p + i * V), *reinterpret_cast<const vec *>(q + i * V));
    if (D % V && static_cast<int>(threadIdx.x) == whole % kWide) {
        vec v = {}, w = {};
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (whole * V + e < D) v[e] = p[whole * V + e], w[e] = q[whole * V + e];
        f(whole * V, D - whole * V, v, w);
    }
}

template <typename T, bool PAST>
__global__ void __launch_bounds__(kWide) k_norm_fwd_wide(NormArgs a) {
    constexpr int V = kVecBytes16<T>;
    typedef Vec<T, V> vec;
    __shared__ Moments red[kWide / kWave];
    const int64_t r = blockIdx.x;
    const int D = static_cast<int>(a.D), first = threadIdx.x * V;
    const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
    const float k = first < D ? to_f32(x[first]) : 0.0f;
    Moments own{};
    pieces(x, D, [&](int, int have, vec v) {
        float d[V];
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] = e < have ? to_f32(static_cast<T>(v[e])) - k : 0.0f;
        own.add<V>(d, have);
    });
    const Moments m = all_moments<kWide>({own.n, k + own.mean, own.m2}, red);
    const float rstd = 1.0f / sqrtf(m.m2 / static_cast<float>(D) + a.eps);
    T *y = static_cast<T *>(a.y) + r * a.D;
    pieces(x, D, [&](int c, int have, vec v) {
        float w[V], b[V], o[V];
        params<V>(w, a.weight, a.pdt, c, D, 1.0f);
        params<V>(b, a.bias, a.pdt, c, D, 0.0f);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf((to_f32(static_cast<T>(v[e])) - m.mean) * rstd, w[e], b[e]);
        Row<T, 1, 1>::template put<PAST>(y, c, D, o);
    });
}

// Rows of more than kLongFrom pieces in the registers of one block, which has a compute unit to itself (2500 x 66000 bfloat16
// 172 to 176 us, 3.8 TB/s; gone through twice 201.  2500 x 50000 116 and 112, 2500 x 40000 95 and 87: there several rows a unit
// come from the L2 again).  Longer ones, as 230,000 columns or 66,000 in float32, are gone through twice (500 x 230000 107 us, 1000
// x 66000 float32 141: 4.3 and 3.7 TB/s).
template <typename T>
__global__ void __launch_bounds__(kLong, 4) k_norm_fwd_long(NormArgs a) {
    typedef Row<T, kLong, kLongR> row;
    constexpr int V = row::V;
    __shared__ float red[kLong / kWave];
    const int D = static_cast<int>(a.D);
    const int64_t r = blockIdx.x;
    row x;
    x.load(static_cast<const T *>(a.x) + r * a.x_stride, D);
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int i = 0; i < kLongR; ++i) {   // the barriers: values are made from the row again rather than kept beside it
#pragma unroll
        for (int e = 0; e < V; ++e) s += x.get(i, e);
        asm volatile("" : "+v"(x.r[i]), "+v"(s));
    }
    const float mean = row_sum<kLong>(s, red) / static_cast<float>(D);
#pragma unroll
    for (int i = 0; i < kLongR; ++i) {
        const int left = D - row::at(i);
        if (left >= V) {
#pragma unroll
            for (int e = 0; e < V; ++e) q = fmaf(x.get(i, e) - mean, x.get(i, e) - mean, q);
        } else if (left > 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) q = e < left ? fmaf(x.get(i, e) - mean, x.get(i, e) - mean, q) : q;
        }
        asm volatile("" : "+v"(x.r[i]), "+v"(q));
    }
    const float rstd = 1.0f / sqrtf(row_sum<kLong>(q, red) / static_cast<float>(D) + a.eps);
    T *y = static_cast<T *>(a.y) + r * a.D;
#pragma unroll
    for (int i = 0; i < kLongR; ++i) {
        const int c = row::at(i);
        asm volatile("" : "+v"(x.r[i]));
        if (c < D) {
            float w[V], b[V], o[V];
            params<V>(w, a.weight, a.pdt, c, D, 1.0f);
            params<V>(b, a.bias, a.pdt, c, D, 0.0f);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf((x.get(i, e) - mean) * rstd, w[e], b[e]);
            row::template put<true>(y, c, D, o);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Per row mean, rstd, mean(dyw), mean(dyw xh).
template <typename T>
__device__ __forceinline__ void wide_stats(const NormArgs &a, int64_t r) {
    constexpr int V = kVecBytes16<T>;
    typedef Vec<T, V> vec;
    __shared__ Moments red[kWide / kWave];
    __shared__ float red2[2 * kWide / kWave];
    const int D = static_cast<int>(a.D), first = threadIdx.x * V;
    const T *x = static_cast<const T *>(a.x) + r * a.x_stride, *dy = static_cast<const T *>(a.dy) + r * a.dy_stride;
    const float k = first < D ? to_f32(x[first]) : 0.0f;
    Moments own{};
    float g1 = 0.0f, g2 = 0.0f;
    pieces2(x, dy, D, [&](int c, int have, vec v, vec g) {
        float w[V], d[V], p1 = 0.0f, p2 = 0.0f;   // a piece's sums first: single terms would be lost beside a long row's
        params<V>(w, a.weight, a.pdt, c, D, 1.0f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            d[e] = e < have ? to_f32(static_cast<T>(v[e])) - k : 0.0f;
            const float gw = to_f32(static_cast<T>(g[e])) * w[e];
            p1 += gw;
            p2 = fmaf(gw, d[e], p2);
        }
        g1 += p1, g2 += p2;
        own.add<V>(d, have);
    });
    const Moments m = all_moments<kWide>({own.n, k + own.mean, own.m2}, red);
    const float rstd = 1.0f / sqrtf(m.m2 / static_cast<float>(D) + a.eps);
    const float2 g = row_sum2<kWide>(g1, rstd * fmaf(k - m.mean, g1, g2), red2);
    if (threadIdx.x == 0) a.stat[r] = make_float4(m.mean, rstd, g.x / static_cast<float>(D), g.y / static_cast<float>(D));
}

// dx of rows r0 .. r1 - 1 and the columns' sums over them, to a part (more: added to what it holds): a thread per 16 bytes of columns.
template <typename T, bool PAST>
__device__ __forceinline__ void wide_columns(const NormArgs &a, int block, int64_t r0, int64_t r1, int to, bool more) {
    constexpr int V = kVecBytes16<T>;
    typedef Vec<T, V> vec;
    const int D = static_cast<int>(a.D);
    const int64_t c64 = (static_cast<int64_t>(block) * kWide + threadIdx.x) * V;
    if (c64 >= D) return;
    const int c = static_cast<int>(c64);
    float dw[V] = {}, db[V] = {}, w[V];
    params<V>(w, a.weight, a.pdt, c, D, 1.0f);
    const T *x = static_cast<const T *>(a.x) + c, *dy = static_cast<const T *>(a.dy) + c;
    T *dx = static_cast<T *>(a.dx);
    auto add = [&](vec xv, vec gv, int64_t r) {
        const float4 st = a.stat[r];
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float g = to_f32(static_cast<T>(gv[e])), xh = (to_f32(static_cast<T>(xv[e])) - st.x) * st.y;
            dw[e] = fmaf(g, xh, dw[e]);
            db[e] += g;
            o[e] = st.y * (g * w[e] - st.z - xh * st.w);
        }
        if (dx) Row<T, 1, 1>::template put<PAST>(dx + r * a.D, c, D, o);
    };
    if (c <= D - V) {
#pragma unroll 2
        for (int64_t r = r0; r < r1; ++r)
            add(*reinterpret_cast<const vec *>(x + r * a.x_stride), *reinterpret_cast<const vec *>(dy + r * a.dy_stride), r);
    } else {
        for (int64_t r = r0; r < r1; ++r) {
            vec xv = {}, gv = {};
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e < D) xv[e] = x[r * a.x_stride + e], gv[e] = dy[r * a.dy_stride + e];
            add(xv, gv, r);
        }
    }
    if (!a.part) return;
    float *part = a.part + static_cast<int64_t>(to) * 2 * a.D;
    flush(part, c, D, dw, more), flush(part + a.D, c, D, db, more);
}

// One launch of a wide backward, at three blocks a compute unit: the columns of the rows [col0, col1), whose statistics the launch before took, and the
// statistics of the next rows [row0, row1) beside them.
struct Round {
    int64_t col0, col1, row0, row1;
    int32_t cols, parts;   // column blocks and parts
};
template <typename T, bool PAST>
__global__ void __launch_bounds__(kWide, 6) k_norm_round(NormArgs a, Round k) {
    const int64_t rows = k.row1 - k.row0;
    if (blockIdx.x < rows) {
        wide_stats<T>(a, k.row0 + blockIdx.x);
    } else {
        const int b = static_cast<int>(blockIdx.x - rows), part = b / k.cols;
        const int64_t n = k.col1 - k.col0;
        wide_columns<T, PAST>(a, b % k.cols, k.col0 + n * part / k.parts, k.col0 + n * (part + 1) / k.parts, part, k.col0 > 0);
    }
}

// The parts' sums, from column c0 on: 32 columns by 8 threads each, which take the parts in turn.
__global__ void __launch_bounds__(kBlock) k_norm_join(NormArgs a, int64_t c0) {
    __shared__ float sum[2][8][32];
    const int col = threadIdx.x % 32, lot = threadIdx.x / 32;
    const int64_t c = c0 + static_cast<int64_t>(blockIdx.x) * 32 + col;
    float dw = 0.0f, db = 0.0f;
    if (c < a.D) {
#pragma unroll 4
        for (int p = lot; p < a.parts; p += 8) {
            dw += a.part[static_cast<int64_t>(p) * 2 * a.D + c];
            db += a.part[(static_cast<int64_t>(p) * 2 + 1) * a.D + c];
        }
    }
    sum[0][lot][col] = dw, sum[1][lot][col] = db;
    __syncthreads();
    if (lot > 1 || c >= a.D) return;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += sum[lot][i][col];
    if (lot == 0 && a.dweight) store_param(a.dweight, a.pdt, c, v);
    if (lot == 1 && a.dbias) store_param(a.dbias, a.pdt, c, v);
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
constexpr int64_t kFused = 16384;   // bytes of the widest row whose columns' sums are kept beside it

// Blocks of a fused backward, and parts of its sums: at least four rows for every thread group, as each part costs its way
// to memory and back (16000 x 1024 bfloat16 in 256, 512, 1024 and 2048 parts 50, 37, 40 and 53 us).
int fused_blocks(int64_t rows, int64_t D, int64_t size) {
    const int64_t bytes = D * size, per = bytes <= 4096 ? kBlock / std::max<int64_t>(8, std::min<int64_t>(64, (bytes + 15) / 16)) : 1;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((rows + 4 * per - 1) / (4 * per), 512)));
}

// A wide backward's rounds of rows: 128 MB of x and dy (96, 128 and 160 MB: 2500 x 66000 bfloat16 386, 380 and 383 us, 1000 x
// 66000 float32 269, 264 and 307, 2500 x 40000 bfloat16 225, 223 and 233, 500 x 230000, of 5, 4 and 3 rounds, 344, 307 and 272),
// and parts of a round: two blocks a compute unit (2500 x 66000: 272, 408, 544 and 816 blocks 455, 404, 398 and 398 us in rounds of
// 96 MB), whose sums go on from round to round.
int64_t round_rows(int64_t rows, int64_t D, int64_t size) {
    return std::max<int64_t>(1, std::min<int64_t>(rows, (int64_t(64) << 20) / (D * size)));
}
int round_parts(int64_t n, int64_t D, int64_t size) {
    const int64_t cols = ((D * size + 15) / 16 + kWide - 1) / kWide;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(n, 544 / cols)));
}

// (two layers after each other on 1000 x 66000 bfloat16 156 us, 167 without; on 500 x 66000 70 and 69)
bool past_caches(const NormArgs &a, int32_t dtype) { return a.rows * a.D * static_cast<int64_t>(dtype_size(dtype)) > kPastCaches; }

void carve(Carver &c, NormArgs &a, int64_t size, bool param) {
    if (a.D * size <= kFused) {
        a.parts = fused_blocks(a.rows, a.D, size);
    } else {
        const int64_t n = round_rows(a.rows, a.D, size);
        a.parts = round_parts(n, a.D, size);
        a.stat = c.take<float4>(static_cast<size_t>(a.rows));
    }
    if (param) a.part = c.take<float>(static_cast<size_t>(a.parts) * 2 * a.D);
}

template <typename T, int L, int R>
void fwd(NormArgs a, hipStream_t s) {
    constexpr int kThreads = L > kBlock ? L : kBlock, kRows = kThreads / L;
    constexpr int64_t kMost = blocks_at_once(kThreads) * kRows;
    const int64_t rows = a.rows;
    for (int64_t r = 0; r < rows; r += kMost) {
        a.rows = std::min(kMost, rows - r);
        hipLaunchKernelGGL((k_norm_fwd<T, L, R>), dim3(static_cast<unsigned>((a.rows + kRows - 1) / kRows)), dim3(kThreads), 0, s, a);
        a.x = static_cast<const T *>(a.x) + kMost * a.x_stride, a.y = static_cast<T *>(a.y) + kMost * a.D;
    }
}

// The threads of a row: as few as hold it in one piece each, up to a wave with four, a block with four, 1024 with four.
template <typename T>
void run_fwd(const NormArgs &a, hipStream_t s) {
    const int64_t p = (a.D + kVecBytes16<T> - 1) / kVecBytes16<T>;   // pieces
    if (p <= 8) fwd<T, 8, 1>(a, s);
    else if (p <= 16) fwd<T, 16, 1>(a, s);
    else if (p <= 32) fwd<T, 32, 1>(a, s);
    else if (p <= 64) fwd<T, 64, 1>(a, s);
    else if (p <= 128) fwd<T, 64, 2>(a, s);
    else if (p <= 256) fwd<T, 64, 4>(a, s);
    else if (p <= 512) fwd<T, 256, 2>(a, s);
    else if (p <= 1024) fwd<T, 256, 4>(a, s);
    else if (p <= 4096) fwd<T, 1024, 4>(a, s);
    else if (p > kLongFrom && p <= kLong * kLongR && a.past)
        hipLaunchKernelGGL(k_norm_fwd_long<T>, dim3(static_cast<unsigned>(a.rows)), dim3(kLong), 0, s, a);
    else if (a.past) hipLaunchKernelGGL((k_norm_fwd_wide<T, true>), dim3(static_cast<unsigned>(a.rows)), dim3(kWide), 0, s, a);
    else hipLaunchKernelGGL((k_norm_fwd_wide<T, false>), dim3(static_cast<unsigned>(a.rows)), dim3(kWide), 0, s, a);
}

template <typename T, int L, int R>
void bwd(const NormArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((k_norm_bwd<T, L, R>), dim3(static_cast<unsigned>(a.parts)), dim3(kBlock), 0, s, a);
}

template <typename T>
void run_bwd(const NormArgs &a, hipStream_t s) {
    const int64_t p = (a.D + kVecBytes16<T> - 1) / kVecBytes16<T>, size = sizeof(T);
    if (a.parts == 0) {   // no rows: the join gives the empty sums
    } else if (a.D * size <= kFused) {
        if (p <= 8) bwd<T, 8, 1>(a, s);
        else if (p <= 16) bwd<T, 16, 1>(a, s);
        else if (p <= 32) bwd<T, 32, 1>(a, s);
        else if (p <= 64) bwd<T, 64, 1>(a, s);
        else if (p <= 128) bwd<T, 64, 2>(a, s);
        else if (p <= 256) bwd<T, 64, 4>(a, s);
        else if (p <= 512) bwd<T, 256, 2>(a, s);
        else bwd<T, 256, 4>(a, s);
    } else {
        const int64_t n = round_rows(a.rows, a.D, size);
        Round k{};
        k.cols = static_cast<int32_t>((p + kWide - 1) / kWide), k.parts = round_parts(n, a.D, size);
        while (k.col1 < a.rows) {
            k.col0 = k.col1, k.col1 = k.row1;
            k.row0 = k.row1, k.row1 = std::min(a.rows, k.row0 + n);
            const int64_t blocks = k.row1 - k.row0 + (k.col1 > k.col0 ? static_cast<int64_t>(k.cols) * k.parts : 0);
            if (a.past) hipLaunchKernelGGL((k_norm_round<T, true>), dim3(static_cast<unsigned>(blocks)), dim3(kWide), 0, s, a, k);
            else hipLaunchKernelGGL((k_norm_round<T, false>), dim3(static_cast<unsigned>(blocks)), dim3(kWide), 0, s, a, k);
        }
    }
    constexpr int64_t kMost = blocks_at_once(kBlock) * 32;
    for (int64_t c = 0; a.part && c < a.D; c += kMost)
        hipLaunchKernelGGL(k_norm_join, dim3(static_cast<unsigned>((std::min(kMost, a.D - c) + 31) / 32)), dim3(kBlock), 0, s, a, c);
}

int check_norm(int64_t rows, int64_t D, int32_t dtype, int32_t pdt, float eps) {
    if (rows < 0 || D < 1 || D >= (int64_t(1) << 31) || rows >= (int64_t(1) << 31))
        return fail(GLIF_EINVAL, "layer norm: rows in [0, 2^31) and D in [1, 2^31)");
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
    a.past = past_caches(a, dtype);
    GLIF_BY_DTYPE(dtype, run_fwd, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

size_t glif_layer_norm_bwd_workspace(int64_t rows, int64_t D, int32_t dtype, int32_t want_params) {
    if (check_norm(rows, D, dtype, dtype, 0.0f)) return 0;
    NormArgs a{};
    a.rows = rows, a.D = D;
    Carver c(nullptr, 0);
    carve(c, a, static_cast<int64_t>(dtype_size(dtype)), want_params != 0);
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
    a.past = past_caches(a, dtype);
    Carver c(ws, ws_bytes);
    carve(c, a, static_cast<int64_t>(dtype_size(dtype)), dweight || dbias);
    if (!c.ok() || (c.off && !ws)) return fail(GLIF_ENOMEM, "layer norm: workspace too small");
    if (rows == 0) a.parts = 0;
    GLIF_BY_DTYPE(dtype, run_bwd, a, static_cast<hipStream_t>(stream));
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
