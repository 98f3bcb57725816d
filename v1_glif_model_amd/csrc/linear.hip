// Linear map with bias, activation and residual in its epilogue, and its backward:
//   pre = x W^T + bias,  y = act(pre) + residual
//   dp = dy act'(pre),  dx = dp W,  dW = dp^T x,  db = sum of dp's rows
// All three products run on the matrix cores with float32 accumulators (16-bit types 16x16x32, float32 16x16x4).
//
// Large products are bound by the matrix cores and what feeds them from LDS (8192^3 bfloat16 802 to 837 us, 1314 to 1370 TFLOP/s
// of 2500); short ones and ones of few tiles by the fill and drain of their blocks and by the way of their operands from memory
// (2500 x 66000 x 512 bfloat16, each in a loop of its own: forward 222 us, dx 259, dW 178; after each other in a training step
// 227, 303 and 202); single ticks by the stream of the weights.
#include "seq.h"

namespace glif {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// C[m][n] = sum_k P(m, k) Q(n, k): P(m, k) is p[m * p_ld + k], or p[k * p_ld + m] where its columns are contiguous;
// likewise Q.
struct GemmArgs {
    const void *p, *q;
    int64_t p_ld, q_ld;        // the stride that is not 1
    int64_t M, N, K;
    // what can be read of an operand whose rows run along k (k_cols >= K) and of one of columns (p_rows >= M, q_rows >= N):
    // more than there is where it is padded (with zeros)
    int64_t k_cols, p_rows, q_rows;
    int64_t k_part;            // k's of a split
    int32_t tiles_m, tiles_n, splits;
    float *part;               // [splits][M][part_ld], where splits > 1
    int64_t part_ld;
    void *c;                   // rows of ldc
    // Likewise, or NULL.  In float32 for every type: a rounding of it would go into every gradient, and float16 does not hold all
    // arguments (16000 x 1024 x 4096 bfloat16 with gelu and gradients 628 us; kept in 16 bits 606).
    float *pre;
    int64_t ldc;
    const void *bias, *residual;
    int64_t ldr;
    int32_t bias_dt, act;
    int32_t past;              // results go past the caches, which keep the operands
};

__device__ __forceinline__ float act_of(float p, int act) {
    switch (act) {
        case GLIF_ACT_RELU: return p < 0.0f ? 0.0f : p;   // NaN stays
        case GLIF_ACT_GELU: return 0.5f * p * (1.0f + erff(p * 0.70710678118654752f));
        case GLIF_ACT_SILU: return p * sigmoid_f(p);
        default: return p;
    }
}

__device__ __forceinline__ float slope_of(float p, int act) {
    switch (act) {
        case GLIF_ACT_RELU: return p <= 0.0f ? 0.0f : 1.0f;
        case GLIF_ACT_GELU:
            return fmaf(p * 0.39894228040143268f, expf(-0.5f * p * p), 0.5f * (1.0f + erff(p * 0.70710678118654752f)));
        case GLIF_ACT_SILU: {
            const float q = sigmoid_f(p);
            return q * fmaf(p, 1.0f - q, 1.0f);
        }
        default: return 1.0f;
    }
}

// One matrix instruction's operands from a row-major LDS row of 32 k's: 16-bit types take 8 consecutive k's a lane.
template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    typedef bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<f16> {
    typedef f16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
// float32: lane l holds four consecutive k's, element i of every lane makes one 16x16x4 product (the order of the k's in
// a sum is free, as long as both operands have it)
template <>
struct Mma<f32> {
    typedef f32 frag __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// ---- tiles in LDS -----------------------------------------------------------------------------------------------------
// An operand's tile is ROWS rows (of m or n) of 128 bytes of k: 64 16-bit values or 32 float32.  LDS gives 256 bytes a clock:
// 16 lanes of 16-byte reads, and those are not neighbours but of two fragments' quarters (measured: permuted by the row mod
// 8, half of the clocks of the reads went to bank conflicts).  So the eight 16-byte chunks of a row are permuted by row / 2
// mod 8, which tells all even and all odd rows of a fragment apart for any chunk.
constexpr int kRowBytes = 128;

__device__ __forceinline__ int lds_at(int row, int chunk) { return row * kRowBytes + (((chunk ^ (row >> 1)) & 7) << 4); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Brings ROWS x 128 bytes of an operand whose rows run along k from memory into LDS by way of registers, NT threads.  Rows
// past the operand's end repeat the last (their products are not written); k's past the part's end are 0.
template <typename T, int ROWS, int NT>
struct Stage {
    static constexpr int kV = 16 / static_cast<int>(sizeof(T));   // values of a chunk
    static constexpr int kBK = 8 * kV;                            // k's of a tile
    static constexpr int kN = ROWS * 8 / NT;                      // chunks a thread takes
    static_assert(ROWS * 8 % NT == 0, "the tile does not divide among the threads");
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    vec r[kN];
    const T *at[kN];

    __device__ __forceinline__ void init(const T *p, int64_t ld, int64_t row0, int64_t rows, int64_t k0) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int u = threadIdx.x + i * NT;
            at[i] = p + min(row0 + (u >> 3), rows - 1) * ld + k0 + (u & 7) * kV;
        }
    }
    // left: the k's from the tile's first one on
    __device__ __forceinline__ void load(int64_t left) {
        if (left >= kBK) {
#pragma unroll
            for (int i = 0; i < kN; ++i) r[i] = *reinterpret_cast<const vec *>(at[i]);
        } else {
            const int have = static_cast<int>(left) - (threadIdx.x & 7) * kV;
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int e = 0; e < kV; ++e) r[i][e] = e < have ? at[i][e] : T(0.0f);
        }
#pragma unroll
        for (int i = 0; i < kN; ++i) at[i] += kBK;
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int u = threadIdx.x + i * NT;
            *reinterpret_cast<u32x4 *>(lds + lds_at(u >> 3, u & 7)) = __builtin_bit_cast(u32x4, r[i]);
        }
    }
};

// Four neighbouring results: bias, activation, residual, and one rounding.  The parts that come from memory are read ahead.
template <typename T>
struct Finish {
    typedef Vec<T, 4> vec;
    f32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
    int64_t n;
    int have;
    __device__ __forceinline__ Finish(const GemmArgs &a, int64_t col) : n(col), have(static_cast<int>(min(static_cast<int64_t>(4), a.N - col))) {
        if (a.bias)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < have) bias[e] = load_param(a.bias, a.bias_dt, n + e);
    }
    __device__ __forceinline__ vec residual(const GemmArgs &a, int64_t m) const {
        vec q = {};
        if (!a.residual) return q;
        const T *p = static_cast<const T *>(a.residual) + m * a.ldr + n;
        if (have == 4) return *reinterpret_cast<const vec *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < have) q[e] = p[e];
        return q;
    }
    template <typename O>
    static __device__ __forceinline__ void write(O *p, f32x4 v, int have, int32_t past) {
        typedef Vec<O, 4> out;
        if (have == 4) {
            const out o = __builtin_convertvector(v, out);
            if (past) {   // kept apart from the other store, or they become one again
                asm volatile("" ::: "memory");
                __builtin_nontemporal_store(o, reinterpret_cast<out *>(p));
                asm volatile("" ::: "memory");
            } else {
                *reinterpret_cast<out *>(p) = o;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < have) p[e] = from_f32<O>(v[e]);
        }
    }
    __device__ __forceinline__ void operator()(const GemmArgs &a, int64_t m, f32x4 v, vec res) const {
        v += bias;
        if (a.pre) write(a.pre + m * a.ldc + n, v, have, a.past);
        if (a.act != GLIF_ACT_NONE) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = act_of(v[e], a.act);
        }
        if (a.residual) v += __builtin_convertvector(res, f32x4);
        write(static_cast<T *>(a.c) + m * a.ldc + n, v, have, a.past);
    }
};

// A wave's TM x TN results by way of a slab of its own in LDS: rows come out whole, and the epilogue stands once.  Quad q of
// row r lies at q ^ r mod the row's quads.
template <typename T, int TM, int TN, int SLAB>
__device__ __forceinline__ void put(const GemmArgs &a, f32x4 (&acc)[TM / 16][TN / 16], char *lds, int64_t m0, int64_t n0, int split) {
    constexpr int kQuads = TN / 4, kRows = SLAB / (TN * 4) < TM ? SLAB / (TN * 4) : TM;
    constexpr int kStep = kWave / kQuads, kAhead = 4;
    static_assert(kRows % 16 == 0 && TM % kRows == 0 && kWave % kQuads == 0 && kRows % (kStep * kAhead) == 0, "slab");
    const int lane = threadIdx.x % kWave, r16 = lane % 16, kq = lane / 16, q = lane % kQuads;
    const int64_t n = n0 + q * 4;
    const Finish<T> finish(a, n);
    f32x4 *slab = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int h = 0; h < TM / kRows; ++h) {
#pragma unroll
        for (int i = 0; i < kRows / 16; ++i)
#pragma unroll
            for (int j = 0; j < TN / 16; ++j) {
                const int r = 16 * i + r16, q = 4 * j + kq;
                slab[r * kQuads + (q ^ (r & (kQuads - 1)))] = acc[h * (kRows / 16) + i][j];
            }
        if (n >= a.N) continue;
        const int left = static_cast<int>(min(a.M - m0 - h * kRows, static_cast<int64_t>(kRows)));
#pragma unroll 1
        for (int r = lane / kQuads; r < kRows; r += kStep * kAhead) {
            f32x4 v[kAhead];
            typename Finish<T>::vec res[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int at = r + u * kStep;
                v[u] = slab[at * kQuads + (q ^ (at & (kQuads - 1)))];
                if (a.residual && a.splits == 1 && at < left) res[u] = finish.residual(a, m0 + h * kRows + at);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int at = r + u * kStep;
                const int64_t m = m0 + h * kRows + at;
                if (at >= left) continue;
                if (a.splits > 1) *reinterpret_cast<f32x4 *>(a.part + (split * a.M + m) * a.part_ld + n) = v[u];
                else finish(a, m, v[u], res[u]);
            }
        }
    }
}

// The block's tile.  Neighbouring tiles share an operand: the XCDs (block id mod 8) take consecutive runs of them, along the
// shorter side.
__device__ __forceinline__ void my_tile(const GemmArgs &a, int &tm, int &tn, int &split) {
    int id = blockIdx.x;
    const int blocks = gridDim.x, x = id & 7, per = blocks >> 3, more = blocks & 7;
    if (blocks >= 8) id = x * per + min(x, more) + (id >> 3);
    split = id / (a.tiles_m * a.tiles_n);
    const int tile = id - split * a.tiles_m * a.tiles_n;
    tm = a.tiles_m <= a.tiles_n ? tile % a.tiles_m : tile / a.tiles_n;
    tn = a.tiles_m <= a.tiles_n ? tile / a.tiles_m : tile % a.tiles_n;
}

// BM x BN of C by WM x WN waves, of k in the split's part, for operands of 16-bit rows of k that start anywhere.  Two tiles of
// each operand in LDS: while one is multiplied, the next comes into registers, and from there into the other (2500 x 66000 x
// 512 bfloat16 forward 264 us; straight into LDS, below, 230).
template <typename T, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM *WN *kWave) k_gemm(GemmArgs a) {
    using M = Mma<T>;
    constexpr int NT = WM * WN * kWave, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
    constexpr int BK = Stage<T, BM, NT>::kBK, kTile = (BM + BN) * kRowBytes;
    __shared__ __attribute__((aligned(16))) char lds[2 * kTile];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, r16 = lane % 16, kq = lane / 16;
    const int wm = wave / WN * TM, wn = wave % WN * TN;
    int tm, tn, split;
    my_tile(a, tm, tn, split);
    const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
    const int64_t k0 = split * a.k_part, k1 = min(a.K, k0 + a.k_part);
    Stage<T, BM, NT> sp;
    Stage<T, BN, NT> sq;
    sp.init(static_cast<const T *>(a.p), a.p_ld, m0, a.M, k0);
    sq.init(static_cast<const T *>(a.q), a.q_ld, n0, a.N, k0);
    f32x4 acc[FM][FN] = {};
    const int steps = static_cast<int>((k1 - k0 + BK - 1) / BK);
    if (steps > 0) {
        sp.load(k1 - k0);
        sq.load(k1 - k0);
        sp.store(lds);
        sq.store(lds + BM * kRowBytes);
        __syncthreads();
    }
    for (int s = 0; s < steps; ++s) {
        const char *cur = lds + (s & 1) * kTile;
        const bool more = s + 1 < steps;
        if (more) {
            const int64_t left = k1 - k0 - static_cast<int64_t>(s + 1) * BK;
            sp.load(left);
            sq.load(left);
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            typename M::frag fp[FM], fq[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i)
                fp[i] = *reinterpret_cast<const typename M::frag *>(cur + lds_at(wm + 16 * i + r16, 4 * kk + kq));
#pragma unroll
            for (int j = 0; j < FN; ++j)
                fq[j] = *reinterpret_cast<const typename M::frag *>(cur + BM * kRowBytes + lds_at(wn + 16 * j + r16, 4 * kk + kq));
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = M::run(fq[j], fp[i], acc[i][j]);   // rows of the result: n
        }
        if (more) {
            char *next = lds + ((s + 1) & 1) * kTile;
            sp.store(next);
            sq.store(next + BM * kRowBytes);
        }
        __syncthreads();
    }
    put<T, TM, TN, 2 * kTile / (WM * WN)>(a, acc, lds + wave * (2 * kTile / (WM * WN)), m0 + wm, n0 + wn, split);
}

#ifdef __HIP_DEVICE_COMPILE__   // the host's pass does not know the builtins
// ---- operands straight into LDS ---------------------------------------------------------------------------------------
// Memory to LDS without registers, 64 x PB bytes of consecutive LDS a wave and instruction; the permutation of the chunks is
// in the addresses that are read.  COL operands lie in LDS as they do in memory, rows of k, and are turned where they are
// read: 16-bit types by the LDS transpose read (16 lanes take 4 k's of 16 m's), float32 by reading single values.  There the
// 16-m pieces of row k are permuted by those bits of k in which the rows of one read differ.
// PB 16 is for rows on 16-byte addresses and of whole chunks, PB 4 for rows on 4-byte ones; a tile of an operand lies within
// 32 bits.
constexpr int kRawBuffer = 0x00020000;   // descriptor word 3: untyped 32-bit offsets
template <typename T, bool COL, int ROWS, int WAVES, int PB>
struct Direct {
    static constexpr int kSize = static_cast<int>(sizeof(T)), kBK = kRowBytes / kSize;
    static constexpr int kLoad = kWave * PB, kN = ROWS * kRowBytes / kLoad / WAVES;    // bytes of an instruction, those of a wave
    static constexpr int kColBytes = ROWS * kSize, kPiece = 16 * kSize;
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    const char *base;              // the next tile's first value, uniform
    uint32_t off[kN];              // of the lane's pieces in a tile
    uint32_t ld;                   // bytes
    int range;                     // of the addresses a load may touch: all, or none

    static __device__ __forceinline__ int col_key(int k) { return (kSize == 2 ? (k & 3) | ((k >> 1) & 4) : (k >> 2) & 3) & (ROWS / 16 - 1); }

    // what lands at lane's place of instruction i: COL (row k, byte of it), else (row, byte of its k's)
    static __device__ __forceinline__ void place(int wave, int lane, int i, int &row, int &at) {
        const int byte = (wave * kN + i) * kLoad + lane * PB;
        if (COL) {
            row = byte / kColBytes, at = byte % kColBytes;
            at = (at / kPiece ^ col_key(row)) * kPiece + at % kPiece;
        } else {
            row = byte / kRowBytes, at = ((byte / 16 ^ (row >> 1)) & 7) * 16 + byte % 16;
        }
    }

    __device__ __forceinline__ void init(const void *p, int64_t stride, int64_t row0, int64_t rows, int64_t k0, int wave, int lane) {
        ld = static_cast<uint32_t>(stride * kSize);
        base = static_cast<const char *>(p) + (COL ? k0 * stride + row0 : row0 * stride + k0) * kSize;
        range = -1;
        const int have = static_cast<int>(min(rows - row0, static_cast<int64_t>(ROWS)));
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            int r, at;
            place(wave, lane, i, r, at);
            off[i] = COL ? r * ld + min(at, have * kSize - PB) : min(r, have - 1) * ld + at;
        }
    }

    // Before the load of a last tile with `left` k's: what would lie past them is read from the tile's first k's, and
    // cleared by clear().
    __device__ __forceinline__ void shorten(int left, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            int r, at;
            place(wave, lane, i, r, at);
            if (COL && r >= left) off[i] -= r * ld;
            if (!COL && at >= left * kSize) off[i] -= at;
        }
    }

    // Every further load is of an empty range.
    __device__ __forceinline__ void stop() { range = 0; }

    __device__ __forceinline__ void load(char *lds, int wave) {
        typedef __attribute__((address_space(3))) void *lptr;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, range, kRawBuffer);
#pragma unroll
        for (int i = 0; i < kN; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lptr)(lds + (wave * kN + i) * kLoad), PB, off[i], 0, 0, 0);
        base += COL ? static_cast<int64_t>(kBK) * ld : kRowBytes;
    }

    static __device__ __forceinline__ void clear(char *lds, int left) {
        for (int u = threadIdx.x; u < ROWS * kRowBytes / 4; u += WAVES * kWave) {
            const int row = COL ? u * 4 / kColBytes : u / 32, at = u * 4 % kRowBytes;
            if (COL ? row >= left : at >= left * kSize)
                *reinterpret_cast<uint32_t *>(lds + (COL ? u * 4 : lds_at(row, at / 16) + at % 16)) = 0u;
        }
    }

    // A wave's reads: fragment i, rows w + 16 i .., of matrix instruction kk of the tile.  What depends on
    // the lane is one of a few offsets (the permutation is an exclusive or of a lane's part and of i's and kk's).
    static constexpr int kReads = !COL ? 1 : kSize == 2 ? 2 : 4;   // LDS reads of a fragment
    static constexpr int kAts = !COL ? 2 : kSize == 2 ? 8 : 4;
    struct Reader {
        int at[kAts];
        __device__ __forceinline__ Reader(int w, int r16, int kq) {
#pragma unroll
            for (int c = 0; c < kAts; ++c) {
                if (!COL) at[c] = lds_at(w + r16, 4 * c + kq);
                else if (kSize == 2) at[c] = (8 * kq + (r16 >> 2)) * kColBytes + ((w / 16 + c) ^ col_key(8 * kq + (r16 >> 2))) * kPiece + (r16 & 3) * 8;
                else at[c] = 4 * kq * kColBytes + ((w / 16 + c) ^ col_key(4 * kq)) * kPiece + r16 * 4;
            }
        }
        __device__ __forceinline__ vec frag(const char *lds, int i, int kk) const {
            if constexpr (!COL) {
                return *reinterpret_cast<const vec *>(lds + at[kk] + i * 16 * kRowBytes);
            } else if constexpr (kSize == 2) {
                typedef short s4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s4 *l4;
                static_assert(ROWS <= 256, "eight fragments a wave");
                const char *p = lds + at[i] + kk * 32 * kColBytes;
                const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l4)(p));
                const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l4)(p + 4 * kColBytes));
                return __builtin_bit_cast(vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            } else {
                vec v;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = *reinterpret_cast<const T *>(lds + at[i & 3] + (kk * 16 + e) * kColBytes + i / 4 * 4 * kPiece);
                return v;
            }
        }
    };
};

#endif

// BM x BN of C by WM x WN waves, of k in the split's part.  Two tiles of each operand in LDS; the second half of a tile's
// operands is in registers before the barrier at which the tile's LDS is given to the loads of the tile after next, and the
// first half of the next tile's is read while that second half is multiplied.
template <typename T, int BM, int BN, int WM, int WN, bool PCOL, bool QCOL, int PB>
__global__ void __launch_bounds__(WM *WN *kWave) k_gemm_direct(GemmArgs a) {
#ifdef __HIP_DEVICE_COMPILE__
    using M = Mma<T>;
    constexpr int W = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
    using P = Direct<T, PCOL, BM, W, PB>;
    using Q = Direct<T, QCOL, BN, W, PB>;
    constexpr int BK = P::kBK, kQAt = BM * kRowBytes, kTile = (BM + BN) * kRowBytes;
    __shared__ __attribute__((aligned(1024))) char lds0[kTile];
    __shared__ __attribute__((aligned(1024))) char lds1[kTile];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r16 = lane % 16, kq = lane / 16;
    const int wm = wave / WN * TM, wn = wave % WN * TN;
    int tm, tn, split;
    my_tile(a, tm, tn, split);
    const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * BN;
    const int64_t k0 = split * a.k_part, k1 = min(a.K, k0 + a.k_part);
    const int steps = static_cast<int>((k1 - k0 + BK - 1) / BK);
    const int tail = static_cast<int>(k1 - k0 - static_cast<int64_t>(steps - 1) * BK);   // k's of the last tile
    P p;
    Q q;
    p.init(a.p, a.p_ld, m0, a.p_rows, k0, wave, lane);
    q.init(a.q, a.q_ld, n0, a.q_rows, k0, wave, lane);
    const typename P::Reader rp(wm, r16, kq);
    const typename Q::Reader rq(wn, r16, kq);
    f32x4 acc[FM][FN] = {};
    typename M::frag fp0[FM], fq0[FN], fp1[FM], fq1[FN];
    auto shorten = [&](int s) {   // before the load of tile s
        if (s + 1 == steps && tail < BK) {
            p.shorten(tail, wave, lane);
            q.shorten(tail, wave, lane);
        }
    };
    auto fetch = [&](char *to) {
        p.load(to, wave);
        q.load(to + kQAt, wave);
    };
    // the tiles that are on their way have landed, and nobody reads the LDS that is loaded next any more
    auto meet = [&](char *landed, bool last) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (last && tail < BK) {
            P::clear(landed, tail);
            Q::clear(landed + kQAt, tail);
            __syncthreads();
        }
    };
    auto half = [&](typename M::frag(&fp)[FM], typename M::frag(&fq)[FN], const char *from, int kk) {
#pragma unroll
        for (int i = 0; i < FM; ++i) fp[i] = rp.frag(from, i, kk);
#pragma unroll
        for (int j = 0; j < FN; ++j) fq[j] = rq.frag(from + kQAt, j, kk);
    };
    auto mul = [&](typename M::frag(&fp)[FM], typename M::frag(&fq)[FN]) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = M::run(fq[j], fp[i], acc[i][j]);   // rows of the result: n
    };
    // A wave issues in order and the loads wait for their turn at the address unit, so they are spread among the matrix
    // instructions; for that they are always there, past the last tile with an empty range (nothing is read).
    auto step = [&](char *cur, char *next, int s) {
        shorten(s + 2);
        half(fp1, fq1, cur, 1);
        mul(fp0, fq0);
        if (s + 2 >= steps) p.stop(), q.stop();
        meet(next, s + 2 == steps);
        fetch(cur);
        half(fp0, fq0, next, 0);   // of no tile after the last, and then not used
        mul(fp1, fq1);
        constexpr int kLoads = P::kN + Q::kN, kMul = FM * FN * (sizeof(T) == 4 ? 4 : 1), kReads = FM * P::kReads + FN * Q::kReads;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, (kReads + kLoads - 1) / kLoads, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, kMul / kLoads, 0);
            __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
        }
    };
    shorten(0);
    fetch(lds0);
    meet(lds0, steps == 1);
    shorten(1);
    if (steps == 1) p.stop(), q.stop();
    fetch(lds1);
    half(fp0, fq0, lds0, 0);
    for (int s = 0;;) {
        step(lds0, lds1, s);
        if (++s == steps) break;
        step(lds1, lds0, s);
        if (++s == steps) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the empty loads still write to LDS
    __syncthreads();
    constexpr int kSlab = 2 * kTile / W;
    char *slab = wave < W / 2 ? lds0 + wave * kSlab : lds1 + (wave - W / 2) * kSlab;
    put<T, TM, TN, kSlab>(a, acc, slab, m0 + wm, n0 + wn, split);
#endif
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
// Products of which one side has at most 16 MT rows (single ticks; a readout of few classes): the other side's 16 rows of a
// block stream from memory straight into operands, each of the block's four waves over a part of the block's k's, and the
// few rows come from the caches.  NFEW: the few are q's rows (n), else p's (m).  Bound by the stream: 5 x 66000 x 512 bfloat16,
// 68 MB of weights, 15 us and 5 for the join of the parts of k.
template <typename T, int MT, bool NFEW>
__global__ void __launch_bounds__(kBlock) k_few(GemmArgs a) {
    using M = Mma<T>;
    constexpr int kV = 16 / static_cast<int>(sizeof(T)), KS = 4 * kV, U = 4, kWaves = kBlock / kWave;
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    __shared__ f32x4 sums[kWaves][MT][kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, r16 = lane % 16, kq = lane / 16;
    const int64_t many = NFEW ? a.M : a.N, few = NFEW ? a.N : a.M;
    const int groups = NFEW ? a.tiles_m : a.tiles_n, split = blockIdx.x / groups;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x - split * groups) * 16;
    // the wave's k's, in whole matrix instructions
    const int64_t b0 = split * a.k_part, b1 = min(a.K, b0 + a.k_part), part = (b1 - b0 + kWaves * KS - 1) / (kWaves * KS) * KS;
    const int64_t k0 = min(b0 + wave * part, b1), k1 = min(k0 + part, b1);
    const T *pm = static_cast<const T *>(NFEW ? a.p : a.q) + min(row0 + r16, many - 1) * (NFEW ? a.p_ld : a.q_ld) + kq * kV;
    const T *pf[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
        pf[i] = static_cast<const T *>(NFEW ? a.q : a.p) + min(static_cast<int64_t>(16 * i + r16), few - 1) * (NFEW ? a.q_ld : a.p_ld) + kq * kV;
    f32x4 acc[MT] = {};
    auto mul = [&](typename M::frag f, typename M::frag w, f32x4 c) { return NFEW ? M::run(f, w, c) : M::run(w, f, c); };   // rows: n
    int64_t k = k0;
    for (; k + U * KS <= k1; k += U * KS) {
        vec w[U], f[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = *reinterpret_cast<const vec *>(pm + k + u * KS);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) f[u][i] = *reinterpret_cast<const vec *>(pf[i] + k + u * KS);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = mul(f[u][i], w[u], acc[i]);
    }
    for (; k < k1; k += KS) {
        const int64_t left = k1 - k - kq * kV;
        auto load = [&](const T *p) {
            if (left >= kV) return *reinterpret_cast<const vec *>(p + k);
            vec v;
#pragma unroll
            for (int e = 0; e < kV; ++e) v[e] = e < left ? p[k + e] : T(0.0f);
            return v;
        };
        const vec w = load(pm);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = mul(load(pf[i]), w, acc[i]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave >= MT) return;
    f32x4 v = sums[0][wave][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w][wave][lane];
    const int64_t m = NFEW ? row0 + r16 : 16 * wave + r16, n = (NFEW ? 16 * wave : row0) + kq * 4;
    if (m >= a.M || n >= a.N) return;
    if (a.splits > 1) {
        *reinterpret_cast<f32x4 *>(a.part + (split * a.M + m) * a.part_ld + n) = v;
    } else {
        const Finish<T> finish(a, n);
        finish(a, m, v, finish.residual(a, m));
    }
}

// The splits' sums and the epilogue: four results by G lanes, which take the splits in turn (their sums are joined by a fixed
// tree).
template <typename T, int G>
__global__ void __launch_bounds__(kBlock) k_gemm_join(GemmArgs a) {
    const int64_t quads = a.part_ld / 4, n4 = a.M * quads, step = static_cast<int64_t>(gridDim.x) * (kBlock / G);
    const int g = threadIdx.x % G;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kBlock / G) + threadIdx.x / G; i < n4; i += step) {
        const int64_t m = i / quads, n = (i - m * quads) * 4;
        const Finish<T> finish(a, n);
        const typename Finish<T>::vec res = finish.residual(a, m);
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        const float *p = a.part + (g * a.M + m) * a.part_ld + n;
#pragma unroll 4
        for (int s = g; s < a.splits; s += G, p += G * a.M * a.part_ld) v += *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
        for (int x = 1; x < G; x <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], x, kWave);
        if (g == 0) finish(a, m, v, res);
    }
}

constexpr int kSlopeCols = 32, kSlopeLots = kBlock / kSlopeCols;
struct SlopeArgs {
    const void *dy;
    const float *pre;    // [M][N]
    int64_t lddy, M, N;
    void *dp;            // [M][lddp] or NULL
    int64_t lddp;
    float *part;         // [parts][N] or NULL
    int32_t act, parts;
};

// dp = dy act'(pre), rounded to the activations' type for the products (zeros past N: the matrix instructions take both
// operands in one type, and a second product for what the rounding leaves would double their time), and the column sums of the
// unrounded values over a chunk of rows: 32 pieces of 16 bytes by 8 rows a block (2500 x 512 bfloat16 with gelu, and the sums' join
// below: a column a thread 18 and 39 us, so 11 and 4).
template <typename T>
__global__ void __launch_bounds__(kBlock) k_slope(SlopeArgs a) {
    constexpr int V = kVecBytes16<T>;
    typedef Vec<T, V> vec;
    __shared__ float sum[kSlopeLots][kSlopeCols * V + 4];
    const int col = threadIdx.x % kSlopeCols, lot = threadIdx.x / kSlopeCols;
    const int64_t n = (static_cast<int64_t>(blockIdx.x) * kSlopeCols + col) * V, cols = a.dp ? a.lddp : a.N;
    const int64_t r0 = a.M * blockIdx.y / a.parts, r1 = a.M * (blockIdx.y + 1) / a.parts;
    const T *dy = static_cast<const T *>(a.dy) + n;
    const float *pre = a.pre + n;
    T *dp = static_cast<T *>(a.dp) + n;
    float s[V] = {};
    if (n + V <= a.N) {
#pragma unroll 2
        for (int64_t m = r0 + lot; m < r1; m += kSlopeLots) {
            const vec g = *reinterpret_cast<const vec *>(dy + m * a.lddy);
            Vec<float, V> p = {};
            vec o;
            if (a.act != GLIF_ACT_NONE) p = *reinterpret_cast<const Vec<float, V> *>(pre + m * a.N);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float v = to_f32(static_cast<T>(g[e])) * slope_of(p[e], a.act);
                o[e] = from_f32<T>(v);
                s[e] += v;
            }
            if (a.dp) *reinterpret_cast<vec *>(dp + m * a.lddp) = o;
        }
    } else if (n < cols) {
        for (int64_t m = r0 + lot; m < r1; m += kSlopeLots) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float v = 0.0f;
                if (n + e < a.N) {
                    v = to_f32(dy[m * a.lddy + e]);
                    if (a.act != GLIF_ACT_NONE) v *= slope_of(pre[m * a.N + e], a.act);
                }
                if (a.dp && n + e < cols) dp[m * a.lddp + e] = from_f32<T>(v);
                s[e] += v;
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int e = 0; e < V; ++e) sum[lot][col * V + e] = s[e];
    __syncthreads();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kSlopeCols * V;
    for (int c = threadIdx.x; c < kSlopeCols * V; c += kBlock) {
        if (first + c >= a.N) continue;
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < kSlopeLots; ++i) t += sum[i][c];
        a.part[static_cast<int64_t>(blockIdx.y) * a.N + first + c] = t;
    }
}

// 16-bit rows onto 16-byte addresses: out [rows][ldo], ldo a multiple of 8, zeros past cols.
__global__ void __launch_bounds__(kBlock) k_repack(const uint16_t *in, int64_t ld, int64_t rows, int64_t cols, uint16_t *out, int64_t ldo) {
    typedef Vec<uint16_t, 8> vec;
    const int64_t per = ldo / 8, n = rows * per;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t r = i / per, c = (i - r * per) * 8;
        const uint16_t *p = in + r * ld + c;
        vec v;
        if (c + 8 <= cols) {
            v = *reinterpret_cast<const vec *>(p);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? p[e] : 0;
        }
        *reinterpret_cast<vec *>(out + i * 8) = v;
    }
}

// The parts' sums: 32 columns by 8 threads, which take the parts in turn.
__global__ void __launch_bounds__(kBlock) k_bias_join(const float *part, int parts, int64_t N, void *dbias, int32_t dt) {
    __shared__ float sum[kSlopeLots][kSlopeCols];
    const int col = threadIdx.x % kSlopeCols, lot = threadIdx.x / kSlopeCols;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * kSlopeCols + col;
    float s = 0.0f;
    if (n < N) {
#pragma unroll 4
        for (int p = lot; p < parts; p += kSlopeLots) s += part[p * N + n];
    }
    sum[lot][col] = s;
    __syncthreads();
    if (lot || n >= N) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < kSlopeLots; ++i) s += sum[i][col];
    store_param(dbias, dt, n, s);
}

// How a product, or one of two pieces of it, is cut up: the tile, and the parts of k whose sums are added afterwards.
enum Kind { kFew16, kFew32, kTile64, kTile128, kTile256 };
struct Piece {
    Kind kind;
    int32_t splits;
    int64_t k_part, part_ld, rows;
    size_t floats() const { return splits > 1 ? static_cast<size_t>(splits) * rows * part_ld : 0; }
};
struct Plan {
    Piece one, two;     // two: of the rows (cut_m) or columns from `cut` on, where that is not 0
    int64_t cut;
    bool cut_m;
    size_t floats() const { return std::max(one.floats(), cut ? two.floats() : 0); }
};

// rr: both operands have k along their rows.
//
// At most 32 rows on one side: k is split until the chip has about eight waves a SIMD to keep the stream of the other side
// going, but no part under 512 k's.  (40 rows by this kernel: 16000 x 4096 x 40 59 us, by 64 x 64 tiles 30.)
//
// Otherwise the cheapest of the tiles and some splits.  A step (128 bytes of k) of a block that is alone on its compute unit
// takes, in us, 16-bit 256 x 256 1.7, 128 x 128 1.0, 64 x 64 0.5, and float32, whose products run at 1/16, 128 x 128 3.0, 64
// x 64 1.1; a step of all of the 1, 2 or 5 blocks that a compute unit holds 1.9, 1.35, 1.2, and 4.3, 2.9 (measured over
// sweeps of tiles and splits at 15 shapes).  Around the steps go 10, 5 and 3; a split costs its sums' way to memory and back
// and the launch that adds them.  Tiles of float32 operands sum over at most 4096 k's up to 64 parts (K of 262144), so that long
// sums do not lose their last digits; few rows are in a wave's parts of k anyway (all-positive float32 terms, K of 66000 with 16500
// to a wave: 3e-6 of the sum), and 16-bit results keep fewer digits than either.
Piece piece_for(int32_t dtype, int64_t M, int64_t N, int64_t K, bool rr, double &best) {
    Piece p{};
    best = 0.0;
    p.rows = M, p.part_ld = (N + 3) / 4 * 4, p.splits = 1, p.kind = kTile128;
    const int64_t size = static_cast<int64_t>(dtype_size(dtype)), bk = kRowBytes / size, steps = std::max<int64_t>((K + bk - 1) / bk, 1);
    p.k_part = steps * bk;
    if (M <= 0 || N <= 0) return p;
    const int64_t few = std::min(M, N), many = std::max(M, N);
    int64_t splits = 1;
    if (rr && few <= 32) {
        p.kind = few <= 16 ? kFew16 : kFew32;
        splits = std::max<int64_t>(1, std::min<int64_t>(2048 / ((many + 15) / 16), K / 512));
        p.k_part = (steps + splits - 1) / splits * bk;
        best = 10.0 + static_cast<double>(many * K * size) / 4e6;   // the stream at 4 TB/s
    } else {
        best = 1e30;
        for (const int tile : {64, 128, 256}) {
            if (size == 4 && tile == 256) continue;
            const int64_t tiles = ((M + tile - 1) / tile) * ((N + tile - 1) / tile);
            const int64_t cap = tile == 256 ? 1 : tile == 128 ? 2 : 5;
            const double alone = size == 2 ? (tile == 256 ? 1.7 : tile == 128 ? 1.0 : 0.5) : (tile == 128 ? 3.0 : 1.1);
            const double full = size == 2 ? (tile == 256 ? 1.9 : tile == 128 ? 1.35 : 1.2) : (tile == 128 ? 4.3 : 2.9);
            const double around = tile == 256 ? 10.0 : tile == 128 ? 5.0 : 3.0;
            for (int64_t c = 1; c <= std::min<int64_t>(64, steps); ++c) {
                const int64_t each = (steps + c - 1) / c, n = (steps + each - 1) / each;
                if (size == 4 && each * bk > 4096 && c < std::min<int64_t>(64, steps)) continue;
                if (c > 1 && each < 4 && !(size == 4 && K > 4096)) break;
                const int64_t unit = (tiles * n + 255) / 256, together = std::min(cap, unit);   // blocks of a compute unit
                const double step = cap == 1 ? full : alone + (full - alone) * static_cast<double>(together - 1) / static_cast<double>(cap - 1);
                const double cost = static_cast<double>(unit) / static_cast<double>(together) * (static_cast<double>(each) * step + around) +
                                    (n > 1 ? 4.0 + static_cast<double>(n * M * N) * 8e-6 / 6.0 : 0.0);
                if (cost < best) best = cost, p.kind = tile == 256 ? kTile256 : tile == 128 ? kTile128 : kTile64, p.k_part = each * bk;
            }
        }
    }
    p.splits = static_cast<int32_t>((steps * bk + p.k_part - 1) / p.k_part);
    return p;
}

// Tiles that are a few more than whole rounds of the chip's blocks cost one round more.  Where it is cheaper, and by more than
// a launch, the whole rounds are one piece, and the rest, as short tiles or with k in parts, is another (2500 x 66000 x 512
// bfloat16, dW of 516 tiles of 256 x 256, 226 us in one, 177 in two).
Plan plan_for(int32_t dtype, int64_t M, int64_t N, int64_t K, bool rr) {
    Plan p{};
    double best;
    p.one = piece_for(dtype, M, N, K, rr, best);
    p.cut_m = M > N;
    const int64_t across = std::min(M, N), along = std::max(M, N);
    if (across <= 32) return p;
    for (const int tile : {128, 256}) {
        if (dtype_size(dtype) == 4 && tile == 256) continue;
        const int64_t slots = tile == 256 ? 256 : 512, wide = (across + tile - 1) / tile;
        const int64_t cut = wide * ((along + tile - 1) / tile) / slots * slots / wide * tile;
        if (cut == 0 || cut >= along) continue;
        double first, rest;
        const Piece one = p.cut_m ? piece_for(dtype, cut, N, K, rr, first) : piece_for(dtype, M, cut, K, rr, first);
        const Piece two = p.cut_m ? piece_for(dtype, M - cut, N, K, rr, rest) : piece_for(dtype, M, N - cut, K, rr, rest);
        if (first + rest + 4.0 < best) best = first + rest + 4.0, p.one = one, p.two = two, p.cut = cut;
    }
    return p;
}

// Whether an operand's rows lie in 16-byte pieces.
bool on_16(const void *p, int64_t ld, int64_t along, size_t size) {
    const int64_t v = 16 / static_cast<int64_t>(size);
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % v == 0 && along % v == 0;
}

// float32 rows may start on any float32; 16-bit rows of k that do not lie on 16 bytes come by way of registers (16-bit
// operands of columns have been put on 16 bytes).
template <typename T, int TILE, int WM, int WN, bool PCOL, bool QCOL>
void launch_tile(GemmArgs &a, hipStream_t s) {
    a.tiles_m = ceil_div(a.M, TILE), a.tiles_n = ceil_div(a.N, TILE);
    const dim3 grid(static_cast<unsigned>(a.tiles_m * a.tiles_n * a.splits)), block(WM * WN * kWave);
    if (on_16(a.p, a.p_ld, PCOL ? a.p_rows : a.k_cols, sizeof(T)) && on_16(a.q, a.q_ld, QCOL ? a.q_rows : a.k_cols, sizeof(T))) {
        hipLaunchKernelGGL((k_gemm_direct<T, TILE, TILE, WM, WN, PCOL, QCOL, 16>), grid, block, 0, s, a);
    } else if constexpr (sizeof(T) == 4) {
        hipLaunchKernelGGL((k_gemm_direct<T, TILE, TILE, WM, WN, PCOL, QCOL, 4>), grid, block, 0, s, a);
    } else if constexpr (!PCOL && !QCOL) {
        if constexpr (TILE == 64) hipLaunchKernelGGL((k_gemm<T, 64, 64, 2, 1>), grid, dim3(2 * kWave), 0, s, a);
        else hipLaunchKernelGGL((k_gemm<T, TILE, TILE, WM, WN>), grid, block, 0, s, a);
    }
}

template <typename T, int MT>
void launch_few(GemmArgs &a, hipStream_t s) {
    const bool nfew = a.N < a.M;
    a.tiles_m = ceil_div(a.M, 16), a.tiles_n = ceil_div(a.N, 16);
    const dim3 grid(static_cast<unsigned>((nfew ? a.tiles_m : a.tiles_n) * a.splits));
    if (nfew) hipLaunchKernelGGL((k_few<T, MT, true>), grid, dim3(kBlock), 0, s, a);
    else hipLaunchKernelGGL((k_few<T, MT, false>), grid, dim3(kBlock), 0, s, a);
}

template <typename T, bool PCOL, bool QCOL>
void launch_piece(GemmArgs a, const Piece &p, float *part, hipStream_t s) {
    a.splits = p.splits, a.k_part = p.k_part, a.part_ld = p.part_ld, a.part = part;
    // a tile's rows of k within 32-bit offsets
    const int64_t ld = std::max(PCOL ? 0 : a.p_ld, QCOL ? 0 : a.q_ld) * static_cast<int64_t>(sizeof(T));
    const int64_t most = ((int64_t(1) << 32) - 1) / std::max<int64_t>(ld, 1);
    if (a.K == 0) {
        a.splits = 0;   // the epilogue of empty sums (the tile kernels load a first tile whatever there is)
    } else if (p.kind == kFew16 || p.kind == kFew32) {
        if constexpr (!PCOL && !QCOL) p.kind == kFew16 ? launch_few<T, 1>(a, s) : launch_few<T, 2>(a, s);
    } else if (sizeof(T) == 2 && p.kind == kTile256 && most >= 256) {
        if constexpr (sizeof(T) == 2) launch_tile<T, 256, 2, 4, PCOL, QCOL>(a, s);
    } else if (p.kind != kTile64 && most >= 128) {
        launch_tile<T, 128, 2, 2, PCOL, QCOL>(a, s);
    } else {
        launch_tile<T, 64, 2, 2, PCOL, QCOL>(a, s);
    }
    if (a.splits != 1) {
        // where the results alone do not fill the chip, lanes over the splits: 5 x 66000 x 512 in 61 parts 14 us -> 4
        const int64_t n4 = a.M * (a.part_ld / 4);
        if (n4 < 32768 && a.splits >= 16)
            hipLaunchKernelGGL((k_gemm_join<T, 16>), dim3(static_cast<unsigned>(ceil_div(n4, kBlock / 16))), dim3(kBlock), 0, s, a);
        else
            hipLaunchKernelGGL((k_gemm_join<T, 1>), dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(n4, kBlock), 8192))),
                               dim3(kBlock), 0, s, a);
    }
}

template <typename T, bool PCOL, bool QCOL>
int launch_gemm(GemmArgs a, const Plan &p, float *part, hipStream_t s) {
    if (a.M == 0 || a.N == 0) return GLIF_OK;
    // (8192^3 bfloat16 1009 us -> 846; 2500 x 512 x 66000, 330 MB of results, 292 -> 271; 2500 x 512 x 12007, 60 MB, 57 and 63)
    a.past = a.M * a.N * static_cast<int64_t>(sizeof(T)) > kPastCaches;
    a.ldc = a.N;
    if (p.cut == 0) {
        launch_piece<T, PCOL, QCOL>(a, p.one, part, s);
        return GLIF_OK;
    }
    GemmArgs b = a;
    auto on = [](auto &at, int64_t by) { at = at ? const_cast<char *>(static_cast<const char *>(at)) + by : nullptr; };
    const int64_t size = sizeof(T);
    if (p.cut_m) {
        a.M = p.cut, b.M -= p.cut, b.p_rows -= p.cut;
        on(b.p, p.cut * size * (PCOL ? 1 : b.p_ld));
        on(b.c, p.cut * size * b.ldc), on(b.residual, p.cut * size * b.ldr);
        if (b.pre) b.pre += p.cut * b.ldc;
    } else {
        a.N = p.cut, b.N -= p.cut, b.q_rows -= p.cut;
        on(b.q, p.cut * size * (QCOL ? 1 : b.q_ld));
        on(b.c, p.cut * size), on(b.residual, p.cut * size);
        if (b.pre) b.pre += p.cut;
        on(b.bias, p.cut * static_cast<int64_t>(dtype_size(b.bias_dt)));
    }
    launch_piece<T, PCOL, QCOL>(a, p.one, part, s);
    launch_piece<T, PCOL, QCOL>(b, p.two, part, s);
    return GLIF_OK;
}

template <typename T>
int gemm_rr(const GemmArgs &a, const Plan &p, float *part, hipStream_t s) { return launch_gemm<T, false, false>(a, p, part, s); }
template <typename T>
int gemm_rc(const GemmArgs &a, const Plan &p, float *part, hipStream_t s) { return launch_gemm<T, false, true>(a, p, part, s); }
template <typename T>
int gemm_cc(const GemmArgs &a, const Plan &p, float *part, hipStream_t s) { return launch_gemm<T, true, true>(a, p, part, s); }

template <typename T>
void run_slope(const SlopeArgs &a, hipStream_t s) {
    if (a.N == 0) return;
    hipLaunchKernelGGL(k_slope<T>, dim3(static_cast<unsigned>(ceil_div(a.dp ? a.lddp : a.N, kSlopeCols * kVecBytes16<T>)),
                                         static_cast<unsigned>(a.parts)),
                       dim3(kBlock), 0, s, a);
}

int row_parts(int64_t M) { return static_cast<int>(std::min<int64_t>(std::max<int64_t>(M / 16, 1), 256)); }

// Rows whose tiles would pass 32-bit offsets.
int check_strides(int64_t a, int64_t b, int64_t c) {
    if (std::max({a, b, c}) >= (1 << 24)) return fail(GLIF_EINVAL, "linear: row strides must be below 2^24");
    return GLIF_OK;
}

int check_linear(int32_t dtype, int32_t bias_dtype, int64_t M, int64_t N, int64_t K, int32_t act) {
    if (!known_dtype(dtype) || (bias_dtype != GLIF_F32 && bias_dtype != dtype))
        return fail(GLIF_EINVAL, "linear: the bias is float32 or of x's type");
    if (M < 0 || N < 0 || K < 0 || M > (1 << 21) || N > (1 << 21) || K >= (1 << 24))
        return fail(GLIF_EINVAL, "linear: M and N in [0, 2^21], K in [0, 2^24)");
    if (act < GLIF_ACT_NONE || act > GLIF_ACT_SILU) return fail(GLIF_EINVAL, "linear: unknown activation");
    return GLIF_OK;
}

struct Back {
    void *dp, *w, *x;     // dp, and the operands put on 16 bytes
    float *part, *sums;   // of the products' splits (one after the other), of the bias's rows
    int32_t parts;
    int64_t np, kp;       // N and K in whole 16 bytes, for 16-bit types
    Plan dx, dw;
};

// repack: some operand of a 16-bit type does not lie on 16 bytes
void carve(Carver &c, Back &b, int32_t dtype, int64_t M, int64_t N, int64_t K, int32_t act, bool repack) {
    const bool half = dtype != GLIF_F32;
    const size_t size = dtype_size(dtype);
    b.parts = row_parts(M);
    b.np = half ? (N + 7) / 8 * 8 : N, b.kp = half ? (K + 7) / 8 * 8 : K;
    b.dx = plan_for(dtype, M, K, N, false), b.dw = plan_for(dtype, N, K, M, false);
    b.sums = c.take<float>(static_cast<size_t>(b.parts * N));
    b.part = c.take<float>(std::max(b.dx.floats(), b.dw.floats()));
    repack = repack && half;
    if (act != GLIF_ACT_NONE || repack) b.dp = c.take<char>(static_cast<size_t>(M * b.np) * size);
    if (repack) {
        b.w = c.take<char>(static_cast<size_t>(N * b.kp) * size);
        b.x = c.take<char>(static_cast<size_t>(M * b.kp) * size);
    }
}

void run_repack(const void *in, int64_t ld, int64_t rows, int64_t cols, void *out, int64_t ldo, hipStream_t s) {
    const int64_t n = rows * (ldo / 8);
    if (n == 0) return;
    hipLaunchKernelGGL(k_repack, dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(n, kBlock), 16384))), dim3(kBlock), 0, s,
                       static_cast<const uint16_t *>(in), ld, rows, cols, static_cast<uint16_t *>(out), ldo);
}

}  // namespace
}  // namespace glif

using namespace glif;

extern "C" {

size_t glif_linear_fwd_workspace(int32_t dtype, int64_t M, int64_t N, int64_t K) {
    if (check_linear(dtype, dtype, M, N, K, 0)) return 0;
    Carver c(nullptr, 0);
    if (const size_t n = plan_for(dtype, M, N, K, true).floats()) c.take<float>(n);
    return c.off;
}

int glif_linear_fwd(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, const void *residual,
                    int64_t ldr, int32_t dtype, int32_t bias_dtype, int64_t M, int64_t N, int64_t K, int32_t activation,
                    void *y, float *pre, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_linear(dtype, bias_dtype, M, N, K, activation)) return rc;
    if (int rc = check_strides(ldx, ldw, 0)) return rc;
    if (M == 0 || N == 0) return GLIF_OK;
    if (!y || (K && (!x || !weight))) return fail(GLIF_EINVAL, "NULL argument");
    GemmArgs a{};
    a.p = x, a.p_ld = ldx, a.q = weight, a.q_ld = ldw, a.M = a.p_rows = M, a.N = a.q_rows = N, a.K = a.k_cols = K;
    a.c = y, a.pre = pre, a.bias = bias, a.residual = residual, a.ldr = ldr, a.bias_dt = bias_dtype, a.act = activation;
    const Plan p = plan_for(dtype, M, N, K, true);
    Carver c(ws, ws_bytes);
    float *part = c.take<float>(p.floats());
    if (!c.ok() || (p.floats() && !ws)) return fail(GLIF_ENOMEM, "linear: workspace too small");
    if (int rc = GLIF_BY_DTYPE(dtype, gemm_rr, a, p, part, static_cast<hipStream_t>(stream))) return rc;
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

size_t glif_linear_bwd_workspace(int32_t dtype, int64_t M, int64_t N, int64_t K, int32_t activation, int32_t unaligned) {
    if (check_linear(dtype, dtype, M, N, K, activation)) return 0;
    Carver c(nullptr, 0);
    Back b{};
    carve(c, b, dtype, M, N, K, activation, unaligned != 0);
    return c.mark();
}

int glif_linear_bwd(const void *dy, int64_t lddy, const float *pre, const void *x, int64_t ldx, const void *weight,
                    int64_t ldw, int32_t dtype, int32_t bias_dtype, int64_t M, int64_t N, int64_t K, int32_t activation,
                    void *dx, void *dweight, void *dbias, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_linear(dtype, bias_dtype, M, N, K, activation)) return rc;
    if (int rc = check_strides(lddy, ldx, ldw)) return rc;
    const bool some = M && N;
    if (some && (!dy || (activation != GLIF_ACT_NONE && !pre) || (dx && K && !weight) || (dweight && K && !x)))
        return fail(GLIF_EINVAL, "NULL argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t size = dtype_size(dtype);
    const bool half = size == 2;
    const bool move_dy = half && (dx || dweight) && !on_16(dy, lddy, N, size);
    const bool move_w = half && dx && !on_16(weight, ldw, K, size), move_x = half && dweight && !on_16(x, ldx, K, size);
    Back b{};
    Carver c(ws, ws_bytes);
    carve(c, b, dtype, M, N, K, activation, move_dy || move_w || move_x);
    if (!c.ok() || (c.off && !ws)) return fail(GLIF_ENOMEM, "linear: workspace too small");
    const void *dp = dy;
    int64_t lddp = lddy, n_cols = N, k_cols = K;
    const bool own_dp = activation != GLIF_ACT_NONE || move_dy;
    if (own_dp || dbias) {
        SlopeArgs a{dy, pre, lddy, M, N, own_dp ? b.dp : nullptr, b.np, dbias ? b.sums : nullptr, activation, b.parts};
        GLIF_BY_DTYPE(dtype, run_slope, a, s);
        if (own_dp) dp = b.dp, lddp = n_cols = b.np;
        if (dbias && N)
            hipLaunchKernelGGL(k_bias_join, dim3(static_cast<unsigned>(ceil_div(N, kSlopeCols))), dim3(kBlock), 0, s, b.sums, b.parts,
                               N, dbias, bias_dtype);
    }
    if (dx) {
        GemmArgs a{};
        if (move_w) run_repack(weight, ldw, N, K, b.w, b.kp, s), weight = b.w, ldw = k_cols = b.kp;
        a.p = dp, a.p_ld = lddp, a.q = weight, a.q_ld = ldw, a.M = a.p_rows = M, a.N = K, a.q_rows = k_cols, a.K = N, a.k_cols = n_cols;
        a.c = dx;
        if (int rc = GLIF_BY_DTYPE(dtype, gemm_rc, a, b.dx, b.part, s)) return rc;
    }
    if (dweight) {
        GemmArgs a{};
        k_cols = K;
        if (move_x) run_repack(x, ldx, M, K, b.x, b.kp, s), x = b.x, ldx = k_cols = b.kp;
        a.p = dp, a.p_ld = lddp, a.q = x, a.q_ld = ldx, a.M = N, a.p_rows = n_cols, a.N = K, a.q_rows = k_cols, a.K = a.k_cols = M;
        a.c = dweight;
        if (int rc = GLIF_BY_DTYPE(dtype, gemm_cc, a, b.dw, b.part, s)) return rc;
    }
    GLIF_HIP(hipGetLastError());
    return GLIF_OK;
}

}  // extern "C"
