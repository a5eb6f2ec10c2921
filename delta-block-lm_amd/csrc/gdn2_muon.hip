// Orthogonalised updates on gfx950: Newton-Schulz products of matrices, and the Muon update of
// parameters with its momentum.
//
//   X = U / (|U| + epsilon)                     |U| the root of the sum of squares
//   A = X X^T,  B = a I + b A + c A A,  X <- B X           `steps` times
//
// on the side whose product is the smaller one (X has m = min(rows, cols) rows and n columns).  All
// products have the form C = L R^T over rows that lie side by side in memory; X is kept in both
// orientations for that.  A and A A are symmetric: the tiles on and above the diagonal are made and
// written twice.
//
// Precision.  An operand of a product goes in as two float16 terms, x = hi + lo, 23 bits (off by
// 2^-23 of itself), and a product as hi hi + hi lo + lo hi into float32 accumulators (lo lo, which is left
// out, is 2^-22 of it at most), at a third of the matrix cores' float16 rate, where their float32 rate is
// a sixteenth.  float16's range is met by powers of two: the largest
// singular values that X, A and B can have follow from the coefficients, no entry is larger, and the
// powers bring those to 2^14; what is below 2^-24 there is 2^-38 of the largest.  Tiles up to 64 sum
// the small products in accumulators of their own, so that a long sum is not rounded three times as often.
// The polynomial is evaluated and the powers taken in 64 bits and rounded once.  Results are off by 0.4
// to 0.8 of what float32 products leave, relative to their root mean square: 1.0e-6 for 2.3e-6 at
// 512 x 512, 1.2e-6 for 3.3e-6 at 512 x 2816, 3.3e-6 for 4.7e-6 at 4096 x 4096.  Where the smaller side
// is at most 64 the sums are short, and the rounding of operands and accumulators would be the larger
// part (8.4e-7 for 7.0e-7 at 8 x 8): the operands are float32 in the same places and go through the
// float64 matrix instructions, which leaves 1.8e-7 to 2.6e-7; a chunk of a 32 x 32 tile takes 0.25 us for
// 0.115.
//
// A step is three launches that depend on each other, two up to 32 rows, whose A is one tile: 2.4 to 4 us
// each for a matrix of 8 x 8 (40 us in all, 5 steps), 6 to 7 at 512 x 512 (102 us), the same in a captured
// graph; all of 4096 x 4096 is 3.4 to 3.5 ms, 1.17 to 1.2 PFLOP/s of float16 products, where the library's
// float16 product reaches 1.2 to 1.28.
#include <float.h>
#include <math.h>

#include "gdn2_common.h"
#include "gdn2_mfma.h"
#include "gdn2_status.h"

namespace gdn2 {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kGroup = 32;    // matrices of one launch
constexpr int kParts = 1024;  // partial sums of a matrix's squares, at most
constexpr int kSplitThreads = 512;
constexpr int kChunk = 32;    // columns of a 128-byte piece of a row
constexpr int64_t kMostBytes = (int64_t)2 << 30;  // of a group's operands

// An operand: rows of `cols` columns (a multiple of the tile), each 128-byte piece 32 columns, their
// first terms and then their second terms, or as float32 (F32 below).
struct Split {
    char *data;
    int cols;
};

__host__ __device__ __forceinline__ int64_t row_bytes(int64_t cols) { return cols * 4; }

// 8 values to the columns col .. col + 7 of a row; col is a multiple of 8.
template <bool F32> __device__ __forceinline__ void store_split(const Split &s, int64_t row, int col, const float *v) {
    char *p = s.data + row * row_bytes(s.cols) + (col & ~(kChunk - 1)) * 4;
    if (F32) {
        __builtin_memcpy(p + (col & (kChunk - 1)) * 4, v, 32);
        return;
    }
    f16x8 hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        hi[j] = (_Float16)v[j];
        lo[j] = (_Float16)(v[j] - (float)hi[j]);
    }
    p += (col & (kChunk - 1)) * 2;
    *reinterpret_cast<f16x8 *>(p) = hi;
    *reinterpret_cast<f16x8 *>(p + 64) = lo;
}

template <bool F32> __device__ __forceinline__ void load_split(const Split &s, int64_t row, int col, float *v) {
    const char *p = s.data + row * row_bytes(s.cols) + (col & ~(kChunk - 1)) * 4;
    if (F32) {
        __builtin_memcpy(v, p + (col & (kChunk - 1)) * 4, 32);
        return;
    }
    p += (col & (kChunk - 1)) * 2;
    const f16x8 hi = *reinterpret_cast<const f16x8 *>(p), lo = *reinterpret_cast<const f16x8 *>(p + 64);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)hi[j] + (float)lo[j];
}

// ---- the inputs -------------------------------------------------------------------------

struct Tensors {
    float *param[kGroup];
    const float *grad[kGroup];
    float *momentum[kGroup];
};

struct Source {
    Tensors t;      // an update's
    View x;         // [matrix, row, column] otherwise
    int bf16, update, nesterov;
    int dense;      // the view's matrices are rows x cols side by side
    float beta;
    int first;      // matrix of the view that the group starts with
    int rows, cols;
    int parts;      // of the squares
};

__device__ __forceinline__ float source_at(const Source &s, int mat, int64_t r, int64_t c) {
    const int64_t i = (s.first + mat) * s.x.s0 + r * s.x.s1 + c * s.x.s2;
    return s.bf16 ? Elem<bf16_t>::load(s.x.data, i) : Elem<float>::load(s.x.data, i);
}

// Four values of a dense matrix from element i, zeros behind its end n.
template <typename T> __device__ __forceinline__ void load4(const T *p, int64_t i, int64_t n, float *v) {
    if (i + 4 <= n) {
        T w[4];
        __builtin_memcpy(w, p + i, sizeof(w));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = Elem<T>::load(w, j);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < n ? Elem<T>::load(p, i + j) : 0.f;
}

// The first n of four values.
template <typename T> __device__ __forceinline__ void store4(T *p, int n, const float *v) {
    if (n == 4) {
        T w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) Elem<T>::store(w, j, v[j]);
        __builtin_memcpy(p, w, sizeof(w));
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < n) Elem<T>::store(p, j, v[j]);
}

// Values (r, c .. c + 3) of what is made orthogonal, zeros outside.
__device__ __forceinline__ void source4(const Source &s, int mat, int64_t r, int64_t c, float *v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = 0.f;
    if (r >= s.rows || c >= s.cols) return;
    const int64_t i = r * s.cols + c, end = (r + 1) * s.cols;
    if (s.update) {
        load4(s.t.momentum[mat], i, end, v);
        if (!s.nesterov) return;
        float g[4];
        load4(s.t.grad[mat], i, end, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = g[j] + s.beta * v[j];
    } else if (s.dense) {
        const int64_t at = (s.first + mat) * s.x.s0;
        if (s.bf16) load4((const bf16_t *)s.x.data + at, i, end, v);
        else load4((const float *)s.x.data + at, i, end, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < s.cols) v[j] = source_at(s, mat, r, c + j);
    }
}

// Sums of squares in 64 bits: of a part of a dense matrix's values, or of every so-manieth row of
// another; an update's momentum first takes the gradient.
template <typename T, bool UPDATE> __global__ void __launch_bounds__(256) ns_squares(Source s, double *partial) {
    __shared__ double red[4];
    const int mat = blockIdx.y;
    double sum = 0;
    if (UPDATE || s.dense) {
        const int64_t n = (int64_t)s.rows * s.cols, per = ((n + s.parts - 1) / s.parts + 3) & ~(int64_t)3;
        const int64_t end = min(n, (blockIdx.x + 1) * per);
        const T *x = UPDATE ? nullptr : (const T *)s.x.data + (s.first + mat) * s.x.s0;
        for (int64_t i = blockIdx.x * per + 4 * (int64_t)threadIdx.x; i < end; i += 4 * 256) {
            float v[4];
            if constexpr (UPDATE) {
                float g[4], m[4];
                load4(s.t.grad[mat], i, end, g);
                load4(s.t.momentum[mat], i, end, m);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m[j] = s.beta * m[j] + g[j];
                    v[j] = s.nesterov ? g[j] + s.beta * m[j] : m[j];
                }
                if (i + 4 <= end) {
                    __builtin_memcpy(s.t.momentum[mat] + i, m, sizeof(m));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (i + j < end) s.t.momentum[mat][i + j] = m[j];
                        else v[j] = 0.f;
                }
            } else {
                load4(x, i, end, v);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) sum += (double)v[j] * v[j];
        }
    } else {
        for (int64_t r = blockIdx.x; r < s.rows; r += s.parts)
            for (int64_t c = threadIdx.x; c < s.cols; c += 256) {
                const double v = source_at(s, mat, r, c);
                sum += v * v;
            }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[mat * kParts + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// U / (|U| + epsilon) times scale, split, in both orientations.  One workgroup a 64 x 64 tile of U.
template <bool F32>
__global__ void __launch_bounds__(kSplitThreads) ns_split(Source s, const double *partial, double epsilon,
                                                          double scale, Split by_rows, Split by_cols, int64_t step) {
    constexpr int N = 64 * 16 / kSplitThreads;  // fours of a thread
    __shared__ float tile[64][65];  // by fours, by eights and down columns over all banks
    __shared__ double red[kSplitThreads / 64];
    const int mat = blockIdx.y, across = by_rows.cols / 64;
    const int r0 = (int)(blockIdx.x / across) * 64, c0 = (int)(blockIdx.x % across) * 64;
    by_rows.data += mat * step, by_cols.data += mat * step;
    float v[N][4];  // on their way while the squares are summed
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = threadIdx.x + k * kSplitThreads;
        source4(s, mat, r0 + (i >> 4), c0 + (i & 15) * 4, v[k]);
    }
    double sum = 0;
    for (int i = threadIdx.x; i < s.parts; i += kSplitThreads) sum += partial[mat * kParts + i];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kSplitThreads / 64; ++w) sum += red[w];
    const double by = scale / (sqrt(sum) + epsilon);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = threadIdx.x + k * kSplitThreads;
#pragma unroll
        for (int j = 0; j < 4; ++j) tile[i >> 4][(i & 15) * 4 + j] = (float)(v[k][j] * by);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 8; i += kSplitThreads) {
        const int a = i >> 3, b = (i & 7) * 8;
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = tile[a][b + j];
        store_split<F32>(by_rows, r0 + a, c0 + b, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = tile[b + j][a];
        store_split<F32>(by_cols, c0 + a, r0 + b, w);
    }
}

// ---- products -------------------------------------------------------------------------------

enum Mode { GRAM, POLY, NEXT, LAST };

struct GemmArgs {
    Split l, r;                // operands: C = L R^T
    Split out, out_t;          // GRAM, POLY: out; NEXT: both
    int64_t l_step, r_step, out_step;  // bytes between matrices
    int tiles_i, tiles_j, tiles;  // tiles of a matrix
    int whole, parts;          // tiles made at once; parts of the others' sums
    float *partial;            // [tile that is not whole][part][T][T]
    int k, stages;             // columns of the operands, and their chunks that are not padding
    float scale;               // of the accumulators
    double a, b, c;            // POLY: of the identity, of A and of the accumulators, in the result's scale
    int whole_poly;            // GRAM: A is one tile, whose polynomial is made at once
    // LAST
    int rows, cols, tall, bf16, first;
    float decay, rate;         // update: param = decay param - rate result
    int update;
    void *result;
    Tensors t;
};

// Tiles of a result.  Four waves multiply, four bring the operands to LDS (two waves do not issue the
// loads as fast as a stage is used: 4096 x 4096 takes 3 % longer).  At 128 two workgroups share a CU, one
// multiplies while the other waits: 0.6 us a stage of each, 0.65 alone; more stages and one workgroup are
// 5 % slower.  At 64 a stage takes 0.2 us, at 32 0.115: the L2's rate into LDS of a CU.  So where 64 leaves
// CUs idle 32 spreads the same sums over four times as many: a product of 512 x 512 takes 6 to 7 us for 8,
// all of it 106 us for 135; 8 of them 284 us for 207.
template <int T> struct Tile {
    static constexpr int WAVES = 4, LOADS = 4, THREADS = 64 * (WAVES + LOADS);
    static constexpr int STAGE = 2 * T * 128;     // bytes: a chunk of T rows of both operands
    static constexpr int STAGES = T == 128 ? 2 : T == 64 ? 4 : 8;
    static constexpr int OPS = STAGE / 1024 / LOADS;  // loads of a wave and stage
    static constexpr int BYTES = STAGES * STAGE;
    static constexpr int F = T / 32;              // 16-row fragments of a wave, 2 x 2 waves
    static_assert((STAGES - 1) * OPS <= 63, "loads on their way fit the memory counter");
    static_assert(BYTES >= T * T * 4 && BYTES <= 160 * 1024, "the result's tile in the stages' place");
};

constexpr int wait_vm(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }
constexpr int kWaitLds = 15 | (3 << 14) | (7 << 4);

__device__ __forceinline__ void stage_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ f32x4 four(const f16x8 &v) { return __builtin_bit_cast(f32x4, v); }

// The stored 16-byte piece of piece x of row r: rows of 128 bytes, 64 banks of 4.
__device__ __forceinline__ int swizzle(int r, int x) { return x ^ ((r >> 1) & 7); }

constexpr int kRowsAtOnce = 4;

// Float (i, j) of a result's tile in LDS: the fours of a row are exchanged by the row, so that writes of
// accumulators (rows 4 apart), reads along rows and reads down columns all spread over the 64 banks.
template <int T> __device__ __forceinline__ int at_tile(int i, int j) {
    const int q = i >> 3;
    const int f = ((q & 1) << 2 | (q & 2) << 2 | (q & 4) >> 2 | (q & 8) >> 2) ^ ((i & 4) << 1);
    return i * T + (j ^ (f << 2 & (T - 1)));
}

// Tile (i, j) of a tile index: all ni x nj, or, for symmetric results, those with i <= j.  Rows of
// tiles go by kRowsAtOnce, columns inside, so that neighbours share both operands.
template <bool SYM> __device__ __forceinline__ void tile_of(int t, int ni, int nj, int *i, int *j) {
    constexpr int R = kRowsAtOnce;
    if (!SYM) {
        const int q = t / (R * nj), rows = min(R, ni - q * R), u = t - q * R * nj;
        *i = q * R + u % rows, *j = u / rows;
        return;
    }
    int q = 0;  // rows q R .. + rows: a triangle of them, then whole columns
    for (;; ++q) {
        const int rows = min(R, ni - q * R), n = rows * (rows + 1) / 2 + rows * (ni - q * R - rows);
        if (t < n) {
            const int corner = rows * (rows + 1) / 2;
            if (t < corner) {
                int c = 0;
                while ((c + 1) * (c + 2) / 2 <= t) ++c;
                *j = q * R + c, *i = q * R + t - c * (c + 1) / 2;
            } else {
                *i = q * R + (t - corner) % rows, *j = q * R + rows + (t - corner) / rows;
            }
            return;
        }
        t -= n;
    }
}

// The polynomial of a tile S that is all of A, in its place: sums in 64 bits, rounded once.  This saves a
// launch of 3 us for 0.3 of work.
template <int T> __device__ __forceinline__ void tile_poly(const GemmArgs &p, float *S, int threads) {
    constexpr int MOST = 2;  // pairs of a thread
    float v[MOST][2];
#pragma unroll
    for (int n = 0; n < MOST; ++n) {
        const int i = threadIdx.x + n * threads, a = i / (T / 2), b = i % (T / 2) * 2;
        if (i >= T * T / 2) break;
        double u0 = 0, u1 = 0;
#pragma unroll 8
        for (int k = 0; k < T; ++k) {
            const double l = S[at_tile<T>(a, k)];
            const float *r = S + at_tile<T>(k, b);
            u0 = fma(l, (double)r[0], u0), u1 = fma(l, (double)r[1], u1);
        }
        const float *m = S + at_tile<T>(a, b);
        v[n][0] = (float)(p.c * u0 + p.b * m[0] + (a == b ? p.a : 0.0));
        v[n][1] = (float)(p.c * u1 + p.b * m[1] + (a == b + 1 ? p.a : 0.0));
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < MOST; ++n) {
        const int i = threadIdx.x + n * threads, a = i / (T / 2), b = i % (T / 2) * 2;
        if (i >= T * T / 2) break;
        float *m = S + at_tile<T>(a, b);
        m[0] = v[n][0], m[1] = v[n][1];
    }
    __syncthreads();
}

// What a product makes of its tile S at (I, J): the next operand, in both orientations where mirror is
// set, or the results.
template <int T, Mode MODE, bool F32>
__device__ __forceinline__ void finish_tile(const GemmArgs &p, int mat, int I, int J, bool mirror, float *S,
                                            int threads) {
    if constexpr (MODE == LAST) {
        const int mr = p.tall ? J : I, mc = p.tall ? I : J;
        for (int i = threadIdx.x; i < T * T / 4; i += threads) {
            const int a = i / (T / 4), b = i % (T / 4) * 4;
            const int64_t r = mr + a, c = mc + b;
            const int n = (int)min((int64_t)4, p.cols - c);  // columns that the result has
            if (r >= p.rows || n <= 0) continue;
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = S[p.tall ? at_tile<T>(b + j, a) : at_tile<T>(a, b + j)];
            const int64_t o = r * p.cols + c;
            if (p.update) {
                float *q = p.t.param[mat] + o, old[4];
                load4(q, 0, n, old);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = p.decay * old[j] - p.rate * v[j];
                store4(q, n, v);
            } else {
                const int64_t at = (int64_t)(p.first + mat) * p.rows * p.cols + o;
                if (p.bf16) store4((bf16_t *)p.result + at, n, v);
                else store4((float *)p.result + at, n, v);
            }
        }
        return;
    }
    Split out = p.out, out_t = MODE == NEXT ? p.out_t : p.out;
    out.data += mat * p.out_step, out_t.data += mat * p.out_step;
    if constexpr (MODE == POLY) {
        Split A = p.l;
        A.data += mat * p.l_step;
        for (int i = threadIdx.x; i < T * T / 8; i += threads) {
            const int a = i / (T / 8), b = i % (T / 8) * 8;
            float v[8];
            load_split<F32>(A, I + a, J + b, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // rounded once
                float &u = S[at_tile<T>(a, b + j)];
                u = (float)(p.c * u + p.b * v[j] + (I + a == J + b + j ? p.a : 0.0));
            }
        }
        __syncthreads();
    }
    if constexpr (MODE == GRAM && F32) {
        if (p.whole_poly) tile_poly<T>(p, S, threads);
    }
    for (int i = threadIdx.x; i < T * T / 8; i += threads) {
        const int a = i / (T / 8), b = i % (T / 8) * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = S[at_tile<T>(a, b + j)];
        store_split<F32>(out, I + a, J + b, v);
        if (mirror) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = S[at_tile<T>(b + j, a)];
            store_split<F32>(out_t, J + a, I + b, v);
        }
    }
}

template <int T, Mode MODE, bool F32> __global__ void __launch_bounds__(Tile<T>::THREADS) ns_product(GemmArgs p) {
    using C = Tile<T>;
    constexpr int F = C::F;
    __shared__ __align__(1024) char lds[C::BYTES];
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    // Neighbouring tiles to one XCD (workgroups go to the eight in turn): first the whole tiles, behind them
    // those that are made in parts of the sum.
    const bool part = (int)blockIdx.x >= p.whole;
    const int first = part ? p.whole : 0, b = blockIdx.x - first;
    const int total = part ? (int)gridDim.x - p.whole : p.whole, x = b & 7, full = total >> 3, more = total & 7;
    const int piece = (b >> 3) + x * full + min(x, more);
    int at = piece, stages = p.stages, from = 0;
    if (part) {
        const int n = piece % p.parts;
        at = p.whole + piece / p.parts;
        from = (int)((int64_t)stages * n / p.parts);
        stages = (int)((int64_t)stages * (n + 1) / p.parts) - from;
    }
    const int mat = at / p.tiles;
    int ti, tj;
    tile_of<SYM>(at % p.tiles, p.tiles_i, p.tiles_j, &ti, &tj);
    const int I = ti * T, J = tj * T;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
    // of the pairs' first terms, and, where registers allow it, of the small products by themselves; a float64
    // accumulator i of a lane is of row 4 i + lane / 16, a float32 one of row 4 (lane / 16) + i
    constexpr bool APART = T <= 64 && !F32;
    f32x4 acc[F][F], low[APART ? F : 1][APART ? F : 1];
    f64x4 sum[F32 ? F : 1][F32 ? F : 1];

    if (w >= C::WAVES) {  // loads
        typedef __attribute__((address_space(1))) const void *gptr;
        typedef __attribute__((address_space(3))) void *lptr;
        const int pw = w - C::WAVES;
        // An operation brings 8 rows of a chunk of the stacked operands.  Where it reads is a uniform
        // address and one of two offsets of the lane.
        const uint32_t row = (uint32_t)row_bytes(p.k);
        const uint32_t lane0 = (l >> 3) * row + swizzle(l >> 3, l & 7) * 16;
        const uint32_t lane8 = (l >> 3) * row + swizzle(8 + (l >> 3), l & 7) * 16;
        const char *left = p.l.data + mat * p.l_step + (int64_t)I * row + from * 128;
        const char *right = p.r.data + mat * p.r_step + (int64_t)J * row + from * 128;
        auto issue = [&](int s) {
            char *slot = lds + (s % C::STAGES) * C::STAGE;
#pragma unroll
            for (int i = 0; i < C::OPS; ++i) {
                const int at = C::LOADS * i + pw, r0 = 8 * at;
                const char *src = (r0 < T ? left + (int64_t)r0 * row : right + (int64_t)(r0 - T) * row) + s * 128;
                __builtin_amdgcn_global_load_lds((gptr)(src + (r0 & 8 ? lane8 : lane0)), (lptr)(slot + at * 1024), 16,
                                                 0, 0);
            }
        };
        for (int s = 0; s < C::STAGES - 1 && s < stages; ++s) issue(s);
        for (int s = 0; s < stages; ++s) {
            if (s + C::STAGES - 2 < stages) __builtin_amdgcn_s_waitcnt(wait_vm((C::STAGES - 2) * C::OPS));
            else __builtin_amdgcn_s_waitcnt(wait_vm(0));
            stage_barrier();  // stage s has landed, stage s - 1 is read
            if (s + C::STAGES - 1 < stages) issue(s + C::STAGES - 1);
        }
    } else {
        const int wi = (w >> 1) * (T / 2), wj = (w & 1) * (T / 2);
        const int n = l & 15, g = l >> 4;
#pragma unroll
        for (int a = 0; a < F; ++a)
#pragma unroll
            for (int b = 0; b < F; ++b) {
                acc[a][b] = zero4();
                if constexpr (APART) low[a][b] = zero4();
                if constexpr (F32) sum[a][b] = f64x4{0., 0., 0., 0.};
            }
        for (int s = 0; s < stages; ++s) {
            __builtin_amdgcn_s_waitcnt(kWaitLds);  // stage s - 1 is read
            stage_barrier();
            const char *L = lds + (s % C::STAGES) * C::STAGE, *R = L + T * 128;
            f16x8 rh[F], rl[F];
#pragma unroll
            for (int b = 0; b < F; ++b) {
                const int row = wj + 16 * b + n;
                rh[b] = *reinterpret_cast<const f16x8 *>(R + row * 128 + swizzle(row, g) * 16);
                rl[b] = *reinterpret_cast<const f16x8 *>(R + row * 128 + swizzle(row, g + 4) * 16);
            }
#pragma unroll
            for (int a = 0; a < F; ++a) {
                const int row = wi + 16 * a + n;
                const f16x8 lh = *reinterpret_cast<const f16x8 *>(L + row * 128 + swizzle(row, g) * 16);
                const f16x8 ll = *reinterpret_cast<const f16x8 *>(L + row * 128 + swizzle(row, g + 4) * 16);
                if constexpr (F32) {
                    // the same pieces hold 4 + 4 columns of float32
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int b = 0; b < F; ++b) {
                            f64x4 &to = sum[a][b];
                            to = __builtin_amdgcn_mfma_f64_16x16x4f64((double)four(lh)[e], (double)four(rh[b])[e], to,
                                                                      0, 0, 0);
                            to = __builtin_amdgcn_mfma_f64_16x16x4f64((double)four(ll)[e], (double)four(rl[b])[e], to,
                                                                      0, 0, 0);
                        }
                    continue;
                }
                // sums of different fragments between those of one
#pragma unroll
                for (int b = 0; b < F; ++b)
                    acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lh, rh[b], acc[a][b], 0, 0, 0);
#pragma unroll
                for (int b = 0; b < F; ++b) {
                    f32x4 &to = APART ? low[a][b] : acc[a][b];
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(lh, rl[b], to, 0, 0, 0);
                }
#pragma unroll
                for (int b = 0; b < F; ++b) {
                    f32x4 &to = APART ? low[a][b] : acc[a][b];
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(ll, rh[b], to, 0, 0, 0);
                }
            }
        }
    }
    // The tile through LDS, so that whole pieces are written in either orientation.
    __syncthreads();
    float *S = reinterpret_cast<float *>(lds);
    if (w < C::WAVES) {
        const int wi = (w >> 1) * (T / 2), wj = (w & 1) * (T / 2);
#pragma unroll
        for (int a = 0; a < F; ++a)
#pragma unroll
            for (int b = 0; b < F; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    int r = 4 * (l >> 4) + i;
                    float v = acc[a][b][i];
                    if constexpr (APART) v += low[a][b][i];
                    if constexpr (F32) r = 4 * i + (l >> 4), v = (float)sum[a][b][i];
                    S[at_tile<T>(wi + 16 * a + r, wj + 16 * b + (l & 15))] = v * p.scale;
                }
    }
    __syncthreads();
    if (part) {
        float4 *to = reinterpret_cast<float4 *>(p.partial + (int64_t)piece * T * T);
        for (int i = threadIdx.x; i < T * T / 4; i += C::THREADS)
            to[i] = *reinterpret_cast<const float4 *>(S + at_tile<T>(i / (T / 4), i % (T / 4) * 4));
        return;
    }
    finish_tile<T, MODE, F32>(p, mat, I, J, !SYM || ti != tj, S, C::THREADS);
}

// The sums of the tiles that were made in parts, in order, at most 64 x 64 of a tile each, four values a
// thread: a wave waits for its loads two times, not eight as with a quarter of the threads.
constexpr int join_side(int tile) { return tile < 64 ? tile : 64; }
constexpr int join_threads(int tile) { return join_side(tile) * join_side(tile) / 4; }

template <int T, Mode MODE, bool F32> __global__ void __launch_bounds__(join_threads(T)) ns_join(GemmArgs p) {
    constexpr int Q = join_side(T), N = T / Q, THREADS = join_threads(T);
    __shared__ __align__(16) float S[Q * Q];
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    const int n = blockIdx.x / (N * N), qi = blockIdx.x / N % N * Q, qj = blockIdx.x % N * Q;
    const int at = p.whole + n;
    int ti, tj;
    tile_of<SYM>(at % p.tiles, p.tiles_i, p.tiles_j, &ti, &tj);
    const int a = threadIdx.x / (Q / 4), b = threadIdx.x % (Q / 4) * 4;
    const float *from = p.partial + (int64_t)n * p.parts * T * T + (qi + a) * T + qj + b;
    double sum[4] = {0, 0, 0, 0};
#pragma unroll 8
    for (int k = 0; k < p.parts; ++k) {
        const float4 v = *reinterpret_cast<const float4 *>(from + (int64_t)k * T * T);
        sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
    }
    *reinterpret_cast<float4 *>(S + at_tile<Q>(a, b)) =
        make_float4((float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]);
    __syncthreads();
    finish_tile<Q, MODE, F32>(p, at / p.tiles, ti * T + qi, tj * T + qj, !SYM || ti != tj, S, THREADS);
}

// ---- host -----------------------------------------------------------------------------------------

struct Plan {
    int tile[LAST + 1];
    bool f32;                    // operands as float32
    int64_t m, n;                // padded
    int64_t x_bytes, xt_bytes, a_bytes;  // of one matrix: X, its transpose, A or B
    int64_t matrix_bytes;
    int group;
};

int check_matrices(const gdn2_matrices_shape *s) {
    if (!s) return fail(GDN2_ERR_ARGUMENT, "shape is null");
    if (s->count < 0 || s->rows < 1 || s->cols < 1)
        return fail(GDN2_ERR_SHAPE, "count must be >= 0, rows and cols nonempty");
    if (s->count > 0x7FFFFFFF || s->rows > (1 << 24) || s->cols > (1 << 24) || s->rows * s->cols > (1 << 30))
        return fail(GDN2_ERR_SHAPE, "too many matrices, rows or columns (2^30 values of a matrix at most)");
    return ok();
}

int64_t padded(int64_t n, int64_t t) { return (n + t - 1) / t * t; }

constexpr int kAtOnce = 512;  // workgroups of large tiles that the card holds

// How the tiles of a product are made: those that fill the card once or more at once, the others, if it
// pays, in parts of their sums that fill it once more, which another kernel joins.  Of several matrices all
// tiles are made alike, so that equal matrices have equal results.
struct Way {
    int tile, parts;
    int64_t whole;
    double time;  // about, in us: a CU's tiles one after another, each with its stages and its result, and the
                  // launch, from the figures at Tile; a part of 64 KB is written and read in 16 ns; a join has
                  // its launch in it, and at 128 more than it takes with the threads it has now (7 to 8 and that)
};

Way way_of(int tile, int64_t tiles, int64_t matrices, int64_t stages, bool f32) {
    const bool small = tile < 128;
    const double stage = f32 ? 0.25 : tile == 32 ? 0.115 : tile == 64 ? 0.2 : 0.6;
    const double result = tile == 32 ? 0.5 : tile == 64 ? 1 : 2, part = tile == 32 ? 0.001 : tile == 64 ? 0.004 : 0.016;
    const double launch = small ? 4 : 5, join = small ? 4.5 : 13;
    // so many workgroups, one or, at 128, two to a CU at once
    auto takes = [&](int64_t n, int64_t chunks) {
        if (!small && n <= 256) return 0.65 * chunks + result;
        return (double)((n + 255) / 256) * (stage * chunks + result);
    };
    tiles *= matrices;
    Way best = {tile, 1, tiles, takes(tiles, stages) + launch};
    // Small tiles all in parts or none: with a rest in parts 1600 x 2100 took 537 us for 509.
    const int64_t most = !small && matrices == 1 ? tiles / kAtOnce * kAtOnce : 0;
    for (int64_t whole = 0;; whole = most) {
        const int64_t rest = tiles - whole;
        const int64_t most_parts = rest ? min(min((int64_t)16, kAtOnce / rest), stages / (small ? 2 : 4)) : 0;
        for (int parts = 2; parts <= most_parts; ++parts) {
            const double time = (whole ? takes(whole, stages) : 0) + takes(rest * parts, (stages + parts - 1) / parts) +
                                launch + join + part * (double)(rest * parts);
            if (time < best.time) best = {tile, parts, whole, time};
        }
        if (whole == most) return best;
    }
}

// Tiles of a result that hold rows and columns of the matrices; what lies behind them is never read as a
// column of an operand.
int tiles_of(int64_t n, int t) { return (int)((n + t - 1) / t); }

// Each product takes the tile that way_of prefers; sizes are padded to 64 or to the larger tile.
Plan plan_of(const gdn2_matrices_shape *s) {
    const int64_t m = s->rows < s->cols ? s->rows : s->cols, n = s->rows < s->cols ? s->cols : s->rows;
    const int64_t count = s->count < kGroup ? s->count : kGroup;
    Plan best{};
    double least = 0;
    for (int pad = 64; pad <= 128; pad += 64) {
        Plan p{};
        p.f32 = m <= 64;
        p.m = padded(m, pad), p.n = padded(n, pad);
        double total = 0;
        for (int mode = GRAM; mode <= NEXT; ++mode) {
            double time = 0;
            for (int t = 32; t <= (p.f32 ? 32 : pad); t *= 2) {
                const int64_t ti = tiles_of(m, t), tiles = mode == NEXT ? ti * tiles_of(n, t) : ti * (ti + 1) / 2;
                const Way w = way_of(t, tiles, count, tiles_of(mode == GRAM ? n : m, kChunk), p.f32);
                if (t == 32 || w.time < time) time = w.time, p.tile[mode] = t;
            }
            total += time;
        }
        if (pad == 64 || total < least) best = p, least = total;
    }
    best.tile[LAST] = best.tile[NEXT];
    best.x_bytes = best.m * row_bytes(best.n), best.xt_bytes = best.n * row_bytes(best.m);
    best.a_bytes = best.m * row_bytes(best.m);
    best.matrix_bytes = 2 * (best.x_bytes + best.xt_bytes + best.a_bytes);
    int64_t g = kMostBytes / best.matrix_bytes;
    if (g > count) g = count;
    best.group = g < 1 ? 1 : (int)g;
    return best;
}

// Parts of a matrix's squares: 1024 values each, as far as they go.
int parts_of(const gdn2_matrices_shape *s) {
    const int64_t n = (s->rows * s->cols + 1023) / 1024;
    return n > kParts ? kParts : (int)n;
}

constexpr size_t kPartialBytes = (size_t)kAtOnce * 128 * 128 * sizeof(float);

size_t workspace_of(const Plan &p) {
    const bool large = p.tile[GRAM] == 128 || p.tile[POLY] == 128 || p.tile[NEXT] == 128;
    return (size_t)p.group * p.matrix_bytes + (size_t)p.group * kParts * sizeof(double) +
           (large ? kPartialBytes : kPartialBytes / 4);
}

// The largest |a t + b t^3 + c t^5| for t in [0, s], and the largest |a + b u + c u^2| for u in [0, s^2].
struct Bounds {
    double x, poly;
};

Bounds bounds_of(const double *k, double s) {
    const double a = k[0], b = k[1], c = k[2];
    auto value = [&](double t) { return fabs(t * (a + t * t * (b + c * t * t))); };
    auto poly = [&](double u) { return fabs(a + u * (b + c * u)); };
    Bounds r = {value(s), fmax(fabs(a), poly(s * s))};
    auto turn = [&](double u) {  // where the derivative in t is zero: a + 3 b u + 5 c u^2 = 0, u = t^2
        if (u > 0 && u < s * s) r.x = fmax(r.x, value(sqrt(u)));
    };
    if (c != 0) {
        const double d = 9 * b * b - 20 * a * c;
        if (d >= 0) turn((-3 * b + sqrt(d)) / (10 * c)), turn((-3 * b - sqrt(d)) / (10 * c));
        const double v = -b / (2 * c);
        if (v > 0 && v < s * s) r.poly = fmax(r.poly, poly(v));
    } else if (b != 0) {
        turn(-a / (3 * b));
    }
    return r;
}

// The power of two that brings a bound to 2^13 .. 2^14.
double power_for(double bound) {
    int e;
    frexp(bound > 1e-30 ? bound : 1e-30, &e);  // bound < 2^e
    return ldexp(1.0, 14 - e);
}

int check_steps(int steps, const double *k, float epsilon) {
    if (steps < 1 || steps > 100) return fail(GDN2_ERR_ARGUMENT, "steps must be 1 to 100");
    if (!k) return fail(GDN2_ERR_ARGUMENT, "coefficients is null");
    if (!(epsilon >= 0) || !(epsilon <= FLT_MAX)) return fail(GDN2_ERR_ARGUMENT, "epsilon must be >= 0 and finite");
    double s = 1;
    for (int i = 0; i < steps; ++i) {
        const Bounds b = bounds_of(k, s);
        s = b.x * 1.001;
        if (!(s < 1e9) || !(b.poly < 1e9))
            return fail(GDN2_ERR_ARGUMENT, "coefficients make the values grow past 1e9 in step %d", i + 1);
    }
    return ok();
}

template <int T, Mode MODE, bool F32> void launch_tiles(const GemmArgs &a, const Way &w, int64_t rest, hipStream_t st) {
    const dim3 grid((unsigned)(w.whole + rest * w.parts));
    hipLaunchKernelGGL((ns_product<T, MODE, F32>), grid, dim3(Tile<T>::THREADS), 0, st, a);
    constexpr int N = T / join_side(T);
    if (rest)
        hipLaunchKernelGGL((ns_join<T, MODE, F32>), dim3((unsigned)(N * N * rest)), dim3(join_threads(T)), 0, st, a);
}

template <Mode MODE> void launch_product(const GemmArgs &a, const Way &w, bool f32, int64_t rest, hipStream_t st) {
    if (f32) launch_tiles<32, MODE, true>(a, w, rest, st);
    else if (w.tile == 32) launch_tiles<32, MODE, false>(a, w, rest, st);
    else if (w.tile == 64) launch_tiles<64, MODE, false>(a, w, rest, st);
    else launch_tiles<128, MODE, false>(a, w, rest, st);
}

// All products of one group of matrices; last holds the fields of the last product's results.
void run_group(const Plan &p, const Source &src, int count, int steps, const double *k, float epsilon,
               const GemmArgs &last, char *ws, hipStream_t st) {
    const bool tall = src.rows > src.cols;
    double *partial = (double *)(ws + (size_t)p.group * p.matrix_bytes);
    // of the first matrix; the others follow at matrix_bytes
    Split X[2], XT[2];
    for (int i = 0; i < 2; ++i) {
        X[i] = {ws + i * (p.x_bytes + p.xt_bytes), (int)p.n};
        XT[i] = {X[i].data + p.x_bytes, (int)p.m};
    }
    const Split A = {ws + 2 * (p.x_bytes + p.xt_bytes), (int)p.m}, B = {A.data + p.a_bytes, (int)p.m};
    // float32 operands need no powers
    auto power = [&](double bound) { return p.f32 ? 1.0 : power_for(bound); };
    const int m = tall ? src.cols : src.rows, n = tall ? src.rows : src.cols;
    double s = 1, sx = power(s);
    const dim3 parts(src.parts, count), threads(256);
    if (src.update) hipLaunchKernelGGL((ns_squares<float, true>), parts, threads, 0, st, src, partial);
    else if (src.bf16) hipLaunchKernelGGL((ns_squares<bf16_t, false>), parts, threads, 0, st, src, partial);
    else hipLaunchKernelGGL((ns_squares<float, false>), parts, threads, 0, st, src, partial);
    const int64_t pr = tall ? p.n : p.m, pc = tall ? p.m : p.n;
    hipLaunchKernelGGL((p.f32 ? ns_split<true> : ns_split<false>), dim3((unsigned)(pr / 64 * (pc / 64)), count),
                       dim3(kSplitThreads), 0, st, src, partial, (double)epsilon, sx, tall ? XT[0] : X[0],
                       tall ? X[0] : XT[0], p.matrix_bytes);
    for (int i = 0; i < steps; ++i) {
        const Split &x = X[i & 1], &xt = XT[i & 1];
        const Bounds b = bounds_of(k, s);
        const double sa = power(s * s), sb = power(b.poly), next = b.x * 1.001;
        GemmArgs g = last;
        g.partial = (float *)(partial + (size_t)p.group * kParts);
        g.l_step = g.r_step = g.out_step = p.matrix_bytes;
        auto run = [&](Mode mode) {
            const int t = p.tile[mode], ti = tiles_of(m, t), tn = tiles_of(n, t);
            g.tiles_i = ti, g.tiles_j = mode >= NEXT ? tn : ti;
            g.tiles = mode >= NEXT ? ti * tn : ti * (ti + 1) / 2;
            // as for a whole group, also where the last one has fewer matrices
            Way w = way_of(t, g.tiles, p.group, g.stages, p.f32);
            const int64_t tiles = (int64_t)g.tiles * count;
            if (p.group > 1) w.whole = w.parts > 1 ? 0 : tiles;
            g.whole = (int)w.whole, g.parts = w.parts;
            switch (mode) {
                case GRAM: launch_product<GRAM>(g, w, p.f32, tiles - w.whole, st); break;
                case POLY: launch_product<POLY>(g, w, p.f32, tiles - w.whole, st); break;
                case NEXT: launch_product<NEXT>(g, w, p.f32, tiles - w.whole, st); break;
                default: launch_product<LAST>(g, w, p.f32, tiles - w.whole, st);
            }
        };
        // A of one tile: B at once
        g.whole_poly = p.f32 && m <= 32;
        g.a = k[0] * sb, g.b = k[1] * sb / sa, g.c = k[2] * sb / (sa * sa);
        g.l = g.r = x, g.out = g.whole_poly ? B : A;
        g.k = (int)p.n, g.stages = tiles_of(n, kChunk);
        g.scale = (float)(sa / (sx * sx));
        run(GRAM);
        g.l = g.r = A, g.out = B, g.k = (int)p.m, g.stages = tiles_of(m, kChunk);
        g.scale = 1;
        if (!g.whole_poly) run(POLY);
        g.l = B, g.r = xt, g.out = X[1 - (i & 1)], g.out_t = XT[1 - (i & 1)];
        const double to = i + 1 < steps ? power(next) : 1;
        g.scale = (float)(to / (sb * sx));
        run(i + 1 < steps ? NEXT : LAST);
        s = next, sx = to;
    }
}

int check_workspace(const void *p, size_t have, size_t need) {
    if (!p || have < need) return fail(GDN2_ERR_WORKSPACE, "workspace is too small: %zu bytes needed", need);
    if ((uintptr_t)p & 15) return fail(GDN2_ERR_ARGUMENT, "workspace must be 16-byte aligned");
    return ok();
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_orthogonalize_workspace_bytes(const gdn2_matrices_shape *shape) {
    if (check_matrices(shape)) return 0;
    return workspace_of(plan_of(shape));
}

int gdn2_orthogonalize(const gdn2_matrices_shape *shape, const gdn2_view *x, void *result, int steps,
                       const double *coefficients, float epsilon, void *workspace, size_t workspace_bytes,
                       void *stream) {
    GDN2_TRY(check_matrices(shape));
    GDN2_TRY(check_view(x, "x", -1, shape->count == 0));
    GDN2_TRY(check_steps(steps, coefficients, epsilon));
    if (shape->count == 0) return ok();
    if (!result) return fail(GDN2_ERR_ARGUMENT, "result must be non-null");
    const Plan p = plan_of(shape);
    GDN2_TRY(check_workspace(workspace, workspace_bytes, workspace_of(p)));
    Source s{};
    s.x = make_view(x), s.bf16 = x->dtype == GDN2_BF16;
    s.rows = (int)shape->rows, s.cols = (int)shape->cols;
    s.dense = s.x.s2 == 1 && s.x.s1 == s.cols;
    GemmArgs last{};
    last.rows = s.rows, last.cols = s.cols, last.tall = s.rows > s.cols, last.bf16 = s.bf16;
    last.result = result;
    s.parts = parts_of(shape);
    for (int64_t i = 0; i < shape->count; i += p.group) {
        s.first = last.first = (int)i;
        const int64_t left = shape->count - i;
        run_group(p, s, (int)(left < p.group ? left : p.group), steps, coefficients, epsilon, last,
                  (char *)workspace, (hipStream_t)stream);
    }
    return launch_status(hipGetLastError(), "gdn2_orthogonalize");
}

int gdn2_muon_update(const gdn2_matrices_shape *shape, const gdn2_muon_tensor *tensors, float lr, float beta,
                     int nesterov, float decay, int steps, const double *coefficients, float epsilon,
                     void *workspace, size_t workspace_bytes, void *stream) {
    GDN2_TRY(check_matrices(shape));
    GDN2_TRY(check_steps(steps, coefficients, epsilon));
    if (shape->count == 0) return ok();
    if (!tensors) return fail(GDN2_ERR_ARGUMENT, "tensors is null");
    for (int64_t i = 0; i < shape->count; ++i)
        if (!tensors[i].param || !tensors[i].grad || !tensors[i].momentum)
            return fail(GDN2_ERR_ARGUMENT, "tensor %lld has a null pointer", (long long)i);
    const Plan p = plan_of(shape);
    GDN2_TRY(check_workspace(workspace, workspace_bytes, workspace_of(p)));
    Source s{};
    s.update = 1, s.nesterov = nesterov != 0, s.beta = beta;
    s.rows = (int)shape->rows, s.cols = (int)shape->cols;
    GemmArgs last{};
    last.rows = s.rows, last.cols = s.cols, last.tall = s.rows > s.cols, last.update = 1;
    last.decay = 1.f - lr * decay;
    s.parts = parts_of(shape);
    last.rate = lr * sqrtf(s.rows > s.cols ? (float)s.rows / (float)s.cols : 1.f);
    for (int64_t i = 0; i < shape->count; i += p.group) {
        const int64_t left = shape->count - i;
        const int n = (int)(left < p.group ? left : p.group);
        for (int j = 0; j < n; ++j) {
            s.t.param[j] = tensors[i + j].param;
            s.t.grad[j] = tensors[i + j].grad;
            s.t.momentum[j] = tensors[i + j].momentum;
        }
        last.t = s.t;
        run_group(p, s, n, steps, coefficients, epsilon, last, (char *)workspace, (hipStream_t)stream);
    }
    return launch_status(hipGetLastError(), "gdn2_muon_update");
}

}  // extern "C"
