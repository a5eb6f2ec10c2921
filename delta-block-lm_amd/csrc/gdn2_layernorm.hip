// Layer norm over rows on gfx950: forward, and backward with the weight's and bias's gradients.
//
//   y = w (x - m) r + b,  m = mean x,  r = 1 / sqrt(mean (x - m)^2 + epsilon)
//   with xh = (x - m) r and c = dy w:  dx = r (c - mean c - xh mean(c xh)),
//   dw = sum over rows of dy xh,  db = sum over rows of dy.
//
// Bound by memory: x is read once and kept in registers between the statistics (the variance about
// the mean, not a difference of squares) and the result.  G threads share a row, E columns each, the
// fewest that hold it: eight rows a wave at width 64, one at 512, a workgroup of 512 at 8192.  Rows
// wider than 32768 are read again for each pass.  The backward's workgroups walk over rows with the
// column sums in registers and write one partial row each, added up in a fixed order by a second launch;
// rows wider than 8192 are read again for their column sums.
#include <math.h>

#include <algorithm>

#include "gdn2_common.h"
#include "gdn2_status.h"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;

struct LnArgs {
    View x, dy;
    int64_t T, H, rows;   // row r = (b, t, h)
    int W;
    float epsilon;
    const float *weight, *bias;
    void *y;              // y or dx, dense
    float *mean, *inverse;
    float *part_w, *part_b;
};

// Threads of a workgroup whose rows have G each: a row of more than one wave has a workgroup of its own.
template <int G> constexpr int kGroup = G > 64 ? G : kThreads;

// The elements of 16 bytes.
template <typename T> constexpr int kPiece = 16 / (int)sizeof(T);

// N adjacent elements, as they are or as floats.  ALIGNED: whole pieces at 16-byte addresses.  Otherwise
// `left` of them are there (the rest is 0), s elements apart; side by side they are read as one piece
// wherever it lies.
template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void fetch_n(const T *p, int64_t s, int left, T (&e)[N]) {
    if (ALIGNED) {
        __builtin_memcpy(e, __builtin_assume_aligned(p, 16), sizeof e);
    } else if (s == 1 && left >= N) {
        __builtin_memcpy(e, p, sizeof e);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = i < left ? p[i * s] : T(0);
    }
}
template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void load_n(const T *p, int64_t s, int left, float (&v)[N]) {
    T e[N];
    fetch_n<T, N, ALIGNED>(p, s, left, e);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Elem<T>::load(e, i);
}
template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void store_n(T *p, int left, const float (&v)[N]) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) Elem<T>::store(e, i, v[i]);
    if (ALIGNED) {
        __builtin_memcpy(__builtin_assume_aligned(p, 16), e, sizeof e);
    } else if (left >= N) {
        __builtin_memcpy(p, e, sizeof e);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = e[i];
    }
}

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float readlane_f(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Sums over the G threads of a row, in every one of them: lane moves inside 16 lanes, K sums at a time
// so that one's waits are the others' work.
template <int G, int K>
__device__ __forceinline__ void row_sum(float (&x)[K], float *red) {
    static_assert(G >= 8, "");
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += dpp_f<0xB1>(x[k]);
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += dpp_f<0x4E>(x[k]);
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += dpp_f<0x141>(x[k]);
    if constexpr (G >= 16)
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] += dpp_f<0x140>(x[k]);
    if constexpr (G == 32)
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] += __shfl_xor(x[k], 16);
    if constexpr (G >= 64)
#pragma unroll
        for (int k = 0; k < K; ++k)
            x[k] = (readlane_f(x[k], 0) + readlane_f(x[k], 16)) + (readlane_f(x[k], 32) + readlane_f(x[k], 48));
    if constexpr (G > 64) {
        constexpr int WAVES = G / 64;
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) red[k * WAVES + wave] = x[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            x[k] = red[k * WAVES];
            for (int i = 1; i < WAVES; ++i) x[k] += red[k * WAVES + i];
        }
    }
}

__device__ __forceinline__ int64_t row_at(const View &x, const LnArgs &p, int64_t r) {
    const uint32_t n = (uint32_t)r, H = (uint32_t)p.H, T = (uint32_t)p.T;
    const uint32_t bt = n / H, h = n % H;
    return (int64_t)(bt / T) * x.s0 + (int64_t)(bt % T) * x.s1 + (int64_t)h * x.s2;
}

// Columns of thread l, piece j: N adjacent ones from N (l + j G).  Pieces past the width read the row's first
// one in their place and become zero afterwards: under a condition each load would wait for the one before.
template <typename T, int G, int E, bool ALIGNED>
struct Row {
    static constexpr int N = kPiece<T>, P = E / N;
    typedef T Raw[P][N];
    float v[P][N];
    static __device__ __forceinline__ void fetch(Raw &r, const void *base, int64_t at, int64_t s, int l, int W) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int c = N * (l + j * G), k = c < W ? c : 0;
            fetch_n<T, N, ALIGNED>(reinterpret_cast<const T *>(base) + at + k * (ALIGNED ? 1 : s), s, W - k, r[j]);
        }
    }
    __device__ __forceinline__ void take(const Raw &r, bool on, int l, int W) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            uint4 q;
            __builtin_memcpy(&q, r[j], 16);
            if (!(on && N * (l + j * G) < W)) q = make_uint4(0, 0, 0, 0);
            T e[N];
            __builtin_memcpy(e, &q, 16);
#pragma unroll
            for (int i = 0; i < N; ++i) v[j][i] = Elem<T>::load(e, i);
        }
    }
    // The columns of a parameter.
    __device__ __forceinline__ void params(const float *w, int l, int W) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int c = N * (l + j * G), k = c < W ? c : 0;
            load_n<float, N, ALIGNED>(w + k, 1, W - k, v[j]);
#pragma unroll
            for (int e = 0; e < N; ++e) v[j][e] = c < W ? v[j][e] : 0.f;
        }
    }
};

// One row a group of G threads.  Bound by memory: bf16 rows read and written, 8192 of 512 columns 5.6 us
// (3.0 TB/s, much of it the launch), 65536 of 512 23 us (5.8 TB/s), of 1024 42 us (6.4 TB/s); 65536 f32 rows
// of 64 7.2 us (4.7 TB/s).
template <typename T, int G, int E, bool ALIGNED>
__global__ void __launch_bounds__(kGroup<G>) ln_forward_kernel(LnArgs p) {
    constexpr int THREADS = kGroup<G>, ROWS = THREADS / G;
    __shared__ float red[G > 64 ? G / 64 : 1];
    typedef Row<T, G, E, ALIGNED> X;
    constexpr int N = X::N;
    const int l = threadIdx.x % G;
    const int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / G;
    typename X::Raw raw;  // a row past the end reads the last one again: row_sum has barriers
    X::fetch(raw, p.x.data, row_at(p.x, p, min(r, p.rows - 1)), p.x.s3, l, p.W);
    X x, w{}, b{};
    w.params(p.weight, l, p.W);
    if (p.bias) b.params(p.bias, l, p.W);
    x.take(raw, true, l, p.W);
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < X::P; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) s[0] += x.v[j][e];
    row_sum<G, 1>(s, red);
    const float W = (float)p.W, m = s[0] / W;
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < X::P; ++j)
        if (N * (l + j * G) < p.W)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                x.v[j][e] -= m;
                if (ALIGNED || N * (l + j * G) + e < p.W) s[0] = fmaf(x.v[j][e], x.v[j][e], s[0]);
            }
    row_sum<G, 1>(s, red);
    if (r >= p.rows) return;
    const float inv = 1.f / sqrtf(s[0] / W + p.epsilon);
    if (l == 0) {
        if (p.mean) p.mean[r] = m;
        if (p.inverse) p.inverse[r] = inv;
    }
    T *y = reinterpret_cast<T *>(p.y) + r * p.W;
#pragma unroll
    for (int j = 0; j < X::P; ++j) {
        const int c = N * (l + j * G);
        if (c >= p.W) continue;
        float o[N];
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = fmaf(x.v[j][e] * inv, w.v[j][e], b.v[j][e]);
        store_n<T, N, ALIGNED>(y + c, p.W - c, o);
    }
}

// dx, and for rows up to 8192 the column sums of the workgroup's rows.  Wider ones leave no registers for
// the sums (2000 bf16 rows of 32768 columns: 336 us with them, 165 with ln_columns).  Bound by memory: bf16
// rows, x and dy read and dx written, with ln_sum_kernel: 8192 of 512 columns 11.4 us (2.2 TB/s, much of it
// the launches), 65536 of 512 37 us (5.5 TB/s), of 1024 81 us (5.0 TB/s); 65536 f32 rows of 64 14 us.
template <typename T, int G, int E, bool ALIGNED>
__global__ void __launch_bounds__(kGroup<G>) ln_backward_kernel(LnArgs p) {
    constexpr int THREADS = kGroup<G>, ROWS = THREADS / G;
    constexpr bool SUMS = G <= 512, AHEAD = SUMS && ALIGNED;
    __shared__ float red[2 * (G > 64 ? G / 64 : 1)];
    __shared__ float cols[ROWS > 1 ? THREADS * E : 1];
    const int l = threadIdx.x % G, g = threadIdx.x / G;
    typedef Row<T, G, E, ALIGNED> X;
    constexpr int N = X::N;
    X w;
    w.params(p.weight, l, p.W);
    float dw[X::P][N], db[X::P][N];
#pragma unroll
    for (int j = 0; j < X::P; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) dw[j][e] = db[j][e] = 0.f;
    const float W = (float)p.W;
    // Every group of the workgroup makes the same number of turns: row_sum has barriers.  The next row is on
    // its way while one is worked on (not for rows off 16 bytes, whose loads have branches: 65536 bf16 rows of
    // 999 took 177 us instead of 124); past the end the last row is read again and adds nothing.
    typename X::Raw rx, rdy;
    float rm, rinv;
    const auto fetch = [&](int64_t r) {
        r = min(r, p.rows - 1);
        X::fetch(rx, p.x.data, row_at(p.x, p, r), p.x.s3, l, p.W);
        X::fetch(rdy, p.dy.data, row_at(p.dy, p, r), p.dy.s3, l, p.W);
        rm = p.mean[r], rinv = p.inverse[r];
    };
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t r = (int64_t)blockIdx.x * ROWS + g;
    if (AHEAD) fetch(r);
    for (; r - g < p.rows; r += step) {
        const bool on = r < p.rows;
        if (!AHEAD) fetch(r);
        X x, dy;
        x.take(rx, on, l, p.W);
        dy.take(rdy, on, l, p.W);
        const float m = on ? rm : 0.f, inv = on ? rinv : 0.f;
        if (AHEAD) fetch(r + step);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < X::P; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float xh = (x.v[j][e] - m) * inv, d = dy.v[j][e];
                if (SUMS) dw[j][e] = fmaf(d, xh, dw[j][e]), db[j][e] += d;
                const float c = d * w.v[j][e];
                s[0] += c;
                s[1] = fmaf(c, xh, s[1]);
                x.v[j][e] = xh, dy.v[j][e] = c;
            }
        row_sum<G, 2>(s, red);
        if (!p.y || !on) continue;
        const float a = s[0] / W, c2 = s[1] / W;
        T *dx = reinterpret_cast<T *>(p.y) + r * p.W;
#pragma unroll
        for (int j = 0; j < X::P; ++j) {
            const int c = N * (l + j * G);
            if (c >= p.W) continue;
            float o[N];
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = inv * ((dy.v[j][e] - a) - x.v[j][e] * c2);
            store_n<T, N, ALIGNED>(dx + c, p.W - c, o);
        }
    }
    if constexpr (!SUMS) return;
    // The workgroup's column sums, over its groups in order.
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float *part = k ? p.part_b : p.part_w;
        if (!part) continue;
        part += (int64_t)blockIdx.x * p.W;
        if constexpr (ROWS == 1) {
#pragma unroll
            for (int j = 0; j < X::P; ++j)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int c = N * (l + j * G) + e;
                    if (c < p.W) part[c] = k ? db[j][e] : dw[j][e];
                }
        } else {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < X::P; ++j)
#pragma unroll
                for (int e = 0; e < N; ++e) cols[g * G * E + N * (l + j * G) + e] = k ? db[j][e] : dw[j][e];
            __syncthreads();
            for (int c = threadIdx.x; c < p.W; c += THREADS) {
                float t = cols[c];
                for (int i = 1; i < ROWS; ++i) t += cols[i * G * E + c];
                part[c] = t;
            }
        }
    }
}

// Rows of any width: one workgroup of 1024, the row read again for each pass.
constexpr int kLong = 1024;

template <typename T>
__global__ void __launch_bounds__(kLong) ln_forward_long(LnArgs p) {
    __shared__ float red[kLong / 64];
    const int64_t r = blockIdx.x;
    const T *x = reinterpret_cast<const T *>(p.x.data) + row_at(p.x, p, r);
    float s[1] = {0.f};
    for (int64_t c = threadIdx.x; c < p.W; c += kLong) s[0] += Elem<T>::load(x, c * p.x.s3);
    row_sum<kLong, 1>(s, red);
    const float m = s[0] / p.W;
    s[0] = 0.f;
    for (int64_t c = threadIdx.x; c < p.W; c += kLong) {
        const float d = Elem<T>::load(x, c * p.x.s3) - m;
        s[0] = fmaf(d, d, s[0]);
    }
    row_sum<kLong, 1>(s, red);
    const float inv = 1.f / sqrtf(s[0] / p.W + p.epsilon);
    if (threadIdx.x == 0) {
        if (p.mean) p.mean[r] = m;
        if (p.inverse) p.inverse[r] = inv;
    }
    for (int64_t c = threadIdx.x; c < p.W; c += kLong)
        Elem<T>::store(p.y, r * p.W + c, fmaf((Elem<T>::load(x, c * p.x.s3) - m) * inv, p.weight[c],
                                              p.bias ? p.bias[c] : 0.f));
}

// dx of one row a workgroup.
template <typename T>
__global__ void __launch_bounds__(kLong) ln_backward_long(LnArgs p) {
    __shared__ float red[2 * kLong / 64];
    const int64_t r = blockIdx.x;
    const T *x = reinterpret_cast<const T *>(p.x.data) + row_at(p.x, p, r);
    const T *dy = reinterpret_cast<const T *>(p.dy.data) + row_at(p.dy, p, r);
    const float m = p.mean[r], inv = p.inverse[r];
    float s[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < p.W; c += kLong) {
        const float d = Elem<T>::load(dy, c * p.dy.s3) * p.weight[c];
        s[0] += d;
        s[1] = fmaf(d, (Elem<T>::load(x, c * p.x.s3) - m) * inv, s[1]);
    }
    row_sum<kLong, 2>(s, red);
    const float a = s[0] / p.W, b = s[1] / p.W;
    for (int64_t c = threadIdx.x; c < p.W; c += kLong) {
        const float d = Elem<T>::load(dy, c * p.dy.s3) * p.weight[c];
        const float xh = (Elem<T>::load(x, c * p.x.s3) - m) * inv;
        Elem<T>::store(p.y, r * p.W + c, inv * ((d - a) - xh * b));
    }
}

// Column sums of wide rows: a piece of columns a thread and every gridDim.y-th row.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) ln_columns(LnArgs p) {
    constexpr int N = kPiece<T>;
    const int64_t c = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * N;
    if (c >= p.W) return;
    const int left = (int)(p.W - c);
    float dw[N], db[N];
#pragma unroll
    for (int e = 0; e < N; ++e) dw[e] = db[e] = 0.f;
#pragma unroll 2
    for (int64_t r = blockIdx.y; r < p.rows; r += gridDim.y) {
        float x[N], d[N];
        load_n<T, N, ALIGNED>(reinterpret_cast<const T *>(p.x.data) + row_at(p.x, p, r) + c * p.x.s3, p.x.s3, left, x);
        load_n<T, N, ALIGNED>(reinterpret_cast<const T *>(p.dy.data) + row_at(p.dy, p, r) + c * p.dy.s3, p.dy.s3, left, d);
        const float m = p.mean[r], inv = p.inverse[r];
#pragma unroll
        for (int e = 0; e < N; ++e) dw[e] = fmaf(d[e], (x[e] - m) * inv, dw[e]), db[e] += d[e];
    }
    const int64_t at = (int64_t)blockIdx.y * p.W + c;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (e >= left) break;
        if (p.part_w) p.part_w[at + e] = dw[e];
        if (p.part_b) p.part_b[at + e] = db[e];
    }
}

// Partial rows -> dweight (blockIdx.y 0) and dbias (1): 16 columns a workgroup, 64 threads of each over
// the partials, then those in order.
__global__ void __launch_bounds__(1024) ln_sum_kernel(const float *pw, const float *pb, int64_t W,
                                                      int64_t n, float *dw, float *db) {
    __shared__ float red[64][17];
    const float *part = blockIdx.y ? pb : pw;
    float *out = blockIdx.y ? db : dw;
    if (!out) return;
    const int col = threadIdx.x & 15, k0 = threadIdx.x >> 4;
    const int64_t c = (int64_t)blockIdx.x * 16 + col;
    float s = 0.f;
    if (c < W)
#pragma unroll 8
        for (int64_t k = k0; k < n; k += 64) s += part[k * W + c];
    red[k0][col] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < W) {
        float t = red[0][col];
#pragma unroll
        for (int i = 1; i < 64; ++i) t += red[i][col];
        out[c] = t;
    }
}

constexpr int64_t kWide = 32768;  // wider rows do not fit the registers of one workgroup,
constexpr int64_t kSums = 8192;   // nor wider ones than this their column sums too

int64_t row_threads(int64_t W) {  // at most, where a row has a group of its own in the grid
    return W <= 1024 ? 64 : W <= 4096 ? 256 : W <= 8192 ? 512 : 1024;
}

int check_ln(const gdn2_rows_shape *s, const gdn2_view *x, const float *weight) {
    if (!s) return fail(GDN2_ERR_ARGUMENT, "shape is null");
    if (s->batch < 0 || s->time < 0 || s->heads < 0 || s->width < 1 || s->width > (1 << 25))
        return fail(GDN2_ERR_SHAPE, "width must be 1..2^25 and the row axes >= 0");
    const int64_t lim = (int64_t)1 << 31;
    if (s->batch >= lim || s->time >= lim || s->heads >= lim ||
        (s->batch && s->time && s->heads > (lim / 2) / s->batch / s->time))
        return fail(GDN2_ERR_SHAPE, "at most 2^30 rows, and widths below 2^31");
    const int64_t rows = s->batch * s->time * s->heads;
    if (rows >= ((int64_t)1 << 32) / row_threads(s->width))  // threads of one launch
        return fail(GDN2_ERR_SHAPE, "too many rows: below 2^26 of up to 1024 columns, 2^24 of up to "
                                    "4096, 2^23 of up to 8192 and 2^22 of wider ones");
    GDN2_TRY(check_view(x, "x", -1, rows == 0));
    if (!weight) return fail(GDN2_ERR_ARGUMENT, "weight is null");
    return GDN2_OK;
}

bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Whether every row is a run of 16-byte pieces.
bool vec_rows(const gdn2_view *v, int64_t W) {
    const int64_t es = v->dtype == GDN2_BF16 ? 2 : 4;
    if (v->stride[3] != 1 || ((uintptr_t)v->data & 15) || W * es % 16) return false;
    for (int d = 0; d < 3; ++d)
        if (v->stride[d] * es % 16) return false;
    return true;
}

template <typename T, int G, int E, bool BWD, bool ALIGNED>
void launch_one(const LnArgs &a, int64_t partials, hipStream_t st) {
    constexpr int THREADS = kGroup<G>, ROWS = THREADS / G;
    const dim3 block(THREADS), every((unsigned)((a.rows + ROWS - 1) / ROWS));
    if constexpr (!BWD) {
        hipLaunchKernelGGL((ln_forward_kernel<T, G, E, ALIGNED>), every, block, 0, st, a);
    } else if constexpr (G <= 512) {
        hipLaunchKernelGGL((ln_backward_kernel<T, G, E, ALIGNED>), dim3((unsigned)partials), block, 0, st, a);
    } else if (a.y) {
        hipLaunchKernelGGL((ln_backward_kernel<T, G, E, ALIGNED>), every, block, 0, st, a);
    }
}

// Threads a row by its width: 8 columns a thread up to 512 (the forward 16 from 257 on), 16 up to 8192 (the
// backward 8 from 1025 to 2048).  bf16 forward and backward with the one and the other: 65536 rows of 512 25 and
// 37 us with 64 x 8, 22 and 39 with 32 x 16; of 1024 41 and 82 with 64 x 16, 48 and 129 with 128 x 8; 20000 of
// 2048 26 and 61 with 128 x 16, 30 and 52 with 256 x 8; 16384 of 4096 46 and 88 with 256 x 16, 55 and 88 with
// 512 x 8.
template <typename T, bool BWD, bool ALIGNED>
void launch_width(const LnArgs &a, int64_t partials, hipStream_t st) {
    if (a.W <= 64) launch_one<T, 8, 8, BWD, ALIGNED>(a, partials, st);
    else if (a.W <= 128) launch_one<T, 16, 8, BWD, ALIGNED>(a, partials, st);
    else if (a.W <= 256) launch_one<T, 32, 8, BWD, ALIGNED>(a, partials, st);
    else if (a.W <= 512) launch_one<T, BWD ? 64 : 32, BWD ? 8 : 16, BWD, ALIGNED>(a, partials, st);
    else if (a.W <= 1024) launch_one<T, 64, 16, BWD, ALIGNED>(a, partials, st);
    else if (a.W <= 2048) launch_one<T, BWD ? 256 : 128, BWD ? 8 : 16, BWD, ALIGNED>(a, partials, st);
    else if (a.W <= 4096) launch_one<T, 256, 16, BWD, ALIGNED>(a, partials, st);
    else if (a.W <= kSums) launch_one<T, 512, 16, BWD, ALIGNED>(a, partials, st);
    else launch_one<T, 1024, 32, BWD, ALIGNED>(a, partials, st);
}

template <typename T>
void launch_columns(const LnArgs &a, bool vec, int64_t partials, hipStream_t st) {
    const int64_t each = kThreads * kPiece<T>;
    const dim3 grid((unsigned)((a.W + each - 1) / each), (unsigned)partials);
    if (vec) hipLaunchKernelGGL((ln_columns<T, true>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((ln_columns<T, false>), grid, dim3(kThreads), 0, st, a);
}

template <bool BWD>
void launch_ln(const LnArgs &a, int dtype, bool vec, int64_t partials, hipStream_t st) {
    const bool bf = dtype == GDN2_BF16;
    if (vec && bf) launch_width<bf16_t, BWD, true>(a, partials, st);
    else if (vec) launch_width<float, BWD, true>(a, partials, st);
    else if (bf) launch_width<bf16_t, BWD, false>(a, partials, st);
    else launch_width<float, BWD, false>(a, partials, st);
}

// Workgroups of the backward, each of which writes a row of column sums, at most.  512 (1024: 65536 bf16 rows of 1024
// 88 us in place of 81, 8192 of 8192 130 in place of 100); 1024 for many rows off 16 bytes, which have no row ahead
// on its way (65536 of 999 118 us, with 512 174); of wide rows fewer, whose sums would weigh as much as they
// (2000 of 32768 165 us, with 128 178).  The order of the sums goes by it.
int64_t partial_rows(int64_t rows, int64_t W, bool vec) {
    return std::max<int64_t>(1, std::min<int64_t>(rows, W > kSums ? 64 : rows >= 32768 && !vec ? 1024 : 512));
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

int gdn2_layer_norm_forward(const gdn2_rows_shape *shape, float epsilon, const gdn2_view *x,
                            const float *weight, const float *bias, void *y, float *mean,
                            float *inverse, void *stream) {
    GDN2_TRY(check_ln(shape, x, weight));
    LnArgs a{};
    a.rows = shape->batch * shape->time * shape->heads;
    if (a.rows == 0) return ok();
    if (!y) return fail(GDN2_ERR_ARGUMENT, "y is null");
    a.x = make_view(x);
    a.T = shape->time, a.H = shape->heads, a.W = (int)shape->width;
    a.epsilon = epsilon;
    a.weight = weight, a.bias = bias;
    a.y = y, a.mean = mean, a.inverse = inverse;
    hipStream_t st = (hipStream_t)stream;
    if (a.W > kWide) {
        if (x->dtype == GDN2_BF16)
            hipLaunchKernelGGL((ln_forward_long<bf16_t>), dim3((unsigned)a.rows), dim3(kLong), 0, st, a);
        else hipLaunchKernelGGL((ln_forward_long<float>), dim3((unsigned)a.rows), dim3(kLong), 0, st, a);
    } else {
        launch_ln<false>(a, x->dtype, vec_rows(x, a.W) && aligned(y) && aligned(weight) && aligned(bias), 0,
                         st);
    }
    return launch_status(hipGetLastError(), "gdn2_layer_norm_forward");
}

size_t gdn2_layer_norm_workspace_bytes(int64_t rows, int64_t width) {
    if (rows < 0 || width < 1) return 0;
    return (size_t)(2 * 4 * partial_rows(rows, width, false) * width);
}

int gdn2_layer_norm_backward(const gdn2_rows_shape *shape, const gdn2_view *x, const float *weight,
                             const float *mean, const float *inverse, const gdn2_view *dy, void *dx,
                             float *dweight, float *dbias, void *workspace, size_t workspace_bytes,
                             void *stream) {
    GDN2_TRY(check_ln(shape, x, weight));
    LnArgs a{};
    a.rows = shape->batch * shape->time * shape->heads;
    GDN2_TRY(check_view(dy, "dy", x->dtype, a.rows == 0));
    if (a.rows && (!mean || !inverse)) return fail(GDN2_ERR_ARGUMENT, "mean and inverse must be non-null");
    a.W = (int)shape->width;
    const bool params = dweight || dbias;
    if (params) {
        if (!workspace || workspace_bytes < gdn2_layer_norm_workspace_bytes(a.rows, a.W))
            return fail(GDN2_ERR_WORKSPACE, "workspace is too small: %zu bytes needed",
                        gdn2_layer_norm_workspace_bytes(a.rows, a.W));
        if ((uintptr_t)workspace & 15) return fail(GDN2_ERR_ARGUMENT, "workspace must be 16-byte aligned");
    }
    a.x = make_view(x), a.dy = make_view(dy);
    a.T = shape->time, a.H = shape->heads;
    a.weight = weight;
    a.mean = const_cast<float *>(mean), a.inverse = const_cast<float *>(inverse);
    a.y = dx;
    const bool bf = x->dtype == GDN2_BF16, views = vec_rows(x, a.W) && vec_rows(dy, a.W);
    const bool vec = views && aligned(dx) && aligned(weight);
    const int64_t n = partial_rows(a.rows, a.W, vec);
    if (params) {
        float *ws = (float *)workspace;
        a.part_w = dweight ? ws : nullptr;
        a.part_b = dbias ? ws + n * a.W : nullptr;
    }
    hipStream_t st = (hipStream_t)stream;
    if (a.rows && a.W > kWide) {
        if (dx) {
            if (bf) hipLaunchKernelGGL((ln_backward_long<bf16_t>), dim3((unsigned)a.rows), dim3(kLong), 0, st, a);
            else hipLaunchKernelGGL((ln_backward_long<float>), dim3((unsigned)a.rows), dim3(kLong), 0, st, a);
        }
    } else if (a.rows && (dx || params)) {
        launch_ln<true>(a, x->dtype, vec, n, st);
    }
    if (a.rows && params && a.W > kSums) {
        if (bf) launch_columns<bf16_t>(a, views, n, st);
        else launch_columns<float>(a, views, n, st);
    }
    if (params)
        hipLaunchKernelGGL(ln_sum_kernel, dim3((unsigned)((a.W + (int64_t)15) / 16), 2), dim3(1024), 0, st,
                           a.part_w, a.part_b, a.W, a.rows ? n : 0, dweight, dbias);
    return launch_status(hipGetLastError(), "gdn2_layer_norm_backward");
}

}  // extern "C"
