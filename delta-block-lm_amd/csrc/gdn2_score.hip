// Scores of given tokens on gfx950: log probability, entropy and the top alternatives of rows of
// logits, and the gradient of the first two.
//
//   z = x / temperature,  m = max x,  s = sum exp((x - m) / temperature)
//   log p_j = (x_j - m) / temperature - log s
//   H       = log s - sum exp(..) (x - m) / temperature / s
//   dx_j    = [dlp (1[j = t] - p_j) - dH p_j (log p_j + H)] / temperature
//
// One workgroup reads a row once: every thread keeps the maximum, s and the entropy's sum of its
// columns, which are joined across the workgroup in a fixed order.  s is held in 64 bits: next to a
// token of probability near 1 the others' sum is far below it, and their part is all that the log
// probability and the entropy are made of.  -inf logits have probability 0 and take no part.
//
// The alternatives need no second sum over the row.  The k-th largest of the threads' maxima is a
// bound that at least k values reach; the few that do are collected and ordered, equal ones by their
// index.  Rows with values that are not finite, with too many values at the bound, or with fewer
// than k that reach it are ordered by k searches for the next value instead.
#include <float.h>
#include <math.h>

#include "gdn2_common.h"
#include "gdn2_status.h"

namespace gdn2 {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kUnroll = 4;     // 16-byte pieces of a thread on their way at once
constexpr int kMaxTop = 64;
constexpr int kList = 1024;    // values that may reach the bound
constexpr float kLowest = -1e30f;  // stands for -inf where it is multiplied by 0

struct ScoreArgs {
    const void *x;
    int64_t rs, cs;
    int64_t rows, width;
    const int64_t *target;
    int64_t ts;
    const float *valid;
    int64_t vs;
    float inv_t;
    int top;
    float *log_probs, *entropy;
    float *top_log_probs;
    int64_t *top_tokens;
    float *stats;  // [rows][3]: m, log s, H
    const float *d_lp, *d_h;
    int64_t d_lp_s, d_h_s;
    void *dx;
};

template <typename T> constexpr int kN = 16 / sizeof(T);

// kN columns from column c of a row, -inf where there are none.
template <typename T, bool UNIT>
__device__ __forceinline__ void load_cols(const ScoreArgs &a, const T *row, int64_t c, float *v) {
    constexpr int N = kN<T>;
    if (UNIT && c + N <= a.width) {
        uint32_t w[4];
        __builtin_memcpy(w, row + c, 16);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
        v[j] = c + j < a.width ? Elem<T>::load(row, (UNIT ? 1 : a.cs) * (c + j)) : -INFINITY;
}

// m: the maximum so far; s, u: the sums of e and of e (x - m) / temperature, e = exp of that.
struct Sums {
    float m;
    double s;
    float u;
};

struct BlockShared {
    float m[kMaxThreads / 64], u[kMaxThreads / 64];
    double s[kMaxThreads / 64];
};

// The sums of the workgroup, in every thread: first the maximum, so that a thread's sums are scaled
// once, then plain sums in a fixed order.
__device__ Sums merge_block(const Sums &a, BlockShared &sh, float inv_t) {
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
    float M = a.m;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) M = fmaxf(M, __shfl_xor(M, d));
    if (waves > 1) {
        if ((threadIdx.x & 63) == 0) sh.m[wave] = M;
        __syncthreads();
        for (int w = 0; w < waves; ++w) M = fmaxf(M, sh.m[w]);
    }
    const float d = fmaxf((a.m - M) * inv_t, kLowest), e = __expf(d);
    double s = a.s * e;
    float u = e * (a.u + (float)a.s * d);
#pragma unroll
    for (int k = 1; k < 64; k *= 2) s += __shfl_xor(s, k), u += __shfl_xor(u, k);
    if (waves > 1) {
        if ((threadIdx.x & 63) == 0) sh.s[wave] = s, sh.u[wave] = u;
        __syncthreads();
        s = 0, u = 0;
        for (int w = 0; w < waves; ++w) s += sh.s[w], u += sh.u[w];
    }
    return {M, s, u};
}

template <typename T, bool UNIT>
__device__ __forceinline__ Sums sum_row(const ScoreArgs &a, const T *row) {
    constexpr int N = kN<T>;
    const float c2 = a.inv_t * 1.4426950408889634f;
    Sums t = {-FLT_MAX, 0.0, 0.f};
    float u2 = 0.f;  // the sum of e (x - m), before the temperature
    const int64_t step = (int64_t)blockDim.x * N;
    for (int64_t c = (int64_t)threadIdx.x * N; c < a.width; c += kUnroll * step) {
        float v[kUnroll][N];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) load_cols<T, UNIT>(a, row, c + i * step, v[i]);
        float cm = t.m;
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) cm = fmaxf(cm, v[i][j]);
        if (cm > t.m) {
            const float d = fmaxf(t.m - cm, kLowest), e = __builtin_amdgcn_exp2f(d * c2);
            u2 = e * (u2 + (float)t.s * d);
            t.s *= e;
            t.m = cm;
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float d = v[i][j] - t.m, e = __builtin_amdgcn_exp2f(d * c2);
                s += e;
                u2 = fmaf(e, fmaxf(d, kLowest), u2);
            }
        t.s += s;
    }
    t.u = u2 * a.inv_t;
    return t;
}

// ---- order of values ------------------------------------------------------------------

// Larger for larger values, NaN the largest, -0 as 0; of equal values larger for the lower index.
__device__ __forceinline__ uint64_t order_of(float v, int64_t i) {
    const uint32_t b = __float_as_uint(v + 0.f);
    const uint32_t key = v != v ? 0xFFFFFFFFu : b ^ ((int32_t)b < 0 ? 0xFFFFFFFFu : 0x80000000u);
    return (uint64_t)key << 32 | (0xFFFFFFFFu - (uint32_t)i);
}

__device__ __forceinline__ int64_t index_of(uint64_t o) { return 0xFFFFFFFFu - (uint32_t)o; }

// The value that was ordered (+0 for -0), of those that are numbers.
__device__ __forceinline__ float value_of(uint64_t o) {
    const uint32_t key = (uint32_t)(o >> 32);
    return __uint_as_float(key ^ ((int32_t)key < 0 ? 0x80000000u : 0xFFFFFFFFu));
}

__device__ __forceinline__ void write_top(const ScoreArgs &a, int64_t r, int rank, int64_t i, float v,
                                          float m, double log_s) {
    a.top_tokens[r * a.top + rank] = i;
    a.top_log_probs[r * a.top + rank] = (float)((double)(v - m) * a.inv_t - log_s);
}

constexpr int kGroups = 256;  // of threads, at most, whose maxima give the bound

struct alignas(16) TopShared {
    union {
        float maxima[kGroups];
        uint64_t list[kList];
    };
    uint64_t best[kMaxThreads / 64];
    float bound;
    int count;
};

// The k values that are next in order, one search of the row each.
template <typename T, bool UNIT>
__device__ void search_top(const ScoreArgs &a, const T *row, int64_t r, float m, double log_s,
                           TopShared &sh) {
    const int waves = blockDim.x >> 6;
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        for (int64_t c = threadIdx.x; c < a.width; c += blockDim.x) {
            const uint64_t o = order_of(Elem<T>::load(row, (UNIT ? 1 : a.cs) * c), c);
            if (o > best && o < last) best = o;
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_xor((unsigned long long)best, d);
            best = o > best ? o : best;
        }
        __syncthreads();  // sh.best is read
        if ((threadIdx.x & 63) == 0) sh.best[threadIdx.x >> 6] = best;
        __syncthreads();
        for (int w = 0; w < waves; ++w) best = sh.best[w] > best ? sh.best[w] : best;
        last = best;
        if (threadIdx.x == 0) {
            const int64_t i = index_of(best);
            write_top(a, r, k, i, Elem<T>::load(row, (UNIT ? 1 : a.cs) * i), m, log_s);
        }
    }
}

template <typename T, bool UNIT>
__device__ void find_top(const ScoreArgs &a, const T *row, int64_t r, float mine, float m, double s,
                         double log_s, TopShared &sh) {
    constexpr int N = kN<T>;
    const int nt = blockDim.x, i0 = threadIdx.x;
    if (!(s >= 1.0 && s < DBL_MAX)) {  // the same in every thread
        search_top<T, UNIT>(a, row, r, m, log_s, sh);
        return;
    }
    // groups of 1, 2 or 4 neighbours, each thread counting a share of the maxima above its group's
    const int groups = min(nt, kGroups), each = nt / groups;
    float top = mine;
    if (each > 1) top = fmaxf(top, __shfl_xor(top, 1));
    if (each > 2) top = fmaxf(top, __shfl_xor(top, 2));
    const int g = i0 / each, share = i0 % each;
    if (share == 0) sh.maxima[g] = top;
    if (i0 == 0) sh.count = 0;
    __syncthreads();
    int rank = 0;
    for (int i = share * (groups / each); i < (share + 1) * (groups / each); i += 4) {
        const float4 o = *reinterpret_cast<const float4 *>(sh.maxima + i);
        rank += (o.x > top || (o.x == top && i < g)) + (o.y > top || (o.y == top && i + 1 < g)) +
                (o.z > top || (o.z == top && i + 2 < g)) + (o.w > top || (o.w == top && i + 3 < g));
    }
    if (each > 1) rank += __shfl_xor(rank, 1);
    if (each > 2) rank += __shfl_xor(rank, 2);
    if (share == 0 && rank == a.top - 1) sh.bound = top;
    __syncthreads();  // maxima are read: their place is the list's
    const float bound = sh.bound;
    if (mine >= bound && mine > -FLT_MAX) {
        const int64_t step = (int64_t)nt * N;
        for (int64_t c = (int64_t)i0 * N; c < a.width; c += kUnroll * step) {
            float v[kUnroll][N];
#pragma unroll
            for (int i = 0; i < kUnroll; ++i) load_cols<T, UNIT>(a, row, c + i * step, v[i]);
#pragma unroll
            for (int i = 0; i < kUnroll; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (v[i][j] >= bound && v[i][j] > -INFINITY) {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < kList) sh.list[at] = order_of(v[i][j], c + i * step + j);
                    }
        }
    }
    __syncthreads();
    const int n = sh.count;  // the list's order differs from run to run, what it holds does not
    if (n < a.top || n > kList) {
        __syncthreads();
        search_top<T, UNIT>(a, row, r, m, log_s, sh);
        return;
    }
    for (int i = i0; i < n; i += nt) {
        const uint64_t o = sh.list[i];
        int before = 0;
        for (int k = 0; k < n; ++k) before += sh.list[k] > o;
        if (before < a.top) write_top(a, r, before, index_of(o), value_of(o), m, log_s);
    }
}

template <typename T, bool UNIT, bool TOP>
__global__ void __launch_bounds__(kMaxThreads) score_forward(ScoreArgs a) {
    __shared__ BlockShared red;
    const int64_t r = blockIdx.x;
    if (a.valid && a.valid[r * a.vs] == 0.f) {
        if (threadIdx.x == 0) {
            a.log_probs[r] = a.entropy[r] = 0.f;
            if (a.stats) a.stats[3 * r] = a.stats[3 * r + 1] = a.stats[3 * r + 2] = 0.f;
        }
        if (TOP && (int)threadIdx.x < a.top) {
            a.top_tokens[r * a.top + threadIdx.x] = 0;
            a.top_log_probs[r * a.top + threadIdx.x] = 0.f;
        }
        return;
    }
    const T *row = (const T *)a.x + r * a.rs;
    const int64_t label = a.target[r * a.ts];
    const float xl = label >= 0 && label < a.width ? Elem<T>::load(row, (UNIT ? 1 : a.cs) * label)
                                                   : __builtin_nanf("");
    const Sums mine = sum_row<T, UNIT>(a, row);
    const Sums t = merge_block(mine, red, a.inv_t);
    const double log_s = log(t.s);
    if (threadIdx.x == 0) {
        const float h = (float)(log_s - (double)t.u / t.s);
        a.log_probs[r] = (float)((double)(xl - t.m) * a.inv_t - log_s);
        a.entropy[r] = h;
        if (a.stats) a.stats[3 * r] = t.m, a.stats[3 * r + 1] = (float)log_s, a.stats[3 * r + 2] = h;
    }
    if constexpr (TOP) {
        __shared__ TopShared sh;
        find_top<T, UNIT>(a, row, r, mine.m, t.m, t.s, log_s, sh);
    }
}

constexpr int kBackThreads = 256;

template <typename T, bool UNIT> __global__ void __launch_bounds__(kBackThreads) score_backward(ScoreArgs a) {
    constexpr int N = kN<T>;
    const int64_t r = blockIdx.x;
    const T *row = (const T *)a.x + r * a.rs;
    T *out = (T *)a.dx + r * a.width;
    const bool on = !a.valid || a.valid[r * a.vs] != 0.f;
    const float m = a.stats[3 * r], log_s = a.stats[3 * r + 1], H = a.stats[3 * r + 2];
    float dl = a.d_lp ? a.d_lp[r * a.d_lp_s] : 0.f;
    const float dh = a.d_h ? a.d_h[r * a.d_h_s] * a.inv_t : 0.f;
    const int64_t label = a.target[r * a.ts];
    if ((label < 0 || label >= a.width) && dl != 0.f) dl = __builtin_nanf("");
    dl *= a.inv_t;
    const int64_t step = (int64_t)kBackThreads * N;
    for (int64_t c = ((int64_t)blockIdx.y * kUnroll * kBackThreads + threadIdx.x) * N; c < a.width;
         c += gridDim.y * kUnroll * step) {
        float v[kUnroll][N];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
            if (on) load_cols<T, UNIT>(a, row, c + i * step, v[i]);
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const int64_t ci = c + i * step;
            if (ci >= a.width) break;
            float o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float lp = fmaxf((v[i][j] - m) * a.inv_t, kLowest) - log_s;
                const float p = __expf(lp);
                float d = p * (-dl - dh * (lp + H));
                if (ci + j == label) d += dl;
                o[j] = on ? d : 0.f;
            }
            if (ci + N <= a.width) {
                uint32_t w[4];
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(o[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w[j] = (uint32_t)f32_to_bf16(o[2 * j]) | ((uint32_t)f32_to_bf16(o[2 * j + 1]) << 16);
                }
                __builtin_memcpy(out + ci, w, 16);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (ci + j < a.width) Elem<T>::store(out, ci + j, o[j]);
            }
        }
    }
}

int check_score(int64_t rows, int64_t width, const gdn2_view *x, const int64_t *target,
                int64_t target_stride, const float *valid, int64_t valid_stride, float temperature,
                ScoreArgs *a) {
    if (rows < 0 || width < 1) return fail(GDN2_ERR_SHAPE, "rows must be >= 0 and width >= 1");
    if (rows > 0x7FFFFFFF || width > 0x7FFFFFFF) return fail(GDN2_ERR_SHAPE, "at most 2^31 - 1 rows and columns");
    GDN2_TRY(check_view(x, "x", -1, rows == 0));
    if (rows && !target) return fail(GDN2_ERR_ARGUMENT, "target is null");
    if (target_stride < 0 || valid_stride < 0) return fail(GDN2_ERR_ARGUMENT, "negative stride");
    if (!(temperature >= FLT_MIN && temperature <= FLT_MAX && 1.f / temperature >= FLT_MIN))
        return fail(GDN2_ERR_ARGUMENT, "temperature must be positive and finite, and its inverse too");
    *a = ScoreArgs{};
    a->x = x->data;
    a->rs = x->stride[0], a->cs = x->stride[1];
    a->rows = rows, a->width = width;
    a->target = target, a->ts = target_stride;
    a->valid = valid, a->vs = valid_stride;
    a->inv_t = 1.f / temperature;
    return ok();
}

// Threads of a row's workgroup: a piece or more for each; many for rows that are few.
int threads_for(int64_t rows, int64_t width, int n) {
    int t = 64;
    const int most = rows >= 512 ? 256 : kMaxThreads;
    while (t < most && width > (int64_t)t * n * 2) t *= 2;
    return t;
}

template <typename T, bool UNIT> void launch_forward(const ScoreArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)a.rows), block(threads_for(a.rows, a.width, kN<T>));
    if (a.top) hipLaunchKernelGGL((score_forward<T, UNIT, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((score_forward<T, UNIT, false>), grid, block, 0, st, a);
}

template <typename T, bool UNIT> void launch_backward(const ScoreArgs &a, hipStream_t st) {
    const int64_t piece = (int64_t)kUnroll * kBackThreads * kN<T>;
    int64_t parts = (a.width + piece - 1) / piece;
    if (parts > 65535) parts = 65535;
    hipLaunchKernelGGL((score_backward<T, UNIT>), dim3((unsigned)a.rows, (unsigned)parts), dim3(kBackThreads),
                       0, st, a);
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

int gdn2_token_score_forward(int64_t rows, int64_t width, const gdn2_view *x, const int64_t *target,
                             int64_t target_stride, const float *valid, int64_t valid_stride,
                             float temperature, int32_t top, float *log_probs, float *entropy,
                             float *top_log_probs, int64_t *top_tokens, float *stats, void *stream) {
    ScoreArgs a;
    GDN2_TRY(check_score(rows, width, x, target, target_stride, valid, valid_stride, temperature, &a));
    if (top < 0 || top > kMaxTop || top > width)
        return fail(GDN2_ERR_SHAPE, "top must be 0 to %d and at most the width", kMaxTop);
    if (rows && (!log_probs || !entropy || (top && (!top_log_probs || !top_tokens))))
        return fail(GDN2_ERR_ARGUMENT, "outputs must be non-null");
    if (rows == 0) return ok();
    a.top = top;
    a.log_probs = log_probs, a.entropy = entropy;
    a.top_log_probs = top_log_probs, a.top_tokens = top_tokens;
    a.stats = stats;
    const bool unit = a.cs == 1;
    hipStream_t st = (hipStream_t)stream;
    if (x->dtype == GDN2_BF16) unit ? launch_forward<bf16_t, true>(a, st) : launch_forward<bf16_t, false>(a, st);
    else unit ? launch_forward<float, true>(a, st) : launch_forward<float, false>(a, st);
    return launch_status(hipGetLastError(), "gdn2_token_score_forward");
}

int gdn2_token_score_backward(int64_t rows, int64_t width, const gdn2_view *x, const int64_t *target,
                              int64_t target_stride, const float *valid, int64_t valid_stride,
                              float temperature, const float *stats, const float *d_log_probs,
                              int64_t d_log_probs_stride, const float *d_entropy,
                              int64_t d_entropy_stride, void *dx, void *stream) {
    ScoreArgs a;
    GDN2_TRY(check_score(rows, width, x, target, target_stride, valid, valid_stride, temperature, &a));
    if (rows && (!stats || !dx)) return fail(GDN2_ERR_ARGUMENT, "stats and dx must be non-null");
    if (d_log_probs_stride < 0 || d_entropy_stride < 0) return fail(GDN2_ERR_ARGUMENT, "negative stride");
    if (rows == 0) return ok();
    a.stats = const_cast<float *>(stats);
    a.d_lp = d_log_probs, a.d_lp_s = d_log_probs_stride;
    a.d_h = d_entropy, a.d_h_s = d_entropy_stride;
    a.dx = dx;
    const bool unit = a.cs == 1;
    hipStream_t st = (hipStream_t)stream;
    if (x->dtype == GDN2_BF16) unit ? launch_backward<bf16_t, true>(a, st) : launch_backward<bf16_t, false>(a, st);
    else unit ? launch_backward<float, true>(a, st) : launch_backward<float, false>(a, st);
    return launch_status(hipGetLastError(), "gdn2_token_score_backward");
}

}  // extern "C"
