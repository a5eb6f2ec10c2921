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
// probability and the entropy are made of.  A thread adds its columns to it by 8 (f32) or 16 (bf16),
// summed in 32 bits; those around such a token are summed again without it.  -inf logits have
// probability 0 and take no part.
//
// The alternatives need no second sum over the row.  The k-th largest of the threads' maxima is a
// bound that at least k values reach; the few that do are collected and ordered, equal ones by their
// index.  Rows with values that are not finite, with too many values at the bound, or with fewer
// than k that reach it are ordered by k searches for the next value instead.
//
// Both passes are bound by the bytes: 8192 rows of 32768, bf16, forward 99 us (5.4 TB/s), backward 190 (5.6).
// Of 8 such rows the forward takes 11 us with 8 alternatives: the latency of reading the row, of its sums'
// join and of the search for the bound.
#include <float.h>
#include <math.h>

#include "gdn2_common.h"
#include "gdn2_status.h"

namespace gdn2 {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kUnroll = 2;     // 16-byte pieces of a thread on their way at once (4: rows of 1000 take a half longer)
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
    int splits;    // workgroups of a row
    struct PartSums *part;  // [rows][splits]
    uint64_t *part_top;     // [rows][splits][top], in order
    const float *d_lp, *d_h;
    int64_t d_lp_s, d_h_s;
    void *dx;
    bool past;     // dx goes past the caches
};

template <typename T> constexpr int kN = 16 / sizeof(T);

// kN columns from column c of a row, -inf from column `to` on.
template <typename T, bool UNIT>
__device__ __forceinline__ void load_cols(const ScoreArgs &a, const T *row, int64_t c, int64_t to, float *v) {
    constexpr int N = kN<T>;
    if (UNIT && c + N <= to) {
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
        v[j] = c + j < to ? Elem<T>::load(row, (UNIT ? 1 : a.cs) * (c + j)) : -INFINITY;
}

// Sums of a part of a row.
struct PartSums {
    double s;
    float m, u;
};

// m: the maximum so far; s, u: the sums of e and of e (x - m) / temperature, e = exp of that.  Of a thread also
// the columns that brought its maximum, and what they added to s.
struct Sums {
    float m;
    double s;
    float u;
    int64_t at;
    float s_at;
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
    return {M, s, u, 0, 0.f};
}

// Columns from .. to of a row.
template <typename T, bool UNIT>
__device__ __forceinline__ Sums sum_row(const ScoreArgs &a, const T *row, int64_t from, int64_t to) {
    constexpr int N = kN<T>;
    const float c2 = a.inv_t * 1.4426950408889634f;
    Sums t = {-FLT_MAX, 0.0, 0.f, from, 0.f};
    float u2 = 0.f;  // the sum of e (x - m), before the temperature
    const int64_t step = (int64_t)blockDim.x * N;
    for (int64_t c = from + (int64_t)threadIdx.x * N; c < to; c += kUnroll * step) {
        float v[kUnroll][N];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) load_cols<T, UNIT>(a, row, c + i * step, to, v[i]);
        float cm = t.m;
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) cm = fmaxf(cm, v[i][j]);
        const bool more = cm > t.m;
        if (more) {
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
        if (more) t.at = c, t.s_at = s;
    }
    t.u = u2 * a.inv_t;
    return t;
}

// A row, or a part of one, whose largest value is more than half of its sum: it is one value, and log s is
// made of the others, of which a thread's float, with the 1 of the largest in it, keeps 24 bits of 1.  The same in
// every thread.
__device__ __forceinline__ bool is_sure(const Sums &t) { return t.s >= 1.0 && t.s < 2.0 && t.m > -FLT_MAX; }

// The thread that has a sure row's largest value: s with the columns around it summed without the 1.  They are
// read again, rather than kept by every thread or summed apart in every step: 8192 rows of 32768, bf16, take 103 to
// 105 us with and without this, 101 for 99 where all of them are sure; 4000 of 5000 17.5 for 15.4.
template <typename T, bool UNIT>
__device__ double sure_sum(const ScoreArgs &a, const T *row, int64_t to, const Sums &mine, double s) {
    constexpr int N = kN<T>;
    const float c2 = a.inv_t * 1.4426950408889634f;
    const int64_t step = (int64_t)blockDim.x * N;
    float others = 0.f;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        float v[N];
        load_cols<T, UNIT>(a, row, mine.at + i * step, to, v);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float d = v[j] - mine.m;
            others += d < 0.f ? __builtin_amdgcn_exp2f(d * c2) : 0.f;
        }
    }
    return 1.0 + ((s - mine.s_at) + others);
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

constexpr int kGroups = 256;  // of threads, at most, whose maxima give the bound: 4 for each alternative,
                              // so that few values lie between the last alternative and the bound

struct alignas(16) TopShared {
    union {
        float maxima[kGroups];
        uint64_t list[kList];
    };
    uint64_t best[kMaxThreads / 64];
    double log_s;
    float bound;
    int count;
};

// Where the alternatives of a row, or of a part of one, go: to the results, or in order to the join.
struct TopOut {
    int64_t r;
    float m;
    uint64_t *part;  // null: the results
};

__device__ __forceinline__ void put_top(const ScoreArgs &a, const TopOut &t, const TopShared &sh, int rank,
                                        uint64_t o, float v) {
    if (t.part) t.part[rank] = o;
    else write_top(a, t.r, rank, index_of(o), v, t.m, sh.log_s);
}

// The values of columns from .. to that are next in order, one search each; behind the last one 0.
template <typename T, bool UNIT>
__device__ void search_top(const ScoreArgs &a, const T *row, int64_t from, int64_t to, const TopOut &out,
                           TopShared &sh) {
    const int waves = blockDim.x >> 6;
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        for (int64_t c = from + threadIdx.x; c < to; c += blockDim.x) {
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
        if (threadIdx.x == 0)
            put_top(a, out, sh, k, best, best ? Elem<T>::load(row, (UNIT ? 1 : a.cs) * index_of(best)) : 0.f);
    }
}

// mine: the largest value of this thread's columns; s: the sum of the exponentials of all of them.
template <typename T, bool UNIT>
__device__ void find_top(const ScoreArgs &a, const T *row, int64_t from, int64_t to, float mine, double s,
                         const TopOut &out, TopShared &sh) {
    constexpr int N = kN<T>;
    const int nt = blockDim.x, i0 = threadIdx.x;
    if (!(s >= 1.0 && s < DBL_MAX)) {  // the same in every thread
        search_top<T, UNIT>(a, row, from, to, out, sh);
        return;
    }
    // groups of neighbours, each thread counting a share of the maxima above its group's
    int each = 1;
    while (each < 16 && nt / (2 * each) >= 4 * a.top && nt / (2 * each) >= 64) each *= 2;
    while (nt / each > kGroups) each *= 2;
    const int groups = nt / each, per = groups / each;
    float top = mine;
    for (int d = 1; d < each; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    const int g = i0 / each, share = i0 % each;
    if (share == 0) sh.maxima[g] = top;
    if (i0 == 0) sh.count = 0;
    __syncthreads();
    int rank = 0;
    for (int i = share * per; i < (share + 1) * per; i += 4) {
        const float4 o = *reinterpret_cast<const float4 *>(sh.maxima + i);
        rank += (o.x > top || (o.x == top && i < g)) + (o.y > top || (o.y == top && i + 1 < g)) +
                (o.z > top || (o.z == top && i + 2 < g)) + (o.w > top || (o.w == top && i + 3 < g));
    }
    for (int d = 1; d < each; d *= 2) rank += __shfl_xor(rank, d);
    if (share == 0 && rank == a.top - 1) sh.bound = top;
    __syncthreads();  // maxima are read: their place is the list's
    // -FLT_MAX, which a thread without a finite value has too, if fewer groups than that have a larger one: every
    // thread lists its values then, so that of equal ones the first are found
    const float bound = sh.bound;
    if (mine >= bound) {
        const int64_t step = (int64_t)nt * N;
        for (int64_t c = from + (int64_t)i0 * N; c < to; c += kUnroll * step) {
            float v[kUnroll][N];
#pragma unroll
            for (int i = 0; i < kUnroll; ++i) load_cols<T, UNIT>(a, row, c + i * step, to, v[i]);
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
        search_top<T, UNIT>(a, row, from, to, out, sh);
        return;
    }
    for (int i = i0; i < n; i += nt) {
        const uint64_t o = sh.list[i];
        int before = 0;
        for (int k = 0; k < n; ++k) before += sh.list[k] > o;
        if (before < a.top) put_top(a, out, sh, before, o, value_of(o));
    }
}

// A row that is not valid: zeros.
__device__ __forceinline__ bool skip_row(const ScoreArgs &a, int64_t r) {
    if (!a.valid || a.valid[r * a.vs] != 0.f) return false;
    if (threadIdx.x == 0) {
        a.log_probs[r] = a.entropy[r] = 0.f;
        if (a.stats) a.stats[3 * r] = a.stats[3 * r + 1] = a.stats[3 * r + 2] = 0.f;
    }
    if ((int)threadIdx.x < a.top) {
        a.top_tokens[r * a.top + threadIdx.x] = 0;
        a.top_log_probs[r * a.top + threadIdx.x] = 0.f;
    }
    return true;
}

template <typename T, bool UNIT>
__device__ __forceinline__ float given_logit(const ScoreArgs &a, const T *row, int64_t r) {
    const int64_t label = a.target[r * a.ts];
    return label >= 0 && label < a.width ? Elem<T>::load(row, (UNIT ? 1 : a.cs) * label) : __builtin_nanf("");
}

// The results of a row by one thread, from its sums and s; log s for the alternatives is read behind a barrier.
template <bool TOP> __device__ __forceinline__ void write_row(const ScoreArgs &a, int64_t r, const Sums &t, double s,
                                                              float xl, TopShared &sh, bool writes) {
    if (!__any(writes)) return;
    const double log_s = log(s);  // in 64 bits: 200 instructions, of one wave
    if (writes) {
        const float h = (float)(log_s - (double)t.u / s);
        a.log_probs[r] = (float)((double)(xl - t.m) * a.inv_t - log_s);
        a.entropy[r] = h;
        if (a.stats) a.stats[3 * r] = t.m, a.stats[3 * r + 1] = (float)log_s, a.stats[3 * r + 2] = h;
        if (TOP) sh.log_s = log_s;
    }
}

template <typename T, bool UNIT, bool TOP>
__global__ void __launch_bounds__(kMaxThreads) score_forward(ScoreArgs a) {
    __shared__ BlockShared red;
    __shared__ TopShared sh;
    const int64_t r = blockIdx.x;
    if (skip_row(a, r)) return;
    const T *row = (const T *)a.x + r * a.rs;
    const float xl = given_logit<T, UNIT>(a, row, r);
    const Sums mine = sum_row<T, UNIT>(a, row, 0, a.width);
    const Sums t = merge_block(mine, red, a.inv_t);
    const bool sure = is_sure(t), writes = sure ? mine.m == t.m : threadIdx.x == 0;
    double s = t.s;
    if (sure && writes) s = sure_sum<T, UNIT>(a, row, a.width, mine, s);
    write_row<TOP>(a, r, t, s, xl, sh, writes);
    if constexpr (TOP) find_top<T, UNIT>(a, row, 0, a.width, mine.m, t.s, TopOut{r, t.m, nullptr}, sh);
}

// Rows that are few and wide: a part of a row each ...
template <typename T, bool UNIT, bool TOP>
__global__ void __launch_bounds__(kMaxThreads) score_part(ScoreArgs a) {
    __shared__ BlockShared red;
    __shared__ TopShared sh;
    const int64_t r = blockIdx.x / a.splits;
    const int part = blockIdx.x % a.splits;
    if (a.valid && a.valid[r * a.vs] == 0.f) return;
    // parts begin at whole pieces
    const int64_t per = ((a.width + a.splits - 1) / a.splits + 15) & ~(int64_t)15;
    const int64_t from = min(part * per, a.width), to = min(from + per, a.width);
    const T *row = (const T *)a.x + r * a.rs;
    const Sums mine = sum_row<T, UNIT>(a, row, from, to);
    const Sums t = merge_block(mine, red, a.inv_t);
    const bool sure = is_sure(t);
    if (sure ? mine.m == t.m : threadIdx.x == 0)
        a.part[blockIdx.x] = {sure ? sure_sum<T, UNIT>(a, row, to, mine, t.s) : t.s, t.m, t.u};
    if constexpr (TOP)
        find_top<T, UNIT>(a, row, from, to, mine.m, t.s, TopOut{r, t.m, a.part_top + (int64_t)blockIdx.x * a.top}, sh);
}

constexpr int kMaxSplits = 24;

// ... and the join of a row's parts.  Of the alternatives' lists, in order each, only what reaches the
// smallest of their ceil(top / splits)-th values can be among the row's.
template <typename T, bool UNIT, bool TOP> __global__ void __launch_bounds__(256) score_join(ScoreArgs a) {
    __shared__ TopShared sh;
    __shared__ uint64_t list[kMaxSplits * kMaxTop];
    const int64_t r = blockIdx.x;
    if (skip_row(a, r)) return;
    const float xl = given_logit<T, UNIT>(a, (const T *)a.x + r * a.rs, r);
    // a lane has a part, every wave the same
    const int lane = threadIdx.x & 63;
    const uint64_t *tops = a.part_top + r * a.splits * a.top;
    const int deep = (a.top + a.splits - 1) / a.splits - 1;
    PartSums q = {0.0, -FLT_MAX, 0.f};
    uint64_t bound = ~0ull;
    if (lane < a.splits) {
        q = a.part[r * a.splits + lane];
        if (TOP) bound = tops[lane * a.top + deep];
    }
    float M = q.m;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) M = fmaxf(M, __shfl_xor(M, k));
    const float d = fmaxf((q.m - M) * a.inv_t, kLowest), e = __expf(d);
    Sums t = {M, q.s * e, e * (q.u + (float)q.s * d), 0, 0.f};
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
        t.s += __shfl_xor(t.s, k), t.u += __shfl_xor(t.u, k);
        if (TOP) bound = min(bound, (uint64_t)__shfl_xor((unsigned long long)bound, k));
    }
    write_row<TOP>(a, r, t, t.s, xl, sh, threadIdx.x == 0);
    if constexpr (TOP) {
        const int n = a.splits * a.top;
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += 256) {
            const uint64_t o = tops[i];
            if (o >= bound && o) list[atomicAdd(&sh.count, 1)] = o;
        }
        __syncthreads();
        const int m = sh.count;
        for (int i = threadIdx.x; i < m; i += 256) {
            const uint64_t o = list[i];
            int before = 0;
            for (int k = 0; k < m; ++k) before += list[k] > o;
            if (before < a.top) {
                // a NaN or an infinity gives the row's sums, -0 gives what 0 does
                write_top(a, r, before, index_of(o), value_of(o), t.m, sh.log_s);
            }
        }
    }
}

constexpr int kBackThreads = 256;
// A gradient larger than the last level of cache is written past it, where the logits stay for a while:
// 8192 rows of 32768, bf16, backward 191 us for 200, forward and backward in turn 282 for 306, with a product
// that reads the gradient behind it 541 for 541.  Of 64 MB the product finds it in the cache: 170 us, 179
// if it was written past.
constexpr int64_t kCache = (int64_t)256 << 20;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T, bool UNIT> __global__ void __launch_bounds__(kBackThreads) score_backward(ScoreArgs a) {
    constexpr int N = kN<T>;
    const int64_t r = blockIdx.x;
    const T *row = (const T *)a.x + r * a.rs;
    T *out = (T *)a.dx + r * a.width;
    const bool on = !a.valid || a.valid[r * a.vs] != 0.f;
    const float m = a.stats[3 * r], log_s = a.stats[3 * r + 1], H = a.stats[3 * r + 2];
    float dl = a.d_lp ? a.d_lp[r * a.d_lp_s] : 0.f;
    const float dh = a.d_h ? a.d_h[r * a.d_h_s] : 0.f;
    const int64_t label = a.target[r * a.ts];
    if ((label < 0 || label >= a.width) && dl != 0.f) dl = __builtin_nanf("");
    const int64_t step = (int64_t)kBackThreads * N;
    for (int64_t c = ((int64_t)blockIdx.y * kUnroll * kBackThreads + threadIdx.x) * N; c < a.width;
         c += gridDim.y * kUnroll * step) {
        float v[kUnroll][N];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
            if (on) load_cols<T, UNIT>(a, row, c + i * step, a.width, v[i]);
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const int64_t ci = c + i * step;
            if (ci >= a.width) break;
            float o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float lp = fmaxf((v[i][j] - m) * a.inv_t, kLowest) - log_s;
                const float p = __expf(lp);
                // p first: p (lp + H) is 0 where p is, and small elsewhere; 1 / temperature may be far larger
                float d = -p * dl - dh * (p * (lp + H));
                if (ci + j == label) d += dl;
                o[j] = on ? d * a.inv_t : 0.f;
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
                if (a.past) __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]}, (u32x4 *)(out + ci));
                else __builtin_memcpy(out + ci, w, 16);
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
    // a workgroup of up to 256 threads a row, 2^32 - 1 threads a launch
    if (rows >= 1 << 24 || width > 0x7FFFFFFF)
        return fail(GDN2_ERR_SHAPE, "at most 2^24 - 1 rows and 2^31 - 1 columns");
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

// Workgroups of a row: more than one where rows are few and wide (one row of 200000 with 32 alternatives:
// 38 us as one, 18 in parts, two launches).  Both sides, in us, bf16, without and with 8 alternatives, as one and in
// parts of the same rule: 8 rows of 32768 7.4, 11.6 and 8.9, 13.3; of 65536 9.8, 16.2 and 9.0, 13.4; 64 rows of 32768
// 7.6, 12.0 and 9.4, 13.8; of 65536 10.2, 16.9 and 9.4, 13.6; of 200000 20.6, 36.8 and 12.4, 19.3.  The limit of 64
// leaves something: 65 rows of 65536 10.1, 16.9 and 10.0, 15.4, 128 of 200000 22.7, 40.5 and 18.1, 28.3.
int splits_for(int64_t rows, int64_t width) {
    if (rows > 64 || width < 65536) return 1;
    int64_t s = width / 8192;
    if (s > 256 / rows) s = 256 / rows;
    return (int)(s > kMaxSplits ? kMaxSplits : s);
}

size_t part_bytes(int64_t rows, int splits, int top) {
    return splits > 1 ? (size_t)rows * splits * (sizeof(PartSums) + sizeof(uint64_t) * top) : 0;
}

template <typename T, bool UNIT> void launch_forward(const ScoreArgs &a, hipStream_t st) {
    if (a.splits > 1) {
        const dim3 parts((unsigned)(a.rows * a.splits)), threads(kMaxThreads), rows((unsigned)a.rows), join(256);
        if (a.top) {
            hipLaunchKernelGGL((score_part<T, UNIT, true>), parts, threads, 0, st, a);
            hipLaunchKernelGGL((score_join<T, UNIT, true>), rows, join, 0, st, a);
        } else {
            hipLaunchKernelGGL((score_part<T, UNIT, false>), parts, threads, 0, st, a);
            hipLaunchKernelGGL((score_join<T, UNIT, false>), rows, join, 0, st, a);
        }
        return;
    }
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

size_t gdn2_token_score_workspace_bytes(int64_t rows, int64_t width, int32_t top) {
    if (rows < 0 || width < 1 || top < 0 || top > kMaxTop) return 0;
    return part_bytes(rows, splits_for(rows, width), top);
}

int gdn2_token_score_forward(int64_t rows, int64_t width, const gdn2_view *x, const int64_t *target,
                             int64_t target_stride, const float *valid, int64_t valid_stride,
                             float temperature, int32_t top, float *log_probs, float *entropy,
                             float *top_log_probs, int64_t *top_tokens, float *stats, void *workspace,
                             size_t workspace_bytes, void *stream) {
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
    a.splits = splits_for(rows, width);
    if (const size_t need = part_bytes(rows, a.splits, top)) {
        if (!workspace || workspace_bytes < need)
            return fail(GDN2_ERR_WORKSPACE, "workspace is too small: %zu bytes needed", need);
        if ((uintptr_t)workspace & 15) return fail(GDN2_ERR_ARGUMENT, "workspace must be 16-byte aligned");
        a.part = (PartSums *)workspace;
        a.part_top = (uint64_t *)(a.part + rows * a.splits);
    }
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
    a.past = rows * width * (x->dtype == GDN2_BF16 ? 2 : 4) > kCache;
    const bool unit = a.cs == 1;
    hipStream_t st = (hipStream_t)stream;
    if (x->dtype == GDN2_BF16) unit ? launch_backward<bf16_t, true>(a, st) : launch_backward<bf16_t, false>(a, st);
    else unit ? launch_backward<float, true>(a, st) : launch_backward<float, false>(a, st);
    return launch_status(hipGetLastError(), "gdn2_token_score_backward");
}

}  // extern "C"
