// Gated linear recurrence on gfx950: forward, backward and the single-token step.
//
//   h_t = exp(g_t) h_{t-1} + x_t,  y_t = h_t                      per channel of [B, T, W]
//   e_t = dy_t + E_{t+1},  E_t = exp(g_t) e_t                     the adjoint, from the last token
//   dx_t = e_t,  dg_t = exp(g_t) h_{t-1} e_t,  d_initial = E_1
//
// A run of tokens acts on the state before it as S + A h, and joining two runs needs only their
// (A, S): the time axis is split over lanes, waves, and, where there are few channels, workgroups.
//   * A workgroup has 128 bytes of channels (64 bf16, 32 f32: one memory line of a token) and up to
//     8 waves; a lane has one 16-byte piece of kL tokens in a row, a wave 8 such runs for each of
//     its 8 pieces, a block is what all waves hold.  Every tensor is read and written once, in
//     lines, and the next block's loads are on their way while a block is worked on.
//   * Inside a block: each lane its own run, the 8 runs of a wave by lane exchanges, the waves
//     through LDS (one barrier a block); then each lane walks its run again from its true state.
//   * Segments: if there are too few workgroups the blocks of a sequence go to several.  A first
//     kernel makes each segment's (A, S), and every segment starts from the joined ones before it:
//     the inputs are read twice, by kernels that fill the card.
// The backward recomputes the states of a block from the state before it, which the forward kept
// (4 bytes a channel for every block), and walks the blocks from the last.
//
// A is carried as half its log2 and its root applied twice, clamped to [2^-126, 2^127]: a state of
// any size meets a decay of any size as it would token by token, zero stays zero, and what is not
// finite stays so.  Logarithms add up almost exactly, so a slow decay is rounded once for what a
// state passes in one step (a block), not once a token.  Half = -inf means that nothing gets through:
// a reset, or a gate whose exp is below 2^-126.  There a state is dropped, not multiplied, so that
// what is not finite does not pass.
#include <math.h>

#include "gdn2_common.h"
#include "gdn2_status.h"

namespace gdn2 {
namespace {

constexpr int kL = 4;         // tokens of a lane's run
constexpr int kPieces = 8;    // 16-byte pieces of channels in a workgroup
constexpr int kRuns = 8;      // runs of a wave: 64 / kPieces
constexpr int kMaxWaves = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNothing = -INFINITY;
constexpr float kTiny = 0x1p-126f, kHuge = 0x1p127f;

template <typename T> constexpr int kN = 16 / sizeof(T);  // channels of a piece

struct RecArgs {
    View x, g, dy;         // [batch, time, channel]
    View valid, reset;     // [batch, time] or null
    View initial;          // [batch, channel] or null
    const float *d_final;  // dense or null
    int64_t T;
    int B, W, slabs;
    int waves, blocks, seg_blocks, segments;
    void *y;               // y, or dx; dense
    void *dg;
    float *final_state;    // final_state, or d_initial
    float *states;         // [block][B][W]: the state before each block
    float *seg_half, *seg_sum;  // [segment][B][W]: half the log2 of its decay, its sum
};

// ---- pieces of a row ------------------------------------------------------------------

template <typename T, int N> struct Piece {
    uint32_t w[N * sizeof(T) / 4];
};

template <typename T, int N> __device__ __forceinline__ float get(const Piece<T, N> &p, int j) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(p.w[j]);
    else return j & 1 ? __uint_as_float(p.w[j >> 1] & 0xFFFF0000u) : __uint_as_float(p.w[j >> 1] << 16);
}

// The first n <= N channels at p, zeros behind them.  UNIT: the channels lie side by side, at any
// address that the type may have.
template <typename T, int N, bool UNIT>
__device__ __forceinline__ void load_piece(Piece<T, N> &r, const T *p, int64_t cs, int n) {
    if (UNIT && n == N) {
        __builtin_memcpy(&r, p, sizeof(r));
        return;
    }
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(T) / 4); ++i) r.w[i] = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (j < n) {
            const T v = p[(UNIT ? 1 : cs) * j];
            if constexpr (sizeof(T) == 4) r.w[j] = __float_as_uint(v);
            else r.w[j >> 1] |= (uint32_t)v << (16 * (j & 1));
        }
}

template <typename T, int N>
__device__ __forceinline__ void store_piece(T *p, const float *v, int n) {
    if (n == N) {
        Piece<T, N> r;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < N; ++j) r.w[j] = __float_as_uint(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < N; j += 2)
                r.w[j >> 1] = (uint32_t)f32_to_bf16(v[j]) | ((uint32_t)f32_to_bf16(v[j + 1]) << 16);
        }
        __builtin_memcpy(p, &r, sizeof(r));
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (j < n) Elem<T>::store(p, j, v[j]);
}

// ---- joining runs ----------------------------------------------------------------------

// The decay of one token: 0 below 2^-126, at most 2^127; log2g is cut to what it uses.
__device__ __forceinline__ float decay_of(float &log2g) {
    log2g = log2g > 127.f ? 127.f : log2g;  // NaN stays
    const float a = __builtin_amdgcn_exp2f(log2g);
    return log2g < -126.f ? 0.f : a;
}

__device__ __forceinline__ float through(float a, float h) { return a == 0.f ? 0.f : a * h; }

// What a run (half the log2 of its decay, -inf if it lets nothing through, and its sum) makes of the
// state before it.
__device__ __forceinline__ float join(float before, float half, float sum) {
    const float r = __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(half), kTiny, kHuge);
    const float t = (before * r) * r;
    return (half == kNothing ? 0.f : t) + sum;
}

// v of the lane D lanes before (UP) or behind this one, id where there is none.
template <int D, bool UP> __device__ __forceinline__ float shifted(float v, float id) {
    const float w = UP ? __shfl_up(v, D) : __shfl_down(v, D);
    const int l = threadIdx.x & 63;
    return (UP ? l >= D : l < 64 - D) ? w : id;
}

template <int N, int D, bool UP> __device__ __forceinline__ void scan_level(float *l, float *s) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float l1 = shifted<D, UP>(l[j], 0.f), s1 = shifted<D, UP>(s[j], 0.f);
        s[j] = join(s1, l[j], s[j]);
        l[j] += l1;
    }
}

// Runs of a wave: on return l, s of everything up to and with this lane's run (from the first run
// on, or, with UP false, from the last one backwards).
template <int N, bool UP> __device__ __forceinline__ void scan_runs(float *l, float *s) {
    scan_level<N, 8, UP>(l, s);
    scan_level<N, 16, UP>(l, s);
    scan_level<N, 32, UP>(l, s);
}

// ---- a lane's run ----------------------------------------------------------------------

struct Place {
    int lane, wave, piece, run;
    int b, seg;
    int c0, n;   // this lane's channels: c0 .. c0 + n
    int c;       // the channel that this lane carries across waves and blocks
    bool owns;   // whether it has one
};

template <typename T> __device__ __forceinline__ Place place(const RecArgs &a) {
    constexpr int N = kN<T>, SLAB = N * kPieces;
    Place p;
    p.lane = threadIdx.x & 63;
    p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    p.piece = p.lane & (kPieces - 1);
    p.run = p.lane / kPieces;
    const unsigned u = blockIdx.x;
    const int slab = u % (unsigned)a.slabs;
    const unsigned rest = u / (unsigned)a.slabs;
    p.b = rest % (unsigned)a.B;
    p.seg = rest / (unsigned)a.B;
    p.c0 = slab * SLAB + p.piece * N;
    p.n = min(max(a.W - p.c0, 0), N);
    p.c = slab * SLAB + (p.lane & (SLAB - 1));
    p.owns = p.lane < SLAB && p.c < a.W;
    return p;
}

template <typename T, int N, bool UNIT>
__device__ __forceinline__ void load_run(Piece<T, N> (&r)[kL], const View &v, const RecArgs &a,
                                         const Place &p, int64_t t) {
    const T *q = (const T *)v.data + p.b * v.s0 + t * v.s1 + (UNIT ? (int64_t)p.c0 : p.c0 * v.s2);
#pragma unroll
    for (int i = 0; i < kL; ++i)
        load_piece<T, N, UNIT>(r[i], q + i * v.s1, v.s2, t + i < a.T ? p.n : 0);
}

struct Masks {
    bool on[kL], cut[kL];
};

__device__ __forceinline__ Masks load_masks(const RecArgs &a, const Place &p, int64_t t) {
    Masks m;
#pragma unroll
    for (int i = 0; i < kL; ++i) {
        m.on[i] = t + i < a.T;
        m.cut[i] = false;
        if (m.on[i] && a.valid.data)
            m.on[i] = ((const float *)a.valid.data)[p.b * a.valid.s0 + (t + i) * a.valid.s1] != 0.f;
        if (m.on[i] && a.reset.data)
            m.cut[i] = ((const float *)a.reset.data)[p.b * a.reset.s0 + (t + i) * a.reset.s1] != 0.f;
    }
    return m;
}

// Decays of a run, and half the log2 of their product: finite, or kNothing.  A gate that is NaN
// counts as 0 there: the sums that it touches are NaN themselves.
template <typename G, int N>
__device__ __forceinline__ void decays(const Piece<G, N> (&g)[kL], const Masks &m, float (&a)[kL][N],
                                       float (&half)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float sum = 0.f;
        bool cut = false;
#pragma unroll
        for (int i = 0; i < kL; ++i) {
            float l = get(g[i], j) * kLog2e;
            float d = decay_of(l);
            d = m.cut[i] ? 0.f : d;
            d = m.on[i] ? d : 1.f;
            l = m.on[i] ? l : 0.f;
            sum += l;
            cut = cut || d == 0.f;
            a[i][j] = d;
        }
        half[j] = cut ? kNothing : sum == sum ? 0.5f * sum : 0.f;
    }
}

// The start state of a segment, in the lanes that own a channel.
__device__ __forceinline__ float start_of(const RecArgs &a, const Place &p, float first, int from,
                                          int to, int step) {
    const int64_t BW = (int64_t)a.B * a.W;
    const int64_t at = (int64_t)p.b * a.W + p.c;
    float st = first;
    for (int s = from; s != to; s += step)
        st = join(st, a.seg_half[s * BW + at], a.seg_sum[s * BW + at]);
    return st;
}

// ---- forward -----------------------------------------------------------------------------

// CARRY: only the segment's (A, S).
template <typename T, typename G, bool UNIT, bool CARRY>
__global__ void __launch_bounds__(64 * kMaxWaves) rec_forward(RecArgs a) {
    constexpr int N = kN<T>, SLAB = N * kPieces;
    __shared__ __align__(16) float tot_l[2][kMaxWaves][SLAB], tot_s[2][kMaxWaves][SLAB];
    __shared__ __align__(16) float in[kMaxWaves][SLAB];
    const Place p = place<T>(a);
    const int BT = a.waves * kRuns * kL;
    const int first = p.seg * a.seg_blocks, last = min(first + a.seg_blocks, a.blocks);
    const int64_t BW = (int64_t)a.B * a.W, at = (int64_t)p.b * a.W + p.c;
    const int ch = p.lane & (SLAB - 1);
    if (CARRY && last == a.blocks) return;  // nothing comes after it

    float state = 0.f, half = 0.f;  // of channel p.c, before the block
    if (!CARRY && p.owns) {
        if (a.initial.data)
            state = ((const float *)a.initial.data)[p.b * a.initial.s0 + p.c * a.initial.s1];
        state = start_of(a, p, state, 0, p.seg, 1);
    }
    int64_t t = (int64_t)first * BT + (p.wave * kRuns + p.run) * kL;
    Piece<T, N> x[kL], xn[kL];
    Piece<G, N> g[kL], gn[kL];
    load_run<T, N, UNIT>(x, a.x, a, p, t);
    load_run<G, N, UNIT>(g, a.g, a, p, t);
    for (int blk = first; blk < last; ++blk, t += BT) {
        const int buf = blk & 1;
        const Masks m = load_masks(a, p, t);
        if (blk + 1 < last) {
            load_run<T, N, UNIT>(xn, a.x, a, p, t + BT);
            load_run<G, N, UNIT>(gn, a.g, a, p, t + BT);
        }
        float d[kL][N], l[N], s[N];
        decays(g, m, d, l);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float h = 0.f;
#pragma unroll
            for (int i = 0; i < kL; ++i) h = through(d[i][j], h) + (m.on[i] ? get(x[i], j) : 0.f);
            s[j] = h;
        }
        scan_runs<N, true>(l, s);
        if (p.run == kRuns - 1) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                tot_l[buf][p.wave][p.piece * N + j] = l[j];
                tot_s[buf][p.wave][p.piece * N + j] = s[j];
            }
        }
        __syncthreads();
        if (!CARRY && a.states && p.wave == 0 && p.owns) a.states[blk * BW + at] = state;
        // The state goes past a block in one step, by the sum of all logarithms.
        float mine = state, all = 0.f, sum = 0.f;
        for (int w = 0; w < a.waves; ++w) {
            const float lw = tot_l[buf][w][ch], sw = tot_s[buf][w][ch];
            if (!CARRY && w < p.wave) mine = join(mine, lw, sw);
            sum = join(sum, lw, sw);
            all += lw;
        }
        state = join(state, all, sum);
        if (CARRY) half += all;
        if (!CARRY) {
            if (p.lane < SLAB) in[p.wave][p.lane] = mine;
            __builtin_amdgcn_wave_barrier();
            // the runs before this lane's in its wave
            float h[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float lb = shifted<8, true>(l[j], 0.f), sb = shifted<8, true>(s[j], 0.f);
                h[j] = join(in[p.wave][p.piece * N + j], lb, sb);
            }
            T *y = (T *)a.y + (p.b * a.T + t) * a.W + p.c0;
#pragma unroll
            for (int i = 0; i < kL; ++i) {
                float o[N];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    h[j] = through(d[i][j], h[j]) + (m.on[i] ? get(x[i], j) : 0.f);
                    o[j] = m.on[i] ? h[j] : 0.f;
                }
                if (t + i < a.T) store_piece<T, N>(y + (int64_t)i * a.W, o, p.n);
            }
        }
#pragma unroll
        for (int i = 0; i < kL; ++i) x[i] = xn[i], g[i] = gn[i];
    }
    if (CARRY) {
        if (p.wave == 0 && p.owns) {
            a.seg_half[p.seg * BW + at] = half;
            a.seg_sum[p.seg * BW + at] = state;
        }
    } else if (p.wave == 0 && p.owns && last == a.blocks) {
        a.final_state[at] = state;
    }
}

// ---- backward ----------------------------------------------------------------------------

template <typename T, typename G, bool UNIT, bool CARRY>
__global__ void __launch_bounds__(64 * kMaxWaves) rec_backward(RecArgs a) {
    constexpr int N = kN<T>, SLAB = N * kPieces;
    __shared__ __align__(16) float tot_l[2][kMaxWaves][SLAB], tot_s[2][kMaxWaves][SLAB],
        tot_e[2][kMaxWaves][SLAB];
    __shared__ __align__(16) float in_h[kMaxWaves][SLAB], in_e[kMaxWaves][SLAB];
    const Place p = place<T>(a);
    const int BT = a.waves * kRuns * kL;
    const int first = p.seg * a.seg_blocks, last = min(first + a.seg_blocks, a.blocks);
    const int64_t BW = (int64_t)a.B * a.W, at = (int64_t)p.b * a.W + p.c;
    const int ch = p.lane & (SLAB - 1);
    if (CARRY && first == 0) return;  // nothing comes before it

    float adj = 0.f, half = 0.f;  // E of channel p.c, behind the block
    if (!CARRY && p.owns) {
        if (a.d_final) adj = a.d_final[at];
        adj = start_of(a, p, adj, a.segments - 1, p.seg, -1);
    }
    int64_t t = (int64_t)(last - 1) * BT + (p.wave * kRuns + p.run) * kL;
    Piece<T, N> x[kL], xn[kL], dy[kL], dyn[kL];
    Piece<G, N> g[kL], gn[kL];
    if (!CARRY) load_run<T, N, UNIT>(x, a.x, a, p, t);
    load_run<G, N, UNIT>(g, a.g, a, p, t);
    load_run<T, N, UNIT>(dy, a.dy, a, p, t);
    for (int blk = last - 1; blk >= first; --blk, t -= BT) {
        const int buf = blk & 1;
        const Masks m = load_masks(a, p, t);
        float state = 0.f;
        if (!CARRY && p.owns) state = a.states[blk * BW + at];
        if (blk > first) {
            if (!CARRY) load_run<T, N, UNIT>(xn, a.x, a, p, t - BT);
            load_run<G, N, UNIT>(gn, a.g, a, p, t - BT);
            load_run<T, N, UNIT>(dyn, a.dy, a, p, t - BT);
        }
        float d[kL][N], l[N], s[N], q[N], e[N];
        decays(g, m, d, l);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float h = 0.f, E = 0.f;
#pragma unroll
            for (int i = 0; i < kL; ++i) {
                if (!CARRY) h = through(d[i][j], h) + (m.on[i] ? get(x[i], j) : 0.f);
                const int k = kL - 1 - i;
                E = through(d[k][j], E + (m.on[k] ? get(dy[k], j) : 0.f));
            }
            s[j] = h, e[j] = E, q[j] = l[j];
        }
        scan_runs<N, false>(q, e);
        if (!CARRY) scan_runs<N, true>(l, s);
        if (p.run == 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                tot_l[buf][p.wave][p.piece * N + j] = q[j];
                tot_e[buf][p.wave][p.piece * N + j] = e[j];
            }
        }
        if (!CARRY && p.run == kRuns - 1) {
#pragma unroll
            for (int j = 0; j < N; ++j) tot_s[buf][p.wave][p.piece * N + j] = s[j];
        }
        __syncthreads();
        float mine_h = state, mine_e = adj, all = 0.f, sum = 0.f;
        for (int w = 0; w < a.waves; ++w) {
            const int v = a.waves - 1 - w;
            const float lv = tot_l[buf][v][ch], ev = tot_e[buf][v][ch];
            if (!CARRY && v > p.wave) mine_e = join(mine_e, lv, ev);
            if (!CARRY && w < p.wave) mine_h = join(mine_h, tot_l[buf][w][ch], tot_s[buf][w][ch]);
            sum = join(sum, lv, ev);
            all += lv;
        }
        adj = join(adj, all, sum);
        if (CARRY) half += all;
        if (!CARRY) {
            if (p.lane < SLAB) in_h[p.wave][p.lane] = mine_h, in_e[p.wave][p.lane] = mine_e;
            __builtin_amdgcn_wave_barrier();
            float carried[kL][N];  // exp(g_t) h_{t-1}
            float E[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float lb = shifted<8, true>(l[j], 0.f), sb = shifted<8, true>(s[j], 0.f);
                float h = join(in_h[p.wave][p.piece * N + j], lb, sb);
#pragma unroll
                for (int i = 0; i < kL; ++i) {
                    carried[i][j] = through(d[i][j], h);
                    h = carried[i][j] + (m.on[i] ? get(x[i], j) : 0.f);
                }
                lb = shifted<8, false>(q[j], 0.f), sb = shifted<8, false>(e[j], 0.f);
                E[j] = join(in_e[p.wave][p.piece * N + j], lb, sb);
            }
            const int64_t o = (p.b * a.T + t) * a.W + p.c0;
#pragma unroll
            for (int i = kL - 1; i >= 0; --i) {
                float ox[N], og[N];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float u = E[j] + (m.on[i] ? get(dy[i], j) : 0.f);
                    ox[j] = m.on[i] ? u : 0.f;
                    og[j] = m.on[i] && d[i][j] != 0.f ? carried[i][j] * u : 0.f;
                    E[j] = through(d[i][j], u);
                }
                if (t + i < a.T) {
                    if (a.y) store_piece<T, N>((T *)a.y + o + (int64_t)i * a.W, ox, p.n);
                    if (a.dg) store_piece<G, N>((G *)a.dg + o + (int64_t)i * a.W, og, p.n);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kL; ++i) x[i] = xn[i], g[i] = gn[i], dy[i] = dyn[i];
    }
    if (CARRY) {
        if (p.wave == 0 && p.owns) {
            a.seg_half[p.seg * BW + at] = half;
            a.seg_sum[p.seg * BW + at] = adj;
        }
    } else if (p.wave == 0 && p.owns && first == 0 && a.final_state) {
        a.final_state[at] = adj;
    }
}

// ---- one token -----------------------------------------------------------------------------

template <typename T, typename G> __global__ void __launch_bounds__(256) rec_step(RecArgs a) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;  // at most 2^30 + 255
    if (i >= (unsigned)a.B * (unsigned)a.W) return;
    const unsigned b = i / (unsigned)a.W, c = i - b * (unsigned)a.W;
    const bool on = !a.valid.data || ((const float *)a.valid.data)[b * a.valid.s0] != 0.f;
    float y = 0.f;
    if (on) {
        const bool cut = a.reset.data && ((const float *)a.reset.data)[b * a.reset.s0] != 0.f;
        float l = Elem<G>::load(a.g.data, b * a.g.s0 + c * a.g.s2) * kLog2e;
        const float d = cut ? 0.f : decay_of(l);
        y = through(d, a.final_state[i]) + Elem<T>::load(a.x.data, b * a.x.s0 + c * a.x.s2);
        a.final_state[i] = y;
    }
    Elem<T>::store(a.y, i, y);
}

// ---- host ------------------------------------------------------------------------------------

// How the time axis is split: a function of the sizes alone, so that both passes agree.
struct Split {
    int slabs, waves, blocks, seg_blocks, segments;
};

constexpr int kWantedGroups = 512;

int check_shape(const gdn2_recurrence_shape *s) {
    if (!s) return fail(GDN2_ERR_ARGUMENT, "shape is null");
    if (s->batch < 1 || s->time < 1 || s->width < 1)
        return fail(GDN2_ERR_SHAPE, "batch, time and width must be nonempty");
    constexpr int64_t most = 1 << 30;
    if (s->batch > most || s->time > most || s->width > most || s->batch * s->width > most)
        return fail(GDN2_ERR_SHAPE, "too many sequences, tokens or channels (2^30 at most)");
    return ok();
}

Split split_of(const gdn2_recurrence_shape *s, int32_t dtype) {
    Split k;
    const int slab = kPieces * (dtype == GDN2_BF16 ? 8 : 4);
    k.slabs = (int)((s->width + slab - 1) / slab);
    k.waves = 1;
    while (k.waves < kMaxWaves && s->time > (int64_t)k.waves * kRuns * kL) k.waves *= 2;
    const int64_t bt = (int64_t)k.waves * kRuns * kL;
    k.blocks = (int)((s->time + bt - 1) / bt);
    const int64_t units = (int64_t)k.slabs * s->batch;
    int64_t segs = units >= kWantedGroups ? 1 : (kWantedGroups + units - 1) / units;
    if (segs > k.blocks) segs = k.blocks;
    k.seg_blocks = (int)((k.blocks + segs - 1) / segs);
    k.segments = (k.blocks + k.seg_blocks - 1) / k.seg_blocks;
    return k;
}

size_t state_bytes(const gdn2_recurrence_shape *s) { return (size_t)4 * s->batch * s->width; }

// Decays and sums of the segments.
size_t segment_bytes(const gdn2_recurrence_shape *s, const Split &k) {
    return k.segments > 1 ? 2 * k.segments * state_bytes(s) : 0;
}

int check_dtype(int32_t dtype) {
    if (dtype != GDN2_F32 && dtype != GDN2_BF16)
        return fail(GDN2_ERR_DTYPE, "dtype must be F32 or BF16 (got %d)", (int)dtype);
    return ok();
}

int check_inputs(const gdn2_recurrence_shape *s, const gdn2_view *x, const gdn2_view *g,
                 const gdn2_view *valid, const gdn2_view *reset) {
    GDN2_TRY(check_shape(s));
    GDN2_TRY(check_view(x, "x", -1, false));
    GDN2_TRY(check_view(g, "g", -1, false));
    if (valid) GDN2_TRY(check_view(valid, "valid", GDN2_F32, true));
    if (reset) GDN2_TRY(check_view(reset, "reset", GDN2_F32, true));
    return ok();
}

RecArgs make_args(const gdn2_recurrence_shape *s, const Split &k, const gdn2_view *x,
                  const gdn2_view *g, const gdn2_view *valid, const gdn2_view *reset) {
    RecArgs a{};
    a.x = make_view(x), a.g = make_view(g);
    a.valid = make_view(valid), a.reset = make_view(reset);
    a.T = s->time, a.B = (int)s->batch, a.W = (int)s->width;
    a.slabs = k.slabs, a.waves = k.waves, a.blocks = k.blocks;
    a.seg_blocks = k.seg_blocks, a.segments = k.segments;
    return a;
}

int check_buffer(const char *name, const void *p, size_t have, size_t need) {
    if (need && (!p || have < need))
        return fail(GDN2_ERR_WORKSPACE, "%s is too small: %zu bytes needed", name, need);
    if ((uintptr_t)p & 15) return fail(GDN2_ERR_ARGUMENT, "%s must be 16-byte aligned", name);
    return ok();
}

int grid_of(const RecArgs &a, int segments, unsigned *out) {
    const int64_t n = (int64_t)a.slabs * a.B * segments;
    if (n > 0x7FFFFFFF) return fail(GDN2_ERR_SHAPE, "too many sequences or channels");
    *out = (unsigned)n;
    return ok();
}

template <typename T, typename G, bool UNIT>
void launch_rec(const RecArgs &a, bool backward, bool carry, unsigned grid, hipStream_t st) {
    const dim3 block(64 * a.waves);
    if (backward) {
        if (carry) hipLaunchKernelGGL((rec_backward<T, G, UNIT, true>), dim3(grid), block, 0, st, a);
        else hipLaunchKernelGGL((rec_backward<T, G, UNIT, false>), dim3(grid), block, 0, st, a);
    } else {
        if (carry) hipLaunchKernelGGL((rec_forward<T, G, UNIT, true>), dim3(grid), block, 0, st, a);
        else hipLaunchKernelGGL((rec_forward<T, G, UNIT, false>), dim3(grid), block, 0, st, a);
    }
}

template <bool UNIT>
void launch_types(const RecArgs &a, int32_t dtype, int32_t gtype, bool backward, bool carry,
                  unsigned grid, hipStream_t st) {
    if (dtype == GDN2_BF16) {
        if (gtype == GDN2_BF16) launch_rec<bf16_t, bf16_t, UNIT>(a, backward, carry, grid, st);
        else launch_rec<bf16_t, float, UNIT>(a, backward, carry, grid, st);
    } else {
        if (gtype == GDN2_BF16) launch_rec<float, bf16_t, UNIT>(a, backward, carry, grid, st);
        else launch_rec<float, float, UNIT>(a, backward, carry, grid, st);
    }
}

int launch_all(const RecArgs &a, int32_t dtype, int32_t gtype, bool backward, void *stream,
               const char *what) {
    unsigned grid;
    GDN2_TRY(grid_of(a, a.segments, &grid));
    const bool unit = a.x.s2 == 1 && a.g.s2 == 1 && (!backward || a.dy.s2 == 1);
    for (int carry = a.segments > 1 ? 1 : 0; carry >= 0; --carry) {
        if (unit) launch_types<true>(a, dtype, gtype, backward, carry, grid, (hipStream_t)stream);
        else launch_types<false>(a, dtype, gtype, backward, carry, grid, (hipStream_t)stream);
    }
    return launch_status(hipGetLastError(), what);
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_recurrence_checkpoint_bytes(const gdn2_recurrence_shape *shape, int32_t dtype, int train) {
    if (check_shape(shape) || check_dtype(dtype)) return 0;
    const Split k = split_of(shape, dtype);
    const size_t n = segment_bytes(shape, k) + (train ? k.blocks * state_bytes(shape) : 0);
    return n ? n : 16;
}

int gdn2_recurrence_scan(const gdn2_recurrence_shape *shape, const gdn2_view *x, const gdn2_view *g,
                         const gdn2_view *valid, const gdn2_view *reset, const gdn2_view *initial,
                         void *output, float *final_state, int train, void *checkpoint,
                         size_t checkpoint_bytes, void *stream) {
    GDN2_TRY(check_inputs(shape, x, g, valid, reset));
    if (initial) GDN2_TRY(check_view(initial, "initial", GDN2_F32, true));
    if (!output || !final_state) return fail(GDN2_ERR_ARGUMENT, "output and final_state must be non-null");
    GDN2_TRY(check_buffer("checkpoint", checkpoint, checkpoint_bytes,
                          gdn2_recurrence_checkpoint_bytes(shape, x->dtype, train)));
    const Split k = split_of(shape, x->dtype);
    RecArgs a = make_args(shape, k, x, g, valid, reset);
    a.initial = make_view(initial);
    a.y = output, a.final_state = final_state;
    float *ck = (float *)checkpoint;
    if (k.segments > 1) {
        a.seg_half = ck, a.seg_sum = ck + segment_bytes(shape, k) / 8;
        ck += segment_bytes(shape, k) / 4;
    }
    if (train) a.states = ck;
    return launch_all(a, x->dtype, g->dtype, false, stream, "gdn2_recurrence_scan");
}

size_t gdn2_recurrence_workspace_bytes(const gdn2_recurrence_shape *shape, int32_t dtype) {
    if (check_shape(shape) || check_dtype(dtype)) return 0;
    const size_t n = segment_bytes(shape, split_of(shape, dtype));
    return n ? n : 16;
}

int gdn2_recurrence_backward(const gdn2_recurrence_shape *shape, const gdn2_view *x,
                             const gdn2_view *g, const gdn2_view *valid, const gdn2_view *reset,
                             const void *checkpoint, size_t checkpoint_bytes,
                             const gdn2_view *d_output, const float *d_final_state, void *dx,
                             void *dg, float *d_initial, void *workspace, size_t workspace_bytes,
                             void *stream) {
    GDN2_TRY(check_inputs(shape, x, g, valid, reset));
    GDN2_TRY(check_view(d_output, "d_output", x->dtype, false));
    GDN2_TRY(check_buffer("checkpoint", checkpoint, checkpoint_bytes,
                          gdn2_recurrence_checkpoint_bytes(shape, x->dtype, 1)));
    GDN2_TRY(check_buffer("workspace", workspace, workspace_bytes,
                          gdn2_recurrence_workspace_bytes(shape, x->dtype)));
    const Split k = split_of(shape, x->dtype);
    RecArgs a = make_args(shape, k, x, g, valid, reset);
    a.dy = make_view(d_output);
    a.d_final = d_final_state;
    a.y = dx, a.dg = dg, a.final_state = d_initial;
    a.states = (float *)checkpoint + segment_bytes(shape, k) / 4;
    if (k.segments > 1) {
        a.seg_half = (float *)workspace;
        a.seg_sum = a.seg_half + segment_bytes(shape, k) / 8;
    }
    return launch_all(a, x->dtype, g->dtype, true, stream, "gdn2_recurrence_backward");
}

int gdn2_recurrence_step(const gdn2_recurrence_shape *shape, const gdn2_view *x, const gdn2_view *g,
                         const gdn2_view *valid, const gdn2_view *reset, float *state, void *output,
                         void *stream) {
    GDN2_TRY(check_inputs(shape, x, g, valid, reset));
    if (shape->time != 1) return fail(GDN2_ERR_SHAPE, "the step takes one token (time == 1)");
    if (!state || !output) return fail(GDN2_ERR_ARGUMENT, "state and output must be non-null");
    RecArgs a = make_args(shape, split_of(shape, x->dtype), x, g, valid, reset);
    a.final_state = state, a.y = output;
    const dim3 grid((unsigned)(((int64_t)a.B * a.W + 255) / 256)), block(256);
    hipStream_t st = (hipStream_t)stream;
    if (x->dtype == GDN2_BF16) {
        if (g->dtype == GDN2_BF16) hipLaunchKernelGGL((rec_step<bf16_t, bf16_t>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((rec_step<bf16_t, float>), grid, block, 0, st, a);
    } else {
        if (g->dtype == GDN2_BF16) hipLaunchKernelGGL((rec_step<float, bf16_t>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((rec_step<float, float>), grid, block, 0, st, a);
    }
    return launch_status(hipGetLastError(), "gdn2_recurrence_step");
}

}  // extern "C"
