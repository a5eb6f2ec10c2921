// Gated linear recurrence on gfx950: forward, backward and the single-token step.
//
//   h_t = exp(g_t) h_{t-1} + x_t,  y_t = h_t                      per channel of [B, T, W]
//   e_t = dy_t + E_{t+1},  E_t = exp(g_t) e_t                     the adjoint, from the last token
//   dx_t = e_t,  dg_t = exp(g_t) h_{t-1} e_t,  d_initial = E_1
//
// A run of tokens acts on the state before it as S + A h, and joining two runs needs only their
// (A, S): the time axis is split over lanes, waves, and, where there are few channels, workgroups.
//   * A workgroup has 64 bytes of channels (32 bf16, 16 f32) and 1 to 8 waves; the two that share a
//     128-byte line go to one XCD, whose L2 reads it once (halves rather than lines: twice the
//     workgroups, 306 us against 443 at 4 x 8192 tokens of 2048 channels, where lines have 128).  A lane
//     has 8 bytes of channels of some tokens in a row, a wave 8 such runs for each of its 8 pieces, a
//     block is what all waves hold.  Every tensor is read and written once.
//   * Inside a block: each lane its own run, the 8 runs of a wave by lane exchanges, the waves
//     through LDS (one barrier a block); then each lane walks its run again from its true state.
//   * Segments: if there are too few workgroups the blocks of a sequence go to several.  A first
//     kernel makes each segment's (A, S), and every segment starts from the joined ones before it:
//     the inputs are read twice, by kernels that fill the card.
// The backward recomputes the states of a block from the state before it, which the forward kept
// (4 bytes a channel for every block), and walks the blocks from the last.
//
// 4 x 8192 tokens of 2048 channels, bf16: forward 122 us, 3.3 TB/s, backward 204.  A block takes 25
// instructions a value, 10 of them the recurrence's own, at two waves a SIMD: 46 % of the time the vector
// units work.  The next block's loads are issued before a block is worked on, but as compiled they are
// waited for before its first multiplication (on entry to the loop the first block's may still be pending,
// and the last block has none behind it), so loads, work and stores of a block follow each other.  It shows
// least where several workgroups share a CU.
//
// A is carried as half its log2 and its root applied twice, clamped to [2^-126, 2^127]: a state of
// any size meets a decay of any size as it would token by token, zero stays zero, and what is not
// finite stays so.  Logarithms add up almost exactly, so a slow decay is rounded once for what a
// state passes in one step (a block), not once a token.  Half = -inf means that nothing gets through:
// a reset, or a gate whose exp is below 2^-126.  There a state is dropped, not multiplied, so that
// what is not finite does not pass.
#include <math.h>

#include <type_traits>

#include "gdn2_common.h"
#include "gdn2_status.h"

// Sums of products are fused where it says fmaf and nowhere else: a wave that takes the way for gates that
// need care gives the bits that it would give without them.
#pragma clang fp contract(off)

namespace gdn2 {
namespace {

constexpr int kMaxWaves = 8;
constexpr int kSlabBytes = 64;  // of a token, a workgroup's channels
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNothing = -INFINITY;
constexpr float kTiny = 0x1p-126f, kHuge = 0x1p127f;

// A lane has 8 bytes of 8 tokens in bf16, of 4 in f32: with runs twice as long registers run out, with
// half as many tokens a block's joining is half of its instructions (4 x 8192 tokens of 2048 channels,
// bf16, forward and backward: 306 us, with runs of 4 tokens 362, with 4-byte pieces of 16 tokens 321).
// WAVES: those of a workgroup, at most.
template <typename T, int W = kMaxWaves> struct Cfg {
    static constexpr int WAVES = W;
    static constexpr int N = 8 / sizeof(T);               // channels of a lane
    static constexpr int L = sizeof(T) == 2 ? 8 : 4;      // tokens of a lane's run
    static constexpr int SLAB = kSlabBytes / sizeof(T);   // channels of a workgroup
    static constexpr int PIECES = SLAB / N, RUNS = 64 / PIECES;
    static constexpr int TOKENS = RUNS * L;               // of a wave
};

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

template <typename T, int N> __device__ __forceinline__ void set(Piece<T, N> &p, const float *v) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < N; ++j) p.w[j] = __float_as_uint(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 2)
            p.w[j >> 1] = (uint32_t)f32_to_bf16(v[j]) | ((uint32_t)f32_to_bf16(v[j + 1]) << 16);
    }
}

// ---- joining runs ----------------------------------------------------------------------

__device__ __forceinline__ float root_of(float half) {
    return __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(half), kTiny, kHuge);
}

// What a run (the root of its decay, 0 if it lets nothing through, and its sum) makes of the state
// before it.
__device__ __forceinline__ float join_root(float before, float r, float sum) {
    const float t = fmaf(before * r, r, sum);
    return r == 0.f ? sum : t;
}

// The same by half the log2 of the decay, kNothing for 0.  CUT: there may be such runs.
template <bool CUT> __device__ __forceinline__ float join(float before, float half, float sum) {
    const float r = root_of(half), t = fmaf(before * r, r, sum);
    return CUT && half == kNothing ? sum : t;
}

// v of the lane D lanes before (UP) or behind this one, 0 where there is none.
template <int D, bool UP> __device__ __forceinline__ float shifted(float v) {
    const float w = UP ? __shfl_up(v, D) : __shfl_down(v, D);
    const int l = threadIdx.x & 63;
    return (UP ? l >= D : l < 64 - D) ? w : 0.f;
}

template <int N, int D, bool UP, bool CUT> __device__ __forceinline__ void scan_level(float *l, float *s) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float l1 = shifted<D, UP>(l[j]), s1 = shifted<D, UP>(s[j]);
        s[j] = join<CUT>(s1, l[j], s[j]);
        l[j] += l1;
    }
}

// Runs of a wave: on return l, s of everything up to and with this lane's run (from the first run
// on, or, with UP false, from the last one backwards).
template <typename C, bool UP, bool CUT> __device__ __forceinline__ void scan_runs(float *l, float *s) {
    if constexpr (C::PIECES <= 4) scan_level<C::N, 4, UP, CUT>(l, s);
    if constexpr (C::PIECES <= 8) scan_level<C::N, 8, UP, CUT>(l, s);
    if constexpr (C::PIECES <= 16) scan_level<C::N, 16, UP, CUT>(l, s);
    if constexpr (C::PIECES <= 32) scan_level<C::N, 32, UP, CUT>(l, s);
}

// ---- a lane's run ----------------------------------------------------------------------

struct Place {
    int lane, wave, piece, run;
    int b, seg;
    int slab0, c0;  // the slab's channels, and this lane's
    int own0;    // the first channel that this workgroup answers for
    int ch, c;   // the channel of the slab, and its number, that this lane carries across waves and blocks
    bool there;  // whether there is one; lanes beyond the slab's channels carry the same ones again
    bool owns;   // whether this lane answers for it
};

// WHOLE: a slab that would reach past the last channel begins earlier; what it shares with the slab
// before it is that one's.
template <typename C, bool WHOLE> __device__ __forceinline__ Place place(const RecArgs &a) {
    Place p;
    p.lane = threadIdx.x & 63;
    p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    p.piece = p.lane & (C::PIECES - 1);
    p.run = p.lane / C::PIECES;
    // Slabs that share 128-byte lines to one XCD: workgroups go to the eight in turn.
    constexpr unsigned G = 128 / kSlabBytes;
    unsigned u = blockIdx.x;
    if (G > 1 && u < gridDim.x / (8 * G) * (8 * G)) {
        const unsigned q = u / (8 * G), r = u % (8 * G);
        u = (q * 8 + r % 8) * G + r / 8;
    }
    const int slab = u % (unsigned)a.slabs;
    const unsigned rest = u / (unsigned)a.slabs;
    p.b = rest % (unsigned)a.B;
    p.seg = rest / (unsigned)a.B;
    p.own0 = slab * C::SLAB;
    p.slab0 = WHOLE ? min(p.own0, a.W - C::SLAB) : p.own0;
    p.c0 = p.slab0 + p.piece * C::N;
    p.ch = p.lane & (C::SLAB - 1);
    p.c = p.slab0 + p.ch;
    p.there = p.c < a.W;
    p.owns = p.lane < C::SLAB && p.c >= p.own0 && p.there;
    return p;
}

// kL tokens of this lane's channels from token t on, t = wave's first token + run kL.  What lies behind
// the last token or channel is read as the last: a lane with such tokens leaves them out, and one with
// such channels writes none.  WHOLE: side by side and near, by a uniform address and a lane's offset.
// Otherwise a load for each value, and the bf16 backward of 8 waves keeps 16 to 19 registers in memory: 16 x 4096
// tokens of 1024 channels, bf16, with tokens side by side forward 262 us for 121 and backward 400 for 194, where a
// copy of one tensor takes 264; with an expanded upstream gradient backward 358.
template <bool WHOLE, typename T, int N, int kL>
__device__ __forceinline__ void load_run(Piece<T, N> (&r)[kL], const View &v, const RecArgs &a,
                                         const Place &p, int64_t first, bool inside) {
    const T *q = (const T *)v.data + p.b * v.s0;
    if (WHOLE) {
        const int64_t from = min(first, a.T - 1);
        const char *base = (const char *)(q + from * v.s1 + p.slab0);
        const uint32_t row = (uint32_t)v.s1 * sizeof(T), piece = p.piece * (N * sizeof(T));
        if (inside) {
            const uint32_t off = p.run * kL * row + piece;
#pragma unroll
            for (int i = 0; i < kL; ++i) __builtin_memcpy(&r[i], base + (int64_t)i * row + off, sizeof(r[i]));
        } else {
            const int most = (int)min(a.T - 1 - from, (int64_t)(64 * kL));
#pragma unroll
            for (int i = 0; i < kL; ++i) {
                const uint32_t off = (uint32_t)min(p.run * kL + i, most) * row + piece;
                __builtin_memcpy(&r[i], base + off, sizeof(r[i]));
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kL; ++i) {
        const T *row = q + min(first + p.run * kL + i, a.T - 1) * v.s1;
#pragma unroll
        for (int k = 0; k < (int)(N * sizeof(T) / 4); ++k) r[i].w[k] = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const T e = row[min(p.c0 + j, a.W - 1) * v.s2];
            if constexpr (sizeof(T) == 4) r[i].w[j] = __float_as_uint(e);
            else r[i].w[j >> 1] |= (uint32_t)e << (16 * (j & 1));
        }
    }
}

// Token first + run L + i of a dense result.
template <bool WHOLE, int L, typename T, int N>
__device__ __forceinline__ void store_piece(void *out, const RecArgs &a, const Place &p, int64_t first, int i,
                                            const float *v) {
    if (WHOLE) {
        char *base = (char *)((T *)out + (p.b * a.T + first + i) * a.W + p.slab0);
        T *q = (T *)(base + (uint32_t)((p.run * L * a.W + p.piece * N) * (int)sizeof(T)));
        if (p.slab0 == p.own0 || p.c0 >= p.own0) {
            Piece<T, N> r;
            set(r, v);
            __builtin_memcpy(q, &r, sizeof(r));
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (p.c0 + j >= p.own0) Elem<T>::store(q, j, v[j]);
        }
        return;
    }
    T *q = (T *)out + (p.b * a.T + first + p.run * L + i) * a.W + p.c0;
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (p.c0 + j < a.W) Elem<T>::store(q, j, v[j]);
}

// Bit i: token i of the run counts, and it is a reset.
struct Masks {
    uint32_t on, cut;
};

// A load and a wait for each token and mask.  16 x 4096 tokens of 1024 channels, bf16, forward and backward: 315 us
// without masks, 367 with a valid of ones alone, 441 with padding and resets (whose blocks take the longer way).
template <int kL> __device__ __forceinline__ Masks load_masks(const RecArgs &a, const Place &p, int64_t first) {
    const int64_t t = first + p.run * kL;
    Masks m = {0, 0};
#pragma unroll
    for (int i = 0; i < kL; ++i) {
        const int64_t at = min(t + i, a.T - 1);
        bool on = t + i < a.T, cut = false;
        if (a.valid.data) on = on && ((const float *)a.valid.data)[p.b * a.valid.s0 + at * a.valid.s1] != 0.f;
        if (a.reset.data) cut = ((const float *)a.reset.data)[p.b * a.reset.s0 + at * a.reset.s1] != 0.f;
        m.on |= (uint32_t)on << i, m.cut |= (uint32_t)(on && cut) << i;
    }
    return m;
}

// Decays of a run, and half the log2 of their product: finite, or kNothing.  A gate that is NaN
// counts as 0 there: the sums that it touches are NaN themselves.  True if a wave's decays need no
// care: all tokens count, all gates are numbers, between 2^-126 and 2^127.
template <bool MASKED, typename G, int N, int kL>
__device__ __forceinline__ bool decays(const Piece<G, N> (&g)[kL], const Masks &m, float (&d)[kL][N],
                                       float (&half)[N]) {
    float lo = 0.f, hi = 0.f, all = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        half[j] = 0.f;
#pragma unroll
        for (int i = 0; i < kL; ++i) {
            const float l = get(g[i], j) * kLog2e;
            d[i][j] = l;
            half[j] += l;
            lo = fminf(lo, l), hi = fmaxf(hi, l);
        }
        all += half[j];
        half[j] *= 0.5f;
    }
    const bool care = !(lo >= -126.f && hi <= 127.f && all == all) ||
                      (MASKED && ((m.on & ((1u << kL) - 1)) != (1u << kL) - 1 || m.cut));
    if (!__any(care)) {
#pragma unroll
        for (int i = 0; i < kL; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) d[i][j] = __builtin_amdgcn_exp2f(d[i][j]);
        return true;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float sum = 0.f;
        bool cut = false;
#pragma unroll
        for (int i = 0; i < kL; ++i) {
            float l = d[i][j];
            l = l > 127.f ? 127.f : l;  // NaN stays
            float v = l < -126.f || (m.cut >> i & 1) ? 0.f : __builtin_amdgcn_exp2f(l);
            const bool on = m.on >> i & 1;
            d[i][j] = v = on ? v : 1.f;
            sum += on ? l : 0.f;
            cut = cut || v == 0.f;
        }
        half[j] = cut ? kNothing : sum == sum ? 0.5f * sum : 0.f;
    }
    return false;
}

// d h + x, or x where nothing gets through.
template <bool PLAIN> __device__ __forceinline__ float next_state(float d, float h, float x) {
    const float t = fmaf(d, h, x);
    return !PLAIN && d == 0.f ? x : t;
}

template <bool PLAIN> __device__ __forceinline__ float through(float d, float h) {
    return !PLAIN && d == 0.f ? 0.f : d * h;
}

// Value j of token i, 0 if the token does not count.
template <bool PLAIN, typename T, int N, int kL>
__device__ __forceinline__ float value(const Piece<T, N> (&x)[kL], const Masks &m, int i, int j) {
    return PLAIN || (m.on >> i & 1) ? get(x[i], j) : 0.f;
}

// The start state of a segment: two loads and a wait for each one before it.  One sequence of 32768 tokens of 32
// to 128 channels, bf16, in 64 segments takes 31 us forward and 35 backward, whose bytes take 1 to 9.
__device__ __forceinline__ float start_of(const RecArgs &a, const Place &p, float first, int from,
                                          int to, int step) {
    const int64_t BW = (int64_t)a.B * a.W;
    const int64_t at = (int64_t)p.b * a.W + p.c;
    float st = first;
    for (int s = from; s != to; s += step)
        st = join<true>(st, a.seg_half[s * BW + at], a.seg_sum[s * BW + at]);
    return st;
}

// What the waves tell each other of a block, twice: a wave that is a block ahead writes the other half.
// Waves that the workgroup does not have let everything through and add nothing.
template <typename C> struct Totals {
    float half[2][C::WAVES][C::SLAB], root[2][C::WAVES][C::SLAB], sum[2][C::WAVES][C::SLAB];
    float in[C::WAVES][C::SLAB];  // the state before each wave's tokens

    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < 2 * C::WAVES * C::SLAB; i += blockDim.x)
            (&half[0][0][0])[i] = 0.f, (&root[0][0][0])[i] = 1.f, (&sum[0][0][0])[i] = 0.f;
    }
    __device__ __forceinline__ void put(int buf, const Place &p, const float *l, const float *s) {
#pragma unroll
        for (int j = 0; j < C::N; ++j) {
            const int c = p.piece * C::N + j;
            half[buf][p.wave][c] = l[j];
            root[buf][p.wave][c] = l[j] == kNothing ? 0.f : root_of(l[j]);
            sum[buf][p.wave][c] = s[j];
        }
    }
    // This lane's channel: the state before its wave's tokens to `in`, and past all waves.  UP: waves in
    // order, or from the last.  A state goes past a block in one step, by the sum of all logarithms.
    template <bool UP> __device__ __forceinline__ float pass(int buf, const Place &p, float state, float *all_out) {
        float r[C::WAVES], s[C::WAVES], all = 0.f, total = 0.f, mine = state;
#pragma unroll
        for (int k = 0; k < C::WAVES; ++k) {
            const int w = UP ? k : C::WAVES - 1 - k;
            r[k] = root[buf][w][p.ch], s[k] = sum[buf][w][p.ch], all += half[buf][w][p.ch];
        }
#pragma unroll
        for (int k = 0; k < C::WAVES; ++k) {
            const int w = UP ? k : C::WAVES - 1 - k;
            const float before = mine;
            mine = join_root(mine, r[k], s[k]);
            if (w == p.wave) in[p.wave][p.ch] = before;
            total = join_root(total, r[k], s[k]);
        }
        __builtin_amdgcn_wave_barrier();
        *all_out = all;
        return join<true>(state, all, total);
    }
};

// ---- forward -----------------------------------------------------------------------------

// A block: the runs' sums, what passes from wave to wave, and the states.
template <typename T, typename G, bool WHOLE, bool CARRY, bool MASKED, typename C>
__device__ __forceinline__ void forward_block(const RecArgs &a, const Place &p, Totals<C> &tot, int buf, int64_t t,
                                              const Piece<T, C::N> (&x)[C::L], const Piece<G, C::N> (&g)[C::L],
                                              const Masks &m, float &state, float &half) {
    constexpr int N = C::N, L = C::L;
    float d[L][N], l[N], s[N];
    const bool plain = decays<MASKED>(g, m, d, l);
    auto sums = [&](auto flag) {
        constexpr bool PLAIN = decltype(flag)::value;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float h = 0.f;
#pragma unroll
            for (int i = 0; i < L; ++i) h = next_state<PLAIN>(d[i][j], h, value<PLAIN>(x, m, i, j));
            s[j] = h;
        }
        scan_runs<C, true, !PLAIN>(l, s);
    };
    if (plain) sums(std::true_type{});
    else sums(std::false_type{});
    if (p.run == C::RUNS - 1) tot.put(buf, p, l, s);
    __syncthreads();
    float all;
    state = tot.template pass<true>(buf, p, state, &all);
    if (CARRY) {
        half += all;
        return;
    }
    auto states = [&](auto flag) {
        constexpr bool PLAIN = decltype(flag)::value;
        float h[N];
#pragma unroll
        for (int j = 0; j < N; ++j)  // past the runs before this lane's in its wave
            h[j] = join<!PLAIN>(tot.in[p.wave][p.piece * N + j], shifted<C::PIECES, true>(l[j]),
                                shifted<C::PIECES, true>(s[j]));
#pragma unroll
        for (int i = 0; i < L; ++i) {
            float o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                h[j] = next_state<PLAIN>(d[i][j], h[j], value<PLAIN>(x, m, i, j));
                o[j] = PLAIN || (m.on >> i & 1) ? h[j] : 0.f;
            }
            if (!MASKED || t + p.run * L + i < a.T) store_piece<WHOLE, L, T, N>(a.y, a, p, t, i, o);
        }
    };
    if (plain) states(std::true_type{});
    else states(std::false_type{});
}

template <typename T, typename G, bool WHOLE, bool CARRY, typename C>
__device__ __forceinline__ void forward_walk(const RecArgs &a, const Place &p, Totals<C> &tot) {
    constexpr int N = C::N, L = C::L;
    const int BT = a.waves * C::TOKENS;
    const int first = p.seg * a.seg_blocks, last = min(first + a.seg_blocks, a.blocks);
    const int64_t BW = (int64_t)a.B * a.W, at = (int64_t)p.b * a.W + p.c;
    const bool masks = a.valid.data || a.reset.data;
    float state = 0.f, half = 0.f;  // of channel p.c, before the block
    if (!CARRY && p.there) {
        if (a.initial.data)
            state = ((const float *)a.initial.data)[p.b * a.initial.s0 + p.c * a.initial.s1];
        state = start_of(a, p, state, 0, p.seg, 1);
    }
    int64_t t = (int64_t)first * BT + p.wave * C::TOKENS;  // this wave's first token
    auto inside = [&](int blk) { return (int64_t)(blk + 1) * BT <= a.T; };
    Piece<T, N> x[L], xn[L];
    Piece<G, N> g[L], gn[L];
    load_run<WHOLE>(x, a.x, a, p, t, inside(first));
    load_run<WHOLE>(g, a.g, a, p, t, inside(first));
    for (int blk = first; blk < last; ++blk, t += BT) {
        if (blk + 1 < last) {
            load_run<WHOLE>(xn, a.x, a, p, t + BT, inside(blk + 1));
            load_run<WHOLE>(gn, a.g, a, p, t + BT, inside(blk + 1));
        }
        if (!CARRY && a.states && p.wave == 0 && p.owns) a.states[blk * BW + at] = state;
        if (masks || !inside(blk))
            forward_block<T, G, WHOLE, CARRY, true>(a, p, tot, blk & 1, t, x, g, load_masks<L>(a, p, t), state, half);
        else
            forward_block<T, G, WHOLE, CARRY, false>(a, p, tot, blk & 1, t, x, g, Masks{~0u, 0}, state, half);
#pragma unroll
        for (int i = 0; i < L; ++i) x[i] = xn[i], g[i] = gn[i];
    }
    if (p.wave != 0 || !p.owns) return;
    if (CARRY) {
        a.seg_half[p.seg * BW + at] = half;
        a.seg_sum[p.seg * BW + at] = state;
    } else if (last == a.blocks) {
        a.final_state[at] = state;
    }
}

// CARRY: only the segment's decay and sum.
template <typename T, typename G, bool WHOLE, bool CARRY, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) rec_forward(RecArgs a) {
    using C = Cfg<T, WAVES>;
    __shared__ __align__(16) Totals<C> tot;
    const Place p = place<C, WHOLE>(a);
    if (CARRY && p.seg == a.segments - 1) return;  // nothing comes after it
    tot.clear();
    __syncthreads();
    forward_walk<T, G, WHOLE, CARRY>(a, p, tot);
}

// ---- backward ----------------------------------------------------------------------------

template <typename T, typename G, bool WHOLE, bool CARRY, bool MASKED, typename C>
__device__ __forceinline__ void backward_block(const RecArgs &a, const Place &p, Totals<C> &fwd, Totals<C> &bwd,
                                               int buf, int64_t t, const Piece<T, C::N> (&x)[C::L],
                                               const Piece<G, C::N> (&g)[C::L], const Piece<T, C::N> (&dy)[C::L],
                                               const Masks &m, float state, float &adj, float &half) {
    constexpr int N = C::N, L = C::L;
    float d[L][N], l[N], s[N], q[N], e[N];
    const bool plain = decays<MASKED>(g, m, d, l);
    auto sums = [&](auto flag) {
        constexpr bool PLAIN = decltype(flag)::value;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float h = 0.f, u = value<PLAIN>(dy, m, L - 1, j);
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (!CARRY) h = next_state<PLAIN>(d[i][j], h, value<PLAIN>(x, m, i, j));
                const int k = L - 1 - i;
                if (k) u = next_state<PLAIN>(d[k][j], u, value<PLAIN>(dy, m, k - 1, j));
            }
            const float E = through<PLAIN>(d[0][j], u);
            s[j] = h, e[j] = E, q[j] = l[j];
        }
        scan_runs<C, false, !PLAIN>(q, e);
        if (!CARRY) scan_runs<C, true, !PLAIN>(l, s);
    };
    if (plain) sums(std::true_type{});
    else sums(std::false_type{});
    if (p.run == 0) bwd.put(buf, p, q, e);
    if (!CARRY && p.run == C::RUNS - 1) fwd.put(buf, p, l, s);
    __syncthreads();
    float all;
    if (!CARRY) fwd.template pass<true>(buf, p, state, &all);
    adj = bwd.template pass<false>(buf, p, adj, &all);
    if (CARRY) {
        half += all;
        return;
    }
    auto grads = [&](auto flag) {
        constexpr bool PLAIN = decltype(flag)::value;
        float carried[L][N], u[N];  // exp(g_t) h_{t-1}, the adjoint
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float h = join<!PLAIN>(fwd.in[p.wave][p.piece * N + j], shifted<C::PIECES, true>(l[j]),
                                   shifted<C::PIECES, true>(s[j]));
#pragma unroll
            for (int i = 0; i < L; ++i) {
                carried[i][j] = through<PLAIN>(d[i][j], h);
                h = next_state<PLAIN>(d[i][j], h, value<PLAIN>(x, m, i, j));
            }
            const float E = join<!PLAIN>(bwd.in[p.wave][p.piece * N + j], shifted<C::PIECES, false>(q[j]),
                                         shifted<C::PIECES, false>(e[j]));
            u[j] = E + value<PLAIN>(dy, m, L - 1, j);
        }
#pragma unroll
        for (int i = L - 1; i >= 0; --i) {
            const bool on = PLAIN || (m.on >> i & 1);
            float ox[N], og[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                ox[j] = on ? u[j] : 0.f;
                og[j] = on && (PLAIN || d[i][j] != 0.f) ? carried[i][j] * u[j] : 0.f;
                if (i) u[j] = next_state<PLAIN>(d[i][j], u[j], value<PLAIN>(dy, m, i - 1, j));
            }
            if (!MASKED || t + p.run * L + i < a.T) {
                if (a.y) store_piece<WHOLE, L, T, N>(a.y, a, p, t, i, ox);
                if (a.dg) store_piece<WHOLE, L, G, N>(a.dg, a, p, t, i, og);
            }
        }
    };
    if (plain) grads(std::true_type{});
    else grads(std::false_type{});
}

template <typename T, typename G, bool WHOLE, bool CARRY, typename C>
__device__ __forceinline__ void backward_walk(const RecArgs &a, const Place &p, Totals<C> &fwd, Totals<C> &bwd) {
    constexpr int N = C::N, L = C::L;
    const int BT = a.waves * C::TOKENS;
    const int first = p.seg * a.seg_blocks, last = min(first + a.seg_blocks, a.blocks);
    const int64_t BW = (int64_t)a.B * a.W, at = (int64_t)p.b * a.W + p.c;
    const bool masks = a.valid.data || a.reset.data;
    float adj = 0.f, half = 0.f;  // E of channel p.c, behind the block
    if (!CARRY && p.there) {
        if (a.d_final) adj = a.d_final[at];
        adj = start_of(a, p, adj, a.segments - 1, p.seg, -1);
    }
    int64_t t = (int64_t)(last - 1) * BT + p.wave * C::TOKENS;  // this wave's first token
    auto inside = [&](int blk) { return (int64_t)(blk + 1) * BT <= a.T; };
    Piece<T, N> x[L], xn[L], dy[L], dyn[L];
    Piece<G, N> g[L], gn[L];
    if (!CARRY) load_run<WHOLE>(x, a.x, a, p, t, inside(last - 1));
    // Where the next block's gates as well do not fit the registers, they are loaded with the block (bf16 with
    // f32 gates, 4 x 8192 tokens of 2048 channels: 228 us for 243).
    constexpr bool LATE = !CARRY && sizeof(T) == 2 && (sizeof(G) == 4 || !WHOLE);
    if (!LATE) load_run<WHOLE>(g, a.g, a, p, t, inside(last - 1));
    load_run<WHOLE>(dy, a.dy, a, p, t, inside(last - 1));
    for (int blk = last - 1; blk >= first; --blk, t -= BT) {
        float state = 0.f;
        if (!CARRY && p.there) state = a.states[blk * BW + at];
        if (LATE) load_run<WHOLE>(g, a.g, a, p, t, inside(blk));
        if (blk > first) {
            if (!CARRY) load_run<WHOLE>(xn, a.x, a, p, t - BT, true);
            if (!LATE) load_run<WHOLE>(gn, a.g, a, p, t - BT, true);
            load_run<WHOLE>(dyn, a.dy, a, p, t - BT, true);
        }
        if (masks || !inside(blk))
            backward_block<T, G, WHOLE, CARRY, true>(a, p, fwd, bwd, blk & 1, t, x, g, dy, load_masks<L>(a, p, t),
                                                     state, adj, half);
        else
            backward_block<T, G, WHOLE, CARRY, false>(a, p, fwd, bwd, blk & 1, t, x, g, dy, Masks{~0u, 0}, state,
                                                      adj, half);
#pragma unroll
        for (int i = 0; i < L; ++i) {
            x[i] = xn[i], dy[i] = dyn[i];
            if (!LATE) g[i] = gn[i];
        }
    }
    if (p.wave != 0 || !p.owns) return;
    if (CARRY) {
        a.seg_half[p.seg * BW + at] = half;
        a.seg_sum[p.seg * BW + at] = adj;
    } else if (first == 0 && a.final_state) {
        a.final_state[at] = adj;
    }
}

template <typename T, typename G, bool WHOLE, bool CARRY, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) rec_backward(RecArgs a) {
    using C = Cfg<T, WAVES>;
    __shared__ __align__(16) Totals<C> fwd, bwd;
    const Place p = place<C, WHOLE>(a);
    if (CARRY && p.seg == 0) return;  // nothing comes before it
    fwd.clear(), bwd.clear();
    __syncthreads();
    backward_walk<T, G, WHOLE, CARRY>(a, p, fwd, bwd);
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
        l = l > 127.f ? 127.f : l;  // NaN stays
        const float d = cut || l < -126.f ? 0.f : __builtin_amdgcn_exp2f(l);
        y = next_state<false>(d, a.final_state[i], Elem<T>::load(a.x.data, b * a.x.s0 + c * a.x.s2));
        a.final_state[i] = y;
    }
    Elem<T>::store(a.y, i, y);
}

// ---- host ------------------------------------------------------------------------------------

// How the time axis is split: a function of the sizes alone, so that both passes agree.
struct Split {
    int slabs, waves, blocks, seg_blocks, segments;
};

// Workgroups that fill the card.  Segments read the inputs twice, so they are taken only to come to one
// workgroup a CU (64 x 2048 tokens of 256 channels, 512 workgroups of 8 waves: 150 us, in two segments 243;
// 4 x 8192 of 2048, 256 workgroups: 306, in two 405).
//
// Each has 8 waves where it has a CU to itself, 4 and 2 where two and four share one, which do not wait for
// each other's barriers.  Forward and backward, in us, with 8, 4 and 2 waves: 256 workgroups (4 x 8192 of
// 2048) 315, 392, 591; 320 (10 x 2048 of 1024) 130, 117, 171; 512 (16 x 4096 of 1024) 345, 291, 390; 1024
// (64 x 2048 of 512) 364, 319, 304; f32, 504 (8 x 509 of 1001) 52, 44, 48; 1024 (8 x 2048 of 2048) 309, 286,
// 271.
constexpr int kWantedGroups = 256;

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
    const bool bf = dtype == GDN2_BF16;
    const int slab = bf ? Cfg<bf16_t>::SLAB : Cfg<float>::SLAB, run = bf ? Cfg<bf16_t>::TOKENS : Cfg<float>::TOKENS;
    k.slabs = (int)((s->width + slab - 1) / slab);
    const int64_t units = (int64_t)k.slabs * s->batch;
    const int most = units <= kWantedGroups ? kMaxWaves : units < 4 * kWantedGroups ? 4 : 2;
    k.waves = 1;
    while (k.waves < most && s->time > (int64_t)k.waves * run) k.waves *= 2;
    const int64_t bt = (int64_t)k.waves * run;
    k.blocks = (int)((s->time + bt - 1) / bt);
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

size_t checkpoint_bytes_of(const gdn2_recurrence_shape *s, const Split &k, int train) {
    return segment_bytes(s, k) + (train ? k.blocks * state_bytes(s) : 0);
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
    if (n * 64 * a.waves > 0xFFFFFFFFll) return fail(GDN2_ERR_SHAPE, "too many sequences or channels for one launch");
    *out = (unsigned)n;
    return ok();
}

template <typename T, typename G, bool WHOLE, bool CARRY, int WAVES>
void launch_kind(const RecArgs &a, bool backward, unsigned grid, hipStream_t st) {
    const dim3 block(64 * a.waves);
    if (backward) hipLaunchKernelGGL((rec_backward<T, G, WHOLE, CARRY, WAVES>), dim3(grid), block, 0, st, a);
    else hipLaunchKernelGGL((rec_forward<T, G, WHOLE, CARRY, WAVES>), dim3(grid), block, 0, st, a);
}

template <typename T, typename G, bool WHOLE>
void launch_rec(const RecArgs &a, bool backward, bool carry, unsigned grid, hipStream_t st) {
    if (carry) launch_kind<T, G, WHOLE, true, kMaxWaves>(a, backward, grid, st);
    else if (a.waves > 4) launch_kind<T, G, WHOLE, false, kMaxWaves>(a, backward, grid, st);
    else if (a.waves > 2) launch_kind<T, G, WHOLE, false, 4>(a, backward, grid, st);
    else launch_kind<T, G, WHOLE, false, 2>(a, backward, grid, st);
}

template <bool WHOLE>
void launch_types(const RecArgs &a, int32_t dtype, int32_t gtype, bool backward, bool carry,
                  unsigned grid, hipStream_t st) {
    if (dtype == GDN2_BF16) {
        if (gtype == GDN2_BF16) launch_rec<bf16_t, bf16_t, WHOLE>(a, backward, carry, grid, st);
        else launch_rec<bf16_t, float, WHOLE>(a, backward, carry, grid, st);
    } else {
        if (gtype == GDN2_BF16) launch_rec<float, bf16_t, WHOLE>(a, backward, carry, grid, st);
        else launch_rec<float, float, WHOLE>(a, backward, carry, grid, st);
    }
}

int launch_all(const RecArgs &a, int32_t dtype, int32_t gtype, bool backward, void *stream,
               const char *what) {
    unsigned grid;
    GDN2_TRY(grid_of(a, a.segments, &grid));
    // whole slabs of channels side by side, a block's offsets, 4 bytes a value at most, in 32 bits
    constexpr int64_t near = (1 << 29) / (kMaxWaves * (Cfg<float>::TOKENS > Cfg<bf16_t>::TOKENS
                                                           ? Cfg<float>::TOKENS : Cfg<bf16_t>::TOKENS));
    auto beside = [&](const View &v) { return v.s2 == 1 && v.s1 <= near; };
    const int slab = dtype == GDN2_BF16 ? Cfg<bf16_t>::SLAB : Cfg<float>::SLAB;
    const bool whole = a.W >= slab && a.W <= near && beside(a.x) && beside(a.g) && (!backward || beside(a.dy));
    hipStream_t st = (hipStream_t)stream;
    for (int carry = a.segments > 1 ? 1 : 0; carry >= 0; --carry) {
        if (whole) launch_types<true>(a, dtype, gtype, backward, carry, grid, st);
        else launch_types<false>(a, dtype, gtype, backward, carry, grid, st);
    }
    return launch_status(hipGetLastError(), what);
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_recurrence_checkpoint_bytes(const gdn2_recurrence_shape *shape, int32_t dtype, int train) {
    if (check_shape(shape) || check_dtype(dtype)) return 0;
    const size_t n = checkpoint_bytes_of(shape, split_of(shape, dtype), train);
    return n ? n : 16;
}

int gdn2_recurrence_scan(const gdn2_recurrence_shape *shape, const gdn2_view *x, const gdn2_view *g,
                         const gdn2_view *valid, const gdn2_view *reset, const gdn2_view *initial,
                         void *output, float *final_state, int train, void *checkpoint,
                         size_t checkpoint_bytes, void *stream) {
    GDN2_TRY(check_inputs(shape, x, g, valid, reset));
    if (initial) GDN2_TRY(check_view(initial, "initial", GDN2_F32, true));
    if (!output || !final_state) return fail(GDN2_ERR_ARGUMENT, "output and final_state must be non-null");
    const Split k = split_of(shape, x->dtype);
    GDN2_TRY(check_buffer("checkpoint", checkpoint, checkpoint_bytes, checkpoint_bytes_of(shape, k, train)));
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
    const Split k = split_of(shape, x->dtype);
    GDN2_TRY(check_buffer("checkpoint", checkpoint, checkpoint_bytes, checkpoint_bytes_of(shape, k, 1)));
    GDN2_TRY(check_buffer("workspace", workspace, workspace_bytes, segment_bytes(shape, k)));
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
