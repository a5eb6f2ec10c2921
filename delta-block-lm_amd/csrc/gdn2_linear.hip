// Linear attention with a decay for each head on gfx950: chunked forward and backward, and the
// recurrent step.
//
// Per (batch, head) and valid token, with a = exp(g):
//   S = a S (0 first at a reset),  S += k v^T,  o = S^T q.
// A chunk of C tokens with start state S0, D_ts = g_{s+1} + .. + g_t, Gam_ts = exp(D_ts) for s <= t
// (0 across a reset), gam_t = exp(g_first + .. + g_t), lam_s = Gam_{last,s}:
//   o_t = sum_{s<=t} Gam_ts (q_t.k_s) v_s + gam_t S0^T q_t,   S_C = gam_C S0 + sum_s lam_s k_s v_s^T.
// The gradients are the same sums with the tensors in other places, R the adjoint at the chunk's end:
//   dq_t = sum_{s<=t} Gam_ts (do_t.v_s) k_s + gam_t S0 do_t      the forward on  (do, v, k)
//   dv_s = sum_{t>=s} Gam_ts (k_s.q_t) do_t + lam_s R^T k_s      time reversed on (k, q, do)
//   dk_s = sum_{t>=s} Gam_ts (v_s.do_t) q_t + lam_s R v_s        time reversed on (v, do, q)
// so one kernel, linear_walk, computes all four from a triple (a, b, c) and a direction:
//   out_t = sum_s Gam (a_t.b_s) c_s + row_t (a_t S),   S' = tot S + sum_s col_s b_s c_s^T.
// The gate's gradient is a sum over the pairs that span a token, dg_t = sum_{u>=t,s<t} W_us with
// W_us = Gam_us (q_u.k_s)(do_u.v_s), cut at the chunk's bounds (linear_gate).  Nothing is subtracted
// over more than one segment, so it keeps float32 accuracy for long memories.
#include <math.h>

#include <algorithm>

#include "gdn2_chunk_tile.h"
#include "gdn2_common.h"
#include "gdn2_status.h"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 64;       // columns of c (and of the state) that a workgroup owns
constexpr float kCut = -110.f;  // exp(g) is 0 in float32 below: such a gate cuts like a reset
constexpr int kWalks = 3;       // walks of one launch (dq, dv, dk)

// Matrix operations of one element type: a fragment holds RB entries of the reduction for 16 rows.
// order() reads a row in the order in which two accumulator tiles hold their 32 rows.
template <typename T> struct Mat;
template <> struct Mat<bf16_t> {
    static constexpr int C = 64, RB = 32, PAD = 8, N = 8;  // N: elements of 16 bytes
    typedef bf16x8_t Frag;
    static __device__ __forceinline__ Frag row(const bf16_t *x, int ld, int r0) {
        return frag(x, ld, r0);
    }
    static __device__ __forceinline__ Frag order(const bf16_t *x, int ld, int r0) {
        const int l = lane_id();
        const bf16_t *p = x + (l & 15) * ld + r0 + 4 * (l >> 4);
        const uint2 u = *reinterpret_cast<const uint2 *>(p), v = *reinterpret_cast<const uint2 *>(p + 16);
        return __builtin_bit_cast(Frag, make_uint4(u.x, u.y, v.x, v.y));
    }
    template <int LD>
    static __device__ __forceinline__ Frag across(const bf16_t *z, int r0, int c0) {
        return frag_tr<LD>(z, r0, c0);
    }
    static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &x, const Frag &y) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc, 0, 0, 0);
    }
};
template <> struct Mat<float> {
    static constexpr int C = 32, RB = 16, PAD = 4, N = 4;
    typedef f32x4 Frag;
    static __device__ __forceinline__ Frag row(const float *x, int ld, int r0) {
        const int l = lane_id();
        return *reinterpret_cast<const f32x4 *>(x + (l & 15) * ld + r0 + 4 * (l >> 4));
    }
    static __device__ __forceinline__ Frag order(const float *x, int ld, int r0) {
        return row(x, ld, r0);
    }
    template <int LD>
    static __device__ __forceinline__ Frag across(const float *z, int r0, int c0) {
        const int l = lane_id();
        const float *p = z + (r0 + 4 * (l >> 4)) * LD + c0 + (l & 15);
        return Frag{p[0], p[LD], p[2 * LD], p[3 * LD]};
    }
    static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &x, const Frag &y) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], acc, 0, 0, 0);
    }
};

// Three bf16 terms hold a float32 to its last bit or two, so a product over them with an exact bf16
// operand keeps float32 accuracy: the state and its update are float32 results.
struct Split3 {
    bf16x8_t t[3];
};
__device__ __forceinline__ Split3 split3(const float (&x)[8]) {
    Split3 s;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const __bf16 a = static_cast<__bf16>(x[e]);
        const float r = x[e] - static_cast<float>(a);
        const __bf16 b = static_cast<__bf16>(r);
        s.t[0][e] = a;
        s.t[1][e] = b;
        s.t[2][e] = static_cast<__bf16>(r - static_cast<float>(b));
    }
    return s;
}

// One walk over the chunks: see the head of the file.
struct Walk {
    View a, b, c;
    const void *dot_x;      // optional: dot_t = sum over columns of row_t (a_t S) dot_x_t
    int64_t dx0, dx1, dx2, dx3;
    int a_vec, b_vec, c_vec;
    int ka, vc;             // widths of a and b, and of c and out
    int rev;                // 1: from the last chunk to the first
    const float *init;      // start state of a segment, or null (zero)
    int64_t i_bh, i_seg, i_row, i_col;
    const float *first;     // start state of the walk's first segment where init has none for it
    int64_t f_b, f_h, f_row, f_col;
    float *fin;             // state after the walk's last segment, or null
    int64_t n_bh, n_row, n_col;
    void *out;              // dense [B, T, H, vc], or null
    float *dots;            // [slices, BH, T]
    float *dot_sums;        // [slices, BH, chunks]
    const float *edge;      // with dots of a reversed walk: the forward's state at the segment's start
    int64_t e_bh, e_seg, e_row, e_col;
    const float *edge_first;
    int64_t ef_b, ef_h, ef_row, ef_col;
    float *edges;           // [slices, BH, segments]: <edge, state at the walk's end of the segment>
    float *seg_state;       // carry walk: state that the segment adds, [BH, segments, ka, vc]
    float *seg_decay;       // [BH, segments]
    int slices;
};

struct WalkArgs {
    Walk w[kWalks];
    int walks;
    int64_t B, T, H;
    View g, valid, reset;   // valid.data, reset.data may be null
    float *totals;          // [BH, chunks]: decay of each chunk, written by the first reversed walk
    int chunks, seg_chunks, segments;
    int first_seg;          // carry walk: the first segment that it covers
    int per_group;          // workgroups of one (batch, head, segment)
};

// Gates of one chunk, from one wave (lane = token).
template <int C>
struct GateTile {
    float hi[C], lo[C];     // sum of g log2(e) up to each token: hi + lo, both float32
    float row[C], col[C];   // factor of the start state and of the token's update (0: none of it)
    float step[C];          // exp(g), 0 at a cut, 1 at padding
    int seg[C];             // cuts up to the token; -1 at padding
    float tot;              // decay of the chunk
};

struct GateIn {
    float g, valid, reset;
};

template <int C>
__device__ __forceinline__ GateIn gate_load(const WalkArgs &p, int64_t b, int64_t h, int64_t chunk) {
    const int l = lane_id();
    const int64_t t = chunk * C + l;
    GateIn x{0.f, 0.f, 0.f};
    if (l < C && t < p.T) {
        x.valid = p.valid.data ? ld4<float>(p.valid, b, t, 0, 0) : 1.f;
        x.reset = p.reset.data ? ld4<float>(p.reset, b, t, 0, 0) : 0.f;
        x.g = ld4<float>(p.g, b, t, h, 0);
    }
    return x;
}

template <int C>
__device__ __forceinline__ void gate_store(const GateIn &x, int rev, GateTile<C> *o) {
    const int l = lane_id();
    const bool val = x.valid != 0.f;
    float g = val ? x.g : 0.f;
    const bool cut = val && (x.reset != 0.f || g < kCut);
    if (cut) g = 0.f;
    int seg = cut;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int z = __shfl_up(seg, d);
        if (l >= d) seg += z;
    }
    // The sums are taken in 64 bits, since differences of float32 sums over a chunk would lose digits,
    // and start again at a cut, so that a gate that is not finite ends there.
    double G = (double)g * 1.4426950408889634;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double y = __shfl_up(G, d);
        const int z = __shfl_up(seg, d);
        if (l >= d && z == seg) G += y;
    }
    const double last = __shfl(G, 63);
    const int end = __shfl(seg, 63);
    if (l < C) {
        const float gam = seg == 0 && val ? exp2f((float)G) : 0.f;
        const float lam = seg == end && val ? exp2f((float)(last - G)) : 0.f;
        o->hi[l] = (float)G;
        o->lo[l] = (float)(G - (double)(float)G);
        o->row[l] = rev ? lam : gam;
        o->col[l] = rev ? gam : lam;
        o->step[l] = cut ? 0.f : val ? expf(g) : 1.f;
        o->seg[l] = val ? seg : -1;
        if (l == 0) o->tot = end == 0 ? exp2f((float)last) : 0.f;
    }
}

// 16 bytes of one row of a sequence tensor; zero beyond its width, past the end and at padding.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const View &x, int vec, int64_t b, int64_t t, int64_t h,
                                            int c0, int width, bool on) {
    constexpr int N = Mat<T>::N;
    if (!on || c0 >= width) return make_uint4(0, 0, 0, 0);
    const T *p = reinterpret_cast<const T *>(x.data) + b * x.s0 + t * x.s1 + h * x.s2;
    if (vec && c0 + N <= width) return *reinterpret_cast<const uint4 *>(p + c0);
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = c0 + i < width ? p[(int64_t)(c0 + i) * x.s3] : T(0);
    uint4 r;
    __builtin_memcpy(&r, e, 16);
    return r;
}

// A tile of C rows and W columns on its way from memory to LDS.
template <typename T, int W>
struct Staged {
    static constexpr int N = Mat<T>::N, C = Mat<T>::C, PIECES = C * W / N / kThreads;
    uint4 r[PIECES];
    __device__ __forceinline__ void load(const View &x, int vec, const WalkArgs &p, int64_t b,
                                         int64_t h, int64_t chunk, int c0, int width) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int n = threadIdx.x + i * kThreads;
            const int64_t t = chunk * C + n / (W / N);
            const bool on = t < p.T && (!p.valid.data || ld4<float>(p.valid, b, t, 0, 0) != 0.f);
            r[i] = load_piece<T>(x, vec, b, t, h, c0 + n % (W / N) * N, width, on);
        }
    }
    template <int LD>
    __device__ __forceinline__ void store(T *tile) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int n = threadIdx.x + i * kThreads;
            *reinterpret_cast<uint4 *>(tile + n / (W / N) * LD + n % (W / N) * N) = r[i];
        }
    }
};

// Four consecutive columns of the output at token t.
template <typename T>
__device__ __forceinline__ void store4(T *out, int64_t row, int col, int width, const f32x4 &x) {
    T *p = out + row * width + col;
    T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) Elem<T>::store(e, i, x[i]);
    if (width % 4 == 0) {
        if (col < width) __builtin_memcpy(__builtin_assume_aligned(p, 4 * sizeof(T)), e, sizeof e);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < width) p[i] = e[i];
    }
}

// Gam of the pair (out token t, source token s), 0 where s is not seen from t.
template <int C>
__device__ __forceinline__ float pair_decay(const GateTile<C> &gt, int rev, int t, int s) {
    const float d = (gt.hi[t] - gt.hi[s]) + (gt.lo[t] - gt.lo[s]);
    const bool on = gt.seg[t] == gt.seg[s] && (rev ? s >= t : s <= t);
    return on ? exp2f(rev ? -d : d) : 0.f;
}

// Sum over the four 16-lane groups of a wave.
__device__ __forceinline__ float groups_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <typename T, int KP>
struct WalkLds {
    static constexpr int C = Mat<T>::C, LDA = KP + Mat<T>::PAD, LDC = kCols + Mat<T>::PAD,
                         LDP = C + Mat<T>::PAD;
    T a[C * LDA], b[C * LDA], c[C * LDC], p[C * LDP];
    GateTile<C> gate;
    float red[4][C];
};

// One workgroup: a segment's chunks in the walk's order, kCols columns of the state.  Each of the four
// waves owns 16 columns, so its part of the state stays in its accumulators, where the state is at
// once the product's operand of the next chunk: neither it nor its update passes through LDS.
// CARRY: only the state that the segment adds and its decay.
template <typename T, int KP, bool CARRY>
__global__ void __launch_bounds__(kThreads, 2) linear_walk(WalkArgs p) {
    typedef Mat<T> M;
    typedef WalkLds<T, KP> L;
    constexpr int C = M::C, TT = C / 16, KT = KP / 16, RB = M::RB, LDA = L::LDA, LDC = L::LDC,
                  LDP = L::LDP, BT = RB / 16;  // BT: accumulator tiles of one fragment
    __shared__ __align__(16) L lds;
    const int lane = lane_id(), wave = threadIdx.x >> 6, n16 = lane & 15, g4 = 4 * (lane >> 4);

    // Workgroups of one group share their inputs: they take neighbouring numbers on one XCD.
    const unsigned total = gridDim.x, xcd = blockIdx.x % 8;
    const unsigned whole = total / 8, rest = total % 8;
    unsigned id = xcd * whole + min(xcd, rest) + blockIdx.x / 8;
    int sub = id % p.per_group;
    id /= p.per_group;
    const int segs = p.segments - (CARRY ? 1 : 0);
    int seg = id % segs;
    const int64_t bh = id / segs, b = bh / p.H, h = bh % p.H;
    int wi = 0;
    while (sub >= p.w[wi].slices) sub -= p.w[wi].slices, ++wi;
    const Walk &w = p.w[wi];
    const int rev = w.rev, col0 = sub * kCols;
    if (CARRY) seg += p.first_seg;

    const int c_lo = seg * p.seg_chunks, c_hi = min(p.chunks, c_lo + p.seg_chunks);
    const int64_t BH = p.B * p.H;

    f32x4 S[KT];
#pragma unroll
    for (int m = 0; m < KT; ++m) S[m] = zero4();
    const bool walk_first = rev ? seg == p.segments - 1 : seg == 0;
    if (!CARRY) {
        const float *src = walk_first ? w.first : w.init;
        if (src) {
            src += walk_first ? b * w.f_b + h * w.f_h : bh * w.i_bh + seg * w.i_seg;
            const int64_t rs = walk_first ? w.f_row : w.i_row, cs = walk_first ? w.f_col : w.i_col;
            const int v = col0 + 16 * wave + n16;
#pragma unroll
            for (int m = 0; m < KT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = 16 * m + g4 + i;
                    if (k < w.ka && v < w.vc) S[m][i] = src[k * rs + v * cs];
                }
        }
    }
    float decay = 1.f;

    Staged<T, KP> sa, sb;
    Staged<T, kCols> sc;
    GateIn gi{};
    const auto fetch = [&](int ci) {
        if (!CARRY) sa.load(w.a, w.a_vec, p, b, h, ci, 0, w.ka);
        sb.load(w.b, w.b_vec, p, b, h, ci, 0, w.ka);
        sc.load(w.c, w.c_vec, p, b, h, ci, col0, w.vc);
        if (wave == 0) gi = gate_load<C>(p, b, h, ci);
    };
    fetch(rev ? c_hi - 1 : c_lo);

    for (int n = c_lo; n < c_hi; ++n) {
        const int ci = rev ? c_lo + c_hi - 1 - n : n;
        __syncthreads();  // the last chunk's tiles are read
        if (!CARRY) sa.template store<LDA>(lds.a);
        sb.template store<LDA>(lds.b);
        sc.template store<LDC>(lds.c);
        if (wave == 0) gate_store<C>(gi, rev, &lds.gate);
        if (n + 1 < c_hi) fetch(rev ? ci - 1 : ci + 1);
        __syncthreads();

        f32x4 acc[TT];
        if (!CARRY) {
            // P_ts = Gam_ts a_t.b_s for the tiles whose block of RB sources is seen from the rows.
            for (int n2 = wave; n2 < TT * TT; n2 += 4) {
                const int tj = n2 / TT, si = n2 % TT;
                if (rev ? si / BT < tj / BT : si / BT > tj / BT) continue;
                f32x4 x = zero4();
#pragma unroll
                for (int r = 0; r < KP; r += RB)
                    M::mma(x, M::row(lds.b + 16 * si * LDA, LDA, r), M::row(lds.a + 16 * tj * LDA, LDA, r));
                const int t = 16 * tj + n16, s = 16 * si + g4;
                T e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float f = pair_decay<C>(lds.gate, rev, t, s + i);
                    Elem<T>::store(e, i, f == 0.f ? 0.f : x[i] * f);
                }
                __builtin_memcpy(__builtin_assume_aligned(lds.p + t * LDP + s, 4 * sizeof(T)), e, sizeof e);
            }
            // acc[j]: rows = the wave's columns, column = token 16 j + n16; the state's part.
#pragma unroll
            for (int j = 0; j < TT; ++j) acc[j] = zero4();
#pragma unroll
            for (int r = 0; r < KP / RB; ++r) {
                if constexpr (sizeof(T) == 2) {
                    const f32x4 u = S[2 * r], v = S[2 * r + 1];
                    const Split3 s3 = split3({u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]});
#pragma unroll
                    for (int j = 0; j < TT; ++j) {
                        const typename M::Frag x = M::order(lds.a + 16 * j * LDA, LDA, r * RB);
                        M::mma(acc[j], s3.t[0], x);
                        if (w.dot_x) {
                            M::mma(acc[j], s3.t[1], x);
                            M::mma(acc[j], s3.t[2], x);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < TT; ++j)
                        M::mma(acc[j], S[r], M::order(lds.a + 16 * j * LDA, LDA, r * RB));
                }
            }
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                const float f = lds.gate.row[16 * j + n16];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][i] = f == 0.f ? 0.f : acc[j][i] * f;
                if (w.dot_x) {
                    const int64_t t = (int64_t)ci * C + 16 * j + n16;
                    float d = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int v = col0 + 16 * wave + g4 + i;
                        if (f != 0.f && v < w.vc)
                            d += acc[j][i] * Elem<T>::load(w.dot_x, b * w.dx0 + t * w.dx1 + h * w.dx2 + v * w.dx3);
                    }
                    d = groups_sum(d);
                    if (lane < 16) lds.red[wave][16 * j + n16] = d;
                }
            }
            __syncthreads();
            if (w.dot_x && wave == 0) {
                const int64_t t = (int64_t)ci * C + lane;
                float d = 0.f;
                if (lane < C) d = (lds.red[0][lane] + lds.red[1][lane]) + (lds.red[2][lane] + lds.red[3][lane]);
                if (lane < C && t < p.T) w.dots[(sub * BH + bh) * p.T + t] = d;
                const float sum = wave_sum(d);
                if (lane == 0) w.dot_sums[(sub * BH + bh) * p.chunks + ci] = sum;
            }
        }
        if (p.totals && wi == 0 && sub == 0 && threadIdx.x == 0) p.totals[bh * p.chunks + ci] = lds.gate.tot;

        // The update, apart from the state: it tells whether b or c held a value that is not finite.
        typename M::Frag cf[C / RB];
#pragma unroll
        for (int r = 0; r < C / RB; ++r) cf[r] = M::template across<LDC>(lds.c, r * RB, 16 * wave);
        f32x4 U[KT];
#pragma unroll
        for (int m = 0; m < KT; ++m) U[m] = zero4();
#pragma unroll
        for (int r = 0; r < C / RB; ++r) {
            const float *f = lds.gate.col + r * RB + (RB / 4) * (lane >> 4);
            if constexpr (sizeof(T) == 2) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(cf[r][e]) * f[e];
                const Split3 s3 = split3(x);
#pragma unroll
                for (int m = 0; m < KT; ++m) {
                    const typename M::Frag y = M::template across<LDA>(lds.b, r * RB, 16 * m);
#pragma unroll
                    for (int q = 0; q < 3; ++q) M::mma(U[m], y, s3.t[q]);
                }
            } else {
                f32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = cf[r][e] * f[e];
#pragma unroll
                for (int m = 0; m < KT; ++m)
                    M::mma(U[m], M::template across<LDA>(lds.b, r * RB, 16 * m), x);
            }
        }
        float z = 0.f;
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) z = fmaf(U[m][i], 0.f, z);
        const float tot = lds.gate.tot;
        decay *= tot;

        if (!__any(z != 0.f)) {  // z is 0 or NaN
            if (!CARRY) {
#pragma unroll
                for (int j = 0; j < TT; ++j) {
#pragma unroll
                    for (int r = 0; r < C / RB; ++r) {
                        if (rev ? r < j / BT : r > j / BT) continue;
                        M::mma(acc[j], cf[r], M::row(lds.p + 16 * j * LDP, LDP, r * RB));
                    }
                    const int64_t t = (int64_t)ci * C + 16 * j + n16;
                    if (w.out && t < p.T)
                        store4<T>(reinterpret_cast<T *>(w.out), (b * p.T + t) * p.H + h,
                                  col0 + 16 * wave + g4, w.vc, acc[j]);
                }
            }
#pragma unroll
            for (int m = 0; m < KT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[m][i] = (tot == 0.f ? 0.f : S[m][i] * tot) + U[m][i];
        } else {
            // A product over masked tokens would spread the value to tokens that do not see it: the
            // wave takes this chunk token by token.
            for (int n2 = 0; n2 < C; ++n2) {
                const int tl = rev ? C - 1 - n2 : n2;
                const int64_t t = (int64_t)ci * C + tl;
                if (t >= p.T) continue;
                const bool val = lds.gate.seg[tl] >= 0;
                const float f = lds.gate.step[tl];
                float o = 0.f;
                if (val) {
                    const float x = Elem<T>::load(lds.c, tl * LDC + 16 * wave + n16);
#pragma unroll
                    for (int m = 0; m < KT; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int k = 16 * m + g4 + i;
                            if (k >= w.ka) continue;  // 0 there, whatever x is
                            if (!rev) S[m][i] = f == 0.f ? 0.f : S[m][i] * f;
                            S[m][i] += Elem<T>::load(lds.b, tl * LDA + k) * x;
                            if (!CARRY) o += Elem<T>::load(lds.a, tl * LDA + k) * S[m][i];
                            if (rev) S[m][i] = f == 0.f ? 0.f : S[m][i] * f;
                        }
                    o = groups_sum(o);
                }
                const int v = col0 + 16 * wave + n16;
                if (!CARRY && w.out && lane < 16 && v < w.vc)
                    Elem<T>::store(w.out, ((b * p.T + t) * p.H + h) * w.vc + v, o);
            }
        }
    }

    const int v = col0 + 16 * wave + n16;
    if (CARRY) {
        float *dst = w.seg_state + (bh * p.segments + seg) * w.ka * w.vc;
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 16 * m + g4 + i;
                if (k < w.ka && v < w.vc) dst[(int64_t)k * w.vc + v] = S[m][i];
            }
        if (threadIdx.x == 0 && sub == 0) w.seg_decay[bh * p.segments + seg] = decay;
        return;
    }
    if (w.fin && (rev ? seg == 0 : seg == p.segments - 1)) {
        float *dst = w.fin + bh * w.n_bh;
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 16 * m + g4 + i;
                if (k < w.ka && v < w.vc) dst[k * w.n_row + v * w.n_col] = S[m][i];
            }
    }
    if (w.edges) {
        const float *e = seg == 0 ? w.edge_first : w.edge;
        float d = 0.f;
        if (e) {
            e += seg == 0 ? b * w.ef_b + h * w.ef_h : bh * w.e_bh + seg * w.e_seg;
            const int64_t rs = seg == 0 ? w.ef_row : w.e_row, cs = seg == 0 ? w.ef_col : w.e_col;
#pragma unroll
            for (int m = 0; m < KT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = 16 * m + g4 + i;
                    if (k < w.ka && v < w.vc) d += S[m][i] * e[k * rs + v * cs];
                }
        }
        d = wave_sum(d);
        __syncthreads();  // wave 0 has read the last chunk's sums
        if (lane == 0) lds.red[wave][0] = d;
        __syncthreads();
        if (threadIdx.x == 0)
            w.edges[(sub * BH + bh) * p.segments + seg] =
                (lds.red[0][0] + lds.red[1][0]) + (lds.red[2][0] + lds.red[3][0]);
    }
}

// Segments' additions -> start states, in place: state[s] = what the segments walked before s left.
// One thread an element; carry over the segments in the walk's order.
struct JoinArgs {
    float *state;        // [BH, segments, K V]
    const float *decay;  // [BH, segments]
    const float *first;  // start state of the walk, or null
    int64_t f_b, f_h, f_row, f_col;
    int64_t H, KV, V;
    int segments, rev;
};

__global__ void __launch_bounds__(kThreads) linear_join(JoinArgs p) {
    const int64_t bh = blockIdx.y, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= p.KV) return;
    float *st = p.state + bh * p.segments * p.KV + i;
    const float *d = p.decay + bh * p.segments;
    float x = 0.f;
    if (p.first)
        x = p.first[bh / p.H * p.f_b + bh % p.H * p.f_h + i / p.V * p.f_row + i % p.V * p.f_col];
    for (int n = 0; n + 1 < p.segments; ++n) {
        const int s = p.rev ? p.segments - 1 - n : n;
        const float add = st[s * p.KV];
        st[s * p.KV] = x;
        x = (d[s] == 0.f ? 0.f : d[s] * x) + add;
    }
    st[(p.rev ? 0 : p.segments - 1) * p.KV] = x;
}

// ---- the gate's gradient -------------------------------------------------------------------------

struct GateGradArgs {
    WalkArgs w;           // g, masks, sizes
    View q, k, v, d_o;
    int q_vec, k_vec, v_vec, o_vec;
    int K, V;
    const float *x, *y;           // dots of the dq and dv walks
    const float *x_sums, *y_sums; // per chunk
    const float *edges;
    const float *totals;
    int x_slices, y_slices;
    float *dg;                    // dense [B, T, H]
};

// One workgroup a chunk: W by matrix products in 64-wide slabs of the channels, prefix sums along
// its rows, and the parts of pairs that reach out of the chunk:
//   dg_t = sum_{u>=t, s<t inside} W_us + sum_{u>=t} x_u + sum_{s<t} y_s + E,
// E the pairs around the whole chunk: edge products at the segment's start, then chunk by chunk.
template <typename T>
__global__ void __launch_bounds__(kThreads) linear_gate(GateGradArgs p) {
    typedef Mat<T> M;
    constexpr int C = M::C, TT = C / 16, RB = M::RB, LD = kCols + M::PAD, LDW = C + 1;
    constexpr int MINE = (TT * (TT + 1) / 2 + 3) / 4;
    __shared__ __align__(16) T xs[C * LD], ys[C * LD];
    __shared__ float W[C * LDW], red[4][64];
    __shared__ GateTile<C> gate;
    const int lane = lane_id(), wave = threadIdx.x >> 6, n16 = lane & 15, g4 = 4 * (lane >> 4);
    const int ci = blockIdx.x % p.w.chunks;
    const int64_t bh = blockIdx.x / p.w.chunks, b = bh / p.w.H, h = bh % p.w.H;
    const int64_t BH = p.w.B * p.w.H;
    GateIn gi{};
    if (wave == 0) {
        gi = gate_load<C>(p.w, b, h, ci);
        gate_store<C>(gi, 0, &gate);
    }
    for (int i = threadIdx.x; i < C * LDW; i += kThreads) W[i] = 0.f;
    f32x4 qk[MINE], ov[MINE];
#pragma unroll
    for (int m = 0; m < MINE; ++m) qk[m] = zero4(), ov[m] = zero4();
    const int kslabs = (p.K + kCols - 1) / kCols, slabs = kslabs + (p.V + kCols - 1) / kCols;
    for (int s = 0; s < slabs; ++s) {
        Staged<T, kCols> a, c;
        const bool first = s < kslabs;
        const int c0 = (first ? s : s - kslabs) * kCols;
        a.load(first ? p.q : p.d_o, first ? p.q_vec : p.o_vec, p.w, b, h, ci, c0, first ? p.K : p.V);
        c.load(first ? p.k : p.v, first ? p.k_vec : p.v_vec, p.w, b, h, ci, c0, first ? p.K : p.V);
        __syncthreads();
        a.template store<LD>(xs);
        c.template store<LD>(ys);
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
            int n = wave + 4 * m, tj = 0;
            if (n >= TT * (TT + 1) / 2) continue;
            while (n > tj) n -= ++tj;  // the lower tiles (tj, si <= tj), row by row
            f32x4 acc = first ? qk[m] : ov[m];
#pragma unroll
            for (int r = 0; r < kCols; r += RB)
                M::mma(acc, M::row(ys + 16 * n * LD, LD, r), M::row(xs + 16 * tj * LD, LD, r));
            if (first) qk[m] = acc;
            else ov[m] = acc;
        }
    }
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
        int n = wave + 4 * m, tj = 0;
        if (n >= TT * (TT + 1) / 2) continue;
        while (n > tj) n -= ++tj;
        const int t = 16 * tj + n16, s = 16 * n + g4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = s + i < t ? pair_decay<C>(gate, 0, t, s + i) : 0.f;
            W[t * LDW + s + i] = f == 0.f ? 0.f : f * qk[m][i] * ov[m][i];
        }
    }
    __syncthreads();
    // lane t of a wave: sum over its rows u >= t of the row's sum before t.
    float r = 0.f;
    for (int u = wave; u < C; u += 4) {
        const float x = lane < C ? W[u * LDW + lane] : 0.f;
        const float y = __shfl_up(x, 1);
        const float pre = wave_scan_add(lane == 0 ? 0.f : y);
        if (u >= lane) r += pre;
    }
    red[wave][lane] = r;
    __syncthreads();
    if (wave != 0) return;
    const int64_t t = (int64_t)ci * C + lane;
    const bool in = lane < C && t < p.w.T;
    float x = 0.f, y = 0.f;
    if (in) {
        for (int s = 0; s < p.x_slices; ++s) x += p.x[(s * BH + bh) * p.w.T + t];
        for (int s = 0; s < p.y_slices; ++s) y += p.y[(s * BH + bh) * p.w.T + t];
    }
    float dg = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    // sum of x over u >= t, and of y over s < t; scans that add only what belongs to them
    float sx = x, sy = __shfl_up(y, 1);
    if (lane == 0) sy = 0.f;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const float a = __shfl_down(sx, d), c = __shfl_up(sy, d);
        if (lane + d < 64) sx += a;
        if (lane >= d) sy += c;
    }
    // E: from the segment's start, or from the last chunk before this one with a cut in it.
    float E = 0.f;
    if (gate.tot != 0.f) {
        const int seg = ci / p.w.seg_chunks, c_lo = seg * p.w.seg_chunks;
        int from = c_lo;  // first chunk whose sums count in full
        bool cut = false;
        for (int c0 = c_lo; c0 < ci; c0 += 64) {
            const int c = c0 + lane;
            const unsigned long long m = __ballot(c < ci && p.totals[bh * p.w.chunks + min(c, ci)] == 0.f);
            if (m) from = c0 + 63 - __clzll(m), cut = true;
        }
        for (int c = from + lane; c < ci; c += 64) {
            float d = 0.f;
            for (int s = 0; s < p.y_slices; ++s) d += p.y_sums[(s * BH + bh) * p.w.chunks + c];
            if (!(cut && c == from))
                for (int s = 0; s < p.x_slices; ++s) d -= p.x_sums[(s * BH + bh) * p.w.chunks + c];
            E += d;
        }
        if (lane == 0 && !cut)
            for (int s = 0; s < p.y_slices; ++s) E += p.edges[(s * BH + bh) * p.w.segments + seg];
        E = wave_sum(E);
        E -= wave_sum(x);
    }
    if (!in) return;
    const bool val = gate.seg[lane] >= 0 && gate.step[lane] != 0.f;
    dg += sx + sy + E;
    p.dg[(b * p.w.T + t) * p.w.H + h] = val ? dg : 0.f;
}

// out[h] = sum over b, t of x[b, t, h]: one workgroup a head, a fixed order.
__global__ void __launch_bounds__(1024) linear_head_sum(const float *x, int64_t rows, int64_t H, float *out) {
    __shared__ float red[16];
    float s = 0.f;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) s += x[r * H + blockIdx.x];
    s = wave_sum(s);
    if (lane_id() == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        float t = red[0];
        for (int i = 1; i < 16; ++i) t += red[i];
        out[blockIdx.x] = t;
    }
}

// ---- one token ---------------------------------------------------------------------------------------

struct StepArgs {
    View q, k, v, g, valid, reset;
    int64_t H;
    int K, V, vec;
    float *state;
    void *out;
};

// One workgroup a (batch, head): CG column groups of four values by 256 / CG rows, each thread four
// rows at a time.  The state is read and written once; bound by that.
template <typename T, int CG>
__global__ void __launch_bounds__(kThreads) linear_step(StepArgs p) {
    constexpr int RG = kThreads / CG, U = 4;
    __shared__ float qs[128], ks[128];
    __shared__ float4 red[RG][CG];
    const int64_t b = blockIdx.x / p.H, h = blockIdx.x % p.H;
    const int cg = threadIdx.x % CG, rg = threadIdx.x / CG, v0 = 4 * cg;
    const bool val = !p.valid.data || ld4<float>(p.valid, b, 0, 0, 0) != 0.f;
    if (!val) {
        if ((int)threadIdx.x < p.V) Elem<T>::store(p.out, (int64_t)blockIdx.x * p.V + threadIdx.x, 0.f);
        return;
    }
    float a = expf(ld4<float>(p.g, b, 0, h, 0));
    if (p.reset.data && ld4<float>(p.reset, b, 0, 0, 0) != 0.f) a = 0.f;
    if ((int)threadIdx.x < p.K) {
        qs[threadIdx.x] = ld4<T>(p.q, b, 0, h, threadIdx.x);
        ks[threadIdx.x] = ld4<T>(p.k, b, 0, h, threadIdx.x);
    }
    float vv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vv[i] = v0 + i < p.V ? ld4<T>(p.v, b, 0, h, v0 + i) : 0.f;
    __syncthreads();
    float *S = p.state + (int64_t)blockIdx.x * p.K * p.V;
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r0 = rg; r0 < p.K; r0 += RG * U) {
        float4 s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = r0 + u * RG;
            s[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k >= p.K || v0 >= p.V) continue;
            const float *src = S + k * p.V + v0;
            if (p.vec) {
                s[u] = *reinterpret_cast<const float4 *>(src);
            } else {
                s[u].x = src[0];
                if (v0 + 1 < p.V) s[u].y = src[1];
                if (v0 + 2 < p.V) s[u].z = src[2];
                if (v0 + 3 < p.V) s[u].w = src[3];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = r0 + u * RG;
            if (k >= p.K || v0 >= p.V) continue;
            const float kk = ks[k], qq = qs[k];
            float x[4] = {s[u].x, s[u].y, s[u].z, s[u].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = (a == 0.f ? 0.f : a * x[i]) + kk * vv[i];
                o[i] += qq * x[i];
            }
            float *dst = S + k * p.V + v0;
            if (p.vec) {
                *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v0 + i < p.V) dst[i] = x[i];
            }
        }
    }
    red[rg][cg] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if ((int)threadIdx.x < p.V) {
        const float *r = reinterpret_cast<const float *>(red);
        float t = 0.f;
        for (int i = 0; i < RG; ++i) t += r[i * 4 * CG + threadIdx.x];
        Elem<T>::store(p.out, (int64_t)blockIdx.x * p.V + threadIdx.x, t);
    }
}

// ---- host ------------------------------------------------------------------------------------------

struct Plan {
    int C, chunks, seg_chunks, segments;
    int64_t BH, KV;
    int kslices, vslices;
};

constexpr int64_t kWantGroups = 512;  // workgroups that fill the card

int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

Plan plan(const gdn2_shape *s, int dtype) {
    Plan p;
    p.C = dtype == GDN2_BF16 ? Mat<bf16_t>::C : Mat<float>::C;
    p.chunks = (int)((s->time + p.C - 1) / p.C);
    p.BH = s->batch * s->heads;
    p.KV = s->keys * s->values;
    p.kslices = (int)((s->keys + kCols - 1) / kCols);
    p.vslices = (int)((s->values + kCols - 1) / kCols);
    // Segments of at least two chunks, as many as fill the card.
    int64_t want = kWantGroups / std::max<int64_t>(1, p.BH * p.vslices);
    want = std::max<int64_t>(1, std::min<int64_t>(want, p.chunks / 2));
    p.seg_chunks = (int)((p.chunks + want - 1) / want);
    p.segments = (p.chunks + p.seg_chunks - 1) / p.seg_chunks;
    return p;
}

struct Layout {
    size_t state, decay, x, y, x_sums, y_sums, edges, totals, dinit, bytes;
};

// Checkpoint: the start states of the segments, and their decays.
Layout checkpoint_layout(const Plan &p) {
    Layout l{};
    l.decay = p.segments > 1 ? round16(4 * p.BH * p.segments * p.KV) : 0;
    l.bytes = l.decay + round16(4 * p.BH * p.segments);
    return l;
}

Layout workspace_layout(const Plan &p, int64_t T) {
    Layout l{};
    size_t n = 0;
    const auto take = [&](int64_t floats) {
        const size_t at = n;
        n += round16(4 * floats);
        return at;
    };
    l.state = take(p.segments > 1 ? p.BH * p.segments * p.KV : 0);
    l.decay = take(p.BH * p.segments);
    l.x = take(p.kslices * p.BH * T);
    l.y = take(p.vslices * p.BH * T);
    l.x_sums = take((int64_t)p.kslices * p.BH * p.chunks);
    l.y_sums = take((int64_t)p.vslices * p.BH * p.chunks);
    l.edges = take((int64_t)p.vslices * p.BH * p.segments);
    l.totals = take(p.BH * p.chunks);
    l.dinit = take(p.BH * T);
    l.bytes = n;
    return l;
}

int check_linear(const gdn2_shape *s, int dtype) {
    if (!s) return fail(GDN2_ERR_ARGUMENT, "shape is null");
    if (s->batch < 1 || s->time < 1 || s->heads < 1)
        return fail(GDN2_ERR_SHAPE, "batch, time and heads must be nonempty");
    if (s->keys < 1 || s->keys > 128 || s->values < 1 || s->values > 128)
        return fail(GDN2_ERR_SHAPE, "key and value widths must be 1..128");
    if (dtype != GDN2_F32 && dtype != GDN2_BF16)
        return fail(GDN2_ERR_DTYPE, "dtype must be F32 or BF16");
    // A launch has at most 2^24 workgroups of 256 threads: 6 for a chunk of 32 or 64 tokens.
    const int64_t lim = (int64_t)1 << 21;
    if (s->batch > lim || s->heads > lim || s->batch * s->heads > lim || s->time > 32 * lim ||
        (s->time + 31) / 32 > lim / (s->batch * s->heads))
        return fail(GDN2_ERR_SHAPE, "too many tokens: batch * heads * ceil(time / 32) must be at most 2^21");
    return GDN2_OK;
}

// 16-byte pieces of every row: unit channel stride, aligned rows.
int vec_rows(const gdn2_view *v) {
    const int64_t es = v->dtype == GDN2_BF16 ? 2 : 4;
    if (v->stride[3] != 1 || ((uintptr_t)v->data & 15)) return 0;
    for (int d = 0; d < 3; ++d)
        if (v->stride[d] * es % 16) return 0;
    return 1;
}

int check_inputs(const gdn2_shape *s, const gdn2_view *q, const gdn2_view *k, const gdn2_view *v,
                 const gdn2_view *g, const gdn2_view *valid, const gdn2_view *reset) {
    GDN2_TRY(check_view(q, "q", -1, false));
    GDN2_TRY(check_linear(s, q->dtype));
    GDN2_TRY(check_view(k, "k", q->dtype, false));
    GDN2_TRY(check_view(v, "v", q->dtype, false));
    GDN2_TRY(check_view(g, "g", GDN2_F32, false));
    if (valid) GDN2_TRY(check_view(valid, "valid", GDN2_F32, true));
    if (reset) GDN2_TRY(check_view(reset, "reset", GDN2_F32, true));
    return GDN2_OK;
}

WalkArgs walk_args(const gdn2_shape *s, const Plan &p, const gdn2_view *g, const gdn2_view *valid,
                   const gdn2_view *reset) {
    WalkArgs a{};
    a.B = s->batch;
    a.T = s->time;
    a.H = s->heads;
    a.g = make_view(g);
    a.valid = make_view(valid);
    a.reset = make_view(reset);
    a.chunks = p.chunks;
    a.seg_chunks = p.seg_chunks;
    a.segments = p.segments;
    return a;
}

Walk make_walk(const gdn2_view *a, const gdn2_view *b, const gdn2_view *c, int64_t ka, int64_t vc, int rev) {
    Walk w{};
    if (a) w.a = make_view(a), w.a_vec = vec_rows(a);
    w.b = make_view(b), w.b_vec = vec_rows(b);
    w.c = make_view(c), w.c_vec = vec_rows(c);
    w.ka = (int)ka;
    w.vc = (int)vc;
    w.rev = rev;
    w.slices = (int)((vc + kCols - 1) / kCols);
    return w;
}

// The start state x [B, H, K, V] of a walk over that state, or over its transpose.
void set_first(Walk *w, const View &x, bool transposed) {
    w->first = (const float *)x.data, w->f_b = x.s0, w->f_h = x.s1;
    w->f_row = transposed ? x.s3 : x.s2, w->f_col = transposed ? x.s2 : x.s3;
}

template <typename T, bool CARRY>
void launch_walk(const WalkArgs &a, const Plan &p, int64_t ka, hipStream_t st) {
    const int64_t segs = p.segments - (CARRY ? 1 : 0);
    const dim3 grid((unsigned)(p.BH * segs * a.per_group)), block(kThreads);
    if (ka <= 64) hipLaunchKernelGGL((linear_walk<T, 64, CARRY>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((linear_walk<T, 128, CARRY>), grid, block, 0, st, a);
}

template <bool CARRY>
hipError_t run_walk(WalkArgs a, const Plan &p, int dtype, hipStream_t st) {
    a.per_group = 0;
    int64_t ka = 0;
    for (int i = 0; i < a.walks; ++i) a.per_group += a.w[i].slices, ka = std::max<int64_t>(ka, a.w[i].ka);
    if (dtype == GDN2_BF16) launch_walk<bf16_t, CARRY>(a, p, ka, st);
    else launch_walk<float, CARRY>(a, p, ka, st);
    return hipGetLastError();
}

// Start states of every segment of a walk over (b, c), from `first` ([B, H, K, V], data may be null).
hipError_t run_carry(const WalkArgs &base, const Plan &p, const gdn2_view *b, const gdn2_view *c,
                     int64_t K, int64_t V, int rev, const View &first, float *state,
                     float *decay, int dtype, hipStream_t st) {
    WalkArgs a = base;
    a.w[0] = make_walk(nullptr, b, c, K, V, rev);
    a.w[0].seg_state = state;
    a.w[0].seg_decay = decay;
    a.walks = 1;
    a.first_seg = rev ? 1 : 0;
    a.totals = nullptr;
    hipError_t e = run_walk<true>(a, p, dtype, st);
    if (e != hipSuccess) return e;
    const JoinArgs j{state,    decay,    (const float *)first.data, first.s0, first.s1, first.s2,
                     first.s3, base.H, K * V, V, p.segments, rev};
    hipLaunchKernelGGL(linear_join, dim3((unsigned)((K * V + kThreads - 1) / kThreads), (unsigned)p.BH),
                       dim3(kThreads), 0, st, j);
    return hipGetLastError();
}

int check_buffer(const void *buf, size_t bytes, size_t need, const char *name) {
    if (!buf || bytes < need)
        return fail(GDN2_ERR_WORKSPACE, "%s of %zu bytes is too small: %zu needed", name, buf ? bytes : 0, need);
    if ((uintptr_t)buf & 15) return fail(GDN2_ERR_ARGUMENT, "%s must be 16-byte aligned", name);
    return GDN2_OK;
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_linear_checkpoint_bytes(const gdn2_shape *shape, int32_t dtype) {
    if (check_linear(shape, dtype) != GDN2_OK) return 0;
    return checkpoint_layout(plan(shape, dtype)).bytes;
}

int gdn2_linear_scan(const gdn2_shape *shape, const gdn2_view *q, const gdn2_view *k,
                     const gdn2_view *v, const gdn2_view *g, const gdn2_view *valid,
                     const gdn2_view *reset, const gdn2_view *initial, void *output,
                     float *final_state, void *checkpoint, size_t checkpoint_bytes, void *stream) {
    GDN2_TRY(check_inputs(shape, q, k, v, g, valid, reset));
    if (initial) GDN2_TRY(check_view(initial, "initial", GDN2_F32, true));
    if (!output || !final_state)
        return fail(GDN2_ERR_ARGUMENT, "output and final_state must be non-null");
    const Plan p = plan(shape, q->dtype);
    const Layout l = checkpoint_layout(p);
    GDN2_TRY(check_buffer(checkpoint, checkpoint_bytes, l.bytes, "checkpoint"));
    if (initial && !initial->data) initial = nullptr;
    const int64_t K = shape->keys, V = shape->values;
    hipStream_t st = (hipStream_t)stream;
    WalkArgs a = walk_args(shape, p, g, valid, reset);
    const View first = make_view(initial);
    float *state = (float *)checkpoint, *decay = (float *)((char *)checkpoint + l.decay);
    if (p.segments > 1) {
        const hipError_t e = run_carry(a, p, k, v, K, V, 0, first, state, decay, q->dtype, st);
        if (e != hipSuccess) return launch_status(e, "gdn2_linear_scan");
    }
    Walk &w = a.w[0];
    w = make_walk(q, k, v, K, V, 0);
    a.walks = 1;
    set_first(&w, first, false);
    w.init = state, w.i_bh = p.segments * p.KV, w.i_seg = p.KV, w.i_row = V, w.i_col = 1;
    w.fin = final_state, w.n_bh = p.KV, w.n_row = V, w.n_col = 1;
    w.out = output;
    return launch_status(run_walk<false>(a, p, q->dtype, st), "gdn2_linear_scan");
}

size_t gdn2_linear_workspace_bytes(const gdn2_shape *shape, int32_t dtype) {
    if (check_linear(shape, dtype) != GDN2_OK) return 0;
    return workspace_layout(plan(shape, dtype), shape->time).bytes;
}

int gdn2_linear_backward(const gdn2_shape *shape, const gdn2_view *q, const gdn2_view *k,
                         const gdn2_view *v, const gdn2_view *g, const gdn2_view *valid,
                         const gdn2_view *reset, const gdn2_view *initial, const void *checkpoint,
                         size_t checkpoint_bytes, const gdn2_view *d_output,
                         const float *d_final_state, void *dq, void *dk, void *dv, float *dg,
                         float *dg_heads, float *d_initial, void *workspace, size_t workspace_bytes,
                         void *stream) {
    GDN2_TRY(check_inputs(shape, q, k, v, g, valid, reset));
    if (initial) GDN2_TRY(check_view(initial, "initial", GDN2_F32, true));
    GDN2_TRY(check_view(d_output, "d_output", q->dtype, false));
    const Plan p = plan(shape, q->dtype);
    const Layout lc = checkpoint_layout(p), l = workspace_layout(p, shape->time);
    GDN2_TRY(check_buffer(checkpoint, checkpoint_bytes, lc.bytes, "checkpoint"));
    GDN2_TRY(check_buffer(workspace, workspace_bytes, l.bytes, "workspace"));
    if (initial && !initial->data) initial = nullptr;
    const int64_t K = shape->keys, V = shape->values, BH = p.BH;
    const int dtype = q->dtype;
    const bool gates = dg || dg_heads;
    hipStream_t st = (hipStream_t)stream;
    const WalkArgs base = walk_args(shape, p, g, valid, reset);
    const auto at = [&](size_t off) { return (float *)((char *)workspace + off); };
    const float *states = (const float *)checkpoint;  // [BH, segments, K, V]
    const View first = make_view(initial), d_final{d_final_state, shape->heads * p.KV, p.KV, V, 1};
    float *adj = at(l.state);
    hipError_t e = hipSuccess;
    if (p.segments > 1) {
        e = run_carry(base, p, q, d_output, K, V, 1, d_final, adj, at(l.decay), dtype, st);
        if (e != hipSuccess) return launch_status(e, "gdn2_linear_backward");
    }
    const int64_t sb = p.segments * p.KV;
    Walk wq = make_walk(d_output, v, k, V, K, 0);  // state transposed: rows V, columns K
    wq.out = dq;
    wq.init = states, wq.i_bh = sb, wq.i_seg = p.KV, wq.i_row = 1, wq.i_col = V;
    set_first(&wq, first, true);
    Walk wv = make_walk(k, q, d_output, K, V, 1);
    wv.out = dv;
    wv.init = adj, wv.i_bh = sb, wv.i_seg = p.KV, wv.i_row = V, wv.i_col = 1;
    set_first(&wv, d_final, false);
    wv.fin = d_initial, wv.n_bh = p.KV, wv.n_row = V, wv.n_col = 1;
    Walk wk = make_walk(v, d_output, q, V, K, 1);
    wk.out = dk;
    wk.init = adj, wk.i_bh = sb, wk.i_seg = p.KV, wk.i_row = 1, wk.i_col = V;
    set_first(&wk, d_final, true);
    if (gates) {
        wq.dot_x = q->data, wq.dx0 = q->stride[0], wq.dx1 = q->stride[1], wq.dx2 = q->stride[2],
        wq.dx3 = q->stride[3];
        wq.dots = at(l.x), wq.dot_sums = at(l.x_sums);
        wv.dot_x = v->data, wv.dx0 = v->stride[0], wv.dx1 = v->stride[1], wv.dx2 = v->stride[2],
        wv.dx3 = v->stride[3];
        wv.dots = at(l.y), wv.dot_sums = at(l.y_sums);
        wv.edges = at(l.edges);
        wv.edge = states, wv.e_bh = sb, wv.e_seg = p.KV, wv.e_row = V, wv.e_col = 1;
        wv.edge_first = (const float *)first.data, wv.ef_b = first.s0, wv.ef_h = first.s1,
        wv.ef_row = first.s2, wv.ef_col = first.s3;
    }
    const bool one = (K <= 64) == (V <= 64);  // one launch covers all three
    for (int n = 0; n < 2; ++n) {
        WalkArgs a = base;
        if (n == 0) {
            if (dv || gates || d_initial) {
                if (gates) a.totals = at(l.totals);
                a.w[a.walks++] = wv;
            }
            if (!one && a.walks == 0) continue;
        }
        if (n == 1 || one) {
            if (dq || gates) a.w[a.walks++] = wq;
            if (dk) a.w[a.walks++] = wk;
        }
        if (a.walks) e = run_walk<false>(a, p, dtype, st);
        if (e != hipSuccess) return launch_status(e, "gdn2_linear_backward");
        if (one) break;
    }
    if (!gates) return ok();
    GateGradArgs ga{};
    ga.w = base;
    ga.q = make_view(q), ga.k = make_view(k), ga.v = make_view(v), ga.d_o = make_view(d_output);
    ga.q_vec = vec_rows(q), ga.k_vec = vec_rows(k), ga.v_vec = vec_rows(v), ga.o_vec = vec_rows(d_output);
    ga.K = (int)K, ga.V = (int)V;
    ga.x = at(l.x), ga.y = at(l.y), ga.x_sums = at(l.x_sums), ga.y_sums = at(l.y_sums);
    ga.edges = at(l.edges), ga.totals = at(l.totals);
    ga.x_slices = p.kslices, ga.y_slices = p.vslices;
    ga.dg = dg ? dg : at(l.dinit);
    const dim3 grid((unsigned)(BH * p.chunks)), block(kThreads);
    if (dtype == GDN2_BF16) hipLaunchKernelGGL((linear_gate<bf16_t>), grid, block, 0, st, ga);
    else hipLaunchKernelGGL((linear_gate<float>), grid, block, 0, st, ga);
    if (dg_heads)
        hipLaunchKernelGGL(linear_head_sum, dim3((unsigned)shape->heads), dim3(1024), 0, st, ga.dg,
                           shape->batch * shape->time, shape->heads, dg_heads);
    return launch_status(hipGetLastError(), "gdn2_linear_backward");
}

int gdn2_linear_step(const gdn2_shape *shape, const gdn2_view *q, const gdn2_view *k,
                     const gdn2_view *v, const gdn2_view *g, const gdn2_view *valid,
                     const gdn2_view *reset, float *state, void *output, void *stream) {
    GDN2_TRY(check_inputs(shape, q, k, v, g, valid, reset));
    if (shape->time != 1) return fail(GDN2_ERR_SHAPE, "a step needs time == 1");
    if (!state || !output) return fail(GDN2_ERR_ARGUMENT, "state and output must be non-null");
    StepArgs a{make_view(q), make_view(k), make_view(v), make_view(g), make_view(valid), make_view(reset),
               shape->heads, (int)shape->keys, (int)shape->values,
               shape->values % 4 == 0 && ((uintptr_t)state & 15) == 0, state, output};
    const dim3 grid((unsigned)(shape->batch * shape->heads)), block(kThreads);
    hipStream_t st = (hipStream_t)stream;
    const bool bf = q->dtype == GDN2_BF16;
    if (shape->values <= 64) {
        if (bf) hipLaunchKernelGGL((linear_step<bf16_t, 16>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((linear_step<float, 16>), grid, block, 0, st, a);
    } else {
        if (bf) hipLaunchKernelGGL((linear_step<bf16_t, 32>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((linear_step<float, 32>), grid, block, 0, st, a);
    }
    return launch_status(hipGetLastError(), "gdn2_linear_step");
}

}  // extern "C"
