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
// The forward and dq are a walk over the chunks in order (linear_walk), from a triple (a, b, c):
//   out_t = sum_s Gam (a_t.b_s) c_s + row_t (a_t S),   S' = tot S + sum_s col_s b_s c_s^T;
// dv and dk share a walk in the other direction (linear_back), with the pairs' decays and the adjoint
// state of both; for widths up to 64 it has dq and the gate's gradient as well.  The gate's gradient is a sum over
// the pairs that span a token,
//   dg_t = sum_{u>=t,s<t} W_us,  W_us = Gam_us (q_u.k_s)(do_u.v_s),
// cut at the chunk's bounds, with x_u = gam_u q_u^T S0 do_u, y_s = lam_s k_s^T R v_s and E = gam <S0, R>:
//   dg_t = sum_{u>=t,s<t inside the chunk} W_us + sum_{u>=t} x_u + sum_{s<t} y_s + E.
// Every chunk has E from its two states (as a sum stepped from chunk to chunk, less x and plus y, it would be what is
// left of much larger numbers after a strong decay).  Where dq has a walk of its own, linear_back leaves it y and
// the adjoint state R of every chunk; in one walk the forward's kept states are S0.  No part is subtracted from
// another, so what spans a token has float32 accuracy, whatever lies around it.
//
// A sequence is cut into segments for parallel work; their start states come from a walk over (b, c) alone,
// a launch of its own for all segments (carry) and a join over them, or, in short sequences, by each
// segment from the sequence's start.  Operands of matrix products are the inputs' type.  In bf16 a float32
// operand goes in as several bf16 terms, so that only the result is rounded: a state has three (float32
// accuracy), a pair weight, and the adjoint state where it makes dk, two.  Those are off by 2^-16, next to a result
// that is rounded to 2^-8 in its turn.
#include <math.h>

#include <algorithm>

#include "gdn2_chunk_tile.h"
#include "gdn2_common.h"
#include "gdn2_status.h"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;
constexpr float kCut = -110.f;  // exp(g) is 0 in float32 below: such a gate cuts like a reset

// Matrix operations of one element type: a fragment holds RB entries of the reduction for 16 rows.
// Lane group g of a fragment has entries 8 g .. 8 g + 7 of a row of bf16 (4 g .. in float32).
//
// place(m, g4): the first of the four rows of a state that a lane (g4 = 4 g) has in accumulator tile m, and the
// columns of tile m of the pair weights.  In bf16 tiles 2 m and 2 m + 1 share 32 rows, eight to each lane
// group, so that a group's accumulators are entries 8 g .. 8 g + 7 at once: a product's other operand is then
// read in 16-byte pieces.  across() reads a tile the other way round, with the rows 4 g .. and 16 + 4 g .. of
// each 32 in group g (a wave's eight rows at a time lie in different banks), which is what the columns of the
// pair weights and the rows of BackLds::D are laid out for; across_place() the same of place()'s columns.
template <typename T> struct Mat;
template <> struct Mat<bf16_t> {
    static constexpr int C = 64, RB = 32, N = 8;  // N: elements of 16 bytes
    typedef bf16x8_t Frag;
    // Elements from row to row in LDS: rows of 64 and of 128 start in banks that 16-byte reads of 16 rows
    // share at most twice, and not at all.
    static __host__ __device__ constexpr int ld(int width) { return width + (width == 128 ? 16 : 8); }
    static __device__ __forceinline__ Frag row(const bf16_t *x, int ld, int r0) {
        return frag(x, ld, r0);
    }
    static __device__ __forceinline__ Frag read_tr(const bf16_t *p, int ld16) {
        const v4s x = lds_tr16(p), y = lds_tr16(p + ld16);
        typedef short v8s __attribute__((ext_vector_type(8)));
        const v8s v = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        return __builtin_bit_cast(Frag, v);
    }
    template <int LD>
    static __device__ __forceinline__ Frag across(const bf16_t *z, int r0, int c0) {
        const int l = lane_id(), i = l & 15;
        return read_tr(z + (r0 + 4 * (l >> 4) + (i >> 2)) * LD + c0 + 4 * (i & 3), 16 * LD);
    }
    template <int LD>
    static __device__ __forceinline__ Frag across_place(const bf16_t *z, int r0, int m) {
        const int l = lane_id(), i = l & 15;
        return read_tr(z + (r0 + 4 * (l >> 4) + (i >> 2)) * LD + place(m, 4 * (i & 3)), 16 * LD);
    }
    static __device__ __forceinline__ constexpr int place(int m, int g4) { return 32 * (m >> 1) + 4 * (m & 1) + 2 * g4; }
    // Entry e of a fragment of across() is row r0 + 4 g + past(e); row_for(i): the row of which it is entry i.
    static __device__ __forceinline__ constexpr int past(int e) { return e + 3 * (e & 4); }
    static __device__ __forceinline__ int row_for(int i) { return (i & ~31) + 4 * ((i >> 3) & 3) + (i & 3) + 4 * (i & 4); }
    static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &x, const Frag &y) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc, 0, 0, 0);
    }
};
template <> struct Mat<float> {
    static constexpr int C = 32, RB = 16, N = 4;
    typedef f32x4 Frag;
    static __host__ __device__ constexpr int ld(int width) { return width + 4; }
    static __device__ __forceinline__ Frag row(const float *x, int ld, int r0) {
        const int l = lane_id();
        return *reinterpret_cast<const f32x4 *>(x + (l & 15) * ld + r0 + 4 * (l >> 4));
    }
    template <int LD>
    static __device__ __forceinline__ Frag across(const float *z, int r0, int c0) {
        const int l = lane_id();
        const float *p = z + (r0 + 4 * (l >> 4)) * LD + c0 + (l & 15);
        return Frag{p[0], p[LD], p[2 * LD], p[3 * LD]};
    }
    template <int LD>
    static __device__ __forceinline__ Frag across_place(const float *z, int r0, int m) { return across<LD>(z, r0, 16 * m); }
    static __device__ __forceinline__ constexpr int place(int m, int g4) { return 16 * m + g4; }
    static __device__ __forceinline__ constexpr int past(int e) { return e; }
    static __device__ __forceinline__ int row_for(int i) { return i; }
    static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &x, const Frag &y) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], acc, 0, 0, 0);
    }
};

// Two bf16 terms hold a float32 to 2^-16 of its value.  The remainder is that of the rounded float32, whatever
// product it came from: the terms are the same bits in every kernel that makes them.
__device__ __forceinline__ void split2(const f32x4 &x, bf16_t (&hi)[4], bf16_t (&lo)[4]) {
#pragma clang fp contract(off)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hi[i] = f32_to_bf16(x[i]);
        lo[i] = f32_to_bf16(x[i] - bf16_to_f32(hi[i]));
    }
}
__device__ __forceinline__ void split2(const f32x4 &x, float (&hi)[4], float (&)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = x[i];
}

// Three bf16 terms hold a float32 to its last bit or two, so a product over them with an exact bf16
// operand keeps float32 accuracy: the state and its update are float32 results.
struct Split3 {
    bf16x8_t t[3];
};
__device__ __forceinline__ Split3 split3(const float (&x)[8]) {
#pragma clang fp contract(off)
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

// The same number, of which the compiler does not know it: what follows from it (addresses, conditions) is made
// where it is used, and not kept in registers through the loop over chunks.  Without it linear_back spills at 64 x 64,
// and its reloads wait for the loads of the next chunk before them: 16 x 512 tokens, 8 heads of 64, both directions
// 77 us in place of 68.
__device__ __forceinline__ int hidden(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The chunks, gates and states of a walk.  Tensor views are [B, T, H, channels].
struct Walk {
    View g, valid, reset;   // valid.data, reset.data may be null
    View first;             // state before the walk, [B, H, rows, columns] (data may be null: zero)
    const float *starts;    // states before every segment, or null: taken from first by a prewalk
    int64_t s_bh;
    int s_row, s_col;
    float *starts_out;      // the prewalk's states before every segment, or null
    float *kept;            // states before every chunk and after the last, [B H, chunks + 1] kept forms, or null
    float *fin;             // state after the walk, [B H, rows, columns], or null
    int64_t T;
    int H;
    int chunks, seg_chunks, segments;
};

// A walk in order: see the head of the file.
struct Forward : Walk {
    View a, b, c, d;        // d: see DOT
    int ka, vc;             // widths of a and b, and of c, d and out
    void *out;              // dense [B, T, H, vc], or null
    const float *y;         // [B H, T], from linear_back
    const float *adj;       // and the adjoint state behind every chunk, [B H, chunks] kept forms
    float *dg;              // dense [B, T, H]
    float *seg_state;       // carry: state that a segment adds, [B H, segments, ka, vc]
    float *seg_decay;       // its root, [B H, segments]
};

// The walk of dv and dk in the other direction, over the adjoint state [K, V].
struct Back : Walk {
    View q, k, v, o;        // o: the output's gradient
    int K, V;
    void *dq, *dk, *dv;     // dense, or null (dq: all in one)
    float *dg;              // dense [B, T, H], or null (all in one)
    float *y, *adj;         // MODE 1: as in Forward
};

// DPP moves of 64 bits; lanes without a source read 0.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double dpp64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)dpp<CTRL, ROWS>((int)(uint32_t)u);
    const uint32_t hi = (uint32_t)dpp<CTRL, ROWS>((int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// One step of a scan that stops at a new segment: adds the source lane's sum if its segment is ours.
// A lane without a source reads 0 for both, and adds 0.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ void seg_step(double &G, int seg1) {
    const double y = dpp64<CTRL, ROWS>(G);
    if (dpp<CTRL, ROWS>(seg1) == seg1) G += y;
}

// Gates of one chunk, from one wave (lane = token).
template <int C>
struct alignas(16) GateTile {
    float hi[C], lo[C];     // sum of g log2(e) in the token's segment: hi + lo, both float32
    float row[C], col[C];   // factor of the start state and of the token's update (0: none of it)
    float step[C];          // the root of exp(g), 0 at a cut, 1 at padding
    int seg[C];             // cuts up to the token; -1 at padding
    float tot;              // decay of the chunk, or NaN if it may grow past float32
    float span;             // decay of the chunk, up to 2^127
    double sum;             // its log2, for a chunk without a cut
};

// Decays can be growth past what float32 holds, which takes a value that is there to infinity, and leaves zero zero.
// A chunk where that may be is taken token by token: its decay is NaN, which shows in the state after it.  There, and
// over chunks that are carried, a decay is its root, applied twice (the largest makes any normal number infinite).
// Only the gate's gradient, which is never made token by token, has growth past 2^127 in a chunk counted as 2^127.
__device__ __forceinline__ float root_exp2(float x) {
    x *= 0.5f;
    return __builtin_amdgcn_exp2f(x > 127.99f ? 127.99f : x);  // NaN stays
}
// A value times a decay given by its root: what was there may be infinite or NaN where a cut leaves nothing of it.
__device__ __forceinline__ float decayed(float x, float root) { return root == 0.f ? 0.f : x * root * root; }

struct GateIn {
    float g, valid, reset;
};

template <int C>
__device__ __forceinline__ GateIn gate_load(const Walk &p, int64_t b, int64_t h, int64_t chunk) {
    const int64_t t = min(chunk * C + lane_id(), p.T - 1);
    const auto at = [&](const View &x) { return reinterpret_cast<const float *>(x.data) + b * x.s0 + t * x.s1; };
    const float *g = at(p.g) + h * p.g.s2;
    return GateIn{*g, p.valid.data ? *at(p.valid) : 1.f, p.reset.data ? *at(p.reset) : 0.f};
}

template <int C, bool REV>
__device__ __forceinline__ void gate_store(const GateIn &x, int left, GateTile<C> *o) {
    const int l = lane_id();
    const bool val = l < left && l < C && x.valid != 0.f;
    float g = val ? x.g : 0.f;
    if (g == INFINITY) g = NAN;  // it makes NaN of a state of zero
    const bool cut = val && (x.reset != 0.f || g < kCut);
    if (cut) g = 0.f;
    const int seg = wave_scan_add((int)cut);
    // The sums are taken in 64 bits, since differences of float32 sums over a chunk would lose digits,
    // and start again at a cut, so that a gate that is not finite ends there.
    double G = (double)g * 1.4426950408889634;
    seg_step<0x111>(G, seg + 1);
    seg_step<0x112>(G, seg + 1);
    seg_step<0x114>(G, seg + 1);
    seg_step<0x118>(G, seg + 1);
    seg_step<0x142, 0xA>(G, seg + 1);
    seg_step<0x143, 0xC>(G, seg + 1);
    const double last = __shfl(G, 63);
    const int end = __builtin_amdgcn_readlane(seg, 63);
    const bool grows = __any(!(g <= 88.f / C));  // e^88 is 2^127; a gate that is NaN, too
    if (l < C) {
        const auto factor = [](float x) { return __builtin_amdgcn_exp2f(x > 127.f ? 127.f : x); };
        const float gam = seg == 0 && val ? factor((float)G) : 0.f;
        const float lam = seg == end && val ? factor((float)(last - G)) : 0.f;
        o->hi[l] = (float)G;
        o->lo[l] = (float)(G - (double)(float)G);
        o->row[l] = REV ? lam : gam;
        o->col[l] = REV ? gam : lam;
        o->step[l] = cut ? 0.f : val ? root_exp2(g * 1.44269504f) : 1.f;
        o->seg[l] = val ? seg : -1;
        if (l == 0) {
            const float span = end == 0 ? factor((float)last) : 0.f;
            o->span = span, o->tot = grows ? NAN : span;
            o->sum = last;
        }
    }
}

// A tile of C rows and W columns on its way from memory to LDS: 16 bytes a thread and turn.  Rows past
// the end and columns past the width read others in their place, and become zero on the way to LDS,
// as do the rows of padding: what they hold is not used.  VEC: unit channel stride, 16-byte aligned
// rows, whole pieces, and offsets inside a chunk below 2^31 bytes.
template <typename T, int W, int THREADS, bool VEC>
struct Staged {
    static constexpr int N = Mat<T>::N, C = Mat<T>::C, PER = W / N, ROWS = THREADS / PER,
                         PIECES = C / ROWS;
    uint4 r[PIECES];
    // base: row 0 of the (batch, head), column 0 of the tile; width: columns there are from it on
    __device__ __forceinline__ void load(const T *base, int64_t s1, int64_t s3, int64_t t0, int left, int width) {
        const int row = threadIdx.x / PER, c = threadIdx.x % PER * N;
        base += t0 * s1;
        if constexpr (VEC) {
            const char *p = reinterpret_cast<const char *>(base);
            const uint32_t step = (uint32_t)s1 * (uint32_t)sizeof(T);
            const uint32_t col = (uint32_t)(c < width ? c : 0) * (uint32_t)sizeof(T);
            if (left >= C) {
                const uint32_t off = (uint32_t)row * step + col;
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
                    r[i] = *reinterpret_cast<const uint4 *>(p + (off + (uint32_t)(i * ROWS) * step));
            } else {
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
                    r[i] = *reinterpret_cast<const uint4 *>(p + ((uint32_t)min(row + i * ROWS, left - 1) * step + col));
            }
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const T *q = base + (int64_t)min(row + i * ROWS, left - 1) * s1;
                if (s3 == 1 && c + N <= width) {  // a whole piece, wherever it lies
                    __builtin_memcpy(&r[i], q + c, 16);
                    continue;
                }
                T e[N];
#pragma unroll
                for (int j = 0; j < N; ++j) e[j] = c + j < width ? q[(int64_t)(c + j) * s3] : T(0);
                __builtin_memcpy(&r[i], e, 16);
            }
        }
    }
    template <int LD>
    __device__ __forceinline__ void store(T *tile, const int *seg, bool masks, int width) const {
        const int row = threadIdx.x / PER, c = threadIdx.x % PER * N;
        T *p = tile + row * LD + c;
        if (!masks) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) *reinterpret_cast<uint4 *>(p + i * ROWS * LD) = r[i];
            return;
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            *reinterpret_cast<uint4 *>(p + i * ROWS * LD) =
                seg[row + i * ROWS] >= 0 && c < width ? r[i] : make_uint4(0, 0, 0, 0);
    }
};

// A chunk's rows of a dense output, from tiles whose rows are four columns from col on and whose columns
// are the tokens 16 j + n16; out is at the chunk's first row, stride the elements between two rows.
template <typename T, int TT, bool VEC>
__device__ __forceinline__ void store_rows(T *out, int64_t stride, int col, int width, int left, const f32x4 (&x)[TT]) {
    const int n16 = hidden(lane_id()) & 15;
    T *p = out + n16 * stride + col;
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        T e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) Elem<T>::store(e, i, x[j][i]);
        if (16 * j + n16 >= left) continue;
        if (VEC) {
            if (col < width) __builtin_memcpy(__builtin_assume_aligned(p + 16 * j * stride, 4 * sizeof(T)), e, sizeof e);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < width) p[16 * j * stride + i] = e[i];
        }
    }
}

// Gam of the pairs of out token t with the sources s .. s + 3, 0 for those that t does not see.
template <int C, bool REV>
__device__ __forceinline__ f32x4 pair_decays(const GateTile<C> &gt, int t, int s) {
    const float ht = gt.hi[t];
    const int st = gt.seg[t];
    const f32x4 hs = *reinterpret_cast<const f32x4 *>(gt.hi + s);
    const int4 ss = *reinterpret_cast<const int4 *>(gt.seg + s);
    const int seg[4] = {ss.x, ss.y, ss.z, ss.w};
    f32x4 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = REV ? hs[i] - ht : ht - hs[i];
    const float lt = gt.lo[t];
    const f32x4 ls = *reinterpret_cast<const f32x4 *>(gt.lo + s);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] += REV ? ls[i] - lt : lt - ls[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool on = seg[i] == st && (REV ? s + i >= t : s + i <= t);
        f[i] = __builtin_amdgcn_exp2f(!on ? -1000.f : f[i] > 127.f ? 127.f : f[i]);  // NaN stays
    }
    return f;
}

// A product times its decay.  Where that is 0 the product is not seen, and may have overflowed.
__device__ __forceinline__ float seen(float x, float f) { return f == 0.f ? 0.f : x * f; }

// Inclusive sums over the lanes of each 16-lane group.
__device__ __forceinline__ void row_scan(float &x) {
    x += dpp<0x111>(x);
    x += dpp<0x112>(x);
    x += dpp<0x114>(x);
    x += dpp<0x118>(x);
}

// Sum over the four 16-lane groups of a wave.
__device__ __forceinline__ float groups_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <typename T, int KP, int CP, bool OUT, bool DOT>
struct WalkLds {
    static constexpr int C = Mat<T>::C, LDA = Mat<T>::ld(KP), LDC = Mat<T>::ld(CP), LDP = Mat<T>::ld(C);
    T b[C * LDA], c[C * LDC];
    // Terms of the pair weights: the second behind the first, with DOT in the place of d once that is read (two
    // workgroups share a unit at 128 x 64).
    static constexpr int TERMS = sizeof(T) == 2 ? 2 : 1, ROOM = DOT ? 1 : TERMS;
    static_assert(LDC >= LDP, "");
    T a[OUT ? C * LDA : 8], p[OUT ? ROOM * C * LDP : 8], d[DOT ? C * LDC : 8];
    // Chunks whose gates are made at a time.  With four and without the sums of DOT three forward workgroups share
    // a unit at 64 x 64 (2048 heads of 8 tokens, bf16: 26 us, by twos 32; a prompt of 3001 tokens, 8 heads, 23.4, 24.1).
    static constexpr int GATES = OUT && !DOT && CP == 64 ? 4 : 8;
    GateTile<C> gate[GATES];
    float red[DOT ? CP / 16 : 1][C], edge[CP / 16];
    float rows[DOT ? C / 16 : 1][C], cols[DOT ? C / 16 : 1][C];  // parts of the pair sums, by tiles of 16 tokens
};

template <typename T, int KP, int VP, bool ALL>
struct BackLds {
    static constexpr int C = Mat<T>::C, LDK = Mat<T>::ld(KP), LDV = Mat<T>::ld(VP), LDP = Mat<T>::ld(C),
                         NW = (KP > VP ? KP : VP) / 16;
    T q[C * LDK], k[C * LDK], v[C * LDV], o[C * LDV];
    // First terms of Gam k.q and Gam v.do (the token-by-token form keeps float sums in pk), and of the adjoint state
    // transposed, [row_for(value)][key].  The second terms take the places of o, k and D once those are read.
    T pk[C * LDP], pv[C * LDP];
    T D[VP * LDK];
    static constexpr int GATES = 8;  // as in WalkLds
    GateTile<C> gate[GATES];
    float red[NW][C], red_q[ALL ? NW : 1][C], edge[VP / 16];
    float rows[ALL ? C / 16 : 1][C], cols[ALL ? C / 16 : 1][C];  // parts of the pair sums, as in WalkLds
    int bad[2];                  // whether any wave's state is not finite, in turn for even and odd chunks
};

// Holds a loaded value where it is: the compiler otherwise moves each load under the condition that
// selects it, one after the other, and waits for every one.
__device__ __forceinline__ void keep(float &x) { asm volatile("" : "+v"(x)); }

__host__ __device__ inline int up32(int n) { return (n + 31) & ~31; }
__host__ __device__ inline int64_t kept_size(int rows, int cols) { return (int64_t)up32(rows) * up32(cols); }

// State of one wave: 16 columns, accumulator tiles of 16 rows (place()).
template <typename T, int KT>
struct State {
    typedef Mat<T> M;
    f32x4 t[KT];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int m = 0; m < KT; ++m) t[m] = zero4();
    }
    // Whether no value of the wave's part is infinite or NaN.
    __device__ __forceinline__ bool finite() const {
        float z = 0.f;
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) z = fmaf(t[m][i], 0.f, z);
        return !__any(z != 0.f);  // z is 0 or NaN
    }
    // Rows and columns of src at strides below 2^22 (32-bit offsets: 64 addresses would spill).  The loads
    // are only issued; settle() waits for them and zeroes what lies outside the state.
    __device__ __forceinline__ void load(const float *src, int rs, int cs, int v, int ka, int vc) {
        const int g4 = 4 * (lane_id() >> 4);
        const uint32_t col = (uint32_t)(min(v, vc - 1) * cs);
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) t[m][i] = src[col + (uint32_t)(min(M::place(m, g4) + i, ka - 1) * rs)];
    }
    __device__ __forceinline__ void settle(int v, int ka, int vc) {
        const int g4 = 4 * (lane_id() >> 4);
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = t[m][i];
                keep(x);
                t[m][i] = M::place(m, g4) + i < ka && v < vc ? x : 0.f;
            }
    }
    // The kept form of a whole state: [columns][rows], both rounded up to 32.
    __device__ __forceinline__ void keep_at(float *dst, int v, int rows, int cols) const {
        if ((v & ~15) >= cols) return;
        dst += v * rows + M::place(0, 4 * (lane_id() >> 4));
#pragma unroll
        for (int m = 0; m < KT; ++m)
            if (M::place(m, 0) < rows) *reinterpret_cast<f32x4 *>(dst + M::place(m, 0)) = t[m];
    }
    // A kept state as it was (the loads are only issued), or its transpose: columns and rows change places.
    __device__ __forceinline__ void load_kept(const float *src, int v, int rows, int cols) {
        zero();
        if ((v & ~15) >= cols) return;
        src += v * rows + M::place(0, 4 * (lane_id() >> 4));
#pragma unroll
        for (int m = 0; m < KT; ++m)
            if (M::place(m, 0) < rows) t[m] = *reinterpret_cast<const f32x4 *>(src + M::place(m, 0));
    }
    __device__ __forceinline__ void load_transposed(const float *src, int v, int rows, int cols) {
        zero();
        if ((v & ~15) >= cols) return;
        v = hidden(v);
        src += M::place(0, 4 * (hidden(lane_id()) >> 4)) * cols + v;
#pragma unroll
        for (int m = 0; m < KT; ++m)
            if (M::place(m, 0) < rows)
#pragma unroll
                for (int i = 0; i < 4; ++i) t[m][i] = src[(uint32_t)((M::place(m, 0) + i) * cols)];
    }
    // The wave's part of the sum of products with another state of the same form, without the columns past the width.
    __device__ __forceinline__ float dot(const State &x, bool column) const {
        float d = 0.f;
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) d = fmaf(t[m][i], x.t[m][i], d);
        return wave_sum(column ? d : 0.f);
    }
    // Dense rows of vc columns.
    __device__ __forceinline__ void store(float *dst, int v, int ka, int vc) const {
        const int g4 = 4 * (lane_id() >> 4);
        if (v >= vc) return;
        dst += M::place(0, g4) * vc + v;
        if (ka == 16 * KT) {
#pragma unroll
            for (int m = 0; m < KT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) dst[(uint32_t)((M::place(m, 0) + i) * vc)] = t[m][i];
            return;
        }
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (M::place(m, g4) + i < ka) dst[(uint32_t)((M::place(m, 0) + i) * vc)] = t[m][i];
    }
};

// The state after the chunk, tot S + sum_s col_s b_s c_s^T, and whether all of it is finite.
template <typename T, int KP>
__device__ __forceinline__ bool update(State<T, KP / 16> &U, const State<T, KP / 16> &S, float tot,
                                       const typename Mat<T>::Frag (&cf)[Mat<T>::C / Mat<T>::RB],
                                       const T *b, const float *col) {
    typedef Mat<T> M;
    constexpr int KT = KP / 16, RB = M::RB, LDA = M::ld(KP);
    U.zero();
#pragma unroll
    for (int r = 0; r < M::C / RB; ++r) {
        const float *f = col + r * RB + 4 * (lane_id() >> 4);
        // Four tiles one after the other: a product waits for none of the others.
        Split3 s3;
        float x[8];
#pragma unroll
        for (int e = 0; e < RB / 4; ++e) x[e] = static_cast<float>(cf[r][e]) * f[M::past(e)];
        if constexpr (sizeof(T) == 2) s3 = split3(x);
#pragma unroll
        for (int m0 = 0; m0 < KT; m0 += 4) {
            typename M::Frag y[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) y[m] = M::template across_place<LDA>(b, r * RB, m0 + m);
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int q = 0; q < 3; ++q)
#pragma unroll
                    for (int m = 0; m < 4; ++m) M::mma(U.t[m0 + m], y[m], s3.t[q]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        U.t[m0 + m] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[m][e], x[e], U.t[m0 + m], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < KT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) U.t[m][i] = fmaf(tot, S.t[m][i], U.t[m][i]);
    return U.finite();
}

// acc[j] += (row t of x) S for the tokens t of tile j: rows = the wave's columns, column = t.
template <typename T, int KP>
__device__ __forceinline__ void state_rows(f32x4 (&acc)[Mat<T>::C / 16], const State<T, KP / 16> &S, const T *x, int ld) {
    typedef Mat<T> M;
#pragma unroll
    for (int r = 0; r < KP / M::RB; ++r) {
        if constexpr (sizeof(T) == 2) {
            const f32x4 u = S.t[2 * r], w = S.t[2 * r + 1];
            const Split3 s3 = split3({u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]});
            typename M::Frag y[M::C / 16];
#pragma unroll
            for (int j = 0; j < M::C / 16; ++j) y[j] = M::row(x + 16 * j * ld, ld, r * M::RB);
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int j = 0; j < M::C / 16; ++j) M::mma(acc[j], s3.t[q], y[j]);
        } else {
#pragma unroll
            for (int j = 0; j < M::C / 16; ++j) M::mma(acc[j], S.t[r], M::row(x + 16 * j * ld, ld, r * M::RB));
        }
    }
}

// The value of the lane's 16-lane group (or of the lane's place in it) among four.
__device__ __forceinline__ float pick(int i, float a, float b, float c, float d) {
    return i < 2 ? (i == 0 ? a : b) : (i == 2 ? c : d);
}

// The wave's part of a dot product per token: its columns of d against acc, summed over the groups; the
// tiles side by side, so that the lane moves of one are the waits of the others.  f: row factors; a row
// with factor 0 gives 0, also where the state is not finite.
template <typename T, int TT>
__device__ __forceinline__ void dot_rows(const f32x4 (&acc)[TT], const float (&f)[TT], const T *d, int ld, float *red) {
    const int lane = hidden(lane_id()), n16 = lane & 15, g4 = 4 * (lane >> 4);
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        T e[4];
        __builtin_memcpy(e, __builtin_assume_aligned(d + (16 * j + n16) * ld + g4, 4 * sizeof(T)), sizeof e);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j] += acc[j][i] * Elem<T>::load(e, i);
        x[j] = f[j] == 0.f ? 0.f : x[j];
    }
    float y[4];
#pragma unroll
    for (int j = 0; j < TT; ++j) y[j] = __shfl_xor(x[j], 16);
#pragma unroll
    for (int j = 0; j < TT; ++j) x[j] += y[j];
#pragma unroll
    for (int j = 0; j < TT; ++j) y[j] = __shfl_xor(x[j], 32);
#pragma unroll
    for (int j = 0; j < TT; ++j) x[j] += y[j];
    if (lane < 16 * TT) red[lane] = pick(lane >> 4, x[0], x[1], x[2], x[3]);
}

// A token's dot product from the waves' parts (one wave, lane = token; 0 past the chunk).
template <int C, int NW, int ALL>
__device__ __forceinline__ float sum_dots(const float (&red)[ALL][C]) {
    const int lane = lane_id();
    float d = 0.f;
    if (lane < C) {
        d = red[0][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) d += red[w][lane];
    }
    return d;
}

// E from the waves' parts of <S0, R>; 0 at a cut, whatever the states hold.
template <int NW>
__device__ __forceinline__ float between(const float (&edge)[NW], float tot) {
    float e = edge[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) e += edge[w];
    return tot == 0.f ? 0.f : tot * e;
}

// The pair sums of a chunk from the parts by tiles, rows[si][t] (over the s of tile si, t of a later tile) and
// cols[tj][s] (over the t of tile tj; of a tile on the diagonal the sums themselves), and the sums of x from
// each token on and of y before it (one wave, lane = token): dg but for E.
//
// Sums from a lane to the end are sums up to it with the lanes turned round: scans add only what belongs to
// them, so that a value that is not finite stays with the tokens that see it.
template <int C>
__device__ __forceinline__ float gate_sums(const float (&rows)[C / 16][C], const float (&cols)[C / 16][C], float x, float y) {
    constexpr int TT = C / 16;
    const int lane = lane_id(), n16 = lane & 15, j = lane / 16;
    // Token t of tile j: rows u >= t of the tile over the tiles to their left, columns s < t of the tile over
    // the tiles below, whole tiles below and to the left, and its own tile.
    float left = 0.f, below = 0.f, dg = 0.f, r0 = 0.f, r1 = 0.f;
    if (lane < C) {
        if (j > 0) left = r0 = rows[0][lane];
        if (j < 1) below += cols[1][lane];
        if constexpr (TT == 4) {
            if (j > 1) left += r1 = rows[1][lane];
            if (j > 2) left += rows[2][lane];
            if (j < 2) below += cols[2][lane];
            if (j < 3) below += cols[3][lane];
        }
        dg = cols[j][lane];
    }
    if (TT == 4) {
        const float f1 = wave_sum(lane >= 32 ? r0 : 0.f);
        const float f2 = wave_sum(lane >= 48 ? r0 + r1 : 0.f);
        dg += j == 1 ? f1 : j == 2 ? f2 : 0.f;
    }
    const int turned = lane ^ 15;
    float up = __shfl(left, turned);
    row_scan(up);
    float before = __shfl_up(below, 1), y_before = __shfl_up(y, 1);
    if (n16 == 0) before = 0.f;
    row_scan(before);
    const float x_on = wave_scan_add(__shfl(x, 63 - lane));
    const float y_sum = wave_scan_add(lane == 0 ? 0.f : y_before);
    return dg + ((__shfl(up, turned) + before) + (__shfl(x_on, 63 - lane) + y_sum));
}

// A chunk token by token, taken where the state before or after it is not finite: products over masked
// tokens, and with factors that are 0, would spread such a value to tokens that do not see it.
template <typename T, int KP, int LDC, bool REV, bool OUT>
__device__ __forceinline__ void walk_tokens(State<T, KP / 16> &S, const T *a, const T *b, const T *c,
                                            const GateTile<Mat<T>::C> &gate, int ka, int v, int vc,
                                            T *out, int64_t stride, int tokens) {
    constexpr int KT = KP / 16, C = Mat<T>::C, LDA = Mat<T>::ld(KP);
    const int g4 = hidden(4 * (lane_id() >> 4));
    v = hidden(v);
#pragma unroll 1
    for (int n = 0; n < C; ++n) {
        const int t = REV ? C - 1 - n : n;
        if (t >= tokens) continue;
        const float f = gate.step[t];
        float o = 0.f;
        if (gate.seg[t] >= 0) {
            const float x = Elem<T>::load(c, t * LDC + v);
#pragma unroll
            for (int m = 0; m < KT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = Mat<T>::place(m, g4) + i;
                    if (k >= ka) continue;  // 0 there, whatever x is
                    if (!REV) S.t[m][i] = decayed(S.t[m][i], f);
                    S.t[m][i] += Elem<T>::load(b, t * LDA + k) * x;
                    if (OUT) o += Elem<T>::load(a, t * LDA + k) * S.t[m][i];
                    if (REV) S.t[m][i] = decayed(S.t[m][i], f);
                }
            o = groups_sum(o);
        }
        if (OUT && out && lane_id() < 16 && v < vc) Elem<T>::store(out, t * stride + v, o);
    }
}

// A workgroup's place: segments that share a (batch, head) take neighbouring numbers on one XCD, the
// longest prewalk first.
struct Place {
    int64_t b, h;
    int bh, seg, nth;  // nth: the segment's place in the walk's order
};
__device__ __forceinline__ Place place(const Walk &p, int segs, bool rev, bool longest_first) {
    const unsigned total = gridDim.x, xcd = blockIdx.x % 8, whole = total / 8, rest = total % 8;
    const unsigned id = xcd * whole + min(xcd, rest) + blockIdx.x / 8;
    Place r;
    r.bh = id / segs;
    r.nth = longest_first ? segs - 1 - (int)(id % segs) : (int)(id % segs);
    r.b = r.bh / p.H, r.h = r.bh % p.H;
    r.seg = rev ? p.segments - 1 - r.nth : r.nth;
    return r;
}

template <typename T>
__device__ __forceinline__ const T *head_rows(const View &x, const Place &at) {
    return reinterpret_cast<const T *>(x.data) + at.b * x.s0 + at.h * x.s2;
}

// The state before a walk's segment: at hand (stored), or the walk's first.
template <typename T, int KT>
__device__ __forceinline__ void start_state(State<T, KT> &S, const Walk &p, const Place &at, bool stored, int v,
                                            int ka, int vc) {
    const float *src = reinterpret_cast<const float *>(p.first.data);
    int rs = (int)p.first.s2, cs = (int)p.first.s3;
    int64_t off = at.b * p.first.s0 + at.h * p.first.s1;
    if (stored) {
        src = p.starts, rs = p.s_row, cs = p.s_col;
        off = at.bh * p.s_bh + at.seg * (int64_t)ka * vc;
    }
    if (src) S.load(src + off, rs, cs, v, ka, vc);
}

// Gates of the next chunks of a walk with n left, from chunk ci on.
template <int C, bool REV, int NW, int GATES>
struct MakeGates {
    static constexpr int EACH = GATES / NW;  // chunks of each wave
    GateIn x[EACH];
    int ci, n;
    __device__ __forceinline__ void load(const Walk &p, const Place &at, int chunk, int left) {
        ci = chunk, n = left;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int k = min((int)(threadIdx.x >> 6) + i * NW, n - 1);
            x[i] = gate_load<C>(p, at.b, at.h, ci + (REV ? -k : k));
        }
    }
    __device__ __forceinline__ void store(const Walk &p, GateTile<C> *gate) const {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int k = (int)(threadIdx.x >> 6) + i * NW;
            const int64_t c = ci + (REV ? -k : k);
            if (k < n) gate_store<C, REV>(x[i], (int)min(p.T - c * C, (int64_t)C), &gate[k]);
        }
    }
};

// One workgroup: a segment's chunks in the walk's order.  Each wave owns 16 columns of the state, so its
// part stays in its accumulators, where it is at once the product's operand of the next chunk: neither
// the state nor its update passes through LDS.  The next chunk's tiles are on their way while one is
// worked on.  Without `starts` a segment's start state is walked to from the sequence's start (prewalk: b
// and c alone).  OUT = false: only the state that the segment adds and its decay (carry; REV: from the
// last chunk to the first).
// DOT: the gate's gradient too, with (a, b, c, d) = (do, v, k, q): the products of the state's part with d
// are its x, and W_us = Gam_us (a_u.b_s)(d_u.c_s).
//
// Bound by latency: a chunk's tiles, weights, products and state wait for each other with two to four waves on
// each SIMD.  bf16: 16 x 512 tokens, 8 heads of 64, forward 26.4 us (52 MB with the kept states, 2.0 TB/s); 4 x 8192
// tokens, 16 heads of 128, forward 205 us (2.6 TB/s), dq and dg 368 us (1.2 GB with the adjoint states, 3.3 TB/s), a
// carry 72 us (3.7 TB/s).  The second terms of the pair weights, and the second and third of the state, are a fifth to
// a quarter of a wide forward.  Rows lie in LDS and states in accumulators as Mat says: with a state by 16 rows a
// tile and rows of 136 a wide forward took an eighth longer, in bank conflicts.  The carry at 128 columns has four
// waves a SIMD; with two it took a fifth longer.
template <typename T, int KP, int CP, bool VEC, bool REV, bool OUT, bool DOT>
__global__ void __launch_bounds__(4 * CP, CP == 64 ? 2 : OUT ? 1 : 4) linear_walk(Forward p) {
    static_assert(!(OUT && REV), "");
    typedef Mat<T> M;
    typedef WalkLds<T, KP, CP, OUT, DOT> L;
    constexpr int C = M::C, TT = C / 16, KT = KP / 16, RB = M::RB, LDA = L::LDA, LDC = L::LDC,
                  LDP = L::LDP, BT = RB / 16;  // BT: accumulator tiles of one fragment
    constexpr int NW = CP / 16;
    __shared__ L lds;
    const int lane = lane_id(), n16 = lane & 15, g4 = 4 * (lane >> 4);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int v = 16 * wave + n16;
    const int segs = p.segments - (OUT ? 0 : 1);
    const Place at = place(p, segs, REV, OUT);
    const int c_lo = at.seg * p.seg_chunks, c_hi = min(p.chunks, c_lo + p.seg_chunks);

    int n = c_hi - c_lo;   // chunks to walk, the last `out` of them with results
    const int out = OUT ? n : 0;
    const bool walked = OUT && !(at.nth > 0 && p.starts);  // from the sequence's start
    if (walked) n = c_hi;
    double sum = 0.;  // carry: log2 of the segment's decay
    bool cut = false;
    int ci = REV ? c_lo + n - 1 : c_hi - n;

    Staged<T, KP, 64 * NW, VEC> sa, sb;
    Staged<T, CP, 64 * NW, VEC> sc, sd;
    const T *pa = head_rows<T>(p.a, at), *pb = head_rows<T>(p.b, at);
    const T *pc = head_rows<T>(p.c, at), *pd = head_rows<T>(p.d, at);
    const auto fetch = [&](int chunk, bool full) {
        const int64_t t0 = (int64_t)chunk * C;
        const int left = (int)min(p.T - t0, (int64_t)C);
        sb.load(pb, p.b.s1, p.b.s3, t0, left, p.ka);
        sc.load(pc, p.c.s1, p.c.s3, t0, left, p.vc);
        if (OUT && full) {
            sa.load(pa, p.a.s1, p.a.s3, t0, left, p.ka);
            if (DOT) sd.load(pd, p.d.s1, p.d.s3, t0, left, p.vc);
        }
    };
    // All first loads are on their way before the first is waited for.
    MakeGates<C, REV, NW, L::GATES> gates;
    gates.load(p, at, ci, n);
    State<T, KT> S;
    S.zero();
    if (OUT) start_state(S, p, at, !walked, v, p.ka, p.vc);
    fetch(ci, n <= out);
    int gi = 0;  // the chunk's place among the gates in LDS
    gates.store(p, lds.gate);
    S.settle(v, p.ka, p.vc);
    __syncthreads();

    const bool odd = p.valid.data || p.ka < KP || p.vc < CP;
    bool fine = S.finite();  // products take a chunk only where the state before it is finite
    const auto across_c = [&](typename M::Frag (&cf)[C / RB]) {
#pragma unroll
        for (int r = 0; r < C / RB; ++r) cf[r] = M::template across<LDC>(lds.c, r * RB, 16 * wave);
    };
    const auto next_gates = [&]() {
        gates.load(p, at, REV ? ci - 1 : ci + 1, n - 1);
        gates.store(p, lds.gate);
        gi = 0;
        __syncthreads();
    };

    for (; n > out; --n, ci += REV ? -1 : 1) {
        const GateTile<C> &gate = lds.gate[gi];
        const bool masks = odd || p.T - (int64_t)ci * C < C;
        sb.template store<LDA>(lds.b, gate.seg, masks, p.ka);
        sc.template store<LDC>(lds.c, gate.seg, masks, p.vc);
        if (n > 1) fetch(REV ? ci - 1 : ci + 1, n - 1 <= out);
        __syncthreads();
        typename M::Frag cf[C / RB];
        across_c(cf);
        State<T, KT> U;
        const bool next = update<T, KP>(U, S, gate.tot, cf, lds.b, gate.col);
        // A cut leaves nothing of the start, whatever the gates before and after it are.
        sum += gate.sum, cut = cut || gate.span == 0.f;
        if (__builtin_expect(fine && next, 1)) {
            S = U;
        } else {
            walk_tokens<T, KP, LDC, REV, false>(S, lds.b, lds.b, lds.c, gate, p.ka, v, p.vc, nullptr, 0,
                                                (int)min(p.T - (int64_t)ci * C, (int64_t)C));
            fine = S.finite();
        }
        __syncthreads();  // the chunk's tiles are read
        if (++gi == L::GATES && n > 1) next_gates();
    }
    if (!OUT) {
        S.store(p.seg_state + ((int64_t)at.bh * p.segments + at.seg) * p.ka * p.vc, v, p.ka, p.vc);
        if (threadIdx.x == 0) p.seg_decay[(int64_t)at.bh * p.segments + at.seg] = cut ? 0.f : root_exp2((float)sum);
        return;
    }
    if (p.starts_out && at.nth > 0)
        S.store(p.starts_out + at.bh * p.s_bh + at.seg * (int64_t)p.ka * p.vc, v, p.ka, p.vc);

    // DOT: the adjoint state behind the chunk, in the form of S.
    const int64_t size = kept_size(p.ka, p.vc);
    const float *adj = DOT ? p.adj + (int64_t)at.bh * p.chunks * size : nullptr;
    State<T, KT> R;
    if constexpr (DOT) R.load_transposed(adj + ci * size, v, up32(p.ka), up32(p.vc));
    for (; n > 0; --n, ++ci) {
        const GateTile<C> &gate = lds.gate[gi];
        const bool masks = odd || p.T - (int64_t)ci * C < C;
        sa.template store<LDA>(lds.a, gate.seg, masks, p.ka);
        sb.template store<LDA>(lds.b, gate.seg, masks, p.ka);
        sc.template store<LDC>(lds.c, gate.seg, masks, p.vc);
        if (DOT) sd.template store<LDC>(lds.d, gate.seg, masks, p.vc);
        if (p.kept) S.keep_at(p.kept + ((int64_t)at.bh * (p.chunks + 1) + ci) * size, v, up32(p.ka), up32(p.vc));
        if (n > 1) fetch(ci + 1, true);
        const int64_t token = (int64_t)ci * C + lane;
        float y_now = 0.f;  // of this chunk, for the wave that adds up dg
        if (DOT && wave == 1) y_now = p.y[at.bh * p.T + min(token, p.T - 1)];
        if constexpr (DOT) {
            const float e = S.dot(R, v < p.vc);
            if (lane == 0) lds.edge[wave] = e;
        }
        __syncthreads();

        // P_ts = Gam_ts a_t.b_s for the tiles whose block of RB sources is seen from the rows: twelve in
        // bf16, three in float32.
        constexpr int MINE = TT == 4 ? (12 + NW - 1) / NW : 1;
        f32x4 y[MINE];
        T lo[MINE][4];
        int tjs[MINE], sis[MINE];
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
            const int id = wave + m * NW;
            int tj = id >> 1, si = id & 1;
            if (TT == 4 && id >= 4) tj = id < 8 ? 2 : 3, si = id & 3;
            tjs[m] = tj, sis[m] = si;
            // none: a wave without a tile, or a block of 16 sources that no row sees
            if ((TT == 4 && 12 % NW && id >= 12) || (TT == 2 && (id >= 4 || si > tj))) {
                tjs[m] = -1;
                continue;
            }
            f32x4 x = zero4();
#pragma unroll
            for (int r = 0; r < KP; r += RB)
                M::mma(x, M::row(lds.b + 16 * si * LDA, LDA, r), M::row(lds.a + 16 * tj * LDA, LDA, r));
            const int t = 16 * tj + n16, s = 16 * si + g4;
            const f32x4 f = pair_decays<C, false>(gate, t, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = seen(x[i], f[i]);
            T hi[4];
            split2(x, hi, lo[m]);
            T *at_p = lds.p + t * LDP + M::place(si, g4);
            __builtin_memcpy(__builtin_assume_aligned(at_p, 4 * sizeof(T)), hi, sizeof hi);
            if (L::ROOM == 2)
                __builtin_memcpy(__builtin_assume_aligned(at_p + C * LDP, 4 * sizeof(T)), lo[m], sizeof hi);
            if (DOT) {
                y[m] = zero4();
#pragma unroll
                for (int r = 0; r < CP; r += RB)
                    M::mma(y[m], M::row(lds.c + 16 * si * LDC, LDC, r), M::row(lds.d + 16 * tj * LDC, LDC, r));
#pragma unroll
                for (int i = 0; i < 4; ++i) y[m][i] = f[i] == 0.f || s + i >= t ? 0.f : x[i] * y[m][i];
            }
        }
        if constexpr (DOT) {
            // By tiles: the sums over s for each row, and over the rows for each s; of a tile on the diagonal, for
            // each of its tokens, the sum over the rows from it on and the s before it.  All tiles of the wave
            // side by side.
            float q[MINE], a[MINE], b[MINE], c[MINE];
#pragma unroll
            for (int m = 0; m < MINE; ++m) q[m] = (y[m][0] + y[m][1]) + (y[m][2] + y[m][3]);
#pragma unroll
            for (int m = 0; m < MINE; ++m)
                a[m] = __shfl_up(q[m], 16), b[m] = __shfl_up(q[m], 32), c[m] = __shfl_up(q[m], 48);
#pragma unroll
            for (int m = 0; m < MINE; ++m) {
                const float pre = (g4 > 0 ? a[m] : 0.f) + (g4 > 4 ? b[m] : 0.f) + (g4 > 8 ? c[m] : 0.f);
                const bool diag = tjs[m] == sis[m];
                float z[4], before = pre;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    z[i] = row16_sum(diag ? (n16 >= g4 + i ? before : 0.f) : y[m][i]);
                    before += y[m][i];
                }
                if (tjs[m] < 0 || sis[m] > tjs[m]) continue;
                const int s = 16 * sis[m] + g4;
                if (n16 < 4) lds.cols[tjs[m]][s + n16] = pick(n16, z[0], z[1], z[2], z[3]);
                if (lane >= 48) lds.rows[sis[m]][16 * tjs[m] + n16] = pre + q[m];  // the last group: all s
            }
        }
        // acc[j]: rows = the wave's columns, column = token 16 j + n16; the state's part.
        f32x4 acc[TT];
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[j] = zero4();
        state_rows<T, KP>(acc, S, lds.a, LDA);
        float f[TT];
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            f[j] = gate.row[16 * j + n16];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = seen(acc[j][i], f[j]);
        }
        if constexpr (DOT) dot_rows<T, TT>(acc, f, lds.d + 16 * wave, LDC, lds.red[wave]);
        __syncthreads();
        if constexpr (DOT) if (wave == 1) {
            const bool in = lane < C && token < p.T;
            const float x = sum_dots<C, NW>(lds.red), y = in ? y_now : 0.f;
            const float dg = gate_sums<C>(lds.rows, lds.cols, x, y) + between<NW>(lds.edge, gate.span);
            const bool on = in && gate.seg[lane] >= 0 && gate.step[lane] != 0.f;
            if (in) p.dg[(at.b * p.T + token) * p.H + at.h] = on ? dg : 0.f;
        }

        constexpr bool LATE = DOT && L::TERMS == 2;
        if constexpr (LATE)
#pragma unroll
            for (int m = 0; m < MINE; ++m)
                if (tjs[m] >= 0)
                    __builtin_memcpy(__builtin_assume_aligned(
                                         lds.d + (16 * tjs[m] + n16) * LDP + M::place(sis[m], g4), 4 * sizeof(T)),
                                     lo[m], sizeof lo[m]);
        typename M::Frag cf[C / RB];
        across_c(cf);
        State<T, KT> U;
        const bool next = update<T, KP>(U, S, gate.tot, cf, lds.b, gate.col);
        if (LATE) __syncthreads();
        const T *const terms[2] = {lds.p, DOT ? lds.d : lds.p + C * LDP};
        T *o = reinterpret_cast<T *>(p.out);
        const int64_t row0 = (at.b * p.T + (int64_t)ci * C) * p.H + at.h;
        const int left = (int)min(p.T - (int64_t)ci * C, (int64_t)C);
        if (__builtin_expect(fine && next, 1)) {
#pragma unroll
            for (int j = 0; j < TT; ++j)
#pragma unroll
                for (int r = 0; r <= j / BT; ++r)
#pragma unroll
                    for (int q = 0; q < L::TERMS; ++q)
                        M::mma(acc[j], cf[r], M::row(terms[q] + 16 * j * LDP, LDP, r * RB));
            if (o)
                store_rows<T, TT, VEC>(o + row0 * p.vc, (int64_t)p.H * p.vc, 16 * wave + g4, p.vc, left, acc);
            S = U;
        } else {
            walk_tokens<T, KP, LDC, false, true>(S, lds.a, lds.b, lds.c, gate, p.ka, v, p.vc,
                                                 o ? o + row0 * p.vc : nullptr, (int64_t)p.H * p.vc, left);
            fine = S.finite();
        }
        if (DOT && n > 1) R.load_transposed(adj + (ci + 1) * size, v, up32(p.ka), up32(p.vc));
        __syncthreads();  // the chunk's tiles are read
        if (++gi == L::GATES && n > 1) next_gates();
    }
    if (at.nth != p.segments - 1) return;
    if (p.fin) S.store(p.fin + (int64_t)at.bh * p.ka * p.vc, v, p.ka, p.vc);
    if (p.kept)
        S.keep_at(p.kept + ((int64_t)at.bh * (p.chunks + 1) + p.chunks) * size, v, up32(p.ka), up32(p.vc));
}

// dv and dk, from the last chunk to the first, and more by MODE.  A wave owns 16 value columns of the adjoint state
// [K, V] and of dv as linear_walk's waves do theirs, and 16 columns of dk; for dk the state goes through LDS, a
// term in the type of the inputs at a time, as each of its values meets all key columns.  (A walk of its own for dk
// read three of the four tensors again, and took its pairs' decays and the state's update a second time.)  MODE 1: also
// y_s = row_s k_s^T S v_s and the adjoint state behind every chunk, for the dq walk.  MODE 2: dq and dg as well,
// from the forward's states before every chunk (all_in_one).
//
// Bound like linear_walk: bf16, 16 x 512 tokens, 8 heads of 64, all in one 46.6 us (78 MB, 1.7 TB/s); 4 x 8192
// tokens, 16 heads of 128, without dq 471 us (1.3 GB with the adjoint states that it leaves, 2.9 TB/s; without those,
// here and in the dq walk, 166 us less), one workgroup of eight waves a unit for its 144 KB of LDS and 256 registers.
template <typename T, int KP, int VP, bool VEC, int MODE>
__global__ void __launch_bounds__(4 * (KP > VP ? KP : VP), (KP > VP ? KP : VP) == 64 ? 2 : 1) linear_back(Back p) {
    typedef Mat<T> M;
    constexpr bool ALL = MODE == 2, DOT = MODE >= 1;
    typedef BackLds<T, KP, VP, ALL> L;
    constexpr int C = M::C, TT = C / 16, KT = KP / 16, RB = M::RB, LDK = L::LDK, LDV = L::LDV,
                  LDP = L::LDP, BT = RB / 16, NW = L::NW, THREADS = 64 * NW;
    __shared__ L lds;
    const int lane = lane_id(), n16 = lane & 15, g4 = 4 * (lane >> 4);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int v = 16 * wave + n16;
    const bool own_v = 16 * wave < VP, own_k = 16 * wave < KP;
    const Place at = place(p, p.segments, true, true);
    const int c_lo = at.seg * p.seg_chunks, c_hi = min(p.chunks, c_lo + p.seg_chunks);
    int n = c_hi - c_lo;
    const int out = n;
    const bool walked = !(at.nth > 0 && p.starts);
    if (walked) n = p.chunks - c_lo;
    int ci = c_lo + n - 1;

    Staged<T, KP, THREADS, VEC> sq, sk;
    Staged<T, VP, THREADS, VEC> sv, so;
    const T *pq = head_rows<T>(p.q, at), *pk = head_rows<T>(p.k, at);
    const T *pv = head_rows<T>(p.v, at), *po = head_rows<T>(p.o, at);
    const auto fetch = [&](int chunk, bool full) {
        const int64_t t0 = (int64_t)chunk * C;
        const int left = (int)min(p.T - t0, (int64_t)C);
        sq.load(pq, p.q.s1, p.q.s3, t0, left, p.K);
        so.load(po, p.o.s1, p.o.s3, t0, left, p.V);
        if (full) {
            sk.load(pk, p.k.s1, p.k.s3, t0, left, p.K);
            sv.load(pv, p.v.s1, p.v.s3, t0, left, p.V);
        }
    };
    MakeGates<C, true, NW, L::GATES> gates;
    gates.load(p, at, ci, n);
    State<T, KT> S;
    S.zero();
    if (own_v) start_state(S, p, at, !walked, v, p.K, p.V);
    fetch(ci, n <= out);
    int gi = 0;
    gates.store(p, lds.gate);
    S.settle(v, p.K, p.V);
    if (threadIdx.x < 2) lds.bad[threadIdx.x] = 0;
    __syncthreads();

    const bool odd = p.valid.data || p.K < KP || p.V < VP;
    bool fine = S.finite();
    const auto across_o = [&](typename M::Frag (&of)[C / RB]) {
#pragma unroll
        for (int r = 0; r < C / RB; ++r) of[r] = M::template across<LDV>(lds.o, r * RB, 16 * wave);
    };
    const auto next_gates = [&]() {
        gates.load(p, at, ci - 1, n - 1);
        gates.store(p, lds.gate);
        gi = 0;
        __syncthreads();
    };

    for (; n > out; --n, --ci) {
        const GateTile<C> &gate = lds.gate[gi];
        const bool masks = odd || p.T - (int64_t)ci * C < C;
        sq.template store<LDK>(lds.q, gate.seg, masks, p.K);
        so.template store<LDV>(lds.o, gate.seg, masks, p.V);
        fetch(ci - 1, n - 1 <= out);
        __syncthreads();
        if (own_v) {
            typename M::Frag of[C / RB];
            across_o(of);
            State<T, KT> U;
            const bool next = update<T, KP>(U, S, gate.tot, of, lds.q, gate.col);
            if (__builtin_expect(fine && next, 1)) {
                S = U;
            } else {
                walk_tokens<T, KP, LDV, true, false>(S, lds.q, lds.q, lds.o, gate, p.K, v, p.V, nullptr, 0,
                                                     (int)min(p.T - (int64_t)ci * C, (int64_t)C));
                fine = S.finite();
            }
        }
        __syncthreads();
        if (++gi == L::GATES) next_gates();
    }

    // ALL: the forward's state before the chunk, transposed: rows = values, the wave's 16 columns = keys.
    const bool gates_too = ALL && p.dg;
    const int64_t size = kept_size(p.K, p.V);
    const float *kept = ALL ? p.kept + (int64_t)at.bh * (p.chunks + 1) * size : nullptr;
    State<T, VP / 16> F;
    State<T, KT> S0;  // gates_too: the same as it is
    if (gates_too) S0.load_kept(kept + ci * size, v, up32(p.K), up32(p.V));

    for (; n > 0; --n, --ci) {
        const GateTile<C> &gate = lds.gate[gi];
        const bool masks = odd || p.T - (int64_t)ci * C < C;
        sq.template store<LDK>(lds.q, gate.seg, masks, p.K);
        sk.template store<LDK>(lds.k, gate.seg, masks, p.K);
        sv.template store<LDV>(lds.v, gate.seg, masks, p.V);
        so.template store<LDV>(lds.o, gate.seg, masks, p.V);
        const auto put_D = [&](int term) {
#pragma unroll
            for (int m = 0; m < KT; ++m) {
                T e[2][4];
                split2(S.t[m], e[0], e[1]);
                __builtin_memcpy(__builtin_assume_aligned(lds.D + M::row_for(v) * LDK + M::place(m, g4), 4 * sizeof(T)),
                                 e[term], sizeof e[0]);
            }
        };
        if (own_v) put_D(0);
        if (MODE == 1 && own_v)
            S.keep_at(p.adj + ((int64_t)at.bh * p.chunks + ci) * size, v, up32(p.K), up32(p.V));
        if (ALL) F.load_transposed(kept + ci * size, v, up32(p.V), up32(p.K));
        if (n > 1) fetch(ci - 1, true);
        if (gates_too) {
            const float e = S.dot(S0, v < p.V);
            if (lane == 0) lds.edge[wave] = e;
        }
        __syncthreads();

        // For out token s and source t >= s: pk = Gam k_s.q_t, pv = Gam v_s.do_t, by tiles as in linear_walk
        // but from the other end.
        constexpr int MINE = TT == 4 ? (12 + NW - 1) / NW : 1;
        f32x4 W[MINE];
        T pk_lo[MINE][4], pv_lo[MINE][4];
        int sjs[MINE], tis[MINE];
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
            const int id = wave + m * NW;
            int sj = id >> 1, ti = id & 1;
            if (TT == 4 && id >= 4) sj = id < 8 ? 2 : 3, ti = id & 3;
            sjs[m] = TT - 1 - sj, tis[m] = TT - 1 - ti;
            const int lane = hidden(lane_id()), n16 = lane & 15, g4 = 4 * (lane >> 4);
            if ((TT == 4 && 12 % NW && id >= 12) || (TT == 2 && (id >= 4 || ti > sj))) {
                sjs[m] = -1;
                continue;
            }
            sj = sjs[m], ti = tis[m];
            f32x4 x = zero4(), y = zero4();
#pragma unroll
            for (int r = 0; r < KP; r += RB)
                M::mma(x, M::row(lds.q + 16 * ti * LDK, LDK, r), M::row(lds.k + 16 * sj * LDK, LDK, r));
#pragma unroll
            for (int r = 0; r < VP; r += RB)
                M::mma(y, M::row(lds.o + 16 * ti * LDV, LDV, r), M::row(lds.v + 16 * sj * LDV, LDV, r));
            const int s = 16 * sj + n16, t = 16 * ti + g4;
            const f32x4 f = pair_decays<C, true>(gate, s, t);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = seen(x[i], f[i]);
                if (ALL) W[m][i] = f[i] == 0.f || t + i <= s ? 0.f : x[i] * y[i];
                y[i] = seen(y[i], f[i]);
            }
            T e[4], g[4];
            split2(x, e, pk_lo[m]);
            split2(y, g, pv_lo[m]);
            const int at_p = s * LDP + M::place(ti, g4);
            __builtin_memcpy(__builtin_assume_aligned(lds.pk + at_p, 4 * sizeof(T)), e, sizeof e);
            __builtin_memcpy(__builtin_assume_aligned(lds.pv + at_p, 4 * sizeof(T)), g, sizeof g);
        }
        if (gates_too) {
            // As in linear_walk, with t along the rows: sums over the s of a tile for each t, over its t for each
            // s, and on the diagonal for each token over the t from it on and the s before it.
            const int lane = hidden(lane_id()), n16 = lane & 15, g4 = 4 * (lane >> 4);
            float q[MINE], a[MINE], b[MINE], c[MINE];
#pragma unroll
            for (int m = 0; m < MINE; ++m) q[m] = (W[m][0] + W[m][1]) + (W[m][2] + W[m][3]);
#pragma unroll
            for (int m = 0; m < MINE; ++m)
                a[m] = __shfl_down(q[m], 16), b[m] = __shfl_down(q[m], 32), c[m] = __shfl_down(q[m], 48);
#pragma unroll
            for (int m = 0; m < MINE; ++m) {
                const float post = (g4 < 12 ? a[m] : 0.f) + (g4 < 8 ? b[m] : 0.f) + (g4 < 4 ? c[m] : 0.f);
                const bool diag = sjs[m] == tis[m];
                float z[4], from = post;
#pragma unroll
                for (int i = 3; i >= 0; --i) {
                    from += W[m][i];
                    z[i] = row16_sum(diag ? (n16 < g4 + i ? from : 0.f) : W[m][i]);
                }
                if (sjs[m] < 0 || tis[m] < sjs[m]) continue;
                const float mine = pick(n16, z[0], z[1], z[2], z[3]);
                const int t = 16 * tis[m] + g4 + n16;
                if (n16 < 4) (diag ? lds.cols[tis[m]] : lds.rows[sjs[m]])[t] = mine;
                if (!diag && lane < 16) lds.cols[tis[m]][16 * sjs[m] + n16] = post + q[m];  // the first group: all t
            }
        }
        // The state's parts: rows = the wave's columns, column = token 16 j + n16.
        f32x4 av[TT], ak[TT];
#pragma unroll
        for (int j = 0; j < TT; ++j) av[j] = ak[j] = zero4();
        const auto dk_state = [&](f32x4 (&acc)[TT]) {  // with the term of the state that is in LDS
#pragma unroll
            for (int r = 0; r < VP; r += RB) {
                const typename M::Frag x = M::template across<LDK>(lds.D, r, 16 * wave);
#pragma unroll
                for (int j = 0; j < TT; ++j) M::mma(acc[j], x, M::row(lds.v + 16 * j * LDV, LDV, r));
            }
        };
        State<T, KT> U;
        U.zero();
        typename M::Frag of[C / RB], kf[ALL ? C / RB : 1];
        bool good = fine;
        if (own_v) {
            state_rows<T, KP>(av, S, lds.k, LDK);
            across_o(of);
            good = update<T, KP>(U, S, gate.tot, of, lds.q, gate.col) && fine;
        }
        if (own_k) {
            dk_state(ak);
            if constexpr (ALL)
#pragma unroll
                for (int r = 0; r < C / RB; ++r) kf[r] = M::template across<LDK>(lds.k, r * RB, 16 * wave);
        }
        f32x4 aq[TT];
        if (ALL) {
#pragma unroll
            for (int j = 0; j < TT; ++j) aq[j] = zero4();
            state_rows<T, VP>(aq, F, lds.o, LDV);
            // A value of k or v that is not finite shows in these products, whatever the state: then dq, too, is
            // taken token by token.
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < TT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) z = fmaf(aq[j][i], 0.f, fmaf(av[j][i], 0.f, fmaf(ak[j][i], 0.f, z)));
            good = good && !__any(z != 0.f);
        }
        float f[TT];
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            f[j] = gate.row[16 * j + n16];
#pragma unroll
            for (int i = 0; i < 4; ++i) av[j][i] = seen(av[j][i], f[j]), ak[j][i] = seen(ak[j][i], f[j]);
        }
        if (DOT && own_v && (!ALL || gates_too)) dot_rows<T, TT>(av, f, lds.v + 16 * wave, LDV, lds.red[wave]);
        if (ALL) {
            float c[TT];
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                c[j] = gate.col[16 * j + n16];  // of the walk in order
#pragma unroll
                for (int i = 0; i < 4; ++i) aq[j][i] = seen(aq[j][i], c[j]);
            }
            if (gates_too) dot_rows<T, TT>(aq, c, lds.q + 16 * wave, LDK, lds.red_q[wave]);
        }
        if (!good && lane == 0) lds.bad[n & 1] = 1;
        __syncthreads();
        const bool bad = lds.bad[n & 1] != 0;
        if (threadIdx.x == 0) lds.bad[(n & 1) ^ 1] = 0;
        if (MODE == 1 && wave == 1) {
            const int64_t t = (int64_t)ci * C + lane;
            const float y = sum_dots<C, VP / 16>(lds.red);
            if (lane < C && t < p.T) p.y[at.bh * p.T + t] = y;
        }
        if constexpr (ALL)
            if (gates_too && wave == 1) {
                const int64_t token = (int64_t)ci * C + lane;
                const float x = sum_dots<C, KP / 16>(lds.red_q), y = sum_dots<C, VP / 16>(lds.red);
                const float dg = gate_sums<C>(lds.rows, lds.cols, x, y) + between<VP / 16>(lds.edge, gate.span);
                const bool on = gate.seg[lane & (C - 1)] >= 0 && gate.step[lane & (C - 1)] != 0.f;
                if (lane < C && token < p.T) p.dg[(at.b * p.T + token) * p.H + at.h] = on ? dg : 0.f;
            }
        const int left = (int)min(p.T - (int64_t)ci * C, (int64_t)C);
        const int64_t row0 = (at.b * p.T + (int64_t)ci * C) * p.H + at.h;
        T *dv = reinterpret_cast<T *>(p.dv), *dk = reinterpret_cast<T *>(p.dk);
        T *dq = ALL && p.dq ? reinterpret_cast<T *>(p.dq) + row0 * p.K : nullptr;
        if (__builtin_expect(!bad, 1)) {
            T *const pk_of[2] = {lds.pk, lds.o}, *const pv_of[2] = {lds.pv, lds.k};
            constexpr int TERMS = sizeof(T) == 2 ? 2 : 1;
            if constexpr (TERMS == 2) {
#pragma unroll
                for (int m = 0; m < MINE; ++m) {
                    if (sjs[m] < 0) continue;
                    const int at_p = (16 * sjs[m] + n16) * LDP + M::place(tis[m], g4);
                    __builtin_memcpy(__builtin_assume_aligned(lds.o + at_p, 8), pk_lo[m], 8);
                    __builtin_memcpy(__builtin_assume_aligned(lds.k + at_p, 8), pv_lo[m], 8);
                }
                if (own_v) put_D(1);
            }
            static_assert(LDV >= LDP && LDK >= LDP, "");
#pragma unroll
            for (int q = 0; q < TERMS; ++q) {
                if (q == 1) {
                    __syncthreads();
                    if (dk && own_k) {
                        f32x4 x[TT];
#pragma unroll
                        for (int j = 0; j < TT; ++j) x[j] = zero4();
                        dk_state(x);
#pragma unroll
                        for (int j = 0; j < TT; ++j) {
                            const float row = gate.row[16 * j + n16];
#pragma unroll
                            for (int i = 0; i < 4; ++i) ak[j][i] += seen(x[j][i], row);
                        }
                    }
                }
                if (dv && own_v) {
#pragma unroll
                    for (int j = 0; j < TT; ++j)
#pragma unroll
                        for (int r = j / BT; r < C / RB; ++r)
                            M::mma(av[j], of[r], M::row(pk_of[q] + 16 * j * LDP, LDP, r * RB));
                }
                if (dk && own_k) {
                    typename M::Frag qf[C / RB];
#pragma unroll
                    for (int r = 0; r < C / RB; ++r) qf[r] = M::template across<LDK>(lds.q, r * RB, 16 * wave);
#pragma unroll
                    for (int j = 0; j < TT; ++j)
#pragma unroll
                        for (int r = j / BT; r < C / RB; ++r)
                            M::mma(ak[j], qf[r], M::row(pv_of[q] + 16 * j * LDP, LDP, r * RB));
                }
                if constexpr (ALL)
                    if (dq) {
#pragma unroll
                        for (int j = 0; j < TT; ++j)
#pragma unroll
                            for (int r = 0; r <= j / BT; ++r)
                                M::mma(aq[j], kf[r], M::template across_place<LDP>(pv_of[q], r * RB, j));
                    }
            }
            if (gates_too && n > 1) S0.load_kept(kept + (ci - 1) * size, v, up32(p.K), up32(p.V));
            if (ALL && dq) store_rows<T, TT, VEC>(dq, (int64_t)p.H * p.K, 16 * wave + g4, p.K, left, aq);
            if (dv && own_v)
                store_rows<T, TT, VEC>(dv + row0 * p.V, (int64_t)p.H * p.V, 16 * wave + g4, p.V, left, av);
            if (dk && own_k)
                store_rows<T, TT, VEC>(dk + row0 * p.K, (int64_t)p.H * p.K, 16 * wave + g4, p.K, left, ak);
            S = U;
        } else {
            if (ALL && dq) {  // from the state before the chunk again
                State<T, VP / 16> G;
                G.load_transposed(kept + ci * size, v, up32(p.V), up32(p.K));
                walk_tokens<T, VP, LDK, false, true>(G, lds.o, lds.v, lds.k, gate, p.V, v, p.K, dq,
                                                     (int64_t)p.H * p.K, left);
            }
            // Token by token, all waves together: see walk_tokens.
            const int v = hidden(16 * wave + n16), g4 = hidden(4 * (lane >> 4));
            float *part = reinterpret_cast<float *>(lds.pk);  // [NW][KP]: dk's sums over a wave's columns
            static_assert(sizeof(lds.pk) >= sizeof(float) * NW * KP, "");
#pragma unroll 1
            for (int t = left - 1; t >= 0; --t) {
                const bool on = gate.seg[t] >= 0;
                const float f = gate.step[t];
                float o = 0.f;
                __syncthreads();  // the last token's sums are read
                if (on && own_v) {
                    const float x = Elem<T>::load(lds.o, t * LDV + v);
                    const float y = v < p.V ? Elem<T>::load(lds.v, t * LDV + v) : 0.f;
#pragma unroll
                    for (int m = 0; m < KT; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int k = Mat<T>::place(m, g4) + i;
                            if (k < p.K) {
                                S.t[m][i] += Elem<T>::load(lds.q, t * LDK + k) * x;
                                o += Elem<T>::load(lds.k, t * LDK + k) * S.t[m][i];
                            }
                            const float d = row16_sum(v < p.V ? S.t[m][i] * y : 0.f);
                            if (n16 == 0) part[wave * KP + k] = d;
                            if (k < p.K) S.t[m][i] = decayed(S.t[m][i], f);
                        }
                    o = groups_sum(o);
                }
                __syncthreads();
                const int64_t row = row0 + (int64_t)t * p.H;
                if (dv && own_v && lane < 16 && v < p.V) Elem<T>::store(dv, row * p.V + v, o);
                if (dk && (int)threadIdx.x < p.K) {
                    float d = 0.f;
                    if (on)
                        for (int w = 0; w < VP / 16; ++w) d += part[w * KP + threadIdx.x];
                    Elem<T>::store(dk, row * p.K + threadIdx.x, d);
                }
            }
            fine = S.finite();
            if (gates_too && n > 1) S0.load_kept(kept + (ci - 1) * size, v, up32(p.K), up32(p.V));
        }
        __syncthreads();  // the chunk's tiles are read
        if (++gi == L::GATES && n > 1) next_gates();
    }

    if (p.fin && own_v && at.seg == 0) S.store(p.fin + (int64_t)at.bh * p.K * p.V, v, p.K, p.V);
}

// Segments' additions -> start states, in place: state[s] = what the segments walked before s left.
// One thread an element; carry over the segments in the walk's order.  Bound by memory: 64 heads of 128 x 128
// and 8 segments 12 us (67 MB, 5.6 TB/s).
struct JoinArgs {
    float *state;        // [BH, segments, K V]
    const float *decay;  // their roots, [BH, segments]
    const float *first;  // start state of the walk, or null
    int64_t f_b, f_h, f_row, f_col;
    int64_t H, KV, V;
    int segments, rev;
};

__global__ void __launch_bounds__(kThreads) linear_join(JoinArgs p) {
    const unsigned blocks = (unsigned)((p.KV + kThreads - 1) / kThreads);
    const int64_t bh = blockIdx.x / blocks, i = (int64_t)(blockIdx.x % blocks) * kThreads + threadIdx.x;
    if (i >= p.KV) return;
    float *st = p.state + bh * p.segments * p.KV + i;
    const float *d = p.decay + bh * p.segments;
    float x = 0.f;
    if (p.first)
        x = p.first[bh / p.H * p.f_b + bh % p.H * p.f_h + i / p.V * p.f_row + i % p.V * p.f_col];
    // Eight segments' additions are read at a time: each store would hold back the next load.
    constexpr int N = 8;
    const int step = p.rev ? -1 : 1;
    int s = p.rev ? p.segments - 1 : 0;
    for (int n = p.segments; n > 0; n -= N, s += step * N) {
        float add[N], f[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = s + step * min(k, max(n - 2, 0));  // the last segment adds nothing that is needed
            add[k] = st[at * p.KV];
            f[k] = d[at];
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (k >= n) break;
            st[(s + step * k) * p.KV] = x;
            x = decayed(x, f[k]) + add[k];
        }
    }
}

// out[h] = sum over b, t of x[b, t, h]: one workgroup a head, a fixed order, in 64 bits, since a thread adds up to
// 2^16 values one after the other.  For 8 x 509 tokens the launch alone (3.9 us).
__global__ void __launch_bounds__(1024) linear_head_sum(const float *x, int64_t rows, int64_t H, float *out) {
    __shared__ double red[16];
    double s = 0.;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) s += x[r * H + blockIdx.x];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if (lane_id() == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = red[0];
        for (int i = 1; i < 16; ++i) t += red[i];
        out[blockIdx.x] = (float)t;
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
// rows at a time.  The state is read and written once; bound by that: 2048 states of 64 x 64 14.3 us (4.8
// TB/s), 8192 of 128 x 128 218 us (4.9 TB/s).
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
    const float g = ld4<float>(p.g, b, 0, h, 0);
    float a = g == INFINITY ? NAN : g < kCut ? 0.f : expf(0.5f * (g > 177.4f ? 177.4f : g));  // a root, as in the chunks
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
                x[i] = decayed(x[i], a) + kk * vv[i];
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
    bool prewalk;  // start states are walked to, instead of carried by a launch of their own
};

// Workgroups that fill the card: two a unit.  Forward and backward of 16 x 512 tokens, 8 heads of 64 / 4 x 8192
// tokens, 16 heads of 128 / 8 x 509 f32 tokens, 8 heads of 64: 68 / 1147 / 74 us; with 1024 68 / 1213 / 74, with
// 256 78 / 1093 / 84.
constexpr int64_t kWantGroups = 512;

int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

Plan plan(const gdn2_shape *s, int dtype) {
    Plan p;
    p.C = dtype == GDN2_BF16 ? Mat<bf16_t>::C : Mat<float>::C;
    p.chunks = (int)((s->time + p.C - 1) / p.C);
    p.BH = s->batch * s->heads;
    p.KV = s->keys * s->values;
    // Segments of at least two chunks (the last one of an odd number has one), as many as fill the card.  (Cut at 16
    // chunks, too, 32 x 2048 bf16 tokens, 16 heads of 64, take 206 us forward and 538 backward in place of 168 and
    // 502, 8 x 8192 tokens, 16 heads of 128, 523 and 1666 in place of 500 and 1626.)  With single chunks a prompt of
    // 3001 tokens, 8 heads of 64, takes 25.9 us in place of 23.6, more to join, but 700 tokens in both directions 45 in
    // place of 55; with three for two where their number is odd 25.6 and 70 (5000 forward 28.5 in place of 29.6).
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(kWantGroups / p.BH, (p.chunks + 1) / 2));
    p.seg_chunks = (int)((p.chunks + want - 1) / want);
    p.segments = (p.chunks + p.seg_chunks - 1) / p.seg_chunks;
    // Walked to where that costs at most a few chunks.  Both directions, 8 heads of 64, walked to and carried: 16 x 384
    // and 16 x 512 bf16 tokens (6 and 8 chunks) 60 and 77, 68 and 82 us; 8 x 250 f32 tokens (8 chunks) 48 and 58; 700
    // bf16 and 300 f32 tokens (11 and 10) 57 and 55, 51 and 50; 8 x 509 f32 tokens (16) 90 and 74.
    p.prewalk = p.chunks <= 8;
    return p;
}

struct Layout {
    size_t state, decay, kept, y, adj, dg, bytes;
};

// Widths for which the backward is one walk, from a state that the forward keeps before every chunk.  Up to 64
// such a state weighs half of what the chunk's four bf16 tensors do, which a dq walk of its own reads again:
// forward and backward of 16 x 512 tokens, 8 heads of 64, 68 us against 117, 8 x 509 f32 tokens 74 against 117.  At 128
// it weighs as much as they, and the walk's registers run out: it took 1.4 times as long as the two.
bool all_in_one(const gdn2_shape *s) { return s->keys <= 64 && s->values <= 64; }

// Checkpoint: the start states of the segments and their decays, and for a backward in one walk the states
// before every chunk and after the last.  A forward that no backward follows needs it only to carry states.
Layout checkpoint_layout(const Plan &p, const gdn2_shape *s, bool train) {
    Layout l{};
    l.decay = p.segments > 1 ? round16(4 * p.BH * p.segments * p.KV) : 0;
    l.kept = l.decay + round16(4 * p.BH * p.segments);
    l.bytes = l.kept;
    if (!train && (p.segments == 1 || p.prewalk)) l.bytes = 16;
    if (train && all_in_one(s)) l.bytes += 4 * p.BH * (p.chunks + 1) * kept_size((int)s->keys, (int)s->values);
    return l;
}

Layout workspace_layout(const Plan &p, const gdn2_shape *s) {
    Layout l{};
    size_t n = 0;
    const auto take = [&](int64_t floats) {
        const size_t at = n;
        n += round16(4 * floats);
        return at;
    };
    l.state = take(p.segments > 1 && !p.prewalk ? p.BH * p.segments * p.KV : 0);
    l.decay = take(p.BH * p.segments);
    const bool all = all_in_one(s);
    l.y = take(all ? 0 : p.BH * s->time);
    l.adj = take(all ? 0 : p.BH * p.chunks * kept_size((int)s->keys, (int)s->values));
    l.dg = take(p.BH * s->time);
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
    // A launch has below 2^32 threads: at most 512 for a chunk of 32 or 64 tokens.
    const int64_t lim = (int64_t)1 << 21;
    if (s->batch > lim || s->heads > lim || s->batch * s->heads > lim || s->time > 32 * lim ||
        (s->time + 31) / 32 > lim / (s->batch * s->heads))
        return fail(GDN2_ERR_SHAPE, "too many tokens: batch * heads * ceil(time / 32) must be at most 2^21");
    return GDN2_OK;
}

// Whether rows are read in 16-byte pieces: unit channel stride, aligned rows, whole pieces.
bool vec_rows(const gdn2_view *v, int64_t width) {
    const int64_t es = v->dtype == GDN2_BF16 ? 2 : 4;
    if (v->stride[3] != 1 || ((uintptr_t)v->data & 15) || width * es % 16) return false;
    for (int d = 0; d < 3; ++d)
        if (v->stride[d] * es % 16) return false;
    return v->stride[1] * es * 64 < ((int64_t)1 << 31);
}

// And results written so: null, or dense at a 16-byte address (rows of whole pieces then all are).
bool vec_out(const void *p) { return ((uintptr_t)p & 15) == 0; }

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

template <typename W>
W base_walk(const gdn2_shape *s, const Plan &p, const gdn2_view *g, const gdn2_view *valid,
               const gdn2_view *reset) {
    W w{};
    w.T = s->time;
    w.H = (int)s->heads;
    w.g = make_view(g);
    w.valid = make_view(valid);
    w.reset = make_view(reset);
    w.chunks = p.chunks;
    w.seg_chunks = p.seg_chunks;
    w.segments = p.segments;
    return w;
}

View transposed(const View &x) { return View{x.data, x.s0, x.s1, x.s3, x.s2}; }

void set_triple(Forward *w, const gdn2_view *a, const gdn2_view *b, const gdn2_view *c, int64_t ka, int64_t vc) {
    w->a = make_view(a), w->b = make_view(b), w->c = make_view(c);
    w->ka = (int)ka;
    w->vc = (int)vc;
}

template <typename T, int KP, int CP, bool REV, bool OUT, bool DOT>
void launch_walk(const Forward &w, bool vec, unsigned grid, hipStream_t st) {
    const dim3 block(4 * CP);
    if (vec) hipLaunchKernelGGL((linear_walk<T, KP, CP, true, REV, OUT, DOT>), dim3(grid), block, 0, st, w);
    else hipLaunchKernelGGL((linear_walk<T, KP, CP, false, REV, OUT, DOT>), dim3(grid), block, 0, st, w);
}

template <typename T, bool REV, bool OUT, bool DOT>
void size_walk(const Forward &w, bool vec, unsigned grid, hipStream_t st) {
    if constexpr (!DOT)  // with it, such widths are linear_back's
        if (w.ka <= 64 && w.vc <= 64) return launch_walk<T, 64, 64, REV, OUT, DOT>(w, vec, grid, st);
    if (w.ka <= 64) launch_walk<T, 64, 128, REV, OUT, DOT>(w, vec, grid, st);
    else if (w.vc <= 64) launch_walk<T, 128, 64, REV, OUT, DOT>(w, vec, grid, st);
    else launch_walk<T, 128, 128, REV, OUT, DOT>(w, vec, grid, st);
}

template <bool REV, bool OUT, bool DOT>
hipError_t run_walk(const Forward &w, const Plan &p, int dtype, bool vec, hipStream_t st) {
    const unsigned grid = (unsigned)(p.BH * (p.segments - (OUT ? 0 : 1)));
    if (dtype == GDN2_BF16) size_walk<bf16_t, REV, OUT, DOT>(w, vec, grid, st);
    else size_walk<float, REV, OUT, DOT>(w, vec, grid, st);
    return hipGetLastError();
}

template <typename T, int KP, int VP, int MODE>
void launch_back(const Back &w, bool vec, unsigned grid, hipStream_t st) {
    const dim3 block(4 * std::max(KP, VP));
    if (vec) hipLaunchKernelGGL((linear_back<T, KP, VP, true, MODE>), dim3(grid), block, 0, st, w);
    else hipLaunchKernelGGL((linear_back<T, KP, VP, false, MODE>), dim3(grid), block, 0, st, w);
}

template <typename T, int MODE>
void size_back(const Back &w, bool vec, unsigned grid, hipStream_t st) {
    if constexpr (MODE == 2) {
        launch_back<T, 64, 64, 2>(w, vec, grid, st);
    } else {
        if (w.K <= 64) launch_back<T, 64, 128, MODE>(w, vec, grid, st);
        else if (w.V <= 64) launch_back<T, 128, 64, MODE>(w, vec, grid, st);
        else launch_back<T, 128, 128, MODE>(w, vec, grid, st);
    }
}

template <int MODE>
hipError_t run_back(const Back &w, const Plan &p, int dtype, bool vec, hipStream_t st) {
    const unsigned grid = (unsigned)(p.BH * p.segments);
    if (dtype == GDN2_BF16) size_back<bf16_t, MODE>(w, vec, grid, st);
    else size_back<float, MODE>(w, vec, grid, st);
    return hipGetLastError();
}

// Start states of every segment of a walk over (b, c) into `state`, from `first`.
template <bool REV>
hipError_t run_carry(Forward w, const Plan &p, const gdn2_view *b, const gdn2_view *c, int64_t K, int64_t V,
                     const View &first, float *state, float *decay, int dtype, bool vec, hipStream_t st) {
    set_triple(&w, nullptr, b, c, K, V);
    w.seg_state = state;
    w.seg_decay = decay;
    hipError_t e = run_walk<REV, false, false>(w, p, dtype, vec, st);
    if (e != hipSuccess) return e;
    const JoinArgs j{state, decay, (const float *)first.data, first.s0, first.s1, first.s2, first.s3,
                     w.H, K * V, V, p.segments, REV};
    hipLaunchKernelGGL(linear_join, dim3((unsigned)((K * V + kThreads - 1) / kThreads * p.BH)),
                       dim3(kThreads), 0, st, j);
    return hipGetLastError();
}

// Rows and columns of a state view at strides that 32-bit offsets reach.
int check_state(const gdn2_view *v, const char *name) {
    GDN2_TRY(check_view(v, name, GDN2_F32, true));
    if (v->data && (v->stride[2] >= (1 << 22) || v->stride[3] >= (1 << 22)))
        return fail(GDN2_ERR_SHAPE, "%s: the key and value strides must be below 2^22", name);
    return GDN2_OK;
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

size_t gdn2_linear_checkpoint_bytes(const gdn2_shape *shape, int32_t dtype, int train) {
    if (check_linear(shape, dtype) != GDN2_OK) return 0;
    return checkpoint_layout(plan(shape, dtype), shape, train != 0).bytes;
}

int gdn2_linear_scan(const gdn2_shape *shape, const gdn2_view *q, const gdn2_view *k,
                     const gdn2_view *v, const gdn2_view *g, const gdn2_view *valid,
                     const gdn2_view *reset, const gdn2_view *initial, void *output,
                     float *final_state, int train, void *checkpoint, size_t checkpoint_bytes,
                     void *stream) {
    GDN2_TRY(check_inputs(shape, q, k, v, g, valid, reset));
    if (initial) GDN2_TRY(check_state(initial, "initial"));
    if (!output || !final_state)
        return fail(GDN2_ERR_ARGUMENT, "output and final_state must be non-null");
    const Plan p = plan(shape, q->dtype);
    const Layout l = checkpoint_layout(p, shape, train != 0);
    GDN2_TRY(check_buffer(checkpoint, checkpoint_bytes, l.bytes, "checkpoint"));
    if (initial && !initial->data) initial = nullptr;
    const int64_t K = shape->keys, V = shape->values;
    const bool vec = vec_rows(q, K) && vec_rows(k, K) && vec_rows(v, V) && vec_out(output);
    hipStream_t st = (hipStream_t)stream;
    Forward w = base_walk<Forward>(shape, p, g, valid, reset);
    const View first = make_view(initial);
    float *state = (float *)checkpoint, *decay = (float *)((char *)checkpoint + l.decay);
    if (p.segments > 1 && !p.prewalk) {
        const hipError_t e = run_carry<false>(w, p, k, v, K, V, first, state, decay, q->dtype, vec, st);
        if (e != hipSuccess) return launch_status(e, "gdn2_linear_scan");
        w.starts = state;
    }
    if (train && all_in_one(shape)) w.kept = (float *)((char *)checkpoint + l.kept);
    else if (train && p.segments > 1 && p.prewalk) w.starts_out = state;
    set_triple(&w, q, k, v, K, V);
    w.first = first;
    w.s_bh = p.segments * p.KV, w.s_row = (int)V, w.s_col = 1;
    w.fin = final_state;
    w.out = output;
    return launch_status(run_walk<false, true, false>(w, p, q->dtype, vec, st), "gdn2_linear_scan");
}

size_t gdn2_linear_workspace_bytes(const gdn2_shape *shape, int32_t dtype) {
    if (check_linear(shape, dtype) != GDN2_OK) return 0;
    return workspace_layout(plan(shape, dtype), shape).bytes;
}

int gdn2_linear_backward(const gdn2_shape *shape, const gdn2_view *q, const gdn2_view *k,
                         const gdn2_view *v, const gdn2_view *g, const gdn2_view *valid,
                         const gdn2_view *reset, const gdn2_view *initial, const void *checkpoint,
                         size_t checkpoint_bytes, const gdn2_view *d_output,
                         const float *d_final_state, void *dq, void *dk, void *dv, float *dg,
                         float *dg_heads, float *d_initial, void *workspace, size_t workspace_bytes,
                         void *stream) {
    GDN2_TRY(check_inputs(shape, q, k, v, g, valid, reset));
    if (initial) GDN2_TRY(check_state(initial, "initial"));
    GDN2_TRY(check_view(d_output, "d_output", q->dtype, false));
    const Plan p = plan(shape, q->dtype);
    const bool all = all_in_one(shape);
    const Layout lc = checkpoint_layout(p, shape, true), l = workspace_layout(p, shape);
    GDN2_TRY(check_buffer(checkpoint, checkpoint_bytes, lc.bytes, "checkpoint"));
    GDN2_TRY(check_buffer(workspace, workspace_bytes, l.bytes, "workspace"));
    if (initial && !initial->data) initial = nullptr;
    const int64_t K = shape->keys, V = shape->values;
    const int dtype = q->dtype;
    const bool gates = dg || dg_heads;
    const bool vec = vec_rows(q, K) && vec_rows(k, K) && vec_rows(v, V) && vec_rows(d_output, V) && vec_out(dq) &&
                     vec_out(dk) && vec_out(dv);
    hipStream_t st = (hipStream_t)stream;
    const Forward base = base_walk<Forward>(shape, p, g, valid, reset);
    const auto at = [&](size_t off) { return (float *)((char *)workspace + off); };
    const float *states = (const float *)checkpoint;  // [B H, segments, K, V]
    const View first = make_view(initial), d_final{d_final_state, shape->heads * p.KV, p.KV, V, 1};
    const bool many = p.segments > 1;
    hipError_t e = hipSuccess;
    if (dk || dv || gates || d_initial || (all && dq)) {
        Back w = base_walk<Back>(shape, p, g, valid, reset);
        if (many && !p.prewalk) {
            float *adj = at(l.state);
            e = run_carry<true>(base, p, q, d_output, K, V, d_final, adj, at(l.decay), dtype, vec, st);
            if (e != hipSuccess) return launch_status(e, "gdn2_linear_backward");
            w.starts = adj;
        }
        w.q = make_view(q), w.k = make_view(k), w.v = make_view(v), w.o = make_view(d_output);
        w.K = (int)K, w.V = (int)V;
        w.dk = dk, w.dv = dv;
        w.first = d_final;
        w.s_bh = p.segments * p.KV, w.s_row = (int)V, w.s_col = 1;
        w.fin = d_initial;
        if (all) {
            w.kept = (float *)((char *)const_cast<void *>(checkpoint) + lc.kept);
            w.dq = dq;
            w.dg = !gates ? nullptr : dg ? dg : at(l.dg);
            e = run_back<2>(w, p, dtype, vec, st);
        } else if (gates) {
            w.y = at(l.y), w.adj = at(l.adj);
            e = run_back<1>(w, p, dtype, vec, st);
        } else {
            e = run_back<0>(w, p, dtype, vec, st);
        }
        if (e != hipSuccess) return launch_status(e, "gdn2_linear_backward");
    }
    if (!all && (dq || gates)) {
        Forward w = base;
        set_triple(&w, d_output, v, k, V, K);  // the state transposed: rows V, columns K
        w.out = dq;
        w.first = transposed(first);
        w.starts = many ? states : nullptr, w.s_bh = p.segments * p.KV, w.s_row = 1, w.s_col = (int)V;
        if (gates) {
            w.d = make_view(q);
            w.y = at(l.y), w.adj = at(l.adj);
            w.dg = dg ? dg : at(l.dg);
            e = run_walk<false, true, true>(w, p, dtype, vec, st);
        } else {
            e = run_walk<false, true, false>(w, p, dtype, vec, st);
        }
        if (e != hipSuccess) return launch_status(e, "gdn2_linear_backward");
    }
    if (dg_heads)
        hipLaunchKernelGGL(linear_head_sum, dim3((unsigned)shape->heads), dim3(1024), 0, st,
                           dg ? dg : at(l.dg),
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
