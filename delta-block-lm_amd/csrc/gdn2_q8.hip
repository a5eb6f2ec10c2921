// SwiGLU that keeps its input in 8 bits for the backward pass, on gfx950.
//
//   forward   a = silu(gate) up;  h = [gate | up] is kept as 8-bit codes with one power of two for
//             each block of 32 columns of a half
//   backward  at the kept values, s = sigmoid(gate):  dgate = da up s (1 + gate (1 - s)),
//             dup = da gate s, and a = gate s up again, which the next weight's gradient reads
//
// A block's scale is 2^e with the smallest e for which its largest magnitude is at most 127 2^e, and a
// code is h 2^-e rounded to the nearest whole number, ties to even: both steps are exact in float32
// apart from that rounding, and a kept value is exact in bf16 (7 bits).  The error is at most 2^(e-1), or 2^e at
// the largest of all values, so below 1/127 of the block's largest magnitude.  Between the passes a token of width M holds
// 2.06 M bytes, where h and a in bf16 hold 6 M.
//
// Bound by memory: eight columns of both halves a thread, 16 bytes of bf16 at a time; the four threads
// of a block share its maximum by lane moves.  bf16, with every byte counted once: 8192 tokens of width 1408
// forward 19 us (4.9 TB/s), backward 20 us (5.9 TB/s); 32768 of 4096 180 us (6.0 TB/s) and 222 us (6.1 TB/s);
// of 1401, whose rows start off 16 bytes, 21 and 31 us.
#include <math.h>

#include "gdn2_common.h"
#include "gdn2_status.h"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 32;  // columns of one exponent
constexpr int kPiece = 8;   // columns of one thread
constexpr int kNan = 255;   // exponent of a block that held a value that is not finite

struct Q8Args {
    const void *h;      // [rows, 2 M] dense
    const void *da;     // [rows, M]
    void *a;            // [rows, M]
    void *dh;           // [rows, 2 M]
    int8_t *codes;      // [rows, 2 M]
    uint8_t *exps;      // [rows, 2 blocks]: e + 127
    uint32_t rows, M, blocks;
    int vec;
};

// 128 sigmoid(x), with v_exp_f32 and v_rcp_f32 (about 1 ulp each).  128 times, because v_rcp_f32 gives 0 for a
// result below the normal numbers, and x sigmoid(x) still is a normal number down to x = -91.8, where sigmoid(x) is
// 2^-132.5.
__device__ __forceinline__ float sigm128(float x) {
    return __builtin_amdgcn_rcpf(0.0078125f + __builtin_amdgcn_exp2f(fmaf(x, -1.4426950408889634f, -7.f)));
}
// The scale goes to the larger factor: a small x would lose bits to it.
__device__ __forceinline__ float silu(float x, float s128) {
    return x < -1.f ? (x * 0.0078125f) * s128 : x * (s128 * 0.0078125f);
}

// Columns [c, c + 8) of a row that starts at p, zero past M.
template <typename T>
__device__ __forceinline__ void load8(const T *p, uint32_t c, uint32_t M, int vec, float (&v)[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 2) {
            const uint4 q = *reinterpret_cast<const uint4 *>(p + c);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        } else {
            const float4 x = *reinterpret_cast<const float4 *>(p + c);
            const float4 y = *reinterpret_cast<const float4 *>(p + c + 4);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
        }
        return;
    }
    T e[8];
    if (c + 8 <= M) {  // a whole piece, wherever it lies
        __builtin_memcpy(e, p + c, sizeof e);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = c + i < M ? p[c + i] : T(0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Elem<T>::load(e, i);
}
template <typename T>
__device__ __forceinline__ void store8(T *p, uint32_t c, uint32_t M, int vec, const float (&v)[8]) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) Elem<T>::store(e, i, v[i]);
    if (vec) {
        __builtin_memcpy(__builtin_assume_aligned(p + c, 16), e, sizeof e);
        return;
    }
    if (c + 8 <= M) {
        __builtin_memcpy(p + c, e, sizeof e);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < M) p[c + i] = e[i];
}

// Exponent (biased) of the block whose four threads hold v.
__device__ __forceinline__ int block_exponent(const float (&v)[8]) {
    uint32_t m = 0;  // the largest magnitude's bits; NaN and infinity are the largest of all
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2));
    if (m >= 0x7F800000u) return kNan;
    // m = 1.f 2^x <= 127 2^e = 1.984375 2^(e + 6)
    const int x = (int)(m >> 23) - 127 - 6 + ((m & 0x7FFFFFu) > 0x7E0000u);
    return min(max(x, -126), 121) + 127;
}
__device__ __forceinline__ float power(int biased) { return __uint_as_float((uint32_t)biased << 23); }

__device__ __forceinline__ void put_codes(int8_t *p, uint32_t c, uint32_t M, int vec,
                                          const float (&v)[8], int ex) {
    // 2^-e = 2^(127 - biased); e <= 121, so it is a normal number.  There values above 127 2^121 take code 127
    // too: with e = 122 they would round to 2^128.
    const float s = ex == kNan ? 0.f : power(254 - ex);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int q = ex == kNan ? 0 : (int)fminf(fmaxf(rintf(v[i] * s), -127.f), 127.f);
        w[i / 4] |= (uint32_t)(q & 255) << (8 * (i % 4));
    }
    if (vec) {
        *reinterpret_cast<uint2 *>(p + c) = make_uint2(w[0], w[1]);
        return;
    }
    if (c + 8 <= M) {
        __builtin_memcpy(p + c, w, sizeof w);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < M) p[c + i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
}
__device__ __forceinline__ void get_values(const int8_t *p, uint32_t c, uint32_t M, int vec, int ex,
                                           float (&v)[8]) {
    const float s = ex == kNan ? __builtin_nanf("") : power(ex);
    if (vec || c + 8 <= M) {
        uint32_t w[2];
        if (vec) __builtin_memcpy(w, __builtin_assume_aligned(p + c, 8), sizeof w);
        else __builtin_memcpy(w, p + c, sizeof w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * s;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < M ? (float)p[c + i] * s : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) q8_forward_kernel(Q8Args p) {
    const uint32_t n = blockIdx.x * kThreads + threadIdx.x, per = p.blocks * (kBlock / kPiece);
    const uint32_t r = n / per, piece = n % per, c = piece * kPiece;
    // The threads of a block of columns leave together, so the lane moves see them all.
    if (r >= p.rows) return;
    const T *h = reinterpret_cast<const T *>(p.h) + (int64_t)r * 2 * p.M;
    float g[8], u[8];
    const bool in = c < p.M;
    const int vec = p.vec;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = u[i] = 0.f;
    if (in) {
        load8<T>(h, c, p.M, vec, g);
        load8<T>(h + p.M, c, p.M, vec, u);
    }
    const int eg = block_exponent(g), eu = block_exponent(u);
    if (!in) return;
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = silu(g[i], sigm128(g[i])) * u[i];
    store8<T>(reinterpret_cast<T *>(p.a) + (int64_t)r * p.M, c, p.M, vec, a);
    int8_t *q = p.codes + (int64_t)r * 2 * p.M;
    put_codes(q, c, p.M, vec, g, eg);
    put_codes(q + p.M, c, p.M, vec, u, eu);
    if (piece % (kBlock / kPiece) == 0) {
        uint8_t *e = p.exps + (int64_t)r * 2 * p.blocks + c / kBlock;
        e[0] = (uint8_t)eg;
        e[p.blocks] = (uint8_t)eu;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) q8_backward_kernel(Q8Args p) {
    const uint32_t n = blockIdx.x * kThreads + threadIdx.x, per = p.blocks * (kBlock / kPiece);
    const uint32_t r = n / per, c = n % per * kPiece;
    if (r >= p.rows || c >= p.M) return;
    const uint8_t *e = p.exps + (int64_t)r * 2 * p.blocks + c / kBlock;
    const int8_t *q = p.codes + (int64_t)r * 2 * p.M;
    float g[8], u[8], d[8], a[8];
    get_values(q, c, p.M, p.vec, e[0], g);
    get_values(q + p.M, c, p.M, p.vec, e[p.blocks], u);
    load8<T>(reinterpret_cast<const T *>(p.da) + (int64_t)r * p.M, c, p.M, p.vec, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s128 = sigm128(g[i]), x = silu(g[i], s128);
        a[i] = x * u[i];
        u[i] = d[i] * u[i] * (s128 * (0.0078125f * fmaf(g[i], fmaf(s128, -0.0078125f, 1.f), 1.f)));
        g[i] = d[i] * x;
    }
    T *dh = reinterpret_cast<T *>(p.dh) + (int64_t)r * 2 * p.M;
    store8<T>(dh, c, p.M, p.vec, u);
    store8<T>(dh + p.M, c, p.M, p.vec, g);
    if (p.a) store8<T>(reinterpret_cast<T *>(p.a) + (int64_t)r * p.M, c, p.M, p.vec, a);
}

int check_q8(int64_t rows, int64_t width, int32_t dtype) {
    if (rows < 0 || width < 1) return fail(GDN2_ERR_SHAPE, "rows must be >= 0 and width >= 1");
    if (dtype != GDN2_F32 && dtype != GDN2_BF16) return fail(GDN2_ERR_DTYPE, "dtype must be F32 or BF16");
    const int64_t lim = ((int64_t)1 << 32) - kThreads;  // threads of one launch
    if (rows > lim || width > ((int64_t)1 << 30) || (rows && (width + kBlock - 1) / kBlock * 4 > lim / rows))
        return fail(GDN2_ERR_SHAPE, "too many values: rows * width must stay below 2^35");
    return GDN2_OK;
}

bool aligned(const void *p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

Q8Args q8_args(int64_t rows, int64_t width) {
    Q8Args a{};
    a.rows = (uint32_t)rows, a.M = (uint32_t)width;
    a.blocks = (uint32_t)((width + kBlock - 1) / kBlock);
    return a;
}

unsigned q8_grid(const Q8Args &a) {
    return (unsigned)(((int64_t)a.rows * a.blocks * (kBlock / kPiece) + kThreads - 1) / kThreads);
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

int gdn2_swiglu_q8_forward(int64_t rows, int64_t width, int32_t dtype, const void *h, void *a,
                           int8_t *codes, uint8_t *exponents, void *stream) {
    GDN2_TRY(check_q8(rows, width, dtype));
    if (rows == 0) return ok();
    if (!h || !a || !codes || !exponents)
        return fail(GDN2_ERR_ARGUMENT, "h, a, codes and exponents must be non-null");
    Q8Args p = q8_args(rows, width);
    p.h = h, p.a = a, p.codes = codes, p.exps = exponents;
    p.vec = width % kPiece == 0 && aligned(h, 16) && aligned(a, 16) && aligned(codes, 8);
    const dim3 grid(q8_grid(p)), block(kThreads);
    if (dtype == GDN2_BF16) hipLaunchKernelGGL((q8_forward_kernel<bf16_t>), grid, block, 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((q8_forward_kernel<float>), grid, block, 0, (hipStream_t)stream, p);
    return launch_status(hipGetLastError(), "gdn2_swiglu_q8_forward");
}

int gdn2_swiglu_q8_backward(int64_t rows, int64_t width, int32_t dtype, const int8_t *codes,
                            const uint8_t *exponents, const void *da, void *dh, void *a,
                            void *stream) {
    GDN2_TRY(check_q8(rows, width, dtype));
    if (rows == 0) return ok();
    if (!codes || !exponents || !da || !dh)
        return fail(GDN2_ERR_ARGUMENT, "codes, exponents, da and dh must be non-null");
    Q8Args p = q8_args(rows, width);
    p.codes = const_cast<int8_t *>(codes), p.exps = const_cast<uint8_t *>(exponents);
    p.da = da, p.dh = dh, p.a = a;
    p.vec = width % kPiece == 0 && aligned(da, 16) && aligned(dh, 16) && aligned(a, 16) && aligned(codes, 8);
    const dim3 grid(q8_grid(p)), block(kThreads);
    if (dtype == GDN2_BF16) hipLaunchKernelGGL((q8_backward_kernel<bf16_t>), grid, block, 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((q8_backward_kernel<float>), grid, block, 0, (hipStream_t)stream, p);
    return launch_status(hipGetLastError(), "gdn2_swiglu_q8_backward");
}

}  // extern "C"
