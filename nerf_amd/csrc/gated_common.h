// What the wide and the narrow kernels of the gated block share (gated_mlp.hip, gated_narrow.hip).
#pragma once
#include "layers_common.h"

namespace gated {

// v_mfma_f32_16x16x32: D[i][j] += sum_k A[i][k] B[k][j].  A lane gives A[l % 16][8 (l / 16) .. + 7] and B[8 (l / 16) .. + 7][l % 16],
// and holds D[4 (l / 16) .. + 3][l % 16].  (Any order of k does, as long as A and B agree on it.)
template <class E> struct Frag;
template <> struct Frag<__bf16> { typedef bf16x8 type; };
template <> struct Frag<_Float16> { typedef f16x8 type; };
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// v_mfma_f32_32x32x16: a lane gives A[l % 32][8 (l / 32) .. + 7], B likewise, and holds D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32].
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// 1 / (1 + e^-g) with the hardware's exponential and reciprocal (1 ulp each): a relative error near |g| * 2^-24, where the
// value itself falls off as e^-|g|; what it adds to act(g) stays below 2^-23 of |g|.  e^-g = inf gives 0, as it should.
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f)); }

// act(g) of N values; the branch is outside of the loop, so that each activation's code stands there once
template <int N> __device__ __forceinline__ void activate(const float (&g)[N], int act, float (&a)[N]) {
    if (act == NERF_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = g[i] > 0.f ? g[i] : (g[i] != g[i] ? g[i] : 0.f);
    } else if (act == NERF_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = g[i] * sigmoid(g[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = 0.5f * g[i] * (1.0f + erff(g[i] * 0.70710678118654752f));
    }
}
// act(g) and act'(g)
template <int N> __device__ __forceinline__ void activate2(const float (&g)[N], int act, float (&a)[N], float (&d)[N]) {
    if (act == NERF_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            a[i] = g[i] > 0.f ? g[i] : (g[i] != g[i] ? g[i] : 0.f);
            d[i] = g[i] > 0.f ? 1.f : 0.f;
        }
    } else if (act == NERF_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float s = sigmoid(g[i]);
            a[i] = g[i] * s;
            d[i] = fmaf(a[i], 1.0f - s, s);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float phi = 0.5f * (1.0f + erff(g[i] * 0.70710678118654752f));
            a[i] = g[i] * phi;
            d[i] = fmaf(g[i] * 0.39894228040143268f, expf(-0.5f * g[i] * g[i]), phi);
        }
    }
}

// a float as P values of E that add up to it: rounded (P = 1), to twice E's bits (P = 2), or as three bf16 (P = 3)
template <class E, int P> __device__ __forceinline__ void cut(float v, E* out) {
    if (P == 1) {
        out[0] = (E)v;
        return;
    }
    asm("" : "+v"(v));      // (one value, rounded once: a product that is converted in the instruction that makes it rounds otherwise)
    if (P == 2) {
        out[0] = (E)v;
        const float near = (float)out[0];
        out[1] = __builtin_fabsf(near) < __builtin_inff() ? (E)(v - near) : (E)0.f;
        return;
    }
    // (without branches: they would stand between the loads and the products of everything that is cut.  A finite value that would
    // round past the largest bf16 is cut off instead; an infinity leaves NaN in the later parts.)
    const float near = (float)(E)v;
    const float hi = __builtin_fabsf(near) < __builtin_inff() ? near : __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    const float r1 = v - hi;        // exact, as is the next difference: each part takes 8 of the bits that are left
    out[0] = (E)hi;
    out[1] = (E)r1;
    out[2] = (E)(r1 - (float)out[1]);
}

// Eight neighbouring elements of a row, as they lie there (Raw) and as what the matrix cores take: P fragments' lanes of E.
template <class T> struct Piece;
// Parts of a hidden value (h, dg, du) between two products.  fp32: as of any other value.  16 bits: rounded to them; its share of an
// output's error is then that of the output's own rounding, 1.4 times as much together, as long as there are enough of them for
// the mean to hold.  Where there are not (`FINE`, nerf_gated_fine), they are held in two parts: little is computed there.
template <class T, bool FINE> constexpr int hidden_parts() { return sizeof(T) == 4 ? 3 : FINE ? 2 : 1; }
template <> struct Piece<__bf16> { typedef __bf16 E; static constexpr int P = 1; };
template <> struct Piece<_Float16> { typedef _Float16 E; static constexpr int P = 1; };
template <> struct Piece<float> { typedef __bf16 E; static constexpr int P = 3; };

template <class T> struct Raw { T v[8]; };
// (zeros behind the row's end; WHOLE: the caller knows that they are in front of it)
template <bool WHOLE, class T> __device__ __forceinline__ Raw<T> raw8(const T* row, int64_t col, int64_t width) {
    Raw<T> r;
    if (WHOLE || col + 8 <= width) {
        __builtin_memcpy(&r, row + col, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = col + i < width ? row[col + i] : (T)0.f;
    }
    return r;
}
template <class E, int P, class T> __device__ __forceinline__ void frags(const Raw<T>& r, typename Frag<E>::type* out) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        E q[P];
        cut<E, P>((float)r.v[i], q);
#pragma unroll
        for (int p = 0; p < P; ++p) out[p][i] = q[p];
    }
}
template <class T> __device__ __forceinline__ void frags(const Raw<T>& r, typename Frag<typename Piece<T>::E>::type* out) {
    frags<typename Piece<T>::E, Piece<T>::P>(r, out);
}
// the product of PA parts by PB: those of the largest orders, small ones first
template <int PA, int PB, class frag> __device__ __forceinline__ f32x4 product(const frag* a, const frag* b, f32x4 c) {
    static_assert(PA == PB ? PA != 2 : PA + PB == 3, "one or three parts each, or one by two");
    if constexpr (PA == 3) {
        c = mfma(a[1], b[1], c);
        c = mfma(a[0], b[2], c);
        c = mfma(a[2], b[0], c);
    }
    if constexpr (PB > 1) c = mfma(a[0], b[1], c);
    if constexpr (PA > 1) c = mfma(a[1], b[0], c);
    return mfma(a[0], b[0], c);
}

// g and u kept for the backward pass: [neurons / 128][rows][2][128], so that what a workgroup keeps (128 hidden values of its rows)
// is one stretch of memory: rows 64 KiB apart, as [rows][2 neurons] would have them, all fall on a few memory channels.
constexpr int kSavedCols = 128;
__host__ __device__ __forceinline__ int64_t saved_at(int64_t r, int64_t c, int64_t rows) {
    return ((c / kSavedCols * rows + r) * 2) * kSavedCols + c % kSavedCols;
}
static inline int64_t saved_floats(int64_t rows, int64_t neurons) { return (neurons + kSavedCols - 1) / kSavedCols * kSavedCols * 2 * rows; }

}  // namespace gated

// Few values in y or x, or few weights: an output's error is the mean over few roundings of hidden values and may stray far from the 1.4
// times of many.  Emulated in 64 bits with hidden values of normal inputs, 150 blocks each, by the smallest of y, h and dx: of 300 values
// (or 200 weights) one block in 5 had an output 1.5 times as far off as one whose hidden values are not rounded, of 1024 one in
// 15 to 25, of 2048 one in 20 to 75, of 4096 (or 3000 weights) at most one in 100.  What two parts cost, for calls of
// 2048 to 4095 values: bf16 1 row of 2048 -> 8192 -> 2048 24.8 us, in one part 22.6; 3 of 1365 -> 4000 -> 1365 20.9 | 19.6; 90 of 40 -> 2000 -> 40 21.1 | 20.8;
// 37 of 64 -> 3000 -> 1536, where every row tile reads both parts of h, 25.4 | 18.2.
static inline bool nerf_gated_fine(int64_t m, int64_t k, int64_t f, int64_t n) {
    const int64_t least = k < f ? (k < n ? k : n) : (f < n ? f : n);
    return m * least < 4096 || (2 * k + n) * f <= 4096;
}

// gated_few.hip: few rows; ws: nerf_gated_few_bytes of workspace.
bool nerf_gated_few_ok(int64_t m);
int64_t nerf_gated_few_bytes(int dtype, int64_t m, int64_t k, int64_t f, int64_t n);
int nerf_gated_few_fwd(const void* params, const void* x, int dtype, int64_t m, int64_t k, int64_t f, int64_t n, int act, void* y,
                       float* saved, void* ws, hipStream_t st);

// gated_narrow.hip: whole blocks of narrow widths in one kernel each way.
bool nerf_gated_narrow_fwd_ok(int dtype, int64_t m, int64_t k, int64_t f, int64_t n);
bool nerf_gated_narrow_bwd_ok(int dtype, int64_t k, int64_t f, int64_t n);
int64_t nerf_gated_narrow_bwd_bytes(int dtype, int64_t m, int64_t k, int64_t f, int64_t n);
int nerf_gated_narrow_fwd(const void* params, const void* x, int dtype, int64_t m, int64_t k, int64_t f, int64_t n, int act, void* y,
                          hipStream_t st);
int nerf_gated_narrow_bwd(const void* params, const void* x, const void* dy, int dtype, int64_t m, int64_t k, int64_t f, int64_t n,
                          int act, void* dx, void* dparams, int dparams_f32, void* ws, hipStream_t st);
