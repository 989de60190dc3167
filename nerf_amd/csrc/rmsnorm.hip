// Root-mean-square norm of rows, with the residual's addition in front of it, and its backward pass.
//
//   s = round(x + residual)          (s = x where there is no residual)
//   r = 1 / sqrt(mean_k(s_k^2) + eps),   n = s * r,   y = round(n * w)
// The norm is of s AS STORED: the backward pass, which has only s, then differentiates exactly what the forward pass computed.
//   dn = dy * w,   ds = (dn - n * mean_k(dn_k * n_k)) * r + dsum,   dx = dresidual = round(ds),   dw = sum_rows dy * n
//
// Bound by HBM: 4 rows moved forward (2 without a residual), 4 (3) backward.  A row is read once and stays in registers between
// the sum and the scaling; r is recomputed backward from s, which has to be read anyway, rather than kept.
// dw: every workgroup walks a fixed set of rows and adds them up in registers (a thread owns the same columns of every row), then
// its row groups in pairs; one partial row per workgroup goes to the workspace, and a second launch adds those in a fixed order: no
// atomics, the same bits every time.
//
// Measured, with a residual: 786432 x 64 fp32 forward 135 us (6.0 TB/s, some of it from the last-level cache), backward 163 + 5 us
// (5.0 TB/s); 16384 x 4096 bf16 109 us (4.9 TB/s) and 127 + 5 us (4.2 TB/s).  One row of 2048: 2.8 us.  Rows that the backward pass reads
// twice, fp32 4096 x 8192: forward 112 us (4.8 TB/s), backward 207 us (2.6 TB/s).
#include <type_traits>

#include "layers_common.h"

namespace {

// Rows that a workgroup does in as many turns or fewer stay with one, which then needs no second launch for dw (fp32, one against
// several: 20 x 64 2.9 | 4.4 us, 64 x 64 4.1 | 4.4, 1000 x 4 4.0 | 4.5; one row a turn, 4 x 2048: 5.6 | 4.9, but a launch less).
constexpr int kOneGroup = 4;
constexpr int kBwdGroups = 1024;        // workgroups of the backward pass at most = rows of partial weight gradients

// Threads of a row: TPR.  A thread holds NV 16-byte pieces of it; piece j starts at column (j * TPR + t) * N.
template <int TPR> struct RowThreads {
    static constexpr int kBlock = TPR > 256 ? TPR : 256;
    static constexpr int kRows = kBlock / TPR;      // rows of a workgroup at a time
};

// N values of the weight, which may be fp32 beside rows of 16 bits
template <int N, class W> __device__ __forceinline__ void load_weight(const W* w, int64_t col, int64_t dim, float* out) {
    if (N == Vec16<W>::N) {
        load_cols(w, col, dim, out);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += Vec16<W>::N) load_cols(w, col + i, dim, out + i);
    }
}

// sum over the TPR threads of a row, given to all of them
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* lds) {
    if constexpr (TPR <= 64) return group_sum<TPR>(v);
    v = group_sum<64>(v);
    constexpr int kWaves = TPR / 64 > 0 ? TPR / 64 : 1;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
    const int w0 = (threadIdx.x / TPR) * kWaves;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += lds[w0 + i];
    __syncthreads();        // (the next sum reuses lds)
    return s;
}

// the largest magnitude of a row, given to all its threads (NaNs aside: the sums show them)
template <int TPR> __device__ __forceinline__ float row_max(float v, float* lds) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    if constexpr (TPR > 64) {
        constexpr int kWaves = TPR / 64;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        const int w0 = (threadIdx.x / TPR) * kWaves;
        for (int i = 0; i < kWaves; ++i) v = fmaxf(v, lds[w0 + i]);
        __syncthreads();
    }
    return v;
}
// Rows whose squares leave fp32's range -- a sum above 2^120, or below 2^-80 with no eps to speak of beside it -- are scaled by the
// power of two that takes the larger of their largest value and eps's root to [1/2, 1), and eps by its square: y is the same.
__device__ __forceinline__ bool out_of_range(float ss, float eps) { return !(ss <= 0x1p120f && (ss >= 0x1p-80f || eps >= 0x1p-100f)); }
__device__ __forceinline__ int row_exponent(float largest, float eps) {
    const float v = fmaxf(largest, sqrtf(eps));
    return v > 0.f && v < __builtin_inff() ? __builtin_amdgcn_frexp_expf(v) : 0;        // (0 / 0 and infinities stay what they are)
}

// two sums at once, one barrier: `lds` (32 floats) must not be the one of the call before (two in turn)
template <int TPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float* lds) {
    if constexpr (TPR <= 64) {
        a = group_sum<TPR>(a);
        b = group_sum<TPR>(b);
    } else {
        a = group_sum<64>(a);
        b = group_sum<64>(b);
        constexpr int kWaves = TPR / 64;
        if ((threadIdx.x & 63) == 0) {
            lds[threadIdx.x >> 6] = a;
            lds[16 + (threadIdx.x >> 6)] = b;
        }
        lds_barrier();
        a = b = 0.f;
        const int w0 = (threadIdx.x / TPR) * kWaves;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            a += lds[w0 + i];
            b += lds[16 + w0 + i];
        }
    }
}

// a 16-byte piece of a row as it lies in memory, zeros behind the row's end; WHOLE: there is no end within a thread's pieces
template <bool WHOLE, class T> __device__ __forceinline__ Vec16<T> piece(const T* row, int64_t col, int64_t dim) {
    if (WHOLE || col + Vec16<T>::N <= dim) return load16(row + col);
    Vec16<T> r;
#pragma unroll
    for (int i = 0; i < Vec16<T>::N; ++i) r.v[i] = col + i < dim ? row[col + i] : (T)0.f;
    return r;
}

template <class T, class W, int TPR, int NV, bool RES>
__global__ __launch_bounds__(RowThreads<TPR>::kBlock) void rmsnorm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                                              const W* __restrict__ w, int64_t rows, int64_t dim,
                                                                              float eps, T* __restrict__ sum, T* __restrict__ y) {
    constexpr int N = Vec16<T>::N;
    __shared__ float lds[16];
    const int t = threadIdx.x % TPR;
    for (int64_t r0 = (int64_t)blockIdx.x * RowThreads<TPR>::kRows; r0 < rows; r0 += (int64_t)gridDim.x * RowThreads<TPR>::kRows) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool live = row < rows;       // (idle threads of the last workgroup still take part in the sums)
    const int64_t at = (live ? row : 0) * dim;
    float s[NV][N];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t col = ((int64_t)j * TPR + t) * N;
        load_cols(x + at, col, live ? dim : 0, s[j]);
        if (RES) {
            float b[N];
            load_cols(res + at, col, live ? dim : 0, b);
#pragma unroll
            for (int i = 0; i < N; ++i) s[j][i] = (float)(T)(s[j][i] + b[i]);
            if (live) store_cols(sum + at, col, dim, s[j]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fmaf(s[j][i], s[j][i], ss);
    }
    ss = row_sum<TPR>(ss, lds);
    float scaled_eps = eps;
    if (out_of_range(ss, eps)) {        // (the same for all threads of the row)
        float largest = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) largest = fmaxf(largest, fabsf(s[j][i]));
        const int e = row_exponent(row_max<TPR>(largest, lds), eps);
        ss = 0.f;
        scaled_eps = ldexpf(eps, -2 * e);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s[j][i] = ldexpf(s[j][i], -e);
                ss = fmaf(s[j][i], s[j][i], ss);
            }
        ss = row_sum<TPR>(ss, lds);
    }
    const float r = 1.0f / sqrtf(ss / (float)dim + scaled_eps);
    if (!live) continue;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t col = ((int64_t)j * TPR + t) * N;
        if (col >= dim) break;
        float o[N], wv[N];
        load_weight<N>(w, col, dim, wv);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = s[j][i] * r * wv[i];
        store_cols(y + at, col, dim, o);
    }
    }
}

// rows wider than the registers of a workgroup hold: the row is read twice (the second time from the caches)
template <class T, class W, bool RES>
__global__ __launch_bounds__(1024) void rmsnorm_fwd_long_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                                const W* __restrict__ w, int64_t rows, int64_t dim, float eps,
                                                                T* __restrict__ sum, T* __restrict__ y) {
    __shared__ float lds[16];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t at = row * dim;
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < dim; c += 1024) {
        float v = (float)x[at + c];
        if (RES) {
            const T q = (T)(v + (float)res[at + c]);
            sum[at + c] = q;
            v = (float)q;
        }
        ss = fmaf(v, v, ss);
    }
    ss = row_sum<1024>(ss, lds);
    const T* s_ = RES ? sum : x;        // (a thread reads back only what it wrote itself)
    int e = 0;
    if (out_of_range(ss, eps)) {
        float largest = 0.f;
        for (int64_t c = threadIdx.x; c < dim; c += 1024) largest = fmaxf(largest, fabsf((float)s_[at + c]));
        e = row_exponent(row_max<1024>(largest, lds), eps);
        ss = 0.f;
        for (int64_t c = threadIdx.x; c < dim; c += 1024) {
            const float v = ldexpf((float)s_[at + c], -e);
            ss = fmaf(v, v, ss);
        }
        ss = row_sum<1024>(ss, lds);
    }
    const float r = 1.0f / sqrtf(ss / (float)dim + ldexpf(eps, -2 * e));
    for (int64_t c = threadIdx.x; c < dim; c += 1024) y[at + c] = (T)(ldexpf((float)s_[at + c], -e) * r * (float)w[c]);
    }
}

template <class T, class W, int TPR, int NV, bool WHOLE>
__global__ __launch_bounds__(RowThreads<TPR>::kBlock) void rmsnorm_bwd_kernel(const T* __restrict__ s_, const W* __restrict__ w,
                                                                              const T* __restrict__ dy, const T* __restrict__ dsum,
                                                                              int64_t rows, int64_t dim, float eps,
                                                                              T* __restrict__ dx, float* __restrict__ part,
                                                                              W* __restrict__ dweight) {
    constexpr int N = Vec16<T>::N, kRows = RowThreads<TPR>::kRows;
    __shared__ float lds[112];      // two sums in turn; those of a scaled row, and its largest value
    extern __shared__ float dwl[];      // [4][dim]: the waves' sums (kRows > 1 only)
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    float dw[NV][N], wv[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t col = ((int64_t)j * TPR + t) * N;
        load_weight<N>(w, col, dim, wv[j]);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[j][i] = 0.f;
    }
    // the next row's pieces travel, as they lie in memory, under this row's sums
    Vec16<T> sn[NV], dn[NV], en[NV];
    auto fetch = [&](int64_t row) {     // (behind the last row that one again: it adds nothing below)
        const int64_t at = (row < rows ? row : rows - 1) * dim;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t col = ((int64_t)j * TPR + t) * N;
            sn[j] = piece<WHOLE>(s_ + at, col, dim);
            dn[j] = piece<WHOLE>(dy + at, col, dim);
            if (dsum) en[j] = piece<WHOLE>(dsum + at, col, dim);
        }
    };
    int turn = 0;
    if (rows > 0) fetch((int64_t)blockIdx.x * kRows + g);
    for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += (int64_t)gridDim.x * kRows, turn ^= 1) {
        const int64_t row = r0 + g;
        const bool live = row < rows;
        const int64_t at = (live ? row : 0) * dim;
        float s[NV][N], d[NV][N];
        Vec16<T> e[NV];
        float ss = 0.f, sd = 0.f;       // sum s^2 and sum dn * s: both at once, mean(dn * n) = sd * r / dim
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            e[j] = en[j];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s[j][i] = (float)sn[j].v[i];
                d[j][i] = (float)dn[j].v[i];
                ss = fmaf(s[j][i], s[j][i], ss);
                sd = fmaf(d[j][i] * wv[j][i], s[j][i], sd);
            }
        }
        fetch(row + (int64_t)gridDim.x * kRows);
        row_sum2<TPR>(ss, sd, lds + 32 * turn);
        int p = 0;
        if (out_of_range(ss, eps)) {        // (the same for all threads of the row)
            float largest = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < N; ++i) largest = fmaxf(largest, fabsf(s[j][i]));
            p = row_exponent(row_max<TPR>(largest, lds + 96), eps);
            ss = sd = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    s[j][i] = ldexpf(s[j][i], -p);
                    ss = fmaf(s[j][i], s[j][i], ss);
                    sd = fmaf(d[j][i] * wv[j][i], s[j][i], sd);
                }
            row_sum2<TPR>(ss, sd, lds + 64);
        }
        const float r = 1.0f / sqrtf(ss / (float)dim + ldexpf(eps, -2 * p));        // (of the scaled row)
        const float c = sd * r / (float)dim, rx = ldexpf(r, -p);
        if (live) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t col = ((int64_t)j * TPR + t) * N;
                if (!WHOLE && col >= dim) break;
                float o[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float n = s[j][i] * r;
                    dw[j][i] = fmaf(d[j][i], n, dw[j][i]);
                    const float ds = (d[j][i] * wv[j][i] - n * c) * rx;
                    o[i] = dsum ? ds + (float)e[j].v[i] : ds;
                }
                if (dx) store_cols<WHOLE>(dx + at, col, dim, o);
            }
        }
    }
    if (!part && !dweight) return;
    // this workgroup's share of the weight's gradient, or all of it where it is the only one
    auto put = [&](int64_t c, float v) {
        if (dweight) dweight[c] = (W)v;
        else part[(int64_t)blockIdx.x * dim + c] = v;
    };
    if constexpr (kRows == 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t col = ((int64_t)j * TPR + t) * N;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col + i < dim) put(col + i, dw[j][i]);
        }
    } else {        // a wave's row groups in pairs, then the waves in order: always the same
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t col = ((int64_t)j * TPR + t) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float v = dw[j][i];
#pragma unroll
                for (int o = TPR; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
                if (lane < TPR && col + i < dim) dwl[wave * dim + col + i] = v;
            }
        }
        __syncthreads();
        for (int64_t c = threadIdx.x; c < dim; c += RowThreads<TPR>::kBlock)
            put(c, (dwl[c] + dwl[dim + c]) + (dwl[2 * dim + c] + dwl[3 * dim + c]));
    }
}

template <class T, class W>
__global__ __launch_bounds__(1024) void rmsnorm_bwd_long_kernel(const T* __restrict__ s_, const W* __restrict__ w,
                                                                const T* __restrict__ dy, const T* __restrict__ dsum, int64_t rows,
                                                                int64_t dim, float eps, T* __restrict__ dx,
                                                                float* __restrict__ part) {
    __shared__ float lds[16];
    float* mine = part + (int64_t)blockIdx.x * dim;
    for (int64_t c = threadIdx.x; c < dim; c += 1024) mine[c] = 0.f;       // (read back by the same thread only)
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t at = row * dim;
        float ss = 0.f, sd = 0.f;
        for (int64_t c = threadIdx.x; c < dim; c += 1024) {
            const float s = (float)s_[at + c];
            ss = fmaf(s, s, ss);
            sd = fmaf((float)dy[at + c] * (float)w[c], s, sd);
        }
        ss = row_sum<1024>(ss, lds);
        sd = row_sum<1024>(sd, lds);
        int p = 0;
        if (out_of_range(ss, eps)) {
            float largest = 0.f;
            for (int64_t c = threadIdx.x; c < dim; c += 1024) largest = fmaxf(largest, fabsf((float)s_[at + c]));
            p = row_exponent(row_max<1024>(largest, lds), eps);
            ss = sd = 0.f;
            for (int64_t c = threadIdx.x; c < dim; c += 1024) {
                const float s = ldexpf((float)s_[at + c], -p);
                ss = fmaf(s, s, ss);
                sd = fmaf((float)dy[at + c] * (float)w[c], s, sd);
            }
            ss = row_sum<1024>(ss, lds);
            sd = row_sum<1024>(sd, lds);
        }
        const float r = 1.0f / sqrtf(ss / (float)dim + ldexpf(eps, -2 * p));        // (of the scaled row)
        const float k = sd * r / (float)dim, rx = ldexpf(r, -p);
        for (int64_t c = threadIdx.x; c < dim; c += 1024) {
            const float n = ldexpf((float)s_[at + c], -p) * r, d = (float)dy[at + c];
            mine[c] = fmaf(d, n, mine[c]);
            const float ds = (d * (float)w[c] - n * k) * rx;
            if (dx) dx[at + c] = (T)(dsum ? ds + (float)dsum[at + c] : ds);
        }
    }
}

// dw[c] = sum over the workgroups' partial rows: 32 columns by 32 threads each, every thread a fixed stripe of the rows
template <class W>
__global__ __launch_bounds__(1024) void rmsnorm_dw_kernel(const float* __restrict__ part, int parts, int64_t dim, W* __restrict__ dw) {
    __shared__ float lds[32][33];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + cx;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < dim) {
        int p = ry;
        for (; p + 96 < parts; p += 128)        // (four rows on their way at a time)
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] += part[(int64_t)(p + 32 * i) * dim + c];
        for (int i = 0; p < parts; p += 32, ++i) a[i & 3] += part[(int64_t)p * dim + c];
    }
    lds[ry][cx] = (a[0] + a[1]) + (a[2] + a[3]);
    for (int o = 16; o > 0; o >>= 1) {
        __syncthreads();
        if (ry < o) lds[ry][cx] += lds[ry + o][cx];
    }
    if (ry == 0 && c < dim) dw[c] = (W)lds[0][cx];
}

// (threads of a row, pieces a thread) by the number of 16-byte pieces in a row: the smallest that holds it in registers
template <class F> int by_row_shape(int64_t pieces, F&& f) {
    if (pieces <= 1) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
    if (pieces <= 4) return f(std::integral_constant<int, 4>(), std::integral_constant<int, 1>());
    if (pieces <= 8) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    if (pieces <= 16) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    if (pieces <= 32) return f(std::integral_constant<int, 32>(), std::integral_constant<int, 1>());
    if (pieces <= 64) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    if (pieces <= 128) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    if (pieces <= 256) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
    if (pieces <= 512) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    if (pieces <= 1024) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
    if (pieces <= 4096) return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
    return -1;
}

unsigned grid_of(int64_t groups) { return (unsigned)(groups < (1 << 20) ? groups : (1 << 20)); }    // (a launch holds under 2^32 threads)
int64_t bwd_groups(int64_t rows) { return rows < kBwdGroups ? (rows > 0 ? rows : 1) : kBwdGroups; }

template <class T, class W>
int fwd_typed(const T* x, const T* res, const W* w, int64_t rows, int64_t dim, float eps, T* sum, T* y, hipStream_t st) {
    const int64_t pieces = ceil_div64(dim, Vec16<T>::N);
    const int rc = by_row_shape(pieces, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
        const unsigned grid = grid_of(ceil_div64(rows, RowThreads<TPR>::kRows));
        if (res)
            rmsnorm_fwd_kernel<T, W, TPR, NV, true><<<grid, RowThreads<TPR>::kBlock, 0, st>>>(x, res, w, rows, dim, eps, sum, y);
        else
            rmsnorm_fwd_kernel<T, W, TPR, NV, false><<<grid, RowThreads<TPR>::kBlock, 0, st>>>(x, res, w, rows, dim, eps, sum, y);
        return 0;
    });
    if (rc < 0) {
        if (res) rmsnorm_fwd_long_kernel<T, W, true><<<grid_of(rows), 1024, 0, st>>>(x, res, w, rows, dim, eps, sum, y);
        else rmsnorm_fwd_long_kernel<T, W, false><<<grid_of(rows), 1024, 0, st>>>(x, res, w, rows, dim, eps, sum, y);
    }
    return nerf_launch_status("nerf_rmsnorm_fwd");
}

template <class T, class W>
int bwd_typed(const T* s, const W* w, const T* dy, const T* dsum, int64_t rows, int64_t dim, float eps, T* dx, W* dw, float* part,
              hipStream_t st) {
    const int64_t pieces = ceil_div64(dim, Vec16<T>::N);
    int groups = 0;
    const int rc = by_row_shape(pieces, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
        if constexpr (TPR > 256) {
            return -1;      // (a row, its successor and the weight's gradient are more than a thread's registers)
        } else {
        const int64_t turns = ceil_div64(rows, RowThreads<TPR>::kRows);     // of a single workgroup
        groups = turns <= kOneGroup ? 1 : (int)bwd_groups(turns);
        const size_t lds = RowThreads<TPR>::kRows > 1 ? (size_t)dim * 16 : 0;       // (at most 1024 columns)
        W* whole = groups == 1 ? dw : nullptr;
        float* share = dw && !whole ? part : nullptr;
        if (dim == (int64_t)TPR * NV * Vec16<T>::N)
            rmsnorm_bwd_kernel<T, W, TPR, NV, true><<<groups, RowThreads<TPR>::kBlock, lds, st>>>(s, w, dy, dsum, rows, dim, eps, dx, share, whole);
        else
            rmsnorm_bwd_kernel<T, W, TPR, NV, false><<<groups, RowThreads<TPR>::kBlock, lds, st>>>(s, w, dy, dsum, rows, dim, eps, dx, share, whole);
        return 0;
        }
    });
    if (rc < 0) {
        groups = (int)bwd_groups(rows);
        rmsnorm_bwd_long_kernel<T, W><<<groups, 1024, 0, st>>>(s, w, dy, dsum, rows, dim, eps, dx, part);
    }
    if (dw && !(rc == 0 && groups == 1)) rmsnorm_dw_kernel<W><<<(unsigned)ceil_div64(dim, 32), 1024, 0, st>>>(part, groups, dim, dw);
    return nerf_launch_status("nerf_rmsnorm_bwd");
}

constexpr int64_t kMaxRows = 0x7fffffff, kMaxDim = 1 << 24;

}  // namespace

extern "C" int nerf_rmsnorm_fwd(const void* x, const void* residual, const void* weight, int dtype, int weight_dtype, int64_t n_rows,
                                int64_t dim, float eps, void* sum, void* y, void* stream) {
    NERF_REQUIRE(nerf_dtype_ok(dtype) && (weight_dtype == dtype || weight_dtype == NERF_F32),
                 "dtype must be NERF_F32, NERF_F16 or NERF_BF16 and the weight's the same or NERF_F32");
    NERF_REQUIRE(n_rows >= 0 && n_rows <= kMaxRows && dim >= 1 && dim <= kMaxDim, "n_rows must be in [0, 2^31), dim in [1, 2^24]");
    NERF_REQUIRE(eps >= 0.f, "eps must not be negative");
    if (n_rows == 0) return 0;
    NERF_REQUIRE(x && weight && y && (!residual || sum), "null pointer (a residual needs sum)");
    hipStream_t st = (hipStream_t)stream;
    int rc = 0;
    NERF_DISPATCH_DTYPE(dtype, {
        rc = weight_dtype == NERF_F32 ? fwd_typed<T, float>((const T*)x, (const T*)residual, (const float*)weight, n_rows, dim, eps, (T*)sum, (T*)y, st)
                                      : fwd_typed<T, T>((const T*)x, (const T*)residual, (const T*)weight, n_rows, dim, eps, (T*)sum, (T*)y, st);
    });
    return rc;
}

extern "C" int64_t nerf_rmsnorm_bwd_workspace_bytes(int64_t n_rows, int64_t dim) {
    if (n_rows < 0 || n_rows > kMaxRows || dim < 1 || dim > kMaxDim) return -1;
    return bwd_groups(n_rows) * dim * 4;
}

extern "C" int nerf_rmsnorm_bwd(const void* sum, const void* weight, const void* dy, const void* dsum, int dtype, int weight_dtype,
                                int64_t n_rows, int64_t dim, float eps, void* dx, void* dweight, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    NERF_REQUIRE(nerf_dtype_ok(dtype) && (weight_dtype == dtype || weight_dtype == NERF_F32),
                 "dtype must be NERF_F32, NERF_F16 or NERF_BF16 and the weight's the same or NERF_F32");
    NERF_REQUIRE(n_rows >= 0 && n_rows <= kMaxRows && dim >= 1 && dim <= kMaxDim, "n_rows must be in [0, 2^31), dim in [1, 2^24]");
    NERF_REQUIRE(eps >= 0.f, "eps must not be negative");
    NERF_REQUIRE(weight && workspace && (n_rows == 0 || (sum && dy)), "null pointer");
    NERF_REQUIRE(nerf_aligned(workspace, 4) && workspace_bytes >= nerf_rmsnorm_bwd_workspace_bytes(n_rows, dim), "workspace too small");
    hipStream_t st = (hipStream_t)stream;
    int rc = 0;
    NERF_DISPATCH_DTYPE(dtype, {
        rc = weight_dtype == NERF_F32
                 ? bwd_typed<T, float>((const T*)sum, (const float*)weight, (const T*)dy, (const T*)dsum, n_rows, dim, eps, (T*)dx, (float*)dweight, (float*)workspace, st)
                 : bwd_typed<T, T>((const T*)sum, (const T*)weight, (const T*)dy, (const T*)dsum, n_rows, dim, eps, (T*)dx, (T*)dweight, (float*)workspace, st);
    });
    return rc;
}
