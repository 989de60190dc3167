// The gated block for few rows (up to 64): bound by reading the weights once.  No tile of rows is worth staging, so the weights go
// from memory straight into the matrix cores' operand registers -- 16 weight rows by 32 k a fragment, 16 bytes a lane -- and the
// waves of a workgroup split k: every wave takes each NW-th run of 64 to 256 k (run_steps), so a workgroup reads whole stretches of its
// rows, and the waves' sums meet in LDS in wave order.  Two launches, h and y; y's tiles are too few for the chip where it is narrow:
// then several workgroups share a tile's k and a third launch adds their sums.
// Rows may start anywhere (16-byte loads at element alignment), so nothing is laid out first.  fp32 is cut into three bf16 parts on
// the way (gated_mlp.hip says why).
//
// Measured: 1 row, 2048 -> 8192 -> 2048 bf16: h 14.3 us (67 MB of weights at 4.7 TB/s), y 10.8 + 3.0 us (33 MB, h in two parts, with its join);
// 37 rows, 1536 -> 4000 -> 1536 fp16: 10.7 and 10.1 + 2.7 us (25 and 12 MB: by the latency of the few turns a wave has; with four row
// tiles in place of three 1.2 us more).  Rows and weights sent for together, all row tiles at a time: 27 us in place of 24 for the one
// row, for want of registers.
#include <type_traits>

#include "gated_common.h"

namespace {

using namespace gated;

// x [m][k] -> [m][ld], zeros in the columns [k, ld)
template <class T> __global__ __launch_bounds__(256) void few_lay_kernel(const T* __restrict__ x, int64_t k, int64_t ld, int64_t count, T* __restrict__ to) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) to[i] = i % ld < k ? x[i / ld * k + i % ld] : (T)0.f;
}

struct Few {
    int64_t k, ldx;         // width of x (and of the weights' rows); its pitch
    int64_t rows;           // weight rows: hidden values, or columns of y
    int64_t ldo;            // pitch of the output; kGate: zeros in the columns [rows, ldo)
    int64_t plane;          // elements from h's first plane to its second; 0: it has one
    int m, act;
};

// 32-k steps of a run -- what a wave has on its way at a time -- as the registers allow
__host__ __device__ constexpr int run_steps(int parts, bool gate, int row_tiles) { return parts == 3 ? (gate ? 2 : 4) : gate || row_tiles > 1 ? 4 : 8; }

// MT: 16-row tiles of x; NW: waves; kGate: both projections and h, or a plain product
// FINE: h in two planes of 16 bits (kGate: p.plane says so)
template <class T, int MT, int NW, bool kGate, bool FINE>
__global__ __launch_bounds__(NW * 64) void few_kernel(const T* __restrict__ w, const T* __restrict__ w2, const T* __restrict__ x, Few p,
                                                      T* __restrict__ out, float* __restrict__ saved, float* __restrict__ part) {
    constexpr int P = Piece<T>::P, G = kGate ? 2 : 1, PX = kGate ? P : hidden_parts<T, FINE>();
    constexpr int XP = PX == 2 ? 2 : 1;     // planes of x
    typedef typename Piece<T>::E E;
    constexpr int kRun = run_steps(P, kGate, MT);
    typedef typename Frag<E>::type frag;
    __shared__ f32x4 sums[NW][G][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int64_t r0 = (int64_t)blockIdx.x * 16, row = r0 + c < p.rows ? r0 + c : p.rows - 1;      // (rows behind the last: not stored)
    const T *wr = w + row * p.k, *wr2 = kGate ? w2 + row * p.k : wr;
    const T* xr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xr[t] = x + (int64_t)min(t * 16 + c, p.m - 1) * p.ldx;
    f32x4 acc[G][MT];
#pragma unroll
    for (int q = 0; q < G; ++q)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t runs = (p.k + 32 * kRun - 1) / (32 * kRun);
    Raw<T> wn[kRun][G];
    // (only the last run can reach behind the rows' end: the others' loads have no branches between them)
    auto whole = [&](int64_t run) { return (run + 1) * 32 * kRun <= p.k; };
    auto fetch = [&](int64_t run) {
        auto load = [&](auto all) {
#pragma unroll
            for (int s = 0; s < kRun; ++s) {
                const int64_t col = (run * kRun + s) * 32 + g * 8;
                wn[s][0] = raw8<decltype(all)::value>(wr, col, p.k);
                if (kGate) wn[s][G - 1] = raw8<decltype(all)::value>(wr2, col, p.k);
            }
        };
        if (whole(run)) load(std::true_type());
        else load(std::false_type());
    };
    // workgroups of one row tile, too, take turns at the runs
    const int64_t stride = (int64_t)NW * gridDim.y, start = (int64_t)blockIdx.y * NW + wave;
    if (start < runs) fetch(start);
    for (int64_t run = start; run < runs; run += stride) {
        Raw<T> wv[kRun][G];
#pragma unroll
        for (int s = 0; s < kRun; ++s)
#pragma unroll
            for (int q = 0; q < G; ++q) wv[s][q] = wn[s][q];
        if (run + stride < runs) fetch(run + stride);       // the next run's weights travel under this run's products
        frag a[kRun][G][P];
#pragma unroll
        for (int s = 0; s < kRun; ++s)
#pragma unroll
            for (int q = 0; q < G; ++q) frags(wv[s][q], a[s][q]);
        Raw<T> xn[kRun][XP];
        const bool all_of_it = whole(run);
        auto rows = [&](int t) {
            auto load = [&](auto all) {
#pragma unroll
                for (int s = 0; s < kRun; ++s)
#pragma unroll
                    for (int q = 0; q < XP; ++q) xn[s][q] = raw8<decltype(all)::value>(xr[t] + q * p.plane, (run * kRun + s) * 32 + g * 8, p.k);
            };
            if (all_of_it) load(std::true_type());
            else load(std::false_type());
        };
        rows(0);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            Raw<T> xv[kRun][XP];
#pragma unroll
            for (int s = 0; s < kRun; ++s)
#pragma unroll
                for (int q = 0; q < XP; ++q) xv[s][q] = xn[s][q];
            if (t + 1 < MT) rows(t + 1);
#pragma unroll
            for (int s = 0; s < kRun; ++s) {
                frag b[PX];
#pragma unroll
                for (int q = 0; q < XP; ++q) frags<T>(xv[s][q], b + q);
#pragma unroll
                for (int q = 0; q < G; ++q) acc[q][t] = product<P, PX>(a[s][q], b, acc[q][t]);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < G; ++q)
#pragma unroll
        for (int t = 0; t < MT; ++t) sums[wave][q][t][lane] = acc[q][t];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 64; i += NW * 64) {
        const int t = i >> 6, l = i & 63, m = t * 16 + (l & 15);
        const int64_t col = r0 + (l >> 4) * 4;
        f32x4 s[G];
#pragma unroll
        for (int q = 0; q < G; ++q) {
            s[q] = sums[0][q][t][l];
            for (int v = 1; v < NW; ++v) s[q] += sums[v][q][t][l];
        }
        if (m >= p.m) continue;
        if (!kGate && part) {       // several workgroups a row tile: [workgroup][row][column]
            float* to = part + ((int64_t)blockIdx.y * p.m + m) * p.ldo + col;
            for (int j = 0; j < 4 && col + j < p.ldo; ++j) to[j] = s[0][j];
            continue;
        }
        float a[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
        if (kGate) {
            const float b[4] = {a[0], a[1], a[2], a[3]};
            activate(b, p.act, a);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (col + j >= p.ldo) break;
            float v = s[0][j];
            if (kGate) {
                const bool in = col + j < p.rows;
                if (saved && in) {
                    saved[saved_at(m, col + j, p.m)] = v;
                    saved[saved_at(m, col + j, p.m) + kSavedCols] = s[G - 1][j];
                }
                v = in ? a[j] * s[G - 1][j] : 0.f;
            }
            T* to = out + m * p.ldo + col + j;
            if (kGate && p.plane) {
                T both[2];
                cut<T, 2>(v, both);
                to[0] = both[0];
                to[p.plane] = both[1];
            } else {
                to[0] = (T)v;
            }
        }
    }
}

template <class T> __global__ __launch_bounds__(256) void few_join_kernel(const float* __restrict__ part, int parts, int64_t count, T* __restrict__ y) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    float a = 0.f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) a += part[p * count + i];
    y[i] = (T)a;
}

int64_t few_ld(int64_t f) { return (f + 31) / 32 * 32; }
// Rows that do not start at multiples of 16 bytes take twice as long to read (48 rows of 831 to 5620: 43 us against 21).  The weights
// are read once either way; x is read by every workgroup, as many 16-row tiles as it has.
bool lays_x(int64_t m, int64_t k, int elem) { return m > 16 && k * elem % 16 != 0; }

// y has few 16-column tiles: as many workgroups each as give every CU two, and none that has no run (bf16, 1 row of 64 -> 2048 -> 512,
// eight runs for one workgroup's waves: 9.3 us, shared by two 11.1; 9 rows of 64 -> 4000 -> 200 fp32, by four 12.4, by three 16.9).
constexpr int kWaves = 8;
int parts_of(int64_t m, int64_t f, int64_t n, int elem) {
    const int64_t want = 2 * kNumCU / ((n + 15) / 16), run = 32 * run_steps(elem == 4 ? 3 : 1, false, m > 16 ? 2 : 1), runs = (f + run - 1) / run;
    const int64_t most = (runs + kWaves - 1) / kWaves;
    return (int)(want < 1 ? 1 : want < most ? want : most < 1 ? 1 : most);
}

template <class T, int MT> int launch(const T* params, const T* x, int64_t m, int64_t k, int64_t f, int64_t n, int act, T* y, float* saved,
                                      T* h, int64_t ldh, float* part, void* xl, hipStream_t st) {
    const int64_t plane = sizeof(T) == 2 && nerf_gated_fine(m, k, f, n) ? m * ldh : 0;
    Few up = {k, k, f, ldh, plane, (int)m, act};
    const Few down = {f, ldh, n, n, plane, (int)m, act};
    const int parts = parts_of(m, f, n, (int)sizeof(T));
    if (lays_x(m, k, (int)sizeof(T))) {
        up.ldx = few_ld(k);
        few_lay_kernel<T><<<(unsigned)ceil_div64(m * up.ldx, 256), 256, 0, st>>>(x, k, up.ldx, m * up.ldx, (T*)xl);
        x = (const T*)xl;
    }
    few_kernel<T, MT, kWaves, true, false><<<(unsigned)(ldh / 16), kWaves * 64, 0, st>>>(params, params + f * k, x, up, h, saved, nullptr);
    const dim3 grid((unsigned)ceil_div64(n, 16), (unsigned)parts);
    const T* wd = params + 2 * f * k;
    if constexpr (sizeof(T) == 2) {
        if (plane) few_kernel<T, MT, kWaves, false, true><<<grid, kWaves * 64, 0, st>>>(wd, wd, h, down, y, nullptr, parts > 1 ? part : nullptr);
        else few_kernel<T, MT, kWaves, false, false><<<grid, kWaves * 64, 0, st>>>(wd, wd, h, down, y, nullptr, parts > 1 ? part : nullptr);
    } else {
        few_kernel<T, MT, kWaves, false, false><<<grid, kWaves * 64, 0, st>>>(wd, wd, h, down, y, nullptr, parts > 1 ? part : nullptr);
    }
    if (parts > 1) few_join_kernel<T><<<(unsigned)ceil_div64(m * n, 256), 256, 0, st>>>(part, parts, m * n, y);
    return nerf_launch_status("nerf_gated_mlp_fwd");
}
template <class T> int by_rows(const T* params, const T* x, int64_t m, int64_t k, int64_t f, int64_t n, int act, T* y, float* saved, T* h,
                               int64_t ldh, float* part, void* xl, hipStream_t st) {
    if (m <= 16) return launch<T, 1>(params, x, m, k, f, n, act, y, saved, h, ldh, part, xl, st);
    if (m <= 32) return launch<T, 2>(params, x, m, k, f, n, act, y, saved, h, ldh, part, xl, st);
    if (m <= 48) return launch<T, 3>(params, x, m, k, f, n, act, y, saved, h, ldh, part, xl, st);
    return launch<T, 4>(params, x, m, k, f, n, act, y, saved, h, ldh, part, xl, st);
}

}  // namespace

bool nerf_gated_few_ok(int64_t m) { return m <= 64; }
static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

int64_t nerf_gated_few_bytes(int dtype, int64_t m, int64_t k, int64_t f, int64_t n) {
    const int parts = parts_of(m, f, n, nerf_dtype_bytes(dtype)), elem = nerf_dtype_bytes(dtype);
    return up256(m * few_ld(f) * 4) +       // (of 16 bits: twice)
           (parts > 1 ? up256(parts * m * n * 4) : 0) + (lays_x(m, k, elem) ? m * few_ld(k) * elem : 0);
}

int nerf_gated_few_fwd(const void* params, const void* x, int dtype, int64_t m, int64_t k, int64_t f, int64_t n, int act, void* y,
                       float* saved, void* ws, hipStream_t st) {
    const int64_t ldh = few_ld(f);
    const int parts = parts_of(m, f, n, nerf_dtype_bytes(dtype));
    char* part = (char*)ws + up256(m * ldh * 4);
    void* xl = part + (parts > 1 ? up256(parts * m * n * 4) : 0);
    int rc = 0;
    NERF_DISPATCH_DTYPE(dtype, rc = by_rows<T>((const T*)params, (const T*)x, m, k, f, n, act, (T*)y, saved, (T*)ws, ldh, (float*)part, xl, st));
    return rc;
}
