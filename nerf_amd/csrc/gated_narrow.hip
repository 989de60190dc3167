// The gated block at field sizes (widths up to 128, few hundred hidden values): one kernel each way, the hidden values never leave the
// registers.  With millions of rows of a hundred bytes the block is bound by reading x and writing y; a hidden value written
// out and read back would be several times that.
//
// Forward: a wave takes 32 rows at a time against all weights, which lie in LDS in the order in which fragments are read
// (1 KiB per 16 x 32 fragment, lane after lane: no bank conflicts).  The rows of a pair of 16-row weight tiles are dealt out
// so that a lane ends up with 8 neighbouring hidden values of its row -- exactly the B fragment of the next product.
//
// Backward: g and u are computed again (cheaper than reading them back).  The waves of a workgroup share 32 rows at a time and
// split the hidden values, 32 each: a wave keeps its five sets of weight fragments and the gradients of its weights in
// registers for the whole launch.  dx is a sum over all hidden values: the waves' partial sums meet in LDS; where a workgroup's
// waves do not cover the hidden values, further launches add their share to the sum so far (fp32).  The weights' gradients need
// the rows along k: dg, du, h (per wave) and x, dy (shared) lie in LDS row by row and are read transposed.  A workgroup
// leaves one partial gradient in the workspace; a last launch adds those in a fixed order.
//
// fp32 is cut into three bf16 parts wherever a product takes it (gated_mlp.hip says why): three fragments in place of one, six
// products.
//
// Measured, 786432 rows, 64 -> 128 -> 64 bf16: forward 60 us (0.64 PFLOP/s, 3.3 TB/s; the matrix cores share their issue slots with the
// activations), backward 182 to 205 + 9 us by card (0.5 PFLOP/s with what it computes again; a tile's products, transposed reads and
// activations follow one another in the one or two waves of a SIMD).  fp32, 65799 rows of the same: 37 and 104 + 6 us.
#include <type_traits>

#include "gated_common.h"

namespace {

using namespace gated;

constexpr int kLdsLimit = 160 * 1024;

__device__ __forceinline__ int pair_row(int tile, int i) { return (tile >> 1) * 32 + 8 * (i >> 2) + 4 * (tile & 1) + (i & 3); }

template <bool WHOLE, class T> __device__ __forceinline__ void put8(T* row, int col, int width, const float* v) {
    if (WHOLE || col + 8 <= width) {
        T r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = (T)v[i];
        __builtin_memcpy(row + col, r, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < width) row[col + i] = (T)v[i];
    }
}
// eight values as fragments' lanes
template <class E, int P> __device__ __forceinline__ void cut8(const float (&v)[8], typename Frag<E>::type* out) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        E q[P];
        cut<E, P>(v[i], q);
#pragma unroll
        for (int p = 0; p < P; ++p) out[p][i] = q[p];
    }
}
template <class T> Raw<T> __device__ __forceinline__ none8() {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = (T)0.f;
    return r;
}

// Widths of rows, for a kernel's loads of eight columns each: kFull: they are multiples of 32; kEight: eight columns or more, so that what
// reaches behind a row's end can be read as the row's last eight and moved into place afterwards, without branches around the loads
// (700000 rows of bf16 48 -> 128 -> 48, with branches | without: forward 61 | 56 us, backward 212 | 184); kAny: the rest.
enum Widths { kAny, kEight, kFull };
template <int W, class T> __device__ __forceinline__ Raw<T> row8(const T* row, int col, int width) {
    return W == kEight ? raw8<true>(row, min(col, width - 8), width) : raw8<W == kFull>(row, col, width);
}
// ... by how many columns it reached behind the end (up to 0: not at all; 8 or more: all of them are zeros)
template <class T> __device__ __forceinline__ void into_place(Raw<T>& v, int behind) {
    if (behind <= 0) return;
#pragma unroll
    for (int by = 4; by > 0; by >>= 1)
        if (behind & by) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = e + by < 8 ? v.v[(e + by) & 7] : (T)0.f;
        }
    if (behind >= 8) v = none8<T>();
}

struct Narrow {
    int64_t m;
    int k, f, n, act;
    // forward: the hidden values [first, first + some 32s) of this launch; `more`: y holds the sum over those before (fp32)
    int first, pairs, more;
};

// KS: 32-column steps of x; NP: pairs of 16-column tiles of y; WIDTHS: of x (kFull: of y, too)
template <class T, int KS, int NP, int WIDTHS, bool FINE>
__global__ __launch_bounds__(512, Piece<T>::P == 1 && KS <= 2 && NP <= 2 && !FINE ? 4 : 2) void narrow_fwd_kernel(
    const T* __restrict__ params, const T* __restrict__ x, Narrow p, T* __restrict__ y) {
    constexpr int P = Piece<T>::P, H = hidden_parts<T, FINE>();
    constexpr bool WHOLE = WIDTHS == kFull;
    typedef typename Piece<T>::E E;
    typedef typename Frag<E>::type frag;
    extern __shared__ __align__(16) char lds_raw[];
    frag* lds = (frag*)lds_raw;
    const int pairs = p.pairs, n_gate = pairs * 2 * KS;     // fragments of the gate (and of the up) weights
    const int n_all = 2 * n_gate + NP * 2 * pairs;
    const T *gate = params, *up = params + (int64_t)p.f * p.k, *down = up + (int64_t)p.f * p.k;
    for (int i = threadIdx.x; i < n_all * 64; i += 512) {
        const int lane = i & 63, which = i >> 6;
        Raw<T> r = none8<T>();
        if (which >= 2 * n_gate) {      // down: [column tile][pair of hidden tiles]
            const int at = which - 2 * n_gate, row = pair_row(at / pairs, lane & 15);
            if (row < p.n) r = raw8<false>(down + (int64_t)row * p.f, p.first + (at % pairs) * 32 + (lane >> 4) * 8, p.f);
        } else {                        // gate, up: [hidden tile][step of k]
            const int at = which < n_gate ? which : which - n_gate, row = p.first + pair_row(at / KS, lane & 15);
            if (row < p.f) r = raw8<false>((which < n_gate ? gate : up) + (int64_t)row * p.k, (at % KS) * 32 + (lane >> 4) * 8, p.k);
        }
        frag q[P];
        frags(r, q);
#pragma unroll
        for (int s = 0; s < P; ++s) lds[(which * P + s) * 64 + lane] = q[s];
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const frag *wg = lds + lane, *wu = lds + n_gate * P * 64 + lane, *wd = lds + 2 * n_gate * P * 64 + lane;
    auto weights = [&](const frag* from, int which, frag (&to)[P]) {
#pragma unroll
        for (int s = 0; s < P; ++s) to[s] = from[(which * P + s) * 64];
    };
    const int64_t tiles = (p.m + 31) / 32, step = (int64_t)gridDim.x * 8;
    int64_t tile = (int64_t)(threadIdx.x >> 6) * gridDim.x + blockIdx.x;     // (few tiles: a CU each)
    Raw<T> xn[2][KS];
    auto fetch = [&](int64_t t) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t r = t * 32 + b * 16 + c;
            const T* row = x + (r < p.m ? r : p.m - 1) * p.k;       // (rows behind the last are computed from it and not stored)
#pragma unroll
            for (int s = 0; s < KS; ++s) xn[b][s] = row8<WIDTHS>(row, s * 32 + g * 8, p.k);
        }
    };
    if (tile < tiles) fetch(tile);
    for (; tile < tiles; tile += step) {
        frag xb[2][KS][P];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (WIDTHS == kEight) into_place(xn[b][s], s * 32 + g * 8 + 8 - p.k);
                frags(xn[b][s], xb[b][s]);
            }
        if (tile + step < tiles) fetch(tile + step);        // the next rows travel under this tile's products
        f32x4 acc[NP][2][2];        // [pair][tile of the pair][row tile]
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int b = 0; b < 2; ++b) acc[i][j][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int h = 0; h < pairs; ++h) {
            f32x4 gv[2][2], uv[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int b = 0; b < 2; ++b) gv[j][b] = uv[j][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    frag a[P];
                    weights(wg, (h * 2 + j) * KS + s, a);
#pragma unroll
                    for (int b = 0; b < 2; ++b) gv[j][b] = product<P, P>(a, xb[b][s], gv[j][b]);
                    weights(wu, (h * 2 + j) * KS + s, a);
#pragma unroll
                    for (int b = 0; b < 2; ++b) uv[j][b] = product<P, P>(a, xb[b][s], uv[j][b]);
                }
            }
            frag hv[2][H];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float ga[8], aa[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) ga[i] = gv[i >> 2][b][i & 3];
                activate(ga, p.act, aa);
#pragma unroll
                for (int i = 0; i < 8; ++i) aa[i] *= uv[i >> 2][b][i & 3];
                cut8<E, H>(aa, hv[b]);
            }
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    frag a[P];
                    weights(wd, (i * 2 + j) * pairs + h, a);
#pragma unroll
                    for (int b = 0; b < 2; ++b) acc[i][j][b] = product<P, H>(a, hv[b], acc[i][j][b]);
                }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t r = tile * 32 + b * 16 + c;
            if (r >= p.m) continue;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                float v[8] = {acc[i][0][b][0], acc[i][0][b][1], acc[i][0][b][2], acc[i][0][b][3],
                              acc[i][1][b][0], acc[i][1][b][1], acc[i][1][b][2], acc[i][1][b][3]};
                if constexpr (P == 3) {
                    if (p.more) {
                        const Raw<T> q = raw8<WHOLE>(y + r * p.n, i * 32 + g * 8, p.n);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] += q.v[e];
                    }
                }
                put8<WHOLE>(y + r * p.n, i * 32 + g * 8, p.n, v);
            }
        }
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------------

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v LdsShort4;

// Eight rows of an LDS tile along k for one column a lane: a fragment with k = rows 8 (l / 16) .. + 7, column l % 16.  The
// transposing read hands every lane of a group of 16 one of 16 columns of 4 rows, to which the group's lanes point in order.
template <class E> __device__ __forceinline__ typename Frag<E>::type turned(const E* tile, int ld, int col, int lane) {
    const int row = 8 * (lane >> 4) + ((lane & 15) >> 2);
    const E* at = tile + row * ld + col + (lane & 3) * 4;
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4*)at);
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4*)(at + 4 * ld));
    const short8v both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Frag<E>::type, both);
}

constexpr int kHidLd = 40;      // elements from row to row of a wave's dg, du and h tiles (32 columns): 80 bytes

// KS, NS: 32-column steps of x and of y; P parts
template <int KS, int NS, int P> struct BwdLds {
    static constexpr int kXLd = KS * 32 + 8, kYLd = NS * 32 + 8, kPartLd = KS * 32 + 4;
    static constexpr int kX = 0, kY = kX + P * 32 * kXLd * 2, kHid = kY + P * 32 * kYLd * 2;
    static constexpr int hid(int waves) { return kHid + waves * 3 * P * 32 * kHidLd * 2; }
    static constexpr int bytes(int waves) { return hid(waves) + waves * 32 * kPartLd * 4; }
};

// What a launch does of the sum over hidden values: values [first, first + 32 a wave), dx = `so_far` + their share, stored rounded in
// dx or in fp32 in `partial` for the next launch.
struct Share {
    int first;
    const float* so_far;
    float* partial;
};

// A wave's registers: 5 sets of weight fragments, 3 of gradients.  Two waves a SIMD where x and y have up to 64 columns of 16 bits,
// one otherwise (`SOLO`).  AHEAD: 8-element chunks of the next rows that a thread holds.  WIDTHS: of x and y.
template <class T, int KS, int NS, int WIDTHS, int AHEAD, bool SOLO, bool FINE>
__global__ __launch_bounds__(SOLO ? 256 : 512) void narrow_bwd_kernel(const T* __restrict__ params, const T* __restrict__ x,
                                                                      const T* __restrict__ dy, Narrow p, Share sh, T* __restrict__ dx,
                                                                      float* __restrict__ part) {
    constexpr int P = Piece<T>::P, H = hidden_parts<T, FINE>(), KT = KS * 2, NT = NS * 2;
    constexpr bool WHOLE = WIDTHS == kFull;
    typedef typename Piece<T>::E E;
    typedef typename Frag<E>::type frag;
    typedef BwdLds<KS, NS, P> L;
    extern __shared__ __align__(16) char lds_raw[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, g = lane >> 4, c = lane & 15;
    E* lx = (E*)(lds_raw + L::kX);
    E* ly = (E*)(lds_raw + L::kY);
    E* hid = (E*)(lds_raw + L::kHid) + wave * 3 * P * 32 * kHidLd;      // [dg, du, h][part][32 rows][kHidLd]
    float* sums = (float*)(lds_raw + L::hid(waves));
    float* mine = sums + wave * 32 * L::kPartLd;
    const T *gate = params, *up = params + (int64_t)p.f * p.k, *down = up + (int64_t)p.f * p.k;
    const int h0 = sh.first + wave * 32;        // this wave's hidden values
    const bool grads = part != nullptr, inputs = dx || sh.partial;

    // weights of this wave: rows of gate / up by steps of k; rows of down^T by steps of n; gate^T, up^T by the hidden values
    frag wg[2][KS][P], wu[2][KS][P], wdt[2][NS][P], wgt[KT][P], wut[KT][P];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = h0 + pair_row(j, c);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            frags(row < p.f ? raw8<false>(gate + (int64_t)row * p.k, s * 32 + g * 8, p.k) : none8<T>(), wg[j][s]);
            frags(row < p.f ? raw8<false>(up + (int64_t)row * p.k, s * 32 + g * 8, p.k) : none8<T>(), wu[j][s]);
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            Raw<T> r;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int col = s * 32 + g * 8 + i;
                r.v[i] = row < p.f && col < p.n ? down[(int64_t)col * p.f + row] : (T)0.f;
            }
            frags(r, wdt[j][s]);
        }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        Raw<T> a, b;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = h0 + g * 8 + i, col = t * 16 + c;
            const bool in = row < p.f && col < p.k;
            a.v[i] = in ? gate[(int64_t)row * p.k + col] : (T)0.f;
            b.v[i] = in ? up[(int64_t)row * p.k + col] : (T)0.f;
        }
        frags(a, wgt[t]);
        frags(b, wut[t]);
    }

    f32x4 dwg[2][KT], dwu[2][KT], dwd[2][NT];       // d(gate), d(up) [hidden tile][k tile]; d(down)^T [hidden tile][n tile]
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int t = 0; t < KT; ++t) dwg[j][t] = dwu[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; ++t) dwd[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const int64_t tiles = (p.m + 31) / 32;
    constexpr int kChunksX = 32 * KS * 4, kChunksY = 32 * NS * 4;       // 8-element chunks of the two row tiles
    // rows behind the last are zeros: they add nothing to the weights' gradients
    auto chunk = [&](int64_t tile, int i) -> Raw<T> {
        const bool of_x = i < kChunksX;
        const int at = of_x ? i : i - kChunksX, per = of_x ? KS * 4 : NS * 4, width = of_x ? p.k : p.n, col = (at % per) * 8;
        const int64_t r = tile * 32 + at / per;
        if constexpr (WIDTHS == kEight) return row8<WIDTHS>((of_x ? x : dy) + (r < p.m ? r : p.m - 1) * width, col, width);
        else return r < p.m ? row8<WIDTHS>((of_x ? x : dy) + r * width, col, width) : none8<T>();
    };
    auto settle = [&](int64_t tile, int i, Raw<T> v) {
        const bool of_x = i < kChunksX;
        const int at = of_x ? i : i - kChunksX, per = of_x ? KS * 4 : NS * 4, ld = of_x ? L::kXLd : L::kYLd, col = (at % per) * 8;
        if constexpr (WIDTHS == kEight) {
            into_place(v, col + 8 - (of_x ? p.k : p.n));
            if (tile * 32 + at / per >= p.m) v = none8<T>();
        }
        E* to = (of_x ? lx : ly) + (at / per) * ld + col;
        frag q[P];
        frags(v, q);
#pragma unroll
        for (int s = 0; s < P; ++s) *(frag*)(to + s * 32 * ld) = q[s];
    };
    for (int i = threadIdx.x; i < kChunksX + kChunksY; i += blockDim.x) settle(blockIdx.x, i, chunk(blockIdx.x, i));

    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        lds_barrier();          // x and dy are there; everybody has read the partial sums of the tile before
        const int64_t next = tile + gridDim.x;
        Raw<T> ahead[AHEAD];    // the next tile's chunks travel under this tile's products (what these do not hold follows later)
        if (WHOLE && (next + 1) * 32 <= p.m) {      // rows side by side: a tile's chunks are one stretch of x and one of dy
            const T *nx = x + next * (32 * KS * 32), *ny = dy + next * (32 * NS * 32) - kChunksX * 8;
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int i = threadIdx.x + q * blockDim.x;
                if (i < kChunksX + kChunksY) __builtin_memcpy(&ahead[q], (i < kChunksX ? nx : ny) + i * 8, sizeof(ahead[q]));
            }
        } else {
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int i = threadIdx.x + q * blockDim.x;
                if constexpr (WIDTHS == kEight) ahead[q] = chunk(next < tiles ? next : tile, min(i, kChunksX + kChunksY - 1));
                else if (next < tiles && i < kChunksX + kChunksY) ahead[q] = chunk(next, i);
            }
        }
        frag second[2][3];      // FINE: the second parts, which take the first ones' place in LDS when those have been used
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int row = b * 16 + c;
            f32x4 gv[2], uv[2], dh[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) gv[j] = uv[j] = dh[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                frag v[P];
#pragma unroll
                for (int q = 0; q < P; ++q) v[q] = *(const frag*)(lx + (q * 32 + row) * L::kXLd + s * 32 + g * 8);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    gv[j] = product<P, P>(wg[j][s], v, gv[j]);
                    uv[j] = product<P, P>(wu[j][s], v, uv[j]);
                }
            }
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                frag v[P];
#pragma unroll
                for (int q = 0; q < P; ++q) v[q] = *(const frag*)(ly + (q * 32 + row) * L::kYLd + s * 32 + g * 8);
#pragma unroll
                for (int j = 0; j < 2; ++j) dh[j] = product<P, P>(wdt[j][s], v, dh[j]);
            }
            float vg[8], vu[8], vh[8];      // dg, du, h: 8 neighbouring hidden values of row c
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float ga[4] = {gv[j][0], gv[j][1], gv[j][2], gv[j][3]};
                float aa[4], da[4];
                activate2(ga, p.act, aa, da);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vg[j * 4 + i] = dh[j][i] * uv[j][i] * da[i];
                    vu[j * 4 + i] = dh[j][i] * aa[i];
                    vh[j * 4 + i] = aa[i] * uv[j][i];
                }
            }
            frag dg[H], du[H], hv[H];
            cut8<E, H>(vg, dg);
            cut8<E, H>(vu, du);
            cut8<E, H>(vh, hv);
#pragma unroll
            for (int q = 0; q < P; ++q) {
                *(frag*)(hid + (q * 32 + row) * kHidLd + g * 8) = dg[q];
                *(frag*)(hid + ((P + q) * 32 + row) * kHidLd + g * 8) = du[q];
                *(frag*)(hid + ((2 * P + q) * 32 + row) * kHidLd + g * 8) = hv[q];
            }
            if constexpr (H == 2) {
                second[b][0] = dg[1];
                second[b][1] = du[1];
                second[b][2] = hv[1];
            }
            if (inputs) {
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
                    s = product<P, H>(wgt[t], dg, s);
                    s = product<P, H>(wut[t], du, s);
                    *(f32x4*)(mine + row * L::kPartLd + t * 16 + g * 4) = s;
                }
            }
        }
        if (grads) {
#pragma unroll
            for (int part_of = 0; part_of < (H == 2 ? 2 : 1); ++part_of) {
                wave_sync();
                if (part_of) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int i = 0; i < 3; ++i) *(frag*)(hid + (i * 32 + b * 16 + c) * kHidLd + g * 8) = second[b][i];
                    wave_sync();
                }
                auto columns = [&](const E* from, int ld, int col, frag (&to)[P]) {
#pragma unroll
                    for (int q = 0; q < P; ++q) to[q] = turned(from + q * 32 * ld, ld, col, lane);
                };
                frag ag[2][P], au[2][P];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    columns(hid, kHidLd, j * 16, ag[j]);
                    columns(hid + P * 32 * kHidLd, kHidLd, j * 16, au[j]);
                }
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    frag v[P];
                    columns(lx, L::kXLd, t * 16, v);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        dwg[j][t] = product<P, P>(ag[j], v, dwg[j][t]);
                        dwu[j][t] = product<P, P>(au[j], v, dwu[j][t]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) columns(hid + 2 * P * 32 * kHidLd, kHidLd, j * 16, ag[j]);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    frag v[P];
                    columns(ly, L::kYLd, t * 16, v);
#pragma unroll
                    for (int j = 0; j < 2; ++j) dwd[j][t] = product<P, P>(ag[j], v, dwd[j][t]);
                }
            }
        }
        lds_barrier();          // partial sums are there; everybody is done with x and dy
        if (inputs) {
            for (int i = threadIdx.x; i < 32 * KS * 4; i += blockDim.x) {
                const int row = i / (KS * 4), col = (i % (KS * 4)) * 8;
                const int64_t r = tile * 32 + row;
                if (r >= p.m || (!WHOLE && col >= p.k)) continue;
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (sh.so_far) {
                    const Raw<float> q = raw8<WHOLE>(sh.so_far + r * p.k, col, p.k);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = q.v[e];
                }
                for (int w = 0; w < waves; ++w) {
                    const f32x4* s = (const f32x4*)(sums + (w * 32 + row) * L::kPartLd + col);
                    const f32x4 s0 = s[0], s1 = s[1];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        v[q] += s0[q];
                        v[4 + q] += s1[q];
                    }
                }
                if (sh.partial) put8<WHOLE>(sh.partial + r * p.k, col, p.k, v);
                else put8<WHOLE>(dx + r * p.k, col, p.k, v);
            }
        }
        if (next < tiles) {
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int i = threadIdx.x + q * blockDim.x;
                if (i < kChunksX + kChunksY) settle(next, i, ahead[q]);
            }
            for (int i = threadIdx.x + AHEAD * blockDim.x; i < kChunksX + kChunksY; i += blockDim.x) settle(next, i, chunk(next, i));
        }
    }
    if (!grads) return;
    float* to = part + (int64_t)blockIdx.x * (2 * p.k + p.n) * p.f;
    float *to_up = to + (int64_t)p.f * p.k, *to_down = to_up + (int64_t)p.f * p.k;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = h0 + j * 16 + g * 4 + i;
            if (row >= p.f) continue;
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int col = t * 16 + c;
                if (col >= p.k) continue;
                to[(int64_t)row * p.k + col] = dwg[j][t][i];
                to_up[(int64_t)row * p.k + col] = dwu[j][t][i];
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int col = t * 16 + c;
                if (col < p.n) to_down[(int64_t)col * p.f + row] = dwd[j][t][i];
            }
        }
}

// the workgroups' partial gradients added up: 32 parameters by 16 threads each, every thread a fixed stripe of the workgroups, then
// those sums in pairs
template <class T>
__global__ __launch_bounds__(512) void narrow_join_kernel(const float* __restrict__ part, int parts, int64_t count, T* __restrict__ out) {
    __shared__ float lds[16][32];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + cx;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < count) {
        int q = ry;
        for (; q + 48 < parts; q += 64)         // (four on their way at a time)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] += part[(int64_t)(q + 16 * j) * count + i];
        for (int j = 0; q < parts; q += 16, ++j) a[j & 3] += part[(int64_t)q * count + i];
    }
    lds[ry][cx] = (a[0] + a[1]) + (a[2] + a[3]);
    for (int o = 8; o > 0; o >>= 1) {
        __syncthreads();
        if (ry < o) lds[ry][cx] += lds[ry + o][cx];
    }
    if (ry == 0 && i < count) out[i] = (T)lds[0][cx];
}

// ---- host -------------------------------------------------------------------------------------------------------------------------

int steps32(int64_t v) { return (int)((v + 31) / 32); }
int step_class(int s) { return s <= 1 ? 1 : s <= 2 ? 2 : 4; }
int parts_of(int dtype) { return dtype == NERF_F32 ? 3 : 1; }
// LDS of 32 hidden values' weights, and how many 32s a forward launch takes
int64_t fwd_lds(int dtype, int64_t k, int64_t n) { return 1024ll * parts_of(dtype) * (4 * step_class(steps32(k)) + 2 * step_class(steps32(n))); }
int fwd_pairs(int dtype, int64_t k, int64_t n) { return (int)(kLdsLimit / fwd_lds(dtype, k, n)); }

// Whether a backward launch has one wave a SIMD (and 128 hidden values a workgroup in place of 256): wider rows or more parts than the
// registers of half a SIMD hold.
bool solo(int dtype, int64_t n) { return dtype == NERF_F32 || n > 64; }
int hidden_of(int dtype, int64_t n) { return solo(dtype, n) ? 128 : 256; }
// Workgroups of a backward launch: as many as the chip holds at a time, by their waves' registers and their LDS (a block of few hidden
// values has workgroups of one wave: 700000 rows of bf16 16 -> 32 -> 16 with two a CU: 221 us, with six 79)
int bwd_groups(int dtype, int64_t m, int64_t k, int64_t f, int64_t n) {
    const int ks = steps32(k) == 1 ? 1 : 2, ns = step_class(steps32(n)), parts = parts_of(dtype), each = hidden_of(dtype, n);
    const int waves = steps32(f < each ? f : each);
    const int lds = parts * 32 * (ks * 32 + ns * 32 + 16) * 2 + waves * (3 * parts * 32 * kHidLd * 2 + 32 * (ks * 32 + 4) * 4);
    const int by_waves = (solo(dtype, n) ? 4 : 8) / waves, by_lds = kLdsLimit / lds;
    const int64_t tiles = (m + 31) / 32, most = (int64_t)kNumCU * (by_waves < by_lds ? by_waves : by_lds);
    return (int)(tiles < most ? tiles : most);
}
int64_t part_bytes(int dtype, int64_t m, int64_t k, int64_t f, int64_t n) {
    return ((int64_t)bwd_groups(dtype, m, k, f, n) * (2 * k + n) * f * 4 + 255) / 256 * 256;
}

template <class T, int KS, int NP, int WIDTHS, bool FINE> int fwd_launch(const T* params, const T* x, const Narrow& p, int lds, T* y, hipStream_t st) {
    static NerfLdsAttrCache cache;
    if (const int rc = nerf_ensure_dynamic_lds((const void*)narrow_fwd_kernel<T, KS, NP, WIDTHS, FINE>, lds, &cache, "nerf_gated_mlp_fwd")) return rc;
    const int64_t groups = ceil_div64(p.m, 32), most = (int64_t)kNumCU * (kLdsLimit / lds < 2 ? 1 : 2);
    narrow_fwd_kernel<T, KS, NP, WIDTHS, FINE><<<(unsigned)(groups < most ? groups : most), 512, lds, st>>>(params, x, p, y);
    return nerf_launch_status("nerf_gated_mlp_fwd");
}
template <class T, int KS, int NP> int fwd_pick(const T* params, const T* x, const Narrow& p, int lds, T* y, hipStream_t st) {
    if constexpr (Piece<T>::P == 1) {
        if (nerf_gated_fine(p.m, p.k, p.f, p.n))
            return p.k >= 8 ? fwd_launch<T, KS, NP, kEight, true>(params, x, p, lds, y, st) : fwd_launch<T, KS, NP, kAny, true>(params, x, p, lds, y, st);
    }
    if (p.k == KS * 32 && p.n == NP * 32) return fwd_launch<T, KS, NP, kFull, false>(params, x, p, lds, y, st);
    return p.k >= 8 ? fwd_launch<T, KS, NP, kEight, false>(params, x, p, lds, y, st) : fwd_launch<T, KS, NP, kAny, false>(params, x, p, lds, y, st);
}
template <class T, int KS> int fwd_by_n(const T* params, const T* x, const Narrow& p, int lds, T* y, hipStream_t st) {
    const int np = step_class(steps32(p.n));
    if (np == 1) return fwd_pick<T, KS, 1>(params, x, p, lds, y, st);
    if constexpr (Piece<T>::P == 1) {
        if (np == 4) return fwd_pick<T, KS, 4>(params, x, p, lds, y, st);
    }
    return fwd_pick<T, KS, 2>(params, x, p, lds, y, st);
}
template <class T> int fwd_by_k(const T* params, const T* x, const Narrow& p, int lds, T* y, hipStream_t st) {
    const int ks = step_class(steps32(p.k));
    if (ks == 1) return fwd_by_n<T, 1>(params, x, p, lds, y, st);
    if constexpr (Piece<T>::P == 1) {
        if (ks == 4) return fwd_by_n<T, 4>(params, x, p, lds, y, st);
    }
    return fwd_by_n<T, 2>(params, x, p, lds, y, st);
}

template <class T, int KS, int NS, int WIDTHS, int AHEAD, bool SOLO, bool FINE = false>
int bwd_launch(const T* params, const T* x, const T* dy, const Narrow& p, const Share& sh, int waves, int groups, T* dx, float* part, hipStream_t st) {
    const int lds = BwdLds<KS, NS, Piece<T>::P>::bytes(waves);
    static NerfLdsAttrCache cache;
    if (const int rc = nerf_ensure_dynamic_lds((const void*)narrow_bwd_kernel<T, KS, NS, WIDTHS, AHEAD, SOLO, FINE>, lds, &cache, "nerf_gated_mlp_bwd")) return rc;
    narrow_bwd_kernel<T, KS, NS, WIDTHS, AHEAD, SOLO, FINE><<<(unsigned)groups, waves * 64, lds, st>>>(params, x, dy, p, sh, dx, part);
    return nerf_launch_status("nerf_gated_mlp_bwd");
}
template <class T, int KS, int NS, bool SOLO>
int bwd_pick(const T* params, const T* x, const T* dy, const Narrow& p, const Share& sh, int waves, int groups, T* dx, float* part, hipStream_t st) {
    const bool whole = p.k == KS * 32 && p.n == NS * 32, eight = p.k >= 8 && p.n >= 8;
    if constexpr (Piece<T>::P == 1) {
        if (nerf_gated_fine(p.m, p.k, p.f, p.n))
            return eight ? bwd_launch<T, KS, NS, kEight, 2, SOLO, true>(params, x, dy, p, sh, waves, groups, dx, part, st)
                         : bwd_launch<T, KS, NS, kAny, 2, SOLO, true>(params, x, dy, p, sh, waves, groups, dx, part, st);
    }
    // Registers are short: four chunks ahead only where a workgroup's threads have more than two each, and neither parts nor ragged widths
    // take registers too (bf16, 700000 rows, two | four: 64 -> 64 -> 64 149 | 129 us, 51 -> 64 -> 64 208 | 272; fp32, 100000 rows,
    // 64 -> 64 -> 64: 136 | 147).
    if constexpr (Piece<T>::P == 1) {
        if (whole && waves * 64 * 2 < 128 * (KS + NS)) return bwd_launch<T, KS, NS, kFull, 4, SOLO>(params, x, dy, p, sh, waves, groups, dx, part, st);
    }
    if (whole) return bwd_launch<T, KS, NS, kFull, 2, SOLO>(params, x, dy, p, sh, waves, groups, dx, part, st);
    return eight ? bwd_launch<T, KS, NS, kEight, 2, SOLO>(params, x, dy, p, sh, waves, groups, dx, part, st)
                 : bwd_launch<T, KS, NS, kAny, 2, SOLO>(params, x, dy, p, sh, waves, groups, dx, part, st);
}
template <class T>
int bwd_by_shape(const T* params, const T* x, const T* dy, const Narrow& p, const Share& sh, int waves, int groups, T* dx, float* part, hipStream_t st) {
    const int ks = steps32(p.k), ns = steps32(p.n);
    if constexpr (Piece<T>::P == 3) {       // fp32: one or two steps each
        if (ks == 1) return ns == 1 ? bwd_pick<T, 1, 1, true>(params, x, dy, p, sh, waves, groups, dx, part, st)
                                    : bwd_pick<T, 1, 2, true>(params, x, dy, p, sh, waves, groups, dx, part, st);
        return ns == 1 ? bwd_pick<T, 2, 1, true>(params, x, dy, p, sh, waves, groups, dx, part, st)
                       : bwd_pick<T, 2, 2, true>(params, x, dy, p, sh, waves, groups, dx, part, st);
    } else {
        if (ns > 2) return bwd_pick<T, 2, 4, true>(params, x, dy, p, sh, waves, groups, dx, part, st);
        if (ks == 1) return ns == 1 ? bwd_pick<T, 1, 1, false>(params, x, dy, p, sh, waves, groups, dx, part, st)
                                    : bwd_pick<T, 1, 2, false>(params, x, dy, p, sh, waves, groups, dx, part, st);
        return ns == 1 ? bwd_pick<T, 2, 1, false>(params, x, dy, p, sh, waves, groups, dx, part, st)
                       : bwd_pick<T, 2, 2, false>(params, x, dy, p, sh, waves, groups, dx, part, st);
    }
}

template <class T>
int bwd_typed(const T* params, const T* x, const T* dy, int dtype, const Narrow& p, T* dx, void* dparams, int dparams_f32, char* ws, hipStream_t st) {
    float* part = dparams ? (float*)ws : nullptr;
    float* partial = (float*)(ws + part_bytes(dtype, p.m, p.k, p.f, p.n));
    const int each = hidden_of(dtype, p.n), groups = bwd_groups(dtype, p.m, p.k, p.f, p.n);
    for (int first = 0; first < p.f; first += each) {
        const int there = p.f - first < each ? p.f - first : each;
        const bool last = first + there == p.f;
        const Share sh = {first, dx && first > 0 ? partial : nullptr, dx && !last ? partial : nullptr};
        if (const int rc = bwd_by_shape(params, x, dy, p, sh, steps32(there), groups, dx, part, st)) return rc;
    }
    if (!dparams) return 0;
    const int64_t count = (2 * (int64_t)p.k + p.n) * p.f;
    const unsigned grid = (unsigned)ceil_div64(count, 32);
    if (dparams_f32) narrow_join_kernel<float><<<grid, 512, 0, st>>>(part, groups, count, (float*)dparams);
    else narrow_join_kernel<T><<<grid, 512, 0, st>>>(part, groups, count, (T*)dparams);
    return nerf_launch_status("nerf_gated_mlp_bwd");
}

}  // namespace

// All weights in LDS at once; in fp32, where y can hold the sum so far, in two halves.  Kernel time, two halves | the wide kernels, fp32
// 51 -> 241 -> 51: 65799 rows 84 | 147 us, 1000 rows 35 | 34 (and four launches); 20 rows 32 | 20 with those for few rows.
bool nerf_gated_narrow_fwd_ok(int dtype, int64_t m, int64_t k, int64_t f, int64_t n) {
    const int64_t most = dtype == NERF_F32 ? 64 : 128;
    return k <= most && n <= most && steps32(f) <= fwd_pairs(dtype, k, n) * (dtype == NERF_F32 && !nerf_gated_few_ok(m) ? 2 : 1);
}
// More than 64 columns of x: its two sets of transposed weights and their gradients do not fit the registers (65799 rows, fp16
// 128 -> 128 -> 128: 258 us here, 143 with the wide kernels); more than 64 of y only, 40 -> 228 -> 100: 170 us against 326.
// Rows do not enter the rule.  Kernel time of a training pass, narrow | wide, at 20, 300, 1000, 4000 rows:
//   bf16 32 ->  64 ->  16:   14 | 38    19 | 60    19 | 66    22 | 69      bf16 50 -> 228 ->  57:   32 | 54    49 | 73    42 | 85    47 | 89
//   fp32 27 ->  64 ->  16:   32 | 71    37 | 103   37 | 102   38 | 115     bf16 40 -> 228 -> 100:   54 | 51    60 | 74    63 | 80    70 | 86
//   fp32 50 -> 228 ->  57:  102 | 75   116 | 112  118 | 120  135 | 135     (65799 rows, fp32 51 -> 241 -> 51: 492 | 766)
bool nerf_gated_narrow_bwd_ok(int dtype, int64_t k, int64_t f, int64_t n) {
    return k <= 64 && n <= (dtype == NERF_F32 ? 64 : 128) && f <= 256;
}
int64_t nerf_gated_narrow_bwd_bytes(int dtype, int64_t m, int64_t k, int64_t f, int64_t n) {
    return part_bytes(dtype, m, k, f, n) + (f > hidden_of(dtype, n) ? m * k * 4 : 0);
}

int nerf_gated_narrow_fwd(const void* params, const void* x, int dtype, int64_t m, int64_t k, int64_t f, int64_t n, int act, void* y,
                          hipStream_t st) {
    const int all = steps32(f), launches = all <= fwd_pairs(dtype, k, n) ? 1 : 2, each = (all + launches - 1) / launches;
    for (int at = 0; at < all; at += each) {
        const int pairs = all - at < each ? all - at : each;
        const Narrow p = {m, (int)k, (int)f, (int)n, act, at * 32, pairs, at > 0};
        const int lds = (int)fwd_lds(dtype, k, n) * pairs;
        int rc = 0;
        NERF_DISPATCH_DTYPE(dtype, rc = fwd_by_k((const T*)params, (const T*)x, p, lds, (T*)y, st));
        if (rc) return rc;
    }
    return 0;
}

int nerf_gated_narrow_bwd(const void* params, const void* x, const void* dy, int dtype, int64_t m, int64_t k, int64_t f, int64_t n,
                          int act, void* dx, void* dparams, int dparams_f32, void* ws, hipStream_t st) {
    const Narrow p = {m, (int)k, (int)f, (int)n, act, 0, 0, 0};
    int rc = 0;
    NERF_DISPATCH_DTYPE(dtype, rc = bwd_typed((const T*)params, (const T*)x, (const T*)dy, dtype, p, (T*)dx, dparams, dparams_f32, (char*)ws, st));
    return rc;
}
