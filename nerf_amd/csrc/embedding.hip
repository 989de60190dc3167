// Row lookup with scaling, and its gradient by sorted indices.
//
//   y[i] = round(scale * table[index[i]])                                   (an index outside the table: a row of zeros)
//   dtable[v] = round(scale * sum over i with index[i] = v of dy[i])                        (rows nobody looked up: zeros)
//
// Backward.  Adding rows into the table with atomics gives other bits every time and serialises on the rows that many positions
// share (every sample of a ray looks up the same image's code).  Here the positions are sorted by index instead -- a stable
// radix sort of (index, position) pairs, 8 bits a pass, as many passes as the table's size has bytes, in one launch where a
// workgroup holds them all -- and every stretch of equal indices is added up in an order that sizes and indices alone decide (the
// positions of a share ascending, then the shares by stripes, below): every bit is the same each time.
//   A GROUP of lanes owns one 16-byte column piece per lane and walks its share of the sorted positions, keeping the running row in
// registers.  A stretch that lies within one share is finished there; one that crosses shares leaves its partial rows (fp32)
// in the workspace -- a share has at most two: the stretch it starts in the middle of and the one it ends in the middle of --
// and a second launch adds those up: a workgroup's threads each every so many-th share, ascending, then the threads' sums.  Rows that nobody looked up have to be zeros: the whole table is cleared by
// spare workgroups of the sort's launches, which leave most of the chip idle.
//
// Measured.  Forward, bound by HBM writes: 786432 rows of 48 fp32 in 33 to 35 us (4.5 TB/s), 32768 of 1000 bf16 in 26 us.  Backward, the same
// sizes: the sort 21 us in one pass and 33 us in two (50000 entries; with 100 MB of table cleared meanwhile), sums 45 and 33 us (3.3 and
// 2.0 TB/s of rows gathered by position), joins 9 and 23 us (the longest stretch: a workgroup for 256 of its columns).
#include "layers_common.h"

namespace {

// ---- forward -----------------------------------------------------------------------------------------------------------------

// One thread per 16-byte piece of an output row.  Bound by HBM writes where the table is small enough for the caches, by
// the reads of both sides otherwise.
template <class T>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const T* __restrict__ table, int64_t entries, int64_t dim, uint32_t pieces,
                                                            const int64_t* __restrict__ index, int64_t rows, float scale,
                                                            T* __restrict__ out) {
    constexpr int N = Vec16<T>::N;
    const int64_t total = rows * pieces;
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < total; k += (int64_t)gridDim.x * 256) {
        const int64_t row = total <= 0xffffffffll ? (int64_t)((uint32_t)k / pieces) : k / pieces;
        const int64_t col = (k - row * pieces) * N;
        const int64_t v = index[row];
        float a[N];
        if (v >= 0 && v < entries) {
            load_cols(table + v * dim, col, dim, a);
#pragma unroll
            for (int i = 0; i < N; ++i) a[i] *= scale;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) a[i] = 0.f;
        }
        store_cols(out + row * dim, col, dim, a);
    }
}

// ---- stable radix sort of (index, position) -----------------------------------------------------------------------------------

// What a launch's workgroups beyond its own clear: bytes [from, to) of the table's gradient (16-byte pieces, and the tail).
struct Clear {
    char* p;
    int64_t from, to;
    uint32_t own;       // workgroups of the launch's own work
};
__device__ __forceinline__ bool clears(const Clear& z) {
    if (blockIdx.x < z.own) return false;
    const int64_t parts = gridDim.x - z.own, part = blockIdx.x - z.own, pieces = (z.to - z.from) / 16;
    for (int64_t i = part * blockDim.x + threadIdx.x; i < pieces; i += parts * blockDim.x) {
        const uint4 zero = {0, 0, 0, 0};
        __builtin_memcpy(z.p + z.from + i * 16, &zero, 16);
    }
    if (part == 0)
        for (int64_t i = z.from + pieces * 16 + threadIdx.x * 2; i < z.to; i += blockDim.x * 2) *(uint16_t*)(z.p + i) = 0;
    return true;
}

// the key of a position: its index, or `entries` (sorts last, adds to nothing) where that is outside the table
__device__ __forceinline__ uint32_t key_of(const int64_t* index, int64_t i, uint32_t entries) {
    const int64_t v = index[i];
    return v >= 0 && v < (int64_t)entries ? (uint32_t)v : entries;
}

// the lanes of a wave that are live and have the same digit as this one
__device__ __forceinline__ uint64_t same_digit(bool live, uint32_t d) {
    uint64_t same = __ballot(live);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const uint64_t m = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? m : ~m;
    }
    return same;
}

// exclusive sum over 256 values, one a thread; `tmp`: four values of LDS
__device__ __forceinline__ uint32_t before_256(uint32_t v, uint32_t* tmp) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
    }
    if (lane == 63) tmp[wave] = inc;
    __syncthreads();
    uint32_t base = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w)
        if (w < wave) base += tmp[w];
    return base + inc - v;
}

// A tile: 4 waves x ROUNDS x 64 pairs.  counts[digit][tile], or [tile][digit] where no scan follows; FIRST: the keys come from the
// indices themselves.
template <bool FIRST, int ROUNDS>
__global__ __launch_bounds__(256) void sort_count_kernel(const int64_t* __restrict__ index, const uint32_t* __restrict__ keys,
                                                         uint32_t n, uint32_t entries, int shift, uint32_t tiles,
                                                         bool scan, uint32_t* __restrict__ counts, uint32_t* __restrict__ list, Clear z) {
    if (clears(z)) return;
    if (FIRST && blockIdx.x == 0 && threadIdx.x == 0) list[0] = 0;      // (nothing to join yet)
    __shared__ uint32_t h[256];
    h[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * (ROUNDS * 256);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = base + r * 256 + threadIdx.x;
        if (i < n) atomicAdd(&h[((FIRST ? key_of(index, i, entries) : keys[i]) >> shift) & 255], 1u);     // (integers: any order)
    }
    __syncthreads();
    counts[scan ? threadIdx.x * tiles + blockIdx.x : blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}

// exclusive sums over the tiles of each digit, a wave a digit, in place; totals[digit]
__global__ __launch_bounds__(256) void sort_scan_kernel(uint32_t* __restrict__ counts, uint32_t tiles, uint32_t* __restrict__ totals,
                                                        Clear z) {
    if (clears(z)) return;
    const int lane = threadIdx.x & 63;
    const uint32_t d = blockIdx.x * 4 + (threadIdx.x >> 6);
    uint32_t* row = counts + d * tiles;
    uint32_t carry = 0;
    for (uint32_t b = 0; b < tiles; b += 256) {
        uint32_t v[4], s = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = b + lane * 4 + i < tiles ? row[b + lane * 4 + i] : 0;
            s += v[i];
        }
        uint32_t inc = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(inc, o, 64);
            if (lane >= o) inc += up;
        }
        uint32_t run = carry + inc - s;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (b + lane * 4 + i < tiles) row[b + lane * 4 + i] = run;
            run += v[i];
        }
        carry += __shfl(inc, 63, 64);
    }
    if (lane == 0) totals[d] = carry;
}

// Every pair to its place: its digit's start + the pairs of that digit in earlier tiles + those before it in this tile.  totals null:
// `starts` are the counts themselves, and every workgroup adds up what it needs of them.
template <bool FIRST, int ROUNDS>
__global__ __launch_bounds__(256) void sort_place_kernel(const int64_t* __restrict__ index, const uint32_t* __restrict__ keys,
                                                         const uint32_t* __restrict__ pos, uint32_t n, uint32_t entries, int shift,
                                                         uint32_t tiles, const uint32_t* __restrict__ starts,
                                                         const uint32_t* __restrict__ totals, uint32_t* __restrict__ keys_out,
                                                         uint32_t* __restrict__ pos_out, Clear z) {
    if (clears(z)) return;
    __shared__ uint32_t h[4][256];      // running count of a digit in a wave's pairs, then the wave's next place
    __shared__ uint32_t tmp[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int w = 0; w < 4; ++w) h[w][threadIdx.x] = 0;
    uint32_t run = 0, all = 0;
    if (totals) {
        all = totals[threadIdx.x];
        run = starts[threadIdx.x * tiles + blockIdx.x];
    } else {
#pragma unroll 8
        for (uint32_t t = 0; t < tiles; ++t) {
            const uint32_t c = starts[t * 256 + threadIdx.x];
            all += c;
            run += t < blockIdx.x ? c : 0;
        }
    }
    run += before_256(all, tmp);        // (ends the clearing, too)
    const uint32_t base = blockIdx.x * (ROUNDS * 256) + wave * (ROUNDS * 64) + lane;
    uint32_t key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = base + r * 64;
        key[r] = i < n ? (FIRST ? key_of(index, i, entries) : keys[i]) : 0;
        if (i < n) atomicAdd(&h[wave][(key[r] >> shift) & 255], 1u);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t c = h[w][threadIdx.x];
        h[w][threadIdx.x] = run;
        run += c;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = base + r * 64, d = (key[r] >> shift) & 255;
        const bool live = i < n;
        const uint64_t same = same_digit(live, d);
        const uint32_t before = (uint32_t)__popcll(same & ((1ull << lane) - 1));
        const uint32_t at = live ? h[wave][d] + before : 0;
        wave_sync();        // every lane of the wave has read its place
        if (live && before == 0) h[wave][d] = at + (uint32_t)__popcll(same);
        wave_sync();
        if (live) {
            keys_out[at] = key[r];
            pos_out[at] = FIRST ? i : pos[i];
        }
    }
}

// the whole sort of up to 4096 pairs in one workgroup: the pairs stay in LDS between the passes
constexpr uint32_t kSmall = 4096;
__global__ __launch_bounds__(256) void sort_small_kernel(const int64_t* __restrict__ index, uint32_t n, uint32_t entries, int passes,
                                                         uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, uint32_t* __restrict__ list,
                                                         Clear z) {
    if (clears(z)) return;
    if (threadIdx.x == 0) list[0] = 0;
    __shared__ uint32_t key[2][kSmall];
    __shared__ uint16_t pos[2][kSmall];
    __shared__ uint32_t h[4][256], tmp[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        key[0][i] = key_of(index, i, entries);
        pos[0][i] = (uint16_t)i;
    }
    const uint32_t per = ((n + 255) / 256) * 64;        // pairs of a wave: whole rounds of 64
    const uint32_t b = min(wave * per, n), e = min(b + per, n);
    for (int p = 0; p < passes; ++p) {
        const int from = p & 1, shift = p * 8;
#pragma unroll
        for (int w = 0; w < 4; ++w) h[w][threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = b + lane; i < e; i += 64) atomicAdd(&h[wave][(key[from][i] >> shift) & 255], 1u);
        __syncthreads();
        uint32_t c[4], all = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) all += c[w] = h[w][threadIdx.x];
        uint32_t run = before_256(all, tmp);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            h[w][threadIdx.x] = run;
            run += c[w];
        }
        __syncthreads();
        for (uint32_t i0 = b; i0 < e; i0 += 64) {
            const uint32_t i = i0 + lane;
            const bool live = i < e;
            const uint32_t k = live ? key[from][i] : 0, d = (k >> shift) & 255;
            const uint64_t same = same_digit(live, d);
            const uint32_t before = (uint32_t)__popcll(same & ((1ull << lane) - 1));
            const uint32_t at = live ? h[wave][d] + before : 0;
            wave_sync();
            if (live && before == 0) h[wave][d] = at + (uint32_t)__popcll(same);
            wave_sync();
            if (live) {
                key[from ^ 1][at] = k;
                pos[from ^ 1][at] = pos[from][i];
            }
        }
        __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        keys_out[i] = key[passes & 1][i];
        pos_out[i] = pos[passes & 1][i];
    }
}

// ---- sums of equal stretches ---------------------------------------------------------------------------------------------------

__global__ __launch_bounds__(256) void clear_kernel(Clear z) { clears(z); }

struct SumShape {
    uint32_t n;             // sorted pairs
    uint32_t entries;
    int64_t dim;
    uint32_t share;         // sorted positions of a group
    uint32_t shares;
    int lanes;              // lanes of a group (a power of two): 16-byte pieces of a row a group covers
};

// list[0]: how many stretches have to be joined (zero before), list[2 ..]: the shares they begin in and their keys.
// Partial rows: part[(share * 2 + which) * dim]: which 0: the stretch that began before the share, 1: the one that goes on behind it.
// A share that lies wholly inside one stretch leaves its sum in 0 alone.
template <class T>
__global__ __launch_bounds__(256) void stretch_sum_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                          const T* __restrict__ dy, SumShape p, float scale, T* __restrict__ dtable,
                                                          float* __restrict__ part, uint32_t* __restrict__ list) {
    constexpr int kAhead = 4;
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & (p.lanes - 1);
    const uint32_t share = blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes;
    const int64_t col = ((int64_t)blockIdx.y * p.lanes + lane) * N;
    if (share >= p.shares || col >= p.dim) return;
    const uint32_t b = share * p.share, e = min(b + p.share, p.n);
    const uint32_t before = b ? keys[b - 1] : 0xffffffffu, after = e < p.n ? keys[e] : 0xffffffffu;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    uint32_t cur = keys[b];
    bool head = cur == before;          // the running stretch began in an earlier share
    auto flush = [&](bool tail) {
        if (cur >= p.entries) return;
        if (head || tail) {
            float* to = part + ((int64_t)share * 2 + (head ? 0 : 1)) * p.dim;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col + i < p.dim) to[col + i] = acc[i];
        } else {
            float o[N];
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = acc[i] * scale;
            store_cols(dtable + (int64_t)cur * p.dim, col, p.dim, o);
        }
    };
    // kAhead rows are on their way while as many are added; the positions they lie at, one step before that
    uint32_t k[kAhead], at[kAhead], kn[kAhead];
    Vec16<T> v[kAhead], vn[kAhead];
    auto where = [&](uint32_t i) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            k[j] = i + j < e ? keys[i + j] : p.entries;
            at[j] = i + j < e ? pos[i + j] : 0;
        }
    };
    auto fetch = [&]() {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            kn[j] = k[j];
            const T* row = dy + (int64_t)at[j] * p.dim;
            if (col + N <= p.dim) vn[j] = load16(row + col);
            else {
#pragma unroll
                for (int c = 0; c < N; ++c) vn[j].v[c] = col + c < p.dim ? row[col + c] : (T)0.f;
            }
        }
    };
    where(b);
    fetch();
    where(b + kAhead);
    for (uint32_t i = b; i < e; i += kAhead) {
        uint32_t kv[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            kv[j] = kn[j];
            v[j] = vn[j];
        }
        if (i + kAhead < e) {
            fetch();
            where(i + 2 * kAhead);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (i + j >= e) break;
            if (kv[j] != cur) {
                flush(false);
                cur = kv[j];
                head = false;
#pragma unroll
                for (int c = 0; c < N; ++c) acc[c] = 0.f;
            }
#pragma unroll
            for (int c = 0; c < N; ++c) acc[c] += (float)v[j].v[c];
        }
    }
    const bool tail = cur == after;
    flush(tail);
    // a stretch that begins here and goes on: to be joined (the order of the list does not matter: its stretches are independent)
    if (tail && !head && cur < p.entries && lane == 0 && blockIdx.y == 0) {
        const uint32_t at = atomicAdd(list, 1u);
        list[2 + 2 * at] = share;
        list[3 + 2 * at] = cur;
    }
}

// The stretches that cross shares: partial 1 of the share a stretch begins in, then partial 0 of the following ones, as long as they
// begin with its key.  L lanes of four columns each by 256 / L threads that take every so many-th share; those sums in order.
template <class T>
__global__ __launch_bounds__(256) void stretch_join_kernel(const uint32_t* __restrict__ keys, SumShape p, float scale,
                                                           const float* __restrict__ part, const uint32_t* __restrict__ list,
                                                           int L, T* __restrict__ dtable) {
    constexpr int kFlight = 4;     // shares' rows on their way (8: 24 in place of 23 us for 2000 stretches, most of two shares; 10 in place of 8 for 100)
    __shared__ f32x4 lds[256];
    const int x = threadIdx.x & (L - 1), y = threadIdx.x / L, stripes = 256 / L;
    const int64_t c = ((int64_t)blockIdx.y * L + x) * 4;
    const uint32_t count = list[0];
    for (uint32_t q = blockIdx.x; q < p.shares; q += gridDim.x) {
        const uint32_t share = list[2 + 2 * q], key = list[3 + 2 * q];     // (there is room for every share; read before `count` is known)
        if (q >= count) break;
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
        auto add = [&](const float* row) {
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] += c + i < p.dim ? row[c + i] : 0.f;
        };
        if (c < p.dim) {
            if (y == 0) add(part + ((int64_t)share * 2 + 1) * p.dim);
            bool on = true;
            for (uint32_t s0 = share + 1 + y; on && s0 < p.shares; s0 += kFlight * stripes) {
                float v[kFlight][4];
                bool mine[kFlight];
#pragma unroll
                for (int j = 0; j < kFlight; ++j) {
                    const uint32_t s = s0 + j * stripes;
                    mine[j] = s < p.shares && keys[s * p.share] == key;
                }
#pragma unroll
                for (int j = 0; j < kFlight; ++j) {     // (only those rows are read: most stretches have one or two)
                    const float* row = part + (int64_t)(s0 + j * stripes) * 2 * p.dim;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[j][i] = mine[j] && c + i < p.dim ? row[c + i] : 0.f;
                }
#pragma unroll
                for (int j = 0; j < kFlight; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) a[i] += v[j][i];
                on = mine[kFlight - 1];
            }
        }
        lds[threadIdx.x] = a;
        __syncthreads();
        if (y == 0 && c < p.dim) {
            for (int i = 1; i < stripes; ++i) a += lds[i * L + x];
            for (int i = 0; i < 4 && c + i < p.dim; ++i) dtable[(int64_t)key * p.dim + c + i] = (T)(a[i] * scale);
        }
        __syncthreads();
    }
}

constexpr int64_t kMaxRows = 0x7fffffff, kMaxEntries = 0x7fffffff, kMaxDim = 1 << 20;

int64_t up16(int64_t bytes) { return (bytes + 15) & ~(int64_t)15; }

// How the sorted positions are shared out: enough shares to fill the chip (256 CUs x 16 waves of groups), none shorter than 16:
// every stretch that crosses shares is written and read once more.
SumShape sum_shape(int64_t entries, int64_t dim, int64_t rows, int elem_bytes) {
    SumShape p = {};
    p.n = (uint32_t)rows;
    p.entries = (uint32_t)entries;
    p.dim = dim;
    const int64_t pieces = ceil_div64(dim, 16 / elem_bytes);
    p.lanes = 1;
    while (p.lanes < 64 && p.lanes < pieces) p.lanes <<= 1;
    const int64_t groups_wanted = (int64_t)kNumCU * 16 * (64 / p.lanes) / ceil_div64(pieces, p.lanes);
    int64_t share = ceil_div64(rows, groups_wanted > 0 ? groups_wanted : 1);
    if (share < 16) share = 16;
    if (ceil_div64(rows, share) > 16384) share = ceil_div64(rows, 16384);
    p.share = (uint32_t)share;
    p.shares = (uint32_t)ceil_div64(rows, share);
    return p;
}

struct Workspace {      // byte offsets
    int64_t keys[2], pos[2], counts, list, part, bytes;
};
// pairs of a sort tile: small ones while there are few, for the chip's sake
int sort_rounds(int64_t n) { return n <= 1048576 ? 4 : 16; }
Workspace workspace_of(const SumShape& p) {
    Workspace w;
    const int64_t n = p.n, tiles = ceil_div64(n, sort_rounds(n) * 256);
    int64_t at = 0;
    for (int i = 0; i < 2; ++i) { w.keys[i] = at; at += up16(n * 4); }
    for (int i = 0; i < 2; ++i) { w.pos[i] = at; at += up16(n * 4); }
    w.counts = at; at += up16((tiles + 1) * 256 * 4);       // (and the digits' totals)
    w.list = at; at += up16((2 + 2 * (int64_t)p.shares) * 4);
    w.part = at; at += (int64_t)p.shares * 2 * p.dim * 4;
    w.bytes = at > 0 ? at : 16;
    return w;
}

// Counts of up to so many tiles are summed by the workgroups that place the pairs, in no launch of their own (a whole
// pass, with | without: 8 tiles 31 | 28 us, 32 tiles 122 | 114, 59 tiles 48 | 50).
constexpr uint32_t kFewTiles = 48;

// The launches of the sort, each with its part of the table's clearing.  Returns which of the two pair buffers holds the result.
template <int ROUNDS>
int sort_pairs(const int64_t* index, const SumShape& p, const Workspace& w, char* ws, int passes, Clear z, hipStream_t st) {
    const uint32_t n = p.n, tiles = (uint32_t)ceil_div64(n, ROUNDS * 256);
    uint32_t *counts = (uint32_t*)(ws + w.counts), *totals = counts + (int64_t)tiles * 256, *list = (uint32_t*)(ws + w.list);
    const int64_t bytes = z.to;
    const bool scan = tiles > kFewTiles;
    const int launches = (scan ? 3 : 2) * passes;
    int done = 0;
    auto grid = [&](uint32_t own) {     // its own workgroups and, behind them, those that clear the next of `launches` parts
        z.own = own;
        z.from = bytes / 16 * done / launches * 16;
        ++done;
        z.to = done == launches ? bytes : bytes / 16 * done / launches * 16;
        const int64_t more = ceil_div64(z.to - z.from, 256 * 16 * 4);
        return dim3((unsigned)(own + (more < 4096 ? more : 4096)));
    };
    int from = 0;
    for (int pass = 0; pass < passes; ++pass) {
        const uint32_t *ki = (const uint32_t*)(ws + w.keys[from]), *pi = (const uint32_t*)(ws + w.pos[from]);
        uint32_t *ko = (uint32_t*)(ws + w.keys[from ^ 1]), *po = (uint32_t*)(ws + w.pos[from ^ 1]);
        const int shift = pass * 8;
        dim3 g = grid(tiles);
        if (pass == 0) sort_count_kernel<true, ROUNDS><<<g, 256, 0, st>>>(index, ki, n, p.entries, shift, tiles, scan, counts, list, z);
        else sort_count_kernel<false, ROUNDS><<<g, 256, 0, st>>>(index, ki, n, p.entries, shift, tiles, scan, counts, list, z);
        if (scan) {
            g = grid(64);
            sort_scan_kernel<<<g, 256, 0, st>>>(counts, tiles, totals, z);
        }
        g = grid(tiles);
        if (pass == 0) sort_place_kernel<true, ROUNDS><<<g, 256, 0, st>>>(index, ki, pi, n, p.entries, shift, tiles, counts, scan ? totals : nullptr, ko, po, z);
        else sort_place_kernel<false, ROUNDS><<<g, 256, 0, st>>>(index, ki, pi, n, p.entries, shift, tiles, counts, scan ? totals : nullptr, ko, po, z);
        from ^= 1;
    }
    return from;
}

}  // namespace

extern "C" int nerf_embedding_fwd(const void* table, int dtype, int64_t n_entries, int64_t dim, const int64_t* index, int64_t n_rows,
                                  float scale, void* out, void* stream) {
    NERF_REQUIRE(nerf_dtype_ok(dtype), "dtype must be NERF_F32, NERF_F16 or NERF_BF16");
    NERF_REQUIRE(n_entries >= 0 && n_entries <= kMaxEntries && n_rows >= 0 && n_rows <= kMaxRows && dim >= 1 && dim <= kMaxDim,
                 "n_entries and n_rows must be in [0, 2^31), dim in [1, 2^20]");
    if (n_rows == 0) return 0;
    NERF_REQUIRE(index && out && (table || n_entries == 0), "null pointer");
    hipStream_t st = (hipStream_t)stream;
    NERF_DISPATCH_DTYPE(dtype, {
        const int64_t pieces = ceil_div64(dim, Vec16<T>::N);
        const int64_t blocks = ceil_div64(n_rows * pieces, 256);
        embedding_fwd_kernel<T><<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, st>>>(
            (const T*)table, n_entries, dim, (uint32_t)pieces, index, n_rows, scale, (T*)out);
    });
    return nerf_launch_status("nerf_embedding_fwd");
}

extern "C" int64_t nerf_embedding_bwd_workspace_bytes(int dtype, int64_t n_entries, int64_t dim, int64_t n_rows) {
    if (!nerf_dtype_ok(dtype) || n_entries < 0 || n_entries > kMaxEntries || n_rows < 0 || n_rows > kMaxRows || dim < 1 || dim > kMaxDim) return -1;
    return workspace_of(sum_shape(n_entries, dim, n_rows, nerf_dtype_bytes(dtype))).bytes;
}

extern "C" int nerf_embedding_bwd(const int64_t* index, const void* dout, int dtype, int64_t n_rows, int64_t n_entries, int64_t dim,
                                  float scale, void* dtable, void* workspace, int64_t workspace_bytes, void* stream) {
    NERF_REQUIRE(nerf_dtype_ok(dtype), "dtype must be NERF_F32, NERF_F16 or NERF_BF16");
    NERF_REQUIRE(n_entries >= 0 && n_entries <= kMaxEntries && n_rows >= 0 && n_rows <= kMaxRows && dim >= 1 && dim <= kMaxDim,
                 "n_entries and n_rows must be in [0, 2^31), dim in [1, 2^20]");
    if (n_entries == 0) return 0;
    NERF_REQUIRE(dtable && (n_rows == 0 || (index && dout && workspace)), "null pointer");
    const SumShape p = sum_shape(n_entries, dim, n_rows, nerf_dtype_bytes(dtype));
    const Workspace w = workspace_of(p);
    NERF_REQUIRE(n_rows == 0 || (nerf_aligned(workspace, 16) && workspace_bytes >= w.bytes), "workspace too small or not 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    const int64_t bytes = n_entries * dim * nerf_dtype_bytes(dtype), clearing = ceil_div64(bytes, 256 * 16 * 4);
    Clear z = {(char*)dtable, 0, bytes, 0};
    if (n_rows == 0) {
        clear_kernel<<<(unsigned)(clearing < 65536 ? clearing : 65536), 256, 0, st>>>(z);
        return nerf_launch_status("nerf_embedding_bwd");
    }
    char* ws = (char*)workspace;
    uint32_t* list = (uint32_t*)(ws + w.list);
    int passes = 1;
    while (passes < 4 && ((uint32_t)n_entries >> (8 * passes)) != 0) ++passes;
    int at = 0;
    if (p.n <= kSmall) {
        z.own = 1;
        sort_small_kernel<<<(unsigned)(1 + (clearing < 65536 ? clearing : 65536)), 256, 0, st>>>(
            index, p.n, p.entries, passes, (uint32_t*)(ws + w.keys[0]), (uint32_t*)(ws + w.pos[0]), list, z);
    } else {
        at = sort_rounds(p.n) == 4 ? sort_pairs<4>(index, p, w, ws, passes, z, st) : sort_pairs<16>(index, p, w, ws, passes, z, st);
    }
    const uint32_t *keys = (const uint32_t*)(ws + w.keys[at]), *pos = (const uint32_t*)(ws + w.pos[at]);
    float* part = (float*)(ws + w.part);
    NERF_DISPATCH_DTYPE(dtype, {
        const dim3 grid((unsigned)ceil_div64(p.shares, 256 / p.lanes), (unsigned)ceil_div64(ceil_div64(dim, Vec16<T>::N), p.lanes));
        stretch_sum_kernel<T><<<grid, 256, 0, st>>>(keys, pos, (const T*)dout, p, scale, (T*)dtable, part, list);
        int L = 1;
        while (L < 64 && L * 4 < dim) L <<= 1;
        const unsigned joins = p.shares < 2048 ? p.shares : 2048;
        stretch_join_kernel<T><<<dim3(joins, (unsigned)ceil_div64(dim, 4 * L)), 256, 0, st>>>(keys, p, scale, part, list, L, (T*)dtable);
    });
    return nerf_launch_status("nerf_embedding_bwd");
}
