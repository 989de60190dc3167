// Gated feed-forward block: y = (act(x Wg^T) * (x Wu^T)) Wd^T, and its backward pass.
//
//   g = x Wg^T,  u = x Wu^T,  h = act(g) * u,  y = h Wd^T              x [M,K], Wg, Wu [F,K], Wd [N,F]
//   dh = dy Wd,  dg = dh * u * act'(g),  du = dh * act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// One tile kernel serves all of these products: an operand may have k along its rows (x, dy, h in the sums over widths) or across
// them (the same buffers in the sums over rows, the weights in dh and dx); the latter is read out of LDS transposed, so nothing
// is ever laid out twice.  Sums are fp32 (the matrix cores' accumulators).
//
// 16-bit types run on v_mfma_f32_32x32x16_{bf16,f16}.  fp32 runs on the same bf16 instruction: a float is cut into three bf16
// (8 + 8 + 8 bits: all 24 of its significand) and the six products of the three largest orders are summed -- what is dropped is
// below 2^-24 of a term, fp32's own rounding.  Six bf16 products cost 6/16 of the fp32 matrix instruction's time.
// Roundings: h, dg and du are rounded to the element type (fp32: cut into three bf16) because the matrix cores read them so;
// g and u are kept in fp32 between the passes, so that the activation's derivative is taken of what the forward pass had.
//
// Measured, 8192 rows, 2048 -> 8192 -> 2048 bf16 (a large library product: 1.2 to 1.5 PFLOP/s at these shapes): g, u and h 567 us (0.97
// PFLOP/s with 537 MB of g and u stored), y 245 us (1.12), dh with dg, du and h again 411 us (0.67: reads g and u), dx 467 us (1.18), the
// weights' gradients 382 us each on average (1.08).  fp32, 4001 rows, 1001 -> 2667 -> 1001: 335, 125, 254, 238 and 202 us each (0.7 to 1.1
// PFLOP/s of bf16 products), laying out 35 us and joins 18 us each.
#include <type_traits>

#include "gated_common.h"

namespace {

using namespace gated;

constexpr int kMaxSegs = 12;

// ---- operands -----------------------------------------------------------------------------------------------------------------

// One product C[i,j] = sum_k A(i,k) B(j,k) among those that are summed.  b2: the second matrix of a gated product (its columns are
// interleaved with b's).
template <class E> struct Seg { const E* a; const E* b; const E* b2; };

// An operand with k along its rows is [m][ld] with zeros in the columns from its width to k; one with k across them is [k][ld],
// of which `ka` (`kb`) rows exist: behind them the last one is read again, against zeros on the other side.
template <class E> struct Operands {
    Seg<E> seg[kMaxSegs];
    int n_segs;
    int64_t lda, ldb;       // in elements, multiples of 32
    int64_t m, n;           // i, j that exist
    int64_t k, ka, kb;      // k: a multiple of 32
};

// ---- epilogues ----------------------------------------------------------------------------------------------------------------
// Each takes four neighbouring columns of one row of the product, from a tile's registers or from summed partial products.

template <class T> __device__ __forceinline__ void put4(T* p, const float* v, int count) {
    if (count >= 4) {
        T o[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        __builtin_memcpy(p, o, sizeof(o));
    } else {
        if (count > 0) p[0] = (T)v[0];
        if (count > 1) p[1] = (T)v[1];
        if (count > 2) p[2] = (T)v[2];
    }
}

template <class E> struct StoreOut {        // C itself, fp32 or E; rows [half, half_ld) are left out, the ones behind follow on
    void* out;
    int64_t m, n, ld, half, half_ld;
    int f32;
    struct Pre {};
    __device__ __forceinline__ Pre pre(int64_t, int64_t) const { return Pre(); }
    static constexpr bool kGated = false;
    __host__ __device__ int64_t rows() const { return m; }
    __host__ __device__ int64_t cols() const { return n; }
    __device__ __forceinline__ bool whole(int64_t r, int64_t c, int rows_, int cols_) const {
        return r + rows_ <= m && c + cols_ <= n && (r + rows_ <= half || r >= half_ld);
    }
    __device__ __forceinline__ void put(int64_t r, int64_t c, const float* v, const float*, Pre) const {
        if (r >= m || c >= n || (r >= half && r < half_ld)) return;
        r -= r >= half_ld ? half_ld - half : 0;
        const int count = (int)(n - c < 4 ? n - c : 4);
        if (f32) put4((float*)out + r * ld + c, v, count);
        else put4((E*)out + r * ld + c, v, count);
    }
    // The same for a tile that lies wholly inside: a thread's column stays, its rows count from the tile's first.
    struct Spot { char* at; uint32_t pitch; };
    __device__ __forceinline__ Spot spot(int64_t r, int64_t c) const {
        r -= r >= half_ld ? half_ld - half : 0;
        return {(char*)out + (r * ld + c) * (f32 ? 4 : (int)sizeof(E)), (uint32_t)ld * (f32 ? 4u : (uint32_t)sizeof(E))};
    }
    __device__ __forceinline__ Pre pre_at(const Spot&, uint32_t) const { return Pre(); }
    __device__ __forceinline__ void put_at(const Spot& s, uint32_t row, const float* v, const float*, Pre) const {
        char* to = s.at + row * s.pitch;
        if (f32) put4((float*)to, v, 4);
        else put4((E*)to, v, 4);
    }
};

template <class E, int P> struct GateOut {      // h = act(g) * u into P planes [m][ld], zeros in the columns [n, ld); g, u kept
    E* h;
    float* saved;       // nullable
    int64_t m, n, ld, plane;
    int act;
    struct Pre {};
    __device__ __forceinline__ Pre pre(int64_t, int64_t) const { return Pre(); }
    static constexpr bool kGated = true;
    __host__ __device__ int64_t rows() const { return m; }
    __host__ __device__ int64_t cols() const { return ld; }
    __device__ __forceinline__ bool whole(int64_t r, int64_t c, int rows_, int cols_) const { return r + rows_ <= m && c + cols_ <= n; }
    __device__ __forceinline__ void hidden(const float* g, const float* u, int count, E (&o)[P][4]) const {
        const float gv[4] = {g[0], g[1], g[2], g[3]};
        float a[4];
        activate(gv, act, a);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            E q[P];
            cut<E, P>(i < count ? a[i] * u[i] : 0.f, q);
#pragma unroll
            for (int p = 0; p < P; ++p) o[p][i] = q[p];
        }
    }
    __device__ __forceinline__ void put(int64_t r, int64_t c, const float* g, const float* u, Pre) const {
        if (r >= m || c >= ld) return;
        E o[P][4];
        const int count = (int)(n - c < 4 ? (n - c < 0 ? 0 : n - c) : 4);
        hidden(g, u, count, o);
#pragma unroll
        for (int p = 0; p < P; ++p) __builtin_memcpy(h + p * plane + r * ld + c, o[p], sizeof(o[p]));     // (ld: a multiple of 32)
        if (saved) {
            float* to = saved + saved_at(r, c, m);
            put4(to, g, count);
            put4(to + kSavedCols, u, count);
        }
    }
    struct Spot { E* h; float* saved; };
    __device__ __forceinline__ Spot spot(int64_t r, int64_t c) const { return {h + r * ld + c, saved ? saved + saved_at(r, c, m) : nullptr}; }
    __device__ __forceinline__ Pre pre_at(const Spot&, uint32_t) const { return Pre(); }
    __device__ __forceinline__ void put_at(const Spot& s, uint32_t row, const float* g, const float* u, Pre) const {
        E o[P][4];
        hidden(g, u, 4, o);
        E* to = s.h + row * (uint32_t)ld;
#pragma unroll
        for (int p = 0; p < P; ++p) __builtin_memcpy(to + p * plane, o[p], sizeof(o[p]));
        if (saved) {
            float* keep = s.saved + row * (2 * kSavedCols);
            put4(keep, g, 4);
            put4(keep + kSavedCols, u, 4);
        }
    }
};

// dh -> dg | du into P planes [rows][pitch] (du from column ld on) and h into P planes [rows][ld]: zeros in the columns [n, ld) and in the
// rows [m, rows)
template <class E, int P> struct GradGateOut {
    const float* saved;
    E *dgu, *h;
    int64_t m, n, ld, pitch, m_ld;        // m_ld: rows of the buffers
    int act;
    struct Pre { float g[4], u[4]; };
    // What the forward pass kept of them.  Behind the last row that row's, behind the last column whatever lies there (`saved` ends
    // on a multiple of 128 columns): `put` takes neither.
    __device__ __forceinline__ Pre pre(int64_t r, int64_t c) const {
        Pre q;
        const float* from = saved + saved_at(r < m ? r : m - 1, c < ld ? c : 0, m);
        __builtin_memcpy(q.g, from, 16);
        __builtin_memcpy(q.u, from + kSavedCols, 16);
        return q;
    }
    static constexpr bool kGated = false;
    __host__ __device__ int64_t rows() const { return m_ld; }
    __host__ __device__ int64_t cols() const { return ld; }
    __device__ __forceinline__ bool whole(int64_t r, int64_t c, int rows_, int cols_) const { return r + rows_ <= m && c + cols_ <= n; }
    struct Out { E g[P][4], u[P][4], h[P][4]; };
    __device__ __forceinline__ void grads(const float* dh, const Pre& q, int count, Out& o) const {
        float a[4], d[4];
        activate2(q.g, act, a, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = i < count;
            E qg[P], qu[P], qh[P];
            cut<E, P>(in ? dh[i] * q.u[i] * d[i] : 0.f, qg);
            cut<E, P>(in ? dh[i] * a[i] : 0.f, qu);
            cut<E, P>(in ? a[i] * q.u[i] : 0.f, qh);
#pragma unroll
            for (int p = 0; p < P; ++p) { o.g[p][i] = qg[p]; o.u[p][i] = qu[p]; o.h[p][i] = qh[p]; }
        }
    }
    __device__ __forceinline__ void store(const Out& o, E* to_g, E* to_h) const {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            __builtin_memcpy(to_g + p * m_ld * pitch, o.g[p], sizeof(o.g[p]));
            __builtin_memcpy(to_g + p * m_ld * pitch + ld, o.u[p], sizeof(o.u[p]));
            __builtin_memcpy(to_h + p * m_ld * ld, o.h[p], sizeof(o.h[p]));
        }
    }
    __device__ __forceinline__ void put(int64_t r, int64_t c, const float* dh, const float*, const Pre& q) const {
        if (r >= m_ld || c >= ld) return;
        Out o;
        grads(dh, q, r < m ? (int)(n - c < 4 ? (n - c < 0 ? 0 : n - c) : 4) : 0, o);
        store(o, dgu + r * pitch + c, h + r * ld + c);
    }
    struct Spot { const float* saved; E *g, *h; };
    __device__ __forceinline__ Spot spot(int64_t r, int64_t c) const { return {saved + saved_at(r, c, m), dgu + r * pitch + c, h + r * ld + c}; }
    __device__ __forceinline__ Pre pre_at(const Spot& s, uint32_t row) const {
        Pre q;
        __builtin_memcpy(q.g, s.saved + row * (2 * kSavedCols), 16);
        __builtin_memcpy(q.u, s.saved + row * (2 * kSavedCols) + kSavedCols, 16);
        return q;
    }
    __device__ __forceinline__ void put_at(const Spot& s, uint32_t row, const float* dh, const float*, const Pre& q) const {
        Out o;
        grads(dh, q, 4, o);
        store(o, s.g + row * (uint32_t)pitch, s.h + row * (uint32_t)ld);
    }
};

// ---- the tile kernel ------------------------------------------------------------------------------------------------------------

typedef __attribute__((address_space(1))) const void GlobalPtr;
typedef __attribute__((address_space(3))) void LdsPtr;

constexpr int kStep = 32;       // k of a step: one matrix instruction's, 64 bytes of a row
constexpr int kBufs = 4;        // steps that are in LDS or on their way there

// One step of both operands' tiles, rows of k along (k = 32 x 2 bytes, `kAlong`) or rows across (a k's B columns).  The loads can
// only fill LDS in lane order, so a lane fetches the 16-byte chunk that belongs in its slot:
//   along:  chunk c of row r lies in slot c ^ ((r >> 2) & 3) of the row's four,
//   across: the pair of chunks p of row k lies in pair p ^ 2 (k & 3) of the row's,
// which spreads what a fragment read touches at a time -- 16 lanes' 16 bytes of as many rows, 32 lanes' 8 bytes of four -- over the
// 64 banks.  (Spread over 32 banks only, half of the LDS's cycles were conflicts.)
template <class E, int BM, int BN> struct Buf {
    E a[BM * kStep];
    E b[BN * kStep];
};
__device__ __forceinline__ int across_turn(int k) { return (k & 3) << 1; }

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v LdsShort4;

// waits until at most N of this wave's loads are under way, then for the other waves
template <int N> __device__ __forceinline__ void arrive() { asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(N) : "memory"); }

// B rows of an operand's tile: where a lane's loads come from and where its fragments lie
template <class E, int B, bool kAcross> struct Side {
    static constexpr int kLoads = B / 64;       // 1 KiB loads of a wave and step
    typedef typename Frag<E>::type frag;
    uint32_t off[kLoads], row[kLoads];          // bytes from the tile's first element in a step; `row`: the part that is the k row's
    uint32_t pitch;                             // bytes from k to k + 1 (across)
    int at[3];                                  // a lane's place in a fragment of 32 rows by 16 k

    // first: the tile's first row; there: rows that exist; pick(r): row r of the tile is the operand's row first + pick(r)
    template <class F> __device__ __forceinline__ void init(int lane, int wave, int64_t first, int64_t there, int64_t ld, F&& pick) {
        pitch = (uint32_t)ld * 2;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            if constexpr (!kAcross) {
                const int r = (j * 4 + wave) * 16 + (lane >> 2), chunk = (lane & 3) ^ ((r >> 2) & 3);
                const int64_t most = there - 1 - first, p = pick(r);
                off[j] = (uint32_t)(((p < most ? p : most) * ld + chunk * 8) * 2);
                row[j] = 0;
            } else {
                constexpr int kRow = B / 8;         // chunks of a k row
                const int k = (j * 4 + wave) * (64 / kRow) + lane / kRow, s = lane % kRow;
                const int64_t chunk = (((s >> 1) ^ across_turn(k)) << 1) | (s & 1), most = ld / 8 - 1 - first / 8;
                off[j] = (uint32_t)((chunk < most ? chunk : most) * 16);
                row[j] = (uint32_t)k;
            }
        }
        const int r = lane & 31, half = lane >> 5;
        if constexpr (!kAcross) {       // row r, chunk 2 kk + half
            at[0] = r * kStep + ((half ^ ((r >> 2) & 3)) * 8);
            at[1] = r * kStep + (((2 + half) ^ ((r >> 2) & 3)) * 8);
        } else {        // k rows 16 kk + 8 half + (l % 16) / 4 (and 4 more), columns 16 (l / 16 % 2) + 4 (l % 4) .. + 3
            const int k = 8 * half + ((lane & 15) >> 2);
            at[0] = k * B + (lane & 3) * 4;
            at[1] = across_turn(k);
            at[2] = (lane >> 4) & 1;
        }
    }
    __device__ __forceinline__ uint32_t offset(int j, uint32_t last) const {        // last: the last k row of this step that exists
        return kAcross ? min(row[j], last) * pitch + off[j] : off[j];
    }
    // rows [32 i, 32 i + 32) from row `base` (a multiple of 32) on, k [16 kk, 16 kk + 16)
    __device__ __forceinline__ frag read(const E* tile, int base, int i, int kk) const {
        if constexpr (!kAcross) {
            return *(const frag*)&tile[(base + i * 32) * kStep + at[kk]];
        } else {
            const int pair = (base >> 4) + 2 * i + at[2];
            const E* p = tile + at[0] + kk * 16 * B + (pair ^ at[1]) * 16;
            const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4*)p);
            const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4*)(p + 4 * B));
            const short8v both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(frag, both);
        }
    }
};

// B x B of C a workgroup of 2 x 2 waves.  Steps of 32 k go straight into LDS, four buffers deep: in step t the products of t
// run from registers while t + 1 is read out of LDS and t + 3 is sent for, into the buffer that t - 1 was read out of a step ago --
// so the barrier between the steps has no LDS read to wait for: every wave has used what it read of t - 1.  A wave's B / 2 x B / 2 piece is what it takes for
// LDS (reads and fills together) to need less time than the products; one wave a SIMD has the registers for it.
template <class E, class Epi, int B, bool kAAcross, bool kBAcross>
__global__ __launch_bounds__(256) void tile_kernel(Operands<E> op, Epi epi, int tiles_m, int tiles_n, float* part) {
#ifdef __HIP_DEVICE_COMPILE__       // (the host's pass knows no buffer descriptors)
    constexpr int T = B / 2, MI = T / 32, kLoads = B / 64;
    typedef typename Frag<E>::type frag;
    __shared__ __align__(128) Buf<E, B, B> buf0;        // (variables of their own: the compiler keeps their accesses apart)
    __shared__ __align__(128) Buf<E, B, B> buf1;
    __shared__ __align__(128) Buf<E, B, B> buf2;
    __shared__ __align__(128) Buf<E, B, B> buf3;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // tiles of one XCD (workgroups go round the eight of them) lie together, 8 tiles of m by all of n
    int tile = blockIdx.x;
    const int tiles = tiles_m * tiles_n, even = tiles & ~7;
    if (tile < even) tile = (tile & 7) * (even >> 3) + (tile >> 3);
    const int group = tile / (8 * tiles_n), in = tile - group * 8 * tiles_n;
    const int gm = min(8, tiles_m - group * 8);
    const int64_t m0 = (int64_t)(group * 8 + in % gm) * B, n0 = (int64_t)(in / gm) * (Epi::kGated ? B / 2 : B);

    const int per_seg = (int)(op.k / kStep), steps = per_seg * op.n_segs;
    const int t0 = (int)((int64_t)steps * blockIdx.y / gridDim.y), count = (int)((int64_t)steps * (blockIdx.y + 1) / gridDim.y) - t0;

    Side<E, B, kAAcross> sa;
    Side<E, B, kBAcross> sb;
    sa.init(lane, wave, m0, op.m, op.lda, [](int r) { return r; });
    // (gated: a wave's T columns are T / 2 of b, then the same T / 2 of b2)
    sb.init(lane, wave, n0, op.n, op.ldb, [](int r) { return Epi::kGated ? (r / T) * (T / 2) + r % (T / 2) : r; });

    // the next step to be sent for; behind the last one it stays where it is (that buffer is not read any more)
    int seg = t0 / per_seg, left = count;
    int64_t k0 = (int64_t)(t0 - seg * per_seg) * kStep;
    auto descriptor = [&](const E* p, int64_t row0, int64_t ld, bool across) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)(across ? p + k0 * ld + row0 : p + row0 * ld + k0), 0, 0x7fffffff, 0x00020000);
    };
    auto ra = descriptor(op.seg[seg].a, m0, op.lda, kAAcross), rb = descriptor(op.seg[seg].b, n0, op.ldb, kBAcross),
         rb2 = Epi::kGated ? descriptor(op.seg[seg].b2, n0, op.ldb, false) : rb;
    uint32_t last_a = (uint32_t)(op.ka - 1 - k0 < 31 ? op.ka - 1 - k0 : 31), last_b = (uint32_t)(op.kb - 1 - k0 < 31 ? op.kb - 1 - k0 : 31);
    auto load_one = [&](Buf<E, B, B>& to, int j) {       // one of a wave's loads of a step
        if (j < kLoads)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (LdsPtr*)&to.a[(j * 4 + wave) * 512], 16, sa.offset(j < kLoads ? j : 0, last_a), 0, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(((j - kLoads) * 4 + wave) * 16 % T >= T / 2 ? rb2 : rb,
                                                     (LdsPtr*)&to.b[((j - kLoads) * 4 + wave) * 512], 16,
                                                     sb.offset(j < kLoads ? 0 : j - kLoads, last_b), 0, 0, 0);
    };
    auto advance = [&]() {
        if (--left > 0) {
            k0 += kStep;
            if (k0 >= op.k) {
                k0 = 0;
                ++seg;
            }
            ra = descriptor(op.seg[seg].a, m0, op.lda, kAAcross);
            rb = descriptor(op.seg[seg].b, n0, op.ldb, kBAcross);
            rb2 = Epi::kGated ? descriptor(op.seg[seg].b2, n0, op.ldb, false) : rb;
            if (kAAcross) last_a = (uint32_t)(op.ka - 1 - k0 < 31 ? op.ka - 1 - k0 : 31);
            if (kBAcross) last_b = (uint32_t)(op.kb - 1 - k0 < 31 ? op.kb - 1 - k0 : 31);
        }
    };
    auto load = [&](Buf<E, B, B>& to) {
#pragma unroll
        for (int j = 0; j < 2 * kLoads; ++j) load_one(to, j);
        advance();
    };

    const int wm = wave >> 1, wn = wave & 1;
    f32x16 acc[MI][MI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;

    frag fa[2][MI], fb[2][2][MI];       // [kk], [set][kk]
    static_assert(MI == kLoads, "a step's reads and loads go out one by one between its rows of products");
    auto step = [&](Buf<E, B, B>& free, const Buf<E, B, B>& next, int set) {
        arrive<2 * kLoads>();       // t + 1 has arrived (t + 2 is on its way); everybody is done with t - 1
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                fb[set ^ 1][kk][i] = sb.read(next.b, wn * T, i, kk);
                load_one(free, kk * MI + i);
#pragma unroll
                for (int j = 0; j < MI; ++j) acc[i][j] = mfma(fb[set][kk][j], fa[kk][i], acc[i][j]);
                fa[kk][i] = sa.read(next.a, wm * T, i, kk);
                __builtin_amdgcn_sched_group_barrier(0x100, kBAcross ? 2 : 1, 0);       // LDS reads
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);                      // load
                __builtin_amdgcn_sched_group_barrier(0x008, MI, 0);                     // products
                __builtin_amdgcn_sched_group_barrier(0x100, kAAcross ? 2 : 1, 0);
            }
        advance();
    };
    load(buf0);
    load(buf1);
    load(buf2);
    arrive<4 * kLoads>();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            fa[kk][i] = sa.read(buf0.a, wm * T, i, kk);
            fb[0][kk][i] = sb.read(buf0.b, wn * T, i, kk);
        }
    for (int t = 0; t + 4 <= count; t += 4) {
        step(buf3, buf1, 0);
        step(buf0, buf2, 1);
        step(buf1, buf3, 0);
        step(buf2, buf0, 1);
    }
    if (count & 3) step(buf3, buf1, 0);
    if ((count & 3) > 1) step(buf0, buf2, 1);
    if ((count & 3) > 2) step(buf1, buf3, 0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (nothing fills or reads these buffers from here on)

    // A lane holds, of every 32 x 32 piece, row lane % 32 and the columns 8 q + 4 (lane / 32) .. + 3 of its four quads q.  Half of the
    // tile's rows at a time go through LDS (32 of them a buffer, quad q of row r in place q ^ (r & 15)), so that whole rows are
    // worked on and stored by neighbouring lanes -- in a loop: unrolled over the registers, the epilogue's code would not fit
    // the instruction cache.
    const int fr = lane & 31, fc = lane >> 5;
    constexpr int kHalf = MI / 2, kQuads = Epi::kGated ? B / 8 : B / 4;     // pieces of a wave; quads of a row
    constexpr int kEach = 32 * kQuads / 256, kBatch = kEach < 4 ? kEach : 4, kBatches = 2 * kHalf * (kEach / kBatch);
    typedef __attribute__((address_space(3))) f32x4 LdsQuad;
    auto stage_of = [&](int k) { return k == 0 ? (LdsQuad*)&buf0 : k == 1 ? (LdsQuad*)&buf1 : k == 2 ? (LdsQuad*)&buf2 : (LdsQuad*)&buf3; };
    // A thread's quads: always the same one of a row; the rows of a batch 256 / kQuads apart.
    const int q = threadIdx.x % kQuads, first_q = Epi::kGated ? (q / (T / 8)) * (T / 4) + q % (T / 8) : q;
    const bool whole = !part && epi.whole(m0, n0, B, Epi::kGated ? B / 2 : B);
    const typename Epi::Spot spot = epi.spot(m0, n0 + q * 4);      // (used where the tile is whole)
    struct Place { int round, lr; };
    auto place = [&](int batch, int z) {
        const int in = batch % (kEach / kBatch) * kBatch + z;
        return Place{batch / (kEach / kBatch), in * (256 / kQuads) + (int)threadIdx.x / kQuads};
    };
    auto row_of = [&](int half, const Place& w) { return (w.round & 1) * T + (half * kHalf + (w.round >> 1)) * 32 + w.lr; };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        typename Epi::Pre ahead[kBatch];        // what the epilogue reads travels a batch ahead
        auto fetch = [&](int batch) {
#pragma unroll
            for (int z = 0; z < kBatch; ++z) ahead[z] = epi.pre_at(spot, row_of(half, place(batch, z)));
        };
        if (whole) fetch(0);
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
            LdsQuad* to = stage_of(2 * i + wm) + fr * (B / 4);
#pragma unroll
            for (int j = 0; j < MI; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x16& x = acc[half * kHalf + i][j];
                    to[((wn * T + j * 32) / 4 + 2 * q + fc) ^ (fr & 15)] = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
                }
        }
        __syncthreads();
        // (loops of their own: the one for whole tiles has no branch in it, its loads and stores wait for nothing but themselves)
        auto staged = [&](const Place& w, float (&v)[4], float (&u)[4]) {
            const LdsQuad* row = stage_of(w.round) + w.lr * (B / 4);
            const f32x4 x = row[first_q ^ (w.lr & 15)], y = Epi::kGated ? row[(first_q + T / 8) ^ (w.lr & 15)] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 4; ++t) { v[t] = x[t]; u[t] = y[t]; }
        };
        if (whole) {
#pragma unroll 1
            for (int batch = 0; batch < kBatches; ++batch) {
                typename Epi::Pre now[kBatch];
#pragma unroll
                for (int z = 0; z < kBatch; ++z) now[z] = ahead[z];
                fetch(batch + 1 < kBatches ? batch + 1 : batch);
#pragma unroll
                for (int z = 0; z < kBatch; ++z) {
                    const Place w = place(batch, z);
                    float v[4], u[4];
                    staged(w, v, u);
                    epi.put_at(spot, row_of(half, w), v, u, now[z]);
                }
            }
        } else {
            const int64_t c = n0 + q * 4, rows_there = epi.rows() - m0, cols = epi.cols();
            const int64_t width = Epi::kGated ? 2 * cols : cols;
            if (c < cols)
#pragma unroll 1
                for (int batch = 0; batch < kBatches; ++batch) {
                    float v[kBatch][4], u[kBatch][4];
                    typename Epi::Pre now[kBatch];
#pragma unroll
                    for (int z = 0; z < kBatch; ++z) {
                        const Place w = place(batch, z);
                        staged(w, v[z], u[z]);
                        if (!part) now[z] = epi.pre(m0 + row_of(half, w), c);
                    }
#pragma unroll
                    for (int z = 0; z < kBatch; ++z) {
                        const int row = row_of(half, place(batch, z));
                        if (row >= rows_there) continue;
                        if (!part) {
                            epi.put(m0 + row, c, v[z], u[z], now[z]);
                        } else {        // split over k: partial products [split][rows][cols]
                            float* to = part + ((int64_t)blockIdx.y * epi.rows() + m0 + row) * width + c;
                            const int there = (int)(cols - c < 4 ? cols - c : 4);
                            put4(to, v[z], there);
                            if (Epi::kGated) put4(to + cols, u[z], there);
                        }
                    }
                }
        }
        __syncthreads();
    }
#endif
}

// Partial products summed, then the epilogue: 256 / stripes quads by `stripes` threads each, every thread every so many-th split,
// those sums in order (a small product has hundreds of splits and few quads: one thread a quad would wait for one load after
// another).
template <class Epi> __global__ __launch_bounds__(256) void join_kernel(Epi epi, const float* __restrict__ part, int splits, int stripes) {
    constexpr int G = Epi::kGated ? 2 : 1;
    __shared__ f32x4 sums[G][256];
    const int lanes = 256 / stripes, x = threadIdx.x % lanes, y = threadIdx.x / lanes;
    const int64_t rows = epi.rows(), cols = epi.cols(), quads = (cols + 3) / 4, width = G * cols, plane = rows * width;
    for (int64_t k0 = (int64_t)blockIdx.x * lanes; k0 < rows * quads; k0 += (int64_t)gridDim.x * lanes) {
        const int64_t k = k0 + x, r = k / quads, c = (k - r * quads) * 4;
        const int count = k < rows * quads ? (int)(cols - c < 4 ? cols - c : 4) : 0;
        f32x4 a[G];
#pragma unroll
        for (int q = 0; q < G; ++q) a[q] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float* p = part + r * width + c;
        auto add = [&](int s, int q, f32x4& to) {
            const float* at = p + s * plane + q * cols;
            if (count == 4) {
                f32x4 v;
                __builtin_memcpy(&v, at, 16);
                to += v;
            } else {
                for (int i = 0; i < count; ++i) to[i] += at[i];
            }
        };
#pragma unroll 4
        for (int s = y; s < splits; s += stripes)
#pragma unroll
            for (int q = 0; q < G; ++q) add(s, q, a[q]);
#pragma unroll
        for (int q = 0; q < G; ++q) sums[q][threadIdx.x] = a[q];
        __syncthreads();
        if (y == 0 && count) {
            for (int i = 1; i < stripes; ++i)
#pragma unroll
                for (int q = 0; q < G; ++q) a[q] += sums[q][i * lanes + x];
            const float v[4] = {a[0][0], a[0][1], a[0][2], a[0][3]};
            const float u[4] = {a[G - 1][0], a[G - 1][1], a[G - 1][2], a[G - 1][3]};
            epi.put(r, c, v, u, epi.pre(r, c));
        }
        __syncthreads();
    }
}

// ---- laying operands out ----------------------------------------------------------------------------------------------------------

// src [rows][cols] -> P planes [rows][ld], zeros in [cols, ld); several matrices a launch, each by its share of the workgroups
template <class T, class E> struct Lay {
    const T* src;
    E* dst;
    int64_t rows, cols, ld;
    unsigned first;     // its first workgroup
};
constexpr int kMostLays = 5;
template <class T, class E> struct Lays {
    Lay<T, E> job[kMostLays];
    int count = 0;
    unsigned groups = 0;
    void add(const T* src, int64_t rows, int64_t cols, int64_t ld, E* dst) {
        job[count++] = {src, dst, rows, cols, ld, groups};
        const int64_t g = ceil_div64(rows * (ld / 4), 256 * 2);
        groups += (unsigned)(g < 1 ? 1 : g < 16384 ? g : 16384);
    }
};
template <class T, class E, int P> __global__ __launch_bounds__(256) void lay_kernel(Lays<T, E> l) {
    int i = 0;
    while (i + 1 < l.count && blockIdx.x >= l.job[i + 1].first) ++i;
    const Lay<T, E> j = l.job[i];
    const int64_t groups = (i + 1 < l.count ? l.job[i + 1].first : gridDim.x) - j.first, quads = j.ld / 4, plane = j.rows * j.ld;
    for (int64_t k = (int64_t)(blockIdx.x - j.first) * 256 + threadIdx.x; k < j.rows * quads; k += groups * 256) {
        const int64_t r = k / quads, c = (k - r * quads) * 4;
        E o[P][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            E q[P];
            cut<E, P>(c + i < j.cols ? (float)j.src[r * j.cols + c + i] : 0.f, q);
#pragma unroll
            for (int p = 0; p < P; ++p) o[p][i] = q[p];
        }
#pragma unroll
        for (int p = 0; p < P; ++p) __builtin_memcpy(j.dst + p * plane + r * j.ld + c, o[p], sizeof(o[p]));
    }
}

template <class T> __global__ __launch_bounds__(256) void fill_zero_kernel(T* __restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = (T)0.f;
}

// ---- host -------------------------------------------------------------------------------------------------------------------------

int64_t up32(int64_t v) { return (v + 31) & ~(int64_t)31; }
int64_t up256(int64_t v) { return (v + 255) & ~(int64_t)255; }
unsigned grid_for(int64_t items) {
    const int64_t b = ceil_div64(items, 256);
    return (unsigned)(b < 1 ? 1 : b < 65536 ? b : 65536);
}

// How a product is cut: tiles of 256 or 128 and splits over k.  A step (32 k) of a 256 tile takes a CU about 1100 cycles; of the two
// 128 tiles that a CU holds at a time, 770 for both (they read twice the LDS a product).  Tiles come in rounds of as many as the
// chip holds, a workgroup spends some 12 steps filling LDS and storing, and splits write and read their partial products
// (a cycle for 2 KiB, the chip's bandwidth) in a launch of their own.  The cheapest by that count is taken.
struct Cut { int tile, splits; };
Cut cut_for(int64_t m, int64_t n, int64_t steps) {
    Cut best = {256, 1};
    double least = 1e300;
    for (int tile = 256; tile >= 128; tile -= 128) {
        const int64_t tiles = ceil_div64(m, tile) * ceil_div64(n, tile), slots = tile == 256 ? kNumCU : 2 * kNumCU;
        if (tiles == 0) break;
        for (int s = 1; s <= 256 && (s == 1 || steps / s >= 4); s += s < 8 ? 1 : s / 4) {
            const int64_t rounds = ceil_div64(tiles * s, slots);
            double cost = (double)rounds * ((double)ceil_div64(steps, s) + 12) * (tile == 256 ? 1100. : 770.);
            if (s > 1) cost += 10000. + (double)m * n * 8 * s / 2048;
            if (cost < least) { least = cost; best = {tile, s}; }
        }
    }
    return best;
}
int64_t part_floats(int64_t m, int64_t n, int64_t steps) {
    const int s = cut_for(m, n, steps).splits;
    return s > 1 ? s * m * n : 0;
}

template <bool kAAcross, bool kBAcross, class E, class Epi>
int run_product(const Operands<E>& op, const Epi& epi, float* part, hipStream_t st) {
    const int64_t rows = epi.rows(), cols = Epi::kGated ? 2 * epi.cols() : epi.cols();
    const Cut cut = cut_for(rows, cols, op.k / kStep * op.n_segs);
    const int64_t tm = ceil_div64(rows, cut.tile), tn = ceil_div64(cols, cut.tile);
    const dim3 grid((unsigned)(tm * tn), (unsigned)cut.splits);
    float* to = cut.splits > 1 ? part : nullptr;
    if (cut.tile == 256) tile_kernel<E, Epi, 256, kAAcross, kBAcross><<<grid, 256, 0, st>>>(op, epi, (int)tm, (int)tn, to);
    else tile_kernel<E, Epi, 128, kAAcross, kBAcross><<<grid, 256, 0, st>>>(op, epi, (int)tm, (int)tn, to);
    if (cut.splits > 1) {
        int stripes = 1;
        while (stripes < 16 && stripes * 8 < cut.splits) stripes *= 2;
        join_kernel<Epi><<<grid_for(rows * ceil_div64(epi.cols(), 4) * stripes), 256, 0, st>>>(epi, part, cut.splits, stripes);
    }
    return 0;
}

// Elements behind a row of dg | du: rows 32 KiB apart, as those of 8192 hidden values would be, fall on a few memory channels (8192 rows,
// dg and du written: 446 us, with 128 bytes between the rows 424; the same for h only slowed its reader down).
constexpr int kPad = 64;
struct Shape {
    int64_t m, k, f, n, kp, fp, np, mp;
    int64_t gp;             // pitch of dg | du
    int planes, hidden, elem;       // operand planes; those of the hidden values; bytes of an element of x, params, y
    Shape(int dtype, int64_t rows, int64_t n_in, int64_t neurons, int64_t n_out)
        : m(rows), k(n_in), f(neurons), n(n_out), kp(up32(n_in)), fp(up32(neurons)), np(up32(n_out)), mp(up32(rows)), gp(2 * fp + kPad),
          planes(dtype == NERF_F32 ? 3 : 1), hidden(dtype == NERF_F32 ? 3 : nerf_gated_fine(rows, n_in, neurons, n_out) ? 2 : 1), elem(nerf_dtype_bytes(dtype)) {}
    int pairs() const { return planes == 3 ? 6 : 1; }               // products that are summed
    int hidden_pairs() const { return planes == 3 ? 6 : hidden; }
    bool lay_k() const { return planes == 3 || k % 32 != 0; }                            // x and the gate / up weights are laid out anew
    bool lay_down() const { return planes == 3 || f % 32 != 0; }
    bool lay_n() const { return planes == 3 || n % 32 != 0; }                            // dy
    int64_t steps(int64_t inner) const { return ceil_div64(inner, kStep) * pairs(); }
    int64_t hidden_steps(int64_t inner) const { return ceil_div64(inner, kStep) * hidden_pairs(); }
};

struct FwdSpace {
    int64_t x, gate, up, down, h, part, bytes;
    explicit FwdSpace(const Shape& s) {
        int64_t at = 0;
        auto take = [&](int64_t b) { const int64_t o = at; at += up256(b); return o; };
        x = s.lay_k() ? take(2 * s.planes * s.m * s.kp) : -1;
        gate = s.lay_k() ? take(2 * s.planes * s.f * s.kp) : -1;
        up = s.lay_k() ? take(2 * s.planes * s.f * s.kp) : -1;
        down = s.lay_down() ? take(2 * s.planes * s.n * s.fp) : -1;
        h = take(2 * s.hidden * s.m * s.fp);
        const int64_t a = part_floats(s.m, 2 * s.fp, s.steps(s.kp)), b = part_floats(s.m, s.n, s.hidden_steps(s.fp));
        part = take(4 * (a > b ? a : b));
        bytes = at;
    }
};

struct BwdSpace {
    int64_t x, dy, gate, up, down, dgu, h, part, bytes;
    explicit BwdSpace(const Shape& s) {
        int64_t at = 0;
        auto take = [&](int64_t b) { const int64_t o = at; at += up256(b); return o; };
        x = s.lay_k() ? take(2 * s.planes * s.m * s.kp) : -1;
        gate = s.lay_k() ? take(2 * s.planes * s.f * s.kp) : -1;
        up = s.lay_k() ? take(2 * s.planes * s.f * s.kp) : -1;
        dy = s.lay_n() ? take(2 * s.planes * s.m * s.np) : -1;
        down = s.lay_down() ? take(2 * s.planes * s.n * s.fp) : -1;
        dgu = take(2 * s.hidden * s.mp * s.gp);
        h = take(2 * s.hidden * s.mp * s.fp);
        const int64_t p[4] = {part_floats(s.mp, s.fp, s.steps(s.np)), part_floats(s.m, s.k, 2 * s.hidden_steps(s.fp)),
                              part_floats(s.fp + s.f, s.k, s.hidden_steps(s.mp)), part_floats(s.n, s.f, s.hidden_steps(s.mp))};
        int64_t most = 0;
        for (int i = 0; i < 4; ++i) most = p[i] > most ? p[i] : most;
        part = take(4 * most);
        bytes = at;
    }
};

// the plane pairs whose products are summed: everything (one plane) or the three largest orders of three planes, small terms first
struct Pair { int a, b; };
const Pair kPairs3[6] = {{1, 1}, {0, 2}, {2, 0}, {0, 1}, {1, 0}, {0, 0}}, kPairs21[2] = {{1, 0}, {0, 0}}, kPairs12[2] = {{0, 1}, {0, 0}};

// na, nb: planes of either side
template <class E> void add_segs(Operands<E>& op, int na, int nb, const E* a, int64_t pa, const E* b, int64_t pb, const E* b2 = nullptr) {
    const Pair* pr = na == 3 ? kPairs3 : na == 2 ? kPairs21 : kPairs12 + (nb == 2 ? 0 : 1);
    const int pairs = na == 3 ? 6 : na > nb ? na : nb;
    for (int i = 0; i < pairs; ++i)
        op.seg[op.n_segs++] = {a + pr[i].a * pa, b + pr[i].b * pb, b2 ? b2 + pr[i].b * pb : nullptr};
}
template <class E> Operands<E> operands(int64_t m, int64_t n, int64_t k, int64_t lda, int64_t ldb, int64_t ka, int64_t kb) {
    Operands<E> op = {};
    op.m = m; op.n = n; op.k = k; op.lda = lda; op.ldb = ldb; op.ka = ka; op.kb = kb;
    return op;
}

// P: planes of the operands, H: of the hidden values
template <class T, class E, int P, int H>
int fwd_typed(const T* params, const T* x, const Shape& s, int act, T* y, float* saved, char* ws, hipStream_t st) {
    const FwdSpace w(s);
    const T *gate = params, *up = params + s.f * s.k, *down = params + 2 * s.f * s.k;
    const E *xa = (const E*)x, *ga = (const E*)gate, *ua = (const E*)up, *da = (const E*)down;
    Lays<T, E> lays;
    auto lay = [&](const T* src, int64_t rows, int64_t cols, int64_t ld, int64_t to) {
        lays.add(src, rows, cols, ld, (E*)(ws + to));
        return (const E*)(ws + to);
    };
    if (s.lay_k()) {
        xa = lay(x, s.m, s.k, s.kp, w.x);
        ga = lay(gate, s.f, s.k, s.kp, w.gate);
        ua = lay(up, s.f, s.k, s.kp, w.up);
    }
    if (s.lay_down()) da = lay(down, s.n, s.f, s.fp, w.down);
    if (lays.count) lay_kernel<T, E, P><<<lays.groups, 256, 0, st>>>(lays);
    E* h = (E*)(ws + w.h);
    float* part = (float*)(ws + w.part);
    Operands<E> op = operands<E>(s.m, s.f, s.kp, s.kp, s.kp, s.kp, s.kp);
    add_segs(op, P, P, xa, s.m * s.kp, ga, s.f * s.kp, ua);
    run_product<false, false>(op, GateOut<E, H>{h, saved, s.m, s.f, s.fp, s.m * s.fp, act}, part, st);
    op = operands<E>(s.m, s.n, s.fp, s.fp, s.fp, s.fp, s.fp);
    add_segs(op, H, P, (const E*)h, s.m * s.fp, da, s.n * s.fp);
    run_product<false, false>(op, StoreOut<E>{y, s.m, s.n, s.n, s.m, s.m, P == 3}, part, st);
    return nerf_launch_status("nerf_gated_mlp_fwd");
}

template <class T, class E, int P, int H>
int bwd_typed(const T* params, const T* x, const T* dy, const float* saved, const Shape& s, int act, T* dx, void* dparams, int dparams_f32,
              char* ws, hipStream_t st) {
    const BwdSpace w(s);
    const T *gate = params, *up = params + s.f * s.k, *down = params + 2 * s.f * s.k;
    const int out_f32 = P == 3 || dparams_f32, out_b = out_f32 ? 4 : 2;
    E *dgu = (E*)(ws + w.dgu), *h = (E*)(ws + w.h);
    float* part = (float*)(ws + w.part);
    const E *xa = (const E*)x, *ga = (const E*)gate, *ua = (const E*)up, *da = (const E*)down, *dya = (const E*)dy;
    Lays<T, E> lays;
    auto lay = [&](const T* src, int64_t rows, int64_t cols, int64_t ld, int64_t to) {
        lays.add(src, rows, cols, ld, (E*)(ws + to));
        return (const E*)(ws + to);
    };
    if (s.lay_n()) dya = lay(dy, s.m, s.n, s.np, w.dy);
    if (s.lay_down()) da = lay(down, s.n, s.f, s.fp, w.down);
    if (s.lay_k() && dx) {
        ga = lay(gate, s.f, s.k, s.kp, w.gate);
        ua = lay(up, s.f, s.k, s.kp, w.up);
    }
    if (s.lay_k() && dparams) xa = lay(x, s.m, s.k, s.kp, w.x);
    if (lays.count) lay_kernel<T, E, P><<<lays.groups, 256, 0, st>>>(lays);
    Operands<E> op = operands<E>(s.m, s.f, s.np, s.np, s.fp, s.np, s.n);
    add_segs(op, P, P, dya, s.m * s.np, da, s.n * s.fp);
    run_product<false, true>(op, GradGateOut<E, H>{saved, dgu, h, s.m, s.f, s.fp, s.gp, s.mp, act}, part, st);
    if (dx) {
        op = operands<E>(s.m, s.k, s.fp, s.gp, s.kp, s.fp, s.f);
        add_segs(op, H, P, (const E*)dgu, s.mp * s.gp, ga, s.f * s.kp);
        add_segs(op, H, P, (const E*)dgu + s.fp, s.mp * s.gp, ua, s.f * s.kp);
        run_product<false, true>(op, StoreOut<E>{dx, s.m, s.k, s.k, s.m, s.m, P == 3}, part, st);
    }
    if (!dparams) return nerf_launch_status("nerf_gated_mlp_bwd");
    op = operands<E>(2 * s.fp, s.k, s.mp, s.gp, s.kp, s.mp, s.m);
    add_segs(op, H, P, (const E*)dgu, s.mp * s.gp, xa, s.m * s.kp);
    run_product<true, true>(op, StoreOut<E>{dparams, s.fp + s.f, s.k, s.k, s.f, s.fp, out_f32}, part, st);
    op = operands<E>(s.n, s.f, s.mp, s.np, s.fp, s.m, s.mp);
    add_segs(op, P, H, dya, s.m * s.np, (const E*)h, s.mp * s.fp);
    run_product<true, true>(op, StoreOut<E>{(char*)dparams + 2 * s.f * s.k * out_b, s.n, s.f, s.f, s.n, s.n, out_f32}, part, st);
    return nerf_launch_status("nerf_gated_mlp_bwd");
}

// f(element, operand element, planes of the operands, planes of the hidden values)
template <class F> int by_type(int dtype, int hidden, F&& f) {
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 3> three;
    if (dtype == NERF_F32) return f(0.f, (__bf16)0.f, three, three);
    if (dtype == NERF_F16) return hidden == 2 ? f((_Float16)0.f, (_Float16)0.f, one, two) : f((_Float16)0.f, (_Float16)0.f, one, one);
    return hidden == 2 ? f((__bf16)0.f, (__bf16)0.f, one, two) : f((__bf16)0.f, (__bf16)0.f, one, one);
}

// The narrow kernels where they apply -- the forward one only where no backward pass needs g and u kept.
bool narrow_fwd(const Shape& s, int dtype, bool keep) { return !keep && nerf_gated_narrow_fwd_ok(dtype, s.m, s.k, s.f, s.n); }
bool narrow_bwd(const Shape& s, int dtype) { return nerf_gated_narrow_bwd_ok(dtype, s.k, s.f, s.n); }
int64_t fwd_bytes(const Shape& s, int dtype, bool keep) {
    if (narrow_fwd(s, dtype, keep && !narrow_bwd(s, dtype))) return 0;
    return nerf_gated_few_ok(s.m) ? nerf_gated_few_bytes(dtype, s.m, s.k, s.f, s.n) : FwdSpace(s).bytes;
}
int64_t bwd_bytes(const Shape& s, int dtype) { return narrow_bwd(s, dtype) ? nerf_gated_narrow_bwd_bytes(dtype, s.m, s.k, s.f, s.n) : BwdSpace(s).bytes; }

constexpr int64_t kMaxRows = 1 << 26, kMaxWidth = 1 << 16;

const char* bad_shape(int dtype, int64_t rows, int64_t n_in, int64_t neurons, int64_t n_out, int act) {
    if (!nerf_dtype_ok(dtype)) return "dtype must be NERF_F32, NERF_F16 or NERF_BF16";
    if (act != NERF_ACT_SILU && act != NERF_ACT_GELU && act != NERF_ACT_RELU) return "activation must be NERF_ACT_SILU, NERF_ACT_GELU or NERF_ACT_RELU";
    if (rows < 0 || rows > kMaxRows || n_in < 1 || n_in > kMaxWidth || neurons < 1 || neurons > kMaxWidth || n_out < 1 || n_out > kMaxWidth)
        return "n_rows must be in [0, 2^26], the widths in [1, 2^16]";
    const int64_t wide = n_in > 2 * neurons ? (n_in > n_out ? n_in : n_out) : (2 * neurons > n_out ? 2 * neurons : n_out);
    if (ceil_div64(rows, 128) * ceil_div64(wide + 64, 128) >= (1 << 23)) return "n_rows times the widest layer is too large for one launch";
    return nullptr;
}

}  // namespace

extern "C" int64_t nerf_gated_mlp_saved_floats(int dtype, int64_t n_rows, int64_t n_in, int64_t n_neurons, int64_t n_out) {
    if (bad_shape(dtype, n_rows, n_in, n_neurons, n_out, NERF_ACT_SILU)) return -1;
    return nerf_gated_narrow_bwd_ok(dtype, n_in, n_neurons, n_out) ? 0 : saved_floats(n_rows, n_neurons);     // (the narrow kernel computes them again)
}

extern "C" int64_t nerf_gated_mlp_fwd_workspace_bytes(int dtype, int64_t n_rows, int64_t n_in, int64_t n_neurons, int64_t n_out) {
    if (bad_shape(dtype, n_rows, n_in, n_neurons, n_out, NERF_ACT_SILU)) return -1;
    return fwd_bytes(Shape(dtype, n_rows, n_in, n_neurons, n_out), dtype, true);
}

extern "C" int64_t nerf_gated_mlp_alone_workspace_bytes(int dtype, int64_t n_rows, int64_t n_in, int64_t n_neurons, int64_t n_out) {
    if (bad_shape(dtype, n_rows, n_in, n_neurons, n_out, NERF_ACT_SILU)) return -1;
    return fwd_bytes(Shape(dtype, n_rows, n_in, n_neurons, n_out), dtype, false);
}

extern "C" int64_t nerf_gated_mlp_bwd_workspace_bytes(int dtype, int64_t n_rows, int64_t n_in, int64_t n_neurons, int64_t n_out) {
    if (bad_shape(dtype, n_rows, n_in, n_neurons, n_out, NERF_ACT_SILU)) return -1;
    return bwd_bytes(Shape(dtype, n_rows, n_in, n_neurons, n_out), dtype);
}

extern "C" int nerf_gated_mlp_fwd(const void* params, const void* x, int dtype, int64_t n_rows, int64_t n_in, int64_t n_neurons,
                                  int64_t n_out, int activation, void* y, float* saved, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
    const char* bad = bad_shape(dtype, n_rows, n_in, n_neurons, n_out, activation);
    NERF_REQUIRE(!bad, bad);
    if (n_rows == 0) return 0;
    const Shape s(dtype, n_rows, n_in, n_neurons, n_out);
    const int64_t need = fwd_bytes(s, dtype, saved != nullptr);
    NERF_REQUIRE(params && x && y && (workspace || need == 0), "null pointer");
    NERF_REQUIRE(nerf_aligned(params, 16) && nerf_aligned(x, 16) && nerf_aligned(workspace, 16), "params, x and workspace must be 16-byte aligned");
    NERF_REQUIRE(workspace_bytes >= need, "workspace too small");
    hipStream_t st = (hipStream_t)stream;
    if (narrow_bwd(s, dtype)) saved = nullptr;
    if (narrow_fwd(s, dtype, saved != nullptr)) return nerf_gated_narrow_fwd(params, x, dtype, s.m, s.k, s.f, s.n, activation, y, st);
    if (nerf_gated_few_ok(s.m)) return nerf_gated_few_fwd(params, x, dtype, s.m, s.k, s.f, s.n, activation, y, saved, workspace, st);
    return by_type(dtype, s.hidden, [&](auto t, auto e, auto p, auto h) {
        typedef decltype(t) T;
        return fwd_typed<T, decltype(e), decltype(p)::value, decltype(h)::value>((const T*)params, (const T*)x, s, activation, (T*)y, saved,
                                                                               (char*)workspace, st);
    });
}

extern "C" int nerf_gated_mlp_bwd(const void* params, const void* x, const void* dy, const float* saved, int dtype, int64_t n_rows,
                                  int64_t n_in, int64_t n_neurons, int64_t n_out, int activation, void* dx, void* dparams,
                                  int dparams_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* bad = bad_shape(dtype, n_rows, n_in, n_neurons, n_out, activation);
    NERF_REQUIRE(!bad, bad);
    NERF_REQUIRE(dparams_dtype == dtype || dparams_dtype == NERF_F32, "dparams_dtype must be dtype or NERF_F32");
    hipStream_t st = (hipStream_t)stream;
    const int64_t count = (2 * n_in + n_out) * n_neurons;
    if (n_rows == 0) {
        if (!dparams) return 0;
        if (dparams_dtype == NERF_F32) fill_zero_kernel<float><<<grid_for(count), 256, 0, st>>>((float*)dparams, count);
        else fill_zero_kernel<uint16_t><<<grid_for(count), 256, 0, st>>>((uint16_t*)dparams, count);
        return nerf_launch_status("nerf_gated_mlp_bwd");
    }
    const Shape s(dtype, n_rows, n_in, n_neurons, n_out);
    NERF_REQUIRE(params && x && dy && workspace && (saved || narrow_bwd(s, dtype)), "null pointer");
    NERF_REQUIRE(nerf_aligned(params, 16) && nerf_aligned(x, 16) && nerf_aligned(dy, 16) && nerf_aligned(workspace, 16),
                 "params, x, dy and workspace must be 16-byte aligned");
    NERF_REQUIRE(workspace_bytes >= bwd_bytes(s, dtype), "workspace too small");
    const int f32 = dparams_dtype == NERF_F32;
    if (narrow_bwd(s, dtype))
        return nerf_gated_narrow_bwd(params, x, dy, dtype, s.m, s.k, s.f, s.n, activation, dx, dparams, f32, workspace, st);
    return by_type(dtype, s.hidden, [&](auto t, auto e, auto p, auto h) {
        typedef decltype(t) T;
        return bwd_typed<T, decltype(e), decltype(p)::value, decltype(h)::value>((const T*)params, (const T*)x, (const T*)dy, saved, s, activation,
                                                                               (T*)dx, dparams, f32, (char*)workspace, st);
    });
}
