// Layer normalisation over the last axis, forward and backward.
//
//   forward    m = mean(x),  s = 1 / sqrt(mean((x - m)^2) + eps),  y = (x - m) s w + b
//   backward   h = (x - m) s,  g = dy w,  dx = s (g - mean(g) - h mean(g h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// The mean of a row far from zero is off by more than its spread allows, so the second sum, over d = x - m with that m, is one
// of d as well as of d^2: c = mean(d) corrects both, mean(d^2) - c^2 is the variance and y = ((x - m) s - c s) w + b.  (A row of
// 5000.3 float32, 3000 long: |y| <= 0.30 without it.)
//
// Both are bound by memory: 2 and 3 rows of traffic.  A row is read once and stays in registers between the statistics
// and the result: G lanes of a wave or a whole block own it, each lane holds PPL packs of E elements of it, and the blocks
// walk down the rows with the next row on its way, so that weights are read (and the backward's column sums kept) in
// registers.  float16 and float32 rows are computed in float32, float64 rows in float64; every result is rounded once, at
// its store.
//
// Measured (rocprofv3): forward of 16384 x 4096 float16 with float32 parameters 48 us (5.6 TB/s; one block per row that
// reads the weights anew 60 us, one wave per row 56), 20011 x 1001 float32 30.5 us (5.3 TB/s: rows off the 16-byte grid);
// backward of 16384 x 4096 float16 80 us + 4.9 for the fold of the column sums (5.0 TB/s), 2049 x 10007 float32 53.5 + 6.6.
// The sum of d beside that of d^2 costs the forward pass about 1 us of the 48 and 4 of the 118 of 1428 x 70000 float16.
// The backward's time does not change with the prefetch distance (0, 1, 2 rows), the threads per row (256 to 1024) or its
// arithmetic (9 against 16 instructions per element): it is what three streams of persistent blocks reach here.
#include "row_ops.hpp"
#include <algorithm>

namespace dpx {
namespace {

struct NormFwd {
    RowMap<4> map; // x, y, mean, rstd
    const void *x, *w, *b;
    void *y, *mean, *rstd;
    int64_t n;
    double eps;
};

// Lane li's j-th pack of a row: packs lie G apart.  A row's last pack is moved back so that it ends with the row (rows
// hold at least E elements); its first `skip` elements belong to the pack before.  Packs beyond the row are that last pack
// again with every element skipped: they add nothing to a sum, and what is stored for skipped elements is what their own lanes
// store there, computed from the same values.
template <int E, int G> struct PackAt {
    int64_t base;
    int skip;
    DPX_D PackAt(int64_t n, int li, int j)
    {
        const int64_t at = ((int64_t)j * G + li) * E;
        base = at + E <= n ? at : n - E;
        const int64_t s = at - base;
        skip = s > E ? E : (int)s;
    }
};

DPX_D float row_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
DPX_D double row_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }
DPX_D float row_sqrt(float v) { return __builtin_sqrtf(v); }
DPX_D double row_sqrt(double v) { return __builtin_sqrt(v); }

// Sums over the G lanes of a row.  Up to 64 lanes: by DPP.  A block: each row of 16 lanes leaves its sums in LDS, and after a
// barrier every row of 16 lanes reads all of them, BT / 256 per lane, and adds them up by DPP again.  `slot` alternates, so
// that the next sum needs no barrier before it writes.
template <int NV, class A> struct alignas(NV * sizeof(A)) SumPart {
    A v[NV];
};
template <int G, int BT, int NV, class A> DPX_D void row_sums(A (&v)[NV], SumPart<NV, A> (*lds)[BT / 16], int slot)
{
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = lanes_fold<(G > 64 ? 16 : G)>(v[i], SumOp{});
    if constexpr (G > 64) {
        if ((threadIdx.x & 15) == 0) {
            SumPart<NV, A> p;
#pragma unroll
            for (int i = 0; i < NV; ++i) p.v[i] = v[i];
            lds[slot][threadIdx.x >> 4] = p;
        }
        __syncthreads();
        constexpr int PER = BT / 256; // (blocks that share a row have 256 threads or more)
        SumPart<NV, A> p[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) p[k] = lds[slot][(threadIdx.x & 15) * PER + k];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = p[0].v[i];
#pragma unroll
            for (int k = 1; k < PER; ++k) v[i] += p[k].v[i];
            v[i] = lanes_fold<16>(v[i], SumOp{});
        }
    }
}

// ---- forward -------------------------------------------------------------------------------------------------------
// A row's statistics from its rounded mean m and the means of d = x - m and d^2.  A mean(d) of up to four roundings of the
// differences is what their own roundings leave and not the mean's error (that of rows about zero is far smaller): it is left out,
// and so is one that is no number.
template <class A> struct NormStats {
    A mean, shift, rstd, shift_rstd;
    DPX_D NormStats(A m, A d, A dd, A eps) : mean(m)
    {
        constexpr A u4 = sizeof(A) == 4 ? A(0x1p-22) : A(0x1p-51);
        shift = d * d > u4 * u4 * dd ? d : A(0);
        const A v = row_fma(-shift, shift, dd);
        rstd = A(1) / row_sqrt((v < 0 ? A(0) : v) + eps); // (NaN stays)
        shift_rstd = -shift * rstd;
    }
    DPX_D A centred(A x) const { return row_fma(x - mean, rstd, shift_rstd); }
    DPX_D A whole_mean() const { return mean + shift; }
};
template <class T, class W, int E, int PPL, int G, int BT> __global__ __launch_bounds__(BT) void norm_fwd_kernel(NormFwd a)
{
    using A = acc_of<T>;
    __shared__ SumPart<1, A> lds[2][BT / 16];
    __shared__ SumPart<2, A> lds2[2][BT / 16];
    constexpr int NG = BT / G;
    const int li = NG > 1 ? threadIdx.x % G : threadIdx.x, gi = NG > 1 ? threadIdx.x / G : 0; // (one row a block: uniform)
    const int64_t n = a.n, rows = a.map.rows, step = (int64_t)gridDim.x * NG;
    const PackAt<E, G> last(n, li, PPL - 1); // only a lane's last pack can be partial
    const A inv_n = A(1) / (A)n;
    // the weights, and the next row, stay in registers as long as they fit
    constexpr bool HOLD = BT < 1024 || PPL <= (E == 8 ? 3 : 5);
    auto weights = [&](int j, A(&w)[E], A(&b)[E]) {
        const int64_t base = PackAt<E, G>(n, li, j).base;
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = 1, b[e] = 0;
        if (a.w) load_vals<E, false>((const W *)a.w + base, w);
        if (a.b) load_vals<E, false>((const W *)a.b + base, b);
    };
    A w[HOLD ? PPL : 1][E], b[HOLD ? PPL : 1][E];
    if constexpr (HOLD)
#pragma unroll
        for (int j = 0; j < PPL; ++j) weights(j, w[j], b[j]);
    struct Row {
        pack<T, E> x[PPL];
        T *y;
    };
    auto fetch = [&](int64_t row, Row &r) {
        const T *x = (const T *)a.x + a.map.template off<0>(row);
        r.y = (T *)a.y + a.map.template off<1>(row);
#pragma unroll
        for (int j = 0; j < PPL; ++j) r.x[j] = load_pack<T, E>(x + PackAt<E, G>(n, li, j).base);
    };
    int64_t row = (int64_t)blockIdx.x * NG + gi;
    Row r;
    if (row < rows) fetch(row, r);
    int slot = 0;
    for (; row < rows; row += step, slot ^= 1) {
        Row next;
        if constexpr (HOLD) fetch(row + step < rows ? row + step : row, next);
        A s[1] = {0};
#pragma unroll
        for (int j = 0; j < PPL; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) s[0] += (j < PPL - 1 || e >= last.skip) ? (A)r.x[j].v[e] : A(0);
        row_sums<G, BT>(s, lds, slot);
        const A mean = s[0] * inv_n;
        A s2[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < PPL; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const A d = (j < PPL - 1 || e >= last.skip) ? (A)r.x[j].v[e] - mean : A(0);
                s2[0] += d;
                s2[1] = row_fma(d, d, s2[1]);
            }
        row_sums<G, BT>(s2, lds2, slot);
        const NormStats<A> st(mean, s2[0] * inv_n, s2[1] * inv_n, (A)a.eps);
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            A o[E];
            if constexpr (!HOLD) weights(j, w[0], b[0]);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = row_fma(st.centred((A)r.x[j].v[e]), w[HOLD ? j : 0][e], b[HOLD ? j : 0][e]);
            store_vals<E, true>(r.y + PackAt<E, G>(n, li, j).base, o);
        }
        if (li == 0) {
            if (a.mean) ((A *)a.mean)[a.map.template off<2>(row)] = st.whole_mean();
            if (a.rstd) ((A *)a.rstd)[a.map.template off<3>(row)] = st.rstd;
        }
        if constexpr (HOLD) r = next;
        else if (row + step < rows) fetch(row + step, r);
    }
}

// Rows too long for a block's registers: blocks of 1024 threads walk down the rows and read each three times (the second and
// third time from a cache; 1428 x 70000 float16 118 us, element by element 334).
// f(base, skip) for the thread's packs of a row; as in PackAt the last one is moved back.  Only its own elements are stored: a
// row may be worked on in place.
template <int E, int BT, class F> DPX_D void each_pack(int64_t n, F f)
{
#pragma unroll 4
    for (int64_t at = (int64_t)threadIdx.x * E; at < n; at += (int64_t)BT * E) {
        const int64_t base = at + E <= n ? at : n - E;
        f(base, (int)(at - base));
    }
}
template <int E, class T, class A> DPX_D void store_own(T *p, int skip, const A (&o)[E])
{
    if (skip == 0) store_vals<E, true>(p, o);
    else
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e >= skip) p[e] = (T)o[e];
}
template <class T, class W, int BT> __global__ __launch_bounds__(BT) void norm_fwd_long_kernel(NormFwd a)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T);
    __shared__ SumPart<1, A> lds[2][BT / 16];
    __shared__ SumPart<2, A> lds2[2][BT / 16];
    const int64_t n = a.n;
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.map.rows; row += gridDim.x, slot ^= 1) {
        const T *x = (const T *)a.x + a.map.template off<0>(row);
        A s[1] = {0};
        each_pack<E, BT>(n, [&](int64_t at, int skip) {
            const pack<T, E> v = load_pack<T, E, false>(x + at);
#pragma unroll
            for (int e = 0; e < E; ++e) s[0] += e >= skip ? (A)v.v[e] : A(0);
        });
        row_sums<BT, BT>(s, lds, slot);
        const A mean = s[0] / (A)n;
        A s2[2] = {0, 0};
        each_pack<E, BT>(n, [&](int64_t at, int skip) {
            const pack<T, E> v = load_pack<T, E, false>(x + at);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const A d = e >= skip ? (A)v.v[e] - mean : A(0);
                s2[0] += d;
                s2[1] = row_fma(d, d, s2[1]);
            }
        });
        row_sums<BT, BT>(s2, lds2, slot);
        const NormStats<A> st(mean, s2[0] / (A)n, s2[1] / (A)n, (A)a.eps);
        T *y = (T *)a.y + a.map.template off<1>(row);
        each_pack<E, BT>(n, [&](int64_t at, int skip) {
            const pack<T, E> v = load_pack<T, E>(x + at);
            A w[E], b[E], o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = 1, b[e] = 0;
            if (a.w) load_vals<E, false>((const W *)a.w + at, w);
            if (a.b) load_vals<E, false>((const W *)a.b + at, b);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = row_fma(st.centred((A)v.v[e]), w[e], b[e]);
            store_own<E>(y + at, skip, o);
        });
        if (threadIdx.x == 0) {
            if (a.mean) ((A *)a.mean)[a.map.template off<2>(row)] = st.whole_mean();
            if (a.rstd) ((A *)a.rstd)[a.map.template off<3>(row)] = st.rstd;
        }
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------
struct NormBwd {
    RowMap<5> map; // dy, x, dx, mean, rstd
    const void *dy, *x, *mean, *rstd, *w;
    void *dx;
    void *part; // [blocks][2][n] sums of dw and db, null when they are not asked for or made by column blocks
    int64_t n;
    int32_t row_blocks; // the blocks beyond them are column blocks, which write dw and db
    void *dw, *db;
};

// Few rows: columns of dw and db by blocks of their own, in the same launch (the statistics are given, so nothing waits for
// the row blocks).  A lane per column, the block's waves share the rows.
template <class T, class W, int BT> DPX_D void norm_grad_columns(const NormBwd &a, acc_of<T> (*lds)[BT / 64][64])
{
    using A = acc_of<T>;
    constexpr int NW = BT / 64, U = 8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = (int)a.map.rows;
    const int64_t col = (int64_t)(blockIdx.x - (uint32_t)a.row_blocks) * 64 + lane, at = col < a.n ? col : a.n - 1;
    A dw = 0, db = 0;
    for (int row = wave; row < rows; row += NW * U) {
        A d[U], h[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = row + u * NW < rows ? row + u * NW : rows - 1;
            const A mean = ((const A *)a.mean)[a.map.template off<3>(r)], rstd = ((const A *)a.rstd)[a.map.template off<4>(r)];
            d[u] = (A)((const T *)a.dy + a.map.template off<0>(r))[at];
            h[u] = ((A)((const T *)a.x + a.map.template off<1>(r))[at] - mean) * rstd;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row + u * NW < rows) {
                dw = row_fma(d[u], h[u], dw);
                db += d[u];
            }
    }
    lds[0][wave][lane] = dw;
    lds[1][wave][lane] = db;
    __syncthreads();
    if (threadIdx.x < 128) {
        const int which = wave;
        A s = lds[which][0][lane];
#pragma unroll
        for (int k = 1; k < NW; ++k) s += lds[which][k][lane];
        if (col < a.n) ((W *)(which ? a.db : a.dw))[col] = (W)s;
    }
}

// A block (or each of its groups of G lanes) walks down the rows, row_blocks apart, and keeps its columns' sums for dw and db in
// registers; at the end they go to the block's slice of the workspace, which norm_grad_fold_kernel adds up in block order.
// AHEAD: the next row is on its way while this one is worked on.
template <class T, class W, int E, int PPL, int G, int BT, int OCC, bool AHEAD>
__global__ __launch_bounds__(BT, OCC) void norm_grad_kernel(NormBwd a)
{
    using A = acc_of<T>;
    constexpr int NG = BT / G;
    __shared__ SumPart<2, A> lds[2][BT / 16];
    __shared__ A columns[2][BT / 64][64];
    extern __shared__ __attribute__((aligned(16))) char cols_raw[]; // NG > 1: [2][n] sums of the block's groups
    if (blockIdx.x >= (uint32_t)a.row_blocks) {
        norm_grad_columns<T, W, BT>(a, columns);
        return;
    }
    const int li = NG > 1 ? threadIdx.x % G : threadIdx.x, gi = NG > 1 ? threadIdx.x / G : 0; // (one row a block: uniform)
    const int64_t n = a.n, step = (int64_t)a.row_blocks * NG;
    const PackAt<E, G> last(n, li, PPL - 1);
    A w[PPL][E], dw[PPL][E], db[PPL][E];
#pragma unroll
    for (int j = 0; j < PPL; ++j) {
        if (a.w) load_vals<E, false>((const W *)a.w + PackAt<E, G>(n, li, j).base, w[j]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (!a.w) w[j][e] = 1;
            dw[j][e] = db[j][e] = 0;
        }
    }
    struct Row {
        pack<T, E> x[PPL], dy[PPL];
        A mean, rstd;
        T *dx;
    };
    auto fetch = [&](int64_t row, Row &r) {
        const T *dy = (const T *)a.dy + a.map.template off<0>(row), *x = (const T *)a.x + a.map.template off<1>(row);
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            const PackAt<E, G> at(n, li, j);
            r.dy[j] = load_pack<T, E>(dy + at.base);
            r.x[j] = load_pack<T, E>(x + at.base);
        }
        r.dx = (T *)a.dx + a.map.template off<2>(row);
        r.mean = ((const A *)a.mean)[a.map.template off<3>(row)];
        r.rstd = ((const A *)a.rstd)[a.map.template off<4>(row)];
    };
    const A inv_n = A(1) / (A)n;
    const bool tail = __builtin_amdgcn_ballot_w64(last.skip != 0) != 0; // some lane of the wave
    int slot = 0;
    int64_t row = (int64_t)blockIdx.x * NG + gi;
    Row r;
    if (AHEAD && row < a.map.rows) fetch(row, r);
    for (; row < a.map.rows; row += step, slot ^= 1) {
        // (loads and stores are never conditional: the wait for the next row's loads then leaves this row's stores in flight)
        Row next;
        if constexpr (!AHEAD) fetch(row, r);
        else fetch(row + step < a.map.rows ? row + step : row, next);
        auto centred = [&](T x) { return ((A)x - r.mean) * r.rstd; };
        A s[2] = {0, 0};
        pack<T, E> dy_last = r.dy[PPL - 1];
        if (tail) // elements that another lane owns add nothing
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < last.skip) dy_last.v[e] = (T)0;
#pragma unroll
        for (int j = 0; j < PPL; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const A h = centred(r.x[j].v[e]), d = (A)(j < PPL - 1 ? r.dy[j] : dy_last).v[e], g = d * w[j][e];
                dw[j][e] = row_fma(d, h, dw[j][e]);
                db[j][e] += d;
                s[0] += g;
                s[1] = row_fma(g, h, s[1]);
            }
        row_sums<G, BT>(s, lds, slot);
        const A c1 = s[0] * inv_n, c2 = s[1] * inv_n;
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            const PackAt<E, G> at(n, li, j);
            A o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const A g = (A)r.dy[j].v[e] * w[j][e];
                o[e] = row_fma(-centred(r.x[j].v[e]), c2, g - c1) * r.rstd;
            }
            store_vals<E, true>(r.dx + at.base, o); // (a last pack's first elements are also the lane's before: the same values)
        }
        if constexpr (AHEAD) r = next;
    }
    if (!a.part) return;
    A *part = (A *)a.part + (int64_t)blockIdx.x * 2 * n;
    if constexpr (NG > 1) {
        A *cols = (A *)cols_raw;
        for (int k = 0; k < NG; ++k) { // group after group: a fixed order of additions
            if (gi == k) {
#pragma unroll
                for (int j = 0; j < PPL; ++j) {
                    const PackAt<E, G> at(n, li, j);
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (e >= at.skip) {
                            cols[at.base + e] = k ? cols[at.base + e] + dw[j][e] : dw[j][e];
                            cols[n + at.base + e] = k ? cols[n + at.base + e] + db[j][e] : db[j][e];
                        }
                }
            }
            __syncthreads();
        }
        for (int64_t i = threadIdx.x; i < 2 * n; i += BT) part[i] = cols[i];
    }
    else {
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            const PackAt<E, G> at(n, li, j);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e >= at.skip) {
                    part[at.base + e] = dw[j][e];
                    part[n + at.base + e] = db[j][e];
                }
        }
    }
}

// Rows too long for registers.  dx: two passes over a row, the second from a cache.
template <class T, class W, int BT> __global__ __launch_bounds__(BT) void norm_grad_long_kernel(NormBwd a)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T);
    __shared__ SumPart<2, A> lds[2][BT / 16];
    const int64_t n = a.n;
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.map.rows; row += gridDim.x, slot ^= 1) {
        const T *dy = (const T *)a.dy + a.map.template off<0>(row), *x = (const T *)a.x + a.map.template off<1>(row);
        const A mean = ((const A *)a.mean)[a.map.template off<3>(row)], rstd = ((const A *)a.rstd)[a.map.template off<4>(row)];
        // h and g of a pack
        auto both = [&](int64_t at, A(&h)[E], A(&g)[E]) {
            const pack<T, E> vx = load_pack<T, E, false>(x + at), vd = load_pack<T, E, false>(dy + at);
            A w[E];
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = 1;
            if (a.w) load_vals<E, false>((const W *)a.w + at, w);
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = ((A)vx.v[e] - mean) * rstd, g[e] = (A)vd.v[e] * w[e];
        };
        A s[2] = {0, 0};
        each_pack<E, BT>(n, [&](int64_t at, int skip) {
            A h[E], g[E];
            both(at, h, g);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e >= skip) {
                    s[0] += g[e];
                    s[1] = row_fma(g[e], h[e], s[1]);
                }
        });
        row_sums<BT, BT>(s, lds, slot);
        const A c1 = s[0] / (A)n, c2 = s[1] / (A)n;
        T *dx = (T *)a.dx + a.map.template off<2>(row);
        each_pack<E, BT>(n, [&](int64_t at, int skip) {
            A h[E], g[E], o[E];
            both(at, h, g);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = row_fma(-h[e], c2, g[e] - c1) * rstd;
            store_own<E>(dx + at, skip, o);
        });
    }
}
// dw and db of such rows: a second reading, by columns and in a launch before that of dx.  A lane per pack, the block's waves share
// the rows of its split, whose sums go to a slice of the workspace.  (The sums kept in the workspace by the blocks that walk
// down the rows: 842 us a call for 3051 x 32768 float16 instead of 222, 302 for 1525 x 16384 float64 instead of 215.)
template <class T, int BT> __global__ __launch_bounds__(BT) void norm_grad_split_kernel(NormBwd a, int splits, uint32_t block0)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T), NW = BT / 64, U = 4;
    __shared__ A lds[NW][2][E][64];
    const int64_t n = a.n;
    const uint32_t strips = (uint32_t)((n + 64 * E - 1) / (64 * E)), block = block0 + blockIdx.x, split = block / strips;
    const int64_t left = (int64_t)(block - split * strips) * 64 * E;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int begin = (int)(a.map.rows * split / splits), end = (int)(a.map.rows * (split + 1) / splits);
    auto base_of = [&](int l) { return left + (int64_t)l * E + E <= n ? left + (int64_t)l * E : n - E; };
    const int64_t at = base_of(lane);
    A dw[E], db[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0;
    for (int row = begin + wave; row < end; row += NW * U) {
        pack<T, E> d[U], x[U];
        A mean[U], rstd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = row + u * NW < end ? row + u * NW : end - 1;
            d[u] = load_pack<T, E, false>((const T *)a.dy + a.map.template off<0>(r) + at);
            x[u] = load_pack<T, E, false>((const T *)a.x + a.map.template off<1>(r) + at);
            mean[u] = ((const A *)a.mean)[a.map.template off<3>(r)];
            rstd[u] = ((const A *)a.rstd)[a.map.template off<4>(r)];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row + u * NW < end)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    dw[e] = row_fma((A)d[u].v[e], ((A)x[u].v[e] - mean[u]) * rstd[u], dw[e]);
                    db[e] += (A)d[u].v[e];
                }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) lds[wave][0][e][lane] = dw[e], lds[wave][1][e][lane] = db[e];
    __syncthreads();
    A *part = (A *)a.part + (int64_t)split * 2 * n;
    for (int i = threadIdx.x; i < 2 * E * 64; i += BT) {
        const int l = i % 64, e = i / 64 % E, which = i / (64 * E);
        A s = lds[0][which][e][l];
#pragma unroll
        for (int k = 1; k < NW; ++k) s += lds[k][which][e][l];
        const int64_t base = base_of(l);
        if (e >= left + (int64_t)l * E - base) part[which * n + base + e] = s; // (elements moved back belong to the lane before)
    }
}

// dw and db: the blocks' sums added up in a fixed order.  32 columns by 16 threads that each take every 16th block, sixteen
// loads at a time.
constexpr int FOLD_COLS = 32, FOLD_ROWS = 16, FOLD_U = 16;
template <class W, class A>
__global__ __launch_bounds__(FOLD_COLS *FOLD_ROWS) void norm_grad_fold_kernel(const A *part, int64_t blocks, int64_t n, W *dw, W *db,
                                                                                   uint32_t block0)
{
    __shared__ A lds[FOLD_ROWS][FOLD_COLS + 1];
    const int c = threadIdx.x % FOLD_COLS, r = threadIdx.x / FOLD_COLS;
    const int64_t col = (int64_t)(block0 + blockIdx.x) * FOLD_COLS + c; // over the 2 n columns of dw and db
    A s = 0;
    if (col < 2 * n)
        for (int64_t k = r; k < blocks; k += FOLD_ROWS * FOLD_U) {
            A v[FOLD_U];
#pragma unroll
            for (int u = 0; u < FOLD_U; ++u) v[u] = k + u * FOLD_ROWS < blocks ? part[(k + u * FOLD_ROWS) * 2 * n + col] : A(0);
#pragma unroll
            for (int u = 0; u < FOLD_U; ++u) s += v[u];
        }
    lds[r][c] = s;
    __syncthreads();
    if (threadIdx.x < FOLD_COLS && col < 2 * n) {
#pragma unroll
        for (int k = 1; k < FOLD_ROWS; ++k) s += lds[k][c];
        if (col < n) dw[col] = (W)s;
        else db[col - n] = (W)s;
    }
}

// ---- dispatch --------------------------------------------------------------------------------------------------------
// Lanes and packs per lane for rows of n elements: the fewest lanes that hold the row, a wave up to 2 packs per lane, then
// blocks of 256, 512 and 1024 threads.  g = 0: the row does not fit.
struct NormShape {
    int e, g, ppl, bt;
};
template <class T> NormShape norm_shape(int64_t n)
{
    constexpr int E = 16 / (int)sizeof(T);
    if (n < E) return {1, 8, 1, 256};
    const int64_t p = (n + E - 1) / E;
    if (p <= 8) return {E, 8, 1, 256};
    if (p <= 16) return {E, 16, 1, 256};
    if (p <= 32) return {E, 32, 1, 256};
    if (p <= 128) return {E, 64, (int)((p + 63) / 64), 256};
    if (p <= 256) return {E, 256, 1, 256};
    for (int bt : {256, 512, 1024}) {
        const int64_t ppl = (p + bt - 1) / bt;
        if (ppl <= (bt == 1024 ? 8 : 4)) return {E, bt, (int)ppl, bt};
    }
    return {0, 0, 0, 1024};
}

// Blocks per CU: as many as keep about 22 KiB of the next rows on their way.  (More streams worse, fewer leaves latency
// uncovered: 16384 x 4096 float16, 8 KiB a block, 2 / 3 / 4 / 5 / 8 blocks a CU: 50.7 / 46.4 / 47.0 / 49.3 / 51.8 us;
// 20011 x 1001 float32, 4 KiB a block: 44.0 / 34.8 / 30.0 / 29.5 / 31.4.)
inline int norm_per_cu(const NormShape &s)
{
    const int bytes = s.bt * s.ppl * 16;
    return std::max(1, std::min(5, (22 * 1024 + bytes / 2) / std::max(bytes, 1)));
}

// calls f(integral constants E, PPL, G, BT) for a shape of norm_shape
template <int E, class F> bool norm_dispatch(const NormShape &s, F &&f)
{
#define DPX_NORM_CASE(E_, P_, G_, B_)                                                                                          \
    if (s.e == (E_) && s.ppl == (P_) && s.g == (G_)) {                                                                         \
        f(std::integral_constant<int, (E_)>{}, std::integral_constant<int, (P_)>{}, std::integral_constant<int, (G_)>{},       \
          std::integral_constant<int, (B_)>{});                                                                                \
        return true;                                                                                                           \
    }
    DPX_NORM_CASE(1, 1, 8, 256)
    DPX_NORM_CASE(E, 1, 8, 256)
    DPX_NORM_CASE(E, 1, 16, 256)
    DPX_NORM_CASE(E, 1, 32, 256)
    DPX_NORM_CASE(E, 1, 64, 256)
    DPX_NORM_CASE(E, 2, 64, 256)
    DPX_NORM_CASE(E, 1, 256, 256)
    DPX_NORM_CASE(E, 2, 256, 256)
    DPX_NORM_CASE(E, 3, 256, 256)
    DPX_NORM_CASE(E, 4, 256, 256)
    DPX_NORM_CASE(E, 3, 512, 512)
    DPX_NORM_CASE(E, 4, 512, 512)
    return false;
}
template <int E, class F> bool norm_dispatch_wide(const NormShape &s, F &&f)
{
    DPX_NORM_CASE(E, 3, 1024, 1024)
    DPX_NORM_CASE(E, 4, 1024, 1024)
    DPX_NORM_CASE(E, 5, 1024, 1024)
    DPX_NORM_CASE(E, 6, 1024, 1024)
    DPX_NORM_CASE(E, 7, 1024, 1024)
    DPX_NORM_CASE(E, 8, 1024, 1024)
#undef DPX_NORM_CASE
    return false;
}

constexpr int64_t MAX_GRID = 0x7fffffff;

template <class T, class W> int norm_fwd_launch(const NormFwd &a, hipStream_t s)
{
    constexpr int E = 16 / (int)sizeof(T);
    const NormShape sh = norm_shape<T>(a.n);
    const int64_t per = sh.g ? sh.bt / sh.g : 1, grid = std::min<int64_t>((a.map.rows + per - 1) / per, (int64_t)device_cus() * norm_per_cu(sh));
    auto run = [&](auto e, auto ppl, auto g, auto bt) {
        hipLaunchKernelGGL((norm_fwd_kernel<T, W, decltype(e)::value, decltype(ppl)::value, decltype(g)::value, decltype(bt)::value>),
                           dim3((unsigned)grid), dim3(bt), 0, s, a);
    };
    if (!norm_dispatch<E>(sh, run) && !norm_dispatch_wide<E>(sh, run))
        hipLaunchKernelGGL((norm_fwd_long_kernel<T, W, 1024>), dim3((unsigned)grid), dim3(1024), 0, s, a);
    const hipError_t rc = hipGetLastError();
    return rc == hipSuccess ? DPX_OK : fail_hip(rc, "layer_norm launch");
}

// Shapes of the backward kernel: like norm_shape, with fewer packs per lane (a pack of E elements costs 2 E registers for the
// column sums, E for the weights and 16 for the row and the next one), and as many blocks as stay resident.
struct GradShape {
    int e, g, ppl, bt, per_cu;
};
template <class T> GradShape grad_shape(int64_t n)
{
    constexpr int E = 16 / (int)sizeof(T);
    if (n < E) return {1, 8, 1, 256, 4};
    const int64_t p = (n + E - 1) / E;
    if (p <= 8) return {E, 8, 1, 256, 4};
    if (p <= 16) return {E, 16, 1, 256, 4};
    if (p <= 32) return {E, 32, 1, 256, 4};
    if (p <= (E == 8 ? 64 : 128)) return {E, 64, (int)((p + 63) / 64), 256, 4};
    if (p <= 256) return {E, 256, 1, 256, 4};
    if (p <= 512) return {E, 512, 1, 512, 2};
    if (p <= 1024) return E == 4 ? GradShape{E, 512, 2, 512, 2} : GradShape{E, 1024, 1, 1024, 1};
    const int64_t ppl = (p + 511) / 512;
    if (ppl <= (E == 8 ? 4 : 8)) return {E, 512, (int)ppl, 512, 1};
    return {0, 0, 0, 1024, 2};
}
template <int E, class F> bool grad_dispatch(const GradShape &s, F &&f)
{
#define DPX_GRAD_CASE(E_, P_, G_, B_, O_, A_)                                                                                  \
    if (s.e == (E_) && s.ppl == (P_) && s.g == (G_)) {                                                                         \
        f(std::integral_constant<int, (E_)>{}, std::integral_constant<int, (P_)>{}, std::integral_constant<int, (G_)>{},       \
          std::integral_constant<int, (B_)>{}, std::integral_constant<int, (O_)>{}, std::integral_constant<bool, (A_)>{});     \
        return true;                                                                                                           \
    }
    DPX_GRAD_CASE(1, 1, 8, 256, 4, true)
    DPX_GRAD_CASE(E, 1, 8, 256, 4, true)
    DPX_GRAD_CASE(E, 1, 16, 256, 4, true)
    DPX_GRAD_CASE(E, 1, 32, 256, 4, true)
    DPX_GRAD_CASE(E, 1, 64, 256, 4, true)
    if constexpr (E < 8) DPX_GRAD_CASE(E, 2, 64, 256, 4, true)
    DPX_GRAD_CASE(E, 1, 256, 256, 4, true)
    DPX_GRAD_CASE(E, 1, 512, 512, 4, true)
    if constexpr (E == 4) {
        DPX_GRAD_CASE(E, 2, 512, 512, 4, true)
    }
    else {
        DPX_GRAD_CASE(E, 1, 1024, 1024, 4, true)
    }
    DPX_GRAD_CASE(E, 3, 512, 512, 2, E != 8)
    DPX_GRAD_CASE(E, 4, 512, 512, 2, E != 8)
    if constexpr (E < 8) {
        DPX_GRAD_CASE(E, 5, 512, 512, 2, E == 4)
        DPX_GRAD_CASE(E, 6, 512, 512, 2, false)
        DPX_GRAD_CASE(E, 7, 512, 512, 2, false)
        DPX_GRAD_CASE(E, 8, 512, 512, 2, false)
    }
#undef DPX_GRAD_CASE
    return false;
}
template <class T> int64_t norm_grad_blocks(int64_t rows, int64_t n)
{
    const GradShape sh = grad_shape<T>(n);
    const int64_t per = sh.g ? sh.bt / sh.g : 1, need = (rows + per - 1) / per, slots = (int64_t)device_cus() * sh.per_cu;
    if (need <= slots) return need;
    const int64_t turns = (need + slots - 1) / slots; // the fewest blocks that need no more turns: they end together
    return (need + turns - 1) / turns;
}

// Up to this many rows dw and db are made by column blocks, one launch instead of two.  A call with a fold / with column
// blocks, us: float32 1024 columns, 16 rows 11.8 / 9.4, 128 rows 11.9 / 9.3, 256 rows 12.0 / 13.0; 10007 columns, 64 rows 16.6 /
// 10.5, 256 rows 26.7 / 16.5; float16 4096 columns, 128 rows 13.8 / 11.1, 1024 rows 26.6 / 35.3.
constexpr int64_t FEW_ROWS = 128;
template <class T> bool norm_grad_columned(int64_t rows, int64_t n) { return rows > 0 && rows <= FEW_ROWS && grad_shape<T>(n).g; }

// slices of the workspace that a fold adds up
template <class T> int64_t norm_grad_parts(int64_t rows, int64_t n)
{
    if (rows == 0 || norm_grad_columned<T>(rows, n)) return 0;
    if (grad_shape<T>(n).g) return norm_grad_blocks<T>(rows, n);
    const int64_t strips = (n * (int64_t)sizeof(T) + 1023) / 1024; // four blocks a CU, 16 rows or more in each
    return std::max<int64_t>(1, std::min((device_cus() * 4 + strips - 1) / strips, rows / 16));
}

template <class T, class W> int norm_grad_launch(NormBwd &a, hipStream_t s)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T);
    const int64_t blocks = norm_grad_blocks<T>(a.map.rows, a.n);
    const GradShape sh = grad_shape<T>(a.n);
    const bool columns = a.dw && norm_grad_columned<T>(a.map.rows, a.n);
    const int64_t parts = norm_grad_parts<T>(a.map.rows, a.n);
    if (blocks > 0) {
        auto run = [&](auto e, auto ppl, auto g, auto bt, auto occ, auto ahead) {
            const size_t lds = (a.part && sh.g < sh.bt) ? (size_t)(2 * a.n) * sizeof(A) : 0;
            auto launch = [&](int64_t row_blocks, int64_t column_blocks) {
                a.row_blocks = (int32_t)row_blocks;
                hipLaunchKernelGGL((norm_grad_kernel<T, W, decltype(e)::value, decltype(ppl)::value, decltype(g)::value,
                                                     decltype(bt)::value, decltype(occ)::value, decltype(ahead)::value>),
                                   dim3((unsigned)(row_blocks + column_blocks)), dim3(bt), lds, s, a);
            };
            const int64_t column_blocks = columns ? (a.n + 63) / 64 : 0;
            const bool in_place = a.dx == a.dy || a.dx == a.x; // then the columns are read before dx is written
            if (columns && in_place) launch(0, column_blocks);
            launch(blocks, in_place ? 0 : column_blocks);
        };
        if (!grad_dispatch<E>(sh, run)) {
            if (a.dw) {
                const int64_t strips = (a.n + 64 * E - 1) / (64 * E);
                if (strips * parts > MAX_GRID) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: rows too long");
                in_launches(strips * parts, 1, 256, [&](int64_t first, int64_t count) {
                    hipLaunchKernelGGL((norm_grad_split_kernel<T, 256>), dim3((unsigned)count), dim3(256), 0, s, a, (int)parts, (uint32_t)first);
                });
            }
            hipLaunchKernelGGL((norm_grad_long_kernel<T, W, 1024>), dim3((unsigned)blocks), dim3(1024), 0, s, a);
        }
    }
    if (a.dw && !columns) {
        const int64_t fold = (2 * a.n + FOLD_COLS - 1) / FOLD_COLS;
        if (fold > MAX_GRID) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: rows too long");
        in_launches(fold, 1, FOLD_COLS * FOLD_ROWS, [&](int64_t first, int64_t count) {
            hipLaunchKernelGGL((norm_grad_fold_kernel<W, A>), dim3((unsigned)count), dim3(FOLD_COLS * FOLD_ROWS), 0, s,
                               (const A *)a.part, parts, a.n, (W *)a.dw, (W *)a.db, (uint32_t)first);
        });
    }
    const hipError_t rc = hipGetLastError();
    return rc == hipSuccess ? DPX_OK : fail_hip(rc, "layer_norm_grad launch");
}

// element types: (data, parameters)
template <class F> int norm_types(int dt, int wdt, F &&f)
{
    if (dt == DPX_HALF && wdt == DPX_HALF) return f(tag<half_t>{}, tag<half_t>{});
    if (dt == DPX_HALF && wdt == DPX_FLOAT) return f(tag<half_t>{}, tag<float>{});
    if (dt == DPX_FLOAT && wdt == DPX_FLOAT) return f(tag<float>{}, tag<float>{});
    if (dt == DPX_DOUBLE && wdt == DPX_DOUBLE) return f(tag<double>{}, tag<double>{});
    return fail(DPX_ERR_NOT_IMPLEMENTED, std::string("layer_norm: parameters of type ") + dtype_name(wdt) + " for data of type " +
                                             dtype_name(dt) + " are not supported");
}
constexpr uint32_t FLOATS = dt_bit(DPX_HALF) | dt_bit(DPX_FLOAT) | dt_bit(DPX_DOUBLE);
int64_t last_extent(const dpx_array_view *v) { return view_ok(v) && v->nd >= 1 ? v->shape[v->nd - 1] : 0; }

int layer_norm_call(const dpx_array_view *x, const dpx_array_view *weight, const dpx_array_view *bias, double eps,
                    const dpx_array_view *y, const dpx_array_view *mean, const dpx_array_view *rstd, hipStream_t stream)
{
    static const char *fn = "layer_norm";
    if (!view_ok(x)) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm: malformed array descriptor for x");
    if (!y) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm: no output array");
    NormFwd a;
    a.n = last_extent(x);
    a.eps = eps;
    const uint32_t acc = dt_bit(acc_dtype(x->dtype));
    const RowArg args[4] = {{"x", x, a.n, FLOATS, false, 0},
                            {"out", y, a.n, dt_bit(x->dtype), true, 1u},
                            {"mean", mean, ROW_SCALAR, acc, true, 0},
                            {"rstd", rstd, ROW_SCALAR, acc, true, 0}};
    char *p[4], *w, *b;
    if (int rc = row_map<4>(fn, args, a.map, p)) return rc;
    if (a.n == 0) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm: the last axis has no elements");
    if (!(eps >= 0) || eps > 1e300) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm: eps must be a number, zero or more");
    if (int rc = row_vector(fn, "weight", weight, a.n, FLOATS, false, &w)) return rc;
    if (int rc = row_vector(fn, "bias", bias, a.n, FLOATS, false, &b)) return rc;
    if (weight && bias && weight->dtype != bias->dtype)
        return fail(DPX_ERR_NOT_IMPLEMENTED, "layer_norm: weight and bias need one type");
    for (const dpx_array_view *o : {y, mean, rstd})
        for (const dpx_array_view *i : {weight, bias})
            if (int rc = row_disjoint(fn, o, "an output", i, "weight or bias")) return rc;
    a.x = p[0], a.y = p[1], a.mean = p[2], a.rstd = p[3], a.w = w, a.b = b;
    const int wdt = weight ? weight->dtype : bias ? bias->dtype : x->dtype;
    return norm_types(x->dtype, wdt, [&](auto t, auto u) {
        if (a.map.rows == 0) return (int)DPX_OK;
        return norm_fwd_launch<typename decltype(t)::type, typename decltype(u)::type>(a, stream);
    });
}

int64_t grad_workspace(const dpx_array_view *x)
{
    if (!view_ok(x) || x->nd < 1 || !row_float(x->dtype)) return 0;
    const int64_t n = last_extent(x);
    if (n == 0) return 0;
    const int64_t rows = view_size(x) / n, parts = x->dtype == DPX_HALF    ? norm_grad_parts<half_t>(rows, n)
                                                   : x->dtype == DPX_FLOAT ? norm_grad_parts<float>(rows, n)
                                                                           : norm_grad_parts<double>(rows, n);
    return parts * 2 * n * itemsize_of(acc_dtype(x->dtype));
}

int layer_norm_grad_call(const dpx_array_view *dy, const dpx_array_view *x, const dpx_array_view *mean, const dpx_array_view *rstd,
                         const dpx_array_view *weight, const dpx_array_view *dx, const dpx_array_view *dweight,
                         const dpx_array_view *dbias, void *workspace, size_t workspace_bytes, hipStream_t stream)
{
    static const char *fn = "layer_norm_grad";
    if (!view_ok(x) || !view_ok(dy)) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: malformed array descriptor");
    if (!mean || !rstd || !dx) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: mean, rstd and dx are needed");
    if ((dweight != nullptr) != (dbias != nullptr))
        return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: dweight and dbias are given together or not at all");
    NormBwd a;
    a.n = last_extent(x);
    const uint32_t acc = dt_bit(acc_dtype(x->dtype));
    const RowArg args[5] = {{"grad", dy, a.n, dt_bit(x->dtype), false, 0},
                            {"x", x, a.n, FLOATS, false, 0},
                            {"dx", dx, a.n, dt_bit(x->dtype), true, 3u},
                            {"mean", mean, ROW_SCALAR, acc, false, 0},
                            {"rstd", rstd, ROW_SCALAR, acc, false, 0}};
    char *p[5], *w, *dw, *db;
    if (int rc = row_map<5>(fn, args, a.map, p)) return rc;
    if (a.n == 0) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: the last axis has no elements");
    if (int rc = row_vector(fn, "weight", weight, a.n, FLOATS, false, &w)) return rc;
    if (int rc = row_vector(fn, "dweight", dweight, a.n, FLOATS, true, &dw)) return rc;
    if (int rc = row_vector(fn, "dbias", dbias, a.n, FLOATS, true, &db)) return rc;
    const int wdt = weight ? weight->dtype : dweight ? dweight->dtype : x->dtype;
    if (dweight && (dweight->dtype != wdt || dbias->dtype != wdt))
        return fail(DPX_ERR_BAD_DTYPE, "layer_norm_grad: dweight and dbias have the type of weight");
    const dpx_array_view *outs[3] = {dx, dweight, dbias}, *ins[5] = {dy, x, mean, rstd, weight};
    static const char *on[3] = {"dx", "dweight", "dbias"}, *in[5] = {"grad", "x", "mean", "rstd", "weight"};
    for (int o = 0; o < 3; ++o) {
        for (int i = o == 0 ? 4 : 0; i < 5; ++i) // (dx against the row arrays: checked above)
            if (int rc = row_disjoint(fn, outs[o], on[o], ins[i], in[i])) return rc;
        for (int q = 0; q < o; ++q)
            if (int rc = row_disjoint(fn, outs[o], on[o], outs[q], on[q])) return rc;
    }
    a.dy = p[0], a.x = p[1], a.dx = p[2], a.mean = p[3], a.rstd = p[4], a.w = w;
    a.part = nullptr, a.dw = dw, a.db = db;
    if (dweight) {
        const size_t need = (size_t)grad_workspace(x);
        if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
            return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed");
        if (need) a.part = workspace;
    }
    return norm_types(x->dtype, wdt, [&](auto t, auto u) {
        if (a.map.rows == 0 && !dweight) return (int)DPX_OK;
        return norm_grad_launch<typename decltype(t)::type, typename decltype(u)::type>(a, stream);
    });
}

} // namespace
} // namespace dpx

using namespace dpx;
extern "C" {
int dpx_layer_norm(const dpx_array_view *x, const dpx_array_view *weight, const dpx_array_view *bias, double eps,
                   const dpx_array_view *y, const dpx_array_view *mean, const dpx_array_view *rstd, void *stream)
{
    return row_entry([&] { return layer_norm_call(x, weight, bias, eps, y, mean, rstd, (hipStream_t)stream); });
}
int64_t dpx_layer_norm_grad_workspace(const dpx_array_view *x) { return grad_workspace(x); }
int dpx_layer_norm_grad(const dpx_array_view *grad, const dpx_array_view *x, const dpx_array_view *mean, const dpx_array_view *rstd,
                        const dpx_array_view *weight, const dpx_array_view *dx, const dpx_array_view *dweight,
                        const dpx_array_view *dbias, void *workspace, size_t workspace_bytes, void *stream)
{
    return row_entry([&] {
        return layer_norm_grad_call(grad, x, mean, rstd, weight, dx, dweight, dbias, workspace, workspace_bytes, (hipStream_t)stream);
    });
}
}
