// Layer normalisation over the last axis, forward and backward.
//
//   forward    m = mean(x),  s = 1 / sqrt(mean((x - m)^2) + eps),  y = (x - m) s w + b
//   backward   h = (x - m) s,  g = dy w,  dx = s (g - mean(g) - h mean(g h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Both are bound by memory: 2 and 3 rows of traffic.  A row is read once and stays in registers between the statistics
// and the result, so G lanes of a wave or a whole block own it and each lane holds PPL packs of E elements of it.
// float16 and float32 rows are computed in float32, float64 rows in float64; every result is rounded once, at its store.
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
// again with every element skipped: their loads are harmless and nothing is stored for them.
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

DPX_D float row_sqrt(float v) { return __builtin_sqrtf(v); }
DPX_D double row_sqrt(double v) { return __builtin_sqrt(v); }

// Sums over the G lanes of a row: inside a wave by DPP, over the waves of a block through LDS (one barrier; `slot`
// alternates so that the next sum needs none before it writes).
template <int G, int BT, int NV, class A> DPX_D void row_sums(A (&v)[NV], A (*lds)[BT / 64][NV], int slot)
{
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = lanes_fold<(G > 64 ? 64 : G)>(v[i], SumOp{});
    if constexpr (G > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < NV; ++i) lds[slot][wave][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            A s = lds[slot][0][i];
#pragma unroll
            for (int k = 1; k < BT / 64; ++k) s += lds[slot][k][i];
            v[i] = s;
        }
    }
}

// ---- forward -------------------------------------------------------------------------------------------------------
template <class T, class W, int E, int PPL, int G, int BT> __global__ __launch_bounds__(BT) void norm_fwd_kernel(NormFwd a)
{
    using A = acc_of<T>;
    __shared__ A lds[2][BT / 64][1];
    const int li = threadIdx.x % G;
    const int64_t row = (int64_t)blockIdx.x * (BT / G) + threadIdx.x / G;
    if (row >= a.map.rows) return;
    const T *x = (const T *)a.x + a.map.template off<0>(row);
    const int64_t n = a.n;
    A v[PPL][E];
#pragma unroll
    for (int j = 0; j < PPL; ++j) load_vals<E, true>(x + PackAt<E, G>(n, li, j).base, v[j]);
    const PackAt<E, G> last(n, li, PPL - 1); // only a lane's last pack can be partial
    A s[1] = {0};
#pragma unroll
    for (int j = 0; j < PPL; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) s[0] += (j < PPL - 1 || e >= last.skip) ? v[j][e] : A(0);
    row_sums<G, BT>(s, lds, 0);
    const A mean = s[0] / (A)n;
    s[0] = 0;
#pragma unroll
    for (int j = 0; j < PPL; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[j][e] -= mean;
            s[0] += (j < PPL - 1 || e >= last.skip) ? v[j][e] * v[j][e] : A(0);
        }
    row_sums<G, BT>(s, lds, 1);
    const A rstd = A(1) / row_sqrt(s[0] / (A)n + (A)a.eps);
    T *y = (T *)a.y + a.map.template off<1>(row);
#pragma unroll
    for (int j = 0; j < PPL; ++j) {
        const PackAt<E, G> at(n, li, j);
        if (at.skip >= E) continue;
        A w[E], b[E], o[E];
        if (a.w) load_vals<E, false>((const W *)a.w + at.base, w);
        if (a.b) load_vals<E, false>((const W *)a.b + at.base, b);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            o[e] = v[j][e] * rstd;
            if (a.w) o[e] *= w[e];
            if (a.b) o[e] += b[e];
        }
        store_vals<E, true>(y + at.base, o);
    }
    if (li == 0) {
        if (a.mean) ((A *)a.mean)[a.map.template off<2>(row)] = mean;
        if (a.rstd) ((A *)a.rstd)[a.map.template off<3>(row)] = rstd;
    }
}

// Rows too long for a block's registers: a block of 1024 threads reads its row three times (the second and third time
// from the memory-side cache), elements BT apart.
template <class T, class W, int BT> __global__ __launch_bounds__(BT) void norm_fwd_long_kernel(NormFwd a)
{
    using A = acc_of<T>;
    __shared__ A lds[2][BT / 64][1];
    const int64_t row = blockIdx.x, n = a.n;
    const T *x = (const T *)a.x + a.map.template off<0>(row);
    A s[1] = {0};
    for (int64_t i = threadIdx.x; i < n; i += BT) s[0] += (A)x[i];
    row_sums<BT, BT>(s, lds, 0);
    const A mean = s[0] / (A)n;
    s[0] = 0;
    for (int64_t i = threadIdx.x; i < n; i += BT) {
        const A d = (A)x[i] - mean;
        s[0] += d * d;
    }
    row_sums<BT, BT>(s, lds, 1);
    const A rstd = A(1) / row_sqrt(s[0] / (A)n + (A)a.eps);
    T *y = (T *)a.y + a.map.template off<1>(row);
    for (int64_t i = threadIdx.x; i < n; i += BT) {
        A o = ((A)x[i] - mean) * rstd;
        if (a.w) o *= (A)((const W *)a.w)[i];
        if (a.b) o += (A)((const W *)a.b)[i];
        y[i] = (T)o;
    }
    if (threadIdx.x == 0) {
        if (a.mean) ((A *)a.mean)[a.map.template off<2>(row)] = mean;
        if (a.rstd) ((A *)a.rstd)[a.map.template off<3>(row)] = rstd;
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------
struct NormBwd {
    RowMap<5> map; // dy, x, dx, mean, rstd
    const void *dy, *x, *mean, *rstd, *w;
    void *dx;
    void *part; // [blocks][2][n] sums of dw and db, null when they are not asked for
    int64_t n;
};

// A block (or each of its groups of G lanes) walks down the rows, gridDim apart, and keeps its columns' sums for dw and db in
// registers; at the end they go to the block's slice of the workspace, which norm_grad_fold_kernel adds up in block order.
template <class T, class W, int E, int PPL, int G, int BT> __global__ __launch_bounds__(BT) void norm_grad_kernel(NormBwd a)
{
    using A = acc_of<T>;
    constexpr int NG = BT / G;
    __shared__ A lds[2][BT / 64][2];
    extern __shared__ __attribute__((aligned(16))) char cols_raw[]; // NG > 1: [2][n] sums of the block's groups
    const int li = threadIdx.x % G, gi = threadIdx.x / G;
    const int64_t n = a.n, step = (int64_t)gridDim.x * NG;
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
    int slot = 0;
    for (int64_t row = (int64_t)blockIdx.x * NG + gi; row < a.map.rows; row += step, slot ^= 1) {
        const T *dy = (const T *)a.dy + a.map.template off<0>(row), *x = (const T *)a.x + a.map.template off<1>(row);
        const A mean = ((const A *)a.mean)[a.map.template off<3>(row)], rstd = ((const A *)a.rstd)[a.map.template off<4>(row)];
        A g[PPL][E], h[PPL][E];
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            const PackAt<E, G> at(n, li, j);
            load_vals<E, true>(dy + at.base, g[j]);
            load_vals<E, true>(x + at.base, h[j]);
        }
        A s[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < PPL; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool mine = j < PPL - 1 || e >= last.skip;
                h[j][e] = (h[j][e] - mean) * rstd;
                const A d = mine ? g[j][e] : A(0);
                dw[j][e] += d * h[j][e];
                db[j][e] += d;
                g[j][e] *= w[j][e];
                const A gw = mine ? g[j][e] : A(0);
                s[0] += gw;
                s[1] += gw * h[j][e];
            }
        row_sums<G, BT>(s, lds, slot);
        const A c1 = s[0] / (A)n, c2 = s[1] / (A)n;
        T *dx = (T *)a.dx + a.map.template off<2>(row);
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            const PackAt<E, G> at(n, li, j);
            if (at.skip >= E) continue;
            A o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = (g[j][e] - c1 - h[j][e] * c2) * rstd;
            store_vals<E, true>(dx + at.base, o);
        }
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

// Rows too long for registers: two passes over the row, the sums for dw and db kept in the block's slice of the workspace
// (each thread adds to its own elements of it).
template <class T, class W, int BT> __global__ __launch_bounds__(BT) void norm_grad_long_kernel(NormBwd a)
{
    using A = acc_of<T>;
    __shared__ A lds[2][BT / 64][2];
    const int64_t n = a.n;
    A *part = a.part ? (A *)a.part + (int64_t)blockIdx.x * 2 * n : nullptr;
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.map.rows; row += gridDim.x, slot ^= 1) {
        const T *dy = (const T *)a.dy + a.map.template off<0>(row), *x = (const T *)a.x + a.map.template off<1>(row);
        const A mean = ((const A *)a.mean)[a.map.template off<3>(row)], rstd = ((const A *)a.rstd)[a.map.template off<4>(row)];
        const bool first = row == (int64_t)blockIdx.x;
        A s[2] = {0, 0};
        for (int64_t i = threadIdx.x; i < n; i += BT) {
            const A h = ((A)x[i] - mean) * rstd, d = (A)dy[i], g = a.w ? d * (A)((const W *)a.w)[i] : d;
            s[0] += g;
            s[1] += g * h;
            if (part) {
                part[i] = first ? d * h : part[i] + d * h;
                part[n + i] = first ? d : part[n + i] + d;
            }
        }
        row_sums<BT, BT>(s, lds, slot);
        const A c1 = s[0] / (A)n, c2 = s[1] / (A)n;
        T *dx = (T *)a.dx + a.map.template off<2>(row);
        for (int64_t i = threadIdx.x; i < n; i += BT) {
            const A h = ((A)x[i] - mean) * rstd, d = (A)dy[i], g = a.w ? d * (A)((const W *)a.w)[i] : d;
            dx[i] = (T)((g - c1 - h * c2) * rstd);
        }
    }
}

// dw and db: the blocks' sums added up in block order.  64 columns by 16 threads that each take every 16th block.
constexpr int FOLD_COLS = 64, FOLD_ROWS = 16;
template <class W, class A>
__global__ __launch_bounds__(FOLD_COLS *FOLD_ROWS) void norm_grad_fold_kernel(const A *part, int64_t blocks, int64_t n, W *dw, W *db)
{
    __shared__ A lds[FOLD_ROWS][FOLD_COLS];
    const int c = threadIdx.x % FOLD_COLS, r = threadIdx.x / FOLD_COLS;
    const int64_t col = (int64_t)blockIdx.x * FOLD_COLS + c; // over the 2 n columns of dw and db
    A s = 0;
    if (col < 2 * n)
        for (int64_t k = r; k < blocks; k += FOLD_ROWS) s += part[k * 2 * n + col];
    lds[r][c] = s;
    __syncthreads();
    if (r == 0 && col < 2 * n) {
#pragma unroll
        for (int k = 1; k < FOLD_ROWS; ++k) s += lds[k][c];
        if (col < n) dw[col] = (W)s;
        else db[col - n] = (W)s;
    }
}

// ---- dispatch --------------------------------------------------------------------------------------------------------
// Lanes and packs per lane for rows of n elements: the fewest lanes that hold the row, a wave up to 4 packs per lane, then
// blocks of 256, 512 and 1024 threads.  g = 0: the row does not fit.
struct NormShape {
    int e, g, ppl, bt;
};
template <class T> NormShape norm_shape(int64_t n, int max_block_ppl)
{
    constexpr int E = 16 / (int)sizeof(T);
    if (n < E) return {1, 8, 1, 256};
    const int64_t p = (n + E - 1) / E;
    if (p <= 8) return {E, 8, 1, 256};
    if (p <= 16) return {E, 16, 1, 256};
    if (p <= 32) return {E, 32, 1, 256};
    if (p <= 256) return {E, 64, (int)((p + 63) / 64), 256};
    for (int bt : {256, 512, 1024}) {
        const int64_t ppl = (p + bt - 1) / bt;
        if (ppl <= (bt == 1024 ? max_block_ppl : 4)) return {E, bt, (int)ppl, bt};
    }
    return {0, 0, 0, 1024};
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
    DPX_NORM_CASE(E, 3, 64, 256)
    DPX_NORM_CASE(E, 4, 64, 256)
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
    const NormShape sh = norm_shape<T>(a.n, 8);
    const int64_t per = sh.g ? sh.bt / sh.g : 1, grid = (a.map.rows + per - 1) / per;
    if (grid > MAX_GRID) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm: too many rows for one launch");
    auto run = [&](auto e, auto ppl, auto g, auto bt) {
        hipLaunchKernelGGL((norm_fwd_kernel<T, W, decltype(e)::value, decltype(ppl)::value, decltype(g)::value, decltype(bt)::value>),
                           dim3((unsigned)grid), dim3(bt), 0, s, a);
    };
    if (!norm_dispatch<E>(sh, run) && !norm_dispatch_wide<E>(sh, run))
        hipLaunchKernelGGL((norm_fwd_long_kernel<T, W, 1024>), dim3((unsigned)grid), dim3(1024), 0, s, a);
    const hipError_t rc = hipGetLastError();
    return rc == hipSuccess ? DPX_OK : fail_hip(rc, "layer_norm launch");
}

// blocks of the backward kernel
template <class T> int64_t norm_grad_blocks(int64_t rows, int64_t n)
{
    const NormShape sh = norm_shape<T>(n, 0);
    const int64_t per = sh.g ? sh.bt / sh.g : 1, need = (rows + per - 1) / per;
    const int64_t want = (int64_t)device_cus() * (sh.bt <= 256 ? 4 : sh.bt == 512 ? 2 : 1);
    return std::min(need, want);
}

template <class T, class W> int norm_grad_launch(NormBwd &a, void *dw, void *db, hipStream_t s)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T);
    const int64_t blocks = norm_grad_blocks<T>(a.map.rows, a.n);
    if (blocks > 0) {
        const NormShape sh = norm_shape<T>(a.n, 0);
        auto run = [&](auto e, auto ppl, auto g, auto bt) {
            const size_t lds = (a.part && sh.g < sh.bt) ? (size_t)(2 * a.n) * sizeof(A) : 0;
            hipLaunchKernelGGL((norm_grad_kernel<T, W, decltype(e)::value, decltype(ppl)::value, decltype(g)::value, decltype(bt)::value>),
                               dim3((unsigned)blocks), dim3(bt), lds, s, a);
        };
        if (!norm_dispatch<E>(sh, run))
            hipLaunchKernelGGL((norm_grad_long_kernel<T, W, 1024>), dim3((unsigned)blocks), dim3(1024), 0, s, a);
    }
    if (dw) {
        const int64_t grid = (2 * a.n + FOLD_COLS - 1) / FOLD_COLS;
        if (grid > MAX_GRID) return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: rows too long");
        hipLaunchKernelGGL((norm_grad_fold_kernel<W, A>), dim3((unsigned)grid), dim3(FOLD_COLS * FOLD_ROWS), 0, s, (const A *)a.part,
                           blocks, a.n, (W *)dw, (W *)db);
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

int64_t grad_blocks(int dt, int64_t rows, int64_t n)
{
    return dt == DPX_HALF ? norm_grad_blocks<half_t>(rows, n) : dt == DPX_FLOAT ? norm_grad_blocks<float>(rows, n) : norm_grad_blocks<double>(rows, n);
}
int64_t grad_workspace(const dpx_array_view *x)
{
    if (!view_ok(x) || x->nd < 1 || !row_float(x->dtype)) return 0;
    const int64_t n = last_extent(x);
    if (n == 0) return 0;
    return grad_blocks(x->dtype, view_size(x) / n, n) * 2 * n * itemsize_of(acc_dtype(x->dtype));
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
    a.part = nullptr;
    if (dweight) {
        const size_t need = (size_t)grad_workspace(x);
        if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
            return fail(DPX_ERR_BAD_ARGUMENT, "layer_norm_grad: a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed");
        a.part = workspace;
    }
    return norm_types(x->dtype, wdt, [&](auto t, auto u) {
        if (a.map.rows == 0 && !dweight) return (int)DPX_OK;
        return norm_grad_launch<typename decltype(t)::type, typename decltype(u)::type>(a, dw, db, stream);
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
