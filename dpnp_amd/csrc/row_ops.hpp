// What the row operators share (layer_norm, distill_topk, process_logits): operators over the last axis of arrays
// whose other dims are rows.  The last axis has unit stride; the rows may lie anywhere (RowMap).  Included by the .hip
// files of the operators; the host part is row_host.cpp.
#pragma once
#include "host.hpp"
#include "types.hpp"
#include <exception>

namespace dpx {

// Element offset of row r in each of NOPS arrays: the row dims after joint collapsing, one dim in nearly every call.
template <int NOPS> struct RowMap {
    int64_t rows;
    int32_t nd;
    int64_t st1[NOPS];                       // nd <= 1: stride of the only dim
    int64_t shape[DPX_MAX_ND];               // nd > 1
    int64_t st[NOPS][DPX_MAX_ND];
    template <int K> DPX_D int64_t off(int64_t r) const
    {
        if (nd <= 1) return r * st1[K];
        int64_t o = 0;
        uint32_t q = (uint32_t)r; // (rows < 2^31, checked on the host: a 64-bit division takes as many registers as a row)
        for (int d = nd - 1; d >= 0; --d) {
            const uint32_t e = (uint32_t)shape[d], t = q / e;
            o += (int64_t)(q - t * e) * st[K][d];
            q = t;
        }
        return o;
    }
};

// statistics, sums and per-row results: float for float16 and float32 data, double for float64
template <class T> using acc_of = std::conditional_t<std::is_same_v<T, double>, double, float>;
constexpr int acc_dtype(int dt) { return dt == DPX_DOUBLE ? DPX_DOUBLE : DPX_FLOAT; }
inline bool row_float(int dt) { return dt == DPX_HALF || dt == DPX_FLOAT || dt == DPX_DOUBLE; }

// ---- host: validation (row_host.cpp) ---------------------------------------------------------------------------------
// One array argument of a row operator.  `v` may be null (not given).  The leading dims are those of the first
// argument's rows (`lead_nd` of them); `width` elements follow along a last axis (width < 0: none).
struct RowArg {
    const char *name;
    const dpx_array_view *v;
    int64_t width;   // extent of the last axis, ROW_SCALAR for a per-row value
    uint32_t dtypes; // bit set of accepted dtype ids
    bool output;
    uint32_t same_as; // outputs: bit set of the arguments it may coincide with exactly (work in place)
};
constexpr int64_t ROW_SCALAR = -1;
constexpr uint32_t dt_bit(int dt) { return 1u << dt; }
// Checks the arguments (args[0] is the array that defines the rows) and fills the row map; ptr[k] receives the address of
// args[k]'s row 0 (null where not given).  DPX_OK with map.rows == 0 for an empty call.
int row_validate(const char *fn, int nargs, const RowArg *args, int64_t &rows, int32_t &nd, int64_t *shape,
                 int64_t (*st)[DPX_MAX_ND], char **ptr);
// a whole 1-d contiguous array of `n` elements (weights): its address, checked
int row_vector(const char *fn, const char *name, const dpx_array_view *v, int64_t n, uint32_t dtypes, bool output,
               char **ptr);
// outputs that are not described by row_validate share no memory with the given views
int row_disjoint(const char *fn, const dpx_array_view *a, const char *an, const dpx_array_view *b, const char *bn);

template <int NOPS>
int row_map(const char *fn, const RowArg (&args)[NOPS], RowMap<NOPS> &m, char *(&ptr)[NOPS])
{
    int64_t st[NOPS][DPX_MAX_ND];
    const int rc = row_validate(fn, NOPS, args, m.rows, m.nd, m.shape, st, ptr);
    if (rc) return rc;
    for (int k = 0; k < NOPS; ++k) {
        m.st1[k] = m.nd == 1 ? st[k][0] : 0;
        for (int d = 0; d < DPX_MAX_ND; ++d) m.st[k][d] = d < m.nd ? st[k][d] : 0;
    }
    return DPX_OK;
}
// A launch holds fewer than 2^32 threads: what needs more blocks is launched in parts.  f(first, count) for `total` things of
// `per` blocks of `threads` threads each.
template <class F> void in_launches(int64_t total, int64_t per, int threads, F &&f)
{
    const int64_t most = 0xffffffff / threads / per;
    for (int64_t first = 0; first < total; first += most) f(first, total - first < most ? total - first : most);
}
// an entry point's body: nothing thrown leaves the library
template <class F> int row_entry(F &&f)
{
    try {
        return f();
    }
    catch (const std::exception &e) {
        return fail(DPX_ERR_HIP, std::string("host failure: ") + e.what());
    }
    catch (...) {
        return fail(DPX_ERR_HIP, "host failure");
    }
}

// ---- device: sums over the lanes that share a row ----------------------------------------------------------------------
// (only for permutations inside a row of 16 lanes: every lane has a source)
template <int CTRL, class A> DPX_D A dpp_get(A v)
{
    constexpr int W = sizeof(A) / 4;
    union {
        A a;
        int w[W];
    } u;
    u.a = v;
#pragma unroll
    for (int i = 0; i < W; ++i) u.w[i] = __builtin_amdgcn_mov_dpp(u.w[i], CTRL, 0xf, 0xf, true);
    return u.a;
}
template <class A> DPX_D A lane_get(A v, int lane)
{
    constexpr int W = sizeof(A) / 4;
    union {
        A a;
        int w[W];
    } u;
    u.a = v;
#pragma unroll
    for (int i = 0; i < W; ++i) u.w[i] = __builtin_amdgcn_readlane(u.w[i], lane);
    return u.a;
}
struct SumOp {
    template <class A> DPX_D A operator()(A a, A b) const { return a + b; }
};
struct MaxOp { // of numbers: a NaN operand gives the other one
    DPX_D float operator()(float a, float b) const { return __builtin_fmaxf(a, b); }
    DPX_D double operator()(double a, double b) const { return __builtin_fmax(a, b); }
};
// op over G neighbouring lanes (8, 16, 32, 64), the result in all of them; all G lanes take part.  Lanes exchange inside a
// row of 16 by DPP (neighbour, pair, mirrored half row, mirrored row: after each step the partners hold equal values, so a
// mirror serves as well as an exclusive-or), the four rows of a wave by lane reads.
template <int G, class Op, class A> DPX_D A lanes_fold(A v, Op op)
{
    static_assert(G == 8 || G == 16 || G == 32 || G == 64);
    v = op(v, dpp_get<0xB1>(v));
    v = op(v, dpp_get<0x4E>(v));
    v = op(v, dpp_get<0x141>(v));
    if constexpr (G >= 16) v = op(v, dpp_get<0x140>(v));
    if constexpr (G == 32) v = op(v, __shfl_xor(v, 16, 64));
    if constexpr (G == 64) v = op(op(lane_get(v, 0), lane_get(v, 16)), op(lane_get(v, 32), lane_get(v, 48)));
    return v;
}

// E elements from p as A: 16-byte packs of the element type (p at any element)
template <int E, bool NT, class T, class A> DPX_D void load_vals(const T *p, A (&out)[E])
{
    constexpr int C = E * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : E;
#pragma unroll
    for (int c = 0; c < E; c += C) {
        const pack<T, C> v = load_pack<T, C, NT>(p + c);
#pragma unroll
        for (int e = 0; e < C; ++e) out[c + e] = (A)v.v[e];
    }
}
template <int E, bool NT, class T, class A> DPX_D void store_vals(T *p, const A (&in)[E])
{
    constexpr int C = E * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : E;
#pragma unroll
    for (int c = 0; c < E; c += C) {
        pack<T, C> v;
#pragma unroll
        for (int e = 0; e < C; ++e) v.v[e] = (T)in[c + e];
        store_pack<T, C, NT>(p + c, v);
    }
}

} // namespace dpx
