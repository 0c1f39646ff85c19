// Distillation from a teacher's top logits, loss and gradient, over rows of V student logits z and K teacher entries
// (logit t_k, token i_k; an entry whose token lies outside [0, V) is absent):
//
//   p = softmax(t / T) over the entries that are there,  q = softmax(z / T) over the vocabulary
//   loss = T^2 sum_k p_k (log p_k - log q[i_k])            (a term with p_k = 0 is 0; no entries: the loss is 0)
//   d loss / d z[v] = T (q[v] P - sum over k with i_k = v of p_k),   P = sum_k p_k: 1, or 0 where no entry is there
//
// The vocabulary is what costs: the loss reads V logits, the gradient reads and writes V.  One pass keeps a running
// maximum m and s = sum exp((z - m) / T) per thread; rows are split over blocks and joined through partials (m, s) in the
// caller's workspace.  Exponentials are taken of z - m (not of z scaled and shifted in one step, whose rounding grows with
// the logits' common offset).  Statistics and sums are float32 (float64 for float64 logits).
#include "row_ops.hpp"
#include <algorithm>

namespace dpx {
namespace {

struct Distill {
    RowMap<6> map; // logits, teacher, tokens, weights, loss, dlogits
    const void *z, *t, *tok, *wt;
    void *loss, *dz;
    void *part; // [rows][splits] pairs (m, s)
    int64_t v, chunk;
    int32_t k, tok64, splits;
    double temp;
};

// e^((x - m) / T) as 2^((x - m) c), c = log2(e) / T
DPX_D float pow2(float x) { return __builtin_amdgcn_exp2f(x); }
DPX_D double pow2(double x) { return ::exp2(x); }
DPX_D float ln(float x) { return ::logf(x); }
DPX_D double ln(double x) { return ::log(x); }
template <class A> DPX_D A neg_inf() { return -(A)__builtin_inff(); }

// running maximum and sum of exponentials.  While m is -inf (nothing but -inf so far) the exponentials are taken relative
// to 0, which leaves the sum at 0 and lets a NaN through.
template <class A> struct Soft {
    A m, s;
};
template <class A> DPX_D A anchor(A m) { return m == neg_inf<A>() ? A(0) : m; }
template <class A> DPX_D Soft<A> soft_join(Soft<A> a, Soft<A> b, A c)
{
    const A m = MaxOp{}(a.m, b.m), z = anchor(m);
    return {m, a.s * pow2((a.m - z) * c) + b.s * pow2((b.m - z) * c)};
}

// over a block: by DPP inside the waves, then through LDS; the result in every thread
template <int BT, class A> DPX_D Soft<A> soft_block(Soft<A> v, A c, A (*lds)[2])
{
    const A m = lanes_fold<64>(v.m, MaxOp{}), z = anchor(m);
    v.s = lanes_fold<64>(v.s * pow2((v.m - z) * c), SumOp{});
    v.m = m;
    if constexpr (BT > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            lds[wave][0] = v.m;
            lds[wave][1] = v.s;
        }
        __syncthreads();
        A mm = lds[0][0];
#pragma unroll
        for (int k = 1; k < BT / 64; ++k) mm = MaxOp{}(mm, lds[k][0]);
        const A zz = anchor(mm);
        A s = 0;
#pragma unroll
        for (int k = 0; k < BT / 64; ++k) s += lds[k][1] * pow2((lds[k][0] - zz) * c);
        v.m = mm;
        v.s = s;
    }
    return v;
}

// the (m, s) of elements [begin, end) of a row, over a block
template <class T, int BT> DPX_D Soft<acc_of<T>> soft_scan(const T *z, int64_t begin, int64_t end, acc_of<T> c)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T), U = 4;
    Soft<A> r{neg_inf<A>(), 0};
    auto take = [&](const A(&x)[E]) {
        A m = r.m;
#pragma unroll
        for (int e = 0; e < E; ++e) m = MaxOp{}(m, x[e]);
        const A a = anchor(m);
        A s = r.s * pow2((r.m - a) * c);
#pragma unroll
        for (int e = 0; e < E; ++e) s += pow2((x[e] - a) * c);
        r.m = m;
        r.s = s;
    };
    int64_t i = begin + (int64_t)threadIdx.x * E;
    for (; i + (int64_t)(U - 1) * BT * E + E <= end; i += (int64_t)U * BT * E) {
        A x[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) load_vals<E, false>(z + i + (int64_t)u * BT * E, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) take(x[u]);
    }
    for (; i + E <= end; i += (int64_t)BT * E) {
        A x[E];
        load_vals<E, false>(z + i, x);
        take(x);
    }
    if (i < end) { // the range's last, partial pack
        A x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = i + e < end ? (A)z[i + e] : neg_inf<A>();
        take(x);
    }
    return r;
}

DPX_D int64_t token_at(const void *tok, int is64, int64_t i)
{
    return is64 ? ((const int64_t *)tok)[i] : (int64_t)((const int32_t *)tok)[i];
}

// The teacher's distribution of a row: p[k] (0 where absent) and token[k] (-1 where absent) in LDS, by a block; returns
// sum(p): 1, 0 with no entry that counts, or NaN.  ends with a barrier.  log_norm: log p_k = (t_k - m) / T - log_norm.
template <class A> struct Teacher {
    A mass, m, log_norm;
};
template <class TT, int BT, class A>
DPX_D Teacher<A> teacher_row(const Distill &a, int64_t row, A inv_t, A c, A *p, int32_t *token, A (*lds)[2])
{
    const TT *t = (const TT *)a.t + a.map.template off<1>(row);
    const int64_t to = a.map.template off<2>(row);
    Soft<A> s{neg_inf<A>(), 0};
    for (int k = threadIdx.x; k < a.k; k += BT) {
        const int64_t i = token_at(a.tok, a.tok64, to + k);
        const bool there = i >= 0 && i < a.v;
        token[k] = there ? (int32_t)i : -1;
        const A x = there ? (A)t[k] : neg_inf<A>();
        p[k] = x;
        s = soft_join(s, Soft<A>{x, there ? pow2((x - anchor(x)) * c) : A(0)}, c);
    }
    s = soft_block<BT>(s, c, lds);
    const bool none = s.m == neg_inf<A>() && s.s == 0;
    const A inv = none ? A(0) : A(1) / s.s;
    for (int k = threadIdx.x; k < a.k; k += BT) p[k] = none ? A(0) : pow2((p[k] - anchor(s.m)) * c) * inv;
    __syncthreads();
    return {none ? A(0) : s.s * inv, anchor(s.m), ln(s.s)};
}

// loss of a row, in thread 0 (a block; p and token from teacher_row)
template <class T, class TT, int BT, class A>
DPX_D A row_loss(const Distill &a, int64_t row, const T *z, Soft<A> q, const Teacher<A> &te, A inv_t, const A *p, const int32_t *token,
                 A (*lds)[2])
{
    const TT *t = (const TT *)a.t + a.map.template off<1>(row);
    const A lq = ln(q.s);
    A sum = 0;
    for (int k = threadIdx.x; k < a.k; k += BT) {
        const A pk = p[k];
        if (token[k] < 0 || pk == 0) continue;
        const A logp = ((A)t[k] - te.m) * inv_t - te.log_norm;
        const A logq = ((A)z[token[k]] - q.m) * inv_t - lq;
        sum += pk * (logp - logq);
    }
    sum = lanes_fold<64>(sum, SumOp{});
    if constexpr (BT > 64) {
        __syncthreads(); // lds was read by the sum before
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6][0] = sum;
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int k = 0; k < BT / 64; ++k) sum += lds[k][0];
    }
    // a NaN among the teacher's logits makes every p NaN; a row without entries gives 0
    return te.mass == 0 ? A(0) : (A)(a.temp * a.temp) * sum;
}

constexpr int DST_BLOCK = 256;

// partials of every row: block (row, split)
template <class T> __global__ __launch_bounds__(DST_BLOCK) void distill_stats_kernel(Distill a)
{
    using A = acc_of<T>;
    __shared__ A lds[DST_BLOCK / 64][2];
    const int64_t row = blockIdx.x / (uint32_t)a.splits;
    const int split = (int)(blockIdx.x - (uint32_t)row * (uint32_t)a.splits);
    const T *z = (const T *)a.z + a.map.template off<0>(row);
    const int64_t begin = split * a.chunk, end = begin + a.chunk < a.v ? begin + a.chunk : a.v;
    const A c = (A)(1.4426950408889634074 / a.temp);
    const Soft<A> r = soft_block<DST_BLOCK>(soft_scan<T, DST_BLOCK>(z, begin, end, c), c, lds);
    if (threadIdx.x == 0) ((Soft<A> *)a.part)[blockIdx.x] = r;
}

// a row's (m, s) from its partials, joined in split order; the same in every thread
template <class A> DPX_D Soft<A> soft_row(const Distill &a, int64_t row, A c)
{
    const Soft<A> *p = (const Soft<A> *)a.part + row * a.splits;
    Soft<A> r = p[0];
    for (int k = 1; k < a.splits; ++k) r = soft_join(r, p[k], c);
    return r;
}

template <class T, class TT> __global__ __launch_bounds__(DST_BLOCK) void distill_loss_kernel(Distill a)
{
    using A = acc_of<T>;
    extern __shared__ __attribute__((aligned(16))) char raw[];
    __shared__ A lds[DST_BLOCK / 64][2];
    A *p = (A *)raw;
    int32_t *token = (int32_t *)(p + a.k);
    const int64_t row = blockIdx.x;
    const T *z = (const T *)a.z + a.map.template off<0>(row);
    const A c = (A)(1.4426950408889634074 / a.temp), inv_t = (A)(1.0 / a.temp);
    const Teacher<A> te = teacher_row<TT, DST_BLOCK, A>(a, row, inv_t, c, p, token, lds);
    const A loss = row_loss<T, TT, DST_BLOCK>(a, row, z, soft_row<A>(a, row, c), te, inv_t, p, token, lds);
    if (threadIdx.x == 0) ((A *)a.loss)[a.map.template off<4>(row)] = loss;
}

// gradient of one chunk of a row.  The gradients at the teacher's tokens are worked out before anything is stored (dz may be
// z); the dense part is stored first, a barrier, then those few over it.  A row of weight 0, and one without entries, gets
// zeros whatever its logits are.
template <class T, class TT> __global__ __launch_bounds__(DST_BLOCK) void distill_grad_kernel(Distill a)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T);
    extern __shared__ __attribute__((aligned(16))) char raw[];
    __shared__ A lds[DST_BLOCK / 64][2];
    A *p = (A *)raw, *fix = p + a.k; // the teacher's distribution; the gradient at each of its tokens
    int32_t *token = (int32_t *)(fix + a.k);
    const int64_t row = blockIdx.x / (uint32_t)a.splits;
    const int split = (int)(blockIdx.x - (uint32_t)row * (uint32_t)a.splits);
    const T *z = (const T *)a.z + a.map.template off<0>(row);
    T *dz = (T *)a.dz + a.map.template off<5>(row);
    const int64_t begin = split * a.chunk, end = begin + a.chunk < a.v ? begin + a.chunk : a.v;
    const A c = (A)(1.4426950408889634074 / a.temp), inv_t = (A)(1.0 / a.temp);
    const Teacher<A> te = teacher_row<TT, DST_BLOCK, A>(a, row, inv_t, c, p, token, lds);
    const Soft<A> q = soft_row<A>(a, row, c);
    const A w = a.wt ? ((const A *)a.wt)[a.map.template off<3>(row)] : A(1);
    const bool zero = te.mass == 0 || w == 0;
    const A coef = (A)a.temp * w, qs = te.mass / q.s;
    for (int k = threadIdx.x; k < a.k; k += DST_BLOCK) {
        const int32_t i = token[k];
        if (zero || i < begin || i >= end) continue;
        A sum = 0; // all entries with this token, in their order
        for (int j = 0; j < a.k; ++j) sum += token[j] == i ? p[j] : A(0);
        fix[k] = coef * (pow2(((A)z[i] - q.m) * c) * qs - sum);
    }
    __syncthreads();
    for (int64_t i = begin + (int64_t)threadIdx.x * E; i < end; i += (int64_t)DST_BLOCK * E) {
        A x[E];
        if (i + E <= end) {
            load_vals<E, false>(z + i, x);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = zero ? A(0) : coef * (pow2((x[e] - q.m) * c) * qs);
            store_vals<E, true>(dz + i, x);
        }
        else
            for (int64_t e = i; e < end; ++e) dz[e] = zero ? (T)0 : (T)(coef * (pow2(((A)z[e] - q.m) * c) * qs));
    }
    __syncthreads();
    for (int k = threadIdx.x; k < a.k; k += DST_BLOCK)
        if (!zero && token[k] >= begin && token[k] < end) dz[token[k]] = (T)fix[k];
}

// ---- host ------------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_GRID = 0x7fffffff;
constexpr int MAX_K = 2048; // the teacher's entries of a row are held in LDS

struct DistillPlan {
    int splits;
    int64_t chunk;
};
// blocks per row: one where the rows alone fill the CUs four times over, else as many as make 1024 blocks, of 4096 elements
// and more
DistillPlan distill_plan(int64_t rows, int64_t v)
{
    const int64_t want = (int64_t)device_cus() * 4;
    int64_t splits = rows >= want ? 1 : (want + rows - 1) / rows;
    splits = std::max<int64_t>(1, std::min(splits, v / 4096));
    int64_t chunk = (v + splits - 1) / splits;
    chunk = (chunk + 255) / 256 * 256;
    return {(int)((v + chunk - 1) / chunk), chunk};
}
int64_t distill_workspace(const dpx_array_view *z)
{
    if (!view_ok(z) || z->nd < 1 || !row_float(z->dtype) || z->shape[z->nd - 1] == 0) return 0;
    const int64_t v = z->shape[z->nd - 1], rows = view_size(z) / v;
    if (rows == 0) return 0;
    return rows * distill_plan(rows, v).splits * 2 * itemsize_of(acc_dtype(z->dtype));
}

template <class T, class TT> int distill_launch(const Distill &a, hipStream_t s)
{
    using A = acc_of<T>;
    const dim3 all((unsigned)(a.map.rows * a.splits)), rows((unsigned)a.map.rows), block(DST_BLOCK);
    hipLaunchKernelGGL((distill_stats_kernel<T>), all, block, 0, s, a);
    hipLaunchKernelGGL((distill_loss_kernel<T, TT>), rows, block, (size_t)a.k * (sizeof(A) + 4), s, a);
    if (a.dz) hipLaunchKernelGGL((distill_grad_kernel<T, TT>), all, block, (size_t)a.k * (2 * sizeof(A) + 4), s, a);
    const hipError_t rc = hipGetLastError();
    return rc == hipSuccess ? DPX_OK : fail_hip(rc, "distill_topk launch");
}

int distill_call(const char *fn, const dpx_array_view *logits, const dpx_array_view *teacher, const dpx_array_view *tokens,
                 const dpx_array_view *weights, double temperature, const dpx_array_view *loss, const dpx_array_view *dlogits,
                 bool grad, void *workspace, size_t workspace_bytes, hipStream_t stream)
{
    const std::string f = std::string(fn) + ": ";
    if (!view_ok(logits) || logits->nd < 1) return fail(DPX_ERR_RANK_MISMATCH, f + "logits needs at least one dimension");
    if (!view_ok(teacher) || !view_ok(tokens) || !loss || (grad && !dlogits))
        return fail(DPX_ERR_BAD_ARGUMENT, f + "missing array");
    if (teacher->nd < 1 || tokens->nd < 1) return fail(DPX_ERR_RANK_MISMATCH, f + "the teacher's arrays need a last axis");
    Distill a;
    const int dt = logits->dtype, acc = acc_dtype(dt);
    const int64_t k = teacher->shape[teacher->nd - 1];
    a.v = logits->shape[logits->nd - 1];
    const uint32_t floats = dt_bit(DPX_HALF) | dt_bit(DPX_FLOAT) | dt_bit(DPX_DOUBLE);
    const RowArg args[6] = {{"logits", logits, a.v, floats, false, 0},
                            {"teacher_logits", teacher, k, dt_bit(dt) | dt_bit(acc), false, 0},
                            {"teacher_tokens", tokens, k, dt_bit(DPX_INT32) | dt_bit(DPX_INT64), false, 0},
                            {"weights", weights, ROW_SCALAR, dt_bit(acc), false, 0},
                            {"loss", loss, ROW_SCALAR, dt_bit(acc), true, 0},
                            {"dlogits", grad ? dlogits : nullptr, a.v, dt_bit(dt), true, 1u}};
    char *p[6];
    if (int rc = row_map<6>(fn, args, a.map, p)) return rc;
    if (!(temperature > 0) || !(temperature <= 1e30)) return fail(DPX_ERR_BAD_ARGUMENT, f + "temperature must be a positive number");
    if (a.v == 0) return fail(DPX_ERR_BAD_ARGUMENT, f + "the last axis of logits has no elements");
    if (a.v > 0x7fffffff) return fail(DPX_ERR_BAD_ARGUMENT, f + "the last axis of logits is too long");
    if (k > MAX_K) return fail(DPX_ERR_BAD_ARGUMENT, f + "at most " + std::to_string(MAX_K) + " teacher entries per row");
    if (a.map.rows == 0) return DPX_OK;
    const DistillPlan pl = distill_plan(a.map.rows, a.v);
    if (a.map.rows * pl.splits > MAX_GRID) return fail(DPX_ERR_BAD_ARGUMENT, f + "too many rows for one launch");
    const size_t need = (size_t)distill_workspace(logits);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
        return fail(DPX_ERR_BAD_ARGUMENT, f + "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed");
    a.z = p[0], a.t = p[1], a.tok = p[2], a.wt = p[3], a.loss = p[4], a.dz = p[5];
    a.part = workspace;
    a.chunk = pl.chunk, a.splits = pl.splits, a.k = (int32_t)k, a.tok64 = tokens->dtype == DPX_INT64, a.temp = temperature;
    if (dt == DPX_HALF && teacher->dtype == DPX_HALF) return distill_launch<half_t, half_t>(a, stream);
    if (dt == DPX_HALF) return distill_launch<half_t, float>(a, stream);
    if (dt == DPX_FLOAT) return distill_launch<float, float>(a, stream);
    return distill_launch<double, double>(a, stream);
}

} // namespace
} // namespace dpx

using namespace dpx;
extern "C" {
int64_t dpx_distill_topk_workspace(const dpx_array_view *logits) { return distill_workspace(logits); }
int dpx_distill_topk(const dpx_array_view *logits, const dpx_array_view *teacher_logits, const dpx_array_view *teacher_tokens,
                     double temperature, const dpx_array_view *loss, void *workspace, size_t workspace_bytes, void *stream)
{
    return row_entry([&] {
        return distill_call("distill_topk", logits, teacher_logits, teacher_tokens, nullptr, temperature, loss, nullptr, false, workspace,
                            workspace_bytes, (hipStream_t)stream);
    });
}
int dpx_distill_topk_grad(const dpx_array_view *logits, const dpx_array_view *teacher_logits, const dpx_array_view *teacher_tokens,
                          const dpx_array_view *weights, double temperature, const dpx_array_view *loss,
                          const dpx_array_view *dlogits, void *workspace, size_t workspace_bytes, void *stream)
{
    return row_entry([&] {
        return distill_call("distill_topk_grad", logits, teacher_logits, teacher_tokens, weights, temperature, loss, dlogits, true,
                            workspace, workspace_bytes, (hipStream_t)stream);
    });
}
}
