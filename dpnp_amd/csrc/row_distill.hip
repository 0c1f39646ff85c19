// Distillation from a teacher's top logits, loss and gradient, over rows of V student logits z and K teacher entries
// (logit t_k, token i_k; an entry whose token lies outside [0, V) is absent):
//
//   p = softmax(t / T) over the entries that are there,  q = softmax(z / T) over the vocabulary
//   loss = T^2 sum_k p_k (log p_k - log q[i_k])            (a term with p_k = 0 is 0; no entries: the loss is 0)
//   d loss / d z[v] = T (q[v] P - sum over k with i_k = v of p_k),   P = sum_k p_k: 1, or 0 where no entry is there
//
// The vocabulary is what costs: the loss reads V logits, the gradient reads and writes V.  Exponentials are taken to base 2,
// relative to the largest logit m as it is: e_v = 2^((z_v - m) c) with c = log2(e) / T, s = sum e_v.  A difference and a product per
// logit; where |m c| is small (form NEAR) one fused multiply-add stands for both, z_v c - M with M = m c rounded, and the factor
// 2^(m c - M) that M's rounding leaves on all of them is taken out of the sum and of the gradient's factor.  Beyond it that
// factor, and then m c itself, leave the type's range, while the differences do not: rows of the type's lowest value have the
// softmax that their differences give.  Statistics and sums are float32 (float64 for float64 logits).
//
// In the logits' own unit the loss is T sum p_k ((t_k - max t) - (z_k - m)) + T^2 P (ln s - ln s_t): a teacher's token that the
// student has masked with the lowest value costs what it should and no infinity.
//
// A block owns a row.  Its logits are read once, HELD packs per thread stay in registers between the sum and the gradient,
// what does not fit is read again while it is still in a cache.  Few long rows are split over blocks that leave (m, s) in the
// caller's workspace, and a second launch joins them.
//
// Measured (rocprofv3): gradient of 2048 x 65536 float16 100 us (5.4 TB/s; its exponentials and the rest of its arithmetic
// take about 50 us of it, which the loads and stores of the other block of the CU hide only in part), of 513 x 100003
// float32 84 us (one row more than two rounds of the 256 CUs; 512 rows 75), loss of 2048 x 131072 float16 87 us (6.2 TB/s;
// with the FAR form 4 more, the gradient 1 to 2 more).
// Tried and not kept: rows that come in while the gradients of the row before go out (persistent blocks, a held pack's
// registers reloaded after its last use: 160 us, the row's state no longer fits the registers); packs held in LDS as well
// (158 us for 513 x 100003); a wave of its own for the teacher's side (a block of 9 waves leaves room for one a CU: 111 us).
#include "row_ops.hpp"
#include <algorithm>

namespace dpx {
namespace {

struct Distill {
    RowMap<6> map; // logits, teacher, tokens, weights, loss, dlogits
    const void *z, *t, *tok, *wt;
    void *loss, *dz;
    void *part; // split rows: [rows][splits] pairs (m, s), then [rows][3 k + 3] values of the teacher's side
    int64_t v, chunk;
    int64_t row0; // first row of the launch
    int32_t k, tok64, splits;
    int32_t table; // gradient: size of the token table
    double temp;
};

DPX_D float pow2(float x) { return __builtin_amdgcn_exp2f(x); }
DPX_D double pow2(double x) { return ::exp2(x); }
DPX_D float ln(float x) { return ::logf(x); }
DPX_D double ln(double x) { return ::log(x); }
DPX_D float fma1(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
DPX_D double fma1(double a, double b, double c) { return __builtin_fma(a, b, c); }
template <class A> DPX_D A neg_inf() { return -(A)__builtin_inff(); }
// (finite for the smallest temperatures too: 0 c is 0)
template <class A> DPX_D A scale_of(const Distill &a)
{
    return (A)__builtin_fmin(1.4426950408889634074 / a.temp, sizeof(A) == 4 ? (double)__FLT_MAX__ : __DBL_MAX__);
}

// Largest logit m and sum of 2^((z - m) c).  While m is -inf (nothing but -inf so far) the exponentials are taken relative
// to 0, which leaves the sum at 0 and lets a NaN through; the maximum itself passes NaN over.
template <class A> struct Soft {
    A m, s;
};
template <class A> DPX_D A anchor(A m) { return m == neg_inf<A>() ? A(0) : m; }
template <class A> DPX_D A far_exp(A x, A m, A c) { return pow2((x - m) * c); }
// 2^(x c - M), M = m c rounded, takes the place of 2^((x - m) c) up to |M| = NEAR_LIMIT: float32's M is off by at most 1 there, so
// the factor 2^(m c - M) between the two stays near 1.  near_factor is its inverse.
// The form is chosen by the row for float32 (BY_ROW), by the temperature for float16, whose largest value is known (a choice by
// the row takes 12 registers more there, which spill: gradient of 4096 x 16000 61 us, not 54); float64 is FAR always, where an
// exponential takes some thirty instructions and one more does not count.
enum Form { NEAR, FAR, BY_ROW };
constexpr float NEAR_LIMIT = 1 << 24;
template <class A> DPX_D bool is_near(A M) { return M >= -NEAR_LIMIT && M <= NEAR_LIMIT; }
template <class A> DPX_D A near_factor(A m, A c, A M) { return pow2(-fma1(m, c, -M)); }
template <class A> DPX_D Soft<A> soft_join(Soft<A> a, Soft<A> b, A c)
{
    const A m = MaxOp{}(a.m, b.m), z = anchor(m);
    return {m, a.s * far_exp(a.m, z, c) + b.s * far_exp(b.m, z, c)};
}
// over G lanes, the result in all of them
template <int G, class A> DPX_D Soft<A> soft_lanes(Soft<A> v, A c)
{
    const A m = lanes_fold<G>(v.m, MaxOp{});
    return {m, lanes_fold<G>(v.s * far_exp(v.m, anchor(m), c), SumOp{})};
}
// over a block of up to 1024 threads, in two halves around a barrier of the caller's
template <class A> DPX_D void soft_leave(Soft<A> v, A c, Soft<A> *lds)
{
    v = soft_lanes<64>(v, c);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
}
template <int BT, class A> DPX_D Soft<A> soft_collect(const Soft<A> *lds, A c)
{
    constexpr int NW = BT / 64;
    static_assert(NW == 2 || NW == 4 || NW == 8 || NW == 16);
    // every row of 16 lanes reads all waves' values (more than once where there are fewer: the duplicates are left out)
    const int lane = threadIdx.x & 15;
    Soft<A> v = lds[lane & (NW - 1)];
    if (lane >= NW) v.s = 0;
    return soft_lanes<16>(v, c);
}

template <class T, int E> DPX_D acc_of<T> pack_max(const pack<T, E> &v)
{
    using A = acc_of<T>;
    T m = v.v[0];
#pragma unroll
    for (int e = 1; e < E; ++e) m = __builtin_elementwise_max(m, v.v[e]);
    return (A)m;
}
template <class T, int E> DPX_D pack<T, E> pack_max2(pack<T, E> a, const pack<T, E> &b)
{
#pragma unroll
    for (int e = 0; e < E; ++e) a.v[e] = __builtin_elementwise_max(a.v[e], b.v[e]);
    return a;
}
// U packs joined into a running (m, s): one rescaling for all of them
template <Form FORM, class T, int E, int U, class A> DPX_D void soft_take(Soft<A> &r, const pack<T, E> *x, A c)
{
    pack<T, E> top = x[0];
#pragma unroll
    for (int u = 1; u < U; ++u) top = pack_max2(top, x[u]);
    const A m = MaxOp{}(r.m, pack_max(top)), z = anchor(m), M = z * c;
    A s[4] = {0, 0, 0, 0}, f = 1;
    auto add = [&](auto exponential) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) s[(u * E + e) & 3] += exponential((A)x[u].v[e]);
    };
    // (a branch of the whole wave)
    if (FORM == NEAR || (FORM == BY_ROW && __builtin_amdgcn_ballot_w64(!is_near(M)) == 0)) {
        add([&](A v) { return pow2(fma1(v, c, -M)); });
        f = near_factor(z, c, M);
    }
    else add([&](A v) { return far_exp(v, z, c); });
    r.s = fma1((s[0] + s[1]) + (s[2] + s[3]), f, r.s * far_exp(r.m, z, c));
    r.m = m;
}

// A run of n logits: packs that start on a 128-byte line, and the elements before them (fewer than LINE) and behind them
// (fewer than E), which the block's first threads take one each.  Rows of an odd length start anywhere, and a wave's 1 KiB
// of packs then takes one line more and shares it with another wave (512 x 100003 float32: 86 us with packs that are
// aligned to 16 bytes only, 76 us).  The order of a row's sum thus goes by where the row starts in its line.
template <class T, int E> struct Run {
    static constexpr int LINE = 128 / (int)sizeof(T);
    const T *z; // first pack
    int head, packs, rest;
    DPX_D Run(const T *z_, int n)
    {
        const int h = (int)((128 - ((uintptr_t)z_ & 127)) & 127) / (int)sizeof(T);
        head = h < n ? h : n;
        z = z_ + head;
        packs = (n - head) / E;
        rest = (n - head) % E;
    }
    template <bool NT> DPX_D pack<T, E> load(int p) const // -inf beyond the run
    {
        pack<T, E> x;
        if (p < packs) return load_pack<T, E, NT>(z + p * E);
#pragma unroll
        for (int e = 0; e < E; ++e) x.v[e] = (T)(-__builtin_inff());
        return x;
    }
    // thread i's single element, relative to the first pack; none: -1
    DPX_D bool single(int i) const { return i < head || (i >= LINE && i < LINE + rest); }
    DPX_D int single_at(int i) const { return i < LINE ? i - head : packs * E + i - LINE; }
    DPX_D T load_rest(int i) const { return single(i) ? z[single_at(i)] : (T)(-__builtin_inff()); }
    // f(z) of every element of pack p; dz: where the first pack goes
    template <class F> DPX_D void store(T *dz, int p, const pack<T, E> &x, F f) const
    {
        acc_of<T> o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = f(x.v[e]);
        if (p < packs) store_vals<E, true>(dz + p * E, o);
    }
    template <class F> DPX_D void store_rest(T *dz, int i, T x, F f) const
    {
        if (single(i)) dz[single_at(i)] = (T)f(x);
    }
};
template <class T, class A> DPX_D Soft<A> soft_one(Soft<A> r, T x, A c) // one element more
{
    const A m = MaxOp{}(r.m, (A)x), z = anchor(m);
    return {m, r.s * far_exp(r.m, z, c) + far_exp((A)x, z, c)};
}

// ---- the teacher's side of a row, by one wave -----------------------------------------------------------------------------
// p[k] (0 where absent), the student's logit zk[k] at the entry's token and the token itself (-1 where absent); in `sum` the
// mass sum(p) (1, 0 with no entry that counts, or NaN), sum p (t - max t) / 2 and the logarithm of the entries' sum.
// (Halves: the difference of two finite logits may not be finite.)
template <class A> struct TeacherSum {
    A mass, half, lns;
    bool repeats; // some token belongs to several entries
};
// The row's tokens in a hash table in LDS (open addressing, at most a quarter full), which tells those of several entries:
// comparing every entry with all others took a block 8 us for 256 entries and 200 us for 1000 more than this.
constexpr uint32_t FREE = ~0u, REPEATED = 1u << 31;
constexpr int table_size(int k)
{
    int n = 64;
    while (n < 4 * k) n *= 2;
    return n;
}
DPX_D uint32_t table_start(uint32_t token) { return (token * 2654435761u) >> 16; } // (2^32 / the golden ratio)
DPX_D bool table_put(uint32_t *table, int n, uint32_t token) // true: it was there already
{
    for (uint32_t at = table_start(token);; ++at) {
        uint32_t *const slot = table + (at & (uint32_t)(n - 1));
        const uint32_t old = atomicCAS(slot, FREE, token);
        if (old == FREE) return false;
        if ((old & ~REPEATED) == token) {
            atomicOr(slot, REPEATED);
            return true;
        }
    }
}
DPX_D bool table_repeated(const uint32_t *table, int n, uint32_t token) // of a token that is there
{
    for (uint32_t at = table_start(token);; ++at) {
        const uint32_t w = table[at & (uint32_t)(n - 1)];
        if ((w & ~REPEATED) == token) return (w & REPEATED) != 0;
    }
}
template <class A> struct Entry {
    int32_t token; // -1: absent
    A t, z;
};
template <class T, class TT, class A> DPX_D Entry<A> teacher_entry(const Distill &a, int64_t row, int k)
{
    Entry<A> f{-1, 0, 0};
    if (k >= a.k) return f;
    const int64_t to = a.map.template off<2>(row) + k;
    const int64_t token = a.tok64 ? ((const int64_t *)a.tok)[to] : (int64_t)((const int32_t *)a.tok)[to];
    f.t = (A)((const TT *)a.t)[a.map.template off<1>(row) + k];
    if (token >= 0 && token < a.v) {
        f.token = (int32_t)token;
        f.z = (A)((const T *)a.z)[a.map.template off<0>(row) + token];
    }
    return f;
}
template <class T, class TT, bool GRAD, class A>
DPX_D TeacherSum<A> teacher_wave(const Distill &a, int64_t row, A c, Entry<A> first, A *p, A *zk, int32_t *token)
{
    const int lane = threadIdx.x & 63;
    uint32_t *const table = (uint32_t *)(token + a.k);
    if constexpr (GRAD) {
        for (int i = lane; i < a.table; i += 64) table[i] = FREE;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); // (the wave's LDS accesses are done in order)
        __builtin_amdgcn_wave_barrier();
    }
    bool repeats = false;
    Soft<A> s{neg_inf<A>(), 0};
    for (int k = lane; k < a.k; k += 64) {
        const Entry<A> f = k < 64 ? first : teacher_entry<T, TT, A>(a, row, k);
        const bool there = f.token >= 0;
        const A x = there ? f.t : neg_inf<A>();
        token[k] = f.token;
        zk[k] = f.z;
        p[k] = x;
        if constexpr (GRAD)
            if (there) repeats |= table_put(table, a.table, (uint32_t)f.token);
        s = soft_join(s, Soft<A>{x, 1}, c);
    }
    s = soft_lanes<64>(s, c);
    const bool none = s.m == neg_inf<A>() && s.s == 0;
    const A inv = none ? A(0) : A(1) / s.s, m = anchor(s.m);
    A half = 0;
    for (int k = lane; k < a.k; k += 64) {
        const A x = p[k], pk = none ? A(0) : far_exp(x, m, c) * inv;
        p[k] = pk;
        if (pk != 0) half += pk * fma1(x, A(0.5), m * A(-0.5));
    }
    return {none ? A(0) : s.s * inv, lanes_fold<64>(half, SumOp{}), ln(s.s), __builtin_amdgcn_ballot_w64(repeats) != 0};
}
// loss of the row from the student's (m, s): by one wave
template <class A> DPX_D A loss_wave(const Distill &a, Soft<A> q, TeacherSum<A> te, const A *p, const A *zk)
{
    A half = 0;
    for (int k = threadIdx.x & 63; k < a.k; k += 64)
        if (p[k] != 0) half += p[k] * fma1(zk[k], A(0.5), q.m * A(-0.5));
    half = lanes_fold<64>(half, SumOp{});
    // (T^2 may be beyond float32 where the loss is not)
    return te.mass == 0 ? A(0)
                        : (A)(2 * a.temp * (double)(te.half - half) + a.temp * a.temp * (double)(te.mass * (ln(q.s) - te.lns)));
}
// all the weight that entry k's token gets, its own and that of other entries with the same token, in their order
template <class A> DPX_D A token_weight(const Distill &a, bool repeats, const A *p, const int32_t *token, int k)
{
    const int32_t i = token[k];
    if (!repeats || i < 0 || !table_repeated((const uint32_t *)(token + a.k), a.table, (uint32_t)i)) return p[k];
    A sum = 0;
#pragma unroll 8
    for (int j = 0; j < a.k; ++j) sum += token[j] == i ? p[j] : A(0);
    return sum;
}

// ---- a block owns a row -----------------------------------------------------------------------------------------------
// HELD packs per thread stay in registers between the sum and the gradient, the others are read again.  The first wave does
// the teacher's side, whose first entries are sent for before the row.  The gradient is stored densely first, a barrier, then
// the values at the teacher's tokens over it (their logits were read at the start: dz may be z).  A row of weight 0, and
// one without entries, gets zeros whatever its logits are.
template <class T, class TT, int BT, int HELD, bool GRAD, Form FORM>
__global__ __launch_bounds__(BT, HELD > 8 ? 4 : GRAD ? 6 : 8) void distill_row_kernel(Distill a)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T), U = 4;
    static_assert(HELD % U == 0);
    extern __shared__ __attribute__((aligned(16))) char raw[];
    __shared__ Soft<A> waves[BT / 64];
    __shared__ TeacherSum<A> teacher;
    A *p = (A *)raw, *zk = p + a.k;
    int32_t *token = (int32_t *)(zk + a.k);
    const int64_t row = a.row0 + blockIdx.x;
    const int tid = (int)threadIdx.x;
    const A c = scale_of<A>(a);
    const T *z = (const T *)a.z + a.map.template off<0>(row);
    T *dz = GRAD ? (T *)a.dz + a.map.template off<5>(row) : nullptr;
    Entry<A> first{};
    if (tid < 64) first = teacher_entry<T, TT, A>(a, row, tid);
    const Run<T, E> run(z, (int)a.v);
    pack<T, E> held[HELD ? HELD : 1];
#pragma unroll
    for (int j = 0; j < HELD; ++j) held[j] = run.template load<true>(j * BT + tid);
    const T rest = run.load_rest(tid);
    if (tid < 64) {
        const TeacherSum<A> te = teacher_wave<T, TT, GRAD>(a, row, c, first, p, zk, token);
        if (tid == 0) teacher = te;
    }
    const A w = GRAD ? (a.wt ? ((const A *)a.wt)[a.map.template off<3>(row)] : A(1)) : A(0);
    Soft<A> r = soft_one(Soft<A>{neg_inf<A>(), 0}, rest, c);
#pragma unroll
    for (int j = 0; j < HELD; j += U) soft_take<FORM, T, E, U>(r, held + j, c);
    for (int q = HELD * BT + tid; q < run.packs; q += U * BT) {
        pack<T, E> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = run.template load<!GRAD>(q + u * BT);
        soft_take<FORM, T, E, U>(r, x, c);
    }
    soft_leave(r, c, waves);
    __syncthreads();
    const Soft<A> q = soft_collect<BT>(waves, c);
    const TeacherSum<A> te = teacher;
    if (tid >= BT - 64) {
        const A loss = loss_wave(a, q, te, p, zk);
        if (tid == BT - 64) ((A *)a.loss)[a.map.template off<4>(row)] = loss;
    }
    if constexpr (GRAD) {
        const bool zero = __builtin_amdgcn_readfirstlane(te.mass == 0 || w == 0); // (the same in all threads)
        const A coef = (A)a.temp * w, f = coef * (te.mass / q.s), M = q.m * c;
        const bool near = FORM == NEAR || (FORM == BY_ROW && __builtin_amdgcn_readfirstlane(is_near(M)));
        T *to = dz + run.head;
        auto reread = [&](int i, auto grad) {
            for (; i < run.packs; i += U * BT) {
                pack<T, E> x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = run.template load<true>(i + u * BT);
#pragma unroll
                for (int u = 0; u < U; ++u) run.store(to, i + u * BT, x[u], grad);
            }
            run.store_rest(to, tid, rest, grad);
        };
        auto dense = [&](auto grad) {
#pragma unroll
            for (int j = 0; j < HELD; ++j) {
                keep_whole(held[j]); // (or the sum's conversions to float are kept for this loop, two registers for one)
                run.store(to, j * BT + tid, held[j], grad);
            }
            reread(HELD * BT + tid, grad);
        };
        if (zero) dense([](T) { return A(0); });
        else if (near) {
            const A g = f * near_factor(q.m, c, M);
            dense([&](T x) { return g * pow2(fma1((A)x, c, -M)); });
        }
        else {
            auto grad = [&](T x) { return f * far_exp((A)x, q.m, c); };
            if constexpr (FORM == BY_ROW) reread(tid, grad); // (rare: the held packs are let go, which saves the registers)
            else dense(grad);
        }
        __syncthreads();
        for (int k = tid; k < a.k; k += BT)
            if (token[k] >= 0)
                dz[token[k]] = (T)(zero ? A(0) : f * far_exp(zk[k], q.m, c) - coef * token_weight(a, te.repeats, p, token, k));
    }
}

// ---- few long rows: split over blocks -------------------------------------------------------------------------------------------
constexpr int DST_BLOCK = 256;
// the teacher's side of a row in the workspace: its TeacherSum, then p, zk and the tokens' weights
template <class A> DPX_D A *teacher_part(const Distill &a, int64_t row)
{
    return (A *)a.part + a.map.rows * a.splits * 2 + row * (3 * (int64_t)a.k + 3);
}

// first launch: block (row, split) leaves (m, s) of its part; the last split of a row the teacher's side
template <class T, class TT, bool GRAD, Form FORM> __global__ __launch_bounds__(DST_BLOCK) void distill_split_kernel(Distill a)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T), U = 4;
    extern __shared__ __attribute__((aligned(16))) char raw[];
    __shared__ Soft<A> waves[DST_BLOCK / 64];
    __shared__ bool repeats;
    A *p = (A *)raw, *zk = p + a.k;
    int32_t *token = (int32_t *)(zk + a.k);
    const int64_t row = blockIdx.x / (uint32_t)(a.splits + 1);
    const int split = (int)(blockIdx.x - (uint32_t)row * (uint32_t)(a.splits + 1)), tid = (int)threadIdx.x;
    const A c = scale_of<A>(a);
    if (split == a.splits) { // a block of its own
        A *to = teacher_part<A>(a, row);
        if (tid < 64) {
            const TeacherSum<A> te = teacher_wave<T, TT, GRAD>(a, row, c, teacher_entry<T, TT, A>(a, row, tid), p, zk, token);
            if (tid == 0) {
                to[0] = te.mass;
                to[1] = te.half;
                to[2] = te.lns;
                repeats = te.repeats;
            }
        }
        __syncthreads();
        for (int k = tid; k < a.k; k += DST_BLOCK) {
            to[3 + k] = p[k];
            to[3 + a.k + k] = zk[k];
            if constexpr (GRAD) to[3 + 2 * a.k + k] = token_weight(a, repeats, p, token, k);
        }
        return;
    }
    const int begin = (int)(split * a.chunk), end = (int)(begin + a.chunk < a.v ? begin + a.chunk : a.v);
    const T *z = (const T *)a.z + a.map.template off<0>(row) + begin;
    const Run<T, E> run(z, end - begin);
    Soft<A> r = soft_one(Soft<A>{neg_inf<A>(), 0}, run.load_rest(tid), c);
    for (int q = tid; q < run.packs; q += U * DST_BLOCK) {
        pack<T, E> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = run.template load<false>(q + u * DST_BLOCK);
        soft_take<FORM, T, E, U>(r, x, c);
    }
    soft_leave(r, c, waves);
    __syncthreads();
    r = soft_collect<DST_BLOCK>(waves, c);
    if (tid == 0) ((Soft<A> *)a.part)[row * a.splits + split] = r;
}

// a row's (m, s) from its parts, the same in every lane: read by the 64 lanes of a wave, joined by DPP
template <class A> DPX_D Soft<A> soft_row(const Distill &a, int64_t row, A c)
{
    const Soft<A> *p = (const Soft<A> *)a.part + row * a.splits;
    Soft<A> r{neg_inf<A>(), 0};
    for (int k = threadIdx.x & 63; k < a.splits; k += 64) r = soft_join(r, p[k], c);
    return soft_lanes<64>(r, c);
}

// second launch: the loss, and with GRAD the gradient of block (row, split)'s part
template <class T, bool GRAD> __global__ __launch_bounds__(GRAD ? DST_BLOCK : 64) void distill_join_kernel(Distill a)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T), U = 4;
    const int splits = GRAD ? a.splits : 1;
    const int64_t row = blockIdx.x / (uint32_t)splits;
    const int split = (int)(blockIdx.x - (uint32_t)row * (uint32_t)splits), tid = (int)threadIdx.x;
    const A c = scale_of<A>(a);
    const A *te = teacher_part<A>(a, row);
    auto loss = [&](Soft<A> q) {
        if (split != 0 || tid >= 64) return;
        const A l = loss_wave(a, q, TeacherSum<A>{te[0], te[1], te[2], false}, te + 3, te + 3 + a.k);
        if (tid == 0) ((A *)a.loss)[a.map.template off<4>(row)] = l;
    };
    if constexpr (!GRAD) loss(soft_row<A>(a, row, c));
    else {
        // everything that does not wait for the row's sum is sent for before it
        const int begin = (int)(split * a.chunk), end = (int)(begin + a.chunk < a.v ? begin + a.chunk : a.v), n = end - begin;
        T *dz = (T *)a.dz + a.map.template off<5>(row) + begin;
        const Run<T, E> run((const T *)a.z + a.map.template off<0>(row) + begin, n);
        T *const first = dz + run.head;
        pack<T, E> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = run.template load<true>(tid + u * DST_BLOCK);
        const T one = run.load_rest(tid);
        const int64_t to = a.map.template off<2>(row);
        struct Named {
            int64_t at;
            A z, weight;
        };
        auto entry = [&](int k) {
            if (k >= a.k) return Named{-1, 0, 0};
            const int64_t token = a.tok64 ? ((const int64_t *)a.tok)[to + k] : (int64_t)((const int32_t *)a.tok)[to + k];
            return Named{token - begin, te[3 + a.k + k], te[3 + 2 * a.k + k]};
        };
        const Named mine = entry(tid);
        const A w = a.wt ? ((const A *)a.wt)[a.map.template off<3>(row)] : A(1), mass = te[0];
        const Soft<A> q = soft_row<A>(a, row, c);
        const bool zero = mass == 0 || w == 0;
        const A coef = (A)a.temp * w, f = coef * (mass / q.s);
        auto grad = [&](T x) { return zero ? A(0) : f * far_exp((A)x, q.m, c); };
        run.store_rest(first, tid, one, grad);
        for (int i = tid;;) {
#pragma unroll
            for (int u = 0; u < U; ++u) run.store(first, i + u * DST_BLOCK, x[u], grad);
            i += U * DST_BLOCK;
            if (i >= run.packs) break;
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = run.template load<true>(i + u * DST_BLOCK);
        }
        loss(q);
        __syncthreads();
        for (int k = tid; k < a.k; k += DST_BLOCK) {
            const Named t = k < DST_BLOCK ? mine : entry(k);
            if (t.at >= 0 && t.at < n) dz[t.at] = (T)(zero ? A(0) : f * far_exp(t.z, q.m, c) - coef * t.weight);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
constexpr int MAX_K = 2048; // the teacher's entries of a row are held in LDS

struct DistillPlan {
    int splits; // 0: a block per row
    int64_t chunk;
};
// A block per row is one launch and reads a row once, but a few long rows leave most of the card idle; split rows cost two
// launches, about 11 us a call.  A call with a block per row / split rows, us (the two ways cross at about the same
// lengths for float16 and float32):
//                            1 row         64 rows       128 rows         and   1 row         64 rows       128 rows
//   float16  65536 gradient   9.8 / 11.8   13.8 / 15.7   15.7 / 18.4   loss    7.2 / 10.2    8.3 / 10.1    8.5 / 10.3
//            90000           12.9 / 11.8   16.9 / 17.6   16.8 / 21.2           8.2 / 10.0   10.7 / 10.1   11.0 / 11.9
//            98304           13.6 / 11.7   15.7 / 16.1   17.2 / 21.1           8.1 / 10.0   10.8 / 10.1   10.8 / 11.9
//           131072           14.7 / 11.9   16.7 / 15.7   17.8 / 22.3           9.8 / 10.2   13.1 / 10.2   13.5 / 12.6
//   float32  65536           10.3 / 11.8   14.6 / 16.6   16.1 / 23.0           7.1 / 10.0    8.6 / 10.1    9.2 / 11.2
//            90000           14.4 / 11.7   18.4 / 19.9   21.0 / 28.1           9.6 / 10.0   11.0 / 10.2   11.8 / 13.1
//            98304           15.2 / 11.8   18.1 / 18.7   22.0 / 29.3           9.2 / 10.0   10.9 / 10.1   12.0 / 13.6
//           131072           19.6 / 11.9   22.4 / 20.6   29.0 / 37.2          11.5 / 10.1   13.7 / 11.0   15.1 / 16.3
//                            1 row         64 rows                     128 rows      192 rows
//   float64  12288 gradient  13.9 / 12.2   17.7 / 14.0   loss 1 row  7.5 / 10.2, 64 rows 8.9 / 10.4
//            16384 gradient  15.6 / 11.6   17.8 / 15.3                 18.8 / 18.3
//                  loss       9.2 / 10.2   10.0 / 10.6                  9.9 / 11.2
//           131072 gradient  76.1 / 11.7   81.5 / 42.1                 91.6 / 75.3   106 / 115
//                  loss      44.1 / 10.3   46.3 / 21.9                               48.7 / 53.2
DistillPlan distill_plan(int64_t rows, int64_t v, bool is_double, bool grad)
{
    const int64_t cus = device_cus();
    if (v <= (!is_double ? 90112 : grad ? 10240 : 18432)) return {0, v};
    if (rows > (is_double ? cus * 5 / 8 : grad ? cus / 4 : cus / 2)) return {0, v};
    int64_t splits = std::max<int64_t>(1, std::min((cus * 4 + rows - 1) / rows, v / 4096));
    int64_t chunk = (v + splits - 1) / splits;
    chunk = (chunk + 255) / 256 * 256;
    return {(int)((v + chunk - 1) / chunk), chunk};
}
int64_t distill_workspace(const dpx_array_view *z, int64_t k)
{
    if (!view_ok(z) || z->nd < 1 || !row_float(z->dtype) || z->shape[z->nd - 1] == 0) return 0;
    const int64_t v = z->shape[z->nd - 1], rows = view_size(z) / v;
    if (rows == 0) return 0;
    const bool is_double = z->dtype == DPX_DOUBLE; // (one size for the loss alone and with its gradient)
    const int64_t splits = std::max(distill_plan(rows, v, is_double, false).splits, distill_plan(rows, v, is_double, true).splits);
    return splits ? rows * (splits * 2 + 3 * k + 3) * itemsize_of(acc_dtype(z->dtype)) : 0;
}

template <class T, class TT, bool GRAD, Form FORM> int distill_launch(Distill &a, hipStream_t s)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T);
    const size_t lds = (size_t)a.k * (2 * sizeof(A) + 4) + (size_t)a.table * 4;
    if (a.splits == 0) {
        const int64_t packs = (a.v + E - 1) / E;
        using std::integral_constant;
        auto run = [&](auto bt, auto held) {
            in_launches(a.map.rows, 1, bt, [&](int64_t first, int64_t rows) {
                a.row0 = first;
                hipLaunchKernelGGL((distill_row_kernel<T, TT, decltype(bt)::value, decltype(held)::value, GRAD, FORM>),
                                   dim3((unsigned)rows), dim3(bt), lds, s, a);
            });
        };
        if constexpr (FORM == FAR && sizeof(T) == 2) run(integral_constant<int, 512>{}, integral_constant<int, 0>{}); // (rare)
        else if constexpr (GRAD) {
            if (packs <= 512) run(integral_constant<int, 128>{}, integral_constant<int, 4>{});
            else if (packs <= 1024) run(integral_constant<int, 256>{}, integral_constant<int, 4>{});
            else if (packs <= 2048) run(integral_constant<int, 256>{}, integral_constant<int, 8>{});
            else if (packs <= 4096) run(integral_constant<int, 512>{}, integral_constant<int, 8>{});
            else if (packs <= 8192) run(integral_constant<int, 512>{}, integral_constant<int, 16>{});
            else run(integral_constant<int, 1024>{}, integral_constant<int, 16>{});
        }
        // (2048 rows of 131072 float16: 85.2 us with 1024 threads, 87 with 512; 8 rows of 32768 float32: 5.2 and 5.6)
        else if (packs <= 1024) run(integral_constant<int, 256>{}, integral_constant<int, 0>{});
        else if (packs <= 4096) run(integral_constant<int, 512>{}, integral_constant<int, 0>{});
        else run(integral_constant<int, 1024>{}, integral_constant<int, 0>{});
    }
    else {
        hipLaunchKernelGGL((distill_split_kernel<T, TT, GRAD, FORM>), dim3((unsigned)(a.map.rows * (a.splits + 1))), dim3(DST_BLOCK), lds, s, a);
        if constexpr (GRAD) hipLaunchKernelGGL((distill_join_kernel<T, true>), dim3((unsigned)(a.map.rows * a.splits)), dim3(DST_BLOCK), 0, s, a);
        else hipLaunchKernelGGL((distill_join_kernel<T, false>), dim3((unsigned)a.map.rows), dim3(64), 0, s, a);
    }
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
    if (a.v > 0x3fffffff) return fail(DPX_ERR_BAD_ARGUMENT, f + "the last axis of logits is too long");
    if (k > MAX_K) return fail(DPX_ERR_BAD_ARGUMENT, f + "at most " + std::to_string(MAX_K) + " teacher entries per row");
    if (a.map.rows == 0) return DPX_OK;
    const DistillPlan pl = distill_plan(a.map.rows, a.v, dt == DPX_DOUBLE, grad);
    const size_t need = (size_t)distill_workspace(logits, k);
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return fail(DPX_ERR_BAD_ARGUMENT, f + "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed");
    a.z = p[0], a.t = p[1], a.tok = p[2], a.wt = p[3], a.loss = p[4], a.dz = p[5];
    a.part = workspace;
    a.chunk = pl.chunk, a.splits = pl.splits, a.k = (int32_t)k, a.tok64 = tokens->dtype == DPX_INT64, a.temp = temperature;
    a.table = grad ? table_size((int)k) : 0;
    auto run = [&](auto t, auto u, auto form) {
        using T = typename decltype(t)::type;
        using TT = typename decltype(u)::type;
        return grad ? distill_launch<T, TT, true, decltype(form)::value>(a, stream)
                    : distill_launch<T, TT, false, decltype(form)::value>(a, stream);
    };
    using std::integral_constant;
    const integral_constant<Form, NEAR> near;
    const integral_constant<Form, FAR> far;
    if (dt == DPX_FLOAT) return run(tag<float>{}, tag<float>{}, integral_constant<Form, BY_ROW>{});
    if (dt == DPX_DOUBLE) return run(tag<double>{}, tag<double>{}, far);
    auto half = [&](auto u) {
        return 65504 * 1.4426950408889634074 / temperature <= NEAR_LIMIT ? run(tag<half_t>{}, u, near) : run(tag<half_t>{}, u, far);
    };
    return teacher->dtype == DPX_HALF ? half(tag<half_t>{}) : half(tag<float>{});
}

} // namespace
} // namespace dpx

using namespace dpx;
extern "C" {
int64_t dpx_distill_topk_workspace(const dpx_array_view *logits, const dpx_array_view *teacher_logits)
{
    if (!view_ok(teacher_logits) || teacher_logits->nd < 1) return 0;
    return distill_workspace(logits, teacher_logits->shape[teacher_logits->nd - 1]);
}
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
