// Host part of the row operators: argument checks and the row map.
#include "row_ops.hpp"
#include <algorithm>
#include <vector>

namespace dpx {

// No two index tuples of the view share an element: sorted by stride, each dim steps over all that lies below it.
// (Sufficient, and true of every slice and permutation of a contiguous array.)
static bool no_self_overlap(const dpx_array_view *v)
{
    std::vector<std::pair<int64_t, int64_t>> d;
    for (int k = 0; k < v->nd; ++k) {
        if (v->shape[k] == 0) return true;
        if (v->shape[k] > 1) d.push_back({v->strides[k] < 0 ? -v->strides[k] : v->strides[k], v->shape[k]});
    }
    std::sort(d.begin(), d.end());
    int64_t below = 0; // largest offset the dims so far reach
    for (auto &[s, n] : d) {
        if (s <= below) return false;
        below += s * (n - 1);
    }
    return true;
}

static int bad(int status, const char *fn, const std::string &what) { return fail(status, std::string(fn) + ": " + what); }

static int check_one(const char *fn, const char *name, const dpx_array_view *v, uint32_t dtypes, bool output)
{
    if (!view_ok(v)) return bad(DPX_ERR_BAD_ARGUMENT, fn, std::string("malformed array descriptor for ") + name);
    if (!(dtypes & dt_bit(v->dtype)))
        return bad(output ? DPX_ERR_BAD_DTYPE : DPX_ERR_NOT_IMPLEMENTED, fn,
                   std::string(name) + " of type " + dtype_name(v->dtype) + " is not supported here");
    if (output && !(v->flags & DPX_WRITABLE)) return bad(DPX_ERR_NOT_WRITABLE, fn, std::string(name) + " is read-only");
    if (output && !no_self_overlap(v))
        return bad(DPX_ERR_NOT_AMPLE, fn, std::string("Memory addressed by ") + name + " is not sufficiently ample.");
    if (view_size(v) != 0 && !v->data) return bad(DPX_ERR_BAD_ARGUMENT, fn, std::string("null data pointer for ") + name);
    return DPX_OK;
}

int row_validate(const char *fn, int nargs, const RowArg *args, int64_t &rows, int32_t &nd, int64_t *shape,
                 int64_t (*st)[DPX_MAX_ND], char **ptr)
{
    const dpx_array_view *first = args[0].v;
    if (!view_ok(first)) return bad(DPX_ERR_BAD_ARGUMENT, fn, std::string("malformed array descriptor for ") + args[0].name);
    if (first->nd < 1) return bad(DPX_ERR_RANK_MISMATCH, fn, std::string(args[0].name) + " needs at least one dimension");
    const int lead = first->nd - 1;
    rows = 1;
    for (int d = 0; d < lead; ++d) rows *= first->shape[d];
    for (int k = 0; k < nargs; ++k) {
        const RowArg &a = args[k];
        ptr[k] = nullptr;
        if (!a.v) continue;
        if (int rc = check_one(fn, a.name, a.v, a.dtypes, a.output)) return rc;
        const bool wide = a.width != ROW_SCALAR;
        if (a.v->nd != lead + (wide ? 1 : 0))
            return bad(DPX_ERR_RANK_MISMATCH, fn, std::string(a.name) + " has " + std::to_string(a.v->nd) +
                                                      " dimensions, " + std::to_string(lead + (wide ? 1 : 0)) + " are needed");
        for (int d = 0; d < lead; ++d)
            if (a.v->shape[d] != first->shape[d])
                return bad(DPX_ERR_SHAPE_MISMATCH, fn, std::string("the leading dimensions of ") + a.name +
                                                           " differ from those of " + args[0].name);
        if (wide) {
            if (a.v->shape[lead] != a.width)
                return bad(DPX_ERR_SHAPE_MISMATCH, fn, std::string("the last axis of ") + a.name + " has length " +
                                                           std::to_string(a.v->shape[lead]) + ", " +
                                                           std::to_string(a.width) + " is needed");
            if (a.width > 1 && a.v->strides[lead] != 1)
                return bad(DPX_ERR_NOT_IMPLEMENTED, fn, std::string(a.name) + " needs unit stride along its last axis");
        }
        for (int j = 0; j < nargs; ++j) {
            if (j == k || !args[j].v || !a.output || (args[j].output && j > k)) continue;
            if (!view_ok(args[j].v) || !views_overlap(a.v, args[j].v)) continue;
            const bool allowed = ((a.same_as >> j) & 1) && views_same_logical(a.v, args[j].v);
            if (!allowed) return bad(DPX_ERR_OVERLAP, fn, std::string(a.name) + " and " + args[j].name + " overlap in memory");
        }
        ptr[k] = (char *)a.v->data;
    }
    // joint collapse of the row dims (args not given have stride 0)
    std::vector<int64_t> strides((size_t)nargs * DPX_MAX_ND, 0), offsets(nargs, 0);
    auto s = reinterpret_cast<int64_t(*)[DPX_MAX_ND]>(strides.data());
    for (int d = 0; d < lead; ++d) {
        shape[d] = first->shape[d];
        for (int k = 0; k < nargs; ++k) s[k][d] = args[k].v ? args[k].v->strides[d] : 0;
    }
    if (rows > 0x7fffffff) return bad(DPX_ERR_BAD_ARGUMENT, fn, "more than 2147483647 rows");
    if (rows == 0) {
        nd = 0;
        return DPX_OK;
    }
    nd = collapse(lead, nargs, shape, s, offsets.data(), false);
    for (int k = 0; k < nargs; ++k) {
        if (ptr[k]) ptr[k] += offsets[k] * itemsize_of(args[k].v->dtype);
        for (int d = 0; d < nd; ++d) st[k][d] = s[k][d];
    }
    return DPX_OK;
}

int row_vector(const char *fn, const char *name, const dpx_array_view *v, int64_t n, uint32_t dtypes, bool output, char **ptr)
{
    *ptr = nullptr;
    if (!v) return DPX_OK;
    if (int rc = check_one(fn, name, v, dtypes, output)) return rc;
    if (v->nd != 1) return bad(DPX_ERR_RANK_MISMATCH, fn, std::string(name) + " must have one dimension");
    if (v->shape[0] != n)
        return bad(DPX_ERR_SHAPE_MISMATCH, fn, std::string(name) + " has length " + std::to_string(v->shape[0]) + ", " +
                                                   std::to_string(n) + " is needed");
    if (n > 1 && v->strides[0] != 1) return bad(DPX_ERR_NOT_IMPLEMENTED, fn, std::string(name) + " needs unit stride");
    *ptr = (char *)v->data;
    return DPX_OK;
}

int row_disjoint(const char *fn, const dpx_array_view *a, const char *an, const dpx_array_view *b, const char *bn)
{
    if (a && b && views_overlap(a, b)) return bad(DPX_ERR_OVERLAP, fn, std::string(an) + " and " + bn + " overlap in memory");
    return DPX_OK;
}

} // namespace dpx
