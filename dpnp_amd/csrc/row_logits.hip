// Logits on their way to a chosen token: penalties for tokens that were there before, biases and a grammar's mask.
// For the logit z of token v in a row, with `said` the number of times v occurs in the row's output tokens:
//
//   z > 0 ? z / repetition : z * repetition      if v is among the row's prompt or output tokens
//   z - frequency * said - presence * [said > 0]
//   z + the sum of the row's biases for v
//   -inf                                         if v's bit in the mask is 0
//
// Bound by memory for a batch (V logits read and written per row), by latency for one sequence.  A block owns CHUNK
// neighbouring tokens of a row.  It scans the row's token lists and counts its own tokens in LDS (integer atomics: the
// counts do not depend on their order), so that no count array of the vocabulary's size exists in memory; then every logit is
// read, changed and written once.  Arithmetic is float32 (float64 for float64 logits).
#include "row_ops.hpp"
#include <algorithm>

namespace dpx {
namespace {

enum { L_Z, L_OUT, L_PROMPT, L_OUTPUT, L_PLEN, L_OLEN, L_REP, L_FREQ, L_PRES, L_BTOK, L_BVAL, L_MASK, L_ARGS };

struct Logits {
    RowMap<L_ARGS> map;
    const void *z, *prompt, *output, *plen, *olen, *rep, *freq, *pres, *btok, *bval, *mask;
    void *out;
    int64_t v;
    int64_t np, no, nb; // entries per row
    int32_t chunks, tok64, btok64;
    double rep0, freq0, pres0; // where no array is given
};

// a token's word in LDS: the count of its occurrences in the output, two bits above
constexpr uint32_t SEEN_PROMPT = 1u << 31, HAS_BIAS = 1u << 30, COUNT = HAS_BIAS - 1;
constexpr int LG_BLOCK = 256;

DPX_D int64_t entry_at(const void *p, int is64, int64_t i)
{
    return is64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}
// entries of a token list that count: the row's length, within the array
DPX_D int64_t entries_of(const void *len, int64_t at, int64_t n)
{
    if (!len) return n;
    const int64_t k = ((const int32_t *)len)[at];
    return k < 0 ? 0 : k < n ? k : n;
}

template <class T, int CHUNK> __global__ __launch_bounds__(LG_BLOCK) void logits_kernel(Logits a)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T);
    __shared__ uint32_t word[CHUNK];
    const int64_t row = blockIdx.x / (uint32_t)a.chunks;
    const int64_t begin = (int64_t)(blockIdx.x - (uint32_t)row * (uint32_t)a.chunks) * CHUNK;
    const int n = (int)(begin + CHUNK < a.v ? CHUNK : a.v - begin);
    for (int i = threadIdx.x * 4; i < CHUNK; i += LG_BLOCK * 4) *(u32x4 *)(word + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    if (a.prompt) {
        const int64_t at = a.map.template off<L_PROMPT>(row), k = entries_of(a.plen, a.map.template off<L_PLEN>(row), a.np);
        for (int64_t i = threadIdx.x; i < k; i += LG_BLOCK) {
            const int64_t t = entry_at(a.prompt, a.tok64, at + i) - begin;
            if (t >= 0 && t < n) atomicOr(&word[t], SEEN_PROMPT);
        }
    }
    if (a.output) {
        const int64_t at = a.map.template off<L_OUTPUT>(row), k = entries_of(a.olen, a.map.template off<L_OLEN>(row), a.no);
        for (int64_t i = threadIdx.x; i < k; i += LG_BLOCK) {
            const int64_t t = entry_at(a.output, a.tok64, at + i) - begin;
            if (t >= 0 && t < n) atomicAdd(&word[t], 1u);
        }
    }
    const int64_t bt = a.btok ? a.map.template off<L_BTOK>(row) : 0, bv = a.btok ? a.map.template off<L_BVAL>(row) : 0;
    if (a.btok)
        for (int64_t i = threadIdx.x; i < a.nb; i += LG_BLOCK) {
            const int64_t t = entry_at(a.btok, a.btok64, bt + i) - begin;
            if (t >= 0 && t < n) atomicOr(&word[t], HAS_BIAS);
        }
    const A rep = a.rep ? (A)((const float *)a.rep)[a.map.template off<L_REP>(row)] : (A)a.rep0;
    const A freq = a.freq ? (A)((const float *)a.freq)[a.map.template off<L_FREQ>(row)] : (A)a.freq0;
    const A pres = a.pres ? (A)((const float *)a.pres)[a.map.template off<L_PRES>(row)] : (A)a.pres0;
    const uint32_t *mask = a.mask ? (const uint32_t *)a.mask + a.map.template off<L_MASK>(row) : nullptr;
    __syncthreads();
    const T *z = (const T *)a.z + a.map.template off<L_Z>(row) + begin;
    T *out = (T *)a.out + a.map.template off<L_OUT>(row) + begin;
    auto change = [&](T z0, int i) -> T {
        const uint32_t w = word[i];
        T r = z0;
        if (w) {
            A x = (A)z0;
            if (w & (SEEN_PROMPT | COUNT)) x = x > 0 ? x / rep : x * rep;
            const uint32_t said = w & COUNT;
            if (said) x = (x - freq * (A)said) - pres;
            if (w & HAS_BIAS) { // the biases of this token added up in their order, then to the logit
                A s = 0;
                for (int64_t k = 0; k < a.nb; ++k)
                    if (entry_at(a.btok, a.btok64, bt + k) == begin + i) s += (A)((const float *)a.bval)[bv + k];
                x += s;
            }
            r = (T)x;
        }
        if (mask && !((mask[(begin + i) >> 5] >> (i & 31)) & 1)) r = (T)(-__builtin_inff());
        return r;
    };
    for (int i = threadIdx.x * E; i < n; i += LG_BLOCK * E) {
        if (i + E <= n) {
            pack<T, E> x = load_pack<T, E>(z + i);
#pragma unroll
            for (int e = 0; e < E; ++e) x.v[e] = change(x.v[e], i + e);
            store_pack<T, E>(out + i, x);
        }
        else
            for (int e = i; e < n; ++e) out[e] = change(z[e], e);
    }
}

constexpr int64_t MAX_GRID = 0x7fffffff;
constexpr int LG_CHUNK = 4096; // a multiple of 32: a chunk starts at a whole word of the mask

template <class T> int logits_launch(Logits &a, hipStream_t s)
{
    a.chunks = (int32_t)((a.v + LG_CHUNK - 1) / LG_CHUNK);
    if (a.map.rows * a.chunks > MAX_GRID) return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: too many rows for one launch");
    hipLaunchKernelGGL((logits_kernel<T, LG_CHUNK>), dim3((unsigned)(a.map.rows * a.chunks)), dim3(LG_BLOCK), 0, s, a);
    const hipError_t rc = hipGetLastError();
    return rc == hipSuccess ? DPX_OK : fail_hip(rc, "process_logits launch");
}

int process_logits_call(const dpx_array_view *logits, const dpx_logits_args *g, const dpx_array_view *out, hipStream_t stream)
{
    static const char *fn = "process_logits";
    if (!g || !out) return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: missing argument");
    if (!view_ok(logits) || logits->nd < 1) return fail(DPX_ERR_RANK_MISMATCH, "process_logits: logits needs at least one dimension");
    for (const dpx_array_view *v : {g->prompt_tokens, g->output_tokens, g->bias_tokens, g->bias_values, g->allowed})
        if (v && (!view_ok(v) || v->nd < 1))
            return fail(DPX_ERR_RANK_MISMATCH, "process_logits: token, bias and mask arrays need a last axis");
    auto last = [](const dpx_array_view *v) { return v ? v->shape[v->nd - 1] : (int64_t)0; };
    Logits a;
    a.v = last(logits);
    a.np = last(g->prompt_tokens), a.no = last(g->output_tokens), a.nb = last(g->bias_tokens);
    const uint32_t floats = dt_bit(DPX_HALF) | dt_bit(DPX_FLOAT) | dt_bit(DPX_DOUBLE), f4 = dt_bit(DPX_FLOAT), i4 = dt_bit(DPX_INT32),
                   ints = i4 | dt_bit(DPX_INT64);
    const RowArg args[L_ARGS] = {{"logits", logits, a.v, floats, false, 0},
                                 {"out", out, a.v, dt_bit(logits->dtype), true, 1u << L_Z},
                                 {"prompt_tokens", g->prompt_tokens, a.np, ints, false, 0},
                                 {"output_tokens", g->output_tokens, a.no, ints, false, 0},
                                 {"prompt_lengths", g->prompt_lengths, ROW_SCALAR, i4, false, 0},
                                 {"output_lengths", g->output_lengths, ROW_SCALAR, i4, false, 0},
                                 {"repetition_penalty", g->repetition, ROW_SCALAR, f4, false, 0},
                                 {"frequency_penalty", g->frequency, ROW_SCALAR, f4, false, 0},
                                 {"presence_penalty", g->presence, ROW_SCALAR, f4, false, 0},
                                 {"bias_tokens", g->bias_tokens, a.nb, ints, false, 0},
                                 {"bias_values", g->bias_values, a.nb, f4, false, 0},
                                 {"allowed", g->allowed, (a.v + 31) / 32, i4 | dt_bit(DPX_UINT32), false, 0}};
    char *p[L_ARGS];
    if (int rc = row_map<L_ARGS>(fn, args, a.map, p)) return rc;
    if ((g->prompt_lengths && !g->prompt_tokens) || (g->output_lengths && !g->output_tokens))
        return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: lengths without tokens");
    if (!g->bias_tokens != !g->bias_values)
        return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: bias_tokens and bias_values are given together or not at all");
    if (g->prompt_tokens && g->output_tokens && g->prompt_tokens->dtype != g->output_tokens->dtype)
        return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: prompt_tokens and output_tokens need one type");
    if (!g->repetition && !(g->repetition_value > 0 && g->repetition_value <= 1e30))
        return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: repetition_penalty must be a positive number");
    for (double v : {g->frequency ? 0.0 : g->frequency_value, g->presence ? 0.0 : g->presence_value})
        if (!(v >= -1e30 && v <= 1e30)) return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: penalties must be finite numbers");
    // a count has 30 bits of its word
    if (a.no > (int64_t)COUNT) return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: output_tokens has too many entries per row");
    if (a.map.rows == 0 || a.v == 0) return DPX_OK;
    a.z = p[L_Z], a.out = p[L_OUT], a.prompt = p[L_PROMPT], a.output = p[L_OUTPUT], a.plen = p[L_PLEN], a.olen = p[L_OLEN];
    a.rep = p[L_REP], a.freq = p[L_FREQ], a.pres = p[L_PRES], a.btok = p[L_BTOK], a.bval = p[L_BVAL], a.mask = p[L_MASK];
    // lists without entries are not there
    if (a.np == 0) a.prompt = a.plen = nullptr;
    if (a.no == 0) a.output = a.olen = nullptr;
    if (a.nb == 0) a.btok = a.bval = nullptr;
    const dpx_array_view *tv = g->prompt_tokens ? g->prompt_tokens : g->output_tokens;
    a.tok64 = tv && tv->dtype == DPX_INT64;
    a.btok64 = g->bias_tokens && g->bias_tokens->dtype == DPX_INT64;
    a.rep0 = g->repetition_value, a.freq0 = g->frequency_value, a.pres0 = g->presence_value;
    if (logits->dtype == DPX_HALF) return logits_launch<half_t>(a, stream);
    if (logits->dtype == DPX_FLOAT) return logits_launch<float>(a, stream);
    return logits_launch<double>(a, stream);
}

} // namespace
} // namespace dpx

using namespace dpx;
extern "C" {
int dpx_process_logits(const dpx_array_view *logits, const dpx_logits_args *args, const dpx_array_view *out, void *stream)
{
    return row_entry([&] { return process_logits_call(logits, args, out, (hipStream_t)stream); });
}
}
