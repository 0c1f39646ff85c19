// Logits on their way to a chosen token: penalties for tokens that were there before, biases and a grammar's mask.
// For the logit z of token v in a row, with `said` the number of times v occurs in the row's output tokens:
//
//   z > 0 ? z / repetition : z * repetition      if v is among the row's prompt or output tokens
//   z - frequency * said - presence * [said > 0]
//   z + the sum of the row's biases for v
//   -inf                                         if v's bit in the mask is 0
//
// Bound by memory for a batch (V logits read and written per row), by latency for one sequence.  No count array of the
// vocabulary's size exists in memory: a block counts the tokens of its part of the vocabulary in LDS (integer atomics: the
// counts do not depend on their order), and every logit is read, changed and written once.  Arithmetic is float32 (float64
// for float64 logits).
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
    int64_t row0;       // first row of the launch
    int64_t np, no, nb; // entries per row
    int32_t steps, groups; // a row's steps (a pack per thread of a block each), and blocks that share them
    int32_t tok64, btok64;
    double rep0, freq0, pres0; // where no array is given
};

// A token's word in LDS: how often the output holds it, whether the prompt does, whether it has a bias.
constexpr uint32_t COUNT = (1u << 30) - 1, SEEN_PROMPT = 1u << 31, HAS_BIAS = 1u << 30;
constexpr int FEW_BIASES = 256; // per row; more of them are added up in a sum per token of the chunk

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

// A row's token list, looked through by a block once per chunk (tokens are below 2^30, entries too: everything is an int).
// HELD packs of 16 bytes per thread are read once and stay in registers; what lies beyond is read again for every chunk.
template <int BT> struct TokenScan {
    static constexpr int HELD = BT >= 512 ? 1 : 2;
    const char *list = nullptr;
    bool is64;
    int k = 0, whole = 0; // entries that count; whole packs of the list (the entries beyond them are read one by one)
    u32x4 raw[HELD];
    int held[4 * HELD];
    // sent for before the row's length is known: the list's extent bounds it
    DPX_D void send(const void *p, int is64_, int64_t at, int64_t extent)
    {
        is64 = is64_ != 0;
#pragma unroll
        for (int h = 0; h < HELD; ++h) raw[h] = u32x4{~0u, ~0u, ~0u, ~0u};
        if (!p) return;
        list = (const char *)p + at * (is64 ? 8 : 4);
        whole = (int)(extent / (is64 ? 2 : 4));
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if ((int)threadIdx.x + h * BT < whole) raw[h] = load_words16<false>(list + ((int)threadIdx.x + h * BT) * 16);
    }
    static constexpr int NONE = 0x7fffffff;
    static DPX_D int narrow(int64_t t) { return t < 0 || t > 0x3fffffff ? NONE : (int)t; }
    DPX_D void arrived(int64_t entries)
    {
        if (!list) return;
        k = (int)entries;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int left = k - ((int)threadIdx.x + h * BT) * (is64 ? 2 : 4);
            int *t = held + 4 * h;
            if (is64) {
                t[0] = narrow((int64_t)(((uint64_t)raw[h][1] << 32) | raw[h][0]));
                t[1] = narrow((int64_t)(((uint64_t)raw[h][3] << 32) | raw[h][2]));
                t[2] = t[3] = NONE;
            }
            else
#pragma unroll
                for (int c = 0; c < 4; ++c) t[c] = narrow((int)raw[h][c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) t[c] = c < left ? t[c] : NONE;
        }
    }
    // calls f(t - begin) for the entries t in [begin, begin + n)
    template <class F> DPX_D void take(int begin, int n, F f) const
    {
        if (!list) return;
        auto one = [&](int token) {
            const uint32_t t = (uint32_t)token - (uint32_t)begin;
            if (t < (uint32_t)n) f((int)t);
        };
#pragma unroll
        for (int c = 0; c < 4 * HELD; ++c) one(held[c]);
        const int packs = whole < HELD * BT ? whole : HELD * BT, c = is64 ? 2 : 4; // what the registers hold
        for (int i = packs * c + (int)threadIdx.x; i < k; i += BT)
            one(narrow(is64 ? ((const int64_t *)list)[i] : (int64_t)((const int32_t *)list)[i]));
    }
};

// A pack's elements whose bit is 0 become -inf: selected by 32-bit words, two float16 at once.
template <class T, int E> DPX_D void keep_allowed(pack<T, E> &x, uint32_t bits)
{
    constexpr int W = E * (int)sizeof(T) / 4;
    union {
        pack<T, E> p;
        uint32_t w[W];
    } u;
    u.p = x;
    auto all = [&](int e) { return (uint32_t)((int32_t)(bits << (31 - e)) >> 31); };
#pragma unroll
    for (int k = 0; k < W; ++k) {
        uint32_t keep, inf;
        if constexpr (sizeof(T) == 2) keep = (all(2 * k) & 0xffffu) | (all(2 * k + 1) & 0xffff0000u), inf = 0xfc00fc00u;
        else if constexpr (sizeof(T) == 4) keep = all(k), inf = 0xff800000u;
        else keep = all(k / 2), inf = k & 1 ? 0xfff00000u : 0u;
        u.w[k] = (u.w[k] & keep) | (inf & ~keep);
    }
    x = u.p;
}

// The sums of a chunk's biases, made by one wave: 64 entries of the row's list at a time, in their order.  A sum lies at its token
// (DENSE), or few sums lie one after the other and a byte per token says where.  Entries of one token among the 64 are found by
// all of them writing their lane to the sum's owner byte: where one does not read itself again, the token's entries are added up
// one after the other, all others at once.  The work goes with the list, whatever is in it, and a token's sum does not depend on
// how the lanes get there.
template <class A, int CHUNK, bool DENSE> struct BiasSums {
    static constexpr int SUMS = DENSE ? CHUNK : FEW_BIASES;
    A sum[SUMS];
    uint8_t owner[SUMS];
    uint8_t at[DENSE ? 4 : CHUNK];
    DPX_D A of(int t) const { return sum[DENSE ? t : at[t]]; }
    static DPX_D void wave_sync() // (a wave's LDS accesses are done in order)
    {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    }
    // lane's entry: token t of the chunk where `in`; `used`: sums so far
    DPX_D void add(uint32_t *word, int lane, bool in, int t, float value, int &used)
    {
        if (__builtin_amdgcn_ballot_w64(in) == 0) return;
        const bool fresh = in && !(atomicOr(&word[t], HAS_BIAS) & HAS_BIAS); // one lane per token that is new
        int k = t;
        if constexpr (!DENSE) {
            const uint64_t who = __builtin_amdgcn_ballot_w64(fresh);
            k = used + __builtin_popcountll(who & (((uint64_t)1 << lane) - 1));
            if (fresh) at[t] = (uint8_t)k;
            used += __builtin_popcountll(who);
        }
        if (fresh) sum[k] = 0;
        wave_sync();
        if (!DENSE && in) k = at[t];
        if (in) owner[k] = (uint8_t)lane;
        wave_sync();
        bool alone = in;
        const bool lost = in && owner[k] != (uint8_t)lane;
        if (__builtin_amdgcn_ballot_w64(lost) != 0) {
            wave_sync();
            if (lost) owner[k] = 255;
            wave_sync();
            alone = in && owner[k] != 255;
            uint64_t todo = __builtin_amdgcn_ballot_w64(in && !alone);
            while (todo) {
                const int first = __builtin_ctzll(todo), sum_k = lane_get(k, first);
                uint64_t same = __builtin_amdgcn_ballot_w64(in && k == sum_k);
                todo &= ~same;
                A s = sum[sum_k];
                for (; same; same &= same - 1) s += (A)lane_get(value, __builtin_ctzll(same));
                if (lane == first) sum[sum_k] = s;
            }
        }
        if (alone) sum[k] += (A)value;
        wave_sync();
    }
};

// A block takes a run of a row's steps, CHUNK neighbouring tokens at a time, the next chunk's logits on their way.  Per chunk
// the lists' tokens are counted in LDS words; then every thread looks at the words of its own packs, and where there are any,
// puts the pack into its place in LDS and processes the named tokens there one by one (a wave runs as many rounds as the most
// named pack of its lanes has, mostly one), clears the words, and stores the pack.
template <class T, int CHUNK, int BT, bool DENSE> __global__ __launch_bounds__(BT, 6) void logits_kernel(Logits a)
{
    using A = acc_of<T>;
    constexpr int E = 16 / (int)sizeof(T), PPT = CHUNK / (BT * E);
    static_assert(PPT * BT * E == CHUNK && CHUNK % 32 == 0 && CHUNK <= 65536);
    __shared__ __attribute__((aligned(16))) uint32_t word[CHUNK];
    __shared__ __attribute__((aligned(16))) T value[BT * E]; // a pack per thread
    __shared__ BiasSums<A, CHUNK, DENSE> biases;
    const uint32_t r = blockIdx.x / (uint32_t)a.groups;
    const int64_t row = a.row0 + r;
    const int group = (int)(blockIdx.x - r * (uint32_t)a.groups), tid = (int)threadIdx.x, v = (int)a.v;
    const T *z = (const T *)a.z + a.map.template off<L_Z>(row);
    T *out = (T *)a.out + a.map.template off<L_OUT>(row);
    const uint8_t *mask = a.mask ? (const uint8_t *)((const uint32_t *)a.mask + a.map.template off<L_MASK>(row)) : nullptr;
    // the packs are laid so that a wave's run of them starts on a 128-byte line of `out` (rows of an odd length start
    // anywhere): the first one starts `shift` elements before the row
    const int shift = (int)((uintptr_t)out / sizeof(T)) & (128 / (int)sizeof(T) - 1);
    // the block's part of the row, in steps of a pack per thread
    constexpr int STEP = BT * E;
    int begin = (int)((int64_t)group * a.steps / a.groups) * STEP - shift;
    const int stop = (int)((int64_t)(group + 1) * a.steps / a.groups) * STEP - shift, end = stop < v ? stop : v;
    // a pack's mask bits: two bytes at once, the last ones of the row at most (positions below 0 or past v are not asked for)
    const int mask_last = (v + 31) / 32 * 4 - 2;
    auto mask_byte = [&](int i) { return i >> 3 < mask_last ? i >> 3 : mask_last; };
    auto allowed = [&](int i) { return (mask[i >> 3] >> (i & 7)) & 1; };
    TokenScan<BT> prompt, output;
    prompt.send(a.prompt, a.tok64, a.map.template off<L_PROMPT>(row), a.np);
    output.send(a.output, a.tok64, a.map.template off<L_OUTPUT>(row), a.no);
    // the last wave looks after the biases
    const int lane = tid - (BT - 64), nb = (int)a.nb;
    const int64_t bt = a.btok ? a.map.template off<L_BTOK>(row) : 0, bv = a.btok ? a.map.template off<L_BVAL>(row) : 0;
    auto bias_token = [&](int k) { return TokenScan<BT>::narrow(entry_at(a.btok, a.btok64, bt + k)); };
    auto bias_value = [&](int k) { return ((const float *)a.bval)[bv + k]; };
    int b_token = TokenScan<BT>::NONE;
    float b_value = 0;
    if (a.btok && lane >= 0 && lane < nb) {
        b_token = bias_token(lane);
        b_value = bias_value(lane);
    }
    auto fetch = [&](int begin, pack<T, E>(&x)[PPT], uint32_t(&ok)[PPT]) {
#pragma unroll
        for (int j = 0; j < PPT; ++j) {
            const int i = begin + (j * BT + tid) * E;
            if (i >= 0 && i + E <= end) {
                x[j] = load_pack<T, E>(z + i);
                if (mask) ok[j] = load_pack<uint16_t, 1, false>((const uint16_t *)(mask + mask_byte(i))).v[0];
            }
            else
#pragma unroll
                for (int e = 0; e < E; ++e) x[j].v[e] = i + e >= 0 && i + e < end ? z[i + e] : (T)0;
        }
    };
    pack<T, E> x[PPT], x2[PPT];
    uint32_t ok[PPT], ok2[PPT];
    fetch(begin, x, ok);
    const bool lists = a.prompt || a.output || a.btok;
    const A rep = a.rep ? (A)((const float *)a.rep)[a.map.template off<L_REP>(row)] : (A)a.rep0;
    const A freq = a.freq ? (A)((const float *)a.freq)[a.map.template off<L_FREQ>(row)] : (A)a.freq0;
    const A pres = a.pres ? (A)((const float *)a.pres)[a.map.template off<L_PRES>(row)] : (A)a.pres0;
    prompt.arrived(entries_of(a.plen, a.map.template off<L_PLEN>(row), a.np));
    output.arrived(entries_of(a.olen, a.map.template off<L_OLEN>(row), a.no));
    if (lists)
        for (int i = tid * 4; i < CHUNK; i += BT * 4) *(u32x4 *)(word + i) = u32x4{0, 0, 0, 0};
    T *mine = value + tid * E;
    for (; begin < end; begin += CHUNK) {
        const int n = end - begin < CHUNK ? end - begin : CHUNK;
        if (begin + CHUNK < end) fetch(begin + CHUNK, x2, ok2);
        if (lists) {
            __syncthreads(); // the words are clear
            prompt.take(begin, n, [&](int t) { atomicOr(&word[t], SEEN_PROMPT); });
            output.take(begin, n, [&](int t) { atomicAdd(&word[t], 1u); });
            if (a.btok && lane >= 0) { // the chunk's biases
                constexpr int B = DENSE ? 4 : 1; // rounds of 64 entries that are sent for together
                int used = 0, token[B];
                float value[B];
                token[0] = b_token, value[0] = b_value;
                for (int k0 = 0; k0 < nb; k0 += 64 * B) {
#pragma unroll
                    for (int q = 0; q < B; ++q) {
                        const int k = k0 + q * 64 + lane;
                        if (k0 + q == 0) continue;
                        token[q] = k < nb ? bias_token(k) : TokenScan<BT>::NONE;
                        value[q] = k < nb ? bias_value(k) : 0.0f;
                    }
#pragma unroll
                    for (int q = 0; q < B; ++q) {
                        const uint32_t t = (uint32_t)token[q] - (uint32_t)begin;
                        asm volatile("" : "+v"(value[q])); // (arrived: a load left pending where no entry is in the chunk would be
                                                           // waited for, and every other with it, by whoever has its register next)
                        biases.add(word, lane, t < (uint32_t)n, (int)t, value[q], used);
                    }
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < PPT; ++j) {
            const int i = (j * BT + tid) * E;
            if (lists) {
                uint32_t w[E], any = 0;
                load_vals<E, false>(word + i, w);
#pragma unroll
                for (int e = 0; e < E; ++e) any |= w[e];
                if (any) {
                    uint32_t named = 0;
#pragma unroll
                    for (int e = 0; e < E; ++e) named |= (w[e] != 0) << e;
                    *(pack<T, E> *)mine = x[j];
                    for (; named; named &= named - 1) {
                        const int e = __builtin_ctz(named);
                        const uint32_t word_e = word[i + e];
                        A r = (A)mine[e];
                        if (word_e & (SEEN_PROMPT | COUNT)) r = r > 0 ? r / rep : r * rep;
                        const uint32_t said = word_e & COUNT;
                        if (said) r = (r - freq * (A)said) - pres;
                        if (a.btok && (word_e & HAS_BIAS)) r += biases.of(i + e);
                        mine[e] = (T)r;
                        word[i + e] = 0;
                    }
                    x[j] = *(const pack<T, E> *)mine;
                }
            }
            const int g = begin + i;
            if (g >= 0 && i + E <= n) {
                if (mask) keep_allowed(x[j], ok[j] >> (g - 8 * mask_byte(g)));
                store_pack<T, E>(out + g, x[j]);
            }
            else
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (g + e >= 0 && i + e < n) out[g + e] = !mask || allowed(g + e) ? x[j].v[e] : (T)(-__builtin_inff());
            x[j] = x2[j];
            ok[j] = ok2[j];
        }
    }
}

template <class T, int CHUNK, int BT, bool DENSE> int logits_launch_as(Logits &a, int64_t slots, hipStream_t s)
{
    constexpr int64_t STEP = BT * (16 / (int)sizeof(T));
    const int64_t span = a.v + 128 / (int64_t)sizeof(T) - 1; // packs may start before the row
    a.steps = (int32_t)((span + STEP - 1) / STEP);
    a.groups = (int32_t)std::max<int64_t>(1, std::min<int64_t>((span + CHUNK - 1) / CHUNK, slots / a.map.rows));
    in_launches(a.map.rows, a.groups, BT, [&](int64_t first, int64_t rows) {
        a.row0 = first;
        hipLaunchKernelGGL((logits_kernel<T, CHUNK, BT, DENSE>), dim3((unsigned)(rows * a.groups)), dim3(BT), 0, s, a);
    });
    const hipError_t rc = hipGetLastError();
    return rc == hipSuccess ? DPX_OK : fail_hip(rc, "process_logits launch");
}
// Chunks and blocks.  With many rows: a chunk of two packs per thread of 512 (float32: three; more spill), three blocks a CU
// that share out each row's steps and keep the next chunk's logits in flight while they count (256 rows of 100003 float16,
// lists of 1800 and 700 tokens, 50 biases, mask: 27.8 us, 3.9 TB/s; a block per chunk, which reads the lists anew and has
// nothing in flight meanwhile: 38.7; 4096 tokens by 256 threads: 30.3).  Without lists there is nothing to keep: a block per
// chunk streams better (mask alone 22.8 against 24.8 us).  With few rows small chunks, so that the row is spread over the CUs
// (1 row of 131072 float32, lists of 700 and 300 tokens: 5.6 us).
// Biases: up to 256 a row in few sums, more in a sum per token, which costs LDS and with it half of the chunk (256 rows of
// 100003 float16 with 50 / 256 of them: 27.0 / 34.4 us, 29.6 / 40.4 with a sum per token; rows of 1000 the same either way).  One
// wave goes through the list for each chunk: 64 rows of 1000 float32 with 300 biases 10.8 us, one row of 16000 with as many
// biases 111, of 131072 with as many 690; 256 rows of 100003 float16 with 2000 155.
// Letting the threads that hold a token process it in LDS, instead of the thread that holds the logit: 28.4 us for the batch and
// 6.4 for the one row (one more barrier).  Where one token in 13 is named (1024 rows of 32000, 2500 different tokens each) the
// holders of the logits take 37 us for float16 and 60 for float32, 20 and 40 of it for the bytes.
template <class T> int logits_launch(Logits &a, hipStream_t s)
{
    constexpr int E = 16 / (int)sizeof(T), CHUNK = 512 * E * (sizeof(T) == 4 ? 3 : 2);
    const int64_t cus = device_cus(), many = (int64_t)1 << 40;
    const bool lists = a.prompt || a.output || a.btok;
    const bool full = a.map.rows * ((a.v + CHUNK - 1) / CHUNK) >= cus * 2;
    if (a.btok && a.nb > FEW_BIASES)
        return full ? logits_launch_as<T, 512 * E, 512, true>(a, cus * 3, s) : logits_launch_as<T, 256 * E, 256, true>(a, many, s);
    return full ? logits_launch_as<T, CHUNK, 512, false>(a, lists ? cus * 3 : many, s) : logits_launch_as<T, 256 * E, 256, false>(a, many, s);
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
    // (a count has 30 bits of its word; positions are ints)
    for (int64_t k : {a.v, a.np, a.no, a.nb})
        if (k >= (1 << 30)) return fail(DPX_ERR_BAD_ARGUMENT, "process_logits: a last axis is too long");
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
