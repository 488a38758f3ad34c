// Kernels that write replies under the pipeline's rules: logit shaping, the choice of a token, the tag-line grammar's masks
// and steps, and the written tokens as text.  The formulas are in include/tagpipe.h.
#include <hip/hip_runtime.h>

#include "tp_reply.h"
#include "tp_launch.h"

namespace tp {

namespace {

constexpr uint32_t SEEN = 0x80000000u;         // a token's count word: stands in the history; below it: how often behind the prompt
constexpr float NEG_INF = -__builtin_inff();

// ---- element types --------------------------------------------------------------------------------------------------------
// Logits of every type are worked on in 32 bits; the one rounding back to 16 bits (to nearest, ties to even) is the store of
// tp_shape_logits.
struct TF32 {
    using S = float;
    static __device__ float up(S v) { return v; }
    static __device__ S down(float v) { return v; }
};
struct TF16 {
    using S = _Float16;
    static __device__ float up(S v) { return (float)v; }
    static __device__ S down(float v) { return (_Float16)v; }
};
struct TBF16 {
    using S = uint16_t;
    static __device__ float up(S v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
    static __device__ S down(float v) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        if (v != v) return (uint16_t)((u >> 16) | 0x40u);
        return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
    }
};

// ---- one row's rules ------------------------------------------------------------------------------------------------------
struct RowRules {
    const int32_t* history;       // null: nothing to count
    uint32_t len, prompt;
    float rep, freq, pres;
    const float* bias;            // null: none
    const uint8_t* mask;          // the mask row's bytes, null: none
};

__device__ inline uint32_t clamp_len(int32_t n, uint32_t cap) { return n < 0 ? 0u : (uint32_t)n > cap ? cap : (uint32_t)n; }

__device__ inline RowRules row_rules(const tp_logits& a, uint64_t row) {
    RowRules r;
    r.len = a.history ? (a.history_len ? clamp_len(a.history_len[row], a.history_cap) : a.history_cap) : 0u;
    if (!a.repetition && !a.frequency && !a.presence) r.len = 0;       // nothing asks what the history holds
    r.history = a.history + row * a.history_stride;
    r.prompt = a.prompt_len ? clamp_len(a.prompt_len[row], a.history_cap) : 0u;
    r.rep = a.repetition ? a.repetition[row] : 1.0f;
    r.freq = a.frequency ? a.frequency[row] : 0.0f;
    r.pres = a.presence ? a.presence[row] : 0.0f;
    r.bias = nullptr;
    if (a.bias) {
        const uint32_t b = a.bias_row ? (uint32_t)a.bias_row[row] : 0u;
        if (b < a.n_bias) r.bias = a.bias + (uint64_t)b * a.bias_stride;
    }
    r.mask = nullptr;
    if (a.mask) {
        const uint32_t m = a.mask_row ? (uint32_t)a.mask_row[row] : 0u;
        if (m < a.n_masks) r.mask = (const uint8_t*)(a.mask + (uint64_t)m * a.mask_stride);
    }
    return r;
}

// The penalties of a token whose count word is c.  -ffp-contract=off: every operation rounds by itself, as the formula says.
__device__ inline float penalised(float x, uint32_t c, const RowRules& r) {
    if (c) {
        x = x > 0.0f ? x / r.rep : x * r.rep;
        const uint32_t n = c & ~SEEN;
        if (n) {
            x = x - r.freq * (float)n;
            x = x - r.pres;
        }
    }
    return x;
}

// ---- block reductions -----------------------------------------------------------------------------------------------------
// Every sum is taken in one fixed order, so that a call's results do not change from run to run.
template <int THREADS>
struct Block {
    static constexpr int WAVES = THREADS / 64;
    struct Lds {
        float f[WAVES];
        uint32_t u[WAVES];
        double d[WAVES];
        uint32_t first, last;
    };
    // the largest value and the lowest index that has it, to every thread
    static __device__ void best(float& v, uint32_t& at, Lds& l) {
        for (int d = 32; d; d >>= 1) {
            const float ov = __shfl_xor(v, d, 64);
            const uint32_t oa = (uint32_t)__shfl_xor((int)at, d, 64);
            if (ov > v || (ov == v && oa < at)) { v = ov; at = oa; }
        }
        if ((threadIdx.x & 63) == 0) { l.f[threadIdx.x >> 6] = v; l.u[threadIdx.x >> 6] = at; }
        __syncthreads();
        v = l.f[0];
        at = l.u[0];
        for (int w = 1; w < WAVES; ++w) {
            const float ov = l.f[w];
            const uint32_t oa = l.u[w];
            if (ov > v || (ov == v && oa < at)) { v = ov; at = oa; }
        }
        __syncthreads();
    }
    static __device__ double sum(double v, Lds& l) {
        for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
        if ((threadIdx.x & 63) == 0) l.d[threadIdx.x >> 6] = v;
        __syncthreads();
        v = l.d[0];
        for (int w = 1; w < WAVES; ++w) v += l.d[w];
        __syncthreads();
        return v;
    }
    // sum of the threads before this one; `total`: of all
    static __device__ double before(double v, double& total, Lds& l) {
        const int lane = (int)(threadIdx.x & 63);
        double incl = v;
        for (int d = 1; d < 64; d <<= 1) {
            const double o = __shfl_up(incl, d, 64);
            if (lane >= d) incl += o;
        }
        if (lane == 63) l.d[threadIdx.x >> 6] = incl;
        __syncthreads();
        double base = 0.0;
        total = 0.0;
        for (int w = 0; w < WAVES; ++w) {
            if (w < (int)(threadIdx.x >> 6)) base += l.d[w];
            total += l.d[w];
        }
        __syncthreads();
        const double excl = __shfl_up(incl, 1, 64);
        return base + (lane ? excl : 0.0);
    }
};

__device__ inline float weight(float z, float best) { return z == best ? 1.0f : expf(z - best); }

// ---- shaping of a dense row, in chunks --------------------------------------------------------------------------------------
// A block takes LOGIT_CHUNK tokens of one row, 16 a thread in two vectors of eight, whose loads stand in flight while the
// block counts the history: a 32 KB LDS table has a word for each of the chunk's tokens, and every thread looks at some of the
// row's whole history for tokens of the chunk.  (Counting needs no second pass over the logits and no device memory; the
// history is read once per chunk, from the L2 after the first.)  A vector whose eight mask bits are all 0 is not loaded.
constexpr int CHUNK_THREADS = 512;
constexpr int CHUNK_VECS = (int)(LOGIT_CHUNK / (CHUNK_THREADS * 8));
static_assert(CHUNK_VECS * CHUNK_THREADS * 8 == (int)LOGIT_CHUNK, "a chunk is whole vectors");

// the first token of this thread's vector v within the chunk
__device__ inline uint32_t vec_at(int v) { return (uint32_t)v * CHUNK_THREADS * 8 + threadIdx.x * 8; }

template <class T>
__device__ void shaped_chunk(const tp_logits& a, const RowRules& r, uint64_t row, uint32_t c0, uint32_t* cnt, float (&x)[CHUNK_VECS][8]) {
    using S = typename T::S;
    const S* l = (const S*)a.logits + row * a.stride + c0;
    const uint32_t n = a.vocab - c0;                                   // tokens from here to the row's end
    uint32_t allowed[CHUNK_VECS];
    S raw[CHUNK_VECS][8] = {};
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v) {
        const uint32_t at = vec_at(v);
        allowed[v] = at < n ? (r.mask ? r.mask[(c0 + at) >> 3] : 0xFFu) : 0u;
    }
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v) {
        const uint32_t at = vec_at(v);
        if (!allowed[v]) continue;
        if (at + 8 <= n) {
            __builtin_memcpy(raw[v], l + at, sizeof raw[v]);           // rows may start at any element
        } else {
            allowed[v] &= 0xFFu >> (8 - (n - at));
#pragma unroll
            for (int j = 0; j < 8; ++j) if (at + j < n) raw[v][j] = l[at + j];
        }
    }
    if (r.len) {
        for (uint32_t k = threadIdx.x * 4; k < LOGIT_CHUNK; k += CHUNK_THREADS * 4) *(uint4*)(cnt + k) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const uint32_t inside = n < LOGIT_CHUNK ? n : LOGIT_CHUNK;
        for (uint32_t k = threadIdx.x; k < r.len; k += CHUNK_THREADS) {
            const uint32_t t = (uint32_t)r.history[k] - c0;
            if (t < inside) {
                if (k >= r.prompt) atomicAdd(&cnt[t], 1u); else atomicOr(&cnt[t], SEEN);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v) {
        const uint32_t at = vec_at(v);
        float b[8];
        if (r.bias && allowed[v]) {
            if (at + 8 <= n) {
                __builtin_memcpy(b, r.bias + c0 + at, sizeof b);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = at + j < n ? r.bias[c0 + at + j] : 0.0f;
            }
        }
        uint32_t c[8] = {};
        if (r.len) __builtin_memcpy(c, __builtin_assume_aligned(cnt + at, 16), sizeof c);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float y = penalised(T::up(raw[v][j]), c[j], r);
            if (r.bias) y = y + b[j];
            x[v][j] = allowed[v] >> j & 1 ? y : NEG_INF;
        }
    }
}

template <class T>
__global__ __launch_bounds__(CHUNK_THREADS) void k_shape(tp_logits a, uint64_t block0, uint32_t chunks, void* out, uint64_t out_stride) {
    using S = typename T::S;
    __shared__ alignas(16) uint32_t cnt[LOGIT_CHUNK];
    const uint64_t b = block0 + blockIdx.x, row = b / chunks;
    const uint32_t c0 = (uint32_t)(b % chunks) * LOGIT_CHUNK;
    float x[CHUNK_VECS][8];
    shaped_chunk<T>(a, row_rules(a, row), row, c0, cnt, x);
    S* o = (S*)out + row * out_stride + c0;
    const uint32_t n = a.vocab - c0;
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v) {
        const uint32_t at = vec_at(v);
        S raw[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[j] = T::down(x[v][j]);
        if (at + 8 <= n) {
            __builtin_memcpy(o + at, raw, sizeof raw);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) if (at + j < n) o[at + j] = raw[j];
        }
    }
}

// ---- the choice -------------------------------------------------------------------------------------------------------------
using CB = Block<CHUNK_THREADS>;

// z = x / T where there is a temperature; a NaN, of x or of an infinity over an infinite temperature, counts as -infinity
__device__ inline float scaled(float x, float t) {
    const float z = t > 0.0f ? x / t : x;
    return z == z ? z : NEG_INF;
}

__device__ inline float temperature_of(const float* temperature, const float* uniform, uint64_t row) {
    const float t = temperature && uniform ? temperature[row] : 0.0f;
    return t > 0.0f ? t : 0.0f;
}

// The chunk's part of the choice out of its shaped logits (z in place of x on return).
__device__ ChoicePart chunk_part(float (&x)[CHUNK_VECS][8], float t, uint32_t c0, CB::Lds& l) {
    float best = NEG_INF;
    uint32_t at = 0xFFFFFFFFu;
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[v][j] = scaled(x[v][j], t);
            if (x[v][j] > best) { best = x[v][j]; at = c0 + vec_at(v) + j; }
        }
    CB::best(best, at, l);
    double s = 0.0;
    if (best > NEG_INF) {
#pragma unroll
        for (int v = 0; v < CHUNK_VECS; ++v) {
            double p = 0.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) p += (double)weight(x[v][j], best);
            s += p;
        }
        s = CB::sum(s, l);
    }
    return ChoicePart{best, (int32_t)at, s};
}

// The lowest token of the chunk whose cumulative weight exceeds `target` (weights against `best`); where rounding or a
// `uniform` of 1 or more leaves none, the last one of a weight above 0.  The thread that holds it returns true, its z in z_out.
__device__ bool pick_in_chunk(const float (&z)[CHUNK_VECS][8], float best, double target, CB::Lds& l, uint32_t& at_out, float& z_out) {
    if (threadIdx.x == 0) { l.first = 0xFFFFFFFFu; l.last = 0; }
    __syncthreads();
    double carry = 0.0;
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v) {
        double w[8], mine = 0.0, total;
#pragma unroll
        for (int j = 0; j < 8; ++j) { w[j] = (double)weight(z[v][j], best); mine += w[j]; }
        double cum = carry + CB::before(mine, total, l);
        uint32_t first = 0xFFFFFFFFu, last = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cum += w[j];
            if (w[j] > 0.0) {
                last = vec_at(v) + j + 1;
                if (first == 0xFFFFFFFFu && cum > target) first = vec_at(v) + j;
            }
        }
        if (first != 0xFFFFFFFFu) atomicMin(&l.first, first);
        if (last) atomicMax(&l.last, last);
        carry += total;
    }
    __syncthreads();
    const uint32_t at = l.first != 0xFFFFFFFFu ? l.first : l.last - 1;
    bool mine = false;
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (at == vec_at(v) + j) { mine = true; z_out = z[v][j]; }
    at_out = at;
    return mine;
}

__device__ inline float log_probability(float z, float best, double sum) { return (float)((z == best ? 0.0 : (double)z - (double)best) - log(sum)); }

template <class T>
__global__ __launch_bounds__(CHUNK_THREADS) void k_choose(tp_logits a, uint64_t block0, uint32_t chunks, const float* temperature, const float* uniform,
                                                          int32_t* tokens, float* logprob, ChoicePart* parts) {
    __shared__ alignas(16) uint32_t cnt[LOGIT_CHUNK];
    __shared__ CB::Lds l;
    const uint64_t b = block0 + blockIdx.x, row = b / chunks;
    const uint32_t c0 = (uint32_t)(b % chunks) * LOGIT_CHUNK;
    float x[CHUNK_VECS][8];
    shaped_chunk<T>(a, row_rules(a, row), row, c0, cnt, x);
    const float t = temperature_of(temperature, uniform, row);
    const ChoicePart p = chunk_part(x, t, c0, l);
    if (chunks > 1) {
        if (threadIdx.x == 0) parts[b] = p;
        return;
    }
    if (p.best > NEG_INF && t > 0.0f) {
        uint32_t at;
        float z;
        if (pick_in_chunk(x, p.best, (double)uniform[row] * p.sum, l, at, z)) {
            tokens[row] = (int32_t)at;
            if (logprob) logprob[row] = log_probability(z, p.best, p.sum);
        }
    } else if (threadIdx.x == 0) {
        const bool none = !(p.best > NEG_INF);
        tokens[row] = none ? -1 : p.token;
        if (logprob) logprob[row] = none ? NEG_INF : (float)-log(p.sum);
    }
}

// Joins the chunks of a row.  A sampled row shapes the one chunk that holds its token again.
template <class T>
__global__ __launch_bounds__(CHUNK_THREADS) void k_choose_join(tp_logits a, uint64_t row0, uint32_t chunks, const float* temperature, const float* uniform,
                                                               int32_t* tokens, float* logprob, const ChoicePart* parts) {
    __shared__ alignas(16) uint32_t cnt[LOGIT_CHUNK];
    __shared__ CB::Lds l;
    __shared__ uint32_t pick_chunk;
    __shared__ double pick_target;
    const uint64_t row = row0 + blockIdx.x;
    const ChoicePart* p = parts + row * chunks;
    float best = NEG_INF;
    uint32_t at = 0xFFFFFFFFu;
    for (uint32_t c = threadIdx.x; c < chunks; c += CHUNK_THREADS) {
        const float v = p[c].best;
        if (v > best) { best = v; at = (uint32_t)p[c].token; }
    }
    CB::best(best, at, l);
    const float t = temperature_of(temperature, uniform, row);
    if (!(best > NEG_INF)) {
        if (threadIdx.x == 0) {
            tokens[row] = -1;
            if (logprob) logprob[row] = NEG_INF;
        }
        return;
    }
    auto share = [&](uint32_t c) { return p[c].best > NEG_INF ? p[c].sum * (p[c].best == best ? 1.0 : exp((double)p[c].best - (double)best)) : 0.0; };
    double s = 0.0;
    for (uint32_t c = threadIdx.x; c < chunks; c += CHUNK_THREADS) s += share(c);
    s = CB::sum(s, l);
    if (!(t > 0.0f)) {
        if (threadIdx.x == 0) {
            tokens[row] = (int32_t)at;
            if (logprob) logprob[row] = (float)-log(s);
        }
        return;
    }
    if (threadIdx.x == 0) {
        const double target = (double)uniform[row] * s;
        double before = 0.0, at_last = 0.0;
        uint32_t c = 0, last = 0;
        for (; c < chunks; ++c) {
            const double w = share(c);
            if (w > 0.0) { last = c; at_last = before; }
            if (w > 0.0 && before + w > target) break;
            before += w;
        }
        const bool found = c < chunks;
        pick_chunk = found ? c : last;
        const double rest = found ? target - before : target - at_last;
        const float pb = p[pick_chunk].best;
        pick_target = rest / (pb == best ? 1.0 : exp((double)pb - (double)best));
    }
    __syncthreads();
    const uint32_t c0 = pick_chunk * LOGIT_CHUNK;
    float x[CHUNK_VECS][8];
    shaped_chunk<T>(a, row_rules(a, row), row, c0, cnt, x);
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[v][j] = scaled(x[v][j], t);
    float z;
    if (pick_in_chunk(x, p[pick_chunk].best, pick_target, l, at, z)) {
        tokens[row] = (int32_t)(c0 + at);
        if (logprob) logprob[row] = log_probability(z, best, s);
    }
}

// ---- the grammar ----------------------------------------------------------------------------------------------------------------

// whether an entry may be taken with `tags` finished tags
__device__ inline bool may(uint32_t move, uint32_t tags, const DevGrammar& g) {
    const uint32_t kind = move >> MOVE_SHIFT;
    return kind == MOVE_INSIDE || (kind == MOVE_COMMA ? tags + 2 <= g.max_tags : tags + 1 >= g.min_tags);
}

struct List { uint32_t lo, hi, tags; };
__device__ inline List list_of(const DevGrammar& g, const int32_t* states, uint64_t row) {
    const uint32_t place = (uint32_t)states[2 * row];
    const int32_t tags = states[2 * row + 1];
    List q{0, 0, tags < 0 ? 0u : tags > 65535 ? 65535u : (uint32_t)tags};
    if (place < g.n_places) { q.lo = g.begin[place]; q.hi = g.begin[place + 1]; }
    return q;
}

// first entry in [lo, hi) whose token is at least t
__device__ inline uint32_t lower_entry(const int32_t* token, uint32_t lo, uint32_t hi, int32_t t) {
    while (lo < hi) {
        const uint32_t m = lo + (hi - lo) / 2;
        if (token[m] < t) lo = m + 1; else hi = m;
    }
    return lo;
}

// A block writes MASK_PIECE words of one row: cleared in LDS, the list's entries that fall into the piece set there, stored
// in 16-byte pieces.
constexpr uint32_t MASK_PIECE = 1024;
__global__ __launch_bounds__(256) void k_grammar_mask(DevGrammar g, const int32_t* states, uint64_t block0, uint32_t pieces, uint32_t* mask, uint64_t mask_stride) {
    __shared__ alignas(16) uint32_t bits[MASK_PIECE];
    const uint64_t b = block0 + blockIdx.x, row = b / pieces;
    const uint32_t w0 = (uint32_t)(b % pieces) * MASK_PIECE, words = (g.n_tokens + 31) / 32;
    List q = list_of(g, states, row);
    *(uint4*)(bits + threadIdx.x * 4) = make_uint4(0, 0, 0, 0);
    const int32_t t0 = (int32_t)(w0 * 32);
    q.lo = lower_entry(g.token, q.lo, q.hi, t0);
    __syncthreads();
    for (uint32_t e = q.lo + threadIdx.x; e < q.hi; e += 256) {
        const uint32_t t = (uint32_t)(g.token[e] - t0);
        if (t >= MASK_PIECE * 32) break;
        if (may(g.move[e], q.tags, g)) atomicOr(&bits[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
    uint32_t* out = mask + row * mask_stride + w0;
    const uint32_t n = words - w0, at = threadIdx.x * 4;
    if (at + 4 <= n) {
        __builtin_memcpy(out + at, bits + at, 16);
    } else {
        for (uint32_t j = at; j < n && j < at + 4; ++j) out[j] = bits[j];
    }
}

// Moves a row on by entry e with its token, and appends it.
__device__ inline void take_entry(const DevGrammar& g, const tp_logits& a, uint64_t row, uint32_t move, int32_t token, int32_t* states, int append) {
    states[2 * row] = (int32_t)(move & MOVE_PLACE);
    if (move >> MOVE_SHIFT == MOVE_COMMA) states[2 * row + 1] += 1;
    if (append) {
        const uint32_t n = clamp_len(a.history_len[row], a.history_cap);
        a.history[row * a.history_stride + n] = token;                   // the caller has seen that there is room
        a.history_len[row] = (int32_t)n + 1;
    }
}

__device__ inline bool has_room(const tp_logits& a, uint64_t row, int append) { return !append || clamp_len(a.history_len[row], a.history_cap) < a.history_cap; }

// The choice among a row's list: a block per row, the list in pieces of STEP_PIECE entries whose tokens, counts and shaped
// logits stand in LDS.  Only the listed tokens' logits are read.  History tokens are found by binary search among the
// piece's (ascending) tokens.
constexpr int STEP_THREADS = 256;
constexpr uint32_t STEP_PIECE = 4096;
using SB = Block<STEP_THREADS>;

struct StepLds {
    int32_t token[STEP_PIECE];
    uint32_t cnt[STEP_PIECE];
    float z[STEP_PIECE];
    SB::Lds l;
};

// z of the m entries from e0 into LDS; an entry that may not be taken has -infinity
template <class T>
__device__ void step_piece(const DevGrammar& g, const tp_logits& a, const RowRules& r, uint64_t row, uint32_t tags, float t, uint32_t e0, uint32_t m, StepLds& s) {
    const typename T::S* l = (const typename T::S*)a.logits + row * a.stride;
    for (uint32_t i = threadIdx.x; i < m; i += STEP_THREADS) {
        const int32_t token = g.token[e0 + i];
        s.token[i] = token;
        s.cnt[i] = 0;
        s.z[i] = may(g.move[e0 + i], tags, g) ? T::up(l[token]) : NEG_INF;
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < r.len; k += STEP_THREADS) {
        const int32_t h = r.history[k];
        const uint32_t i = lower_entry(s.token, 0, m, h);
        if (i < m && s.token[i] == h) {
            if (k >= r.prompt) atomicAdd(&s.cnt[i], 1u); else atomicOr(&s.cnt[i], SEEN);
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < m; i += STEP_THREADS) {
        if (!may(g.move[e0 + i], tags, g)) continue;
        float y = penalised(s.z[i], s.cnt[i], r);
        if (r.bias) y = y + r.bias[s.token[i]];
        s.z[i] = scaled(y, t);
    }
    __syncthreads();
}

template <class T>
__global__ __launch_bounds__(STEP_THREADS) void k_grammar_step(DevGrammar g, tp_logits a, uint64_t row0, const float* temperature, const float* uniform,
                                                               int32_t* states, int32_t* tokens, float* logprob, int append) {
    __shared__ StepLds s;
    const uint64_t row = row0 + blockIdx.x;
    const List q = list_of(g, states, row);
    const RowRules r = row_rules(a, row);
    const float t = temperature_of(temperature, uniform, row);
    const bool room = has_room(a, row, append);
    // largest z, the entry that has it first, and the sum of the weights against it, over all pieces
    float best = NEG_INF;
    uint32_t at = 0xFFFFFFFFu;
    double sum = 0.0;
    for (uint32_t p = q.lo; p < q.hi; p += STEP_PIECE) {
        const uint32_t m = q.hi - p < STEP_PIECE ? q.hi - p : STEP_PIECE;
        step_piece<T>(g, a, r, row, q.tags, t, p, m, s);
        float pb = NEG_INF;
        uint32_t pa = 0xFFFFFFFFu;
        for (uint32_t i = threadIdx.x; i < m; i += STEP_THREADS)
            if (s.z[i] > pb) { pb = s.z[i]; pa = p + i; }
        SB::best(pb, pa, s.l);
        if (pb > best) {
            sum = best > NEG_INF ? sum * (double)weight(best, pb) : 0.0;
            best = pb;
            at = pa;
        }
        if (best > NEG_INF) {
            double w = 0.0;
            for (uint32_t i = threadIdx.x; i < m; i += STEP_THREADS) w += (double)weight(s.z[i], best);
            sum += SB::sum(w, s.l);
        }
    }
    if (!(best > NEG_INF) || !room) {
        if (threadIdx.x == 0) {
            tokens[row] = -1;
            if (logprob) logprob[row] = NEG_INF;
        }
        return;
    }
    float z = best;
    if (t > 0.0f) {
        const double target = (double)uniform[row] * sum;
        double carry = 0.0;
        uint32_t found = 0xFFFFFFFFu, last = 0xFFFFFFFFu;
        float z_last = NEG_INF;
        for (uint32_t p = q.lo; p < q.hi && found == 0xFFFFFFFFu; p += STEP_PIECE) {
            const uint32_t m = q.hi - p < STEP_PIECE ? q.hi - p : STEP_PIECE;
            if (q.hi - q.lo > STEP_PIECE) step_piece<T>(g, a, r, row, q.tags, t, p, m, s);   // else the one piece still stands there
            if (threadIdx.x == 0) { s.l.first = 0xFFFFFFFFu; s.l.last = 0; }
            const uint32_t run = (m + STEP_THREADS - 1) / STEP_THREADS;       // each thread's entries stand side by side
            const uint32_t i0 = threadIdx.x * run < m ? threadIdx.x * run : m, i1 = i0 + run < m ? i0 + run : m;
            double mine = 0.0, total;
            for (uint32_t i = i0; i < i1; ++i) mine += (double)weight(s.z[i], best);
            double cum = carry + SB::before(mine, total, s.l);
            uint32_t f = 0xFFFFFFFFu, lst = 0;
            for (uint32_t i = i0; i < i1; ++i) {
                const double w = (double)weight(s.z[i], best);
                cum += w;
                if (w > 0.0) {
                    lst = i + 1;
                    if (f == 0xFFFFFFFFu && cum > target) f = i;
                }
            }
            if (f != 0xFFFFFFFFu) atomicMin(&s.l.first, f);
            if (lst) atomicMax(&s.l.last, lst);
            __syncthreads();
            const uint32_t first = s.l.first, behind = s.l.last;
            if (first != 0xFFFFFFFFu) { found = p + first; z = s.z[first]; }
            if (behind) { last = p + behind - 1; z_last = s.z[behind - 1]; }
            carry += total;
            __syncthreads();
        }
        if (found == 0xFFFFFFFFu) { found = last; z = z_last; }
        at = found;
    }
    if (threadIdx.x == 0) {
        const int32_t token = g.token[at];
        tokens[row] = token;
        if (logprob) logprob[row] = log_probability(z, best, sum);
        take_entry(g, a, row, g.move[at], token, states, append);
    }
}

// The move by the caller's own tokens: a thread per row.
__global__ __launch_bounds__(256) void k_grammar_advance(DevGrammar g, tp_logits a, int32_t* states, const int32_t* tokens, int append) {
    const uint64_t row = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= a.rows) return;
    const int32_t token = tokens[row];
    if (token == -1 || !has_room(a, row, append)) return;
    const List q = list_of(g, states, row);
    const uint32_t e = lower_entry(g.token, q.lo, q.hi, token);
    if (e < q.hi && g.token[e] == token && may(g.move[e], q.tags, g)) take_entry(g, a, row, g.move[e], token, states, append);
    else states[2 * row] = -1;
}

// ---- the lines ------------------------------------------------------------------------------------------------------------------

struct Written { uint32_t first, last; };
__device__ inline Written written(const int32_t* begin, const int32_t* len, uint32_t width, uint64_t row) {
    return Written{begin ? clamp_len(begin[row], width) : 0u, len ? clamp_len(len[row], width) : width};
}

// a wave per row: the bytes of its text
__global__ __launch_bounds__(256) void k_line_sizes(DevGrammar g, const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t block0, uint64_t rows, uint32_t* sizes) {
    const uint64_t row = (block0 + blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const Written w = written(begin, len, width, row);
    uint32_t n = 0;
    for (uint64_t k = w.first + (threadIdx.x & 63); k < w.last; k += 64) {
        const uint32_t t = (uint32_t)tokens[row * stride + k];
        if (t < g.n_tokens) n += g.text_begin[t + 1] - g.text_begin[t];
    }
    for (int d = 32; d; d >>= 1) n += (uint32_t)__shfl_xor((int)n, d, 64);
    if ((threadIdx.x & 63) == 0) sizes[row] = n;
}

// a wave per row: a lane copies one token's bytes
__global__ __launch_bounds__(256) void k_line_text(DevGrammar g, const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t block0, uint64_t rows,
                                                   const uint64_t* offsets, uint8_t* arena, uint64_t capacity) {
    const uint64_t row = (block0 + blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const uint32_t lane = threadIdx.x & 63;
    const Written w = written(begin, len, width, row);
    uint64_t at = offsets[row];
    for (uint64_t k0 = w.first; k0 < w.last; k0 += 64) {
        uint32_t from = 0, n = 0;
        if (k0 + lane < w.last) {
            const uint32_t t = (uint32_t)tokens[row * stride + k0 + lane];
            if (t < g.n_tokens) { from = g.text_begin[t]; n = g.text_begin[t + 1] - from; }
        }
        uint32_t incl = n;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)incl, d, 64);
            if ((int)lane >= d) incl += o;
        }
        const uint64_t to = at + incl - n;
        for (uint32_t j = 0; j < n; ++j) if (to + j < capacity) arena[to + j] = g.text[from + j];
        at += (uint32_t)__shfl((int)incl, 63, 64);
    }
    if (row == rows - 1 && lane < 16 && at + lane < capacity) arena[at + lane] = 0;
}

constexpr uint64_t MAX_BLOCKS = (uint64_t)1 << 22;   // of one launch: its threads stay below 2^32

template <class F>
hipError_t in_ranges(uint64_t blocks, F&& launch) {
    for (uint64_t b = 0; b < blocks; b += MAX_BLOCKS) {
        launch(b, (unsigned)(blocks - b < MAX_BLOCKS ? blocks - b : MAX_BLOCKS));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <class F>
hipError_t by_type(int32_t type, F&& f) {
    return type == TP_T_F32 ? f(TF32{}) : type == TP_T_F16 ? f(TF16{}) : f(TBF16{});
}

}  // namespace

hipError_t launch_shape(const tp_logits& io, void* out, uint64_t out_stride) {
    const uint32_t chunks = logit_chunks(io.vocab);
    return by_type(io.type, [&](auto tag) {
        using T = decltype(tag);
        return in_ranges(io.rows * chunks, [&](uint64_t b, unsigned n) {
            hipLaunchKernelGGL(k_shape<T>, dim3(n), dim3(CHUNK_THREADS), 0, (hipStream_t)io.stream, io, b, chunks, out, out_stride);
        });
    });
}

hipError_t launch_choose(const tp_logits& io, const float* temperature, const float* uniform, int32_t* tokens, float* logprob, ChoicePart* parts) {
    const uint32_t chunks = logit_chunks(io.vocab);
    return by_type(io.type, [&](auto tag) {
        using T = decltype(tag);
        hipError_t e = in_ranges(io.rows * chunks, [&](uint64_t b, unsigned n) {
            hipLaunchKernelGGL(k_choose<T>, dim3(n), dim3(CHUNK_THREADS), 0, (hipStream_t)io.stream, io, b, chunks, temperature, uniform, tokens, logprob, parts);
        });
        if (e != hipSuccess || chunks == 1) return e;
        return in_ranges(io.rows, [&](uint64_t b, unsigned n) {
            hipLaunchKernelGGL(k_choose_join<T>, dim3(n), dim3(CHUNK_THREADS), 0, (hipStream_t)io.stream, io, b, chunks, temperature, uniform, tokens, logprob, parts);
        });
    });
}

hipError_t launch_grammar_mask(const DevGrammar& g, const int32_t* states, uint64_t rows, uint32_t* mask, uint64_t mask_stride, hipStream_t s) {
    const uint32_t pieces = ((g.n_tokens + 31) / 32 + MASK_PIECE - 1) / MASK_PIECE;
    return in_ranges(rows * pieces, [&](uint64_t b, unsigned n) {
        hipLaunchKernelGGL(k_grammar_mask, dim3(n), dim3(256), 0, s, g, states, b, pieces, mask, mask_stride);
    });
}

hipError_t launch_grammar_step(const DevGrammar& g, const tp_logits& io, const float* temperature, const float* uniform, int32_t* states,
                               int32_t* tokens, float* logprob, int append) {
    if (!io.logits) {
        hipLaunchKernelGGL(k_grammar_advance, dim3((unsigned)((io.rows + 255) / 256)), dim3(256), 0, (hipStream_t)io.stream, g, io, states, tokens, append);
        return hipGetLastError();
    }
    return by_type(io.type, [&](auto tag) {
        using T = decltype(tag);
        return in_ranges(io.rows, [&](uint64_t b, unsigned n) {
            hipLaunchKernelGGL(k_grammar_step<T>, dim3(n), dim3(STEP_THREADS), 0, (hipStream_t)io.stream, g, io, b, temperature, uniform, states, tokens, logprob, append);
        });
    });
}

hipError_t launch_grammar_lines(const DevGrammar& g, const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t rows,
                                uint8_t* arena, uint64_t capacity, uint64_t* offsets, void* workspace, hipStream_t s) {
    uint32_t* sizes = (uint32_t*)workspace;
    uint64_t* tiles = (uint64_t*)((uint8_t*)workspace + (rows + 4) / 4 * 16);
    hipError_t e = in_ranges((rows + 3) / 4, [&](uint64_t b, unsigned n) {
        hipLaunchKernelGGL(k_line_sizes, dim3(n), dim3(256), 0, s, g, tokens, stride, width, begin, len, b, rows, sizes);
    });
    if (e != hipSuccess) return e;
    e = launch_scan_u32(sizes, rows, offsets, tiles, nullptr, nullptr, s);
    if (e != hipSuccess) return e;
    return in_ranges((rows + 3) / 4, [&](uint64_t b, unsigned n) {
        hipLaunchKernelGGL(k_line_text, dim3(n), dim3(256), 0, s, g, tokens, stride, width, begin, len, b, rows, offsets, arena, capacity);
    });
}

}  // namespace tp
