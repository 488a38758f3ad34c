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

// ---- wave reductions --------------------------------------------------------------------------------------------------------
// Every sum is taken in one fixed order, so that a call's results do not change from run to run.
template <int CTRL, int ROWS>
__device__ inline float dpp(float old, float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
}
__device__ inline float read_lane(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }

__device__ inline float wave_max(float v) {
    v = fmaxf(v, dpp<0x111, 0xF>(v, v));   // row_shr:1, 2, 4, 8
    v = fmaxf(v, dpp<0x112, 0xF>(v, v));
    v = fmaxf(v, dpp<0x114, 0xF>(v, v));
    v = fmaxf(v, dpp<0x118, 0xF>(v, v));
    v = fmaxf(v, dpp<0x142, 0xA>(v, v));   // row_bcast:15 into rows 1 and 3
    v = fmaxf(v, dpp<0x143, 0xC>(v, v));   // row_bcast:31 into rows 2 and 3
    return read_lane(v, 63);
}
__device__ inline float wave_sum(float v) {
    v += dpp<0x111, 0xF>(0.0f, v);
    v += dpp<0x112, 0xF>(0.0f, v);
    v += dpp<0x114, 0xF>(0.0f, v);
    v += dpp<0x118, 0xF>(0.0f, v);
    v += dpp<0x142, 0xA>(0.0f, v);
    v += dpp<0x143, 0xC>(0.0f, v);
    return read_lane(v, 63);
}
__device__ inline double wave_sum(double v) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
// sum of the lanes up to and including this one
__device__ inline double wave_scan(double v) {
    const int lane = (int)(threadIdx.x & 63);
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// ---- weights ------------------------------------------------------------------------------------------------------------------
// exp((x - best) / T) as 2^((x - best) * k), k = log2(e) / T.  The difference is taken first: it is small where the weight counts,
// so that the rounding of k and of the product (each half a step, relative) moves a weight by less than |ln w| steps of 2^-23, where dividing
// every x by T would move it by as many steps as z is large.  k stays a normal number, so that neither 0 * k nor -infinity * k is a NaN.
__device__ inline float weight_scale(float t) {
    return t > 0.0f ? fminf(fmaxf(1.44269504088896341f / t, 1.17549435e-38f), 3.40282347e38f) : 1.44269504088896341f;
}
__device__ inline float weight(float x, float best, float k) {
    if (best == -NEG_INF) return x == best ? 1.0f : 0.0f;
    return __builtin_amdgcn_exp2f((x - best) * k);
}
__device__ inline float temperature_of(const float* temperature, const float* uniform, uint64_t row) {
    const float t = temperature && uniform ? temperature[row] : 0.0f;
    return t > 0.0f ? t : 0.0f;
}
__device__ inline float log_probability(float x, float best, float t, double sum) {
    return (float)((x == best ? 0.0 : ((double)x - (double)best) / (t > 0.0f ? (double)t : 1.0)) - log(sum));
}
// a NaN counts as -infinity in a choice
__device__ inline float countable(float x) { return fmaxf(x, NEG_INF); }

// What a barrier of THREADS threads is: a single wave needs none, since its LDS accesses happen in order; the compiler must
// only keep them so.  (One wave of a larger block may then work on its own.)
template <int THREADS>
__device__ inline void block_sync() {
    if constexpr (THREADS == 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}
template <int THREADS>
__device__ inline bool block_any(bool v) {
    if constexpr (THREADS == 64) {
        const bool any = __ballot(v) != 0;
        block_sync<64>();
        return any;
    } else {
        return __syncthreads_or(v) != 0;
    }
}

// ---- shaping of a dense row, in windows -----------------------------------------------------------------------------------------
// THREADS threads take a window of THREADS * VECS * 8 tokens of one row, VECS vectors of eight each, whose loads stand in flight while the
// history is worked on.  Of the history only the tokens inside the window count: their counts are taken in an LDS table (a word
// per token; only the words that are hit are cleared), then one thread per distinct token works the penalties out, with the token's logit
// of its own load, and leaves the result in the token's word and a bit in a bitmap.  A vector then looks at one byte of the bitmap:
// the penalties' arithmetic, a division among it, is done once per repeated token instead of once per token of the row, and a
// window that the history does not reach stops after the first look.  A vector whose eight mask bits are all 0 is not loaded.
template <int THREADS, int VECS>
struct Window {
    static constexpr uint32_t TOKENS = THREADS * VECS * 8;
    struct Lds {
        alignas(16) uint32_t word[TOKENS];
        alignas(16) uint32_t seen[TOKENS / 32];
    };
    // the first token of this thread's vector v within the window
    static __device__ uint32_t at(int v) { return (uint32_t)v * THREADS * 8 + threadIdx.x * 8; }

    // whether the history has a token inside the window of `inside` tokens from w0; if so their penalised logits stand in LDS
    template <class T>
    static __device__ bool repeated(const RowRules& r, const typename T::S* l, uint32_t w0, uint32_t inside, Lds& s) {
        if (!r.len) return false;
        const uint32_t tid = threadIdx.x, h0 = tid < r.len ? (uint32_t)r.history[tid] - w0 : 0xFFFFFFFFu;
        bool any = h0 < inside;
        if (any) s.word[h0] = 0;
        for (uint32_t k = tid + THREADS; k < r.len; k += THREADS) {
            const uint32_t t = (uint32_t)r.history[k] - w0;
            if (t < inside) { s.word[t] = 0; any = true; }
        }
        for (uint32_t k = tid; k < TOKENS / 32; k += THREADS) s.seen[k] = 0;
        if (!block_any<THREADS>(any)) return false;
        auto count = [&](uint32_t k, uint32_t t) { if (t < inside) { if (k >= r.prompt) atomicAdd(&s.word[t], 1u); else atomicOr(&s.word[t], SEEN); } };
        count(tid, h0);
        for (uint32_t k = tid + THREADS; k < r.len; k += THREADS) count(k, (uint32_t)r.history[k] - w0);
        block_sync<THREADS>();
        auto claim = [&](uint32_t t) {
            if (t >= inside) return;
            const uint32_t bit = 1u << (t & 31);
            if (!(atomicOr(&s.seen[t >> 5], bit) & bit)) s.word[t] = __builtin_bit_cast(uint32_t, penalised(T::up(l[t]), s.word[t], r));
        };
        claim(h0);
        for (uint32_t k = tid + THREADS; k < r.len; k += THREADS) claim((uint32_t)r.history[k] - w0);
        block_sync<THREADS>();
        return true;
    }

    template <class T>
    static __device__ void shaped(const tp_logits& a, const RowRules& r, uint64_t row, uint32_t w0, Lds& s, float (&x)[VECS][8]) {
        using S = typename T::S;
        const S* l = (const S*)a.logits + row * a.stride + w0;
        const uint32_t n = a.vocab - w0;                                   // tokens from here to the row's end
        uint32_t allowed[VECS];
        S raw[VECS][8] = {};
#pragma unroll
        for (int v = 0; v < VECS; ++v) allowed[v] = at(v) < n ? (r.mask ? r.mask[(w0 + at(v)) >> 3] : 0xFFu) : 0u;
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            if (!allowed[v]) continue;
            if (at(v) + 8 <= n) {
                __builtin_memcpy(raw[v], l + at(v), sizeof raw[v]);           // rows may start at any element
            } else {
                allowed[v] &= 0xFFu >> (8 - (n - at(v)));
#pragma unroll
                for (int j = 0; j < 8; ++j) if (at(v) + j < n) raw[v][j] = l[at(v) + j];
            }
        }
        const bool hits = repeated<T>(r, l, w0, n < TOKENS ? n : TOKENS, s);
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[v][j] = T::up(raw[v][j]);
            const uint32_t hit = hits ? ((const uint8_t*)s.seen)[at(v) >> 3] : 0u;
            if (hit) {
                float y[8];
                __builtin_memcpy(y, __builtin_assume_aligned(s.word + at(v), 16), sizeof y);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[v][j] = hit >> j & 1 ? y[j] : x[v][j];
            }
            if (r.bias && allowed[v]) {
                float b[8];
                if (at(v) + 8 <= n) {
                    __builtin_memcpy(b, r.bias + w0 + at(v), sizeof b);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) b[j] = at(v) + j < n ? r.bias[w0 + at(v) + j] : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) x[v][j] = x[v][j] + b[j];
            }
            if (allowed[v] != 0xFFu) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[v][j] = allowed[v] >> j & 1 ? x[v][j] : NEG_INF;
            }
        }
    }
};

constexpr int CHUNK_THREADS = 512;
constexpr int CHUNK_VECS = (int)(LOGIT_CHUNK / (CHUNK_THREADS * 8));
using Chunk = Window<CHUNK_THREADS, CHUNK_VECS>;
static_assert(Chunk::TOKENS == LOGIT_CHUNK, "a chunk is whole vectors");

template <class T>
__global__ __launch_bounds__(CHUNK_THREADS) void k_shape(tp_logits a, uint64_t block0, uint32_t chunks, void* out, uint64_t out_stride) {
    using S = typename T::S;
    __shared__ Chunk::Lds s;
    const uint64_t b = block0 + blockIdx.x, row = b / chunks;
    const uint32_t c0 = (uint32_t)(b % chunks) * LOGIT_CHUNK;
    float x[CHUNK_VECS][8];
    Chunk::shaped<T>(a, row_rules(a, row), row, c0, s, x);
    S* o = (S*)out + row * out_stride + c0;
    const uint32_t n = a.vocab - c0;
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v) {
        const uint32_t at = Chunk::at(v);
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
// The first launch reads the logits once: per chunk the largest x and, against it, the sums of the weights of 16 segments of 512
// tokens.  The second joins a row's chunks with one wave: the token's chunk by a scan of the chunks' sums, its segment
// by a scan of the segments', and the token itself in the one segment, which the wave shapes again (1 KB of the row).  A row of
// one chunk does both in the first launch.  Segment sums are 32-bit sums of at most 512 weights in a tree of 9 levels; everything above is summed in 64.
constexpr int SEGMENT = 512;
using Segment = Window<64, 1>;
static_assert(Segment::TOKENS == SEGMENT && CHUNK_SEGMENTS * SEGMENT == LOGIT_CHUNK && CHUNK_VECS * CHUNK_THREADS / 64 == CHUNK_SEGMENTS, "a wave's vector of a chunk is a segment");

struct ChunkLds {
    float max[CHUNK_THREADS / 64];
    uint32_t first;
    ChoicePart part;
};

// The chunk's part of the choice; `out` is complete for the whole block after the next barrier.
__device__ void chunk_part(float (&x)[CHUNK_VECS][8], float t, uint32_t c0, ChunkLds& l, ChoicePart* out) {
    const int wave = (int)(threadIdx.x >> 6);
    float best = NEG_INF;
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[v][j] = countable(x[v][j]);
            best = fmaxf(best, x[v][j]);
        }
    best = wave_max(best);
    if ((threadIdx.x & 63) == 0) l.max[wave] = best;
    if (threadIdx.x == 0) l.first = 0xFFFFFFFFu;
    __syncthreads();
    best = l.max[0];
#pragma unroll
    for (int w = 1; w < CHUNK_THREADS / 64; ++w) best = fmaxf(best, l.max[w]);
    best = read_lane(best, 0);                                            // the same in every lane: the cases below are branches of the wave
    const float k = weight_scale(t);
#pragma unroll
    for (int v = 0; v < CHUNK_VECS; ++v) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = best > NEG_INF ? weight(x[v][j], best, k) : 0.0f;
        const float sum = wave_sum(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
        if ((threadIdx.x & 63) == 0) out->sum[v * (CHUNK_THREADS / 64) + wave] = sum;
    }
    if (t == 0.0f) {                                                      // the lowest token of the largest x
        uint32_t first = 0xFFFFFFFFu;
#pragma unroll
        for (int v = CHUNK_VECS - 1; v >= 0; --v)
#pragma unroll
            for (int j = 7; j >= 0; --j) if (x[v][j] == best) first = c0 + Chunk::at(v) + j;
        if (first != 0xFFFFFFFFu) atomicMin(&l.first, first);
        __syncthreads();
    }
    if (threadIdx.x == 0) { out->best = best; out->token = (int32_t)l.first; }
}

// Joins a row's chunks: all lanes of one wave.
template <class T>
__device__ void join_row(const tp_logits& a, uint64_t row, uint32_t chunks, const ChoicePart* p, float t, const float* uniform, int32_t* tokens, float* logprob, Segment::Lds& s) {
    const uint32_t lane = threadIdx.x & 63;
    float best = NEG_INF;
    for (uint32_t c = lane; c < chunks; c += 64) best = fmaxf(best, p[c].best);
    best = wave_max(best);
    if (!(best > NEG_INF)) {
        if (lane == 0) {
            tokens[row] = -1;
            if (logprob) logprob[row] = NEG_INF;
        }
        return;
    }
    const float k = weight_scale(t);
    auto share = [&](uint32_t c) {
        if (c >= chunks || !(p[c].best > NEG_INF)) return 0.0;
        double w = 0.0;
#pragma unroll
        for (int i = 0; i < CHUNK_SEGMENTS; ++i) w += (double)p[c].sum[i];
        return w * (double)weight(p[c].best, best, k);
    };
    double sum = 0.0;
    uint32_t greedy = 0xFFFFFFFFu;
    for (uint32_t c = lane; c < chunks; c += 64) {
        sum += share(c);
        if (p[c].best == best && (uint32_t)p[c].token < greedy) greedy = (uint32_t)p[c].token;
    }
    sum = wave_sum(sum);
    if (t == 0.0f) {
        for (int d = 32; d; d >>= 1) {
            const uint32_t o = (uint32_t)__shfl_xor((int)greedy, d, 64);
            greedy = o < greedy ? o : greedy;
        }
        if (lane == 0) {
            tokens[row] = (int32_t)greedy;
            if (logprob) logprob[row] = (float)-log(sum);
        }
        return;
    }
    // Where rounding, or a `uniform` of 1 or more, leaves no place whose cumulative weight exceeds the target, the last place
    // of a weight above 0 is taken, at every level.
    double target = (double)uniform[row] * sum;
    uint32_t chunk = 0;
    {
        double carry = 0.0, before = 0.0;
        bool found = false;
        for (uint32_t c0 = 0; c0 < chunks && !found; c0 += 64) {
            const double w = share(c0 + lane), incl = carry + wave_scan(w);
            const uint64_t live = __ballot(w > 0.0), over = __ballot(w > 0.0 && incl > target);
            if (live) {
                found = over != 0;
                const int at = found ? __builtin_ctzll(over) : 63 - __builtin_clzll(live);
                chunk = c0 + (uint32_t)at;
                before = __shfl(incl - w, at, 64);
            }
            carry = __shfl(incl, 63, 64);
        }
        target = (target - before) / (double)weight(p[chunk].best, best, k);
    }
    uint32_t segment;
    {
        const double w = lane < CHUNK_SEGMENTS ? (double)p[chunk].sum[lane] : 0.0, incl = wave_scan(w);
        const uint64_t live = __ballot(w > 0.0), over = __ballot(w > 0.0 && incl > target);
        segment = (uint32_t)(over ? __builtin_ctzll(over) : 63 - __builtin_clzll(live));
        target -= __shfl(incl - w, (int)segment, 64);
    }
    const float chunk_best = p[chunk].best;
    const uint32_t w0 = chunk * LOGIT_CHUNK + segment * SEGMENT;
    float x[1][8];
    Segment::shaped<T>(a, row_rules(a, row), row, w0, s, x);
    double cum = 0.0;
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        w[j] = weight(countable(x[0][j]), chunk_best, k);
        cum += (double)w[j];
    }
    double run = wave_scan(cum) - cum;
    uint32_t first = 8, last = 8;
    float x_first = 0.0f, x_last = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        run += (double)w[j];
        if (w[j] > 0.0f) {
            last = (uint32_t)j; x_last = x[0][j];
            if (first == 8 && run > target) { first = (uint32_t)j; x_first = x[0][j]; }
        }
    }
    const uint64_t over = __ballot(first < 8), live = __ballot(last < 8);
    const uint32_t at = (uint32_t)(over ? __builtin_ctzll(over) : 63 - __builtin_clzll(live));
    if (lane == at) {
        tokens[row] = (int32_t)(w0 + lane * 8 + (over ? first : last));
        if (logprob) logprob[row] = log_probability(over ? x_first : x_last, best, t, sum);
    }
}

template <class T>
__global__ __launch_bounds__(CHUNK_THREADS) void k_choose(tp_logits a, uint64_t block0, uint32_t chunks, const float* temperature, const float* uniform,
                                                          int32_t* tokens, float* logprob, ChoicePart* parts) {
    __shared__ union { Chunk::Lds chunk; Segment::Lds segment; } s;
    __shared__ ChunkLds l;
    const uint64_t b = block0 + blockIdx.x, row = b / chunks;
    const uint32_t c0 = (uint32_t)(b % chunks) * LOGIT_CHUNK;
    float x[CHUNK_VECS][8];
    Chunk::shaped<T>(a, row_rules(a, row), row, c0, s.chunk, x);
    const float t = temperature_of(temperature, uniform, row);
    chunk_part(x, t, c0, l, chunks > 1 ? parts + b : &l.part);
    if (chunks > 1) return;
    __syncthreads();
    if (threadIdx.x < 64) join_row<T>(a, row, 1, &l.part, t, uniform, tokens, logprob, s.segment);
}

template <class T>
__global__ __launch_bounds__(64) void k_choose_join(tp_logits a, uint64_t row0, uint32_t chunks, const float* temperature, const float* uniform,
                                                    int32_t* tokens, float* logprob, const ChoicePart* parts) {
    __shared__ Segment::Lds s;
    const uint64_t row = row0 + blockIdx.x;
    join_row<T>(a, row, chunks, parts + row * chunks, temperature_of(temperature, uniform, row), uniform, tokens, logprob, s);
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

// first entry in [lo, hi) whose token is at least t, by one thread
__device__ inline uint32_t lower_entry(const uint2* entry, uint32_t lo, uint32_t hi, uint32_t t) {
    while (lo < hi) {
        const uint32_t m = lo + (hi - lo) / 2;
        if (entry[m].x < t) lo = m + 1; else hi = m;
    }
    return lo;
}
// the same by a wave, 64 probes a step: the loads of a step are in flight together, where one thread's would follow one another
__device__ inline uint32_t lower_entry_wave(const uint2* entry, uint32_t lo, uint32_t hi, uint32_t t) {
    while (lo < hi) {
        const uint32_t step = (hi - lo + 63) / 64, m = lo + (threadIdx.x & 63) * step;
        const uint32_t below = (uint32_t)__popcll(__ballot(m < hi && entry[m].x < t));   // the probes ascend: the first `below` of them
        if (below == 0) return lo;
        const uint32_t last = lo + (below - 1) * step;
        lo = last + 1;
        hi = last + step < hi ? last + step : hi;
    }
    return lo;
}

// A block writes MASK_PIECE words of one row: cleared in LDS, the list's entries that fall into the piece set there, stored
// in 16-byte pieces.  Of a list longer than a few rounds of the block only the piece's own part is read.
constexpr uint32_t MASK_PIECE = 1024;
__global__ __launch_bounds__(256) void k_grammar_mask(DevGrammar g, const int32_t* states, uint64_t block0, uint32_t pieces, uint32_t* mask, uint64_t mask_stride) {
    __shared__ alignas(16) uint32_t bits[MASK_PIECE];
    const uint64_t b = block0 + blockIdx.x, row = b / pieces;
    const uint32_t w0 = (uint32_t)(b % pieces) * MASK_PIECE, words = (g.n_tokens + 31) / 32;
    List q = list_of(g, states, row);
    *(uint4*)(bits + threadIdx.x * 4) = make_uint4(0, 0, 0, 0);
    const uint32_t t0 = w0 * 32;
    if (t0 && q.hi - q.lo > 1024) q.lo = lower_entry_wave(g.entry, q.lo, q.hi, t0);
    __syncthreads();
    for (uint32_t e = q.lo + threadIdx.x; e < q.hi; e += 256) {
        const uint2 en = g.entry[e];
        const uint32_t t = en.x - t0;
        if (en.x >= t0 + MASK_PIECE * 32) break;
        if (en.x >= t0 && may(en.y, q.tags, g)) atomicOr(&bits[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
    uint32_t* out = mask + row * mask_stride + w0;
    const uint32_t n = words - w0, at = threadIdx.x * 4;
    if (at + 4 <= n) {
        __builtin_memcpy(out + at, __builtin_assume_aligned(bits + at, 16), 16);
    } else {
        for (uint32_t j = at; j < n && j < at + 4; ++j) out[j] = bits[j];
    }
}

// Moves a row on by an entry, and appends its token.
__device__ inline void take_entry(const tp_logits& a, uint64_t row, uint2 entry, int32_t* states, int append) {
    states[2 * row] = (int32_t)(entry.y & MOVE_PLACE);
    if (entry.y >> MOVE_SHIFT == MOVE_COMMA) states[2 * row + 1] += 1;
    if (append) {
        const uint32_t n = clamp_len(a.history_len[row], a.history_cap);
        a.history[row * a.history_stride + n] = (int32_t)entry.x;            // the caller has seen that there is room
        a.history_len[row] = (int32_t)n + 1;
    }
}

__device__ inline bool has_room(const tp_logits& a, uint64_t row, int append) { return !append || clamp_len(a.history_len[row], a.history_cap) < a.history_cap; }

// The choice among a row's list.  THREADS threads hold EACH entries apiece: entry, logit and bias of all of them are loaded before any is used,
// so that a list costs two rounds of memory latency (entries, then what they point to) whatever its length up to
// THREADS * EACH.  Only the listed tokens' logits are read.  History tokens are looked up among the list's ascending tokens in LDS.  A
// longer list is worked on in pieces, twice: for the largest x and the sum, and for the place.
template <int THREADS, int EACH>
struct Step {
    static constexpr uint32_t PIECE = THREADS * EACH;
    static constexpr int WAVES = THREADS / 64, SEGMENTS = WAVES * EACH;      // a wave's 64 entries of one round are a segment, in token order
    struct Lds {
        uint32_t token[PIECE];
        uint32_t cnt[PIECE];
        float sum[SEGMENTS];
        float max[WAVES];
        uint32_t first;
    };

    // x of the m entries from e0: entry i of the piece is thread i % THREADS's number i / THREADS; -infinity where it may not be taken
    template <class T>
    static __device__ void shaped(const DevGrammar& g, const tp_logits& a, const RowRules& r, uint64_t row, uint32_t tags, uint32_t e0, uint32_t m, Lds& s, uint2 (&en)[EACH], float (&x)[EACH]) {
        const typename T::S* l = (const typename T::S*)a.logits + row * a.stride;
        const uint32_t tid = threadIdx.x;
        bool ok[EACH];
        typename T::S raw[EACH];
        float b[EACH];
#pragma unroll
        for (int v = 0; v < EACH; ++v) en[v] = (uint32_t)v * THREADS + tid < m ? g.entry[e0 + v * THREADS + tid] : make_uint2(0xFFFFFFFFu, 0);
#pragma unroll
        for (int v = 0; v < EACH; ++v) {
            ok[v] = en[v].x != 0xFFFFFFFFu && may(en[v].y, tags, g);
            raw[v] = ok[v] ? l[en[v].x] : (typename T::S)0;
            b[v] = ok[v] && r.bias ? r.bias[en[v].x] : 0.0f;
        }
        uint32_t c[EACH] = {};
        if (r.len) {
            block_sync<THREADS>();                                           // the piece before is done with the tables
#pragma unroll
            for (int v = 0; v < EACH; ++v)
                if ((uint32_t)v * THREADS + tid < m) { s.token[v * THREADS + tid] = en[v].x; s.cnt[v * THREADS + tid] = 0; }
            block_sync<THREADS>();
            for (uint32_t k = tid; k < r.len; k += THREADS) {
                const uint32_t h = (uint32_t)r.history[k];
                uint32_t lo = 0, hi = m;
                while (lo < hi) {
                    const uint32_t mid = (lo + hi) / 2;
                    if (s.token[mid] < h) lo = mid + 1; else hi = mid;
                }
                if (lo < m && s.token[lo] == h) {
                    if (k >= r.prompt) atomicAdd(&s.cnt[lo], 1u); else atomicOr(&s.cnt[lo], SEEN);
                }
            }
            block_sync<THREADS>();
#pragma unroll
            for (int v = 0; v < EACH; ++v) if ((uint32_t)v * THREADS + tid < m) c[v] = s.cnt[v * THREADS + tid];
        }
#pragma unroll
        for (int v = 0; v < EACH; ++v) {
            float y = penalised(T::up(raw[v]), c[v], r);
            if (r.bias) y = y + b[v];
            x[v] = ok[v] ? countable(y) : NEG_INF;
        }
    }

    // the largest value of the block, in every thread
    static __device__ float block_max(float v, Lds& s) {
        v = wave_max(v);
        if constexpr (WAVES > 1) {
            if ((threadIdx.x & 63) == 0) s.max[threadIdx.x >> 6] = v;
            block_sync<THREADS>();
            v = wave_max(s.max[threadIdx.x % WAVES]);
            block_sync<THREADS>();
        }
        return v;
    }
    // the segments' sums of the weights against `best`, into LDS
    static __device__ void segment_sums(const float (&x)[EACH], float best, float k, Lds& s) {
#pragma unroll
        for (int v = 0; v < EACH; ++v) {
            const float w = wave_sum(best > NEG_INF ? weight(x[v], best, k) : 0.0f);
            if ((threadIdx.x & 63) == 0) s.sum[v * WAVES + (threadIdx.x >> 6)] = w;
        }
        block_sync<THREADS>();
    }
    static __device__ double segment(const Lds& s, uint32_t i) { return i < (uint32_t)SEGMENTS ? (double)s.sum[i] : 0.0; }
    static __device__ double piece_sum(const Lds& s) {
        double w = 0.0;
        for (uint32_t i = threadIdx.x & 63; i < (uint32_t)SEGMENTS; i += 64) w += (double)s.sum[i];
        return wave_sum(w);
    }

    template <class T>
    static __device__ void run(const DevGrammar& g, const tp_logits& a, uint64_t row, const List& q, const float* temperature, const float* uniform, int32_t* states,
                               int32_t* tokens, float* logprob, int append, Lds& s) {
        const RowRules r = row_rules(a, row);
        const float t = temperature_of(temperature, uniform, row), k = weight_scale(t);
        const bool one = q.hi - q.lo <= PIECE, room = has_room(a, row, append);
        const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
        uint2 en[EACH];
        float x[EACH], best = NEG_INF;
        double sum = 0.0;
        for (uint32_t p = q.lo; p < q.hi; p += PIECE) {
            shaped<T>(g, a, r, row, q.tags, p, q.hi - p < PIECE ? q.hi - p : PIECE, s, en, x);
            float pb = NEG_INF;
#pragma unroll
            for (int v = 0; v < EACH; ++v) pb = fmaxf(pb, x[v]);
            pb = read_lane(block_max(pb, s), 0);
            if (pb > best) {
                sum = best > NEG_INF ? sum * (double)weight(best, pb, k) : 0.0;
                best = pb;
            }
            segment_sums(x, best, k, s);
            sum += piece_sum(s);
            if (!one) block_sync<THREADS>();                                 // before the next piece's sums
        }
        if (!(best > NEG_INF) || !room) {
            if (threadIdx.x == 0) {
                tokens[row] = -1;
                if (logprob) logprob[row] = NEG_INF;
            }
            return;
        }
        // Greedy: the first entry of the largest x.  Sampled: the first whose cumulative weight exceeds the target; where there is none (rounding, or
        // a `uniform` of 1 or more) the last of a weight above 0.
        const double target = t > 0.0f ? (double)uniform[row] * sum : 0.0;
        double carry = 0.0;
        bool found = false, mine = false;
        uint2 entry = make_uint2(0, 0);
        float x_at = best;
        for (uint32_t p = q.lo; p < q.hi && !found; p += PIECE) {
            if (!one) shaped<T>(g, a, r, row, q.tags, p, q.hi - p < PIECE ? q.hi - p : PIECE, s, en, x);
            if (t == 0.0f) {
                if (threadIdx.x == 0) s.first = 0xFFFFFFFFu;
                block_sync<THREADS>();
#pragma unroll
                for (int v = 0; v < EACH; ++v) if (x[v] == best) atomicMin(&s.first, (uint32_t)v * THREADS + threadIdx.x);
                block_sync<THREADS>();
                const uint32_t first = s.first;
                found = first != 0xFFFFFFFFu;
#pragma unroll
                for (int v = 0; v < EACH; ++v) if (found && first == (uint32_t)v * THREADS + threadIdx.x) { mine = true; entry = en[v]; }
                if (!one) block_sync<THREADS>();
                continue;
            }
            if (!one) segment_sums(x, best, k, s);
            // the piece's segment: every wave finds it
            int at = -1;
            double before = 0.0, in_piece = 0.0;
            for (uint32_t i0 = 0; i0 < (uint32_t)SEGMENTS && !found; i0 += 64) {
                const double w = segment(s, i0 + lane), incl = carry + in_piece + wave_scan(w);
                const uint64_t live = __ballot(w > 0.0), over = __ballot(w > 0.0 && incl > target);
                if (live) {
                    found = over != 0;
                    const int to = found ? __builtin_ctzll(over) : 63 - __builtin_clzll(live);
                    at = (int)i0 + to;
                    before = __shfl(incl - w, to, 64);
                }
                in_piece = __shfl(incl, 63, 64) - carry;
            }
            if (at >= 0) mine = false;                                       // a later place than any before
            if (at >= 0 && at % WAVES == wave) {
                float xs = NEG_INF;
                uint2 es = make_uint2(0, 0);
#pragma unroll
                for (int v = 0; v < EACH; ++v) if (v == at / WAVES) { xs = x[v]; es = en[v]; }
                const float w = weight(xs, best, k);
                const double incl = before + wave_scan((double)w);
                const uint64_t live = __ballot(w > 0.0f), over = __ballot(w > 0.0f && incl > target);
                const int to = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(live);
                if (lane == to) { mine = true; entry = es; x_at = xs; }
            }
            carry += in_piece;
            if (!one) block_sync<THREADS>();
        }
        if (mine) {
            tokens[row] = (int32_t)entry.x;
            if (logprob) logprob[row] = log_probability(x_at, best, t, sum);
            take_entry(a, row, entry, states, append);
        }
    }
};

// A block per row.  Most places of a tag line have a handful of tokens, and the places where a tag begins thousands: a list of up to 64
// is the work of one wave, which needs no barrier, and the block's other waves are done at once.
constexpr int STEP_THREADS = 1024;
using LongStep = Step<STEP_THREADS, 8>;
using ShortStep = Step<64, 1>;

template <class T>
__global__ __launch_bounds__(STEP_THREADS) void k_grammar_step(DevGrammar g, tp_logits a, uint64_t row0, const float* temperature, const float* uniform,
                                                               int32_t* states, int32_t* tokens, float* logprob, int append) {
    __shared__ union { LongStep::Lds l; ShortStep::Lds s; } lds;
    const uint64_t row = row0 + blockIdx.x;
    const List q = list_of(g, states, row);
    if (q.hi - q.lo > ShortStep::PIECE) {
        __syncthreads();                                                     // every wave has read the state before one moves it
        LongStep::run<T>(g, a, row, q, temperature, uniform, states, tokens, logprob, append, lds.l);
    } else if (threadIdx.x < 64) {
        ShortStep::run<T>(g, a, row, q, temperature, uniform, states, tokens, logprob, append, lds.s);
    }
}

// The move by the caller's own tokens: a thread per row.
__global__ __launch_bounds__(256) void k_grammar_advance(DevGrammar g, tp_logits a, int32_t* states, const int32_t* tokens, int append) {
    const uint64_t row = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= a.rows) return;
    const int32_t token = tokens[row];
    if (token == -1 || !has_room(a, row, append)) return;
    const List q = list_of(g, states, row);
    const uint32_t e = token < 0 ? q.hi : lower_entry(g.entry, q.lo, q.hi, (uint32_t)token);
    const uint2 entry = e < q.hi ? g.entry[e] : make_uint2(0xFFFFFFFFu, 0);
    if (entry.x == (uint32_t)token && may(entry.y, q.tags, g)) take_entry(a, row, entry, states, append);
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
        if (t < g.n_tokens) n += g.span[t].y;
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
        uint2 span = make_uint2(0, 0);
        if (k0 + lane < w.last) {
            const uint32_t t = (uint32_t)tokens[row * stride + k0 + lane];
            if (t < g.n_tokens) span = g.span[t];
        }
        uint32_t incl = span.y;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)incl, d, 64);
            if ((int)lane >= d) incl += o;
        }
        const uint64_t to = at + incl - span.y;
        for (uint32_t j = 0; j < span.y; ++j) if (to + j < capacity) arena[to + j] = g.text[span.x + j];
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
            hipLaunchKernelGGL(k_choose_join<T>, dim3(n), dim3(64), 0, (hipStream_t)io.stream, io, b, chunks, temperature, uniform, tokens, logprob, parts);
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
