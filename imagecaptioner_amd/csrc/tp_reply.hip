// Kernels that write replies under the pipeline's rules: logit shaping, the choice of a token, the tag-line grammar's masks
// and steps, and the written tokens as text.  The formulas are in include/tagpipe.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "tp_reply.h"
#include "tp_launch.h"

namespace tp {

namespace {

constexpr uint32_t SEEN = 0x80000000u;         // a token's count word: stands in the history; below it: how often behind the prompt
constexpr float NEG_INF = -__builtin_inff();

// ---- element types --------------------------------------------------------------------------------------------------------
// Pointers into device memory as the kernels hold them: told to be global memory, so that their accesses are global ones with
// the row's start in scalar registers.
template <class E>
using Glob = const E __attribute__((address_space(1)))*;
template <class E>
__device__ inline Glob<E> glob(const E* p) { return (Glob<E>)p; }
typedef uint32_t Words4 __attribute__((ext_vector_type(4)));
template <class E> struct At;                     // four words at an address that is only a multiple of an element's size
template <> struct At<uint16_t> { typedef Words4 W __attribute__((aligned(2))); };
template <> struct At<uint32_t> { typedef Words4 W __attribute__((aligned(4))); };

// Logits of every type are worked on in 32 bits; the one rounding back to 16 bits (to nearest, ties to even) is the store of
// tp_shape_logits.  S: an element's bits; VEC: groups of four words that eight elements take.
struct TF32 {
    using S = uint32_t;
    static constexpr int VEC = 2;
    static __device__ float up(S v) { return __builtin_bit_cast(float, v); }
    static __device__ S down(float v) { return __builtin_bit_cast(uint32_t, v); }
    static __device__ void up8(const Words4 (&d)[2], float (&x)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = up(d[j >> 2][j & 3]);
    }
    static __device__ void down8(const float (&x)[8], Words4 (&d)[2]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j >> 2][j & 3] = down(x[j]);
    }
};
template <class T>
struct Pairs {                                      // two elements a word
    static __device__ void up8(const Words4 (&d)[1], float (&x)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            x[j] = T::up((uint16_t)d[0][j >> 1]);
            x[j + 1] = T::up((uint16_t)(d[0][j >> 1] >> 16));
        }
    }
    static __device__ void down8(const float (&x)[8], Words4 (&d)[1]) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) d[0][j >> 1] = (uint32_t)T::down(x[j]) | (uint32_t)T::down(x[j + 1]) << 16;
    }
};
struct TF16 : Pairs<TF16> {
    using S = uint16_t;
    static constexpr int VEC = 1;
    static __device__ float up(S v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ S down(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};
struct TBF16 : Pairs<TBF16> {
    using S = uint16_t;
    static constexpr int VEC = 1;
    static __device__ float up(S v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
    static __device__ S down(float v) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        if (v != v) return (uint16_t)((u >> 16) | 0x40u);
        return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
    }
};

// ---- one row's rules ------------------------------------------------------------------------------------------------------
struct RowRules {
    Glob<int32_t> history;        // `len` of them
    uint32_t len, prompt;
    float rep, freq, pres;
    Glob<float> bias;             // null: none
    Glob<uint8_t> mask;           // the mask row's bytes, null: none
};

__device__ inline uint32_t clamp_len(int32_t n, uint32_t cap) { return n < 0 ? 0u : (uint32_t)n > cap ? cap : (uint32_t)n; }

// Every rule is one load from where it stands or from a zero, and none waits for another: a row's block begins with one round of
// memory latency instead of one per rule.
__device__ const uint32_t no_rule[1] = {0};
__device__ inline RowRules row_rules(const tp_logits& a, uint64_t row) {
    const auto none = glob((const float*)no_rule);
    const auto none_i = glob((const int32_t*)no_rule);
    const int32_t len = *(a.history_len ? glob(a.history_len) + row : none_i), prompt = *(a.prompt_len ? glob(a.prompt_len) + row : none_i);
    const float rep = *(a.repetition ? glob(a.repetition) + row : none), freq = *(a.frequency ? glob(a.frequency) + row : none), pres = *(a.presence ? glob(a.presence) + row : none);
    const uint32_t bias = (uint32_t)*(a.bias_row ? glob(a.bias_row) + row : none_i), mask = (uint32_t)*(a.mask_row ? glob(a.mask_row) + row : none_i);
    RowRules r;
    const bool asked = a.history && (a.repetition || a.frequency || a.presence);       // else nothing asks what the history holds
    r.len = asked ? (a.history_len ? clamp_len(len, a.history_cap) : a.history_cap) : 0u;
    r.history = glob(a.history) + row * a.history_stride;
    r.prompt = clamp_len(prompt, a.history_cap);
    r.rep = a.repetition ? rep : 1.0f;
    r.freq = freq;
    r.pres = pres;
    r.bias = a.bias && bias < a.n_bias ? glob(a.bias) + (uint64_t)bias * a.bias_stride : nullptr;
    r.mask = a.mask && mask < a.n_masks ? (Glob<uint8_t>)(glob(a.mask) + (uint64_t)mask * a.mask_stride) : nullptr;
    return r;
}
template <class T>
__device__ inline Glob<typename T::S> logit_row(const tp_logits& a, uint64_t row) { return glob((const typename T::S*)a.logits) + row * a.stride; }

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
__device__ inline float read_lane(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }

// One instruction a step (the waits are for the step before, whose result another lane reads); a NaN is passed over.
__device__ inline float wave_max(float v) {
    asm("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:1 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:2 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:4 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n\t"
        "s_nop 1" : "+v"(v));
    return read_lane(v, 63);
}
// sum of the lanes up to and including this one
__device__ inline uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}
template <int CTRL, int ROWS>
__device__ inline double dpp(double v) {                                      // 0 where no lane is the source
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline double read_lane(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline double wave_scan(double v) {
    v += dpp<0x111, 0xF>(v);
    v += dpp<0x112, 0xF>(v);
    v += dpp<0x114, 0xF>(v);
    v += dpp<0x118, 0xF>(v);
    v += dpp<0x142, 0xA>(v);
    v += dpp<0x143, 0xC>(v);
    return v;
}
__device__ inline double wave_sum(double v) { return read_lane(wave_scan(v), 63); }
// in the last of eight neighbouring lanes, their sum
__device__ inline double eight_lanes_sum(double v) {
    v += dpp<0x111, 0xF>(v);
    v += dpp<0x112, 0xF>(v);
    v += dpp<0x114, 0xF>(v);
    return v;
}

// ---- weights ------------------------------------------------------------------------------------------------------------------
// z = x / T is rounded to 32 bits, as the formula says, by the quotient's own rounding: with 131072 tokens a border between two of them lies in every
// hundred-thousandth of the weight, and unrounded quotients choose another token than the rounded ones in one row of 1100 (28 of 30720).
// A token's weight is 2^(z * LOG2E - c), c = best * LOG2E rounded once for the tokens that are summed together: one fused multiply-add and one power.  c is no
// more than a common scale, known exactly to whoever joins sums of different c, so that a weight is off by LOG2E's rounding and the fma's, each half a step
// relative in the exponent, and by the power's own step.  From |c| = 2^30 on, neighbouring numbers lie so far apart that only the largest z weighs anything, and c's own rounding
// (32 at the most below it) would grow out of the powers' range.
constexpr float LOG2E = 1.44269504088896341f;
struct Scale {
    float c, best;
    bool equal;                   // weigh by equality with the largest
    __device__ Scale(float best_) : c(best_ * LOG2E), best(best_), equal(!(fabsf(best_ * LOG2E) < 0x1p30f)) {}
    __device__ float weight(float z) const { return equal ? (z == best ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(__builtin_fmaf(z, LOG2E, -c)); }
    // what a sum of the weights of another scale counts for in this one's
    __device__ double of(float other_best) const { return equal || !(other_best > NEG_INF) ? (other_best == best ? 1.0 : 0.0) : (double)__builtin_amdgcn_exp2f(other_best * LOG2E - c); }
    // ln of the weight's share of `sum`: of the weight as it was summed, so that a token that is alone has 0 exactly; of its exponent where that is
    // next to nothing
    __device__ float log_share(float z, double sum) const {
        const float w = weight(z);
        return (float)(w > 1e-30f ? log((double)w / sum) : ((double)z * (double)LOG2E - (double)c) * 0.69314718055994531 - log(sum));
    }
};
__device__ inline float temperature_of(const float* temperature, const float* uniform, uint64_t row) {
    const float t = temperature && uniform ? temperature[row] : 0.0f;
    return t > 0.0f ? t : 0.0f;
}
// a NaN counts as -infinity in a choice
__device__ inline float countable(float x) { return x == x ? x : NEG_INF; }
// the z of the weights, never a NaN; temper: the temperature, 1 where the largest is chosen
__device__ inline float z_of(float x, float temper) { return countable(x / temper); }
// The same quotient of many x by two operations.  hi + lo is 1 / temper to 48 bits, hi below it, so that x * hi + x * lo is off by 2^-46 before the one
// rounding that matters; with lo above 0 an infinite x gives the infinity that it should.  A temper out of bounds gives NaNs, whoever has them divides.
struct Inverse {
    float hi, lo;
    __device__ Inverse(float temper) {
        hi = 1.0f / temper;
        float rest = __builtin_fmaf(-hi, temper, 1.0f);
        if (rest < 0.0f) {
            hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, hi) - 1);
            rest = __builtin_fmaf(-hi, temper, 1.0f);
        }
        lo = fmaxf(rest * hi, 1.17549435e-38f);
        if (!(temper > 1e-30f && temper < 1e30f)) hi = __builtin_nanf("");
    }
    __device__ float z(float x) const { return __builtin_fmaf(x, hi, x * lo); }
};
__device__ inline float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

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

// ---- a row in segments ----------------------------------------------------------------------------------------------------------
constexpr uint32_t SEGMENT = REPLY_SEGMENT;
constexpr int VECS = (int)(SEGMENT / (64 * 8));
extern __shared__ __attribute__((aligned(16))) uint32_t dynamic_lds[];

// A wave's segment of a row: two vectors of eight tokens a lane, the lane's second 512 tokens behind its first.  A vector that the row's end cuts is loaded
// from eight tokens before the end instead, so that every lane loads alike; its first `cut` tokens belong to the vector before and
// are left out by their bits of `take`.  (TINY: a vocabulary of fewer than eight tokens, loaded one by one.)
template <class T>
struct Held {
    Words4 d[VECS][T::VEC], b[VECS][2];                                       // logits, biases
    uint32_t take[VECS];                                                      // tokens that are this lane's, inside the row and allowed by the mask
};
__device__ inline uint32_t lane_at(uint32_t segment) { return segment * SEGMENT + (threadIdx.x & 63) * 8; }
// how far the vector at t reaches over the end of n tokens: 0 not, 8 it lies behind it
__device__ inline uint32_t cut_of(uint32_t t, uint32_t n) { return t + 8 <= n ? 0u : t < n ? t + 8 - n : 8u; }

template <class E>
using Vec = const typename At<E>::W __attribute__((address_space(1)));

// The mask's bytes of a segment, any segment.  The logits of eight tokens that are all forbidden are not loaded, so the loads wait for these; whoever goes through
// several segments loads the bytes a segment ahead.
__device__ inline void load_mask(const RowRules& r, uint32_t w0, uint32_t n, uint32_t segment, uint32_t (&bits)[VECS]) {
    if (!r.mask) return;
#pragma unroll
    for (int v = 0; v < VECS; ++v) bits[v] = r.mask[(w0 + std::min(lane_at(segment) + v * 512, n - 1)) >> 3];
}

// `n`: tokens from the window's start to the row's end
// The loads go through the caches, where logits that a product has just written still are if it writes them to one place step after step, as a loop over an allocator's blocks does: choosing
// for 512 rows of 131072 behind such a product takes 37 us instead of the 41 of loads past them, for 512 of 50021 23.0 instead of 23.7.  With three places in turn it takes 44.5
// instead of 42, 23.2 instead of 23.9; where nothing is in the caches 42.2 instead of 41.2, 24.1 instead of 23.9.
// BIAS_LAST: behind the logits where those wait for nothing (choosing for 512 rows: 43.8 -> 42.9 us), before them in shaping (256 rows: 53.0 -> 51.9).
template <class T, bool TINY, bool BIAS_LAST>
__device__ inline void load_segment(const RowRules& r, Glob<typename T::S> row, uint32_t w0, uint32_t n, uint32_t segment, const uint32_t (&bits)[VECS], Held<T>& h) {
    using S = typename T::S;
    const uint32_t at = lane_at(segment);
    if (r.bias && !TINY && !BIAS_LAST) {
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            auto* from = (Vec<uint32_t>*)(r.bias + w0 + (int32_t)std::min((int32_t)(at + v * 512), (int32_t)n - 8));
            h.b[v][0] = from[0];
            h.b[v][1] = from[1];
        }
    }
    if constexpr (TINY) {
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            const uint32_t t = at + v * 512, cut = cut_of(t, n);
            h.take[v] = cut < 8 ? (r.mask ? bits[v] : 0xFFu) << cut & 0xFFu : 0u;
#pragma unroll
            for (int g = 0; g < T::VEC; ++g) h.d[v][g] = Words4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t e = cut < 8 && (uint32_t)j >= cut ? (uint32_t)row[j - cut] : 0u;
                if constexpr (sizeof(S) == 4) h.d[v][j >> 2][j & 3] = e;
                else h.d[v][0][j >> 1] |= e << (16 * (j & 1));
            }
        }
        return;
    }
    if (r.mask) {
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            const uint32_t t = at + v * 512;
            h.take[v] = bits[v] << cut_of(t, n) & 0xFFu;
            if (h.take[v])
#pragma unroll
                for (int g = 0; g < T::VEC; ++g) {
                    auto* from = (Vec<S>*)(row + (int32_t)std::min((int32_t)t, (int32_t)n - 8)) + g;
                    h.d[v][g] = *from;
                }
        }
    } else {
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            const uint32_t t = at + v * 512;
            h.take[v] = 0xFFu << cut_of(t, n) & 0xFFu;
#pragma unroll
            for (int g = 0; g < T::VEC; ++g) {
                auto* from = (Vec<S>*)(row + (int32_t)std::min((int32_t)t, (int32_t)n - 8)) + g;
                h.d[v][g] = *from;
            }
        }
    }
    if (r.bias && BIAS_LAST) {
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            auto* from = (Vec<uint32_t>*)(r.bias + w0 + (int32_t)std::min((int32_t)(at + v * 512), (int32_t)n - 8));
            h.b[v][0] = from[0];
            h.b[v][1] = from[1];
        }
    }
}
// the bias, and -infinity where `take` has no bit
template <class T, bool TINY>
__device__ inline void finish_segment(const RowRules& r, uint32_t n, uint32_t segment, const Held<T>& h, const uint32_t (&take)[VECS], float (&x)[VECS][8]) {
    const uint32_t at = lane_at(segment);
    if (r.bias) {
        if constexpr (TINY) {
#pragma unroll
            for (int v = 0; v < VECS; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) if (take[v] >> j & 1) x[v][j] = x[v][j] + r.bias[j - cut_of(at + v * 512, n)];
        } else {
#pragma unroll
            for (int v = 0; v < VECS; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[v][j] = x[v][j] + __builtin_bit_cast(float, (uint32_t)h.b[v][j >> 2][j & 3]);
        }
    }
#pragma unroll
    for (int v = 0; v < VECS; ++v)
        if (take[v] != 0xFFu) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)take[v], j, 1);   // all ones or none
                x[v][j] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x[v][j]) & keep) | (0xFF800000u & ~keep));
            }
        }
}

// A row's history as a block of THREADS threads goes through it: HELD entries a thread in registers, loaded before
// anything else is, the others again from memory in every pass.
template <int THREADS, int HELD>
struct History {
    static constexpr int HELD_ENTRIES = HELD;
    uint32_t token[HELD];                                                     // as they stand there: nothing waits for them here
    __device__ inline void load(const RowRules& r, uint32_t w0) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const uint32_t k = threadIdx.x % THREADS + i * THREADS;
            token[i] = k < r.len ? (uint32_t)r.history[k] : w0 - 1;              // no token: a distance of 2^32 - 1
        }
    }
    // f(whether the entry counts for frequency and presence, distance from w0, number among the held or -1), for distances below `inside`
    template <class F>
    __device__ inline void each(const RowRules& r, uint32_t w0, uint32_t inside, F&& f) const {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (token[i] - w0 < inside) f(threadIdx.x % THREADS + i * THREADS >= r.prompt, token[i] - w0, i);
        for (uint32_t k = threadIdx.x % THREADS + HELD * THREADS; k < r.len; k += THREADS) {
            const uint32_t h = (uint32_t)r.history[k] - w0;
            if (h < inside) f(k >= r.prompt, h, -1);
        }
    }
};

// ---- shaping ------------------------------------------------------------------------------------------------------------------------
// Bound by reading and writing the logits once: 256 rows of 131071 float32 with 1500 entries of history take 52 us (270 MB, 5.2 TB/s).  A block takes 8192 tokens of one row, a segment a wave; the loads stand in flight while the
// block counts the history in an LDS table of a word per token, of which it clears all and every thread looks at some of the
// row's whole history.  The penalties are worked out where a token's word is not 0.  (The choice below keeps only as many words as
// the history has entries and works each repeated token out once; here, with the vector units idle, its longer chain of
// barriers costs more than it saves: 77 against 54 us for 256 x 131071 float32 with 1500 entries of history.)
// Blocks of SHAPE_FEW waves where a row has no more segments: 4096 rows of 1000 tokens 18.9 -> 8.3 us a pass, of 2048 19.5 -> 10.2, 512 rows as before.
constexpr int SHAPE_WAVES = 8, SHAPE_FEW = 2;

template <class T, bool TINY, bool MASKED, int WAVES>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(8))) void k_shape(tp_logits a, uint64_t row0, void* out, uint64_t out_stride) {
    using S = typename T::S;
    using V = typename At<S>::W __attribute__((address_space(1)));
    constexpr uint32_t THREADS = WAVES * 64, TOKENS = WAVES * SEGMENT;
    __shared__ alignas(16) uint32_t cnt[TOKENS];
    const uint64_t row = row0 + blockIdx.y;
    const uint32_t w0 = blockIdx.x * TOKENS, n = a.vocab - w0;
    const uint32_t g = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), at = lane_at(g);
    auto* o = (S __attribute__((address_space(1)))*)((S*)out + row * out_stride + w0);
    RowRules r = row_rules(a, row);
    if (!MASKED) r.mask = nullptr;                                            // as it is: 256 rows of 131072 bfloat16 take 22.5 us instead of 24.5
    History<THREADS, 4> history;
    history.load(r, w0);
    Held<T> h;
    uint32_t bits[VECS];
    load_mask(r, w0, n, g, bits);
    load_segment<T, TINY, false>(r, logit_row<T>(a, row) + w0, w0, n, g, bits, h);
    if (r.len) {
        for (uint32_t k = threadIdx.x * 4; k < TOKENS; k += THREADS * 4) *(uint4*)(cnt + k) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        history.each(r, w0, std::min(n, TOKENS), [&](bool counted, uint32_t t, int) { if (counted) atomicAdd(&cnt[t], 1u); else atomicOr(&cnt[t], SEEN); });
        __syncthreads();
    }
    if (g * SEGMENT >= n) return;
    float x[VECS][8];
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
        T::up8(h.d[v], x[v]);
        if (r.len) {
            const uint32_t t = at + v * 512, cut = cut_of(t, n);
            if (cut == 0) {
                uint32_t c[8];
                __builtin_memcpy(c, __builtin_assume_aligned(cnt + t, 16), sizeof c);
                if (c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[v][j] = penalised(x[v][j], c[j], r);
                }
            } else if (cut < 8) {
#pragma unroll
                for (int j = 0; j < 8; ++j) if ((uint32_t)j >= cut) x[v][j] = penalised(x[v][j], cnt[t + j - cut], r);
            }
        }
    }
    finish_segment<T, TINY>(r, n, g, h, h.take, x);
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
        const uint32_t t = at + v * 512, cut = cut_of(t, n);
        Words4 d[T::VEC];
        T::down8(x[v], d);
        if (cut == 0) {
#pragma unroll
            for (int k = 0; k < T::VEC; ++k) {
                // Past the caches where a store fills whole lines (64 rows of bfloat16 10.7 -> 9.2 us, shaping and then choosing 26.2 -> 25.0; in 32 bits, where it fills halves,
                // 256 rows 51.7 -> 56.8).
                if constexpr (T::VEC == 1) __builtin_nontemporal_store(d[k], (V*)(o + t) + k);
                else ((V*)(o + t))[k] = d[k];
            }
        } else if (cut < 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) if ((uint32_t)j >= cut) o[t + j - cut] = T::down(x[v][j]);
        }
    }
}

// ---- repeated tokens of a window ------------------------------------------------------------------------------------------------
// For the choice, which the vector units bound: the tokens of the history inside a window of a row are marked in a bitmap, a prefix sum over
// its words ranks them, and the distinct ones' counts are taken in an array as long as the history has room for.  One
// thread per distinct token then works its z out, with a load of the token's own logit, and puts it in the count's place.  The
// vectors leave these tokens out: the penalties' arithmetic, a division among it, is done once per repeated token instead
// of once per token of the row.  The first segment's loads are in flight meanwhile.
template <int WAVES, int SEGS>
struct Window {
    static constexpr int THREADS = WAVES * 64;
    static constexpr uint32_t TOKENS = (uint32_t)WAVES * SEGS * SEGMENT, WORDS = TOKENS / 32;
    static constexpr int MINE = (int)((WORDS + THREADS - 1) / THREADS);    // bitmap words of a thread
    struct Lds {
        alignas(16) uint32_t seen[WORDS];
        union {
            uint32_t claimed[WORDS];
            alignas(16) float lane_sum[TOKENS / (8 * VECS)];                  // what the choice makes of every lane's tokens, when `claimed` is done with
        };
        uint32_t rank[WORDS + 1];                                             // distinct tokens before the word
        uint32_t wave[WAVES];
    };
    // `value`, in dynamic LDS: the distinct tokens' z, in token order; as many words as the history has entries, or the window tokens

    static __device__ uint32_t tid() { return threadIdx.x % THREADS; }
    static __device__ uint32_t rank_of(const Lds& l, uint32_t t) { return l.rank[t >> 5] + (uint32_t)__popc(l.seen[t >> 5] & ((1u << (t & 31)) - 1)); }

    // How many distinct tokens of the window of `inside` tokens from w0 the history has; their z stand in `value`.
    template <class T, class H>
    static __device__ uint32_t repeated(const RowRules& r, float temper, const H& history, Glob<typename T::S> row, uint32_t w0, uint32_t inside, Lds& l, uint32_t* value) {
        if (!r.len) return 0;
        const uint32_t words = (inside + SEGMENT - 1) / SEGMENT * (SEGMENT / 32);      // the bitmap's, in whole segments
        for (uint32_t k = tid(); k < words; k += THREADS) l.seen[k] = l.claimed[k] = 0;
        typename T::S held[H::HELD_ENTRIES];                                    // the held entries' own logits and biases, wanted at the end
        float held_bias[H::HELD_ENTRIES];
#pragma unroll
        for (int i = 0; i < H::HELD_ENTRIES; ++i) {
            const uint32_t t = history.token[i] - w0;
            held[i] = t < inside ? row[t] : (typename T::S)0;
            held_bias[i] = t < inside && r.bias ? r.bias[w0 + t] : 0.0f;
        }
        block_sync<THREADS>();
        bool any = false;
        history.each(r, w0, inside, [&](bool, uint32_t t, int) { atomicOr(&l.seen[t >> 5], 1u << (t & 31)); any = true; });
        if (!block_any<THREADS>(any)) return 0;
        uint32_t n[MINE], mine = 0;
#pragma unroll
        for (int i = 0; i < MINE; ++i) { n[i] = tid() * MINE + i < words ? (uint32_t)__popc(l.seen[tid() * MINE + i]) : 0u; mine += n[i]; }
        const uint32_t incl = wave_scan(mine);
        uint32_t before = incl - mine, distinct = 0;
        if constexpr (WAVES > 1) {
            if ((tid() & 63) == 63) l.wave[tid() >> 6] = incl;
            block_sync<THREADS>();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) { if (w < (int)(tid() >> 6)) before += l.wave[w]; distinct += l.wave[w]; }
        } else {
            distinct = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
        }
#pragma unroll
        for (int i = 0; i < MINE; ++i) if (tid() * MINE + i < words) { l.rank[tid() * MINE + i] = before; before += n[i]; }
        if (tid() == 0) l.rank[words] = distinct;
        for (uint32_t k = tid(); k < distinct; k += THREADS) value[k] = 0;
        block_sync<THREADS>();
        history.each(r, w0, inside, [&](bool counted, uint32_t t, int) { if (counted) atomicAdd(&value[rank_of(l, t)], 1u); else atomicOr(&value[rank_of(l, t)], SEEN); });
        block_sync<THREADS>();
        history.each(r, w0, inside, [&](bool, uint32_t t, int at) {
            const uint32_t bit = 1u << (t & 31);
            if (atomicOr(&l.claimed[t >> 5], bit) & bit) return;
            const uint32_t i = rank_of(l, t);
            typename T::S logit = 0;
            float b = 0.0f;
            if (at < 0) {
                logit = row[t];
                if (r.bias) b = r.bias[w0 + t];
            }
#pragma unroll
            for (int h = 0; h < H::HELD_ENTRIES; ++h) if (at == h) { logit = held[h]; b = held_bias[h]; }
            float x = penalised(T::up(logit), value[i], r);
            if (r.bias) x = x + b;
            if (r.mask && !(r.mask[(w0 + t) >> 3] >> (t & 7) & 1)) x = NEG_INF;
            value[i] = __builtin_bit_cast(uint32_t, z_of(x, temper));
        });
        block_sync<THREADS>();
        return distinct;
    }
};

// ---- the choice -------------------------------------------------------------------------------------------------------------
// The first launch reads the logits once and leaves of every segment the sum of its weights and the z that they are relative to.  The second joins a
// row with one wave: the token's segment by a scan of the segments' shares, and the token in that segment, which
// the wave shapes again (1024 tokens of the row).  A row of one window does both in the first launch.  A lane's sixteen weights of a segment are summed in
// 32 bits (five roundings, one more where repeated tokens are among them), everything above in 64: sums in 64 bits from the first weight on take 53.5 us instead of 42.0 for
// 512 rows of 131072 (their LDS leaves one block a unit), 16.6 instead of 16.2 for 48 of 50021.  Against the formula with 64-bit sums, 131072 tokens and temperatures
// of 0.5 .. 1.2, 7 rows of 30720 got another token, always the border's other side, and the border within 2e-8 of the weight from the random number.
//
// What bounds it: 512 rows of 131072 bfloat16 (134 MB, 26 us at a copy's rate) with 256 tokens of history and a bias take 42 us: the vector units
// spend some 260 instructions a segment (powers: 16, four times as long), 29 us of work; the block's start (rules, history and repeated tokens: 6 us) and the join of
// the row (4 us) are chains of latency that no other block hides, since all rows are at work at once.
using OneSegment = Window<1, 1>;
// A block has eight waves of up to 16 segments.  Two blocks share a unit, for their LDS, and so a wave may have 128 registers: with sixteen waves of 64, which had to
// store some of them and copied others, 512 rows of 131072 took 42.0 us instead of 41.1, 48 rows of 50021 under masks 18.5 instead of 17.5, one row of 131072 13.9 instead of 12.8.
// Where there are more rows than units and they have up to 16 segments, blocks of four waves: more rows at work at once hide each other's start and join (sixteen waves / four:
// 4096 rows of 16384 115 / 49 us, 512 of 8000 13.8 / 11.7; with eight waves 300 rows of 16384 14.2 / 13.5, 256 rows 11.6 / 12.1).  So they are for up to four
// segments in any case: the other waves would have nothing to do.
constexpr int CHOICE_WAVES = 8, MOST_SEGS = 16;                               // waves of a block, segments of a wave at the most
constexpr int FEW_WAVES = 4, FEW_SEGS = 4;

// x of a segment without its repeated tokens, which are value[i0 .. i1)
template <class T, bool TINY, class Lds>
__device__ inline void segment_x(const RowRules& r, uint32_t n, uint32_t g, const Held<T>& h, uint32_t distinct, const Lds& l, float (&x)[VECS][8], uint32_t& i0, uint32_t& i1) {
    uint32_t take[VECS];
    i0 = i1 = 0;
#pragma unroll
    for (int v = 0; v < VECS; ++v) take[v] = h.take[v];
    if (distinct) {
        i0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)l.rank[g * (SEGMENT / 32)]);
        i1 = (uint32_t)__builtin_amdgcn_readfirstlane((int)l.rank[(g + 1) * (SEGMENT / 32)]);
        if (i1 > i0) {
#pragma unroll
            for (int v = 0; v < VECS; ++v) {
                const uint32_t t = lane_at(g) + v * 512;
                take[v] &= ~((uint32_t)((const uint8_t*)l.seen)[t >> 3] << cut_of(t, n));
            }
        }
    }
#pragma unroll
    for (int v = 0; v < VECS; ++v) T::up8(h.d[v], x[v]);
    finish_segment<T, TINY>(r, n, g, h, take, x);
}
// the largest z; a NaN among the x may hide others, or be passed over
__device__ inline float segment_largest(const float (&x)[VECS][8], float temper, const uint32_t* value, uint32_t i0, uint32_t i1) {
    float best = NEG_INF;
#pragma unroll
    for (int v = 0; v < VECS; ++v)
#pragma unroll
        for (int j = 0; j < 8; j += 2) best = max3(best, x[v][j], x[v][j + 1]);
    best = z_of(best, temper);                                                      // the quotients are in the order of the x
    for (uint32_t i = i0 + (threadIdx.x & 63); i < i1; i += 64) best = fmaxf(best, __builtin_bit_cast(float, value[i]));
    return wave_max(best);
}

// The lane's sum of a segment's weights.  They are taken against `ref`, and only where they outgrow it, or there is none, against
// the segment's own largest z, which is the wave's `ref` from then on: the shares that the join works with do not mind what they are
// relative to, and the largest need not be found.  With `greedy` it is the segment's largest in any case.
// A NaN among the weights has the segment done again, by divisions and without the NaNs.
template <class T, bool TINY, class Lds, class Next>
__device__ inline float segment_part(const RowRules& r, uint32_t n, uint32_t g, const Held<T>& h, float temper, const Inverse& inverse, bool greedy, float& ref, uint32_t distinct, const Lds& l,
                                          const uint32_t* value, Next&& next) {
    float x[VECS][8];
    uint32_t i0, i1;
    static_assert(VECS == 2, "");
    // A grammar's mask leaves most segments without a token (making the mask and choosing under it for 1024 rows of 131072: 108 -> 58 us; 48 rows of 50021 under masks that leave every
    // segment a few: 17.7 -> 18.5).
    const bool empty = r.mask && __ballot((h.take[0] | h.take[1]) != 0) == 0;
    segment_x<T, TINY>(r, n, g, h, distinct, l, x, i0, i1);
    next();                                                                   // `h` is free for the loads of the wave's next segment
    if (empty) {
        if (greedy) ref = NEG_INF;
        return 0.0f;
    }
    auto repeated = [&](const Scale& scale) {
        double more = 0.0;                                                    // up to sixteen, one after another
        for (uint32_t i = i0 + (threadIdx.x & 63); i < i1; i += 64) more += (double)scale.weight(__builtin_bit_cast(float, value[i]));
        return more;
    };
    if (greedy || ref == NEG_INF) ref = segment_largest(x, temper, value, i0, i1);
    Scale scale(ref);
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(inverse.z(x[v][j]), LOG2E, -scale.c));
        sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    }
    if (i1 > i0) sum = (float)((double)sum + repeated(scale));
    if (__ballot(!(sum < 1e30f)) || scale.equal) {                                      // outgrown, or a NaN, or no scale to go by
#pragma unroll
        for (int v = 0; v < VECS; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[v][j] = z_of(x[v][j], temper);
        ref = segment_largest(x, 1.0f, value, i0, i1);
        scale = Scale(ref);
        sum = 0.0f;
#pragma unroll
        for (int v = 0; v < VECS; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += scale.weight(x[v][j]);
        sum = ref == NEG_INF ? 0.0f : (float)((double)sum + repeated(scale));
    }
    return sum;
}

// Joins a row's segments: all lanes of one wave.  Tables: Chunk where the row's own window stands in LDS (`distinct` of it), OneSegment
// where the segment's repeated tokens are still to be found.
template <class T, class Tables, bool TINY>
__device__ void join_row(const tp_logits& a, const RowRules& r, uint64_t row, uint32_t segments, const ChoicePart* p, float t, const float* uniform, int32_t* tokens,
                         float* logprob, uint32_t distinct, typename Tables::Lds& l, uint32_t* value) {
    constexpr bool HERE = Tables::TOKENS > SEGMENT;
    const uint32_t lane = threadIdx.x & 63;
    float best = NEG_INF;
    for (uint32_t c = lane; c < segments; c += 64) best = fmaxf(best, p[c].best);
    best = wave_max(best);
    if (!(best > NEG_INF)) {
        if (lane == 0) {
            tokens[row] = -1;
            if (logprob) logprob[row] = NEG_INF;
        }
        return;
    }
    const float temper = t > 0.0f ? t : 1.0f;
    const Scale scale(best);
    auto share = [&](uint32_t c) { return c < segments ? p[c].sum * scale.of(p[c].best) : 0.0; };
    double sum = 0.0;
    for (uint32_t c = lane; c < segments; c += 64) sum += share(c);
    sum = wave_sum(sum);
    // Greedy: the first segment that has the largest z.  Sampled: the first whose cumulative share exceeds the target; where there is none (rounding,
    // or a `uniform` of 1 or more) the last of a share above 0, and so within the segment.
    double target = t > 0.0f ? (double)uniform[row] * sum : 0.0, carry = 0.0, before = 0.0;
    uint32_t segment = 0;
    bool found = false;
    for (uint32_t c0 = 0; c0 < segments && !found; c0 += 64) {
        const double w = share(c0 + lane), incl = carry + wave_scan(w);
        const uint64_t live = __ballot(w > 0.0);
        const uint64_t over = t > 0.0f ? __ballot(w > 0.0 && incl > target) : __ballot(c0 + lane < segments && p[c0 + lane].best == best);
        if (over || (live && t > 0.0f)) {
            found = over != 0;
            const int to = found ? __builtin_ctzll(over) : 63 - __builtin_clzll(live);
            segment = c0 + (uint32_t)to;
            before = read_lane(incl - w, to);
        }
        carry = read_lane(incl, 63);
    }
    const Scale within(p[segment].best);
    target = (target - before) / scale.of(within.best);
    const uint32_t w0 = segment * SEGMENT, n = a.vocab - w0, l0 = HERE ? w0 : 0;             // l0: the segment's start within the tables
    const auto from = logit_row<T>(a, row) + w0;
    Held<T> h;
    uint32_t bits[VECS];
    load_mask(r, w0, n, 0, bits);
    if constexpr (HERE) {
        load_segment<T, TINY, false>(r, from, w0, n, 0, bits, h);
    } else {
        History<64, 8> history;
        history.load(r, w0);
        load_segment<T, TINY, false>(r, from, w0, n, 0, bits, h);
        distinct = OneSegment::repeated<T>(r, temper, history, from, w0, std::min(n, SEGMENT), l, value);
    }
    uint32_t at = 0;
    float x_at = best;
    bool done = false;
    double run = 0.0;
    float xs[VECS][8];
#pragma unroll
    for (int v = 0; v < VECS; ++v) T::up8(h.d[v], xs[v]);
    finish_segment<T, TINY>(r, n, 0, h, h.take, xs);
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
        float (&x)[8] = xs[v];
        const uint32_t t0 = l0 + lane_at(0) + v * 512, cut = cut_of(lane_at(0) + v * 512, n);
        const uint32_t hit = distinct && cut < 8 ? (uint32_t)((const uint8_t*)l.seen)[t0 >> 3] << cut & 0xFFu : 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = z_of(x[j], temper);
        if (hit) {
            uint32_t i = Tables::rank_of(l, t0);
#pragma unroll
            for (int j = 0; j < 8; ++j) if (hit >> j & 1) x[j] = __builtin_bit_cast(float, value[i++]);
        }
        float w[8];
        double mine = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = within.weight(x[j]);
            mine += (double)w[j];
        }
        const double incl = run + wave_scan(mine);
        run = read_lane(incl, 63);
        if (done) continue;
        uint32_t first = 8, last = 8;
        float x_first = best, x_last = best;
        if (t > 0.0f) {
            double cum = incl - mine;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                cum += (double)w[j];
                if (w[j] > 0.0f) {
                    last = (uint32_t)j; x_last = x[j];
                    if (first == 8 && cum > target) { first = (uint32_t)j; x_first = x[j]; }
                }
            }
        } else {
#pragma unroll
            for (int j = 7; j >= 0; --j) if (x[j] == best) first = (uint32_t)j;
        }
        const uint64_t over = __ballot(first < 8), live = __ballot(last < 8);
        if (!over && !live) continue;
        done = over != 0;
        const int to = done ? __builtin_ctzll(over) : 63 - __builtin_clzll(live);
        at = (uint32_t)v * 512 + (uint32_t)to * 8 + (uint32_t)__builtin_amdgcn_readlane((int)((done ? first : last) - cut), to);
        x_at = read_lane(done ? x_first : x_last, to);
    }
    // The token's own segment is now known to 64 bits: where the token has nearly all the weight, its logarithm is that of a number next to 1, and the
    // segment's sum in 32 bits would have rounded the rest away.
    sum += (run - p[segment].sum) * scale.of(within.best);
    if (lane == 0) {
        tokens[row] = (int32_t)(w0 + at);
        if (logprob) logprob[row] = scale.log_share(x_at, sum);
    }
}

template <class T, bool TINY, bool MASKED, int WAVES>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(4))) void k_choose(tp_logits a, uint64_t row0, uint32_t segs, const float* temperature,
                                                                                              const float* uniform, int32_t* tokens, float* logprob, ChoicePart* parts) {
    constexpr int SEGS = WAVES == CHOICE_WAVES ? MOST_SEGS : FEW_SEGS;
    using Chunk = Window<WAVES, SEGS>;
    __shared__ typename Chunk::Lds l;
    __shared__ ChoicePart here[WAVES * SEGS];
    __shared__ float largest[WAVES];
    const uint64_t row = row0 + blockIdx.y;
    const uint32_t chunks = gridDim.x, window = segs * WAVES * SEGMENT, w0 = blockIdx.x * window, n = a.vocab - w0, segments = reply_segments(a.vocab);
    const float t = temperature_of(temperature, uniform, row), temper = t > 0.0f ? t : 1.0f;
    const Inverse inverse(temper);
    RowRules r = row_rules(a, row);
    if (!MASKED) r.mask = nullptr;                                            // as it is: without the masks' registers 512 rows take 42.0 us instead of 42.9
    const auto from = logit_row<T>(a, row) + w0;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), last = std::min(segs * WAVES, reply_segments(n));
    History<WAVES * 64, 16 / WAVES> history;
    history.load(r, w0);
    Held<T> h;
    uint32_t bits[VECS];
    load_mask(r, w0, n, wave, bits);
    if (wave < last) load_segment<T, TINY, true>(r, from, w0, n, wave, bits, h);
    load_mask(r, w0, n, wave + WAVES, bits);
    const uint32_t distinct = Chunk::template repeated<T>(r, temper, history, from, w0, std::min(n, window), l, dynamic_lds);
    ChoicePart* out = parts + row * segments + w0 / SEGMENT;
    float ref = NEG_INF;
    if (t > 0.0f) {                                                           // the largest of the waves' first segments, a number near the row's largest: small exponents round less
        if (wave < last) {
            float x[VECS][8];
            uint32_t i0, i1;
            segment_x<T, TINY>(r, n, wave, h, distinct, l, x, i0, i1);
            ref = segment_largest(x, temper, dynamic_lds, i0, i1);
        }
        if ((threadIdx.x & 63) == 0) largest[wave] = ref;
        __syncthreads();
        ref = wave_max(largest[threadIdx.x % WAVES]);
    }
    for (uint32_t g = wave; g < last; g += WAVES) {
        const float sum = segment_part<T, TINY>(r, n, g, h, temper, inverse, t == 0.0f, ref, distinct, l, dynamic_lds, [&] {
            if (g + WAVES < last) load_segment<T, TINY, true>(r, from, w0, n, g + WAVES, bits, h);
            load_mask(r, w0, n, g + 2 * WAVES, bits);
        });
        l.lane_sum[g * 64 + (threadIdx.x & 63)] = sum;
        if ((threadIdx.x & 63) == 0) here[g].best = ref;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < last * 8; i += WAVES * 64) {           // eight threads a segment
        const float4 a0 = *(const float4*)(l.lane_sum + i * 8), a1 = *(const float4*)(l.lane_sum + i * 8 + 4);
        const double sum = eight_lanes_sum((((double)a0.x + a0.y) + ((double)a0.z + a0.w)) + (((double)a1.x + a1.y) + ((double)a1.z + a1.w)));
        if (i % 8 == 7) {
            const uint32_t g = i / 8;
            if (chunks > 1) out[g] = ChoicePart{sum, here[g].best}; else here[g].sum = sum;
        }
    }
    if (chunks > 1) return;
    __syncthreads();
    if (threadIdx.x < 64) join_row<T, Chunk, TINY>(a, r, row, segments, here, t, uniform, tokens, logprob, distinct, l, dynamic_lds);
}

template <class T>
__global__ __launch_bounds__(64) void k_choose_join(tp_logits a, uint64_t row0, const float* temperature, const float* uniform, int32_t* tokens, float* logprob,
                                                    const ChoicePart* parts) {
    __shared__ OneSegment::Lds l;
    const uint64_t row = row0 + blockIdx.x;
    const uint32_t segments = reply_segments(a.vocab);
    join_row<T, OneSegment, false>(a, row_rules(a, row), row, segments, parts + row * segments, temperature_of(temperature, uniform, row), uniform, tokens, logprob, 0, l, dynamic_lds);
}

// ---- the grammar ----------------------------------------------------------------------------------------------------------------

// whether an entry may be taken with `tags` finished tags
__device__ inline bool may(uint32_t move, uint32_t tags, const DevGrammar& g) {
    const uint32_t kind = move >> MOVE_SHIFT;
    return kind == MOVE_INSIDE || (kind == MOVE_COMMA ? tags + 2 <= g.max_tags : tags + 1 >= g.min_tags);
}

struct List { uint32_t lo, hi, tags; };
__device__ inline List list_of(const DevGrammar& g, const int32_t* states, uint64_t row) {
    const uint32_t place = (uint32_t)glob(states)[2 * row];
    const int32_t tags = glob(states)[2 * row + 1];
    List q{0, 0, tags < 0 ? 0u : tags > 65535 ? 65535u : (uint32_t)tags};
    if (place < g.n_places) { q.lo = glob(g.begin)[place]; q.hi = glob(g.begin)[place + 1]; }
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
// in 16-byte pieces.  Of a list longer than a few rounds of the block only the piece's own part is read.  Bound by the blocks of the long
// lists: 1024 rows over 131072 tokens (17 MB of mask, 4 us at a copy's rate) take 6.0 us.
constexpr uint32_t MASK_PIECE = 1024, MASK_AHEAD = 2;   // (4 ahead: 7.3 us, 1: 7.2)
__global__ __launch_bounds__(256) void k_grammar_mask(DevGrammar g, const int32_t* states, uint64_t row0, uint32_t* mask, uint64_t mask_stride) {
    __shared__ alignas(16) uint32_t bits[MASK_PIECE];
    const uint64_t row = row0 + blockIdx.y;
    const uint32_t w0 = blockIdx.x * MASK_PIECE, words = (g.n_tokens + 31) / 32;
    List q = list_of(g, states, row);
    *(uint4*)(bits + threadIdx.x * 4) = make_uint4(0, 0, 0, 0);
    const uint32_t t0 = w0 * 32;
    if (t0 && q.hi - q.lo > 256 * MASK_AHEAD) q.lo = lower_entry_wave(g.entry, q.lo, q.hi, t0);
    __syncthreads();
    const auto entries = (Glob<unsigned long long>)glob((const unsigned long long*)g.entry);
    for (uint32_t e0 = q.lo + threadIdx.x; e0 < q.hi; e0 += 256 * MASK_AHEAD) {
        unsigned long long en[MASK_AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < MASK_AHEAD; ++i) en[i] = e0 + i * 256 < q.hi ? entries[e0 + i * 256] : 0xFFFFFFFFull;
#pragma unroll
        for (uint32_t i = 0; i < MASK_AHEAD; ++i) {
            const uint32_t t = (uint32_t)en[i] - t0;                          // beyond the piece where the entry is one of another piece, or none
            if (t < MASK_PIECE * 32 && may((uint32_t)(en[i] >> 32), q.tags, g)) atomicOr(&bits[t >> 5], 1u << (t & 31));
        }
        if ((uint32_t)en[MASK_AHEAD - 1] >= t0 + MASK_PIECE * 32) break;       // ascending: so is whatever follows
    }
    __syncthreads();
    uint32_t* out = mask + row * mask_stride + w0;
    const uint32_t n = words - w0, at = threadIdx.x * 4;
    if (at + 4 <= n) {
        __builtin_nontemporal_store(*(const Words4*)(bits + at), (At<uint32_t>::W*)(out + at));   // past the caches: 7.0 -> 6.0 us
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
// THREADS * EACH.  Only the listed tokens' logits are read.  The history goes through a hash table in LDS, a part of THREADS * RECALL entries at a time,
// in which every entry of the list looks its token up.  (Looking every history token up in the sorted list takes a binary search of
// dependent LDS reads: 3.4 of the 8.5 us that a list of 4781 took.)  A list longer than THREADS * EACH is worked on in pieces,
// twice: for the largest x and the sum, and for the place.  ONE: there is none.
template <int THREADS, int EACH, int RECALL, bool ONE>
struct Step {
    static constexpr uint32_t PIECE = THREADS * EACH;
    static constexpr int WAVES = THREADS / 64, SEGMENTS = WAVES * EACH;      // a wave's 64 entries of one round are a segment, in token order
    static constexpr uint32_t SLOTS = 2 * THREADS * RECALL, EMPTY = 0xFFFFFFFFu;   // at most half of the slots are taken: a search ends
    static_assert((SLOTS & (SLOTS - 1)) == 0, "a power of two");
    struct Lds {
        alignas(16) uint32_t key[SLOTS];
        alignas(16) uint32_t cnt[SLOTS];
        double sum[SEGMENTS];
        alignas(16) float weight[EACH == 1 ? 4 : PIECE];
        float max[WAVES];
        uint32_t first;
    };
    static __device__ uint32_t slot_of(uint32_t token) { return (token * 0x9E3779B1u) >> (32 - __builtin_ctz(SLOTS)); }

    // The history's entries [k0, k0 + THREADS * RECALL) as the threads take them.
    static __device__ void remember(const RowRules& r, uint32_t k0, uint32_t (&token)[RECALL]) {
#pragma unroll
        for (int i = 0; i < RECALL; ++i) { const uint32_t k = k0 + i * THREADS + threadIdx.x; token[i] = k < r.len ? (uint32_t)r.history[k] : EMPTY; }
    }
    // their table
    static __device__ void put_down(const DevGrammar& g, const RowRules& r, uint32_t k0, const uint32_t (&token)[RECALL], Lds& s) {
        const uint32_t tid = threadIdx.x;
#pragma unroll
        for (uint32_t i = tid * 4; i < SLOTS; i += THREADS * 4) {
            *(uint4*)(s.key + i) = make_uint4(EMPTY, EMPTY, EMPTY, EMPTY);
            *(uint4*)(s.cnt + i) = make_uint4(0, 0, 0, 0);
        }
        block_sync<THREADS>();
#pragma unroll
        for (int i = 0; i < RECALL; ++i) {
            if (token[i] >= g.n_tokens) continue;                               // none: EMPTY among them
            uint32_t h = slot_of(token[i]);
            for (;; h = (h + 1) & (SLOTS - 1)) {
                const uint32_t was = atomicCAS(&s.key[h], EMPTY, token[i]);
                if (was == EMPTY || was == token[i]) break;
            }
            if (k0 + i * THREADS + tid >= r.prompt) atomicAdd(&s.cnt[h], 1u); else atomicOr(&s.cnt[h], SEEN);
        }
        block_sync<THREADS>();
    }
    // what the table adds to the count words of the thread's entries
    static __device__ void look_up(const uint2 (&en)[EACH], const Lds& s, uint32_t (&c)[EACH]) {
        uint32_t found[EACH];
#pragma unroll
        for (int v = 0; v < EACH; ++v) found[v] = s.key[slot_of(en[v].x)];
#pragma unroll
        for (int v = 0; v < EACH; ++v) {
            uint32_t h = slot_of(en[v].x);
            while (found[v] != EMPTY && found[v] != en[v].x) { h = (h + 1) & (SLOTS - 1); found[v] = s.key[h]; }
            if (found[v] != EMPTY) {
                const uint32_t n = s.cnt[h];
                c[v] = (c[v] + (n & ~SEEN)) | (n & SEEN);
            }
        }
    }

    // z of the m entries from e0: entry i of the piece is thread i % THREADS's number i / THREADS; -infinity where it may not be taken.  The history's table is made
    // while the entries are on their way, and asked while their logits are.
    template <class T>
    static __device__ void shaped(const DevGrammar& g, const tp_logits& a, const RowRules& r, float temper, uint64_t row, uint32_t tags, uint32_t e0, uint32_t m, Lds& s, uint2 (&en)[EACH], float (&x)[EACH]) {
        const auto l = logit_row<T>(a, row);
        const auto entries = (Glob<unsigned long long>)(glob((const unsigned long long*)g.entry) + e0);
        const uint32_t tid = threadIdx.x;
        bool ok[EACH];
        typename T::S raw[EACH];
        float b[EACH];
        unsigned long long e[EACH];
        uint32_t token[RECALL];
        remember(r, 0, token);
#pragma unroll
        for (int v = 0; v < EACH; ++v) e[v] = (uint32_t)v * THREADS + tid < m ? entries[v * THREADS + tid] : (unsigned long long)EMPTY;
        if (r.len) {
            block_sync<THREADS>();                                               // the piece before has asked its table
            put_down(g, r, 0, token, s);
        }
#pragma unroll
        for (int v = 0; v < EACH; ++v) {
            en[v] = make_uint2((uint32_t)e[v], (uint32_t)(e[v] >> 32));
            ok[v] = en[v].x != EMPTY && may(en[v].y, tags, g);
            raw[v] = ok[v] ? l[en[v].x] : (typename T::S)0;
            b[v] = ok[v] && r.bias ? r.bias[en[v].x] : 0.0f;
        }
        uint32_t c[EACH] = {};
        if (r.len) look_up(en, s, c);
        for (uint32_t k0 = THREADS * RECALL; k0 < r.len; k0 += THREADS * RECALL) {
            remember(r, k0, token);
            block_sync<THREADS>();
            put_down(g, r, k0, token, s);
            look_up(en, s, c);
        }
#pragma unroll
        for (int v = 0; v < EACH; ++v) {
            float y = penalised(T::up(raw[v]), c[v], r);
            if (r.bias) y = y + b[v];
            x[v] = ok[v] ? z_of(y, temper) : NEG_INF;
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
    static __device__ void segment_sums(const float (&x)[EACH], float best, Lds& s) {
        const Scale scale(best);
        if constexpr (EACH == 1) {
            const double w = wave_sum(best > NEG_INF ? (double)scale.weight(x[0]) : 0.0);
            if ((threadIdx.x & 63) == 0) s.sum[threadIdx.x >> 6] = w;
        } else {                                                              // eight threads a segment, eight neighbours each: three steps of 64 bits instead of 48
            static_assert(EACH == 8, "");
#pragma unroll
            for (int v = 0; v < EACH; ++v) s.weight[v * THREADS + threadIdx.x] = best > NEG_INF ? scale.weight(x[v]) : 0.0f;
            block_sync<THREADS>();
            const float4 a0 = *(const float4*)(s.weight + threadIdx.x * 8), a1 = *(const float4*)(s.weight + threadIdx.x * 8 + 4);
            const double w = eight_lanes_sum((((double)a0.x + a0.y) + ((double)a0.z + a0.w)) + (((double)a1.x + a1.y) + ((double)a1.z + a1.w)));
            if (threadIdx.x % 8 == 7) s.sum[threadIdx.x / 8] = w;
        }
        block_sync<THREADS>();
    }
    static __device__ double segment(const Lds& s, uint32_t i) { return i < (uint32_t)SEGMENTS ? s.sum[i] : 0.0; }
    static __device__ double piece_sum(const Lds& s) {
        double w = 0.0;
        for (uint32_t i = threadIdx.x & 63; i < (uint32_t)SEGMENTS; i += 64) w += s.sum[i];
        return wave_sum(w);
    }

    template <class T>
    static __device__ void run(const DevGrammar& g, const tp_logits& a, const RowRules& r, uint64_t row, const List& q, float t, float u, int32_t* states,
                               int32_t* tokens, float* logprob, int append, Lds& s) {
        const float temper = t > 0.0f ? t : 1.0f;
        const bool one = ONE || q.hi - q.lo <= PIECE, room = has_room(a, row, append);
        const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
        uint2 en[EACH];
        float x[EACH], best = NEG_INF;
        double sum = 0.0;
        for (uint32_t p = q.lo; p < q.hi; p += PIECE) {
            shaped<T>(g, a, r, temper, row, q.tags, p, q.hi - p < PIECE ? q.hi - p : PIECE, s, en, x);
            float pb = NEG_INF;
#pragma unroll
            for (int v = 0; v < EACH; ++v) pb = fmaxf(pb, x[v]);
            pb = read_lane(block_max(pb, s), 0);
            if (pb > best) {
                sum = best > NEG_INF ? sum * Scale(pb).of(best) : 0.0;
                best = pb;
            }
            segment_sums(x, best, s);
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
        const Scale scale(best);
        const double target = t > 0.0f ? (double)u * sum : 0.0;
        double carry = 0.0;
        bool found = false, mine = false;
        uint2 entry = make_uint2(0, 0);
        float x_at = best;
        for (uint32_t p = q.lo; p < q.hi && !found; p += PIECE) {
            if (!one) shaped<T>(g, a, r, temper, row, q.tags, p, q.hi - p < PIECE ? q.hi - p : PIECE, s, en, x);
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
            if (!one) segment_sums(x, best, s);
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
                    before = read_lane(incl - w, to);
                }
                in_piece = read_lane(incl, 63) - carry;
            }
            if (at >= 0) mine = false;                                       // a later place than any before
            if (at >= 0 && at % WAVES == wave) {
                float xs = NEG_INF;
                uint2 es = make_uint2(0, 0);
#pragma unroll
                for (int v = 0; v < EACH; ++v) if (v == at / WAVES) { xs = x[v]; es = en[v]; }
                const float w = scale.weight(xs);
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
            if (logprob) logprob[row] = scale.log_share(x_at, sum);
            take_entry(a, row, entry, states, append);
        }
    }
};

// A block per row.  Most places of a tag line have a handful of tokens, and the places where a tag begins thousands: a list of up to 64
// is the work of one wave, which needs no barrier, and the block's other waves are done at once.  Bound by latency: 256 rows over
// 131072 tokens and lists of up to 4781 take 14 us, of which the bytes (1.3 MB, 0.3 us) are next to nothing; rules and list, entries, their
// logits, the sums and the choice each wait for what comes before.
// The block is as large as the grammar's longest list asks for: 256 threads up to 2048 entries, 512 up to 4096, 1024 beyond.  A unit holds as many more rows, and a row's start
// costs fewer idle waves: 4096 rows with lists of up to 759 take 22.6 us in 256 threads, 39.0 in 512, 89.8 in 1024, up to 2259 47.4 in 512 and 102 in 1024 (and 43.9 in
// 256, in two pieces, but 256 rows 19.0 instead of 11.4).
using ShortStep = Step<64, 1, 4, true>;

template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_grammar_step(DevGrammar g, tp_logits a, uint64_t row0, const float* temperature, const float* uniform,
                                                               int32_t* states, int32_t* tokens, float* logprob, int append) {
    using LongStep = Step<THREADS, 8, 1024 / THREADS, THREADS < 1024>;
    __shared__ union { typename LongStep::Lds l; ShortStep::Lds s; } lds;
    const uint64_t row = row0 + blockIdx.x;
    // with the rules, not when it is wanted: 256 rows 15.05 -> 14.73 us (the choice, whose join loads more at once, is slower that way)
    const float t = temperature_of(temperature, uniform, row), u = temperature && uniform ? uniform[row] : 0.0f;
    const RowRules r = row_rules(a, row);
    const List q = list_of(g, states, row);
    const bool many = q.hi - q.lo > ShortStep::PIECE;
    __syncthreads();                                                         // every wave has read the state before one moves it
    if (many) {
        LongStep::template run<T>(g, a, r, row, q, t, u, states, tokens, logprob, append, lds.l);
    } else if (threadIdx.x < 64) {
        ShortStep::run<T>(g, a, r, row, q, t, u, states, tokens, logprob, append, lds.s);
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

// Sixteen rows a block, a wave each: first the bytes of every row's text and of the block's, then, each block adding the blocks before
// it up, where a row begins, and its text.  (Rows beyond LINES_DIRECT are added up by the scan of the caption offsets instead.)
// Up to LINES_ALONE rows one launch does both, every block finding the sizes of the rows before it as well: two launches / one, a pass, 8.7 / 5.4 us for 16 rows of 32 tokens,
// 9.0 / 6.4 for 32 of 128, 11.5 / 11.6 for 64 of 300, 7.6 / 10.4 for 128 of 32.
// A wave takes 64 tokens at a time, the next 64's texts and the 64 tokens behind those in flight (256 at a time, loaded together: 8192 rows of 300 in 22.2 us a pass
// instead of 20.4, for their registers and their bursts); a text stands beside
// their sizes in 16 bytes up to a length of 15.  Bound by the gathers (64 cache lines a wave's load) and by LDS: 8192 rows of up to 300 tokens (7 MB of
// tokens, 13 of text: 4.5 us at a copy's rate) take 5 us for the sizes (10 without the table of lengths in LDS) and 15 to 17 for the texts.
// A wave of the sizes holds SIZE_AHEAD times 64 tokens: 3, 4, 5, 6 and 8 are within 3 % of one another for 8192 rows of 128 to 1200 tokens (8 is 4 % ahead for 1000 rows of 2000).
constexpr uint32_t LINE_ROWS = 16, LINE_THREADS = LINE_ROWS * 64, SIZE_AHEAD = 5;
constexpr uint64_t LINES_DIRECT = 65536, LINES_ALONE = 64;

// The bytes of a row's text, by a wave.  `between` is called when the first tokens' loads are in flight.  TABLE: the lengths of all tokens stand in LDS, four bits each; a
// token's length costs a cache line otherwise.
template <bool TABLE, class F>
__device__ inline uint32_t row_bytes(const DevGrammar& g, Glob<int32_t> t, const Written& w, F&& between) {
    const uint32_t lane = threadIdx.x & 63;
    const auto bytes = glob(g.bytes);
    uint32_t n = 0, id[SIZE_AHEAD];
    auto load = [&](uint32_t k0) {
#pragma unroll
        for (uint32_t q = 0; q < SIZE_AHEAD; ++q) id[q] = k0 + q * 64 + lane < w.last ? (uint32_t)t[k0 + q * 64 + lane] : 0xFFFFFFFFu;
    };
    load(w.first);
    between();
    for (uint32_t k0 = w.first; k0 < w.last; k0 += SIZE_AHEAD * 64) {
        if (k0 != w.first) load(k0);
        uint32_t of[SIZE_AHEAD];
#pragma unroll
        for (uint32_t q = 0; q < SIZE_AHEAD; ++q) {
            if constexpr (TABLE) of[q] = id[q] < g.n_tokens ? dynamic_lds[id[q] >> 3] >> (id[q] % 8 * 4) & 15u : 0u;
            else of[q] = id[q] < g.n_tokens ? (uint32_t)bytes[id[q]] : 0u;
        }
#pragma unroll
        for (uint32_t q = 0; q < SIZE_AHEAD; ++q) {
            if (TABLE && of[q] == 15) of[q] = bytes[id[q]];
            n += of[q] == LONG_TOKEN ? glob((const uint32_t*)g.record)[id[q] * 4ull + 1] : of[q];
        }
    }
    return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(n), 63);
}

template <bool TABLE>
__global__ __launch_bounds__(LINE_THREADS) void k_line_sizes(DevGrammar g, const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t block0,
                                                             uint64_t rows, uint32_t* sizes, unsigned long long* sums) {
    __shared__ uint32_t of_row[LINE_ROWS];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint64_t row = (block0 + blockIdx.x) * LINE_ROWS + wave;
    const Written w = row < rows ? written(begin, len, width, row) : Written{0, 0};
    const uint32_t n = row_bytes<TABLE>(g, glob(tokens) + row * stride, w, [&] {
        if constexpr (TABLE) {
            const uint32_t pieces = (g.n_tokens + 31) / 32;
            for (uint32_t i = threadIdx.x; i < pieces; i += LINE_THREADS) ((uint4*)dynamic_lds)[i] = g.quarter[i];
            __syncthreads();
        }
    });
    if (lane == 0 && row < rows) sizes[row] = n;
    if (!sums) return;
    if (lane == 0) of_row[wave] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned long long sum = 0;
        for (uint32_t w = 0; w < LINE_ROWS; ++w) sum += of_row[w];
        sums[block0 + blockIdx.x] = sum;
    }
}

// A wave's text on its way out: collected in LDS at the place it has within its 16-byte pieces of memory, and stored by whole pieces.  Texts are put there
// eight bytes at a time by two OR operations on aligned words of eight bytes (a byte at a time takes four times as many LDS operations), so the words are 0
// where nothing has been put yet.
constexpr uint32_t LINE_STAGE = 1024;
typedef unsigned long long Bytes8 __attribute__((aligned(1)));
typedef uint8_t __attribute__((address_space(1)))* OutBytes;
struct Staged {
    unsigned long long* word;     // LINE_STAGE bytes and two words
    OutBytes piece;               // memory of the first word, a multiple of 16
    OutBytes end;                 // the arena's end: nothing is stored at or behind it
    uint32_t from, n;             // bytes [from, n) are to be stored; from is 0 but in a row's first piece

    __device__ uint8_t byte(uint32_t i) const { return ((const uint8_t*)word)[i]; }
    __device__ void clear(uint32_t lane) {
        block_sync<64>();
        *(uint4*)(word + lane * 2) = make_uint4(0, 0, 0, 0);
        if (lane < 2) word[LINE_STAGE / 8 + lane] = 0;
        block_sync<64>();
    }
    __device__ void start(OutBytes at, uint32_t lane) {
        from = n = (uint32_t)((uintptr_t)at & 15);
        piece = at - from;
        clear(lane);
    }
    // the low `count` (up to 8) bytes of `text` to byte i
    __device__ void put(uint32_t i, unsigned long long text, uint32_t count) {
        if (!count) return;
        const uint32_t shift = (i & 7) * 8;
        text &= ~0ull >> (64 - 8 * count);
        atomicOr(word + (i >> 3), text << shift);
        if ((i & 7) + count > 8) atomicOr(word + (i >> 3) + 1, text >> (64 - shift));
    }
    // the pieces that are full
    __device__ void flush(uint32_t lane) {
        const uint32_t full = n / 16;
        if (!full) return;
        block_sync<64>();
        if (lane < 16 && lane >= from && piece + lane < end) piece[lane] = byte(lane);
        for (uint32_t c = 1 + lane; c < full; c += 64) {
            const OutBytes to = piece + c * 16;
            const Words4 d = *(const Words4*)(word + c * 2);
            if (to + 16 <= end) *(Words4 __attribute__((address_space(1)))*)to = d;
            else for (uint32_t j = 0; j < 16; ++j) if (to + j < end) to[j] = byte(c * 16 + j);
        }
        const unsigned long long rest = lane < 2 ? word[full * 2 + lane] : 0ull;    // the last piece's bytes, 0 from n on
        clear(lane);
        if (lane < 2) word[lane] = rest;
        block_sync<64>();
        piece += full * 16;
        n &= 15;
        from = 0;
    }
    __device__ void finish(uint32_t lane) {
        flush(lane);
        block_sync<64>();
        if (lane >= from && lane < n && piece + lane < end) piece[lane] = byte(lane);
    }
};

// ALONE: no launch has found the sizes, the block finds those of its rows and of all rows before.
template <bool ALONE>
__global__ __launch_bounds__(LINE_THREADS) void k_line_text(DevGrammar g, const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t block0,
                                                            uint64_t rows, const uint32_t* sizes, const unsigned long long* sums, uint64_t* offsets, uint8_t* arena, uint64_t capacity) {
    __shared__ alignas(16) unsigned long long stage[LINE_ROWS][LINE_STAGE / 8 + 2];
    __shared__ unsigned long long before[LINE_ROWS];
    __shared__ uint32_t here[LINE_ROWS];
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const uint64_t b = block0 + blockIdx.x, row = b * LINE_ROWS + wave;
    const bool mine = row < rows;
    const Written w = mine ? written(begin, len, width, row) : Written{0, 0};
    const auto t = glob(tokens) + row * stride;
    const auto record = glob((const Words4*)g.record);
    auto token = [&](uint32_t k0) { return k0 + lane < w.last ? (uint32_t)t[k0 + lane] : 0xFFFFFFFFu; };
    auto text_of = [&](uint32_t id) { return id < g.n_tokens ? record[id] : Words4{0, 0, 0, 0}; };
    Words4 next = text_of(token(w.first));                                       // in flight while the row's place is found
    uint32_t id = token(w.first + 64);
    uint64_t at = 0;
    if (ALONE || sums) {
        unsigned long long sum = 0;
        if constexpr (ALONE) {
            const uint32_t own = row_bytes<false>(g, t, w, [] {});
            for (uint64_t q = wave; q < b * LINE_ROWS; q += LINE_ROWS) sum += row_bytes<false>(g, glob(tokens) + q * stride, written(begin, len, width, q), [] {});
            if (lane == 0) here[wave] = own;
        } else {
            for (uint64_t i = threadIdx.x; i < b; i += LINE_THREADS) sum += sums[i];
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
            if (wave == 0 && lane < LINE_ROWS) here[lane] = b * LINE_ROWS + lane < rows ? sizes[b * LINE_ROWS + lane] : 0u;
        }
        if (lane == 0) before[wave] = sum;
        __syncthreads();
        sum = lane < LINE_ROWS ? before[lane] + (lane < wave ? here[lane] : 0u) : 0ull;   // the blocks before, a wave's share a lane, and the block's rows before this one
        for (int d = 8; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
        at = sum;                                                                 // of the first sixteen lanes
        at = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at);
        if (mine && lane == 0) {
            offsets[row] = at;
            if (row == rows - 1) offsets[rows] = at + here[wave];
        }
    } else if (mine) {
        at = offsets[row];
    }
    if (!mine) return;
    const auto text = glob(g.text);
    const OutBytes out = (OutBytes)arena;
    Staged s;
    s.word = stage[wave];
    s.end = out + capacity;
    s.start(out + at, lane);
    for (uint32_t k0 = w.first; k0 < w.last; k0 += 64) {
        const Words4 rec = next;
        next = text_of(id);
        id = token(k0 + 128);
        const uint32_t kind = rec[3] >> 24, n = kind == LONG_TOKEN ? rec[1] : kind;
        const uint32_t incl = wave_scan(n), all = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63), to = incl - n;
        if (all <= LINE_STAGE - 16) {
            s.flush(lane);
            const uint32_t d = s.n + to;                                      // a flush leaves at most 15 bytes
            if (kind != LONG_TOKEN) {
                s.put(d, (unsigned long long)rec[1] << 32 | rec[0], n < 8 ? n : 8);
                if (n > 8) s.put(d + 8, (unsigned long long)rec[3] << 32 | rec[2], n - 8);
            } else {
                for (uint32_t j = 0; j < n; j += 8)                           // the texts are followed by eight bytes of room
                    s.put(d + j, *(const Bytes8 __attribute__((address_space(1)))*)(text + rec[0] + j), n - j < 8 ? n - j : 8);
            }
            s.n += all;
        } else {                                                              // texts longer than the stage: a lane stores its token's
            s.finish(lane);
            const OutBytes d = s.piece + s.n + to;
            for (uint32_t j = 0; j < n; ++j)
                if (d + j < s.end) d[j] = kind == LONG_TOKEN ? text[rec[0] + j] : (uint8_t)((j < 8 ? j < 4 ? rec[0] : rec[1] : j < 12 ? rec[2] : rec[3]) >> (8 * (j & 3)));
            s.start(s.piece + s.n + all, lane);
        }
    }
    s.finish(lane);
    if (row == rows - 1) {
        const OutBytes d = s.piece + s.n;
        if (lane < 16 && d + lane < s.end) d[lane] = 0;
    }
}

constexpr uint64_t MAX_BLOCKS = (uint64_t)1 << 21;   // of one launch: its threads stay below 2^32

template <class F>
hipError_t in_ranges(uint64_t blocks, F&& launch) {
    for (uint64_t b = 0; b < blocks; b += MAX_BLOCKS) {
        launch(b, (unsigned)(blocks - b < MAX_BLOCKS ? blocks - b : MAX_BLOCKS));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// the same for a grid of `columns` blocks a row: f(first row, rows)
template <class F>
hipError_t in_row_ranges(uint64_t rows, uint32_t columns, F&& launch) {
    const uint64_t most = std::max<uint64_t>(1, std::min<uint64_t>(65535, MAX_BLOCKS / columns));
    for (uint64_t r = 0; r < rows; r += most) {
        launch(r, (unsigned)std::min(most, rows - r));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <class F>
hipError_t by_type(int32_t type, F&& f) {
    return type == TP_T_F32 ? f(TF32{}) : type == TP_T_F16 ? f(TF16{}) : f(TBF16{});
}
// f(type, whether the vocabulary is smaller than a vector)
template <class F>
hipError_t by_type_and_size(const tp_logits& io, F&& f) {
    return by_type(io.type, [&](auto tag) { return io.vocab < 8 ? f(tag, std::true_type{}) : f(tag, std::false_type{}); });
}

}  // namespace

hipError_t load_reply_kernels() {
    hipFuncAttributes attr;                                                    // of one of them: they are one code object
    return hipFuncGetAttributes(&attr, (const void*)k_grammar_mask);
}

hipError_t launch_shape(const tp_logits& io, void* out, uint64_t out_stride) {
    const bool few = reply_segments(io.vocab) <= SHAPE_FEW;
    const uint32_t chunks = few ? 1 : (reply_segments(io.vocab) + SHAPE_WAVES - 1) / SHAPE_WAVES;
    return by_type_and_size(io, [&](auto tag, auto tiny) {
        using T = decltype(tag);
        return in_row_ranges(io.rows, chunks, [&](uint64_t r, unsigned n) {
            auto launch = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, dim3(chunks, n), dim3(waves * 64), 0, (hipStream_t)io.stream, io, r, out, out_stride); };
            if constexpr (decltype(tiny)::value) launch(k_shape<T, true, true, SHAPE_FEW>, SHAPE_FEW);
            else if (few) launch(io.mask ? k_shape<T, false, true, SHAPE_FEW> : k_shape<T, false, false, SHAPE_FEW>, SHAPE_FEW);
            else launch(io.mask ? k_shape<T, false, true, SHAPE_WAVES> : k_shape<T, false, false, SHAPE_WAVES>, SHAPE_WAVES);
        });
    });
}

// Segments a wave of the choice takes, one after another.  Where a window holds the row (131072 tokens) its history is read once and
// no second launch joins it; but a unit works on a segment for some 0.15 us, and fewer long rows than units leave the others idle: they are split.
// Split / not, us a pass: one row of 20000 14.8 / 11.3, of 32768 14.5 / 12.9, of 50021 14.5 / 14.7, of 65536 14.2 / 16.7, 128 rows of 50021 19.0 / 16.3;
// one row of 131072 14.7 / 24.1, 48 17.9 / 26.0, 128 23.1 / 26.2, 200 29.8 / 26.6.
// Up to 131072 tokens, that is: a window has no more (its tables' LDS), so longer rows are split in any case, and the powers of two split them unevenly.  The rule / the best of
// windows of 32768, 65536, 81920, 98304 and 131072 tokens: one row of 151936 13.5 / 16.2, 48 18.6 / 18.4, 160 40.7 / 28.3 (65536), 512 76.7 / 58.0 (81920); of 262144 13.2 / 16.1,
// 21.7 / 21.6, 40.1 / 34.5 (98304), 82 / 82.
// A window must also keep its repeated tokens in 64 KB of LDS.
static uint32_t window_segments(const tp_logits& io) {
    uint32_t segs = 1;
    const bool whole = reply_segments(io.vocab) <= 64 || io.rows >= 160;
    while (segs < MOST_SEGS && segs * CHOICE_WAVES * SEGMENT < io.vocab && (whole || io.rows * ((io.vocab + 2 * segs * CHOICE_WAVES * SEGMENT - 1) / (2 * segs * CHOICE_WAVES * SEGMENT)) >= 256)) segs *= 2;
    while (segs > 1 && io.history && std::min(io.history_cap, segs * CHOICE_WAVES * SEGMENT) > 16384) segs /= 2;
    return segs;
}

hipError_t launch_choose(const tp_logits& io, const float* temperature, const float* uniform, int32_t* tokens, float* logprob, ChoicePart* parts) {
    const uint32_t segments = reply_segments(io.vocab);
    const bool few = segments <= FEW_WAVES || (segments <= FEW_WAVES * FEW_SEGS && io.rows > 256);
    const uint32_t segs = few ? (segments + FEW_WAVES - 1) / FEW_WAVES : window_segments(io), window = segs * (few ? FEW_WAVES : CHOICE_WAVES) * SEGMENT, chunks = (io.vocab + window - 1) / window;
    const uint32_t lds = io.history ? std::min(io.history_cap, window) * 4 : 0, lds_one = io.history ? std::min(io.history_cap, SEGMENT) * 4 : 0;
    return by_type_and_size(io, [&](auto tag, auto tiny) {
        using T = decltype(tag);
        hipError_t e = in_row_ranges(io.rows, chunks, [&](uint64_t r, unsigned n) {
            auto launch = [&](auto kernel, int waves) {
                hipLaunchKernelGGL(kernel, dim3(chunks, n), dim3(waves * 64), lds, (hipStream_t)io.stream, io, r, segs, temperature, uniform, tokens, logprob, parts);
            };
            if constexpr (decltype(tiny)::value) launch(k_choose<T, true, true, FEW_WAVES>, FEW_WAVES);
            else if (few) launch(io.mask ? k_choose<T, false, true, FEW_WAVES> : k_choose<T, false, false, FEW_WAVES>, FEW_WAVES);
            else launch(io.mask ? k_choose<T, false, true, CHOICE_WAVES> : k_choose<T, false, false, CHOICE_WAVES>, CHOICE_WAVES);
        });
        if (e != hipSuccess || chunks == 1) return e;
        return in_ranges(io.rows, [&](uint64_t b, unsigned n) {
            hipLaunchKernelGGL(k_choose_join<T>, dim3(n), dim3(64), lds_one, (hipStream_t)io.stream, io, b, temperature, uniform, tokens, logprob, parts);
        });
    });
}

hipError_t launch_grammar_mask(const DevGrammar& g, const int32_t* states, uint64_t rows, uint32_t* mask, uint64_t mask_stride, hipStream_t s) {
    const uint32_t columns = ((g.n_tokens + 31) / 32 + MASK_PIECE - 1) / MASK_PIECE;
    return in_row_ranges(rows, columns, [&](uint64_t r, unsigned n) {
        hipLaunchKernelGGL(k_grammar_mask, dim3(columns, n), dim3(256), 0, s, g, states, r, mask, mask_stride);
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
            const int threads = g.longest_list <= 2048 ? 256 : g.longest_list <= 4096 ? 512 : 1024;
            const auto kernel = threads == 256 ? k_grammar_step<T, 256> : threads == 512 ? k_grammar_step<T, 512> : k_grammar_step<T, 1024>;
            hipLaunchKernelGGL(kernel, dim3(n), dim3(threads), 0, (hipStream_t)io.stream, g, io, b, temperature, uniform, states, tokens, logprob, append);
        });
    });
}

// The lengths in LDS: up to 64 KB of them, so that two blocks share a compute unit, and where there are blocks for every unit and tokens enough to pay for the table.
// Without / with it, us a pass, of 131072 tokens: 8192 rows of 300 tokens 22.9 / 19.9, of 192 16.4 / 15.3, of 128 13.8 / 13.7; 4096 rows of 300 15.5 / 14.4, of 128
// 10.5 / 10.8; 2048 rows of 300 13.0 / 12.7; of 32768 tokens: 8192 rows of 300 19.4 / 18.1, of 128 12.3 / 12.4.
static bool line_sizes_by_table(const DevGrammar& g, uint64_t rows, uint32_t width) {
    return g.n_tokens <= 131072 && rows >= 256 * LINE_ROWS && width >= 192;
}

hipError_t launch_grammar_lines(const DevGrammar& g, const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t rows,
                                uint8_t* arena, uint64_t capacity, uint64_t* offsets, void* workspace, hipStream_t s) {
    uint32_t* sizes = (uint32_t*)workspace;
    unsigned long long* sums = (unsigned long long*)((uint8_t*)workspace + (rows + 4) / 4 * 16);
    const uint64_t blocks = (rows + LINE_ROWS - 1) / LINE_ROWS;
    const bool direct = rows <= LINES_DIRECT;
    if (rows <= LINES_ALONE) {
        hipLaunchKernelGGL(k_line_text<true>, dim3((unsigned)blocks), dim3(LINE_THREADS), 0, s, g, tokens, stride, width, begin, len, 0, rows, nullptr, nullptr, offsets, arena, capacity);
        return hipGetLastError();
    }
    const bool table = line_sizes_by_table(g, rows, width);
    hipError_t e = in_ranges(blocks, [&](uint64_t b, unsigned n) {
        if (table) hipLaunchKernelGGL(k_line_sizes<true>, dim3(n), dim3(LINE_THREADS), (g.n_tokens + 31) / 32 * 16, s, g, tokens, stride, width, begin, len, b, rows, sizes, direct ? sums : nullptr);
        else hipLaunchKernelGGL(k_line_sizes<false>, dim3(n), dim3(LINE_THREADS), 0, s, g, tokens, stride, width, begin, len, b, rows, sizes, direct ? sums : nullptr);
    });
    if (e != hipSuccess) return e;
    if (!direct) e = launch_scan_u32(sizes, rows, offsets, (uint64_t*)sums, nullptr, nullptr, s);
    if (e != hipSuccess) return e;
    return in_ranges(blocks, [&](uint64_t b, unsigned n) {
        hipLaunchKernelGGL(k_line_text<false>, dim3(n), dim3(LINE_THREADS), 0, s, g, tokens, stride, width, begin, len, b, rows, sizes, direct ? sums : nullptr, offsets, arena, capacity);
    });
}

}  // namespace tp
