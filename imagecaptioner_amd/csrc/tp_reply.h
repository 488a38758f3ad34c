// Launchers of the kernels that write replies (tp_reply.hip), used by the C ABI layer (tp_api.cpp).
#pragma once
#include <hip/hip_runtime_api.h>
#include <hip/hip_vector_types.h>
#include <stdint.h>

#include "../../include/tagpipe.h"
#include "tp_grammar.hpp"

namespace tp {

constexpr uint32_t LONG_TOKEN = 255;

// A compiled grammar in device memory.
struct DevGrammar {
    const uint32_t* begin;        // HostGrammar::begin
    const uint2* entry;           // per entry: token, move
    const uint8_t* bytes;         // per token: its bytes, or LONG_TOKEN
    const uint4* quarter;         // per token four bits, 32 tokens an element: its bytes, or 15 for 15 and more
    const uint4* record;          // per token: up to 15 bytes of text and their number in the last byte; of a longer one where it starts in
                                  //   `text`, its bytes, and LONG_TOKEN in the last byte
    const uint8_t* text;          // the tokens' bytes, and eight behind them
    uint32_t n_tokens, n_places;  // places 0 .. n_places - 1 (the end among them)
    uint32_t min_tags, max_tags, longest_list;
};

// Loads the kernels' code on the current device, so that the first call of one may already be a captured one.
hipError_t load_reply_kernels();
hipError_t launch_shape(const tp_logits& io, void* out, uint64_t out_stride);
hipError_t launch_choose(const tp_logits& io, const float* temperature, const float* uniform, int32_t* tokens, float* logprob, ChoicePart* parts);
hipError_t launch_grammar_mask(const DevGrammar& g, const int32_t* states, uint64_t rows, uint32_t* mask, uint64_t mask_stride, hipStream_t s);
hipError_t launch_grammar_step(const DevGrammar& g, const tp_logits& io, const float* temperature, const float* uniform, int32_t* states,
                               int32_t* tokens, float* logprob, int append);
hipError_t launch_grammar_lines(const DevGrammar& g, const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t rows,
                                uint8_t* arena, uint64_t capacity, uint64_t* offsets, void* workspace, hipStream_t s);

}  // namespace tp
