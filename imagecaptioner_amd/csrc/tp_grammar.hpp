// Host-side compiler of the tag-line grammar over a token list (tp_grammar_create), and the argument checks of the entry
// points that write replies.  Nothing here needs a device.
#pragma once
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/tagpipe.h"

namespace tp {

// An entry's move: the place behind the token, and in the two top bits what the token does.
constexpr uint32_t MOVE_PLACE = 0x3FFFFFFFu, MOVE_SHIFT = 30;
enum : uint32_t { MOVE_INSIDE = 0, MOVE_COMMA = 1, MOVE_END = 2 };

struct HostGrammar {
    tp_grammar_info info{};
    uint32_t min_tags = 0, max_tags = 0;
    std::vector<uint32_t> begin;          // per place, one more than there are: its entries
    std::vector<int32_t> token;           // per entry, ascending within a place
    std::vector<uint32_t> move;           // per entry
    std::vector<uint8_t> text;            // the tokens' bytes, back to back
    std::vector<uint32_t> text_begin;     // n_tokens + 1
};

struct HostTables;
// The tags the line ingest keeps: valid and not dropped, and with a vocabulary file a member of it (where the vocabulary is not
// strict another table string would be kept too, but the caller's list does not have it); and the same of what NormalizeTag makes of them.
// With `spaces`, those that a line may hold with ' ' for every '_'.
std::vector<std::string> reply_tags(const HostTables& ht, bool spaces = false);

// Throws ConfigError.  tags: the texts a tag may have, in any order, with repeats, before '_' becomes ' '.
void compile_grammar(const tp_grammar_config& cfg, std::vector<std::string> tags, HostGrammar& out);

// nullptr when the arguments can be run, else what is wrong with them.
const char* check_grammar_config(const tp_grammar_config* cfg);
const char* check_logits(const tp_logits* io, bool logits_needed);
const char* check_shape(const tp_logits* io, const void* out, uint64_t out_stride);
const char* check_choose(const tp_logits* io, const float* temperature, const float* uniform, const int32_t* tokens, const float* logprob,
                         const void* workspace, uint64_t workspace_bytes);
const char* check_mask(uint32_t n_tokens, const int32_t* states, uint64_t rows, const uint32_t* mask, uint64_t mask_stride);
const char* check_step(uint32_t n_tokens, const tp_logits* io, const float* temperature, const float* uniform, const int32_t* states,
                       const int32_t* tokens, const float* logprob, int append);
const char* check_lines(const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t rows, const uint8_t* arena, uint64_t capacity, const uint64_t* offsets,
                        const void* workspace, uint64_t workspace_bytes);

constexpr uint64_t MAX_REPLY_ROWS = (uint64_t)1 << 31;
// The choice of a token joins segments of a row: of each the sum of its weights, and the z that they are relative to.
constexpr uint32_t REPLY_SEGMENT = 1024;
constexpr uint32_t reply_segments(uint32_t vocab) { return (vocab + REPLY_SEGMENT - 1) / REPLY_SEGMENT; }
struct ChoicePart { double sum; float best; };
uint64_t choose_workspace(uint64_t rows, uint32_t vocab);
uint64_t lines_workspace(uint64_t rows);

}  // namespace tp
