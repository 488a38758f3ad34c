// Test-only host build of the tag-line grammar's compiler and of the argument checks of the entry points that write replies.
#include <cstring>
#include <memory>
#include <string>

#include "../../imagecaptioner_amd/csrc/tp_grammar.hpp"
#include "../../imagecaptioner_amd/csrc/tp_tables.hpp"

using namespace tp;

static std::string g_error;

extern "C" {

const char* rsim_last_error() { return g_error.c_str(); }

// cfg->tags, or the tags of the tables that `tables` configures
HostGrammar* rsim_compile(const tp_grammar_config* cfg, const tp_config* tables) {
    if (const char* e = check_grammar_config(cfg)) { g_error = e; return nullptr; }
    try {
        std::vector<std::string> tags;
        if (cfg->tags) {
            for (uint64_t t = 0; t < cfg->n_tags; ++t) tags.emplace_back((const char*)cfg->tags + cfg->tag_offsets[t], (size_t)(cfg->tag_offsets[t + 1] - cfg->tag_offsets[t]));
        } else {
            HostTables ht;
            compile_tables(*tables, ht);
            tags = reply_tags(ht, cfg->spaces != 0);
        }
        std::unique_ptr<HostGrammar> g(new HostGrammar());
        compile_grammar(*cfg, tags, *g);
        return g.release();
    } catch (const std::exception& e) {
        g_error = e.what();
        return nullptr;
    }
}
void rsim_destroy(HostGrammar* g) { delete g; }
void rsim_info(const HostGrammar* g, tp_grammar_info* out) { *out = g->info; }
const uint32_t* rsim_begin(const HostGrammar* g) { return g->begin.data(); }
const int32_t* rsim_token(const HostGrammar* g) { return g->token.data(); }
const uint32_t* rsim_move(const HostGrammar* g) { return g->move.data(); }
const uint8_t* rsim_text(const HostGrammar* g) { return g->text.data(); }
const uint32_t* rsim_text_begin(const HostGrammar* g) { return g->text_begin.data(); }

const char* rsim_check_shape(const tp_logits* io, const void* out, uint64_t out_stride) { return check_shape(io, out, out_stride); }
const char* rsim_check_choose(const tp_logits* io, const float* t, const float* u, const int32_t* tokens, const float* lp, const void* ws, uint64_t bytes) {
    return check_choose(io, t, u, tokens, lp, ws, bytes);
}
const char* rsim_check_mask(uint32_t n, const int32_t* states, uint64_t rows, const uint32_t* mask, uint64_t stride) { return check_mask(n, states, rows, mask, stride); }
const char* rsim_check_step(uint32_t n, const tp_logits* io, const float* t, const float* u, const int32_t* states, const int32_t* tokens, const float* lp, int append) {
    return check_step(n, io, t, u, states, tokens, lp, append);
}
const char* rsim_check_lines(const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t rows, const uint8_t* arena,
                             uint64_t capacity, const uint64_t* offsets, const void* ws, uint64_t bytes) {
    return check_lines(tokens, stride, width, begin, len, rows, arena, capacity, offsets, ws, bytes);
}
uint64_t rsim_choose_workspace(uint64_t rows, uint32_t vocab) { return choose_workspace(rows, vocab); }
uint64_t rsim_lines_workspace(uint64_t rows) { return lines_workspace(rows); }
}
