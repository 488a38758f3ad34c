// The tag-line grammar's compiler: see tp_grammar.hpp and tp_grammar_create in include/tagpipe.h.
#include "tp_grammar.hpp"

#include <algorithm>
#include <cstring>

#include "tp_tables.hpp"

namespace tp {

namespace {

constexpr uint32_t NONE = 0xFFFFFFFFu;
constexpr uint64_t MAX_ENTRIES = (uint64_t)1 << 28;

struct Span { const uint8_t* p; uint32_t n; };

// The prefixes of the tags as a tree.  The tags are added in ascending order, so a node's number is its prefix's place among
// the sorted prefixes, and the children of a node ascend along the sibling chain.
struct PrefixTree {
    struct Node { uint32_t first = NONE, last = NONE, next = NONE; uint8_t byte = 0; bool whole = false; };
    std::vector<Node> nodes{Node()};
    void add(const std::string& s) {
        uint32_t at = 0;
        for (char ch : s) {
            const uint8_t b = (uint8_t)ch;
            const uint32_t l = nodes[at].last;
            if (l != NONE && nodes[l].byte == b) { at = l; continue; }
            const uint32_t n = (uint32_t)nodes.size();
            nodes.emplace_back();
            nodes[n].byte = b;
            if (l == NONE) nodes[at].first = n; else nodes[l].next = n;
            nodes[at].last = n;
            at = n;
        }
        nodes[at].whole = true;
    }
};

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
size_t type_bytes(int32_t t) { return t == TP_T_F32 ? 4 : 2; }
uint64_t mask_words(uint32_t vocab) { return ((uint64_t)vocab + 31) / 32; }
// a tag as a line of the grammar spells it
std::string spelled(std::string tag, bool spaces) {
    if (spaces) std::replace(tag.begin(), tag.end(), '_', ' ');
    return tag;
}
// rows * stride elements of `bytes` stay below 2^62
bool fits(uint64_t rows, uint64_t stride, uint64_t bytes) { return stride == 0 || rows <= ((uint64_t)1 << 62) / bytes / stride; }

}  // namespace

uint64_t choose_workspace(uint64_t rows, uint32_t vocab) {
    // a vocabulary that any launch's window holds needs none
    return vocab > 16 * REPLY_SEGMENT && rows <= MAX_REPLY_ROWS ? (rows * reply_segments(vocab) * sizeof(ChoicePart) + 15) / 16 * 16 : 0;
}

uint64_t lines_workspace(uint64_t rows) { return rows <= MAX_REPLY_ROWS ? (rows + 4) / 4 * 16 + (rows / 16 + 4) * 8 : 0; }

const char* check_grammar_config(const tp_grammar_config* cfg) {
    if (!cfg || cfg->struct_size != sizeof(tp_grammar_config)) return "tp_grammar_config is null or has the wrong struct_size";
    if (!cfg->token_offsets || !cfg->tokens) return "no token list";
    if (cfg->n_tokens < 1 || cfg->n_tokens > (1u << 24)) return "n_tokens must be 1 .. 2^24";
    for (uint32_t t = 0; t < cfg->n_tokens; ++t) if (cfg->token_offsets[t + 1] < cfg->token_offsets[t]) return "token_offsets must be non-decreasing";
    if (cfg->token_offsets[cfg->n_tokens] - cfg->token_offsets[0] >= ((uint64_t)1 << 32)) return "the tokens' texts take 4 GiB or more";
    if (cfg->end_token < 0 || (uint32_t)cfg->end_token >= cfg->n_tokens) return "end_token is not a token";
    if (cfg->min_tags < 1 || cfg->min_tags > cfg->max_tags || cfg->max_tags > 65535) return "1 <= min_tags <= max_tags <= 65535 is needed";
    if (cfg->spaces > 1) return "spaces must be 0 or 1";
    if (cfg->tags) {
        if (!cfg->tag_offsets) return "tags without tag_offsets";
        for (uint64_t t = 0; t < cfg->n_tags; ++t) if (cfg->tag_offsets[t + 1] < cfg->tag_offsets[t]) return "tag_offsets must be non-decreasing";
    }
    return nullptr;
}

const char* check_logits(const tp_logits* io, bool logits_needed) {
    if (!io || io->struct_size != sizeof(tp_logits)) return "tp_logits is null or has the wrong struct_size";
    if (io->type != TP_T_F32 && io->type != TP_T_F16 && io->type != TP_T_BF16) return "type must be TP_T_F32, TP_T_F16 or TP_T_BF16";
    if (io->vocab < 1 || io->vocab > (1u << 24)) return "vocab must be 1 .. 2^24";
    if (io->rows > MAX_REPLY_ROWS) return "at most 2^31 rows";
    if (!io->logits && logits_needed && io->rows) return "no logits";
    if (io->logits) {
        if (io->stride < io->vocab) return "stride is less than vocab";
        if (!fits(io->rows, io->stride, 4)) return "rows times stride is too large";
        if (!aligned(io->logits, type_bytes(io->type))) return "logits are not aligned to their type";
    }
    if (io->history) {
        if (io->history_cap > 0x7FFFFFFFu) return "history_cap must be below 2^31";
        if (io->history_stride < io->history_cap) return "history_stride is less than history_cap";
        if (!fits(io->rows, io->history_stride, 4)) return "rows times history_stride is too large";
    } else if (io->history_len || io->prompt_len) return "history_len or prompt_len without a history";
    if (io->bias) {
        if (io->n_bias < 1) return "bias needs n_bias of at least 1";
        if (io->bias_stride < io->vocab) return "bias_stride is less than vocab";
        if (!fits(io->n_bias, io->bias_stride, 4)) return "n_bias times bias_stride is too large";
    } else if (io->bias_row) return "bias_row without a bias";
    if (io->mask) {
        if (io->n_masks < 1) return "mask needs n_masks of at least 1";
        if (io->mask_stride < mask_words(io->vocab)) return "mask_stride is less than (vocab + 31) / 32";
        if (!fits(io->n_masks, io->mask_stride, 4)) return "n_masks times mask_stride is too large";
    } else if (io->mask_row) return "mask_row without a mask";
    for (const void* p : {(const void*)io->history, (const void*)io->history_len, (const void*)io->prompt_len, (const void*)io->repetition, (const void*)io->frequency,
                          (const void*)io->presence, (const void*)io->bias, (const void*)io->bias_row, (const void*)io->mask, (const void*)io->mask_row})
        if (!aligned(p, 4)) return "an array of 32-bit values is not aligned to 4";
    return nullptr;
}

const char* check_shape(const tp_logits* io, const void* out, uint64_t out_stride) {
    if (const char* e = check_logits(io, true)) return e;
    if (io->rows == 0) return nullptr;
    if (!out) return "no output";
    const uint64_t bytes = type_bytes(io->type);
    if (out_stride < io->vocab) return "out_stride is less than vocab";
    if (!fits(io->rows, out_stride, 4)) return "rows times out_stride is too large";
    if (!aligned(out, bytes)) return "out is not aligned to its type";
    const uintptr_t a = (uintptr_t)io->logits, b = (uintptr_t)out;
    const uint64_t na = ((io->rows - 1) * io->stride + io->vocab) * bytes, nb = ((io->rows - 1) * out_stride + io->vocab) * bytes;
    if (a < b + nb && b < a + na && !(a == b && (out_stride == io->stride || io->rows == 1))) return "out overlaps the logits without being them";
    return nullptr;
}

const char* check_choose(const tp_logits* io, const float* temperature, const float* uniform, const int32_t* tokens, const float* logprob,
                         const void* workspace, uint64_t workspace_bytes) {
    if (const char* e = check_logits(io, true)) return e;
    if (io->rows == 0) return nullptr;
    if (!tokens) return "no tokens output";
    if (!aligned(temperature, 4) || !aligned(uniform, 4) || !aligned(tokens, 4) || !aligned(logprob, 4)) return "an array of 32-bit values is not aligned to 4";
    const uint64_t need = choose_workspace(io->rows, io->vocab);
    if (need && (!workspace || workspace_bytes < need)) return "the workspace is smaller than tp_choose_workspace says";
    if (need && !aligned(workspace, 16)) return "the workspace is not aligned to 16";
    return nullptr;
}

const char* check_mask(uint32_t n_tokens, const int32_t* states, uint64_t rows, const uint32_t* mask, uint64_t mask_stride) {
    if (rows > MAX_REPLY_ROWS) return "at most 2^31 rows";
    if (rows == 0) return nullptr;
    if (!states || !mask) return "null argument";
    if (mask_stride < mask_words(n_tokens)) return "mask_stride is less than (n_tokens + 31) / 32";
    if (!fits(rows, mask_stride, 4)) return "rows times mask_stride is too large";
    if (!aligned(states, 4) || !aligned(mask, 4)) return "an array of 32-bit values is not aligned to 4";
    return nullptr;
}

const char* check_step(uint32_t n_tokens, const tp_logits* io, const float* temperature, const float* uniform, const int32_t* states,
                       const int32_t* tokens, const float* logprob, int append) {
    if (const char* e = check_logits(io, false)) return e;
    if (io->vocab != n_tokens) return "vocab is not the grammar's n_tokens";
    if (io->mask || io->mask_row) return "tp_grammar_step takes its mask from the grammar: io->mask must be null";
    if (append != 0 && append != 1) return "append must be 0 or 1";
    if (append && (!io->history || !io->history_len)) return "append needs a history and history_len";
    if (io->rows == 0) return nullptr;
    if (!states || !tokens) return "null argument";
    for (const void* p : {(const void*)states, (const void*)tokens, (const void*)temperature, (const void*)uniform, (const void*)logprob})
        if (!aligned(p, 4)) return "an array of 32-bit values is not aligned to 4";
    return nullptr;
}

const char* check_lines(const int32_t* tokens, uint64_t stride, uint32_t width, const int32_t* begin, const int32_t* len, uint64_t rows, const uint8_t* arena, uint64_t capacity, const uint64_t* offsets,
                        const void* workspace, uint64_t workspace_bytes) {
    if (rows > MAX_REPLY_ROWS) return "at most 2^31 rows";
    if (!offsets) return "no offsets";
    if (!aligned(offsets, 8)) return "offsets are not aligned to 8";
    if (rows == 0) return nullptr;
    if (width > 0x7FFFFFFFu) return "width must be below 2^31";
    if (stride < width) return "stride is less than width";
    if (!fits(rows, stride, 4)) return "rows times stride is too large";
    if ((!tokens && width) || (!arena && capacity)) return "null argument";
    if (!aligned(tokens, 4) || !aligned(begin, 4) || !aligned(len, 4)) return "an array of 32-bit values is not aligned to 4";
    if (!workspace || workspace_bytes < lines_workspace(rows)) return "the workspace is smaller than tp_lines_workspace says";
    if (!aligned(workspace, 16)) return "the workspace is not aligned to 16";
    return nullptr;
}

std::vector<std::string> reply_tags(const HostTables& ht, bool spaces) {
    // A phrase or a fence inside a force-allowed tag would make the whole line look bad, and one with a comma is cut up.  FL_PHRASE is the string's as it stands, and most
    // phrases hold a blank: with `spaces` other tags come to hold one ("unable_to_stand").
    const uint32_t want = FL_VALID | FL_LEN2 | (ht.known_found ? FL_KNOWN : 0u), without = FL_DROP | FL_PHRASE | FL_FENCE | FL_SPLIT;
    // What the ingest judges is not the string but what NormalizeTag makes of it, an alias's target among others, and it normalises three times: the line's parts
    // (Program.cs:599-601), the candidates (:622-631) and the selected tags (:693-697).  The caption's tags are normalised further, to where the string stays the same (or a circle
    // of aliases closes): all of those must be known too.
    constexpr int SELECTED = 3, FURTHER = 64;
    auto kept = [&](uint32_t id) {
        for (int hop = 1; hop <= FURTHER; ++hop) {
            const uint32_t to = ht.next[id], f = ht.flags[to];
            if (hop == 1 && (!(f & FL_LEN2) || (f & FL_SPLIT))) return false;
            if (hop <= SELECTED && ((f & FL_DROP) || (hop > 1 && !(f & FL_VALID)))) return false;
            if (hop >= SELECTED && ht.known_found && !(f & FL_KNOWN)) return false;
            if (hop >= SELECTED && to == id) break;
            id = to;
        }
        return true;
    };
    // A blank at a tag's end would be trimmed off with the comma's, and another tag read.  (None begins with '_'.)
    auto spellable = [&](const std::string& s) { return !spaces || (s.back() != '_' && !holds_phrase(spelled(s, true))); };
    std::vector<std::string> tags;
    for (uint32_t i = 0; i < ht.scalars.n_public; ++i)
        if ((ht.flags[i] & want) == want && !(ht.flags[i] & without) && kept(i) && spellable(ht.strings[i])) tags.push_back(ht.strings[i]);
    return tags;
}

void compile_grammar(const tp_grammar_config& cfg, std::vector<std::string> tags, HostGrammar& out) {
    out = HostGrammar();
    out.min_tags = cfg.min_tags;
    out.max_tags = cfg.max_tags;
    for (std::string& t : tags) {
        t = spelled(std::move(t), cfg.spaces != 0);
        if (t.empty() || t.front() == ' ' || t.back() == ' ') throw ConfigError("a tag of the grammar is empty, or begins or ends with a space: \"" + t + "\"");
        for (char ch : t) if (ch == ',' || (uint8_t)ch < 0x20) throw ConfigError("a tag of the grammar holds a comma or a control character: \"" + t + "\"");
    }
    std::sort(tags.begin(), tags.end(), [](const std::string& a, const std::string& b) {
        const int c = std::memcmp(a.data(), b.data(), std::min(a.size(), b.size()));
        return c ? c < 0 : a.size() < b.size();
    });
    tags.erase(std::unique(tags.begin(), tags.end()), tags.end());
    if (tags.empty()) throw ConfigError("the grammar has no tags");
    uint64_t bytes = 0;
    for (const std::string& t : tags) bytes += t.size();
    if (bytes >= (1u << 24)) throw ConfigError("the grammar's tags take 16 MiB or more");

    PrefixTree tree;
    for (const std::string& t : tags) tree.add(t);
    const uint32_t P = (uint32_t)tree.nodes.size();

    const uint64_t base = cfg.token_offsets[0];
    out.text.assign(cfg.tokens + base, cfg.tokens + cfg.token_offsets[cfg.n_tokens]);
    out.text_begin.resize((size_t)cfg.n_tokens + 1);
    for (uint32_t t = 0; t <= cfg.n_tokens; ++t) out.text_begin[t] = (uint32_t)(cfg.token_offsets[t] - base);
    // The end token has no text in a line, whatever the list spells for it: its bytes are cut out.
    {
        const uint32_t e = (uint32_t)cfg.end_token, n = out.text_begin[e + 1] - out.text_begin[e];
        if (n) {
            out.text.erase(out.text.begin() + out.text_begin[e], out.text.begin() + out.text_begin[e + 1]);
            for (uint32_t t = e + 1; t <= cfg.n_tokens; ++t) out.text_begin[t] -= n;
        }
    }
    auto text = [&](uint32_t t) { return Span{out.text.data() + out.text_begin[t], out.text_begin[t + 1] - out.text_begin[t]}; };

    // The tokens in the order of their texts: the tokens that go on with given bytes are a range of it, and those that end there
    // stand first in the range.
    std::vector<uint32_t> order;
    uint32_t longest = 0;
    for (uint32_t t = 0; t < cfg.n_tokens; ++t) {
        const uint32_t n = text(t).n;
        longest = std::max(longest, n);
        if (n) order.push_back(t);
    }
    std::sort(order.begin(), order.end(), [&](uint32_t a, uint32_t b) {
        const Span x = text(a), y = text(b);
        const int c = std::memcmp(x.p, y.p, std::min(x.n, y.n));
        return c ? c < 0 : x.n != y.n ? x.n < y.n : a < b;
    });

    bool used[256] = {}, alone[256] = {};
    used[(uint8_t)','] = used[(uint8_t)' '] = true;
    for (const std::string& t : tags) for (char ch : t) used[(uint8_t)ch] = true;
    for (uint32_t t : order) if (text(t).n == 1) alone[text(t).p[0]] = true;
    for (int b = 0; b < 256; ++b)
        if (used[b] && !alone[b])
            throw ConfigError("the token list has no token for the single byte " + std::to_string(b) + ", which tag lines use: a line could come to a place with no way on");

    // Every place's tokens: walk the texts that may follow it and the token order side by side.
    struct Walk { uint32_t place, lo, hi, depth; bool comma; };
    struct Entry { uint32_t token, move; };
    std::vector<Walk> todo;
    std::vector<Entry> got;
    out.begin.reserve((size_t)P + 3);
    for (uint32_t s = 0; s <= P; ++s) {
        out.begin.push_back((uint32_t)out.token.size());
        got.clear();
        todo.assign(1, Walk{s, 0, (uint32_t)order.size(), 0, false});
        while (!todo.empty()) {
            Walk w = todo.back();
            todo.pop_back();
            while (w.lo < w.hi && text(order[w.lo]).n == w.depth) got.push_back(Entry{order[w.lo++], w.place | (w.comma ? MOVE_COMMA : MOVE_INSIDE) << MOVE_SHIFT});
            if (w.lo >= w.hi) continue;
            auto on = [&](uint8_t b, uint32_t place, bool comma) {
                const uint32_t d = w.depth;
                const auto first = order.begin() + w.lo, last = order.begin() + w.hi;
                const auto lo = std::partition_point(first, last, [&](uint32_t t) { return text(t).p[d] < b; });
                const auto hi = std::partition_point(lo, last, [&](uint32_t t) { return text(t).p[d] <= b; });
                if (lo != hi) todo.push_back(Walk{place, (uint32_t)(lo - order.begin()), (uint32_t)(hi - order.begin()), d + 1, comma});
            };
            if (w.place == P) { on(' ', 0, w.comma); continue; }
            const auto& node = tree.nodes[w.place];
            if (node.whole && !w.comma) on(',', P, true);
            for (uint32_t c = node.first; c != NONE; c = tree.nodes[c].next) on(tree.nodes[c].byte, c, w.comma);
        }
        if (s < P && tree.nodes[s].whole) got.push_back(Entry{(uint32_t)cfg.end_token, (P + 1) | MOVE_END << MOVE_SHIFT});
        std::sort(got.begin(), got.end(), [](const Entry& a, const Entry& b) { return a.token < b.token; });
        if (out.token.size() + got.size() > MAX_ENTRIES) throw ConfigError("the grammar over this token list has more than 2^28 entries");
        out.info.longest_list = std::max(out.info.longest_list, (uint32_t)got.size());
        for (const Entry& e : got) { out.token.push_back((int32_t)e.token); out.move.push_back(e.move); }
    }
    out.begin.push_back((uint32_t)out.token.size());       // the end: nothing follows
    out.begin.push_back((uint32_t)out.token.size());
    out.info.n_tokens = cfg.n_tokens;
    out.info.n_prefixes = P;
    out.info.n_tags = (uint32_t)tags.size();
    out.info.longest_token = longest;
    out.info.n_entries = out.token.size();
}

}  // namespace tp
