"""The operators that write a captioning model's reply under the tag pipeline's own rules, as measured cases.

A language model that runs beside the pipeline answers token by token.  Between its logits and the tag line that
tp_run_lines_device reads stand five operators:

  shape   penalties for repeated tokens, biases and allowed-token masks on logits
  choose  the same, and the token that they leave the choice of, with its log-probability
  mask    the allowed-token masks of the tag-line grammar, for rows of grammar states
  step    one step of writing tag lines: shaping, choice and the grammar's move
  lines   the rows' tokens as one arena of line bytes with offsets

`own` says which side runs: the plain form in elementary torch operations, or the framework's kernels.
"""
import functools
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MIN_TAGS, MAX_TAGS = 3, 42          # a line of fewer than three tags falls back (Program.cs:297), one of more than 42 is cut (Program.cs:38)


def listed():
    return [
        # one reply being written, a small vocabulary: latency
        {"name": "shape one row", "op": "shape", "rows": 1, "vocab": 32768, "type": "bf16", "history": 64, "biases": 1, "masks": 0, "density": 1.0},
        # a batch of replies with an allowed-token mask and a bias table per request kind
        {"name": "shape 64 rows", "op": "shape", "rows": 64, "vocab": 131072, "type": "bf16", "history": 512, "biases": 4, "masks": 64, "density": 0.3},
        # a large batch of 32-bit logits over an odd vocabulary: the largest
        {"name": "shape 256 odd rows f32", "op": "shape", "rows": 256, "vocab": 131071, "type": "f32", "history": 1500, "biases": 1, "masks": 16, "density": 0.6},
        # one reply, sampled, nothing masked
        {"name": "choose one row", "op": "choose", "rows": 1, "vocab": 131072, "type": "bf16", "history": 300, "biases": 0, "masks": 0, "density": 1.0},
        # an odd vocabulary in half precision, sparse masks of the caller's own
        {"name": "choose 48 odd rows f16", "op": "choose", "rows": 48, "vocab": 50021, "type": "f16", "history": 200, "biases": 2, "masks": 48, "density": 0.02},
        # a large batch: the logits' one read is what it costs
        {"name": "choose 512 rows", "op": "choose", "rows": 512, "vocab": 131072, "type": "bf16", "history": 256, "biases": 1, "masks": 0, "density": 1.0},
        # masks for a caller's own sampler: a few rows, and a large batch
        {"name": "mask 16 rows", "op": "mask", "rows": 16, "vocab": 32768, "tags": 5800},
        {"name": "mask 1024 rows", "op": "mask", "rows": 1024, "vocab": 131072, "tags": 5800},
        # writing one tag line, and a batch of them: the step that a captioning loop runs for every token
        {"name": "step one row", "op": "step", "rows": 1, "vocab": 32768, "tags": 5800, "type": "bf16", "history": 100, "biases": 0},
        {"name": "step 256 rows", "op": "step", "rows": 256, "vocab": 131072, "tags": 5800, "type": "bf16", "history": 200, "biases": 1},
        # finished replies as the pipeline's input: a batch, and a whole directory's
        {"name": "lines 32 rows", "op": "lines", "rows": 32, "vocab": 32768, "tags": 5800, "tokens": 128},
        {"name": "lines 8192 rows", "op": "lines", "rows": 8192, "vocab": 131072, "tags": 5800, "tokens": 300},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shape", "choose", "mask", "step", "lines"])
    if op in ("shape", "choose"):
        vocab = _log_int(rng, 1000, 131072)
        rows = _log_int(rng, 1, min(512, max(1, (256 if op == "shape" else 400) * 131071 // vocab)))
        masks = rng.choice([0, 1, rows])
        return {"op": op, "rows": rows, "vocab": vocab, "type": rng.choice(["bf16", "f16", "f32"]) if rows <= 256 else "bf16", "history": _log_int(rng, 1, 1500),
                "biases": rng.choice([0, 1, 3]), "masks": masks, "density": rng.choice([0.01, 0.2, 0.7]) if masks else 1.0}
    vocab, tags = rng.choice([8192, 32768, 50021, 131072]), rng.choice([500, 5800])
    if op == "mask":
        return {"op": op, "rows": _log_int(rng, 1, 1024), "vocab": vocab, "tags": tags}
    if op == "step":
        return {"op": op, "rows": _log_int(rng, 1, 256), "vocab": vocab, "tags": tags, "type": rng.choice(["bf16", "f16", "f32"]), "history": _log_int(rng, 1, 600), "biases": rng.choice([0, 1, 3])}
    return {"op": op, "rows": _log_int(rng, 1, 8192), "vocab": vocab, "tags": tags, "tokens": _log_int(rng, 8, 300)}


# ---- the tags and the tokens that a user's program starts with ---------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _tag_texts(count):
    """`count` distinct two-word tags, as a vocabulary file holds them."""
    rng = random.Random(count)
    syllables = [c + v for c in "bdfgklmnprtvz" for v in "aeou"]
    words = sorted({"".join(rng.choice(syllables) for _ in range(rng.randint(1, 3))) for _ in range(4 * int(math.sqrt(count)) + 40)})
    tags = set()
    while len(tags) < count:
        tags.add(rng.choice(words) + "_" + rng.choice(words))
    return tuple(sorted(tags))


@functools.lru_cache(maxsize=None)
def _token_texts(vocab, count):
    """A token list: the 256 single bytes, pieces of tag lines, pieces that no tag line holds, and the end token (the last id, no text)."""
    rng = random.Random(vocab * 7 + count)
    tags = _tag_texts(count)
    pieces, tries = {b", "}, 0
    while len(pieces) < (vocab - 257) * 2 // 5 and tries < vocab:
        tries += 1
        tag = rng.choice(tags)
        at, n = rng.randrange(len(tag) - 1), rng.randint(2, 8)
        piece = tag[at:at + n].encode()
        pieces.add(b" " + piece if not at and rng.random() < 0.3 else piece + b"," if at + n >= len(tag) and rng.random() < 0.1 else piece)
    while len(pieces) < vocab - 257:
        pieces.add(("%s%x" % (rng.choice(["Q", "X", " J", "9"]), rng.randrange(1 << 30))).encode())
    pieces = sorted(pieces)
    rng.shuffle(pieces)
    return tuple(bytes([b]) for b in range(256)) + tuple(pieces) + (b"",)


@functools.lru_cache(maxsize=None)
def _plain_grammar(vocab, count):
    """The tag-line grammar as lists: for every state the tokens that may come next, ascending, with the state behind each.

    A state is the place a line has come to: the n-th of the sorted distinct prefixes of the tags (the empty one, 0, is where a tag begins),
    or n_prefixes behind a tag's comma, or n_prefixes + 1 behind the end.  Kind 0: the token stays within the tag, 1: it holds the comma
    that ends the tag, 2: the end token."""
    tags, tokens = [t.encode() for t in _tag_texts(count)], _token_texts(vocab, count)
    prefixes = sorted({t[:n] for t in tags for n in range(len(t) + 1)})
    place = {p: i for i, p in enumerate(prefixes)}
    whole, after_comma, end = set(tags), len(prefixes), len(prefixes) + 1
    grown = [[] for _ in prefixes]                     # per prefix the ids of the prefixes one byte longer
    for p in prefixes[1:]:
        grown[place[p[:-1]]].append(place[p])

    def behind_comma(tail):                            # where what follows a comma leads, None: nowhere
        return after_comma if not tail else place.get(tail[1:]) if tail[:1] == b" " else None

    by_text, by_head, by_tail = {}, {}, []
    for i, t in enumerate(tokens[:-1]):
        by_text.setdefault(t, []).append(i)
        if t.count(b",") == 1:
            head, tail = t.split(b",")
            to = behind_comma(tail)
            if to is not None:
                by_head.setdefault(head, []).append((i, to))
        if t[:1] == b" ":
            by_tail.append(i)
    longest = max(len(t) for t in tokens)
    lists = []
    for s, p in enumerate(prefixes):
        got, todo = [], [s]
        while todo:
            q = todo.pop()
            piece = prefixes[q][len(p):]
            got += [(i, 0, q) for i in by_text.get(piece, ())] if piece else []
            if prefixes[q] in whole:
                got += [(i, 1, to) for i, to in by_head.get(piece, ())]
            if len(piece) < longest:
                todo += grown[q]
        if p in whole:
            got.append((vocab - 1, 2, end))
        lists.append(sorted(got))
    got = []
    for i in by_tail:                                  # behind the comma: a space, and what may begin a tag
        head, *tail = tokens[i][1:].split(b",")
        if not tail and head in place:
            got.append((i, 0, place[head]))
        elif len(tail) == 1 and head in whole and behind_comma(tail[0]) is not None:
            got.append((i, 1, behind_comma(tail[0])))
    lists += [sorted(got), []]
    begin = np.zeros(len(lists) + 1, np.int64)
    begin[1:] = np.cumsum([len(x) for x in lists])
    flat = np.array([e for x in lists for e in x], np.int64).reshape(-1, 3)
    return {"begin": begin, "token": flat[:, 0], "kind": flat[:, 1], "next": flat[:, 2], "states": len(lists)}


@functools.lru_cache(maxsize=None)
def _grammar_on(device, vocab, count):
    g = {k: torch.as_tensor(v, device=device) if not isinstance(v, int) else v for k, v in _plain_grammar(vocab, count).items()}
    g["key"] = torch.repeat_interleave(torch.arange(g["states"], device=device), g["begin"].diff()) * vocab + g["token"]
    return g


@functools.lru_cache(maxsize=None)
def _own_pipe(count):
    from imagecaptioner_amd import Config, TagPipe
    return TagPipe(Config(vocabulary="\n".join(_tag_texts(count)).encode()) if count else Config())


@functools.lru_cache(maxsize=None)
def _own_grammar(vocab, count):
    return _own_pipe(count).tag_grammar(_token_texts(vocab, count), end_token=vocab - 1, min_tags=MIN_TAGS, max_tags=MAX_TAGS)


@functools.lru_cache(maxsize=None)
def _token_bytes_on(device, vocab, count):
    tokens = _token_texts(vocab, count)
    begin = np.zeros(len(tokens) + 1, np.int64)
    begin[1:] = np.cumsum([len(t) for t in tokens])
    return torch.as_tensor(np.frombuffer(b"".join(tokens), np.uint8).copy(), device=device), torch.as_tensor(begin, device=device)


# ---- inputs ----------------------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=device).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=device)

    def whole(high, *shape):
        return torch.randint(high, shape, generator=gen, device=device, dtype=torch.int32)

    s = {"op": case["op"], "rows": rows, "vocab": vocab, "tags": case.get("tags", 0)}
    if case["op"] in ("mask", "step"):
        n = _plain_grammar(vocab, case["tags"])["states"]
        at = whole(n, rows)                                  # lines of every length being written: starts, middles of tags, finished ones
        at = torch.where(uniform(rows) < 0.15, torch.zeros_like(at), at)
        at = torch.where(uniform(rows) < 0.03, torch.full_like(at, n - 1), at)
        s["states"] = torch.stack([at, whole(MAX_TAGS, rows)], 1)
    if case["op"] in ("shape", "choose", "step"):
        logits = torch.randn(rows, vocab, generator=gen, device=device).mul_(3.0)
        logits.add_(uniform(rows, vocab).gt_(0.999), alpha=6.0)     # a few likely tokens a row
        s["logits"] = logits.to(TYPES[case["type"]])
        h = case["history"]
        spread = uniform(rows, h).pow_(3.0)                          # written tokens, some of them again and again
        s["history"] = (spread * (vocab - 1)).to(torch.int32)
        s["history_len"] = torch.where(uniform(rows) < 0.5, whole(h + 1, rows), torch.full_like(s["history"][:, 0], h))
        s["prompt_len"] = (uniform(rows) * 0.3 * s["history_len"]).to(torch.int32)
        s["repetition"] = 1.0 + 0.3 * uniform(rows)
        s["frequency"], s["presence"] = 0.5 * uniform(rows), 0.5 * uniform(rows)
        if case["biases"]:
            s["bias"] = torch.randn(case["biases"], vocab, generator=gen, device=device)
            s["bias_row"] = whole(case["biases"] + 1, rows) - 1 if case["biases"] > 1 else whole(1, rows)      # some rows without one
        if case.get("masks"):
            words = (vocab + 31) // 32
            m = case["masks"]
            s["mask"] = torch.empty(m, words, device=device, dtype=torch.int32)
            for at in range(0, m, 64):
                bits = uniform(min(64, m - at), words * 32).lt_(case["density"]).to(torch.int32)
                s["mask"][at:at + 64] = _packed(bits)
            if m > 2:
                s["mask"][m // 2] = 0                                # a row that its mask leaves nothing
            s["mask_row"] = torch.arange(rows, device=device, dtype=torch.int32) if m == rows else whole(m, rows)
    if case["op"] in ("choose", "step"):
        s["temperature"] = torch.where(uniform(rows) < 0.25, torch.zeros(rows, device=device), 0.5 + 0.7 * uniform(rows))
        s["uniform"] = uniform(rows)
    if case["op"] == "lines":
        n = case["tokens"]
        s["tokens"] = whole(vocab, rows, n)
        s["lengths"] = torch.where(uniform(rows) < 0.5, whole(n + 1, rows), torch.full_like(s["tokens"][:, 0], n))
        s["longest"] = max(len(t) for t in _token_texts(vocab, case["tags"]))
        s["arena"] = torch.zeros(rows * n * s["longest"] + 16, device=device, dtype=torch.uint8)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    device = s.get("logits", s.get("states", s.get("tokens"))).device
    if own:
        s["pipe"] = _own_pipe(s["tags"])
        if s["tags"]:
            s["grammar"] = _own_grammar(s["vocab"], s["tags"])
    elif s["op"] in ("mask", "step"):
        s["lists"] = _grammar_on(device, s["vocab"], s["tags"])
    elif s["op"] == "lines":
        s["token_bytes"], s["token_begin"] = _token_bytes_on(device, s["vocab"], s["tags"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------

def _packed(bits):
    """Truth values (as int32, a multiple of 32 a row) as words, token t in bit t % 32 of word t // 32."""
    weight = torch.ones(32, device=bits.device, dtype=torch.int64) << torch.arange(32, device=bits.device)
    words = (bits.view(bits.shape[0], -1, 32) * weight).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _plain_counts(s):
    """Per row and token: how often it stands in the history behind the prompt, and whether it stands in the history at all."""
    rows, vocab = s["rows"], s["vocab"]
    at = torch.arange(s["history"].shape[1], device=s["history"].device)
    token = s["history"].long()
    inside = at < s["history_len"][:, None]
    behind = inside & (at >= s["prompt_len"][:, None])
    zero = torch.zeros(rows, vocab, device=token.device)
    return zero.scatter_add(1, token, behind.float()), zero.scatter_add(1, token, inside.float()) > 0


def _plain_shaped(s):
    x = s["logits"].float()
    count, seen = _plain_counts(s)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = torch.where(count > 0, x - s["presence"][:, None], x)
    if "bias" in s:
        row = s["bias_row"].long()
        x = torch.where((row >= 0)[:, None], x + s["bias"][row.clamp(min=0)], x)
    return x


def _plain_masked(s, x):
    if "mask" not in s:
        return x
    t = torch.arange(s["vocab"], device=x.device)
    allowed = (s["mask"][s["mask_row"].long()][:, t // 32] >> (t % 32).to(torch.int32)) & 1
    return x.masked_fill(allowed == 0, -math.inf)


def _plain_choice(s, x):
    t = s["temperature"][:, None]
    z = torch.where(t > 0, x / t, x)
    best = z.max(1, keepdim=True).values
    w = torch.where(z == best, torch.ones_like(z), (z - best).exp())
    w = torch.where(x > -math.inf, w, torch.zeros_like(w)).double()
    cum = w.cumsum(1)
    total = cum[:, -1:]
    first = (x == x.max(1, keepdim=True).values).to(torch.int32).argmax(1, keepdim=True)
    drawn = (cum > s["uniform"].double()[:, None] * total).to(torch.int32).argmax(1, keepdim=True)
    token = torch.where(t > 0, drawn, first)
    logprob = (z.gather(1, token).double() - best.double() - total.log()).float()
    none = best == -math.inf
    return torch.where(none, -1, token)[:, 0].to(torch.int32), torch.where(none, -math.inf, logprob)[:, 0]


def _plain_allowed(s):
    g, states = s["lists"], s["states"].long()
    at, tags = states[:, 0], states[:, 1]
    n = g["begin"][at + 1] - g["begin"][at]
    row = torch.repeat_interleave(torch.arange(s["rows"], device=at.device), n)
    entry = torch.arange(row.shape[0], device=at.device) - (n.cumsum(0) - n)[row] + g["begin"][at][row]
    kind, tags = g["kind"][entry], tags[row]
    ok = (kind == 0) | ((kind == 1) & (tags + 2 <= MAX_TAGS)) | ((kind == 2) & (tags + 1 >= MIN_TAGS))
    allowed = torch.zeros(s["rows"], (s["vocab"] + 31) // 32 * 32, device=at.device, dtype=torch.bool)
    allowed[row[ok], g["token"][entry[ok]]] = True
    return allowed


def _plain_step(s):
    g, at = s["lists"], s["states"].long()
    x = _plain_shaped(s).masked_fill(~_plain_allowed(s)[:, :s["vocab"]], -math.inf)
    token, logprob = _plain_choice(s, x)
    entry = torch.searchsorted(g["key"], at[:, 0] * s["vocab"] + token.clamp(min=0).long()).clamp(max=g["key"].shape[0] - 1)
    moved = torch.stack([g["next"][entry], at[:, 1] + (g["kind"][entry] == 1)], 1)
    return token, logprob, torch.where((token >= 0)[:, None], moved, at).to(torch.int32)


def _plain_lines(s):
    tokens = s["tokens"].long()
    inside = torch.arange(tokens.shape[1], device=tokens.device) < s["lengths"][:, None]
    begin = s["token_begin"][tokens]
    n = torch.where(inside, s["token_begin"][tokens + 1] - begin, 0)
    offsets = torch.cat([n.new_zeros(1), n.sum(1).cumsum(0)])
    n, begin = n.view(-1), begin.view(-1)
    source = torch.repeat_interleave(begin - (n.cumsum(0) - n), n)
    source = source + torch.arange(source.shape[0], device=tokens.device)
    arena = torch.zeros_like(s["arena"])
    arena[:source.shape[0]] = s["token_bytes"][source]
    return arena, offsets


def run(s):
    if own:
        return _own_run(s)
    if s["op"] == "shape":
        return _plain_masked(s, _plain_shaped(s)).to(s["logits"].dtype)
    if s["op"] == "choose":
        return _plain_choice(s, _plain_masked(s, _plain_shaped(s)))
    if s["op"] == "mask":
        return _packed(_plain_allowed(s).to(torch.int32))
    if s["op"] == "step":
        return _plain_step(s)
    return _plain_lines(s)


def _own_run(s):
    if s["op"] == "mask":
        return s["grammar"].mask(s["states"])
    if s["op"] == "lines":
        return s["grammar"].lines(s["tokens"], s["lengths"], arena=s["arena"])
    rules = {k: s.get(k) for k in ("history", "history_len", "prompt_len", "repetition", "frequency", "presence", "bias", "bias_row")}
    if s["op"] == "step":
        states = s["states"].clone()
        token, logprob = s["grammar"].step(states, s["logits"], temperature=s["temperature"], uniform=s["uniform"], **rules)
        return token, logprob, states
    rules.update(mask=s.get("mask"), mask_row=s.get("mask_row"))
    if s["op"] == "shape":
        return s["pipe"].shape_logits(s["logits"], **rules)
    return s["pipe"].choose_tokens(s["logits"], temperature=s["temperature"], uniform=s["uniform"], **rules)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------

def work(case):
    rows, vocab, op = case["rows"], case["vocab"], case["op"]
    history = rows * (4 * 0.75 * case.get("history", 0) + 32)
    if op in ("shape", "choose"):
        logits = rows * vocab * BYTES[case["type"]] * case["density"]
        tables = case["biases"] * vocab * 4 + case["masks"] * vocab / 8
        written = rows * vocab * BYTES[case["type"]] if op == "shape" else rows * 8
        return {"bytes": logits + tables + history + written, "flops": rows * vocab * case["density"] * (6 if op == "shape" else 10)}
    if op == "lines":
        texts = _token_texts(vocab, case["tags"])
        tokens = rows * case["tokens"] * 0.75
        return {"bytes": tokens * (4 + sum(map(len, texts)) / len(texts)) + rows * 12, "flops": tokens}
    begin = _plain_grammar(vocab, case["tags"])["begin"]
    n = 0.15 * float(begin[1]) + 0.85 * float(begin[-1]) / (len(begin) - 1)       # entries of a state's list, as the states are spread
    if op == "mask":
        return {"bytes": rows * (vocab / 8 + 8 + 4 * n), "flops": rows * n}
    return {"bytes": rows * (n * (4 + BYTES[case["type"]]) + 24) + history, "flops": rows * n * 10}


# ---- the operators' definition in 64 bits ----------------------------------------------------------------------------------------------

def _exact_row(s, r):
    """Row r's shaped logits before any mask, from the definition."""
    x = s["logits"][r].astype(np.float64)
    end, prompt = int(s["history_len"][r]), int(s["prompt_len"][r])
    all_of, counted = s["history"][r, :end], s["history"][r, prompt:end]
    seen = np.unique(all_of)
    x[seen] = np.where(x[seen] > 0, x[seen] / float(s["repetition"][r]), x[seen] * float(s["repetition"][r]))
    tokens, count = np.unique(counted, return_counts=True)
    x[tokens] -= float(s["frequency"][r]) * count + float(s["presence"][r])
    if "bias" in s and s["bias_row"][r] >= 0:
        x += s["bias"][s["bias_row"][r]]
    return x


def _exact_choice(s, r, x):
    """(token, log-probability) of a row whose forbidden tokens are -inf."""
    if not np.any(x > -np.inf):
        return -1, -np.inf
    t = float(s["temperature"][r])
    z = x / t if t > 0 else x
    w = np.exp(z - z.max())
    token = int(np.argmax(np.cumsum(w) > float(s["uniform"][r]) * np.cumsum(w)[-1])) if t > 0 else int(np.argmax(x))
    return token, z[token] - z.max() - np.log(w.sum())


def exact(case, seed):
    if case["op"] not in ("shape", "choose", "step"):
        return None
    s = {k: (v.float() if v.is_floating_point() else v).cpu().numpy() if torch.is_tensor(v) else v for k, v in _inputs(case, seed).items()}
    rows, vocab = case["rows"], case["vocab"]
    g = _plain_grammar(vocab, case["tags"]) if case["op"] == "step" else None
    out = np.empty((rows, vocab)) if case["op"] == "shape" else None
    token, logprob, states = np.empty(rows, np.int32), np.empty(rows), np.empty((rows, 2), np.int32)
    for r in range(rows):
        x = _exact_row(s, r)
        if g is not None:
            at, tags = (int(v) for v in s["states"][r])
            lo, hi = g["begin"][at], g["begin"][at + 1]
            ids, kind = g["token"][lo:hi], g["kind"][lo:hi]
            keep = ids[(kind == 0) | ((kind == 1) & (tags + 2 <= MAX_TAGS)) | ((kind == 2) & (tags + 1 >= MIN_TAGS))]
            y = np.full(vocab, -np.inf)
            y[keep] = x[keep]
            x = y
        elif "mask" in s:
            bits = np.unpackbits(s["mask"][s["mask_row"][r]].view(np.uint8), bitorder="little")[:vocab]
            x = np.where(bits, x, -np.inf)
        if out is not None:
            out[r] = x
            continue
        token[r], logprob[r] = _exact_choice(s, r, x)
        if g is not None:
            states[r] = at, tags
            if token[r] >= 0:
                e = lo + int(np.searchsorted(ids, token[r]))
                states[r] = g["next"][e], tags + (g["kind"][e] == 1)
    if out is not None:
        return out
    return (token, logprob) if g is None else (token, logprob, states)
