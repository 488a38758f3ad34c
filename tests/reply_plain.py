"""Plain 64-bit restatement of the entry points that write replies (include/tagpipe.h): numpy and Python sets, one token and one row at a
time, sharing nothing with the kernels or with the grammar's compiler."""
import math

import numpy as np

NONE = -1


def shaped_row(l, history=(), prompt=0, rep=1.0, freq=0.0, pres=0.0, bias=None, allowed=None):
    """x of a row in 64 bits."""
    x = np.asarray(l, dtype=np.float64).copy()
    n = len(x)
    seen, count = set(), {}
    for k, t in enumerate(history):
        t = int(t)
        if not 0 <= t < n:
            continue
        seen.add(t)
        if k >= prompt:
            count[t] = count.get(t, 0) + 1
    with np.errstate(invalid="ignore", over="ignore"):
        for t in seen:
            x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
            if t in count:
                x[t] = x[t] - freq * count[t] - pres
        if bias is not None:
            x = x + bias
    if allowed is not None:
        x = np.where(allowed, x, -np.inf)
    return x


def weights_row(x, temperature):
    """(z, weights) of a row; a NaN counts as -infinity."""
    x = np.where(np.isnan(x), -np.inf, x)
    z = x / temperature if temperature > 0 else x
    m = z.max()
    if m == -np.inf:
        return z, np.zeros(len(z))
    with np.errstate(invalid="ignore"):
        return z, np.where(z == m, 1.0, np.exp(z - m))


def choose_row(x, temperature=0.0, uniform=None):
    """(token, log-probability)."""
    t = temperature if uniform is not None and temperature > 0 else 0.0
    z, w = weights_row(x, t)
    if not w.any():
        return NONE, -math.inf
    cum = np.cumsum(w)
    if t > 0:
        above = np.nonzero((cum > uniform * cum[-1]) & (w > 0))[0]
        token = int(above[0]) if len(above) else int(np.nonzero(w)[0][-1])
    else:
        token = int(np.argmax(np.where(np.isnan(x), -np.inf, x)))
    return token, (0.0 if z[token] == z.max() else z[token] - z.max()) - math.log(w.sum())


def bits_of(words, vocab):
    """Truth values of packed mask words."""
    return np.unpackbits(np.ascontiguousarray(words).view(np.uint8), bitorder="little")[:vocab].astype(bool)


class PlainGrammar:
    def __init__(self, tags, tokens, end_token, min_tags=3, max_tags=42, spaces=False):
        self.tags = sorted({(t.replace("_", " ") if spaces else t).encode() for t in tags})
        self.whole = set(self.tags)
        self.prefixes = sorted({t[:n] for t in self.tags for n in range(len(t) + 1)})
        self.place = {p: i for i, p in enumerate(self.prefixes)}
        self.tokens, self.end_token, self.min_tags, self.max_tags = list(tokens), end_token, min_tags, max_tags
        self.after_comma, self.end = len(self.prefixes), len(self.prefixes) + 1

    def go(self, state, token):
        """The state behind `token`, or None where it is not allowed."""
        at, tags = state
        if not 0 <= at <= self.after_comma or not 0 <= token < len(self.tokens):
            return None
        if token == self.end_token:
            ends = at < self.after_comma and self.prefixes[at] in self.whole and tags + 1 >= self.min_tags
            return (self.end, tags) if ends else None
        text = self.tokens[token]
        if not text or text.count(b",") > 1:
            return None
        for i in range(len(text)):
            b = text[i:i + 1]
            if at == self.after_comma:
                if b != b" ":
                    return None
                at = 0
            elif b == b",":
                if self.prefixes[at] not in self.whole or tags + 2 > self.max_tags:
                    return None
                at, tags = self.after_comma, tags + 1
            else:
                at = self.place.get(self.prefixes[at] + b)
                if at is None:
                    return None
        return at, tags

    def allowed(self, state):
        return np.array([self.go(state, t) is not None for t in range(len(self.tokens))])

    def text(self, row):
        return b"".join(self.tokens[t] for t in row if 0 <= t < len(self.tokens) and t != self.end_token)


def token_list(rng, tags, size, spaces=False):
    """The 256 single bytes, pieces of tag lines, pieces no line holds, one of two commas, an empty one, a repeated one; the end token is the last."""
    pieces = {b", ", b",,", b"a, b, c", b"Zz%", b""}
    while len(pieces) < size - 258:
        line = ", ".join(rng.choice(tags) for _ in range(3))
        line = line.replace("_", " ") if spaces else line
        at = rng.randrange(len(line))
        pieces.add(line[at:at + rng.randint(2, 7)].encode() if rng.random() < 0.8 else b"Q%x" % rng.randrange(1 << 20))
    pieces = sorted(pieces)
    rng.shuffle(pieces)
    return [bytes([b]) for b in range(256)] + pieces + [pieces[0], b"</s>"]


TAGS = ["1girl", "solo", "long_hair", "long_hair_bow", "blue_eyes", "blue_sky", "smile", "school_uniform", "standing", "class_room", "hat", "hats", "a", "ab"]
