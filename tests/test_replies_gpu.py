"""The entry points that write replies (shape_logits, choose_tokens, the tag-line grammar, run_tokens) on the GPU, against the plain 64-bit
restatement in reply_plain.py and, for the captions, against the oracle."""
import math
import random

import numpy as np
import pytest

from helpers import Config, Oracle, assert_same_results
from reply_plain import TAGS, PlainGrammar, bits_of, choose_row, shaped_row, token_list, weights_row

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF32 = 2.0 ** -24                                    # half a step of a 32-bit float, relative


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x), device="cuda", dtype=dtype)


@pytest.fixture(scope="module")
def pipe():
    from imagecaptioner_amd import TagPipe
    return TagPipe(Config(vocabulary="\n".join(TAGS).encode()))


class Rules:
    """Random rules for rows of logits: the tensors the calls take and what the plain form needs of them."""

    def __init__(self, rng, rows, vocab, history=0, bias=0, mask=0, density=0.5, odd=False):
        self.rows, self.vocab = rows, vocab
        self.args, self.cap = {}, history
        if history:
            hot = rng.integers(0, vocab, size=max(1, history // 3))
            self.history = np.where(rng.random((rows, history)) < 0.6, rng.choice(hot, size=(rows, history)), rng.integers(0, vocab, size=(rows, history))).astype(np.int32)
            self.len = rng.integers(0, history + 1, size=rows).astype(np.int32)
            self.len[0] = history
            self.prompt = (rng.random(rows) * 0.5 * history).astype(np.int32)
            if odd:                                    # tokens that are none, lengths outside the room, prompts behind the end
                self.history[:, ::5] = rng.choice([-1, -7, vocab, vocab + 5, 2 ** 31 - 1, -2 ** 31], size=self.history[:, ::5].shape)
                self.len[rows // 2] = history + 9
                self.len[rows // 3] = -4
                self.prompt[-1], self.prompt[0] = history + 3, -2
            self.rep = rng.uniform(0.7, 1.6, rows).astype(np.float32)
            self.freq, self.pres = rng.uniform(-0.5, 0.8, rows).astype(np.float32), rng.uniform(-0.5, 0.8, rows).astype(np.float32)
            self.args.update(history=dev(self.history), history_len=dev(self.len), prompt_len=dev(self.prompt), repetition=dev(self.rep),
                             frequency=dev(self.freq), presence=dev(self.pres))
        self.n_bias, self.n_mask = bias, mask
        if bias:
            self.bias = rng.normal(size=(bias, vocab)).astype(np.float32)
            self.bias_row = rng.integers(-1, bias + (2 if odd else 0), size=rows).astype(np.int32)
            self.args.update(bias=dev(self.bias), bias_row=dev(self.bias_row))
        if mask:
            words = (vocab + 31) // 32
            self.mask = np.packbits(rng.random((mask, words * 32)) < density, axis=1, bitorder="little").view(np.int32).copy()
            if mask > 1:
                self.mask[mask - 1] = 0
            self.mask_row = rng.integers(-1 if odd else 0, mask + (2 if odd else 0), size=rows).astype(np.int32)
            self.args.update(mask=dev(self.mask), mask_row=dev(self.mask_row))

    def plain(self, l, r):
        """(x in 64 bits, the largest size an intermediate value has, allowed)"""
        kw, size = {}, np.abs(np.asarray(l, np.float64))
        if self.cap:
            n = min(max(int(self.len[r]), 0), self.cap)
            h = self.history[r, :n]
            rep, freq, pres = float(self.rep[r]), float(self.freq[r]), float(self.pres[r])
            kw.update(history=h, prompt=min(max(int(self.prompt[r]), 0), self.cap), rep=rep, freq=freq, pres=pres)
            size = size * max(rep, 1 / rep)
            tokens, count = np.unique(h[(h >= 0) & (h < self.vocab)], return_counts=True)
            size[tokens] += abs(freq) * count + abs(pres)
        if self.n_bias and 0 <= self.bias_row[r] < self.n_bias:
            kw["bias"] = self.bias[self.bias_row[r]].astype(np.float64)
            size = size + np.abs(kw["bias"])
        allowed = np.ones(self.vocab, bool)
        if self.n_mask and 0 <= self.mask_row[r] < self.n_mask:
            allowed = bits_of(self.mask[self.mask_row[r]], self.vocab)
        return shaped_row(l, allowed=allowed, **kw), size, allowed


def check_shaped(got, l, rules, dtype):
    """Five 32-bit operations at most (the repetition, freq * n, three sums), each off by half a step of an intermediate value, then one rounding to the type."""
    half = torch.finfo(dtype).eps / 2
    got = got.double().cpu().numpy()
    for r in range(rules.rows):
        x, size, allowed = rules.plain(l[r], r)
        assert np.all(got[r][~allowed] == -np.inf), r
        with np.errstate(invalid="ignore"):
            bound = 5 * HALF32 * size * 1.001 + (half * np.abs(x) * 1.01 + 2.0 ** -25 if dtype != torch.float32 else 0)   # 2^-25: half of fp16's smallest step
            ok = np.where(np.isfinite(x), np.abs(got[r] - x) <= bound, (got[r] == x) | (np.isnan(got[r]) & np.isnan(x)))
        assert ok[allowed].all(), (r, np.nonzero(~ok & allowed)[0][:5])


def make_logits(rng, rows, vocab, dtype, scale=3.0):
    t = dev(rng.normal(size=(rows, vocab)) * scale, torch.float32).to(dtype)
    return t, t.double().cpu().numpy()


@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 8), (5, 100), (2, 8191), (3, 8192), (4, 8193), (7, 50021), (1, 70000)])
def test_shape(pipe, name, rows, vocab):
    rng = np.random.default_rng(rows * vocab)
    logits, l = make_logits(rng, rows, vocab, TYPES[name])
    for kw in (dict(history=40, bias=2, mask=rows), dict(history=700, odd=True, mask=3, bias=1), dict(), dict(mask=2, density=0.02), dict(bias=1), dict(history=1)):
        rules = Rules(rng, rows, vocab, **kw)
        check_shaped(pipe.shape_logits(logits, **rules.args), l, rules, TYPES[name])


@pytest.mark.parametrize("name", sorted(TYPES))
def test_shape_in_place_strided_and_unaligned(pipe, name):
    rng = np.random.default_rng(3)
    dtype, rows, vocab, stride = TYPES[name], 5, 9001, 9013
    for first in (0, 1, 3):                                               # rows of any alignment
        room = torch.full((rows * stride + 8,), 7.0, device="cuda", dtype=dtype)
        view = room[first:first + rows * stride].view(rows, stride)[:, :vocab]
        src, l = make_logits(rng, rows, vocab, dtype)
        view.copy_(src)
        before = room.clone()
        rules = Rules(rng, rows, vocab, history=90, bias=2, mask=rows)
        apart = pipe.shape_logits(view, **rules.args)
        check_shaped(apart, l, rules, dtype)
        assert torch.equal(room, before)                                 # inputs stay as they are
        assert pipe.shape_logits(view, out=view, **rules.args) is view
        assert torch.equal(view, apart)
        gaps = torch.ones_like(room, dtype=torch.bool)
        gaps[first:first + rows * stride].view(rows, stride)[:, :vocab] = False
        assert torch.equal(room[gaps], before[gaps])                     # what lies between and behind the rows too


def test_shape_rules_in_views(pipe):
    """Tables, masks and histories that are parts of larger tensors."""
    rng = np.random.default_rng(4)
    rows, vocab = 6, 5003
    logits, l = make_logits(rng, rows, vocab, torch.float32)
    rules = Rules(rng, rows, vocab, history=30, bias=3, mask=4)
    wide = {k: torch.zeros(v.shape[0], v.shape[1] + 13, device="cuda", dtype=v.dtype) for k, v in rules.args.items() if v.dim() == 2}
    for k, w in wide.items():
        w[:, 5:5 + rules.args[k].shape[1]] = rules.args[k]
    args = {k: wide[k][:, 5:5 + v.shape[1]] if k in wide else v for k, v in rules.args.items()}
    check_shaped(pipe.shape_logits(logits, **args), l, rules, torch.float32)
    rules.len[:] = 30                                                       # no lengths: every row is full, and ends at its width
    full = {k: v for k, v in args.items() if k != "history_len"}
    check_shaped(pipe.shape_logits(logits, **full), l, rules, torch.float32)


@pytest.mark.parametrize("name", sorted(TYPES))
def test_masked_places_may_hold_anything(pipe, name):
    vocab = 300
    bad = [math.inf, -math.inf, math.nan, torch.finfo(TYPES[name]).min, torch.finfo(TYPES[name]).max]
    l = np.zeros((2, vocab))
    l[:, ::3] = np.resize(bad, l[:, ::3].shape)
    l[:, 1::3] = np.arange(100) % 37
    allowed = np.arange(vocab) % 3 != 0
    mask = dev(np.packbits(np.resize(allowed, 320), bitorder="little").view(np.int32)[None])
    logits = dev(l, torch.float32).to(TYPES[name])
    out = pipe.shape_logits(logits, mask=mask, bias=torch.ones(vocab, device="cuda")).double().cpu().numpy()
    assert np.all(out[:, ~allowed] == -np.inf) and np.array_equal(out[:, allowed], l[:, allowed] + 1)
    token, logprob = pipe.choose_tokens(logits, mask=mask)
    assert token.tolist() == [3 * 36 + 1] * 2 and torch.isfinite(logprob).all()
    nothing = torch.zeros_like(mask)
    assert torch.all(pipe.shape_logits(logits, mask=nothing) == -math.inf)
    token, logprob = pipe.choose_tokens(logits, mask=nothing)
    assert token.tolist() == [-1, -1] and torch.all(logprob == -math.inf)
    # not masked: infinities and NaN go through the formula
    out = pipe.shape_logits(logits, bias=torch.ones(vocab, device="cuda")).double().cpu().numpy()
    want = logits.double().cpu().numpy()[:, ::3]
    assert np.array_equal(np.isnan(out[:, ::3]), np.isnan(want)) and np.array_equal(out[:, ::3] == -np.inf, want == -np.inf)


def check_choice(token, logprob, xs, sizes, temperature, uniform):
    """The token against the 64-bit distribution.  z = x / T is off by e = (5 + 1) half steps of the largest intermediate over T.  A weight is 2^(z * log2 e - c): log2 e and
    the fused product are off by two half steps relative, which moves the weight by 2 half steps times |ln w|, taken as 4;
    the power itself is off by one step (two half steps), and a sum of 1024 weights by six roundings to 32 bits, taken as 10.  u * sum may fall on the other side of
    a border by that share of the sum."""
    for r, x in enumerate(xs):
        t = float(temperature[r]) if temperature is not None and uniform is not None and temperature[r] > 0 else 0.0
        got, lp = int(token[r]), float(logprob[r])
        z, w = weights_row(x, t)
        if not w.any():
            assert got == -1 and lp == -math.inf, r
            continue
        fine = np.isfinite(z) & (sizes[r] < np.inf)
        e = 6 * HALF32 * (sizes[r][fine].max() if fine.any() else 0) / (t or 1.0)
        spread = np.abs(z[fine] - z[fine].max()) if fine.any() else np.zeros(1)
        live = spread[spread < 104]                                       # expf is 0 below -104
        share = 2 * e + 4 * HALF32 * (live.max() if len(live) else 0) + (2 + 10) * HALF32
        assert 0 <= got < len(x) and w[got] > 0, r
        if t > 0:
            cum, total = np.cumsum(w), w.sum()
            target = min(max(float(uniform[r]), 0.0), 1.0) * total
            assert cum[got] >= target - share * total and cum[got] - w[got] <= target + share * total, (r, got)
        else:
            assert z[got] >= z.max() - 2 * e, (r, got)
        want = (0.0 if z[got] == z.max() else z[got] - z.max()) - math.log(w.sum())
        assert abs(lp - want) <= 2 * e + 2 * share + 2 * HALF32 * abs(want), (r, lp, want)


@pytest.mark.parametrize("rows,vocab", [(2, 50021), (3, 9000), (5, 3000), (1, 200001), (520, 17000)])
def test_long_histories(pipe, rows, vocab):
    """More history than a launch keeps of it at once, most of it distinct."""
    rng = np.random.default_rng(rows)
    logits, l = make_logits(rng, rows, vocab, torch.float16)
    rules = Rules(rng, rows, vocab, history=20000 if rows < 500 else 4200, bias=1)
    rules.history[:, ::2] = rng.integers(0, vocab, size=rules.history[:, ::2].shape)
    rules.args["history"] = dev(rules.history)
    temperature, uniform = choice_numbers(rng, rows)
    some = range(rows) if rows < 500 else [0, 1, 2, 259, 519]
    got = pipe.shape_logits(logits, **rules.args)
    token, logprob = (v.cpu().numpy() for v in pipe.choose_tokens(logits, temperature=dev(temperature), uniform=dev(uniform), **rules.args))
    if rows < 500:
        check_shaped(got, l, rules, torch.float16)
    xs, sizes, _ = zip(*(rules.plain(l[r], r) for r in some))
    some = list(some)
    check_choice(token[some], logprob[some], xs, sizes, temperature[some], uniform[some])


def choice_numbers(rng, rows):
    temperature = np.where(rng.random(rows) < 0.3, 0.0, rng.uniform(0.3, 1.5, rows)).astype(np.float32)
    uniform = rng.random(rows).astype(np.float32)
    uniform[0] = 0.0
    if rows > 2:
        uniform[1], temperature[1], uniform[2], temperature[2] = np.float32(1 - 2.0 ** -24), 0.9, 0.0, 0.8
    return temperature, uniform


@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (9, 100), (4, 8192), (5, 8193), (260, 9000), (6, 50021), (33, 20000), (2, 300001)])
def test_choose(pipe, name, rows, vocab):
    rng = np.random.default_rng(rows + vocab)
    logits, l = make_logits(rng, rows, vocab, TYPES[name])
    temperature, uniform = choice_numbers(rng, rows)
    for kw in (dict(history=50, bias=2, mask=rows), dict(), dict(history=300, odd=True, bias=1, mask=2), dict(mask=rows, density=0.003)):
        rules = Rules(rng, rows, vocab, **kw)
        xs, sizes, _ = zip(*(rules.plain(l[r], r) for r in range(rows)))
        for tu in (dict(temperature=dev(temperature), uniform=dev(uniform)), dict()):
            token, logprob = pipe.choose_tokens(logits, **tu, **rules.args)
            check_choice(token.cpu().numpy(), logprob.cpu().numpy(), xs, sizes, temperature if tu else None, uniform if tu else None)
            again = pipe.choose_tokens(logits, **tu, **rules.args)
            assert torch.equal(token, again[0]) and torch.equal(logprob, again[1])          # the same bits every time


@pytest.mark.parametrize("vocab", [9, 8192, 20011])
def test_choose_ties_and_specials(pipe, vocab):
    l = np.full((9, vocab), -1.0)
    rng = np.random.default_rng(vocab)
    ties = [np.sort(rng.choice(vocab, size=4, replace=False)) for _ in range(9)]
    for r, at in enumerate(ties):
        l[r, at] = 5.0
    l[1, ties[1]] = math.inf                                             # infinities share the weight
    l[2, ties[2]] = math.nan                                             # a NaN is never chosen
    l[3, :] = -math.inf                                                  # nothing to choose
    l[4, :] = -math.inf
    l[4, ties[4][2]] = -3e38                                             # one token left
    temperature = np.array([0, 0, 0, 1, 1, 1, math.nan, -1, math.inf], np.float32)
    uniform = np.array([0.9, 0.9, 0.9, 0.5, 0.5, 1.5, 0.5, 0.5, 0.999999], np.float32)
    temperature[5] = 1e-3                                                # only the four ties have a weight: u >= 1 takes the last of them
    for name, dtype in TYPES.items():
        token, logprob = pipe.choose_tokens(dev(l, torch.float32).to(dtype), temperature=dev(temperature), uniform=dev(uniform))
        token, logprob = token.cpu().numpy(), logprob.cpu().numpy()
        first = int(np.nonzero(l[2] == -1.0)[0][0])
        left = int(ties[4][2]) if name != "f16" else -1                 # fp16 has no such number: -infinity
        assert token[:8].tolist() == [ties[0][0], ties[1][0], first, -1, left, ties[5][3], ties[6][0], ties[7][0]], name
        assert abs(token[8] - 0.999999 * vocab) <= 1 + vocab * 1e-6     # an infinite temperature: every token weighs the same
        lp = [0] * 8 + [-math.log(vocab)]
        lp[0] = lp[6] = lp[7] = -math.log(4 + (vocab - 4) * math.exp(-6))
        lp[1] = lp[5] = -math.log(4)
        lp[2] = -math.log(vocab - 4)
        lp[3] = -math.inf
        lp[4] = 0.0 if left >= 0 else -math.inf
        assert np.allclose(logprob, lp, rtol=1e-6, atol=1e-6), (name, logprob, lp)          # 4 half steps of each weight and of the logarithm
    u = dev(np.float32([-0.5, 0.0, 0.5, 0.9999999]))
    flat = torch.zeros(4, vocab, device="cuda")
    token, _ = pipe.choose_tokens(flat, temperature=torch.ones(4, device="cuda"), uniform=u)
    assert token.tolist() == [0, 0, int(0.5 * vocab), vocab - 1]        # cumulative weights k + 1 > u * vocab: exact in 64 bits


@pytest.mark.parametrize("vocab", [7, 4000, 140000])
def test_extreme_temperatures(pipe, vocab):
    """z = x / T in 32 bits: far above 1 every token weighs the same, far below the largest x is alone, and where the quotients overflow those that do share the weight."""
    rng = np.random.default_rng(vocab)
    l = rng.permutation(vocab).astype(np.float32) / 64 + 1.0
    l[rng.random(vocab) < 0.3] *= -1
    flat, sharp, over = [1e29, 1e31, 3e38, np.inf], [1e-29, 1e-31, 1e-33], [1e-40, 2e-45]
    temperature = np.array(flat + sharp + over, np.float32)
    uniform = rng.random(len(temperature)).astype(np.float32)
    rows = len(temperature)
    logits = dev(np.repeat(l[None], rows, 0))
    for rules, left in ((dict(), np.ones(vocab, bool)), (dict(mask=dev(np.packbits(np.pad(np.arange(vocab) % 3 == 1, (0, -vocab % 32)), bitorder="little").view(np.int32)[None])), np.arange(vocab) % 3 == 1)):
        token, logprob = pipe.choose_tokens(logits, temperature=dev(temperature), uniform=dev(uniform), **rules)
        at = np.nonzero(left)[0]
        up = np.nonzero(left & (l > 0))[0]
        for r in range(rows):
            of = at if r < len(flat) else up if r >= len(flat) + len(sharp) else [at[np.argmax(l[at])]]
            k = int(np.searchsorted(of, int(token[r])))
            assert of[k] == int(token[r]) and abs(k - float(uniform[r]) * len(of)) <= 1, (r, int(token[r]))       # cumulative weights are whole numbers: exact
            assert abs(float(logprob[r]) + math.log(len(of))) <= 2 * HALF32 * math.log(max(len(of), 2)), r


@pytest.mark.parametrize("vocab", [7, 4000, 140000])
def test_large_logits(pipe, vocab):
    """Whole multiples of every size of unit, which no operation before the weights rounds."""
    rng = np.random.default_rng(vocab)
    units = [2.0 ** p for p in (-3, 0, 5, 10, 16, 20, 23, 24, 26, 28, 29, 30, 31, 40, 64, 100, 120)]
    l = np.concatenate([rng.integers(lo, hi, (len(units), vocab)) * np.array(units)[:, None] for lo, hi in ((-6, 7), (100, 108), (-108, -100))])
    rows = len(l)
    temperature, uniform = np.where(np.arange(rows) % 2, 1.0, 0.5).astype(np.float32), rng.random(rows).astype(np.float32)
    token, logprob = (v.cpu().numpy() for v in pipe.choose_tokens(dev(l, torch.float32), temperature=dev(temperature), uniform=dev(uniform)))
    assert np.isfinite(logprob).all()
    check_choice(token, logprob, list(l), [np.zeros(vocab)] * rows, temperature, uniform)


@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", [(40, 50021), (3, 300001), (260, 140000)])
def test_choose_under_masks_that_empty_segments(pipe, name, rows, vocab):
    rng = np.random.default_rng(rows)
    logits, l = make_logits(rng, rows, vocab, TYPES[name])
    rules = Rules(rng, rows, vocab, history=60, bias=1, mask=5, density=2e-4)
    allowed = bits_of(rules.mask[0], vocab).nonzero()[0]
    rules.history[:, ::4] = rng.choice(allowed, size=rules.history[:, ::4].shape)                                  # repeated and allowed
    rules.mask[1], rules.mask[2] = 0, 0
    rules.mask[1, -1] = 1                                                 # one token near the end, in a segment behind empty ones
    rules.mask[2, 3] = 1 << 7
    rules.args.update(history=dev(rules.history), mask=dev(rules.mask))
    temperature, uniform = choice_numbers(rng, rows)
    some = list(range(rows)) if rows < 100 else list(range(0, rows, 20))
    for tu in (dict(temperature=dev(temperature), uniform=dev(uniform)), dict()):
        token, logprob = (v.cpu().numpy() for v in pipe.choose_tokens(logits, **tu, **rules.args))
        xs, sizes, _ = zip(*(rules.plain(l[r], r) for r in some))
        check_choice(token[some], logprob[some], xs, sizes, temperature[some] if tu else None, uniform[some] if tu else None)


@pytest.mark.parametrize("name", sorted(TYPES))
def test_signalling_nans(pipe, name):
    """NaNs of either kind among the logits, in every position of a lane's eight, hide no larger number beside them."""
    bits = {"f32": (torch.int32, [0x7F800001, -0x7FFFFF, 0x7FC00000]), "f16": (torch.int16, [0x7C01, -0x3FF, 0x7E00]), "bf16": (torch.int16, [0x7F81, -0x7F, 0x7FC0])}[name]
    rows, vocab = 64, 3001
    rng = np.random.default_rng(77)
    logits, l = make_logits(rng, rows, vocab, TYPES[name])
    at = rng.random((rows, vocab)) < 0.4
    raw = logits.view(bits[0])
    raw[dev(at)] = dev(rng.choice(bits[1], size=int(at.sum())), bits[0])
    l[at] = np.nan
    token, logprob = pipe.choose_tokens(logits)
    assert token.tolist() == np.nanargmax(l, axis=1).tolist()
    temperature, uniform = choice_numbers(rng, rows)
    token, logprob = pipe.choose_tokens(logits, temperature=dev(temperature), uniform=dev(uniform))
    check_choice(token.cpu().numpy(), logprob.cpu().numpy(), [np.where(at[r], -np.inf, l[r]) for r in range(rows)], [np.abs(np.nan_to_num(l[r])) for r in range(rows)], temperature, uniform)
    shaped = pipe.shape_logits(logits).double().cpu().numpy()
    assert np.array_equal(np.isnan(shaped), at) and np.array_equal(shaped[~at], l[~at])


@pytest.mark.parametrize("rows,vocab,history", [(65537, 12, 3), (2 ** 21 + 3, 1, 1), (70001, 40, 0)])
def test_more_rows_than_a_launch_takes(pipe, rows, vocab, history):
    """Integers a 16-bit float holds: every value and every choice of the largest is exact."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    logits = torch.randint(-60, 60, (rows, vocab), generator=gen, device="cuda").to(torch.float16)
    rules, want = {}, logits.double()
    if history:
        h = torch.randint(0, vocab, (rows, history), generator=gen, device="cuda", dtype=torch.int32)
        rules = dict(history=h, presence=torch.full((rows,), 2.0, device="cuda"), frequency=torch.full((rows,), 3.0, device="cuda"))
        count = torch.zeros(rows, vocab, device="cuda", dtype=torch.float64).scatter_add_(1, h.long(), torch.ones(rows, history, device="cuda", dtype=torch.float64))
        want = want - 3 * count - 2 * (count > 0)
    bits = torch.randint(-2 ** 31, 2 ** 31 - 1, (5, (vocab + 31) // 32), generator=gen, device="cuda").to(torch.int32)
    pick = torch.arange(rows, device="cuda", dtype=torch.int32) % 5
    rules.update(mask=bits, mask_row=pick)
    allowed = (bits[pick.long()][:, torch.arange(vocab, device="cuda") // 32] >> (torch.arange(vocab, device="cuda", dtype=torch.int32) % 32)) & 1
    want = torch.where(allowed > 0, want, -math.inf)
    assert torch.equal(pipe.shape_logits(logits, **rules).double(), want)
    token, _ = pipe.choose_tokens(logits, **rules)
    best = want.max(1).values
    first = torch.where(want == best[:, None], torch.arange(vocab, device="cuda"), vocab).min(1).values
    assert torch.equal(token.long(), torch.where(best > -math.inf, first, -1))


def test_the_largest_vocabulary(pipe):
    """2^24 tokens, and an odd million: windows, segments and history tables of a row's last tokens."""
    rng = np.random.default_rng(78)
    for vocab in (2 ** 24, 1200003):
        logits, l = make_logits(rng, 2, vocab, torch.bfloat16, scale=1.0)
        rules = Rules(rng, 2, vocab, history=300, bias=1, mask=2)
        rules.history[:, :3] = [vocab - 1, vocab - 2, vocab - 1025]
        rules.mask[:, -40:], rules.mask_row[:] = -1, 0
        rules.args.update(history=dev(rules.history), mask=dev(rules.mask), mask_row=dev(rules.mask_row))
        check_shaped(pipe.shape_logits(logits, **rules.args), l, rules, torch.bfloat16)
        xs, sizes, _ = zip(*(rules.plain(l[r], r) for r in range(2)))
        temperature, uniform = np.float32([1, 0.8]), np.float32([0.9999999, 0.3])
        for tu in (dict(temperature=dev(temperature), uniform=dev(uniform)), dict()):
            token, logprob = pipe.choose_tokens(logits, **tu, **rules.args)
            check_choice(token.cpu().numpy(), logprob.cpu().numpy(), xs, sizes, temperature if tu else None, uniform if tu else None)


def test_rows_beyond_32_bit_offsets(pipe):
    """Rows that start 2^32 elements and more into their tensors."""
    far, vocab = 2 ** 32 + 3, 1000
    rng = np.random.default_rng(8)
    room = torch.empty(far + vocab, device="cuda", dtype=torch.bfloat16)
    logits = room.as_strided((2, vocab), (far, 1))
    src, l = make_logits(rng, 2, vocab, torch.bfloat16)
    logits.copy_(src)
    wide = torch.empty(2 ** 31 + 40, device="cuda", dtype=torch.int32)
    history = wide.as_strided((2, 30), (2 ** 31 + 5, 1))
    rules = Rules(rng, 2, vocab, history=30, bias=1, mask=2)
    history.copy_(rules.args["history"])
    rules.args["history"] = history
    check_shaped(pipe.shape_logits(logits, **rules.args), l, rules, torch.bfloat16)
    apart = pipe.shape_logits(logits, **rules.args)
    assert torch.equal(pipe.shape_logits(logits, out=logits, **rules.args), apart)
    del room, logits
    xs, sizes, _ = zip(*(rules.plain(l[r], r) for r in range(2)))
    token, logprob = pipe.choose_tokens(src, **rules.args)
    check_choice(token.cpu().numpy(), logprob.cpu().numpy(), xs, sizes, None, None)
    tokens = [bytes([b]) for b in range(256)] + [b"", b"hat, "]
    g = pipe.tag_grammar(tokens, 256)
    history.copy_(dev(np.array([[257, 104] * 15, [97, 257] * 15]), torch.int32))
    arena, offsets = g.lines(history)
    assert bytes(arena[:int(offsets[2])].cpu().numpy()) == b"hat, h" * 15 + b"ahat, " * 15
    torch.cuda.empty_cache()


# ---- the grammar -------------------------------------------------------------------------------------------------------------------

def small_grammar(pipe, seed=1, size=600, **kw):
    tokens = token_list(random.Random(seed), TAGS, size, kw.get("spaces", False))
    kept = [t for t in TAGS if len(t) > 1]                                # the line ingest drops a tag of one character (Program.cs:600)
    return pipe.tag_grammar(tokens, len(tokens) - 1, **kw), PlainGrammar(kept, tokens, len(tokens) - 1, **kw), tokens


def every_state(plain):
    at = list(range(-2, plain.end + 3))
    return np.array([(a, t) for a in at for t in sorted({0, 1, plain.min_tags - 2, plain.min_tags - 1, plain.max_tags - 2, plain.max_tags - 1, plain.max_tags}) if t >= 0], np.int32)


@pytest.mark.parametrize("kw", [dict(), dict(spaces=True, min_tags=1, max_tags=2), dict(min_tags=2, max_tags=2)])
def test_grammar_mask(pipe, kw):
    g, plain, tokens = small_grammar(pipe, **kw)
    states = every_state(plain)
    mask = g.mask(dev(states)).cpu().numpy()
    for r, s in enumerate(states):
        assert np.array_equal(bits_of(mask[r], len(tokens)), plain.allowed((int(s[0]), int(s[1])))), s
        assert not np.unpackbits(mask[r].view(np.uint8), bitorder="little")[len(tokens):].any()
    words = mask.shape[1]
    room = torch.full((len(states), words + 3), -9, device="cuda", dtype=torch.int32)
    g.mask(dev(states), out=room[:, 1:1 + words])
    assert np.array_equal(room[:, 1:1 + words].cpu().numpy(), mask) and torch.all(room[:, 0] == -9) and torch.all(room[:, 1 + words:] == -9)


def words_grammar(pipe, count=9000, vocab=70001):
    """A place with more tokens than one block's tables hold, over a vocabulary of several mask pieces."""
    rng = random.Random(5)
    letters = "bcdfghjklmnpqrstvwxz"
    tags = sorted({"".join(rng.choice(letters) for _ in range(4)) for _ in range(count)})
    pieces = sorted({t[:n].encode() for t in tags for n in (2, 3, 4)})
    rng.shuffle(pieces)
    tokens = [bytes([b]) for b in range(256)] + pieces
    tokens += [b"Q%d" % i for i in range(vocab - 1 - len(tokens))] + [b""]
    order = list(range(256, len(tokens) - 1))
    rng.shuffle(order)
    tokens[256:-1] = [tokens[i] for i in order]
    return pipe.tag_grammar(tokens, len(tokens) - 1, tags=tags), PlainGrammar(tags, tokens, len(tokens) - 1), tokens


@pytest.fixture(scope="module")
def wide_grammar(pipe):
    return words_grammar(pipe)


def test_grammar_mask_of_long_lists(wide_grammar):
    g, plain, tokens = wide_grammar
    assert g.info.longest_list > 9000
    states = np.array([(0, 0), (plain.place[b"bc"] if b"bc" in plain.place else 1, 3), (plain.place[plain.tags[7]], 41), (plain.place[plain.tags[8]], 1),
                       (plain.after_comma, 2), (plain.end, 3)], np.int32)
    mask = g.mask(dev(states)).cpu().numpy()
    for r, s in enumerate(states):
        assert np.array_equal(bits_of(mask[r], len(tokens)), plain.allowed((int(s[0]), int(s[1])))), s


def check_step(g, plain, tokens, states, name, rules, l, logits, temperature, uniform, append=False):
    rows = len(states)
    moving = dev(states)
    args = dict(rules.args)
    tu = dict(temperature=dev(temperature), uniform=dev(uniform)) if temperature is not None else {}
    token, logprob = g.step(moving, logits, append=append, **tu, **args)
    token, logprob, moved = token.cpu().numpy(), logprob.cpu().numpy(), moving.cpu().numpy()
    xs, sizes = [], []
    for r in range(rows):
        x, size, _ = rules.plain(l[r], r)
        xs.append(np.where(plain.allowed((int(states[r, 0]), int(states[r, 1]))), x, -np.inf))
        sizes.append(size)
    room = [not append or min(max(int(rules.len[r]), 0), rules.cap) < rules.cap for r in range(rows)]
    with_room = [r for r in range(rows) if room[r]]
    check_choice(token[with_room], logprob[with_room], [xs[r] for r in with_room], [sizes[r] for r in with_room],
                 temperature[with_room] if temperature is not None else None, uniform[with_room] if uniform is not None else None)
    for r in range(rows):
        s = (int(states[r, 0]), int(states[r, 1]))
        if not room[r]:
            assert token[r] == -1 and logprob[r] == -math.inf
        want = s if token[r] < 0 else plain.go(s, int(token[r]))
        assert tuple(moved[r]) == want, (r, s, token[r], moved[r])
    if append:
        history, length = args["history"].cpu().numpy(), args["history_len"].cpu().numpy()
        for r in range(rows):
            n = min(max(int(rules.len[r]), 0), rules.cap)
            if token[r] >= 0:
                assert length[r] == n + 1 and history[r, n] == token[r]
                assert np.array_equal(np.delete(history[r], n), np.delete(rules.history[r], n))
            else:
                assert length[r] == rules.len[r] and np.array_equal(history[r], rules.history[r])
    return token


@pytest.mark.parametrize("name", sorted(TYPES))
def test_grammar_step(pipe, name):
    g, plain, tokens = small_grammar(pipe)
    rng = np.random.default_rng(21)
    states = every_state(plain)
    rows = len(states)
    logits, l = make_logits(rng, rows, len(tokens), TYPES[name])
    temperature, uniform = choice_numbers(rng, rows)
    for kw in (dict(), dict(history=60, bias=2), dict(history=20, odd=True, bias=1)):
        rules = Rules(rng, rows, len(tokens), **kw)
        check_step(g, plain, tokens, states, name, rules, l, logits, temperature, uniform)
        check_step(g, plain, tokens, states, name, rules, l, logits, None, None)
    rules = Rules(rng, rows, len(tokens), history=12)
    rules.len[::4] = 12                                                   # full rows get no token
    rules.args["history_len"] = dev(rules.len)
    check_step(g, plain, tokens, states, name, rules, l, logits, temperature, uniform, append=True)


def test_grammar_step_on_long_lists(wide_grammar):
    g, plain, tokens = wide_grammar
    rng = np.random.default_rng(22)
    states = np.array([(0, 0)] * 9 + [(plain.after_comma, 2), (plain.place[plain.tags[11]], 4), (0, 41)], np.int32)
    logits, l = make_logits(rng, len(states), len(tokens), torch.bfloat16, scale=1.0)
    temperature, uniform = choice_numbers(rng, len(states))
    uniform[3:9], temperature[3:9] = [0.1, 0.3, 0.5, 0.7, 0.9, 1.5], 1.2  # a token of every piece, and the last
    for kw in (dict(), dict(history=800, bias=1)):
        rules = Rules(rng, len(states), len(tokens), **kw)
        check_step(g, plain, tokens, states, "bf16", rules, l, logits, temperature, uniform)
        check_step(g, plain, tokens, states, "bf16", rules, l, logits, None, None)


@pytest.mark.parametrize("count,lo,hi", [(800, 1500, 2048), (1800, 2049, 4096), (3500, 4097, 8192)])
def test_grammar_step_by_the_longest_list(pipe, count, lo, hi):
    g, plain, tokens = words_grammar(pipe, count, 20011)
    assert lo <= g.info.longest_list <= hi, g.info.longest_list
    rng = np.random.default_rng(count)
    states = np.array([(0, 0)] * 9 + [(plain.after_comma, 2), (plain.place[plain.tags[11]], 4), (0, 41), (plain.place[plain.tags[5][:1]], 3)], np.int32)
    logits, l = make_logits(rng, len(states), len(tokens), torch.float16, scale=1.0)
    temperature, uniform = choice_numbers(rng, len(states))
    uniform[3:9], temperature[3:9] = [0.1, 0.3, 0.5, 0.7, 0.9, 1.5], 1.2
    for kw in (dict(), dict(history=1300, bias=1)):                       # 1024 entries of history go into a table at once
        rules = Rules(rng, len(states), len(tokens), **kw)
        check_step(g, plain, tokens, states, "f16", rules, l, logits, temperature, uniform)
        check_step(g, plain, tokens, states, "f16", rules, l, logits, None, None)


def test_grammar_step_of_large_logits(pipe, wide_grammar):
    for g, plain, tokens in (small_grammar(pipe), wide_grammar):
        rng = np.random.default_rng(29)
        units = np.array([2.0 ** p for p in (-3, 0, 10, 24, 29, 30, 64, 120)])
        states = np.zeros((len(units), 2), np.int32)
        l = rng.integers(100, 108, (len(units), len(tokens))) * units[:, None]
        temperature, uniform = np.ones(len(units), np.float32), rng.random(len(units)).astype(np.float32)
        rules = Rules(rng, len(units), len(tokens))
        token, logprob = (v.cpu().numpy() for v in g.step(dev(states), dev(l, torch.float32), temperature=dev(temperature), uniform=dev(uniform)))
        allowed = plain.allowed((0, 0))
        check_choice(token, logprob, [np.where(allowed, x, -np.inf) for x in l], [np.zeros(len(tokens))] * len(units), temperature, uniform)


def test_step_is_choose_under_the_grammars_mask(pipe, wide_grammar):
    rng = np.random.default_rng(23)
    for g, plain, tokens in (small_grammar(pipe), wide_grammar):
        rows = 64
        states = np.stack([rng.integers(0, plain.end + 1, rows), rng.integers(0, 42, rows)], 1).astype(np.int32)
        states[::4, 0] = 0
        logits, _ = make_logits(rng, rows, len(tokens), torch.float32)
        rules = Rules(rng, rows, len(tokens), history=100, bias=2)
        tu = [dev(v) for v in choice_numbers(rng, rows)]
        token, logprob = g.step(dev(states), logits, temperature=tu[0], uniform=tu[1], **rules.args)
        mask = g.mask(dev(states))
        other, logprob2 = pipe.choose_tokens(logits, temperature=tu[0], uniform=tu[1], mask=mask, mask_row=torch.arange(rows, device="cuda", dtype=torch.int32), **rules.args)
        assert torch.equal(token, other)
        assert torch.allclose(logprob[token >= 0], logprob2[token >= 0], rtol=1e-6, atol=1e-6) and torch.equal(logprob[token < 0], logprob2[token < 0])


def test_grammar_on_more_rows_than_a_launch_takes(pipe):
    tokens = [b"a", b"b", b",", b" ", b"ab", b"", b"b, "]
    g, plain = pipe.tag_grammar(tokens, 5, tags=["ab", "aba"], min_tags=2), PlainGrammar(["ab", "aba"], tokens, 5, min_tags=2)
    rows = 2 ** 21 + 70003
    gen = torch.Generator(device="cuda").manual_seed(4)
    kinds = every_state(plain)
    which = torch.randint(0, len(kinds), (rows,), generator=gen, device="cuda")
    states = dev(kinds)[which]
    logits = torch.randn(rows, 7, generator=gen, device="cuda")
    mask = g.mask(states)
    want = dev(np.array([np.packbits(plain.allowed((int(a), int(b))), bitorder="little")[0] for a, b in kinds], np.int32))[which]
    assert torch.equal(mask[:, 0], want)
    allowed = (want[:, None] >> torch.arange(7, device="cuda", dtype=torch.int32)) & 1
    x = torch.where(allowed > 0, logits, -math.inf)
    token, _ = g.step(states, logits)
    best = x.max(1)
    assert torch.equal(token.long(), torch.where(best.values > -math.inf, best.indices, -1))
    to = {(k, t): plain.go((int(s[0]), int(s[1])), t) for k, s in enumerate(kinds) for t in range(7) if plain.allowed((int(s[0]), int(s[1])))[t]}
    table = np.repeat(kinds[:, None, :], 8, axis=1)                        # [.., 7]: no token, the state stays
    for (k, t), s in to.items():
        table[k, t] = s
    went = dev(table)[which, torch.where(token < 0, 7, token.long())]
    assert torch.equal(states, went)
    again = dev(kinds)[which]
    g.advance(again, token)
    assert torch.equal(again, went)


def test_grammar_advance(pipe):
    g, plain, tokens = small_grammar(pipe)
    rng = np.random.default_rng(24)
    states = np.repeat(every_state(plain), 4, axis=0)
    given = rng.integers(-1, len(tokens), len(states)).astype(np.int32)
    for r in range(0, len(states), 2):                                    # every other token is an allowed one
        ok = np.nonzero(plain.allowed((int(states[r, 0]), int(states[r, 1]))))[0]
        if len(ok):
            given[r] = rng.choice(ok)
    given[5], given[9] = len(tokens) + 7, -3
    moving = dev(states)
    g.advance(moving, dev(given))
    for r, got in enumerate(moving.cpu().numpy()):
        s = (int(states[r, 0]), int(states[r, 1]))
        want = s if given[r] == -1 else plain.go(s, int(given[r])) or (-1, s[1])
        assert tuple(got) == want, (r, s, given[r])
    history, length = torch.full((len(states), 2), -5, device="cuda", dtype=torch.int32), dev(np.arange(len(states)) % 3, torch.int32)
    again = dev(states)
    g.advance(again, dev(given), history=history, history_len=length, append=True)
    for r in range(len(states)):
        s, n = (int(states[r, 0]), int(states[r, 1])), r % 3
        to = plain.go(s, int(given[r]))
        if n == 2 or given[r] == -1:                                      # a full row does not move
            assert tuple(again[r].tolist()) == s and history[r].tolist() == [-5, -5] and int(length[r]) == n
        elif to is None:
            assert tuple(again[r].tolist()) == (-1, s[1]) and int(length[r]) == n
        else:
            assert tuple(again[r].tolist()) == to and history[r, n] == given[r] and int(length[r]) == n + 1


# ---- the lines ----------------------------------------------------------------------------------------------------------------------

def lines_of(plain, rows, first, last):
    return [plain.text(row[a:b]) for row, a, b in zip(rows, first, last)]


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 300), (5, 64), (4, 65), (64, 70), (65, 20), (70, 131), (4100, 9), (4099, 200), (70001, 2)])
def test_lines(pipe, rows, width):
    g, plain, tokens = small_grammar(pipe)
    rng = np.random.default_rng(rows * width)
    t = rng.integers(-2, len(tokens) + 2, (rows, width)).astype(np.int32)
    first, last = rng.integers(0, width // 2 + 1, rows).astype(np.int32), rng.integers(0, width + 1, rows).astype(np.int32)
    first[0], last[0] = 0, width
    first[-1], last[-1] = (-3, width + 5) if rows > 1 else (first[-1], last[-1])
    a, b = np.clip(first, 0, width), np.clip(last, 0, width)
    for args, texts in ((dict(), lines_of(plain, t, [0] * rows, [width] * rows)), (dict(lengths=dev(last)), lines_of(plain, t, [0] * rows, b)),
                        (dict(lengths=dev(last), begin=dev(first)), lines_of(plain, t, a, b))):
        want = b"".join(texts)
        arena, offsets = g.lines(dev(t), **args)
        offs = offsets.cpu().numpy()
        assert np.array_equal(offs, np.cumsum([0] + [len(x) for x in texts]))
        assert bytes(arena[:len(want) + 16].cpu().numpy()) == (want + b"\0" * 16)[:arena.shape[0]]
        for cut in {0, 1, len(want) // 2, len(want), len(want) + 5}:      # a smaller arena: nothing at or behind its end
            room = torch.full((len(want) + 64,), 0x55, device="cuda", dtype=torch.uint8)
            _, o2 = g.lines(dev(t), arena=room[:cut], **args)
            got = bytes(room.cpu().numpy())
            assert torch.equal(o2, offsets) and got[:cut] == (want + b"\0" * 16)[:cut] and set(got[cut:]) <= {0x55}, cut
    wide = torch.full((rows, width + 3), 65, device="cuda", dtype=torch.int32)
    wide[:, 1:1 + width] = dev(t)
    arena, offsets = g.lines(wide[:, 1:1 + width])
    assert bytes(arena[:int(offsets[-1])].cpu().numpy()) == b"".join(lines_of(plain, t, [0] * rows, [width] * rows))


def test_lines_of_long_tokens(pipe):
    """Texts around and beyond the 1008 bytes that 64 tokens are collected in, at every offset within 16 bytes."""
    rng = random.Random(3)
    texts = [bytes(rng.choice(b"abcdef") for _ in range(n)) for n in (1, 7, 8, 9, 15, 16, 17, 31, 63, 250, 1000, 1007, 1008, 1009, 1024, 5000)]
    tokens = [bytes([b]) for b in range(256)] + texts + [b""]
    g = pipe.tag_grammar(tokens, len(tokens) - 1)
    plain = PlainGrammar(["ab"], tokens, len(tokens) - 1)
    rows = []
    for r in range(64):
        row = [ord("x")] * (r % 17) + [256 + rng.randrange(len(texts)) for _ in range(r % 5)] + [256] * (70 if r % 3 else 0) + [256 + (r % len(texts))]
        rows.append(row + [-1] * (100 - len(row)))
    t = np.array(rows, np.int32)
    arena, offsets = g.lines(dev(t))
    want = [plain.text(row) for row in rows]
    assert offsets.tolist() == np.cumsum([0] + [len(x) for x in want]).tolist()
    assert bytes(arena[:int(offsets[-1])].cpu().numpy()) == b"".join(want)
    for first in range(1, 16):                                             # an arena of any alignment
        room = torch.full((int(offsets[-1]) + 64,), 0x55, device="cuda", dtype=torch.uint8)
        g.lines(dev(t), arena=room[first:first + int(offsets[-1])])
        got = bytes(room.cpu().numpy())
        assert got[first:first + int(offsets[-1])] == b"".join(want) and set(got[:first] + got[first + int(offsets[-1]):]) == {0x55}


def test_nothing_to_do(pipe):
    g, plain, tokens = small_grammar(pipe)
    empty = torch.zeros(0, len(tokens), device="cuda")
    assert pipe.shape_logits(empty).shape == (0, len(tokens))
    assert [len(x) for x in pipe.choose_tokens(empty)] == [0, 0]
    assert g.mask(g.start(0)).shape[0] == 0 and len(g.step(g.start(0), empty)[0]) == 0
    arena, offsets = g.lines(torch.zeros(0, 4, device="cuda", dtype=torch.int32))
    assert offsets.tolist() == [0]
    arena, offsets = g.lines(torch.zeros(3, 0, device="cuda", dtype=torch.int32))
    assert offsets.tolist() == [0] * 4
    assert pipe.run_tokens(g, torch.zeros(0, 4, device="cuda", dtype=torch.int32)).n_files == 0
    one = torch.ones(2, 9, device="cuda")
    none = torch.zeros(2, 0, device="cuda", dtype=torch.int32)
    assert torch.equal(pipe.shape_logits(one, history=none, history_len=torch.ones(2, device="cuda", dtype=torch.int32), repetition=torch.full((2,), 2.0, device="cuda")), one)


# ---- together -------------------------------------------------------------------------------------------------------------------------

def write_replies(pipe, g, plain, rng, rows, steps, prompt=3):
    """Replies written from random logits; returns (history, history_len, prompt_len, the states)."""
    vocab = g.info.n_tokens
    history = torch.randint(0, vocab, (rows, prompt + steps), device="cuda", dtype=torch.int32)
    prompt_len = torch.full((rows,), prompt, device="cuda", dtype=torch.int32)
    length = prompt_len.clone()
    states = g.start(rows)
    rep = torch.full((rows,), 1.3, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    bias = torch.zeros(vocab, device="cuda")
    bias[vocab - 1] = 3.0                                                  # an end that comes
    for _ in range(steps):
        logits = torch.randn(rows, vocab, generator=gen, device="cuda").mul_(2.0).to(torch.bfloat16)
        g.step(states, logits, temperature=torch.ones(rows, device="cuda"), uniform=torch.rand(rows, generator=gen, device="cuda"), append=True,
               history=history, history_len=length, prompt_len=prompt_len, repetition=rep, bias=bias)
    return history, length, prompt_len, states


@pytest.mark.parametrize("spaces", [False, True])
def test_written_replies_become_captions(pipe, spaces):
    g, plain, tokens = small_grammar(pipe, spaces=spaces, max_tags=12)
    rng = np.random.default_rng(31)
    rows = 200
    history, length, prompt, states = write_replies(pipe, g, plain, rng, rows, 150)
    ended = (states[:, 0] == g.end_place).cpu().numpy()
    assert ended.mean() > 0.9
    rows_of = [h[3:n] for h, n in zip(history.cpu().numpy(), length.cpu().numpy())]
    texts = [plain.text(r) for r in rows_of]
    for r, text in enumerate(texts):
        tags = text.split(b", ")
        if ended[r]:
            assert rows_of[r][-1] == len(tokens) - 1 and 3 <= len(tags) <= 12 and set(tags) <= plain.whole, text
    got = pipe.run_tokens(g, history, length, begin=prompt)
    cfg = Config(vocabulary="\n".join(TAGS).encode())
    want = Oracle(cfg).run_texts([t.decode() for t in texts])
    assert_same_results(got, want, pipe.histogram_dict(got.histogram), "written replies")
    assert not (got.verdicts["flags"][ended] & 0x10).any()                 # no finished line is rejected
    same = pipe.run_texts([t.decode() for t in texts])
    assert np.array_equal(same.captions, got.captions) and np.array_equal(same.fired, got.fired) and np.array_equal(same.facet_choice, got.facet_choice)


def test_a_captured_loop_replays(pipe):
    """Steps, masks, choices and lines in one graph, replayed with new logits; every replay equals the eager calls."""
    g, plain, tokens = small_grammar(pipe)
    rows, vocab, steps = 17, len(tokens), 5
    rng = np.random.default_rng(33)
    logits, uniform = torch.empty(steps, rows, vocab, device="cuda", dtype=torch.bfloat16), torch.empty(steps, rows, device="cuda")
    temperature, rep = torch.ones(rows, device="cuda"), torch.full((rows,), 1.2, device="cuda")
    big = torch.empty(2, 20000, device="cuda")

    def loop():
        states = g.start(rows)
        history, length = torch.zeros(rows, steps, device="cuda", dtype=torch.int32), torch.zeros(rows, device="cuda", dtype=torch.int32)
        picks = []
        for k in range(steps):
            picks += g.step(states, logits[k], temperature=temperature, uniform=uniform[k], history=history, history_len=length, repetition=rep, append=True)
        mask = g.mask(states)
        free = pipe.choose_tokens(logits[0], mask=mask, mask_row=torch.arange(rows, device="cuda", dtype=torch.int32))
        wide = pipe.choose_tokens(big, temperature=temperature[:2], uniform=uniform[0, :2])
        shaped = pipe.shape_logits(logits[1], history=history, history_len=length, repetition=rep)
        arena, offsets = g.lines(history, length)
        return [*picks, states, mask, *free, *wide, shaped, offsets], arena

    def fill():
        logits.copy_(dev(rng.normal(size=logits.shape) * 3, torch.float32))
        uniform.copy_(dev(rng.random(uniform.shape), torch.float32))
        big.copy_(dev(rng.normal(size=big.shape), torch.float32))
    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loop()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, held_arena = loop()
    for _ in range(4):
        fill()
        graph.replay()
        torch.cuda.synchronize()
        want, arena = loop()
        for a, b in zip(held, want):
            assert torch.equal(a, b)
        n = int(want[-1][-1])
        assert torch.equal(held_arena[:n], arena[:n])


def test_run_tokens_finds_the_sizes_first_where_the_bound_is_large(pipe, monkeypatch):
    from imagecaptioner_amd import replies
    g, plain, tokens = small_grammar(pipe, max_tags=12)
    history, length, prompt, _ = write_replies(pipe, g, plain, np.random.default_rng(36), 40, 60)
    want = pipe.run_tokens(g, history, length, begin=prompt)
    monkeypatch.setattr(replies, "MOST_ARENA", 100)
    got = pipe.run_tokens(g, history, length, begin=prompt)
    assert np.array_equal(want.captions, got.captions) and np.array_equal(want.caption_offsets, got.caption_offsets)
    assert pipe.run_tokens(g, history[:0], length[:0]).n_files == 0


def test_gradients_are_refused_or_reported(pipe):
    """What is given requires no gradient, and a backward pass whose kept values are shaped in place says so."""
    x = torch.randn(2, 50, device="cuda")
    one = torch.ones(2, device="cuda")
    for rules in (dict(bias=torch.zeros(50, device="cuda", requires_grad=True)), dict(repetition=one.clone().requires_grad_(), history=torch.zeros(2, 3, device="cuda", dtype=torch.int32)),
                  dict(out=torch.zeros(2, 50, device="cuda", requires_grad=True))):
        with pytest.raises(ValueError, match="gradient"):
            pipe.shape_logits(x, **rules)
        with torch.no_grad():
            pipe.shape_logits(x, **rules)
    with pytest.raises(ValueError, match="gradient"):
        pipe.choose_tokens(x, temperature=one.clone().requires_grad_(), uniform=one)
    leaf = x.clone().requires_grad_()
    kept = leaf.exp()                                                      # its backward pass multiplies by what it holds
    pipe.shape_logits(kept.detach(), out=kept.detach(), bias=torch.ones(50, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()


def test_two_streams_at_once(pipe):
    g, plain, tokens = small_grammar(pipe)
    rng = np.random.default_rng(35)
    logits = [make_logits(rng, 40, 30000, torch.float32)[0] for _ in range(2)]
    tu = [dev(v) for v in choice_numbers(rng, 40)]
    want = [pipe.choose_tokens(x, temperature=tu[0], uniform=tu[1]) for x in logits]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(pipe.choose_tokens(logits[k], temperature=tu[0], uniform=tu[1]))
    torch.cuda.synchronize()
    for k in range(2):
        for token, logprob in got[k]:
            assert torch.equal(token, want[k][0]) and torch.equal(logprob, want[k][1])


def test_binding_refusals(pipe):
    from imagecaptioner_amd import TagPipeError
    g, plain, tokens = small_grammar(pipe)
    x = torch.zeros(2, len(tokens), device="cuda")
    i32 = dict(device="cuda", dtype=torch.int32)
    for call in (lambda: pipe.shape_logits(x.cpu()), lambda: pipe.shape_logits(x.double()), lambda: pipe.shape_logits(x[0]), lambda: pipe.shape_logits(x.t()),
                 lambda: pipe.shape_logits(x.requires_grad_(True)) if not x.requires_grad else None,
                 lambda: pipe.shape_logits(x.detach(), out=torch.zeros(2, 5, device="cuda")), lambda: pipe.shape_logits(x.detach(), out=x.detach().half()),
                 lambda: pipe.shape_logits(x.detach(), history=torch.zeros(2, 3, device="cuda")), lambda: pipe.shape_logits(x.detach(), history=torch.zeros(3, 3, **i32)),
                 lambda: pipe.shape_logits(x.detach(), history_len=torch.zeros(2, **i32)), lambda: pipe.shape_logits(x.detach(), bias=torch.zeros(7, device="cuda")),
                 lambda: pipe.shape_logits(x.detach(), bias_row=torch.zeros(2, **i32)), lambda: pipe.shape_logits(x.detach(), mask=torch.zeros(2, 3, **i32)),
                 lambda: pipe.shape_logits(x.detach(), bias=torch.zeros(0, len(tokens), device="cuda")), lambda: pipe.shape_logits(x.detach(), repetition=torch.ones(2).half().cuda()),
                 lambda: pipe.choose_tokens(x.detach(), temperature=torch.ones(2, device="cuda")), lambda: pipe.choose_tokens(x.detach(), temperature=1.0),
                 lambda: g.step(g.start(3), x.detach()), lambda: g.step(g.start(2).long(), x.detach()), lambda: g.mask(torch.zeros(2, 3, **i32)),
                 lambda: g.mask(torch.zeros(2, 4, **i32)[:, :2]), lambda: g.lines(torch.zeros(2, 3, device="cuda")), lambda: g.lines(torch.zeros(2, 3, **i32), torch.zeros(3, **i32)),
                 lambda: pipe.tag_grammar(tokens, -1), lambda: pipe.tag_grammar(tokens, len(tokens) - 1, max_tags=1 << 33)):
        with pytest.raises((ValueError, AttributeError)):
            call()
    x = x.detach()
    for call in (lambda: pipe.shape_logits(x[:1].expand(2, -1)), lambda: pipe.shape_logits(x, out=x.view(-1).as_strided((2, len(tokens)), (len(tokens) - 1, 1))),
                 lambda: g.step(g.start(2), x[:, :-1].contiguous()), lambda: g.step(g.start(2), x, append=True), lambda: g.step(g.start(2), x, mask=torch.zeros(len(tokens) // 32 + 1, **i32)[None]),
                 lambda: pipe.tag_grammar(tokens, len(tokens) - 1, tags=[]), lambda: pipe.tag_grammar([b"a"], 0), lambda: pipe.tag_grammar(tokens, len(tokens) - 1, min_tags=9, max_tags=8)):
        with pytest.raises(TagPipeError):
            call()


def test_the_grammar_outlives_its_context():
    from imagecaptioner_amd import TagPipe
    p = TagPipe(Config(vocabulary="\n".join(TAGS).encode()))
    g, plain, tokens = small_grammar(p)
    p.close()
    states = np.array([(0, 0), (plain.place[b"solo"], 2)], np.int32)
    mask = g.mask(dev(states)).cpu().numpy()
    for r, s in enumerate(states):
        assert np.array_equal(bits_of(mask[r], len(tokens)), plain.allowed((int(s[0]), int(s[1]))))
    g.close()
