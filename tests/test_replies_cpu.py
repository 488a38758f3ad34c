"""The tag-line grammar's compiler against the plain restatement, and what the entry points that write replies refuse: host code, no GPU."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

from helpers import ROOT, Config, shipped_config
from reply_plain import TAGS, PlainGrammar, token_list
from imagecaptioner_amd._abi import TP_T_BF16, TP_T_F32, tp_grammar_config, tp_grammar_info, tp_logits
from imagecaptioner_amd.replies import _pack


@pytest.fixture(scope="module")
def sim():
    d = os.path.join(ROOT, "tests", "hostsim")
    subprocess.check_call(["make", "-C", d, "-s"])
    L = C.CDLL(os.path.join(d, "libtp_replysim.so"))
    V, U = C.c_void_p, C.c_uint64
    L.rsim_last_error.restype = C.c_char_p
    L.rsim_compile.restype = V
    L.rsim_compile.argtypes = [V, V]
    L.rsim_destroy.argtypes = [V]
    L.rsim_info.argtypes = [V, V]
    for name in ("begin", "token", "move", "text", "text_begin"):
        f = getattr(L, "rsim_" + name)
        f.restype, f.argtypes = V, [V]
    for name, args in (("shape", [V, V, U]), ("choose", [V] * 6 + [U]), ("mask", [C.c_uint32, V, U, V, U]), ("step", [C.c_uint32] + [V] * 6 + [C.c_int]),
                       ("lines", [V, U, C.c_uint32, V, V, U, V, U, V, V, U])):
        f = getattr(L, "rsim_check_" + name)
        f.restype, f.argtypes = C.c_char_p, args
    for name, args in (("choose", [U, C.c_uint32]), ("lines", [U])):
        f = getattr(L, "rsim_%s_workspace" % name)
        f.restype, f.argtypes = U, args
    return L


def compiled(sim, tokens, end_token, tags=None, tables=None, min_tags=3, max_tags=42, spaces=0, **fields):
    """Dict of the compiled grammar's arrays, or the refusal's text."""
    text, offsets = _pack(tokens)
    cfg = tp_grammar_config()
    cfg.struct_size = C.sizeof(tp_grammar_config)
    cfg.n_tokens, cfg.tokens, cfg.token_offsets = len(tokens), text.ctypes.data, offsets.ctypes.data
    cfg.end_token, cfg.min_tags, cfg.max_tags, cfg.spaces = end_token, min_tags, max_tags, spaces
    if tags is not None:
        tag_text, tag_offsets = _pack(tags)
        cfg.tags, cfg.tag_offsets, cfg.n_tags = tag_text.ctypes.data, tag_offsets.ctypes.data, len(tags)
    for k, v in fields.items():
        setattr(cfg, k, v)
    h = sim.rsim_compile(C.byref(cfg), C.byref(tables.struct) if tables is not None else None)
    if not h:
        return sim.rsim_last_error().decode()
    info = tp_grammar_info()
    sim.rsim_info(h, C.byref(info))

    def grab(name, n, dt):
        if not n:
            return np.zeros(0, dt)
        p = getattr(sim, "rsim_" + name)(h)
        return np.frombuffer(C.string_at(p, n * np.dtype(dt).itemsize), dtype=dt).copy()
    begin = grab("begin", info.n_prefixes + 3, np.uint32)
    out = {"info": info, "begin": begin, "token": grab("token", int(info.n_entries), np.int32), "move": grab("move", int(info.n_entries), np.uint32),
           "text_begin": grab("text_begin", info.n_tokens + 1, np.uint32)}
    out["text"] = grab("text", int(out["text_begin"][-1]), np.uint8).tobytes()
    sim.rsim_destroy(h)
    return out


def check_against_plain(g, plain):
    assert g["info"].n_prefixes == len(plain.prefixes) and g["info"].n_tags == len(plain.tags) and len(g["begin"]) == len(plain.prefixes) + 3
    for at in range(plain.end + 1):
        lo, hi = int(g["begin"][at]), int(g["begin"][at + 1])
        got = list(zip(g["token"][lo:hi].tolist(), (g["move"][lo:hi] & 0x3FFFFFFF).tolist(), (g["move"][lo:hi] >> 30).tolist()))
        want = []
        for t in range(len(plain.tokens)):
            to = plain.go((at, plain.min_tags - 1), t)          # enough tags to end, and room for one more
            if to is not None:
                want.append((t, to[0], 2 if t == plain.end_token else to[1] - (plain.min_tags - 1)))
        assert got == want, (at, plain.prefixes[at] if at < len(plain.prefixes) else at)


@pytest.mark.parametrize("spaces", [0, 1])
@pytest.mark.parametrize("seed,size", [(1, 300), (2, 700)])
def test_every_place_has_the_tokens_of_the_plain_grammar(sim, seed, size, spaces):
    rng = random.Random(seed)
    tokens = token_list(rng, TAGS, size, spaces)
    g = compiled(sim, tokens, len(tokens) - 1, TAGS, spaces=spaces)
    check_against_plain(g, PlainGrammar(TAGS, tokens, len(tokens) - 1, spaces=bool(spaces)))
    assert g["text"] == b"".join(tokens[:-1])                   # the end token has no text in a line
    assert g["info"].longest_token == max(len(t) for t in tokens[:-1])
    assert g["info"].longest_list == max(np.diff(g["begin"].astype(np.int64)))


def test_random_tags(sim):
    rng = random.Random(9)
    for _ in range(6):
        tags = sorted({"".join(rng.choice("ab_c") for _ in range(rng.randint(1, 6))) for _ in range(rng.randint(1, 40))})
        tokens = token_list(rng, tags, 420)
        end = rng.randrange(256, len(tokens))
        check_against_plain(compiled(sim, tokens, end, tags * 2, min_tags=1, max_tags=rng.choice([2, 5])), PlainGrammar(tags, tokens, end, 1, 5))


def test_tags_come_from_the_tables(sim):
    tokens = [bytes([b]) for b in range(256)] + [b""]
    cfg = Config(vocabulary=b"long_hair\nblue_eyes\nwatermark\nsolo\n:odd\nx\nsmile\nbad_one", denylist=b"bad_one")
    g = compiled(sim, tokens, 256, tables=cfg)
    check_against_plain(g, PlainGrammar(["long_hair", "blue_eyes", "solo", "smile"], tokens, 256))      # watermark and bad_one are dropped, :odd is invalid, x too short
    assert compiled(sim, tokens, 256, tables=shipped_config())["info"].n_tags > 100
    assert compiled(sim, tokens, 256, tables=Config())["info"].n_tags > 0                              # no vocabulary: the tables' own tags


def test_grammar_refusals(sim):
    tokens = [bytes([b]) for b in range(256)] + [b"", b"lo"]
    ok = dict(tokens=tokens, end_token=256, tags=TAGS)
    assert isinstance(compiled(sim, **ok), dict)

    def refused(text, **change):
        got = compiled(sim, **{**ok, **change})
        assert isinstance(got, str) and text in got, (got, change)
    refused("no tags", tags=[])
    refused("holds a comma", tags=["a,b"])
    refused("holds a comma or a control", tags=["a\tb"])
    refused("empty", tags=["solo", ""])
    refused("begins or ends with a space", tags=["solo "])
    refused("begins or ends with a space", tags=["_solo"], spaces=1)
    refused("end_token", end_token=258)
    refused("end_token", end_token=-1)
    refused("min_tags", min_tags=0)
    refused("min_tags", min_tags=5, max_tags=4)
    refused("min_tags", max_tags=65536)
    refused("spaces", spaces=2)
    refused("struct_size", struct_size=8)
    refused("n_tokens", n_tokens=0)
    refused("no token for the single byte 44", tokens=[t for t in tokens if t != b","], end_token=255)
    refused("no token for the single byte 95", tokens=[t if t != b"_" else b"zz" for t in tokens])
    refused("no token for the single byte 108", end_token=ord("l"))                                 # the end token's own text does not count
    assert compiled(sim, tokens=[t if t != b"Z" else b"zz" for t in tokens], end_token=256, tags=TAGS)   # a byte no line uses may be missing


def logits_io(**fields):
    io = tp_logits()
    io.struct_size = C.sizeof(tp_logits)
    io.type, io.rows, io.vocab, io.logits, io.stride = TP_T_F32, 3, 100, 4096, 100
    for k, v in fields.items():
        setattr(io, k, v)
    return io


HISTORY = dict(history=4096, history_stride=10, history_cap=10)
BIAS = dict(bias=4096, bias_stride=100, n_bias=2)
MASK = dict(mask=4096, mask_stride=4, n_masks=2)


@pytest.mark.parametrize("text,fields", [
    ("struct_size", dict(struct_size=8)), ("type", dict(type=3)), ("type", dict(type=-1)), ("vocab", dict(vocab=0)), ("vocab", dict(vocab=(1 << 24) + 1)),
    ("rows", dict(rows=(1 << 31) + 1)), ("no logits", dict(logits=None)), ("stride", dict(stride=99)), ("too large", dict(stride=1 << 62)),
    ("aligned", dict(logits=4098)), ("history_cap", dict(HISTORY, history_stride=9)), ("history_cap", dict(HISTORY, history_cap=1 << 31, history_stride=1 << 32)),
    ("too large", dict(HISTORY, history_stride=1 << 62)), ("without a history", dict(history_len=4096)), ("without a history", dict(prompt_len=4096)),
    ("n_bias", dict(BIAS, n_bias=0)), ("bias_stride", dict(BIAS, bias_stride=99)), ("too large", dict(BIAS, bias_stride=1 << 62)), ("without a bias", dict(bias_row=4096)),
    ("n_masks", dict(MASK, n_masks=0)), ("mask_stride", dict(MASK, mask_stride=3)), ("too large", dict(MASK, mask_stride=1 << 62)), ("without a mask", dict(mask_row=4096)),
    ("aligned", dict(HISTORY, history=4097)), ("aligned", dict(repetition=4098)), ("aligned", dict(frequency=4097)), ("aligned", dict(presence=4097)),
    ("aligned", dict(BIAS, bias_row=4097)), ("aligned", dict(MASK, mask=4097)), ("aligned", dict(MASK, mask_row=4098)),
])
def test_logit_refusals(sim, text, fields):
    io = logits_io(**fields)
    for got in (sim.rsim_check_shape(C.byref(io), 1 << 20, 1 << 62 if "stride" in fields and fields["stride"] > 100 else 100),
                sim.rsim_check_choose(C.byref(io), None, None, 4096, None, None, 0)):
        assert got is not None and text in got.decode(), (got, fields)
    if "mask" not in fields and text != "no logits":
        got = sim.rsim_check_step(io.vocab, C.byref(io), None, None, 4096, 4096, None, 0)
        assert got is not None and text in got.decode(), (got, fields)


def test_accepted_arguments(sim):
    io = logits_io(**HISTORY, **BIAS, **MASK)
    assert sim.rsim_check_shape(C.byref(io), 1 << 20, 100) is None
    assert sim.rsim_check_choose(C.byref(io), 4096, 4096, 4096, 4096, None, 0) is None
    io = logits_io(**HISTORY, **BIAS)
    assert sim.rsim_check_step(100, C.byref(io), 4096, 4096, 4096, 4096, 4096, 0) is None
    io.history_len = 4096
    assert sim.rsim_check_step(100, C.byref(io), 4096, 4096, 4096, 4096, 4096, 1) is None
    for rows in (0, 3):                                                     # no rows: pointers may be null
        io = logits_io(rows=rows, logits=None if not rows else 4096)
        assert (sim.rsim_check_shape(C.byref(io), None, 0) is None) == (rows == 0)
        assert (sim.rsim_check_choose(C.byref(io), None, None, None, None, None, 0) is None) == (rows == 0)


def test_shape_output_refusals(sim):
    io = logits_io(type=TP_T_BF16, logits=1 << 20, stride=128)
    ok = lambda out, stride: sim.rsim_check_shape(C.byref(io), out, stride)
    bytes_ = (2 * 128 + 100) * 2
    assert ok(1 << 20, 128) is None                                          # in place
    assert ok((1 << 20) + bytes_, 100) is None                               # right behind
    assert ok((1 << 20) - bytes_, 128) is None                               # right before
    for out, stride, text in ((None, 100, "no output"), (1 << 21, 99, "out_stride"), ((1 << 21) + 1, 100, "aligned"), (1 << 21, 1 << 62, "too large"),
                              (1 << 20, 100, "overlaps"), ((1 << 20) + 2, 128, "overlaps"), ((1 << 20) + bytes_ - 2, 100, "overlaps")):
        got = ok(out, stride)
        assert got is not None and text in got.decode(), (out, stride, got)
    io.rows = 1
    assert ok(1 << 20, 100) is None                                          # one row: its stride does not matter


def test_choose_mask_step_and_lines_refusals(sim):
    big = logits_io(vocab=100_000, stride=100_000)
    need = sim.rsim_choose_workspace(3, 100_000)
    assert need >= 3 * 16 and sim.rsim_choose_workspace(3, 100) == 0
    for args, text in (((None, None, None, None, 4096, need), "no tokens"), ((None, None, 4096, None, None, 0), "workspace"), ((None, None, 4096, None, 4096, need - 1), "workspace"),
                       ((None, None, 4096, None, 4104, need), "aligned to 16"), ((4097, None, 4096, None, 4096, need), "aligned"), ((None, 4097, 4096, None, 4096, need), "aligned"),
                       ((None, None, 4097, None, 4096, need), "aligned"), ((None, None, 4096, 4097, 4096, need), "aligned")):
        got = sim.rsim_check_choose(C.byref(big), *args)
        assert got is not None and text in got.decode(), (args, got)
    for args, text in (((100, None, 3, 4096, 4), "null"), ((100, 4096, 3, None, 4), "null"), ((100, 4096, 3, 4096, 3), "mask_stride"), ((100, 4097, 3, 4096, 4), "aligned"),
                       ((100, 4096, 3, 4097, 4), "aligned"), ((100, 4096, (1 << 31) + 1, 4096, 4), "rows"), ((100, 4096, 3, 4096, 1 << 62), "too large")):
        got = sim.rsim_check_mask(*args)
        assert got is not None and text in got.decode(), (args, got)
    assert sim.rsim_check_mask(100, None, 0, None, 0) is None
    for n, fields, args, text in ((99, {}, (None, None, 4096, 4096, None, 0), "n_tokens"), (100, MASK, (None, None, 4096, 4096, None, 0), "mask must be null"),
                                  (100, {}, (None, None, 4096, 4096, None, 1), "append needs"), (100, HISTORY, (None, None, 4096, 4096, None, 1), "append needs"),
                                  (100, {}, (None, None, 4096, 4096, None, 2), "append must"), (100, {}, (None, None, None, 4096, None, 0), "null"),
                                  (100, {}, (None, None, 4096, None, None, 0), "null"), (100, {}, (None, None, 4097, 4096, None, 0), "aligned"),
                                  (100, {}, (4097, None, 4096, 4096, None, 0), "aligned"), (100, {}, (None, None, 4096, 4096, 4097, 0), "aligned")):
        io = logits_io(**fields)
        got = sim.rsim_check_step(n, C.byref(io), *args)
        assert got is not None and text in got.decode(), (fields, args, got)
    io = logits_io(logits=None)
    assert sim.rsim_check_step(100, C.byref(io), None, None, 4096, 4096, None, 0) is None        # no logits: the caller's own tokens
    ws = sim.rsim_lines_workspace(3)
    base = [4096, 10, 10, None, None, 3, 4096, 100, 4096, 4096, ws]
    assert sim.rsim_check_lines(*base) is None
    for at, v, text in ((0, None, "null"), (0, 4097, "aligned"), (1, 9, "stride"), (2, 1 << 31, "width"), (3, 4097, "aligned"), (4, 4097, "aligned"), (5, (1 << 31) + 1, "rows"),
                        (6, None, "null"), (8, None, "no offsets"), (8, 4100, "aligned"), (9, None, "workspace"), (9, 4104, "aligned to 16"), (10, ws - 1, "workspace"),
                        (1, 1 << 62, "too large")):
        args = list(base)
        args[at] = v
        got = sim.rsim_check_lines(*args)
        assert got is not None and text in got.decode(), (at, v, got)


def test_null_handles_are_refused_by_the_library():
    from imagecaptioner_amd import load_library
    L = load_library()
    io = logits_io()
    assert L.tp_shape_logits(None, C.byref(io), 4096, 100) == -1
    assert L.tp_choose_tokens(None, C.byref(io), None, None, 4096, None, None, 0) == -1
    assert not L.tp_grammar_create(None, None) and b"null" in L.tp_last_error()
    assert L.tp_grammar_get_info(None, None) == -1
    assert L.tp_grammar_mask(None, 4096, 1, 4096, 4, None) == -1
    assert L.tp_grammar_step(None, C.byref(io), None, None, 4096, 4096, None, 0) == -1
    assert L.tp_grammar_lines(None, 4096, 1, 1, None, None, 1, 4096, 1, 4096, 4096, 100, None) == -1
    L.tp_grammar_destroy(None)


def test_the_torch_module_refuses_without_a_device():
    """Everything is checked before the library is called: with tensors of the host there is nothing else to do."""
    import torch

    from imagecaptioner_amd.replies import _native
    native = _native()
    x, i = torch.zeros(2, 40), torch.zeros(2, dtype=torch.int32)
    states = torch.zeros(2, 2, dtype=torch.int32)
    for text, call in (("logits must be a Float tensor", lambda: native.shape(None, 0, 0, x, None, {})), ("logits must be a tensor", lambda: native.shape(None, 0, 0, 7, None, {})),
                       ("float32, float16 or bfloat16", lambda: native.choose(None, 0, 0, x.double(), None, None, {})), ("states must be", lambda: native.mask(None, 0, 0, states, 2, None)),
                       ("states must be", lambda: native.step(None, 0, 0, states, x, None, None, False, {})), ("states must be", lambda: native.advance(None, 0, 0, states, 40, i, False, {})),
                       ("tokens must be a Int tensor", lambda: native.lines(None, 0, 0, x, None, None, None, 5)), ("requires a gradient", lambda: native.shape(None, 0, 0, x.clone().requires_grad_(), None, {}))):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(TypeError):
        native.shape(None, 0, 0, x, None)
    # device -1 is the host's: the checks of the rules, up to the library's own refusal of a context that is none
    from imagecaptioner_amd import TagPipeError
    for error, text, rules in ((ValueError, "history_len or prompt_len without a history", dict(history_len=i)), (ValueError, "bias_row without a bias", dict(bias_row=i)),
                               (ValueError, "mask must be", dict(mask=torch.zeros(2, 3, dtype=torch.int32))), (ValueError, "bias must be", dict(bias=torch.zeros(39))), (ValueError, "bias has 0 rows", dict(bias=torch.zeros(0, 40))),
                               (ValueError, "history must be", dict(history=x)), (ValueError, r"history must be .*\(2, -1\)", dict(history=torch.zeros(3, 4, dtype=torch.int32))),
                               (ValueError, r"repetition must be .*\(2,\)", dict(repetition=torch.ones(3))), (ValueError, "repetition must be .*not contiguous", dict(repetition=torch.ones(4)[::2])),
                               (TypeError, "unexpected keyword argument 'penalty'", dict(penalty=i)), (TagPipeError, "null argument", dict(bias=None, mask=torch.zeros(2, dtype=torch.int32)))):
        with pytest.raises(error, match=text):
            native.shape(None, -1, 0, x, None, rules)
    with pytest.raises(ValueError, match="a temperature needs"):
        native.choose(None, -1, 0, x, torch.ones(2), None, {})
    with pytest.raises(ValueError, match="one state per row"):
        native.step(None, -1, 0, torch.zeros(3, 2, dtype=torch.int32), x, None, None, False, {})


def test_struct_layouts_match_the_header(tmp_path):
    from imagecaptioner_amd import _abi
    names = ("tp_logits", "tp_grammar_config", "tp_grammar_info")
    checks = ['printf("%%zu\\n", sizeof(%s));' % n for n in names]
    checks += ['printf("%%zu\\n", offsetof(%s, %s));' % (n, f) for n in names for f, _ in getattr(_abi, n)._fields_]
    (tmp_path / "p.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tagpipe.h"\nint main(void) { %s return 0; }' % " ".join(checks))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "p"), str(tmp_path / "p.c")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "p")]).split()]
    want = [C.sizeof(getattr(_abi, n)) for n in names] + [getattr(getattr(_abi, n), f).offset for n in names for f, _ in getattr(_abi, n)._fields_]
    assert got == want
