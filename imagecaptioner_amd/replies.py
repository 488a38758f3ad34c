"""Writing the replies: the torch side of tp_shape_logits, tp_choose_tokens and the tag-line grammar (include/tagpipe.h).

A captioning model that runs on the pipeline's GPU leaves its logits there, one row per reply.  The calls here work on
torch tensors of that device, on torch's current stream, without waiting for it, so they can be captured into a graph:

    pipe = TagPipe(Config(vocabulary="top_tags.txt"))
    grammar = pipe.tag_grammar(token_texts, end_token=2)
    states = grammar.start(rows)
    for _ in range(steps):
        logits = model(history, history_len)                    # [rows, vocab]
        grammar.step(states, logits, history=history, history_len=history_len, prompt_len=prompt_len, repetition=repetition, append=True)
    result = pipe.run_tokens(grammar, history, history_len, begin=prompt_len)

Nothing here has a gradient: the calls shape what a model answers while it answers.
"""
import ctypes as C

import numpy as np

from ._abi import TP_E_CAPACITY, VERDICT_DTYPE, tp_counters, tp_device_io, tp_grammar_config, tp_grammar_info, tp_logits
from .tagpipe import BatchResult, TagPipeError, load_library

_TYPES = None


def _torch():
    global _TYPES
    import torch
    if _TYPES is None:
        _TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    return torch


def _stream(torch, device):
    return torch.cuda.current_stream(device).cuda_stream


def _tensor(name, t, device, dtype, shape):
    """t's data pointer after the checks every argument gets; -1 in `shape` takes any size.  The last axis must be dense."""
    if t.dtype is not dtype or t.get_device() != device:
        raise ValueError("%s must be a %s tensor on cuda:%d, got %s on %s" % (name, dtype, device, t.dtype, t.device))
    if t.dim() != len(shape) or any(want not in (-1, got) for want, got in zip(shape, t.shape)):
        raise ValueError("%s must have the shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    if shape and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("%s must be dense along its last axis" % name)
    return t.data_ptr() or None


def _row_stride(t):
    """Elements between rows; where there is one row at most, its length."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def logit_rules(device, rows, vocab, *, history=None, history_len=None, prompt_len=None, repetition=None, frequency=None, presence=None,
                bias=None, bias_row=None, mask=None, mask_row=None):
    """A tp_logits without its logits.

    history int32 [rows, n] with history_len int32 [rows] (every row is full without it); entries before prompt_len int32 [rows] count as
    repeated but not for frequency and presence.  repetition, frequency, presence: float32 [rows].
    bias float32 [n, vocab] (or [vocab]) with bias_row int32 [rows]: which one a row takes, -1 none; row 0 for all without it.
    mask int32 [n, (vocab + 31) // 32] (or one row) with mask_row likewise: token t is allowed when bit t % 32 of word t // 32 is set."""
    torch = _torch()
    io = tp_logits()
    io.struct_size = C.sizeof(tp_logits)
    io.rows, io.vocab = rows, vocab
    i32, f32 = torch.int32, torch.float32
    if history is not None:
        io.history = _tensor("history", history, device, i32, (rows, -1))
        io.history_stride, io.history_cap = _row_stride(history), history.shape[1]
        if history_len is not None:
            io.history_len = _tensor("history_len", history_len, device, i32, (rows,))
        if prompt_len is not None:
            io.prompt_len = _tensor("prompt_len", prompt_len, device, i32, (rows,))
        if io.history is None:                                # no rows, or rows of no room: there is no history, whatever the lengths say
            io.history_len = io.prompt_len = None
    elif history_len is not None or prompt_len is not None:
        raise ValueError("history_len or prompt_len without a history")
    if repetition is not None:
        io.repetition = _tensor("repetition", repetition, device, f32, (rows,))
    if frequency is not None:
        io.frequency = _tensor("frequency", frequency, device, f32, (rows,))
    if presence is not None:
        io.presence = _tensor("presence", presence, device, f32, (rows,))
    if bias is not None:
        bias = bias if bias.dim() == 2 else bias[None]
        io.bias = _tensor("bias", bias, device, f32, (-1, vocab))
        io.bias_stride, io.n_bias = _row_stride(bias), bias.shape[0]
        if bias_row is not None:
            io.bias_row = _tensor("bias_row", bias_row, device, i32, (rows,))
        if bias.shape[0] == 0:
            raise ValueError("bias has no rows")
    elif bias_row is not None:
        raise ValueError("bias_row without a bias")
    if mask is not None:
        mask = mask if mask.dim() == 2 else mask[None]
        io.mask = _tensor("mask", mask, device, i32, (-1, (vocab + 31) // 32))
        io.mask_stride, io.n_masks = _row_stride(mask), mask.shape[0]
        if mask_row is not None:
            io.mask_row = _tensor("mask_row", mask_row, device, i32, (rows,))
        if mask.shape[0] == 0:
            raise ValueError("mask has no rows")
    elif mask_row is not None:
        raise ValueError("mask_row without a mask")
    io.stream = _stream(torch, device)
    return io


def _with_logits(device, logits, rules):
    torch = _torch()
    if logits.dim() != 2 or logits.dtype not in _TYPES:
        raise ValueError("logits must be a float32, float16 or bfloat16 tensor [rows, vocab], got %s %s" % (logits.dtype, tuple(logits.shape)))
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("logits require a gradient, which this call does not have: detach them")
    io = logit_rules(device, logits.shape[0], logits.shape[1], **rules)
    io.logits = _tensor("logits", logits, device, logits.dtype, (-1, -1))
    io.type, io.stride = _TYPES[logits.dtype], _row_stride(logits)
    return io


def _choice_inputs(device, rows, temperature, uniform):
    torch = _torch()
    t = None if temperature is None else _tensor("temperature", temperature, device, torch.float32, (rows,))
    u = None if uniform is None else _tensor("uniform", uniform, device, torch.float32, (rows,))
    if t is not None and u is None and rows:
        raise ValueError("a temperature needs `uniform`, the random numbers of the choice")
    return t, u


def shape_logits(pipe, logits, out, rules):
    torch = _torch()
    device = pipe._cfg.struct.device
    io = _with_logits(device, logits, rules)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    to = _tensor("out", out, device, logits.dtype, tuple(logits.shape))
    pipe._check(pipe._L.tp_shape_logits(pipe._h, C.byref(io), to, _row_stride(out)))
    return out


def choose_tokens(pipe, logits, temperature, uniform, rules):
    torch = _torch()
    device = pipe._cfg.struct.device
    io = _with_logits(device, logits, rules)
    rows = logits.shape[0]
    t, u = _choice_inputs(device, rows, temperature, uniform)
    need = pipe._L.tp_choose_workspace(rows, logits.shape[1])
    workspace = torch.empty(need, dtype=torch.uint8, device=logits.device)       # torch's own pool keeps it apart per stream and per graph
    tokens = torch.empty(rows, dtype=torch.int32, device=logits.device)
    logprob = torch.empty(rows, dtype=torch.float32, device=logits.device)
    pipe._check(pipe._L.tp_choose_tokens(pipe._h, C.byref(io), t, u, tokens.data_ptr(), logprob.data_ptr(), workspace.data_ptr(), need))
    return tokens, logprob


def _pack(texts):
    bs = [t.encode("utf-8") if isinstance(t, str) else bytes(t) for t in texts]
    offsets = np.zeros(len(bs) + 1, dtype=np.uint64)
    if bs:
        offsets[1:] = np.cumsum([len(b) for b in bs], dtype=np.uint64)
    return np.frombuffer(b"".join(bs) + b"\0", dtype=np.uint8), offsets


class TagGrammar:
    """The grammar of a tag line over a model's token list, resident on the device (tp_grammar_create)."""

    def __init__(self, pipe, tokens, end_token, min_tags=3, max_tags=42, spaces=False, tags=None):
        self._L = load_library()
        self._h = None
        text, offsets = _pack(tokens)
        cfg = tp_grammar_config()
        cfg.struct_size = C.sizeof(tp_grammar_config)
        for name, v, top in (("min_tags", min_tags, 65535), ("max_tags", max_tags, 65535), ("end_token", end_token, 2 ** 24)):
            if not 0 <= v <= top:                              # ctypes would cut a larger number
                raise ValueError("%s must be 0 .. %d, got %d" % (name, top, v))
        cfg.n_tokens, cfg.tokens, cfg.token_offsets = len(offsets) - 1, text.ctypes.data, offsets.ctypes.data
        cfg.end_token, cfg.min_tags, cfg.max_tags, cfg.spaces = int(end_token), int(min_tags), int(max_tags), int(bool(spaces))
        if tags is not None:
            tag_text, tag_offsets = _pack(tags)
            cfg.tags, cfg.tag_offsets, cfg.n_tags = tag_text.ctypes.data, tag_offsets.ctypes.data, len(tag_offsets) - 1
        self._h = self._L.tp_grammar_create(pipe._h, C.byref(cfg))
        if not self._h:
            raise TagPipeError(-2, self._L.tp_last_error().decode("utf-8", "replace"))
        self.info = tp_grammar_info()
        self._check(self._L.tp_grammar_get_info(self._h, C.byref(self.info)))
        self.device = pipe._cfg.struct.device
        self.end_place = self.info.n_prefixes + 1

    def _check(self, rc):
        if rc != 0:
            raise TagPipeError(rc, self._L.tp_last_error().decode("utf-8", "replace"))

    def close(self):
        if getattr(self, "_h", None):
            self._L.tp_grammar_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def start(self, rows):
        """States of `rows` empty lines: int32 [rows, 2], the place and the number of finished tags."""
        torch = _torch()
        return torch.zeros(rows, 2, dtype=torch.int32, device="cuda:%d" % self.device)

    def _states(self, states):
        torch = _torch()
        p = _tensor("states", states, self.device, torch.int32, (-1, 2))
        if states.shape[0] > 1 and states.stride(0) != 2:
            raise ValueError("states must be dense")
        return p

    def mask(self, states, out=None):
        """tp_grammar_mask: the allowed-token masks of rows of states, int32 [rows, (n_tokens + 31) // 32]."""
        torch = _torch()
        p, rows, words = self._states(states), states.shape[0], (self.info.n_tokens + 31) // 32
        if out is None:
            out = torch.empty(rows, words, dtype=torch.int32, device=states.device)
        to = _tensor("out", out, self.device, torch.int32, (rows, words))
        self._check(self._L.tp_grammar_mask(self._h, p, rows, to, _row_stride(out), _stream(torch, self.device)))
        return out

    def step(self, states, logits, *, temperature=None, uniform=None, append=False, **rules):
        """tp_grammar_step: (tokens int32 [rows], log-probabilities float32 [rows]); `states` move on in place, and with append=True the
        tokens go to the end of `history` and `history_len` rises.  -1: the row's line is at its end, or nothing is left to choose."""
        torch = _torch()
        p, rows = self._states(states), states.shape[0]
        io = _with_logits(self.device, logits, rules)
        if logits.shape[0] != rows:
            raise ValueError("one state per row of logits")
        t, u = _choice_inputs(self.device, rows, temperature, uniform)
        tokens = torch.empty(rows, dtype=torch.int32, device=states.device)
        logprob = torch.empty(rows, dtype=torch.float32, device=states.device)
        self._check(self._L.tp_grammar_step(self._h, C.byref(io), t, u, p, tokens.data_ptr(), logprob.data_ptr(), int(append)))
        return tokens, logprob

    def advance(self, states, tokens, *, history=None, history_len=None, append=False):
        """tp_grammar_step by the caller's own tokens (int32 [rows]): `states` move on in place; to place -1 where a token is not allowed."""
        torch = _torch()
        p, rows = self._states(states), states.shape[0]
        io = logit_rules(self.device, rows, self.info.n_tokens, history=history, history_len=history_len)
        given = _tensor("tokens", tokens, self.device, torch.int32, (rows,))
        self._check(self._L.tp_grammar_step(self._h, C.byref(io), None, None, p, given, None, int(append)))

    def lines(self, tokens, lengths=None, begin=None, arena=None):
        """tp_grammar_lines: (arena uint8, offsets int64 [rows + 1]) of rows of tokens int32 [rows, n], from begin to below lengths (int32
        [rows]).  A given arena bounds what is written: compare offsets[rows] with its size."""
        torch = _torch()
        p, (rows, n) = _tensor("tokens", tokens, self.device, torch.int32, (-1, -1)), tokens.shape
        le = None if lengths is None else _tensor("lengths", lengths, self.device, torch.int32, (rows,))
        be = None if begin is None else _tensor("begin", begin, self.device, torch.int32, (rows,))
        if arena is None:
            arena = torch.empty(rows * n * self.info.longest_token + 16, dtype=torch.uint8, device=tokens.device)
        to = _tensor("arena", arena, self.device, torch.uint8, (-1,))
        offsets = torch.zeros(1, dtype=torch.int64, device=tokens.device) if rows == 0 else torch.empty(rows + 1, dtype=torch.int64, device=tokens.device)
        need = self._L.tp_lines_workspace(rows)
        workspace = torch.empty(need, dtype=torch.uint8, device=tokens.device)
        self._check(self._L.tp_grammar_lines(self._h, p, _row_stride(tokens), n, be, le, rows, to, arena.shape[0], offsets.data_ptr(), workspace.data_ptr(), need,
                                             _stream(torch, self.device)))
        return arena, offsets


def run_tokens(pipe, grammar, tokens, lengths, begin):
    torch = _torch()
    if grammar.device != pipe._cfg.struct.device:
        raise ValueError("the grammar is on another device than the context")
    arena, offsets = grammar.lines(tokens, lengths, begin)
    rows, info, device = tokens.shape[0], pipe.info, tokens.device

    def zeros(n, dtype):
        return torch.zeros(max(n, 1), dtype=dtype, device=device)
    text_bytes = int(offsets[rows])
    capacity = 2 * text_bytes + 512 * rows + 64
    while True:
        captions, caption_offsets = torch.empty(capacity, dtype=torch.uint8, device=device), zeros(rows + 1, torch.int64)
        verdicts, histogram, counters = zeros(16 * rows, torch.uint8), zeros(info.n_strings + 1, torch.int64), zeros(8, torch.int64)
        fired, facets = zeros(rows * info.fired_words, torch.int32), zeros(rows * info.n_facets, torch.int16)
        io = tp_device_io()
        io.arena, io.offsets, io.n_files = arena.data_ptr(), offsets.data_ptr(), rows
        io.captions, io.caption_capacity, io.caption_offsets = captions.data_ptr(), capacity, caption_offsets.data_ptr()
        io.verdicts, io.histogram, io.counters = verdicts.data_ptr(), histogram.data_ptr(), counters.data_ptr()
        io.fired, io.facet_choice, io.stream = fired.data_ptr(), facets.data_ptr(), _stream(torch, device)
        try:
            total = pipe.run_lines_device(io)
            break
        except TagPipeError as e:
            if e.code != TP_E_CAPACITY:
                raise
            capacity = e.required

    def host(t, n, dtype):
        return t.cpu().numpy()[:n].view(dtype).copy()
    hist = host(histogram, info.n_strings + 1, np.uint64)
    counts = tp_counters.from_buffer_copy(host(counters, 8, np.uint64).tobytes())
    return BatchResult(host(captions[:total], total, np.uint8), host(caption_offsets, rows + 1, np.uint64), host(verdicts, 16 * rows, np.uint8).view(VERDICT_DTYPE),
                       counts.as_dict(), hist[:info.n_strings].copy(), int(hist[info.n_strings]), host(fired, rows * info.fired_words, np.uint32).reshape(rows, info.fired_words),
                       host(facets, rows * info.n_facets, np.uint16).reshape(rows, info.n_facets))
