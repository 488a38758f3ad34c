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
import struct

import numpy as np

from ._abi import TP_E_CAPACITY, VERDICT_DTYPE, tp_counters, tp_device_io, tp_grammar_config, tp_grammar_info
from .tagpipe import BatchResult, TagPipeError, load_library

# A decoding loop makes these calls once per token, and the host's part of a small call takes longer than the GPU's: arguments are
# checked with as few tensor queries as will do, and tp_logits is packed in one go (the layout of _abi.tp_logits).
_LOGITS = struct.Struct("@IiQIIPQPQPPPPPPQPPQPIIP")
_torch_module = None
_TYPES = None


def _torch():
    global _torch_module, _TYPES
    if _torch_module is None:
        import torch
        _TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        _torch_module = torch
    return _torch_module


def _stream(torch, device):
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)                 # the same number without a Stream object around it
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


def _refuse(name, t, device, dtype, shape):
    if t.requires_grad and _torch_module.is_grad_enabled():
        raise ValueError("%s requires a gradient, which this call does not have: detach it" % name)
    raise ValueError("%s must be a %s tensor of the shape %s on cuda:%d, dense along its last axis, got %s %s with strides %s on %s" % (
        name, dtype, shape, device, t.dtype, tuple(t.shape), t.stride(), t.device))


def _vec(name, t, device, dtype, rows):
    """A dense vector's data pointer."""
    if t.dtype is not dtype or t.get_device() != device or t.shape != (rows,) or not t.is_contiguous() or (t.requires_grad and _torch_module.is_grad_enabled()):
        _refuse(name, t, device, dtype, "(%d,)" % rows)
    return t.data_ptr()


def _table(name, t, device, dtype, rows, columns):
    """A table's data pointer, rows, columns and elements between rows (its columns where there is one row at most); rows or columns -1: any."""
    if t.dtype is not dtype or t.get_device() != device or t.dim() != 2 or (t.requires_grad and _torch_module.is_grad_enabled()):
        _refuse(name, t, device, dtype, "(%d, %d)" % (rows, columns))
    r, c = t.shape
    stride, dense = t.stride()
    if (rows != -1 and r != rows) or (columns != -1 and c != columns) or (c > 1 and dense != 1):
        _refuse(name, t, device, dtype, "(%d, %d)" % (rows, columns))
    return t.data_ptr(), r, c, stride if r > 1 else c


def logit_rules(device, type_, rows, vocab, logits, stride, *, history=None, history_len=None, prompt_len=None, repetition=None, frequency=None, presence=None,
                bias=None, bias_row=None, mask=None, mask_row=None):
    """A packed tp_logits.

    history int32 [rows, n] with history_len int32 [rows] (every row is full without it); entries before prompt_len int32 [rows] count as
    repeated but not for frequency and presence.  repetition, frequency, presence: float32 [rows].
    bias float32 [n, vocab] (or [vocab]) with bias_row int32 [rows]: which one a row takes, -1 none; row 0 for all without it.
    mask int32 [n, (vocab + 31) // 32] (or one row) with mask_row likewise: token t is allowed when bit t % 32 of word t // 32 is set."""
    torch = _torch()
    i32, f32 = torch.int32, torch.float32
    h = h_cap = h_stride = h_len = prompt = b = b_stride = b_row = n_bias = m = m_stride = m_row = n_masks = 0
    if history is not None:
        h, _, h_cap, h_stride = _table("history", history, device, i32, rows, -1)
        if history_len is not None:
            h_len = _vec("history_len", history_len, device, i32, rows)
        if prompt_len is not None:
            prompt = _vec("prompt_len", prompt_len, device, i32, rows)
        if not h:                                            # no rows, or rows of no room: there is no history, whatever the lengths say
            h_len = prompt = 0
    elif history_len is not None or prompt_len is not None:
        raise ValueError("history_len or prompt_len without a history")
    if bias is not None:
        b, n_bias, _, b_stride = _table("bias", bias if bias.dim() == 2 else bias[None], device, f32, -1, vocab)
        if bias_row is not None:
            b_row = _vec("bias_row", bias_row, device, i32, rows)
        if not n_bias:
            raise ValueError("bias has no rows")
    elif bias_row is not None:
        raise ValueError("bias_row without a bias")
    if mask is not None:
        m, n_masks, _, m_stride = _table("mask", mask if mask.dim() == 2 else mask[None], device, i32, -1, (vocab + 31) // 32)
        if mask_row is not None:
            m_row = _vec("mask_row", mask_row, device, i32, rows)
        if not n_masks:
            raise ValueError("mask has no rows")
    elif mask_row is not None:
        raise ValueError("mask_row without a mask")
    return _LOGITS.pack(_LOGITS.size, type_, rows, vocab, h_cap, logits, stride, h, h_stride, h_len, prompt,
                        0 if repetition is None else _vec("repetition", repetition, device, f32, rows),
                        0 if frequency is None else _vec("frequency", frequency, device, f32, rows),
                        0 if presence is None else _vec("presence", presence, device, f32, rows),
                        b, b_stride, b_row, m, m_stride, m_row, n_bias, n_masks, _stream(torch, device))


def _with_logits(device, logits, rules):
    """(packed tp_logits, rows, vocab)"""
    _torch()
    dtype = logits.dtype
    if dtype not in _TYPES:
        raise ValueError("logits must be a float32, float16 or bfloat16 tensor [rows, vocab], got %s" % dtype)
    p, rows, vocab, stride = _table("logits", logits, device, dtype, -1, -1)
    return logit_rules(device, _TYPES[dtype], rows, vocab, p, stride, **rules), rows, vocab


def _choice_inputs(device, rows, temperature, uniform):
    torch = _torch()
    t = None if temperature is None else _vec("temperature", temperature, device, torch.float32, rows)
    u = None if uniform is None else _vec("uniform", uniform, device, torch.float32, rows)
    if t and not u:
        raise ValueError("a temperature needs `uniform`, the random numbers of the choice")
    return t, u


def shape_logits(pipe, logits, out, rules):
    device = pipe._device
    io, rows, vocab = _with_logits(device, logits, rules)
    if out is None:
        out = logits.new_empty((rows, vocab))
        to, stride = out.data_ptr(), vocab
    else:
        to, _, _, stride = _table("out", out, device, logits.dtype, rows, vocab)
        _torch().autograd.graph.increment_version(out)           # a backward pass that has kept what `out` held finds it changed
    pipe._check(pipe._L.tp_shape_logits(pipe._h, io, to, stride))
    return out


def choose_tokens(pipe, logits, temperature, uniform, rules):
    torch = _torch()
    device = pipe._device
    io, rows, vocab = _with_logits(device, logits, rules)
    t, u = _choice_inputs(device, rows, temperature, uniform)
    need = pipe._L.tp_choose_workspace(rows, vocab)
    workspace = logits.new_empty((need,), dtype=torch.uint8) if need else None   # torch's own pool keeps it apart per stream and per graph
    tokens = logits.new_empty((rows,), dtype=torch.int32)
    logprob = logits.new_empty((rows,), dtype=torch.float32)
    pipe._check(pipe._L.tp_choose_tokens(pipe._h, io, t, u, tokens.data_ptr(), logprob.data_ptr(), workspace.data_ptr() if need else None, need))
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
        self.device = pipe._device
        self.end_place = self.info.n_prefixes + 1
        self._words = (self.info.n_tokens + 31) // 32

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
        p, rows, _, stride = _table("states", states, self.device, _torch().int32, -1, 2)
        if stride != 2:
            raise ValueError("states must be dense")
        return p, rows

    def mask(self, states, out=None):
        """tp_grammar_mask: the allowed-token masks of rows of states, int32 [rows, (n_tokens + 31) // 32]."""
        p, rows = self._states(states)
        words = self._words
        if out is None:
            out = states.new_empty((rows, words))
            to, stride = out.data_ptr(), words
        else:
            to, _, _, stride = _table("out", out, self.device, states.dtype, rows, words)
        self._check(self._L.tp_grammar_mask(self._h, p, rows, to, stride, _stream(_torch(), self.device)))
        return out

    def step(self, states, logits, *, temperature=None, uniform=None, append=False, **rules):
        """tp_grammar_step: (tokens int32 [rows], log-probabilities float32 [rows]); `states` move on in place, and with append=True the
        tokens go to the end of `history` and `history_len` rises.  -1: the row's line is at its end, or nothing is left to choose."""
        p, rows = self._states(states)
        io, of_logits, _ = _with_logits(self.device, logits, rules)
        if of_logits != rows:
            raise ValueError("one state per row of logits")
        t, u = _choice_inputs(self.device, rows, temperature, uniform)
        tokens = states.new_empty((rows,))
        logprob = states.new_empty((rows,), dtype=_torch().float32)
        self._check(self._L.tp_grammar_step(self._h, io, t, u, p, tokens.data_ptr(), logprob.data_ptr(), bool(append)))
        return tokens, logprob

    def advance(self, states, tokens, *, history=None, history_len=None, append=False):
        """tp_grammar_step by the caller's own tokens (int32 [rows]): `states` move on in place; to place -1 where a token is not allowed."""
        p, rows = self._states(states)
        io = logit_rules(self.device, 0, rows, self.info.n_tokens, 0, 0, history=history, history_len=history_len)
        self._check(self._L.tp_grammar_step(self._h, io, None, None, p, _vec("tokens", tokens, self.device, states.dtype, rows), None, bool(append)))

    def lines(self, tokens, lengths=None, begin=None, arena=None):
        """tp_grammar_lines: (arena uint8, offsets int64 [rows + 1]) of rows of tokens int32 [rows, n], from begin to below lengths (int32
        [rows]).  A given arena bounds what is written: compare offsets[rows] with its size."""
        torch = _torch()
        i32 = torch.int32
        p, rows, n, stride = _table("tokens", tokens, self.device, i32, -1, -1)
        le = None if lengths is None else _vec("lengths", lengths, self.device, i32, rows)
        be = None if begin is None else _vec("begin", begin, self.device, i32, rows)
        if arena is None:
            arena = tokens.new_empty((rows * n * self.info.longest_token + 16,), dtype=torch.uint8)
        to = _vec("arena", arena, self.device, torch.uint8, arena.numel())
        offsets = tokens.new_empty((rows + 1,), dtype=torch.int64) if rows else tokens.new_zeros((1,), dtype=torch.int64)
        need = self._L.tp_lines_workspace(rows)
        workspace = tokens.new_empty((need,), dtype=torch.uint8)
        self._check(self._L.tp_grammar_lines(self._h, p, stride, n, be, le, rows, to, arena.numel(), offsets.data_ptr(), workspace.data_ptr(), need,
                                             _stream(torch, self.device)))
        return arena, offsets


# An arena for rows of nothing but the longest token is made up to this many bytes; beyond it (a token list may hold a token of a hundred
# spaces) the texts' sizes are found first, at the price of doing the work twice.
MOST_ARENA = 1 << 30


def run_tokens(pipe, grammar, tokens, lengths, begin):
    torch = _torch()
    if grammar.device != pipe._device:
        raise ValueError("the grammar is on another device than the context")
    arena = None
    if tokens.numel() * grammar.info.longest_token > MOST_ARENA:
        _, offsets = grammar.lines(tokens, lengths, begin, arena=tokens.new_empty((0,), dtype=torch.uint8))
        arena = tokens.new_empty((int(offsets[-1]) + 16,), dtype=torch.uint8)
    arena, offsets = grammar.lines(tokens, lengths, begin, arena)
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
        io.fired, io.facet_choice, io.stream = fired.data_ptr(), facets.data_ptr(), _stream(torch, pipe._device)
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
