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

from ._abi import TP_E_CAPACITY, VERDICT_DTYPE, tp_counters, tp_device_io, tp_grammar_config, tp_grammar_info
from .tagpipe import BatchResult, TagPipeError, load_library

_native_module = None
_torch_module = None


def _native():
    """The module that checks the tensors, makes the outputs and calls the library (csrc/tp_torch.cpp)."""
    global _native_module, _torch_module
    if _native_module is None:
        import torch
        L = load_library()
        try:
            from . import _tp_torch
        except ImportError as e:
            raise TagPipeError(-3, "the torch module is not built or does not fit this torch (run `python -m imagecaptioner_amd.build`): %s" % e) from e

        here = "torch module for %s %s" % (torch.__version__, torch.version.git_version)
        if _tp_torch.built_for != here:
            raise TagPipeError(-3, "this is a %s, and the module is a %s (run `python -m imagecaptioner_amd.build`)" % (here, _tp_torch.built_for))

        def failed(rc):
            raise TagPipeError(rc, L.tp_last_error().decode("utf-8", "replace"))
        _tp_torch.bind(*(C.cast(f, C.c_void_p).value for f in (L.tp_shape_logits, L.tp_choose_workspace, L.tp_choose_tokens, L.tp_grammar_mask, L.tp_grammar_step,
                                                              L.tp_lines_workspace, L.tp_grammar_lines)), failed)
        _native_module, _torch_module = _tp_torch, torch
    return _native_module


def _torch():
    _native()
    return _torch_module


def _stream(device):
    raw = getattr(_torch_module._C, "_cuda_getCurrentRawStream", None)         # the same number without a Stream object around it
    return raw(device) if raw is not None else _torch_module.cuda.current_stream(device).cuda_stream


def shape_logits(pipe, logits, out, rules):
    native, device = _native(), pipe._device
    return native.shape(pipe._h, device, _stream(device), logits, out, rules)


def choose_tokens(pipe, logits, temperature, uniform, rules):
    native, device = _native(), pipe._device
    return native.choose(pipe._h, device, _stream(device), logits, temperature, uniform, rules)


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
        self._n_tokens, self._longest, self._words = self.info.n_tokens, self.info.longest_token, (self.info.n_tokens + 31) // 32

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

    def mask(self, states, out=None):
        """tp_grammar_mask: the allowed-token masks of rows of states, int32 [rows, (n_tokens + 31) // 32]."""
        native = _native()
        return native.mask(self._h, self.device, _stream(self.device), states, self._words, out)

    def step(self, states, logits, *, temperature=None, uniform=None, append=False, **rules):
        """tp_grammar_step: (tokens int32 [rows], log-probabilities float32 [rows]); `states` move on in place, and with append=True the
        tokens go to the end of `history` and `history_len` rises.  -1: the row's line is at its end, or nothing is left to choose.  `rules` are
        those of TagPipe.shape_logits, without a mask."""
        native = _native()
        return native.step(self._h, self.device, _stream(self.device), states, logits, temperature, uniform, append, rules)

    def advance(self, states, tokens, *, history=None, history_len=None, append=False):
        """tp_grammar_step by the caller's own tokens (int32 [rows]): `states` move on in place; to place -1 where a token is not allowed."""
        native = _native()
        native.advance(self._h, self.device, _stream(self.device), states, self._n_tokens, tokens, append, {"history": history, "history_len": history_len})

    def _capturing(self):
        with _torch_module.cuda.device(self.device):
            return _torch_module.cuda.is_current_stream_capturing()

    def lines(self, tokens, lengths=None, begin=None, arena=None):
        """tp_grammar_lines: (arena uint8, offsets int64 [rows + 1]) of rows of tokens int32 [rows, n], from begin to below lengths (int32
        [rows]).  A given arena bounds what is written: compare offsets[rows] with its size.  Without one it is made for rows of nothing but the
        longest token, up to MOST_ARENA bytes; beyond those the texts' sizes are found first, for which the call waits (a captured call cannot, and
        makes the large one)."""
        native = _native()
        if arena is None and isinstance(tokens, _torch_module.Tensor) and tokens.numel() * self._longest > MOST_ARENA and not self._capturing():
            _, offsets = self.lines(tokens, lengths, begin, arena=tokens.new_empty((0,), dtype=_torch_module.uint8))
            arena = tokens.new_empty((int(offsets[-1]) + 16,), dtype=_torch_module.uint8)
        return native.lines(self._h, self.device, _stream(self.device), tokens, lengths, begin, arena, self._longest)


# Most bytes of an arena that is made for the largest texts there could be: a token list may hold a token of a hundred spaces, or of a megabyte.  Finding the
# sizes first does the work twice.
MOST_ARENA = 1 << 30


def run_tokens(pipe, grammar, tokens, lengths, begin):
    torch = _torch()
    if grammar.device != pipe._device:
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
        io.fired, io.facet_choice, io.stream = fired.data_ptr(), facets.data_ptr(), _stream(pipe._device)
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
