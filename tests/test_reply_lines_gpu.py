"""The text of written tokens where its bound is far from its size and as the first work of a process, and replies under tables with aliases, on the GPU."""
import os
import random
import subprocess
import sys

import numpy as np
import pytest

from helpers import ROOT, Config, Oracle, assert_same_results
from reply_plain import TAGS, PlainGrammar, token_list
from test_reply_tags_cpu import ALIASES, WORDS, lexicon

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pipe():
    from imagecaptioner_amd import TagPipe
    return TagPipe(Config(vocabulary="\n".join(TAGS).encode()))


def test_one_long_token_does_not_make_a_large_arena(pipe):
    """A token of a megabyte in the list: 300 x 400 tokens are bounded by 126 GB and hold 120 KB."""
    tokens = [bytes([b]) for b in range(256)] + [b"x" * (1 << 20), b""]
    g = pipe.tag_grammar(tokens, len(tokens) - 1)
    rows = np.random.default_rng(4).integers(97, 123, (300, 400)).astype(np.int32)
    t = torch.as_tensor(rows, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    arena, offsets = g.lines(t)
    assert torch.cuda.max_memory_allocated() - before < 8 << 20
    want = rows.astype(np.uint8).tobytes()
    assert offsets.tolist() == list(range(0, 300 * 400 + 1, 400)) and bytes(arena.cpu().numpy()) == want + b"\0" * 16
    t[7, 3] = 256                                                          # and a text that does hold it
    arena, offsets = g.lines(t, torch.full((300,), 390, device="cuda", dtype=torch.int32))
    want = [bytes(r[:390].astype(np.uint8)) for r in rows]
    want[7] = want[7][:3] + tokens[256] + want[7][4:]
    assert offsets.tolist() == np.cumsum([0] + [len(x) for x in want]).tolist() and bytes(arena.cpu().numpy()) == b"".join(want) + b"\0" * 16


def test_a_captured_call_makes_the_large_arena(pipe, monkeypatch):
    from imagecaptioner_amd import replies
    monkeypatch.setattr(replies, "MOST_ARENA", 100)
    tokens = [bytes([b]) for b in range(256)] + [b""]
    g, plain = pipe.tag_grammar(tokens, 256), PlainGrammar(TAGS, tokens, 256)
    t = torch.full((70, 9), 98, device="cuda", dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g.lines(t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        arena, offsets = g.lines(t)
    for letter in (99, 100, 101):
        t.fill_(letter)
        graph.replay()
        torch.cuda.synchronize()
        eager, eager_offsets = g.lines(t)
        assert torch.equal(offsets, eager_offsets) and arena.numel() == 70 * 9 + 16
        assert bytes(arena[:640].cpu().numpy()) == bytes(eager[:640].cpu().numpy()) == bytes([letter]) * 630 + b"\0" * 10
        assert plain.text(t[0].tolist()) * 70 == bytes(arena[:630].cpu().numpy())


FIRST = """
import numpy as np, torch
from imagecaptioner_amd import Config, TagPipe
pipe = TagPipe(Config(vocabulary=b"solo\\nsmile\\nhat"))
tokens = [bytes([b]) for b in range(256)] + [b""]
g = pipe.tag_grammar(tokens, 256)
rows = 70001                                          # so many are placed by the scan of the caption offsets
t = torch.as_tensor(np.random.default_rng(5).integers(97, 123, (rows, 2)).astype(np.int32), device="cuda")
states, logits = torch.zeros(5, 2, device="cuda", dtype=torch.int32), torch.randn(5, 257, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):                         # nothing of the reply calls has run before
    arena, offsets = g.lines(t)
    mask = g.mask(states)
    shaped = pipe.shape_logits(logits, mask=mask, mask_row=torch.arange(5, device="cuda", dtype=torch.int32))
    token, logprob = g.step(states, logits)
for _ in range(3):
    states.zero_()
    t.copy_(t.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert bytes(arena[:2 * rows].cpu().numpy()) == t.cpu().numpy().astype(np.uint8).tobytes()
    assert np.array_equal(offsets.cpu().numpy(), np.arange(rows + 1) * 2)
    assert torch.equal(token, shaped.argmax(1).int()) and (shaped > -1e30).sum(1).tolist() == [2] * 5    # 's' and 'h' begin a line
print("captured first calls replay")
"""


def test_the_first_call_of_a_process_may_be_captured():
    done = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "captured first calls replay" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("spaces", [False, True])
def test_replies_under_aliases_are_taken(spaces):
    """Tables with aliases to kept, unknown and dropped tags, and tags that spell a phrase with blanks: no finished reply is refused and none of its tags is lost."""
    from imagecaptioner_amd import TagPipe
    cfg = Config(vocabulary="\n".join(WORDS).encode(), lexicon=lexicon(ALIASES), trigger="solo")
    pipe, oracle, rng = TagPipe(cfg), Oracle(cfg), random.Random(8)
    tokens = token_list(rng, WORDS, 500, spaces)
    g = pipe.tag_grammar(tokens, len(tokens) - 1, spaces=spaces, max_tags=9)
    rows, steps, vocab = 300, 120, len(tokens)
    gen = torch.Generator(device="cuda").manual_seed(9)
    history, length = torch.zeros(rows, steps, device="cuda", dtype=torch.int32), torch.zeros(rows, device="cuda", dtype=torch.int32)
    states, bias = g.start(rows), torch.zeros(vocab, device="cuda")
    bias[vocab - 1] = 3.0                                                  # an end that comes
    for _ in range(steps):
        g.step(states, torch.randn(rows, vocab, generator=gen, device="cuda").mul_(2.0), temperature=torch.ones(rows, device="cuda"),
               uniform=torch.rand(rows, generator=gen, device="cuda"), append=True, history=history, history_len=length, bias=bias)
    ended = (states[:, 0] == g.end_place).cpu().numpy()
    assert ended.mean() > 0.9
    texts = [b"".join(tokens[t] for t in row[:n] if t != vocab - 1).decode() for row, n in zip(history.cpu().numpy(), length.cpu().numpy())]
    got, want = pipe.run_tokens(g, history, length), oracle.run_texts(texts)
    assert_same_results(got, want, pipe.histogram_dict(got.histogram), "replies under aliases")
    assert not (got.verdicts["flags"][ended] & 0x10).any() and not got.verdicts["n_dropped"][ended].any()
    for r in np.nonzero(ended)[0]:
        kept = {oracle.normalize_tag(t) for t in texts[r].split(", ")}
        assert len(texts[r].split(", ")) >= 3 and got.verdicts["n_candidates"][r] == len(kept) and got.verdicts["n_selected"][r] == len(kept | {"solo", "1girl"}), texts[r]
