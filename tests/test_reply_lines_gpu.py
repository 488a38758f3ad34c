"""The text of written tokens where its bound is far from its size, and as the first work of a process, on the GPU."""
import os
import subprocess
import sys

import numpy as np
import pytest

from helpers import ROOT, Config
from reply_plain import TAGS, PlainGrammar

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
