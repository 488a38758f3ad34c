#!/usr/bin/env python3
"""How often a sampled token of tp_choose_tokens lies on the other side of a border between two tokens than a program's that takes the formula in
other precisions, on rows of 131072 logits:

  rounded     z = x / T rounded to 32 bits, as the formula of tagpipe.h says, weights and sums in 64 bits
  unrounded   z = x / T in 64 bits as well

and how far that border is from the random number, as a share of the row's weight.  python3 tools/choice_borders.py [calls of 512 rows]"""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from imagecaptioner_amd import Config, TagPipe

ROWS, VOCAB = 512, 131072


def chosen(z, uniform):
    """(tokens, cumulative shares) by 64-bit weights of the z given."""
    w = (z.double() - z.double().amax(1, keepdim=True)).exp_()
    cum = w.cumsum(1)
    cum /= cum[:, -1:].clone()
    return (cum > uniform.double()[:, None]).int().argmax(1).int(), cum


def main():
    calls = int(sys.argv[1]) if len(sys.argv) > 1 else 40
    pipe = TagPipe(Config(vocabulary=b"solo"))
    pairs = {"call against rounded": 0, "call against unrounded": 0, "rounded against unrounded": 0}
    farthest = 0.0
    for k in range(calls):
        gen = torch.Generator(device="cuda").manual_seed(k)
        logits = torch.randn(ROWS, VOCAB, generator=gen, device="cuda").mul_(3.0)
        logits += 6.0 * (torch.rand(ROWS, VOCAB, generator=gen, device="cuda") > 0.999)
        logits = logits.bfloat16()
        temperature = torch.rand(ROWS, generator=gen, device="cuda") * 0.7 + 0.5
        uniform = torch.rand(ROWS, generator=gen, device="cuda")
        call = pipe.choose_tokens(logits, temperature=temperature, uniform=uniform)[0]
        unrounded, cum = chosen(logits.double() / temperature.double()[:, None], uniform)
        del cum
        rounded, cum = chosen(logits.float() / temperature[:, None], uniform)
        pairs["call against unrounded"] += int((call != unrounded).sum())
        pairs["rounded against unrounded"] += int((rounded != unrounded).sum())
        other = (call != rounded).nonzero()[:, 0].tolist()
        pairs["call against rounded"] += len(other)
        for r in other:
            a, b = sorted((int(call[r]), int(rounded[r])))
            farthest = max(farthest, abs(float(cum[r, a]) - float(uniform[r])), abs(float(cum[r, b - 1]) - float(uniform[r])))
    for name, n in pairs.items():
        print("%-26s %3d of %d rows another token (%.1e)" % (name, n, calls * ROWS, n / (calls * ROWS)))
    print("call against rounded: the border is at most %.1e of the row's weight from the random number" % farthest)


if __name__ == "__main__":
    main()
