#!/usr/bin/env python3
"""Beam search over a small recurrent model whose lm_head is MXFP4, on one MI355X.

Each beam keeps a cache of the hidden states of its tokens; a step's hidden state is the last
token's embedding plus the mean of its cache. The step's logits come from ``LmHeadMx4`` (hidden
states quantised in the call), ``BeamSearch.step`` chooses the continuations and moves every beam's
cache to the beams that survived. Weights are random: the example shows the calls, not a language.

Usage: python examples/beam_search_mx4.py [--groups G] [--beams B] [--steps N] [--vocab V] [--hidden H]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from tabby_amd import beam, mx4


class Model:
    """An embedding table and an lm_head of random weights, the latter held in MXFP4."""

    def __init__(self, vocab: int, hidden: int, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.vocab, self.hidden = vocab, hidden
        self.embed = torch.randn(vocab, hidden, device="cuda", generator=g)
        weight = torch.randn(vocab, hidden, device="cuda", generator=g) * (3.0 / hidden ** 0.5)
        self.head = mx4.LmHeadMx4(mx4.Mx4Matrix.quantize(weight))

    def hidden_states(self, tokens, cache, length: int):
        """The step's hidden states [rows, hidden] of each row's last token, kept in ``cache``
        [rows, capacity, hidden] at position ``length``."""
        h = self.embed[tokens.long()]
        if length:
            h = h + cache[:, :length].float().mean(1)
        cache[:, length] = h.to(cache.dtype)
        return h


def search(model: Model, prompt, beams: int, steps: int, end_ids=()):
    """The best ``steps`` tokens after each group's last prompt token (int32 [groups]):
    [(token ids, score)], and the ``BeamSearch``."""
    groups = int(prompt.shape[0])
    run = beam.BeamSearch(groups, beams, model.vocab, steps, end_ids=end_ids)
    cache = torch.zeros(groups * beams, steps, model.hidden, dtype=torch.bfloat16, device="cuda")
    tokens = prompt.repeat_interleave(beams)
    for length in range(steps):
        logits = model.head.logits(model.hidden_states(tokens, cache, length))
        lengths = torch.full((groups,), length + 1, dtype=torch.int32, device="cuda")
        tokens = run.step(logits, states=[cache], lengths=lengths)
    return run.best(), run


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--groups", type=int, default=4)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--vocab", type=int, default=151936)
    ap.add_argument("--hidden", type=int, default=896)
    args = ap.parse_args(argv)
    model = Model(args.vocab, args.hidden)
    prompt = torch.arange(args.groups, dtype=torch.int32, device="cuda") % args.vocab
    search(model, prompt, args.beams, 2)
    torch.cuda.synchronize()
    start = time.perf_counter()
    best, _ = search(model, prompt, args.beams, args.steps)
    took = time.perf_counter() - start
    for g, (ids, score) in enumerate(best):
        print(f"group {g}: {score:9.4f}  {ids}")
    print(f"{took / args.steps * 1e6:.0f} us a step: {args.groups} searches of {args.beams} beams over "
          f"{args.vocab} tokens")
    return best


if __name__ == "__main__":
    main()
