#!/usr/bin/env python3
"""Speculative decoding with two small models whose lm_heads are FP8, on one MI355X.

The next token's distribution of either model depends on the last token alone: its embedding is the hidden
state. A step lets the draft model propose ``drafts`` tokens a request, one after another, then computes the
target's logits after each of them in one product (``LmHeadFp8``, hidden states quantised in the call), and
``DraftVerify`` accepts as many as the target's distribution allows and draws the token after them. The draft
model's own draws are the same call with nothing drafted. Weights are random: the example shows the calls, not a
language.

Usage: python examples/speculative_fp8.py [--requests R] [--drafts N] [--steps S] [--vocab V] [--hidden H]
"""
from __future__ import annotations

import argparse
import os
import sys
import time
from typing import NamedTuple

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np
import torch

from tabby_amd import draft, fp8, sampler


class Model:
    """An embedding table and an lm_head of random weights, the latter held in FP8; ``near`` makes a model whose
    head is another's with noise added."""

    def __init__(self, vocab: int, hidden: int, seed: int = 0, near: "Model" = None, noise: float = 0.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.vocab, self.hidden = vocab, hidden
        if near is None:
            self.embed = torch.randn(vocab, hidden, device="cuda", generator=g).to(torch.bfloat16)
            self.weight = torch.randn(vocab, hidden, device="cuda", generator=g) * (3.0 / hidden ** 0.5)
        else:
            self.embed = near.embed
            self.weight = near.weight + noise / hidden ** 0.5 * torch.randn(vocab, hidden, device="cuda", generator=g)
        self.head = fp8.LmHeadFp8(fp8.Fp8Matrix.quantize(self.weight, block_rows=fp8.BLOCK))

    def logits(self, tokens):
        """Logits [n, vocab] of what follows each of ``tokens`` (int32 [n])."""
        return self.head.logits(self.embed[tokens.long()])


class Step(NamedTuple):
    """A step's inputs and what came of them."""

    logits: "object"        # [requests * (drafts + 1), vocab]
    draft_logits: "object"  # [requests * drafts, vocab]
    drafts: "object"        # int32 [requests * drafts]
    uniforms: "object"      # float64 [requests * drafts]
    lasts: "object"         # float64 [requests]
    verified: draft.Verified


class Speculation:
    """The two models, the requests' settings, and the workspaces."""

    def __init__(self, target: Model, proposer: Model, settings, drafts: int, seed: int = 0):
        self.target, self.proposer, self.settings, self.drafts = target, proposer, list(settings), drafts
        requests = len(self.settings)
        self.verify = draft.DraftVerify(target.vocab, requests, drafts)
        self.draw = draft.DraftVerify(target.vocab, requests, 0)
        self.random = np.random.default_rng(seed)
        self.none_int = torch.empty(0, dtype=torch.int32, device="cuda")
        self.none_float = torch.empty(0, dtype=torch.float64, device="cuda")
        whole = any(s.temperature > 0 and (s.topK == 0 or s.topK > draft.POOL_MAX) for s in self.settings)
        self.flags = sampler.TABBY_FLAG_FULL_VOCAB if whole else 0

    def _params(self, uniforms):
        packed = sampler.make_params(self.settings, len(self.settings), uniforms)
        return torch.from_numpy(packed.view(np.uint8).copy()).cuda()

    def step(self, tokens) -> Step:
        """One step after each request's last token (int32 [requests])."""
        requests, last = len(self.settings), tokens
        proposed, rows = [], []
        for _ in range(self.drafts):
            logits = self.proposer.logits(last)
            last = self.draw(logits, self.none_int, self._params(self.random.random(requests)), self.none_float,
                             flags=self.flags).tokens.view(-1)
            proposed.append(last)
            rows.append(logits)
        drafts = torch.stack(proposed, 1)  # [requests, drafts]
        logits = self.target.logits(torch.cat([tokens.view(-1, 1), drafts], 1).view(-1))
        draft_logits = torch.stack(rows, 1).view(requests * self.drafts, -1)
        uniforms = torch.from_numpy(self.random.random(requests * self.drafts)).cuda()
        lasts = self.random.random(requests)
        drafts = drafts.reshape(-1)
        verified = self.verify(logits, drafts, self._params(lasts), uniforms, draft_logits=draft_logits, flags=self.flags)
        return Step(logits, draft_logits, drafts, uniforms, torch.from_numpy(lasts), verified)

    def generate(self, tokens, count: int):
        """At least ``count`` tokens after each of ``tokens``: a list to each request, and the steps that it took."""
        made = [[] for _ in self.settings]
        steps = 0
        while min(len(m) for m in made) < count:
            verified = self.step(tokens).verified
            steps += 1
            ids, accepted = verified.tokens.tolist(), verified.accepted.tolist()
            for m, row, n in zip(made, ids, accepted):
                m += row[:n + 1]
            tokens = torch.tensor([m[-1] for m in made], dtype=torch.int32, device="cuda")
        return made, steps


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--steps", type=int, default=32, help="tokens a request")
    ap.add_argument("--vocab", type=int, default=151936)
    ap.add_argument("--hidden", type=int, default=896)
    args = ap.parse_args(argv)
    target = Model(args.vocab, args.hidden)
    proposer = Model(args.vocab, args.hidden, seed=1, near=target, noise=0.5)
    run = Speculation(target, proposer, [sampler.SamplingParams(0.7, 40, 0.9)] * args.requests, args.drafts)
    prompt = torch.arange(args.requests, dtype=torch.int32, device="cuda") % args.vocab
    run.generate(prompt, 2)
    torch.cuda.synchronize()
    start = time.perf_counter()
    made, steps = run.generate(prompt, args.steps)
    took = time.perf_counter() - start
    for r, ids in enumerate(made):
        print(f"request {r}: {ids[:args.steps]}")
    print(f"{took / steps * 1e6:.0f} us a step of {args.drafts} drafted tokens, {sum(map(len, made)) / steps / args.requests:.2f} "
          f"tokens a request and step")
    return made


if __name__ == "__main__":
    main()
