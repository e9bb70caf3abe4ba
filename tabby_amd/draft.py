"""Speculative decoding's verification on the GPU: how many of a request's drafted tokens the target's
distribution accepts, and the token that follows them.

It stands where ``sampler.GpuSampler`` has a sampled token (the reference's encodeSampling and
sampleFromTopK, src/engine/forward.ts:522-601, src/engine/sampler.ts:147-212): a smaller model, or a
lookup in the prompt, proposes a request's next tokens, the target computes the logits of all of
them at once, and what comes out is distributed as if the target had drawn every token by itself,
under the sampler's own settings.

Calls are asynchronous on the given stream (default: torch's current one) and check their arguments
before any GPU work; ``DraftVerify.verify`` reads back.
"""
from __future__ import annotations

import ctypes
from typing import List, NamedTuple, Sequence, Union

import numpy as np
import torch

from .beam import _int32, _used_here
from .mx4 import INT32_MAX, call_on, dtype_code, on_device, rows_of
from .sampler import (PARAMS_DTYPE, SamplingError, SamplingParams, SeededRandom, TABBY_FLAG_FULL_VOCAB, TABBY_OK, _check,
                      load_library, make_params)

POOL_MAX = 128     # larger pools need TABBY_FLAG_FULL_VOCAB, as the whole vocabulary does
DRAFTS_MAX = 63


class Verified(NamedTuple):
    """What a request's drafted tokens came to."""

    tokens: "object"    # int32 [requests, drafts + 1]: the accepted ones, one more, then -1
    accepted: "object"  # int32 [requests]


class VerifyOutcome(NamedTuple):
    """A request's new tokens: those of its drafted ones that were accepted, and one more."""

    tokens: List[int]
    accepted: int


class DraftVerify:
    """The verification, with its workspace for up to ``requests_max`` requests of ``drafts_max`` drafted
    tokens over ``vocab_max`` tokens (tabby_draft_verify_device). Calls that may overlap need an object
    each."""

    def __init__(self, vocab_max: int, requests_max: int = 1, drafts_max: int = 4, device="cuda"):
        if max(vocab_max, requests_max, drafts_max) > INT32_MAX:
            raise ValueError("vocab_max, requests_max and drafts_max must fit 32 bits")
        size = ctypes.c_int64()
        _check(load_library().tabby_draft_workspace(requests_max, drafts_max, vocab_max, ctypes.byref(size)))
        self.vocab_max, self.requests_max, self.drafts_max = int(vocab_max), int(requests_max), int(drafts_max)
        self.workspace_bytes = size.value
        self.workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
        self._streams = set()

    def __call__(self, logits, drafts, params, uniforms, draft_logits=None, offsets=None, status=None, flags: int = 0,
                 stream=None) -> Verified:
        """``logits`` [rows, vocab] (float32, float16, bfloat16): request r's rows, one more than it has
        drafted tokens, are offsets[r] to offsets[r + 1] - 1 (``offsets`` int32 [requests + 1]; without it
        every request has as many). ``drafts`` int32 and ``uniforms`` float64 [rows - requests], one request
        after another, as the rows of ``draft_logits`` that the tokens were drawn from, of the logits' type;
        without those the tokens were certain. ``params`` a uint8 tensor of PARAMS_DTYPE entries, one to a
        request: the settings that both sides are sampled with, and the uniform of the last draw. ``flags``
        TABBY_FLAG_FULL_VOCAB where a request that is not greedy has top_k 0 or above ``POOL_MAX``. ``status``
        int32 [requests] receives each request's tabby_status; a request that fails has no tokens."""
        x = rows_of(logits, "logits")
        code = dtype_code(x.dtype)
        device = x.device
        rows, vocab = x.shape
        size = PARAMS_DTYPE.itemsize
        if params.dtype != torch.uint8 or not params.is_contiguous() or params.numel() % size or not params.numel():
            raise ValueError(f"params must be a contiguous uint8 tensor of {size} bytes to a request")
        requests = params.numel() // size
        on_device(device, params, uniforms, self.workspace)
        total = rows - requests
        if offsets is None:
            if rows % requests:
                raise ValueError(f"logits have {rows} rows, which {requests} requests do not share evenly")
            most, offsets_at = rows // requests - 1, None
        else:
            most, offsets_at = self.drafts_max, _int32(offsets, (requests + 1,), "offsets", device)
        if requests > self.requests_max or most > self.drafts_max or vocab > self.vocab_max:
            raise ValueError(f"{requests} requests x {most} drafted tokens x {vocab} tokens exceed the object's "
                             f"{self.requests_max} x {self.drafts_max} x {self.vocab_max}")
        if not 0 <= total <= requests * most:
            raise ValueError(f"logits have {rows} rows, {requests} requests of up to {most} drafted tokens "
                             f"{requests} to {requests * (most + 1)}")
        drafts_at = _int32(drafts.view(-1) if drafts.is_contiguous() else drafts, (total,), "drafts", device)
        if uniforms.dtype != torch.float64 or not uniforms.is_contiguous() or uniforms.numel() != total:
            raise ValueError(f"uniforms must be a contiguous float64 tensor of {total} entries")
        draft_at, draft_stride = None, 0
        if draft_logits is not None and total:
            y = rows_of(draft_logits, "draft_logits")
            on_device(device, y)
            if y.dtype != x.dtype or tuple(y.shape) != (total, vocab):
                raise ValueError(f"draft_logits must be {x.dtype} [{total}, {vocab}], got {y.dtype} {tuple(y.shape)}")
            draft_at, draft_stride = y.data_ptr(), y.stride(0)
        status_at = None if status is None else _int32(status, (requests,), "status", device)
        ctx, handle = call_on(device, stream)
        with ctx:
            _used_here(self._streams, device, handle, self.workspace)
            tokens = torch.empty_strided((requests, most + 1), (most + 1, 1), dtype=torch.int32, device=device)
            accepted = torch.empty_strided((requests,), (1,), dtype=torch.int32, device=device)
            _check(load_library().tabby_draft_verify_device(
                x.data_ptr(), code, x.stride(0), rows, draft_at, draft_stride, drafts_at, uniforms.data_ptr(), offsets_at,
                requests, most, vocab, params.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), status_at,
                self.workspace.data_ptr(), self.workspace_bytes, flags, handle))
        return Verified(tokens, accepted)

    def verify(self, logits, drafts: Sequence[Sequence[int]], params: Union[SamplingParams, Sequence[SamplingParams]],
               rng: Union[SeededRandom, Sequence[SeededRandom]], draft_logits=None, stream=None) -> List[VerifyOutcome]:
        """The same from host values (reads back): each request's drafted tokens as a list, its settings and its
        random numbers. A SeededRandom is advanced, in the order of the requests, once per drafted token
        and once more for a request with temperature > 0, not at all for a greedy one; a list holds one to
        a request."""
        requests = len(drafts)
        if not requests:
            raise ValueError("drafts must hold a list of tokens to each request")
        lengths = [len(d) for d in drafts]
        if max(lengths) > self.drafts_max:
            raise ValueError(f"{max(lengths)} drafted tokens exceed the object's {self.drafts_max}")
        settings = [params] * requests if isinstance(params, SamplingParams) else list(params)
        generators = [rng] * requests if isinstance(rng, SeededRandom) else list(rng)
        if len(generators) != requests:
            raise ValueError(f"expected {requests} random number generators, got {len(generators)}")
        packed = make_params(settings, requests, None)  # refuses bad temperatures before any number is drawn
        uniforms = []
        for r, (setting, generator) in enumerate(zip(settings, generators)):
            drawn = setting.temperature > 0
            uniforms += [generator.next() if drawn else 0.0 for _ in range(lengths[r])]
            packed[r]["uniform"] = generator.next() if drawn else 0.0
        vocab = int(logits.shape[-1])
        whole = any(p.temperature > 0 and (p.topK == 0 or p.topK > POOL_MAX) for p in settings) and vocab > POOL_MAX
        device = logits.device
        ctx, _ = call_on(device, stream)
        with ctx:
            status = torch.empty(requests, dtype=torch.int32, device=device)
            got = self(logits, torch.tensor([t for d in drafts for t in d], dtype=torch.int32, device=device),
                       torch.from_numpy(packed.view(np.uint8).copy()).to(device),
                       torch.tensor(uniforms, dtype=torch.float64, device=device), draft_logits=draft_logits,
                       offsets=torch.tensor(np.cumsum([0] + [n + 1 for n in lengths]), dtype=torch.int32, device=device),
                       status=status, flags=TABBY_FLAG_FULL_VOCAB if whole else 0)
            tokens, accepted, codes = got.tokens.tolist(), got.accepted.tolist(), status.tolist()
        for r, code in enumerate(codes):
            if code != TABBY_OK:
                raise SamplingError(code, f"request {r}: its settings, a drafted token or a row of logits cannot be used")
        return [VerifyOutcome(t[:n + 1], n) for t, n in zip(tokens, accepted)]
