"""Beam search on the GPU: the selection over a group's beams and the vocabulary, the
reordering of cached states, and one decode step that runs both.

It stands where ``sampler.GpuSampler`` has a sampled token (the reference's encodeSampling and
sampleFromTopK, src/engine/forward.ts:522-601, src/engine/sampler.ts:147-212): a request that is
searched keeps ``beams`` sequences and their cache rows (src/engine/kvcache.ts:14-104), a batch
holds ``groups`` of them, and row ``g * beams + b`` is beam ``b`` of group ``g``.

Every call is asynchronous on the given stream (default: torch's current one) and checks its
arguments before any GPU work.
"""
from __future__ import annotations

import ctypes
from typing import List, NamedTuple, Optional, Sequence

from .mx4 import call_on, dtype_code, on_device, rows_of
from .sampler import SamplingError, TABBY_EDOMAIN, TABBY_EEMPTY, _check, load_library

BEAMS_MAX = 64
COUNT_MAX = 128


class BeamChoice(NamedTuple):
    """The continuations kept, best first, [groups, count] each; -1, -1 and -inf where there are
    fewer."""

    tokens: "object"   # int32
    parents: "object"  # int32, the beam within the group
    scores: "object"   # float32


def _int32(t, shape, what, device):
    import torch
    if t.dtype != torch.int32 or not t.is_contiguous() or tuple(t.shape) != shape:
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape}")
    on_device(device, t)


def pack_mask(mask):
    """Truth values [rows, vocab] as the words ``BeamSelect`` takes: int32 [rows, ceil(vocab / 32)],
    entry t at bit t % 32 of word t // 32."""
    import torch
    rows, vocab = mask.shape
    padded = torch.nn.functional.pad(mask.bool(), (0, -vocab % 32)).view(rows, -1, 32)
    bits = torch.arange(32, device=mask.device, dtype=torch.int64)
    words = (padded.to(torch.int64) << bits).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


class BeamSelect:
    """The selection, with its workspace for up to ``groups_max`` groups of ``beams_max`` beams over
    ``vocab_max`` tokens, ``count_max`` continuations kept (tabby_beam_select_device). Calls that may
    overlap need an object each."""

    def __init__(self, vocab_max: int, groups_max: int = 1, beams_max: int = 4, count_max: int = 8, device="cuda"):
        import torch
        size = ctypes.c_int64()
        _check(load_library().tabby_beam_workspace(groups_max, beams_max, vocab_max, count_max, ctypes.byref(size)))
        self.vocab_max, self.groups_max = int(vocab_max), int(groups_max)
        self.beams_max, self.count_max = int(beams_max), int(count_max)
        self.workspace = torch.empty(size.value, dtype=torch.uint8, device=device)

    def __call__(self, logits, scores, count: int, allowed=None, done=None, pad_id: int = 0, status=None,
                 stream=None) -> BeamChoice:
        """``logits`` [groups * beams, vocab] (float32, float16, bfloat16); ``scores`` float32
        [groups, beams]; ``allowed`` the words of ``pack_mask``; ``done`` int32 [groups, beams], nonzero
        for an ended beam, whose one continuation is ``pad_id`` at its own score; ``status`` int32
        [groups] receives each group's tabby_status."""
        import torch
        x = rows_of(logits, "logits")
        code = dtype_code(x.dtype)
        device = x.device
        if scores.dtype != torch.float32 or scores.dim() != 2 or not scores.is_contiguous():
            raise ValueError("scores must be a contiguous float32 tensor [groups, beams]")
        groups, beams = int(scores.shape[0]), int(scores.shape[1])
        rows, vocab, count = int(x.shape[0]), int(x.shape[1]), int(count)
        if rows != groups * beams:
            raise ValueError(f"logits have {rows} rows, scores {groups} x {beams}")
        if groups > self.groups_max or beams > self.beams_max or vocab > self.vocab_max or count > self.count_max:
            raise ValueError(f"{groups} groups x {beams} beams x {vocab} tokens, {count} kept, exceed the object's "
                             f"{self.groups_max} x {self.beams_max} x {self.vocab_max}, {self.count_max}")
        on_device(device, scores, self.workspace)
        if allowed is not None:
            _int32(allowed, (rows, -(-vocab // 32)), "allowed", device)
        if done is not None:
            _int32(done, (groups, beams), "done", device)
        if status is not None:
            _int32(status, (groups,), "status", device)
        if count < 1:
            raise ValueError(f"count must be between 1 and {self.count_max}, got {count}")
        ctx, handle = call_on(device, stream)
        with ctx:
            found = torch.empty((3, groups, count), dtype=torch.int32, device=device)
            tokens, parents, kept = found[0], found[1], found[2].view(torch.float32)
            _check(load_library().tabby_beam_select_device(
                x.data_ptr(), code, x.stride(0), groups, beams, vocab, scores.data_ptr(),
                allowed.data_ptr() if allowed is not None else None, done.data_ptr() if done is not None else None,
                int(pad_id), count, tokens.data_ptr(), parents.data_ptr(), kept.data_ptr(),
                status.data_ptr() if status is not None else None, self.workspace.data_ptr(),
                self.workspace.numel(), handle))
        return BeamChoice(tokens, parents, kept)


def _geometry(states, rows: int, what: str):
    """(segments, capacity, unit bytes, row stride, segment stride) of states of one shape: [rows,
    positions], [rows, positions, width] or [rows, segments, positions, width]."""
    s = states[0]
    if not s.is_cuda:
        raise ValueError(f"{what} must be device (cuda) tensors")
    if s.dim() not in (2, 3, 4) or s.shape[0] != rows or s.numel() == 0:
        raise ValueError(f"{what} must be [rows, positions], [rows, positions, width] or [rows, segments, positions, "
                         f"width] with {rows} rows, got {tuple(s.shape)}")
    for o in states[1:]:
        if o.shape != s.shape or o.stride() != s.stride() or o.dtype != s.dtype:
            raise ValueError(f"{what} must all be of one shape, layout and type")
    on_device(s.device, *states[1:])
    size = s.element_size()
    position = 1 if s.dim() < 4 else 2
    capacity = int(s.shape[position])
    width = int(s.shape[position + 1]) if s.dim() > 2 else 1
    if (s.dim() > 2 and width > 1 and s.stride(-1) != 1) or (capacity > 1 and s.stride(position) != width):
        raise ValueError(f"{what}: a segment's positions must lie one after another")
    segments = int(s.shape[1]) if s.dim() == 4 else 1
    return segments, capacity, width * size, s.stride(0) * size, (s.stride(1) * size if s.dim() == 4 else 0)


def reorder_states(states: Sequence, parents, lengths=None, out: Optional[Sequence] = None, stream=None) -> List:
    """Row (g, b) of every state becomes row (g, parents[g, b]), in the first lengths[g] positions
    (all, without ``lengths``); a row whose parent is outside the group (-1) stays. ``states`` are
    tensors of one shape and layout, [groups * beams, positions], [rows, positions, width] or
    [rows, segments, positions, width]; they are moved in place, or into ``out``, whose rest
    stays. Returns the tensors written."""
    import torch
    states = list(states)
    out = states if out is None else list(out)
    if not states or len(out) != len(states):
        raise ValueError("states must not be empty, and out must hold as many")
    if parents.dim() != 2:
        raise ValueError("parents must be [groups, beams]")
    groups, beams = int(parents.shape[0]), int(parents.shape[1])
    shape = _geometry(states, groups * beams, "states")
    if out is not states and (_geometry(out, groups * beams, "out") != shape or out[0].dtype != states[0].dtype):
        raise ValueError("out must be laid out like states")
    device = states[0].device
    on_device(device, out[0])
    _int32(parents, (groups, beams), "parents", device)
    if lengths is not None:
        _int32(lengths, (groups,), "lengths", device)
    n = len(states)
    pointers = ctypes.c_void_p * n
    src = pointers(*[s.data_ptr() for s in states])
    dst = src if out is states else pointers(*[s.data_ptr() for s in out])
    ctx, handle = call_on(device, stream)
    with ctx:
        _check(load_library().tabby_beam_reorder_device(
            src, dst, n, groups, beams, *shape, parents.data_ptr(),
            lengths.data_ptr() if lengths is not None else None, handle))
    return out


class BeamSearch:
    """The decode loop's state of ``groups`` searches of ``beams`` beams: scores, ended beams, the
    tokens so far, and the cached states that ``step`` keeps in line with them. An ended beam stays
    among its group's, at its score, until ``beams`` better ones push it out."""

    def __init__(self, groups: int, beams: int, vocab: int, max_tokens: int, end_ids: Sequence[int] = (),
                 pad_id: int = 0, device="cuda"):
        import torch
        self.groups, self.beams, self.max_tokens, self.pad_id = groups, beams, max_tokens, pad_id
        self.select = BeamSelect(vocab_max=vocab, groups_max=groups, beams_max=beams, count_max=beams, device=device)
        # One live beam per group to begin with: the beams' rows are alike until the first step.
        self.scores = torch.full((groups, beams), float("-inf"), device=device)
        self.scores[:, 0] = 0.0
        self.done = torch.zeros((groups, beams), dtype=torch.int32, device=device)
        self.tokens = torch.full((groups * beams, max_tokens), pad_id, dtype=torch.int32, device=device)
        self.status = torch.zeros(groups, dtype=torch.int32, device=device)
        self.end_ids = torch.tensor(list(end_ids), dtype=torch.int32, device=device)
        self.length = 0

    def step(self, logits, states: Sequence = (), lengths=None, allowed=None):
        """One step from the beams' logits: chooses, moves ``states`` and the tokens to the surviving
        beams and appends the new tokens; returns them, int32 [groups * beams]."""
        import torch
        if self.length >= self.max_tokens:
            raise ValueError(f"the search holds {self.max_tokens} tokens")
        choice = self.select(logits, self.scores, self.beams, allowed=allowed, done=self.done, pad_id=self.pad_id,
                             status=self.status)
        if states:
            reorder_states(states, choice.parents, lengths=lengths)
        reorder_states([self.tokens], choice.parents)
        reorder_states([self.done.view(-1, 1)], choice.parents)
        new = torch.where(choice.tokens < 0, self.pad_id, choice.tokens)
        self.tokens[:, self.length] = new.view(-1)
        if self.end_ids.numel():
            self.done |= torch.isin(new, self.end_ids).to(torch.int32)
        self.scores = choice.scores.contiguous()
        self.length += 1
        return new.view(-1)

    def finished(self) -> bool:
        """Whether every beam that has a score has ended (reads back)."""
        return bool(((self.done != 0) | (self.scores == float("-inf"))).all())

    def best(self):
        """Each group's best sequence and its score: a list of (token ids, score) (reads back)."""
        status = self.status.tolist()
        for g, code in enumerate(status):
            if code in (TABBY_EEMPTY, TABBY_EDOMAIN):
                raise SamplingError(code, f"group {g}: " + ("no continuation" if code == TABBY_EEMPTY else
                                                            "a logit or score is NaN or +inf"))
        tokens = self.tokens.view(self.groups, self.beams, -1)[:, 0, :self.length].tolist()
        ends = set(self.end_ids.tolist())
        out = []
        for ids, score in zip(tokens, self.scores[:, 0].tolist()):
            stop = next((i + 1 for i, t in enumerate(ids) if t in ends), len(ids))
            out.append((ids[:stop], score))
        return out
