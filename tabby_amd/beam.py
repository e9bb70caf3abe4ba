"""Beam search on the GPU: the selection over a group's beams and the vocabulary, the
reordering of cached states, and one decode step that runs both.

It stands where ``sampler.GpuSampler`` has a sampled token (the reference's encodeSampling and
sampleFromTopK, src/engine/forward.ts:522-601, src/engine/sampler.ts:147-212): a request that is
searched keeps ``beams`` sequences and their cache rows (src/engine/kvcache.ts:14-104), a batch
holds ``groups`` of them, and row ``g * beams + b`` is beam ``b`` of group ``g``.

Every call is asynchronous on the given stream (default: torch's current one) and checks its
arguments before any GPU work; what reads back (``BeamSearch.finished``, ``best``) does so on the
current one.
"""
from __future__ import annotations

import ctypes
from typing import List, NamedTuple, Optional, Sequence

import torch

from .mx4 import INT32_MAX, call_on, dtype_code, on_device, rows_of
from .sampler import SamplingError, TABBY_EDOMAIN, TABBY_EEMPTY, _check, load_library

BEAMS_MAX = 64
COUNT_MAX = 128


def _used_here(seen, device, handle, *tensors):
    """Tells the allocator that an object's own tensors are used on the current stream (`handle`; once for each in
    `seen`): the object may be dropped while the stream still works with them."""
    if handle not in seen:
        seen.add(handle)
        for t in tensors:
            t.record_stream(torch.cuda.current_stream(device))


class BeamChoice(NamedTuple):
    """The continuations kept, best first, [groups, count] each; -1, -1 and -inf where there are
    fewer."""

    tokens: "object"   # int32
    parents: "object"  # int32, the beam within the group
    scores: "object"   # float32


def _int32(t, shape, what, device):
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape}")
    on_device(device, t)
    return t.data_ptr()


def pack_mask(mask):
    """Truth values [rows, vocab] as the words ``BeamSelect`` takes: int32 [rows, ceil(vocab / 32)],
    entry t at bit t % 32 of word t // 32."""
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
        if max(groups_max, beams_max, vocab_max, count_max) > INT32_MAX:
            raise ValueError("groups_max, beams_max, vocab_max and count_max must fit 32 bits")
        size = ctypes.c_int64()
        _check(load_library().tabby_beam_workspace(groups_max, beams_max, vocab_max, count_max, ctypes.byref(size)))
        self.vocab_max, self.groups_max = int(vocab_max), int(groups_max)
        self.beams_max, self.count_max = int(beams_max), int(count_max)
        self.workspace_bytes = size.value
        self.workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
        self._streams = set()

    def __call__(self, logits, scores, count: int, allowed=None, done=None, pad_id: int = 0, status=None,
                 stream=None) -> BeamChoice:
        """``logits`` [groups * beams, vocab] (float32, float16, bfloat16); ``scores`` float32
        [groups, beams]; ``allowed`` the words of ``pack_mask``; ``done`` int32 [groups, beams], nonzero
        for an ended beam, whose one continuation is ``pad_id`` at its own score; ``status`` int32
        [groups] receives each group's tabby_status."""
        x = rows_of(logits, "logits")
        code = dtype_code(x.dtype)
        device = x.device
        if scores.dtype != torch.float32 or scores.dim() != 2 or not scores.is_contiguous():
            raise ValueError("scores must be a contiguous float32 tensor [groups, beams]")
        groups, beams = scores.shape
        rows, vocab = x.shape
        count = int(count)
        if rows != groups * beams:
            raise ValueError(f"logits have {rows} rows, scores {groups} x {beams}")
        if groups > self.groups_max or beams > self.beams_max or vocab > self.vocab_max or count > self.count_max:
            raise ValueError(f"{groups} groups x {beams} beams x {vocab} tokens, {count} kept, exceed the object's "
                             f"{self.groups_max} x {self.beams_max} x {self.vocab_max}, {self.count_max}")
        if count < 1:
            raise ValueError(f"count must be between 1 and {self.count_max}, got {count}")
        if pad_id > INT32_MAX:
            raise ValueError(f"pad_id must fit 32 bits, got {pad_id}")
        on_device(device, scores, self.workspace)
        allowed_at = None if allowed is None else _int32(allowed, (rows, -(-vocab // 32)), "allowed", device)
        done_at = None if done is None else _int32(done, (groups, beams), "done", device)
        status_at = None if status is None else _int32(status, (groups,), "status", device)
        ctx, handle = call_on(device, stream)
        with ctx:
            _used_here(self._streams, device, handle, self.workspace)
            tokens, parents, kept = torch.empty_strided(
                (3, groups, count), (groups * count, count, 1), dtype=torch.int32, device=device).unbind()
            at, size = tokens.data_ptr(), 4 * groups * count
            _check(load_library().tabby_beam_select_device(
                x.data_ptr(), code, x.stride(0), groups, beams, vocab, scores.data_ptr(), allowed_at, done_at,
                int(pad_id), count, at, at + size, at + 2 * size, status_at, self.workspace.data_ptr(),
                self.workspace_bytes, handle))
        return BeamChoice(tokens, parents, kept.view(torch.float32))


def _geometry(states, rows: int, what: str):
    """(segments, capacity, unit bytes, row stride, segment stride) of states of one shape, [rows,
    positions], [rows, positions, width] or [rows, segments, positions, width], and their addresses."""
    s = states[0]
    dtype, shape, strides, dims = s.dtype, s.shape, s.stride(), s.dim()
    if not s.is_cuda:
        raise ValueError(f"{what} must be device (cuda) tensors")
    if dims not in (2, 3, 4) or shape[0] != rows or s.numel() == 0:
        raise ValueError(f"{what} must be [rows, positions], [rows, positions, width] or [rows, segments, positions, "
                         f"width] with {rows} rows, got {tuple(shape)}")
    index = s.get_device()
    for o in states:
        if o.shape != shape or o.stride() != strides or o.dtype is not dtype:
            raise ValueError(f"{what} must all be of one shape, layout and type")
        if o.get_device() != index:
            raise ValueError(f"tensors lie on {s.device} and on {o.device}")
    addresses = [o.data_ptr() for o in states]
    size = s.element_size()
    position = 1 if dims < 4 else 2
    capacity = shape[position]
    width = shape[position + 1] if dims > 2 else 1
    if (dims > 2 and width > 1 and strides[-1] != 1) or (capacity > 1 and strides[position] != width):
        raise ValueError(f"{what}: a segment's positions must lie one after another")
    segments = shape[1] if dims == 4 else 1
    if segments > INT32_MAX or rows > INT32_MAX:
        raise ValueError(f"{what}'s rows and segments must fit 32 bits, got {tuple(shape)}")
    return (segments, capacity, width * size, strides[0] * size, strides[1] * size if dims == 4 else 0), addresses


def reorder_states(states: Sequence, parents, lengths=None, out: Optional[Sequence] = None, stream=None) -> List:
    """Row (g, b) of every state becomes row (g, parents[g, b]), in the first lengths[g] positions
    (all, without ``lengths``); a row whose parent is outside the group (-1) stays. ``states`` are
    tensors of one shape and layout, [groups * beams, positions], [rows, positions, width] or
    [rows, segments, positions, width]; they are moved in place, or into ``out``, whose rest
    stays. What is written must not overlap another of the tensors: a cache that layers share is
    listed once. Returns the tensors written."""
    states = list(states)
    out = states if out is None else list(out)
    n = len(states)
    if not n or len(out) != n:
        raise ValueError("states must not be empty, and out must hold as many")
    if parents.dim() != 2:
        raise ValueError("parents must be [groups, beams]")
    groups, beams = parents.shape
    shape, addresses = _geometry(states, groups * beams, "states")
    pointers = ctypes.c_void_p * n
    src = dst = pointers(*addresses)
    device = states[0].device
    if out is not states:
        out_shape, addresses = _geometry(out, groups * beams, "out")
        if out_shape != shape or out[0].dtype != states[0].dtype:
            raise ValueError("out must be laid out like states")
        on_device(device, out[0])
        dst = pointers(*addresses)
    parents_at = _int32(parents, (groups, beams), "parents", device)
    lengths_at = None if lengths is None else _int32(lengths, (groups,), "lengths", device)
    ctx, handle = call_on(device, stream)
    with ctx:
        _check(load_library().tabby_beam_reorder_device(src, dst, n, groups, beams, *shape, parents_at, lengths_at, handle))
    return out


class BeamSearch:
    """The decode loop's state of ``groups`` searches of ``beams`` beams: scores, ended beams, the
    tokens so far, and the cached states that ``step`` keeps in line with them. An ended beam stays
    among its group's, at its score, until ``beams`` better ones push it out."""

    def __init__(self, groups: int, beams: int, vocab: int, max_tokens: int, end_ids: Sequence[int] = (),
                 pad_id: int = 0, device="cuda"):
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
        self._streams = set()

    def step(self, logits, states: Sequence = (), lengths=None, allowed=None, stream=None):
        """One step from the beams' logits: chooses, moves ``states`` and the tokens to the surviving
        beams and appends the new tokens; returns them, int32 [groups * beams]. A step is not captured
        into a graph, where it would stay the same step: ``BeamSelect`` and ``reorder_states`` are. The
        caller orders a stream's steps after those of another, and after the object's making."""
        if self.length >= self.max_tokens:
            raise ValueError(f"the search holds {self.max_tokens} tokens")
        device = self.scores.device
        ctx, handle = call_on(device, stream)
        with ctx:
            if torch.cuda.is_current_stream_capturing():
                raise ValueError("a step of a search cannot be captured: the next one has other scores and another place")
            # Scores and status are replaced below, and may be an earlier stream's.
            here = torch.cuda.current_stream(device)
            self.scores.record_stream(here)
            self.status.record_stream(here)
            _used_here(self._streams, device, handle, self.tokens, self.done, self.end_ids)
            status = torch.empty_like(self.status)
            choice = self.select(logits, self.scores, self.beams, allowed=allowed, done=self.done, pad_id=self.pad_id,
                                 status=status)
            self.status = torch.where(self.status == 0, status, self.status)  # a group's first failure
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

    def best(self, strict: bool = True):
        """Each group's best sequence and its score: a list of (token ids, score) (reads back). A group that
        failed raises its SamplingError, or is None in the list where not ``strict``."""
        status = self.status.tolist()
        failed = {g: code for g, code in enumerate(status) if code in (TABBY_EEMPTY, TABBY_EDOMAIN)}
        if strict:
            for g, code in failed.items():
                raise SamplingError(code, f"group {g}: " + ("no continuation" if code == TABBY_EEMPTY else
                                                            "a logit or score is NaN or +inf"))
        tokens = self.tokens.view(self.groups, self.beams, -1)[:, 0, :self.length].tolist()
        ends = set(self.end_ids.tolist())
        out = []
        for g, (ids, score) in enumerate(zip(tokens, self.scores[:, 0].tolist())):
            stop = next((i + 1 for i, t in enumerate(ids) if t in ends), len(ids))
            out.append(None if g in failed else (ids[:stop], score))
        return out
