"""Beam search on the device: the choice over beams and vocabulary (`beam_select`) and the beams' states moved to where their children are
(`beam_reorder`); libmoshi_tlm.so, include/moshi_tlm.h.

    r = beam_select(logits, scores, lengths=lengths, finished=finished, eos=2, length_penalty=0.6)
    beam_reorder([state, history], r.parents)                 # row b * beams + i: what row b * beams + r.parents[b, i] was
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _capi

_DTYPES = {torch.bfloat16: _capi.MMI_BF16, torch.float32: _capi.MMI_F32}


@dataclass
class BeamChoice:
    """The new beams, best first; every field is [requests, beams]."""
    scores: torch.Tensor                 # fp32: sums of log probabilities
    parents: torch.Tensor                # int32: beam that it continues
    tokens: torch.Tensor                 # int32: token that it appends
    finished: Optional[torch.Tensor]     # bool: it ends with `eos` (None without an end token)
    lengths: Optional[torch.Tensor]      # int32: tokens that it has (None without lengths)


def _library(device: torch.device, lib: Optional[_capi.Lib]) -> _capi.Lib:
    if lib is None:
        if device.type != "cuda":
            raise RuntimeError("moshi_amd.beam runs on an MI355X (device='cuda'); there is no CPU path")
        lib = _capi.load_tlm()
    return lib


def beam_select(logits: torch.Tensor, scores: torch.Tensor, lengths: Optional[torch.Tensor] = None, finished: Optional[torch.Tensor] = None, eos: int = -1,
                length_penalty: float = 0.0, lib: Optional[_capi.Lib] = None) -> BeamChoice:
    """Of every request's candidates (beam, token) the best `beams`.

    Args:
        logits: [requests * beams, vocab], bf16 or fp32.  scores: fp32 [requests, beams], sums of log probabilities so far; -inf: no such beam
            (all but one at a request's start).
        lengths: int32 [requests, beams], tokens so far; needed for a length penalty.
        finished: bool [requests, beams]; a finished beam has one candidate, `eos` at the score and length it has.
        length_penalty: candidates are ranked by score / length ** length_penalty.
    Equal ranks go to the lower beam, then the lower token.  At most 32 beams.
    """
    device = logits.device
    lib = _library(device, lib)
    if scores.dim() != 2 or logits.dim() != 2 or logits.shape[0] != scores.numel():
        raise AssertionError("logits are [requests * beams, vocab], scores [requests, beams]")
    if logits.dtype not in _DTYPES or (logits.stride(1) != 1 and logits.numel()):
        raise ValueError("logits are bf16 or fp32, a row's side by side")
    want = [("scores", scores, torch.float32), ("lengths", lengths, torch.int32), ("finished", finished, torch.bool)]
    for name, t, dtype in want:
        if t is not None and (t.shape != scores.shape or t.dtype != dtype or not t.is_contiguous() or t.device != device):
            raise ValueError(f"{name} is a contiguous {dtype} tensor [requests, beams] on the logits' device")
    if length_penalty and lengths is None:
        raise ValueError("a length penalty needs lengths")
    batch, beams = scores.shape
    vocab = logits.shape[1]
    new = lambda dtype: torch.empty((batch, beams), dtype=dtype, device=device)  # noqa: E731
    r = BeamChoice(new(torch.float32), new(torch.int32), new(torch.int32), new(torch.bool) if eos >= 0 else None, None if lengths is None else new(torch.int32))
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    with _capi.device_scope(device):
        need = lib.mmi_beam_select_workspace(batch, beams, vocab)
        lib.check(min(0, need))
        work = torch.empty(need, dtype=torch.uint8, device=device)
        lib.check(lib.mmi_beam_select(batch, beams, vocab, _DTYPES[logits.dtype], ptr(logits), logits.stride(0), ptr(scores), ptr(lengths), ptr(finished), int(eos),
                                      float(length_penalty), ptr(r.scores), ptr(r.parents), ptr(r.tokens), ptr(r.finished), ptr(r.lengths), ptr(work), need,
                                      _capi.stream_ptr(device)))
    return r


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, lib: Optional[_capi.Lib] = None) -> None:
    """In place, for every tensor [requests * beams, ...] of any type: row b * beams + i becomes a copy of what row b * beams + parents[b, i] was.
    parents: int32 [requests, beams]; one outside the request leaves its row alone.  A row's elements lie together; no two tensors share memory."""
    device = parents.device
    lib = _library(device, lib)
    if parents.dim() != 2 or parents.dtype != torch.int32 or not parents.is_contiguous():
        raise ValueError("parents is a contiguous int32 tensor [requests, beams]")
    batch, beams = parents.shape
    n = len(states)
    at, stride, size = (C.c_void_p * max(1, n))(), (C.c_int64 * max(1, n))(), (C.c_int64 * max(1, n))()
    k = 0
    for t in states:
        if t.dim() < 1 or t.shape[0] != batch * beams:
            raise AssertionError("states are [requests * beams, ...]")
        if t.device != device or not (t.is_contiguous() or t[:1].is_contiguous()):
            raise ValueError("a state's rows are contiguous, on the parents' device")
        if t.numel():
            item = t.element_size()
            at[k], size[k] = t.data_ptr(), t.numel() // t.shape[0] * item
            stride[k] = t.stride(0) * item if t.shape[0] > 1 else size[k]
            k += 1
    with _capi.device_scope(device):
        lib.check(lib.mmi_beam_reorder(k, at, stride, size, batch, beams, parents.data_ptr(), _capi.stream_ptr(device)))
