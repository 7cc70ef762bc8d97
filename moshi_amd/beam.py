"""Beam search on the device: the choice over beams and vocabulary (`beam_select`) and the beams' states moved to where their children are
(`beam_reorder`); libmoshi_tlm.so, include/moshi_tlm.h.

    r = beam_select(logits, scores, lengths=lengths, finished=finished, eos=2, length_penalty=0.6)
    beam_reorder([state, history], r.parents)                 # row b * beams + i: what row b * beams + r.parents[b, i] was
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Dict, Optional, Sequence

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


_on: Dict[torch.device, _capi.LaunchOn] = {}
_need: Dict[tuple, int] = {}             # bytes that a selection of (requests, beams, vocabulary) works in
_I32, _F32, _BOOL = torch.int32, torch.float32, torch.bool


def _place(device: torch.device, lib: Optional[_capi.Lib]):
    if lib is None:
        if device.type != "cuda":
            raise RuntimeError("moshi_amd.beam runs on an MI355X (device='cuda'); there is no CPU path")
        lib = _capi.load_tlm()
    on = _on.get(device)
    if on is None:
        on = _on[device] = _capi.LaunchOn(device)
    return lib, on


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
    device, shape = logits.device, scores.shape
    lib, on = _place(device, lib)
    if len(shape) != 2 or logits.dim() != 2 or logits.shape[0] != shape[0] * shape[1]:
        raise AssertionError("logits are [requests * beams, vocab], scores [requests, beams]")
    (batch, beams), vocab, dtype, (row, step) = shape, logits.shape[1], _DTYPES.get(logits.dtype), logits.stride()
    if dtype is None or (step != 1 and vocab > 1):
        raise ValueError("logits are bf16 or fp32, a row's side by side")
    where = logits.get_device()
    for name, t, kind in (("scores", scores, _F32), ("lengths", lengths, _I32), ("finished", finished, _BOOL)):
        if t is not None and (t.dtype is not kind or t.shape != shape or t.get_device() != where or not t.is_contiguous()):
            raise ValueError(f"{name} is a contiguous {kind} tensor [requests, beams] on the logits' device")
    if length_penalty and lengths is None:
        raise ValueError("a length penalty needs lengths")
    need = _need.get((batch, beams, vocab))
    if need is None:
        need = lib.mmi_beam_select_workspace(batch, beams, vocab)
        lib.check(min(0, need))
        if len(_need) > 4096:
            _need.clear()
        _need[batch, beams, vocab] = need
    parents, tokens, grown = torch.empty((3, batch, beams), dtype=_I32, device=device).unbind()
    r = BeamChoice(torch.empty(shape, dtype=_F32, device=device), parents, tokens, torch.empty(shape, dtype=_BOOL, device=device) if eos >= 0 else None,
                   None if lengths is None else grown)
    work = torch.empty(need, dtype=torch.uint8, device=device)
    lib.check(on.call(lib.mmi_beam_select, batch, beams, vocab, dtype, logits.data_ptr(), row, scores.data_ptr(), None if lengths is None else lengths.data_ptr(),
                      None if finished is None else finished.data_ptr(), eos, length_penalty, r.scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                      None if eos < 0 else r.finished.data_ptr(), None if lengths is None else grown.data_ptr(), work.data_ptr(), need))
    return r


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, lib: Optional[_capi.Lib] = None) -> None:
    """In place, for every tensor [requests * beams, ...] of any type: row b * beams + i becomes a copy of what row b * beams + parents[b, i] was.
    parents: int32 [requests, beams]; one outside the request leaves its row alone.  A row's elements lie together; no two tensors share memory."""
    lib, on = _place(parents.device, lib)
    if parents.dim() != 2 or parents.dtype is not _I32 or not parents.is_contiguous():
        raise ValueError("parents is a contiguous int32 tensor [requests, beams]")
    (batch, beams), where = parents.shape, parents.get_device()
    total, at, stride, size = batch * beams, [], [], []
    for t in states:
        if t.dim() < 1 or t.shape[0] != total:
            raise AssertionError("states are [requests * beams, ...]")
        if t.get_device() != where:
            raise ValueError("a state's rows are contiguous, on the parents' device")
        nbytes = t.nbytes
        if not nbytes:
            continue
        at.append(t.data_ptr())
        size.append(nbytes // total)
        if t.is_contiguous():
            stride.append(nbytes // total)
        else:
            if not t[:1].is_contiguous():
                raise ValueError("a state's rows are contiguous, on the parents' device")
            stride.append(t.stride(0) * t.element_size())
    n = len(at)
    lib.check(on.call(lib.mmi_beam_reorder, n, (C.c_void_p * n)(*at), (C.c_int64 * n)(*stride), (C.c_int64 * n)(*size), batch, beams, parents.data_ptr()))
