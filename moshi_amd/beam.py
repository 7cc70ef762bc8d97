"""Beam search on the device: the choice over beams and vocabulary (`beam_select`) and the beams' states moved to where their children are
(`beam_reorder`); libmoshi_tlm.so, include/moshi_tlm.h.  `beam_search` runs them over a `TokenLM`.

    r = beam_select(logits, scores, lengths=lengths, finished=finished, eos=2, length_penalty=0.6)
    beam_reorder([state, history], r.parents)                 # row b * beams + i: what row b * beams + r.parents[b, i] was

    best = beam_search(lm, prompts, beams=4, max_new_tokens=64, eos=2)[0][0].tokens
"""
from __future__ import annotations

from array import array
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _capi
from .tlm import TokenLM

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
        eos: token that ends a beam; negative: none does.
        length_penalty: candidates are ranked by score / length ** length_penalty; between -16 and 16.
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
    if eos >= vocab > 0:
        raise ValueError("the end token is outside the vocabulary")
    eos = max(eos, -1)
    need = _need.get((batch, beams, vocab))
    if need is None:
        need = lib.mmi_beam_select_workspace(batch, beams, vocab)
        lib.check(min(0, need))
        if len(_need) > 4096:
            _need.clear()
        _need[batch, beams, vocab] = need
    like = torch.empty_like                                # (a third of what `empty` with its arguments takes)
    parents, tokens = like(scores, dtype=_I32), like(scores, dtype=_I32)
    r = BeamChoice(like(scores), parents, tokens, like(scores, dtype=_BOOL) if eos >= 0 else None, None if lengths is None else like(lengths))
    work = scores.new_empty(need, dtype=torch.uint8)
    lib.check(on.call(lib.mmi_beam_select, batch, beams, vocab, dtype, logits.data_ptr(), row, scores.data_ptr(), None if lengths is None else lengths.data_ptr(),
                      None if finished is None else finished.data_ptr(), eos, length_penalty, r.scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                      None if eos < 0 else r.finished.data_ptr(), None if lengths is None else r.lengths.data_ptr(), work.data_ptr(), need))
    return r


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, lib: Optional[_capi.Lib] = None) -> None:
    """In place, for every tensor [requests * beams, ...] of any type: row b * beams + i becomes a copy of what row b * beams + parents[b, i] was.
    parents: int32 [requests, beams]; one outside the request leaves its row alone.  A row's elements lie together; no two tensors share memory,
    with the parents among them (views of one buffer's rows, as far apart from row to row, may lie between one another)."""
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
    lists = [array("q", x) for x in (at, stride, size)]
    lib.check(on.call(lib.mmi_beam_reorder, len(at), *[x.buffer_info()[0] for x in lists], batch, beams, parents.data_ptr()))


@dataclass
class BeamHypothesis:
    tokens: List[int]                    # what follows the prompt, an end token included
    score: float                         # sum of their log probabilities


def beam_pages(lm_pages, prompt: int, beams: int, max_new_tokens: int, page: int) -> int:
    """Cache pages that one request's search may come to hold; lm_pages(n): pages of a sequence of n tokens.  The beams share the prompt's full pages."""
    total = lm_pages(prompt + max_new_tokens - 1)
    shared = min(total, prompt // page)
    return shared + beams * (total - shared)


@torch.no_grad()
def beam_search(lm: TokenLM, prompts: Sequence[Sequence[int]], beams: int = 4, max_new_tokens: int = 64, eos: int = -1, length_penalty: float = 0.0,
                step_tokens: int = 2048) -> List[List[BeamHypothesis]]:
    """For every prompt the `beams` continuations that the search ends with, best first (by score / length ** length_penalty).  A search ends when
    all its beams have ended with `eos` (-1: no end token), or after max_new_tokens.

    As many prompts run together as the model's slots (`beams` each), its pages and `step_tokens` allow.  BufferError when not even one does.
    """
    prompts = [[int(t) for t in p] for p in prompts]
    if beams < 1 or max_new_tokens < 1 or any(not p for p in prompts):
        raise ValueError("a search needs a beam, a prompt and at least one new token")
    if not abs(length_penalty) <= 16:
        raise ValueError("a length penalty is between -16 and 16")
    if not -1 <= eos < lm.vocab:
        raise ValueError("the end token is outside the vocabulary")
    if any(t < 0 or t >= lm.vocab for p in prompts for t in p):
        raise ValueError("token outside the vocabulary")
    for p in prompts:
        if lm.max_positions and len(p) + max_new_tokens - 1 > lm.max_positions:
            raise ValueError(f"the request reaches position {len(p) + max_new_tokens - 1}, the model has {lm.max_positions}")
    step_tokens = min(int(step_tokens), lm.max_step_tokens)
    need = [beam_pages(lambda n: lm.pages_needed(-1, n), len(p), beams, max_new_tokens, lm.page_tokens) for p in prompts]
    out: List[List[BeamHypothesis]] = []
    while len(out) < len(prompts):
        first, room = len(out), min(lm.free_slots, step_tokens) // beams
        n, pages = first, lm.free_pages
        while n < len(prompts) and n - first < room and need[n] <= pages:
            pages -= need[n]
            n += 1
        if n == first:
            raise BufferError(f"the search needs {beams} slots, {need[n]} pages and {beams} tokens a step; there are {lm.free_slots}, {lm.free_pages} and {step_tokens}")
        out += _search(lm, prompts[first:n], beams, max_new_tokens, eos, length_penalty, step_tokens)
    return out


def _prefill(lm: TokenLM, prompts: List[List[int]], slots: List[int], step_tokens: int) -> torch.Tensor:
    """Logits behind every prompt, [prompts, vocab]."""
    logits, entries, budget = torch.empty((len(prompts), lm.vocab), dtype=_F32, device=lm.device), [], step_tokens
    done = 0

    def run():
        nonlocal entries, budget, done
        n = sum(len(w) for _, _, w in entries)
        if n:
            lm.step(entries, out=logits[done:done + n])
        else:
            lm.step(entries)
        entries, budget, done = [], step_tokens, done + n

    for prompt, slot in zip(prompts, slots):
        fed = 0
        while fed < len(prompt):
            take = min(budget, len(prompt) - fed)
            fed += take
            budget -= take
            entries.append((slot, prompt[fed - take:fed], [take - 1] if fed == len(prompt) else []))
            if not budget:
                run()
    if entries:
        run()
    return logits


def _search(lm: TokenLM, prompts: List[List[int]], beams: int, max_new_tokens: int, eos: int, length_penalty: float, step_tokens: int) -> List[List[BeamHypothesis]]:
    device, opened = lm.device, []
    result: List[List[BeamHypothesis]] = [[] for _ in prompts]
    try:
        for _ in range(len(prompts) * beams):
            opened.append(lm.open())
        slots = [opened[i:i + beams] for i in range(0, len(opened), beams)]
        live = list(range(len(prompts)))
        trace: List[List[Tuple[List[int], List[int]]]] = [[] for _ in prompts]      # parents and tokens of every step
        logits = _prefill(lm, prompts, [s[0] for s in slots], step_tokens).repeat_interleave(beams, dim=0)
        scores = torch.full((len(prompts), beams), float("-inf"), device=device)
        scores[:, 0] = 0.0
        lengths = torch.zeros((len(prompts), beams), dtype=_I32, device=device)
        finished = None
        while True:
            r = beam_select(logits, scores, lengths, finished, eos, length_penalty, lib=lm._lib)
            scores, lengths, finished = r.scores, r.lengths, r.finished
            parents, tokens, size, ended = torch.stack([r.parents, r.tokens, lengths, lengths.new_zeros(lengths.shape) if finished is None else finished.int()]).tolist()
            for i, p, t in zip(live, parents, tokens):
                trace[i].append((p, t))
            last = len(trace[live[0]]) == max_new_tokens
            stay = [] if last else [j for j in range(len(live)) if not all(ended[j])]
            if len(stay) < len(live):
                sums = scores.tolist()
                for j in set(range(len(live))).difference(stay):
                    result[live[j]] = _hypotheses(trace[live[j]], sums[j], size[j])
                    for s in slots[j]:
                        lm.close(s)
                        opened.remove(s)
                if not stay:
                    return result
                at = torch.tensor(stay, device=device)
                scores, lengths, finished = scores[at], lengths[at], None if finished is None else finished[at]
                live, slots, parents, tokens = ([x[j] for j in stay] for x in (live, slots, parents, tokens))
            lm.reorder(slots, parents)
            logits = lm.step([(s, [t], [0]) for row, toks in zip(slots, tokens) for s, t in zip(row, toks)])
    finally:
        for s in opened:
            lm.close(s)


def _hypotheses(trace: List[Tuple[List[int], List[int]]], sums: List[float], size: List[int]) -> List[BeamHypothesis]:
    out = []
    for i, (score, n) in enumerate(zip(sums, size)):
        if score == float("-inf"):
            continue
        back, tokens = i, []
        for parents, toks in reversed(trace):
            tokens.append(toks[back])
            back = parents[back]
        out.append(BeamHypothesis(tokens[::-1][:n], score))
    return out
