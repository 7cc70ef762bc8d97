"""Cases for the token language models' operators - the 8-bit paged cache, its attention, beam selection and reordering - run on the kernel
simulator (test_operators_sim.py) and on the GPU (test_e_operators_gpu.py), against plain restatements in 64 bits."""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import List

import numpy as np
import pytest
import torch

from moshi_amd.beam import beam_reorder, beam_search, beam_select
from moshi_amd.kv_cache import PagedKVCache

F32, BF16 = torch.float32, torch.bfloat16
TOP = {"int8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -100


# ---- the cache in 64 bits -------------------------------------------------------------------------------------------------------
def code64(x, codes):
    """The nearest code's value, ties to even: int8 integers, or e4m3 (3 bits behind the leading one, smallest step 2^-9)."""
    if codes == "int8":
        return x.round().clamp(-127, 127)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    return ((x / torch.exp2(e - 3)).round() * torch.exp2(e - 3)).clamp(-448, 448)


def rotate64(x, pos, rot, base, halves):
    """x [rows, heads, dim] float64."""
    if not rot:
        return x
    a = pos.double()[:, None, None] * torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
    i = torch.arange(rot // 2)
    p, q = (i, i + rot // 2) if halves else (2 * i, 2 * i + 1)
    y = x.clone()
    y[..., p], y[..., q] = x[..., p] * a.cos() - x[..., q] * a.sin(), x[..., p] * a.sin() + x[..., q] * a.cos()
    return y


class Cache64:
    """Values [pages, heads, 64, n] (codes, as float64) and scales [pages, heads, 4] of one side of a cache."""

    def __init__(self, codes, values, scales):
        self.codes, self.v, self.s = codes, values, scales

    @classmethod
    def of(cls, cache: PagedKVCache, side: str):
        x = getattr(cache, side).cpu().to(torch.float32).double()
        return cls("int8" if cache.k.dtype == torch.int8 else "e4m3", (x if side == "k" else x.transpose(2, 3)).contiguous(), getattr(cache, side + "_scale").cpu().double())

    def append(self, x, page_of, pos):
        """x [rows, heads, n] for positions pos, pos + 1, ..; page_of(position): page or -1."""
        n = len(x)
        for b in range(pos // 16 * 16, pos + n, 16):
            page, part, lo, hi = page_of(b), b % 64 // 16, max(b, pos), min(b + 16, pos + n)
            if page < 0:
                continue
            new = x[lo - pos:hi - pos].transpose(0, 1)                                    # [heads, rows, n]
            for h in range(x.shape[1]):
                at = slice(b % 64, b % 64 + lo - b)
                big = new[h].abs().max()
                scale = torch.clamp(big, min=TINY) / TOP[self.codes]
                before = self.s[page, h, part]
                if lo > b:
                    scale = torch.maximum(scale, before)
                if not torch.isfinite(big) or (lo > b and not torch.isfinite(before)):
                    self.s[page, h, part] = math.nan
                    self.v[page, h, b % 64:b % 64 + hi - b] = 0
                    continue
                if lo > b and scale != before:
                    self.v[page, h, at] = code64(self.v[page, h, at] * (before / scale), self.codes)
                self.v[page, h, b % 64 + lo - b:b % 64 + hi - b] = code64(new[h] / scale, self.codes)
                self.s[page, h, part] = scale

    def values(self, page):
        return self.v[page] * self.s[page].repeat_interleave(16, dim=-1)[..., None]        # [heads, 64, n]


@dataclass
class Case:
    """Sequences of a call: what they hold, what they bring (`single`: one row each, without `rows`)."""
    past: List[int]
    rows: List[int]
    kv_heads: int = 2
    rep: int = 2
    dim: int = 64
    vdim: int = 64
    codes: str = "int8"
    dtype: torch.dtype = BF16
    rot: int = 0
    halves: bool = False
    window: int = 0
    keep: int = 0
    sink: bool = False
    single: bool = False
    extra_rows: int = 0                  # rows behind the last sequence
    seed: int = 0
    missing: List[tuple] = field(default_factory=list)      # (sequence, page index, page number in the table)
    base: float = 1e4
    spread: float = 1.0                  # of the values' magnitudes from token to token
    wide_table: int = 0                  # unused entries of the page table behind the ones needed

    @property
    def total(self):
        return sum(self.rows) + self.extra_rows


def build(c: Case, dev, lib, fill=True, strided=False):
    """The cache with a random past (token by token magnitudes that differ), the call's tensors, and the plain cache."""
    g = torch.Generator().manual_seed(c.seed + 100)
    need = [-(-(max(p, 0) + r) // 64) for p, r in zip(c.past, c.rows)]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).tolist()
    ld = max(need) + c.wide_table
    table = torch.full((len(need), max(ld, 1)), -1, dtype=torch.int32)
    at = 0
    for e, n in enumerate(need):
        table[e, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    for e, i, page in c.missing:
        table[e, i] = page
    cache = PagedKVCache.empty(pages, c.kv_heads, c.dim, c.vdim, c.codes, dev, rot_dim=c.rot, rot_base=c.base, rot_halves=c.halves, lib=lib)
    if fill:
        def noise(t):                    # any byte at all, where nothing is read it must not matter
            return torch.randint(-128, 128, t.shape, generator=g, dtype=torch.int8).to(dev)
        k, v = noise(cache.k.view(torch.int8)), noise(cache.v.view(torch.int8))
        cache.k.view(torch.int8).copy_(k)
        cache.v.view(torch.int8).copy_(v)
        for s in (cache.k_scale, cache.v_scale):
            s.copy_(torch.where(torch.rand(s.shape, generator=g) < 0.2, math.nan, 1e30))
        for e, p in enumerate(c.past):
            if p > 0:
                for side in "kv":
                    put_past(c, cache, table[e], p, side, g)
    T = c.total

    def rows(heads, n):
        x = torch.randn((T, heads, n + (8 if strided else 0)), generator=g) * torch.exp(c.spread * torch.randn((T, 1, 1), generator=g))
        x = x.to(c.dtype).to(dev)
        return x[..., 3:n + 3] if strided else x

    q, k, v = rows(c.kv_heads * c.rep, c.dim), rows(c.kv_heads, c.dim), rows(c.kv_heads, c.vdim)
    q.mul_(0.125)                        # scores of a few units: their own roundings stay small beside a wrong weight
    starts = torch.cumsum(torch.tensor([0] + c.rows), 0).to(torch.int32).to(dev)
    args = (table.to(dev), torch.tensor(c.past, dtype=torch.int32).to(dev), None if c.single else starts)
    return cache, q, k, v, args


def put_past(c, cache, table, n, side, g):
    """Random codes and scales for a sequence's first n tokens, written to the arrays directly (both layouts are documented)."""
    dim = c.dim if side == "k" else c.vdim
    for b in range(0, n, 16):
        page = int(table[b // 64])
        if page < 0 or page >= cache.pages:
            continue
        m = min(16, n - b)
        x = code64(torch.randn((c.kv_heads, m, dim), generator=g).double() * TOP[c.codes] / 3.5, c.codes).float()
        arr = getattr(cache, side).view(torch.int8) if c.codes == "int8" else getattr(cache, side)
        y = x.to(torch.int8) if c.codes == "int8" else x.to(torch.float8_e4m3fn)
        raw = arr.view(torch.int8)
        if side == "k":
            raw[page, :, b % 64:b % 64 + m] = y.view(torch.int8).to(raw.device)
        else:
            raw[page, :, :, b % 64:b % 64 + m] = y.view(torch.int8).transpose(1, 2).to(raw.device)
        getattr(cache, side + "_scale")[page, :, b % 64 // 16] = ((0.5 + torch.rand((c.kv_heads,), generator=g)) / TOP[c.codes] * 3).to(raw.device)


def page_finder(c, table, cache):
    def of(e):
        def page_of(pos):
            i = pos // 64
            p = int(table[e, i]) if i < table.shape[1] else -1
            return p if 0 <= p < cache.pages else -1
        return page_of
    return of


def sequences(c: Case):
    row = 0
    for e, (p, n) in enumerate(zip(c.past, c.rows)):
        yield e, p, n, row
        row += n


APPENDS = {
    "first_token": Case([0], [1], single=True),
    "single_tokens": Case([0, 1, 15, 16, 63, 64, 200, 37], [1] * 8, single=True, kv_heads=3, codes="int8"),
    "single_tokens_e4m3": Case([5, 31, 32, 79, 128], [1] * 5, single=True, kv_heads=5, codes="e4m3", dtype=F32, spread=2.0),
    "portions": Case([0, 7, 16, 100, 63], [40, 9, 16, 1, 66], kv_heads=2, rot=32, halves=True),
    "portions_e4m3": Case([3, 0, 61], [30, 16, 5], kv_heads=1, codes="e4m3", rot=64, halves=False, dtype=F32, spread=2.0),
    "rotated_part_of_odd_sizes": Case([9, 250], [20, 3], dim=80, vdim=48, rot=24, halves=True),
    "pairs_side_by_side": Case([9, 250], [20, 3], dim=48, vdim=16, rot=8, codes="e4m3"),
    "largest_heads": Case([30], [21], dim=256, vdim=256, rot=256, halves=True, kv_heads=1),
    "smallest_heads": Case([30], [21], dim=16, vdim=16, kv_heads=4, dtype=F32),
    "far": Case([(1 << 22) + 5], [1], single=True, rot=64, halves=True, dtype=F32),
    "nothing_to_append": Case([5, 12, 30], [0, 3, 0]),
    "rows_behind": Case([5, 12], [2, 3], extra_rows=4),
    "pages_that_are_not_there": Case([60, 0], [10, 70], missing=[(0, 1, -1), (1, 0, 1 << 30)]),
    "passed_over": Case([-1, 4, -7], [1, 1, 1], single=True),
}


def check_append(name, dev, lib, strided=False):
    """Scales to fp32 rounding; every code within half a step of what it is rounded from; every other byte as it was."""
    c = APPENDS[name]
    far = c.past[0] > 1 << 20
    if far:                              # one page stands for all: the table is short of nothing but memory
        c = Case(**{**c.__dict__, "past": [5]})
    cache, _, k, v, args = build(c, dev, lib, strided=strided)
    table = args[0].cpu()
    if far:
        args = (args[0][:, :1].expand(1, (1 << 22) // 64 + 1).contiguous(), torch.tensor([(1 << 22) + 5], dtype=torch.int32, device=args[0].device), args[2])
        c = Case(**{**c.__dict__, "past": [(1 << 22) + 5]})
    before = {side: Cache64.of(cache, side) for side in "kv"}
    raw = {side: (getattr(cache, side).view(torch.int8).cpu().clone(), getattr(cache, side + "_scale").cpu().clone()) for side in "kv"}
    cache.append(k, v, *args)
    finder = page_finder(c, args[0].cpu(), cache)
    for side, x in (("k", k), ("v", v)):
        x = x.detach().cpu().double()
        want, got = Cache64(c.codes, before[side].v.clone(), before[side].s.clone()), Cache64.of(cache, side)
        touched = torch.zeros(want.v.shape[:3], dtype=torch.bool)
        for e, p, n, row in sequences(c):
            if p < 0 or not n:
                continue
            y = x[row:row + n]
            if side == "k":
                y = rotate64(y, torch.arange(p, p + n), c.rot, c.base, c.halves)
            want.append(y, finder(e), p)
            for b in range(p // 16 * 16, p + n):
                if finder(e)(b) >= 0:
                    touched[finder(e)(b), :, b % 64] = True
        live = touched.view(touched.shape[0], touched.shape[1], 4, 16).any(-1)
        # the largest magnitude passes a rotation (two products, one sum: 3 half steps, and an angle good to 2 steps) and a division
        assert torch.allclose(got.s[live], want.s[live], rtol=2 ** -21, atol=0)
        gv, wv = got.values(slice(None)), want.values(slice(None))
        step = want.s.repeat_interleave(16, dim=2)[..., None] * (1.0 if c.codes == "int8" else torch.exp2(torch.floor(torch.log2(want.v.abs().clamp(min=2.0 ** -6))) - 3))
        # equal but for values beside a border between two codes, which may fall on either side of it
        off = ((gv - wv).abs() / step.expand_as(wv))[touched]
        assert off.max() <= 1.01 and (off > 1e-3).double().mean() <= 2e-3, (off.max(), (off > 1e-3).double().mean())
        keep = ~touched.to(cache.k.device).cpu()
        now = getattr(cache, side).view(torch.int8).cpu()
        a, b = (now, raw[side][0]) if side == "k" else (now.transpose(2, 3), raw[side][0].transpose(2, 3))
        assert torch.equal(a[keep], b[keep])
        assert torch.equal(getattr(cache, side + "_scale").cpu()[~live].view(torch.int32), raw[side][1][~live].view(torch.int32))
    # what it is read back as
    if c.total == sum(c.rows) and min(c.past) >= 0:
        kr, vr = cache.read(*args, tokens=c.total, dtype=F32)
        for got, side in ((kr, "k"), (vr, "v")):
            have = Cache64.of(cache, side)
            for e, p, n, row in sequences(c):
                for i in range(n):
                    page = finder(e)(p + i)
                    want = have.values(page)[:, (p + i) % 64] if page >= 0 else torch.zeros_like(got[row + i].cpu().double())
                    assert torch.allclose(got[row + i].cpu().double(), want, rtol=2 ** -23, atol=0)


def check_append_order(dev, lib, codes):
    """Token by token, in portions, at once: the same scales, and values within the roundings that a growing scale costs."""
    g = torch.Generator().manual_seed(3)
    n, heads, dim = 70, 2, 32
    x = (torch.randn((n, heads, dim), generator=g) * torch.exp(torch.randn((n, 1, 1), generator=g))).to(dev)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=dev)
    out = []
    for cuts in ([n], [1] * n, [13, 30, 27]):
        cache = PagedKVCache.empty(2, heads, dim, dim, codes, dev, lib=lib)
        at = 0
        for m in cuts:
            cache.append(x[at:at + m], x[at:at + m], table, torch.tensor([at], dtype=torch.int32, device=dev), torch.tensor([0, m], dtype=torch.int32, device=dev))
            at += m
        out.append([t.cpu() for t in (cache.k_scale, cache.v_scale, *cache.read(table, torch.zeros(1, dtype=torch.int32, device=dev),
                                                                               torch.tensor([0, n], dtype=torch.int32, device=dev), tokens=n))])
    for other in out[1:]:
        assert torch.equal(out[0][0], other[0]) and torch.equal(out[0][1], other[1])
        for a, b in zip(out[0][2:], other[2:]):
            # at most 16 growths, each half a step of a scale that is then at most the last one
            scale = a.abs().view(n, -1).amax(dim=1).max()
            limit = (8.5 / 127 if codes == "int8" else 16 * 2 ** -4) * scale
            assert (a - b).abs().max() <= limit


def check_not_finite(dev, lib, codes):
    """A NaN or an infinity poisons its block of its head, for whoever sees it, and nothing else; a block that starts anew is clean."""
    c = Case([0], [40], kv_heads=2, rep=1, dim=32, vdim=32, codes=codes, dtype=F32)
    for bad in (math.nan, math.inf, -math.inf):
        for side in "kv":
            cache, q, k, v, args = build(c, dev, lib)
            t = {"k": k, "v": v}[side]
            t[20, 1, 5] = bad                                  # position 20, block 1, head 1
            cache.append(k, v, *args)
            scale = getattr(cache, side + "_scale").cpu()[int(args[0][0, 0])]
            nan = torch.zeros(scale.shape, dtype=torch.bool)
            nan[1, 1] = True
            assert torch.equal(scale[:, :3].isnan(), nan[:, :3])
            out = cache.attend(q, *args).cpu()
            assert out[:, 0].isfinite().all() and out[:16, 1].isfinite().all() and out[20:, 1].isnan().any(dim=-1).all()
            # a later token of the same block keeps it so; a window that has left it behind does not see it
            assert cache.attend(q, *args, window=4).cpu()[36:, 1].isfinite().all()
            fresh = torch.zeros_like(k[:16])
            cache.append(fresh, fresh, args[0], torch.tensor([16], dtype=torch.int32, device=dev), torch.tensor([0, 16], dtype=torch.int32, device=dev))
            assert getattr(cache, side + "_scale").cpu()[int(args[0][0, 0]), :, 1].isfinite().all()


ATTENDS = {
    "first_token": Case([0], [1], single=True),
    "single_tokens": Case([0, 1, 15, 16, 63, 64, 200], [1] * 7, single=True, kv_heads=2, rep=4),
    "single_fp32": Case([3, 70, 131], [1] * 3, single=True, kv_heads=1, rep=3, dtype=F32, dim=80, vdim=48),
    "own_heads": Case([90, 17], [1, 1], single=True, kv_heads=3, rep=1, codes="e4m3"),
    "more_than_a_tile_of_heads": Case([90, 17], [1, 1], single=True, kv_heads=1, rep=20),
    "rotated": Case([190, 64], [1, 1], single=True, rot=64, halves=True, kv_heads=1, rep=5),
    "rotated_side_by_side": Case([190, 64], [1, 1], single=True, rot=32, codes="e4m3", dtype=F32),
    "window": Case([190, 64, 10, 129], [1] * 4, single=True, window=50, rep=4),
    "window_one": Case([190, 64], [1, 1], single=True, window=1),
    "window_that_keeps": Case([300, 64, 3], [1] * 3, single=True, window=40, keep=5, codes="e4m3"),
    "keeps_pages": Case([300, 64], [1] * 2, single=True, window=3, keep=70, sink=True),
    "sink": Case([30, 0], [1, 1], single=True, sink=True, dtype=F32),
    "many_splits": Case([1300], [1], single=True, kv_heads=1, rep=2, dim=16, vdim=16, wide_table=3),
    "largest_heads": Case([70], [1], single=True, kv_heads=1, rep=2, dim=256, vdim=256, rot=256, halves=True),
    "largest_heads_fp32": Case([70], [1], single=True, kv_heads=1, rep=2, dim=256, vdim=240, dtype=F32, codes="e4m3"),
    "values_wider_than_keys": Case([70], [1], single=True, dim=16, vdim=144, rep=1),
    "portion": Case([0], [37], kv_heads=1, rep=4),
    "portions": Case([0, 7, 16, 100], [40, 9, 1, 17], kv_heads=2, rep=2, rot=64, halves=True),
    "portion_behind_a_past": Case([150], [33], kv_heads=1, rep=5, codes="e4m3", rot=32),
    "portions_window": Case([0, 130, 90], [70, 20, 1], kv_heads=1, rep=4, window=33, keep=3, sink=True),
    "portions_fp32": Case([20, 0, 5], [30, 1, 18], kv_heads=1, rep=3, dim=128, vdim=112, dtype=F32, rot=128, halves=True),
    "portion_of_own_heads": Case([10], [70], kv_heads=2, rep=1, dim=48, vdim=32),
    "portion_largest_heads": Case([40], [20], kv_heads=1, rep=2, dim=256, vdim=256, rot=128),
    "portion_largest_heads_fp32": Case([40], [10], kv_heads=1, rep=2, dim=240, vdim=256, dtype=F32, codes="e4m3"),
    "portion_splits": Case([520], [9], kv_heads=1, rep=3, dim=16, vdim=32, wide_table=9),
    "empty_sequences": Case([5, 12, 30, 2], [0, 25, 0, 1], kv_heads=1, rep=2),
    "rows_behind": Case([5, 12], [2, 20], extra_rows=5, rep=4),
    "pages_that_are_not_there": Case([200, 130], [1, 1], single=True, missing=[(0, 1, -1), (1, 0, 1 << 30), (1, 1, -5)]),
    "nothing_to_see": Case([70, 3], [1, 1], single=True, missing=[(0, 0, -1), (0, 1, -1), (1, 0, -3)]),
    "portion_with_missing_pages": Case([100], [40], rep=4, kv_heads=1, missing=[(0, 1, -1)], codes="e4m3"),
    "passed_over": Case([-1, 4, -7], [1, 1, 1], single=True),
    "many_short_sequences": Case([3 * i for i in range(70)], [1] * 70, kv_heads=1, rep=2, dim=16, vdim=16),
}


def attend64(c: Case, cache, q, args, scale=None):
    """Outputs, the largest magnitude among the values, and for every row the largest sum over dimensions of |query x key| times the scale."""
    finder = page_finder(c, args[0].cpu(), cache)
    k64, v64 = Cache64.of(cache, "k"), Cache64.of(cache, "v")
    q = q.detach().cpu().double()
    scale = c.dim ** -0.5 if scale is None else scale
    out = torch.full((c.total, q.shape[1], c.vdim), math.nan, dtype=torch.float64)
    size, top = torch.zeros(c.total), 0.0
    for e, p, n, row in sequences(c):
        if p < 0 or not n:
            continue
        pages = [finder(e)(64 * i) for i in range((p + n + 63) // 64)]
        keys = torch.cat([k64.values(max(i, 0)) for i in pages], dim=1)
        vals = torch.cat([v64.values(max(i, 0)) for i in pages], dim=1)
        there = torch.tensor([i >= 0 for i in pages]).repeat_interleave(64)
        x = rotate64(q[row:row + n], torch.arange(p, p + n), c.rot, c.base, c.halves)
        for i in range(n):
            t = torch.arange(len(there))
            seen = there & (t <= p + i)
            if c.window:
                seen &= (p + i - t < c.window) | (t < c.keep)
            out[row + i] = 0.0
            if not seen.any():
                continue
            for h in range(q.shape[1]):
                kk, vv = keys[h // c.rep][seen], vals[h // c.rep][seen]
                s = kk @ x[i, h] * scale
                w = torch.exp(s - s.max())
                total = w.sum() + (torch.exp(-s.max()) if c.sink else 0.0)
                out[row + i, h] = (w / total) @ vv
                size[row + i] = max(size[row + i], float((kk.abs() @ x[i, h].abs()).max() * abs(scale)))
                top = max(top, float(vv.abs().max()))
    return out, size, top


def check_attend(name, dev, lib, strided=False):
    c = ATTENDS[name]
    cache, q, k, v, args = build(c, dev, lib, strided=strided)
    cache.append(k, v, *args)
    held = torch.full((c.total, c.kv_heads * c.rep, c.vdim), 7.0, dtype=c.dtype, device=q.device)
    got = cache.attend(q, *args, window=c.window, keep_first=c.keep, sink=c.sink, out=held)
    assert got is held
    want, size, top = attend64(c, cache, q, args)
    # a score is a sum of products whose queries are off by half a step h of their operands (fp16 2^-11 / 2; two parts: 2^-23) and whose sum, in fp32, by
    # dim half steps of 2^-23 / 2; a weight by twice a score's error, by h, by the exponential's 2^-22 and by the sum's rounding; outputs by that times the largest value,
    # and by their own rounding
    h = 2.0 ** -12 if c.dtype == BF16 else 2.0 ** -23
    off = 2 * size * (h + c.dim * 2.0 ** -24) + h + 2.0 ** -20
    limit = (off[:, None, None] * top + want.abs() * (torch.finfo(c.dtype).eps / 2)).double()
    got = got.cpu().double()
    for e, p, n, row in sequences(c):
        if p < 0:
            assert (got[row:row + n] == 7).all()
        else:
            assert got[row:row + n].isfinite().all()
            assert ((got - want).abs() <= limit)[row:row + n].all(), float(((got - want).abs() / limit)[row:row + n].max())
    assert (got[sum(c.rows):] == 7).all()
    again = cache.attend(q, *args, window=c.window, keep_first=c.keep, sink=c.sink)
    used = torch.cat([torch.arange(row, row + n) for e, p, n, row in sequences(c) if p >= 0])
    assert torch.equal(again.cpu()[used], held.cpu()[used])


def check_extreme_scores(dev, lib):
    """Scores far apart, all at the largest finite magnitudes' side, tiny values beside large ones: no overflow on the way, no sum lost."""
    c = Case([130], [1], single=True, kv_heads=1, rep=2, dim=32, vdim=32, dtype=F32)
    for qs, vs in ((1e4, 1.0), (1e-30, 1.0), (1e18, 1e18), (1.0, 1e-30), (0.0, 1e30)):
        cache, q, k, v, args = build(c, dev, lib, fill=False)
        g = torch.Generator().manual_seed(9)
        past = [torch.randn((131, 1, 32), generator=g).to(dev) for _ in range(2)]
        past[1][:16] *= 1e-6                                   # a first block of small values, as first tokens have
        at = (args[0], torch.zeros(1, dtype=torch.int32, device=dev), torch.tensor([0, 131], dtype=torch.int32, device=dev))
        cache.append(past[0], past[1] * vs, *at)
        q = q * qs
        got = cache.attend(q, *args).cpu().double()
        want, size, top = attend64(c, cache, q, args)
        h = 2.0 ** -23
        limit = (2 * size.max() * (h + 32 * 2.0 ** -24) + h + 2.0 ** -20) * top + want.abs() * 2.0 ** -24
        assert got.isfinite().all() and ((got - want).abs() <= limit).all(), (qs, vs)
    # all the weight on a block of small values, beside a block of large ones: its own precision is what counts
    cache, q, k, v, args = build(c, dev, lib, fill=False)
    keys, vals = torch.zeros((131, 1, 32), device=dev), torch.randn((131, 1, 32), generator=torch.Generator().manual_seed(4)).to(dev)
    keys[3, 0, 0] = 1.0
    vals[:16] *= 1e-5
    cache.append(keys, vals, *at)
    q = torch.zeros_like(q)
    q[..., 0] = 400.0
    got, held = cache.attend(q, *args).cpu(), cache.read(*at, tokens=131)[1].cpu()[3]
    assert torch.allclose(got[0].double(), held.double().expand_as(got[0]), rtol=2.0 ** -20, atol=1e-12)


def check_refusals(dev, lib):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    new = lambda **kw: PagedKVCache.empty(**{**dict(pages=3, kv_heads=2, dim=32, device=dev, lib=lib), **kw})  # noqa: E731
    for bad in (dict(dim=24), dict(dim=272), dict(vdim=8), dict(vdim=288)):
        with pytest.raises(NotImplementedError):
            new(**bad)
    for bad in (dict(rot_dim=12), dict(rot_dim=40), dict(rot_dim=-8), dict(codes="int4"), dict(rot_dim=16, rot_base=0.0), dict(rot_dim=16, rot_base=math.inf)):
        with pytest.raises(ValueError):
            new(**bad)
    with pytest.raises(AssertionError):
        new(pages=0)
    c = new()
    with pytest.raises(AssertionError):
        PagedKVCache(c.k, c.v[:2], c.k_scale, c.v_scale, lib=lib)
    with pytest.raises(AssertionError):
        PagedKVCache(c.k, c.v, c.k_scale[:, :, :3], c.v_scale, lib=lib)
    with pytest.raises(ValueError):
        PagedKVCache(c.k, c.v.view(torch.float8_e4m3fn), c.k_scale, c.v_scale, lib=lib)
    with pytest.raises(ValueError):
        PagedKVCache(c.k.transpose(0, 1).contiguous().transpose(0, 1), c.v, c.k_scale, c.v_scale, lib=lib)
    x, table, pos = torch.zeros((2, 2, 32), dtype=BF16, device=dev), i32([0], [1]).view(2, 1), i32(0, 0)
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    for args, kind in (((x[:, :1], x, table, pos), AssertionError), ((x, x[:1], table, pos), AssertionError), ((x, x.float(), table, pos), AssertionError),
                       ((x.half(), x.half(), table, pos), ValueError), ((x, x, table.long(), pos), ValueError), ((x, x, table, pos.long()), ValueError),
                       ((x, x, table[:1], pos), AssertionError), ((x, x, table, pos[:1]), AssertionError), ((x, x, table, pos, i32(0, 1)), AssertionError),
                       ((x[:1], x[:1], table, pos), AssertionError), ((x.transpose(1, 2).contiguous().transpose(1, 2), x, table, pos), ValueError),
                       ((x, x, table[:, :0], pos), ValueError)):
        with pytest.raises(kind):
            c.append(*args)
    q = torch.zeros((2, 4, 32), dtype=BF16, device=dev)
    for kw, kind in ((dict(q=q[:, :3]), AssertionError), (dict(window=-1), ValueError), (dict(keep_first=-1), ValueError), (dict(scale=math.nan), ValueError),
                     (dict(scale=math.inf), ValueError), (dict(out=q.float()), AssertionError), (dict(out=q[:1]), AssertionError), (dict(q=q[..., :16]), AssertionError)):
        with pytest.raises(kind):
            c.attend(**{**dict(q=q, table=table, positions=pos), **kw})
    with pytest.raises(ValueError):
        c.read(table, pos, i32(0, 1, 2))
    with pytest.raises(ValueError):
        c.read(table, pos, dtype=torch.float16)
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(before, (c.k, c.v, c.k_scale, c.v_scale)))
    # nothing to do: nothing done, no row touched
    none = torch.zeros((0, 2, 32), dtype=BF16, device=dev)
    c.append(none, none, table[:0], pos[:0])
    assert c.attend(torch.zeros((0, 4, 32), dtype=BF16, device=dev), table[:0], pos[:0]).shape == (0, 4, 32)
    # arguments that only the C entry can be given
    import ctypes as C
    from moshi_amd import _capi
    s = _capi.KVSeqs(2, 2, None, pos.data_ptr(), table.data_ptr(), 1)
    call = lambda **kw: lib.mmi_kv_attend(*{**dict(cache=C.byref(c._desc), seqs=C.byref(s), dtype=_capi.MMI_BF16, heads=4, q=q.data_ptr(), qr=128, qh=32, o=q.data_ptr(), orow=128, oh=32,  # noqa: E731
                                                   scale=1.0, window=0, keep=0, sink=0, w=None, n=0, stream=None), **kw}.values())
    for kw in (dict(q=None), dict(o=None), dict(qr=-1), dict(o=q.data_ptr() + 2), dict(cache=None), dict(seqs=None)):
        assert call(**kw) == _capi.MMI_ERR_INVALID
    assert call(dtype=_capi.MMI_F16) == _capi.MMI_ERR_UNSUPPORTED
    assert call(seqs=C.byref(_capi.KVSeqs(2, 3, None, pos.data_ptr(), table.data_ptr(), 1))) == _capi.MMI_ERR_SHAPE
    assert call(seqs=C.byref(_capi.KVSeqs(-1, 3, None, pos.data_ptr(), table.data_ptr(), 1))) == _capi.MMI_ERR_INVALID
    long = C.byref(_capi.KVSeqs(2, 2, None, pos.data_ptr(), table.data_ptr(), 100))
    assert lib.mmi_kv_attend_workspace(C.byref(c._desc), long, 4, 0, 0) > 0 and call(seqs=long) == _capi.MMI_ERR_INVALID


# ---- beam search ----------------------------------------------------------------------------------------------------------------
def select64(logits, scores, lengths=None, finished=None, eos=-1, penalty=0.0):
    """Best candidates by sorting all of them: NaN counts as -infinity, equal ranks go to the lower beam, then the lower token."""
    B, K = scores.shape
    V = logits.shape[1]
    x = logits.cpu().double().view(B, K, V).numpy()
    out = []
    for b in range(B):
        total, rank = np.full((K, V), -np.inf), np.full((K, V), -np.inf)
        for k in range(K):
            done = finished is not None and bool(finished[b, k])
            n = max(1, (int(lengths[b, k]) if lengths is not None else 0) + (0 if done else 1))
            if done:
                total[k, eos] = float(scores[b, k])
            else:
                with np.errstate(all="ignore"):
                    top = np.max(x[b, k])
                    total[k] = float(scores[b, k]) + x[b, k] - (top + np.log(np.sum(np.exp(x[b, k] - top))))
            total[k][np.isnan(total[k])] = -np.inf
            rank[k] = total[k] / float(n) ** penalty if penalty else total[k]
        order = np.argsort(-rank.reshape(-1), kind="stable")[:K]
        parents, tokens = order // V, order % V
        fin = np.array([(finished is not None and bool(finished[b, p])) or t == eos for p, t in zip(parents, tokens)])
        lens = np.array([(int(lengths[b, p]) if lengths is not None else 0) + (0 if finished is not None and bool(finished[b, p]) else 1) for p in parents])
        out.append((total.reshape(-1)[order], parents, tokens, fin, lens))
    return [np.stack(t) for t in zip(*out)]


SELECTS = {
    "one_beam": dict(batch=2, beams=1, vocab=100),
    "four": dict(batch=1, beams=4, vocab=5000),
    "odd_rows": dict(batch=3, beams=3, vocab=1027),
    "bf16_ties": dict(batch=2, beams=8, vocab=2500, dtype=BF16, coarse=True),
    "all_equal": dict(batch=1, beams=6, vocab=1500, equal=True),
    "thirty_two": dict(batch=1, beams=32, vocab=1300),
    "more_beams_than_tokens": dict(batch=2, beams=8, vocab=3),
    "one_token": dict(batch=2, beams=5, vocab=1),
    "start": dict(batch=3, beams=4, vocab=700, start=True),
    "finished": dict(batch=4, beams=6, vocab=900, finished=0.5, penalty=0.7),
    "all_finished": dict(batch=2, beams=4, vocab=90, finished=1.1, penalty=1.0),
    "negative_penalty": dict(batch=2, beams=4, vocab=300, finished=0.3, penalty=-0.5),
    "masked": dict(batch=2, beams=4, vocab=3000, masked=-math.inf),
    "masked_lowest": dict(batch=2, beams=4, vocab=3000, masked=-3.4028234663852886e38),
    "masked_all_but_two": dict(batch=1, beams=4, vocab=2100, masked=-math.inf, left=2),
    "masked_altogether": dict(batch=2, beams=3, vocab=1100, masked=-math.inf, left=0),
    "not_finite": dict(batch=2, beams=4, vocab=1200, spoil=True),
    "strided": dict(batch=2, beams=3, vocab=513, pad=6),
    # more candidates than are ranked at once
    "many": dict(batch=2, beams=32, vocab=9000),
    "many_finished": dict(batch=1, beams=20, vocab=12100, finished=0.4, penalty=0.8),
    "many_bf16_ties": dict(batch=1, beams=24, vocab=10007, dtype=BF16, coarse=True),
    "many_start": dict(batch=1, beams=32, vocab=5000, start=True),
    "many_equal": dict(batch=1, beams=16, vocab=17000, equal=True),
    "many_equal_lists": dict(batch=1, beams=32, vocab=33 * 1024, equal=True),
    "many_masked_all_but_two": dict(batch=1, beams=24, vocab=9000, masked=-math.inf, left=2),
    "many_masked_lowest": dict(batch=1, beams=24, vocab=9000, masked=-3.4028234663852886e38),
    "many_not_finite": dict(batch=1, beams=24, vocab=9000, spoil=True),
}


def check_select(name, dev, lib):
    o = dict(dtype=F32, coarse=False, equal=False, start=False, finished=0.0, penalty=0.0, masked=None, left=900, spoil=False, pad=0)
    o.update(SELECTS[name])
    g = torch.Generator().manual_seed(len(name))
    B, K, V = o["batch"], o["beams"], o["vocab"]
    x = torch.randn((B * K, V + o["pad"]), generator=g) * 3
    if o["coarse"]:
        x = (x * 2).round() / 2
    if o["equal"]:
        x[:] = 1.25
    if o["masked"] is not None:
        for r in range(B * K):
            x[r, torch.randperm(V, generator=g)[o["left"]:]] = o["masked"]
    if o["spoil"]:
        x[1, 7], x[2, 9], x[5, 1100] = math.nan, math.inf, -math.inf
    x = x.to(o["dtype"]).to(dev)[:, :V]
    scores = (-20 * torch.rand((B, K), generator=g))
    if o["start"]:
        scores[:, 1:] = -math.inf
    lengths = torch.randint(1, 20, (B, K), generator=g, dtype=torch.int32)
    finished = torch.rand((B, K), generator=g) < o["finished"] if o["finished"] else None
    eos = V // 2
    want = select64(x, scores, lengths, finished, eos, o["penalty"])
    r = beam_select(x, scores.to(dev), lengths.to(dev), None if finished is None else finished.to(dev), eos=eos, length_penalty=o["penalty"], lib=lib)
    got = [t.cpu().numpy() for t in (r.scores, r.parents, r.tokens, r.finished, r.lengths)]
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]), (got[1:3], want[1:3])
    assert np.array_equal(got[3], want[3]) and np.array_equal(got[4], want[4])
    # a score: one fp32 rounding, and the logarithm of a sum that is good to 2^-22
    assert np.array_equal(np.isfinite(got[0]), np.isfinite(want[0]))
    fin = np.isfinite(want[0])
    assert (np.abs(got[0] - want[0])[fin] <= np.abs(want[0])[fin] * 2.0 ** -24 + 2.0 ** -22).all()
    bare = beam_select(x, scores.to(dev), lib=lib)
    assert bare.finished is None and bare.lengths is None
    plain = select64(x, scores)
    assert np.array_equal(bare.parents.cpu().numpy(), plain[1]) and np.array_equal(bare.tokens.cpu().numpy(), plain[2])


def check_select_refusals(dev, lib):
    x, s = torch.zeros((6, 50), device=dev), torch.zeros((2, 3), device=dev)
    n, f = torch.ones((2, 3), dtype=torch.int32, device=dev), torch.zeros((2, 3), dtype=torch.bool, device=dev)
    for args, kw, kind in (((x[:5], s), {}, AssertionError), ((x.half(), s), {}, ValueError), ((x, s.double()), {}, ValueError), ((x, s, n.long()), {}, ValueError),
                           ((x, s, n, f), {}, ValueError), ((x, s, n, f), dict(eos=50), ValueError), ((x, s), dict(length_penalty=1.0), ValueError),
                           ((x, s, n), dict(length_penalty=math.nan), ValueError), ((x.t().contiguous().t(), s), {}, ValueError), ((x, s.t().contiguous().t()), {}, ValueError),
                           ((torch.zeros((33, 50), device=dev), torch.zeros((1, 33), device=dev)), {}, NotImplementedError), ((x, s[:, :1].expand(2, 3)), {}, ValueError)):
        with pytest.raises(kind):
            beam_select(*args, lib=lib, **kw)
    assert beam_select(torch.zeros((0, 50), device=dev), torch.zeros((0, 3), device=dev), lib=lib).scores.shape == (0, 3)
    with pytest.raises((ValueError, AssertionError)):
        beam_select(torch.zeros((6, 0), device=dev), s, lib=lib)


def check_reorder(dev, lib, beams):
    g = torch.Generator().manual_seed(beams)
    B = 3
    rows = B * beams
    shapes = [((rows, 7, 33), F32), ((rows, 4), torch.int32), ((rows, 129), BF16), ((rows, 13), torch.uint8), ((rows, 3), torch.bool), ((rows,), torch.int64), ((rows, 0, 5), F32),
              ((rows, 1000), F32)]
    states = [torch.randint(0, 2 if dt == torch.bool else 200, s, generator=g).to(dt) for s, dt in shapes]
    big = torch.randn((rows, 40, 24), generator=g)
    for trial in range(3):
        parents = torch.randint(0, beams, (B, beams), generator=g, dtype=torch.int32)
        if trial == 1:
            parents[0] = torch.arange(beams)                   # nothing moves
            parents[1] = torch.arange(beams).flip(0)           # every row changes places
        if trial == 2:
            parents[2, 0], parents[0, -1] = -1, beams          # no such parent: those rows stay
        at = torch.where((parents >= 0) & (parents < beams), parents.long(), torch.arange(beams)) + beams * torch.arange(B)[:, None]
        mine = [t.clone().to(dev) for t in states]
        pad = big.clone().to(dev)
        view = pad[:, 8:24]                                    # rows apart from one another
        beam_reorder([*mine, view], parents.to(dev), lib=lib)
        for t, m in zip(states, mine):
            assert torch.equal(m.cpu(), t[at.flatten()])
        assert torch.equal(view.cpu(), big[at.flatten()][:, 8:24]) and torch.equal(pad.cpu()[:, :8], big[:, :8]) and torch.equal(pad.cpu()[:, 24:], big[:, 24:])
    many = [torch.full((rows, 1 + i % 3), i, dtype=torch.int16, device=dev) + torch.arange(rows, dtype=torch.int16, device=dev)[:, None] for i in range(101)]
    ref = [t.cpu()[at.flatten()] for t in many]
    beam_reorder(many, parents.to(dev), lib=lib)
    assert all(torch.equal(t.cpu(), r) for t, r in zip(many, ref))


def check_reorder_refusals(dev, lib):
    p = torch.zeros((2, 3), dtype=torch.int32, device=dev)
    t = torch.zeros((6, 8), device=dev)
    for states, parents, kind in (([t, t], p, ValueError), ([t, t[:, 2:6]], p, ValueError), ([t[:5]], p, AssertionError), ([t], p.long(), ValueError), ([t], p[0], ValueError),
                                  ([t.t().contiguous().t()], p, ValueError), ([torch.zeros((33, 2), device=dev)], torch.zeros((1, 33), dtype=torch.int32, device=dev), NotImplementedError),
                                  ([t[:1].expand(6, 8)], p, ValueError)):
        with pytest.raises(kind):
            beam_reorder(states, parents, lib=lib)
    beam_reorder([], p, lib=lib)
    beam_reorder([t[:0]], p[:0], lib=lib)


# ---- the token language models over a cache in 8 bits ---------------------------------------------------------------------------
from moshi_amd.config import GroupedAttentionConfig  # noqa: E402
from moshi_amd.tlm import TokenLM  # noqa: E402
from moshi_amd.weights import random_token_lm_state_dict  # noqa: E402
from oracle.token_lm_oracle import TokenLMOracle  # noqa: E402
from tests import tlm_cases as tc  # noqa: E402


class EightBitOracle(TokenLMOracle):
    """The oracle with grouped attention over a cache in 8 bits, fed in the given portions (the last one repeats)."""

    def __init__(self, state_dict, cfg, codes, cuts):
        super().__init__(state_dict, cfg)
        self.codes, self.cuts = codes, cuts

    def mixer(self, i, h):
        m = self.cfg.layers[i].mixer
        if not isinstance(m, GroupedAttentionConfig):
            return super().mixer(i, h)
        p, T = f"l{i}.mix.", len(h)
        rows = lambda name, heads, n: torch.from_numpy((h @ self.w[p + name].T).reshape(T, heads, n))  # noqa: E731
        q, k, v = rows("q", m.heads, m.dim), rows("k", m.kv_heads, m.dim), rows("v", m.kv_heads, m.vdim)
        pages = T // 64 + 1
        held = [Cache64(self.codes, torch.zeros((pages, m.kv_heads, 64, n), dtype=torch.float64), torch.zeros((pages, m.kv_heads, 4), dtype=torch.float64)) for n in (m.dim, m.vdim)]
        out = torch.zeros((T, m.heads, m.vdim), dtype=torch.float64)
        at, n = 0, 0
        while at < T:
            b = min(T, at + self.cuts[min(n, len(self.cuts) - 1)])
            for cache, x in zip(held, (k, v)):
                cache.append(x[at:b], lambda pos: pos // 64, at)
            keys, vals = [torch.cat([c.values(j) for j in range(pages)], dim=1) for c in held]
            t, pos = torch.arange(64 * pages)[None], torch.arange(at, b)[:, None]
            seen = t <= pos
            if m.window:
                seen &= (pos - t < m.window) | (t < m.keep_first)
            for head in range(m.heads):
                g = head // (m.heads // m.kv_heads)
                s = (q[at:b, head] @ keys[g].T * m.scale).masked_fill(~seen, -math.inf)
                if m.sink:
                    s = torch.cat([s, torch.zeros((b - at, 1), dtype=torch.float64)], dim=1)
                out[at:b, head] = torch.softmax(s, dim=1)[:, :64 * pages] @ vals[g]
            at, n = b, n + 1
        return out.reshape(T, -1).numpy() @ self.w[p + "o"].T


# Beside the models' own: one code of the largest value on the other side of a border, where all of a row's weight is on it
ONE_CODE = {"int8": 1 / 127, "e4m3": 2.0 ** -4}


def check_token_lm(name, dev, lib, dtype, codes, n=90, cut_sets=((90,), (21, 1), (3, 40, 1, 1, 30)), **kw):
    cfg = tc.MECHANISMS[name]
    sd = random_token_lm_state_dict(cfg, seed=5)
    toks = tc.tokens_of(cfg, n)
    for cuts in cut_sets:
        lm = TokenLM(sd, cfg, device=dev, dtype=dtype, lib=lib, kv_cache=codes, **{**dict(max_slots=6, max_tokens=1024), **kw})
        want = EightBitOracle(sd, cfg, codes, cuts).logits(toks)
        assert tc.rel(tc.run_cut(lm, toks, list(cuts)), want) < tc.TOL[dtype] + ONE_CODE[codes], cuts


def check_token_lm_batch(dev, lib, dtype, codes, name="grouped_attention"):
    """Portions beside single tokens, sequences left out of steps, slots taken again: each sequence as if it were alone."""
    cfg = tc.MECHANISMS[name]
    sd = random_token_lm_state_dict(cfg, seed=5)
    lm = TokenLM(sd, cfg, device=dev, dtype=dtype, lib=lib, kv_cache=codes, max_slots=5, max_tokens=2048)
    rng = np.random.default_rng(3)
    for first in (0, 5):
        seqs = [tc.tokens_of(cfg, m, seed=first + i) for i, m in enumerate((131, 1, 64, 40, 66))]
        slots, at, cuts, got = [lm.open() for _ in seqs], [0] * 5, [[] for _ in seqs], [[] for _ in seqs]
        while any(a < len(s) for a, s in zip(at, seqs)):
            entries, who = [], []
            for i in rng.permutation(5):
                left = len(seqs[i]) - at[i]
                if left == 0 or rng.random() < 0.25:
                    continue
                m = min(left, int(rng.choice([1, 1, 2, 5, 17, 64, 70])))
                entries.append((slots[i], seqs[i][at[i]:at[i] + m], list(range(m))))
                who.append((i, m))
                at[i] += m
            if not entries:
                continue
            logits = lm.step(entries).cpu().numpy()
            row = 0
            for i, m in who:
                got[i].append(logits[row:row + m])
                cuts[i].append(m)
                row += m
        for i, s in enumerate(seqs):
            want = EightBitOracle(sd, cfg, codes, cuts[i]).logits(s)
            assert tc.rel(np.concatenate(got[i]), want) < tc.TOL[dtype] + ONE_CODE[codes], (i, cuts[i])
        for s in slots:
            lm.close(s)
        assert lm.free_pages == lm.total_pages


def check_token_lm_refusals(dev, lib):
    cfg = tc.MECHANISMS["mingru"]
    with pytest.raises(NotImplementedError, match="grouped attention"):
        TokenLM(random_token_lm_state_dict(cfg, seed=1), cfg, device=dev, lib=lib, kv_cache="int8")
    with pytest.raises(ValueError):
        TokenLM({}, tc.MECHANISMS["grouped_attention"], device=dev, lib=lib, kv_cache="int4")


# ---- beams --------------------------------------------------------------------------------------------------------------------
def check_token_lm_reorder(name, dev, lib, dtype=F32, codes=None, lengths=((20, 64, 1, 130, 63), (65, 7, 90, 90, 128)), tail=70):
    """Sequences that became copies of others, against sequences that had those tokens from the start: the same batches, so the same bits."""
    cfg = tc.MECHANISMS[name]
    sd = random_token_lm_state_dict(cfg, seed=5)
    beams, parents = 5, [[[3, 1, 1, 0, 3], [2, 2, 2, 2, 2]], [[0, 0, 4, 4, 1], [4, 3, 2, 1, 0]]]
    seqs = [[tc.tokens_of(cfg, n, seed=9 * g + i) for i, n in enumerate(row)] for g, row in enumerate(lengths)]
    a, b = (TokenLM(sd, cfg, device=dev, dtype=dtype, lib=lib, kv_cache=codes, max_slots=11, max_tokens=64 * 60) for _ in range(2))
    a.open()                                               # (slots need not start at the first)
    sa, sb = ([[m.open() for _ in range(beams)] for _ in range(2)] for m in (a, b))
    rng = np.random.default_rng(1)
    for g in range(2):
        for i in range(beams):
            a.step([(sa[g][i], seqs[g][i], [])])
    at = parents[0]
    a.reorder(sa, at)
    for g in range(2):
        for i in range(beams):
            b.step([(sb[g][i], seqs[g][at[g][i]], [])])
    fed = [[[] for _ in range(beams)] for _ in range(2)]

    def step_both():
        toks = rng.integers(0, cfg.vocab, (2, beams)).tolist()
        ya, yb = (m.step([(s[g][i], [toks[g][i]], [0]) for g in range(2) for i in range(beams)]) for m, s in ((a, sa), (b, sb)))
        assert torch.equal(ya, yb)
        for g in range(2):
            for i in range(beams):
                fed[g][i].append(toks[g][i])

    for _ in range(tail):
        step_both()
    assert [[a.position(s) for s in row] for row in sa] == [[b.position(s) for s in row] for row in sb]
    # and again: b's sequences step by step, in batches like the first ones
    a.reorder(sa, parents[1])
    for row in sb:
        for s in row:
            b.close(s)
    sb = [[b.open() for _ in range(beams)] for _ in range(2)]
    src = [[at[g][parents[1][g][i]] for i in range(beams)] for g in range(2)]
    for g in range(2):
        for i in range(beams):
            b.step([(sb[g][i], seqs[g][src[g][i]], [])])
    for n in range(tail):
        b.step([(sb[g][i], [fed[g][parents[1][g][i]][n]], [0]) for g in range(2) for i in range(beams)])
    for _ in range(3):
        step_both()
    a.reorder(sa, [list(range(beams))] * 2)                # nothing moves
    step_both()
    for m, s in ((a, sa), (b, sb)):
        for row in s:
            for slot in row:
                m.close(slot)
        assert m.free_pages == m.total_pages


def check_token_lm_reorder_pool(dev, lib):
    """Shared pages are counted once, given back with their last holder, and a reordering that the pool cannot hold leaves everything as it was."""
    cfg = tc.MECHANISMS["grouped_attention_no_window"]
    sd = random_token_lm_state_dict(cfg, seed=5)
    lm = TokenLM(sd, cfg, device=dev, dtype=F32, lib=lib, max_slots=5, max_tokens=64 * 6)
    s = [lm.open() for _ in range(4)]
    toks = tc.tokens_of(cfg, 200)
    lm.step([(s[0], toks[:130], [])])                      # two full pages and two tokens of a third
    assert lm.free_pages == 3
    lm.reorder([s], [[0, 0, 0, 0]])
    assert lm.free_pages == 0 and [lm.position(x) for x in s] == [130] * 4
    lm.reorder([s], [[1, 0, 3, 3]])                        # partly filled pages change hands: none more is needed
    assert lm.free_pages == 0
    with pytest.raises(BufferError):
        lm.step([(x, toks[130:192 + 1], []) for x in s])   # (a page more each)
    lm.close(s[1])
    assert lm.free_pages == 1
    s[1] = lm.open()
    lm.step([(s[1], [1], [])])
    before = lm.step([(s[0], [5], [0]), (s[2], [5], [0])])
    with pytest.raises(BufferError):
        e = lm.open()
        lm.reorder([[s[0], e]], [[0, 0]])
    assert lm.free_pages == 0 and lm.position(e) == 0 and lm.position(s[0]) == 131
    y = lm.step([(s[0], [9], [0]), (s[2], [9], [0])])
    assert torch.equal(before[0], before[1]) and torch.equal(y[0], y[1])
    lm.close(s[0])                                         # its own page alone: the others still hold the first two
    assert lm.free_pages == 1
    for x in (s[1], s[2], s[3], e):
        lm.close(x)
    assert lm.free_pages == 6
    for slots, parents, kind in (([[0]], [[0]], Exception), ([[0, 0]], [[0, 1]], Exception)):
        with pytest.raises(kind):
            lm.reorder(slots, parents)                     # no open sequence
    s = [lm.open() for _ in range(4)]
    for slots, parents in (([s], [[0, 1, 2, 4]]), ([s], [[0, 1, 2, -1]]), ([s[:2] + s[:2]], [[0, 0, 0, 0]]), ([s], [[0]]), ([s, s[:3]], [[0] * 4] * 2)):
        with pytest.raises(ValueError):
            lm.reorder(slots, parents)
    lm.reorder([], [])


class _Beams64:
    """The search in 64 bits, every sequence computed anew; `gap`: the least difference of rank between what a step kept and what it left."""

    def __init__(self, orc, prompt, beams, steps, eos, alpha):
        self.gap = math.inf
        held = [(0.0, [], False)]
        rank = lambda c: c[0] / len(c[1]) ** alpha  # noqa: E731
        for _ in range(steps):
            new = []
            for score, toks, done in held:
                if done:
                    new.append((score, toks, True))
                    continue
                p = self.log_probs(orc, prompt, toks)
                new += [(score + p[t], toks + [t], t == eos) for t in range(len(p))]
            new.sort(key=rank, reverse=True)
            if len(new) > beams:
                self.gap = min(self.gap, rank(new[beams - 1]) - rank(new[beams]))
            held = new[:beams]
            if all(d for _, _, d in held):
                break
        self.held = held

    @staticmethod
    def log_probs(orc, prompt, toks):
        y = np.asarray(orc.logits(prompt + toks)[-1], np.float64)
        return y - y.max() - np.log(np.exp(y - y.max()).sum())


def check_beam_search(dev, lib, name, dtype=F32, codes=None, beams=4, steps=9, alpha=0.0, room=None, **kw):
    cfg = tc.MECHANISMS[name]
    sd = random_token_lm_state_dict(cfg, seed=5)
    cuts = (16, 1)
    orc = EightBitOracle(sd, cfg, codes, cuts) if codes else TokenLMOracle(sd, cfg)
    prompts = [tc.tokens_of(cfg, n, seed=n) for n in (16, 16, 16)] if codes else [tc.tokens_of(cfg, n, seed=n) for n in (5, 60, 1)]
    eos = int(np.argmax(orc.logits(prompts[0] + [int(np.argmax(orc.logits(prompts[0])[-1]))])[-1]))      # the second token of the first one's likeliest
    lm = TokenLM(sd, cfg, device=dev, dtype=dtype, lib=lib, kv_cache=codes, **{**dict(max_slots=3 * beams, max_tokens=64 * 2 * 3 * beams), **kw})
    got = beam_search(lm, prompts, beams, steps, eos, alpha, **({} if codes else {"step_tokens": 14}))
    assert lm.free_pages == lm.total_pages and lm.free_slots == lm.max_slots
    same = 0
    for prompt, hyps in zip(prompts, got):
        want = _Beams64(orc, prompt, beams, steps, eos, alpha)
        # a logit is off by at most its row's RMS error times sqrt(vocab); log p by twice that (itself and the sum), a score by that per token
        rms = math.sqrt(float(np.mean(np.square(orc.logits(prompt)))))
        off = (tc.TOL[dtype] + (ONE_CODE[codes] if codes else 0)) * rms * math.sqrt(cfg.vocab) * 2
        assert len(hyps) == beams
        ranks = [h.score / len(h.tokens) ** alpha for h in hyps]
        assert ranks == sorted(ranks, reverse=True)
        for h in hyps:
            assert 1 <= len(h.tokens) <= steps and eos not in h.tokens[:-1] and (len(h.tokens) == steps or h.tokens[-1] == eos)
            p = sum(_Beams64.log_probs(orc, prompt, h.tokens[:i])[t] for i, t in enumerate(h.tokens))
            assert abs(h.score - p) <= off * len(h.tokens)
        if want.gap > 2 * off * steps:
            assert sorted(h.tokens for h in hyps) == sorted(t for _, t, _ in want.held)
            same += 1
    return same


def check_beam_search_of_one(dev, lib, name="mixed"):
    """One beam is greedy decoding; more requests than fit wait for the first ones' slots and pages."""
    from moshi_amd.token_batcher import TokenBatcher
    cfg = tc.MECHANISMS[name]
    lm = TokenLM(random_token_lm_state_dict(cfg, seed=5), cfg, device=dev, dtype=F32, lib=lib, max_slots=2, max_tokens=64 * 3)
    prompts = [tc.tokens_of(cfg, n, seed=n) for n in (3, 70, 64, 9)]
    want = TokenBatcher(lm).generate(prompts, 6)
    assert [h[0].tokens for h in beam_search(lm, prompts, 1, 6)] == want
    with pytest.raises(BufferError):
        beam_search(lm, prompts, 3, 6)
    with pytest.raises(BufferError):
        beam_search(lm, [tc.tokens_of(cfg, 150)], 2, 6)
    for bad in (([[]], 1, 1), ([[1]], 0, 1), ([[1]], 1, 0), ([[cfg.vocab]], 1, 1), ([[-1]], 1, 1), ([[1]], 1, 1, cfg.vocab)):
        with pytest.raises(ValueError):
            beam_search(lm, *bad)
    assert beam_search(lm, [], 2, 4) == [] and lm.free_slots == 2 and lm.free_pages == lm.total_pages


# ---- calls that the documentation allows, at its edges ----------------------------------------------------------------------------
def _filled(dev, lib, pages, tokens, codes="int8", dim=32):
    """A cache of one head with one sequence's tokens in pages 0, 1, ..; the values it holds, in 64 bits."""
    g = torch.Generator().manual_seed(4)
    cache = PagedKVCache.empty(pages, 1, dim, codes=codes, device=dev, lib=lib)
    k, v = [torch.randn((tokens, 1, dim), generator=g).to(dev) for _ in range(2)]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    cache.append(k, v, table, i32(0), i32(0, tokens))
    held = [x[:, 0].double().cpu() for x in cache.read(table, i32(0), i32(0, tokens), tokens=tokens)]
    return cache, table, held, i32, g


def check_position_past_the_table(dev, lib, codes="int8"):
    """Far behind the last page that the table names, the kept first tokens (more of them than it names) are all there is to see."""
    cache, table, (k, v), i32, g = _filled(dev, lib, 8, 512, codes)
    for n in (1, 20):
        q = torch.randn((n, 2, 32), generator=g).to(dev)
        for keep in (2000, 100):
            got = cache.attend(q, table, i32(10000), None if n == 1 else i32(0, n), window=64, keep_first=keep)
            s = torch.einsum("rhd,td->rht", q.double().cpu(), k[:keep]) * 32 ** -0.5
            want = torch.softmax(s, dim=-1) @ v[:keep]
            # operands of 22 bits, sums in 32: as for the other fp32 cases
            assert torch.allclose(got.double().cpu(), want, rtol=2.0 ** -16, atol=2.0 ** -18), (n, keep)
        assert not cache.attend(q, table, i32(10000), None if n == 1 else i32(0, n), window=64).any()


def check_rows_in_no_order(dev, lib):
    """Row starts that do not ascend are no sequences; whatever becomes of those rows, the memory beside the tensors stays as it is."""
    cache, table, _, i32, g = _filled(dev, lib, 8, 300)
    tables = table.expand(4, 8).contiguous()
    for rows in ((0, 40, 10, 60, 25), (60, 0, 60, 0, 60), (50, 40, 30, 20, 10), (-5, 70, 1 << 30, -(1 << 30), 3)):
        q = torch.full((60 + 128, 2, 32), 7.0, device=dev)
        out = torch.full((60 + 128, 2, 32), 7.0, device=dev)
        q[64:124] = torch.randn((60, 2, 32), generator=g).to(dev)
        cache.attend(q[64:124], tables, i32(100, 200, 299, 0), i32(*rows), out=out[64:124])
        assert (out[:64] == 7).all() and (out[124:] == 7).all(), rows
        before = [t.clone() for t in (cache.k_scale, cache.v_scale)]
        big = torch.full((60 + 128, 1, 32), 1e30, device=dev)                         # (what lies beside the rows would show in a scale)
        big[64:124] = 0.01
        cache.append(big[64:124], big[64:124], tables, i32(100, 200, 299, 0), i32(*rows))
        assert max(float(t.max()) for t in (cache.k_scale, cache.v_scale)) <= max(float(t.max()) for t in before), rows
        kv = cache.read(tables, i32(100, 200, 299, 0), i32(*rows), tokens=60)
        assert kv[0].shape == (60, 1, 32)


# ---- value scales of a sequence's blocks far apart -------------------------------------------------------------------------------------
def _ramp(first, last):
    return lambda t: 2.0 ** (first + (last - first) * t)


# mags: of the values, levels: scores (natural logarithms), both functions of the place 0 .. 1 in the sequence; nothing: pages that the caller's own scales say
# hold zeros; negative: pages whose scales are negative
FAR = {
    "zeros_in_a_page": dict(c=Case([40], [24], kv_heads=1, rep=2, dim=32, vdim=32), mags=lambda t: 0.0 if t < 0.5 else 1.0, levels=lambda t: 5.0 if t < 0.5 else 0.0),
    "zeros_first": dict(c=Case([639], [1], single=True, kv_heads=1, rep=2, dim=32, vdim=32), mags=lambda t: 0.0 if t < 0.5 else 1.0, levels=lambda t: 3.0 if t < 0.5 else 0.0),
    "zeros_last": dict(c=Case([600], [40], kv_heads=1, rep=2, dim=32, vdim=32, codes="e4m3", dtype=F32), mags=lambda t: 1.0 if t < 0.5 else 0.0, levels=lambda t: 0.0 if t < 0.5 else 6.0),
    "zeros_alone": dict(c=Case([90], [40], kv_heads=1, rep=2, dim=32, vdim=32), mags=lambda t: 0.0, levels=lambda t: 0.0),
    "scale_of_zero": dict(c=Case([127], [1], single=True, kv_heads=2, rep=2, dim=32, vdim=32), mags=lambda t: 1.0, levels=lambda t: 1.0 if t < 0.5 else 0.0, nothing=(0,)),
    "scale_of_zero_portion": dict(c=Case([100], [60], kv_heads=2, rep=2, dim=32, vdim=48, codes="e4m3"), mags=lambda t: 1.0, levels=lambda t: 2.0 if t < 0.4 else 0.0, nothing=(0, 2)),
    "scale_of_zero_fp32_sink": dict(c=Case([300], [1], single=True, kv_heads=1, rep=3, dim=32, vdim=32, dtype=F32, sink=True), mags=lambda t: 1.0, levels=lambda t: 0.0, nothing=(1, 3)),
    "large_behind_likelier_zeros": dict(c=Case([639], [1], single=True, kv_heads=1, rep=2, dim=32, vdim=32, dtype=F32), mags=lambda t: 0.0 if t < 0.5 else 2.0 ** 20,
                                        levels=lambda t: 9.0 if t < 0.5 else 0.0),
    "large_behind_likelier_zeros_portion": dict(c=Case([600], [40], kv_heads=1, rep=2, dim=32, vdim=32, dtype=F32, codes="e4m3"), mags=lambda t: 0.0 if t < 0.5 else 2.0 ** 40,
                                                levels=lambda t: 9.0 if t < 0.5 else 0.0),
    "growing": dict(c=Case([1299], [1], single=True, kv_heads=1, rep=2, dim=32, vdim=32, dtype=F32), mags=_ramp(-110, 110), levels=lambda t: 0.0),
    "growing_portion": dict(c=Case([1270], [30], kv_heads=1, rep=2, dim=32, vdim=32, sink=True), mags=_ramp(-110, 110), levels=lambda t: 0.0),
    "shrinking": dict(c=Case([1299], [1], single=True, kv_heads=1, rep=2, dim=32, vdim=32, dtype=F32, codes="e4m3"), mags=_ramp(110, -110), levels=lambda t: 0.0),
    "shrinking_against_scores": dict(c=Case([1270], [30], kv_heads=1, rep=2, dim=32, vdim=32, dtype=F32), mags=_ramp(60, -60), levels=lambda t: 70 * t),
    "negative_scales": dict(c=Case([200], [1], single=True, kv_heads=2, rep=2, dim=32, vdim=32), mags=lambda t: 1.0, levels=lambda t: 0.0, negative=(0, 2)),
    "negative_scales_portion": dict(c=Case([200], [30], kv_heads=2, rep=2, dim=32, vdim=32, codes="e4m3", dtype=F32), mags=lambda t: 4.0, levels=lambda t: t, negative=(1,)),
}
# pages that are not split, so that a sum runs over many of them (long on the simulator)
FAR_LARGE = {
    "zeros_below_unsplit": dict(c=Case([620], [20], kv_heads=400, rep=1, dim=16, vdim=16), mags=lambda t: 0.0 if t < 0.8 else 1.0,
                                levels=lambda t: 5.6 * math.log(2) if 0.1 <= t < 0.8 else 0.0),
    "large_behind_likelier_zeros_unsplit": dict(c=Case([620], [20], kv_heads=400, rep=1, dim=16, vdim=16), mags=lambda t: 0.0 if t < 0.5 else 2.0 ** 60, levels=lambda t: 8.0 if t < 0.5 else 0.0),
}


def check_blocks_far_apart(name, dev, lib):
    """Blocks of zeros, of values 2^220 apart, of scales of zero or below it: no sum overflows and none is lost, whichever kernel, split or not."""
    o = {**FAR, **FAR_LARGE}[name]
    c, g = o["c"], torch.Generator().manual_seed(len(name))
    cache, q, _, _, args = build(c, dev, lib, fill=False)
    n = c.past[0] + c.rows[0]
    at = torch.arange(n) / n
    mags, levels = [torch.tensor([o[f](float(t)) for t in at], dtype=torch.float64).float() for f in ("mags", "levels")]
    keys = 0.1 * torch.randn((n, c.kv_heads, c.dim), generator=g)
    keys[..., 0] = levels[:, None]
    vals = torch.randn((n, c.kv_heads, c.vdim), generator=g) * mags[:, None, None]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cache.append(keys.to(dev), vals.to(dev), args[0], i32(0), i32(0, n))
    table = args[0][0].tolist()
    for i in o.get("nothing", ()):
        cache.v_scale[table[i]] = 0.0
    for i in o.get("negative", ()):
        cache.v_scale[table[i]] *= -1.0
    q = torch.randn(q.shape, generator=g) * 0.1
    q[..., 0] = c.dim ** 0.5                               # (times the softmax's factor: one)
    q = q.to(c.dtype).to(dev)
    got = cache.attend(q, *args, sink=c.sink).cpu().double()
    want, size, top = attend64(c, cache, q, args)
    h = 2.0 ** -12 if c.dtype == BF16 else 2.0 ** -23      # (check_attend)
    off = 2 * size * (h + c.dim * 2.0 ** -24) + h + 2.0 ** -20
    limit = off[:, None, None].double() * top + want.abs() * (torch.finfo(c.dtype).eps / 2)
    assert got.isfinite().all() and ((got - want).abs() <= limit).all(), float(((got - want).abs() / limit).max())


def check_select_penalties(dev, lib):
    """Length penalties at the ends of what is taken, with beams at -infinity and few candidates that are not: as in 64 bits.  Beyond: refused."""
    g = torch.Generator().manual_seed(2)
    B, K, V = 3, 4, 700
    for bad in (16.001, -16.001, 110.0, 300.0, -300.0, math.inf, -math.inf, math.nan):
        with pytest.raises(ValueError, match="penalty"):
            beam_select(torch.zeros((K, V), device=dev), torch.zeros((1, K), device=dev), torch.ones((1, K), dtype=torch.int32, device=dev), length_penalty=bad, lib=lib)
    for penalty in (16.0, -16.0, 1.0):
        for longest in (30, 2 ** 31 - 2):
            x = torch.full((B * K, V), -math.inf)
            x[:, :3] = torch.randn((B * K, 3), generator=g)
            x[2 * K:] = torch.randn((K, V), generator=g)
            x[4:6] = -math.inf
            scores = -20 * torch.rand((B, K), generator=g)
            scores[0, 1:] = -math.inf                          # three candidates for four places
            scores[2, 2] = 0.0
            lengths = torch.randint(longest // 2, longest, (B, K), generator=g, dtype=torch.int32)
            finished = torch.zeros((B, K), dtype=torch.bool)
            finished[1, 2:], finished[2, :2] = True, True
            scores[1, 3] = -math.inf
            want = select64(x, scores, lengths, finished, 2, penalty)
            r = beam_select(x.to(dev), scores.to(dev), lengths.to(dev), finished.to(dev), eos=2, length_penalty=penalty, lib=lib)
            got = [t.cpu().numpy() for t in (r.scores, r.parents, r.tokens, r.finished, r.lengths)]
            assert all(np.array_equal(a, b) for a, b in zip(got[1:], want[1:])), (penalty, longest, got, want)
            fin = np.isfinite(want[0])
            assert np.array_equal(np.isfinite(got[0]), fin) and (np.abs(got[0] - want[0])[fin] <= np.abs(want[0])[fin] * 2.0 ** -24 + 2.0 ** -22).all()


def check_keeps_everything(dev, lib, codes="int8"):
    """A window that keeps more first positions than there can be, and one longer than any sequence, hide nothing."""
    cache, table, _, i32, g = _filled(dev, lib, 8, 500, codes)
    for n in (1, 20):
        q = torch.randn((n, 2, 32), generator=g).to(dev)
        args = (q, table, i32(500 - n), None if n == 1 else i32(0, n))
        want = cache.attend(*args)
        assert want.any()
        for window, keep in ((10, 2 ** 31 - 64), (10, 2 ** 31 - 63), (1, 2 ** 31 - 1), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1)):
            # the same keys in the same order, whatever the splits: sums in another order at most
            assert torch.allclose(cache.attend(*args, window=window, keep_first=keep), want, rtol=2.0 ** -16, atol=2.0 ** -18), (n, window, keep)


def check_token_lm_keeps_everything(dev, lib, codes):
    from dataclasses import replace
    cfg = tc.MECHANISMS["grouped_attention_no_window"]
    sd, toks, out = random_token_lm_state_dict(cfg, seed=5), tc.tokens_of(cfg, 150), []
    for window, keep in ((0, 0), (9, 2 ** 31 - 1), (9, 2 ** 31 - 63), (2 ** 31 - 1, 2 ** 31 - 1)):
        layers = [replace(x, mixer=replace(x.mixer, window=window, keep_first=keep)) if isinstance(x.mixer, GroupedAttentionConfig) else x for x in cfg.layers]
        lm = TokenLM(sd, replace(cfg, layers=layers), device=dev, dtype=F32, lib=lib, kv_cache=codes, max_slots=2, max_tokens=256)
        out.append(tc.run_cut(lm, toks, [100, 1]))
        assert tc.rel(out[-1], out[0]) < 1e-5, (window, keep)      # fp32 sums in another order


from contextlib import contextmanager  # noqa: E402


@contextmanager
def _new_memory_is_nan():
    """torch.empty and its like give NaN (the largest integers), not what the memory happens to hold."""
    torch.use_deterministic_algorithms(True, warn_only=True)
    try:
        yield
    finally:
        torch.use_deterministic_algorithms(False)


# `first`: rows before the first sequence; a negative past: passed over, with as many rows as it brings
RESTS = {
    "single_tokens": (Case([-1, 4, -7, 70, -2], [1] * 5, single=True, rep=20, kv_heads=1), 0),
    "single_tokens_fp32": (Case([-1, -3], [1] * 2, single=True, dtype=F32, codes="e4m3", vdim=48), 0),
    "behind": (Case([5, 12], [2, 20], extra_rows=5, rep=4), 0),
    "before_and_behind": (Case([70, 3], [30, 1], extra_rows=3, dtype=F32, dim=32, vdim=80), 4),
    "portions_passed_over": (Case([-1, 40, -64, 9, -5], [18, 3, 1, 25, 7], extra_rows=2, rep=3, codes="e4m3"), 1),
    "all_passed_over": (Case([-1, -1], [18, 3], extra_rows=2), 3),
}


def check_rest(name, dev, lib):
    """Rows that no sequence brings: zeros in new tensors, in `out` as they were; the others the same either way."""
    c, first = RESTS[name]
    c = Case(**{**c.__dict__, "extra_rows": c.extra_rows + first})
    cache, q, k, v, args = build(c, dev, lib)
    if not c.single:
        args = (args[0], args[1], args[2] + first)
    cache.append(k, v, *args)
    brought = torch.zeros(c.total, dtype=torch.bool)
    for e, p, n, row in sequences(c):
        brought[row + first:row + first + n] = p >= 0
    held = torch.full((c.total, c.kv_heads * c.rep, c.vdim), 7.0, dtype=c.dtype, device=dev)
    cache.attend(q, *args, out=held)
    with _new_memory_is_nan():
        fresh = cache.attend(q, *args)
        got = cache.read(*args, tokens=c.total, dtype=c.dtype)
    held, fresh, got = held.cpu(), fresh.cpu(), [t.cpu() for t in got]
    assert (held[~brought] == 7).all() and (fresh[~brought] == 0).all() and torch.equal(held[brought], fresh[brought]) and fresh[brought].isfinite().all()
    for t in got:
        assert (t[~brought] == 0).all() and t[brought].isfinite().all() and (t[brought] != 0).flatten(1).any(dim=1).all()
    with _new_memory_is_nan():                                # no sequence at all
        none = (args[0][:0], args[1][:0], torch.zeros(1, dtype=torch.int32, device=dev))
        assert not cache.attend(q, *none).any() and not any(t.any() for t in cache.read(*none, tokens=c.total))
    held = torch.full_like(fresh, 7.0).to(dev)
    assert (cache.attend(q, *none, out=held) == 7).all()


def check_flags(dev, lib):
    import ctypes as C
    from moshi_amd import _capi
    cache, table, _, i32, g = _filled(dev, lib, 2, 70)
    pos, q = i32(69), torch.randn((1, 2, 32), generator=g).to(dev)
    s, out = _capi.KVSeqs(1, 1, None, pos.data_ptr(), table.data_ptr(), 2), torch.zeros_like(q)
    for flags, status in ((0, 0), (1, 0), (2, 0), (3, 0), (4, _capi.MMI_ERR_INVALID), (-1, _capi.MMI_ERR_INVALID)):
        need = lib.mmi_kv_attend_workspace(C.byref(cache._desc), C.byref(s), 2, 0, 0)
        work = torch.empty(max(1, need), dtype=torch.uint8, device=dev)
        assert lib.mmi_kv_attend(C.byref(cache._desc), C.byref(s), _capi.MMI_F32, 2, q.data_ptr(), 64, 32, out.data_ptr(), 64, 32, 0.1, 0, 0, flags, work.data_ptr(), need,
                                 _capi.stream_ptr(out.device)) == status


def check_reorder_views(dev, lib):
    """Views of one buffer whose rows lie between one another's move like tensors of their own; views that share a byte, and parents among the rows, are refused."""
    g = torch.Generator().manual_seed(6)
    parents = torch.tensor([[2, 0, 1, 1], [3, 3, 0, 2]], dtype=torch.int32)
    at = parents.long().flatten() + torch.tensor([0] * 4 + [4] * 4)
    kv = torch.randn((8, 2, 3, 8), generator=g)
    mine = kv.clone().to(dev)
    beam_reorder([mine[:, 0], mine[:, 1]], parents.to(dev), lib=lib)
    assert torch.equal(mine.cpu(), kv[at])
    wide = torch.randint(0, 200, (8, 100), generator=g, dtype=torch.uint8)
    mine, more = wide.clone().to(dev), kv.clone().to(dev)
    beam_reorder([mine[:, 60:], more, mine[:, :7], mine[:, 7:20], mine[:, 33:34]], parents.to(dev), lib=lib)
    want = wide.clone()
    for part in (slice(60, 100), slice(0, 20), slice(33, 34)):
        want[:, part] = wide[at][:, part]
    assert torch.equal(mine.cpu(), want) and torch.equal(more.cpu(), kv[at])
    # a buffer of rows that a second one begins inside, whole rows later: apart only where the parts are
    flat = torch.zeros(480, dtype=torch.int32, device=dev)
    rows = lambda first, n, step=40: torch.as_strided(flat, (8, n), (step, 1), first)  # noqa: E731
    beam_reorder([rows(0, 10), rows(90, 10), rows(20, 10)], parents.to(dev), lib=lib)
    for views in ([rows(0, 10), rows(9, 5)], [rows(0, 10), rows(85, 10)], [rows(0, 10), rows(115, 10)], [rows(0, 10), rows(35, 6)], [rows(0, 10), rows(20, 10), rows(25, 3)],
                  [rows(0, 10), rows(20, 4, 41)], [rows(5, 10), rows(0, 6)]):
        before = flat.clone()
        with pytest.raises(ValueError, match="share"):
            beam_reorder(views, parents.to(dev), lib=lib)
        assert torch.equal(before, flat)
    p = flat[40 * 3 + 12:40 * 3 + 20].view(2, 4)               # parents between rows: nobody's
    p.copy_(parents)
    beam_reorder([rows(0, 12), rows(20, 20)], p, lib=lib)
    assert torch.equal(p.cpu(), parents)
    for views in ([rows(0, 13)], [rows(19, 4)], [flat[:320].view(8, 40)], [rows(20, 10), rows(12, 1)]):
        with pytest.raises(ValueError, match="share"):
            beam_reorder(views, p, lib=lib)
    # rows without a byte share nothing; one row of one tensor may have any distance to its next
    beam_reorder([flat[:80].view(8, 10), flat[:80].view(8, 10)[:, :0]], parents.to(dev), lib=lib)
    # more tensors than the entry takes: refused before any of them is looked at
    import ctypes as C
    from moshi_amd import _capi
    place = _capi.LaunchOn(torch.device(dev, 0) if dev == "cuda" else torch.device(dev))
    one = (C.c_int64 * 1)(flat.data_ptr())
    assert place.call(lib.mmi_beam_reorder, (1 << 16) + 1, one, one, one, 2, 4, p.data_ptr()) == _capi.MMI_ERR_SHAPE
    assert place.call(lib.mmi_beam_reorder, 1, one, (C.c_int64 * 1)(1 << 60), (C.c_int64 * 1)(4), 2, 4, p.data_ptr()) == _capi.MMI_ERR_SHAPE


def check_output_rows(dev, lib):
    """Outputs whose rows or heads share memory are refused; rows within heads, and gaps, are taken."""
    cache, table, _, i32, g = _filled(dev, lib, 2, 70)
    q = torch.randn((3, 2, 32), generator=g).to(dev)
    args = (q, table, i32(67), i32(0, 3))
    want = cache.attend(*args)
    flat = torch.full((400,), 7.0, device=dev)
    view = lambda row, head: torch.as_strided(flat, (3, 2, 32), (row, head, 1))  # noqa: E731
    for row, head in ((64, 32), (32, 96), (32, 100), (100, 36), (80, 48), (96, 64), (64, 200)):
        flat.fill_(7.0)
        out = view(row, head)
        assert cache.attend(*args, out=out) is out and torch.equal(out, want), (row, head)
        out.fill_(7.0)
        assert (flat == 7).all()
    for row, head in ((0, 32), (32, 0), (64, 0), (32, 32), (60, 32), (64, 28), (28, 200), (90, 64), (48, 32)):
        with pytest.raises(ValueError, match="share"):
            cache.attend(*args, out=view(row, head))
    assert (flat == 7).all()
    one = (q[:1], table, i32(67))
    out = view(0, 32)[:1]
    assert torch.equal(cache.attend(*one, out=out), cache.attend(*one))      # (a row alone has no distance)


def check_wide_integers(dev, lib):
    """Integers beyond 32 bits mean what they say: windows are no shorter for it, and an end token is outside the vocabulary."""
    cache, table, _, i32, g = _filled(dev, lib, 2, 70)
    q = torch.randn((1, 2, 32), generator=g).to(dev)
    want = cache.attend(q, table, i32(69))
    for kw in (dict(window=2 ** 31), dict(window=2 ** 32 + 3), dict(window=2 ** 63), dict(window=3, keep_first=2 ** 31), dict(window=3, keep_first=2 ** 32 + 1)):
        assert torch.allclose(cache.attend(q, table, i32(69), **kw), want, rtol=2.0 ** -16, atol=2.0 ** -18), kw
    x, s = torch.zeros((3, 50), device=dev), torch.zeros((1, 3), device=dev)
    for eos in (50, 2 ** 32 + 3, 2 ** 63):
        with pytest.raises(ValueError, match="end token"):
            beam_select(x, s, eos=eos, lib=lib)
    assert beam_select(x, s, eos=49, lib=lib).finished.shape == (1, 3) and beam_select(x, s, eos=-5, lib=lib).finished is None


# ---- the search's choices, whatever the model's rounding -------------------------------------------------------------------------------
def _search64(lm, prompts, beams, steps, eos, alpha, step_tokens):
    """Beam search that ranks in 64 bits what the model says of sequences fed from their start, in slots of their own for every step: same batches, no reordering."""
    from moshi_amd.beam import _prefill
    R = len(prompts)
    scores = torch.full((R, beams), -math.inf)
    scores[:, 0] = 0.0
    lengths, finished = torch.zeros((R, beams), dtype=torch.int32), torch.zeros((R, beams), dtype=torch.bool)
    paths, live, was_live = [[[] for _ in range(beams)] for _ in range(R)], list(range(R)), []
    for n in range(steps):
        slots = [[lm.open() for _ in range(beams)] for _ in range(R)]
        for i in range(beams):                             # (a beam at a time: the same portions as where one sequence stands for all)
            first = _prefill(lm, prompts, [s[i] for s in slots], step_tokens).cpu()
        logits = first.repeat_interleave(beams, dim=0).view(R, beams, -1)
        for k, who in enumerate(was_live):
            y = lm.step([(slots[r][i], [paths[r][i][k]], [0]) for r in who for i in range(beams)]).cpu().view(len(who), beams, -1)
            for at, r in enumerate(who):
                logits[r] = y[at]
        for row in slots:
            for s in row:
                lm.close(s)
        total, parents, tokens, fin, lens = select64(logits[live].flatten(0, 1), scores[live], lengths[live], finished[live], eos, alpha)
        for at, r in enumerate(live):
            paths[r] = [paths[r][int(p)] + [int(t)] for p, t in zip(parents[at], tokens[at])]
            scores[r], lengths[r], finished[r] = torch.from_numpy(total[at]).float(), torch.from_numpy(lens[at]), torch.from_numpy(fin[at])
        live = [r for r in live if not finished[r].all()]
        if not live:
            break
        was_live.append(list(live))
    return [[(paths[r][i][:int(lengths[r, i])], float(scores[r, i])) for i in range(beams) if scores[r, i] > -math.inf] for r in range(R)]


def check_beam_search_choices(dev, lib, name, dtype=F32, codes=None, beams=4, steps=7, alpha=0.0):
    """Every hypothesis, token by token, is the one that the model's own logits lead to."""
    cfg = tc.MECHANISMS[name]
    sd = random_token_lm_state_dict(cfg, seed=5)
    prompts = [tc.tokens_of(cfg, n, seed=n) for n in (5, 61, 16)]
    lm = TokenLM(sd, cfg, device=dev, dtype=dtype, lib=lib, kv_cache=codes, max_slots=3 * beams, max_tokens=64 * 3 * 3 * beams)
    probe = beam_search(lm, prompts, beams, steps, -1, alpha, step_tokens=14)
    assert all(len(set(tuple(h.tokens) for h in hyps)) == beams for hyps in probe)
    for eos in (-1, probe[0][0].tokens[1], probe[1][-1].tokens[2]):      # none; tokens that beams end with early, all of a request's perhaps
        got = beam_search(lm, prompts, beams, steps, eos, alpha, step_tokens=14)
        want = _search64(lm, prompts, beams, steps, eos, alpha, 14)
        assert [[h.tokens for h in hyps] for hyps in got] == [[t for t, _ in hyps] for hyps in want], eos
        # a score: a rounding and the error of a sum's logarithm for every token
        for a, b in zip([h.score for hyps in got for h in hyps], [s for hyps in want for _, s in hyps]):
            assert abs(a - b) <= steps * (abs(b) * 2.0 ** -24 + 2.0 ** -22)
    for bad in (16.5, -17.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="penalty"):
            beam_search(lm, prompts, beams, steps, -1, bad)
    assert lm.free_pages == lm.total_pages and lm.free_slots == lm.max_slots


def check_long_tables(dev, lib):
    """Page tables with more entries than there are positions: no more splits, whose first pages would leave 31 bits."""
    import ctypes as C
    from moshi_amd import _capi
    cache, _, _, i32, _ = _filled(dev, lib, 2, 70)
    here = i32(0, 1)
    for row0 in (None, here.data_ptr()):
        need = [lib.mmi_kv_attend_workspace(C.byref(cache._desc), C.byref(_capi.KVSeqs(1, 1, row0, here.data_ptr(), here.data_ptr(), ld)), 2, 0, 0)
                for ld in (1 << 25, (1 << 25) + 1, 1 << 30, (1 << 31) - 1)]
        assert need[0] > 0 and need == [need[0]] * 4, need


def check_wide_negative_integers(dev, lib):
    """Below 32 bits too: a negative window is none, and no token ends a beam."""
    cache, table, _, i32, g = _filled(dev, lib, 2, 70)
    q = torch.randn((1, 2, 32), generator=g).to(dev)
    for kw in (dict(window=-2 ** 32), dict(window=-2 ** 32 + 3), dict(window=3, keep_first=-2 ** 32), dict(keep_first=-2 ** 63)):
        with pytest.raises(ValueError):
            cache.attend(q, table, i32(69), **kw)
    x, s = torch.zeros((3, 50), device=dev), torch.zeros((1, 3), device=dev)
    n, f = torch.ones((1, 3), dtype=torch.int32, device=dev), torch.ones((1, 3), dtype=torch.bool, device=dev)
    with pytest.raises(ValueError):                        # (finished beams need an end token)
        beam_select(x, s, n, f, eos=-2 ** 32 + 5, lib=lib)
    assert beam_select(x, s, n, eos=-2 ** 32 + 5, lib=lib).finished is None


def check_reorder_of_too_long_rows(dev, lib):
    """A row beyond what a launch takes is refused before the tensors in front of it have moved."""
    import ctypes as C
    from moshi_amd import _capi
    place = _capi.LaunchOn(torch.device(dev, 0) if dev == "cuda" else torch.device(dev))
    states = [torch.arange(8, dtype=torch.int32, device=dev).view(4, 2) + 100 * i for i in range(60)]
    before, parents = [t.clone() for t in states], torch.tensor([[3, 2, 1, 0]], dtype=torch.int32, device=dev)
    at = [t.data_ptr() for t in states] + [1 << 44]        # (never read: the lengths are refused)
    ints = lambda x: (C.c_int64 * len(x))(*x)  # noqa: E731
    for size in ((1 << 30) + 1, 16 << 30):
        lists = [ints(x) for x in (at, [8] * 60 + [size], [8] * 60 + [size])]
        assert place.call(lib.mmi_beam_reorder, 61, *lists, 1, 4, parents.data_ptr()) == _capi.MMI_ERR_SHAPE
        assert all(torch.equal(a, b) for a, b in zip(states, before))
