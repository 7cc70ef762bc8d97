"""`PagedKVCache` - keys and values of token sequences in 8 bits, in pages of 64 tokens, and the attention over them (libmoshi_tlm.so,
include/moshi_tlm.h).

    cache = PagedKVCache.empty(pages=1024, kv_heads=8, dim=128, codes="int8", rot_dim=128, rot_base=1e4)
    cache.append(k, v, table, positions, rows)                # rotate, round to 8 bits, write
    out = cache.attend(q, table, positions, rows, window=1024, keep_first=4)

Which page holds what is the caller's: `table` [sequences, pages of a sequence] int32 names them, `positions` [sequences] int32 says where the
sequence's first row of this call stands, and `rows` [sequences + 1] int32 where its rows lie in the tensors (None: one row each, a decoding
step).  All three are device tensors and are read when the kernels run, so a captured graph replays with what they hold then.  A page
number outside the cache stands for no page: rows that belong there are not written, and nothing is seen of it.  A sequence at a negative
position is passed over: an unused place of a batch.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch

from . import _capi

PAGE_TOKENS, BLOCK_TOKENS = 64, 16
_LONGEST = 2 ** 31 - 1                   # no sequence has more positions
_SINK, _ZERO_REST, _SINK_ZERO_REST = _capi.MMI_KV_SINK, _capi.MMI_KV_ZERO_REST, _capi.MMI_KV_SINK | _capi.MMI_KV_ZERO_REST
_CODES = {torch.int8: _capi.MMI_I8, torch.float8_e4m3fn: _capi.MMI_F8E4M3}
_NAMES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_DTYPES = {torch.bfloat16: _capi.MMI_BF16, torch.float32: _capi.MMI_F32}


class PagedKVCache:
    """The cache's four arrays and how its keys are rotated.

    Args:
        k, v: codes, [pages, kv_heads, 64, dim] and [pages, kv_heads, vdim, 64]; torch.int8 or torch.float8_e4m3fn, contiguous.  Head sizes
            are multiples of 16 up to 256.
        k_scale, v_scale: fp32 [pages, kv_heads, 4]: what a code of each 16 tokens and head is multiplied by.
        rot_dim: leading dimensions of keys and queries that are rotated by their positions (a multiple of 8; 0: none), pair i by
            position * rot_base ** (-2 i / rot_dim); rot_halves: partners lie rot_dim / 2 apart instead of side by side.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, rot_dim: int = 0, rot_base: float = 1e4,
                 rot_halves: bool = False, lib: Optional[_capi.Lib] = None):
        if k.dim() != 4 or v.dim() != 4 or k.shape[2] != PAGE_TOKENS or v.shape[3] != PAGE_TOKENS or k.shape[:2] != v.shape[:2]:
            raise AssertionError("codes are [pages, kv_heads, 64, dim] and [pages, kv_heads, vdim, 64]")
        if k.dtype not in _CODES or v.dtype != k.dtype:
            raise ValueError("codes are int8 or float8_e4m3fn, the same for keys and values")
        shape = (k.shape[0], k.shape[1], PAGE_TOKENS // BLOCK_TOKENS)
        if k_scale.shape != shape or v_scale.shape != shape or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise AssertionError("scales are fp32 [pages, kv_heads, 4]")
        self.device = k.device
        if not all(t.is_contiguous() and t.device == self.device for t in (k, v, k_scale, v_scale)):
            raise ValueError("the cache's arrays are contiguous and on one device")
        if lib is None:
            if self.device.type != "cuda":
                raise RuntimeError("moshi_amd.PagedKVCache runs on an MI355X (device='cuda'); there is no CPU path")
            lib = _capi.load_tlm()
        if rot_dim and not (rot_base > 0 and math.isfinite(rot_base)):
            raise ValueError("rot_base must be positive")
        self._lib = lib
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, _, self.dim = k.shape
        self.vdim = v.shape[2]
        self.rot_dim, self.rot_base, self.rot_halves = int(rot_dim), float(rot_base), bool(rot_halves)
        self._freq = None
        if rot_dim:
            turns = [rot_base ** (-2.0 * i / rot_dim) / (2.0 * math.pi) for i in range(rot_dim // 2)]
            self._freq = torch.tensor(turns, dtype=torch.float64, device=self.device)
        self._desc = _capi.KVCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), self.pages, self.kv_heads, self.dim, self.vdim, _CODES[k.dtype],
                                       self.rot_dim, int(self.rot_halves), self._freq.data_ptr() if rot_dim else None)
        self._on = _capi.LaunchOn(self.device)
        self._where = k.get_device()
        self._need = {}
        self._workspace(_capi.KVSeqs(), (0, 0, 0, self.kv_heads, 0, 0, True))      # (sizes that the kernels do not take are refused here)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, dim: int, vdim: Optional[int] = None, codes: str = "int8", device: torch.device | str = "cuda", **rotation) -> "PagedKVCache":
        """A cache that holds nothing.  codes: "int8" (steps of 1/127 of a block's largest value) or "e4m3" (3 bits behind the leading one)."""
        if codes not in _NAMES:
            raise ValueError("codes are 'int8' or 'e4m3'")
        vdim = dim if vdim is None else vdim
        k = torch.zeros((pages, kv_heads, PAGE_TOKENS, dim), dtype=torch.int8, device=device).view(_NAMES[codes])
        v = torch.zeros((pages, kv_heads, vdim, PAGE_TOKENS), dtype=torch.int8, device=device).view(_NAMES[codes])
        scales = [torch.zeros((pages, kv_heads, PAGE_TOKENS // BLOCK_TOKENS), device=device) for _ in range(2)]
        return cls(k, v, *scales, **rotation)

    # ---- arguments --------------------------------------------------------------------------------------------------
    def _seqs(self, table: torch.Tensor, positions: torch.Tensor, rows: Optional[torch.Tensor], total: int) -> _capi.KVSeqs:
        where, (n, *more), shape = self._where, positions.shape, table.shape
        if more or len(shape) != 2 or shape[0] != n or (rows is not None and rows.shape != (n + 1,)):
            raise AssertionError("table is [sequences, pages], positions [sequences], rows [sequences + 1]")
        for t in (table, positions) if rows is None else (table, positions, rows):
            if t.dtype is not torch.int32 or t.get_device() != where or not t.is_contiguous():
                raise ValueError("table, positions and rows are contiguous int32 tensors on the cache's device")
        if rows is None and total != n:
            raise AssertionError(f"{total} rows for {n} sequences: without `rows` every sequence brings one")
        return _capi.KVSeqs(n, total, None if rows is None else rows.data_ptr(), positions.data_ptr(), table.data_ptr(), shape[1])

    def _rows(self, t: torch.Tensor, name: str, heads: Optional[int], dim: int):
        """Heads and type of a tensor of rows, and its address and strides."""
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
            raise AssertionError(f"{name} is [rows, {'heads' if heads is None else heads}, {dim}]")
        dtype = _DTYPES.get(t.dtype)
        if dtype is None or t.get_device() != self._where:
            raise ValueError(f"{name} is bf16 or fp32, on the cache's device")
        if stride[2] != 1 and t.numel():
            raise ValueError(f"a head's dimensions lie side by side in {name}")
        return shape[1], dtype, (t.data_ptr(), stride[0], stride[1])

    def _workspace(self, seqs: _capi.KVSeqs, key) -> int:
        """Bytes that an attention of these sizes (sequences, rows, pages of a sequence, heads, window, first tokens, one row each?) works in."""
        need = self._need.get(key)
        if need is None:
            need = self._lib.mmi_kv_attend_workspace(C.byref(self._desc), C.byref(seqs), *key[3:6])
            self._lib.check(min(0, need))
            if len(self._need) > 4096:
                self._need.clear()
            self._need[key] = need
        return need

    # ---- computation -------------------------------------------------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, rows: Optional[torch.Tensor] = None) -> None:
        """Write the rows' keys [rows, kv_heads, dim] (rotated on the way) and values [rows, kv_heads, vdim], bf16 or fp32, to their pages.
        The pages that two sequences of a call write to are different ones."""
        seqs = self._seqs(table, positions, rows, k.shape[0])
        (_, dtype, kp), (_, vtype, vp) = self._rows(k, "k", self.kv_heads, self.dim), self._rows(v, "v", self.kv_heads, self.vdim)
        if dtype != vtype or v.shape[0] != seqs.rows:
            raise AssertionError("keys and values come in the same number and type")
        self._lib.check(self._on.call(self._lib.mmi_kv_append, C.byref(self._desc), C.byref(seqs), dtype, *kp, *vp))

    def attend(self, q: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, rows: Optional[torch.Tensor] = None, scale: Optional[float] = None, window: int = 0,
               keep_first: int = 0, sink: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of queries [rows, heads, dim] over the positions up to their own, those rows' keys having been appended: [rows, heads, vdim]
        in the queries' type.  scale: default dim ** -0.5.  window > 0: the last `window` positions and the first `keep_first`.  sink: one is
        added to the softmax's denominator.  Rows that see nothing are zeros.  Rows that no sequence brings - behind the last one, or of one that
        is passed over - are zeros too in a new tensor, and left as they were in `out`, whose rows and heads lie apart."""
        if window >> 31 or keep_first >> 31:                   # (below 0, or beyond 31 bits)
            if window < 0 or keep_first < 0:
                raise ValueError("a window, and the first positions kept beside it, are not negative")
            window, keep_first = min(window, _LONGEST), min(keep_first, _LONGEST)
        heads, dtype, qp = self._rows(q, "q", None, self.dim)
        total = q.shape[0]
        seqs = self._seqs(table, positions, rows, total)
        if out is None:
            flags = _SINK_ZERO_REST if sink else _ZERO_REST
            out = torch.empty_like(q) if self.vdim == self.dim and q.is_contiguous() else q.new_empty((total, heads, self.vdim))
            op = (out.data_ptr(), heads * self.vdim, self.vdim)
            if not positions.shape[0]:
                out.zero_()
        else:
            flags = _SINK if sink else 0
            if out.shape != (total, heads, self.vdim) or out.dtype != q.dtype:
                raise AssertionError("out is [rows, heads, vdim] in the queries' type")
            op = self._rows(out, "out", heads, self.vdim)[2]
        need = self._workspace(seqs, (seqs.n, total, seqs.table_ld, heads, window, keep_first, rows is None))
        work = q.new_empty(need, dtype=torch.uint8) if need else None
        self._lib.check(self._on.call(self._lib.mmi_kv_attend, C.byref(self._desc), C.byref(seqs), dtype, heads, *qp, *op, self.dim ** -0.5 if scale is None else scale, window,
                                      keep_first, flags, work.data_ptr() if need else None, need))
        return out

    def read(self, table: torch.Tensor, positions: torch.Tensor, rows: Optional[torch.Tensor] = None, tokens: Optional[int] = None,
             dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values the cache holds for those positions (keys as they were rotated): [tokens, kv_heads, dim] and [tokens, kv_heads, vdim];
        zeros where there is no page, and in rows that no sequence brings.  tokens: rows[-1] (without `rows`: one for each sequence)."""
        if rows is not None and tokens is None:
            raise ValueError("tokens is needed beside rows")
        total = positions.shape[0] if rows is None else int(tokens)
        if dtype not in _DTYPES:
            raise ValueError("dtype must be torch.bfloat16 or torch.float32")
        seqs = self._seqs(table, positions, rows, total)
        k = self.k_scale.new_empty((total, self.kv_heads, self.dim), dtype=dtype)
        v = torch.empty_like(k) if self.vdim == self.dim else k.new_empty((total, self.kv_heads, self.vdim))
        if not seqs.n:
            return k.zero_(), v.zero_()
        self._lib.check(self._on.call(self._lib.mmi_kv_read, C.byref(self._desc), C.byref(seqs), _DTYPES[dtype], k.data_ptr(), v.data_ptr()))
        return k, v
