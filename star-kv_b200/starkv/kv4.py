"""Paged 4-bit key / value cache for layers whose K / V projections are not factored.

The latent cache (``ops.LatentCache``) pays off where a layer's learned ranks are
small; a layer whose ranks stay near the head dimension keeps its whole heads
here instead, 5 bits a value (4-bit codes, fp16 scale and centre per 32 channels),
in pages that sequences of a batch share a pool of:

    cache = KV4Cache(num_pages, num_kv_heads, page_size=64)
    cache.write(k, v, block_table, start)                       # prompt or newest tokens, quantised
    out = cache.attend(q, block_table, lengths, scaling)        # newest 1..n queries, dense
    pages = cache.select(q, block_table, lengths, 64)           # pages a score bound keeps
    out = cache.attend(q, block_table, lengths, scaling, pages=pages)
    k, v = cache.read(block_table, start, num_tokens)           # back to whole heads

Every op launches on the current torch stream, takes its positions, lengths and
page lists from the GPU (so a step can be captured in a CUDA graph) and goes
through ``libstarkv.so`` (``starkv_kv4_*`` in ``include/starkv.h``, which specifies
the layout and the arithmetic); there is no CPU path.
"""

from __future__ import annotations

import copy
import ctypes as C
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import StarKVError, check, load
from .ops import _DT

# Argument blocks (the mirrors of _lib, packed in one call: a ctypes structure
# costs several microseconds to fill field by field).
_CACHE = struct.Struct("4P4i")
_IO = struct.Struct("2P3q3qPq2P4i")
_ATTENTION = struct.Struct("3P3q3qPqPP2qPPNf7i")
_SELECT = struct.Struct("P3qPq3PN8i")

_TOKEN_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_QUERY_DTYPES = (torch.float16, torch.bfloat16)

# The checks below run on every call of a decode step, several calls a layer: they
# compare device indices and torch.Size tuples instead of building objects.
_device_now = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _ints(t: torch.Tensor, name: str, shape, index: int) -> int:
    if t.dtype != torch.int32 or t.get_device() != index:
        raise StarKVError(f"{name} must be an int32 tensor on cuda:{index}")
    if t.shape != shape or not t.is_contiguous():
        raise StarKVError(f"{name} must be contiguous of shape {shape}, got {tuple(t.shape)}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, shape, dtypes, index: int):
    """Checks a (B, tokens, heads, 128) tensor; returns its element strides."""
    if t.get_device() != index:
        raise StarKVError(f"{name} must be on cuda:{index}")
    if t.dtype not in dtypes:
        raise StarKVError(f"{name} must be one of {dtypes}, got {t.dtype}")
    if t.shape != shape:
        raise StarKVError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    st = t.stride()
    if st[3] != 1:
        raise StarKVError(f"{name} channels must be contiguous")
    if 1 in shape:                       # the stride of a dimension of one is never used
        st = tuple([0 if n == 1 else s for n, s in zip(shape, st)])
    return st


def _output(t: torch.Tensor, name: str):
    if not t.is_contiguous() and any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
        raise StarKVError(f"{name} must not repeat elements (stride 0)")


# The newest few streams' scratch: an attention workspace is 32 MB, and programs go through many
# streams.  What is dropped goes back to its own stream's pool of torch's allocator, which hands
# it out behind the work that still uses it.
_WORKSPACES = {}
_MAX_WORKSPACES = 8


def release_workspaces() -> None:
    """Give the scratch of all streams back to torch's allocator."""
    _WORKSPACES.clear()


def _workspace(kind: str, index: int, size, zeroed: int) -> torch.Tensor:
    """Scratch of one kind for the current stream, of ``size()`` bytes at least (its
    first ``zeroed`` bytes cleared when made; every call leaves them clear for the
    next).  A call under graph capture gets its own, cleared by the graph, so replays
    never share one with eager calls."""
    capturing = torch.cuda.is_current_stream_capturing()
    key = (kind, index, _stream_of(index))
    ws = None if capturing else _WORKSPACES.get(key)
    need = size()
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, dtype=torch.uint8, device=f"cuda:{index}")
        ws[:zeroed].zero_()
        if not capturing:
            _WORKSPACES.pop(key, None)
            held = [k for k in list(_WORKSPACES) if k[0] == kind]
            for k in held[:max(0, len(held) + 1 - _MAX_WORKSPACES)]:
                _WORKSPACES.pop(k, None)
            _WORKSPACES[key] = ws
    return ws


_attention_bytes = 0


def _attention_size() -> int:
    global _attention_bytes
    if not _attention_bytes:
        n = C.c_size_t(0)
        check(load().starkv_kv4_workspace_size(C.byref(n)), "starkv_kv4_workspace_size")
        _attention_bytes = int(n.value)
    return _attention_bytes


class KV4Cache:
    """A pool of ``num_pages`` pages of ``page_size`` tokens (16, 32, 64 or 128) for
    ``num_kv_heads`` KV heads of dimension 128.

    ``data``: uint8 (num_pages, num_kv_heads, page_size / 16, 2560).  With
    ``page_bounds`` each full page also carries int8 bounds of its keys
    (``bounds``, ``bound_scales``), which ``select`` scores.  Which pages belong to
    which sequence is the caller's: ``block_table`` (B, W) int32 names sequence b's
    pages in order."""

    def __init__(self, num_pages: int, num_kv_heads: int, page_size: int = 64, device="cuda",
                 page_bounds: bool = True):
        if page_size not in (16, 32, 64, 128):
            raise StarKVError(f"page_size must be 16, 32, 64 or 128, got {page_size}")
        if num_pages <= 0 or num_kv_heads <= 0:
            raise StarKVError("KV4Cache needs at least one page and one KV head")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise StarKVError("KV4Cache lives on a CUDA device")
        data = torch.zeros(num_pages, num_kv_heads, page_size // 16, 2560, dtype=torch.uint8, device=dev)
        bounds = scales = None
        if page_bounds:
            bounds = torch.zeros(num_pages, num_kv_heads, 2, 128, dtype=torch.int8, device=dev)
            scales = torch.zeros(num_pages, num_kv_heads, dtype=torch.float32, device=dev)
        self._hold(data, bounds, scales, torch.zeros(1, dtype=torch.int32, device=dev))

    @classmethod
    def from_tensors(cls, data: torch.Tensor, bounds: Optional[torch.Tensor], bound_scales: Optional[torch.Tensor],
                     error_word: torch.Tensor) -> "KV4Cache":
        """A cache over the tensors of another (``data``, ``bounds``, ``bound_scales``,
        ``error_word``), for code that passes them one by one."""
        if data.dim() != 4 or data.shape[3] != 2560 or data.dtype != torch.uint8 or not data.is_cuda:
            raise StarKVError("data must be a uint8 (pages, heads, page_size / 16, 2560) CUDA tensor")
        pages, heads = data.shape[:2]
        ok = data.is_contiguous() and data.shape[2] in (1, 2, 4, 8) and pages > 0 and heads > 0
        ok = ok and (bounds is None) == (bound_scales is None)
        parts = [(error_word, torch.int32, (1,))]
        if bounds is not None:
            parts += [(bounds, torch.int8, (pages, heads, 2, 128)), (bound_scales, torch.float32, (pages, heads))]
        for t, dtype, shape in parts:
            ok = ok and t.dtype == dtype and t.shape == shape and t.is_contiguous() and t.device == data.device
        if not ok:
            raise StarKVError("the tensors are not those of a KV4Cache")
        self = cls.__new__(cls)
        self._hold(data, bounds, bound_scales, error_word)
        return self

    def _hold(self, data, bounds, bound_scales, error_word):
        self.data, self.bounds, self.bound_scales, self.error_word = data, bounds, bound_scales, error_word
        self.num_pages, self.num_kv_heads, self.page_size = data.shape[0], data.shape[1], data.shape[2] * 16
        self.device = data.device
        self._index = self.device.index
        self._block = _CACHE.pack(data.data_ptr(), 0 if bounds is None else bounds.data_ptr(),
                                  0 if bounds is None else bound_scales.data_ptr(), error_word.data_ptr(),
                                  self.num_pages, self.num_kv_heads, self.page_size, 128)
        self._lib = load()

    def __deepcopy__(self, memo) -> "KV4Cache":
        """A pool of its own with the same contents (the argument block holds addresses)."""
        parts = (self.data, self.bounds, self.bound_scales, self.error_word)
        return self.from_tensors(*[copy.deepcopy(t, memo) for t in parts])

    def __reduce__(self):
        return self.from_tensors, (self.data, self.bounds, self.bound_scales, self.error_word)

    def nbytes(self) -> int:
        """Device bytes of the pool (codes, parameters and bounds)."""
        return sum(t.numel() * t.element_size() for t in (self.data, self.bounds, self.bound_scales) if t is not None)

    def _table(self, t: torch.Tensor):
        if t.dtype != torch.int32 or t.get_device() != self._index or t.dim() != 2:
            raise StarKVError(f"block_table must be an int32 (B, W) tensor on {self.device}")
        (B, W), (st, unit) = t.shape, t.stride()
        if W == 0 or (W > 1 and unit != 1):
            raise StarKVError("block_table must have W > 0 and contiguous rows")
        return B, W, t.data_ptr(), st

    def _call(self, fn, args: bytes, what: str):
        """One C call on the pool's device and its current stream."""
        if _device_now() == self._index:
            rc = fn(self._block, args, _stream_of(self._index))
        else:
            with torch.cuda.device(self._index):
                rc = fn(self._block, args, _stream_of(self._index))
        if rc:
            check(rc, what)

    def _io(self, fn, what, k, v, ks, vs, table, start, count):
        B, W, tp, ts = table
        a = _IO.pack(k.data_ptr(), v.data_ptr(), *ks[:3], *vs[:3], tp, ts,
                     _ints(start, "start", (B,), self._index),
                     0 if count is None else _ints(count, "count", (B,), self._index), _DT[k.dtype], B, k.shape[1], W)
        self._call(fn, a, what)

    def write(self, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, start: torch.Tensor,
              count: Optional[torch.Tensor] = None) -> None:
        """Quantise k / v (B, T, num_kv_heads, 128; fp32, fp16 or bf16, rows of any
        stride that is a multiple of 16 bytes) into positions start[b] .. start[b] +
        count[b] - 1 (count: int32 (B,), T when None).  Filling a page's last slot
        writes the page's bounds."""
        table = self._table(block_table)
        shape = (table[0], k.shape[1] if k.dim() == 4 else -1, self.num_kv_heads, 128)
        ks = _rows(k, "k", shape, _TOKEN_DTYPES, self._index)
        vs = _rows(v, "v", shape, (k.dtype,), self._index)
        self._io(self._lib.starkv_kv4_write, "starkv_kv4_write", k, v, ks, vs, table, start, count)

    def read(self, block_table: torch.Tensor, start: torch.Tensor, num_tokens: int,
             count: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Positions start[b] .. start[b] + num_tokens - 1 as (k, v), each (B,
        num_tokens, num_kv_heads, 128) of ``dtype`` (or into ``out``); rows past count[b]
        are 0."""
        table = self._table(block_table)
        shape = (table[0], int(num_tokens), self.num_kv_heads, 128)
        if out is None:
            if num_tokens < 0:
                raise StarKVError("num_tokens must not be negative")
            if dtype not in _TOKEN_DTYPES:
                raise StarKVError(f"dtype must be one of {_TOKEN_DTYPES}, got {dtype}")
            B, T, H, _ = shape
            ks = vs = (T * H * 128, H * 128, 128, 1)
            k, v = torch.empty_strided((2, *shape), (B * ks[0], *ks), dtype=dtype, device=self.device).unbind(0)
        else:
            k, v = out
            ks = _rows(k, "out[0]", shape, _TOKEN_DTYPES, self._index)
            vs = _rows(v, "out[1]", shape, (k.dtype,), self._index)
            _output(k, "out[0]")
            _output(v, "out[1]")
        self._io(self._lib.starkv_kv4_read, "starkv_kv4_read", k, v, ks, vs, table, start, count)
        return k, v

    def _queries(self, q: torch.Tensor, batch: int):
        """q as (B, Q, Hq, 128) and its strides; a (B, Hq, 128) q is one query token."""
        q4 = q.unsqueeze(1) if q.dim() == 3 else q
        if q4.dim() != 4 or q4.shape[2] == 0 or q4.shape[2] % self.num_kv_heads:
            raise StarKVError(f"q must be (B, Hq, 128) or (B, Q, Hq, 128), Hq a multiple of {self.num_kv_heads}")
        return q4, _rows(q4, "q", (batch, q4.shape[1], q4.shape[2], 128), _QUERY_DTYPES, self._index)

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, scaling: float,
               mask: Optional[torch.Tensor] = None, pages: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False,
               ws: Optional[torch.Tensor] = None):
        """Attention of each sequence's newest Q tokens, q (B, Q, Hq, 128) or (B, Hq,
        128), over its first lengths[b] positions (the queries' own included, written
        before): query i attends to positions up to lengths[b] - Q + i.

        mask: additive fp32 (B, L), -inf excludes a position.  pages: int32 (B,
        num_kv_heads, n) page ordinals to attend within (``select``).  Returns out of
        q's shape and dtype (or in ``out``), and with ``return_lse`` the fp32 log-sum-exp
        (q's shape without the channels); a query with nothing to attend to gets 0 and
        -inf.  ws: scratch of one's own, ``starkv_kv4_workspace_size`` bytes on a 16-byte
        boundary, its first 1024 zeroed before its first use (each call leaves them zero)."""
        B, W, tp, ts = self._table(block_table)
        q4, qs = self._queries(q, B)
        Q, Hq = q4.shape[1], q4.shape[2]
        index = self._index
        lp = _ints(lengths, "lengths", (B,), index)
        if out is None:
            # empty_strided: the cheapest of torch's allocating calls
            os_ = (Q * Hq * 128, Hq * 128, 128, 1)
            o4 = torch.empty_strided((B, Q, Hq, 128), os_, dtype=q.dtype, device=self.device)
            out = o4 if q4 is q else o4[:, 0]
        else:
            o4 = out.unsqueeze(1) if q.dim() == 3 and out.dim() == 3 else out
            os_ = _rows(o4, "out", q4.shape, _TOKEN_DTYPES, index)
            _output(o4, "out")
        mp = mstride = mwidth = 0
        if mask is not None:
            if mask.dtype != torch.float32 or mask.get_device() != index or mask.dim() != 2 or mask.shape[0] != B:
                raise StarKVError(f"mask must be an fp32 (B, L) tensor on {self.device}")
            if mask.shape[1] > 1 and mask.stride(1) != 1:
                raise StarKVError("mask rows must be contiguous")
            mp, mstride, mwidth = mask.data_ptr(), mask.stride(0), mask.shape[1]
        pp = n = 0
        if pages is not None:
            if pages.dim() != 3 or pages.shape[2] == 0:
                raise StarKVError("pages must be (B, num_kv_heads, n), n > 0")
            n = pages.shape[2]
            pp = _ints(pages, "pages", (B, self.num_kv_heads, n), index)
        lse = None
        if return_lse:
            lse = torch.empty_strided((B, Q, Hq), (Q * Hq, Hq, 1), dtype=torch.float32, device=self.device)
            lse_out = lse if q4 is q else lse[:, 0]
        if ws is None:
            ws = _workspace("attention", index, _attention_size, 1024)
        elif ws.get_device() != index or not ws.is_contiguous():
            raise StarKVError(f"ws must be contiguous on {self.device}")
        a = _ATTENTION.pack(q4.data_ptr(), o4.data_ptr(), lse.data_ptr() if return_lse else 0,
                            *qs[:3], *os_[:3], tp, ts, lp, mp, mstride, mwidth, pp, ws.data_ptr(),
                            ws.numel() * ws.element_size(), scaling, n, _DT[q.dtype], _DT[out.dtype], B, Q, Hq, W)
        self._call(self._lib.starkv_kv4_attention, a, "starkv_kv4_attention")
        return (out, lse_out) if return_lse else out

    def select(self, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, num_pages: int,
               first: int = 1, last: int = 1, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Page ordinals to attend to, int32 (B, num_kv_heads, num_pages) ascending, then
        -1: the sequence's first ``first`` and last ``last`` pages and, among the others,
        those whose bound on q.k (over the KV head's query heads and tokens) is
        highest; every page where there are no more than ``num_pages``."""
        if self.bounds is None:
            raise StarKVError("this KV4Cache was made without page_bounds")
        B, W, tp, ts = self._table(block_table)
        q4, qs = self._queries(q, B)
        lp = _ints(lengths, "lengths", (B,), self._index)
        shape = (B, self.num_kv_heads, int(num_pages))
        if out is None:
            if num_pages <= 0:
                raise StarKVError("num_pages must be positive")
            n = shape[2]
            out = torch.empty_strided(shape, (self.num_kv_heads * n, n, 1), dtype=torch.int32, device=self.device)
        op = _ints(out, "out", shape, self._index)
        # counters (65536 ints), then a score a page
        ws = _workspace("select", self._index, lambda: 262144 + 4 * B * self.num_kv_heads * W, 262144)
        a = _SELECT.pack(q4.data_ptr(), *qs[:3], tp, ts, lp, op, ws.data_ptr(), ws.numel(), _DT[q.dtype], B,
                         q4.shape[1], q4.shape[2], W, num_pages, first, last)
        self._call(self._lib.starkv_kv4_select, a, "starkv_kv4_select")
        return out

    def read_error(self) -> int:
        """Read and clear the pool's device error word (synchronises): 0, or a code of
        ``ERRORS``."""
        code = int(self.error_word.item())
        if code:
            self.error_word.zero_()
        return code


#: Codes of the device error word.
ERRORS = {0x101: "a bulk copy never completed", 0x201: "a block table names a page outside the pool",
          0x202: "a position or length lies outside the block table"}
