"""Rotary positions from the tokens' positions, queries and keys in one launch.

    rope = Rope(128, base=500000.0, scaling=config.rope_scaling)     # one for all layers
    q, k = rope.apply(q, k, positions)

The counterpart of ``attention.apply_rotary_pos_emb_custom`` (the reference's RoPE helper,
LlamaLoRaAttention_headwise.py:22-29), which multiplies by tables of sines in the model's
type, rounding each product: here a token's angles come from its position, exact modulo a
turn at any distance, and a value is rounded once (``starkv_rope`` in ``include/starkv.h``).
"""

from __future__ import annotations

import math
import struct
from typing import List, Optional, Sequence, Tuple, Union

import torch

from ._lib import StarKVError, check, load
from .kv4 import _TOKEN_DTYPES, _device_now, _output, _stream_of
from .ops import _DT

# starkv_rope_args: the tensors, their strides, the positions, the rest
_STRIDES, _REST = struct.Struct("12q"), struct.Struct("2qPf10i4x")
_ROPE = struct.Struct(f"4P{_STRIDES.size}sP{_REST.size}s")
_MAX_PLANS = 64

# What a scaling may hold: read below, or without a say in the angles of the types that are taken
_SCALING_KEYS = frozenset((
    "rope_type", "type", "rope_theta", "partial_rotary_factor", "factor", "low_freq_factor", "high_freq_factor",
    "original_max_position_embeddings", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim",
    "short_factor", "long_factor", "max_position_embeddings", "finetuned"))


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None) -> Tuple[List[float], float]:
    """The angle per position of each of rotary_dim / 2 channel pairs, in 64 bits, and the factor of
    the sines and cosines.

    scaling: None, or a model configuration's ``rope_scaling`` / ``rope_parameters``, of
    ``rope_type`` "default", "linear" (factor), "llama3" (factor, low_freq_factor,
    high_freq_factor, original_max_position_embeddings) or "yarn" (factor,
    original_max_position_embeddings, beta_fast, beta_slow, truncate, attention_factor); a
    ``rope_theta`` in it is the base; of a ``partial_rotary_factor`` rotary_dim is the outcome (``Rope``
    works it out).  Entries of None count as absent, unknown ones (sections of several positions, a
    dictionary for each kind of layer) are refused."""
    s = {name: value for name, value in (scaling or {}).items() if value is not None or name == "truncate"}
    unknown = sorted(map(str, s.keys() - _SCALING_KEYS))
    if unknown:
        raise StarKVError(f"scaling entries that are not understood: {', '.join(unknown)}")
    base = float(s.get("rope_theta", base))
    kind = s.get("rope_type", s.get("type", "default"))
    if rotary_dim <= 0 or rotary_dim % 2 or not base > 0 or base == 1.0 or not math.isfinite(base):
        raise StarKVError("rotary_dim must be even and positive, base positive and not 1")

    def number(name, default=None):
        value = s.get(name)
        value = default if value is None else value
        if value is None or not float(value) > 0 or not math.isfinite(float(value)):
            raise StarKVError(f"{kind} scaling needs a positive {name}")
        return float(value)

    f = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if kind == "default":
        return f, 1.0
    factor = number("factor")
    if kind == "linear":
        return [x / factor for x in f], 1.0
    if kind == "llama3":
        old, low, high = number("original_max_position_embeddings"), number("low_freq_factor"), number("high_freq_factor")
        if high <= low:
            raise StarKVError("llama3 scaling needs high_freq_factor > low_freq_factor")
        for i, x in enumerate(f):
            t = min(1.0, max(0.0, (old * x / (2.0 * math.pi) - low) / (high - low)))
            f[i] = (1.0 - t) * x / factor + t * x
        return f, 1.0
    if kind == "yarn":
        old = number("original_max_position_embeddings")
        # the pair that makes n turns over the original context
        pair = lambda n: rotary_dim * math.log(old / (2.0 * math.pi * n)) / (2.0 * math.log(base))  # noqa: E731
        lo, hi = pair(number("beta_fast", 32.0)), pair(number("beta_slow", 1.0))
        if s.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
        for i, x in enumerate(f):
            e = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f[i] = (1.0 - e) * x + e * x / factor
        for name in ("mscale", "mscale_all_dim"):
            if s.get(name):
                raise StarKVError(f"yarn scaling with {name} is not supported; give attention_factor")
        return f, number("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)
    raise StarKVError(f"unknown rope_type {kind!r}")


class _Turn(torch.autograd.Function):
    """The turn is linear and its transpose is the inverse turn with the same factor, so the gradients
    of q and k are those of the outputs turned back; recorded again where they need gradients."""

    @staticmethod
    def forward(ctx, rope, inverse, positions, q, k):
        ctx.rope, ctx.inverse = rope, inverse
        ctx.save_for_backward(positions)             # autograd refuses positions that were written since
        return rope._turn(q, k, positions, inverse, None)

    @staticmethod
    def backward(ctx, *grads):
        positions, = ctx.saved_tensors
        # a gradient may be repeated elements (that of a sum); channels have to follow one another
        sides = [g if g.stride(-1) == 1 else g.contiguous() for g, needed in zip(grads, ctx.needs_input_grad[3:]) if needed]
        back = ctx.rope.apply(sides[0], sides[1] if len(sides) == 2 else None, positions, inverse=not ctx.inverse)
        found = iter(back if len(sides) == 2 else (back,))
        return (None, None, None, *(next(found) if needed else None for needed in ctx.needs_input_grad[3:]))


def rotary_channels(head_dim: int, rotary_dim: Optional[int] = None, scaling: Optional[dict] = None) -> int:
    """How many channels of a head turn: ``rotary_dim``, or the part of head_dim that scaling's
    ``partial_rotary_factor`` says, or all."""
    part = (scaling or {}).get("partial_rotary_factor")
    if part is not None:
        if not 0 < float(part) <= 1:
            raise StarKVError(f"partial_rotary_factor must be above 0 and at most 1, got {part}")
        part = int(head_dim * float(part))
        if rotary_dim is not None and rotary_dim != part:
            raise StarKVError(f"rotary_dim {rotary_dim} is not the scaling's partial_rotary_factor of head_dim, {part}")
        rotary_dim = part
    rotary_dim = head_dim if rotary_dim is None else rotary_dim
    if rotary_dim <= 0 or rotary_dim % 2 or rotary_dim > head_dim:
        raise StarKVError(f"rotary_dim must be even, positive and at most head_dim {head_dim}, got {rotary_dim}")
    return rotary_dim


class Rope:
    """Rotary positions of heads of ``head_dim``, of which the first ``rotary_dim`` channels (by default
    all, or ``scaling``'s ``partial_rotary_factor`` of them) turn: pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with ``interleaved``.

    Frequencies come from ``base`` and ``scaling`` (``rope_frequencies``), or are given:
    ``frequencies`` (rotary_dim / 2 numbers, e.g. a model's ``inv_freq``) and ``factor``."""

    def __init__(self, head_dim: int, base: float = 10000.0, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 scaling: Optional[dict] = None, frequencies: Optional[Union[Sequence[float], torch.Tensor]] = None,
                 factor: float = 1.0, device="cuda"):
        rotary_dim = rotary_channels(head_dim, rotary_dim, scaling)
        if frequencies is None:
            frequencies, factor = rope_frequencies(rotary_dim, base, scaling)
        elif scaling is not None:
            raise StarKVError("scaling and frequencies exclude each other")
        else:
            if isinstance(frequencies, torch.Tensor):
                frequencies = frequencies.double().tolist()
            frequencies = [float(f) for f in frequencies]
        if len(frequencies) != rotary_dim // 2 or not all(map(math.isfinite, [*frequencies, factor])):
            raise StarKVError(f"frequencies must be {rotary_dim // 2} finite numbers, factor one")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise StarKVError("Rope lives on a CUDA device")
        self.frequencies = tuple(frequencies)
        self._hold(head_dim, torch.tensor(turns_of(frequencies), dtype=torch.int64, device=dev), factor, interleaved)

    @classmethod
    def from_turns(cls, head_dim: int, turns: torch.Tensor, factor: float = 1.0, interleaved: bool = False) -> "Rope":
        """A Rope over the ``turns`` of another, for code that passes tensors."""
        if turns.dtype != torch.int64 or turns.dim() != 1 or not turns.is_cuda or not turns.is_contiguous() or \
                not 0 < 2 * turns.shape[0] <= head_dim:
            raise StarKVError("turns must be int64 (rotary_dim / 2,) on a CUDA device")
        self = cls.__new__(cls)
        self.frequencies = None
        self._hold(head_dim, turns, factor, interleaved)
        return self

    def _hold(self, head_dim, turns, factor, interleaved):
        self.head_dim, self.rotary_dim, self.interleaved = int(head_dim), 2 * turns.shape[0], bool(interleaved)
        self.factor, self.turns = float(factor), turns
        self.device, self._index = turns.device, turns.device.index
        self._turns, self._fn = turns.data_ptr(), load().starkv_rope
        # What follows from shapes, strides and types alone, of calls into new tensors or in place, so that
        # a decode step's checks are made once: 8.9 us of the host a call, 11.9 without, 5.2 in place
        self._plans = {}

    def __deepcopy__(self, memo) -> "Rope":
        """Modules that share one may be copied: the turns are, the library is not."""
        new = Rope.from_turns(self.head_dim, self.turns.clone(), self.factor, self.interleaved)
        new.frequencies = self.frequencies
        memo[id(self)] = new
        return new

    def __reduce__(self):
        return Rope.from_turns, (self.head_dim, self.turns, self.factor, self.interleaved)

    def _side(self, t: torch.Tensor, name: str, lead, dtype):
        """Checks a side; returns its strides of batch, token and head."""
        shape, st = t.shape, t.stride()
        if t.get_device() != self._index or t.dtype != dtype or shape[:-2] != lead or shape[-1] != self.head_dim:
            if t.get_device() != self._index:
                raise StarKVError(f"{name} must be on {self.device}")
            if t.dtype != dtype:
                raise StarKVError(f"{name} must be {dtype}, got {t.dtype}")
            raise StarKVError(f"{name} must be (tokens, heads, {self.head_dim}) or (B, tokens, heads, {self.head_dim}), "
                              f"tokens alike, got {tuple(shape)}")
        if st[-1] != 1 and self.head_dim > 1:
            raise StarKVError(f"{name} channels must be contiguous")
        if 1 in shape:                       # the stride of a dimension of one is never used
            st = [0 if n == 1 else s for n, s in zip(shape, st)]
        return st[:3] if len(lead) == 2 else (0, st[0], st[1])

    def apply(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inverse: bool = False, out=None):
        """q (and k) turned by the tokens' positions: (B, T, heads, head_dim), or (tokens, heads,
        head_dim) for packed prompts, fp32, fp16 or bf16, any strides whose channels are
        contiguous; positions int32 or int64 of the leading shape, or (T,) for every
        sequence, on the GPU.  ``inverse`` turns back (what was turned by the same
        positions).  Returns new tensors, or writes ``out`` (a tensor, or a
        pair with k), which may be the inputs themselves.  Without k (None) one tensor.
        Where q or k needs a gradient autograd records the call, and ``out`` is refused."""
        if torch.is_grad_enabled():
            needs = q.requires_grad or k is not None and k.requires_grad
            if out is None:
                if needs:
                    return _Turn.apply(self, inverse, positions, q, k)
            elif needs or any(o.requires_grad for o in (out if isinstance(out, (tuple, list)) else (out,))):
                raise StarKVError("out is for tensors without a gradient; without it new ones are recorded")
        return self._turn(q, k, positions, inverse, out)

    def _turn(self, q, k, positions, inverse, out):
        key = None
        if k is not None and (out is None or type(out) is tuple and len(out) == 2 and out[0] is q and out[1] is k):
            key = (q.shape, q.stride(), k.shape, k.stride(), positions.shape, positions.stride(), q.dtype, k.dtype,
                   positions.dtype, inverse, out is None)
            plan = self._plans.get(key)
            if plan is not None and q.get_device() == k.get_device() == positions.get_device() == self._index:
                strides, rest, dense = plan
                qp, kp = q.data_ptr(), k.data_ptr()
                if out is not None:
                    if qp != kp:
                        self._launch(_ROPE.pack(qp, kp, qp, kp, strides, positions.data_ptr(), rest))
                        return q, k
                elif dense:
                    oq, ok = torch.empty_like(q), torch.empty_like(k)
                    self._launch(_ROPE.pack(qp, kp, oq.data_ptr(), ok.data_ptr(), strides, positions.data_ptr(), rest))
                    return oq, ok
        dtype = q.dtype
        if dtype not in _TOKEN_DTYPES:
            raise StarKVError(f"q must be one of {_TOKEN_DTYPES}, got {dtype}")
        if not 3 <= q.dim() <= 4:
            raise StarKVError(f"q must be (tokens, heads, {self.head_dim}) or (B, tokens, heads, {self.head_dim})")
        lead = q.shape[:-2]
        qs = self._side(q, "q", lead, dtype)
        ks = (0, 0, 0) if k is None else self._side(k, "k", lead, dtype)
        if out is None:
            oq, qos = (torch.empty_like(q), qs) if q.is_contiguous() else self._new(q, lead)
            if k is None:
                ok, kos = None, (0, 0, 0)
            else:
                ok, kos = (torch.empty_like(k), ks) if k.is_contiguous() else self._new(k, lead)
        else:
            oq, ok = (out, None) if k is None else self._pair(out)
            qos = self._placed(oq, "out[0]", q, qs, lead)
            kos = (0, 0, 0) if k is None else self._placed(ok, "out[1]", k, ks, lead)
            if k is not None:
                for a, b in ((oq, k), (ok, q), (oq, ok)):
                    if a.numel() and a.data_ptr() == b.data_ptr():
                        raise StarKVError("the two sides must be apart")
                # (in place the two may lie between one another, as heads of a joint projection do)
                if oq.data_ptr() != q.data_ptr() and _overlap(oq, k) or ok.data_ptr() != k.data_ptr() and _overlap(ok, q):
                    raise StarKVError("an output that is not its input must be apart from the other side's too")
        wide = positions.dtype == torch.int64
        if positions.get_device() != self._index or not (wide or positions.dtype == torch.int32):
            raise StarKVError(f"positions must be int32 or int64 on {self.device}")
        B, T = (1, *lead) if len(lead) == 1 else lead
        if positions.shape == lead:
            ps = positions.stride()
            ps = ps if len(lead) == 2 else (0, ps[0])
        elif positions.shape == (T,) or positions.shape == (1, T):
            ps = (0, positions.stride(-1))
        else:
            raise StarKVError(f"positions must have shape {tuple(lead)} or ({T},), got {tuple(positions.shape)}")
        if k is None:
            kp = okp = kh = 0
        else:
            kp, okp, kh = k.data_ptr(), ok.data_ptr(), k.shape[-2]
        strides = _STRIDES.pack(*qs, *ks, *qos, *kos)
        rest = _REST.pack(*ps, self._turns, self.factor, wide, _DT[dtype], B, T, q.shape[-2], kh, self.head_dim,
                          self.rotary_dim, self.interleaved, inverse)
        self._launch(_ROPE.pack(q.data_ptr(), kp, oq.data_ptr(), okp, strides, positions.data_ptr(), rest))
        if key is not None:
            if len(self._plans) >= _MAX_PLANS:
                self._plans.clear()
            self._plans[key] = strides, rest, q.is_contiguous() and k.is_contiguous()
        return oq if k is None else (oq, ok)

    def _launch(self, a: bytes):
        if _device_now() == self._index:
            rc = self._fn(a, _stream_of(self._index))
        else:
            with torch.cuda.device(self._index):
                rc = self._fn(a, _stream_of(self._index))
        if rc:
            check(rc, "starkv_rope")

    def _new(self, x: torch.Tensor, lead):
        """A contiguous tensor of x's shape and its strides (empty_like, which is cheaper, keeps x's order)."""
        row, T = x.shape[-2] * self.head_dim, lead[-1]
        st = (T * row, row, self.head_dim)
        return torch.empty_strided(x.shape, (*st[3 - len(lead) - 1:], 1), dtype=x.dtype, device=self.device), st

    @staticmethod
    def _pair(out):
        out = tuple(out)
        if len(out) != 2:
            raise StarKVError("out must be a pair where k is given")
        return out

    def _placed(self, o: torch.Tensor, name: str, x: torch.Tensor, xs, lead):
        if o.shape != x.shape:
            raise StarKVError(f"{name} must have shape {tuple(x.shape)}, got {tuple(o.shape)}")
        st = self._side(o, name, lead, x.dtype)
        _output(o, name)
        if not (o.data_ptr() == x.data_ptr() and tuple(st) == tuple(xs)) and _overlap(o, x):
            raise StarKVError(f"{name} must be its input itself or apart from it")
        return st


def turns_of(frequencies: Sequence[float]) -> List[int]:
    """frequencies / 2 pi modulo 1 in units of 2^-64, as signed 64-bit numbers."""
    found = []
    for f in frequencies:
        # n = f / 2 pi * 2^64, in whole numbers: 2 pi = TAU / 2^120
        num, den = f.as_integer_ratio()
        n = ((num << 185) // (den * _TAU) + 1 >> 1) & (1 << 64) - 1
        found.append(n - (1 << 64) if n >> 63 else n)
    return found


# 2 pi * 2^120, from Machin's formula pi / 4 = 4 atan(1 / 5) - atan(1 / 239) in whole numbers
def _atan_inverse(n: int, bits: int) -> int:
    total, term, k = 0, (1 << bits) // n, 1
    while term:
        total += term // k if k % 4 == 1 else -(term // k)
        term //= n * n
        k += 2
    return total


_TAU = 8 * (4 * _atan_inverse(5, 140) - _atan_inverse(239, 140)) >> 20


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))

    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1
