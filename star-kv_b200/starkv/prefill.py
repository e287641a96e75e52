"""Prompt (prefill) attention of the compressed-KV layer on the B200.

The reference's prefill (model.py:429-449) rebuilds full keys and values from
the latents and runs causal SDPA over them.  Here the rebuild is two plain GEMMs
per layer (``X_k U_k^T`` per KV head, ``X_v U_v^T`` once; cuBLAS) plus RoPE of
the keys, and the attention is the library's own tcgen05 flash-attention kernel
(``starkv_prefill_attention``): GQA by head index (no repeated K / V), the
values read in place from the (B, T, Hkv*128) product, the output written in
the (B, T, Hq, 128) order ``o_proj`` reads.

``packed_attention`` is the form for prompts of different lengths in one batch without
padding, and for pieces that continue earlier prompts (``starkv_packed_attention``).
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Sequence, Tuple, Union

import torch

from . import ops
from ._lib import StarKVError, check, load
from .kv4 import _QUERY_DTYPES, _TOKEN_DTYPES, _device_now, _ints, _output, _stream_of, _workspace
from .ops import _DT

# starkv_packed_args, packed in one call
_PACKED = struct.Struct("5P8q5PNP2qf6i4x")


def rebuild_keys(k_lat: torch.Tensor, k_u_heads: Sequence[torch.Tensor], k_ranks: Sequence[int],
                 cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """RoPE(X_k U_k^T) per KV head (model.py:431-432): k_lat (B, T, sum r_h) ->
    (B, Hkv, T, 128).  cos / sin: (B or 1, T, 128) tables of positions 0..T-1."""
    B, T, _ = k_lat.shape
    out = torch.empty(B, len(k_ranks), T, 128, dtype=k_lat.dtype, device=k_lat.device)
    c0 = 0
    for h, (r, u) in enumerate(zip(k_ranks, k_u_heads)):
        out[:, h] = torch.matmul(k_lat[..., c0:c0 + r], u.to(k_lat.dtype).T)
        c0 += r
    half = 64
    rot = torch.cat([-out[..., half:], out[..., :half]], dim=-1)
    return out * cos[:, None] + rot * sin[:, None]


def rebuild_values(v_lat: torch.Tensor, v_u_weight: torch.Tensor, num_kv_heads: int) -> torch.Tensor:
    """X_v U_v^T split into heads (model.py:437-441): (B, T, R) -> a (B, Hkv, T, 128)
    strided view of the (B, T, Hkv*128) product."""
    B, T, _ = v_lat.shape
    full = torch.matmul(v_lat, v_u_weight.to(v_lat.dtype).T)
    return full.view(B, T, num_kv_heads, 128).transpose(1, 2)


def prompt_attention(q_rot: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, scaling: float,
                     out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Causal attention of q_rot (B, Hq, T, 128) over keys / values (B, Hkv, T, 128)
    on the tensor cores; returns (B, Hq, T, 128) (a view of a (B, T, Hq, 128)
    tensor, so ``out.transpose(1, 2).reshape(B, T, -1)`` costs no copy)."""
    B, Hq, T, _ = q_rot.shape
    out = torch.empty(B, T, Hq, 128, dtype=out_dtype or q_rot.dtype, device=q_rot.device).transpose(1, 2)
    return ops.prefill_attention(q_rot, keys, values, scaling, out=out)


_packed_bytes = 0


def _packed_size() -> int:
    global _packed_bytes
    if not _packed_bytes:
        n = C.c_size_t(0)
        check(load().starkv_packed_workspace_size(C.byref(n)), "starkv_packed_workspace_size")
        _packed_bytes = int(n.value)
    return _packed_bytes


def _packed_rows(t: torch.Tensor, name: str, dtypes, index: int):
    """Checks a (rows, heads, 128) tensor; returns its strides of rows and heads."""
    if t.get_device() != index:
        raise StarKVError(f"{name} must be on cuda:{index}")
    if t.dtype not in dtypes:
        raise StarKVError(f"{name} must be one of {dtypes}, got {t.dtype}")
    shape, st = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != 128 or shape[1] == 0 or st[2] != 1:
        raise StarKVError(f"{name} must be (rows, heads, 128) with contiguous channels, got {tuple(shape)}")
    return (0 if shape[0] <= 1 else st[0]), (0 if shape[1] == 1 else st[1])


Ranges = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _ranges(t: Ranges, name: str, index: int):
    """(batch, address of the first rows, address behind the last) of cumulated lengths or a pair."""
    if isinstance(t, torch.Tensor):
        if t.dim() != 1 or t.shape[0] == 0:
            raise StarKVError(f"{name} must be int32 (batch + 1,), or a pair of (batch,)")
        at = _ints(t, name, t.shape, index)
        return t.shape[0] - 1, at, at + 4
    start, end = t
    if start.dim() != 1:
        raise StarKVError(f"{name} must be int32 (batch + 1,), or a pair of (batch,)")
    return start.shape[0], _ints(start, name, start.shape, index), _ints(end, name, start.shape, index)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: Ranges, cu_k: Ranges, scaling: float,
                     causal: bool = True, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                     error_word: Optional[torch.Tensor] = None, ws: Optional[torch.Tensor] = None):
    """Attention of packed sequences: q (total_q, Hq, 128), k / v (total_k, Hkv, 128), fp16 or
    bf16, strides of rows and heads multiples of 8 elements.

    cu_q, cu_k: int32 (batch + 1,) cumulated lengths on the GPU (sequence b has rows cu[b] ..
    cu[b + 1] - 1), or a pair (first rows, rows behind the last), int32 (batch,) each, which may
    leave gaps, as left padding does, and name keys twice (rows of q
    belong to one sequence at most).  A sequence's newest query sits on its newest key: with n
    queries and m keys, query i attends to keys 0 .. m - n + i, or to all without ``causal``.

    Returns out of q's shape and dtype (or in ``out``, of any of the three types) and with
    ``return_lse`` the fp32 log-sum-exp (total_q, Hq); a query with nothing to attend to gets 0
    and -inf.  Rows of no sequence stay as they are in an ``out`` that is given; in a new one
    they are 0 (-inf) where ranges are pairs, and undefined before cu_q[0] and from cu_q[batch]
    on.  error_word: int32 (1,), set to a code of ``kv4.ERRORS`` where ranges leave the tensors
    (they are cut off there) or a copy never lands; without it the device has one, which
    ``read_packed_error`` reads.  ws: scratch of one's own,
    ``starkv_packed_workspace_size`` bytes, its first 4096 zeroed before its first use (each
    call leaves them zero)."""
    index = q.get_device()
    if index < 0:
        raise StarKVError("q must be a CUDA tensor")
    qs = _packed_rows(q, "q", _QUERY_DTYPES, index)
    ks = _packed_rows(k, "k", (q.dtype,), index)
    vs = _packed_rows(v, "v", (q.dtype,), index)
    if v.shape != k.shape or q.shape[1] % k.shape[1]:
        raise StarKVError(f"k and v must have one shape, and q's heads be a multiple of theirs: {tuple(q.shape)}, "
                          f"{tuple(k.shape)}, {tuple(v.shape)}")
    batch, q0, q1 = _ranges(cu_q, "cu_q", index)
    batch_k, k0, k1 = _ranges(cu_k, "cu_k", index)
    if batch != batch_k:
        raise StarKVError(f"cu_q has {batch} sequences, cu_k {batch_k}")
    total, heads = q.shape[0], q.shape[1]
    gaps = batch == 0 or not isinstance(cu_q, torch.Tensor)
    if out is None:
        if gaps:
            out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        else:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        os_ = (heads * 128, 128)
    else:
        if out.shape != q.shape:
            raise StarKVError(f"out must have shape {tuple(q.shape)}, got {tuple(out.shape)}")
        os_ = _packed_rows(out, "out", _TOKEN_DTYPES, index)
        _output(out, "out")
    lse = None
    if return_lse:
        lse = torch.empty_strided((total, heads), (heads, 1), dtype=torch.float32, device=q.device)
        if gaps:
            lse.fill_(float("-inf"))
    if ws is None:
        ws = _workspace("packed", index, _packed_size, 4096)
    elif ws.get_device() != index or not ws.is_contiguous():
        raise StarKVError(f"ws must be contiguous on cuda:{index}")
    err = 0 if error_word is None else _ints(error_word, "error_word", (1,), index)
    a = _PACKED.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
                     *qs, *ks, *vs, *os_, q0, q1, k0, k1, ws.data_ptr(), ws.numel() * ws.element_size(), err,
                     total, k.shape[0], scaling, _DT[q.dtype], _DT[out.dtype], batch, heads, k.shape[1], causal)
    fn = load().starkv_packed_attention
    if _device_now() == index:
        rc = fn(a, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = fn(a, _stream_of(index))
    if rc:
        check(rc, "starkv_packed_attention")
    return (out, lse) if return_lse else out


def read_packed_error(device="cuda") -> int:
    """Read and clear the device's error word of ``packed_attention`` calls that were given none, behind
    what the current stream holds (synchronises): 0, or a code of ``kv4.ERRORS``."""
    code = C.c_int(0)
    with torch.cuda.device(torch.device(device)):
        check(load().starkv_packed_read_error(C.byref(code), torch.cuda.current_stream().cuda_stream), "starkv_packed_read_error")
    return int(code.value)
