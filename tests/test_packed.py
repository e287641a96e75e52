"""Packed attention's refusals on the host (no CUDA calls)."""

import ctypes as C

import pytest
import torch

from starkv import _lib, prefill
from starkv._lib import StarKVError


def _args(**kw):
    a = _lib.PackedArgs()
    for i, name in enumerate(("q", "k", "v", "out", "workspace", "q_start", "q_end", "k_start", "k_end")):
        setattr(a, name, 0x1000 * (i + 1))
    for st, heads in ((a.q_strides, 8), (a.k_strides, 2), (a.v_strides, 2), (a.out_strides, 8)):
        st[0], st[1] = heads * 128, 128
    n = C.c_size_t(0)
    assert _lib.load().starkv_packed_workspace_size(C.byref(n)) == 0
    a.workspace_bytes = n.value
    a.total_q, a.total_k, a.batch, a.num_q_heads, a.num_kv_heads = 10, 20, 1, 8, 2
    a.scaling, a.dtype, a.out_dtype, a.causal = 0.1, _lib.F16, _lib.F16, 1
    for name, value in kw.items():
        if isinstance(value, tuple):
            getattr(a, name)[value[0]] = value[1]
        else:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("rc,kw", [
    (2, dict(dtype=_lib.F32)), (1, dict(out_dtype=9)), (1, dict(batch=-1)), (1, dict(total_q=-1)), (1, dict(total_k=-1)),
    (1, dict(num_q_heads=0)), (1, dict(num_kv_heads=0)), (1, dict(num_q_heads=7)), (2, dict(num_q_heads=258)), (2, dict(total_q=1 << 30)),
    (1, dict(scaling=0.0)), (1, dict(scaling=-1.0)), (1, dict(scaling=float("nan"))), (1, dict(scaling=float("inf"))),
    (1, dict(q=0)), (1, dict(k=0)), (1, dict(v=0)), (1, dict(out=0)), (1, dict(q_start=0)), (1, dict(k_end=0)), (1, dict(workspace=0)),
    (1, dict(q_end=0x7002)), (1, dict(lse=0x10001)), (1, dict(error_word=0x10002)), (4, dict(workspace_bytes=4096)), (4, dict(workspace=0x5008)),
    (1, dict(q=0x1008)), (1, dict(out=0x4004)), (1, dict(q_strides=(0, 1028))), (1, dict(k_strides=(1, -128))),
    (2, dict(k_strides=(0, 0))), (2, dict(v_strides=(1, 0))), (2, dict(out_strides=(1, 0)))])
def test_c_refusals(rc, kw):
    lib = _lib.load()
    a = _args(**kw)
    assert lib.starkv_packed_attention(C.byref(a), None) == rc
    assert lib.starkv_last_error()


def test_c_null():
    assert _lib.load().starkv_packed_attention(None, None) == 1
    assert _lib.load().starkv_packed_workspace_size(None) == 1


def test_c_read_error_null():
    assert _lib.load().starkv_packed_read_error(None, None) == 1


def test_no_cpu_path():
    q, cu = torch.zeros(4, 2, 128, dtype=torch.float16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(StarKVError):
        prefill.packed_attention(q, q, q, cu, cu, 1.0)
