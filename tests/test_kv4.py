"""The paged 4-bit cache on a machine without a GPU: the argument blocks match the
library's structs, the host checks refuse, and the oracle's quantiser has the
properties its specification states."""

import ctypes as C

import numpy as np
import pytest
import torch

import kv4_oracle as O
from starkv import _lib, kv4


@pytest.mark.parametrize("which,mirror,packed", [(0, _lib.KV4Cache, kv4._CACHE), (1, _lib.KV4IoArgs, kv4._IO),
                                                 (2, _lib.KV4AttentionArgs, kv4._ATTENTION),
                                                 (3, _lib.KV4SelectArgs, kv4._SELECT)])
def test_argument_blocks(which, mirror, packed):
    assert _lib.load().starkv_kv4_struct_size(which) == C.sizeof(mirror) == packed.size
    # packed in field order, arrays spread out
    n = sum(f[1]._length_ if hasattr(f[1], "_length_") else 1 for f in mirror._fields_)
    got = mirror.from_buffer_copy(packed.pack(*range(1, n + 1)))
    flat = []
    for name, *_ in mirror._fields_:
        v = getattr(got, name)
        flat += list(v) if hasattr(v, "_length_") else [v]
    assert [int(x) for x in flat] == list(range(1, n + 1))


def test_no_cpu_path():
    with pytest.raises(_lib.StarKVError):
        kv4.KV4Cache(4, 2, device="cpu")
    lib = _lib.load()
    z = b"\0" * 256
    for fn in (lib.starkv_kv4_write, lib.starkv_kv4_read, lib.starkv_kv4_attention, lib.starkv_kv4_select):
        assert fn(z, z, None) == 1                              # null cache: refused before any CUDA call


@pytest.mark.parametrize("field,value,status", [("head_dim", 64, 2), ("page_size", 48, 2), ("num_pages", 0, 1),
                                                ("num_kv_heads", 0, 1), ("data", 8, 1), ("bounds", 0, 1)])
def test_pool_checks(field, value, status):
    c = _lib.KV4Cache(data=256, bounds=256, bound_scales=256, error_word=256, num_pages=4, num_kv_heads=2,
                      page_size=64, head_dim=128)
    setattr(c, field, value)
    a = _lib.KV4IoArgs()
    assert _lib.load().starkv_kv4_write(C.byref(c), C.byref(a), None) == status


def test_oracle_quantiser():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 128)) * 10.0 ** rng.uniform(-3, 3, (50, 1))
    x = x.astype(np.float16).astype(np.float64)
    c, s, m = O.quantise(x)
    assert c.min() == -8 and c.max() == 7
    g = x.reshape(50, 4, 32)
    # half a step, plus what rounding the centre to fp16 may cut off at an end
    room = 0.5 * s + np.abs(m) * 2.0 ** -11 + np.abs(s) * 16 * 2.0 ** -11 + 2.0 ** -24
    assert (np.abs(O.values(x).reshape(50, 4, 32) - g) <= room[..., None] * 1.01).all()
    assert (O.values(np.full((1, 128), 0.1)) == np.float64(np.float16(0.1))).all()


def test_oracle_bounds_hold():
    """A page's score is not below q.k of any of its tokens by more than the rounding of q."""
    rng = np.random.default_rng(1)
    page = O.values(rng.standard_normal((32, 128)))
    up, lo, t = O.bounds(page)
    assert (up * t >= page.max(0) - 1e-5).all() and (lo * t <= page.min(0) + 1e-5).all()
    q = rng.standard_normal((3, 128))
    u = np.abs(q).max(-1) / 127
    a = np.rint(q / u[:, None])
    score = (np.where(a > 0, a * up, a * lo).sum(-1) * u * t)
    slack = 0.5 * u * np.abs(page).sum(-1).max()
    assert (score >= (q @ page.T).max(-1) - slack - 1e-3).all()


def test_oracle_attention_is_softmax():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((2, 3, 128)), rng.standard_normal((9, 128)), rng.standard_normal((9, 128))
    out, lse, w = O.attend(q, k, v, 0.1)
    x = torch.from_numpy(q[1] @ k.T * 0.1)
    assert np.allclose(out[1], (torch.softmax(x, -1) @ torch.from_numpy(v)).numpy())
    assert np.allclose(lse[1], torch.logsumexp(x, -1).numpy())
    assert (w[0][:, 8] == 0).all() and np.allclose(w.sum(-1), 1)
    out, lse, _ = O.attend(q, k[:1], v[:1], 0.1)                # one token, two queries: the first sees nothing
    assert (out[0] == 0).all() and np.isneginf(lse[0]).all() and np.allclose(out[1], v[:1])


def test_decode_masks_of_every_kind():
    """Boolean and whole-number masks keep or drop positions; floating masks are added."""
    from starkv.attention import LlamaCustomAttention as A
    inf = float("inf")
    keep = torch.tensor([[False, True, True, True, True], [True, True, True, False, True]])
    want = torch.tensor([[-inf, 0, 0, 0], [0, 0, 0, -inf]])
    rows = torch.stack([torch.ones_like(keep), keep], 1)[:, None]      # (2, 1, 2, 5): the last row counts
    for m in (keep, keep.long(), keep.to(torch.uint8), rows, rows.int()):
        got = A._decode_mask(m, 2, 4)
        assert got.dtype == torch.float32 and got.is_contiguous() and torch.equal(got, want)
    assert torch.equal(A._decode_mask(keep[:1], 2, 4), want[:1].expand(2, 4))
    add = torch.tensor([[-inf, 0.5, -65504.0, 1.0]], dtype=torch.float16)
    for m in (add, add[:, None, None]):
        assert torch.equal(A._decode_mask(m, 2, 4), add.float().expand(2, 4))
    assert A._decode_mask(None, 2, 4) is None


def test_rows_that_differ_by_causality_only():
    from starkv.kv4_attention import causal_rows
    B, T, n = 2, 4, 9
    pad = torch.ones(B, 1, 1, n, dtype=torch.bool)
    pad[0, ..., :3] = False
    keep = pad & torch.ones(T, n, dtype=torch.bool).tril(n - T)
    wide = torch.cat([keep, torch.ones(B, 1, T, 2, dtype=torch.bool)], -1)     # columns past n do not count
    for dtype in (torch.bool, torch.float16, torch.float32):
        for m in (keep, wide):
            add = m if dtype == torch.bool else torch.zeros(m.shape, dtype=dtype).masked_fill(~m, torch.finfo(dtype).min)
            assert causal_rows(add, n)
    inf = torch.zeros(keep.shape).masked_fill(~keep, float("-inf"))
    assert causal_rows(inf, n)
    for at in ((0, 0, 1, 5), (1, 0, 0, 8), (0, 0, 0, 0)):         # a dropped one, a newer one seen, padding seen
        for m in (keep.clone(), inf.clone()):
            m[at] = not keep[at] if m.dtype == torch.bool else (float("-inf") if keep[at] else 0.0)
            assert not causal_rows(m, n)
    bias = inf.clone()
    bias[1, 0, 2, 4] = 0.5
    assert not causal_rows(bias, n)


def test_keep_pages_that_cannot_hold_the_first_and_the_newest():
    from types import SimpleNamespace
    from starkv.kv4_attention import KV4Attention
    cfg = SimpleNamespace(hidden_size=256, num_attention_heads=2, num_key_value_heads=1, attention_bias=False)
    for keep in (1, -1):
        with pytest.raises(ValueError):
            KV4Attention(cfg, keep_pages=keep)
    assert [KV4Attention(cfg, keep_pages=k).keep_pages for k in (0, 2, 64)] == [0, 2, 64]


def test_module_is_built_like_the_latent_ones():
    """The positional arguments mean the same in both, and the attributes that model code reads are there."""
    from transformers import LlamaConfig
    from starkv.attention import LlamaCustomAttention
    from starkv.kv4_attention import KV4Attention
    cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=2, attention_bias=False)
    a, b = LlamaCustomAttention(cfg, 3, 32), KV4Attention(cfg, 3, 32, keep_pages=2)
    for name in ("config", "layer_idx", "attention_dropout", "hidden_size", "num_heads", "num_key_value_heads",
                 "num_key_value_groups", "head_dim", "is_causal", "scaling", "decomp_goup_num"):
        assert getattr(a, name) == getattr(b, name), name
    assert b.page_size == 64 and b.keep_pages == 2
    assert KV4Attention(cfg, 3, page_size=32).page_size == 32
    with pytest.raises(TypeError):
        KV4Attention(cfg, 3, 1, 32)


@pytest.mark.parametrize("field,value", [("bounds", 264), ("bounds", 257), ("bound_scales", 258), ("error_word", 257)])
def test_pool_alignment(field, value):
    """The kernels store words of 16 and 4 bytes there."""
    c = _lib.KV4Cache(data=256, bounds=256, bound_scales=256, error_word=256, num_pages=4, num_kv_heads=2,
                      page_size=64, head_dim=128)
    setattr(c, field, value)
    lib = _lib.load()
    for fn, a in ((lib.starkv_kv4_write, _lib.KV4IoArgs()), (lib.starkv_kv4_read, _lib.KV4IoArgs()),
                  (lib.starkv_kv4_attention, _lib.KV4AttentionArgs()), (lib.starkv_kv4_select, _lib.KV4SelectArgs())):
        assert fn(C.byref(c), C.byref(a), None) == 1
        assert b"aligned" in lib.starkv_last_error()
