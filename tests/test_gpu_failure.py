"""Device-side failure paths of the K kernel and of the 4-bit attention, made without
faulting the GPU.

A test hook shortens every device wait to 20 ms and makes the first CTA's
producer never issue one unit's staging copy.  The waits on that stage run
out; the kernel records an error code in the workspace's first word, its roles
leave their loops, wait (bounded) for their copies and MMAs in flight, free
TMEM and return.  The host reads the code, and the next normal step on the same
device still matches the oracle."""

import numpy as np
import pytest

import starkv_oracle as O
from starkv import ops
from starkv.harness import build_step
from starkv.synthetic import make_layer, make_spec

pytestmark = pytest.mark.gpu
REL_L2, MAX_ABS = 2e-3, 1e-2
DEV_WAIT_COPY, DEV_WAIT_MMA = 0x101, 0x102


def test_timed_out_wait_reports_and_the_device_recovers(cuda):
    spec = make_spec("c1", seed=31, num_q_heads=8, batch=2, context=3000)
    data = make_layer(spec)
    st = build_step(data, cuda)
    L = st.layer
    L.append(st.k_new, st.v_new)
    assert ops.read_device_error(device=cuda) == 0
    try:
        ops.set_test_hooks(wait_limit_ns=20_000_000, skip_copy_unit=1)
        L.attend(st.q)
        code = ops.read_device_error(device=cuda)
    finally:
        ops.set_test_hooks()
    assert code in (DEV_WAIT_COPY, DEV_WAIT_MMA), hex(code)
    out = L.attend(st.q, out=None).float().cpu().numpy()
    assert ops.read_device_error(device=cuda) == 0
    ref = O.layer_reference(data)
    assert O.rel_l2(out, ref) <= 1e-2           # model-dtype output (fp16)
    assert np.abs(out - ref).max() <= 2e-2


@pytest.mark.parametrize("lens,Hkv,G,Q,skip", [
    ([4000], 1, 4, 1, 0),                       # a tile a warp
    ([8000] * 4, 8, 1, 1, 0), ([8000] * 4, 8, 1, 1, 5), ([8000] * 4, 8, 1, 1, 6),   # the first, a later, a last tile of the ring
    ([5000, 3000, 1, 0, 77] * 8, 4, 4, 1, 3),   # segments that end inside the stretch
    ([6000] * 4, 8, 4, 4, 2),                   # 16 columns
])
@pytest.mark.parametrize("masked", [False, True])
def test_timed_out_tile_of_the_4_bit_attention(cuda, lens, Hkv, G, Q, skip, masked):
    """The copy of one tile is withheld: the call reports it and returns, and the next calls on
    the same workspace give what they gave before."""
    import torch
    from starkv.kv4 import KV4Cache
    B, n = len(lens), max(lens)
    W = -(-n // 64)
    g = torch.Generator(device=cuda).manual_seed(5)
    draw = lambda *s: torch.randn(*s, generator=g, device=cuda).half()  # noqa: E731
    cache = KV4Cache(B * W, Hkv, device=cuda)
    table = torch.arange(B * W, dtype=torch.int32, device=cuda).view(B, W)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
    cache.write(draw(B, n, Hkv, 128), draw(B, n, Hkv, 128), table, torch.zeros_like(lengths), lengths)
    q = draw(B, Q, Hkv * G, 128)
    mask = None
    if masked:
        mask = torch.zeros(B, n, device=cuda)
        mask[:, ::7] = float("-inf")
    attend = lambda: cache.attend(q, table, lengths, 128 ** -0.5, mask=mask, return_lse=True)  # noqa: E731
    want = attend()
    assert cache.read_error() == 0
    try:
        ops.set_test_hooks(wait_limit_ns=20_000_000, skip_copy_unit=skip)
        attend()
        assert cache.read_error() == DEV_WAIT_COPY
    finally:
        ops.set_test_hooks()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, attend()))
    assert cache.read_error() == 0
