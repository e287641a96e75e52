"""Rotary positions on the host: frequencies, their fixed-point form, refusals."""

import ctypes as C
import math

import pytest

from starkv import _lib, rope
from starkv.rope import rope_frequencies, rotary_channels, turns_of

LLAMA3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)
YARN = dict(rope_type="yarn", factor=32.0, original_max_position_embeddings=4096)


@pytest.mark.parametrize("dim,base,scaling", [(128, 10000.0, None), (64, 500000.0, LLAMA3), (128, 500000.0, LLAMA3),
                                              (128, 10000.0, YARN), (64, 1000000.0, dict(YARN, factor=4.0, beta_fast=16.0)),
                                              (128, 10000.0, dict(rope_type="linear", factor=4.0))])
def test_frequencies_are_those_of_transformers(dim, base, scaling):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    got, factor = rope_frequencies(dim, base, scaling)
    if scaling is None:
        want, wf = [base ** (-2 * i / dim) for i in range(dim // 2)], 1.0
    else:
        cfg = LlamaConfig(hidden_size=dim, num_attention_heads=1, head_dim=dim, max_position_embeddings=131072,
                          rope_parameters=dict(scaling, rope_theta=base))
        want, wf = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
        want = want.tolist()
    # theirs are fp32 through a few operations: some roundings of 2^-24, more where the exponent is far from 0
    assert factor == pytest.approx(wf, rel=1e-6)
    for a, b in zip(got, want):
        assert a == pytest.approx(b, rel=16 * 2.0 ** -24)


def test_turns():
    assert abs(turns_of([2 * math.pi])[0]) < 1 << 12    # a whole turn, as near as 64-bit floats have it
    for f in (1.0, 0.3, 1e-6, 5e-9, -0.25):
        t = turns_of([f])[0] % (1 << 64) / 2.0 ** 64
        assert math.sin(2 * math.pi * t) == pytest.approx(math.sin(f), rel=1e-12, abs=1e-18)
    # pi to 120 bits: sin of a large whole angle through the fixed point
    n = turns_of([1.0])[0] * 1000003 % (1 << 64)
    assert math.sin(2 * math.pi * (n / 2.0 ** 64)) == pytest.approx(math.sin(1000003.0), abs=1e-12)


@pytest.mark.parametrize("scaling", [dict(rope_type="longrope", factor=2.0), dict(rope_type="linear"), dict(rope_type="linear", factor=0.0),
                                     dict(LLAMA3, high_freq_factor=1.0), dict(YARN, mscale=1.0), dict(rope_type="yarn", factor=2.0)])
def test_scaling_refusals(scaling):
    with pytest.raises(_lib.StarKVError):
        rope_frequencies(64, 10000.0, scaling)


@pytest.mark.parametrize("kw", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=130), dict(frequencies=[1.0]),
                                dict(frequencies=[float("nan")] * 64), dict(base=1.0), dict(base=-1.0), dict(device="cpu"),
                                dict(frequencies=[1.0] * 64, scaling=LLAMA3)])
def test_constructor_refusals(kw):
    with pytest.raises(_lib.StarKVError):
        rope.Rope(128, **kw)


def _args(**kw):
    a = _lib.RopeArgs()
    a.x[0] = a.out[0] = 0x1000
    a.positions, a.turns = 0x2000, 0x3000
    a.batch, a.num_tokens, a.head_dim, a.rotary_dim, a.dtype = 1, 4, 128, 128, _lib.F16
    a.num_heads[0] = 2
    for name, value in kw.items():
        if isinstance(value, tuple):
            getattr(a, name)[value[0]] = value[1]
        else:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [dict(dtype=7), dict(rotary_dim=130), dict(rotary_dim=3), dict(rotary_dim=0), dict(batch=-1),
                                dict(num_tokens=-1), dict(num_heads=(0, -2)), dict(positions=0), dict(turns=0), dict(x=(0, 0)),
                                dict(out=(0, 0)), dict(num_heads=(1, 2)), dict(positions=0x2002), dict(turns=0x3004),
                                dict(x=(0, 0x1001)), dict(wide_positions=1, positions=0x2004)])
def test_c_refusals(kw):
    lib = _lib.load()
    a = _args(**kw)
    assert lib.starkv_rope(C.byref(a), None) == 1
    assert lib.starkv_last_error()


def test_c_negative_strides_refused():
    a = _args()
    a.x_strides[0][1] = -128
    assert _lib.load().starkv_rope(C.byref(a), None) == 1
    assert _lib.load().starkv_rope(None, None) == 1


@pytest.mark.parametrize("dim,base,scaling", [(64, 150000.0, dict(YARN, truncate=False)), (64, 150000.0, dict(YARN, truncate=True)),
                                              (64, 150000.0, dict(YARN, truncate=None)), (128, 10000.0, dict(YARN, truncate=False, beta_fast=16.0)),
                                              (128, 1000000.0, dict(YARN, truncate=False, factor=4.0, beta_slow=2.0)),
                                              (64, 500000.0, dict(LLAMA3, truncate=False))])
def test_truncate(dim, base, scaling):
    """Whether yarn's ramp begins and ends on whole pairs.  Theirs is fp32, off by 16 u (u = 2^-24) as above;
    and its ramp e = (i - lo) / (hi - lo) by u for the rounding of each end, u lo / (hi - lo) and
    u hi / (hi - lo), and for the subtraction, the division and 1 - e: 8 u where lo + hi <= 5 (hi - lo), as
    it is here.  The ramp is multiplied by the unscaled frequency, which is up to `factor` times the result."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    got, factor = rope_frequencies(dim, base, scaling)
    cfg = LlamaConfig(hidden_size=dim, num_attention_heads=1, head_dim=dim, max_position_embeddings=131072,
                      rope_parameters=dict(scaling, rope_theta=base))
    want, wf = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
    assert factor == pytest.approx(wf, rel=1e-6) and len(want) == len(got)
    for i, (a, b) in enumerate(zip(got, want.tolist())):
        assert abs(a - b) <= 2.0 ** -24 * (16 * b + 8 * base ** (-2 * i / dim))


@pytest.mark.parametrize("head,part", [(64, 0.5), (128, 0.25), (80, 0.4), (96, 1.0)])
@pytest.mark.parametrize("scaling", [dict(rope_type="default"), LLAMA3, YARN, dict(rope_type="linear", factor=4.0)])
def test_part_of_a_head(head, part, scaling):
    """A configuration's partial_rotary_factor says how many channels turn, as in transformers."""
    scaling = dict(scaling, partial_rotary_factor=part, rope_theta=500000.0)
    n = rotary_channels(head, None, scaling)
    assert n == int(head * part) == rotary_channels(head, n, scaling)
    got, _ = rope_frequencies(n, scaling=scaling)
    if scaling["rope_type"] == "default":
        want = [500000.0 ** (-2 * i / n) for i in range(n // 2)]
    else:
        from transformers import LlamaConfig
        from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
        cfg = LlamaConfig(hidden_size=head, num_attention_heads=1, head_dim=head, max_position_embeddings=131072, rope_parameters=scaling)
        want = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")[0].tolist()
    assert len(want) == len(got) == n // 2
    for a, b in zip(got, want):
        assert a == pytest.approx(b, rel=16 * 2.0 ** -24)
    for other in (n - 2, n + 2):
        with pytest.raises(_lib.StarKVError):
            rope.Rope(head, rotary_dim=other, scaling=scaling)


@pytest.mark.parametrize("part", [0.0, -0.5, 1.5, float("nan"), 0.02, 0.4])
def test_part_of_a_head_refusals(part):
    """Outside 0 to 1, or no even number of channels (1 and 25 of 64)."""
    with pytest.raises(_lib.StarKVError):
        rope.Rope(64, scaling=dict(rope_type="default", partial_rotary_factor=part))


@pytest.mark.parametrize("extra", [dict(mrope_section=[8, 12, 12]), dict(llama_4_scaling_beta=0.1), dict(some_new_factor=2.0)])
@pytest.mark.parametrize("scaling", [dict(rope_type="default"), LLAMA3, YARN])
def test_unknown_entries_are_refused(scaling, extra):
    with pytest.raises(_lib.StarKVError):
        rope_frequencies(64, 10000.0, dict(scaling, **extra))
    # a dictionary for each kind of layer is not one
    with pytest.raises(_lib.StarKVError):
        rope_frequencies(64, 10000.0, dict(full_attention=scaling, sliding_attention=dict(rope_type="default")))


def test_entries_without_a_say():
    """None counts as absent; what other types read, and notes, change nothing (nor do they in transformers)."""
    plain = rope_frequencies(64, 10000.0, YARN)
    assert rope_frequencies(64, 10000.0, dict(YARN, finetuned=True, max_position_embeddings=131072, low_freq_factor=2.0, some_new_factor=None,
                                              rope_theta=None, attention_factor=None, beta_fast=None)) == plain
    assert rope_frequencies(64, 10000.0, dict({k: v for k, v in YARN.items() if k != "rope_type"}, rope_type=None, type="yarn")) == plain
    assert rope_frequencies(64, 10000.0, dict(rope_type=None, factor=4.0)) == rope_frequencies(64)
