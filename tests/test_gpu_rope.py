"""Rotary positions on the GPU against the formula in 64 bits."""

import math

import pytest
import torch

from starkv._lib import StarKVError
from starkv.rope import Rope

pytestmark = pytest.mark.gpu

LLAMA3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)
YARN = dict(rope_type="yarn", factor=32.0, original_max_position_embeddings=4096)
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def reference(rope, x, positions, inverse=False):
    """The turned x in 64 bits. Angles: positions of up to 2^31 times frequencies of 53 bits, reduced by
    64-bit arithmetic: off by 2^-22 rad at 2^31, by 2^-33 at 10^6."""
    r = rope.rotary_dim
    f = torch.tensor(rope.frequencies, dtype=torch.float64, device=x.device)
    lead = x.shape[:-2]
    angle = positions.to(torch.float64).expand(lead)[..., None, None] * f
    c, s = torch.cos(angle) * rope.factor, torch.sin(angle) * rope.factor
    if inverse:
        s = -s
    y = x.double().clone()
    one, two = (slice(0, r, 2), slice(1, r, 2)) if rope.interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = y[..., one].clone(), y[..., two].clone()
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size = torch.zeros_like(y)
    size[..., one] = size[..., two] = (a.abs() + b.abs()) * rope.factor
    return y, size


def close(got, want, size, angle=0.0):
    """Half a step of the type for the last rounding, and inside fp32: the fraction of a turn has 24 bits
    (pi 2^-24), sine and cosine 2 units of 2^-24, factor, product and sum one each: below 2^-20 of
    |a| + |b| in all. Half a step of fp16 is at least 2^-25 in absolute terms."""
    eps = torch.finfo(got.dtype).eps / 2
    bound = eps * (want.abs() + 2.0 ** -20 * size) + (2.0 ** -20 + angle) * size + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


def make(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head,rotary", [(128, 128), (128, 64), (128, 32), (64, 24), (80, 32), (96, 2), (256, 256), (6, 6), (5, 2), (7, 6)])
def test_layouts(cuda, dtype, interleaved, head, rotary):
    rope = Rope(head, rotary_dim=rotary, interleaved=interleaved)
    q, k = make((2, 5, 3, head), dtype), make((2, 5, 1, head), dtype, 1)
    pos = torch.tensor([[0, 1, 2, 3, 4], [777, 131071, 5, 5, 1000000]], device=cuda)
    a, b = rope.apply(q, k, pos)
    for got, x in ((a, q), (b, k)):
        close(got, *reference(rope, x, pos))
        assert torch.equal(got[..., rotary:], x[..., rotary:])
    assert torch.equal(rope.apply(q, None, pos), a)


@pytest.mark.parametrize("tokens,heads", [(1, (32, 8)), (1, (1, 1)), (3, (71, 1)), (257, (5, 5)), (2049, (32, 8)), (1, (300, 300))])
@pytest.mark.parametrize("scaling", [None, LLAMA3, YARN])
def test_sizes(cuda, tokens, heads, scaling):
    rope = Rope(128, base=500000.0, scaling=scaling)
    q, k = make((tokens, heads[0], 128), torch.bfloat16), make((tokens, heads[1], 128), torch.bfloat16, 1)
    pos = torch.arange(tokens, device=cuda, dtype=torch.int32) + 4000
    a, b = rope.apply(q, k, pos)
    close(a, *reference(rope, q, pos))
    close(b, *reference(rope, k, pos))


def test_far_and_negative_positions(cuda):
    rope = Rope(128)
    q = make((6, 2, 128), torch.float32)
    pos = torch.tensor([0, -1, -1000000, 2 ** 31 - 1, -2 ** 31, 16777217], device=cuda, dtype=torch.int32)
    close(rope.apply(q, None, pos), *reference(rope, q, pos), angle=2.0 ** -21)
    assert torch.equal(rope.apply(q, None, pos), rope.apply(q, None, pos.long()))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_in_place_and_broadcast_positions(cuda, dtype):
    rope = Rope(128, rotary_dim=96)
    fused = make((2, 9, 12 * 128), dtype)
    q, k = fused[..., :8 * 128].view(2, 9, 8, 128), fused[..., 8 * 128:10 * 128].view(2, 9, 2, 128)
    before, v = fused.clone(), fused[..., 10 * 128:].clone()
    pos = torch.arange(9, device=cuda)
    a, b = rope.apply(q, k, pos)
    wide = rope.apply(q, k, torch.stack([pos, pos]))
    assert torch.equal(a, wide[0]) and torch.equal(b, wide[1]) and torch.equal(fused, before)
    # heads ahead of tokens, odd offsets that leave only single elements aligned
    t = rope.apply(q.transpose(1, 2).contiguous().transpose(1, 2), None, pos)
    assert torch.equal(t, a)
    odd = torch.empty(q.numel() + 1, dtype=dtype, device=cuda)[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(rope.apply(odd, None, pos), a)
    got = rope.apply(q, k, pos, out=(q, k))
    assert got[0] is q and torch.equal(q, a) and torch.equal(k, b) and torch.equal(fused[..., 10 * 128:], v)


def test_inverse_is_the_transposed_map(cuda):
    """<y, R x> = <R' y, x>: the inverse is the gradient; and it undoes the turn where the factor is 1."""
    for kw in (dict(), dict(interleaved=True, rotary_dim=64), dict(scaling=YARN)):
        rope = Rope(128, **kw)
        x, y = make((33, 4, 128), torch.float32), make((33, 4, 128), torch.float32, 1)
        pos = torch.arange(33, device=cuda) * 1013
        a = (y.double() * rope.apply(x, None, pos).double()).sum()
        b = (rope.apply(y, None, pos, inverse=True).double() * x.double()).sum()
        # 33 * 4 * 128 terms of about one, each off by up to 2^-20
        assert abs(float(a - b)) < 33 * 4 * 128 * 2.0 ** -20
        close(rope.apply(x, None, pos, inverse=True), *reference(rope, x, pos, inverse=True))
        # differences: the map is linear, so a step of any size gives its derivative
        d = torch.autograd.functional.jvp(lambda t: reference(rope, t, pos)[0], x.double(), y.double())[1]
        assert float((rope.apply(x + y, None, pos).double() - rope.apply(x, None, pos).double() - d).abs().max()) < 2.0 ** -17
        if rope.factor == 1.0:
            back = rope.apply(rope.apply(x, None, pos), None, pos, inverse=True)
            assert float((back - x).abs().max()) < 2.0 ** -18


def test_not_finite_stays_in_its_pair(cuda):
    rope = Rope(128)
    x = make((4, 2, 128), torch.bfloat16)
    y = x.clone()
    y[2, 1, 5], y[1, 0, 100] = float("nan"), float("inf")
    pos = torch.arange(4, device=cuda) + 7
    a, b = rope.apply(x, None, pos), rope.apply(y, None, pos)
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[2, 1, [5, 69]] = touched[1, 0, [100, 36]] = True
    assert torch.equal(a[~touched], b[~touched])
    assert bool(b[2, 1, [5, 69]].isnan().all()) and not bool(b[1, 0, [100, 36]].isfinite().any())


def test_given_frequencies_and_empty(cuda):
    f = torch.tensor([1.0, 0.1, 1e-3, 2 * math.pi + 0.25])
    rope = Rope(8, frequencies=f, factor=1.5)
    x = make((1, 40, 3, 8), torch.float32)
    pos = torch.arange(40, device=cuda)
    close(rope.apply(x, None, pos), *reference(rope, x, pos))
    assert rope.apply(x[:, :0], None, pos[:0]).shape == (1, 0, 3, 8)
    assert rope.apply(x[:0], None, pos).shape == (0, 40, 3, 8)


def test_stream_and_graph(cuda):
    rope = Rope(128)
    q, k = make((1, 1, 32, 128), torch.float16), make((1, 1, 8, 128), torch.float16, 1)
    pos = torch.zeros(1, 1, dtype=torch.int64, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope.apply(q, k, pos)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, b = rope.apply(q, k, pos)
        pos.add_(1)
    for i in range(3):
        g.replay()
        want = rope.apply(q, k, torch.full_like(pos, i))
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_strides_beyond_31_bits(cuda):
    rope = Rope(128)
    big = torch.zeros(2 ** 32 + 4096, dtype=torch.float16, device="cuda")
    x = big.as_strided((2, 2, 2, 128), (2 ** 31 + 1024, 2 ** 31 + 1024 - 512, 128, 1), 8)
    x[:, :, 0], x[:, :, 1] = make((128,), torch.float16), make((128,), torch.float16, 1)
    before, pos = x.clone(), torch.tensor([[5], [6]], device=cuda)
    x, before = x[:, 1:], before[:, 1:]
    a = rope.apply(x, None, pos)
    close(a, *reference(rope, before, pos))
    assert rope.apply(x, None, pos, out=x) is x and torch.equal(x, a)


def test_calls_of_one_shape(cuda):
    """A shape's second call gives what the first would, for other tensors, values and directions, and
    refuses what the first would."""
    rope = Rope(128, scaling=LLAMA3)
    pos = torch.tensor([[7], [123456]], device=cuda)
    for i in range(3):
        q, k = make((2, 1, 4, 128), torch.float16, 2 * i), make((2, 1, 2, 128), torch.float16, 2 * i + 1)
        for inverse in (False, True):
            a, b = rope.apply(q, k, pos + i, inverse=inverse)
            assert a.data_ptr() not in (q.data_ptr(), k.data_ptr()) and b.data_ptr() not in (q.data_ptr(), k.data_ptr())
            for got, x in ((a, q), (b, k)):
                close(got, *reference(rope, x, pos + i, inverse))
            c, d = q.clone(), k.clone()
            e, f = rope.apply(c, d, pos + i, inverse=inverse, out=(c, d))
            assert e is c and f is d and torch.equal(c, a) and torch.equal(d, b)
            for wide in (pos.int() + i, (pos + i).expand(2, 1), (pos[:1] + i)[:, 0]):
                if wide.shape == (1,):
                    assert torch.equal(rope.apply(q[:1], k[:1], wide, inverse=inverse)[0], a[:1])
                else:
                    assert torch.equal(rope.apply(q, k, wide, inverse=inverse)[1], b)
        packed = make((2, 1, 6, 128), torch.float16, i)                    # strides of a joint projection
        a, b = rope.apply(packed[:, :, :4], packed[:, :, 4:], pos)
        close(a, *reference(rope, packed[:, :, :4], pos))
        close(b, *reference(rope, packed[:, :, 4:], pos))
        same = make((2, 1, 4, 128), torch.float16)
        rope.apply(same, same.clone(), pos), rope.apply(same, same, pos)
        ok = same.clone()
        rope.apply(same, ok, pos, out=(same, ok))
        for bad in (lambda: rope.apply(same, same, pos, out=(same, same)), lambda: rope.apply(same, ok, pos.cpu()),
                    lambda: rope.apply(same.cpu(), ok, pos), lambda: rope.apply(same, ok.cpu(), pos),
                    lambda: rope.apply(same, ok.bfloat16(), pos), lambda: rope.apply(same, ok, pos.float())):
            with pytest.raises(StarKVError):
                bad()
    for n in range(1, 80):                                                 # more shapes than are kept
        x = make((1, n, 1, 128), torch.bfloat16, n)
        a, b = rope.apply(x, x, torch.arange(n, device=cuda))
        assert torch.equal(a, b) and torch.equal(a, rope.apply(x, None, torch.arange(n, device=cuda)))


def test_refusals(cuda):
    rope = Rope(128)
    q, pos = make((2, 3, 4, 128), torch.float16), torch.zeros(2, 3, dtype=torch.int64, device=cuda)
    for bad in (lambda: rope.apply(q.double(), None, pos), lambda: rope.apply(q, q.float(), pos),
                lambda: rope.apply(q[..., :64], None, pos), lambda: rope.apply(q, q[:1], pos), lambda: rope.apply(q, None, pos.float()),
                lambda: rope.apply(q, None, pos[:, :2]), lambda: rope.apply(q, None, pos.cpu()), lambda: rope.apply(q.cpu(), None, pos),
                lambda: rope.apply(q.transpose(-1, -2), None, pos), lambda: rope.apply(q, None, pos, out=q[:, :, :2]),
                lambda: rope.apply(q, None, pos, out=q[:, :1].expand(2, 3, 4, 128)),
                lambda: rope.apply(q[:, :2], None, pos[:, :2], out=q[:, 1:]), lambda: rope.apply(q, q.clone(), pos, out=(q,)),
                lambda: rope.apply(q, q.clone(), pos, out=(q, q))):
        with pytest.raises(StarKVError):
            bad()


def test_part_of_a_head_from_the_scaling(cuda):
    """The constructor takes the turned channels from partial_rotary_factor."""
    rope = Rope(128, scaling=dict(YARN, rope_theta=500000.0, truncate=False, partial_rotary_factor=0.25))
    assert rope.rotary_dim == 32
    q, pos = make((9, 3, 128), torch.float32), torch.arange(9, device=cuda) * 1000
    got = rope.apply(q, None, pos)
    close(got, *reference(rope, q, pos))
    assert torch.equal(got[..., 32:], q[..., 32:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("needs", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("kw", [dict(), dict(interleaved=True, rotary_dim=64, scaling=YARN)])
def test_gradients(cuda, dtype, needs, kw):
    """Against the formula: the transposed map, that is the inverse turn, with one rounding."""
    rope = Rope(128, **kw)
    x = [make((2, 5, h, 128), dtype, h).requires_grad_(n) for h, n in zip((4, 2), needs)]
    pos = torch.tensor([[0, 3, 77, 5, 9], [1, 2, 3, 4, 100000]], device=cuda)
    for inverse in (False, True):
        got = rope.apply(*x, pos, inverse=inverse)
        with torch.no_grad():
            plain = rope.apply(*x, pos, inverse=inverse)
        assert all(torch.equal(a, b) for a, b in zip(got, plain)) and not any(b.requires_grad for b in plain)
        assert got[0].grad_fn is not None and got[1].grad_fn is got[0].grad_fn
        up = [make(t.shape, dtype, 7 + i) for i, t in enumerate(got)]
        sides = [i for i in (0, 1) if needs[i]]
        grads = torch.autograd.grad(got, [x[i] for i in sides], up)
        for i, g in zip(sides, grads):
            close(g, *reference(rope, up[i], pos, inverse=not inverse))
    # one side, and a gradient that is one repeated number
    if needs[0]:
        g, = torch.autograd.grad(rope.apply(x[0], None, pos).sum(), x[0])
        close(g, *reference(rope, torch.ones_like(g), pos, inverse=True))


def test_gradients_by_differences(cuda):
    """The map is linear: the difference of two calls is the derivative along their distance, but for
    the calls' own errors (2^-20 of some values of one to eight, 9 * 3 * 128 of them times |up|)."""
    rope = Rope(128, scaling=YARN)
    x, d, up = (make((9, 3, 128), torch.float32, i) for i in range(3))
    pos = torch.arange(9, device=cuda) * 311
    x.requires_grad_()
    y = rope.apply(x, None, pos)
    g, = torch.autograd.grad(y, x, up, create_graph=True)
    with torch.no_grad():
        want = (up.double() * (rope.apply(x + d, None, pos).double() - y.double())).sum()
    assert abs(float((g.detach().double() * d.double()).sum() - want)) < 9 * 3 * 128 * 2.0 ** -18
    # the gradient's gradient: of <g, d> by up, the turned d
    up2 = up.clone().requires_grad_()
    g, = torch.autograd.grad(rope.apply(x, None, pos), x, up2, create_graph=True)
    back, = torch.autograd.grad(g, up2, d)
    close(back, *reference(rope, d, pos))


def test_gradient_refusals(cuda):
    rope = Rope(128)
    q, k, pos = make((3, 4, 128), torch.float32), make((3, 2, 128), torch.float32, 1), torch.arange(3, device=cuda)
    leaf = q.clone().requires_grad_()
    before = k.clone()
    for bad in (lambda: rope.apply(leaf, k, pos, out=(leaf, k)), lambda: rope.apply(k, leaf, pos, out=(k, leaf)),
                lambda: rope.apply(leaf, None, pos, out=torch.empty_like(q)), lambda: rope.apply(q, None, pos, out=torch.empty_like(leaf).requires_grad_()),
                lambda: rope.apply(k, leaf * 1, pos, out=[k, torch.empty_like(q)])):
        with pytest.raises(StarKVError):
            bad()
    assert torch.equal(k, before) and torch.equal(leaf.detach(), q)
    with torch.no_grad():                                                  # nothing is recorded: in place as asked
        want = rope.apply(leaf, None, pos)
        assert torch.equal(rope.apply(leaf, None, pos, out=leaf), want)
    # positions that were written in between are not those of the call
    leaf = q.clone().requires_grad_()
    y = rope.apply(leaf, k, pos)
    pos.add_(1)
    with pytest.raises(RuntimeError):
        y[0].sum().backward()


def test_an_output_over_the_other_side_is_refused(cuda):
    rope = Rope(128)
    buf = make((2, 6, 8, 128), torch.float16)
    pos = torch.arange(6, device=cuda)
    q, k = buf[0], make((6, 8, 128), torch.float16, 1)
    for oq, ok in ((torch.empty_like(q), buf.view(-1)[128:128 + k.numel()].view(k.shape)),             # ok over q, a head on
                   (torch.empty_like(q), buf.view(12, 8, 128)[5:11])):                                              # and by its last token
        with pytest.raises(StarKVError):
            rope.apply(q, k, pos, out=(oq, ok))
        with pytest.raises(StarKVError):
            rope.apply(k, q, pos, out=(ok, oq))
    # behind the other side's input, into the two halves of one buffer, and in place between one another
    a, b = rope.apply(q, k, pos)
    ok = buf[1]
    rope.apply(q, k, pos, out=(torch.empty_like(q), ok))
    assert torch.equal(ok, b)
    both = torch.empty(6, 16, 128, dtype=torch.float16, device=cuda)
    rope.apply(q, k, pos, out=(both[:, :8], both[:, 8:]))
    assert torch.equal(both[:, :8], a) and torch.equal(both[:, 8:], b)
    both = torch.cat([q, k], 1)
    rope.apply(both[:, :8], both[:, 8:], pos, out=(both[:, :8], both[:, 8:]))
    assert torch.equal(both[:, :8], a) and torch.equal(both[:, 8:], b)
