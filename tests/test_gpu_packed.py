"""Packed attention on the GPU against the formula in 64 bits."""

import math

import pytest
import torch

from starkv import _lib, prefill
from starkv._lib import StarKVError
from starkv.prefill import packed_attention

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def make(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def cumulated(lengths):
    return torch.tensor([0, *lengths], device="cuda").cumsum(0).to(torch.int32)


def reference(q, k, v, rq, rk, scale=SCALE, causal=True):
    """out, lse, and what their errors scale with: sum of w |v|, the largest sum of |q k|. Masked keys
    are left out, whatever they hold."""
    G = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    size, grown = torch.zeros_like(out), torch.zeros_like(lse)
    for (q0, q1), (k0, k1) in zip(rq, rk):
        n, m = q1 - q0, k1 - k0
        for h in range(q.shape[1]):
            a, b, c = q[q0:q1, h].double(), k[k0:k1, h // G].double(), v[k0:k1, h // G].double()
            seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
            if causal:
                seen = seen.tril(m - n)
            rows = seen.any(1)
            if not bool(rows.any()):
                continue
            s = (a @ b.T * scale).masked_fill(~seen, -math.inf)
            w = torch.softmax(s[rows], -1)
            # the product over what is seen only: 0 * NaN does not count
            clean = torch.where(c.isfinite(), c, torch.zeros_like(c))
            o = w @ clean
            for key in (~c.isfinite()).any(1).nonzero()[:, 0].tolist():
                odd = torch.where(c[key].isfinite(), torch.zeros_like(c[key]), c[key])
                o += torch.where(seen[rows][:, key, None], odd, torch.zeros_like(odd))
            at = q0 + rows.nonzero()[:, 0]
            out[at, h], lse[at, h] = o, torch.logsumexp(s[rows], -1)
            size[at, h] = w @ clean.abs()
            grown[at, h] = (a.abs() @ b.abs().T * scale).masked_fill(~seen, 0).amax(1)[rows]
    return out, lse, size, grown


def close(got, lse, want, dtype, keys):
    """Scores: 128 products in 8 matrix instructions, each sum off by 2^-22 of what is summed, 2^-19
    of sum |q k| in all; the exponential 2^-20. Both move a weight and the sum of the weights. The
    weight's rounding is half a step, the output's too; a weight is held to 2^-34 of the row's
    largest at least (fp16)."""
    out, want_lse, size, grown = want
    eps = torch.finfo(dtype).eps / 2
    d = (grown * 2.0 ** -19 + 2.0 ** -20)[..., None]
    top = size.amax(-1, keepdim=True)
    last = torch.finfo(got.dtype).eps / 2
    bound = (eps + 2 * d) * size * 1.01 + last * out.abs() * 1.01 + keys * 2.0 ** -33 * top + 2.0 ** -25
    off = (got.double() - out).abs()
    finite = out.isfinite()
    assert bool((off <= bound)[finite].all()), float((off / bound)[finite].max())
    odd = ~finite
    assert torch.equal(got[odd].double().nan_to_num(7e7, 8e8, -8e8), out[odd].nan_to_num(7e7, 8e8, -8e8))
    if lse is not None:
        live = want_lse > -math.inf
        assert torch.equal(lse > -math.inf, live)
        lb = d[..., 0] * 2 + want_lse.abs() * 2.0 ** -22
        assert bool(((lse.double() - want_lse).abs() <= lb)[live].all())
    assert not bool(got[size.sum(-1) == 0][:, :0].any())


def run_case(nq, nk, heads, dtype, causal=True, seed=0, out_dtype=None):
    q, k, v = make((sum(nq), heads[0], 128), dtype, seed), make((sum(nk), heads[1], 128), dtype, seed + 1), make((sum(nk), heads[1], 128), dtype, seed + 2)
    cq, ck = cumulated(nq), cumulated(nk)
    out = None if out_dtype is None else torch.empty(q.shape, dtype=out_dtype, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got, lse = packed_attention(q, k, v, cq, ck, SCALE, causal=causal, out=out, return_lse=True, error_word=err)
    assert int(err) == 0
    pairs = lambda c: list(zip(c.tolist()[:-1], c.tolist()[1:]))  # noqa: E731
    close(got, lse, reference(q, k, v, pairs(cq), pairs(ck), causal=causal), dtype, max(nk))
    return q, k, v, cq, ck, got, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
def test_one_prompt(cuda, dtype, n):
    run_case([n], [n], (4, 2), dtype)


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 8), (5, 5), (14, 2), (12, 4), (71, 1), (128, 1), (65, 1), (32, 8)])
def test_head_layouts(cuda, heads):
    run_case([1, 100, 0, 37], [1, 100, 0, 300], heads, torch.bfloat16)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk", [([5, 0, 300, 1], [5, 0, 300, 1]), ([1, 1, 1], [1000, 1, 0]), ([10, 200], [3, 130]), ([300, 300], [0, 129]),
                                   ([0], [50]), ([64], [5000]), ([1], [20000]), ([700, 3], [2000, 3000]), ([130] * 9, [0, 1, 127, 128, 129, 130, 131, 256, 257])])
def test_ragged(cuda, nq, nk, causal):
    run_case(nq, nk, (8, 2), torch.float16, causal)


def test_many_sequences(cuda):
    nq = [(i * 7) % 5 for i in range(1500)]
    nk = [n + (i * 13) % 40 for i, n in enumerate(nq)]
    run_case(nq, nk, (4, 2), torch.bfloat16)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_output_types(cuda, out_dtype):
    run_case([200, 33], [200, 700], (4, 1), torch.bfloat16, out_dtype=out_dtype)


def test_same_result_every_time_and_clear_workspace(cuda):
    q, k, v, cq, ck, got, lse = run_case([64, 1, 17], [9000, 16384, 30], (8, 2), torch.bfloat16)
    ws = torch.zeros(prefill._packed_size(), dtype=torch.uint8, device="cuda")
    for _ in range(5):
        again, l2 = packed_attention(q, k, v, cq, ck, SCALE, return_lse=True, ws=ws)
        assert torch.equal(again, got) and torch.equal(l2, lse)
        assert not bool(ws[:4096].any())


def test_strided_inputs_and_rows_left_alone(cuda):
    fused = make((300, 12 * 128), torch.float16)
    q, k, v = fused[:, :8 * 128].view(300, 8, 128), fused[:, 8 * 128:10 * 128].view(300, 2, 128), fused[:, 10 * 128:].view(300, 2, 128)
    cu = torch.tensor([10, 140, 250], dtype=torch.int32, device="cuda")
    out = torch.full((300, 8, 256), 3.0, dtype=torch.float16, device="cuda")[..., :128]
    got = packed_attention(q, k, v, cu, cu, SCALE, out=out)
    assert got is out and bool((out[:10] == 3).all()) and bool((out[250:] == 3).all())
    close(out[10:250], None, [t[10:250] for t in reference(q, k, v, [(10, 140), (140, 250)], [(10, 140), (140, 250)])], torch.float16, 140)
    # heads ahead of rows
    t = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    assert torch.equal(packed_attention(t(q), t(k), t(v), cu, cu, SCALE)[10:250], out[10:250])


def test_rows_beyond_31_bits(cuda):
    """Rows of one tensor that reach 2.4e9 elements: keys, values, queries and outputs; with history
    enough to be cut among the SMs."""
    rows, wide = 600_000, 4096
    big = torch.empty(rows, wide, dtype=torch.float16, device="cuda")
    view = lambda at: big[:, at:at + 128].view(rows, 1, 128)  # noqa: E731
    k, v, q, out = (view(at) for at in (0, 128, 256, 512))
    for i, x in enumerate((k, v, q)):
        x.copy_(make((rows, 1, 128), torch.float16, i))
    out.fill_(7.0)
    first, n = rows - 20_000, 70
    v[-5, 0, 3] = math.inf                                        # an odd value near the end
    rq, rk = [(rows - n, rows)], [(first, rows)]
    pair = lambda r: tuple(torch.tensor([x[i] for x in r], dtype=torch.int32, device="cuda") for i in (0, 1))  # noqa: E731
    got, lse = packed_attention(q, k, v, pair(rq), pair(rk), SCALE, out=out, return_lse=True)
    assert got is out and bool((out[:rows - n] == 7.0).all())
    want = reference(q[-n:].contiguous(), k[first:].contiguous(), v[first:].contiguous(), [(0, n)], [(0, rows - first)])
    close(got[-n:].contiguous(), lse[-n:], want, torch.float16, rows - first)


def test_pairs_of_ranges_as_left_padding(cuda):
    B, T = 3, 200
    q, k, v = (make((B * T, h, 128), torch.bfloat16, h) for h in (4, 2, 2))
    k2 = make((B * T, 2, 128), torch.bfloat16, 9)
    pad = torch.tensor([0, 77, 199], dtype=torch.int32, device="cuda")
    ends = torch.arange(1, B + 1, dtype=torch.int32, device="cuda") * T
    starts = ends - T + pad
    r = list(zip(starts.tolist(), ends.tolist()))
    dirty = [x.clone() for x in (q, k, k2)]
    for b, n in enumerate(pad.tolist()):
        for x in dirty:
            x[b * T:b * T + n] = float("nan")
    out, lse = packed_attention(*dirty, (starts, ends), (starts, ends), SCALE, return_lse=True)
    close(out, lse, reference(q, k, k2, r, r), torch.bfloat16, T)
    for b, n in enumerate(pad.tolist()):
        assert not bool(out[b * T:b * T + n].any()) and bool((lse[b * T:b * T + n] == -math.inf).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nk", [([300, 50], [300, 50]), ([40, 3], [4000, 700])])
def test_not_finite_stays_with_those_that_see_it(cuda, dtype, nq, nk):
    q, k, v = make((sum(nq), 4, 128), dtype), make((sum(nk), 2, 128), dtype, 1), make((sum(nk), 2, 128), dtype, 2)
    v[nk[0] - 20, 1, 7], v[nk[0] - 3, 0, 100], v[nk[0] + 5, 0, 3] = float("nan"), float("inf"), float("-inf")
    v[nk[0] - 1, 0, 100], v[10, 0, 64] = float("-inf"), float("inf")
    k[nk[0] - 5, 1, 9], k[nk[0] + 48] = float("nan"), float("inf")
    pairs = lambda n: [(0, n[0]), (n[0], n[0] + n[1])]  # noqa: E731
    got, lse = packed_attention(q, k, v, cumulated(nq), cumulated(nk), SCALE, return_lse=True)
    want = reference(q, k, v, pairs(nq), pairs(nk))
    # rows that see a NaN or infinite key are NaN as a whole
    bad = want[1].isnan() | (want[1] == math.inf) | want[3].isnan()
    assert bool(bad.any()) and not bool(bad.all())
    assert bool(got[bad].isnan().all()) and bool(lse[bad].isnan().all())
    ok = ~bad
    close(got[ok], lse[ok], [t[ok] for t in want], dtype, max(nk))


def test_extreme_scores(cuda):
    for scale, big in ((SCALE, 60.0), (1e-30, 1.0), (30.0, 1.0), (1e-6, 200.0)):
        q, k, v = make((70, 2, 128), torch.bfloat16) * big, make((500, 1, 128), torch.bfloat16, 1), make((500, 1, 128), torch.bfloat16, 2)
        cq, ck = cumulated([70]), cumulated([500])
        got, lse = packed_attention(q, k, v, cq, ck, scale, return_lse=True)
        close(got, lse, reference(q, k, v, [(0, 70)], [(0, 500)], scale=scale), torch.bfloat16, 500)
    # scores far beyond what fp32 resolves: the largest takes all, and nothing overflows
    q = make((70, 2, 128), torch.bfloat16) * 1e30
    got, lse = packed_attention(q, k, v, cq, ck, SCALE, return_lse=True)
    best = (q[:, 0].double() @ k[:, 0].double().T).masked_fill(~torch.ones(70, 500, dtype=torch.bool, device="cuda").tril(430), -math.inf).argmax(1)
    assert torch.equal(got[:, 0], v[best, 0]) and bool(lse.isfinite().all())
    # scores that fall along the keys, and rise: the reference never, or always, moves
    for sign in (1, -1):
        q = torch.ones(1, 1, 128, dtype=torch.float16, device="cuda")
        k = (torch.linspace(3, -3, 700, device="cuda") * sign)[:, None, None].expand(700, 1, 128).half().contiguous()
        v = make((700, 1, 128), torch.float16)
        got, lse = packed_attention(q, k, v, cumulated([1]), cumulated([700]), SCALE, return_lse=True)
        close(got, lse, reference(q, k, v, [(0, 1)], [(0, 700)]), torch.float16, 700)


def test_long_tail_of_small_weights(cuda):
    """One key outweighs each of 30000 others by 2^25: together they still count (fp16 weights
    relative to the largest alone would all round to nothing)."""
    n = 30001
    k = torch.zeros(n, 1, 128, dtype=torch.float16, device="cuda")
    k[777, 0, 0] = 25 * math.log(2.0)
    q = torch.zeros(1, 1, 128, dtype=torch.float16, device="cuda")
    q[0, 0, 0] = 1
    v = torch.full((n, 1, 128), 1000.0, dtype=torch.float16, device="cuda")
    v[777] = 0
    got, lse = packed_attention(q, k, v, cumulated([1]), cumulated([n]), 1.0, return_lse=True, out=torch.empty(1, 1, 128, device="cuda"))
    w = math.exp(-float(k[777, 0, 0]))
    want = 1000.0 * 30000 * w / (1 + 30000 * w)
    assert float(got[0, 0, 0]) == pytest.approx(want, rel=2.0 ** -8)     # 2^-34 absolute in 2^-25: 2^-9 each


def test_bad_ranges_are_cut_off(cuda):
    q, k, v = make((50, 2, 128), torch.float16), make((80, 1, 128), torch.float16, 1), make((80, 1, 128), torch.float16, 2)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = packed_attention(q, k, v, (i(0, 30, 45), i(20, 99, 40)), (i(0, -5, 0), i(20, 1000, 9)), SCALE, error_word=err)
    assert int(err) == 0x203
    close(out, None, reference(q, k, v, [(0, 20), (30, 50)], [(0, 20), (0, 80)]), torch.float16, 80)


def test_empty_calls(cuda):
    q, k = make((0, 2, 128), torch.float16), make((9, 1, 128), torch.float16)
    assert packed_attention(q, k, k, cumulated([0]), cumulated([9]), SCALE).shape == (0, 2, 128)
    q = make((9, 2, 128), torch.float16)
    out, lse = packed_attention(q, k[:0], k[:0], cumulated([9]), cumulated([0]), SCALE, return_lse=True)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not bool(packed_attention(q, k, k, none, none, SCALE).any())


def test_graph_and_streams(cuda):
    q, k, v = make((90, 8, 128), torch.bfloat16), make((9000, 2, 128), torch.bfloat16, 1), make((9000, 2, 128), torch.bfloat16, 2)
    cases = [([90, 0], [9000, 0]), ([1, 89], [3000, 6000]), ([45, 45], [0, 45])]
    cq, ck = cumulated(cases[0][0]), cumulated(cases[0][1])
    want = [packed_attention(q, k, v, cumulated(a), cumulated(b), SCALE) for a, b in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        packed_attention(q, k, v, cq, ck, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = packed_attention(q, k, v, cq, ck, SCALE)
        graphs.append((g, out))
    for (a, b), w in zip(cases, want):
        cq.copy_(cumulated(a))
        ck.copy_(cumulated(b))
        for g, _ in graphs:                              # two graphs at once, on streams of their own
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
            torch.cuda.current_stream().wait_stream(s)
        eager = packed_attention(q, k, v, cq, ck, SCALE)
        n = sum(a)
        for got in (eager, *(o for _, o in graphs)):
            assert torch.equal(got[:n], w[:n])


def test_refusals(cuda):
    q, k = make((9, 4, 128), torch.float16), make((20, 2, 128), torch.float16)
    cq, ck = cumulated([9]), cumulated([20])
    for bad in (lambda: packed_attention(q.float(), k.float(), k.float(), cq, ck, SCALE), lambda: packed_attention(q, k.bfloat16(), k, cq, ck, SCALE),
                lambda: packed_attention(q, k, k[:19], cq, ck, SCALE), lambda: packed_attention(q[:, :3], k, k, cq, ck, SCALE),
                lambda: packed_attention(q, k, k, cq.long(), ck, SCALE), lambda: packed_attention(q, k, k, cq, cumulated([10, 10]), SCALE),
                lambda: packed_attention(q, k, k, cq.cpu(), ck, SCALE), lambda: packed_attention(q.cpu(), k, k, cq, ck, SCALE),
                lambda: packed_attention(q[..., :64], k, k, cq, ck, SCALE), lambda: packed_attention(q, k, k, cq, ck, 0.0),
                lambda: packed_attention(q, k, k, cq, ck, -1.0), lambda: packed_attention(q, k, k, cq, ck, float("nan")),
                lambda: packed_attention(q, k, k, cq, ck, float("inf")), lambda: packed_attention(q, k[:1].expand(20, 2, 128), k, cq, ck, SCALE),
                lambda: packed_attention(q, k, k, cq, ck, SCALE, out=torch.empty(9, 4, 64, device="cuda")),
                lambda: packed_attention(q, k, k, cq, ck, SCALE, ws=torch.zeros(64, dtype=torch.uint8, device="cuda")),
                lambda: packed_attention(make((9, 260, 128), torch.float16), k, k, cq, ck, SCALE),
                lambda: packed_attention(make((9, 4 * 128 + 4), torch.float16)[:, 4:].view(9, 4, 128), k, k, cq, ck, SCALE)):
        with pytest.raises(StarKVError):
            bad()
    assert _lib.load().starkv_packed_attention(None, None) == 1


@pytest.mark.parametrize("skip", [0, 1, 2, 5, 6])
@pytest.mark.parametrize("nq,nk", [([3000], [3000]), ([64, 1], [9000, 16000]), ([300] * 60, [300] * 60)])
def test_timed_out_copy(cuda, skip, nq, nk):
    """A tile of the first CTA is withheld: the call reports it and returns, and the next calls on the
    same workspace give what they gave before."""
    from starkv import ops
    q, k, v = make((sum(nq), 8, 128), torch.float16), make((sum(nk), 2, 128), torch.float16, 1), make((sum(nk), 2, 128), torch.float16, 2)
    cq, ck = cumulated(nq), cumulated(nk)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = packed_attention(q, k, v, cq, ck, SCALE, error_word=err)
    assert int(err) == 0
    try:
        ops.set_test_hooks(wait_limit_ns=20_000_000, skip_copy_unit=skip)
        packed_attention(q, k, v, cq, ck, SCALE, error_word=err)
        # 16000 keys are 125 tiles in 32 parts, the first of 3: six tiles of keys and values, and no second piece
        assert int(err) in (0x101, 0x102) or (nq == [64, 1] and skip >= 6 and int(err) == 0)
    finally:
        ops.set_test_hooks()
    err.zero_()
    for _ in range(3):
        assert torch.equal(packed_attention(q, k, v, cq, ck, SCALE, error_word=err), want)
    assert int(err) == 0


@pytest.mark.parametrize("batch", [4, 300, 1500])
def test_ends_far_below_zero(cuda, batch):
    """Ends near -2^31 behind starts inside the tensors: such a sequence has no rows and the error word says
    so, in the table of up to 256 sequences and beyond; the others are what they are without it."""
    q, k, v = make((2 * batch, 2, 128), torch.float16), make((2 * batch, 1, 128), torch.float16, 1), make((2 * batch, 1, 128), torch.float16, 2)
    starts = torch.arange(batch, dtype=torch.int32, device="cuda") * 2
    pairs = [(2 * b, 2 * b + 2) for b in range(0, batch, 2)]
    live = torch.zeros(2 * batch, dtype=torch.bool, device="cuda")
    live.view(-1, 4)[:, :2] = True
    want = [t[live] for t in reference(q, k, v, pairs, pairs)]
    for low in (-2 ** 31, -2 ** 31 + 1, -2 ** 31 + batch, -1):
        for which in ("q", "k"):
            ends = {"q": starts + 2, "k": starts + 2}
            ends[which][1::2] = low
            out, err = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
            packed_attention(q, k, v, (starts, ends["q"]), (starts, ends["k"]), SCALE, out=out, error_word=err)
            assert int(err) == 0x203
            close(out[live], None, want, torch.float16, 2)
            # without queries rows are left alone, without keys they are 0
            assert bool((out[~live] == (7.0 if which == "q" else 0.0)).all())


def test_errors_of_calls_without_a_word(cuda):
    """They are in the device's word: of the entry point, the torch.library op and a replayed graph; calls
    with a word of their own leave it alone."""
    from starkv import ops, torch_ops  # noqa: F401
    from starkv.prefill import read_packed_error
    q, k = make((20, 2, 128), torch.float16, 1), make((20, 1, 128), torch.float16, 2)
    good, bad = cumulated([20]), cumulated([21])
    read_packed_error()
    want = packed_attention(q, k, k, good, good, SCALE)
    assert read_packed_error() == 0
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for run in (lambda: packed_attention(q, k, k, bad, bad, SCALE), lambda: torch.ops.starkv.packed_attn(q, k, k, bad, bad, SCALE)[0]):
        assert torch.equal(run(), want) and read_packed_error(q.device) == 0x203 and read_packed_error() == 0
    packed_attention(q, k, k, bad, bad, SCALE, error_word=err)
    assert int(err) == 0x203 and read_packed_error() == 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = packed_attention(q, k, k, good, good, SCALE)
    for cu, code in (([20], 0), ([21], 0x203), ([20], 0)):
        good.copy_(cumulated(cu))
        g.replay()
        assert torch.equal(out, want) and read_packed_error() == code
    try:
        ops.set_test_hooks(wait_limit_ns=20_000_000, skip_copy_unit=1)
        packed_attention(q, k, k, good, good, SCALE)
        assert read_packed_error() in (0x101, 0x102)
    finally:
        ops.set_test_hooks()
    assert torch.equal(packed_attention(q, k, k, good, good, SCALE), want) and read_packed_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk", [([300, 40], [100, 0]), ([5, 700, 1], [0, 257, 3]), ([600], [599]), ([3], [0])])
def test_rows_that_see_nothing_are_zero(cuda, dtype, causal, nq, nk):
    """Exactly 0 and -inf, also into memory that held NaN."""
    q, k, v = make((sum(nq), 4, 128), dtype), make((sum(nk), 2, 128), dtype, 1), make((sum(nk), 2, 128), dtype, 2)
    for out_dtype in (dtype, torch.float32):
        out = torch.full(q.shape, math.nan, dtype=out_dtype, device="cuda")
        _, lse = packed_attention(q, k, v, cumulated(nq), cumulated(nk), SCALE, causal=causal, out=out, return_lse=True)
        idle = torch.cat([torch.arange(n, device="cuda") < (n - m if causal else n if m == 0 else 0) for n, m in zip(nq, nk)])
        assert bool(idle.any()) or not causal
        assert torch.equal(out[idle], torch.zeros_like(out[idle])) and bool((lse[idle] == -math.inf).all())
        assert bool(out[~idle].isfinite().all()) and bool(lse[~idle].isfinite().all())


@pytest.mark.parametrize("kv_heads,batch", [(8, 4_000_000), (1, 30_000_000)])
def test_rows_given_to_too_many_sequences(cuda, kv_heads, batch):
    """All rows to every sequence: 128 pairs of tiles a KV head, 4e9 pieces of work, which 31 bits do not
    number.  The call says so and leaves its outputs alone; the next one is as before."""
    n = 128 * 256
    q, k = make((n, kv_heads, 128), torch.float16), make((5, kv_heads, 128), torch.float16, 1)
    good = packed_attention(q, k, k, cumulated([n]), cumulated([5]), SCALE, causal=False)
    i = lambda x: torch.full((batch,), x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, err = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    packed_attention(q, k, k, (i(0), i(n)), (i(0), i(5)), SCALE, causal=False, out=out, error_word=err)
    assert int(err) == 0x203 and bool((out == 7.0).all())
    assert torch.equal(packed_attention(q, k, k, cumulated([n]), cumulated([5]), SCALE, causal=False, error_word=err), good)


def test_many_idle_rows_beside_a_long_history(cuda):
    """Two million queries with nothing to see beside cut histories."""
    nq, nk = [2_000_000, 3, 1], [700, 40_000, 30_000]
    q, k, v = make((sum(nq), 1, 128), torch.float16), make((sum(nk), 1, 128), torch.float16, 1), make((sum(nk), 1, 128), torch.float16, 2)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got, lse = packed_attention(q, k, v, cumulated(nq), cumulated(nk), SCALE, return_lse=True, error_word=err)
    assert int(err) == 0
    idle = nq[0] - nk[0]
    assert not bool(got[:idle].any()) and bool((lse[:idle] == -math.inf).all())
    live = torch.arange(idle, sum(nq), device="cuda")
    want = reference(q[live], k, v, [(0, 700), (700, 703), (703, 704)], [(0, 700), (700, 40_700), (40_700, 70_700)])
    close(got[live], lse[live], want, torch.float16, 40_000)
