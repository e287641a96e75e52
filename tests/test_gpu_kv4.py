"""The paged 4-bit cache on the B200 against the 64-bit oracle.

Read-back is exact: every step of the quantiser is specified in IEEE fp32.

Attention tolerances (u = 2^-11, the half-ulp of an fp16 number).  A softmax
weight w becomes an fp16 factor and its product with a token's scale s is rounded
to fp16 again, so the coded part s * c of a value carries at most 2u of w |s c| and
the centre m at most u of w |m|.  Scores: products are exact and summed in fp32;
with A = scaling * max_t sum_d |q_d| (16 s + |m|) the sum of 128 + 8 terms (some
tensor-core additions truncate) is off by at most 2^-15 A, which moves every weight
by that factor at most twice (numerator and denominator).  Hence, in fp32,
    |out - ref| <= (2u (1 + 2u) + 2 * 2^-15 A + 2^-18) sum_t w (|s c| + |m|)
    |lse - ref| <= 2^-15 A + 2^-20 (1 + |ref|)
and rounding the output once adds u |ref| (fp16) or 2^-8 |ref| (bf16)."""

import numpy as np
import pytest
import torch

import kv4_oracle as O
from starkv import StarKVError
from starkv.kv4 import KV4Cache, ERRORS

pytestmark = pytest.mark.gpu
U = 2.0 ** -11
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SCALING = 128 ** -0.5


def rnd(shape, dtype, seed, dev, outliers=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(shape, generator=g, device=dev)
    if outliers:
        x = x * (1 + 7 * (torch.rand(shape[-2:], generator=g, device=dev) < 0.02))
    return x.to(dtype)


def table_of(B, W, dev, seed=0, num_pages=None):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(num_pages or B * W, generator=g)[:B * W].to(torch.int32).view(B, W).to(dev)


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def f64(t):
    return t.double().cpu().numpy()


class Made:
    """A cache of B sequences with the stored values of each as the oracle has them."""

    def __init__(self, dev, lens, Hkv, page, dtype, seed=0, garbage=True, spare=3):
        B = len(lens)
        n = max(1, max(lens))
        W = -(-n // page) + 1
        self.cache = KV4Cache(B * W + spare, Hkv, page_size=page, device=dev)
        if garbage:                                             # NaN / infinite parameters wherever nothing is written
            self.cache.data.fill_(0xFF)
        self.table = table_of(B, W, dev, seed, B * W + spare)
        self.k, self.v = rnd((B, n, Hkv, 128), dtype, seed + 1, dev), rnd((B, n, Hkv, 128), dtype, seed + 2, dev)
        self.lens, self.lengths, self.page, self.Hkv, self.dev = lens, ints(lens, dev), page, Hkv, dev
        self.cache.write(self.k, self.v, self.table, ints([0] * B, dev), self.lengths)

    def stored(self, b, h):
        return tuple(O.values(f64(t[b, :self.lens[b], h])) for t in (self.k, self.v))


def check_attention(made, q, mask=None, pages=None, out_dtype=F32, **kw):
    B, Q, Hq, _ = q.shape
    G = Hq // made.Hkv
    out = torch.empty(q.shape, dtype=out_dtype, device=q.device)
    got, lse = made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask, pages=pages, out=out,
                                 return_lse=True, **kw)
    torch.cuda.synchronize()
    assert got is out and made.cache.read_error() == 0
    got, lse = f64(got), f64(lse)
    for b in range(B):
        n = made.lens[b]
        for h in range(made.Hkv):
            qq = f64(q[b, :, h * G:(h + 1) * G])
            k, v = made.stored(b, h)
            keep = None
            if pages is not None:
                keep = np.isin(np.arange(n) // made.page, [p for p in pages[b, h].tolist() if p >= 0])
            ref, rlse, w = O.attend(qq, k, v, SCALING, keep, None if mask is None else f64(mask[b]))
            o, l = got[b, :, h * G:(h + 1) * G], lse[b, :, h * G:(h + 1) * G]
            empty = np.isneginf(rlse)
            assert (o[empty] == 0).all() and np.isneginf(l[empty]).all()
            if n == 0:
                continue
            _, s, m = O.quantise(f64(made.k[b, :n, h]))
            A = SCALING * np.max(np.einsum("qgje,nj->qgn", np.abs(qq).reshape(Q, G, 4, 32), 16 * s + np.abs(m)))
            c, s, m = O.quantise(f64(made.v[b, :n, h]))
            size = (np.abs(s[..., None] * c) + np.abs(m)[..., None]).reshape(n, 128)
            tol = (2 * U * (1 + 2 * U) + 2 * 2.0 ** -15 * A + 2.0 ** -18) * (w @ size)
            tol += np.abs(ref) * {F32: 0.0, F16: U, BF16: 2.0 ** -8}[out_dtype] + 2.0 ** -24
            bad = np.abs(o - ref) > tol
            assert not bad.any(), (b, h, np.abs(o - ref).max(), (np.abs(o - ref) / tol).max())
            live = ~empty
            ltol = 2.0 ** -15 * A + 2.0 ** -20 * (1 + np.abs(rlse[live]))
            assert (np.abs(l[live] - rlse[live]) <= ltol).all(), np.abs(l[live] - rlse[live]).max()
    return got


# ------------------------------------------------------------------ write and read
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("start,count", [((0, 0, 0), (1, 16, 200)), ((15, 64, 127), (1, 0, 2)), ((5, 63, 100), (37, 65, 199))])
def test_write_reads_back_exactly(cuda, dtype, page, start, count):
    B, T, H = 3, 200, 3
    W = -(-(max(start) + T) // page)
    cache = KV4Cache(B * W, H, page_size=page, device=cuda)
    table = table_of(B, W, cuda, 7)
    k, v = rnd((B, T, H, 128), dtype, 1, cuda), rnd((B, T, H, 128), dtype, 2, cuda)
    cache.write(k, v, table, ints(start, cuda), ints(count, cuda))
    for out in (F32, dtype):
        rk, rv = cache.read(table, ints(start, cuda), T, ints(count, cuda), dtype=out)
        for got, x in ((rk, k), (rv, v)):
            want = torch.from_numpy(O.values(f64(x))).to(torch.float32).to(out)
            for b in range(B):
                want[b, count[b]:] = 0
            assert torch.equal(got.cpu(), want)
    assert cache.read_error() == 0


def test_writes_in_pieces_give_the_same_pool(cuda):
    """Tokens written one by one, in odd pieces or at once leave the same bytes and bounds."""
    H, page, n = 2, 64, 150
    k, v = rnd((1, n, H, 128), F16, 3, cuda), rnd((1, n, H, 128), F16, 4, cuda)
    table = table_of(1, 3, cuda, 1)
    pools = []
    for pieces in ([n], [1] * n, [7, 13, 44, 1, 63, 22]):
        cache = KV4Cache(3, H, page_size=page, device=cuda)
        at = 0
        for m in pieces:
            cache.write(k[:, at:at + m], v[:, at:at + m], table, ints([at], cuda))
            at += m
        assert at == n
        pools.append((cache.data, cache.bounds, cache.bound_scales))
    for other in pools[1:]:
        assert all(torch.equal(a, b) for a, b in zip(pools[0], other))


def test_bounds_are_of_the_full_pages(cuda):
    H, page, n = 3, 32, 101
    made = Made(cuda, [n], H, page, BF16, seed=11)
    for h in range(H):
        keys, _ = made.stored(0, h)
        for p in range(n // page):
            up, lo, t = O.bounds(keys[p * page:(p + 1) * page])
            at = int(made.table[0, p])
            assert np.array_equal(f64(made.cache.bounds[at, h, 0]), up)
            assert np.array_equal(f64(made.cache.bounds[at, h, 1]), lo)
            assert float(made.cache.bound_scales[at, h]) == t


def test_write_special_values(cuda):
    """Constant groups are kept exactly, infinities saturate, a NaN takes its group of
    32 with it and nothing else."""
    x = torch.zeros(1, 4, 1, 128, device=cuda)
    x[0, 0] = 3.25
    x[0, 1, 0, 5] = float("inf")
    x[0, 2, 0, 70] = float("nan")
    x[0, 3] = torch.linspace(-1e30, 1e30, 128, device=cuda)
    cache = KV4Cache(1, 1, page_size=16, device=cuda)
    table = ints([[0]], cuda)
    cache.write(x, x, table, ints([0], cuda))
    for got in cache.read(table, ints([0], cuda), 4, dtype=F32):
        got = got[0, :, 0].cpu()
        assert (got[0] == 3.25).all()
        assert torch.isfinite(got[1]).all() and got[1, 5] > 60000 and (got[1, 32:] == 0).all()
        nan = torch.isnan(got[2])
        assert nan[64:96].all() and not nan[:64].any() and not nan[96:].any()
        want = torch.from_numpy(O.values(f64(x[0, 3, 0]))).float()
        assert torch.equal(got[3], want) and torch.isfinite(got[3]).all()


def test_strided_inputs_and_outputs(cuda):
    """Heads-first storage, a fused qkv tensor and padded rows are read and written in place."""
    B, T, H = 2, 50, 4
    table = table_of(B, 1, cuda)
    start = ints([3, 0], cuda)
    fused = rnd((B, T, 3 * H, 128), F16, 5, cuda)
    first = rnd((B, H, T, 128), F16, 6, cuda).transpose(1, 2)
    wide = rnd((B, T, H, 136), F16, 7, cuda)[..., :128]
    for k, v in ((fused[:, :, :H], fused[:, :, 2 * H:]), (first, wide)):
        cache = KV4Cache(2, H, device=cuda)
        cache.write(k, v, table, start)
        out = (torch.full((B, H, T, 128), 9.0, dtype=F16, device=cuda).transpose(1, 2),
               torch.full((B, T, H, 256), 9.0, dtype=F16, device=cuda)[..., 128:])
        got = cache.read(table, start, T, out=out)
        for g, x in zip(got, (k, v)):
            assert torch.equal(g.cpu(), torch.from_numpy(O.values(f64(x))).float().to(F16))


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("Hkv,G,Q", [(2, 1, 1), (1, 4, 1), (2, 8, 1), (3, 5, 1), (1, 4, 4), (1, 3, 5), (2, 7, 3), (1, 8, 6)])
def test_attention_matches_the_oracle(cuda, dtype, page, Hkv, G, Q):
    lens = [1, 16, 0, 15, 17, 64, 333]
    made = Made(cuda, lens, Hkv, page, dtype, seed=Hkv * 100 + G * 10 + Q)
    check_attention(made, rnd((len(lens), Q, Hkv * G, 128), dtype, 5, cuda))


@pytest.mark.parametrize("lens", [[5000], [2049, 1, 777, 0, 4096], [16] * 70 + [1500] + [3] * 5])
@pytest.mark.parametrize("Hkv,G,Q", [(2, 4, 1), (1, 4, 4)])
def test_attention_split_over_the_machine(cuda, lens, Hkv, G, Q):
    made = Made(cuda, lens, Hkv, 64, F16, seed=len(lens))
    check_attention(made, rnd((len(lens), Q, Hkv * G, 128), F16, 6, cuda))


@pytest.mark.parametrize("B,Hkv,G,Q,top", [(300, 8, 4, 1, 130), (500, 4, 1, 1, 60), (200, 4, 4, 4, 90), (64, 8, 4, 1, 700), (1300, 1, 2, 1, 40)])
def test_attention_many_short_sequences(cuda, B, Hkv, G, Q, top):
    """Stretches that hold the end of one sequence, several whole ones and the start of another."""
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(0, top, B)]
    made = Made(cuda, lens, Hkv, 16, F16, seed=B)
    check_attention(made, rnd((B, Q, Hkv * G, 128), F16, 7, cuda))


@pytest.mark.parametrize("out_dtype", [F16, BF16])
def test_attention_output_types(cuda, out_dtype):
    made = Made(cuda, [100, 40], 2, 32, F16, seed=8)
    check_attention(made, rnd((2, 1, 4, 128), F16, 9, cuda), out_dtype=out_dtype)


@pytest.mark.parametrize("Q,G", [(1, 1), (2, 4), (3, 8)])
def test_attention_masks(cuda, Q, G):
    """-inf everywhere, -inf in runs and alone, the type's lowest value (added like any
    other number: alone it leaves the weights as they were, beside 0 it takes none), a
    bias, and a mask narrower than the sequence."""
    lens = [300] * 6
    made = Made(cuda, lens, 2, 64, F16, seed=21)
    mask = torch.zeros(6, 300, device=cuda)
    mask[0] = float("-inf")
    mask[1, :137] = float("-inf")
    mask[2, ::3] = float("-inf")
    mask[3, 100:] = torch.finfo(F32).min
    mask[4] = torch.randn(300, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda) * 3
    mask[5, :299] = float("-inf")
    q = rnd((6, Q, 2 * G, 128), F16, 22, cuda)
    check_attention(made, q, mask=mask)
    # every position at the type's lowest value: the scores vanish beside it, the mean of the values is left
    low = torch.full((6, 300), torch.finfo(F32).min, device=cuda)
    out = made.cache.attend(q, made.table, made.lengths, SCALING, mask=low, out=torch.empty(q.shape, device=cuda))
    for h in range(2):
        mean = O.values(f64(made.v[2, :, h])).mean(0)
        if Q == 1:
            assert np.abs(f64(out[2, 0, h * G]) - mean).max() <= 2 * U * 8
    narrow = made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask[:, :137].contiguous())
    wide = mask.clone()
    wide[:, 137:] = 0
    assert torch.equal(narrow, made.cache.attend(q, made.table, made.lengths, SCALING, mask=wide))


def test_attention_ignores_what_is_masked(cuda):
    """NaN keys and values at masked positions and past the length change nothing."""
    lens = [200, 90]
    made = Made(cuda, lens, 1, 64, F16, seed=31, garbage=False)
    q = rnd((2, 1, 4, 128), F16, 32, cuda)
    mask = torch.zeros(2, 200, device=cuda)
    mask[:, 10:50] = float("-inf")
    before = made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask)
    nan = torch.full((2, 40, 1, 128), float("nan"), dtype=F16, device=cuda)
    made.cache.write(nan, nan, made.table, ints([10, 10], cuda))
    made.cache.write(nan, nan, made.table, made.lengths)          # right behind the last token
    after = made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask)
    assert torch.equal(before, after) and torch.isfinite(after).all()


@pytest.mark.parametrize("scale", [1e-4, 1.0, 300.0, 4000.0])
def test_attention_value_ranges(cuda, scale):
    """Values far below and above one: the fp16 factors of P.V are scaled to fit."""
    made = Made(cuda, [700, 31], 1, 64, F32, seed=41)
    made.v = (made.v * scale).clamp(-60000, 60000)
    made.cache.write(made.k, made.v, made.table, ints([0, 0], cuda), made.lengths)
    check_attention(made, rnd((2, 1, 4, 128), F16, 42, cuda))


def test_attention_large_and_small_queries(cuda):
    made = Made(cuda, [260], 1, 64, BF16, seed=51)
    q = rnd((1, 3, 4, 128), BF16, 52, cuda)
    q[0, 0] *= 1e-20
    q[0, 1] *= 20
    q[0, 2, 1] = 0
    check_attention(made, q)


def test_attention_is_the_same_every_time_and_on_any_stream(cuda):
    lens = [3000, 17, 1024]
    made = Made(cuda, lens, 2, 64, F16, seed=61)
    q = rnd((3, 1, 8, 128), F16, 62, cuda)
    want = made.cache.attend(q, made.table, made.lengths, SCALING)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [made.cache.attend(q, made.table, made.lengths, SCALING) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want, g) for g in got)


def test_step_in_a_cuda_graph(cuda):
    """write, select and attend captured once, replayed as the sequences grow."""
    made = Made(cuda, [1000, 500], 2, 64, F16, seed=71)
    lengths = made.lengths.clone()
    k, v = rnd((2, 1, 2, 128), F16, 72, cuda), rnd((2, 1, 2, 128), F16, 73, cuda)
    q = rnd((2, 1, 8, 128), F16, 74, cuda)
    start = lengths.clone()

    def step():
        made.cache.write(k, v, made.table, start)
        pages = made.cache.select(q, made.table, lengths, 4)
        return made.cache.attend(q, made.table, lengths, SCALING), made.cache.attend(q, made.table, lengths, SCALING, pages=pages)

    lengths += 1
    want0 = [t.clone() for t in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want0, got))
    start += 1
    lengths += 1
    graph.replay()
    got = [t.clone() for t in got]
    assert all(torch.equal(a, b) for a, b in zip(step(), got))


def test_pool_offsets_past_32_bits(cuda):
    """Pages whose bytes start beyond 2^32."""
    H, page = 32, 64
    per = H * page * 160
    n = (1 << 32) // per + 4
    cache = KV4Cache(n, H, page_size=page, device=cuda)
    table = ints([[n - 1, 1, n - 2]], cuda)
    k, v = rnd((1, 150, H, 128), F16, 81, cuda), rnd((1, 150, H, 128), F16, 82, cuda)
    cache.write(k, v, table, ints([0], cuda))
    rk, rv = cache.read(table, ints([0], cuda), 150)
    assert torch.equal(rk.cpu(), torch.from_numpy(O.values(f64(k))).float().to(F16))
    assert torch.equal(rv.cpu(), torch.from_numpy(O.values(f64(v))).float().to(F16))
    q = rnd((1, 1, H, 128), F16, 83, cuda)
    big = cache.attend(q, table, ints([150], cuda), SCALING)
    small = KV4Cache(3, H, page_size=page, device=cuda)
    t2 = ints([[0, 1, 2]], cuda)
    small.write(k, v, t2, ints([0], cuda))
    assert torch.equal(big, small.attend(q, t2, ints([150], cuda), SCALING))
    assert torch.equal(cache.select(q, table, ints([150], cuda), 2), small.select(q, t2, ints([150], cuda), 2))


# ------------------------------------------------------------------ selected pages
@pytest.mark.parametrize("page,Hkv,G,Q,keep", [(16, 2, 1, 1, 7), (16, 1, 4, 2, 2), (32, 3, 5, 1, 12), (64, 2, 8, 1, 5), (128, 1, 1, 3, 3)])
def test_selection_and_attention_over_it(cuda, page, Hkv, G, Q, keep):
    lens = [1, 0, page * keep, page * keep + 1, page * 20 + 5, page * 11]
    made = Made(cuda, lens, Hkv, page, F16, seed=page + keep)
    q = rnd((len(lens), Q, Hkv * G, 128), F16, 91, cuda)
    pages = made.cache.select(q, made.table, made.lengths, keep)
    for b, n in enumerate(lens):
        for h in range(Hkv):
            keys, _ = made.stored(b, h)
            want = O.select(f64(q[b, :, h * G:(h + 1) * G]).reshape(-1, 128), keys, page, keep)
            assert pages[b, h].tolist() == want + [-1] * (keep - len(want)), (b, h)
    check_attention(made, q, pages=pages)
    mask = torch.zeros(len(lens), max(lens), device=cuda)
    mask[:, ::2] = float("-inf")
    check_attention(made, q, pages=pages, mask=mask)


@pytest.mark.parametrize("pages_n", [2500, 9000])
def test_selection_among_many_pages(cuda, pages_n):
    """More pages than one thread's registers hold, and more than all of them do."""
    n = pages_n * 16 - 7
    made = Made(cuda, [n, 40 * 16], 1, 16, F16, seed=pages_n, garbage=False)
    q = rnd((2, 1, 2, 128), F16, 92, cuda)
    pages = made.cache.select(q, made.table, made.lengths, 33, first=2, last=3)
    for b, m in enumerate((n, 40 * 16)):
        want = O.select(f64(q[b]).reshape(-1, 128), made.stored(b, 0)[0], 16, 33, 2, 3)
        assert pages[b, 0].tolist() == want
    assert torch.equal(pages, made.cache.select(q, made.table, made.lengths, 33, first=2, last=3))


def test_selection_first_last_and_ties(cuda):
    """Identical pages tie: the lower ones win; first / last pages are always in."""
    page, n = 16, 16 * 12
    cache = KV4Cache(12, 1, page_size=page, device=cuda)
    table = table_of(1, 12, cuda, 3)
    k = rnd((1, page, 1, 128), F16, 95, cuda).repeat(1, 12, 1, 1)
    cache.write(k, k, table, ints([0], cuda))
    q = rnd((1, 1, 2, 128), F16, 96, cuda)
    for first, last, want in ((1, 1, [0, 1, 2, 3, 11]), (0, 2, [0, 1, 2, 10, 11]), (2, 3, [0, 1, 9, 10, 11])):
        assert cache.select(q, table, ints([n], cuda), 5, first, last)[0, 0].tolist() == want


def test_attention_over_given_pages(cuda):
    """Hand-made lists: any order, -1 anywhere, none at all, and pages past the sequence."""
    made = Made(cuda, [500, 500, 30], 1, 32, F16, seed=99)
    pages = ints([[[9, 2, -1, 15]], [[-1, -1, -1, -1]], [[0, 7, 15, -1]]], cuda)
    q = rnd((3, 1, 4, 128), F16, 98, cuda)
    out = check_attention(made, q, pages=pages)
    assert (out[1] == 0).all()


# ------------------------------------------------------------------ refusals
def test_refusals(cuda):
    H = 2
    cache = KV4Cache(4, H, page_size=32, device=cuda)
    table, start = table_of(2, 2, cuda), ints([0, 0], cuda)
    k = torch.zeros(2, 5, H, 128, dtype=F16, device=cuda)
    q = torch.zeros(2, 1, 4, 128, dtype=F16, device=cuda)
    with pytest.raises(StarKVError):
        KV4Cache(4, H, page_size=48, device=cuda)
    with pytest.raises(StarKVError):
        KV4Cache(4, H, device="cpu")
    bad_io = [
        dict(k=k[..., :64], v=k[..., :64]), dict(k=k.double(), v=k.double()), dict(k=k, v=k.bfloat16()),
        dict(k=k.cpu(), v=k.cpu()), dict(k=k[:1], v=k[:1]), dict(k=k[:, :, :1], v=k[:, :, :1]),
        dict(table=table.long()), dict(table=table[:, :0]), dict(start=start.long()), dict(start=start[:1]),
        dict(count=ints([1], cuda)), dict(k=torch.zeros(2, 5, H, 129, dtype=F16, device=cuda)[..., 1:], v=k),
        dict(k=k.transpose(2, 3).contiguous().transpose(2, 3), v=k),
    ]
    for bad in bad_io:
        a = dict(k=k, v=k, table=table, start=start, count=None)
        a.update(bad)
        with pytest.raises(StarKVError):
            cache.write(a["k"], a["v"], a["table"], a["start"], a["count"])
    with pytest.raises(StarKVError):
        cache.read(table, start, 5, dtype=torch.int8)
    with pytest.raises(StarKVError):
        cache.read(table, start, 5, out=(k[:, :1].expand(2, 5, H, 128), k.clone()))
    bad_attend = [
        dict(q=q.float()), dict(q=q[:, :, :3]), dict(q=q[:1]), dict(lengths=start.long()), dict(mask=torch.zeros(2, 5, device=cuda).half()),
        dict(mask=torch.zeros(1, 5, device=cuda)), dict(pages=ints([[[0]]], cuda)), dict(out=torch.empty(2, 1, 2, 128, device=cuda)),
        dict(ws=torch.zeros(16, dtype=torch.uint8, device=cuda)),
    ]
    for bad in bad_attend:
        a = dict(q=q, lengths=start, mask=None, pages=None, out=None, ws=None)
        a.update(bad)
        with pytest.raises(StarKVError):
            cache.attend(a["q"], table, a["lengths"], 1.0, mask=a["mask"], pages=a["pages"], out=a["out"], ws=a["ws"])
    for args in ((1, 1, 1), (0, 0, 0), (4, 1, 0), (4, -1, 1)):
        with pytest.raises(StarKVError):
            cache.select(q, table, start, *args)
    with pytest.raises(StarKVError):
        KV4Cache(4, H, page_bounds=False, device=cuda).select(q, table, start, 2)


def test_bad_pages_and_positions_set_the_error_word(cuda):
    """The kernels' own checks: what lies outside is skipped and reported, the rest is done."""
    H = 2
    cache = KV4Cache(4, H, page_size=16, device=cuda)
    k = rnd((2, 20, H, 128), F16, 1, cuda)
    good = ints([[0, 1], [2, 3]], cuda)
    bad = ints([[0, 4], [-1, 3]], cuda)
    start = ints([0, 0], cuda)
    cache.write(k, k, bad, start)
    assert cache.read_error() == 0x201 and 0x201 in ERRORS and cache.read_error() == 0
    got, _ = cache.read(good, start, 20, dtype=F32)
    want = torch.from_numpy(O.values(f64(k))).float()
    assert torch.equal(got[0, :16].cpu(), want[0, :16]) and (got[0, 16:] == 0).all()
    assert (got[1, :16] == 0).all() and torch.equal(got[1, 16:].cpu(), want[1, 16:])
    cache.write(k, k, good, ints([20, -3], cuda))                 # past the table; before its start
    assert cache.read_error() == 0x202
    cache.write(k, k, good, start)
    q = rnd((2, 1, 4, 128), F16, 2, cuda)
    cache.attend(q, good, ints([33, 5], cuda), SCALING)           # a length past the table
    assert cache.read_error() == 0x202
    want = cache.attend(q, good, ints([16, 20], cuda), SCALING)
    assert cache.read_error() == 0
    got = cache.attend(q, ints([[0, 77], [2, 3]], cuda), ints([20, 20], cuda), SCALING)
    assert cache.read_error() == 0x201 and torch.equal(got, want)
    cache.read(good, ints([30, 0], cuda), 5)
    assert cache.read_error() == 0x202


def test_torch_ops_match_the_cache(cuda):
    """torch.ops.starkv.kv4_* give what the KV4Cache methods give."""
    from starkv import torch_ops  # noqa: F401
    o = torch.ops.starkv
    made = Made(cuda, [300, 77], 2, 32, F16, seed=13, garbage=False)
    c, q = made.cache, rnd((2, 1, 4, 128), F16, 14, cuda)
    other = KV4Cache(c.num_pages, 2, 32, device=cuda)
    o.kv4_write(other.data, other.bounds, other.bound_scales, other.error_word, made.k, made.v, made.table,
                ints([0, 0], cuda), made.lengths)
    assert all(torch.equal(getattr(c, n), getattr(other, n)) for n in ("data", "bounds", "bound_scales"))
    kv = o.kv4_read(c.data, c.error_word, made.table, ints([0, 5], cuda), 50, F16)
    k, v = c.read(made.table, ints([0, 5], cuda), 50, dtype=F16)
    assert torch.equal(kv[0], k) and torch.equal(kv[1], v)
    pages = o.kv4_select(c.data, c.bounds, c.bound_scales, c.error_word, q, made.table, made.lengths, 4)
    assert torch.equal(pages, c.select(q, made.table, made.lengths, 4))
    out, lse = o.kv4_attn(c.data, c.error_word, q, made.table, made.lengths, SCALING, None, pages)
    want, wlse = c.attend(q, made.table, made.lengths, SCALING, pages=pages, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    with pytest.raises(StarKVError):
        KV4Cache.from_tensors(c.data[:, :1], None, None, c.error_word)
    with pytest.raises(StarKVError):
        KV4Cache.from_tensors(c.data, c.bounds, None, c.error_word)


def test_single_query_shape(cuda):
    """(B, Hq, 128) queries give (B, Hq, 128) outputs, the same as one token of (B, 1, Hq, 128)."""
    made = Made(cuda, [100, 33], 2, 16, F16, seed=5)
    q = rnd((2, 1, 4, 128), F16, 6, cuda)
    a, la = made.cache.attend(q, made.table, made.lengths, SCALING, return_lse=True)
    b, lb = made.cache.attend(q[:, 0], made.table, made.lengths, SCALING, return_lse=True)
    assert b.shape == (2, 4, 128) and lb.shape == (2, 4)
    assert torch.equal(a[:, 0], b) and torch.equal(la[:, 0], lb)
    assert torch.equal(made.cache.select(q, made.table, made.lengths, 3), made.cache.select(q[:, 0], made.table, made.lengths, 3))


def test_empty_calls(cuda):
    cache = KV4Cache(2, 1, device=cuda)
    none = torch.zeros(0, 1, dtype=torch.int32, device=cuda)
    z = torch.zeros(0, dtype=torch.int32, device=cuda)
    cache.write(torch.zeros(0, 3, 1, 128, device=cuda), torch.zeros(0, 3, 1, 128, device=cuda), none, z)
    cache.write(torch.zeros(1, 0, 1, 128, device=cuda), torch.zeros(1, 0, 1, 128, device=cuda), ints([[0]], cuda), ints([0], cuda))
    assert cache.read(ints([[0]], cuda), ints([0], cuda), 0)[0].shape == (1, 0, 1, 128)
    assert cache.attend(torch.zeros(0, 1, 2, 128, dtype=F16, device=cuda), none, z, 1.0).shape == (0, 1, 2, 128)
    assert cache.select(torch.zeros(0, 2, 128, dtype=F16, device=cuda), none, z, 2).shape == (0, 1, 2)
    assert cache.read_error() == 0


def test_unaligned_workspaces_are_refused(cuda):
    """The kernels read and write 16 bytes at a time in the attention's workspace, 4 in the selection's."""
    import ctypes as C
    from starkv import _lib, kv4
    lib = _lib.load()
    cache = KV4Cache(4, 2, page_size=32, device=cuda)
    table, lengths = table_of(2, 2, cuda), ints([40, 3], cuda)
    q = torch.zeros(2, 1, 4, 128, dtype=F16, device=cuda)
    need = kv4._attention_size()
    room = torch.zeros(need + 64, dtype=torch.uint8, device=cuda)
    base = -room.data_ptr() % 16
    for off in (1, 2, 4, 8, 15):
        with pytest.raises(StarKVError):
            cache.attend(q, table, lengths, SCALING, ws=room[base + off:])
    got = cache.attend(q, table, lengths, SCALING, ws=room[base + 16:])
    assert torch.equal(got, cache.attend(q, table, lengths, SCALING))
    n = C.c_size_t(0)
    assert lib.starkv_kv4_select_workspace_size(cache._block, 2, 2, C.byref(n)) == 0
    room = torch.zeros(n.value + 64, dtype=torch.uint8, device=cuda)
    out = torch.empty(2, 2, 2, dtype=torch.int32, device=cuda)
    for off, status in ((1, 4), (2, 4), (3, 4), (4, 0)):
        a = _lib.KV4SelectArgs(q=q.data_ptr(), q_strides=q.stride()[:3], block_table=table.data_ptr(), table_stride=2,
                               lengths=lengths.data_ptr(), pages_out=out.data_ptr(), workspace=room.data_ptr() + off,
                               workspace_bytes=n.value, q_dtype=1, batch=2, num_queries=1, num_q_heads=4, table_width=2,
                               num_selected=2, num_first=1, num_last=1)
        assert lib.starkv_kv4_select(cache._block, C.byref(a), None) == status
    torch.cuda.synchronize()
    assert out.cpu()[0, 0].tolist() == [0, 1]


@pytest.mark.parametrize("Q,G", [(1, 1), (1, 4), (3, 8)])
def test_nan_in_a_mask(cuda, Q, G):
    """A NaN in a mask is added like any number: the queries that may attend there are NaN, and only they."""
    lens = [300, 300, 70]
    made = Made(cuda, lens, 2, 64, F16, seed=23, garbage=False)
    q = rnd((3, Q, 2 * G, 128), F16, 24, cuda)
    clean = torch.zeros(3, 300, device=cuda)
    clean[1, 290:] = float("-inf")
    mask = clean.clone()
    mask[0, 17] = mask[1, 280] = float("nan")
    mask[2, 70:] = float("nan")                               # past the length
    want, wlse = made.cache.attend(q, made.table, made.lengths, SCALING, mask=clean, return_lse=True)
    out, lse = made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask, return_lse=True)
    assert torch.isnan(out[:2]).all() and torch.isnan(lse[:2]).all()
    assert torch.equal(out[2], want[2]) and torch.equal(lse[2], wlse[2])
    if Q > 1:                                                 # where only the newest query attends
        mask = clean.clone()
        mask[0, 299] = float("nan")
        out, lse = made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask, return_lse=True)
        assert torch.isnan(out[0, -1]).all() and torch.equal(out[0, :-1], want[0, :-1]) and torch.equal(lse[0, :-1], wlse[0, :-1])


@pytest.mark.parametrize("Q,G", [(1, 1), (1, 4), (3, 8)])
def test_masks_of_the_largest_magnitudes(cuda, Q, G):
    """Numbers near the ends of fp32 are kept apart: positions at -3e38 weigh nothing beside one at
    -2.5e38, which weighs nothing beside 0, and the log-sum-exp is the largest of them."""
    low = torch.finfo(F32).min
    made = Made(cuda, [300] * 7, 2, 64, F16, seed=25)
    q = rnd((7, Q, 2 * G, 128), F16, 26, cuda)
    mask = torch.full((7, 300), low, device=cuda)
    mask[1, 40] = -3e38
    mask[2, 40] = -2.5e38
    mask[2, 41:] = -3.3e38
    mask[3, :], mask[3, 40] = torch.finfo(BF16).min, -1e38
    mask[4, :], mask[4, 40] = -1e38, 2.5e38
    mask[5, :], mask[5, 40], mask[5, 41] = 0, 1e38, 3e38
    mask[6, 40] = -9e37
    out = torch.empty(q.shape, device=cuda)
    _, lse = made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask, out=out, return_lse=True)
    want = [low, -3e38, -2.5e38, -1e38, 2.5e38, 3e38, -9e37]
    assert np.abs(f64(lse) / np.array(want)[:, None, None] - 1).max() <= 2.0 ** -20
    for b in range(1, 7):                                     # one position takes all: its value, rounded twice at most
        for h in range(2):
            v = O.values(f64(made.v[b, 41 if b == 5 else 40, h]))
            _, s, m = O.quantise(f64(made.v[b, 41 if b == 5 else 40, h]))
            tol = 2 * U * (8 * s + np.abs(m)).repeat(32)
            assert (np.abs(f64(out[b, :, h * G:(h + 1) * G]) - v) <= tol).all(), b


@pytest.mark.parametrize("scaling,size", [(1e-25, 1e-20), (-1e-30, 1e-12), (1e-38, 1.0), (0.0, 1.0), (1e-35, 1e30), (1e20, 1e-25)])
def test_scalings_of_any_size(cuda, scaling, size):
    """Products of queries and scaling below fp32's range leave the mean of the values, the others their softmax."""
    lens, Q, G = [77, 5, 0, 333], 2, 4
    made = Made(cuda, lens, 1, 64, BF16, seed=27)
    q = (rnd((4, Q, G, 128), BF16, 28, cuda).float() * size).to(BF16)
    mask = torch.zeros(4, 333, device=cuda)
    mask[3, :100] = float("-inf")
    for m in (None, mask):
        out = torch.empty(q.shape, device=cuda)
        _, lse = made.cache.attend(q, made.table, made.lengths, scaling, mask=m, out=out, return_lse=True)
        for b, n in enumerate(lens):
            k, v = made.stored(b, 0)
            ref, rlse, w = O.attend(f64(q[b]), k, v, float(np.float32(scaling)), None, None if m is None else f64(m[b]))
            empty = np.isneginf(rlse)
            assert (f64(out[b])[empty] == 0).all() and np.isneginf(f64(lse[b])[empty]).all()
            if n:                                             # scores are below 0.1: 2^-15 of that does not show
                _, s, mm = O.quantise(f64(made.v[b, :n, 0]))
                big = (8 * s + np.abs(mm)).max()
                assert np.abs(f64(out[b]) - ref).max() <= (2 * U + 2.0 ** -15) * big
                assert np.abs(f64(lse[b])[~empty] - rlse[~empty]).max() <= 2.0 ** -15


def test_nan_scaling(cuda):
    made = Made(cuda, [77, 1, 0], 1, 64, F16, seed=29)
    q = rnd((3, 2, 4, 128), F16, 30, cuda)
    out, lse = made.cache.attend(q, made.table, made.lengths, float("nan"), return_lse=True)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and torch.isnan(out[1, 1]).all()
    assert (out[1, 0] == 0).all() and (out[2] == 0).all() and torch.isneginf(lse[2]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hkv,G,Q,n", [(1, 4, 2, 77), (2, 1, 4, 33), (1, 4, 4, 16), (1, 3, 5, 130), (2, 8, 6, 64), (1, 2, 3, 3)])
def test_nan_in_newer_tokens_does_not_reach_older_queries(cuda, dtype, Hkv, G, Q, n):
    """A NaN key or value of a newer draft is the newer queries' alone, and a value's only in its 32 channels."""
    made = Made(cuda, [n, n], Hkv, 16, F32, seed=33, garbage=False)
    made.k, made.v = made.k.clamp(-3, 3), made.v.clamp(-3, 3)         # scales below 1: no other exponent without one
    made.cache.write(made.k, made.v, made.table, ints([0, 0], cuda))
    q = rnd((2, Q, Hkv * G, 128), dtype, 34, cuda)
    mask = torch.zeros(2, n, device=cuda)
    for m in (None, mask):
        want, wlse = made.cache.attend(q, made.table, made.lengths, SCALING, mask=m, return_lse=True)
        for i in range(1, Q):                                         # position of query i
            k, v = made.k.clone(), made.v.clone()
            v[0, n - Q + i, :, 70] = float("nan")
            k[1, n - Q + i, :, 5] = float("nan")
            made.cache.write(k, v, made.table, ints([0, 0], cuda))
            out, lse = made.cache.attend(q, made.table, made.lengths, SCALING, mask=m, return_lse=True)
            assert torch.equal(out[:, :i], want[:, :i]) and torch.equal(lse[:, :i], wlse[:, :i])
            bad = torch.isnan(out[0, i:])
            assert bad[..., 64:96].all() and not bad[..., :64].any() and not bad[..., 96:].any()
            assert torch.equal(lse[0], wlse[0]) and torch.isnan(lse[1, i:]).all() and torch.isnan(out[1, i:]).all()
        made.cache.write(made.k, made.v, made.table, ints([0, 0], cuda))
    mask[:, n - 1] = float("-inf")                                    # masked for all: nobody's
    want = made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask)
    v = made.v.clone()
    v[:, n - 1] = float("nan")
    made.cache.write(made.k, v, made.table, ints([0, 0], cuda))
    assert torch.equal(want, made.cache.attend(q, made.table, made.lengths, SCALING, mask=mask))


def test_workspaces_of_many_streams_are_bounded(cuda):
    """The scratch of a few streams is kept, whichever come, and can be let go."""
    from starkv import kv4
    made = Made(cuda, [3000, 17, 1024], 2, 64, F16, seed=63)
    q = rnd((3, 1, 8, 128), F16, 64, cuda)
    want = made.cache.attend(q, made.table, made.lengths, SCALING)
    pages = made.cache.select(q, made.table, made.lengths, 4)
    torch.cuda.synchronize()
    kv4.release_workspaces()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    streams = [torch.cuda.Stream() for _ in range(20)]
    got = []
    for _ in range(2):
        for st in streams:
            with torch.cuda.stream(st):
                got.append((made.cache.attend(q, made.table, made.lengths, SCALING), made.cache.select(q, made.table, made.lengths, 4)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, pages) for a, b in got)
    assert len({s.cuda_stream for s in streams}) > 10 >= kv4._MAX_WORKSPACES
    assert torch.cuda.memory_allocated() - before <= kv4._MAX_WORKSPACES * (kv4._attention_size() + (1 << 20)) + (4 << 20)
    kv4.release_workspaces()
    del got
    assert torch.cuda.memory_allocated() - before <= 1 << 20
    assert torch.equal(want, made.cache.attend(q, made.table, made.lengths, SCALING))


def test_copies_have_pools_of_their_own(cuda):
    """copy.deepcopy (a prompt's cache reused) and pickling: the copy holds the same tokens, and
    writing into one leaves the other as it is; a shallow copy shares the pool."""
    import copy
    import pickle
    from starkv.attention import StarKVCache
    from starkv.kv4_attention import KV4State
    made = Made(cuda, [300, 77], 2, 64, F16, seed=65, garbage=False)
    q = rnd((2, 1, 8, 128), F16, 66, cuda)
    want = made.cache.attend(q, made.table, made.lengths, SCALING)
    whole = StarKVCache(400)
    whole.kv4_states[0] = KV4State(2, 400, 2, 64, cuda, page_bounds=True)
    whole.kv4_states[0].append(made.k, made.v)
    other = copy.deepcopy(whole)
    new = rnd((2, 1, 2, 128), F16, 67, cuda)
    before = [t.clone() for t in whole.kv4_states[0].history(F32)]
    other.kv4_states[0].append(new, new)
    assert (other.get_seq_length(), whole.get_seq_length()) == (301, 300)
    assert all(torch.equal(a, b) for a, b in zip(before, whole.kv4_states[0].history(F32)))
    assert all(torch.equal(a, b[:, :300]) for a, b in zip(before, other.kv4_states[0].history(F32)))
    for twin in (copy.deepcopy(made.cache), pickle.loads(pickle.dumps(made.cache))):
        assert twin.data.data_ptr() != made.cache.data.data_ptr() and torch.equal(twin.bounds, made.cache.bounds)
        twin.write(new, new, made.table, ints([0, 0], cuda))
        assert not torch.equal(twin.attend(q, made.table, made.lengths, SCALING), want)
        assert torch.equal(made.cache.attend(q, made.table, made.lengths, SCALING), want)
    bare = copy.deepcopy(KV4Cache(3, 1, page_bounds=False, device=cuda))
    assert bare.bounds is None and bare.num_pages == 3
    shared = copy.copy(made.cache)
    assert shared.data is made.cache.data and torch.equal(shared.attend(q, made.table, made.lengths, SCALING), want)


@pytest.mark.parametrize("scale,grow", [(1e-5, 1), (1e-4, 1), (1e-3, 1), (1e-2, 1), (1.0, 1), (1e-5, 40), (1e-5, 3000), (1e-4, 100), (0.05, 40)])
def test_attention_to_many_small_values_behind_one_peak(cuda, scale, grow):
    """One key holds nearly all the weight, the others 2^-20 of its weight each, so many in a warp's
    stretch that together they are some hundredths; the values may be far below one and grow on the
    way.  The bound at the head of this file without its absolute part: what the small weights add is
    not lost below fp16's range."""
    B, H, page, n = 8, 32, 128, 131072
    W = n // page
    k = rnd((1, n, 1, 128), F16, 71, cuda)
    v = rnd((1, n, 1, 128), F32, 72, cuda).clamp(-3, 3)
    v[..., ::32] = 4.0                                        # code 7 in every token: losses do not average out
    at = torch.arange(n, device=cuda)[None, :, None, None] / 128 % 100 / 100    # again and again within a stretch's length
    v = v * scale * torch.where(at > 0.6, float(grow), torch.where(at > 0.3, grow ** 0.5, 1.0))
    cache = KV4Cache(B * W, H, page_size=page, device=cuda, page_bounds=False)
    table = table_of(B, W, cuda, 5)
    cache.write(k.float().expand(B, n, H, 128), v.expand(B, n, H, 128), table, ints([0] * B, cuda))
    mask = torch.full((B, n), -14.0, device=cuda)
    mask[:, 37] = 0
    q = torch.zeros(B, 1, H, 128, dtype=F16, device=cuda)
    out = torch.empty(q.shape, device=cuda)
    cache.attend(q, table, ints([n] * B, cuda), SCALING, mask=mask, out=out)
    vals = O.values(f64(v[0, :, 0]))
    c, s, m = O.quantise(f64(v[0, :, 0]))
    w = np.exp(f64(mask[0]))
    w /= w.sum()
    size = (np.abs(s[..., None] * c) + np.abs(m)[..., None]).reshape(n, 128)
    tol = (2 * U * (1 + 2 * U) + 2.0 ** -18) * (w @ size)
    err = np.abs(f64(out[:, 0]) - w @ vals)                   # the same tokens in every sequence and head
    assert (err <= tol).all(), (err / tol).max()
