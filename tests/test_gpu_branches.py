"""A prompt's way through layers of whole heads with the operators together: rotary positions by
kernel, packed attention, continuations behind one prompt; modules, the end-to-end loop and
the torch.library ops."""

import copy
import math
import pickle

import pytest
import torch

from starkv import StarKVError, torch_ops  # noqa: F401
from starkv.attention import StarKVCache, apply_rotary_pos_emb_custom
from starkv.e2e import build_model, forward_tokens, generate, generate_branches, generate_graphed
from starkv.kv4 import KV4Cache
from starkv.kv4_attention import KV4Attention, KV4Branches, join_attention
from starkv.prefill import packed_attention
from starkv.rope import Rope

pytestmark = pytest.mark.gpu


class Config:
    hidden_size, num_attention_heads, num_key_value_heads, attention_bias = 1024, 8, 2, False


def rel(a, b):
    return float(torch.linalg.vector_norm(a.double() - b.double()) / torch.linalg.vector_norm(b.double()))


def make(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_operators_together(cuda, dtype):
    """Ragged prompts: turned, attended packed, their keys into pages; then one token each over the
    pages, against 64-bit attention on the turned heads (the cache's 4-bit values read back)."""
    Hq, Hkv, lengths = 8, 2, [5, 130, 64, 1]
    N = sum(lengths)
    cu = torch.tensor([0, *lengths], device=cuda).cumsum(0).to(torch.int32)
    qkv = make((N, (Hq + 2 * Hkv) * 128), dtype, 1)
    q, k, v = (t.view(N, -1, 128) for t in qkv.split([Hq * 128, Hkv * 128, Hkv * 128], -1))
    pos = torch.cat([torch.arange(n, device=cuda) for n in lengths])
    rope = Rope(128, base=500000.0)
    rope.apply(q, k, pos, out=(q, k))
    out, lse = packed_attention(q, k, v, cu, cu, 128 ** -0.5, return_lse=True)
    eps = torch.finfo(dtype).eps / 2
    for b, n in enumerate(lengths):
        s = slice(int(cu[b]), int(cu[b + 1]))
        x, kk, vv = q[s].double(), k[s].double().repeat_interleave(4, 1), v[s].double().repeat_interleave(4, 1)
        z = (torch.einsum("ihd,jhd->hij", x, kk) * 128 ** -0.5).masked_fill(~torch.ones(n, n, dtype=torch.bool, device=cuda).tril(), -math.inf)
        w = torch.softmax(z, -1)
        want = torch.einsum("hij,jhd->ihd", w, vv)
        size = torch.einsum("hij,jhd->ihd", w, vv.abs())
        # half a step for the weights and one for the output; 2^-13 for the scores of some tens (see test_gpu_packed)
        assert bool(((out[s].double() - want).abs() <= (eps + 2.0 ** -13) * size + eps * want.abs() + 2.0 ** -25).all())
    # the longest prompt becomes the prefix of three sequences with a token each
    page, s = 64, slice(int(cu[1]), int(cu[2]))
    cache = KV4Cache(6, Hkv, page_size=page)
    ptable, table = torch.tensor([4, 0, 2], dtype=torch.int32, device=cuda), torch.tensor([[1], [3], [5]], dtype=torch.int32, device=cuda)
    zero = torch.zeros(3, dtype=torch.int32, device=cuda)
    cache.write(k[None, s], v[None, s], ptable[None], zero[:1])
    nq, nk, nv = make((3, 1, Hq, 128), dtype, 2), make((3, 1, Hkv, 128), dtype, 3), make((3, 1, Hkv, 128), dtype, 4)
    nq, nk = rope.apply(nq, nk, torch.full((3, 1), 130, device=cuda))
    cache.write(nk, nv, table, zero)
    plen = torch.tensor([130], dtype=torch.int32, device=cuda)
    got = cache.attend_shared(nq, ptable, plen, table, zero + 1, 128 ** -0.5)
    pk, pv = (t[0].double() for t in cache.read(ptable[None], zero[:1], 130, dtype=torch.float32))
    for b in range(3):
        ok, ov = (t[0].double() for t in cache.read(table[b:b + 1], zero[:1], 1, dtype=torch.float32))
        kk, vv = torch.cat([pk, ok]).repeat_interleave(4, 1), torch.cat([pv, ov]).repeat_interleave(4, 1)
        w = torch.softmax(torch.einsum("hd,jhd->hj", nq[b, 0].double(), kk) * 128 ** -0.5, -1)
        want, size = torch.einsum("hj,jhd->hd", w, vv), torch.einsum("hj,jhd->hd", w, vv.abs())
        group = size.unflatten(-1, (4, 32)).amax(-1, keepdim=True).expand(Hq, 4, 32).flatten(-2)
        assert bool(((got[b, 0].double() - want).abs() <= 2.0 ** -8 * group + eps * want.abs()).all())     # 8 u of the group's largest


@torch.no_grad()
@pytest.mark.parametrize("pieces", [[1, 1, 1], [4, 16, 1], [40, 1, 33, 3]])
def test_module_branches_match_separate_sequences(cuda, pieces):
    """Branches of one prompt against the prompt repeated for each. Both are within u = 2^-11 (weights,
    values, output: some 4 u of sum w |v|) of the same numbers, but for pieces that the one attends
    to from exact heads and the other from 4-bit history alike; relative to the outputs 5e-3."""
    torch.manual_seed(3)
    m = KV4Attention(Config(), layer_idx=0, rope=Rope(128)).to(cuda, torch.float16)
    for p in m.parameters():
        p.data.normal_(0, 0.05)
    B, P = 5, 150
    prompt = make((1, P, 1024), torch.float16, 1)
    one, many = StarKVCache(P), StarKVCache(P + 100)
    a, _ = m(prompt, None, None, past_key_values=one)
    b, _ = m(prompt.expand(B, -1, -1), None, None, past_key_values=many)
    assert torch.equal(a.expand_as(b), b)
    cache = one.branch(B, 100)
    assert cache.get_seq_length() == P and isinstance(cache.kv4_states[0], KV4Branches)
    for i, T in enumerate(pieces):
        x = make((B, T, 1024), torch.float16, 10 + i)
        got, _ = m(x, None, None, past_key_values=cache)
        want, _ = m(x, None, None, past_key_values=many)
        assert rel(got, want) < 5e-3, T
        assert cache.get_seq_length() == many.get_seq_length()
    # rejected drafts are forgotten, the prompt is not
    cache.crop(P + 1)
    many.crop(P + 1)
    x = make((B, 2, 1024), torch.float16, 99)
    assert rel(m(x, None, None, past_key_values=cache)[0], m(x, None, None, past_key_values=many)[0]) < 5e-3
    with pytest.raises(ValueError):
        cache.crop(P - 1)
    # the first cache goes on by itself
    x = make((1, 1, 1024), torch.float16, 7)
    assert one.get_seq_length() == P and cache.get_seq_length() == P + 3


@torch.no_grad()
def test_branch_refusals(cuda):
    m = KV4Attention(Config(), layer_idx=0, rope=Rope(128)).to(cuda, torch.float16)
    with pytest.raises(ValueError):
        StarKVCache(10).branch(2, 3)
    cache = StarKVCache(20)
    m(make((2, 20, 1024), torch.float16, 1), None, None, past_key_values=cache)
    with pytest.raises(ValueError):
        cache.branch(2, 3)                               # two sequences
    cache = StarKVCache(20)
    m(make((1, 20, 1024), torch.float16, 1), None, None, past_key_values=cache)
    new = cache.branch(2, 64)
    with pytest.raises(StarKVError):
        m(make((3, 1, 1024), torch.float16, 1), None, None, past_key_values=new)
    with pytest.raises(NotImplementedError):
        m(make((2, 1, 1024), torch.float16, 1), None, torch.zeros(2, 1, 1, 21, device=cuda), past_key_values=new)
    with pytest.raises(ValueError):
        m(make((2, 65, 1024), torch.float16, 1), None, None, past_key_values=new)


@torch.no_grad()
def test_module_rope_is_that_of_the_tables(cuda):
    """Turned by kernel against fp32 tables of sines: one rounding of fp16, not three."""
    torch.manual_seed(1)
    m = KV4Attention(Config(), layer_idx=0, rope=Rope(128)).to(cuda, torch.float16)
    x = make((2, 9, 1024), torch.float16, 1)
    inv = 1.0 / 10000.0 ** (torch.arange(0, 128, 2, device=cuda).double() / 128)
    pos = torch.arange(9, device=cuda) + 300
    ang = torch.cat([pos[:, None] * inv] * 2, -1)[None]
    q, k, v = m.heads(x, None, None, pos)
    m.rope = None
    q2, k2, v2 = m.heads(x.float().half(), ang.cos().float(), ang.sin().float())
    for a, b in ((q, q2), (k, k2)):
        assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -10 * float(b.abs().max())
    assert torch.equal(v, v2)


def test_rope_copies_and_pickles(cuda):
    rope = Rope(128, scaling=dict(rope_type="linear", factor=2.0))
    x, pos = make((7, 2, 128), torch.float32, 1), torch.arange(7, device=cuda)
    want = rope.apply(x, None, pos)
    for other in (copy.deepcopy(rope), pickle.loads(pickle.dumps(rope))):
        assert torch.equal(other.apply(x, None, pos), want)


@torch.no_grad()
def test_end_to_end(cuda):
    kw = dict(num_layers=2, hidden=512, heads=4, kv_heads=2, mlp=1024, vocab=1000, v_block_kv=2, quantized=False, seed=3, device=cuda,
              max_positions=1024, kv4_layers=range(2))
    model, plain = build_model(kernel_rope=True, **kw), build_model(**kw)
    g = torch.Generator(device=cuda).manual_seed(1)
    prompt = torch.randint(0, 1000, (1, 300), generator=g, device=cuda)
    starts = torch.randint(0, 1000, (6, 3), generator=g, device=cuda)
    # logits of the first step of every branch: behind the one prompt, and each as a prompt of its own
    one = StarKVCache(300, quantized=False)
    a = forward_tokens(model, prompt, 0, one)
    b = forward_tokens(plain, prompt, 0, StarKVCache(300, quantized=False))
    assert rel(a, b) < 1e-2                              # tables rounded to fp16 against exact angles: 2^-11 a layer and head
    many = StarKVCache(310, quantized=False)
    forward_tokens(model, prompt.expand(6, -1), 0, many)
    got, want = forward_tokens(model, starts, 300, one.branch(6, 10)), forward_tokens(model, starts, 300, many)
    assert rel(got, want) < 1e-2
    ids, _ = generate_branches(model, prompt, starts, 8)
    assert ids.shape == (6, 8) and torch.equal(ids, generate_branches(model, prompt, starts, 8)[0])
    assert torch.equal(ids[:, 0], got.argmax(-1))
    # the graphed loop turns by positions on the GPU
    assert torch.equal(generate(model, prompt, 6)[0], generate_graphed(model, prompt, 6)[0])


def test_torch_library_ops(cuda):
    q, k, v = make((30, 4, 128), torch.float16, 1), make((50, 2, 128), torch.float16, 2), make((50, 2, 128), torch.float16, 3)
    cq, ck = torch.tensor([0, 10, 30], dtype=torch.int32, device=cuda), torch.tensor([0, 25, 50], dtype=torch.int32, device=cuda)
    got = torch.ops.starkv.packed_attn(q, k, v, cq, ck, 0.1)
    want = packed_attention(q, k, v, cq, ck, 0.1, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rope = Rope(128, rotary_dim=64, interleaved=True)
    pos = torch.arange(30, device=cuda)
    got = torch.ops.starkv.rope(q, k[:30], pos, rope.turns, rope.factor, True)
    want = rope.apply(q, k[:30], pos)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    cache = KV4Cache(3, 2, page_size=16)
    zero = torch.zeros(2, dtype=torch.int32, device=cuda)
    ptable, table = torch.tensor([1], dtype=torch.int32, device=cuda), torch.tensor([[0], [2]], dtype=torch.int32, device=cuda)
    cache.write(k[None, :16], v[None, :16], ptable[None], zero[:1])
    cache.write(k[:2, None], v[:2, None], table, zero)
    args = (q[:2, None], ptable, zero[:1] + 16, table, zero + 1, 0.1)
    got = torch.ops.starkv.kv4_attn_shared(cache.data, cache.error_word, *args)
    want = cache.attend_shared(*args, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_join_attention(cuda):
    a, b = torch.randn(5, 128, device=cuda), torch.randn(5, 128, device=cuda)
    la, lb = torch.tensor([0.0, -math.inf, 3.0, -math.inf, 100.0], device=cuda), torch.tensor([0.0, 1.0, -math.inf, -math.inf, -100.0], device=cuda)
    a[1] = a[3] = b[2] = b[3] = 0
    got = join_attention(a, la, b, lb)
    for i, want in enumerate(((a[0] + b[0]) / 2, b[1], a[2], 0 * a[3], a[4])):
        assert torch.allclose(got[i], want, rtol=2.0 ** -20, atol=0)


def module(dtype=torch.float16, seed=3, **kw):
    torch.manual_seed(seed)
    m = KV4Attention(Config(), layer_idx=0, **kw).to("cuda", dtype)
    for p in m.parameters():
        p.data.normal_(0, 0.05)
    return m


@torch.no_grad()
@pytest.mark.parametrize("T", [1, 3, 40])
def test_projections_are_not_written_over(cuda, T):
    """A forward hook that keeps a projection's output has it as it was."""
    m = module(rope=Rope(128))
    kept = []
    for proj in (m.q_proj, m.k_proj):
        proj.register_forward_hook(lambda mod, args, out: kept.append((out, out.clone())))
    cache = StarKVCache(100)
    m(make((2, 30, 1024), torch.float16, 1), None, None, past_key_values=cache)
    m(make((2, T, 1024), torch.float16, 2), None, None, past_key_values=cache)
    assert len(kept) == 4 and all(torch.equal(a, b) for a, b in kept)


@pytest.mark.parametrize("train", ["all", "keys"])
def test_projections_get_their_gradients(cuda, train):
    """A piece behind a history (which goes through torch's attention) with the kernel's positions,
    against the same in 64 bits from the history that the cache reads back."""
    m = module(rope=Rope(128))
    for name, p in m.named_parameters():
        p.requires_grad_(train == "all" or name.startswith("k_proj"))
    B, P, T = 2, 37, 20
    cache = StarKVCache(P + T)
    with torch.no_grad():
        m(make((B, P, 1024), torch.float16, 1), None, None, past_key_values=cache)
    x, up = make((B, T, 1024), torch.float16, 2), make((B, T, 1024), torch.float16, 4)
    hk, hv = (t.double() for t in cache.kv4_states[0].history(torch.float32))
    y, _ = m(x, None, None, past_key_values=cache)
    y.backward(up)
    w = {n: p.detach().double().requires_grad_() for n, p in m.named_parameters()}
    heads = lambda n: (x.double() @ w[n + ".weight"].T).view(B, T, -1, 128)  # noqa: E731
    f = torch.tensor(m.rope.frequencies, dtype=torch.float64, device=cuda)
    angle = (torch.arange(P, P + T, device=cuda).double()[:, None] * f)[:, None]

    def turn(t):
        a, b = t[..., :64], t[..., 64:]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    k, v = torch.cat([hk, turn(heads("k_proj"))], 1), torch.cat([hv, heads("v_proj")], 1)
    s = torch.einsum("bihd,bjhd->bhij", turn(heads("q_proj")), k.repeat_interleave(4, 2)) * m.scaling
    s = s.masked_fill(~torch.ones(T, P + T, dtype=torch.bool, device=cuda).tril(P), -math.inf)
    o = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v.repeat_interleave(4, 2)).reshape(B, T, -1)
    (o @ w["o_proj.weight"].T).backward(up.double())
    for n, p in m.named_parameters():
        if p.requires_grad:
            # eight roundings of 2^-11 one after the other (projections, turn, scores, weights, outputs, gradients of
            # each); they are independent over the sums that a gradient is, so of its norm at most that
            assert rel(p.grad, w[n].grad) <= 8 * 2.0 ** -11, n
        else:
            assert p.grad is None


def masks_of(B, T, n):
    """A causal mask of the newest T of n tokens in the forms that models make."""
    seen = torch.ones(T, n, dtype=torch.bool, device="cuda").tril(n - T).expand(B, 1, T, n)
    for low in (-math.inf, torch.finfo(torch.float16).min):
        yield torch.zeros(seen.shape, dtype=torch.float16, device="cuda").masked_fill(~seen, low)
    yield seen
    yield torch.nn.functional.pad(seen[:1].long(), (0, 5))                  # wider than what is held


@torch.no_grad()
@pytest.mark.parametrize("T", [2, 16, 17, 40])
def test_branches_take_causal_masks(cuda, T):
    m, B, P = module(rope=Rope(128)), 3, 90
    one = StarKVCache(P)
    m(make((1, P, 1024), torch.float16, 1), None, None, past_key_values=one)
    x, first = make((B, T, 1024), torch.float16, 2), make((B, 1, 1024), torch.float16, 5)

    def run(mask):
        cache = one.branch(B, 60)
        m(first, None, None, past_key_values=cache)
        return m(x, None, mask, past_key_values=cache)[0]

    want = run(None)
    for mask in masks_of(B, T, P + 1 + T):
        assert torch.equal(run(mask), want)
    # what a mask says beyond causality is refused, and nothing is written
    for at, value in (((0, 0, T - 1, 3), False), ((1, 0, 0, P), False), ((2, 0, 0, P + 2), True)):
        mask = torch.ones(T, P + 1 + T, dtype=torch.bool, device=cuda).tril(P + 1).expand(B, 1, -1, -1).clone()
        mask[at] = value
        cache = one.branch(B, 60)
        m(first, None, None, past_key_values=cache)
        for bad in (mask, mask[..., :-1], torch.cat([mask, mask], 1), mask[:, :, 1:]):
            with pytest.raises(NotImplementedError):
                m(x, None, bad, past_key_values=cache)
        assert cache.get_seq_length() == P + 1 and torch.equal(m(x, None, None, past_key_values=cache)[0], want)


@torch.no_grad()
@pytest.mark.parametrize("attention", ["sdpa", "eager"])
def test_branches_through_a_transformers_model(cuda, attention):
    """Tokens, drafts and longer pieces of branches by the model's own forward, which makes the masks,
    against the layers called one by one."""
    kw = dict(num_layers=2, hidden=512, heads=4, kv_heads=2, mlp=1024, vocab=1000, v_block_kv=2, quantized=False, seed=3, device=cuda,
              max_positions=1024, kv4_layers=range(2), kernel_rope=True)
    model = build_model(**kw)
    model.config._attn_implementation = attention
    g = torch.Generator(device=cuda).manual_seed(1)
    prompt = torch.randint(0, 1000, (1, 300), generator=g, device=cuda)
    one = StarKVCache(300, quantized=False)
    forward_tokens(model, prompt, 0, one)
    by_hand, by_model = one.branch(4, 70), one.branch(4, 70)
    at = 300
    for T in (3, 40, 5) if attention == "eager" else (1, 3, 40, 1, 16):
        ids = torch.randint(0, 1000, (4, T), generator=g, device=cuda)
        want = forward_tokens(model, ids, at, by_hand)
        pos = torch.arange(at, at + T, device=cuda)[None]
        got = model(input_ids=ids, position_ids=pos, past_key_values=by_model, use_cache=True).logits[:, -1]
        # the same kernels on the same numbers, but for the model's own fp16 tables of sines, which are not used
        assert torch.equal(got, want), T
        at += T
        assert by_model.get_seq_length() == by_hand.get_seq_length() == at


@torch.no_grad()
@pytest.mark.parametrize("first", [1, 16, 40])
def test_reset_of_branches(cuda, first):
    """After reset branches are sequences that share nothing: as a new cache of theirs, from the first
    token on."""
    m, B = module(rope=Rope(128)), 3
    one = StarKVCache(70)
    m(make((1, 70, 1024), torch.float16, 1), None, None, past_key_values=one)
    cache = one.branch(B, 64)
    m(make((B, 5, 1024), torch.float16, 2), None, None, past_key_values=cache)
    for _ in range(2):
        cache.reset()
        assert cache.get_seq_length() == 0
        new = StarKVCache(64)
        for i, T in enumerate((first, 1, 7, 1)):
            x = make((B, T, 1024), torch.float16, 10 + i)
            got, want = (m(x, None, None, past_key_values=c)[0] for c in (cache, new))
            # (of a first piece of up to 16 tokens, one attends to its own tokens' 4-bit heads and the other to exact ones)
            assert i == 0 and 1 < first <= 16 or rel(got, want) < 5e-3, T
            assert cache.get_seq_length() == new.get_seq_length()
        cache.crop(first + 1)
        assert cache.get_seq_length() == first + 1
        with pytest.raises(ValueError):
            m(make((B, 64, 1024), torch.float16, 9), None, None, past_key_values=cache)
    # the cache it came from is as it was
    assert one.get_seq_length() == 70
    one.reset()
    assert one.get_seq_length() == 0


@torch.no_grad()
@pytest.mark.parametrize("own", [0, 3])
def test_pieces_of_branches_report_errors(cuda, own):
    """A wait that runs out in a longer piece's attention, behind the prompt or among the own tokens, is in
    the layer's error word; the next piece is what it was."""
    from starkv import ops
    m, B, P, T = module(rope=Rope(128)), 3, 2000, 40
    one = StarKVCache(P)
    m(make((1, P, 1024), torch.float16, 1), None, None, past_key_values=one)
    x = make((B, T, 1024), torch.float16, 2)

    def run():
        cache = one.branch(B, 60)
        if own:
            m(make((B, own, 1024), torch.float16, 3), None, None, past_key_values=cache)
        return cache.kv4_states[0].cache, m(x, None, None, past_key_values=cache)[0]

    pool, want = run()
    assert pool.read_error() == 0
    try:
        cache = one.branch(B, 60)
        if own:
            m(make((B, own, 1024), torch.float16, 3), None, None, past_key_values=cache)
        ops.set_test_hooks(wait_limit_ns=20_000_000, skip_copy_unit=1)
        m(x, None, None, past_key_values=cache)
        assert cache.kv4_states[0].cache.read_error() in (0x101, 0x102)
    finally:
        ops.set_test_hooks()
    for _ in range(2):
        pool, got = run()
        assert pool.read_error() == 0 and torch.equal(got, want)


@torch.no_grad()
def test_refused_calls_of_branches_leave_no_token(cuda):
    m, B = module(rope=Rope(128)), 2
    one = StarKVCache(30)
    m(make((1, 30, 1024), torch.float16, 1), None, None, past_key_values=one)
    cache, x = one.branch(B, 40), make((B, 3, 1024), torch.float16, 2)
    want = m(x, None, None, past_key_values=cache)[0]
    for n, bad in enumerate((dict(keep_pages=4), dict(mask=torch.zeros(B, 1, 3, 5, device=cuda)), dict(batch=B + 1), dict(tokens=70))):
        cache = one.branch(B, 40)
        st = cache.kv4_states[0]
        m.keep_pages = bad.get("keep_pages", 0)
        y = make((bad.get("batch", B), bad.get("tokens", 3), 1024), torch.float16, 3)
        with pytest.raises((NotImplementedError, ValueError, StarKVError)):
            m(y, None, bad.get("mask"), past_key_values=cache)
        m.keep_pages = 0
        assert cache.get_seq_length() == 30 and not bool(st.lengths.any()), n
        assert torch.equal(m(x, None, None, past_key_values=cache)[0], want), n
