"""Left-padded batches through transformers' own model code with ``KV4Attention`` layers:
each sequence of the batch against the same sequence alone.

Tolerance.  The first layer's keys and values come from the same embeddings and the same
positions, so they differ by at most an fp16 rounding (another shape of the projection's
product).  A rounding of 2^-11 moves a 4-bit code, whose step is about a fifteenth of a range
of four standard deviations, in at most one value of a hundred, by one step: 0.1 x 4 / 15 of the
values' own size, 2.7e-2, where nothing averages out.  Attending to padding shows as order 1."""

import pytest
import torch

from starkv.attention import StarKVCache
from starkv.e2e import build_model

pytestmark = pytest.mark.gpu
TOLERANCE = 2.7e-2


def rel(a, b):
    return float(torch.linalg.vector_norm(a.double() - b.double()) / torch.linalg.vector_norm(b.double()))


def small_model(cuda, kv4_layers, quantized=False, **kw):
    return build_model(num_layers=2, hidden=512, heads=4, kv_heads=2, mlp=1024, vocab=1000, v_block_kv=2,
                       quantized=quantized, seed=11, device=cuda, max_positions=512, kv4_layers=kv4_layers, **kw)


def first_layer(model):
    """Keeps what the first layer's attention returns."""
    seen = []
    model.model.layers[0].self_attn.register_forward_hook(lambda m, a, out: seen.append(out[0]))
    return seen


def four_dims(keep, T, dtype):
    """The padding mask keep (B, n) with causality as an additive mask of the newest T tokens."""
    B, n = keep.shape
    ok = keep[:, None].bool() & torch.ones(T, n, dtype=torch.bool, device=keep.device).tril(n - T)
    return torch.zeros(B, 1, T, n, dtype=dtype, device=keep.device).masked_fill_(~ok[:, None], torch.finfo(dtype).min)


@torch.no_grad()
def run_padded(model, seqs, steps, kind):
    """The prompt seqs[b] left-padded to one length, then `steps` token counts at once; returns
    the first layer's outputs, one a call."""
    dev = model.device
    seen = first_layer(model)
    P = max(len(s) for s, _ in seqs)
    cache = StarKVCache(P + sum(steps) + 8)
    prompt = torch.stack([torch.cat([s.new_zeros(P - len(s)), s]) for s, _ in seqs])
    keep = torch.stack([torch.arange(P, device=dev) >= P - len(s) for s, _ in seqs]).long()
    model(input_ids=prompt, attention_mask=keep, position_ids=(keep.cumsum(1) - 1).clamp(min=0), past_key_values=cache,
          use_cache=True)
    at = 0
    for T in steps:
        ids = torch.stack([new[at:at + T] for _, new in seqs])
        at += T
        keep = torch.cat([keep, keep.new_ones(len(seqs), T)], 1)
        mask = keep if kind == "2d" else four_dims(keep, T, torch.float16)
        out = model(input_ids=ids, attention_mask=mask, position_ids=keep.cumsum(1)[:, -T:] - 1, past_key_values=cache,
                    use_cache=True)
        assert torch.isfinite(out.logits).all()
    return seen


def sequences(dev, lens, more):
    g = torch.Generator(device=dev).manual_seed(12)
    draw = lambda n: torch.randint(1, 1000, (n,), generator=g, device=dev)  # noqa: E731
    return [(draw(n), draw(more)) for n in lens]


def check_padded(cuda, steps, kind, lens=(40, 150, 7)):
    model = small_model(cuda, (0, 1))
    seqs = sequences(cuda, lens, sum(steps))
    got = run_padded(model, seqs, steps, kind)
    for b, (s, new) in enumerate(seqs):
        alone = run_padded(small_model(cuda, (0, 1)), [(s, new)], steps, kind)
        for x, y in zip(got[1:], alone[1:]):
            assert rel(x[b], y[0]) <= TOLERANCE, (b, x.shape, rel(x[b], y[0]))


@pytest.mark.parametrize("kind", ["2d", "additive"])
def test_decode_steps(cuda, kind):
    """``2d``: transformers makes a boolean 4-D mask of the padding mask."""
    check_padded(cuda, (1, 1, 1), kind)


@pytest.mark.parametrize("quantized", [False, True])
@torch.no_grad()
def test_latent_layers_take_boolean_masks(cuda, quantized):
    """A boolean decode mask gives the latent layers what the additive one does."""
    outs = []
    for kind in (torch.bool, torch.long, torch.float16):
        model = small_model(cuda, (), quantized)
        g = torch.Generator(device=cuda).manual_seed(13)
        ids = torch.randint(0, 1000, (2, 40), generator=g, device=cuda)
        cache = StarKVCache(64, quantized=quantized)
        model(input_ids=ids, past_key_values=cache, use_cache=True)
        keep = torch.ones(2, 1, 1, 41, dtype=torch.bool, device=cuda)
        keep[0, ..., :17] = False
        mask = keep.to(kind) if kind != torch.float16 else torch.zeros(keep.shape, dtype=kind, device=cuda).masked_fill_(~keep, float("-inf"))
        x = torch.randn(2, 1, 512, generator=g, device=cuda).half()
        cos, sin = model.model.rotary_emb(x, torch.full((2, 1), 40, device=cuda))
        attn = model.model.layers[0].self_attn
        outs.append(attn(x, (cos, sin), mask, **({"past_key_values_upper": cache} if quantized else {"past_key_values": cache}))[0])
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("kind", ["2d", "additive"])
def test_drafts(cuda, kind):
    check_padded(cuda, (3, 1, 4), kind)


def with_rows(q, k, v, rows, scaling):
    """64-bit attention of q (B, T, Hq, 128) over k / v (B, n, Hkv, 128) with the additive mask rows (B, T, n)."""
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    grp = q.shape[1] // k.shape[1]
    s = q @ k.repeat_interleave(grp, 1).transpose(-1, -2) * scaling + rows[:, None].double()
    return (torch.softmax(s, -1) @ v.repeat_interleave(grp, 1)).transpose(1, 2)


@pytest.mark.parametrize("kind", ["bool", "additive", "later"])
@torch.no_grad()
def test_draft_masks_whose_rows_differ(cuda, kind):
    """A draft's tree: a token attends to the history and its own ancestors; ``later``: and a
    token that comes after it.  Within 2e-3 as in test_gpu_kv4_attention.py."""
    attn = small_model(cuda, (0, 1)).model.layers[0].self_attn
    attn.o_proj = torch.nn.Identity()
    B, P, T = 2, 90, 5
    g = torch.Generator(device=cuda).manual_seed(14)
    x = torch.randn(B, P + T, 512, generator=g, device=cuda).half() * 20
    one = torch.ones(B, 1, 128, device=cuda, dtype=torch.float16)     # no rotation
    pos = (one, one * 0)
    cache = StarKVCache(128)
    attn(x[:, :P], pos, None, past_key_values=cache)
    keep = torch.ones(B, 1, T, P + T, dtype=torch.bool, device=cuda)
    keep[0, ..., :33] = False                                         # padding
    tree = torch.tensor([[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 1, 0, 1, 0], [1, 0, 1, 0, 1]], device=cuda).bool()
    if kind == "later":
        tree[1, 4] = True
    keep[..., P:] = tree
    rows = torch.zeros(keep.shape, dtype=torch.float16, device=cuda).masked_fill_(~keep, float("-inf"))
    out, _ = attn(x[:, P:], pos, keep if kind == "bool" else rows, past_key_values=cache)
    q, _, _ = attn.heads(x[:, P:], *pos)
    want = with_rows(q, *cache.kv4_states[0].history(torch.float32), rows[:, 0], attn.scaling)
    assert rel(out, want.flatten(2)) <= 2e-3
    # the same rows from a CUDA graph, which cannot look at them
    state, held = cache.kv4_states[0], P
    def again():
        state.lengths.fill_(held)
        state.length = held
        return attn(x[:, P:], pos, keep, past_key_values=cache)[0]
    if kind == "bool":
        again()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = again()
        graph.replay()
        assert torch.equal(got, out)


def state_of(cuda, n, page=64, B=1, seed=15):
    """A KV4State with n random tokens a sequence, 2 KV heads."""
    from starkv.kv4_attention import KV4State
    st = KV4State(B, n + 64, 2, page, cuda, page_bounds=True)
    g = torch.Generator(device=cuda).manual_seed(seed)
    draw = lambda *s: torch.randn(*s, generator=g, device=cuda).half()  # noqa: E731
    st.append(draw(B, n, 2, 128), draw(B, n, 2, 128))
    return st, draw


@pytest.mark.parametrize("page,T,over", [(64, 4, 1), (64, 16, 1), (64, 16, 15), (64, 16, 0), (16, 16, 1), (16, 5, 4), (32, 2, 1), (128, 1, 5)])
def test_kept_pages_hold_the_drafts_themselves(cuda, page, T, over):
    """T drafts whose newest `over` tokens are in the last page: every query's own position is
    among the pages kept, whatever the others score and however few are asked for."""
    n = page * 20 + over
    st, draw = state_of(cuda, n, page)
    for keep in (1, 2, 8):
        q = draw(1, T, 8, 128)
        pages = st.select(q, keep)
        own = set(range((n - T) // page, (n - 1) // page + 1))
        for h in range(2):
            got = [p for p in pages[0, h].tolist() if p >= 0]
            assert own <= set(got) and 0 in got and len(got) == len(set(got)) and len(got) >= keep
        # rows that see everything up to themselves, one by one over the same pages
        rows = torch.where(torch.ones(T, n, device=cuda).tril(n - T) > 0, 0.0, float("-inf"))[None]
        a, b = st.attend(q, 128 ** -0.5, keep_pages=keep), st.attend_rows(q, 128 ** -0.5, rows, keep_pages=keep)
        hide = torch.full((1, T, n), float("-inf"), device=cuda)
        k, v = st.history(torch.float32)
        for h in range(2):
            kept = torch.isin(torch.arange(n, device=cuda) // page, pages[0, h])
            want = with_rows(q[:, :, 4 * h:4 * h + 4], k[:, :, h:h + 1], v[:, :, h:h + 1], torch.where(kept, rows, hide), 128 ** -0.5)
            assert rel(a[:, :, 4 * h:4 * h + 4], want) <= 2e-3
        assert torch.isfinite(b).all()
        if T == 1:
            assert rel(b, a) <= 2e-3


@torch.no_grad()
def test_module_drafts_with_kept_pages(cuda):
    """Fewest pages, drafts over the end of a page: the first page and the drafts' own."""
    attn = small_model(cuda, (0, 1), kv4_keep_pages=2).model.layers[0].self_attn
    attn.o_proj = torch.nn.Identity()
    P, T = 64 * 6 - 3, 5
    g = torch.Generator(device=cuda).manual_seed(16)
    x = torch.randn(1, P + T, 512, generator=g, device=cuda).half() * 20
    one = torch.ones(1, 1, 128, device=cuda, dtype=torch.float16)
    cache = StarKVCache(512)
    attn(x[:, :P], (one, one * 0), None, past_key_values=cache)
    out, _ = attn(x[:, P:], (one, one * 0), None, past_key_values=cache)
    n = P + T
    at = torch.arange(n, device=cuda)
    ok = (at[None] <= torch.arange(P, n, device=cuda)[:, None]) & ((at < 64) | (at >= 64 * 5))
    q, _, _ = attn.heads(x[:, P:], one, one * 0)
    want = with_rows(q, *cache.kv4_states[0].history(torch.float32), torch.where(ok, 0.0, float("-inf"))[None], attn.scaling)
    assert rel(out, want.flatten(2)) <= 2e-3


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float16).min, torch.finfo(torch.float32).min])
def test_kept_pages_leave_padding_out(cuda, low):
    """A sequence behind whole pages of padding keeps the pages it keeps alone; padding that ends
    inside a page, a sequence that is all padding, and a mask narrower than the sequence."""
    from starkv.kv4_attention import KV4State
    page, n, pads = 64, 64 * 16 + 9, (64 * 7, 0, 64 * 3 + 10, 64 * 16 + 9, 64 * 15)
    st, draw = state_of(cuda, n, page, B=5)
    q = draw(5, 2, 8, 128)
    mask = torch.zeros(5, n, device=cuda)
    for b, m in enumerate(pads):
        mask[b, :m] = low
    pages = st.select(q, 5, mask)
    k, v = st.history(torch.float16)
    out = st.attend(q, 128 ** -0.5, mask, keep_pages=5)
    for b in (0, 1):
        alone = KV4State(1, n + 64, 2, page, cuda, page_bounds=True)
        alone.append(k[b:b + 1, pads[b]:], v[b:b + 1, pads[b]:])
        # stored values quantise to other codes than the tokens did: the same pool is needed for the same bounds
        alone.cache.data[:st.width - pads[b] // page].copy_(st.cache.data[b * st.width + pads[b] // page:(b + 1) * st.width])
        alone.cache.bounds[:st.width - pads[b] // page].copy_(st.cache.bounds[b * st.width + pads[b] // page:(b + 1) * st.width])
        alone.cache.bound_scales[:st.width - pads[b] // page].copy_(st.cache.bound_scales[b * st.width + pads[b] // page:(b + 1) * st.width])
        assert torch.equal(alone.select(q[b:b + 1], 5) + pads[b] // page, pages[b:b + 1])
        want = alone.attend(q[b:b + 1], 128 ** -0.5, keep_pages=5)
        assert rel(out[b:b + 1], want) <= 2e-3
    assert (pages[2, :, 0] == 3).all() and (pages[2].amin() >= 3) and (pages[2, :, -2:].cpu() == torch.tensor([15, 16])).all()
    assert (pages[4].cpu() == torch.tensor([15, 16, -1, -1, -1])).all()
    assert (pages[3, :, 0] == 16).all() and st.cache.read_error() == 0
    if low == float("-inf"):
        assert (out[3] == 0).all()
    # positions past the mask count
    assert torch.equal(st.select(q, 5, mask[:, :64 * 7]), st.select(q, 5, torch.cat([mask[:, :64 * 7], torch.zeros_like(mask[:, 64 * 7:])], 1)))


@torch.no_grad()
def test_padded_batch_with_kept_pages(cuda):
    """Through transformers' code: a short sequence beside a long one keeps all its own pages,
    as it does alone."""
    seqs = sequences(cuda, (400, 160), 2)
    got = run_padded(small_model(cuda, (0, 1), kv4_keep_pages=4), seqs, (1, 1), "2d")
    alone = run_padded(small_model(cuda, (0, 1), kv4_keep_pages=4), seqs[1:], (1, 1), "2d")
    for x, y in zip(got[1:], alone[1:]):
        assert rel(x[1], y[0]) <= TOLERANCE


@torch.no_grad()
def test_keep_pages_set_after_the_prompt(cuda):
    """keep_pages may change from step to step."""
    outs = []
    for late in (False, True):
        attn = small_model(cuda, (0, 1), kv4_keep_pages=0 if late else 3).model.layers[0].self_attn
        g = torch.Generator(device=cuda).manual_seed(17)
        x = torch.randn(1, 401, 512, generator=g, device=cuda).half() * 20
        one = torch.ones(1, 1, 128, device=cuda, dtype=torch.float16)
        cache = StarKVCache(512)
        attn(x[:, :400], (one, one * 0), None, past_key_values=cache)
        attn.keep_pages = 3
        outs.append(attn(x[:, 400:], (one, one * 0), None, past_key_values=cache)[0])
    assert torch.equal(*outs)


@pytest.mark.parametrize("kv4_layers", [(0, 1), (0,), ()])
@torch.no_grad()
def test_rejected_drafts_are_forgotten(cuda, kv4_layers):
    """StarKVCache.crop: drafts (single tokens where a layer holds latents) that are taken back leave
    no trace, over a page's end, with page bounds and after a reset."""
    model = small_model(cuda, kv4_layers, kv4_keep_pages=3)
    from starkv.e2e import forward_tokens
    model.starkv_quantized = False
    g = torch.Generator(device=cuda).manual_seed(18)
    ids = torch.randint(0, 1000, (2, 230), generator=g, device=cuda)
    P = 62
    step = 6 if kv4_layers == (0, 1) else 1
    plain, cache = StarKVCache(256), StarKVCache(256)
    for c in (plain, cache):
        forward_tokens(model, ids[:, :P], 0, c)
    for turn in range(2):
        wrong = torch.randint(0, 1000, (2, 2 * step), generator=g, device=cuda)
        for i in range(2):
            forward_tokens(model, wrong[:, i * step:(i + 1) * step], P + i * step, cache)
        assert cache.get_seq_length() == P + 2 * step
        cache.crop(P + 1 if turn else -2 * step)
        if turn:
            cache.crop(P)
        assert all(cache.get_seq_length(i) == P for i in range(2))
        for i in range(70):
            a = forward_tokens(model, ids[:, P + i:P + i + 1], P + i, cache)
            b = forward_tokens(model, ids[:, P + i:P + i + 1], P + i, plain)
            assert torch.equal(a, b), i
        P += 70
    cache.crop(1000)
    assert cache.get_seq_length() == P
    cache.reset()
    assert cache.get_seq_length() == 0
    assert torch.equal(forward_tokens(model, ids[:, :100], 0, cache), forward_tokens(model, ids[:, :100], 0, StarKVCache(256)))
