"""``KV4Attention`` (whole heads in the paged 4-bit cache) in its three uses, against
64-bit attention over what the cache reads back, and the mixed end-to-end loop.

Tolerance: fp16 queries, keys and projections as the module has them; the attention's
own error is bounded by 2^-10 of sum w |v| (see test_gpu_kv4.py) and the output
projection rounds once more, so rel-L2 <= 2e-3 as for the latent modules."""

import pytest
import torch

from starkv.attention import StarKVCache
from starkv.e2e import build_model, forward_tokens, generate, generate_graphed
from starkv.kv4_attention import KV4Attention, KV4State

pytestmark = pytest.mark.gpu


class Config:
    hidden_size, num_attention_heads, num_key_value_heads, attention_bias = 1024, 8, 2, False


def tables(start, T, dev):
    inv = 1.0 / 10000.0 ** (torch.arange(0, 128, 2, device=dev).float() / 128)
    ang = torch.arange(start, start + T, device=dev).float()[:, None] * inv
    emb = torch.cat([ang, ang], -1)[None]
    return emb.cos().half(), emb.sin().half()


def reference(m, q, k, v, mask=None):
    """64-bit attention of the newest queries, through the module's output projection."""
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    grp = q.shape[1] // k.shape[1]
    s = q @ k.repeat_interleave(grp, 1).transpose(-1, -2) * m.scaling
    T, n = s.shape[-2:]
    s = s.masked_fill(~torch.ones(T, n, dtype=torch.bool, device=s.device).tril(n - T), float("-inf"))
    if mask is not None:
        s = s + mask[:, None, None].double()
    o = torch.softmax(s, -1) @ v.repeat_interleave(grp, 1)
    return o.transpose(1, 2).flatten(2) @ m.o_proj.weight.double().T


def rel(a, b):
    return float(torch.linalg.vector_norm(a.double() - b) / torch.linalg.vector_norm(b))


@pytest.fixture
def module(cuda):
    torch.manual_seed(3)
    m = KV4Attention(Config(), layer_idx=0).to(cuda, torch.float16)
    for p in m.parameters():
        p.data.normal_(0, 0.05)
    return m


@torch.no_grad()
def test_prompt_decode_and_continuation(cuda, module):
    B, P = 2, 150
    cache = StarKVCache(capacity=400)
    g = torch.Generator(device=cuda).manual_seed(4)
    at = 0
    for T in (P, 1, 1, 5, 30, 1):                          # prompt, tokens, a draft, a longer continuation, a token
        x = torch.randn(B, T, 1024, generator=g, device=cuda, dtype=torch.float16)
        pos = tables(at, T, cuda)
        q, k, v = module.heads(x, *pos)
        st = cache.kv4_states.get(0)
        old = st.history(torch.float32) if at else None
        out, _ = module(x, pos, None, past_key_values=cache)
        st = cache.kv4_states[0]
        at += T
        assert st.length == at == cache.get_seq_length(0) and st.lengths.tolist() == [at] * B
        if T == P:                                         # exact heads
            want = reference(module, q, k, v)
        elif T > 16:                                       # history from the pages, the new tokens exact
            want = reference(module, q, *(torch.cat([o, n.float()], 1) for o, n in zip(old, (k, v))))
        else:
            want = reference(module, q, *st.history(torch.float32))
        assert out.shape == (B, T, 1024) and rel(out, want) <= 2e-3, (T, rel(out, want))
    assert st.cache.read_error() == 0


@torch.no_grad()
def test_decode_mask_and_kept_pages(cuda, module):
    B, P = 2, 200
    cache = StarKVCache(capacity=256)
    g = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn(B, P, 1024, generator=g, device=cuda, dtype=torch.float16)
    module(x, tables(0, P, cuda), None, past_key_values=cache)
    y = torch.randn(B, 1, 1024, generator=g, device=cuda, dtype=torch.float16)
    mask = torch.zeros(B, 1, 1, P + 1, device=cuda, dtype=torch.float16)
    mask[0, ..., :70] = float("-inf")
    out, _ = module(y, tables(P, 1, cuda), mask, past_key_values=cache)
    st = cache.kv4_states[0]
    q, _, _ = module.heads(y, *tables(P, 1, cuda))
    assert rel(out, reference(module, q, *st.history(torch.float32), mask=mask[:, 0, 0].float())) <= 2e-3
    kept = KV4State(B, 256, 2, 64, cuda, page_bounds=True)
    k, v = st.history(torch.float16)
    kept.append(k, v)
    few = kept.attend(q, module.scaling, keep_pages=2)      # first and last page of four
    pages = torch.zeros(B, P + 1, dtype=torch.bool, device=cuda)
    pages[:, :64] = pages[:, 192:] = True
    hide = torch.where(pages, 0.0, float("-inf"))
    want = kept.attend(q, module.scaling, mask=hide)
    assert torch.allclose(few.float(), want.float(), rtol=2e-3, atol=2e-3)
    every = kept.attend(q, module.scaling, keep_pages=9)
    assert torch.allclose(every.float(), kept.attend(q, module.scaling).float(), rtol=2e-3, atol=2e-3)


def test_refusals(cuda, module):
    x = torch.zeros(1, 1, 1024, device=cuda, dtype=torch.float16)
    with pytest.raises(TypeError):
        module(x, tables(0, 1, cuda), None)
    with pytest.raises(ValueError):                         # a full cache
        cache = StarKVCache(capacity=64)
        with torch.no_grad():
            module(torch.zeros(1, 65, 1024, device=cuda, dtype=torch.float16), tables(0, 65, cuda), None, past_key_values=cache)

    class Narrow(Config):
        num_attention_heads = 16
    with pytest.raises(ValueError):
        KV4Attention(Narrow())


@pytest.mark.parametrize("keep", [0, 2])
def test_mixed_layers_graphed_loop_matches_eager(cuda, keep):
    """Latent and whole-head layers in one model: the graph-replayed loop gives the eager loop's tokens."""
    model = build_model(num_layers=3, hidden=512, heads=4, kv_heads=4, mlp=1024, vocab=1000, v_block_kv=2,
                        quantized=True, seed=7, device=cuda, max_positions=1024, kv4_layers=(0, 2), kv4_keep_pages=keep)
    g = torch.Generator(device=cuda).manual_seed(3)
    for B in (1, 3):
        prompt = torch.randint(0, 1000, (B, 150), generator=g, device=cuda)
        a, _ = generate(model, prompt, 45)                  # past a page's end
        b, _ = generate_graphed(model, prompt, 45)
        assert torch.equal(a, b)


def test_mixed_layers_decode_matches_recompute(cuda):
    """A token decoded through the caches against the whole sequence through the prompt
    path: logits differ by the 4-bit heads only (5 bits a value: rel-L2 within 0.2)."""
    model = build_model(num_layers=2, hidden=512, heads=4, kv_heads=2, mlp=1024, vocab=1000, v_block_kv=2,
                        quantized=False, seed=3, device=cuda, max_positions=512, kv4_layers=(1,))
    g = torch.Generator(device=cuda).manual_seed(1)
    seq = torch.randint(0, 1000, (2, 81), generator=g, device=cuda)
    cache = StarKVCache(90)
    forward_tokens(model, seq[:, :-1], 0, cache)
    got = forward_tokens(model, seq[:, -1:], 80, cache)
    want = forward_tokens(model, seq, 0, StarKVCache(90))
    assert rel(got.float(), want.double()) <= 0.2


@pytest.mark.parametrize("kv4_layers", [(0,), (0, 1), ()])
def test_graphed_loop_with_a_cache_that_the_prompt_fills(cuda, kv4_layers):
    """One new token needs no slot: the loop from graphs gives the eager loop's, as it does where the
    last step fills the cache."""
    model = build_model(num_layers=2, hidden=512, heads=4, kv_heads=2, mlp=1024, vocab=1000, v_block_kv=2,
                        quantized=False, seed=3, device=cuda, max_positions=512, kv4_layers=kv4_layers)
    g = torch.Generator(device=cuda).manual_seed(1)
    prompt = torch.randint(0, 1000, (2, 64), generator=g, device=cuda)
    for new, capacity in ((1, 64), (1, 65), (65, 128)):
        a, b = {}, {}
        want, _ = generate(model, prompt, new, capacity, a)
        got, per = generate_graphed(model, prompt, new, capacity, b)
        assert torch.equal(want, got) and got.shape == (2, new) and per >= 0 and b["prompt_s"] > 0
