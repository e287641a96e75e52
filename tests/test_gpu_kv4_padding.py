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
