"""Llama attention with whole key / value heads in the paged 4-bit cache.

``KV4Attention`` stands beside the latent modules (``starkv.attention``) in one model
and one ``StarKVCache``: layers whose learned ranks stay near the head dimension keep
their dense ``k_proj`` / ``v_proj`` and hold their heads in 4 bits here, the others
hold latents.  The latent modules' constructor arguments (its own by keyword) and
attributes, and either's forward arguments by keyword, so the decoder layer's code does
not change.

* prompt: keys (rotated) and values are written into pages; the attention runs over
  the exact heads with the prompt kernel (``starkv.prefill``);
* a longer piece that continues a prompt: the history is read back from the
  pages, attention by torch SDPA over both;
* decode, and up to ``MAX_DRAFT`` tokens at once: write, then attention over the
  pages; with ``keep_pages`` set, over the pages that ``KV4Cache.select`` keeps.

The kernel takes one mask row a sequence and is causal by itself.  A mask with a row for
each of several tokens goes to it in one call where the rows differ by causality only,
and a token at a time where they do not (a draft's tree).
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import prefill
from .attention import LlamaCustomAttention, StarKVCache, additive_mask, apply_rotary_pos_emb_custom
from .kv4 import KV4Cache

MAX_DRAFT = 16


def causal_rows(mask: torch.Tensor, n: int) -> bool:
    """Whether the rows of mask (B, 1, T, >= n) are its last one with the positions behind
    each token dropped (-inf, or the lowest number of the mask's type).  Synchronises."""
    T = mask.shape[2]
    rows = additive_mask(mask[:, 0, :, :n])
    seen = torch.ones(T, n, dtype=torch.bool, device=mask.device).tril(n - T)
    low = torch.finfo(mask.dtype).min if mask.is_floating_point() else float("-inf")
    return bool(torch.where(seen, rows == rows[:, -1:], rows <= low).all())


class KV4State:
    """One layer's pages of a fixed batch: sequence b owns ``pages_per_sequence``
    consecutive pages of the pool.  ``lengths`` (int32, on the GPU) is what the kernels
    read, ``length`` the same number on the host."""

    def __init__(self, batch: int, capacity: int, num_kv_heads: int, page_size: int, device, page_bounds: bool):
        self.width = -(-capacity // page_size)
        self.cache = KV4Cache(batch * self.width, num_kv_heads, page_size, device, page_bounds)
        self.block_table = torch.arange(batch * self.width, dtype=torch.int32, device=device).view(batch, self.width)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.length = 0

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Write k / v (B, T, Hkv, 128) behind the tokens held."""
        if self.length + k.shape[1] > self.width * self.cache.page_size:
            raise ValueError(f"the cache holds {self.width * self.cache.page_size} tokens")
        self.cache.write(k, v, self.block_table, self.lengths)
        self.lengths.add_(k.shape[1])
        self.length += k.shape[1]

    def crop(self, length: int) -> None:
        """Forgets the tokens from ``length`` on; their slots are written anew."""
        self.lengths.fill_(length)
        self.length = length

    def select(self, q: torch.Tensor, keep_pages: int, mask: Optional[torch.Tensor] = None,
               newest: Optional[int] = None) -> torch.Tensor:
        """The pages (``KV4Cache.select``) of queries q (B, T, Hq, 128) among the ``newest``
        tokens (T of them when None).  The first page and those that may hold the newest
        tokens, whose own positions they are, always count; more than ``keep_pages`` where
        those alone are more.

        With an additive mask (B, L) a sequence begins at the first position that it does not
        drop (-inf, or at most fp16's lowest number): pages of left padding are neither the
        first page nor scored."""
        newest = newest or q.shape[1]
        page = self.cache.page_size
        last = 1 + -(-(newest - 1) // page)
        keep = max(keep_pages, 1 + last)
        if mask is None:
            return self.cache.select(q, self.block_table, self.lengths, keep, 1, last)
        live = mask > torch.finfo(torch.float16).min
        lead = torch.where(live.any(1), live.int().argmax(1), mask.shape[1])
        skip = torch.minimum(lead, self.lengths - 1).clamp_(min=0) // page
        at = (skip[:, None] + torch.arange(self.width, device=skip.device)).clamp_(max=self.width - 1)
        skip = skip.int()
        pages = self.cache.select(q, self.block_table.gather(1, at), self.lengths - skip * page, keep, 1, last)
        return torch.where(pages >= 0, pages + skip[:, None, None], pages)

    def attend(self, q: torch.Tensor, scaling: float, mask: Optional[torch.Tensor] = None,
               keep_pages: int = 0) -> torch.Tensor:
        """The newest tokens' queries (B, T, Hq, 128) over the pages, or over the best
        ``keep_pages`` of them."""
        pages = self.select(q, keep_pages, mask) if keep_pages else None
        return self.cache.attend(q, self.block_table, self.lengths, scaling, mask=mask, pages=pages)

    def attend_rows(self, q: torch.Tensor, scaling: float, rows: torch.Tensor, keep_pages: int = 0) -> torch.Tensor:
        """``attend`` with a mask row for each token, rows (B, T, length): a call a token, in
        which its row says what it attends to, the newer tokens too."""
        out = []
        for i in range(q.shape[1]):
            qi = q[:, i:i + 1]
            pages = self.select(qi, keep_pages, rows[:, i], newest=q.shape[1]) if keep_pages else None
            out.append(self.cache.attend(qi, self.block_table, self.lengths, scaling, mask=rows[:, i], pages=pages))
        return torch.cat(out, 1)

    def history(self, dtype: torch.dtype):
        """All tokens held as (k, v), each (B, length, Hkv, 128)."""
        return self.cache.read(self.block_table, torch.zeros_like(self.lengths), self.length, dtype=dtype)


class KV4Attention(nn.Module):
    """``keep_pages``: pages a decode step attends to (0: all of them; from 2 on, the first and
    the newest token's are always among them)."""

    def __init__(self, config, layer_idx: Optional[int] = None, decomp_goup_num: Optional[int] = 1, *,
                 page_size: int = 64, keep_pages: int = 0):
        super().__init__()
        self.config = config
        self.layer_idx = layer_idx
        self.attention_dropout = getattr(config, "attention_dropout", 0.0)
        self.hidden_size = config.hidden_size
        self.num_heads = config.num_attention_heads
        self.num_key_value_heads = config.num_key_value_heads
        self.num_key_value_groups = self.num_heads // self.num_key_value_heads
        self.head_dim = config.hidden_size // config.num_attention_heads
        self.is_causal = True
        self.decomp_goup_num = decomp_goup_num           # nothing is factored here
        if self.head_dim != 128:
            raise ValueError("the 4-bit cache takes heads of dimension 128")
        if keep_pages < 0 or keep_pages == 1:
            raise ValueError("keep_pages must be 0, or 2 and more (the first page and the newest token's)")
        self.scaling = self.head_dim ** -0.5
        self.page_size, self.keep_pages = page_size, keep_pages
        bias = config.attention_bias
        self.q_proj = nn.Linear(config.hidden_size, self.num_heads * 128, bias=bias)
        self.k_proj = nn.Linear(config.hidden_size, self.num_key_value_heads * 128, bias=bias)
        self.v_proj = nn.Linear(config.hidden_size, self.num_key_value_heads * 128, bias=bias)
        self.o_proj = nn.Linear(self.num_heads * 128, config.hidden_size, bias=bias)

    def state(self, cache: StarKVCache, batch: int, device) -> KV4State:
        st = cache.kv4_states.get(self.layer_idx)
        if st is None:
            # with bounds (2.5 % of the pool) whatever keep_pages is: it may be set later
            st = KV4State(batch, cache.capacity, self.num_key_value_heads, self.page_size, device, True)
            cache.kv4_states[self.layer_idx] = st
        return st

    def heads(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
        """Rotated queries and keys and the values of x (B, T, hidden), each (B, T, heads, 128)."""
        B, T, _ = x.shape
        q = self.q_proj(x).view(B, T, self.num_heads, 128).transpose(1, 2)
        k = self.k_proj(x).view(B, T, self.num_key_value_heads, 128).transpose(1, 2)
        q = apply_rotary_pos_emb_custom(q, cos, sin)
        k = apply_rotary_pos_emb_custom(k, cos, sin)
        return q.transpose(1, 2), k.transpose(1, 2), self.v_proj(x).view(B, T, self.num_key_value_heads, 128)

    def forward(self, hidden_states, position_embeddings, attention_mask, position_ids=None, past_key_values=None,
                cache_position=None, past_key_values_upper=None, **kwargs):
        cache = past_key_values if past_key_values is not None else past_key_values_upper
        if not isinstance(cache, StarKVCache):
            raise TypeError("KV4Attention takes a StarKVCache as past_key_values")
        B, T, _ = hidden_states.shape
        q, k, v = self.heads(hidden_states, *position_embeddings)
        st = self.state(cache, B, hidden_states.device)
        before = st.length
        if T > MAX_DRAFT and before:
            old_k, old_v = st.history(k.dtype)
            keys, values = torch.cat([old_k, k], 1), torch.cat([old_v, v], 1)
        else:
            keys, values = k, v
        st.append(k, v)
        if T <= MAX_DRAFT and (before or T == 1):
            by_row = attention_mask is not None and attention_mask.dim() == 4 and attention_mask.shape[2] == T > 1
            # a graph cannot ask what the mask holds
            if by_row and (torch.cuda.is_current_stream_capturing() or not causal_rows(attention_mask, st.length)):
                rows = additive_mask(attention_mask[:, 0, :, :st.length]).expand(B, T, st.length)
                out = st.attend_rows(q, self.scaling, rows, self.keep_pages)
            else:
                mask = LlamaCustomAttention._decode_mask(attention_mask, B, st.length)
                out = st.attend(q, self.scaling, mask, self.keep_pages)
        elif attention_mask is None and not before:
            out = prefill.prompt_attention(q.transpose(1, 2), keys.transpose(1, 2), values.transpose(1, 2), self.scaling)
            out = out.transpose(1, 2)
        else:
            grp = self.num_key_value_groups
            n = keys.shape[1]
            if attention_mask is None:
                mask = torch.ones(T, n, dtype=torch.bool, device=q.device).tril(n - T)
            else:
                mask = attention_mask[:, :, :, :n]
            out = F.scaled_dot_product_attention(q.transpose(1, 2), keys.transpose(1, 2).repeat_interleave(grp, 1),
                                                 values.transpose(1, 2).repeat_interleave(grp, 1), attn_mask=mask,
                                                 scale=self.scaling).transpose(1, 2)
        return self.o_proj(out.reshape(B, T, self.num_heads * 128)), None
