"""Cases of the paged 4-bit key / value cache: writing tokens into it, reading
them back, attention over it, and attention over the pages that a bound on the
scores selects.

The quantiser (all steps IEEE fp32, round half to even): per token, KV head and
group of 32 channels, x clamped to +-65504,
    s = fp16((max - min) / 15),  m = fp16(min + 8 s),  inv = s > 0 ? 1 / s : 0,
    c = clamp(rint((x - m) * inv), -8, 7),   value = s * c + m.
A page that is full carries, per KV head and channel, int8 bounds of its keys:
    t = max|value| / 127,  up = min(ceil(max / t), 127),  lo = max(floor(min / t), -127).
A page's score for query columns q_j (int8 codes a_j with scale u_j = max|q_j| / 127):
    max_j (u_j * sum_d (a_j,d > 0 ? a_j,d * up_d : a_j,d * lo_d)) * t.
"""

import math
import os
import sys

import torch

own = False

D, GROUP = 128, 32
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the newest token of one conversation, a 32-head layer; it fills the last slot of its page
        dict(name="append_one", op="write", batch=1, tokens=1, context=4095, kv_heads=32, page=64, dtype="fp16", ragged=False),
        # a serving batch's newest tokens, every sequence at a place of its own
        dict(name="append_batch64", op="write", batch=64, tokens=1, context=8191, kv_heads=8, page=64, dtype="bf16", ragged=True),
        # prompts of different lengths entering the cache together (Llama-3.1-8B key / value heads)
        dict(name="prompt_4x32k", op="write", batch=4, tokens=32768, context=0, kv_heads=8, page=64, dtype="bf16", ragged=True),
        # an earlier turn of an odd length brought back for a prompt that continues it
        dict(name="read_turn_1001", op="read", batch=1, tokens=1001, context=39, kv_heads=8, page=64, dtype="bf16", ragged=False),
        # long shared documents brought back whole
        dict(name="read_4x32k", op="read", batch=4, tokens=32768, context=0, kv_heads=32, page=64, dtype="fp16", ragged=False),
        # two short conversations, one token each: latency counts
        dict(name="attend_777", op="attend", batch=2, queries=1, context=777, kv_heads=8, group=1, page=64, dtype="fp16", ragged=False, masked=False),
        # one long conversation, Llama-3.1-8B heads: few rows, the context is split
        dict(name="attend_1x32k", op="attend", batch=1, queries=1, context=32769, kv_heads=8, group=4, page=64, dtype="bf16", ragged=False, masked=False),
        # a serving batch of mixed lengths in small pages
        dict(name="attend_64x8k_mixed", op="attend", batch=64, queries=1, context=8192, kv_heads=8, group=4, page=16, dtype="bf16", ragged=True, masked=False),
        # four drafted tokens a sequence checked at once, left-padded prompts masked out
        dict(name="attend_draft4", op="attend", batch=8, queries=4, context=16384, kv_heads=8, group=4, page=64, dtype="fp16", ragged=True, masked=True),
        # batch 16 at 32K, 32 heads, no sharing of KV heads: the largest
        dict(name="attend_16x32k", op="attend", batch=16, queries=1, context=32768, kv_heads=32, group=1, page=64, dtype="fp16", ragged=False, masked=False),
        # one conversation of 16K that attends to 32 of its 256 pages
        dict(name="sparse_1x16k", op="sparse", batch=1, queries=1, context=16384, kv_heads=32, group=1, page=64, dtype="fp16", ragged=False, select=32),
        # batch 4 at 131072, 64 pages of 2048 a KV head
        dict(name="sparse_4x128k", op="sparse", batch=4, queries=1, context=131072, kv_heads=8, group=4, page=64, dtype="bf16", ragged=False, select=64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "sparse"])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 16, 32])
    c = dict(op=op, kv_heads=kv_heads, page=rng.choice([16, 32, 64, 64, 128]), dtype=rng.choice(["fp16", "bf16"]), ragged=rng.random() < 0.6)
    if op in ("write", "read"):
        c["batch"] = _log_int(rng, 1, 64)
        most = (1 << (20 if op == "write" else 22)) // (kv_heads * c["batch"])
        c["tokens"] = _log_int(rng, 1, max(1, min(32768, most)))
        c["context"] = rng.choice([0, _log_int(rng, 1, 4096)])
        return c
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    if op == "attend":
        c["batch"] = _log_int(rng, 1, 64)
        c["context"] = _log_int(rng, 16, max(16, min(131072, (1 << 24) // (kv_heads * c["batch"]))))
        c["queries"] = rng.choice([1, 1, 1, 2, 3, 4, 6])
        c["masked"] = rng.random() < 0.3
    else:
        c["batch"] = _log_int(rng, 1, 16)
        c["context"] = _log_int(rng, 1024, max(1024, min(131072, (1 << 22) // (kv_heads * c["batch"]))))
        c["queries"] = rng.choice([1, 1, 2])
        c["select"] = _log_int(rng, 4, 64)
    c["group"] = group
    return c


# ------------------------------------------------- lengths, from the case alone
def _counts(c):
    """New (write) or wanted (read) tokens of each sequence."""
    n, B = c["tokens"], c["batch"]
    return [max(0, n - (b * n) // (2 * B)) if c["ragged"] else n for b in range(B)]


def _starts(c):
    """The first position that is written or read."""
    n, B = c["context"], c["batch"]
    return [(n * (b + 1)) // B if c["ragged"] else n for b in range(B)]


def _lengths(c):
    """Tokens a sequence holds when it is attended to; ragged batches hold an empty one too."""
    n, B = c["context"], c["batch"]
    if not c["ragged"]:
        return [n] * B
    return [0 if B > 2 and b == 1 else max(1, (n * (b + 1)) // B - (b % 3)) for b in range(B)]


def _table_width(c):
    most = c["context"] + c["tokens"] if c["op"] in ("write", "read") else c["context"]
    return max(1, -(-most // c["page"]))


def work(case):
    Hkv, per = case["kv_heads"], 80  # bytes of one token's key (or value) of one head: 64 of codes, 16 of (s, m)
    if case["op"] in ("write", "read"):
        n = sum(_counts(case)) * Hkv
        # write: read K and V, write them packed; then, as read does, read them packed and write them whole
        per_token = 2 * 2 * D + 2 * per if case["op"] == "read" else 2 * (2 * 2 * D + 2 * per)
        return {"bytes": n * per_token, "flops": n * 2 * D * (2 if case["op"] == "read" else 10)}
    G, Q, ps = case["group"], case["queries"], case["page"]
    qbytes = case["batch"] * Q * Hkv * G * D * 2 * 2
    total_b, total_f = qbytes, 0
    for n in _lengths(case):
        if case["op"] == "sparse":
            pages = -(-n // ps)
            kept = min(n, case["select"] * ps)
            if pages > case["select"]:
                total_b += Hkv * (n // ps) * (2 * D + 4)
                total_f += Hkv * (n // ps) * G * Q * 2 * D
        else:
            kept = n
            total_b += 4 * n if case["masked"] else 0
        total_b += Hkv * kept * 2 * per
        total_f += Hkv * kept * G * Q * 4 * D
    return {"bytes": total_b, "flops": total_f}


# ------------------------------------------------------------------ the inputs
def _gen(seed, n):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + n) % (1 << 62))


def _values(c, seed, n, shape):
    """N(0, 1) with 1 % of the channels eight times as large, in the case's type."""
    g = _gen(seed, n)
    wide = 1.0 + 7.0 * (torch.rand(shape[-2:], generator=g, device="cuda") < 0.01)
    x = torch.empty(shape, dtype=DTYPES[c["dtype"]], device="cuda").normal_(generator=g)
    return x.mul_(wide.to(x.dtype))


def _inputs(c, seed):
    """What both forms and the 64-bit definition start from."""
    B, H, ps, W = c["batch"], c["kv_heads"], c["page"], _table_width(c)
    x = {"table": torch.randperm(B * W, generator=_gen(seed, 1), device="cuda").to(torch.int32).view(B, W)}
    if c["op"] in ("write", "read"):
        n, x["first"], x["count"] = c["tokens"], _starts(c), _counts(c)
    else:
        n, x["first"], x["count"] = c["context"], [0] * B, _lengths(c)
        x["q"] = _values(c, seed, 4, (B, c["queries"], H * c["group"], D))
        if c.get("masked"):
            L = W * ps
            pad = torch.rand(B, generator=_gen(seed, 5), device="cuda") * 0.3 * torch.tensor(x["count"], device="cuda")
            mask = torch.where(torch.arange(L, device="cuda") < pad[:, None], float("-inf"), 0.0)
            if B > 1:
                mask[0] = float("-inf")  # a sequence that is all padding
            x["mask"] = mask.contiguous()
    x["k"], x["v"] = _values(c, seed, 2, (B, n, H, D)), _values(c, seed, 3, (B, n, H, D))
    for name in ("first", "count"):
        x[name] = torch.tensor(x[name], dtype=torch.int32, device="cuda")
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    B, H, ps, W = case["batch"], case["kv_heads"], case["page"], _table_width(case)
    if own:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        path = os.path.join(root, "star-kv_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from starkv.kv4 import KV4Cache
        cache = KV4Cache(B * W, H, page_size=ps, device="cuda")
    else:
        cache = _Plain(B * W, H, ps)
    state = dict(case=case, cache=cache, table=x["table"], first=x["first"], count=x["count"], scaling=D ** -0.5)
    if case["op"] == "write":
        state["k"], state["v"] = x["k"], x["v"]
    else:
        if own:
            cache.write(x["k"], x["v"], x["table"], x["first"], x["count"])
        else:
            cache.write(x["k"], x["v"], x["table"], x["first"], x["count"], bounds=case["op"] == "sparse")
        for name in ("q", "mask"):
            state[name] = x.get(name)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    c, cache, table = state["case"], state["cache"], state["table"]
    dtype, first, count = DTYPES[c["dtype"]], state["first"], state["count"]
    if c["op"] == "write":
        cache.write(state["k"], state["v"], table, first, count)
        k, v = cache.read(table, first, c["tokens"], count, dtype=dtype)
        return {"k": k, "v": v}
    if c["op"] == "read":
        k, v = cache.read(table, first, c["tokens"], count, dtype=dtype)
        return {"k": k, "v": v}
    if c["op"] == "attend":
        out, lse = cache.attend(state["q"], table, count, state["scaling"], mask=state["mask"], return_lse=True)
        return {"out": out, "lse": lse}
    pages = cache.select(state["q"], table, count, c["select"])
    out, lse = cache.attend(state["q"], table, count, state["scaling"], pages=pages, return_lse=True)
    return {"pages": pages, "out": out, "lse": lse}


def _number(value, dtype=torch.float32):
    """A divisor on the GPU: torch multiplies by the reciprocal of a Python number instead of dividing by it."""
    return torch.full((), value, dtype=dtype, device="cuda")


class _Plain:
    """The operators in elementary torch operations, fp32 inside."""

    def __init__(self, num_pages, heads, page):
        self.page, self.heads = page, heads
        z = lambda *s, dtype: torch.zeros(num_pages, heads, *s, dtype=dtype, device="cuda")  # noqa: E731
        self.codes = [z(page, D // 2, dtype=torch.uint8) for _ in range(2)]
        self.params = [z(page, D // GROUP, 2, dtype=torch.float16) for _ in range(2)]
        self.up, self.lo = z(D, dtype=torch.int8), z(D, dtype=torch.int8)
        self.unit = z(dtype=torch.float32)

    def _quantise(self, x):
        x = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (D // GROUP, GROUP))
        low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        s = ((high - low) / _number(15.0)).half().float()
        m = (low + 8.0 * s).half().float()
        inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
        c = ((x - m) * inv).round().clamp(-8, 7).add(8).to(torch.uint8).flatten(-2)
        return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([s, m], -1).half()

    def _values(self, codes, params):
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().sub_(8.0).unflatten(-1, (D // GROUP, GROUP))
        p = params.float()
        return c.mul_(p[..., :1]).add_(p[..., 1:]).flatten(-2)

    def _where(self, table, first, count, n):
        """(live, page, slot) of the n positions from `first` on, each (B, n)."""
        i = torch.arange(n, device="cuda")
        pos = (first[:, None] + i).long()
        live = i < count[:, None]
        at = (pos // self.page).clamp(max=table.shape[1] - 1)
        return live, table.long().gather(1, at), pos % self.page

    def write(self, k, v, table, first, count, bounds=True):
        n = k.shape[1]
        live, page, slot = self._where(table, first, count, n)
        page, slot = page[live], slot[live]
        for x, codes, params in zip((k, v), self.codes, self.params):
            c, p = self._quantise(x)
            codes[page, :, slot], params[page, :, slot] = c[live], p[live]
        if not bounds:
            return
        at = torch.arange(table.shape[1], device="cuda")
        done = ((at + 1) * self.page <= (first + count)[:, None]) & ((at + 1) * self.page > first[:, None])
        full = table[done].long()
        x = self._values(self.codes[0][full], self.params[0][full])
        high, low = x.amax(-2), x.amin(-2)
        t = torch.maximum(high.abs(), low.abs()).amax(-1, keepdim=True) / _number(127.0)
        u = torch.where(t > 0, t, torch.ones_like(t))
        self.up[full] = (high / u).ceil().clamp(max=127).to(torch.int8)
        self.lo[full] = (low / u).floor().clamp(min=-127).to(torch.int8)
        self.unit[full] = t[..., 0]

    def read(self, table, first, n, count, dtype):
        live, page, slot = self._where(table, first, count, n)
        out = []
        for codes, params in zip(self.codes, self.params):
            x = self._values(codes[page, :, slot], params[page, :, slot])
            out.append(x.where(live[..., None, None], torch.zeros_like(x)).to(dtype))
        return out

    def select(self, q, table, lengths, most, first=1, last=1):
        B, W, H = table.shape[0], table.shape[1], self.heads
        x = q.float().view(B, q.shape[1], H, -1, D).transpose(1, 2).flatten(2, 3)
        u = x.abs().amax(-1, keepdim=True) / _number(127.0)
        a = torch.where(u > 0, x / torch.where(u > 0, u, torch.ones_like(u)), torch.zeros_like(x)).round()
        up, lo = self.up[table.long()].transpose(1, 2).float(), self.lo[table.long()].transpose(1, 2).float()
        # whole numbers below 2^24: the sums are exact in fp32
        dots = a.clamp(min=0) @ up.transpose(-1, -2) + a.clamp(max=0) @ lo.transpose(-1, -2)
        score = (dots * u).amax(2) * self.unit[table.long()].transpose(1, 2)
        at = torch.arange(W, device="cuda")
        n = ((lengths + self.page - 1) // self.page)[:, None, None]
        score = torch.where((at < first) | (at >= n - last), torch.full_like(score, float("inf")), score)
        score = torch.where(at < n, score, torch.full_like(score, float("-inf"))) + 0.0
        best = score.sort(dim=-1, descending=True, stable=True).indices[..., :most]
        if best.shape[-1] < most:
            best = torch.cat([best, best.new_full((B, H, most - best.shape[-1]), W)], -1)
        best = torch.where(best < n, best, torch.full_like(best, 1 << 30)).sort(-1).values
        return torch.where(best < (1 << 30), best, torch.full_like(best, -1)).to(torch.int32)

    def attend(self, q, table, lengths, scaling, mask=None, pages=None, return_lse=True):
        B, Q, H, ps = q.shape[0], q.shape[1], self.heads, self.page
        x = q.float().view(B, Q, H, -1, D).permute(0, 2, 1, 3, 4)
        G = x.shape[3]
        heads = torch.arange(H, device="cuda")[:, None]
        if pages is None:
            listed = torch.arange(table.shape[1], device="cuda").expand(B, H, -1)
        else:
            listed = pages.long()
        phys = table.long()[:, None].expand(B, H, -1).gather(2, listed.clamp(min=0))
        k, v = (self._values(c[phys, heads], p[phys, heads]).flatten(2, 3) for c, p in zip(self.codes, self.params))
        pos = (listed[..., None] * ps + torch.arange(ps, device="cuda")).masked_fill((listed < 0)[..., None], 1 << 30).flatten(2)
        end = (lengths[:, None] - Q + 1 + torch.arange(Q, device="cuda"))[:, None, :, None, None]
        s = (x.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (Q, G)) * scaling
        s = s.masked_fill(pos[:, :, None, None, :] >= end, float("-inf"))
        if mask is not None:
            s = s + mask[:, None, None, None, :s.shape[-1]]
        top = s.amax(-1, keepdim=True)
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        w = e / torch.where(total > 0, total, torch.ones_like(total))
        out = (w.flatten(2, 3) @ v).unflatten(2, (Q, G)).permute(0, 2, 1, 3, 4).reshape(q.shape).to(q.dtype)
        lse = (top + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(B, Q, H * G)
        return out, lse


# ------------------------------------------------------- the definition in 64 bits
def _exact_codes(x):
    """(c, s, m) in 64 bits. The quantiser's steps are defined in fp32: each is taken in 64 bits and
    rounded to fp32, which gives the same (sums, products and quotients of fp32 numbers)."""
    r = lambda t: t.float().double()  # noqa: E731
    x = torch.clamp(x.double(), -65504.0, 65504.0).reshape(*x.shape[:-1], D // GROUP, GROUP)
    low, high = x.min(-1, keepdim=True)[0], x.max(-1, keepdim=True)[0]
    s = r(r(high - low) / _number(15.0, torch.float64)).float().half().double()
    m = r(low + 8.0 * s).float().half().double()
    inv = r(torch.where(s > 0, 1.0 / s.clamp(min=2.0 ** -30), 0.0 * s))
    return torch.clamp(torch.round(r(r(x - m) * inv)), -8, 7), s, m


def _exact_values(x):
    c, s, m = _exact_codes(x)
    return (s * c + m).reshape(x.shape)


def exact(case, seed):
    x = _inputs(case, seed)
    B, H, ps = case["batch"], case["kv_heads"], case["page"]
    first, count = x["first"].tolist(), x["count"].tolist()
    if case["op"] in ("write", "read"):
        if x["k"].numel() > 1 << 29:
            return None
        found = {}
        for name in ("k", "v"):
            t = _exact_values(x[name])
            for b in range(B):
                t[b, count[b]:] = 0
            found[name] = t
        return found
    Q, G = case["queries"], case["group"]
    out = torch.zeros(B, Q, H * G, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Q, H * G), -math.inf, dtype=torch.float64, device="cuda")
    sparse = case["op"] == "sparse"
    chosen = torch.full((B, H, case["select"]), -1, dtype=torch.int32, device="cuda") if sparse else None
    for b in range(B):
        n = count[b]
        for h0 in range(0, H, 4):
            hs = range(h0, min(H, h0 + 4))
            if not n:
                continue
            k, v = (_exact_values(x[t][b, :n, h0:hs.stop].transpose(0, 1)) for t in ("k", "v"))
            for i, h in enumerate(hs):
                q = x["q"][b, :, h * G:(h + 1) * G].double()
                keep = torch.ones(n, dtype=torch.bool, device="cuda")
                if sparse:
                    kept = _exact_select(k[i], q.reshape(-1, D), ps, case["select"])
                    chosen[b, h, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
                    keep = torch.isin(torch.arange(n, device="cuda") // ps, torch.tensor(kept, device="cuda"))
                s = torch.einsum("qgd,nd->qgn", q, k[i]) / math.sqrt(D)
                for j in range(Q):
                    ok = keep & (torch.arange(n, device="cuda") < n - Q + 1 + j)
                    add = x["mask"][b, :n].double() if "mask" in x else torch.zeros(n, dtype=torch.float64, device="cuda")
                    ok = ok & (add > -math.inf)
                    if not bool(ok.any()):
                        continue
                    z = s[j][:, ok] + add[ok]
                    lse[b, j, h * G:(h + 1) * G] = torch.logsumexp(z, -1)
                    out[b, j, h * G:(h + 1) * G] = torch.softmax(z, -1) @ v[i][ok]
    found = {"out": out, "lse": lse}
    if sparse:
        found["pages"] = None
    return found


def _exact_select(k, q, ps, most):
    """Ordinals of the pages kept for one KV head: k (n, D) and q (columns, D) in 64 bits."""
    r = lambda t: t.float().double()  # noqa: E731
    n = k.shape[0]
    pages, full = -(-n // ps), n // ps
    if pages <= most:
        return list(range(pages))
    x = r(k[:full * ps]).reshape(full, ps, D)
    high, low = x.max(1)[0], x.min(1)[0]
    t = r(torch.maximum(high.abs(), low.abs()).max(-1)[0] / _number(127.0, torch.float64))
    safe = torch.where(t > 0, t, t + 1)[:, None]
    up, lo = torch.clamp(torch.ceil(r(high / safe)), max=127), torch.clamp(torch.floor(r(low / safe)), min=-127)
    u = r(q.abs().max(-1)[0] / _number(127.0, torch.float64))
    a = torch.round(r(q / torch.where(u > 0, u, u + 1)[:, None]))
    dots = (torch.where(a > 0, a, 0 * a)[:, None] * up + torch.where(a < 0, a, 0 * a)[:, None] * lo).sum(-1)
    score = r(r(dots * u[:, None]).max(0)[0] * t).tolist() + [0.0] * (pages - full)
    order = sorted(range(1, pages - 1), key=lambda p: (-score[p], p))
    return sorted([0, pages - 1] + order[:most - 2])
