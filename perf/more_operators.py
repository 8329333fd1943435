"""Performance cases of a decoding step's further operators: the 8-bit cache, a mixture-of-experts layer for a few tokens, sampling.

* ``append``    ``ops.paged.paged_append`` on float8_e4m3fn pages: rotation, QK norm, value embedding, and K / V into 8 bits with a
  power of two for each 16 tokens and KV head, which grows when a token does not fit (earlier tokens are then written again)
* ``attention`` ``ops.paged.paged_attention`` on such pages (GQA, left window)
* ``moe``       ``ops.moe.moe_tokens``: router, top-k, ReLU^2 experts and shared expert of a few tokens
* ``sample``    ``ops.sampling.sample_logits``: temperature, top-k, top-p and min-p, a token for each row from a given number

``own`` selects the framework's operators; otherwise ``run`` evaluates their plain form with elementary torch operations, in 32 bits,
and in 64 where a comparison hangs on them (the experts' choice, the sampled token).
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 2.0 ** -23  # of the QK norm
BLOCK = 16        # tokens that share a scale


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one user, one token, the benchmark model's heads (10 query, 5 KV heads of 128): latency
        dict(name="append one token", op="append", dtype="bf16", B=1, t=1, heads=10, kv_heads=5, dim=128, page=64,
             length=778, ragged=False, norm=True, ve=True),
        # a decode step of a busy server: one token for each of 192 rows of unequal length
        dict(name="append 192 rows", op="append", dtype="fp16", B=192, t=1, heads=12, kv_heads=12, dim=128, page=16,
             length=3001, ragged=True, norm=True, ve=False),
        # prompts of up to 2048 tokens enter the cache, value embeddings on
        dict(name="append 8 prompts of 2048", op="append", dtype="bf16", B=8, t=2048, heads=10, kv_heads=5, dim=128,
             page=64, length=2048, ragged=True, norm=True, ve=True),
        # one user at about a thousand tokens
        dict(name="attention 1 x 1001", op="attention", dtype="bf16", B=1, t=1, heads=10, kv_heads=5, dim=128, page=64,
             length=1001, ragged=False, window=-1),
        # a server's batch with unequal lengths and one KV head for 16 query heads
        dict(name="attention 64 ragged 8192", op="attention", dtype="bf16", B=64, t=1, heads=16, kv_heads=1, dim=128,
             page=64, length=8192, ragged=True, window=-1),
        # four drafted tokens are verified at once in a sliding-window layer, heads of 64
        dict(name="attention 24 x 4 window", op="attention", dtype="fp16", B=24, t=4, heads=12, kv_heads=12, dim=64,
             page=16, length=6007, ragged=True, window=1023),
        # long contexts, the benchmark model's heads: bandwidth
        dict(name="attention 16 x 32768", op="attention", dtype="bf16", B=16, t=1, heads=10, kv_heads=5, dim=128,
             page=64, length=32768, ragged=False, window=-1),
        # one user, one token, the benchmark's MoE layer (64 experts of 1024, top 8, one shared)
        dict(name="moe one token", op="moe", dtype="bf16", T=1, width=2048, hidden=1024, experts=64, top_k=8, shared=1),
        # a dozen users on the same layer
        dict(name="moe 12 tokens", op="moe", dtype="bf16", T=12, width=2048, hidden=1024, experts=64, top_k=8, shared=1),
        # the scaling recipe's layer (256 experts of width / 4): nearly every expert is wanted by a few of 64 tokens
        dict(name="moe 64 tokens 256 experts", op="moe", dtype="bf16", T=64, width=1280, hidden=320, experts=256, top_k=8, shared=1),
        # one user, a vocabulary of 32768, top-k and top-p on the head's own bf16 logits
        dict(name="sample 1 x 32768", op="sample", dtype="bf16", B=1, vocab=32768, k=True, p=True, m=False, mask=False),
        # a server's batch on the benchmark's vocabulary, a setting for each row, after penalties and a grammar mask
        dict(name="sample 224 x 65536", op="sample", dtype="fp32", B=224, vocab=65536, k=True, p=True, m=True, mask=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "moe", "moe", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("append", "attention"):
        heads, kv_heads = rng.choice([(10, 5), (12, 12), (16, 1), (16, 4), (6, 6), (8, 2), (12, 3)])
        dim = rng.choice([64, 128, 128])
        page = rng.choice([16, 32, 48, 64, 128])
    if op == "append":
        B = _log(rng, 1, 256)
        t = rng.choice([1, 1, _log(rng, 2, max(2, min(2048, 8 * 2048 * 15 // (B * (heads + 2 * kv_heads)))))])
        before = _log(rng, 1, max(1, min(4096, 2 ** 28 // (B * kv_heads * dim)))) - 1
        return dict(op=op, dtype=dtype, B=B, t=t, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    length=t + before, ragged=rng.random() < 0.6, norm=rng.random() < 0.8, ve=rng.random() < 0.5)
    if op == "attention":
        length = _log(rng, 1, 32768)
        t = min(length, rng.choice([1, 1, 1, 2, 3, 5, 8]))
        most = 16 * 32768 * 5 * 128 // (length * kv_heads * dim)
        return dict(op=op, dtype=dtype, B=_log(rng, 1, max(1, min(256, most))), t=t, heads=heads, kv_heads=kv_heads,
                    dim=dim, page=page, length=length, ragged=rng.random() < 0.6,
                    window=rng.choice([-1, -1, _log(rng, 1, 4096)]))
    if op == "moe":
        width, experts = 8 * _log(rng, 16, 256), rng.choice([4, 8, 32, 48, 64, 128, 256])
        hidden = 8 * _log(rng, 8, max(8, min(512, 64 * 1024 * 2048 // (experts * width) // 8)))
        return dict(op=op, dtype=dtype, T=_log(rng, 1, 64), width=width, hidden=hidden, experts=experts,
                    top_k=rng.choice([k for k in (1, 2, 3, 4, 6, 8) if k <= experts]), shared=rng.choice([0, 1, 1, 2]))
    vocab = _log(rng, 1000, 131072)
    return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), B=_log(rng, 1, max(1, min(256, 224 * 65536 // vocab))),
                vocab=vocab, k=rng.random() < 0.5, p=rng.random() < 0.6, m=rng.random() < 0.4, mask=rng.random() < 0.4)


def _spans(case):
    """Of each row: the tokens in the cache before the call, and the new ones.  A row may bring fewer tokens than t."""
    B, t, length = case["B"], case["t"], case["length"]
    if not case["ragged"]:
        return [(length - t, t)] * B
    rng = random.Random(B * 100003 + length)
    spans = []
    for b in range(B):
        count = t if t <= 16 or b == 0 else _log(rng, t // 4, t)
        total = length if b == 0 else max(count, _log(rng, max(1, length // 16), length))
        spans.append((total - count, count))
    return spans


# ------------------------------------------------------------------------------------------ inputs
def _pages(case, spans, gen):
    """An 8-bit cache whose pages are handed out in random order; what lies behind a row's last token is older data.  Blocks' keys
    reach 3.5 to 28, their values 1.8 to 14."""
    page, Hk, D = case["page"], case["kv_heads"], case["dim"]
    need = [-(-(s + c) // page) for s, c in spans]
    total = sum(need)
    order = torch.randperm(total + 3, generator=gen, device="cuda").to(torch.int32)
    columns = max(need)
    table = torch.full((case["B"], columns), -1, dtype=torch.int32, device="cuda")
    first = torch.tensor([0] + need, device="cuda").cumsum(0)
    at = torch.arange(columns, device="cuda")[None]
    there = at < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(there, order[(first[:-1, None] + at).clamp(max=total - 1)], table)

    def codes():
        x = torch.randn(total + 3, Hk, page, D, generator=gen, device="cuda", dtype=torch.bfloat16) * 80
        return x.clamp(-448, 448).to(torch.float8_e4m3fn)

    def scales(low):
        return torch.exp2(torch.randint(low, low + 4, (total + 3, Hk, page // BLOCK), generator=gen, device="cuda").float())
    return codes(), codes(), scales(-7), scales(-8), table.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(*shape, generator=gen, device="cuda")

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s, dtype = dict(op=case["op"]), DTYPES[case["dtype"]]
    if case["op"] in ("append", "attention"):
        B, t, H, Hk, D = case["B"], case["t"], case["heads"], case["kv_heads"], case["dim"]
        spans = _spans(case)
        s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"] = _pages(case, spans, gen)
        s["start"], s["count"] = ints([a for a, _ in spans]), ints([c for _, c in spans])
        if case["op"] == "attention":
            s["q"] = normal(B, t, H, D, scale=1.2, dtype=dtype)
            s["longest"], s["window"] = max(a + c for a, c in spans), case["window"]
            return s
        # q, k and v as one projection gives them
        packed = normal(B, t, H + 2 * Hk, D, dtype=dtype)
        s["q"], s["k"], s["v"] = packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]
        angle = torch.outer(torch.arange(20480, device="cuda"),
                            100000.0 ** (-torch.arange(0, D, 2, device="cuda") / D))
        s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
        s["norm"] = 1.2 if case["norm"] else None
        s["ve"] = normal(B, t, Hk, D, dtype=dtype) if case["ve"] else None
        s["ve_gate"] = normal(B, t, Hk, dtype=dtype) if case["ve"] else None
        # the blocks that get tokens: their rows, and which of its row's new blocks each is
        s["written"] = torch.tensor([(b, j) for b, (a, c) in enumerate(spans) for j in range((a % BLOCK + c + BLOCK - 1) // BLOCK)],
                                    device="cuda").T
        return s
    if case["op"] == "moe":
        T, d, F, E = case["T"], case["width"], case["hidden"], case["experts"]

        def weights(*shape):
            return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype) * shape[-1] ** -0.5
        s["x"] = normal(T, d, dtype=dtype)
        s["router"] = normal(E, d, scale=d ** -0.5)
        s["bias"] = normal(E, scale=2e-3)  # as load balancing leaves it
        s["w_fc"], s["w_proj"] = weights(E, F, d), weights(E, d, F)
        s["shared_fc"] = weights(case["shared"] * F, d) if case["shared"] else None
        s["shared_proj"] = weights(d, case["shared"] * F) if case["shared"] else None
        s["top_k"] = case["top_k"]
        return s
    B, V = case["B"], case["vocab"]
    padded = -(-V // 64) * 64  # the head's rows are padded to 64
    logits = 15.0 * torch.tanh(normal(B, padded, scale=4.0) / 15.0)
    if case["mask"]:  # a grammar allows about half
        logits = torch.where(uniform(B, padded) < 0.5, logits, -math.inf)
    s["logits"] = logits.to(dtype)[:, :V]
    s["uniform"] = uniform(B)
    rows = torch.arange(B, device="cuda")
    temperature = uniform(B, lo=0.4, hi=1.5)
    s["temperature"] = torch.where(rows % 16 == 5, 0.0, temperature)  # some rows take the largest logit
    k = torch.exp(uniform(B, lo=math.log(2.0), hi=math.log(1200.0))).to(torch.int32)
    s["top_k"] = torch.where(rows % 4 == 3, 0, k).to(torch.int32) if case["k"] else None  # 0: off in this row
    s["top_p"] = torch.where(rows % 8 == 6, 1.0, uniform(B, lo=0.5, hi=0.99)) if case["p"] else None
    s["min_p"] = torch.where(rows % 2 == 0, 0.0, uniform(B, lo=0.01, hi=0.2)) if case["m"] else None
    return s


# ------------------------------------------------------------------------------------------ one pass
_operators = None


def _own():
    """The framework's operators, looked up once as a program's imports are."""
    global _operators
    if _operators is None:
        from nexttransformer_b200.ops.moe import moe_tokens
        from nexttransformer_b200.ops.paged import paged_append, paged_attention
        from nexttransformer_b200.ops.sampling import sample_logits
        _operators = paged_append, paged_attention, moe_tokens, sample_logits
    return _operators


def run(s):
    op = s["op"]
    if not own:
        return _PLAIN[op](s)
    paged_append, paged_attention, moe_tokens, sample_logits = _own()
    if op == "append":
        q = paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["start"], s["count"],
                         cos=s["cos"], sin=s["sin"], qk_scale=s["norm"], ve=s["ve"], ve_gate=s["ve_gate"],
                         k_scale=s["k_scale"], v_scale=s["v_scale"])
        return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]
    if op == "attention":
        return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["start"], s["count"],
                               window=s["window"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if op == "moe":
        return moe_tokens(s["x"], s["router"], s["w_fc"], s["w_proj"], s["top_k"], bias=s["bias"],
                          shared_fc=s["shared_fc"], shared_proj=s["shared_proj"])
    return sample_logits(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                         min_p=s["min_p"])


def _power_of_two(top):
    """The smallest power of two, from 2^-100 on, whose 448-fold reaches `top`."""
    fraction, exponent = torch.frexp(top)              # top = fraction 2^exponent, 0.5 <= fraction < 1
    exponent = exponent - 9 + (fraction > 0.875).int()  # 448 = 0.875 * 2^9
    return torch.ldexp(torch.ones_like(top), torch.where(top > 0, exponent, -100).clamp(-100, 120))


def _quantised(x, pages, scale, s):
    """Writes the new tokens x [B, t, Hk, D] into the pages, block by block."""
    B, t, Hk, D = x.shape
    columns, page = s["table"].shape[1], pages.shape[2]
    start, count = s["start"].long(), s["count"].long()
    blocks = (t + 2 * BLOCK - 2) // BLOCK
    first = start // BLOCK * BLOCK                                       # position of the first block's first slot
    position = first[:, None] + torch.arange(blocks * BLOCK, device=x.device)
    new = position - start[:, None]                                      # the call's token in this slot
    is_new = ((new >= 0) & (new < count[:, None])).view(B, blocks, BLOCK)
    values = x.gather(1, new.clamp(0, t - 1)[:, :, None, None].expand(-1, -1, Hk, D)).view(B, blocks, BLOCK, Hk, D)
    held = is_new[..., None, None]
    need = _power_of_two(torch.where(held, values.abs(), 0.0).amax((2, 4)))   # [B, blocks, Hk]
    at = position[:, ::BLOCK]
    numbers = s["table"].long().gather(1, (at // page).clamp(max=columns - 1))
    row, block = s["written"]
    number, slot = numbers[row, block], (at % page)[row, block]
    old = scale[number, :, slot // BLOCK]                                # [blocks written, Hk]
    continued = (start > at[:, 0])[row] & (block == 0)
    grown = torch.where(continued[:, None], torch.maximum(old, need[row, block]), need[row, block])
    slots = slot[:, None] + torch.arange(BLOCK, device=x.device)
    where = number[:, None], slice(None), slots
    codes = pages[where].float()                                         # [blocks written, BLOCK, Hk, D]
    earlier = (position.view(B, blocks, BLOCK) < start[:, None, None])[row, block][..., None, None]
    codes = torch.where(earlier, codes * (old / grown)[:, None, :, None], codes)
    codes = torch.where(held[row, block], values[row, block] / grown[:, None, :, None], codes)
    pages[where] = codes.to(pages.dtype)
    scale[number, :, slot // BLOCK] = grown


def _plain_append(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    B, t, H, D = q.shape
    new = torch.arange(t, device=q.device)
    position = s["start"].long()[:, None] + new
    clipped = position.clamp(max=s["cos"].shape[0] - 1)
    cos, sin = s["cos"][clipped].float()[:, :, None], s["sin"][clipped].float()[:, :, None]

    def turned(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        y = torch.cat((a * cos + b * sin, b * cos - a * sin), -1)
        if s["norm"] is None:
            return y
        return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * s["norm"]

    if s["ve"] is not None:
        v = v + 3 * torch.sigmoid(s["ve_gate"].float())[..., None] * s["ve"].float()
    _quantised(turned(k), s["k_pages"], s["k_scale"], s)
    _quantised(v, s["v_pages"], s["v_scale"], s)
    q = torch.where((new < s["count"][:, None])[:, :, None, None], turned(q), 0.0)
    return q.to(s["q"].dtype), s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _plain_attention(s):
    B, t, H, D = s["q"].shape
    Hk, page = s["k_pages"].shape[1], s["k_pages"].shape[2]
    key = torch.arange(s["longest"], device=s["q"].device)
    number = s["table"].long()[:, key // page].clamp(min=0)

    def held(pages, scale):  # [B, Hk, keys, D]
        x = pages.view(torch.uint8)[number, :, key % page].view(torch.float8_e4m3fn).float()
        return (x * scale[number, :, key % page // BLOCK][..., None]).transpose(1, 2)
    K, V = held(s["k_pages"], s["k_scale"]), held(s["v_pages"], s["v_scale"])
    q = s["q"].float().reshape(B, t, Hk, H // Hk, D).transpose(1, 2)                           # [B, Hk, t, g, D]
    score = (q.flatten(2, 3) @ K.transpose(-1, -2)).view(B, Hk, t, H // Hk, -1) / math.sqrt(D)
    new = torch.arange(t, device=key.device)
    position = s["start"].long()[:, None] + new
    seen = (key <= position[..., None]) & (new < s["count"][:, None])[..., None]
    if s["window"] >= 0:
        seen = seen & (key >= position[..., None] - s["window"])
    seen = seen[:, None, :, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    return (p.flatten(2, 3) @ V).view(B, Hk, t, H // Hk, D).transpose(1, 2).reshape(B, t, H, D).to(s["q"].dtype)


def _plain_moe(s):
    x, k = s["x"].float(), s["top_k"]
    T, E = x.shape[0], s["router"].shape[0]
    logits = s["x"].double() @ s["router"].double().T      # the choice between experts hangs on small differences
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    choice = torch.sort(p + s["bias"].double(), dim=-1, descending=True, stable=True).indices[:, :k]
    c = p.gather(1, choice)
    c = (c / c.sum(-1, keepdim=True)).float()
    if T * k <= E:  # the chosen experts' weights
        h = (s["w_fc"][choice].float() @ x[:, None, :, None]).clamp(min=0).square()
        y = ((s["w_proj"][choice].float() @ h)[..., 0] * c[..., None]).sum(1)
    else:           # every expert for every token, and a weight of zero where it was not chosen
        h = torch.einsum("td,efd->etf", x, s["w_fc"].float()).clamp(min=0).square()
        h = h * torch.zeros(T, E, device=x.device).scatter_(1, choice, c).T[..., None]
        y = torch.einsum("etf,edf->td", h, s["w_proj"].float())
    if s["shared_fc"] is not None:
        y = y + (x @ s["shared_fc"].float().T).clamp(min=0).square() @ s["shared_proj"].float().T
    return y.to(s["x"].dtype)


def _plain_sample(s):
    x, T = s["logits"].double(), s["temperature"].double()[:, None]
    B, V = x.shape
    less = x - x.amax(-1, keepdim=True)
    w = torch.where(T > 0, torch.exp(less / torch.where(T > 0, T, 1.0)), (less == 0).double())
    w, order = torch.sort(w, dim=-1, descending=True, stable=True)
    rank = torch.arange(V, device=x.device)
    keep = (T > 0) | (rank == 0)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep = keep & ((k <= 0) | (rank < k))
    w = torch.where(keep, w, 0.0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        mass = w.cumsum(-1)
        keep = keep & ((p >= 1) | (mass - w < p * mass[:, -1:]) | (rank == 0))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    mass = w.cumsum(-1)
    token = (mass <= s["uniform"].double()[:, None] * mass[:, -1:]).sum(-1).clamp(max=V - 1)
    chance = w.gather(1, token[:, None])[:, 0] / mass[:, -1]
    return token, torch.log(chance).float()


_PLAIN = dict(append=_plain_append, attention=_plain_attention, moe=_plain_moe, sample=_plain_sample)


# ------------------------------------------------------------------------------------------ work and definition
def work(case):
    if case["op"] == "append":
        spans = _spans(case)
        new, Hk, D = sum(c for _, c in spans), case["kv_heads"], case["dim"]
        blocks = sum((s + c - 1) // BLOCK - s // BLOCK + 1 for s, c in spans if c)
        # q, k, v (and ve) and the angles in, q out in 16 bits; keys and values out in 8; scales in and out
        each = D * (2 * (case["heads"] + 2 * Hk + (Hk if case["ve"] else 0) + 1) + 2 * case["heads"] + 2 * Hk)
        return {"bytes": new * each + blocks * Hk * 16 + 12 * case["B"],
                "flops": new * (case["heads"] + 2 * Hk) * D * 6}
    if case["op"] == "attention":
        keys = pairs = 0
        for start, count in _spans(case):
            first = max(0, start - case["window"]) if case["window"] >= 0 else 0
            keys += start + count - first
            pairs += sum(min(start + i, case["window"] if case["window"] >= 0 else start + i) + 1 for i in range(count))
        rows = sum(c for _, c in _spans(case)) * case["heads"] * case["dim"]
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] + keys * case["kv_heads"] // 2 + 4 * rows +
                4 * (keys // case["page"] + 2 * case["B"]), "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "moe":
        T, d, F, E, k = case["T"], case["width"], case["hidden"], case["experts"], case["top_k"]
        wanted = E * (1 - (1 - k / E) ** T) + case["shared"]  # distinct experts, on average
        return {"bytes": int(wanted * 4 * d * F) + 4 * E * d + 4 * T * d,
                "flops": 4 * T * (k + case["shared"]) * d * F + 2 * T * E * d}
    B, V = case["B"], case["vocab"]
    return {"bytes": B * (V * (4 if case["dtype"] == "fp32" else 2) + 32), "flops": 8 * B * V}


def exact(case, seed):
    """The operators by their definitions in 64 bits, a row (or an expert) at a time."""
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s, _spans(case))
    if case["op"] == "attention":
        return _exact_attention(s, _spans(case))
    return _exact_moe(s) if case["op"] == "moe" else _exact_sample(s)


def _exact_append(s, spans):
    cos, sin = s["cos"].double(), s["sin"].double()
    q_out = torch.zeros_like(s["q"], dtype=torch.float64)
    caches = [(s[n + "_pages"].double(), s[n + "_scale"].double()) for n in "kv"]
    page = s["k_pages"].shape[2]
    for b, (start, count) in enumerate(spans):
        rows = slice(start, start + count)
        turn = torch.complex(cos[rows], -sin[rows])[:, None]  # a rotation by minus the angle

        def turned(x):
            half = x.shape[-1] // 2
            y = torch.view_as_real(torch.complex(x[..., :half], x[..., half:]) * turn)
            y = torch.cat((y[..., 0], y[..., 1]), -1)
            return y if s["norm"] is None else s["norm"] * y / ((y * y).mean(-1, keepdim=True) + EPS).sqrt()

        q, k, v = (x[b, :count].double() for x in (s["q"], s["k"], s["v"]))
        q_out[b, :count] = turned(q)
        if s["ve"] is not None:
            v = v + 3 / (1 + torch.exp(-s["ve_gate"][b, :count].double()))[..., None] * s["ve"][b, :count].double()
        last = start + count - 1
        at = torch.arange(start // BLOCK, last // BLOCK + 1, device=q.device)     # blocks of the row
        number, slot = s["table"][b].long()[at * BLOCK // page], at * BLOCK % page
        slots = slot[:, None] + torch.arange(BLOCK, device=q.device)
        before = start % BLOCK
        for (codes, scale), x in zip(caches, (turned(k), v)):
            whole = torch.zeros(len(at) * BLOCK, *x.shape[1:], dtype=torch.float64, device=q.device)
            whole[before:before + count] = x
            whole = whole.view(len(at), BLOCK, *x.shape[1:])
            top = whole.abs().amax((1, 3))
            power = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(-100, 120))
            power = torch.where(top > 448 * power, 2 * power, torch.where(top <= 224 * power, power / 2, power))
            power = torch.where(top == 0, 2.0 ** -100, power)
            if before:
                old = scale[number[0], :, slot[0] // BLOCK].clone()
                power[0] = torch.maximum(power[0], old)
                whole[0, :before] = (codes[number[0], :, slot[0]:slot[0] + before] * old[:, None, None]).transpose(0, 1)
            new = _rounded(whole / power[:, None, :, None])
            old = codes[number[:, None], :, slots]
            position = at[:, None] * BLOCK + torch.arange(BLOCK, device=q.device)
            codes[number[:, None], :, slots] = torch.where((position <= last)[..., None, None], new, old)
            scale[number, :, slot // BLOCK] = power
    return q_out, caches[0][0], caches[1][0], caches[0][1], caches[1][1]


def _rounded(x):
    """To the nearest number with a sign, three bits behind the leading one and 2^-9 as the smallest step; ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_attention(s, spans):
    B, t, H, D = s["q"].shape
    Hk, page = s["k_pages"].shape[1:3]
    out = torch.zeros(B, t, H, D, dtype=torch.float64, device=s["q"].device)
    for b, (start, count) in enumerate(spans):
        total = start + count
        pages = s["table"][b, :-(-total // page)].long()
        K, V = ((s[n + "_pages"][pages].double() * s[n + "_scale"][pages].double().repeat_interleave(BLOCK, 2)[..., None])
                .transpose(0, 1).reshape(Hk, -1, D)[:, :total] for n in "kv")
        for i in range(count):
            first = max(0, start + i - s["window"]) if s["window"] >= 0 else 0
            q = s["q"][b, i].double().view(Hk, H // Hk, D)
            p = torch.softmax(torch.einsum("hgd,hkd->hgk", q, K[:, first:start + i + 1]) * D ** -0.5, -1)
            out[b, i] = torch.einsum("hgk,hkd->hgd", p, V[:, first:start + i + 1]).reshape(H, D)
    return out


def _exact_moe(s):
    x, k = s["x"].double(), s["top_k"]
    p = torch.softmax((s["router"].double() @ x.T).T, -1)
    taken = torch.zeros_like(p)
    score = p + s["bias"].double()
    rows = torch.arange(len(x), device=x.device)
    for _ in range(k):
        best = torch.where(taken > 0, -math.inf, score).argmax(-1)
        taken[rows, best] = 1.0
    c = p * taken / (p * taken).sum(-1, keepdim=True)
    y = torch.zeros_like(x)
    for e in torch.nonzero(taken.sum(0))[:, 0].tolist():
        who = torch.nonzero(taken[:, e])[:, 0]
        h = torch.relu(x[who] @ s["w_fc"][e].double().T) ** 2
        y[who] += c[who, e, None] * (h @ s["w_proj"][e].double().T)
    if s["shared_fc"] is not None:
        y += (torch.relu(x @ s["shared_fc"].double().T) ** 2) @ s["shared_proj"].double().T
    return y


def _exact_sample(s):
    tokens, chances = [], []
    B, V = s["logits"].shape
    for b in range(B):
        x = s["logits"][b].double()
        k, p, m = (None if s[n] is None else s[n][b].item() for n in ("top_k", "top_p", "min_p"))
        T = s["temperature"][b].item()
        if T <= 0:
            tokens.append(int(torch.nonzero(x == x.max())[0, 0]))
            chances.append(0.0)
            continue
        order = torch.argsort(x, descending=True, stable=True)
        if k:
            order = order[:k]
        w = torch.exp((x[order] - x[order[0]]) / T)
        n = len(order)
        if p is not None and p < 1:
            upto = torch.cumsum(w, 0)
            n = 1 + int((upto[:-1] < p * upto[-1]).sum())
        if m is not None:
            n = max(1, min(n, int((w >= m).sum())))
        kept, back = torch.sort(order[:n])
        mass = torch.cumsum(w[:n][back], 0)
        at = min(int(torch.searchsorted(mass, s["uniform"][b].double() * mass[-1], right=True)), n - 1)
        tokens.append(int(kept[at]))
        chances.append(float(torch.log(w[:n][back][at] / mass[-1])))
    return torch.tensor(tokens, device="cuda"), torch.tensor(chances, device="cuda", dtype=torch.float64)
