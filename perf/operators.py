"""Performance cases of the serving operators: what one generated token asks of them, from the smallest call to the largest.

* ``append``    ``ops.paged.paged_append``: rotation, QK norm and value embedding of new tokens, K / V written into a paged cache
* ``attention`` ``ops.paged.paged_attention``: new query tokens over the paged cache (GQA, left window)
* ``delta``     ``ops.delta_recurrent.delta_recurrent``: the gated delta rule token by token with a carried fp32 state
* ``logits``    ``ops.logits.adjust_logits``: penalties for repeated tokens, sparse biases and a grammar bit mask

``own`` selects the framework's operators; otherwise ``run`` evaluates their plain form in 32 bits with elementary torch operations.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 2.0 ** -23  # of the QK norm


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
        # one user, one token, Gated DeltaNet with the hybrid configurations' 12 heads of 128
        dict(name="delta one token", op="delta", kind="gdn", dtype="bf16", B=1, T=1, heads=12, dim=128, ragged=False),
        # a server's batch, KDA (a decay for each feature)
        dict(name="delta 160 rows", op="delta", kind="kda", dtype="bf16", B=160, T=1, heads=12, dim=128, ragged=False),
        # short prompts pass through the recurrence
        dict(name="delta 4 x 389 tokens", op="delta", kind="gdn", dtype="bf16", B=4, T=389, heads=12, dim=128,
             ragged=True),
        # one user, a vocabulary of 32768, a few hundred tokens so far
        dict(name="logits 1 x 32768", op="logits", dtype="bf16", B=1, vocab=32768, tokens=307, bias=0, mask=False),
        # a server's batch on the benchmark's vocabulary, everything switched on
        dict(name="logits 224 x 65536", op="logits", dtype="bf16", B=224, vocab=65536, tokens=2048, bias=48, mask=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "delta", "logits"])
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
                    length=t + before, ragged=rng.random() < 0.6, norm=rng.random() < 0.8,
                    ve=rng.random() < 0.5)
    if op == "attention":
        length = _log(rng, 1, 32768)
        t = min(length, rng.choice([1, 1, 1, 2, 3, 5, 8]))
        most = 16 * 32768 * 5 * 128 // (length * kv_heads * dim)
        return dict(op=op, dtype=dtype, B=_log(rng, 1, max(1, min(256, most))), t=t, heads=heads, kv_heads=kv_heads,
                    dim=dim, page=page, length=length, ragged=rng.random() < 0.6,
                    window=rng.choice([-1, -1, _log(rng, 1, 4096)]))
    if op == "delta":
        heads, T = rng.choice([1, 4, 6, 12, 16]), rng.choice([1, 1, 1, _log(rng, 2, 389)])
        most = min(128 * 12 // heads, 512 if T == 1 else 4 * 389 * 12 // (T * heads))
        return dict(op=op, kind=rng.choice(["deltanet", "gdn", "kda"]), dtype=dtype, B=_log(rng, 1, max(1, most)),
                    T=T, heads=heads, dim=rng.choice([64, 128, 128]), ragged=T > 1 and rng.random() < 0.6)
    vocab = _log(rng, 1000, 131072)
    return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), B=_log(rng, 1, max(1, min(256, 128 * 65536 // vocab))),
                vocab=vocab, tokens=_log(rng, 1, 2048), bias=rng.choice([0, 1, 48, 300]), mask=rng.random() < 0.5)


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


def _counts(case):
    """Of each row of a delta-rule case: its tokens."""
    if not case["ragged"]:
        return [case["T"]] * case["B"]
    rng = random.Random(case["B"] * 100003 + case["T"])
    return [case["T"] if b == 0 else _log(rng, 1, case["T"]) for b in range(case["B"])]


# ------------------------------------------------------------------------------------------ inputs
def _pages(case, spans, gen, dtype):
    """A cache whose pages are handed out in random order; what lies behind a row's last token is older data."""
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
    k = torch.randn(total + 3, Hk, page, D, generator=gen, device="cuda", dtype=dtype) * 1.2
    v = torch.randn(total + 3, Hk, page, D, generator=gen, device="cuda", dtype=dtype)
    return k, v, table.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = dict(op=case["op"])
    if case["op"] in ("append", "attention"):
        dtype = DTYPES[case["dtype"]]
        B, t, H, Hk, D = case["B"], case["t"], case["heads"], case["kv_heads"], case["dim"]
        spans = _spans(case)
        s["k_pages"], s["v_pages"], s["table"] = _pages(case, spans, gen, dtype)
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
        # the rows of the flattened [B * t] that are real tokens
        s["real"] = torch.tensor([b * t + i for b, (_, c) in enumerate(spans) for i in range(c)], device="cuda")
        return s
    if case["op"] == "delta":
        dtype = DTYPES[case["dtype"]]
        B, T, H, D, kind = case["B"], case["T"], case["heads"], case["dim"], case["kind"]
        s["q"], s["k"], s["v"] = (normal(B, T, H, D, dtype=dtype) for _ in range(3))
        s["beta"] = torch.sigmoid(normal(B, T, H)).to(dtype)
        s["g"] = None
        if kind == "gdn":  # decays as the layer's initialisation gives them
            rate = torch.rand(H, generator=gen, device="cuda") * 16
            step = torch.exp(torch.rand(H, generator=gen, device="cuda") * math.log(100.0)) * 1e-3
            s["g"] = -rate * torch.nn.functional.softplus(normal(B, T, H) + torch.log(torch.expm1(step)))
        elif kind == "kda":
            s["g"] = -torch.nn.functional.softplus(normal(B, T, H, D) - 3.0)
        s["state"] = normal(B + 2, H, D, D, scale=0.3)
        s["slots"] = torch.randperm(B + 2, generator=gen, device="cuda")[:B].to(torch.int32)
        s["count"] = ints(_counts(case))
        s["scale"] = D ** -0.5
        return s
    B, V, L = case["B"], case["vocab"], case["tokens"]
    padded = -(-V // 64) * 64  # the head's rows are padded to 64
    cap = 15.0
    logits = cap * torch.tanh(normal(B, padded, scale=4.0) / cap)
    s["logits"] = logits.to(torch.float32 if case["dtype"] == "fp32" else DTYPES[case["dtype"]])[:, :V]
    s["tokens"] = (V * torch.rand(B, L, generator=gen, device="cuda") ** 3).to(torch.int32).clamp(max=V - 1)
    rng = random.Random(B * 100003 + L)
    length = [L if b == 0 else _log(rng, 1, L) for b in range(B)]
    s["length"], s["prompt"] = ints(length), ints([n // 3 for n in length])
    s["repetition"] = 1.0 + 0.3 * torch.rand(B, generator=gen, device="cuda")
    s["presence"] = torch.rand(B, generator=gen, device="cuda")
    s["frequency"] = 0.5 * torch.rand(B, generator=gen, device="cuda")
    K = case["bias"]
    s["bias_ids"] = torch.randint(0, V, (B, K), generator=gen, device="cuda", dtype=torch.int32) if K else None
    s["bias"] = normal(B, K, scale=3.0) if K else None
    s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=gen, device="cuda",
                                 dtype=torch.int64).to(torch.int32) if case["mask"] else None
    return s


# ------------------------------------------------------------------------------------------ one pass
_operators = None


def _own():
    """The framework's operators, looked up once as a program's imports are."""
    global _operators
    if _operators is None:
        from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
        from nexttransformer_b200.ops.logits import adjust_logits
        from nexttransformer_b200.ops.paged import paged_append, paged_attention
        _operators = paged_append, paged_attention, delta_recurrent, adjust_logits
    return _operators


def run(s):
    op = s["op"]
    if not own:
        return _PLAIN[op](s)
    paged_append, paged_attention, delta_recurrent, adjust_logits = _own()
    if op == "append":
        q = paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["start"], s["count"],
                         cos=s["cos"], sin=s["sin"], qk_scale=s["norm"], ve=s["ve"], ve_gate=s["ve_gate"])
        return q, s["k_pages"], s["v_pages"]
    if op == "attention":
        return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["start"], s["count"],
                               window=s["window"])
    if op == "delta":
        o = delta_recurrent(s["q"], s["k"], s["v"], s["state"], s["beta"], s["g"], scale=s["scale"], l2norm=True,
                            slots=s["slots"], count=s["count"])
        return o, s["state"]
    return adjust_logits(s["logits"], tokens=s["tokens"], length=s["length"], prompt=s["prompt"],
                         repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                         bias_ids=s["bias_ids"], bias=s["bias"], allowed=s["allowed"])


def _plain_append(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    B, t, H, D = q.shape
    Hk, page = k.shape[2], s["k_pages"].shape[2]
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

    q, k = turned(q), turned(k)
    if s["ve"] is not None:
        v = v + 3 * torch.sigmoid(s["ve_gate"].float())[..., None] * s["ve"].float()
    real = s["real"]
    position = position.reshape(-1)[real]
    at = s["table"].long()[real // t, position // page], slice(None), position % page
    s["k_pages"][at] = k.reshape(B * t, Hk, D)[real].to(s["k_pages"].dtype)
    s["v_pages"][at] = v.reshape(B * t, Hk, D)[real].to(s["v_pages"].dtype)
    q = torch.where((new < s["count"][:, None])[:, :, None, None], q, 0.0)
    return q.to(s["q"].dtype), s["k_pages"], s["v_pages"]


def _plain_attention(s):
    B, t, H, D = s["q"].shape
    Hk, page = s["k_pages"].shape[1], s["k_pages"].shape[2]
    key = torch.arange(s["longest"], device=s["q"].device)
    at = s["table"].long()[:, key // page].clamp(min=0), slice(None), key % page
    K, V = s["k_pages"][at].float().transpose(1, 2), s["v_pages"][at].float().transpose(1, 2)  # [B, Hk, keys, D]
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


def _plain_delta(s):
    q, k, v, beta = s["q"].float(), s["k"].float(), s["v"].float(), s["beta"].float()
    B, T, H, D = q.shape
    q = q / q.norm(dim=-1, keepdim=True).clamp(min=1e-12) * s["scale"]
    k = k / k.norm(dim=-1, keepdim=True).clamp(min=1e-12)
    decay = None if s["g"] is None else torch.exp(s["g"]).reshape(B, T, H, -1, 1)
    slots = s["slots"].long()
    S = s["state"][slots]
    real = torch.arange(T, device=q.device) < s["count"][:, None]
    outputs = []
    for i in range(T):
        new = S if decay is None else S * decay[:, i]
        wrong = v[:, i] - (k[:, i, :, :, None] * new).sum(-2)
        new = new + k[:, i, :, :, None] * (beta[:, i, :, None] * wrong)[:, :, None]
        keep = real[:, i, None, None]
        S = torch.where(keep[..., None], new, S)
        outputs.append(torch.where(keep, (q[:, i, :, :, None] * S).sum(-2), 0.0))
    s["state"][slots] = S
    return torch.stack(outputs, 1).to(s["q"].dtype), s["state"]


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    at = torch.arange(s["tokens"].shape[1], device=x.device)
    said, tokens = at < s["length"][:, None], s["tokens"].long()
    answer = said & (at >= s["prompt"][:, None])
    seen = torch.zeros_like(x).scatter_add_(1, tokens, said.float()) > 0
    times = torch.zeros_like(x).scatter_add_(1, tokens, answer.float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * times - torch.where(times > 0, s["presence"][:, None], 0.0)
    if s["bias"] is not None:
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"].long(), s["bias"])
    if s["allowed"] is not None:
        ids = torch.arange(V, device=x.device)
        x = torch.where((s["allowed"][:, ids // 32] >> (ids % 32)) & 1 == 1, x, -math.inf)
    return x


_PLAIN = dict(append=_plain_append, attention=_plain_attention, delta=_plain_delta, logits=_plain_logits)


# ------------------------------------------------------------------------------------------ work and definition
def work(case):
    if case["op"] == "append":
        new = sum(c for _, c in _spans(case))
        per_token = case["heads"] + 2 * case["kv_heads"]
        each = 2 * case["dim"] * (2 * per_token + (case["kv_heads"] if case["ve"] else 0) + 1)
        return {"bytes": new * each + 12 * case["B"], "flops": new * per_token * case["dim"] * 6}
    if case["op"] == "attention":
        keys = pairs = 0
        for start, count in _spans(case):
            first = max(0, start - case["window"]) if case["window"] >= 0 else 0
            keys += start + count - first
            pairs += sum(min(start + i, case["window"] if case["window"] >= 0 else start + i) + 1 for i in range(count))
        rows = sum(c for _, c in _spans(case)) * case["heads"] * case["dim"]
        return {"bytes": 4 * keys * case["kv_heads"] * case["dim"] + 4 * rows + 4 * (keys // case["page"] + 2 * case["B"]),
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "delta":
        tokens, D = sum(_counts(case)) * case["heads"], case["dim"]
        gate = {"deltanet": 0, "gdn": 4, "kda": 4 * D}[case["kind"]]
        return {"bytes": 8 * case["B"] * case["heads"] * D * D + tokens * (8 * D + 2 + gate), "flops": 8 * tokens * D * D}
    B, V = case["B"], case["vocab"]
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": B * (V * (size + 4) + (V // 8 if case["mask"] else 0) + 4 * case["tokens"] + 8 * case["bias"]),
            "flops": 4 * B * V}


def exact(case, seed):
    """The operators by their definitions in 64 bits, a row at a time."""
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s, _spans(case))
    if case["op"] == "attention":
        return _exact_attention(s, _spans(case))
    if case["op"] == "delta":
        return _exact_delta(s, _counts(case))
    return _exact_logits(s)


def _exact_append(s, spans):
    page = s["k_pages"].shape[2]
    cos, sin = s["cos"].double(), s["sin"].double()
    k_pages, v_pages, q_out = s["k_pages"].double(), s["v_pages"].double(), torch.zeros_like(s["q"], dtype=torch.float64)
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
        k = turned(k)
        where = torch.arange(start, start + count, device=q.device)
        pages = s["table"][b].long()[where // page]
        k_pages[pages, :, where % page] = k
        v_pages[pages, :, where % page] = v
    return q_out, k_pages, v_pages


def _exact_attention(s, spans):
    B, t, H, D = s["q"].shape
    Hk, page = s["k_pages"].shape[1:3]
    out = torch.zeros(B, t, H, D, dtype=torch.float64, device=s["q"].device)
    for b, (start, count) in enumerate(spans):
        total = start + count
        pages = s["table"][b, :-(-total // page)].long()
        K, V = (x[pages].transpose(0, 1).reshape(Hk, -1, D)[:, :total].double() for x in (s["k_pages"], s["v_pages"]))
        for i in range(count):
            first = max(0, start + i - s["window"]) if s["window"] >= 0 else 0
            q = s["q"][b, i].double().view(Hk, H // Hk, D)
            p = torch.softmax(torch.einsum("hgd,hkd->hgk", q, K[:, first:start + i + 1]) * D ** -0.5, -1)
            out[b, i] = torch.einsum("hgk,hkd->hgd", p, V[:, first:start + i + 1]).reshape(H, D)
    return out


def _exact_delta(s, counts):
    q, k, v, beta = (s[n].double() for n in ("q", "k", "v", "beta"))
    q = torch.nn.functional.normalize(q, dim=-1) * s["scale"]
    k = torch.nn.functional.normalize(k, dim=-1)
    state, out = s["state"].double(), torch.zeros_like(v)
    slots = s["slots"].tolist()
    for i in range(max(counts)):
        rows = [b for b, c in enumerate(counts) if i < c]
        S = state[[slots[b] for b in rows]]
        if s["g"] is not None:
            g = s["g"][rows, i].double()
            S = S * torch.exp(g if g.dim() == 3 else g[..., None])[..., None]
        ki, qi = k[rows, i], q[rows, i]
        u = beta[rows, i][..., None] * (v[rows, i] - torch.einsum("bhk,bhkv->bhv", ki, S))
        out[rows, i] = torch.einsum("bhk,bhkv->bhv", qi, S) + (qi * ki).sum(-1, keepdim=True) * u
        state[[slots[b] for b in rows]] = S + torch.einsum("bhk,bhv->bhkv", ki, u)
    return out, state


def _exact_logits(s):
    x = s["logits"].double()
    V = x.shape[1]
    for b, (n, p) in enumerate(zip(s["length"].tolist(), s["prompt"].tolist())):
        history = s["tokens"][b, :n].long()
        times = torch.bincount(history[p:], minlength=V).double()
        seen = history.unique()
        r = s["repetition"][b].double()
        old = x[b, seen]
        x[b, seen] = torch.maximum(old, old * 0) / r + torch.minimum(old, old * 0) * r
        x[b] -= s["frequency"][b].double() * times + s["presence"][b].double() * times.clamp(max=1)
        if s["bias"] is not None:
            x[b].index_add_(0, s["bias_ids"][b].long(), s["bias"][b].double())
        if s["allowed"] is not None:
            bits = torch.stack([(s["allowed"][b].long() >> i) & 1 for i in range(32)], -1).flatten()[:V]
            x[b][bits == 0] = -math.inf
    return x
