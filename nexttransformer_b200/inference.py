"""Autoregressive decoding for the dense shell: a KV-cache engine and plain prefix re-run sampling.

``KVCache`` holds per-layer keys/values [B, T_max, Hk, D] and the position; ``decode`` runs the
shell block by block on the new tokens only (RoPE offset by the cache position, sliding windows
honoured, the smear gate reading the cached previous embedding).  Methods other than the dense
shell decode by re-running the full prefix, as the reference's ``generate`` does.

``PagedCache``, ``decode_paged`` and ``generate_batch`` serve many rows of unequal length at once, dense
models and delta-rule hybrids (DeltaNet, GDN, KDA layers between the shell's attention) alike: keys and values
lie in pages that rows take and give back (``ops.paged``), linear layers carry their convolution inputs and
recurrent state (``ops.delta_recurrent``), and next-token logits pass ``ops.logits.adjust_logits`` before they
are sampled.  The cache may be held in 8 bits, the experts of a mixture-of-experts model may be laid out for a few tokens
(``serve_experts``, ``ops.moe.moe_tokens``), and ``ops.sampling.sample_logits`` draws with top-p and min-p.
"""
import torch
import torch.nn.functional as F

from nexttransformer_b200.models.linear import LinearMixer
from nexttransformer_b200.models.moe import MoEFFN
from nexttransformer_b200.models.shell import Block, CausalSelfAttention, apply_rotary_emb, norm
from nexttransformer_b200.ops._ext import check_errors
from nexttransformer_b200.ops.logits import adjust_logits
from nexttransformer_b200.ops.paged import BLOCK, paged_append, paged_attention
from nexttransformer_b200.ops.sampling import sample_logits


class KVCache:
    def __init__(self, batch, max_len, n_layer, n_kv_head, head_dim, device, dtype):
        self.k = torch.zeros(n_layer, batch, max_len, n_kv_head, head_dim, device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)
        self.pos = 0
        self.prev_embedding = None


def supports_cache(model):
    return all(type(b) is Block and type(b.attn) is CausalSelfAttention for b in model.transformer.h)


@torch.no_grad()
def decode(model, idx, cache):
    """Logits of the last position after appending `idx` [B, t] to the cache."""
    B, t = idx.shape
    T0 = cache.pos
    cos, sin = model.cos[:, T0:T0 + t], model.sin[:, T0:T0 + t]
    x = norm(model.transformer.wte(idx).to(model.cos.dtype))
    prev = cache.prev_embedding
    cache.prev_embedding = x[:, -1:]
    gate_in = x
    if t > 1:
        g = model.smear_lambda.to(x.dtype) * torch.sigmoid(model.smear_gate(x[:, 1:, :24]))
        x = torch.cat((x[:, :1], x[:, 1:] + g * x[:, :-1]), 1)
    if prev is not None:
        g0 = model.smear_lambda.to(x.dtype) * torch.sigmoid(model.smear_gate(gate_in[:, :1, :24]))
        x = torch.cat((x[:, :1] + g0 * prev, x[:, 1:]), 1)
    x0 = x
    n = len(model.transformer.h)
    backout = None
    for i, blk in enumerate(model.transformer.h):
        x = model.resid_lambdas[i] * x + model.x0_lambdas[i] * x0
        a = blk.attn
        h = norm(x)
        ve = model.value_embeds[str(i)](idx).to(x.dtype) if str(i) in model.value_embeds else None
        q, k, v = a.project(h, ve, (cos, sin))
        cache.k[i, :, T0:T0 + t] = k
        cache.v[i, :, T0:T0 + t] = v
        K, V = cache.k[i, :, :T0 + t], cache.v[i, :, :T0 + t]
        w = model.window_sizes[i][0]
        qi = torch.arange(T0, T0 + t, device=idx.device)[:, None]
        kj = torch.arange(T0 + t, device=idx.device)[None, :]
        mask = (kj <= qi) & ((qi - kj) <= w if w >= 0 else torch.ones_like(kj, dtype=torch.bool))
        y = F.scaled_dot_product_attention(q.transpose(1, 2), K.transpose(1, 2), V.transpose(1, 2), attn_mask=mask,
                                           enable_gqa=K.shape[2] != q.shape[2])
        x = x + a.c_proj(y.transpose(1, 2).reshape(B, t, -1))
        x = x + blk.mlp(norm(x))
        if i == n // 2:
            backout = x
    cache.pos += t
    return model.readout(x[:, -1:], backout[:, -1:] if backout is not None else None)[:, -1]


@torch.no_grad()
def generate(model, tokens, max_tokens, temperature=1.0, top_k=None, seed=42, use_cache=True):
    """Yield sampled token ids after the prompt `tokens` (list of ints), batch 1."""
    dev = model.get_device()
    g = torch.Generator(device=dev).manual_seed(seed) if temperature > 0 else None
    ids = torch.tensor([tokens], dtype=torch.long, device=dev)
    cache = None
    if use_cache and supports_cache(model):
        cfg = model.shell
        cache = KVCache(1, len(tokens) + max_tokens, cfg.n_layer, cfg.n_kv_head, cfg.head_dim, dev, model.cos.dtype)
        logits = decode(model, ids, cache)
    for _ in range(max_tokens):
        if cache is None:
            logits = model(ids)[:, -1]
        logits = logits.float()
        if top_k:
            v, _ = torch.topk(logits, min(top_k, logits.size(-1)))
            logits[logits < v[:, [-1]]] = -float("inf")
        if temperature > 0:
            nxt = torch.multinomial(F.softmax(logits / temperature, -1), 1, generator=g)
        else:
            nxt = logits.argmax(-1, keepdim=True)
        ids = torch.cat((ids, nxt), 1)
        yield int(nxt.item())
        if cache is not None:
            logits = decode(model, nxt, cache)


# ------------------------------------------------------------------------------------------ many rows
def supports_paged(model):
    """True when ``decode_paged`` serves the model: plain blocks on one ordinary trunk whose mixers are the
    shell's attention or a delta-rule mixer; on CUDA in bf16 or fp16 with heads of 64 or 128."""
    from nexttransformer_b200.models.config import LOOPED, RESIDUAL
    c = getattr(model, "config", None)
    if c is not None and (c.method in LOOPED | RESIDUAL or model.plugin is not None):
        return False
    for b in model.transformer.h:
        linear = type(b) is Block and type(b.attn) is LinearMixer and b.attn.kind in ("deltanet", "gdn", "kda")
        if not linear and not (type(b) is Block and type(b.attn) is CausalSelfAttention):
            return False
        dim = b.attn.config.head_dim if linear else b.attn.head_dim
        if model.cos.is_cuda and (dim not in (64, 128) or model.cos.dtype == torch.float32):
            return False
    return True


class PagedCache:
    """What ``rows`` rows of a model carry from token to token.

    Attention layers share one pool of ``pages`` pages of ``page`` tokens (by default enough for every row to
    reach ``max_len``); ``reserve`` gives a row the pages for its next tokens, ``release`` takes them back and
    clears the row.  ``dtype`` is what keys and values are held in: the model's type, or ``torch.float8_e4m3fn`` with a scale
    for each 16 tokens and KV head (half the memory, and half of what attention reads).
    """

    def __init__(self, model, rows, max_len, page=64, pages=None, dtype=None):
        if not supports_paged(model):
            raise ValueError("this model has layers that the paged decoder does not serve")
        cfg, device = model.shell, model.get_device()
        held, dtype = model.cos.dtype if dtype is None else dtype, model.cos.dtype
        if held not in (dtype, torch.float8_e4m3fn):
            raise ValueError("the cache is held in the model's type or in float8_e4m3fn")
        if held == torch.float8_e4m3fn and page % BLOCK:
            raise ValueError(f"a float8_e4m3fn cache has pages of a multiple of {BLOCK} tokens")
        self.rows, self.page, self.columns = rows, page, -(-max_len // page)
        pages = rows * self.columns if pages is None else pages
        mixers = [b.attn for b in model.transformer.h]
        attention = [i for i, a in enumerate(mixers) if type(a) is CausalSelfAttention]
        linear = [i for i, a in enumerate(mixers) if type(a) is LinearMixer]
        shape = (len(attention), pages, cfg.n_kv_head, page, cfg.head_dim)
        keys, values = torch.zeros(shape, device=device, dtype=held), torch.zeros(shape, device=device, dtype=held)
        self.pages = {i: (keys[n], values[n]) for n, i in enumerate(attention)}
        self.scales = {i: {} for i in attention}
        if held == torch.float8_e4m3fn:
            shape = (2, *shape[:3], page // BLOCK)
            k_scale, v_scale = torch.zeros(shape, device=device)
            self.scales = {i: dict(k_scale=k_scale[n], v_scale=v_scale[n]) for n, i in enumerate(attention)}
        self.linear = {}
        for i in linear:
            c = mixers[i].config
            self.linear[i] = (torch.zeros(rows, mixers[i].q_conv.size - 1, 3 * c.width, device=device, dtype=dtype),
                              torch.zeros(rows, c.heads, c.head_dim, c.head_dim, device=device, dtype=torch.float32))
        self.table = torch.full((rows, self.columns), -1, dtype=torch.int32, device=device)
        self.start = torch.zeros(rows, dtype=torch.int32, device=device)
        self.prev_embedding = torch.zeros(rows, 1, cfg.n_embd, device=device, dtype=dtype)
        self.lengths = [0] * rows                       # the host's copy of start
        self.free = list(range(pages))[::-1]
        self.held = [[] for _ in range(rows)]

    def reserve(self, counts):
        """Pages for ``counts[row]`` more tokens of every row; raises when the pool is empty, and then takes none."""
        needs = []
        for row, n in enumerate(counts):
            if n and self.lengths[row] + n > self.columns * self.page:
                raise ValueError(f"row {row} would pass the cache's {self.columns * self.page} tokens")
            needs.append(max(0, -(-(self.lengths[row] + n) // self.page) - len(self.held[row])))
        if sum(needs) > len(self.free):
            raise RuntimeError("the paged cache has no free pages left")
        new = []
        for row, need in enumerate(needs):
            for _ in range(need):
                new.append((row, len(self.held[row]), self.free[-1]))
                self.held[row].append(self.free.pop())
        if new:
            row, column, number = torch.tensor(new, device=self.table.device).t()
            self.table[row, column] = number.int()

    def advance(self, counts, count):
        self.lengths = [a + n for a, n in zip(self.lengths, counts)]
        self.start += count

    def release(self, row):
        self.free += self.held[row][::-1]
        self.held[row], self.lengths[row] = [], 0
        self.table[row] = -1
        self.start[row] = 0
        self.prev_embedding[row] = 0
        for conv, state in self.linear.values():
            conv[row] = 0
            state[row] = 0


def serve_experts(model):
    """Lay the experts of a mixture-of-experts model out for decoding (``MoEFFN.serve``), once its weights are what is to be
    served; ``decode_paged`` then sends calls of up to 64 tokens through ``ops.moe.moe_tokens``.  Other layers are left alone."""
    for b in model.transformer.h:
        if isinstance(b.mlp, MoEFFN):
            b.mlp.serve(model.cos.dtype)


@torch.no_grad()
def decode_paged(model, idx, cache, counts=None):
    """Append ``idx [rows, t]`` to the cache and return logits ``[rows, V]`` of each row's last new token.

    ``counts`` (a list; t each by default) says how many of a row's t tokens are real; a row with 0 keeps its
    state, and its logits mean nothing.  It does not wait for the device; ``ops._ext.check_errors`` does, and raises
    for what the kernels recorded.
    """
    B, t = idx.shape
    if B != cache.rows:
        raise ValueError("one line of tokens for each row of the cache")
    counts = [t] * B if counts is None else list(counts)
    if any(not 0 <= n <= t for n in counts):
        raise ValueError("a row's count lies between 0 and the number of tokens given")
    if max(a + n for a, n in zip(cache.lengths, counts)) > model.cos.shape[1]:
        raise ValueError("sequence longer than the rotary cache")
    cache.reserve(counts)
    count = torch.tensor(counts, dtype=torch.int32, device=idx.device)
    slots = torch.arange(B, dtype=torch.int32, device=idx.device)
    last = (count.long() - 1).clamp(min=0)[:, None, None].expand(-1, 1, model.shell.n_embd)
    x = norm(model.transformer.wte(idx).to(model.cos.dtype))
    before = torch.cat((cache.prev_embedding, x[:, :-1]), 1)
    smear = model.smear_lambda.to(x.dtype) * torch.sigmoid(model.smear_gate(x[..., :24]))
    cache.prev_embedding = torch.where((count > 0)[:, None, None], x.gather(1, last), cache.prev_embedding)
    # the first token of a row has nothing before it: prev_embedding is zero there
    x = x + smear * before
    x0 = x
    cos, sin = model.cos[0, :, 0], model.sin[0, :, 0]
    n = len(model.transformer.h)
    backout = None
    for i, blk in enumerate(model.transformer.h):
        x = model.resid_lambdas[i] * x + model.x0_lambdas[i] * x0
        a = blk.attn
        h = norm(x)
        ve = model.value_embeds[str(i)](idx).to(x.dtype) if str(i) in model.value_embeds else None
        if i in cache.linear:
            y = a.step(h, ve, *cache.linear[i], slots, count)
        else:
            q, k, v = a.projections(h)
            q = q.view(B, t, a.n_head, a.head_dim)
            k, v = (z.view(B, t, a.n_kv_head, a.head_dim) for z in (k, v))
            gate = None
            if ve is not None and a.ve_gate is not None:
                gate = a.ve_gate(h[..., :a.ve_gate_channels])
                ve = ve.view(B, t, a.n_kv_head, a.head_dim)
            q = paged_append(q, k, v, *cache.pages[i], cache.table, cache.start, count, cos=cos, sin=sin, qk_scale=1.2,
                             ve=ve if gate is not None else None, ve_gate=gate, **cache.scales[i])
            y = paged_attention(q, *cache.pages[i], cache.table, cache.start, count, window=model.layer_window(i), **cache.scales[i])
            y = a.c_proj(y.view(B, t, -1))
        x = x + y
        x = x + (blk.mlp.step if isinstance(blk.mlp, MoEFFN) else blk.mlp)(norm(x))
        if i == n // 2:
            backout = x
    cache.advance(counts, count)
    return model.readout(x.gather(1, last), backout.gather(1, last) if backout is not None else None)[:, -1]


def _drawn_by_softmax(logits, temperature, top_k, g):
    """Next tokens ``[B, 1]`` by ``torch.multinomial``, and which rows permit no token or hold a NaN."""
    if top_k:
        v, _ = torch.topk(logits, min(top_k, logits.size(-1)))
        logits = logits.masked_fill(logits < v[:, [-1]], -float("inf"))
    # a row whose largest logit is not finite (over a small temperature, too) has a softmax of NaN, which sampling on
    # CUDA answers with a device assert: its largest logits share the choice; rows that have none are told apart below
    top = logits.amax(-1, keepdim=True)
    scaled = logits / temperature if temperature > 0 else logits
    scaled = torch.where(scaled.amax(-1, keepdim=True).isfinite(), scaled,
                         torch.where(top.isnan() | (logits == top), 0.0, -torch.inf))
    nxt = torch.multinomial(F.softmax(scaled, -1), 1, generator=g) if temperature > 0 else scaled.argmax(-1, keepdim=True)
    return nxt, top == -torch.inf, top.isnan()


@torch.no_grad()
def generate_batch(model, prompts, max_tokens, temperature=1.0, top_k=None, seed=42, stop=(), repetition=None,
                   presence=None, frequency=None, bias=None, allowed=None, page=64, top_p=None, min_p=None, cache_dtype=None):
    """Sample up to ``max_tokens`` tokens after each of ``prompts`` (lists of ints); a list of lists comes back.

    A row ends behind a token of ``stop``.  ``repetition``, ``presence`` and ``frequency`` are numbers, ``bias`` a
    dict from token to what is added to its logit, ``allowed`` a callable that gets the answers so far (a list
    of lists) and returns the grammar's bit masks for the next tokens, int32 ``[rows, ceil(V / 32)]`` (see
    ``ops.logits.adjust_logits``).  A row that it allows nothing ends there; rows that have ended may have any mask.  A
    bias of inf settles the choice; a NaN among a row's logits raises, as does at the end whatever the kernels recorded
    (``ops._ext.check_errors``).

    With ``top_p`` or ``min_p``, or where ``temperature`` or ``top_k`` is a list with one value for each prompt (as all four may
    be), tokens are drawn by ``ops.sampling.sample_logits`` from numbers of the seed's generator.  ``cache_dtype`` is the cache's
    (``PagedCache``).
    """
    if not prompts or any(not p for p in prompts):
        raise ValueError("every prompt needs at least one token")
    dev, B = model.get_device(), len(prompts)
    lengths = [len(p) for p in prompts]
    filters = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    drawn = top_p is not None or min_p is not None or any(isinstance(v, (list, tuple)) for v in filters.values())
    for name, v in filters.items():
        if isinstance(v, (list, tuple)):
            if len(v) != B:
                raise ValueError(f"{name}: one value for each prompt")
            filters[name] = torch.tensor(v, dtype=torch.int32 if name == "top_k" else torch.float32, device=dev)
    cache = PagedCache(model, B, max(lengths) + max_tokens, page, dtype=cache_dtype)
    g = torch.Generator(device=dev).manual_seed(seed) if drawn or temperature > 0 else None
    history = torch.zeros(B, max(lengths) + max_tokens, dtype=torch.int32)
    for row, p in enumerate(prompts):
        history[row, :len(p)] = torch.tensor(p, dtype=torch.int32)
    history = history.to(dev)
    prompt = torch.tensor(lengths, dtype=torch.int32, device=dev)
    length = prompt.clone()

    def each(value):
        return None if value is None else torch.full((B,), float(value), device=dev)
    penalties = dict(repetition=each(repetition), presence=each(presence), frequency=each(frequency))
    if bias:
        ids, values = torch.tensor(list(bias), dtype=torch.int32), torch.tensor([float(v) for v in bias.values()])
        penalties.update(bias_ids=ids.to(dev).expand(B, -1).contiguous(), bias=values.to(dev).expand(B, -1).contiguous())
    answers, live = [[] for _ in prompts], [True] * B
    logits = decode_paged(model, history[:, :max(lengths)].long(), cache, lengths)
    for step in range(max_tokens):
        logits = adjust_logits(logits, tokens=history, length=length, prompt=prompt, **penalties,
                               allowed=None if allowed is None else allowed(answers).to(dev))
        if drawn:
            token, _ = sample_logits(logits, torch.rand(B, generator=g, device=dev), **filters)
            nxt, nothing, broken = token.clamp(min=0)[:, None], token[:, None] == -1, token[:, None] == -2
        else:
            nxt, nothing, broken = _drawn_by_softmax(logits, temperature, top_k, g)
        for row, (token, nothing, broken) in enumerate(torch.cat((nxt, nothing, broken), 1).tolist()):
            if live[row] and broken:
                raise RuntimeError(f"NaN among the logits of row {row}")
            if live[row] and not nothing:
                answers[row].append(token)
            live[row] = live[row] and not nothing and token not in stop
        if step + 1 == max_tokens or not any(live):
            break
        counts = [int(alive) for alive in live]
        history.scatter_(1, length.long()[:, None], nxt.int())
        length += torch.tensor(counts, dtype=torch.int32, device=dev)
        logits = decode_paged(model, nxt, cache, counts)
    if history.is_cuda:
        check_errors()
    return answers
