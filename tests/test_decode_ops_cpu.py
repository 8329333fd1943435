"""The 8-bit cache, the experts of a few tokens and sampling: plain forms, refusals, the engine that uses them; on the CPU."""
import math
from dataclasses import replace

import pytest
import torch

from nexttransformer_b200.models import build_model
from nexttransformer_b200.models.config import debug_config
from nexttransformer_b200.ops.moe import moe_tokens
from nexttransformer_b200.ops.paged import paged_append, paged_attention
from nexttransformer_b200.ops.sampling import sample_logits

F8 = torch.float8_e4m3fn


def _model(method, seed=3, **extra):
    c = replace(debug_config(method), **extra) if extra else debug_config(method)
    m = build_model(c, "cpu", seed=seed).eval()
    with torch.no_grad():
        for b in m.transformer.h:
            b.attn.c_proj.weight.normal_(0, .05)
        m.smear_lambda.fill_(.7)
        m.lm_head.weight.normal_(0, .3)
    return c, m


def _cache(P, Hk, page, D, dtype=F8):
    return (torch.zeros(P, Hk, page, D).to(dtype), torch.zeros(P, Hk, page, D).to(dtype), torch.zeros(P, Hk, page // 16),
            torch.zeros(P, Hk, page // 16))


def _rotary(n, D):
    a = torch.outer(torch.arange(n).float(), 10000.0 ** (-torch.arange(0, D, 2) / D))
    return a.cos(), a.sin()


@pytest.mark.parametrize("first,n", [(0, 1), (0, 16), (0, 40), (5, 3), (5, 11), (5, 12), (15, 2), (16, 5), (37, 30)])
def test_plain_append_in_8_bits(first, n):
    """A row's tokens arrive as `first` in ones and `n` at once; each value lies within half a step of its block's final scale for each
    time that it was rounded, and the scale is the least power of two that reaches the block's largest."""
    torch.manual_seed(first * 100 + n)
    Hk, D, page, total = 2, 32, 32, first + n
    k_pages, v_pages, k_scale, v_scale = _cache(4, Hk, page, D)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    k = torch.randn(1, total, Hk, D) * torch.exp2(torch.randint(-6, 7, (1, total, 1, 1)).float())
    v = torch.randn(1, total, Hk, D)
    q = torch.randn(1, total, 4, D)
    cos, sin = _rotary(100, D)
    rest = dict(cos=cos, sin=sin, k_scale=k_scale, v_scale=v_scale)
    for i in range(first):
        paged_append(q[:, i:i + 1], k[:, i:i + 1], v[:, i:i + 1], k_pages, v_pages, table, torch.tensor([i], dtype=torch.int32), **rest)
    got = paged_append(q[:, first:], k[:, first:], v[:, first:], k_pages, v_pages, table, torch.tensor([first], dtype=torch.int32), **rest)
    wide = [torch.zeros(4, Hk, page, D) for _ in "kv"]
    ref = paged_append(q, k, v, *wide, table, torch.tensor([0], dtype=torch.int32), cos=cos, sin=sin)
    assert torch.equal(got, ref[:, first:])
    for codes, scale, exact in ((k_pages, k_scale, wide[0]), (v_pages, v_scale, wide[1])):
        for p in range(0, total, 16):
            at = int(table[0, p // page]), slice(None), slice(p % page, p % page + min(16, total - p))
            x, s = exact[at], scale[at[0], :, p % page // 16]
            top = x.abs().amax((1, 2))
            assert (top <= 448 * s).all() and (top > 224 * s).all() and torch.equal(torch.exp2(torch.log2(s).round()), s)
            step = torch.exp2(torch.floor(torch.log2((x / s[:, None, None]).abs().clamp(min=2.0 ** -6))) - 3) * s[:, None, None]
            # rounded once where it arrived, and under the smallest step once more for each growth: these add up to one step
            off = (codes[at].float() * s[:, None, None] - x).abs()
            assert (off <= 0.5 * step * 1.00001 + 2.0 ** -9 * s[:, None, None]).all()
    assert (k_pages.float()[1] == 0).all() and (k_scale[1] == 0).all()


def test_plain_append_in_8_bits_of_what_is_not_finite():
    k_pages, v_pages, k_scale, v_scale = _cache(1, 1, 16, 16)
    k = torch.ones(1, 2, 1, 16)
    k[0, 0, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    v = torch.zeros(1, 2, 1, 16)
    cos, sin = torch.ones(4, 8), torch.zeros(4, 8)
    paged_append(k, k, v, k_pages, v_pages, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), cos=cos, sin=sin,
                 k_scale=k_scale, v_scale=v_scale)
    back = k_pages.float() * k_scale[..., None]
    # channels 8 to 10 are the others' rotated partners: x_8 cos - x_0 sin with sin 0 is NaN where x_0 is not finite
    odd = torch.tensor([i % 8 < 3 for i in range(16)])
    assert torch.equal(back[0, 0, 0].isnan(), odd)
    assert (back[0, 0, 0][~odd] == 1).all() and (back[0, 0, 1] == 1).all()
    assert (v_pages.float() == 0).all() and v_scale[0, 0, 0] == 2.0 ** -100


@pytest.mark.parametrize("t,window", [(1, -1), (3, -1), (4, 7), (1, 0)])
def test_plain_attention_in_8_bits(t, window):
    """That of the numbers that the codes stand for."""
    torch.manual_seed(t)
    codes = [torch.randn(5, 2, 32, 16).mul(60).to(F8) for _ in "kv"]
    scales = [torch.exp2(torch.randint(-8, -3, (5, 2, 2)).float()) for _ in "kv"]
    wide = [c.float() * s.repeat_interleave(16, 2)[..., None] for c, s in zip(codes, scales)]
    q = torch.randn(2, t, 6, 16)
    table = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32)
    start = torch.tensor([40 - t, 3], dtype=torch.int32)
    got = paged_attention(q, *codes, table, start, window=window, k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(got, paged_attention(q, *wide, table, start, window=window))


def test_refusals_of_the_8_bit_cache():
    k_pages, v_pages, k_scale, v_scale = _cache(2, 2, 16, 16)
    q, table, start = torch.randn(1, 1, 4, 16), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def refused(kp, vp, ks, vs, match="k_scale and v_scale"):
        with pytest.raises(RuntimeError, match=match):
            paged_attention(q, kp, vp, table, start, k_scale=ks, v_scale=vs)
        with pytest.raises(RuntimeError, match=match):
            paged_append(q, q[:, :, :2], q[:, :, :2], kp, vp, table, start, cos=torch.ones(4, 8), sin=torch.ones(4, 8), k_scale=ks, v_scale=vs)
    refused(k_pages, v_pages, None, None)
    refused(k_pages, v_pages, k_scale, None)
    refused(k_pages.float(), v_pages.float(), k_scale, v_scale)
    refused(k_pages, v_pages.float(), k_scale, v_scale)
    refused(k_pages, v_pages, k_scale[:1], v_scale)
    refused(k_pages, v_pages, k_scale.double(), v_scale)
    with pytest.raises(RuntimeError, match="share a scale"):
        paged_append(q, q[:, :, :2], q[:, :, :2], k_pages, v_pages, table, start, cos=torch.ones(4, 8), sin=torch.ones(4, 8),
                     k_scale=k_scale, v_scale=v_scale[:1].expand(2, 2, 1))
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no backward"):
        paged_attention(q, k_pages, v_pages, table, start, k_scale=k_scale.clone().requires_grad_(), v_scale=v_scale)


# ------------------------------------------------------------------------------------------ sampling
def _by_hand(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """The definition, one row with Python's numbers."""
    x = [float(v) for v in x]
    top = max(x)
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if T <= 0:
        return order[0], 0.0
    w = {i: math.exp((x[i] - top) / T) if x[i] > -math.inf else 0.0 for i in order}
    if k > 0:
        order = order[:k]
    if p < 1:
        total, before, kept = math.fsum(w[i] for i in order), 0.0, []
        for i in order:
            if kept and before >= p * total:
                break
            kept.append(i)
            before += w[i]
        order = kept
    order = [i for j, i in enumerate(order) if j == 0 or w[i] >= min(m, 1.0)]
    total, upto = math.fsum(w[i] for i in order), 0.0
    for i in sorted(order):
        upto += w[i]
        if upto > u * total:
            return i, math.log(w[i] / total)


@pytest.mark.parametrize("V", [1, 2, 7, 50])
@pytest.mark.parametrize("T,k,p,m", [(1.0, 0, 1.0, 0.0), (0.5, 3, 1.0, 0.0), (2.0, 0, 0.7, 0.0), (1.0, 0, 1.0, 0.2), (0.8, 9, 0.6, 0.05),
                                     (0.0, 5, 0.5, 0.5), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 3.0)])
def test_plain_sampling(V, T, k, p, m):
    torch.manual_seed(V)
    x = torch.randn(20, V) * 2
    x[3] = x[3].round()                    # equal logits
    if V > 2:
        x[4, 1::2] = -math.inf             # not permitted
    u = torch.rand(20)
    T, p, m = (float(torch.tensor(v)) for v in (T, p, m))
    tokens, logprobs = sample_logits(x, u, temperature=T, top_k=k, top_p=p, min_p=m)
    rows = [torch.full((20,), v) for v in (T, p, m)]
    again, _ = sample_logits(x, u, temperature=rows[0], top_k=torch.full((20,), k, dtype=torch.int32), top_p=rows[1], min_p=rows[2])
    assert torch.equal(tokens, again) and tokens.dtype == torch.long and logprobs.dtype == torch.float32
    for b in range(20):
        token, logprob = _by_hand(x[b], float(u[b]), T, k, p, m)
        assert tokens[b] == token and abs(logprobs[b] - logprob) <= 1e-6 + 2.0 ** -22 * abs(logprob)


def test_plain_sampling_of_odd_rows():
    x = torch.zeros(6, 5)
    x[0] = -math.inf
    x[1, 3] = math.nan
    x[2, 1] = x[2, 4] = math.inf
    x[3, :4] = -math.inf
    u = torch.tensor([0.1, 0.1, 0.6, 0.9, 1.0, math.nan])
    tokens, logprobs = sample_logits(x, u, top_p=0.9)
    assert tokens.tolist() == [-1, -2, 4, 4, 4, 0]
    assert logprobs[0] == -math.inf and logprobs[1].isnan() and abs(logprobs[2] - math.log(0.5)) < 1e-6 and logprobs[3] == 0
    with pytest.raises(RuntimeError, match="B, V"):
        sample_logits(x[0], u)
    with pytest.raises(RuntimeError, match="one entry for each row"):
        sample_logits(x, u, top_p=torch.ones(5))
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no backward"):
        sample_logits(x.clone().requires_grad_(), u)


# ------------------------------------------------------------------------------------------ experts
@pytest.mark.parametrize("T,shared", [(1, 1), (7, 0), (5, 2)])
def test_plain_experts_equal_the_layer(T, shared):
    from nexttransformer_b200.models.moe import MoEFFN
    torch.manual_seed(T)
    layer = MoEFFN(32, 8, 3, 24, shared=shared).eval()
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0, 0.3)
        layer.expert_bias.normal_(0, 0.05)
        x = torch.randn(T, 32)
        ref = layer(x)
        assert torch.equal(layer.step(x), ref)       # not laid out: the layer itself
        layer.serve(torch.float32)
        load = layer.load.clone()
        assert torch.allclose(layer.step(x), ref, rtol=1e-5, atol=1e-5 * ref.abs().max().item())
        assert torch.equal(layer.load, load)
        many = torch.randn(65, 32)
        assert torch.allclose(layer.step(many), layer(many))


def test_plain_experts_refusals_and_ties():
    x, router = torch.randn(2, 16), torch.zeros(4, 16)
    w_fc, w_proj = torch.randn(4, 8, 16), torch.randn(4, 16, 8)
    for bad in (dict(x=x[0]), dict(router=router[:, :8]), dict(w_proj=w_proj[:3]), dict(top_k=0), dict(top_k=5), dict(shared_fc=w_fc[0])):
        a = dict(dict(x=x, router=router, w_fc=w_fc, w_proj=w_proj, top_k=2), **bad)
        with pytest.raises(RuntimeError):
            moe_tokens(**a)
    got = moe_tokens(x, router, w_fc, w_proj, 2)      # all equal: experts 0 and 1, a half each
    ref = sum(0.5 * torch.relu(x @ w_fc[e].T).square() @ w_proj[e].T for e in (0, 1))
    assert torch.allclose(got, ref, rtol=1e-5, atol=1e-5)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no backward"):
        moe_tokens(x.clone().requires_grad_(), router, w_fc, w_proj, 2)


def test_laid_out_experts_change_together():
    """What was laid out stays of one state of the weights until it is laid out again."""
    from nexttransformer_b200.models.moe import MoEFFN
    torch.manual_seed(3)
    layer, x = MoEFFN(32, 8, 3, 24, shared=1).eval(), torch.randn(5, 32)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0, 0.3)
        before = layer(x)
        layer.serve(torch.float32)
        for p in (*layer.parameters(), layer.expert_bias):
            p.normal_(0, 0.3)
        after = layer(x)
        assert not torch.allclose(before, after, rtol=1e-2)
        assert torch.allclose(layer.step(x), before, rtol=1e-5, atol=1e-5 * before.abs().max().item())
        layer.serve(torch.float32)
        assert torch.allclose(layer.step(x), after, rtol=1e-5, atol=1e-5 * after.abs().max().item())


# ------------------------------------------------------------------------------------------ the engine
def test_decode_with_laid_out_experts():
    """Ragged prompts and pausing rows against the same without: the same layer, so the same logits but for the sums' order."""
    from nexttransformer_b200.inference import PagedCache, decode_paged, serve_experts
    c, m = _model("moe")
    ids = torch.randint(0, c.vocab_size, (3, 5))
    logits = []
    for laid_out in (False, True):
        if laid_out:
            serve_experts(m)
        cache = PagedCache(m, 3, 12, page=16)
        a = decode_paged(m, ids, cache, [5, 1, 3])
        b = decode_paged(m, ids[:, :1], cache, [1, 0, 1])
        logits.append(torch.cat((a, b[[0, 2]])))
    assert torch.allclose(*logits, atol=2e-4)


def test_decode_over_an_8_bit_cache():
    """The first layer's keys and values, which see the same tokens in both caches, lie within half a step of each other; a row's pages
    are begun anew after its release."""
    from nexttransformer_b200.inference import PagedCache, decode_paged
    c, m = _model("dense")
    ids = torch.randint(0, c.vocab_size, (2, 9))
    cache, other = PagedCache(m, 2, 32, page=16, dtype=F8), PagedCache(m, 2, 32, page=16)
    for x in (cache, other):
        decode_paged(m, ids, x, [9, 4])
    for i, (k, v) in cache.pages.items():
        assert k.dtype == F8 and k.element_size() == 1
        for wide, codes, scale in zip(other.pages[i], (k, v), cache.scales[i].values()):
            held = codes.float() * scale.repeat_interleave(16, 2)[..., None]
            for b, n in enumerate((9, 4)):
                page = int(cache.table[b, 0])
                if i == 0:  # the first layer saw the same tokens
                    x, s = wide[page, :, :n], scale[page, :, 0][:, None, None]
                    assert ((held[page, :, :n] - x).abs() <= 2.0 ** -4 * x.abs() * 1.00001 + 2.0 ** -10 * s).all()
    assert cache.lengths == [9, 4]
    a = decode_paged(m, ids[:, :1], cache, [1, 0])
    assert a.isfinite().all()
    cache.release(0)
    decode_paged(m, ids[:, :3], cache, [3, 0])
    assert cache.lengths == [3, 4]
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedCache(m, 1, 32, page=24, dtype=F8)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        PagedCache(m, 2, 32, dtype=torch.float16)


def test_generate_batch_draws_with_filters():
    from nexttransformer_b200.inference import generate_batch
    c, m = _model("dense")
    prompts = [[3, 1, 4], [1], [5, 9]]
    greedy = generate_batch(m, prompts, 6, temperature=0)
    assert generate_batch(m, prompts, 6, top_p=1e-6) == greedy
    assert generate_batch(m, prompts, 6, min_p=1.0) == greedy
    assert generate_batch(m, prompts, 6, top_k=[1, 1, 1]) == greedy
    assert generate_batch(m, prompts, 6, temperature=0, top_p=0.5) == greedy
    one = generate_batch(m, prompts, 6, temperature=[0.0, 1.5, 0.0], top_p=0.9, seed=1)
    assert [one[0], one[2]] == [greedy[0], greedy[2]]
    assert one == generate_batch(m, prompts, 6, temperature=[0.0, 1.5, 0.0], top_p=0.9, seed=1)
    eight = generate_batch(m, prompts, 6, top_p=0.9, min_p=0.01, cache_dtype=F8)
    assert all(len(a) == 6 for a in eight)
    with pytest.raises(ValueError, match="one value for each prompt"):
        generate_batch(m, prompts, 2, top_p=[0.5])
    # rows that may say nothing end, a NaN raises
    none = torch.zeros(3, -(-c.vocab_size // 32), dtype=torch.int32)
    none[1] = -1
    assert [len(a) for a in generate_batch(m, prompts, 3, top_p=0.9, allowed=lambda answers: none)] == [0, 3, 0]
    with torch.no_grad():
        m.lm_head.weight[2] = math.nan
    with pytest.raises(RuntimeError, match="NaN among the logits of row 0"):
        generate_batch(m, prompts, 2, top_p=0.9)


def test_generate_cli_with_filters(tmp_path, monkeypatch, capsys):
    from nexttransformer_b200 import generate
    c, m = _model("moe")
    monkeypatch.setattr("nexttransformer_b200.models.load_model", lambda *a, **k: (m, None))
    f = tmp_path / "prompts.txt"
    f.write_text("1 2 3\n4\n")
    generate.main(["--checkpoint", "x", "--batch", str(f), "--tokens", "3", "--top-p", "0.8", "--min-p", "0.01", "--cache-8bit", "--serve-experts"])
    assert [len(line.split()) for line in capsys.readouterr().out.splitlines()] == [3, 3]
    generate.main(["--checkpoint", "x", "--prompt", "1 2", "--tokens", "2", "--top-p", "0.8"])
    assert len(capsys.readouterr().out.splitlines()) == 1
