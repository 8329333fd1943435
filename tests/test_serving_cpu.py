"""The serving operators' plain forms, the paged decoder and batched generation on the CPU."""
import math
from dataclasses import replace

import pytest
import torch

from nexttransformer_b200.models import build_model
from nexttransformer_b200.models.config import debug_config


def _model(method, seed=3, **extra):
    c = replace(debug_config(method), **extra) if extra else debug_config(method)
    m = build_model(c, "cpu", seed=seed).eval()
    with torch.no_grad():
        for b in m.transformer.h:
            b.attn.c_proj.weight.normal_(0, .05)
            if hasattr(b.mlp, "c_proj"):
                b.mlp.c_proj.weight.normal_(0, .05)
        m.smear_lambda.fill_(.7)
        m.lm_head.weight.normal_(0, .3)
    return c, m


@pytest.mark.parametrize("method", ["dense", "gdn_hybrid_swa", "gdn_hybrid", "deltanet", "kda", "kda_no_ve"])
def test_paged_decode_matches_full_forward(method):
    """Ragged prompts at once, then token by token with a row pausing, against the full forward of every prefix."""
    from nexttransformer_b200.inference import PagedCache, decode_paged
    c, m = _model(method)
    torch.manual_seed(0)
    rows = torch.randint(0, c.vocab_size, (3, 12))
    have = [5, 1, 3]
    cache = PagedCache(m, 3, 12, page=16)
    logits = decode_paged(m, rows[:, :5], cache, have)

    def check(active):
        for r in active:
            full = m(rows[r:r + 1, :have[r]])[:, -1]
            assert torch.allclose(logits[r], full[0], atol=2e-4), (method, r, have, (logits[r] - full[0]).abs().max())
    check(range(3))
    for counts in ([1, 1, 1], [1, 0, 1], [1, 2, 0], [2, 1, 3]):
        t = max(counts)
        new = torch.stack([torch.nn.functional.pad(rows[r, have[r]:have[r] + n], (0, t - n)) for r, n in enumerate(counts)])
        logits = decode_paged(m, new, cache, counts)
        have = [a + n for a, n in zip(have, counts)]
        check([r for r, n in enumerate(counts) if n])
    assert cache.lengths == have == cache.start.tolist()


def test_paged_cache_gives_pages_back():
    from nexttransformer_b200.inference import PagedCache, decode_paged
    c, m = _model("gdn_hybrid_swa")
    cache = PagedCache(m, 2, 64, page=16, pages=3)
    ids = torch.randint(0, c.vocab_size, (2, 12))
    first = decode_paged(m, ids, cache)
    assert len(cache.free) == 1
    decode_paged(m, ids[:, :6], cache, [6, 0])
    with pytest.raises(RuntimeError, match="no free pages"):
        decode_paged(m, ids[:, :6], cache, [0, 6])
    cache.release(0)
    cache.release(1)
    assert sorted(cache.free) == [0, 1, 2] and (cache.table == -1).all()
    assert torch.equal(decode_paged(m, ids, cache), first)
    with pytest.raises(ValueError, match="count"):
        decode_paged(m, ids, cache, [13, 0])
    with pytest.raises(ValueError, match="line of tokens"):
        decode_paged(m, ids[:1], cache)
    with pytest.raises(ValueError, match="pass the cache"):
        PagedCache(m, 1, 16, page=16).reserve([17])


def test_unsupported_models_are_refused():
    from nexttransformer_b200.inference import PagedCache, supports_paged
    for method in ("mla_nope", "ouro", "hc", "gla", "nsa"):
        m = build_model(debug_config(method), "cpu", seed=0)
        assert not supports_paged(m)
        with pytest.raises(ValueError, match="paged decoder"):
            PagedCache(m, 1, 16)


def test_generate_batch_equals_single_greedy():
    from nexttransformer_b200.inference import generate, generate_batch
    c, m = _model("dense")
    prompts = [[3, 1, 4, 1, 5], [9, 2], [6]]
    # sequence_len bounds the plain forward, not the cached one
    single = [list(generate(m, p, 6, temperature=0)) for p in prompts]
    assert generate_batch(m, prompts, 6, temperature=0, page=16) == single
    stop = single[0][2]
    ended = generate_batch(m, prompts, 6, temperature=0, page=16, stop=(stop,))
    for whole, cut in zip(single, ended):
        assert cut == whole[:whole.index(stop) + 1 if stop in whole else None]


def test_generate_batch_penalties_and_masks():
    from nexttransformer_b200.inference import generate_batch
    c, m = _model("gdn_hybrid")
    prompts = [[1, 2, 3], [4]]
    V = c.vocab_size
    answers = generate_batch(m, prompts, 5, temperature=0, page=16, frequency=1e6, presence=1.0)
    assert all(len(set(a)) == 5 for a in answers)                      # nothing twice
    answers = generate_batch(m, prompts, 4, temperature=0, page=16, repetition=1e9, bias={7: 1e4})
    assert all(a[0] == 7 for a in answers)

    def only(token):
        mask = torch.zeros(2, -(-V // 32), dtype=torch.int64)
        mask[:, token // 32] = 1 << (token % 32)
        return torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).int()
    got = generate_batch(m, prompts, 3, temperature=1.0, page=16, allowed=lambda done: only(31 + len(done[0])))
    assert got == [[31, 32, 33]] * 2
    with pytest.raises(ValueError, match="prompt"):
        generate_batch(m, [[]], 1)


def test_generate_cli_batch(tmp_path, monkeypatch, capsys):
    import nexttransformer_b200.generate as cli
    import nexttransformer_b200.models as models
    c, m = _model("dense")
    monkeypatch.setattr(models, "load_model", lambda *a, **k: (m, None))
    (tmp_path / "prompts").write_text("1 2 3\n4\n")
    cli.main(["--checkpoint", "x", "--batch", str(tmp_path / "prompts"), "--tokens", "4", "--temperature", "0"])
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 2 and all(len(line.split()) == 4 for line in lines)
    cli.main(["--checkpoint", "x", "--prompt", "1 2 3", "--tokens", "2", "--temperature", "0", "--bias", "5:1000"])
    assert capsys.readouterr().out.split() == ["5", "5"]


# ------------------------------------------------------------------------------------------ plain forms
def test_plain_paged_operators():
    """One row by hand: pages out of order, a window, GQA."""
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    torch.manual_seed(1)
    H, Hk, D, page = 4, 2, 8, 16
    kp, vp = torch.zeros(4, Hk, page, D), torch.zeros(4, Hk, page, D)
    table = torch.tensor([[2, 0, -1]], dtype=torch.int32)
    angle = torch.rand(64, D // 2)
    q, k, v = torch.randn(1, 20, H, D), torch.randn(1, 20, Hk, D), torch.randn(1, 20, Hk, D)
    start = torch.zeros(1, dtype=torch.int32)
    out_q = paged_append(q, k, v, kp, vp, table, start, torch.tensor([19]), cos=angle.cos(), sin=angle.sin())
    turn = torch.polar(torch.ones(19, 1, D // 2), -angle[:19, None])
    ref_k = torch.view_as_real(torch.complex(*k[0, :19].chunk(2, -1)) * turn)
    ref_k = torch.cat((ref_k[..., 0], ref_k[..., 1]), -1)
    assert torch.allclose(kp[2].transpose(0, 1), ref_k[:16], atol=1e-6) and torch.allclose(kp[0, :, :3].transpose(0, 1), ref_k[16:], atol=1e-6)
    assert torch.equal(vp[0, :, 2], v[0, 18]) and (kp[0, :, 3:] == 0).all() and (out_q[0, 19:] == 0).all()
    y = paged_attention(out_q, kp, vp, table, start, torch.tensor([19]), window=5)
    for i, h in ((0, 0), (4, 3), (18, 1)):
        lo = max(0, i - 5)
        p = torch.softmax(ref_k[lo:i + 1, h // 2] @ out_q[0, i, h] / math.sqrt(D), 0)
        assert torch.allclose(y[0, i, h], p @ v[0, lo:i + 1, h // 2], atol=1e-5)
    assert (y[0, 19:] == 0).all()
    with pytest.raises(RuntimeError, match="page number"):
        paged_attention(q[:, :1], kp, vp, table, torch.tensor([40], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="page table"):
        paged_attention(q[:, :1], kp, vp, table, torch.tensor([48], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="rotary"):
        paged_append(q[:, :1], k[:, :1], v[:, :1], kp, vp, table, torch.tensor([9]), cos=angle[:9], sin=angle[:9])
    with pytest.raises(RuntimeError, match="backward"):
        paged_attention(q.requires_grad_(), kp, vp, table, start)


def test_plain_delta_recurrent():
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    torch.manual_seed(2)
    q, k, v = (torch.randn(2, 3, 1, 4) for _ in range(3))
    beta, g, state = torch.rand(2, 3, 1), -torch.rand(2, 3, 1, 4), torch.randn(3, 1, 4, 4)
    ref = state[2, 0].clone()
    o = delta_recurrent(q, k, v, state, beta, g, scale=.5, l2norm=True, slots=torch.tensor([2, -1]), count=torch.tensor([2, 3]))
    for t in range(2):
        kk, qq = k[0, t, 0] / k[0, t, 0].norm(), q[0, t, 0] / q[0, t, 0].norm()
        ref = ref * g[0, t, 0].exp()[:, None]
        ref = ref + torch.outer(kk, beta[0, t, 0] * (v[0, t, 0] - kk @ ref))
        assert torch.allclose(o[0, t, 0], .5 * qq @ ref, atol=1e-6)
    assert torch.allclose(state[2, 0], ref, atol=1e-6) and (o[0, 2] == 0).all() and (o[1] == 0).all()
    with pytest.raises(RuntimeError, match="slot"):
        delta_recurrent(q, k, v, state, beta, g, slots=torch.tensor([0, 3]))


def test_plain_adjust_logits():
    from nexttransformer_b200.ops.logits import adjust_logits
    x = torch.tensor([[2., -2., 1., 0., 5.]])
    got = adjust_logits(x, tokens=torch.tensor([[0, 1, 1, 4, 9]]), length=torch.tensor([4]), prompt=torch.tensor([1]),
                        repetition=torch.tensor([2.]), presence=torch.tensor([.5]), frequency=torch.tensor([.25]),
                        bias_ids=torch.tensor([[2, 2, -1]]), bias=torch.tensor([[1., 2., 3.]]),
                        allowed=torch.tensor([[0b01111]], dtype=torch.int32))
    assert torch.allclose(got, torch.tensor([[1., -4 - .5 - .5, 4., 0., -math.inf]]))
