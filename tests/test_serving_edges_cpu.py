"""The serving engine and the operators' plain forms where they can go wrong, on the CPU."""
import math

import pytest
import torch

from tests.test_serving_cpu import _model


@pytest.mark.parametrize("method", ["dense", "gdn_hybrid_swa"])
@pytest.mark.parametrize("fault", ["pool", "limit"])
def test_a_refused_reservation_takes_nothing(method, fault):
    """Rows before the one that cannot be served want a page too; nothing of the cache moves, and after a release the same
    call gives what a cache that never refused gives."""
    from nexttransformer_b200.inference import PagedCache, decode_paged
    c, m = _model(method)
    torch.manual_seed(4)
    ids = torch.randint(0, c.vocab_size, (3, 16))
    new = torch.randint(0, c.vocab_size, (3, 2))
    calm, cache = (PagedCache(m, 3, 48, page=16, pages=n) for n in (9, 4 if fault == "pool" else 9))
    for x in (calm, cache):
        decode_paged(m, ids, x)
    if fault == "limit":                       # row 2 stands at the cache's end
        for x in (calm, cache):
            decode_paged(m, ids, x, [0, 0, 16])
            decode_paged(m, ids, x, [0, 0, 16])

    def books():
        return [list(h) for h in cache.held], list(cache.free), list(cache.lengths), cache.table.clone(), cache.start.clone()
    before = books()
    with pytest.raises((RuntimeError, ValueError), match="no free pages" if fault == "pool" else "pass the cache"):
        decode_paged(m, new, cache)
    for a, b in zip(before, books()):
        assert torch.equal(a, b) if torch.is_tensor(a) else a == b
    cache.release(2)
    calm.release(2)
    counts = [2, 2, 0]
    for _ in range(2):
        assert torch.equal(decode_paged(m, new, cache, counts)[:2], decode_paged(m, new, calm, counts)[:2])
    assert sorted(cache.free + sum(cache.held, [])) == list(range(len(cache.free) + sum(map(len, cache.held))))


@pytest.mark.parametrize("temperature", [0, 1.0])
@pytest.mark.parametrize("top_k", [None, 5])
def test_a_grammar_that_allows_nothing(temperature, top_k):
    """An ended answer's mask does not matter; a running answer that may not go on ends without a token; the others go on."""
    from nexttransformer_b200.inference import generate_batch
    c, m = _model("dense")
    prompts, words = [[3, 1, 4], [9, 2], [6]], -(-c.vocab_size // 32)

    def one(token):
        mask = [0] * words
        mask[token // 32] = 1 << (token % 32)
        return mask

    def grammar(done):   # row 0: 7 then stop token 8, then nothing; row 1: 5 for ever; row 2: 10, 11, then nothing
        first = [one(7), one(8)][len(done[0])] if len(done[0]) < 2 else [0] * words
        last = [one(10), one(11)][len(done[2])] if len(done[2]) < 2 else [0] * words
        return torch.tensor([first, one(5), last], dtype=torch.int32)
    got = generate_batch(m, prompts, 6, temperature=temperature, top_k=top_k, page=16, stop=(8,), allowed=grammar)
    assert got == [[7, 8], [5] * 6, [10, 11]]
    nothing = generate_batch(m, prompts, 6, temperature=temperature, top_k=top_k, page=16,
                             allowed=lambda done: torch.zeros(3, words, dtype=torch.int32))
    assert nothing == [[], [], []]


@pytest.mark.parametrize("temperature", [0, 1.0])
def test_logits_that_are_not_finite(temperature):
    """NaN names its row; an infinite bias settles the choice."""
    from nexttransformer_b200.inference import generate_batch
    c, m = _model("dense")
    with torch.no_grad():
        m.transformer.wte.weight[7] = math.nan
    with pytest.raises(RuntimeError, match="row 1"):
        generate_batch(m, [[3, 1], [7], [2]], 2, temperature=temperature, page=16)
    for bias in ({7: -1e9, 5: 1e6}, {7: -math.inf, 5: math.inf}, {7: -1e38, 5: 3e38}):
        assert generate_batch(m, [[3, 1], [2]], 2, temperature=temperature, top_k=3, page=16, bias=bias) == [[5, 5]] * 2
    assert generate_batch(m, [[3, 1]], 2, temperature=temperature * 1e-40, page=16, bias={7: -math.inf, 5: 9.0}) == [[5, 5]]


# what each operator is called with where every tensor that may carry a gradient is given
def _serving_calls(device, dtype):
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    from nexttransformer_b200.ops.logits import adjust_logits
    from nexttransformer_b200.ops.paged import paged_append, paged_attention

    def ones(*shape, dtype=dtype):
        return torch.ones(*shape, device=device, dtype=dtype)

    def zeros(*shape):
        return torch.zeros(*shape, device=device, dtype=torch.int32)
    q, kv, pages, rope = ones(1, 1, 4, 64), ones(1, 1, 2, 64), ones(1, 2, 16, 64), ones(16, 32)
    cache = dict(k_pages=pages, v_pages=pages.clone(), table=zeros(1, 1), start=zeros(1))
    per_row = ones(1, dtype=torch.float32)
    return {
        "append": (paged_append, dict(q=q, k=kv, v=kv, cos=rope, sin=rope, ve=kv, ve_gate=kv[..., 0], **cache)),
        "attention": (paged_attention, dict(q=q, **cache)),
        "delta": (delta_recurrent, dict(q=kv, k=kv, v=kv, beta=kv[..., 0], g=ones(1, 1, 2, dtype=torch.float32),
                                        state=ones(1, 2, 64, 64, dtype=torch.float32))),
        "logits": (adjust_logits, dict(logits=ones(1, 32), tokens=zeros(1, 3), repetition=per_row, presence=per_row,
                                       frequency=per_row, bias_ids=zeros(1, 1), bias=ones(1, 1, dtype=torch.float32))),
    }


@pytest.mark.parametrize("op,name", [
    *(("append", n) for n in ("q", "k", "v", "k_pages", "v_pages", "cos", "sin", "ve", "ve_gate")),
    *(("attention", n) for n in ("q", "k_pages", "v_pages")),
    *(("delta", n) for n in ("q", "k", "v", "beta", "g", "state")),
    *(("logits", n) for n in ("logits", "repetition", "presence", "frequency", "bias")),
])
def test_no_gradient_is_dropped(op, name):
    """Whichever argument wants a gradient is refused while gradients are recorded, and welcome under no_grad."""
    call, args = _serving_calls("cpu", torch.float32)[op]
    call(**args)
    args[name] = args[name].detach().clone().requires_grad_()
    with pytest.raises(RuntimeError, match="backward"):
        call(**args)
    with torch.no_grad():
        call(**args)


def test_check_errors_tells_everything_at_once(monkeypatch):
    """Reading clears the records, so an error that is read and not told would be lost."""
    from nexttransformer_b200.ops import _ext

    class Recorded:
        gemm, serving = [7, 0x10, 0, 0, 0, 0, 0, 0], [2, 5, 2, 3]

        def read_errors(self):
            got, Recorded.gemm = Recorded.gemm, [0] * 8
            return got

        def read_serving_errors(self):
            got, Recorded.serving = Recorded.serving, [0] * 4
            return got
    monkeypatch.setattr(_ext, "ext", Recorded)
    with pytest.raises(RuntimeError) as said:
        _ext.check_errors()
    for words in ("gemm code 7 at 0x10", "page number lies outside the cache (row 5)", "slot outside the states (row 3)"):
        assert words in str(said.value)
    _ext.check_errors()


@pytest.mark.parametrize("t,window", [(1, 0), (1, 20), (3, 20), (3, 100)])
def test_plain_attention_reads_nothing_before_every_window(t, window):
    """Pages before the oldest key that a token sees may have been given back, and their memory may hold anything."""
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(6)
    n, H, Hk, D, page = 77, 4, 2, 8, 16
    K, V = torch.randn(n, Hk, D), torch.randn(n, Hk, D)
    q = torch.randn(1, t, H, D)
    start = n - t
    first = max(0, start - window)
    kp, vp = (torch.full((5, Hk, page, D), math.nan) for _ in range(2))
    for x, pages in ((K, kp), (V, vp)):
        for p in range(first, n):
            pages[p // page, :, p % page] = x[p]
    table = torch.arange(5, dtype=torch.int32)[None]
    table[0, :first // page] = -1
    got = paged_attention(q, kp, vp, table, torch.tensor([start], dtype=torch.int32), window=window)
    for i in range(t):
        lo = max(0, start + i - window)
        for h in range(H):
            p = torch.softmax(K[lo:start + i + 1, h // 2].double() @ q[0, i, h].double() / math.sqrt(D), 0)
            assert torch.allclose(got[0, i, h].double(), p @ V[lo:start + i + 1, h // 2].double(), atol=1e-5)


def test_paged_decode_of_a_mixture_of_experts():
    """Ragged prompts and pausing rows: what stands behind a row's count changes no other token's experts."""
    from tests.test_serving_cpu import test_paged_decode_matches_full_forward
    test_paged_decode_matches_full_forward("moe")
