"""Serving operators where they can go wrong: precision of single probabilities, bad pages, NaN, launch forms of large calls.

Bounds are derived beside each test; u is the relative rounding of the output's type (2^-8 bf16, 2^-11 fp16).
"""
import math

import pytest
import torch

from tests.test_serving_gpu import DEV, U, make_cache

pytestmark = pytest.mark.gpu


def ints(*values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def pages_of(K, V, page, dtype):
    """Keys and values [n, D] of one row and head as pages in order, with their table."""
    n, D = K.shape
    P = -(-n // page)
    k, v = (torch.nn.functional.pad(x, (0, 0, 0, P * page - n)).view(P, 1, page, D).to(DEV, dtype) for x in (K, V))
    return k, v, torch.arange(P, device=DEV, dtype=torch.int32)[None]


@pytest.mark.parametrize("keys", [3, 40, 1001, 9000])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype,heads,kv_heads,t", [(torch.bfloat16, 10, 5, 1), (torch.float16, 16, 1, 1), (torch.bfloat16, 4, 2, 3)])
def test_attention_of_a_query_that_is_not_finite(keys, bad, dtype, heads, kv_heads, t):
    """Its scores are NaN or infinite whatever the keys are, so its output is NaN, in one piece or joined from many; the
    other queries' outputs stay what they are (up to roundings: probabilities to 2^-16, the output to u)."""
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(22)
    rows = [keys, keys, 17 + t]
    k, v, table = make_cache(rows, kv_heads, 64, 128, dtype)
    start = ints(*(n - t for n in rows))
    q = torch.randn(3, t, heads, 128, device=DEV).to(dtype)
    clean = paged_attention(q, k, v, table, start).float()
    q[0, t - 1, heads // 2, 5] = bad
    q[2, 0, 0, 127] = bad
    got = paged_attention(q, k, v, table, start).float()
    hit = torch.zeros(3, t, heads, dtype=torch.bool, device=DEV)
    hit[0, t - 1, heads // 2], hit[2, 0, 0] = True, True
    assert torch.isnan(got[hit]).all()
    top = v.float().nan_to_num(0.0).abs().max()
    assert ((got - clean)[~hit].abs() <= 1.02 * U[dtype] * clean[~hit].abs() + 2.0 ** -15 * top).all()


@pytest.mark.parametrize("dtype,D,H,Hk,page,t,window,rows,bad", [
    # bad: (row, page column, number in the table)
    (torch.bfloat16, 128, 10, 5, 64, 1, -1, [(1000, 1), (300, 1)], [(0, 7, -1), (0, 15, 1 << 30)]),
    (torch.float16, 64, 4, 4, 16, 1, -1, [(40, 1), (9, 1)], [(0, 0, -5)]),
    (torch.bfloat16, 128, 16, 1, 32, 5, 200, [(500, 5), (12, 3), (95, 5)], [(0, 12, -1), (0, 11, 99999), (2, 1, -1)]),
    (torch.float16, 128, 6, 2, 48, 33, -1, [(0, 33), (200, 20)], [(1, 2, -1)]),
    (torch.bfloat16, 64, 12, 3, 16, 1, -1, [(9000, 1)], [(0, j, -1) for j in range(100, 300)]),
    (torch.bfloat16, 128, 2, 1, 64, 1, -1, [(70, 1), (70, 1)], [(0, 0, -1), (0, 1, -1)]),   # nothing is left of row 0
])
def test_attention_leaves_out_what_has_no_page(dtype, D, H, Hk, page, t, window, rows, bad):
    """Keys whose page is not in the cache take no part; the others' softmax is theirs alone, and the error is reported.

    Bound: probabilities held to 2^-16 (and in fp16 to 2^-25 of the largest a key), of values weighed with them, and u of the
    output.
    """
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(23)
    k, v, table = make_cache([s + c for s, c in rows], Hk, page, D, dtype)
    q = (torch.randn(len(rows), t, H, D, device=DEV) * 1.2).to(dtype)
    missing = torch.zeros(len(rows), table.shape[1] * page, dtype=torch.bool, device=DEV)
    broken = table.clone()
    for b, column, number in bad:
        broken[b, column] = number
        missing[b, column * page:(column + 1) * page] = True
    check_errors()
    got = paged_attention(q, k, v, broken, ints(*(s for s, _ in rows)), ints(*(c for _, c in rows)), window=window)
    with pytest.raises(RuntimeError, match="page number"):
        check_errors()
    top = v.float().nan_to_num(0.0).abs().max().double()
    for b, (s, c) in enumerate(rows):
        for i in range(c):
            key = torch.arange(max(0, s + i - window) if window >= 0 else 0, s + i + 1, device=DEV)
            key = key[~missing[b, key]]
            if not len(key):
                assert (got[b, i] == 0).all()
                continue
            at = table[b].long()[key // page], slice(None), key % page
            K, V = k[at].double(), v[at].double()
            p = torch.softmax(torch.einsum("hgd,khd->hgk", q[b, i].double().view(Hk, H // Hk, D), K) * D ** -0.5, -1)
            ref, held = (torch.einsum("hgk,khd->hgd", p, x).reshape(H, D) for x in (V, V.abs()))
            slack = 2.0 ** -15 * held + (len(key) * 2.0 ** -25 * top if dtype == torch.float16 else 0)
            assert ((got[b, i].double() - ref).abs() <= 1.02 * U[dtype] * ref.abs() + slack).all(), (b, i)
        assert (got[b, c:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [0, 6, 10, 12, 14, 16])
@pytest.mark.parametrize("keys,B", [(32, 64), (700, 1), (5000, 300)])
def test_attention_beside_a_key_that_takes_nearly_all(dtype, gap, keys, B):
    """A first key with value zero whose score lies `gap` above the others': the output is made of small probabilities only.

    Scores are exact up to their rounding in powers of two, below 2^-20, and exp2 is good to 2^-22.  A probability is held to
    2^-16 of itself in bf16 and to 2^-22 in fp16, there with at most 2^-32 of the largest lost; sums of up to 5000 equal
    numbers in fp32 may drift by 2^-24 for each 16 of them, 2^-15.7.  In all 2^-14 of the output besides its rounding, and
    2^-32 of the value a key.
    """
    from nexttransformer_b200.ops.paged import paged_attention
    K, V = torch.zeros(keys, 64), torch.full((keys, 64), 1000.0)
    K[0, 0], V[0] = gap, 0
    V[1::2, 1] = -500.0
    k, v, table = pages_of(K, V, 16, dtype)
    q = torch.zeros(B, 1, 1, 64, device=DEV, dtype=dtype)
    q[..., 0] = 1
    got = paged_attention(q, k, v, table.expand(B, -1).contiguous(), torch.full((B,), keys - 1, device=DEV, dtype=torch.int32),
                          scale=1.0).double().cpu()[:, 0, 0]
    p = torch.softmax(k.reshape(-1, 64)[:keys, 0].double().cpu(), 0)
    values = v.reshape(-1, 64)[:keys].double().cpu()
    ref, held = p @ values, p @ values.abs()
    slack = 2.0 ** -14 * held + (keys * 2.0 ** -32 * 1000 * p[0] if dtype == torch.float16 else 0)
    assert ((got - ref).abs() <= 1.02 * U[dtype] * ref.abs() + slack).all(), ((got - ref).abs() / ref.abs()).max().item()



@pytest.mark.parametrize("op,name", [
    *(("append", n) for n in ("q", "k", "v", "k_pages", "v_pages", "cos", "sin", "ve", "ve_gate")),
    *(("attention", n) for n in ("q", "k_pages", "v_pages")),
    *(("delta", n) for n in ("q", "k", "v", "beta", "g", "state")),
    *(("logits", n) for n in ("logits", "repetition", "presence", "frequency", "bias")),
])
def test_no_gradient_is_dropped(op, name):
    """Whichever argument wants a gradient is refused while gradients are recorded, and welcome under no_grad."""
    from tests.test_serving_edges_cpu import _serving_calls
    call, args = _serving_calls(DEV, torch.bfloat16)[op]
    call(**args)
    args[name] = args[name].detach().clone().requires_grad_()
    with pytest.raises(RuntimeError, match="backward"):
        call(**args)
    with torch.no_grad():
        call(**args)


def test_check_errors_waits_for_other_streams():
    """Streams of their own do not wait for the default stream, on which the error words are read, nor it for them."""
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_attention
    k, v, table = make_cache([20], 2, 16, 64, torch.bfloat16, fill=0.0)
    q = torch.ones(1, 1, 4, 64, device=DEV, dtype=torch.bfloat16)
    start, bad = ints(3), torch.full_like(table, -1)
    paged_attention(q, k, v, table, start)
    check_errors()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        paged_attention(q, k, v, table, start)          # what a stream's first call sets up is not part of the wait
        side.synchronize()
        torch.cuda._sleep(200_000_000)                   # about a tenth of a second
        paged_attention(q, k, v, bad, start)
    with pytest.raises(RuntimeError, match="page number"):
        check_errors()


def small_model(**extra):
    from dataclasses import replace
    from nexttransformer_b200.models import build_model
    from nexttransformer_b200.models.config import candidate_config
    from tests.test_families_gpu import compute_dtype
    c = replace(candidate_config("dense"), layers=2, width=256, heads=2, kv_heads=1, vocab_size=512, sequence_len=256,
                mlp_width=1024, scale="custom", window_pattern="L", **extra)
    with compute_dtype(torch.bfloat16):
        return c, build_model(c, DEV, seed=0).eval()


def test_generate_batch_raises_for_what_the_kernels_recorded(monkeypatch):
    """A cache whose table loses a row's pages: the kernels leave them out, and the answers are not handed over."""
    from nexttransformer_b200.inference import PagedCache, generate_batch
    from nexttransformer_b200.ops._ext import check_errors
    c, m = small_model()
    check_errors()
    assert [len(a) for a in generate_batch(m, [[1, 2, 3], [4]], 3)] == [3, 3]
    reserve = PagedCache.reserve

    def forgetful(cache, counts):
        reserve(cache, counts)
        cache.table[1] = -1
    monkeypatch.setattr(PagedCache, "reserve", forgetful)
    with pytest.raises(RuntimeError, match="page number lies outside the cache .row 1."):
        generate_batch(m, [[1, 2, 3], [4]], 3)
    check_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 11])
def test_delta_recurrent_of_unaligned_views(dtype, T):
    """Heads that start on any element, as slices of wider projections do: the same bits as from copies."""
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    torch.manual_seed(24)
    B, H, D = 2, 3, 128
    q, k, v = (torch.randn(B, T, H, D + 5, device=DEV).to(dtype)[..., i:D + i] for i in (1, 2, 3))
    g = -torch.rand(B, T, H, D + 5, device=DEV)[..., 3:D + 3]
    beta = torch.rand(B, T, H, device=DEV)
    state = torch.randn(B, H, D, D, device=DEV) * .3
    copy = state.clone()
    got = delta_recurrent(q, k, v, state, beta, g, l2norm=True)
    assert torch.equal(got, delta_recurrent(*(x.contiguous() for x in (q, k, v)), copy, beta, g.contiguous(), l2norm=True))
    assert torch.equal(state, copy)
