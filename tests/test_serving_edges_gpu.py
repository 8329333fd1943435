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
    """Its scores are NaN, or infinite of both signs with these keys, so its output is NaN, in one piece or joined from many;
    the other queries' outputs stay what they are (up to roundings: probabilities to 2^-16, the output to u)."""
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


# ------------------------------------------------------------------------------------------ precision of the attention
def tight_attention(q, k, v, table, rows, window, some=None):
    """Asserts what the kernel claims: the output's rounding, and 2^-14 of the values weighed with their probabilities.

    A score is a sum of D products in fp32 on tensor cores, off by at most D / 16 + 1 roundings of 2^-23 of its largest partial
    sum, which is below 20 for these inputs: 2^-15.6 in powers of two.  A probability is held to 2^-16; exp2, totals and
    joins are good to 2^-19.
    """
    from nexttransformer_b200.ops.paged import paged_attention
    B, t, H, D = q.shape
    Hk, page = k.shape[1:3]
    got = paged_attention(q, k, v, table, ints(*(s for s, _ in rows)), ints(*(c for _, c in rows)), window=window)
    assert torch.isfinite(got.float()).all()
    for b in range(B) if some is None else some:
        s, c = rows[b]
        assert (got[b, c:] == 0).all()
        if not c:
            continue
        key = torch.arange(max(0, s - window) if window >= 0 else 0, s + c, device=DEV)
        at = table[b].long()[key // page], slice(None), key % page
        K, V = k[at].double(), v[at].double()
        for i0 in range(0, c, 64):
            n = min(64, c - i0)
            pos = torch.arange(s + i0, s + i0 + n, device=DEV)[:, None]
            seen = (key <= pos) & (key >= pos - window if window >= 0 else True)
            score = torch.einsum("ihgd,khd->hgik", q[b, i0:i0 + n].double().view(n, Hk, H // Hk, D), K) * D ** -0.5
            p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            ref, held = (torch.einsum("hgik,khd->ihgd", p, x).reshape(n, H, D) for x in (V, V.abs()))
            err = (got[b, i0:i0 + n].double() - ref).abs()
            assert (err <= 1.02 * U[got.dtype] * ref.abs() + 2.0 ** -14 * held + 2.0 ** -25).all(), (b, i0, (err / held).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,Hk,page,t,window,rows", [
    (128, 8, 2, 64, 1, -1, [(9000, 1)]),                                      # over many CTAs
    (128, 2, 1, 64, 1, 5000, [(30000, 1), (17, 1)]),
    (64, 16, 1, 128, 8, -1, [(9000, 8)]),
    (128, 10, 5, 64, 1, -1, [(0, 1), (1, 1), (15, 1), (16, 1), (63, 1), (64, 1), (1000, 1), (2500, 1), (8191, 1)]),
    (64, 12, 12, 16, 4, 1023, [(6000, 4), (1020, 4), (90, 3), (200, 0), (3000, 4)]),
    (128, 12, 3, 16, 5, -1, [(1200, 5), (77, 1), (640, 4), (4000, 5)]),
    (128, 16, 4, 64, 9, 100, [(3000, 9), (5, 9)]),
    (128, 16, 1, 64, 11, -1, [(40, 11), (3000, 2), (0, 11)]),
])
def test_attention_to_its_own_precision(dtype, D, H, Hk, page, t, window, rows):
    """A tile of 16 keys left out or counted twice among 9000 moves an output by several times this bound."""
    torch.manual_seed(25)
    k, v, table = make_cache([s + c for s, c in rows], Hk, page, D, dtype)
    tight_attention((torch.randn(len(rows), t, H, D, device=DEV) * 1.2).to(dtype), k, v, table, rows, window)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("keys,page,B,H,Hk,t,window", [
    (17, 16, 1, 1, 1, 1, -1), (1000, 64, 1, 4, 2, 1, -1), (8192, 64, 1, 1, 1, 1, -1), (8183, 48, 2, 2, 2, 1, -1),
    (40000, 128, 1, 2, 1, 1, -1), (3001, 16, 5, 16, 1, 2, 777), (513, 32, 2, 12, 3, 9, -1), (2000, 64, 40, 8, 8, 1, -1),
])
def test_attention_weighs_each_tile_once(dtype, D, keys, page, B, H, Hk, t, window):
    """Equal scores, and tile j of 16 keys has value 1 in channel j % D: an output channel is the share of its tiles' keys,
    off by the output's rounding and those of 1 / n and the joins, 2^-20."""
    from nexttransformer_b200.ops.paged import paged_attention
    channel = torch.arange(keys) // 16 % D
    g = torch.Generator().manual_seed(26)
    P = -(-keys // page)
    order = torch.randperm(P + 1, generator=g)[:P]
    V = torch.nn.functional.one_hot(channel, D).float()
    v = torch.full((P + 1, Hk, page, D), math.nan)
    for j in range(P):
        v[order[j], :, :min(page, keys - j * page)] = V[j * page:(j + 1) * page]
    v = v.to(DEV, dtype)
    k = torch.randn(v.shape, device=DEV).to(dtype).masked_fill(torch.isnan(v), math.nan)
    table = order.int().to(DEV)[None].expand(B, -1).contiguous()
    start = torch.full((B,), keys - t, device=DEV, dtype=torch.int32)
    got = paged_attention(torch.zeros(B, t, H, D, device=DEV, dtype=dtype), k, v, table, start, window=window).double().cpu()
    for i in range(t):
        seen = channel[max(0, keys - t + i - window) if window >= 0 else 0:keys - t + i + 1]
        ref = torch.bincount(seen, minlength=D).double() / len(seen)
        assert ((got[:, i] - ref).abs() <= (1.02 * U[dtype] + 2.0 ** -20) * ref).all(), i


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("heads", [1, 16])
def test_attention_difference_of_neighbouring_probabilities(dtype, D, heads):
    """Channel d sees key 2 d with value 1024 and key 2 d + 1 with value -1024, whose scores differ by about 2^-14: the output is
    the difference of two nearly equal probabilities, and shows how exactly each is held.

    The scores are below 2^-6 and exact, so the probabilities lie between 0.98 and 1 of the largest.  Two bf16 numbers hold such
    a one to 2^-18, two of fp16 to 2^-22; exp2 is good to 2^-22, and the products of the parts add two roundings of at most
    2^-23: together less than 2^-17 of p_j + p_{j+1}, besides the output's rounding.  One bf16 number alone is 2^-9 off.
    """
    from nexttransformer_b200.ops.paged import paged_attention
    g = torch.Generator().manual_seed(21)
    x = (torch.rand(D, generator=g) * .5 + .5).to(dtype).float()
    K, V = torch.zeros(2 * D, D), torch.zeros(2 * D, D)
    K[0::2, 0], K[1::2, 0] = x, x - 2.0 ** -8     # both types hold both
    V[0::2], V[1::2] = 1024 * torch.eye(D), -1024 * torch.eye(D)
    k, v, table = pages_of(K, V, 64, dtype)
    q = torch.zeros(1, 1, heads, D, device=DEV, dtype=dtype)
    q[..., 0] = 1
    got = paged_attention(q, k, v, table, ints(2 * D - 1), scale=2.0 ** -6).double().cpu()[0, 0]
    p = 1024 * torch.softmax(k.reshape(-1, D)[:2 * D, 0].double().cpu() / 64, 0)
    ref, held = p[0::2] - p[1::2], p[0::2] + p[1::2]
    assert (ref > 2.0 ** -14).all()   # a normal number in fp16
    assert ((got - ref).abs() <= 1.02 * U[dtype] * ref + 2.0 ** -17 * held).all(), ((got - ref).abs() / held).max().item()


# ------------------------------------------------------------------------------------------ forms of large calls
@pytest.mark.parametrize("dtype,D,H,Hk,page,B,t", [
    # enough heads and tokens that a thread takes five heads (blocks x groups of five heads at least twice the SMs)
    (torch.bfloat16, 128, 10, 5, 64, 3, 700), (torch.float16, 128, 10, 5, 16, 3, 700), (torch.bfloat16, 128, 16, 1, 32, 4, 333),
    (torch.float16, 128, 12, 12, 48, 2, 401), (torch.bfloat16, 64, 8, 2, 16, 5, 1000), (torch.float16, 64, 16, 1, 64, 3, 1111),
    (torch.bfloat16, 64, 12, 12, 128, 2, 777), (torch.float16, 128, 3, 1, 16, 6000, 1),
])
@pytest.mark.parametrize("norm,ve", [(True, True), (False, False), (True, False)])
def test_append_of_many_tokens(dtype, D, H, Hk, page, B, t, norm, ve):
    """Ragged prompts behind what rows hold already.  fp32 inside (1e-5 covers it), one rounding."""
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_append
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-B * t // (2048 // D)) * ((H + 2 * Hk + 4) // 5) >= 2 * sms
    torch.manual_seed(27)
    rows = [((b * 37) % 90, max(0, t - (b * 111) % (t + 1))) for b in range(B)]
    kp, vp, table = make_cache([s + c for s, c in rows], Hk, page, D, dtype, fill=7.0)
    before = kp.clone(), vp.clone()
    packed = torch.randn(B, t, H + 2 * Hk, D, device=DEV).to(dtype)
    q, k, v = packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]
    angle = torch.outer(torch.arange(2048, device=DEV), 1e5 ** (-torch.arange(0, D, 2, device=DEV) / D))
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    e = torch.randn(B, t, Hk, D, device=DEV).to(dtype) if ve else None
    gate = torch.randn(B, t, Hk, device=DEV).to(dtype) if ve else None
    start, count = (ints(*(r[i] for r in rows)) for i in (0, 1))
    got = paged_append(q, k, v, kp, vp, table, start, count, cos=cos, sin=sin, qk_scale=1.2 if norm else None, ve=e,
                       ve_gate=gate)
    check_errors()
    b, i = (torch.tensor(x, device=DEV) for x in zip(*((b, i) for b, (_, c) in enumerate(rows) for i in range(c))))
    pos = start.long()[b] + i
    c, sn = cos[pos].double()[:, None], sin[pos].double()[:, None]

    def turn(x):
        x1, x2 = x[b, i].double().chunk(2, -1)
        y = torch.cat((x1 * c + x2 * sn, x2 * c - x1 * sn), -1)
        return 1.2 * y / (y.pow(2).mean(-1, keepdim=True) + 2.0 ** -23).sqrt() if norm else y
    qr, kr, vr = torch.zeros(q.shape, dtype=torch.float64, device=DEV), before[0].double(), before[1].double()
    qr[b, i] = turn(q)
    at = table.long()[b, pos // page], slice(None), pos % page
    kr[at] = turn(k)
    vr[at] = v[b, i].double() + (3 * torch.sigmoid(gate[b, i].double())[..., None] * e[b, i].double() if ve else 0)
    for x, r in ((got, qr), (kp, kr), (vp, vr)):
        assert ((x.double() - r).abs() <= 1.02 * U[dtype] * r.abs() + 1e-5).all()
    written = torch.zeros(kp.shape[:3], dtype=torch.bool, device=DEV)
    written[at] = True
    for x, old in zip((kp, vp), before):
        assert torch.equal(x[~written], old[~written])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V,L,K,mask,pad", [
    # B x ceil(V / 8192) pieces: at least twice the SMs take 8192 entries each
    (101, 20000, 1500, 40, True, 48), (101, 20001, 1100, 33, True, 63), (300, 4097, 70, 300, False, 0), (150, 8193, 3000, 5, True, 3),
])
def test_adjust_logits_of_a_large_batch(dtype, B, V, L, K, mask, pad):
    from tests.test_serving_gpu import test_adjust_logits
    assert B * -(-V // 8192) >= 2 * torch.cuda.get_device_properties(0).multi_processor_count
    test_adjust_logits(dtype, B, V, L, K, mask, pad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,H,T", [(128, 30, 50), (64, 60, 21)])
def test_delta_recurrent_without_decay_at_32_columns(dtype, D, H, T):
    from tests.test_serving_gpu import test_delta_recurrent
    assert 6 * H * (D // 32) >= torch.cuda.get_device_properties(0).multi_processor_count
    test_delta_recurrent(dtype, "deltanet", D, H, T, [T, 3, T, 17, 0, T], [5, 4, 3, 2, 1, 0], True)


@pytest.mark.parametrize("dtype,H,Hk,B,t,window", [
    (torch.bfloat16, 16, 1, 3, 720, -1), (torch.float16, 16, 1, 3, 720, 100), (torch.bfloat16, 8, 2, 2100, 1, -1),
])
def test_attention_with_a_cta_for_each_row(dtype, H, Hk, B, t, window):
    """More rows, or row tiles of 16 queries, than the line of work holds (2048), heads of 128: prompts and large batches."""
    torch.manual_seed(28)
    assert B * -(-t * (H // Hk) // 16) > 2048
    rows = [((b * 53) % 200, max(1, t - b * 7)) if t > 1 else ((b * 7) % 90, 1) for b in range(B)]
    k, v, table = make_cache([s + c for s, c in rows], Hk, 16, 128, dtype)
    q = (torch.randn(B, t, H, 128, device=DEV) * 1.2).to(dtype)
    tight_attention(q, k, v, table, rows, window, list(range(0, B, 1 + B // 30)))


# ------------------------------------------------------------------------------------------ streams and graphs
def test_attention_on_three_streams_at_once():
    """Rows of which each takes many CTAs, on two streams and as a graph on a third, waiting for nothing but a common start:
    every result has the bits of the call alone."""
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(29)
    k, v, table = make_cache([4000, 3000, 5000], 1, 64, 128, torch.bfloat16)
    start = ints(3999, 2999, 4999)
    q = [torch.randn(3, 1, 8, 128, device=DEV).bfloat16() for _ in range(3)]
    alone = [paged_attention(x, k, v, table, start) for x in q]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [paged_attention(q[2], k, v, table, start) for _ in range(40)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(3):
        for x in held:
            x.zero_()
        got = [[], []]
        torch.cuda._sleep(20_000_000)      # all three queues fill meanwhile
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[2]):
            graph.replay()
        for _ in range(40):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    got[i].append(paged_attention(q[i], k, v, table, start))
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(x, alone[i]) for x in got[i])
        assert all(torch.equal(x, alone[2]) for x in held)


CAPTURE = """
import torch
from nexttransformer_b200.ops.paged import paged_attention
torch.manual_seed(30)
P = 64
k, v = (torch.randn(P, 1, 64, 128, device="cuda").bfloat16() for _ in range(2))
table = torch.arange(P, device="cuda", dtype=torch.int32)[None]
start = torch.tensor([P * 64 - 1], device="cuda", dtype=torch.int32)
q = torch.randn(1, 1, 4, 128, device="cuda").bfloat16()
torch.cuda.synchronize()
first = torch.cuda.CUDAGraph()
with torch.cuda.graph(first):               # no call came before: the graph clears counters of its own
    a = paged_attention(q, k, v, table, start)
first.replay()
alone = paged_attention(q, k, v, table, start)
assert torch.equal(a, alone)
many = torch.cuda.CUDAGraph()
with torch.cuda.graph(many):                # more calls than there are counters set aside for graphs
    held = [paged_attention(q, k, v, table, start) for _ in range(2100)]
side = torch.cuda.Stream()
for _ in range(2):
    for x in (a, *held):
        x.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        many.replay()
    first.replay()
    eager = [paged_attention(q, k, v, table, start) for _ in range(50)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, alone) for x in (a, *held, *eager))
print("fine")
"""


def test_attention_captured_without_counters_set_aside():
    """In a process of its own: a capture before any other call, and more captured calls than have counters set aside."""
    import subprocess
    import sys
    done = subprocess.run([sys.executable, "-c", CAPTURE], capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and done.stdout.split()[-1] == "fine", done.stderr[-2000:]


@pytest.mark.parametrize("T", [1, 4, 300])
def test_delta_recurrent_captured(T):
    """A graph keeps the early launch of the walk through the blocks (T = 4), and segments (T = 300 of 128 heads)."""
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    torch.manual_seed(31)
    B, H, D = 8, 16, 128
    q, k, v = (torch.randn(B, T, H, D, device=DEV).bfloat16() for _ in range(3))
    beta, g = torch.rand(B, T, H, device=DEV), -torch.rand(B, T, H, device=DEV)
    first = torch.randn(B, H, D, D, device=DEV) * .3
    alone = first.clone()
    want = [delta_recurrent(q, k, v, alone, beta, g, l2norm=True) for _ in range(3)]
    state = first.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [delta_recurrent(q, k, v, state, beta, g, l2norm=True) for _ in range(3)]
    for _ in range(2):
        state.copy_(first)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want)) and torch.equal(state, alone)
