"""The 8-bit cache, the experts of a few tokens and sampling on the GPU, against definitions in 64 bits.

u is half a unit in the last place (2^-8 bf16, 2^-11 fp16); every tolerance is derived beside its use.
"""
import math

import pytest
import torch

from tests.test_serving_gpu import U, oracle_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn


def make_cache8(rows, Hk, page, D, spare=2, seed=0, low=-9, high=-5):
    """8-bit pages in random order for rows of n tokens.  Behind a row's last token codes are NaN, and so are the scales of blocks
    without a token.  Also the numbers that the codes stand for."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in rows]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g).int()
    table = torch.full((len(rows), max(1, max(need))), -1, dtype=torch.int32)
    codes = [torch.full((P, Hk, page, D), math.nan).to(F8) for _ in "kv"]
    scales = [torch.full((P, Hk, page // 16), math.nan) for _ in "kv"]
    at = 0
    for b, n in enumerate(rows):
        table[b, :need[b]] = order[at:at + need[b]]
        for j in range(need[b]):
            m, p = min(page, n - j * page), order[at + j]
            for c, s in zip(codes, scales):
                c[p, :, :m] = (torch.randn(Hk, m, D, generator=g) * 80).clamp(-448, 448).to(F8)
                s[p, :, :-(-m // 16)] = torch.exp2(torch.randint(low, high, (Hk, -(-m // 16)), generator=g).float())
        at += need[b]
    codes, scales = [c.to(DEV) for c in codes], [s.to(DEV) for s in scales]
    return *codes, *scales, table.to(DEV)


def stands_for(codes, scale):
    return codes.double() * scale.double().repeat_interleave(16, 2)[..., None]


def check8(got, ref, v, keys, scores):
    """The output is rounded once (u |ref|).  Scores of size up to `scores` (their terms' sum) come from fp32 sums of D products, half a
    unit each: 2^-24 scores * 4 covers 128 terms' drift; a score's error moves an output by twice itself times max |v|.  Probabilities
    are two fp16 numbers (2^-22 of each) beside fp16 queries and one (2^-12) beside bf16 queries, and lose 2^-32 of the largest a key:
    their sum times |v| is at most max |v|, so that is what it moves an output by.  (A first build held two in both.)"""
    top = v.nan_to_num(0.0).abs().max().item()
    slack = top * (2 * scores * 2.0 ** -22 + (2.0 ** -20 if got.dtype == torch.float16 else 1.01 * 2.0 ** -12) + keys * 2.0 ** -32) + 1e-30
    err = (got.double() - ref).abs()
    assert torch.isfinite(got.float()).all()
    assert (err <= 1.02 * U[got.dtype] * ref.abs() + slack).all(), (err - U[got.dtype] * ref.abs()).max().item() / slack


CASES = [
    # dtype, D, H, Hk, page, t, window, (start, count) per row
    (torch.bfloat16, 128, 10, 5, 64, 1, -1, [(0, 1), (1, 1), (14, 1), (15, 1), (16, 1), (62, 1), (63, 1), (64, 1), (700, 1)]),
    (torch.float16, 128, 4, 4, 16, 1, -1, [(0, 1), (31, 1), (300, 1)]),
    (torch.bfloat16, 64, 16, 1, 48, 1, 37, [(0, 1), (36, 1), (37, 1), (38, 1), (53, 1), (400, 1)]),
    (torch.float16, 64, 12, 12, 16, 4, 20, [(0, 4), (0, 1), (13, 3), (90, 4), (200, 0)]),
    (torch.bfloat16, 128, 12, 3, 32, 5, 0, [(0, 5), (29, 5), (77, 2)]),
    (torch.bfloat16, 128, 40, 1, 64, 1, -1, [(0, 1), (130, 1)]),
    (torch.float16, 128, 6, 6, 128, 33, 50, [(0, 33), (64, 20), (7, 0)]),
    (torch.bfloat16, 64, 6, 2, 16, 1, -1, [(0, 0), (40, 0), (40, 1)]),
    (torch.bfloat16, 128, 8, 2, 64, 1, -1, [(9000, 1)]),
    (torch.float16, 64, 2, 1, 64, 1, 5000, [(30000, 1), (17, 1)]),
    (torch.bfloat16, 64, 4, 2, 16, 3, -1, [(b * 7 % 90, 3) for b in range(500)]),
]


@pytest.mark.parametrize("dtype,D,H,Hk,page,t,window,rows", CASES)
def test_attention_in_8_bits(dtype, D, H, Hk, page, t, window, rows):
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(1)
    k, v, ks, vs, table = make_cache8([s + c for s, c in rows], Hk, page, D)
    start, count = ([r[i] for r in rows] for i in (0, 1))
    q = (torch.randn(len(rows), t, H, D, device=DEV) * 1.2).to(dtype)
    args = (torch.tensor(start, device=DEV, dtype=torch.int32), torch.tensor(count, device=DEV, dtype=torch.int32))
    got = paged_attention(q, k, v, table, *args, window=window, k_scale=ks, v_scale=vs)
    K, V = stands_for(k, ks), stands_for(v, vs)
    # |q| |k| of D channels: 1.2 * 80 * 2^-6 at most, times D ** 0.5 for the scale
    check8(got, oracle_attention(q, K, V, table, start, count, window), V, max(s + c for s, c in rows), 1.5 * D ** 0.5)
    for b, c in enumerate(count):
        assert (got[b, c:] == 0).all()
    assert torch.equal(got, paged_attention(q, k, v, table, *args, window=window, k_scale=ks, v_scale=vs))
    check_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,t,keys", [(4, 1, 700), (16, 1, 3000), (2, 2, 40)])
def test_attention_in_8_bits_with_scales_far_apart(dtype, heads, t, keys):
    """Blocks' scales from 2^-20 to 2^6 (values) beside each other, scales that are no powers of two, queries of 1e-20 to 1e3."""
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(heads)
    k, v, ks, vs, table = make_cache8([keys, 5], 2, 16, 64, seed=3)
    vs = vs * torch.exp2(torch.randint(-11, 12, vs.shape, device=DEV).float()) * (1 + torch.rand(vs.shape, device=DEV))
    ks = ks * (1 + torch.rand(ks.shape, device=DEV))
    q = torch.randn(2, t, heads, 64, device=DEV)
    if dtype == torch.bfloat16:
        q[:, :, 0] *= 1e-20
    q[:, :, -1] *= 8
    q = q.to(dtype)
    start = [keys - t, 5 - t]
    got = paged_attention(q, k, v, table, torch.tensor(start, device=DEV, dtype=torch.int32), k_scale=ks, v_scale=vs)
    K, V = stands_for(k, ks), stands_for(v, vs)
    check8(got, oracle_attention(q, K, V, table, start, [t, t], -1), V, keys, 8 * 3 * 64 ** 0.5)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("keys", [3, 1001])
def test_attention_in_8_bits_of_a_query_that_is_not_finite(bad, dtype, keys):
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(keys)
    k, v, ks, vs, table = make_cache8([keys] * 3, 2, 16, 128)
    q = torch.randn(3, 1, 4, 128, device=DEV).to(dtype)
    start = torch.full((3,), keys - 1, device=DEV, dtype=torch.int32)
    clean = paged_attention(q, k, v, table, start, k_scale=ks, v_scale=vs)
    q[1, 0, 2, 77] = bad
    got = paged_attention(q, k, v, table, start, k_scale=ks, v_scale=vs)
    hit = torch.zeros(3, 1, 4, 128, dtype=torch.bool, device=DEV)
    hit[1, 0, 2] = True
    assert torch.equal(got[~hit], clean[~hit])
    # an infinite query has a score of +inf at some key (their signs differ), and so gives NaN
    signs = stands_for(k, ks)[table[1].long()][:, 1].reshape(-1, 128)[:keys, 77].sign() * (1 if bad != -math.inf else -1)
    if math.isnan(bad) or (signs > 0).any():
        assert got[hit].isnan().all()


def test_attention_in_8_bits_leaves_out_what_has_no_page():
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(5)
    k, v, ks, vs, table = make_cache8([100, 100], 2, 16, 64)
    q = torch.randn(2, 1, 4, 64, device=DEV).bfloat16()
    start = torch.tensor([99, 99], device=DEV, dtype=torch.int32)
    lost = table.clone()
    lost[0, 2] = k.shape[0] + 7
    lost[0, 4] = -1
    got = paged_attention(q, k, v, lost, start, k_scale=ks, v_scale=vs)
    with pytest.raises(RuntimeError, match="page number lies outside the cache .row 0"):
        check_errors()
    kept = torch.tensor([i for i in range(100) if i // 16 not in (2, 4)], device=DEV)
    at = table[0].long()[kept // 16], slice(None), kept % 16
    K, V = stands_for(k, ks)[at], stands_for(v, vs)[at]
    p = torch.softmax(torch.einsum("hgd,khd->hgk", q[0, 0].double().view(2, 2, 64), K) / 8, -1)
    ref = torch.einsum("hgk,khd->hgd", p, V).reshape(4, 64)
    check8(got[0, 0], ref, V, 100, 1.5 * 8)
    assert torch.equal(got[1], paged_attention(q, k, v, table, start, k_scale=ks, v_scale=vs)[1])


def test_8_bit_cache_behind_32_bits():
    """Pages whose offsets pass 2^32 bytes, written and read."""
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    P, Hk, page, D = 70000, 4, 128, 128
    k = torch.zeros(P, Hk, page, D, device=DEV, dtype=torch.uint8).view(F8)
    v = torch.zeros(P, Hk, page, D, device=DEV, dtype=torch.uint8).view(F8)
    assert k.numel() > 2 ** 32
    ks, vs = torch.zeros(P, Hk, page // 16, device=DEV), torch.zeros(P, Hk, page // 16, device=DEV)
    torch.manual_seed(0)
    x = torch.randn(1, 20, 8 + 2 * Hk, D, device=DEV).bfloat16()
    table = torch.tensor([[P - 1]], device=DEV, dtype=torch.int32)
    zero = torch.zeros(1, device=DEV, dtype=torch.int32)
    cos, sin = torch.ones(64, D // 2, device=DEV).bfloat16(), torch.zeros(64, D // 2, device=DEV).bfloat16()
    args = dict(cos=cos, sin=sin, k_scale=ks, v_scale=vs)
    q = paged_append(x[:, :, :8], x[:, :, 8:12], x[:, :, 12:], k, v, table, zero, **args)
    got = paged_attention(q, k, v, table, zero, k_scale=ks, v_scale=vs)
    check_errors()
    K, V = stands_for(k[-1:], ks[-1:]), stands_for(v[-1:], vs[-1:])
    assert ((K[0, :, :20].transpose(0, 1) - x[0, :, 8:12].double()).abs() <= 2.0 ** -4 * x[0, :, 8:12].double().abs() + 2.0 ** -10 * ks.max()).all()
    check8(got, oracle_attention(q, K, V, table * 0, [0], [20], -1), V, 20, 1.5 * D ** 0.5)


# ------------------------------------------------------------------------------------------ append
def rule(top):
    return 2.0 ** max(-100, min(120, math.ceil(math.log2(top / 448)))) if top > 0 else 2.0 ** -100


APPENDS = [
    # dtype, D, H, Hk, page, t, norm, ve, (start, count) per row
    (torch.bfloat16, 128, 10, 5, 64, 1, True, True, [(0, 1), (1, 1), (15, 1), (16, 1), (63, 1), (64, 1), (700, 0), (701, 1)]),
    (torch.float16, 64, 12, 12, 16, 1, False, False, [(3, 1), (31, 1), (300, 1)]),
    (torch.bfloat16, 64, 6, 2, 48, 5, True, False, [(0, 5), (13, 5), (44, 3), (47, 5), (90, 0)]),
    (torch.float16, 128, 4, 1, 16, 40, True, True, [(0, 40), (7, 33), (16, 1), (31, 18)]),
    (torch.bfloat16, 128, 16, 4, 128, 17, False, True, [(0, 17), (120, 17), (5, 11), (5, 12)]),
    (torch.bfloat16, 128, 7, 7, 32, 700, True, False, [(0, 700), (9, 691), (3, 90), (20, 1), (16, 512), (1, 16), (2, 600), (40, 699)]),  # many tokens
]


@pytest.mark.parametrize("dtype,D,H,Hk,page,t,norm,ve,rows", APPENDS)
def test_append_in_8_bits(dtype, D, H, Hk, page, t, norm, ve, rows):
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_append
    torch.manual_seed(2)
    B = len(rows)
    k, v, ks, vs, table = make_cache8([s + c for s, c in rows], Hk, page, D, low=-14, high=-3)
    old = [x.clone() for x in (k, v, ks, vs)]
    packed = torch.randn(B, t, H + 2 * Hk, D, device=DEV)
    packed *= torch.exp2(torch.randint(-3, 4, (B, t, 1, 1), device=DEV).float())
    packed = packed.to(dtype)
    q, kin, vin = packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]
    angle = torch.outer(torch.arange(1500, device=DEV), 1e4 ** (-torch.arange(0, D, 2, device=DEV) / D))
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    extra = torch.randn(B, t, Hk, D, device=DEV).to(dtype) if ve else None
    gate = torch.randn(B, t, Hk, device=DEV).to(dtype) if ve else None
    start, count = (torch.tensor([r[i] for r in rows], device=DEV, dtype=torch.int32) for i in (0, 1))
    out = paged_append(q, kin, vin, k, v, table, start, count, cos=cos, sin=sin, qk_scale=1.2 if norm else None, ve=extra, ve_gate=gate,
                       k_scale=ks, v_scale=vs)
    check_errors()
    for b, (s, n) in enumerate(rows):
        assert (out[b, n:] == 0).all()
        if not n:
            continue
        at = torch.arange(s, s + n, device=DEV)
        c, si = cos[at].double()[:, None], sin[at].double()[:, None]

        def turned(x):
            x, y = x.double().chunk(2, -1)
            z = torch.cat((x * c + y * si, y * c - x * si), -1)
            return 1.2 * z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 2.0 ** -23) if norm else z
        ref = turned(q[b, :n])
        # rounded once; rotation and norm in fp32: a dozen roundings of 2^-24 of the head's largest
        assert ((out[b, :n].double() - ref).abs() <= 1.02 * U[dtype] * ref.abs() + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True)).all()
        new_v = vin[b, :n].double()
        if ve:
            new_v = new_v + 3 * torch.sigmoid(gate[b, :n].double())[..., None] * extra[b, :n].double()
        for new, codes, scale, before, scale_before in ((turned(kin[b, :n]), k, ks, old[0], old[2]), (new_v, v, vs, old[1], old[3])):
            for p0 in range(s // 16 * 16, s + n, 16):
                page_no, slot = int(table[b, p0 // page]), p0 % page
                lo, hi = max(p0, s) - s, min(p0 + 16, s + n) - s
                x = new[lo:hi].transpose(0, 1)                       # [Hk, tokens, D]
                got_s = scale[page_no, :, slot // 16].double()
                for h in range(Hk):
                    top = x[h].abs().max().item()
                    held = scale_before[page_no, h, slot // 16].item() if p0 < s else 0.0
                    # near a power of two the fp32 maximum may fall to its other side
                    assert got_s[h].item() in [max(held, rule(top * f)) for f in (1 - 2.0 ** -20, 1, 1 + 2.0 ** -20)]
                f = got_s[:, None, None]
                first = max(p0, s) - p0 + slot
                step = torch.exp2(torch.floor(torch.log2((x / f).abs().clamp(min=2.0 ** -6))) - 3) * f
                off = (codes[page_no, :, first:first + hi - lo].double() * f - x).abs()
                # half a step, and fp32's own error before it
                assert (off <= 0.5 * step + 2.0 ** -20 * x.abs().amax(-1, keepdim=True)).all()
                if p0 < s:   # the block's earlier codes stand for what they stood for, but for one more rounding where the scale grew
                    e = slice(slot, first)
                    was = before[page_no, :, e].double() * scale_before[page_no, :, slot // 16].double()[:, None, None]
                    now = codes[page_no, :, e].double() * f
                    assert ((now - was).abs() <= 2.0 ** -10 * f * (f > scale_before[page_no, :, slot // 16].double()[:, None, None])).all()
                e = slice(first + hi - lo, slot + 16)                # behind the new tokens nothing is touched
                assert torch.equal(codes[page_no, :, e].view(torch.uint8), before[page_no, :, e].view(torch.uint8))
    # rows without new tokens and spare pages as they were
    used = {int(table[b, p // page]) for b, (s, n) in enumerate(rows) for p in range(s, s + n)}
    rest = torch.tensor([p for p in range(k.shape[0]) if p not in used], device=DEV)
    for x, y in zip((k, v), old):
        assert torch.equal(x.view(torch.uint8)[rest], y.view(torch.uint8)[rest])
    for x, y in zip((ks, vs), old[2:]):
        assert torch.equal(x.view(torch.int32)[rest], y.view(torch.int32)[rest])


@pytest.mark.parametrize("t", [1, 6])
def test_append_in_8_bits_layouts_and_what_is_not_finite(t):
    """One layer of a token-major cache, scales in a wider tensor, another stream; NaN and infinities become NaN and set no scale."""
    from nexttransformer_b200.ops.paged import paged_append
    torch.manual_seed(3)
    whole = torch.zeros(2, 6, 16, 2, 128, device=DEV).to(F8)        # [kv, page, token, head, channel]
    k, v = whole[0].transpose(1, 2), whole[1].transpose(1, 2)
    scales = torch.zeros(6, 2, 1, 3, device=DEV)
    ks, vs = scales[..., 0], scales[..., 2]
    x = torch.randn(2, t, 8, 128, device=DEV).half()
    x[1, 0, 6, :2] = torch.tensor([math.inf, math.nan])
    x[1, t - 1, 7, 5] = 60000.0
    table = torch.tensor([[3], [5]], device=DEV, dtype=torch.int32)
    start = torch.tensor([0, 2], device=DEV, dtype=torch.int32)
    cos, sin = torch.ones(20, 64, device=DEV).half(), torch.zeros(20, 64, device=DEV).half()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = paged_append(x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], k, v, table, start, cos=cos, sin=sin, k_scale=ks, v_scale=vs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q, x[:, :, :4])
    for b in range(2):
        for codes, scale, new in ((k, ks, x[b, :, 4:6]), (v, vs, x[b, :, 6:])):
            s = scale[int(table[b, 0]), :, 0].double()
            s0 = int(start[b])
            got = codes[int(table[b, 0]), :, s0:s0 + t].double() * s[:, None, None]
            ref = new.double().transpose(0, 1)
            assert torch.equal(got.isnan(), ~ref.isfinite())
            fine = ref.isfinite()
            top = torch.where(fine, ref.abs(), 0.0).amax((1, 2))
            assert s.tolist() == [rule(a) for a in top.tolist()]
            step = torch.exp2(torch.floor(torch.log2((ref / s[:, None, None]).abs().clamp(2.0 ** -6, 500))) - 3) * s[:, None, None]
            assert ((got - ref).abs() <= 0.5 * step)[fine].all()
    assert (whole[:, [0, 1, 2, 4]].float() == 0).all() and (scales[..., 1] == 0).all()


def test_8_bit_refusals_and_device_checks():
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    k, v, ks, vs, table = make_cache8([20], 2, 16, 64)
    q = torch.randn(1, 1, 4, 64, device=DEV).bfloat16()
    start = torch.tensor([20], device=DEV, dtype=torch.int32)
    good = dict(q=q, k_pages=k, v_pages=v, table=table, start=start, k_scale=ks, v_scale=vs)
    for change, match in ((dict(k_scale=None), "k_scale and v_scale"), (dict(k_pages=k.float().bfloat16(), v_pages=v.float().bfloat16()), "k_scale and v_scale"),
                          (dict(v_pages=v.float().bfloat16()), "float8_e4m3fn"), (dict(k_scale=ks.half()), "k_scale"), (dict(k_scale=ks[:, :1]), "k_scale"),
                          (dict(k_scale=ks.cpu()), "k_scale"), (dict(q=q.float()), "bf16 or fp16"),
                          (dict(k_pages=k.view(torch.uint8).view(torch.float8_e5m2), v_pages=v.view(torch.uint8).view(torch.float8_e5m2)), "float8_e4m3fn")):
        with pytest.raises(RuntimeError, match=match):
            paged_attention(**dict(good, **change))
    cos, sin = torch.ones(21, 32, device=DEV).bfloat16(), torch.zeros(21, 32, device=DEV).bfloat16()
    before = [x.clone() for x in (k, v, ks, vs)]

    def append(t, tab, at, match):
        x = torch.randn(1, t, 8, 64, device=DEV).bfloat16()
        paged_append(x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], k, v, tab, torch.tensor([at], device=DEV, dtype=torch.int32), cos=cos, sin=sin,
                     k_scale=ks, v_scale=vs)
        with pytest.raises(RuntimeError, match=match):
            check_errors()
    for t in (1, 2):
        append(t, torch.tensor([[-1, k.shape[0]]], device=DEV, dtype=torch.int32), 15 if t == 2 else 3, "outside the cache")
        append(t, table[:, :1].contiguous(), 16, "behind the row's page table")
        append(t, table, 21, "behind the rotary table")
    for x, y in zip((k, v, ks, vs), before):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    x = torch.randn(1, 1, 8, 64, device=DEV).bfloat16()
    with pytest.raises(RuntimeError, match="share a scale"):
        paged_append(x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], k, v, table, start, cos=cos, sin=sin, k_scale=ks, v_scale=vs[:1].expand_as(vs))
    with pytest.raises(RuntimeError, match="no backward"):
        paged_attention(**dict(good, k_scale=ks.clone().requires_grad_()))


# ------------------------------------------------------------------------------------------ sampling
def both(logits, u, **kw):
    """The kernel's tokens have to be the 64-bit form's, logprobs to fp32 (a share's own rounding moves its log by 2^-24)."""
    from nexttransformer_b200.ops.sampling import sample_logits
    got, logprob = sample_logits(logits, u, **kw)
    ref, its = sample_logits(logits.cpu(), u.cpu(), **{k: v.cpu() if torch.is_tensor(v) else v for k, v in kw.items()})
    assert got.dtype == torch.long and torch.equal(got.cpu(), ref)
    its = its.double()
    close = (logprob.cpu().double() - its).abs() <= 2.0 ** -22 * its.abs() + 2.0 ** -23
    assert (close | (logprob.cpu() == its) | (its.isnan() & logprob.cpu().isnan())).all()
    again = sample_logits(logits, u, **kw)
    assert torch.equal(again[0], got) and torch.equal(again[1].view(torch.int32), logprob.view(torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 33, 4097, 32768, 50257, 131072, 524288])
def test_sampling(V, dtype):
    torch.manual_seed(V)
    B = 5
    x, u = (torch.randn(B, V, device=DEV) * 3).to(dtype), torch.rand(B, device=DEV)
    rows = dict(top_k=torch.tensor([1, 2, 0, 900, V], device=DEV, dtype=torch.int32), top_p=torch.tensor([0.5, 0.0, 1.0, 0.3, 0.999], device=DEV),
                min_p=0.01, temperature=torch.tensor([0.7, 1.0, 0.0, 2.0, 0.3], device=DEV))
    for kw in (dict(), dict(top_k=17), dict(top_p=0.9), dict(top_p=0.99, temperature=2.0), dict(min_p=0.05), rows,
               dict(top_k=max(1, V // 2), top_p=0.5, temperature=1e30), dict(top_p=0.5, temperature=1e-30), dict(top_p=math.nan, min_p=math.nan)):
        both(x, u, **kw)
    both(x, torch.tensor([0.0, 1.0, -3.0, math.nan, 0.99999994], device=DEV), top_p=0.95)


@pytest.mark.parametrize("V", [2, 1000, 32769, 300001])
def test_sampling_of_equal_and_odd_logits(V):
    torch.manual_seed(V)
    B = 5
    u = torch.rand(B, device=DEV)
    equal = torch.zeros(B, V, device=DEV)
    near = 5 + torch.randint(0, 3, (B, V), device=DEV).float() * 2.0 ** -20
    holes = torch.where(torch.rand(B, V, device=DEV) < 0.5, torch.randn(B, V, device=DEV), -math.inf)
    holes[1] = -math.inf
    holes[2, -1] = math.nan
    holes[3, V // 2] = holes[3, V - 1] = math.inf
    holes[4, 0] = -0.0
    for x in (equal, near, holes, torch.cat((equal[:, :-1], equal[:, :1] + 1), 1)):
        for kw in (dict(), dict(top_k=max(1, V // 3)), dict(top_p=0.37), dict(top_k=max(1, V // 2), top_p=0.37), dict(min_p=5.0),
                   dict(temperature=math.inf, top_p=0.5), dict(temperature=0.0)):
            both(x, u, **kw)


def test_sampling_layouts_streams_and_capture():
    from nexttransformer_b200.ops.sampling import sample_logits
    torch.manual_seed(9)
    wide = torch.randn(300, 1001, device=DEV)
    both(wide[:, 1:1000], torch.rand(300, device=DEV), top_p=0.8)            # rows on any element
    both(wide.bfloat16()[::2, :1000], torch.rand(150, device=DEV), top_k=5)
    x, u, out = torch.randn(7, 40000, device=DEV), torch.rand(7, device=DEV), []
    ref = sample_logits(x, u, top_p=0.9, top_k=100)
    side = [torch.cuda.Stream() for _ in range(3)]
    for s in side:                                                           # beside each other
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out.append([sample_logits(x, u, top_p=0.9, top_k=100) for _ in range(5)])
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, ref[0]) and torch.equal(b, ref[1]) for o in out for a, b in o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, _ = sample_logits(x, u, top_p=0.9, top_k=100)
    for seed in range(3):
        torch.manual_seed(seed)
        x.normal_()
        u.uniform_()
        graph.replay()
        assert torch.equal(tokens, sample_logits(x, u, top_p=0.9, top_k=100)[0])
    assert sample_logits(x[:0], u[:0])[0].shape == (0,)


def test_sampling_refusals():
    from nexttransformer_b200.ops.sampling import sample_logits
    x, u = torch.randn(3, 64, device=DEV), torch.rand(3, device=DEV)
    for args, kw, match in (((x[0], u), {}, "B, V"), ((x.t(), u), {}, "B, V"), ((x.double(), u), {}, "bf16, fp16 or fp32"), ((x, u[:2]), {}, "uniform"),
                            ((x, u.cpu()), {}, "uniform"), ((x, u), dict(top_k=u), "top_k"), ((x, u), dict(top_p=u[:2]), "top_p"),
                            ((x, u), dict(temperature=u.double()), "temperature"), ((torch.empty(1, 524289, device=DEV), u[:1]), {}, "524288"),
                            ((x[:, :0], u), {}, "vocabularies")):
        with pytest.raises(RuntimeError, match=match):
            sample_logits(*args, **kw)
    with pytest.raises(RuntimeError, match="no backward"):
        sample_logits(x.requires_grad_(), u)


# ------------------------------------------------------------------------------------------ experts
def experts(x, router, w_fc, w_proj, k, bias=None, shared_fc=None, shared_proj=None):
    """The definition in 64 bits, and the sum of the magnitudes of the last products."""
    x = x.double()
    p = torch.softmax(x @ router.double().T, -1)
    score = p + (0 if bias is None else bias.double())
    best, choice = torch.sort(score, dim=-1, descending=True, stable=True)
    if k < best.shape[1]:  # no token's choice hangs on fp32's last digits (or they are equal, and the lower wins)
        gap = best[:, k - 1] - best[:, k]
        assert ((gap > 1e-6) | (gap == 0) | gap.isnan()).all()
    choice = choice[:, :k]
    share = p.gather(1, choice)
    share = share / share.sum(-1, keepdim=True)
    y, size = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[0]):
        for e, c in zip(choice[t].tolist(), share[t]):
            h = c * torch.relu(w_fc[e].double() @ x[t]) ** 2
            y[t] += w_proj[e].double() @ h
            size[t] += w_proj[e].double().abs() @ h
        if shared_fc is not None:
            h = torch.relu(shared_fc.double() @ x[t]) ** 2
            y[t] += shared_proj.double() @ h
            size[t] += shared_proj.double().abs() @ h
    return y, size


def make_experts(T, d, F, E, shared, dtype, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, s=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEV) * s).to(dtype)
    a = dict(x=normal(T, d, s=scale, dtype=dtype), router=normal(E, d, s=d ** -0.5 / scale), w_fc=normal(E, F, d, s=d ** -0.5, dtype=dtype),
             w_proj=normal(E, d, F, s=F ** -0.5, dtype=dtype), bias=normal(E, s=2e-3))
    if shared:
        a.update(shared_fc=normal(shared, d, s=d ** -0.5, dtype=dtype), shared_proj=normal(d, shared, s=shared ** -0.5, dtype=dtype))
    return a


def check_experts(got, ref, size, dtype, steps):
    """The output is rounded once, and a hidden value is held as two numbers, 2^-16 of it in bf16 and 2^-22 in fp16.  Sums on the matrix
    units are chains of 16 products a step, each of which may cut its fp32 partial sum, by 2^-23 of it: steps * 2^-23 for a chain.
    In a hidden value (a chain of d / 16) the square doubles that, and partial sums are about as large as the values' spread, whose
    product with |v| is up to twice v^2 on average: four times.  `steps`: d / 4 for these, and the length of the outer chain."""
    slack = ((2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -22) + steps * 2.0 ** -23) * size + 1e-30
    if dtype == torch.float16:
        slack = slack + 2.0 ** -24  # its smallest step
    assert ((got.double() - ref).abs() <= 1.02 * U[dtype] * ref.abs() + slack).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,d,F,E,k,shared", [
    (1, 256, 128, 8, 2, 128), (1, 8, 8, 1, 1, 0), (2, 2048, 264, 64, 8, 264), (3, 72, 200, 5, 5, 8), (8, 640, 136, 33, 4, 0),
    (9, 640, 136, 32, 4, 136), (17, 128, 64, 4, 1, 64), (33, 136, 72, 3, 2, 0), (64, 320, 80, 256, 8, 80), (64, 64, 24, 2, 2, 4000),
    (5, 8192, 16, 512, 16, 0), (20, 5888, 24, 6, 2, 8), (31, 5896, 8, 6, 2, 0), (64, 6144, 16, 5, 1, 0), (64, 8192, 8, 300, 2, 8), (64, 1280, 320, 4, 2, 320), (12, 512, 1024, 16, 16, 1024)])
def test_experts_of_a_few_tokens(T, d, F, E, k, shared, dtype):
    from nexttransformer_b200.ops.moe import moe_tokens
    a = make_experts(T, d, F, E, shared, dtype, seed=T * 1000 + d)
    got = moe_tokens(top_k=k, **a)
    ref, size = experts(a["x"], a["router"], a["w_fc"], a["w_proj"], k, a["bias"], a.get("shared_fc"), a.get("shared_proj"))
    check_experts(got, ref, size, dtype, d / 4 + (k * F + shared) / 16)
    assert torch.equal(got, moe_tokens(top_k=k, **a))


def test_experts_large_small_and_odd_tokens():
    """fp16 hidden values beyond 65504; rows far apart; a token with a NaN or an infinity leaves the others alone; equal routers."""
    from nexttransformer_b200.ops.moe import moe_tokens
    a = make_experts(4, 128, 64, 8, 64, torch.float16, seed=1)
    a["x"] = (a["x"].float() * 300).half()
    a["router"] /= 300
    for n in ("w_proj", "shared_proj"):
        a[n] = a[n] * 2.0 ** -10
    ref, size = experts(a["x"], a["router"], a["w_fc"], a["w_proj"], 2, a["bias"], a["shared_fc"], a["shared_proj"])
    assert (torch.relu(a["x"].double() @ a["shared_fc"].double().T) ** 2).max() > 65504
    got = moe_tokens(top_k=2, **a)
    check_experts(got, ref, size, torch.float16, 32 + 12)
    a = make_experts(20, 256, 64, 16, 64, torch.bfloat16, seed=2)
    clean = moe_tokens(top_k=4, **a)
    a["x"] = torch.nn.functional.pad(a["x"], (0, 40))[:, :256]           # rows 296 elements apart
    assert torch.equal(moe_tokens(top_k=4, **a), clean)
    a["x"][3, 7], a["x"][11, 0] = math.nan, math.inf
    got = moe_tokens(top_k=4, **a)
    keep = [t for t in range(20) if t not in (3, 11)]
    assert got[3].isnan().all() and not got[11].isfinite().any() and torch.equal(got[keep], clean[keep])
    a = make_experts(6, 64, 32, 40, 0, torch.bfloat16, seed=3)
    a["router"].zero_()
    a.pop("bias")
    ref, size = experts(a["x"], a["router"], a["w_fc"], a["w_proj"], 3)   # experts 0, 1 and 2, a third each
    check_experts(moe_tokens(top_k=3, **a), ref, size, torch.bfloat16, 16 + 6)
    a["x"].zero_()
    assert (moe_tokens(top_k=3, **a) == 0).all()
    assert moe_tokens(a["x"][:0], a["router"], a["w_fc"], a["w_proj"], 3).shape == (0, 64)


def test_experts_behind_32_bits():
    """The last expert's weights lie behind 2^32 bytes (2^31 elements)."""
    from nexttransformer_b200.ops.moe import moe_tokens
    E, F, d = 260, 2048, 4096
    w_fc, w_proj = (torch.empty(*s, device=DEV, dtype=torch.bfloat16) for s in ((E, F, d), (E, d, F)))
    assert w_fc.numel() > 2 ** 31
    torch.manual_seed(4)
    w_fc[-1], w_proj[-1] = torch.randn(F, d, device=DEV) * d ** -0.5, torch.randn(d, F, device=DEV) * F ** -0.5
    x, bias = torch.randn(3, d, device=DEV).bfloat16(), torch.zeros(E, device=DEV)
    bias[-1] = 10.0
    got = moe_tokens(x, torch.zeros(E, d, device=DEV), w_fc, w_proj, 1, bias=bias)
    ref, size = experts(x, torch.zeros(1, d, device=DEV), w_fc[-1:], w_proj[-1:], 1)
    check_experts(got, ref, size, torch.bfloat16, 1024 + 128)


def test_experts_on_streams_and_captured():
    from nexttransformer_b200.ops.moe import moe_tokens
    sets = [make_experts(T, 256, 128, 32, 128, torch.bfloat16, seed=T) for T in (1, 9, 40)]
    refs = [moe_tokens(top_k=4, **a) for a in sets]
    streams, out = [torch.cuda.Stream() for _ in sets], []
    for s, a in zip(streams, sets):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out.append([moe_tokens(top_k=4, **a) for _ in range(8)])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(y, ref) for ys, ref in zip(out, refs) for y in ys)
    graphs = []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h = moe_tokens(top_k=4, **a)
            y = moe_tokens(h, *(a[n] for n in ("router", "w_fc", "w_proj")), 4)
        graphs.append((g, y))
    for (g, y), a, ref in zip(graphs, sets, refs):
        a["x"].mul_(1)  # the inputs are the graph's own
        g.replay()
    for (g, y), a, ref in zip(graphs, sets, refs):
        assert torch.equal(y, moe_tokens(ref, a["router"], a["w_fc"], a["w_proj"], 4))


def test_experts_refusals():
    from nexttransformer_b200.ops.moe import moe_tokens
    a = make_experts(4, 64, 32, 8, 32, torch.bfloat16)
    for change, match in ((dict(x=torch.zeros(65, 64, device=DEV).bfloat16()), "64 tokens"), (dict(x=a["x"].float()), "bf16 or fp16"),
                          (dict(x=a["x"][:, :60]), "multiple of 8"), (dict(x=a["x"].half()), "w_fc"), (dict(router=a["router"].bfloat16()), "router"),
                          (dict(router=a["router"].cpu()), "router"), (dict(top_k=9), "top_k"), (dict(top_k=0), "top_k"),
                          (dict(w_fc=a["w_fc"].transpose(1, 2)), "contiguous"), (dict(w_proj=a["w_proj"][:7]), "w_fc"),
                          (dict(shared_proj=None), "go together"), (dict(bias=a["bias"].half()), "bias"), (dict(bias=a["bias"][:4]), "bias"),
                          (dict(w_fc=a["w_fc"][:, :12].contiguous(), w_proj=a["w_proj"][:, :, :12].contiguous()), "multiple of 8")):
        with pytest.raises(RuntimeError, match=match):
            moe_tokens(**dict(dict(a, top_k=2), **change))
    with pytest.raises(RuntimeError, match="no backward"):
        moe_tokens(**dict(a, top_k=2, w_fc=a["w_fc"].clone().requires_grad_()))


# ------------------------------------------------------------------------------------------ together
def test_a_decoding_step_of_all_four():
    """Prompt and three steps through the 8-bit cache, the experts and the sampler, each against its definition on the inputs it got."""
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.moe import moe_tokens
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    torch.manual_seed(11)
    B, H, Hk, D, page, V = 6, 8, 2, 64, 32, 5000
    d = H * D
    dtype = torch.bfloat16
    w = make_experts(B, d, 128, 16, 128, dtype, seed=5)
    w.pop("x")
    proj = (torch.randn((H + 2 * Hk) * D, d, device=DEV) * d ** -0.5).to(dtype)
    head = (torch.randn(V, d, device=DEV) * d ** -0.5).to(dtype)
    k, v = (torch.zeros(2 * B, Hk, page, D, device=DEV).to(F8) for _ in "kv")
    ks, vs = (torch.zeros(2 * B, Hk, page // 16, device=DEV) for _ in "kv")
    table = torch.randperm(2 * B, device=DEV).int().view(B, 2)
    angle = torch.outer(torch.arange(64, device=DEV), 1e4 ** (-torch.arange(0, D, 2, device=DEV) / D))
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    lengths = [20, 3, 16, 1, 30, 9]
    start, count = torch.zeros(B, device=DEV, dtype=torch.int32), torch.tensor(lengths, device=DEV, dtype=torch.int32)
    x = torch.randn(B, 30, d, device=DEV).to(dtype)
    at = [0] * B
    for step in range(4):
        t = x.shape[1]
        qkv = (x @ proj.T).view(B, t, H + 2 * Hk, D)
        q = paged_append(qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:], k, v, table, start, count, cos=cos, sin=sin, qk_scale=1.2,
                         k_scale=ks, v_scale=vs)
        y = paged_attention(q, k, v, table, start, count, k_scale=ks, v_scale=vs)
        K, V_ = stands_for(k, ks), stands_for(v, vs)
        new = lengths if step == 0 else [1] * B
        check8(y, oracle_attention(q, K, V_, table, at, new, -1), V_, 40, 1.2 * 1.2 * D ** 0.5)
        last = torch.tensor([n - 1 for n in new], device=DEV)
        rows = y.view(B, t, d)[torch.arange(B, device=DEV), last]
        z = moe_tokens(rows, w["router"], w["w_fc"], w["w_proj"], 4, bias=w["bias"], shared_fc=w["shared_fc"], shared_proj=w["shared_proj"])
        ref, size = experts(rows, w["router"], w["w_fc"], w["w_proj"], 4, w["bias"], w["shared_fc"], w["shared_proj"])
        check_experts(z, ref, size, dtype, d / 4 + 40)
        both(z @ head.T, torch.rand(B, device=DEV), top_p=0.9, top_k=50, temperature=0.8)
        at = [a + n for a, n in zip(at, new)]
        start, count = start + count, torch.ones_like(count)
        x = torch.randn(B, 1, d, device=DEV).to(dtype)
    check_errors()


def test_generation_with_all_four():
    """A mixture-of-experts model in bf16: its layer on laid-out experts against the grouped products of its forward, and answers of a
    batch with an 8-bit cache and filters, the same twice."""
    from dataclasses import replace
    from nexttransformer_b200.inference import generate_batch, serve_experts
    from nexttransformer_b200.models import build_model
    from nexttransformer_b200.models.config import debug_config
    from nexttransformer_b200.models.moe import MoEFFN
    c = replace(debug_config("moe"), width=256, heads=4, kv_heads=2, moe_ffn=64)
    m = build_model(c, DEV, seed=1).eval()
    layer = next(b.mlp for b in m.transformer.h if isinstance(b.mlp, MoEFFN))
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0, 0.05)
        serve_experts(m)
        x = torch.randn(7, 1, 256, device=DEV).to(m.cos.dtype)
        got, ref = layer.step(x).double(), layer(x).double()
    # the layer rounds hidden values and each expert's product: 2 u of the magnitudes, which are a few times the result's size
    assert (got - ref).norm() <= 4 * U[torch.bfloat16] * ref.norm()
    prompts = [[1, 2, 3], [4], list(range(20))]
    answers = [generate_batch(m, prompts, 12, top_p=0.9, min_p=0.01, temperature=[0.5, 1.0, 0.0], cache_dtype=F8) for _ in range(2)]
    assert answers[0] == answers[1] and all(len(a) == 12 for a in answers[0])


def test_laid_out_experts_follow_the_kernel_state():
    """Where the kernel state keeps all of a layer's bf16 weights, one update reaches all of what ``step`` reads."""
    from dataclasses import replace
    from nexttransformer_b200.inference import serve_experts
    from nexttransformer_b200.models import build_model
    from nexttransformer_b200.models.config import debug_config
    from nexttransformer_b200.models.moe import MoEFFN
    c = replace(debug_config("moe"), width=256, heads=4, kv_heads=2, moe_ffn=128)
    m = build_model(c, DEV, seed=2).eval()
    m.fused_state()
    layer = next(b.mlp for b in m.transformer.h if isinstance(b.mlp, MoEFFN))
    serve_experts(m)
    assert layer._w_fc is not None and layer._served["w_fc"] is layer._w_fc
    x = torch.randn(9, 256, device=DEV).to(m.cos.dtype)
    results = []
    with torch.no_grad():
        for _ in range(2):
            for p in (*layer.parameters(), layer.expert_bias):
                p.normal_(0, 0.05)
            m.refresh_shadows()
            results.append((layer.step(x).double(), layer(x).double()))
    for got, ref in results:    # the layer's own roundings, as above
        assert (got - ref).norm() <= 4 * U[torch.bfloat16] * ref.norm()


def test_8_bit_cache_captured_and_on_two_streams():
    """A step (append and attention) captured once and replayed over several positions, across a block's border, beside the same on another
    stream: both equal eager steps bit for bit."""
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    B, H, Hk, D = 5, 8, 2, 128
    lengths = [13, 0, 31, 200, 64]
    cos, sin = torch.ones(300, D // 2, device=DEV).bfloat16(), torch.zeros(300, D // 2, device=DEV).bfloat16()
    torch.manual_seed(9)
    news = [torch.randn(B, 1, H + 2 * Hk, D, device=DEV).bfloat16() for _ in range(6)]

    def state():
        k, v, ks, vs, table = make_cache8([n + 8 for n in lengths], Hk, 32, D)
        return dict(k=k, v=v, ks=ks, vs=vs, table=table, x=torch.zeros_like(news[0]), start=torch.tensor(lengths, device=DEV, dtype=torch.int32))

    def step(s):
        x = s["x"]
        q = paged_append(x[:, :, :H], x[:, :, H:H + Hk], x[:, :, H + Hk:], s["k"], s["v"], s["table"], s["start"], cos=cos, sin=sin, qk_scale=1.2,
                         k_scale=s["ks"], v_scale=s["vs"])
        y = paged_attention(q, s["k"], s["v"], s["table"], s["start"], k_scale=s["ks"], v_scale=s["vs"])
        s["start"] += 1
        return y

    first = state()
    states = [first] + [{n: t.clone() for n, t in first.items()} for _ in range(2)]
    eager = []
    for x in news:
        states[0]["x"].copy_(x)
        eager.append(step(states[0]).clone())
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for s, stream in zip(states[1:], streams):
        keep = {n: t.clone() for n, t in s.items()}
        with torch.cuda.stream(stream):
            step(s)                                     # once before capture
            for n, t in keep.items():
                s[n].copy_(t)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(step(s))
        graphs.append(graph)
    got = [[], []]
    for x in news:
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                states[1 + i]["x"].copy_(x)
                graphs[i].replay()
                got[i].append(outs[i].clone())
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(got[i], eager):
            assert torch.equal(a, b)
        for n in ("k", "v", "ks", "vs"):
            assert torch.equal(states[1 + i][n].view(torch.uint8), states[0][n].view(torch.uint8))
    check_errors()
