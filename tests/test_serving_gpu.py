"""Serving operators (paged append and attention, recurrent delta rule, logits adjustment) against 64-bit definitions.

Tolerances follow from the roundings: u is half a unit in the last place of the output type (2^-8 bf16, 2^-11 fp16).
Attention may round its probabilities to the cache's type before it multiplies them by V, which moves an output by
at most u max|v| (fp16: and 2^-25 max|v| a key where they fall below the normal range), and rounds the output once.
Everything else is fp32.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DEV = "cuda"


def make_cache(rows, Hk, page, D, dtype, spare=2, seed=0, fill=float("nan")):
    """Pages in random order for rows of (start + count) tokens; every slot behind a row's last token holds `fill`."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in rows]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g).int()
    table = torch.full((len(rows), max(1, max(need))), -1, dtype=torch.int32)
    k = torch.full((P, Hk, page, D), fill)
    v = torch.full((P, Hk, page, D), fill)
    at = 0
    for b, n in enumerate(rows):
        table[b, :need[b]] = order[at:at + need[b]]
        for j in range(need[b]):
            m = min(page, n - j * page)
            k[order[at + j], :, :m] = torch.randn(Hk, m, D, generator=g) * 1.2
            v[order[at + j], :, :m] = torch.randn(Hk, m, D, generator=g)
        at += need[b]
    return k.to(DEV, dtype), v.to(DEV, dtype), table.to(DEV)


def oracle_attention(q, k_pages, v_pages, table, start, count, window, scale=None):
    B, t, H, D = q.shape
    Hk, page = k_pages.shape[1:3]
    out = torch.zeros(B, t, H, D, dtype=torch.float64, device=DEV)
    scale = D ** -0.5 if scale is None else scale
    for b in range(B):
        for i in range(count[b]):
            pos = start[b] + i
            lo = max(0, pos - window) if window >= 0 else 0
            key = torch.arange(lo, pos + 1, device=DEV)
            at = table[b].long()[key // page], slice(None), key % page
            K, V = k_pages[at].double(), v_pages[at].double()
            qq = q[b, i].double().view(Hk, H // Hk, D)
            p = torch.softmax(torch.einsum("hgd,khd->hgk", qq, K) * scale, -1)
            out[b, i] = torch.einsum("hgk,khd->hgd", p, V).reshape(H, D)
    return out


def check_attention(got, ref, v_pages, keys):
    u = U[got.dtype]
    top = v_pages.float().nan_to_num(0.0).abs().max().item()
    slack = 1.02 * u * top + (keys * 2.0 ** -25 * top if got.dtype == torch.float16 else 0.0) + 1e-5
    err = (got.double() - ref).abs()
    assert torch.isfinite(got.float()).all()
    assert (err <= 1.02 * u * ref.abs() + slack).all(), err.max().item()


CASES = [
    # dtype, D, H, Hk, page, t, window, (start, count) per row
    (torch.bfloat16, 128, 10, 5, 64, 1, -1, [(0, 1), (1, 1), (14, 1), (15, 1), (16, 1), (62, 1), (63, 1), (64, 1), (700, 1)]),
    (torch.float16, 128, 4, 4, 16, 1, -1, [(0, 1), (31, 1), (300, 1)]),
    (torch.bfloat16, 64, 16, 1, 48, 1, 37, [(0, 1), (36, 1), (37, 1), (38, 1), (53, 1), (400, 1)]),
    (torch.float16, 64, 12, 12, 16, 4, 20, [(0, 4), (0, 1), (13, 3), (90, 4), (200, 0)]),
    (torch.bfloat16, 128, 12, 3, 32, 5, 0, [(0, 5), (29, 5), (77, 2)]),
    (torch.bfloat16, 128, 16, 1, 64, 3, -1, [(0, 3), (5, 2), (1000, 3)]),
    (torch.bfloat16, 128, 40, 1, 64, 1, -1, [(0, 1), (130, 1)]),          # 40 query heads on one KV head
    (torch.float16, 128, 6, 6, 128, 33, 50, [(0, 33), (64, 20), (7, 0)]),  # a chunk of a prompt
    (torch.bfloat16, 64, 6, 2, 16, 1, -1, [(0, 0), (40, 0), (40, 1)]),     # rows without tokens
    (torch.bfloat16, 128, 8, 2, 64, 1, -1, [(9000, 1)]),                   # one row over many CTAs
    (torch.bfloat16, 128, 2, 1, 64, 1, 5000, [(30000, 1), (17, 1)]),
]


@pytest.mark.parametrize("dtype,D,H,Hk,page,t,window,rows", CASES)
def test_paged_attention(dtype, D, H, Hk, page, t, window, rows):
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(1)
    k, v, table = make_cache([s + c for s, c in rows], Hk, page, D, dtype)
    start, count = ([r[i] for r in rows] for i in (0, 1))
    q = (torch.randn(len(rows), t, H, D, device=DEV) * 1.2).to(dtype)
    args = (torch.tensor(start, device=DEV, dtype=torch.int32), torch.tensor(count, device=DEV, dtype=torch.int32))
    got = paged_attention(q, k, v, table, *args, window=window)
    check_attention(got, oracle_attention(q, k, v, table, start, count, window), v, max(s + c for s, c in rows))
    for b, c in enumerate(count):
        assert (got[b, c:] == 0).all()
    assert torch.equal(got, paged_attention(q, k, v, table, *args, window=window))   # bitwise reproducible
    check_errors()


def test_paged_attention_many_rows():
    """More rows than a CTA has threads to line them up."""
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(2)
    rows = [(b * 7) % 90 for b in range(500)]
    k, v, table = make_cache([r + 1 for r in rows], 2, 16, 64, torch.bfloat16)
    q = torch.randn(500, 1, 4, 64, device=DEV).bfloat16()
    got = paged_attention(q, k, v, table, torch.tensor(rows, device=DEV, dtype=torch.int32))
    check_attention(got, oracle_attention(q, k, v, table, rows, [1] * 500, -1), v, 90)


@pytest.mark.parametrize("dtype,D,H,Hk,page,t,window,rows", [
    (torch.bfloat16, 128, 12, 3, 16, 5, -1, [(0, 5), (1200, 5), (77, 1), (640, 4)]),        # 20 query rows: 2 strips
    (torch.float16, 64, 10, 5, 48, 9, 30, [(0, 9), (500, 9), (31, 8), (32, 0)]),            # 18: the second almost empty
    (torch.bfloat16, 128, 16, 4, 64, 9, -1, [(3000, 9), (5, 9)]),                           # 36: 4 strips, one empty
    (torch.float16, 128, 16, 1, 32, 5, 100, [(0, 5), (2500, 5), (95, 5), (300, 1)]),        # 80: 8, three empty
    (torch.bfloat16, 64, 16, 1, 128, 8, -1, [(9000, 8)]),                                   # 128: 8 strips over many CTAs
    (torch.bfloat16, 128, 16, 1, 64, 11, -1, [(40, 11), (700, 2), (0, 11)]),                # 176: two items a row
    (torch.float16, 128, 8, 2, 16, 50, 64, [(0, 50), (333, 41), (20, 33)]),                 # 200, windowed
])
def test_paged_attention_strips(dtype, D, H, Hk, page, t, window, rows):
    """More query rows a KV head than one warp holds: warps beside each other, items behind each other."""
    test_paged_attention(dtype, D, H, Hk, page, t, window, rows)


@pytest.mark.parametrize("B,t,H,Hk", [(2100, 1, 4, 2), (2060, 5, 4, 1)])
def test_paged_attention_of_more_rows_than_a_line_holds(B, t, H, Hk):
    """More rows than the CTAs line up: a CTA for each (row, KV head).  Every 97th row is compared."""
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(12)
    rows = [(b * 7) % 90 for b in range(B)]
    k, v, table = make_cache([r + t for r in rows], Hk, 16, 64, torch.bfloat16)
    q = torch.randn(B, t, H, 64, device=DEV).bfloat16()
    got = paged_attention(q, k, v, table, torch.tensor(rows, device=DEV, dtype=torch.int32))
    some = list(range(0, B, 97)) + [B - 1]
    check_attention(got[some], oracle_attention(q[some], k, v, table[some], [rows[b] for b in some], [t] * len(some), -1), v, 95)


def test_paged_attention_layouts_scale_and_stream():
    """Query rows inside a packed projection, one layer of a token-major cache, another stream, a given scale."""
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(3)
    rows = [33, 150]
    k, v, table = make_cache(rows, 3, 32, 128, torch.float16)
    big = torch.full((2, k.shape[0], 32, 3, 128), float("nan"), device=DEV, dtype=torch.float16)
    big[1] = k.transpose(1, 2)
    k = big[1].transpose(1, 2)
    packed = torch.randn(2, 2, 12, 128, device=DEV).half()
    q = packed[:, :, 3:9]
    start = torch.tensor([31, 148], device=DEV, dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention(q, k, v, table, start, scale=0.25)
    torch.cuda.current_stream().wait_stream(side)
    check_attention(got, oracle_attention(q, k, v, table, [31, 148], [2, 2], -1, 0.25), v, 150)


def test_paged_attention_scores_of_any_size():
    """Large scores: the running maximum moves by hundreds between tiles; one key takes all."""
    from nexttransformer_b200.ops.paged import paged_attention
    torch.manual_seed(4)
    k, v, table = make_cache([500], 1, 16, 128, torch.bfloat16)
    k.nan_to_num_(0.0)
    k *= torch.linspace(-40, 40, k.shape[0], device=DEV)[:, None, None, None].bfloat16()
    q = torch.randn(1, 1, 8, 128, device=DEV).bfloat16() * 4
    got = paged_attention(q, k, v, table, torch.tensor([499], device=DEV, dtype=torch.int32))
    check_attention(got, oracle_attention(q, k, v, table, [499], [1], -1), v, 500)


def test_paged_offsets_behind_32_bits():
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    torch.manual_seed(5)
    P = 2 ** 31 // (16 * 128) + 8
    k = torch.empty(P, 1, 16, 128, device=DEV, dtype=torch.bfloat16)
    v = torch.empty_like(k)
    k[-8:], v[-8:] = torch.randn(8, 1, 16, 128, device=DEV), torch.randn(8, 1, 16, 128, device=DEV)
    table = torch.tensor([[P - 3, P - 6]], device=DEV, dtype=torch.int32)
    start = torch.tensor([20], device=DEV, dtype=torch.int32)
    ones = torch.ones(32, 64, device=DEV, dtype=torch.bfloat16)
    new = torch.randn(1, 1, 4, 128, device=DEV).bfloat16()
    q = paged_append(new[:, :, :2], new[:, :, 2:3], new[:, :, 3:], k, v, table, start, cos=ones, sin=ones * 0)
    assert torch.equal(k[P - 6, 0, 4], new[0, 0, 2]) and torch.equal(v[P - 6, 0, 4], new[0, 0, 3])
    got = paged_attention(q, k, v, table, start)
    check_attention(got, oracle_attention(q, k, v, table, [20], [1], -1), v[-8:], 21)


@pytest.mark.parametrize("dtype,D,H,Hk,page,t,norm,ve,rows", [
    (torch.bfloat16, 128, 10, 5, 64, 1, True, True, [(0, 1), (63, 1), (64, 1), (200, 1)]),
    (torch.float16, 64, 3, 3, 16, 5, True, False, [(0, 5), (12, 4), (40, 0)]),
    (torch.bfloat16, 64, 4, 1, 48, 70, False, True, [(0, 70), (47, 33)]),
    (torch.float16, 128, 2, 1, 32, 1, False, False, [(5, 1)]),
])
def test_paged_append(dtype, D, H, Hk, page, t, norm, ve, rows):
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_append
    torch.manual_seed(6)
    B = len(rows)
    kp, vp, table = make_cache([s + c for s, c in rows], Hk, page, D, dtype, fill=7.0)
    before = kp.clone(), vp.clone()
    packed = torch.randn(B, t, H + 2 * Hk, D, device=DEV).to(dtype)
    q, k, v = packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]
    angle = torch.outer(torch.arange(512, device=DEV), 1e5 ** (-torch.arange(0, D, 2, device=DEV) / D))
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    e = torch.randn(B, t, Hk, D, device=DEV).to(dtype) if ve else None
    gate = torch.randn(B, t, Hk, device=DEV).to(dtype) if ve else None
    start, count = (torch.tensor([r[i] for r in rows], device=DEV, dtype=torch.int32) for i in (0, 1))
    got = paged_append(q, k, v, kp, vp, table, start, count, cos=cos, sin=sin, qk_scale=1.2 if norm else None, ve=e,
                       ve_gate=gate)
    check_errors()
    kr, vr, qr = before[0].double(), before[1].double(), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    written = torch.zeros(kp.shape[:3], dtype=torch.bool, device=DEV)
    for b, (s, n) in enumerate(rows):
        for i in range(n):
            c, sn = cos[s + i].double(), sin[s + i].double()

            def turn(x):
                x1, x2 = x.double().chunk(2, -1)
                y = torch.cat((x1 * c + x2 * sn, x2 * c - x1 * sn), -1)
                return 1.2 * y / (y.pow(2).mean(-1, keepdim=True) + 2.0 ** -23).sqrt() if norm else y
            qr[b, i] = turn(q[b, i])
            at = int(table[b, (s + i) // page]), slice(None), (s + i) % page
            kr[at] = turn(k[b, i])
            vr[at] = v[b, i].double() + (3 * torch.sigmoid(gate[b, i].double())[:, None] * e[b, i].double() if ve else 0)
            written[at] = True
    u = U[dtype]
    for x, r in ((got, qr), (kp, kr), (vp, vr)):  # fp32 inside (1e-5 covers it), one rounding
        assert ((x.double() - r).abs() <= 1.02 * u * r.abs() + 1e-5).all()
    for x, old in zip((kp, vp), before):
        assert torch.equal(x[~written], old[~written])


def test_paged_refusals():
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    k, v, table = make_cache([20], 2, 16, 64, torch.bfloat16)
    q = torch.zeros(1, 1, 4, 64, device=DEV, dtype=torch.bfloat16)
    start = torch.zeros(1, device=DEV, dtype=torch.int32)
    good = dict(q=q, k_pages=k, v_pages=v, table=table, start=start)
    for bad in (dict(q=q.float()), dict(q=q[..., :32]), dict(q=q[:, :, :3]), dict(k_pages=k.half()), dict(v_pages=v[:1]),
                dict(k_pages=k[:, :, :8], v_pages=v[:, :, :8]), dict(table=table.long()), dict(start=start.long()),
                dict(start=torch.zeros(2, device=DEV, dtype=torch.int32)), dict(table=table.cpu()), dict(k_pages=k.cpu()),
                dict(q=torch.zeros(1, 1, 4, 65, device=DEV, dtype=torch.bfloat16)[..., 1:])):
        with pytest.raises(RuntimeError):
            paged_attention(**{**good, **bad})
    with pytest.raises(RuntimeError, match="backward"):
        paged_attention(**{**good, "q": q.clone().requires_grad_()})
    cos = torch.ones(32, 32, device=DEV, dtype=torch.bfloat16)
    new = dict(good, k=q[:, :, :2], v=q[:, :, :2], cos=cos, sin=cos)
    for bad in (dict(cos=cos.float()), dict(cos=cos[:, :16]), dict(sin=cos[:16]), dict(k=q), dict(ve=q[:, :, :2]),
                dict(ve=q[:, :, :2], ve_gate=q[:, :, :2, 0].float()), dict(count=start.float())):
        with pytest.raises(RuntimeError):
            paged_append(**{**new, **bad})


def test_paged_device_checks():
    """Positions and page numbers are checked where they are read; the host raises afterwards."""
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    k, v, table = make_cache([20, 20], 2, 16, 64, torch.bfloat16, fill=0.0)
    before = k.clone()
    q = torch.ones(2, 1, 4, 64, device=DEV, dtype=torch.bfloat16)
    cos = torch.ones(64, 32, device=DEV, dtype=torch.bfloat16)

    def append(start, table, cos=cos):
        return paged_append(q, q[:, :, :2], q[:, :, :2], k, v, table, torch.tensor(start, device=DEV, dtype=torch.int32),
                            cos=cos, sin=cos)
    append([-1, 40], table)
    with pytest.raises(RuntimeError, match="page table.*row 1"):
        check_errors()
    append([5, -1], torch.full_like(table, 1 << 30))
    with pytest.raises(RuntimeError, match="page number.*row 0"):
        check_errors()
    append([5, -3], table, cos[:4])
    with pytest.raises(RuntimeError, match="rotary.*row 0"):
        check_errors()
    assert torch.equal(k, before)
    out = paged_attention(q, k, v, torch.full_like(table, -7), torch.tensor([5, -1], device=DEV, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="page number.*row 0"):
        check_errors()
    assert (out[1] == 0).all()
    paged_attention(q, k, v, table, torch.tensor([3, 32], device=DEV, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="page table.*row 1"):
        check_errors()
    check_errors()


# ------------------------------------------------------------------------------------------ delta rule
def oracle_delta(q, k, v, state, beta, g, scale, l2norm, slots, count):
    q, k, v, beta = (x.double() for x in (q, k, v, beta))
    if l2norm:
        q, k = (x / x.norm(dim=-1, keepdim=True).clamp(min=1e-12) for x in (q, k))
    state, out = state.double(), torch.zeros_like(v)
    for b in range(q.shape[0]):
        if slots[b] < 0:
            continue
        S = state[slots[b]]
        for t in range(count[b]):
            if g is not None:
                a = g[b, t].double().exp()
                S = S * (a[:, None, None] if a.dim() == 1 else a[..., None])
            u = beta[b, t, :, None] * (v[b, t] - torch.einsum("hk,hkv->hv", k[b, t], S))
            S = S + k[b, t, :, :, None] * u[:, None]
            out[b, t] = torch.einsum("hk,hkv->hv", q[b, t] * scale, S)
        state[slots[b]] = S
    return out, state


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind,D,H,T,count,slots,l2norm", [
    ("gdn", 128, 3, 1, [1, 1], [0, 1], True),
    ("kda", 128, 2, 1, [1, 0, 1], [3, 1, 0], True),
    ("deltanet", 64, 1, 8, [8, 7, 0], [2, 0, 1], True),
    ("gdn", 64, 2, 9, [9, 1], [1, -1], False),
    ("kda", 64, 1, 17, [17, 16, 3], [0, 1, 2], True),
    ("deltanet", 128, 2, 70, [70, 41], [0, 1], True),
    ("gdn", 128, 1, 65, [65], [4], True),
    ("gdn", 128, 30, 50, [50, 3, 50, 17, 50, 50], [5, 4, 3, 2, 1, 0], True),   # columns 32 a CTA
    ("kda", 64, 40, 33, [33, 33, 8, 33, 33], [0, 1, 2, 3, 4], True),
])
def test_delta_recurrent(dtype, kind, D, H, T, count, slots, l2norm):
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    torch.manual_seed(7)
    B, scale = len(count), D ** -0.5
    packed = (torch.randn(B, T, 3 * H, D, device=DEV) * (1.0 if l2norm else D ** -0.5)).to(dtype)
    q, k, v = packed[:, :, :H], packed[:, :, H:2 * H], packed[:, :, 2 * H:]
    beta = torch.rand(B, T, H, device=DEV).to(dtype if T % 2 else torch.float32)
    g = {"deltanet": None, "gdn": -torch.rand(B, T, H, device=DEV) * 2, "kda": -torch.rand(B, T, H, D, device=DEV)}[kind]
    state = torch.randn(6, H, D, D, device=DEV) * 0.3
    ref, ref_state = oracle_delta(q, k, v, state, beta, g, scale, l2norm, slots, count)
    ints = dict(slots=torch.tensor(slots, device=DEV, dtype=torch.int32), count=torch.tensor(count, device=DEV, dtype=torch.int32))
    first = state.clone()
    got = delta_recurrent(q, k, v, state, beta, g, scale=scale, l2norm=l2norm, **ints)
    check_errors()
    # fp32 sums of D terms of size 1, T steps that do not amplify: 1e-6 a step
    slack = 2e-6 * (T + 4)
    assert ((state.double() - ref_state).abs() <= slack).all(), (state.double() - ref_state).abs().max()
    assert ((got.double() - ref).abs() <= 1.02 * U[dtype] * ref.abs() + slack).all()
    for s in set(range(6)) - {s for s, c in zip(slots, count) if c}:
        assert torch.equal(state[s], first[s])
    again = first.clone()
    assert torch.equal(got, delta_recurrent(q, k, v, again, beta, g, scale=scale, l2norm=l2norm, **ints))
    assert torch.equal(again, state)


def test_delta_recurrent_in_pieces_and_zero_vectors():
    """A run of tokens equals the same tokens in several calls, bitwise where the cuts keep its blocks of eight and
    within twice the bound of test_delta_recurrent elsewhere; zero queries and keys stay zero under the norm."""
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    torch.manual_seed(8)
    q, k, v = (torch.randn(2, 21, 2, 128, device=DEV) for _ in range(3))
    k[0, 3], q[1, 5] = 0.0, 0.0
    beta, g = torch.rand(2, 21, 2, device=DEV), -torch.rand(2, 21, 2, device=DEV)
    whole = torch.zeros(2, 2, 128, 128, device=DEV)
    o = delta_recurrent(q, k, v, whole, beta, g, l2norm=True)
    for cuts, slack in (((0, 8, 16, 21), 0.0), ((0, 1, 9, 21), 4e-6 * (21 + 4))):
        state = torch.zeros_like(whole)
        cut = [delta_recurrent(*(x[:, a:b] for x in (q, k, v)), state, beta[:, a:b], g[:, a:b], l2norm=True)
               for a, b in zip(cuts, cuts[1:])]
        assert (torch.cat(cut, 1) - o).abs().max() <= slack and (state - whole).abs().max() <= slack
    assert (o[1, 5] == 0).all() and torch.isfinite(o).all()


def test_delta_recurrent_in_segments():
    """More blocks than the workspace holds: the state passes through memory between segments of a call."""
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    torch.manual_seed(12)
    B, T, H, D = 8, 300, 16, 128
    q, k, v = (torch.randn(B, T, H, D, device=DEV).bfloat16() for _ in range(3))
    beta, g = torch.rand(B, T, H, device=DEV), -torch.rand(B, T, H, device=DEV)
    count = [300, 1, 0, 199, 200, 201, 256, 77]
    state = torch.randn(B, H, D, D, device=DEV) * 0.3
    ref, ref_state = oracle_delta(q, k, v, state, beta, g, 1.0, True, list(range(B)), count)
    got = delta_recurrent(q, k, v, state, beta, g, l2norm=True, count=torch.tensor(count, device=DEV, dtype=torch.int32))
    slack = 2e-6 * (T + 4)
    assert ((state.double() - ref_state).abs() <= slack).all()
    assert ((got.double() - ref).abs() <= 1.02 * U[torch.bfloat16] * ref.abs() + slack).all()


def test_delta_recurrent_state_behind_32_bits():
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    torch.manual_seed(9)
    N = 2 ** 31 // 128 ** 2 + 4
    state = torch.empty(N, 1, 128, 128, device=DEV)
    state[-4:] = 0
    q, k, v = (torch.randn(1, 1, 1, 128, device=DEV) for _ in range(3))
    one = torch.ones(1, 1, 1, device=DEV)
    delta_recurrent(q, k, v, state, one, slots=torch.tensor([N - 2], device=DEV, dtype=torch.int32))
    torch.testing.assert_close(state[N - 2, 0], k[0, 0, 0][:, None] * v[0, 0, 0], rtol=1e-6, atol=1e-6)
    assert (state[[N - 4, N - 3, N - 1]] == 0).all()


def test_delta_recurrent_refusals():
    from nexttransformer_b200.ops._ext import check_errors
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    x = torch.zeros(2, 1, 2, 64, device=DEV, dtype=torch.bfloat16)
    state, beta = torch.zeros(2, 2, 64, 64, device=DEV), torch.zeros(2, 1, 2, device=DEV)
    good = dict(q=x, k=x, v=x, state=state, beta=beta)
    for bad in (dict(q=x.half()), dict(k=x[:, :, :1]), dict(state=state.bfloat16()), dict(state=state[:1]),
                dict(state=state.transpose(-1, -2)), dict(beta=beta[:1]), dict(beta=beta.double()),
                dict(g=beta.bfloat16()), dict(g=beta[..., None]), dict(count=torch.ones(2, device=DEV)),
                dict(q=x[..., :32], k=x[..., :32], v=x[..., :32])):
        with pytest.raises(RuntimeError):
            delta_recurrent(**{**good, **bad})
    with pytest.raises(RuntimeError, match="backward"):
        delta_recurrent(**{**good, "v": x.clone().requires_grad_()})
    o = delta_recurrent(**good, slots=torch.tensor([0, 2], device=DEV, dtype=torch.int32))
    assert (o == 0).all()
    with pytest.raises(RuntimeError, match="slot.*row 1"):
        check_errors()


# ------------------------------------------------------------------------------------------ logits
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V,L,K,mask,pad", [
    (1, 1, 1, 1, True, 0), (3, 31, 5, 0, True, 33), (2, 1000, 0, 40, False, 24), (5, 4099, 700, 3, True, 0),
    (200, 8192, 64, 33, True, 64), (2, 50001, 3000, 300, True, 47),
])
def test_adjust_logits(dtype, B, V, L, K, mask, pad):
    from nexttransformer_b200.ops.logits import _plain, adjust_logits
    torch.manual_seed(10)
    full = (torch.randn(B, V + pad, device=DEV) * 5).to(dtype)
    logits = full[:, :V]
    few = max(1, V // 50)
    tokens = torch.randint(-1, V + 1, (B, L), device=DEV, dtype=torch.int32)
    tokens[:, ::2] = tokens[:, ::2] % few
    length = torch.randint(0, L + 2, (B,), device=DEV, dtype=torch.int32)
    prompt = torch.randint(0, L + 2, (B,), device=DEV, dtype=torch.int32)
    r, p, f = 1 + torch.rand(B, device=DEV), torch.rand(B, device=DEV), torch.rand(B, device=DEV)
    ids = torch.randint(-1, V + 1, (B, K), device=DEV, dtype=torch.int32)
    if K > 2:
        ids[:, 2] = ids[:, 0]
    bias = torch.randn(B, K, device=DEV)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), device=DEV).int() if mask else None
    if mask:
        allowed[0] = 0                      # a row that allows nothing
        full[B - 1, 0] = float("nan")       # a masked NaN is masked
        allowed[B - 1, 0] &= ~1
    args = (tokens, length, prompt, r, p, f, ids, bias, allowed)
    names = ("tokens", "length", "prompt", "repetition", "presence", "frequency", "bias_ids", "bias", "allowed")
    got = adjust_logits(logits, **dict(zip(names, args)))
    ref = _plain(logits.cpu(), *(None if x is None else x.cpu() for x in args))
    assert got.dtype == torch.float32 and got.shape == (B, V)
    if mask:
        assert (got[0] == -math.inf).all() and got[B - 1, 0] == -math.inf
    # a few fp32 roundings of numbers below 3000 (a count of at most L times a frequency below 1)
    torch.testing.assert_close(got.cpu(), ref, rtol=1e-6, atol=1e-3 if L > 1000 else 1e-4)
    assert torch.equal(got, adjust_logits(logits, **dict(zip(names, args))))
    # each part alone
    torch.testing.assert_close(adjust_logits(logits).cpu(), logits.float().cpu(), rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(adjust_logits(logits, tokens=tokens, repetition=r).cpu(),
                               _plain(logits.cpu(), tokens.cpu(), None, None, r.cpu(), None, None, None, None, None),
                               rtol=1e-6, atol=0, equal_nan=True)


def test_adjust_logits_refusals():
    from nexttransformer_b200.ops.logits import adjust_logits
    x = torch.zeros(2, 64, device=DEV)
    ints = torch.zeros(2, 3, device=DEV, dtype=torch.int32)
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.t()), dict(tokens=ints.long()),
                dict(tokens=ints[:1]), dict(repetition=x[:, 0].double()), dict(presence=x[:1, 0]), dict(bias=x),
                dict(bias_ids=ints, bias=x[:, :2]), dict(allowed=ints[:, :1]), dict(length=ints[0]), dict(tokens=ints.cpu())):
        with pytest.raises(RuntimeError):
            adjust_logits(**{"logits": x, **bad})
    with pytest.raises(RuntimeError, match="backward"):
        adjust_logits(x.clone().requires_grad_())


# ------------------------------------------------------------------------------------------ together
def test_operators_under_graph_capture():
    """The operators can be captured; a replay on another stream, beside eager calls, sees the buffers' new contents."""
    from nexttransformer_b200.ops.delta_recurrent import delta_recurrent
    from nexttransformer_b200.ops.logits import adjust_logits
    from nexttransformer_b200.ops.paged import paged_append, paged_attention
    torch.manual_seed(11)
    k, v, table = make_cache([3000, 40], 2, 16, 128, torch.bfloat16, fill=0.0)
    start = torch.tensor([2990, 30], device=DEV, dtype=torch.int32)
    angle = torch.rand(4096, 64, device=DEV)
    cos, sin = angle.cos().bfloat16(), angle.sin().bfloat16()
    new = torch.randn(2, 1, 8, 128, device=DEV).bfloat16()
    state, beta = torch.zeros(2, 2, 128, 128, device=DEV), torch.rand(2, 1, 2, device=DEV)
    tokens = torch.randint(0, 500, (2, 9), device=DEV, dtype=torch.int32)
    two = torch.full((2,), 2.0, device=DEV)

    def step():
        q = paged_append(new[:, :, :4], new[:, :, 4:6], new[:, :, 6:], k, v, table, start, cos=cos, sin=sin, qk_scale=1.2)
        y = paged_attention(q, k, v, table, start)
        z = delta_recurrent(y[:, :, :2], y[:, :, 2:], y[:, :, :2], state, beta, l2norm=True)
        return y, z, adjust_logits(z.reshape(2, -1), tokens=tokens, repetition=two)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    side = torch.cuda.Stream()
    for seed in (1, 2):
        torch.manual_seed(seed)
        new.copy_(torch.randn_like(new))
        start += 1
        state.zero_()
        eager = [t.clone() for t in step()]
        state.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("method,extra", [("dense", dict(layers=2, window_pattern="SL", kv_heads=1)),
                                          ("gdn_hybrid_swa", dict(layers=4, backend="fla_chunk64", sliding_window=128)),
                                          ("kda", dict(layers=2, backend="fla_chunk64"))])
def test_paged_decode_of_a_model(method, extra):
    """Prompts and steps through the kernels against the same weights in fp64: no further off than twice the plain
    bf16 forward is, which measures what bf16 activations alone cost."""
    from dataclasses import replace
    from nexttransformer_b200.inference import PagedCache, decode_paged, generate_batch
    from nexttransformer_b200.models import build_model
    from nexttransformer_b200.models.config import candidate_config
    from nexttransformer_b200.ops._ext import check_errors
    from tests.test_families_gpu import compute_dtype
    c = replace(candidate_config(method), width=256, heads=2, vocab_size=512, sequence_len=256, mlp_width=1024,
                scale="custom", **{"window_pattern": "L", **extra})
    with compute_dtype(torch.bfloat16):
        m = build_model(c, DEV, seed=0).eval()
    with torch.no_grad():
        for b in m.transformer.h:
            b.attn.c_proj.weight.normal_(0, .05)
            b.mlp.c_proj.weight.normal_(0, .05)
        m.smear_lambda.fill_(.5)
        m.lm_head.weight.normal_(0, .2)
    with compute_dtype(torch.float64):
        oracle = build_model(c, "cpu", seed=0)
        oracle.load_state_dict(m.state_dict())
        oracle = oracle.double().eval()
        oracle.cos, oracle.sin = m.cos.cpu().double(), m.sin.cpu().double()
    torch.manual_seed(5)
    ids = torch.randint(0, c.vocab_size, (3, 200), device=DEV)
    have = [150, 1, 63]
    cache = PagedCache(m, 3, 200, page=16)
    with torch.no_grad():
        got = [decode_paged(m, ids[:, :150], cache, have)]
        for _ in range(2):
            got.append(decode_paged(m, torch.stack([ids[r, n:n + 1] for r, n in enumerate(have)]), cache))
            have = [n + 1 for n in have]
        check_errors()
        for step, n0 in ((0, [150, 1, 63]), (2, [152, 3, 65])):
            for r, n in enumerate(n0):
                with compute_dtype(torch.float64):
                    ref = oracle(ids[r:r + 1, :n].cpu())[0, -1].float()
                plain = (m(ids[r:r + 1, :n])[0, -1].cpu() - ref).norm() / ref.norm()
                mine = (got[step][r].cpu() - ref).norm() / ref.norm()
                assert mine <= 2 * plain + 2e-3, (step, r, mine.item(), plain.item())
        answers = generate_batch(m, [ids[0, :9].tolist(), [1]], 5, temperature=.8, top_k=20, frequency=.5, repetition=1.1)
    check_errors()
    assert all(len(a) == 5 and all(0 <= t < c.vocab_size for t in a) for a in answers)
