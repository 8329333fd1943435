"""Edges of the decoding operators on the GPU: rows, weights and values where a kernel's ways of computing part, against 64 bits."""
import math

import pytest
import torch

import tests.test_decode_ops_gpu as ops
from tests.test_decode_ops_gpu import F8, both, check_experts, experts, make_experts, stands_for
from tests.test_serving_gpu import U

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------------------ sampling
@pytest.mark.parametrize("B,V,allowed", [
    (5, 8000, 40), (60, 8000, 300), (100, 20000, 40), (100, 20000, 3500),   # two CTAs a row
    (5, 32768, 40), (5, 32768, 9000), (224, 65536, 60), (74, 65536, 4000),  # four
    (7, 131072, 300), (2, 131072, 20000), (3, 300001, 20000), (9, 1000, 30)])  # eight, eight, eight, one
def test_sampling_with_fewer_permitted_tokens_than_top_k(B, V, allowed):
    """A mask leaves fewer tokens than top-k asks for, so that the k-th has no weight and top-p goes by all that are left."""
    torch.manual_seed(B + V)
    place = torch.rand(B, V, device=DEV).argsort(-1)
    x = torch.where(place < allowed, torch.randn(B, V, device=DEV) * 2, -math.inf)
    u = torch.rand(B, device=DEV)
    k = min(V, allowed + 10)
    both(x, u, top_k=k, top_p=0.9)
    both(x.bfloat16(), u, top_k=k, top_p=0.9, temperature=0.6, min_p=0.01)
    both(x, u, top_k=k)
    # some rows with a k that is reached, and some without a token
    x[::3, 1:] = -math.inf
    some = torch.where(torch.arange(B, device=DEV) % 2 == 0, k, max(1, allowed // 2)).int()
    both(x, u, top_k=some, top_p=0.8)


# what a call may ask for: drawn by one CTA from a few, by sums up to a border, and from a whole row
WAYS = [dict(), dict(top_k=17), dict(top_p=0.37), dict(top_k=7000, top_p=0.9), dict(min_p=0.02), dict(top_k=40, top_p=0.5, min_p=0.3)]


@pytest.mark.parametrize("V,dtype", [(700, torch.bfloat16), (32768, torch.float32), (32768, torch.bfloat16), (131072, torch.float32)])
def test_sampling_at_low_temperatures(V, dtype):
    """The largest logit's weight is 1 whatever top / T is: one largest, and many that share the choice."""
    torch.manual_seed(V)
    single = torch.randn(6, V, device=DEV) * 4 + torch.tensor([15.0, -20.0, 3.0, 0.0, 31.0, 14.3], device=DEV)[:, None]
    many = torch.where(torch.rand(6, V, device=DEV) < 0.4, 14.3, single.clamp(max=10.0))
    u = torch.rand(6, device=DEV)
    for x in (single, many):
        for T in (1e-9, 1e-12, 1e-14, 1e-15, 1e-16, 1e-17, 1e-18, 1e-20, 1e-24, 1e-38, 1e-44):
            for kw in WAYS:
                both(x.to(dtype), u, temperature=T, **kw)
    T = torch.tensor([1e-9, 1e-16, 1e-17, 1e-20, 0.7, 1e-24], device=DEV)
    for kw in WAYS:
        both(single.to(dtype), u, temperature=T, **kw)


@pytest.mark.parametrize("V,dtype", [(700, torch.float32), (700, torch.bfloat16), (32768, torch.float32), (131072, torch.bfloat16)])
def test_sampling_of_large_logits(V, dtype):
    """Logits as a bias of 1e18 leaves them, and rows that are large altogether."""
    torch.manual_seed(V + 1)
    rows = torch.randn(4, V, device=DEV)
    u = torch.rand(4, device=DEV)
    for size in (1e9, 6e15, 1e17, 1e19, 1e30, 3e38):
        for sign in (1, -1):
            one, equal, some = rows.clone(), torch.full_like(rows, sign * size), rows.clone()
            one[:, V // 3] = size if sign > 0 else one[:, V // 3]
            if sign < 0:
                one = one - size                     # most of them equal, by rounding
            some[:, 5::7] = sign * size              # a seventh of the row above, or below, the rest
            for x in (one, equal, some):
                for T in (0.3, 1.0):
                    for kw in WAYS:
                        both(x.to(dtype), u, temperature=T, **kw)
        both((rows * min(size, 1e37)).to(dtype), u, temperature=min(size, 1e37) / 2, top_p=0.9)
        both((rows * min(size, 1e37)).to(dtype), u, temperature=min(size, 1e37) / 2, top_k=50)


@pytest.mark.parametrize("V,dtype", [(50, torch.float32), (700, torch.bfloat16), (32768, torch.float32)])
def test_sampling_where_logits_lie_further_apart_than_fp32_reaches(V, dtype):
    torch.manual_seed(V + 2)
    x = ((torch.rand(4, V, device=DEV) * 2 - 1) * 3.3e38).to(dtype)
    x[:, 0], x[:, -1] = 3.3e38, -3.3e38
    u = torch.rand(4, device=DEV)
    for T in (1e36, 1e37, 1e38, 3e38, math.inf):
        for kw in (*WAYS, dict(top_k=V - 1), dict(top_p=0.999)):
            both(x, u, temperature=T, **kw)


# ------------------------------------------------------------------------------------------ experts
@pytest.mark.parametrize("scale", [1.0, 0.1, 0.03, 0.01, 0.001])
@pytest.mark.parametrize("T,d,F,E,k,shared", [
    (1, 256, 64, 16, 8, 64), (5, 2048, 128, 32, 8, 0), (12, 2048, 64, 16, 16, 64), (13, 136, 72, 16, 8, 0), (16, 64, 24, 3, 2, 1000),
    (20, 320, 80, 32, 8, 80), (64, 128, 64, 16, 10, 64)])
def test_fp16_experts_of_small_tokens(T, d, F, E, k, shared, scale):
    """Small tokens have small hidden values, whose squares must not fall between fp16's steps.

    As `check_experts`: a hidden value is 2^-22 of itself off, or 2^-30 where that is more.  The latter, over the products of an output (a
    row of W2 has a norm of sqrt(k) or sqrt(k + 1) here, at most 4.2, and the errors have independent signs), is 2^-30 * 4.2 * 6 at the outside, less than
    the 2^-25 that the output's smallest half step leaves of the 2^-24 there."""
    from nexttransformer_b200.ops.moe import moe_tokens
    a = make_experts(T, d, F, E, shared, torch.float16, seed=T * 100 + d, scale=scale)
    got = moe_tokens(top_k=k, **a)
    ref, size = experts(a["x"], a["router"], a["w_fc"], a["w_proj"], k, a["bias"], a.get("shared_fc"), a.get("shared_proj"))
    check_experts(got, ref, size, torch.float16, d / 4 + (k * F + shared) / 16)
    assert torch.equal(got, moe_tokens(top_k=k, **a))


def test_fp16_experts_of_large_and_small_hidden_values():
    """The same layer for tokens of 1e-2 to 3e2 beside each other: hidden values of 1e-6 to 1e5."""
    from nexttransformer_b200.ops.moe import moe_tokens
    for T in (6, 15, 30):
        a = make_experts(T, 256, 64, 16, 64, torch.float16, seed=T)
        size_of = torch.logspace(-2, 2.5, T, device=DEV)
        a["x"] = (a["x"].float() * size_of[:, None]).half()
        a["router"] /= 300
        for n in ("w_proj", "shared_proj"):
            a[n] = a[n] * 2.0 ** -6
        ref, size = experts(a["x"], a["router"], a["w_fc"], a["w_proj"], 4, a["bias"], a["shared_fc"], a["shared_proj"])
        check_experts(moe_tokens(top_k=4, **a), ref, size, torch.float16, 64 + 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,d,F", [(1, 64, 64), (6, 2048, 72), (7, 136, 200), (12, 2048, 64), (16, 72, 136), (20, 136, 72), (64, 64, 24)])
def test_weights_that_are_not_finite_reach_the_tokens_that_chose_them(T, d, F, dtype):
    from nexttransformer_b200.ops.moe import moe_tokens
    a = make_experts(T, d, F, 12, 64, dtype, seed=T)
    a["bias"][7] = -5.0                                                   # nobody's
    clean = moe_tokens(top_k=2, **a)
    assert torch.isfinite(clean).all()
    score = torch.softmax(a["x"].double() @ a["router"].double().T, -1) + a["bias"].double()
    choice = score.topk(2).indices
    for e in (7, int(choice[0, 0]), int(choice[-1, 1])):
        hit = (choice == e).any(-1)
        for bad in (math.inf, -math.inf, math.nan):
            b = dict(a, w_proj=a["w_proj"].clone(), w_fc=a["w_fc"])
            b["w_proj"][e, 9, F // 2] = bad                               # one channel of y
            got = moe_tokens(top_k=2, **b)
            assert torch.equal(got[~hit], clean[~hit]) and not got[hit, 9].isfinite().any()
            got[:, 9] = clean[:, 9]
            assert torch.equal(got, clean)
            b = dict(a, w_fc=a["w_fc"].clone())
            b["w_fc"][e, F - 1, d // 2] = bad                             # one hidden value
            got = moe_tokens(top_k=2, **b)
            assert torch.equal(got[~hit], clean[~hit])
            if math.isnan(bad):
                assert got[hit].isnan().all()


# ------------------------------------------------------------------------------------------ attention in 8 bits
def check_keys(got, q, k, v, table, start, window=-1):
    """Attention in 64 bits over what the codes stand for, with a bound for each output from the keys that its query sees.

    The output is rounded once (u |out|).  A score, a sum of D products in fp32, is 2^-22 of its terms' sum off, which moves a probability
    p by twice that.  p is held as one fp16 number beside bf16 queries (2^-11 of it at most, half a step), two beside fp16 ones (2^-22), and below 2^-14 of the
    largest as a multiple of 2^-24 after a factor of 2^7 * 2^-8 at the least (a tile's scale may be 2^-7 of the unit, itself rounded up to
    a power of two): 2^-25 / 2^-1 of the largest probability, which is at most 1, 2^-24, and never more than p itself.  Where a tile's scale is the
    largest, the factor is 2^6 at the least, and it is 2^-31.  fp32 sums of n terms: n * 2^-24 of their size."""
    B, t, H, D = q.shape
    Hk, page = k.shape[1:3]
    group = H // Hk
    for b in range(B):
        for i in range(t):
            pos = start[b] + i
            key = torch.arange(max(0, pos - window) if window >= 0 else 0, pos + 1, device=DEV)
            at = table[b].long()[key // page], slice(None), key % page
            K, V = k[at], v[at].abs()
            qq = q[b, i].double().view(Hk, group, D)
            s = torch.einsum("hgd,khd->hgk", qq, K) * D ** -0.5
            terms = torch.einsum("hgd,khd->hgk", qq.abs(), K.abs()) * D ** -0.5
            p = torch.softmax(s, -1)
            ref = torch.einsum("hgk,khd->hgd", p, v[at])
            largest = V.amax(-1) >= V.amax((0, 2)) / 256                                   # [key, head]
            lost = torch.where(largest.T[:, None], 2.0 ** -31, 2.0 ** -24)
            each = p * (2 * terms.amax(-1, keepdim=True) * 2.0 ** -22 + (1.01 * 2.0 ** -11 if got.dtype == torch.bfloat16 else 2.0 ** -21) + len(key) * 2.0 ** -24)
            slack = torch.einsum("hgk,khd->hgd", each + torch.minimum(p, lost), V)
            err = (got[b, i].double().view(Hk, group, D) - ref).abs()
            assert torch.isfinite(got[b, i].float()).all()
            assert (err <= 1.02 * U[got.dtype] * ref.abs() + slack + 2.0 ** -25).all(), ((err - U[got.dtype] * ref.abs()) / slack).max().item()


def make_far_apart(rows, Hk, D, page, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    columns = -(-max(rows) // page)
    P = len(rows) * columns
    table = torch.randperm(P, generator=g, device=DEV).int().view(len(rows), columns)
    k, v = ((torch.randn(P, Hk, page, D, generator=g, device=DEV) * 80).clamp(-448, 448).to(F8) for _ in "kv")
    ks, vs = (torch.full((P, Hk, page // 16), 2.0 ** -7, device=DEV) for _ in "kv")
    return k, v, ks, vs, table


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("larger", [12, 20, 30, 100])
@pytest.mark.parametrize("H,Hk,D,first,t", [(4, 2, 64, 30, 4), (8, 1, 128, 700, 12), (2, 2, 128, 9, 40)])
def test_attention_in_8_bits_before_a_block_of_larger_values(H, Hk, D, first, t, larger, dtype):
    """Queries that a later block of the same call is hidden from: its values are 2^12 to 2^100 times theirs."""
    from nexttransformer_b200.ops.paged import paged_attention
    k, v, ks, vs, table = make_far_apart([first + t] * 2, Hk, D, 16, seed=first)
    last = (first + t - 1) // 16
    vs[table[:, last].long()] *= 2.0 ** larger
    q = torch.randn(2, t, H, D, device=DEV).to(dtype)
    start = torch.full((2,), first, device=DEV, dtype=torch.int32)
    got = paged_attention(q, k, v, table, start, k_scale=ks, v_scale=vs)
    seen = last * 16 - first                           # queries that do not see it
    assert 0 < seen < t
    check_keys(got[:, :seen], q[:, :seen], stands_for(k, ks), stands_for(v, vs), table, [first] * 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("keys,larger,window", [(40, 20, -1), (700, 24, -1), (3000, 16, -1), (9000, 20, -1), (600, 30, 100)])
def test_attention_in_8_bits_beside_blocks_of_larger_values(keys, larger, window, dtype):
    """Blocks whose values are 2^16 to 2^30 times the others', and whose keys the queries all but pass by."""
    from nexttransformer_b200.ops.paged import paged_attention
    H = Hk = 3
    D, page = 64, 32
    k, v, ks, vs, table = make_far_apart([keys] * 2, Hk, D, page, seed=keys)
    q = (torch.randn(2, 1, H, D, device=DEV) * 0.5).to(dtype)
    blocks = -(-keys // 16)
    for b in range(2):
        for j in {0, 1, blocks // 3, blocks // 2, max(0, blocks - 3)} - {blocks - 1}:
            at, half = table[b, j * 16 // page].long(), j * 16 % page // 16
            vs[at, :, half] *= 2.0 ** larger
            # scores of about -80: against the query's signs
            ks[at, :, half] = 1.0
            k[at, :, half * 16:half * 16 + 16] = (q[b, 0].float().sign() * -28.0)[:, None].expand(Hk, 16, D).to(F8)
    if dtype == torch.bfloat16:
        vs[table[:, -1].long()] *= 2.0 ** -20          # and a last one far below
    start = torch.full((2,), keys - 1, device=DEV, dtype=torch.int32)
    got = paged_attention(q, k, v, table, start, window=window, k_scale=ks, v_scale=vs)
    check_keys(got, q, stands_for(k, ks), stands_for(v, vs), table, [keys - 1] * 2, window)


def test_attention_in_8_bits_reads_scales_that_share_memory():
    from nexttransformer_b200.ops.paged import paged_attention
    k, v, _, _, table = make_far_apart([70], 2, 64, 32, seed=1)
    shape = (*k.shape[:2], 2)
    one, heads = torch.full((1, 1, 1), 2.0 ** -7, device=DEV).expand(shape), torch.tensor([2.0 ** -8, 2.0 ** -6], device=DEV)[None, :, None].expand(shape)
    q, start = torch.randn(1, 1, 4, 64, device=DEV).bfloat16(), torch.tensor([69], device=DEV, dtype=torch.int32)
    got = paged_attention(q, k, v, table, start, k_scale=one, v_scale=heads)
    assert torch.equal(got, paged_attention(q, k, v, table, start, k_scale=one.contiguous(), v_scale=heads.contiguous()))


# ------------------------------------------------------------------------------------------ append in 8 bits
@pytest.mark.parametrize("dtype,D,H,Hk,page,t,norm,ve,rows", [
    (torch.float16, 64, 10, 2, 16, 512, True, True, [(0, 512), (9, 300)]),                  # 10240 heads of tokens
    (torch.bfloat16, 64, 10, 5, 64, 511, False, True, [(7, 511), (0, 16)]),                 # just below
    (torch.bfloat16, 128, 1, 1, 48, 700, True, False, [(b, 700 - 40 * b) for b in range(16)]),
    (torch.float16, 128, 16, 4, 32, 40, True, True, [(b * 5 % 37, b % 41) for b in range(20)])])
def test_append_in_8_bits_of_many_and_few_heads(dtype, D, H, Hk, page, t, norm, ve, rows):
    ops.test_append_in_8_bits(dtype, D, H, Hk, page, t, norm, ve, rows)


@pytest.mark.parametrize("H,Hk,D,dtype", [(10, 5, 128, torch.bfloat16), (12, 12, 64, torch.float16), (16, 1, 128, torch.bfloat16)])
def test_append_in_8_bits_of_a_batch_and_of_its_rows(H, Hk, D, dtype):
    """Rows of a large call and of small ones are written alike, to the bit."""
    from nexttransformer_b200.ops.paged import paged_append
    torch.manual_seed(H)
    B, t, page = 6, 400, 32
    x = torch.randn(B, t, H + 2 * Hk, D, device=DEV).to(dtype)
    table = torch.randperm(B * 16, device=DEV).int().view(B, 16)
    start = torch.tensor([0, 5, 16, 31, 100, 111], device=DEV, dtype=torch.int32)
    count = torch.tensor([400, 1, 33, 400, 399, 16], device=DEV, dtype=torch.int32)
    angle = torch.outer(torch.arange(512, device=DEV), 1e4 ** (-torch.arange(0, D, 2, device=DEV) / D))
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    held, out = [], []
    for parts in ([slice(0, B)], [slice(b, b + 1) for b in range(B)]):
        k, v = (torch.zeros(B * 16, Hk, page, D, device=DEV).to(F8) for _ in "kv")
        ks, vs = (torch.zeros(B * 16, Hk, 2, device=DEV) for _ in "kv")
        out.append(torch.cat([paged_append(x[p, :, :H], x[p, :, H:H + Hk], x[p, :, H + Hk:], k, v, table[p], start[p], count[p], cos=cos, sin=sin,
                                           qk_scale=1.2, k_scale=ks, v_scale=vs) for p in parts]))
        held.append((k.view(torch.uint8), v.view(torch.uint8), ks, vs))
    assert torch.equal(*out) and all(torch.equal(a, b) for a, b in zip(*held))


# ------------------------------------------------------------------------------------------ the layer
@pytest.mark.parametrize("dtype,d,F,E,k,shared", [
    (torch.bfloat16, 64, 60, 8, 2, 0), (torch.bfloat16, 60, 64, 8, 2, 1), (torch.float16, 64, 40, 20, 17, 1), (torch.bfloat16, 64, 8, 520, 2, 0),
    (torch.bfloat16, 8200, 8, 4, 2, 0), (torch.float32, 64, 32, 8, 2, 1)])
def test_layers_that_the_kernel_does_not_take_decode_through_forward(dtype, d, F, E, k, shared):
    from nexttransformer_b200.models.moe import MoEFFN
    torch.manual_seed(F)
    layer = MoEFFN(d, E, k, F, shared=shared).eval().to(DEV)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0, 0.1)
        x = torch.randn(2, 3, d, device=DEV).to(dtype)
        assert torch.isfinite(layer(x)).all()
        layer.serve(dtype)
        assert layer.step(x).shape == x.shape
        layer.forward = lambda x: x + 1                # (its own sums are atomics, in any order)
        assert torch.equal(layer.step(x), x + 1)


def test_a_step_of_rows_that_are_a_part_of_wider_ones():
    from nexttransformer_b200.models.moe import MoEFFN
    torch.manual_seed(1)
    layer = MoEFFN(64, 8, 2, 32, shared=1).eval().to(DEV)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0, 0.1)
        layer.serve(torch.bfloat16)
        wide = torch.randn(5, 71, device=DEV).bfloat16()
        for rows in (5, 1):
            x = wide[:rows, 3:67]
            assert x.data_ptr() % 16 and torch.equal(layer.step(x), layer.step(x.clone(memory_format=torch.contiguous_format)))


# ------------------------------------------------------------------------------------------ the engine
def test_generation_at_low_temperatures_and_with_large_biases():
    """Answers of a temperature that leaves the largest logit alone are the greedy ones, and a bias of 1e18 settles the choice."""
    from dataclasses import replace
    from nexttransformer_b200.inference import generate_batch
    from nexttransformer_b200.models import build_model
    from nexttransformer_b200.models.config import debug_config
    c = replace(debug_config("dense"), width=256, heads=4, kv_heads=2)
    m = build_model(c, DEV, seed=1).eval()
    with torch.no_grad():
        m.lm_head.weight.normal_(0, 0.3)
    prompts = [[1, 2, 3], [4], list(range(20))]
    greedy = generate_batch(m, prompts, 8, temperature=0.0)
    for T in (1e-15, 1e-18, 1e-20):
        assert generate_batch(m, prompts, 8, temperature=T, top_p=0.9) == greedy
        assert generate_batch(m, prompts, 8, temperature=[T] * 3, top_k=[0, 3, 50], min_p=0.1) == greedy
    for T in (0.7, 1.0):
        assert generate_batch(m, prompts, 4, temperature=T, top_p=0.9, bias={9: 1e18}) == [[9] * 4] * 3
