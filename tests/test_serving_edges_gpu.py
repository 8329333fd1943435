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
