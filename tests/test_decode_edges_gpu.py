"""Edges of the decoding operators on the GPU: rows, weights and values where a kernel's ways of computing part, against 64 bits."""
import math

import pytest
import torch

from tests.test_decode_ops_gpu import both

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
