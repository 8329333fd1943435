"""Edges of the decoding operators that need no GPU."""
import pytest
import torch

from nexttransformer_b200.ops.moe import tokens_supported


@pytest.mark.parametrize("change,taken", [
    ({}, True), (dict(dtype=torch.float16, Fs=24), True), (dict(d=8, F=8, E=1, top_k=1), True), (dict(d=8192, E=512, top_k=16), True),
    (dict(dtype=torch.float32), False), (dict(d=60), False), (dict(d=8200), False), (dict(F=60), False), (dict(F=65544), False), (dict(E=513), False),
    (dict(E=32, top_k=17), False), (dict(Fs=20), False)])
def test_what_the_experts_of_a_few_tokens_take(change, taken):
    assert tokens_supported(**dict(dict(dtype=torch.bfloat16, d=64, F=32, E=8, top_k=2), **change)) is taken
