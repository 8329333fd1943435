"""Edges of the decoding operators that need no GPU."""
import pytest
import torch

from nexttransformer_b200.ops.moe import tokens_supported
from nexttransformer_b200.ops.paged import paged_attention


@pytest.mark.parametrize("change,taken", [
    ({}, True), (dict(dtype=torch.float16, Fs=24), True), (dict(d=8, F=8, E=1, top_k=1), True), (dict(d=8192, E=512, top_k=16), True),
    (dict(dtype=torch.float32), False), (dict(d=60), False), (dict(d=8200), False), (dict(F=60), False), (dict(F=65544), False), (dict(E=513), False),
    (dict(E=32, top_k=17), False), (dict(Fs=20), False)])
def test_what_the_experts_of_a_few_tokens_take(change, taken):
    assert tokens_supported(**dict(dict(dtype=torch.bfloat16, d=64, F=32, E=8, top_k=2), **change)) is taken


def test_a_step_calls_the_forward_hooks_of_a_layer():
    from nexttransformer_b200.models.moe import MoEFFN
    torch.manual_seed(2)
    layer, x, seen = MoEFFN(32, 8, 3, 24, shared=1).eval(), torch.randn(5, 32), []
    with torch.no_grad():
        layer.serve(torch.float32)
        plain = layer.step(x)
        for register, value in ((layer.register_forward_hook, lambda m, a, out: seen.append(out)),
                                (layer.register_forward_pre_hook, lambda m, a: seen.append(a[0]))):
            hook = register(value)
            out = layer.step(x)
            assert len(seen) == 1 and seen.pop() is (out if register == layer.register_forward_hook else x)
            hook.remove()
        assert torch.equal(layer.step(x), plain) and not seen


def test_attention_in_8_bits_reads_scales_that_share_memory():
    torch.manual_seed(4)
    k, v = (torch.randn(3, 2, 32, 16).mul(60).to(torch.float8_e4m3fn) for _ in "kv")
    q, table, start = torch.randn(1, 1, 4, 16), torch.tensor([[2, 0]], dtype=torch.int32), torch.tensor([50], dtype=torch.int32)
    one, heads = torch.full((1, 1, 1), 2.0 ** -5).expand(3, 2, 2), torch.tensor([2.0 ** -6, 2.0 ** -4])[None, :, None].expand(3, 2, 2)
    got = paged_attention(q, k, v, table, start, k_scale=one, v_scale=heads)
    assert torch.equal(got, paged_attention(q, k, v, table, start, k_scale=one.contiguous(), v_scale=heads.contiguous()))
