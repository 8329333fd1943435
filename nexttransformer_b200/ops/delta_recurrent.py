"""The gated delta rule in its recurrent form, with a state carried from call to call.

``delta_recurrent`` runs DeltaNet (no decay), Gated DeltaNet (a log decay per head) and KDA (one per
feature) token by token on ``state [states, H, D, D]`` (fp32, updated in place):

    S <- diag(e^g) S,   S <- S + k (beta (v - k^T S))^T,   o = q^T S

It is the form for decoding and for prompts that have to leave their final state; training uses the chunk
form of ``ops.linear_attention``.  On CUDA a run of tokens is taken eight at a time from the call's start, so a run
cut elsewhere than behind a multiple of eight gives the same up to rounding, not bit for bit.  CUDA tensors run ``csrc/delta_step.cu`` (bf16, fp16 or fp32, heads of 64 or
128), CPU tensors ``models.linear.recurrent_scan``.  It has no backward.
"""
import torch
import torch.nn.functional as F

from nexttransformer_b200.ops._ext import ext
from nexttransformer_b200.ops.paged import _inference_only


def delta_recurrent(q, k, v, state, beta, g=None, *, scale=1.0, l2norm=False, slots=None, count=None):
    """Outputs ``[B, T, H, D]`` of T tokens per row; ``state`` holds the rows' states afterwards.

    ``q``, ``k``, ``v [B, T, H, D]``, ``beta [B, T, H]``, ``g`` (fp32 log decay) ``[B, T, H]`` or
    ``[B, T, H, D]``.  Queries are scaled by ``scale``; with ``l2norm`` queries and keys are L2-normalised
    before.  ``slots [B]`` (int32): the state of each row (row b's is b by default; a negative one leaves the
    row out; no two rows share one).  ``count [B]``: how many of a row's T tokens are real; the others change
    nothing and give zeros.
    """
    if q.is_cuda:
        return ext().delta_step(q, k, v, state, beta, g, scale, l2norm, slots, count)
    _inference_only(q, k, v, state, beta, g)
    return _plain(q, k, v, state, beta, g, scale, l2norm, slots, count)


def _plain(q, k, v, state, beta, g, scale, l2norm, slots, count):
    from nexttransformer_b200.models.linear import recurrent_scan
    B, T, H, D = q.shape
    if k.shape != q.shape or v.shape != q.shape or beta.shape != q.shape[:3]:
        raise RuntimeError("q, k and v must be [B, T, H, D], beta [B, T, H]")
    if g is not None and g.shape not in (q.shape, q.shape[:3]):
        raise RuntimeError("g must be an fp32 log decay, [B, T, H] or [B, T, H, D]")
    if state.dtype != torch.float32 or state.shape[1:] != (H, D, D) or (slots is None and state.shape[0] < B):
        raise RuntimeError("state must be contiguous fp32 [states, H, D, D]")
    if l2norm:
        q, k = F.normalize(q.float(), dim=-1), F.normalize(k.float(), dim=-1)
    out = torch.zeros(v.shape, dtype=v.dtype)
    kind = "deltanet" if g is None else "gdn" if g.dim() == 3 else "kda"
    for b in range(B):
        s, n = b if slots is None else int(slots[b]), T if count is None else max(0, min(int(count[b]), T))
        if s >= state.shape[0]:
            raise RuntimeError(f"delta_recurrent: slot outside the states (row {b})")
        if s < 0 or n == 0:
            continue
        decay = None if g is None else g[b:b + 1, :n].exp()
        decay = decay.unsqueeze(-1) if kind == "gdn" else decay
        o, final = recurrent_scan(q[b:b + 1, :n].float() * scale, k[b:b + 1, :n].float(), v[b:b + 1, :n].float(),
                                  kind=kind, decay=decay, beta=beta[b:b + 1, :n].float(),
                                  initial_state=state[s:s + 1])
        out[b, :n] = o[0].to(v.dtype)
        state[s] = final[0]
    return out
