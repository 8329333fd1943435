"""What a serving loop does to next-token logits before it samples: penalties, biases, a grammar mask.

``adjust_logits`` is one pass over the logits (``csrc/logits.cu``; CPU tensors run the plain form below).  It
has no backward.
"""
import torch

from nexttransformer_b200.ops._ext import ext
from nexttransformer_b200.ops.paged import _inference_only


def adjust_logits(logits, *, tokens=None, length=None, prompt=None, repetition=None, presence=None, frequency=None,
                  bias_ids=None, bias=None, allowed=None):
    """fp32 logits ``[B, V]`` of ``logits [B, V]`` (bf16, fp16 or fp32, any row stride), in this order:

    * tokens that occur in the row's history ``tokens [B, L]`` (int32; the first ``length [B]`` count, ids
      outside the vocabulary are ignored): ``x / repetition`` where ``x > 0``, ``x * repetition`` elsewhere;
    * tokens that occur ``n`` times in the answer, which is the history without its first ``prompt [B]``
      tokens: ``x - frequency n - presence``;
    * ``x + bias`` for the ids in ``bias_ids [B, K]`` (outside the vocabulary: ignored; repeated: all are added);
    * ``-inf`` where the bit of ``allowed [B, ceil(V / 32)]`` (int32, token ``i`` in bit ``i % 32`` of word
      ``i // 32``) is 0, whatever the logit is.  A row that allows nothing is ``-inf`` throughout.

    ``repetition``, ``presence`` and ``frequency`` are fp32 ``[B]``; what is None is left out.
    """
    if logits.is_cuda:
        return ext().adjust_logits(logits, tokens, length, prompt, repetition, presence, frequency, bias_ids, bias,
                                   allowed)
    _inference_only(logits, repetition, presence, frequency, bias)
    return _plain(logits, tokens, length, prompt, repetition, presence, frequency, bias_ids, bias, allowed)


def _plain(logits, tokens, length, prompt, repetition, presence, frequency, bias_ids, bias, allowed):
    if logits.dim() != 2:
        raise RuntimeError("logits must be [B, V] with contiguous rows")
    if (bias_ids is None) != (bias is None):
        raise RuntimeError("bias_ids and bias go together")
    B, V = logits.shape
    if allowed is not None and (allowed.shape[0] != B or allowed.shape[1] < -(-V // 32)):
        raise RuntimeError("allowed must be [B, ceil(V / 32)]")
    x = logits.float().clone()
    for b in range(B):
        if tokens is not None:
            n = tokens.shape[1] if length is None else max(0, min(int(length[b]), tokens.shape[1]))
            first = 0 if prompt is None else max(0, min(int(prompt[b]), n))
            history, at = tokens[b, :n].long(), torch.arange(n)
            known = (history >= 0) & (history < V)
            times = torch.bincount(history[known & (at >= first)], minlength=V)
            seen = torch.bincount(history[known], minlength=V) > 0
            if repetition is not None:
                x[b] = torch.where(seen, torch.where(x[b] > 0, x[b] / repetition[b], x[b] * repetition[b]), x[b])
            if frequency is not None:
                x[b] = torch.where(times > 0, x[b] - frequency[b] * times, x[b])
            if presence is not None:
                x[b] = torch.where(times > 0, x[b] - presence[b], x[b])
        if bias is not None:
            known = (bias_ids[b] >= 0) & (bias_ids[b] < V)
            x[b].index_add_(0, bias_ids[b][known].long(), bias[b][known])
        if allowed is not None:
            ids = torch.arange(V)
            x[b] = torch.where((allowed[b].long()[ids // 32] >> (ids % 32)) & 1 == 1, x[b], -torch.inf)
    return x
