"""A token for each row of next-token logits: temperature, top-k, top-p, min-p, drawn with numbers that the caller gives.

``sample_logits`` is one launch (``csrc/sampling.cu``; CPU tensors run the plain form below), which reads rows of up to 131072 logits once and
longer ones again in each pass.  It has no backward and draws no random numbers of its own, so a call's result depends on its
arguments alone.
"""
import torch

from nexttransformer_b200.ops._ext import ext
from nexttransformer_b200.ops.paged import _inference_only


def sample_logits(logits, uniform, *, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """``(tokens, logprobs)``, int64 and fp32 ``[B]``, of ``logits [B, V]`` (bf16, fp16 or fp32, any row stride; on CUDA
    up to 524288 tokens) and ``uniform [B]``, fp32 numbers in [0, 1).

    With the weights ``w = exp((x - max x) / temperature)`` and tokens ordered by falling logit, equal ones by rising
    index, a row keeps

    * its first ``top_k`` tokens (all, where it is 0 or less),
    * of these, the tokens before which less than ``top_p`` of their mass lies (all, from 1 on),
    * of these, the tokens with ``w >= min_p`` (all, where it is 0 or less; from 1 on those with the largest logit),

    and always the first.  The token is the smallest index up to which more than ``uniform`` of the kept mass lies, its
    logprob the log of its share of that mass.  Masses are exact sums of weights held as whole multiples of 2^-50 of the largest (2^-42 with
    524288 tokens): what lies closer to a border than they do may fall to its other side.  ``temperature``, ``top_p`` and ``min_p`` are numbers or fp32 ``[B]``, ``top_k`` is a
    number or int32 ``[B]``; None leaves a part out (a temperature is 1 then), and so does a NaN in ``top_p`` or ``min_p``.  A
    temperature of 0 or less, or a NaN, takes the first token.  A ``uniform`` outside [0, 1) counts as the nearest number inside, NaN as 0.

    Logits of -inf are never drawn; where the largest are inf, they share the choice.  A row without any permitted token
    gives token -1 (logprob -inf), a row with a NaN -2 (logprob NaN).
    """
    if logits.is_cuda:
        return tuple(ext().sample_logits(logits, uniform, temperature, top_k, top_p, min_p))
    _inference_only(logits, uniform, *(v for v in (temperature, top_k, top_p, min_p) if torch.is_tensor(v)))
    return _plain(logits, uniform, temperature, top_k, top_p, min_p)


def _plain(logits, uniform, temperature, top_k, top_p, min_p):
    if logits.dim() != 2 or logits.shape[1] < 1 or uniform.shape != logits.shape[:1]:
        raise RuntimeError("logits must be [B, V] with contiguous rows, uniform [B]")
    B, V = logits.shape

    def rows(value, none, name):
        if torch.is_tensor(value) and value.shape != (B,):
            raise RuntimeError(f"{name} must have one entry for each row")
        if isinstance(value, float):
            value = torch.tensor(value)  # in 32 bits, as for the kernel
        value = torch.as_tensor(none if value is None else value).double()
        return torch.where(value.isnan(), none, value).expand(B)
    T, k = rows(temperature, 0.0, "temperature"), rows(top_k, 0, "top_k")
    if temperature is None:
        T = torch.ones(B, dtype=torch.float64)
    p, m = rows(top_p, 1.0, "top_p"), rows(min_p, 0.0, "min_p")
    u = uniform.double().nan_to_num(0.0).clamp(0.0, 1.0 - 2.0 ** -24)
    tokens, logprobs = torch.empty(B, dtype=torch.long), torch.empty(B)
    for b in range(B):
        x = logits[b].double()
        top = x.max()
        if x.isnan().any() or top == -torch.inf:
            tokens[b], logprobs[b] = (-2, torch.nan) if x.isnan().any() else (-1, -torch.inf)
            continue
        if top == torch.inf:
            x, top = torch.where(x == torch.inf, 0.0, -torch.inf).double(), 0.0
        order = torch.sort(x, descending=True, stable=True).indices
        if T[b] <= 0:
            tokens[b], logprobs[b] = order[0], 0.0
            continue
        w = torch.where(x == -torch.inf, 0.0, torch.exp((x - top) / T[b]))[order]
        keep = torch.ones(V, dtype=torch.bool)
        if k[b] > 0:
            keep[int(min(k[b], V)):] = False
        w = w * keep
        if p[b] < 1:
            mass = w.cumsum(0)
            keep &= mass - w < p[b] * mass[-1]
        if m[b] > 0:
            keep &= (w >= m[b]) if m[b] < 1 else (x == top)[order]
        keep[0] = True
        kept = torch.zeros(V, dtype=torch.float64).index_add_(0, order, w * keep)
        mass = kept.cumsum(0)
        token = int(torch.searchsorted(mass, u[b] * mass[-1], right=True).clamp(max=int(kept.nonzero()[-1])))
        tokens[b], logprobs[b] = token, torch.log(kept[token] / mass[-1])
    return tokens, logprobs
