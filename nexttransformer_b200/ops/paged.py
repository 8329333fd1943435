"""Paged key-value cache: appending rotated keys and values, and attention over the pages.

Keys and values lie in pages ``[P, Hk, page, D]`` (bf16 or fp16, heads of 64 or 128, ``page`` a multiple of
16): token ``p`` of row ``b`` is in page ``table[b, p // page]`` at slot ``p % page``.  ``start [B]`` (int32)
is how many tokens a row holds before the call (negative: the row is left out), ``count [B]`` how many of the call's
``t`` tokens are real (all by default); what stands behind a row's count is neither written nor attended to and gives
zeros.  Strides are free as long as rows, tokens and heads start on 16-byte boundaries.

Pages may also be held in 8 bits (``float8_e4m3fn``) beside bf16 or fp16 queries.  Then ``k_scale`` and ``v_scale``, fp32
``[P, Hk, page / 16]``, go with them: 16 tokens of a page and head share a scale, and a key is its code times its scale.
``paged_append`` chooses it: the smallest power of two (2^-100 to 2^120) whose 448-fold reaches the largest number that the
block's tokens had so far; a call that begins a block chooses anew, one that continues it may raise the scale, and then
the block's earlier codes are written again.  So a block of 16 tokens takes tokens of one row only in a call, and no other call
at the same time.  What is not finite becomes NaN and does not count for the scale.  Blocks may share a scale in memory where it is only
read, by ``paged_attention``.

* ``paged_append``    rotates and QK-normalises new queries and keys, adds the gated value embedding, writes
  keys and values into the pages and returns the queries;
* ``paged_attention`` attends from the new tokens to the row's keys, causally and through an optional left
  window.

CUDA tensors run the kernels of ``csrc/paged.cu``; CPU tensors the plain form below, in any float type.  The
kernels check positions and page numbers themselves: nothing is written to a page outside the cache, keys in one (or
behind the table) take no part in the softmax, and ``ops._ext.check_errors`` raises for it; the plain form raises at once.
Neither operator has a backward.
"""
import torch

from nexttransformer_b200.ops._ext import ext


def _inference_only(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("serving operators have no backward: call them under torch.no_grad()")


def paged_append(q, k, v, k_pages, v_pages, table, start, count=None, *, cos, sin, qk_scale=None, ve=None,
                 ve_gate=None, k_scale=None, v_scale=None):
    """Write the new tokens' keys and values into the pages; return the rotated queries ``[B, t, H, D]``.

    ``q [B, t, H, D]``, ``k`` / ``v [B, t, Hk, D]``: raw projections, which may be slices of one.
    ``cos`` / ``sin [positions, D / 2]``: queries and keys are rotated by -theta at their position, then, with
    ``qk_scale``, RMS-normalised and scaled by it.  ``ve`` (like ``v``) and ``ve_gate [B, t, Hk]``: values
    become ``v + 3 sigmoid(ve_gate) ve``.
    """
    if q.is_cuda:
        return ext().paged_append(q, k, v, k_pages, v_pages, table, start, count, cos, sin, qk_scale, ve, ve_gate, k_scale,
                                  v_scale)
    _inference_only(q, k, v, k_pages, v_pages, cos, sin, ve, ve_gate, k_scale, v_scale)
    return _append_plain(q, k, v, k_pages, v_pages, table, start, count, cos, sin, qk_scale, ve, ve_gate, k_scale, v_scale)


def paged_attention(q, k_pages, v_pages, table, start, count=None, *, window=-1, scale=None, k_scale=None, v_scale=None):
    """Attention of the new tokens ``q [B, t, H, D]`` over the pages, which hold their keys already.

    Token ``i`` of a row stands at position ``start + i`` and sees the positions up to its own, with
    ``window >= 0`` at most ``window`` back.  ``scale`` defaults to ``D ** -0.5``.  Keys and values that one of a
    call's tokens sees have to be finite: one that only some of them see meets the others with probability zero,
    which does not remove a NaN.  What no token sees (behind the row's tokens, before every window) may hold anything.
    A query with a NaN gives NaN, and so does one with a score of inf; where every score is -inf the kernel gives zeros, as
    for a token without keys (the plain form NaN).

    Sums are fp32.  Over pages in 8 bits a probability is one fp16 number beside bf16 queries (2^-11 of it, below the output's rounding), two beside
    fp16 ones.
    """
    if q.is_cuda:
        return ext().paged_attention(q, k_pages, v_pages, table, start, count, window, scale, k_scale, v_scale)
    _inference_only(q, k_pages, v_pages, k_scale, v_scale)
    return _attention_plain(q, k_pages, v_pages, table, start, count, window, scale, k_scale, v_scale)


# ------------------------------------------------------------------------------ plain form (CPU)
BLOCK = 16  # tokens that share a scale


def _check_plain(q, k_pages, v_pages, table, start, count, k_scale, v_scale):
    if q.dim() != 4 or k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] != q.shape[3]:
        raise RuntimeError("q [B, t, H, D] and pages [P, Hk, page, D] expected")
    if q.shape[2] % k_pages.shape[1]:
        raise RuntimeError("KV heads must divide query heads")
    if k_pages.shape[2] % 16:
        raise RuntimeError("tokens per page must be a multiple of 16")
    f8 = k_pages.dtype == torch.float8_e4m3fn
    if (v_pages.dtype == torch.float8_e4m3fn) != f8 or f8 != (k_scale is not None) or f8 != (v_scale is not None):
        raise RuntimeError("float8_e4m3fn pages go with k_scale and v_scale, other pages without")
    for s in (k_scale, v_scale) if f8 else ():
        if s.dtype != torch.float32 or s.shape != (*k_pages.shape[:2], k_pages.shape[2] // BLOCK):
            raise RuntimeError("k_scale and v_scale must be fp32 [P, Hk, page / 16]")
    B, t = q.shape[:2]
    if table.shape[0] != B or start.shape != (B,) or (count is not None and count.shape != (B,)):
        raise RuntimeError("table, start and count must have one entry for each row")
    counts = [t] * B if count is None else [max(0, min(int(c), t)) for c in count]
    starts = [int(s) for s in start]
    return starts, [n if s >= 0 else 0 for s, n in zip(starts, counts)]


def _pages_of(table, b, positions, k_pages):
    page = k_pages.shape[2]
    if len(positions) and int(positions[-1]) // page >= table.shape[1]:
        raise RuntimeError(f"paged cache: a position lies behind the row's page table (row {b})")
    at = table[b].long()[positions // page]
    if len(at) and not (0 <= int(at.min()) and int(at.max()) < k_pages.shape[0]):
        raise RuntimeError(f"paged cache: a page number lies outside the cache (row {b})")
    return at, slice(None), positions % page


def _append_coded(x, pages, scale, at, first):
    """Tokens ``x [n, Hk, D]`` of a row, the first at slot ``first`` of a block, into 8-bit pages at ``at``."""
    page, head, slot = at
    for low in range(-first, len(x), BLOCK):                     # a block's first slot, as a token of the call
        new = slice(max(low, 0), low + BLOCK)
        p, begin = page[new][0], int(slot[new][0]) // BLOCK * BLOCK
        y = x[new].float().transpose(0, 1)                       # [Hk, tokens, D]
        y = torch.where(y.isfinite(), y, torch.nan)
        fraction, exponent = torch.frexp(y.abs().nan_to_num(0.0).amax((1, 2)))
        need = torch.where(fraction > 0, exponent - 9 + (fraction > 0.875).int(), -100).clamp(-100, 120)  # 448 = 0.875 2^9
        need = torch.ldexp(torch.ones(len(need)), need)
        if low < 0:
            old = scale[p, :, begin // BLOCK].clone()
            need = torch.maximum(need, old)
            codes = pages[p, :, begin:begin - low].float() * (old / need)[:, None, None]
            pages[p, :, begin:begin - low] = codes.to(pages.dtype)
        scale[p, :, begin // BLOCK] = need
        pages[p, :, int(slot[new][0]):int(slot[new][0]) + y.shape[1]] = (y / need[:, None, None]).to(pages.dtype)


def _decoded(pages, scale, at):
    """Keys or values at ``at`` of 8-bit pages, as the numbers that they stand for."""
    page, head, slot = at
    return pages.view(torch.uint8)[at].view(pages.dtype).float() * scale[page, :, slot // BLOCK][..., None]


def _append_plain(q, k, v, k_pages, v_pages, table, start, count, cos, sin, qk_scale, ve, ve_gate, k_scale, v_scale):
    from nexttransformer_b200.models.shell import apply_rotary_emb, norm
    starts, counts = _check_plain(q, k_pages, v_pages, table, start, count, k_scale, v_scale)
    if any(n > 1 and step == 0 for s in (k_scale, v_scale) if s is not None for n, step in zip(s.shape, s.stride())):
        raise RuntimeError("blocks may not share a scale in memory")
    if (ve is None) != (ve_gate is None):
        raise RuntimeError("ve and ve_gate go together")
    if ve is not None:
        v = v + 3 * torch.sigmoid(ve_gate)[..., None] * ve
    out = torch.zeros(q.shape, dtype=q.dtype)
    for b, (s, n) in enumerate(zip(starts, counts)):
        if s + n > cos.shape[0] and n:
            raise RuntimeError(f"paged cache: a position lies behind the rotary table (row {b})")
        positions = torch.arange(s, s + n)
        turn = cos[positions][:, None], sin[positions][:, None]
        qb, kb = apply_rotary_emb(q[b, :n], *turn), apply_rotary_emb(k[b, :n], *turn)
        if qk_scale is not None:
            qb, kb = norm(qb) * qk_scale, norm(kb) * qk_scale
        at = _pages_of(table, b, positions, k_pages)
        out[b, :n] = qb
        if k_scale is not None:
            if n:
                _append_coded(kb, k_pages, k_scale, at, s % BLOCK)
                _append_coded(v[b, :n], v_pages, v_scale, at, s % BLOCK)
            continue
        k_pages[at] = kb.to(k_pages.dtype)
        v_pages[at] = v[b, :n].to(v_pages.dtype)
    return out


def _attention_plain(q, k_pages, v_pages, table, start, count, window, scale, k_scale, v_scale):
    starts, counts = _check_plain(q, k_pages, v_pages, table, start, count, k_scale, v_scale)
    B, t, H, D = q.shape
    Hk = k_pages.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=q.dtype)
    for b, (s, n) in enumerate(zip(starts, counts)):
        if not n:
            continue
        key = torch.arange(max(0, s - window) if window >= 0 else 0, s + n)   # what one of the tokens sees
        at = _pages_of(table, b, key, k_pages)
        if k_scale is not None:
            K, V = _decoded(k_pages, k_scale, at).transpose(0, 1), _decoded(v_pages, v_scale, at).transpose(0, 1)
        else:
            K, V = k_pages[at].transpose(0, 1).float(), v_pages[at].transpose(0, 1).float()  # [Hk, keys, D]
        Q = q[b, :n].float().reshape(n, Hk, H // Hk, D).permute(1, 2, 0, 3)                  # [Hk, g, n, D]
        position = torch.arange(s, s + n)[:, None]
        seen = key <= position
        if window >= 0:
            seen = seen & (key >= position - window)
        score = (Q @ K[:, None].transpose(-1, -2) * scale).masked_fill(~seen, -torch.inf)
        out[b, :n] = (torch.softmax(score, -1) @ V[:, None]).permute(2, 0, 1, 3).reshape(n, H, D).to(q.dtype)
    return out
