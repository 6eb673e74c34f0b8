"""Eager PyTorch formulations of the fused ops (``force_reference=True``).

Same names and semantics as ``nuvla_forge/kernels/reference.py``: the
reference's own non-fused path, which its ``force_reference`` switch selects
and its DiT/nuVLA models run with ``fused=False``.  These run on whatever
device the inputs live on, through ATen; they are never chosen implicitly.
The parity oracle the tests use is a separate NumPy restatement (``oracle/``).

The last three (token log probabilities, embedding lookup, dropout) have no
counterpart there.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def _expand_cond(c: torch.Tensor, tokens_per_sample: int) -> torch.Tensor:
    """[B, N] -> [B*T, N]; row m belongs to sample m // T (reference.py:17-19)."""
    return c.repeat_interleave(tokens_per_sample, dim=0)


def adaln_residual_rmsnorm_ref(x, y, gate, weight, scale, shift, tokens_per_sample, eps=1e-6):
    """h = x + gate*y;  out = rmsnorm(h) * w * (1 + scale) + shift  (reference.py:22-66).

    Returns (h, out); out is cast to x.dtype, h keeps the promoted dtype of
    ``x + gate * y`` exactly as the reference's eager expression does.
    """
    t = tokens_per_sample
    g = _expand_cond(gate, t)
    s = _expand_cond(scale, t)
    sh = _expand_cond(shift, t)
    h = x + g * y
    hf = h.float()
    rstd = torch.rsqrt(hf.pow(2).mean(dim=-1, keepdim=True) + eps)
    out = hf * rstd * weight.float() * (1.0 + s.float()) + sh.float()
    return h, out.to(x.dtype)


def swiglu_ref(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """silu(a) * b in fp32, cast to a.dtype (reference.py:69-74)."""
    return (F.silu(a.float()) * b.float()).to(a.dtype)


def chunked_cross_entropy_ref(hidden, lm_weight, targets, ignore_index=-100):
    """Unchunked mean cross entropy over hidden @ lm_weight.T (reference.py:77-96)."""
    logits = F.linear(hidden.float(), lm_weight.float())
    return F.cross_entropy(logits, targets, ignore_index=ignore_index, reduction="mean")


def token_logprobs_ref(hidden, lm_weight, targets, top_k=0, chunk_size=1024, ignore_index=-100):
    """(logprobs, entropy, top_logprobs, top_ids) over hidden @ lm_weight.T in fp32, rows taken
    ``chunk_size`` at a time; the last two are None for ``top_k`` 0.  Rows whose target is
    ``ignore_index`` or outside [0, V) give 0 (and id -1) and no gradient, whatever they hold; a
    logit of -inf has no part in the entropy; alternatives go by their logits, NaN by none."""
    v, w, parts = lm_weight.shape[0], lm_weight.float(), []
    for at in range(0, max(hidden.shape[0], 1), chunk_size):
        tg = targets[at:at + chunk_size]
        live = (tg != ignore_index) & (tg >= 0) & (tg < v)
        # rows left out: zeros before the product (their gradient stops there) and after it (an
        # infinity in w makes a NaN of 0)
        h = torch.where(live[:, None], hidden[at:at + chunk_size], 0.0).float()
        z = torch.where(live[:, None], F.linear(h, w), 0.0)
        logp = z.log_softmax(-1)
        own = logp.gather(1, torch.where(live, tg, 0)[:, None])[:, 0]
        ent = -(logp.exp() * logp.clamp(min=-200.0)).sum(-1)  # exp(-200) is 0: 0 * -inf is not
        got = [torch.where(live, own, 0.0), torch.where(live, ent, 0.0)]
        if top_k:
            idx = torch.sort(z.detach(), dim=-1, descending=True, stable=True)[1]  # NaN first
            place = torch.arange(top_k, device=z.device) + z.isnan().sum(-1, keepdim=True)
            idx = idx.gather(1, place.clamp(max=v - 1))
            got += [torch.where(live[:, None], logp.detach().gather(1, idx), 0.0),
                    torch.where(live[:, None] & (place < v), idx, -1)]
        parts.append(got)
    out = [torch.cat([got[i] for got in parts]) for i in range(len(parts[0]))]
    return tuple(out) if top_k else (*out, None, None)


def embedding_ref(ids, table, scale, padding_idx, out_dtype):
    """scale * table[ids] in fp32, cast to ``out_dtype``; 0 for ids outside [0, V), no gradient
    from positions that hold ``padding_idx``."""
    live = ((ids >= 0) & (ids < table.shape[0]))[..., None]
    rows = table[torch.where(live[..., 0], ids, 0).long()].float()
    if padding_idx is not None:
        rows = torch.where((ids == padding_idx)[..., None], rows.detach(), rows)
    return torch.where(live, rows * scale, 0.0).to(out_dtype)


def _philox_words(seed, block, offset):
    """The four 32-bit words of Philox4x32-10 under key ``seed`` (an int or int64 tensor) for the
    counters (block, offset), as int64."""
    low = 0xFFFFFFFF
    k0, k1 = seed & low, (seed >> 32) & low
    c0, c1 = block & low, (block >> 32) & low
    c2, c3 = (torch.full_like(block, x & low) for x in (offset, offset >> 32))
    for r in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # wraps; the low 64 bits are the product's
        c0, c1, c2, c3 = (((b >> 32) & low) ^ c1 ^ ((k0 + r * 0x9E3779B9) & low), b & low,
                          ((a >> 32) & low) ^ c3 ^ ((k1 + r * 0xBB67AE85) & low), a & low)
    return c0, c1, c2, c3


def dropout_keep(shape, threshold, seed, offset, device):
    """The mask of ``fused_dropout``: True where an element is kept."""
    n = math.prod(shape)
    if isinstance(seed, torch.Tensor):
        seed = seed.reshape(())
    words = torch.stack(_philox_words(seed, torch.arange((n + 7) // 8, device=device), offset), 1)
    parts = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)
    return (parts[:n] >= threshold).view(shape)


def dropout_ref(x, threshold, seed, offset, residual):
    """residual + (kept ? x * 65536 / (65536 - threshold) : 0) in fp32, cast to the residual's
    type (x's without one)."""
    keep = dropout_keep(x.shape, threshold, seed, offset, x.device)
    f = 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0
    y = torch.where(keep, x.float() * f, 0.0)
    return y.to(x.dtype) if residual is None else (y + residual.float()).to(residual.dtype)
