"""Attention with its gradient on MI355X.

``fused_attention`` makes one pass over the keys with a running maximum and sum
(``nf_attention_fwd``): the probabilities are never stored, and the backward
(``nf_attention_bwd``) forms them again from each row's log-sum-exp.  Query, key and
value are read where a projection left them, [B, T, heads, D] with any strides; the
query heads of a group share a key head, whose gradients sum over them in a fixed
order: the same bits every run.  A few query rows over many keys (one generated token
for each request, a planner's waypoints) are split along the keys and joined.
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from .reference import attention_ref
from .utils import check_devices, device_of, first_order_only, use_fused

MAX_HEAD = 128  # widest head the kernels take
MAX_SCALE = 2.0 ** 127  # times log2(e) is still an fp32 number


def _vector_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` where its rows are whole 16-byte vectors (zeros past D), a copy of it where not."""
    e, d = 16 // t.element_size(), t.shape[-1]
    far = (1 << 30) // t.element_size()
    sb, st, sh = (0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3]))
    whole = (d % e == 0 and t.data_ptr() % 16 == 0 and (t.stride(-1) == 1 or d == 1)
             and not (sb % e or st % e or sh % e)
             and st <= far // 512 and 130 * st + t.shape[2] * sh < far)
    if whole:
        return t
    # written out, not padded by the library: that keeps the order of t's axes, the tokens
    # innermost where they are
    rows = torch.empty(*t.shape[:3], d + -d % e, dtype=t.dtype, device=t.device)
    rows[..., :d] = t
    rows[..., d:] = 0
    return rows


def _strides(t: torch.Tensor) -> list[int]:
    return [0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])]


def _mask(key_mask):
    """``key_mask`` with its keys side by side, and the bytes from sample to sample."""
    if key_mask is None:
        return None, 0
    m = key_mask if key_mask.stride(1) == 1 or key_mask.shape[1] == 1 else key_mask.contiguous()
    return m, 0 if m.shape[0] == 1 else m.stride(0)


class _FusedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, causal, scale, keep):
        b, tq, h, d = q.shape
        tk, hk = k.shape[1:3]
        q2, k2, v2 = (_vector_rows(t) for t in (q, k, v))
        mask, mask_b = _mask(key_mask)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dt, L = _lib.dtype_code(q), _lib.lib()
        sizes = (b, tq, tk, h, hk, d)
        n_state = L.nf_attention_state_bytes(*sizes, dt) if keep else 0
        n_ws = L.nf_attention_fwd_workspace(*sizes, causal, dt)
        state, ws = (torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
                     for n in (n_state, n_ws))
        with device_of(q):
            _lib.check(
                L.nf_attention_fwd(q2.data_ptr(), *_strides(q2), k2.data_ptr(), *_strides(k2),
                                   v2.data_ptr(), *_strides(v2), _lib.ptr(mask), mask_b, *sizes,
                                   causal, scale, dt, out.data_ptr(), _lib.ptr(state), n_state,
                                   _lib.ptr(ws), n_ws, _lib.stream_of(q)),
                "nf_attention_fwd",
            )
        if keep:
            ctx.save_for_backward(q2, k2, v2, out, state, mask)
            ctx.call = (sizes, causal, scale)
        return out

    @staticmethod
    def backward(ctx, grad):
        q, k, v, out, state, key_mask = ctx.saved_tensors
        # what a saved-tensor hook gives back may lie in memory in another way
        q, k, v, out, state = (*map(_vector_rows, (q, k, v)), out.contiguous(), state.contiguous())
        sizes, causal, scale = ctx.call
        b, tq, tk, h, hk, d = sizes
        check_devices("fused_attention backward", "the forward's q", dict(dout=grad),
                      device=q.device)
        g = _vector_rows(grad.to(q.dtype))
        mask, mask_b = _mask(key_mask)
        dq, dk, dv = (torch.empty(shape, dtype=q.dtype, device=q.device) if need else None
                      for shape, need in zip(((b, tq, h, d), (b, tk, hk, d), (b, tk, hk, d)),
                                             ctx.needs_input_grad))
        dt, L = _lib.dtype_code(q), _lib.lib()
        n_ws = L.nf_attention_bwd_workspace(*sizes, causal, dt)
        ws = torch.empty(n_ws, dtype=torch.uint8, device=q.device)
        with device_of(q):
            _lib.check(
                L.nf_attention_bwd(q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k),
                                   v.data_ptr(), *_strides(v), _lib.ptr(mask), mask_b,
                                   out.data_ptr(), g.data_ptr(), *_strides(g), *sizes, causal,
                                   scale, dt, state.data_ptr(), state.numel(), _lib.ptr(dq),
                                   _lib.ptr(dk), _lib.ptr(dv), ws.data_ptr(), n_ws,
                                   _lib.stream_of(q)),
                "nf_attention_bwd",
            )
        return first_order_only("fused_attention", (grad,), (dq, dk, dv, None, None, None, None))


def _check(q, k, v, key_mask, scale):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"fused_attention: {name} [B, T, heads, D] expected, got "
                             f"{tuple(t.shape)}")
        _lib.dtype_code(t)
        if t.dtype != q.dtype:
            raise TypeError(f"fused_attention: {name} is {t.dtype}; expected q's {q.dtype}")
    if v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"fused_attention: shape mismatch: q {tuple(q.shape)}, k "
                         f"{tuple(k.shape)}, v {tuple(v.shape)}")
    if q.shape[3] == 0 or k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"fused_attention: {q.shape[2]} query heads over {k.shape[2]} key heads "
                         f"of {q.shape[3]}")
    if key_mask is not None:
        if key_mask.dtype != torch.bool:
            raise TypeError(f"fused_attention: key_mask is {key_mask.dtype}; expected bool")
        if key_mask.shape != k.shape[:2]:
            raise ValueError(f"fused_attention: key_mask [B, Tk] = {tuple(k.shape[:2])} expected, "
                             f"got {tuple(key_mask.shape)}")
    if not abs(scale) <= MAX_SCALE:
        raise ValueError(f"fused_attention: scale must be finite in fp32 (at most 2^127), got {scale}")
    check_devices("fused_attention", "q", dict(q=q, k=k, v=v, key_mask=key_mask))


def fused_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False,
                    key_mask: torch.Tensor | None = None, scale: float | None = None,
                    force_reference: bool = False) -> torch.Tensor:
    """``softmax(scale q k^T) v`` over the keys that each row may attend.

    Args:
        q: [B, Tq, H, D], fp32, bf16 or fp16; any strides.  q, k and v are read where they
            lie if their rows are whole 16-byte vectors, a token's stride is at most 2 MiB, and
            130 token strides and the heads' strides together span less than 1 GiB; else a
            copy is made in each call (a cache stored head by head, [B, Hk, T, D], from 1 GiB
            a sample on).
        k, v: [B, Tk, Hk, D], q's type; H a multiple of Hk, up to 32768 times it: query head h
            attends key head h // (H / Hk).  At most about 2^28 keys over all samples' key heads,
            and as many rows.
        causal: query i attends keys up to i + Tk - Tq: the last query sees every key.
        key_mask: bool [B, Tk]; False: no query attends the key.  What such a key and its
            value hold, NaN or infinity too, changes no bit of any result (the unfilled part of
            a cache, padding).
        scale: multiplies the logits, in fp32; 1 / sqrt(D) by default.
        force_reference: run the eager formulation instead.

    Returns:
        [B, Tq, H, D], contiguous, q's type.  A row that may attend no key gives zeros and
        takes no part in any gradient, whatever its query and its output's gradient hold.

    Logits, statistics and sums are fp32; for their products the probabilities (and the logits'
    gradients) are rounded to the inputs' type, or to two terms of it where few rows or keys
    make a block's waves share them: a sample's 16-bit results may differ by that rounding with the
    size of the batch that it is in.  A NaN or an infinity in a key or value that some row may
    attend, or in the query or the gradient of a row that attends one, can reach other rows of its
    head and the gradients of other keys in the same sample.  First derivatives only on the device.
    Host tensors, heads wider than 128 and calls without a key take the eager formulation.
    """
    fused = use_fused(q, "fused_attention", force_reference)
    s = None if scale is None else float(scale)
    if s is None and q.dim() == 4 and q.shape[3]:
        s = 1.0 / math.sqrt(q.shape[3])
    if fused and s is not None:  # the plain call runs in C++; any other (None) takes what follows
        out = _lib.native().attention(q, k, v, key_mask, bool(causal), s)
        if out is not None:
            return out
    _check(q, k, v, key_mask, 1.0 if s is None else s)
    if not fused or q.shape[3] > MAX_HEAD or q.numel() == 0 or k.numel() == 0:
        return attention_ref(q, k, v, bool(causal), key_mask, s)
    keep = torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v))
    return _FusedAttention.apply(q, k, v, key_mask, bool(causal), s, keep)
