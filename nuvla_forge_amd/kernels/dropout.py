"""Dropout from a counter-based generator, its mask never stored, on MI355X.

``fused_dropout`` adds an optional residual in the same pass and forms the mask
from the element's index (``nf_dropout``): the backward computes it again.  The
generator is Philox4x32-10; an element takes 16 bits of it, so ``p`` acts in steps
of 2^-16 and kept elements are scaled by the exact inverse of what is kept.

The same ``seed`` and ``offset`` give the same mask on the device and on the host,
for every element type and every stride: it belongs to the element's place in
row-major order.  A program keeps one seed (a step counter, say, in an int64 tensor
on the device: a captured graph reads what it holds at replay) and gives each call
site an offset of its own.
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from .reference import dropout_ref
from .utils import check_devices, device_of, use_fused


def dropout_threshold(p: float) -> int:
    """``p`` in 65536ths, as the kernel takes it."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"fused_dropout: p must be in [0, 1], got {p}")
    return math.floor(p * 65536 + 0.5)


def _check(x, seed, offset, residual):
    _lib.dtype_code(x)
    if not 0 <= offset < 1 << 63:
        raise ValueError(f"fused_dropout: offset must be in [0, 2^63), got {offset}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"fused_dropout: a seed tensor holds one int64, got {seed.numel()} "
                             f"of {seed.dtype}")
    elif not -(1 << 63) <= seed < 1 << 63:
        raise ValueError(f"fused_dropout: seed must fit 64 bits, got {seed}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"fused_dropout: shape mismatch {tuple(x.shape)} vs residual "
                             f"{tuple(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"fused_dropout: residual is {residual.dtype}; expected {x.dtype} or "
                            "float32")
    check_devices("fused_dropout", "x", dict(
        x=x, residual=residual, seed=seed if isinstance(seed, torch.Tensor) else None))


def _launch(x, residual, out, threshold, seed, offset):
    by_ptr = isinstance(seed, torch.Tensor)
    with device_of(x):
        _lib.check(
            _lib.lib().nf_dropout(x.data_ptr(), _lib.ptr(residual), out.data_ptr(), x.numel(),
                                  threshold, seed.data_ptr() if by_ptr else None,
                                  0 if by_ptr else seed, offset, _lib.dtype_code(x),
                                  _lib.dtype_code(out), _lib.stream_of(x)),
            "nf_dropout",
        )
    return out


class _FusedDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed, offset, out_dtype):
        x = x.contiguous()
        r = None if residual is None else residual.contiguous()
        out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
        _launch(x, r, out, threshold, seed, offset)
        ctx.call = (threshold, seed if not isinstance(seed, torch.Tensor) else None, offset)
        ctx.x_dtype = x.dtype
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)  # one changed in place before the backward raises
        return out

    @staticmethod
    def backward(ctx, dout):
        threshold, seed, offset = ctx.call
        if seed is None:
            (seed,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:  # linear in dout, and so the operator once more
            dx = _FusedDropout.apply(dout, None, threshold, seed, offset, ctx.x_dtype)
        return dx, dout if ctx.needs_input_grad[1] else None, None, None, None, None


def fused_dropout(x: torch.Tensor, p: float, seed: int | torch.Tensor, offset: int = 0,
                  residual: torch.Tensor | None = None, force_reference: bool = False
                  ) -> torch.Tensor:
    """``residual + dropout(x, p)`` (``residual`` may be left out).

    Args:
        x: any shape, fp32, bf16 or fp16.
        p: the probability of dropping an element, in steps of 2^-16 (1: all).
        seed: the generator's 64-bit key: an int, or an int64 tensor of one element
            on x's device, read there when the kernel runs.
        offset: the second half of the generator's counter: calls with different
            offsets draw independent masks under one seed.
        residual: same shape, x's type or fp32; the result has its type.
        force_reference: run the eager formulation instead.

    A dropped element gives 0 (or the residual) whatever x holds there.  The mask is
    computed again in the backward, from the seed as it was in the forward: a seed
    tensor that was changed in place in between raises.  Host tensors take the eager
    formulation, with the same mask.  Derivatives of any order.
    """
    threshold = dropout_threshold(p)
    fused = use_fused(x, "fused_dropout", force_reference)
    if fused:  # the plain call runs in C++; any other (None) takes the Function below
        out = _lib.native().dropout(x, residual, threshold, seed, offset)
        if out is not None:
            return out
    _check(x, seed, offset, residual)
    if not fused:
        return dropout_ref(x, threshold, seed, offset, residual)
    return _FusedDropout.apply(x, residual, threshold, seed, offset,
                               x.dtype if residual is None else residual.dtype)
