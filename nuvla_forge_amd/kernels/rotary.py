"""Rotary positions over several axes (time, height, width) on MI355X.

``fused_rotary`` turns the heads of q and k in one launch (``nf_rotary``), each pair by
the coordinate of its axis: the angles are formed in the kernel, once a token, in 64 bits,
so there is no table to keep and no last position that one would hold.  The gradient turns back.
"""

from __future__ import annotations

import ctypes
import math

import torch

from .. import _lib
from .reference import rotary_ref
from .utils import check_devices, device_of, use_fused

MAX_PAIRS, MAX_HEAD = 256, 1024  # pairs and elements of a head that the kernel takes
_POS_KIND = {torch.int64: 0, torch.int32: 1, torch.float32: 2}


def _rows(t):
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _launch(q, k, positions, call, inverse):
    """q and k (either may be None) turned."""
    sections, base, joint, interleaved = call
    like = q if q is not None else k
    outs = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)
            for t in (q, k)]
    args = []
    for t, out in zip((q, k), outs):
        t = _rows(t)
        args += ([None, 0, 0, 0, None, 0] if t is None
                 else [t.data_ptr(), *t.stride()[:3], out.data_ptr(), t.shape[2]])
    b, t, _, d = like.shape
    shared = positions.dim() == 2 or positions.shape[0] == 1
    with device_of(like):
        _lib.check(
            _lib.lib().nf_rotary(*args, positions.data_ptr(),
                                 0 if shared else t * positions.shape[-1],
                                 _POS_KIND[positions.dtype], b, t, d,
                                 (ctypes.c_int32 * len(sections))(*sections), len(sections), base,
                                 joint, interleaved, inverse, _lib.dtype_code(like),
                                 _lib.stream_of(like)),
            "nf_rotary",
        )
    return tuple(outs)


class _FusedRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, call, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)  # one changed in place before the backward raises
        ctx.call = (call, inverse)
        return _launch(q, k, positions, call, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        positions = positions.contiguous()  # a saved-tensor hook may have moved them
        call, inverse = ctx.call
        want = [g if need else None for g, need in zip((dq, dk), ctx.needs_input_grad)]
        check_devices("fused_rotary backward", "the forward's positions",
                      dict(dq=want[0], dk=want[1]), device=positions.device)
        if want != [None, None]:  # linear: the operator once more, the other way
            want = _FusedRotary.apply(*want, positions, call, not inverse)
        return *want, None, None, None


def _check(q, k, positions, sections, base, ladder):
    for name, t in (("q", q), ("k", k)):
        if t is None:
            continue
        if t.dim() != 4:
            raise ValueError(f"fused_rotary: {name} [B, T, heads, D] expected, got "
                             f"{tuple(t.shape)}")
        _lib.dtype_code(t)
        if t.dtype != q.dtype:
            raise TypeError(f"fused_rotary: {name} is {t.dtype}; expected q's {q.dtype}")
        if t.shape[:2] != q.shape[:2] or t.shape[3] != q.shape[3]:
            raise ValueError(f"fused_rotary: shape mismatch {tuple(q.shape)} vs {name} "
                             f"{tuple(t.shape)}")
    if ladder not in ("axis", "joint"):
        raise ValueError(f"fused_rotary: ladder is {ladder!r}; expected 'axis' or 'joint'")
    if not 1 <= len(sections) <= 4 or any(n < 0 for n in sections):
        raise ValueError(f"fused_rotary: sections {tuple(sections)}: 1 to 4 numbers of pairs "
                         "expected")
    if not 1 <= sum(sections) <= q.shape[3] // 2:
        raise ValueError(f"fused_rotary: {sum(sections)} pairs in heads of {q.shape[3]}")
    if not (base > 0.0 and math.isfinite(base)):
        raise ValueError(f"fused_rotary: base must be positive, got {base}")
    if positions.dtype not in _POS_KIND:
        raise TypeError(f"fused_rotary: positions are {positions.dtype}; expected int64, int32 or "
                        "float32")
    n, (b, t) = len(sections), q.shape[:2]
    if positions.shape not in ((t, n), (1, t, n), (b, t, n)):
        raise ValueError(f"fused_rotary: positions [B, T, axes] = {(b, t, n)} or [T, axes] "
                         f"expected, got {tuple(positions.shape)}")
    check_devices("fused_rotary", "q", dict(q=q, k=k, positions=positions))


def fused_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, sections,
                 base: float = 10000.0, ladder: str = "axis", interleaved: bool = False,
                 force_reference: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q and k with every pair of a head turned by its token's position.

    Args:
        q: [B, T, H, D], fp32, bf16 or fp16, any strides.
        k: [B, T, Hk, D], q's type, or None.
        positions: [B, T, axes] or [T, axes], int64, int32 or fp32 (fractions of a patch):
            each token's coordinates.  They take no gradient.
        sections: how many pairs each axis (1 to 4 of them) turns, in the order of the
            pairs; their sum P is at most D / 2, and elements past 2 P stay as they are.
        base, ladder: pair frequencies.  "axis": ``base ** (-i / n)`` for the i-th of an
            axis's n pairs, a ladder for each axis (images, video).  "joint":
            ``base ** (-j / P)`` for the j-th of all pairs, so that a token with equal
            coordinates (text) turns as by one position.
        interleaved: pair j is elements (2 j, 2 j + 1) instead of (j, P + j).
        force_reference: run the eager formulation instead.

    Returns:
        (q, k) turned, contiguous; k is None where it was.

    Angles are formed in 64 bits: those of up to about 2^27 turns to fp32's precision, farther
    ones off by 2^-52 of themselves.  Linear in q and k: derivatives of any order.  Host
    tensors, more than 256 pairs and heads wider than 1024 take the eager formulation; on the
    device q and k have at most 65536 heads together.
    """
    fused = use_fused(q, "fused_rotary", force_reference)
    if fused and type(sections) in (tuple, list):
        # the plain call runs in C++; any other (None) takes what follows
        out = _lib.native().rotary(q, k, positions, tuple(sections), float(base), ladder,
                                   bool(interleaved))
        if out is not None:
            return out
    sections = tuple(int(n) for n in sections)
    _check(q, k, positions, sections, base, ladder)
    call = (sections, float(base), ladder == "joint", bool(interleaved))
    empty = q.numel() == 0 or (k is not None and k.numel() == 0)
    if not fused or empty or sum(sections) > MAX_PAIRS or q.shape[3] > MAX_HEAD:
        return tuple(None if t is None else rotary_ref(t, positions, *call) for t in (q, k))
    return _FusedRotary.apply(q, k, positions.detach().contiguous(), call, False)
