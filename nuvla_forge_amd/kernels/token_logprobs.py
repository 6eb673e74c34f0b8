"""Log probabilities of given tokens on the language-model head, on MI355X MFMA.

``chunked_token_logprobs`` gives, for every row of hidden states, the log probability
of one token under ``softmax(hidden @ lm_weight.T)``, the entropy of that distribution
and, where asked, its ``top_k`` most probable tokens, without a full logit tensor: what
policy-gradient training, scoring and reporting alternatives need of a head whose mean
loss ``chunked_cross_entropy`` computes.  Both per-token values have gradients.

The device path is two calls, as the cross entropy's.  ``nf_token_logprobs_fwd`` compacts
the rows that count on the device and keeps them with each row's largest logit, the logarithm
of its sum and its entropy and, where a backward will follow and one chunk takes every row
(bf16, more than 128 rows), the exponential of every logit in 16 bits;
``nf_token_logprobs_bwd`` forms the logits' gradient from those, or from the logits formed
again, and runs the cross entropy's gradient products.  No call synchronises with the host.

Element types and ``chunk_size`` are the cross entropy's: bf16 inputs, or any under bf16
autocast, run bf16 MFMA with fp32 accumulation; fp32 inputs bf16 products over three-part
operands; others are widened to fp32.  ``chunk_size`` bounds what the forward keeps of the
logits, and what the backward holds of their gradient with its accumulator, each by the bytes
of an fp32 [chunk_size, V] tile plus an fp32 [V, D] accumulator.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from .chunked_ce import _compute_dtype, chunk_rows_for
from .reference import token_logprobs_ref
from .utils import check_devices, device_of, first_order_only, use_fused

MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    """What ``chunked_token_logprobs`` returns; the last two are None for ``top_k`` 0."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor | None
    top_ids: torch.Tensor | None


def _check(hidden, lm_weight, targets, top_k):
    if hidden.dim() != 2 or lm_weight.dim() != 2 or hidden.shape[1] != lm_weight.shape[1]:
        raise ValueError(f"hidden [M, D] and lm_weight [V, D] expected, got "
                         f"{tuple(hidden.shape)} and {tuple(lm_weight.shape)}")
    if targets.shape != (hidden.shape[0],):
        raise ValueError(f"targets must be [M={hidden.shape[0]}], got {tuple(targets.shape)}")
    if 0 in lm_weight.shape:
        raise ValueError(f"lm_weight must not be empty, got {tuple(lm_weight.shape)}")
    if not 0 <= top_k <= min(MAX_TOP_K, lm_weight.shape[0]):
        raise ValueError(f"top_k must be in [0, {min(MAX_TOP_K, lm_weight.shape[0])}], got {top_k}")
    check_devices("chunked_token_logprobs", "hidden",
                  dict(hidden=hidden, lm_weight=lm_weight, targets=targets))


def _from_vector(x):
    """``x`` (contiguous) from a whole 16-byte vector on: a copy of a view that begins between
    two, which every kernel of the call would read element by element."""
    whole = x.data_ptr() % 16 == 0 or x.shape[1] * x.element_size() % 16 != 0
    return x if whole else x.clone()


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, lm_weight, targets, top_k, chunk_rows, ignore_index):
        (m, d), v, dev = hidden.shape, lm_weight.shape[0], hidden.device
        cdt = _compute_dtype(hidden, lm_weight)
        h, w = (_from_vector(x.to(cdt).contiguous()) for x in (hidden, lm_weight))
        tg = targets.to(torch.int64).contiguous()
        logprobs = torch.empty(m, dtype=torch.float32, device=dev)
        entropy = torch.empty_like(logprobs)
        top_lp = torch.empty((m, top_k), dtype=torch.float32, device=dev)
        top_ids = torch.empty((m, top_k), dtype=torch.int64, device=dev)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_lp, top_ids)
        ctx.types = (hidden.dtype, lm_weight.dtype)
        ctx.shape = (m, d, v, chunk_rows, _lib.dtype_code(cdt))
        if m == 0:
            ctx.save_for_backward(w)
            return logprobs, entropy, top_lp, top_ids
        L, code = _lib.lib(), _lib.dtype_code(cdt)
        # what a backward reads instead of forming the logits again (asked of the inputs: inside
        # a Function no gradient is being recorded)
        keep = any(ctx.needs_input_grad[:2])
        ctx.keep = keep
        st_bytes = L.nf_token_logprobs_state_bytes(m, d, v, chunk_rows, keep, code)
        ws_bytes = L.nf_token_logprobs_fwd_workspace(m, d, v, chunk_rows, top_k, code)
        if not st_bytes or not ws_bytes:
            raise ValueError(f"chunked_token_logprobs: shape M={m} D={d} V={v} is beyond the "
                             "kernels")
        state = torch.empty(st_bytes, dtype=torch.uint8, device=dev)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        with device_of(hidden):
            _lib.check(
                L.nf_token_logprobs_fwd(h.data_ptr(), w.data_ptr(), tg.data_ptr(), m, d, v,
                                        ignore_index, chunk_rows, top_k, keep, code,
                                        logprobs.data_ptr(), entropy.data_ptr(),
                                        top_lp.data_ptr(), top_ids.data_ptr(), state.data_ptr(),
                                        st_bytes, ws.data_ptr(), ws_bytes,
                                        _lib.stream_of(hidden)),
                "nf_token_logprobs_fwd",
            )
        ctx.save_for_backward(w, state)
        return logprobs, entropy, top_lp, top_ids

    @staticmethod
    def backward(ctx, g_lp, g_ent, _g_top, _g_ids):
        none = (None,) * 6
        if g_lp is None and g_ent is None:
            return none
        w, *rest = ctx.saved_tensors
        m, d, v, chunk_rows, code = ctx.shape
        need_h, need_w = ctx.needs_input_grad[:2]
        dh = torch.empty((m, d), dtype=ctx.types[0], device=w.device) if need_h else None
        dw = torch.empty((v, d), dtype=ctx.types[1], device=w.device) if need_w else None
        if m == 0:
            return dh, None if dw is None else dw.zero_(), *none[2:]
        (state,) = rest
        check_devices("chunked_token_logprobs backward", "the forward's hidden",
                      dict(grad_logprobs=g_lp, grad_entropy=g_ent), device=w.device)
        g, h = (None if t is None else t.to(torch.float32).contiguous() for t in (g_lp, g_ent))
        L = _lib.lib()
        ws_bytes = L.nf_token_logprobs_bwd_workspace(m, d, v, chunk_rows, code)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=w.device)
        # a gradient of a type the kernels do not write is cast to from fp32
        wide = [t if t in _lib.DTYPE_CODE else torch.float32 for t in ctx.types]
        oh = dh if dh is None or dh.dtype == wide[0] else torch.empty_like(dh, dtype=wide[0])
        ow = dw if dw is None or dw.dtype == wide[1] else torch.empty_like(dw, dtype=wide[1])
        with device_of(w):
            _lib.check(
                L.nf_token_logprobs_bwd(w.data_ptr(), m, d, v, chunk_rows, ctx.keep, code,
                                        state.data_ptr(), state.numel(), _lib.ptr(g),
                                        _lib.ptr(h), _lib.ptr(oh), _lib.dtype_code(wide[0]),
                                        _lib.ptr(ow), _lib.dtype_code(wide[1]), ws.data_ptr(),
                                        ws_bytes, _lib.stream_of(w)),
                "nf_token_logprobs_bwd",
            )
        return first_order_only("chunked_token_logprobs", (g_lp, g_ent),
                                (None if oh is None else oh.to(ctx.types[0]),
                                 None if ow is None else ow.to(ctx.types[1]), *none[2:]))


def chunked_token_logprobs(
    hidden: torch.Tensor,
    lm_weight: torch.Tensor,
    targets: torch.Tensor,
    top_k: int = 0,
    chunk_size: int = 1024,
    ignore_index: int = -100,
    force_reference: bool = False,
) -> TokenLogprobs:
    """Log probability of ``targets`` under ``softmax(hidden @ lm_weight.T)``, the entropy
    and the most probable tokens of each row.

    Args:
        hidden: [M, D] pre-projection hidden states.
        lm_weight: [V, D] output embedding.
        targets: [M] int64 token ids, ``ignore_index`` to leave a row out.
        top_k: how many of the most probable tokens to report, 0 to 32.
        chunk_size: memory budget, as in ``chunked_cross_entropy``.
        ignore_index: target value of rows that are left out; targets outside [0, V)
            leave their row out too.
        force_reference: run the eager row-chunk loop instead.

    Returns:
        ``TokenLogprobs(logprobs, entropy, top_logprobs, top_ids)``: fp32 [M], fp32 [M],
        fp32 [M, top_k] in falling order and int64 [M, top_k] (equal ones: the lower token
        first).  Rows left out give 0, their alternatives token -1, and no gradient.
        ``logprobs`` and ``entropy`` carry gradients, the alternatives none.  A row with a
        NaN among its logits has NaN values, and -1 for alternatives it cannot order.

    Second derivatives are not supported on the device: taking one raises.

    Host tensors run the eager row-chunk loop.
    """
    fused = use_fused(hidden, "chunked_token_logprobs", force_reference)
    if fused:  # the plain call runs in C++; any other (None) takes the Function below
        out = _lib.native().token_logprobs(
            hidden, lm_weight, targets, top_k, chunk_size, ignore_index,
            _lib.dtype_code(_compute_dtype(hidden, lm_weight)))
        if out is not None:
            return TokenLogprobs(*out) if top_k else TokenLogprobs(out[0], out[1], None, None)
    _check(hidden, lm_weight, targets, top_k)
    chunk_rows = chunk_rows_for(chunk_size)
    if not fused:
        return TokenLogprobs(*token_logprobs_ref(hidden, lm_weight, targets, top_k, chunk_rows,
                                                 ignore_index))
    lp, ent, top_lp, top_ids = _TokenLogprobs.apply(hidden, lm_weight, targets, int(top_k),
                                                    chunk_rows, int(ignore_index))
    return TokenLogprobs(lp, ent, *((top_lp, top_ids) if top_k else (None, None)))
