"""Embedding lookup with scaling, its gradient by sorted tokens, on MI355X.

``embedding_lookup`` gathers scaled rows of a vocabulary table in one pass
(``nf_embedding_fwd``), in the table's type or, from an fp32 table, in 16 bits: the
cast that autocast would add is part of it.  The gradient (``nf_embedding_bwd``)
sorts the tokens by id, sums each id's rows in fp32 in a fixed order and writes
every row of the table's gradient once: bit-identical run to run, however often one
token repeats, where scattered atomic sums are not.
"""

from __future__ import annotations

import torch

from .. import _lib
from .reference import embedding_ref
from .utils import check_devices, device_of, use_fused


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx, out_dtype):
        flat = ids.reshape(-1).to(torch.int64).contiguous()
        m, (v, d) = flat.numel(), table.shape
        # rows of unit stride that do not overlap, else a copy
        rows = (table.stride(1) == 1 or d == 1) and (table.stride(0) >= d or v == 1)
        t = table if rows else table.contiguous()
        out = torch.empty((m, d), dtype=out_dtype, device=t.device)
        with device_of(t):
            _lib.check(
                _lib.lib().nf_embedding_fwd(flat.data_ptr(), t.data_ptr(), max(t.stride(0), d),
                                            scale, m, d, v, out.data_ptr(), _lib.dtype_code(t),
                                            _lib.dtype_code(out), _lib.stream_of(t)),
                "nf_embedding_fwd",
            )
        ctx.save_for_backward(flat)
        ctx.call = (v, d, scale, -1 if padding_idx is None else padding_idx, table.dtype)
        return out.view(*ids.shape, d)

    @staticmethod
    def backward(ctx, dout):
        (flat,) = ctx.saved_tensors
        g = dout.reshape(-1, ctx.call[1])
        return None, _EmbeddingGrad.apply(g, flat, *ctx.call), None, None, None


class _EmbeddingGrad(torch.autograd.Function):
    """The lookup's gradient, [V, D]: linear in dout, its own gradient the lookup again."""

    @staticmethod
    def forward(ctx, dout, flat, v, d, scale, pad, dtype):
        g = dout.contiguous()
        check_devices("embedding_lookup backward", "the forward's ids", dict(dout=g),
                      device=flat.device)
        m = flat.numel()
        dtable = torch.empty((v, d), dtype=dtype, device=g.device)
        L = _lib.lib()
        nbytes = L.nf_embedding_bwd_workspace(m, d, v)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=g.device)
        with device_of(g):
            _lib.check(
                L.nf_embedding_bwd(g.data_ptr(), flat.data_ptr(), pad, scale, m, d, v,
                                   dtable.data_ptr(), _lib.dtype_code(g),
                                   _lib.dtype_code(dtable), ws.data_ptr(), nbytes,
                                   _lib.stream_of(g)),
                "nf_embedding_bwd",
            )
        ctx.save_for_backward(flat)
        ctx.call = (scale, pad, g.dtype)
        return dtable

    @staticmethod
    def backward(ctx, gg):
        (flat,) = ctx.saved_tensors
        scale, pad, dtype = ctx.call
        # the padding id's rows, which gave nothing, get nothing: as those outside the table
        ids = flat if pad < 0 else flat.masked_fill(flat == pad, -1)
        return _EmbeddingLookup.apply(ids, gg, scale, None, dtype), *(None,) * 6


def embedding_lookup(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
                     padding_idx: int | None = None, out_dtype: torch.dtype | None = None,
                     force_reference: bool = False) -> torch.Tensor:
    """``scale * table[ids]``.

    Args:
        ids: integer token ids, any shape.
        table: [V, D] embedding table (a row stride is fine), fp32, bf16 or fp16.
        scale: what the rows are multiplied by, in fp32, before their one rounding.
        padding_idx: an id in [0, V) that is looked up like any other and gives no
            gradient.
        out_dtype: the table's type (the default), or bf16 / fp16 from an fp32 table.
        force_reference: run the eager formulation instead.

    Returns:
        [*ids.shape, D].  An id outside [0, V) gives a row of zeros and no gradient: the
        call reads nothing back to the host, so it cannot raise for one.

    The gradient has the table's type and is the same bits every run; derivatives of any
    order.  Host tensors take the eager formulation.
    """
    fused = use_fused(table, "embedding_lookup", force_reference)
    if fused and table.dim() == 2 and (padding_idx is None or 0 <= padding_idx < table.shape[0]):
        # the plain call runs in C++; any other (None) takes the Function below
        out = _lib.native().embedding(ids, table, float(scale),
                                      -1 if padding_idx is None else padding_idx,
                                      _lib.DTYPE_CODE.get(out_dtype or table.dtype))
        if out is not None:
            return out
    if table.dim() != 2 or 0 in table.shape:
        raise ValueError(f"embedding_lookup: table [V, D] expected, got {tuple(table.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"embedding_lookup: ids are {ids.dtype}; expected int64 or int32")
    if padding_idx is not None and not 0 <= padding_idx < table.shape[0]:
        raise ValueError(f"embedding_lookup: padding_idx {padding_idx} outside "
                         f"[0, {table.shape[0]})")
    out_dtype = table.dtype if out_dtype is None else out_dtype
    _lib.dtype_code(table), _lib.dtype_code(out_dtype)
    if out_dtype != table.dtype and table.dtype != torch.float32:
        raise TypeError(f"embedding_lookup: rows of a {table.dtype} table in {out_dtype}; expected "
                        f"{table.dtype}")
    check_devices("embedding_lookup", "table", dict(table=table, ids=ids))
    if not fused:
        return embedding_ref(ids, table, scale, padding_idx, out_dtype)
    return _EmbeddingLookup.apply(ids, table, float(scale), padding_idx, out_dtype)
