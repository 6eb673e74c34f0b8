"""Attention and the rotary positions on the GPU: calls at the edges of what the documentation
allows (layouts that need a copy, rows that attend nothing, axes of no length, odd arguments).
"""

from __future__ import annotations

import math

import pytest
import torch

from nuvla_forge_amd import _lib
from nuvla_forge_amd.kernels import fused_attention, fused_rotary

from .helpers import assert_graph_replays_match, gen, note, randn
from .test_gpu_block_ops import _check, _mask, _qkv, _run
from .test_gpu_token_ops_edges import route  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16


def _same(want, got, what=""):
    for name, a, b in zip(("out", "dq", "dk", "dv"), want, got, strict=True):
        assert torch.equal(a, b), f"{what} {name}"


# ---------------------------------------------------------------------------
# layouts
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, d", [(BF16, 100), (F16, 100), (BF16, 7), (F32, 90), (F32, 1)])
@pytest.mark.parametrize("tq", [1, 70])
def test_attention_token_axis_innermost(cuda, route, tq, dtype, d):
    """Heads of no whole vectors whose tokens lie side by side, or are one: operands, gradients
    and saved tensors give the bits of their dense copies."""
    note(f"attention tokens innermost {tq} {d} {dtype} {route}")
    q, k, v, do = _qkv(2, tq, 70, 4, 2, d, dtype, cuda)
    m = _mask("random", 2, 70, cuda)
    want = _run(q, k, v, do, key_mask=m)

    def inner(x, order):  # the same values, the axes stored in this order
        back = [order.index(i) for i in range(4)]
        return x.permute(order).contiguous().permute(back)

    for order in ((0, 2, 3, 1), (0, 3, 2, 1), (3, 2, 0, 1), (1, 3, 0, 2)):
        a, b, c, e = (inner(x, order) for x in (q, k, v, do))
        _same(want, _run(a, b, c, do, key_mask=m), f"operands {order}")
        _same(want, _run(q, k, v, e, key_mask=m), f"gradient {order}")
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x, o=order: (
                inner(x, o) if x.dim() == 4 else x)):
            _same(want, _run(a, b, c, e, key_mask=m), f"saved {order}")
    one = [x[:, :1, :1, :1].expand(x.shape) for x in (q, k, v, do)]
    _same(_run(*(x.contiguous() for x in one)), _run(*one), "broadcast")


@pytest.mark.parametrize("dtype, d", [(BF16, 100), (F32, 90)])
def test_attention_before_a_convolution_over_tokens(cuda, route, dtype, d):
    """What follows takes [B, H D, T], and gives its gradient in that order."""
    note(f"attention before a convolution {d} {dtype} {route}")
    q, k, v, _ = _qkv(2, 70, 70, 2, 2, d, dtype, cuda)
    w = randn((3, 2 * d, 1), gen(5), dtype, cuda)
    seen = []

    def step(keep):
        x = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = fused_attention(*x, causal=True)
        out.register_hook(lambda g: (seen.append(g), keep(g))[1])
        y = torch.matmul(w[:, :, 0].float(), out.float().flatten(2).transpose(1, 2).contiguous())
        return [out, *torch.autograd.grad(y.sum(), x)]

    # the gradient as the product's backward leaves it, tokens innermost or not, and its dense copy
    _same(step(lambda g: g.contiguous()), step(lambda g: g))
    g = seen[0].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    assert g.stride(1) == 1
    _same(step(lambda _: g.contiguous()), step(lambda _: g))


# ---------------------------------------------------------------------------
# rows that attend no key, axes of no length
# ---------------------------------------------------------------------------
def _padded(kind, b, tk, dev):
    """Masks that leave a sample's first keys out, one sample none, one all of them."""
    if kind is None:
        return None
    m = torch.ones(b, tk, dtype=torch.bool)
    for i in range(b):
        m[i, : i * tk // (b + 1)] = False
    if kind == "holes":
        m &= torch.rand(b, tk, generator=gen(b)) > 0.3
    m[-1] = False
    return m.to(dev)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("mask", [None, "left", "holes"])
@pytest.mark.parametrize("b, tq, tk, h, hk, d", [
    (3, 20, 9, 4, 2, 64), (3, 200, 150, 4, 2, 72), (3, 33, 200, 6, 2, 128), (2, 5, 3, 3, 1, 40),
    (4, 1, 70, 4, 2, 32), (70, 150, 130, 8, 4, 72), (70, 150, 150, 8, 4, 128), (66, 70, 70, 9, 3, 32),
    (2, 2300, 2000, 4, 2, 64), (3, 2000, 2000, 2, 1, 128)])
def test_attention_rows_without_a_key_reach_no_gradient(cuda, b, tq, tk, h, hk, d, mask, dtype):
    """NaN, infinities and the type's largest values in the queries and output gradients of rows
    that attend no key change no bit of any result."""
    note(f"attention keyless rows {b} {tq} {tk} {h} {hk} {d} {mask} {dtype}")
    q, k, v, do = _qkv(b, tq, tk, h, hk, d, dtype, cuda)
    m = _padded(mask, b, tk, cuda)
    live = torch.ones(b, tk, dtype=torch.bool, device=cuda) if m is None else m
    seen = torch.arange(tq, device=cuda) + tk - tq  # the row's last key
    count = torch.cat([torch.zeros(b, 1, device=cuda), live.float().cumsum(1)], 1)
    bare = count.gather(1, (seen + 1).clamp(min=0).expand(b, tq)) == 0
    if not bare.any():
        bare = torch.zeros_like(bare)
    want = _run(q, k, v, do, causal=True, key_mask=m)
    for x in want[:2]:
        assert (x[bare] == 0).all()
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max):
        fill = torch.tensor(bad, dtype=dtype, device=cuda)
        q2, do2 = (torch.where(bare[..., None, None], fill, t) for t in (q, do))
        _same(want, _run(q2, k, v, do, causal=True, key_mask=m), f"q {bad}")
        _same(want, _run(q2, k, v, do2, causal=True, key_mask=m), f"q, dout {bad}")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b, t, h, hk, d", [(2, 300, 4, 2, 64), (2, 2000, 4, 2, 128), (70, 140, 8, 4, 96)])
def test_attention_blocks_without_a_key_give_zeros(cuda, b, t, h, hk, d, dtype):
    """Stretches of keys that the mask drops whole, at either end and between, causal or not: zero
    gradients there, whatever the rows hold elsewhere."""
    note(f"attention dropped blocks {b} {t} {h} {hk} {d} {dtype}")
    q, k, v, do = _qkv(b, t, t, h, hk, d, dtype, cuda)
    m = torch.ones(b, t, dtype=torch.bool, device=cuda)
    m[0, : t // 2] = False
    m[1, t // 2:] = False
    m[-1, t // 4: 3 * t // 4] = False
    for causal in (False, True):
        _check(q, k, v, do, causal=causal, key_mask=m)
        got = _run(q, k, v, do, causal=causal, key_mask=m)
        for x in got[2:]:
            assert (x[~m] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b, tk, hk, d", [(1, 1, 1, 1), (2, 70, 2, 64), (3, 1001, 5, 33)])
def test_attention_gradients_of_no_rows_are_zeros(cuda, b, tk, hk, d, dtype):
    """The C entry over keys without a query: dk and dv are empty sums, and what lies behind them
    stays; also inside a captured graph."""
    note(f"attention no rows {b} {tk} {hk} {d} {dtype}")
    dt = _lib.dtype_code(dtype)
    n = b * tk * hk * d
    empty = torch.empty(256, dtype=torch.uint8, device=cuda)
    p = empty.data_ptr()

    def call(dk, dv, stream):
        return _lib.lib().nf_attention_bwd(
            *(p, 0, 0, 0) * 3, None, 0, p, p, 0, 0, 0, b, 0, tk, 2 * hk, hk, d, 1, 1.0, dt, p, 0, None,
            dk, dv, None, 0, stream)

    def outs():
        return [torch.full((n + 64,), 5.0, dtype=dtype, device=cuda) for _ in range(2)]

    x = outs()
    stream = _lib.stream_of(x[0])
    for pick in ((True, True), (True, False), (False, True), (False, False)):
        x = outs()
        assert call(*(t.data_ptr() if w else None for t, w in zip(x, pick)), stream) == 0
        for t, w in zip(x, pick):
            assert (t[:n] == (0.0 if w else 5.0)).all() and (t[n:] == 5.0).all()
    x = outs()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        assert call(x[0].data_ptr(), x[1].data_ptr(), _lib.stream_of(x[0])) == 0
    for _ in range(3):
        for t in x:
            t.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all((t[:n] == 0).all() and (t[n:] == 5.0).all() for t in x)


def test_attention_without_rows_through_the_public_call(cuda, route):
    note(f"attention without rows {route}")
    q, k, v, _ = _qkv(2, 3, 40, 4, 2, 64, BF16, cuda)
    x = [t.detach().requires_grad_(True) for t in (q[:, :0], k, v)]
    out = fused_attention(*x)
    assert out.shape == (2, 0, 4, 64)
    got = torch.autograd.grad(out, x, torch.empty_like(out))
    assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(got, x))


def test_attention_gradients_of_no_rows_outside_device_memory_are_refused(cuda):
    """The one call that looks at no operand asks the runtime where its gradients are, before any
    launch."""
    note("attention no rows, a gradient on the host")
    host, dev = torch.full((64,), 5.0), torch.full((64,), 5.0, device=cuda)
    p = dev.data_ptr()
    for dk, dv in ((host.data_ptr(), p), (p, host.data_ptr()), (4096, None)):
        rc = _lib.lib().nf_attention_bwd(
            *(p, 0, 0, 0) * 3, None, 0, p, p, 0, 0, 0, 1, 0, 4, 2, 1, 16, 1, 1.0, 0, p, 0, None, dk, dv,
            None, 0, _lib.stream_of(dev))
        assert rc == -1 and "nf_attention_bwd" in _lib.lib().nf_last_error().decode()
    assert (dev == 5.0).all() and (host == 5.0).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [24, 32, 57, 64, 88, 96, 120, 128])
def test_attention_results_that_turn_in_one_place(cuda, d, dtype):
    """Blocks whose wavefronts have rows, or keys, of their own lay dk and then dv out in the same
    LDS: each is the one of a call for it alone, and both are right."""
    note(f"attention results in turn {d} {dtype}")
    q, k, v, do = _qkv(64, 130, 130, 4, 4, d, dtype, cuda)
    want = _check(q, k, v, do)
    for i in (1, 2):
        x = [t.detach().requires_grad_(i == j) for j, t in enumerate((q, k, v))]
        got = torch.autograd.grad(fused_attention(*x), x[i], do)[0]
        assert torch.equal(got, want[1 + i])


# ---------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, 2e38, math.inf, -math.inf, math.nan])
def test_attention_scale_beyond_fp32_is_refused(cuda, route, scale):
    note(f"attention scale {scale} {route}")
    q, k, v, _ = _qkv(2, 3, 4, 4, 2, 64, BF16, cuda)
    with pytest.raises(ValueError, match="fused_attention: scale"):
        fused_attention(q, k, v, scale=scale)


@pytest.mark.parametrize("scale", [2.0 ** 127, -2.0 ** 127, 2.0 ** -149, 1e-300])
def test_attention_scales_at_the_ends_of_fp32(cuda, route, scale):
    """Logits of 0 stay 0: each row's output is its values' mean, its queries' gradient 0 or what
    the scale makes of it."""
    note(f"attention scale {scale} {route}")
    q, k, v, do = _qkv(2, 3, 8, 4, 2, 64, F32, cuda)
    out, _, dk, dv = _run(torch.zeros_like(q), k, v, do, scale=scale)
    want = _run(torch.zeros_like(q), k, v, do, scale=1.0)
    assert torch.equal(out, want[0]) and torch.equal(dv, want[3]) and (dk == 0).all()


@pytest.mark.parametrize("shape", [(), (2,), (3,), (1, 1, 3, 2), (0, 2)])
def test_rotary_positions_of_the_wrong_dimensions_are_refused(cuda, route, shape):
    note(f"rotary positions {shape} {route}")
    q = randn((2, 3, 4, 16), gen(0), BF16, cuda)
    with pytest.raises(ValueError, match="fused_rotary: positions"):
        fused_rotary(q, None, torch.zeros(shape, dtype=torch.long, device=cuda), (4, 4))


# ---------------------------------------------------------------------------
# calls that copy their operands, in graphs and under what sees or replaces a call
# ---------------------------------------------------------------------------
def _copied(t, d, dtype, dev):
    """Operands of no whole vectors, k and the mask with their tokens innermost."""
    q, k, v, do = _qkv(2, t, 70, 4, 2, d, dtype, dev)
    k = k.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    return (q, k, v, do), _mask("random", 2, 70, dev).t().contiguous().t()


@pytest.mark.parametrize("dtype, d", [(BF16, 100), (F32, 90)])
@pytest.mark.parametrize("t", [1, 70])
def test_attention_with_copies_in_a_graph(cuda, t, dtype, d):
    note(f"attention copies in a graph {t} {d} {dtype}")
    args, m = _copied(t, d, dtype, cuda)

    def make():
        x = [a.clone(memory_format=torch.preserve_format).requires_grad_(True) for a in args[:3]]

        def step():
            out = fused_attention(*x, causal=True, key_mask=m)
            return [out.detach(), *torch.autograd.grad(out, x, args[3])]

        return step

    assert_graph_replays_match(make)


@pytest.mark.parametrize("dtype, d", [(BF16, 100), (F32, 90)])
def test_attention_with_copies_under_modes_and_create_graph(cuda, route, dtype, d):
    from torch.utils._python_dispatch import TorchDispatchMode

    note(f"attention copies under modes {d} {dtype} {route}")
    (q, k, v, do), m = _copied(70, d, dtype, cuda)
    want = _run(q, k, v, do, causal=True, key_mask=m)

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, a=(), kw=None):
            return func(*a, **(kw or {}))

    with Dispatch():
        _same(want, _run(q, k, v, do, causal=True, key_mask=m), "mode")
    op = lambda *x: fused_attention(*x, causal=True, key_mask=m)  # noqa: E731
    traced = torch.jit.trace(op, (q, k, v), check_trace=False)
    assert torch.equal(traced(q, k, v), want[0])
    x = [t.detach().requires_grad_(True) for t in (q, k, v)]
    up = do.clone().requires_grad_(True)
    got = torch.autograd.grad(op(*x), x, up, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want[1:], got))
    for leaf in (*x, up):
        with pytest.raises(RuntimeError, match="fused_attention: second derivatives"):
            torch.autograd.grad(sum((t.float() ** 2).sum() for t in got), leaf, retain_graph=True,
                                allow_unused=True)


def test_attention_rows_without_a_key_in_a_graph_and_on_two_streams(cuda):
    """A batch padded on the left, NaN in the padding: replays and calls on other streams give the
    bits of zeros there."""
    note("attention keyless rows in a graph")
    (q, k, v, do) = _qkv(3, 150, 150, 4, 2, 64, BF16, cuda)
    m = torch.arange(150, device=cuda)[None] >= torch.tensor([[0], [61], [149]], device=cuda)
    pad = ~m[..., None, None]
    want = _run(*(t.masked_fill(pad, 0.0) for t in (q, k, v, do)), causal=True, key_mask=m)
    args = [t.masked_fill(pad, math.nan) for t in (q, k, v, do)]

    def make():
        x = [t.clone().requires_grad_(True) for t in args[:3]]

        def step():
            out = fused_attention(*x, causal=True, key_mask=m)
            return [out.detach(), *torch.autograd.grad(out, x, args[3])]

        return step

    _same(want, make()())
    assert_graph_replays_match(make)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            got.append(make()())
    torch.cuda.synchronize()
    for x in got:
        _same(want, x)
