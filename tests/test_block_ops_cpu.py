"""Attention and the rotary positions without a GPU: the eager formulations that host tensors
take, the 64-bit restatements against differences, the refusals of the Python entries and of the
C ABI.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from nuvla_forge_amd import _lib
from nuvla_forge_amd.kernels import fused_attention, fused_rotary
from nuvla_forge_amd.kernels import attention
from nuvla_forge_amd.kernels.utils import DeviceMismatchError

from .block_ops_ref import attention64, near, rotary64, within

NF_OK, NF_ERR_ARG, NF_ERR_DTYPE, NF_ERR_WORKSPACE = 0, -1, -2, -3
FAKE = 4096  # a non-null pointer value; every call below returns before using it
BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16


def _err() -> str:
    return _lib.lib().nf_last_error().decode()


def _qkv(b, tq, tk, h, hk, d, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(b, t, n, d, generator=g).to(dtype) for t, n in ((tq, h), (tk, hk), (tk, hk))]


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b, tq, tk, h, hk, d, causal, mask", [
    (2, 5, 9, 4, 2, 8, False, False), (1, 7, 7, 3, 3, 5, True, True), (2, 9, 4, 2, 1, 6, True, False),
    (3, 1, 11, 4, 4, 16, False, True)])
def test_attention_eager(b, tq, tk, h, hk, d, causal, mask, dtype):
    q, k, v = (t.requires_grad_(True) for t in _qkv(b, tq, tk, h, hk, d, dtype))
    m = None
    if mask:
        m = torch.rand(b, tk, generator=torch.Generator().manual_seed(1)) > 0.4
        m[0] = False
    out = fused_attention(q, k, v, causal=causal, key_mask=m)
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(2)).to(dtype)
    got = (out, *torch.autograd.grad(out, [q, k, v], dout))
    want = attention64(q, k, v, dout, causal, m)
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        assert x.dtype == dtype
        within(x, want[name], want["tol_" + name], name)


def test_attention64_gradient_against_differences():
    """Central differences in 64 bits: the error of step s is s^2 / 6 times a third derivative of
    order 1, beside 2^-52 / s from the values' rounding."""
    q, k, v = (t.double() for t in _qkv(2, 4, 5, 4, 2, 3))
    m = torch.ones(2, 5, dtype=torch.bool)
    m[0, 1] = m[1, 4] = False
    dout = torch.randn(2, 4, 4, 3, generator=torch.Generator().manual_seed(3)).double()

    def value(*x):  # attention64 takes any type of tensor in 64 bits
        return float((_plain64(*x, True, m) * dout).sum())

    want = attention64(*(t.float() for t in (q, k, v)), dout.float(), True, m)
    base = [t.float().double() for t in (q, k, v)]
    dout = dout.float().double()
    s = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        for at in torch.randperm(base[i].numel(), generator=torch.Generator().manual_seed(i))[:12]:
            hi, lo = ([t.clone() for t in base] for _ in range(2))
            hi[i].view(-1)[at] += s
            lo[i].view(-1)[at] -= s
            d = (value(*hi) - value(*lo)) / (2 * s)
            assert abs(d - float(want[name].reshape(-1)[at])) < 1e-6, (name, at)


def _plain64(q, k, v, causal, mask):
    """softmax(q k^T / sqrt(d)) v, row by row, as the definition reads."""
    out = torch.zeros_like(q)
    for b in range(q.shape[0]):
        for i in range(q.shape[1]):
            for h in range(q.shape[2]):
                j = h * k.shape[2] // q.shape[2]
                keys = [n for n in range(k.shape[1])
                        if mask[b, n] and not (causal and n > i + k.shape[1] - q.shape[1])]
                if keys:
                    z = torch.stack([(q[b, i, h] * k[b, n, j]).sum() for n in keys])
                    p = torch.softmax(z / math.sqrt(q.shape[3]), 0)
                    out[b, i, h] = sum(p[n] * v[b, keys[n], j] for n in range(len(keys)))
    return out


def test_attention64_is_the_definition():
    q, k, v = _qkv(2, 4, 6, 4, 2, 5)
    m = torch.tensor([[True, False, True, True, True, False], [False] * 6])
    near(_plain64(*(t.double() for t in (q, k, v)), True, m),
         attention64(q, k, v, causal=True, key_mask=m)["out"], 0, 0, "out", slack=1e-14)


def test_attention_masked_places_are_never_read_on_the_host():
    q, k, v = _qkv(2, 3, 6, 2, 2, 4)
    m = torch.tensor([[True, True, False, True, False, False], [False] * 6])
    want = fused_attention(q, k, v, key_mask=m)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(F32).min):
        kb, vb = (torch.where(m[..., None, None], t, bad).requires_grad_(True) for t in (k, v))
        out = fused_attention(q, kb, vb, key_mask=m)
        assert torch.equal(out, want) and (out[1] == 0).all()
        for x in torch.autograd.grad(out.sum(), [kb, vb]):
            assert x.isfinite().all() and (x[~m] == 0).all()


def test_attention_without_keys_or_rows():
    q, k, v = (t.requires_grad_(True) for t in _qkv(2, 3, 4, 2, 1, 4))
    out = fused_attention(q, k[:, :0], v[:, :0])
    assert out.shape == q.shape and (out == 0).all()
    assert (torch.autograd.grad(out.sum(), q)[0] == 0).all()
    assert fused_attention(q[:, :0], k, v).shape == (2, 0, 2, 4)
    assert fused_attention(q[:0], k[:0], v[:0], causal=True).shape == (0, 3, 2, 4)


def test_attention_refusals():
    q, k, v = _qkv(2, 3, 4, 4, 2, 8)
    mask = torch.ones(2, 4, dtype=torch.bool)
    for bad in ((q[0], k, v), (q, k, v[:, :3]), (q, k[:1], v[:1]), (q[..., :4], k, v),
                (q[:, :, :3], k, v), (q, k[:, :, :0], v[:, :, :0])):
        with pytest.raises(ValueError, match="fused_attention"):
            fused_attention(*bad)
    for bad in ((q.double(), k.double(), v.double()), (q, k.half(), v), (q, k, v.bfloat16())):
        with pytest.raises(TypeError):
            fused_attention(*bad)
    with pytest.raises(TypeError, match="key_mask"):
        fused_attention(q, k, v, key_mask=mask.float())
    for m in (mask[:1], mask[:, :3], mask[0]):
        with pytest.raises(ValueError, match="key_mask"):
            fused_attention(q, k, v, key_mask=m)
    for s in (math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            fused_attention(q, k, v, scale=s)
    with pytest.raises(DeviceMismatchError, match="v is on meta"):
        fused_attention(q, k, v.to("meta"))
    with pytest.raises(DeviceMismatchError, match="key_mask is on meta"):
        fused_attention(q, k, v, key_mask=mask.to("meta"))


def _fwd(**over):
    a = dict(q=FAKE, qs=(64, 64, 16), k=FAKE, ks=(64, 64, 16), v=FAKE, vs=(64, 64, 16), mask=None,
             mb=0, B=1, Tq=2, Tk=2, H=4, Hk=4, D=16, causal=0, scale=0.25, dtype=1,
             out=FAKE, state=FAKE, state_bytes=1 << 20, ws=FAKE, ws_bytes=1 << 20)
    a.update(over)
    return _lib.lib().nf_attention_fwd(
        a["q"], *a["qs"], a["k"], *a["ks"], a["v"], *a["vs"], a["mask"], a["mb"], a["B"], a["Tq"],
        a["Tk"], a["H"], a["Hk"], a["D"], a["causal"], a["scale"], a["dtype"], a["out"],
        a["state"], a["state_bytes"], a["ws"], a["ws_bytes"], None)


def _bwd(**over):
    a = dict(q=FAKE, qs=(64, 64, 16), k=FAKE, ks=(64, 64, 16), v=FAKE, vs=(64, 64, 16), mask=None,
             mb=0, out=FAKE, g=FAKE, gs=(64, 64, 16), B=1, Tq=2, Tk=2, H=4, Hk=4, D=16, causal=0,
             scale=0.25, dtype=1, state=FAKE, state_bytes=1 << 20, dq=FAKE, dk=FAKE, dv=FAKE,
             ws=FAKE, ws_bytes=1 << 20)
    a.update(over)
    return _lib.lib().nf_attention_bwd(
        a["q"], *a["qs"], a["k"], *a["ks"], a["v"], *a["vs"], a["mask"], a["mb"], a["out"],
        a["g"], *a["gs"], a["B"], a["Tq"], a["Tk"], a["H"], a["Hk"], a["D"], a["causal"], a["scale"],
        a["dtype"],
        a["state"], a["state_bytes"], a["dq"], a["dk"], a["dv"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("call", [_fwd, _bwd])
def test_attention_c_abi_refusals(call):
    assert call(dtype=7) == NF_ERR_DTYPE
    for over in (dict(H=6), dict(Hk=0), dict(H=-4), dict(D=0), dict(D=129), dict(B=-1), dict(Tq=-1),
                 dict(Tk=-1), dict(Tk=0), dict(scale=math.nan), dict(scale=math.inf),
                 dict(B=1 << 31), dict(Tq=1 << 31), dict(Tk=1 << 31), dict(B=1 << 22),
                 dict(q=None), dict(k=None), dict(v=None), dict(q=FAKE + 2), dict(qs=(64, 60, 16)),
                 dict(ks=(64, 64, 12)), dict(vs=(4, 64, 16)), dict(ks=(64, -64, 16)),
                 dict(qs=(64, 1 << 22, 16)), dict(Hk=1, qs=(64, 64, 1 << 28)), dict(out=None),
                 dict(state=FAKE + 8), dict(mask=FAKE, mb=-1)):
        assert call(**over) == NF_ERR_ARG, over
        assert "nf_attention" in _err()
    for over in (dict(state_bytes=0), dict(state_bytes=256)):
        assert call(**over) == NF_ERR_WORKSPACE, over
    # nothing to do
    assert call(B=0) == NF_OK and call(Tq=0) == NF_OK


def test_attention_c_abi_refuses_groups_beyond_the_row_division():
    """x / G by a 32-bit reciprocal is exact for all x < G + 128 up to the limit; beyond it the
    quotient of G - 1 can be 1."""
    def quotient(x, g):
        return x * -(-2 ** 32 // g) >> 32

    for g in (2, 3, 7, 127, 129, 32765, 32767, 32768):
        assert all(quotient(x, g) == x // g for x in (0, 1, g - 1, g, 2 * g - 1, g + 127) if
                   x < g + 128)
    assert quotient(100_002, 100_003) == 1
    L = _lib.lib()
    assert L.nf_attention_state_bytes(1, 1, 1, 32768, 1, 8, 1) > 0
    assert L.nf_attention_state_bytes(1, 1, 1, 32769, 1, 8, 1) == 0
    for f in (L.nf_attention_fwd_workspace, L.nf_attention_bwd_workspace):
        assert f(1, 1, 1, 32769, 1, 8, 0, 1) == 0


def test_attention_c_abi_workspaces():
    L = _lib.lib()
    # many rows: no split; a few rows over many keys: partial sums
    assert L.nf_attention_fwd_workspace(8, 1176, 1176, 6, 6, 64, 0, 1) == 0
    few = L.nf_attention_fwd_workspace(1, 1, 65536, 8, 2, 128, 0, 1)
    assert few > 0
    assert _fwd(Tq=1, Tk=65536, H=4, Hk=4, ws_bytes=16) == NF_ERR_WORKSPACE
    assert _fwd(Tq=1, Tk=65536, H=4, Hk=4, ws=None) == NF_ERR_ARG
    assert _bwd(ws_bytes=16) == NF_ERR_WORKSPACE and _bwd(ws=None) == NF_ERR_ARG
    assert _bwd(g=None) == NF_ERR_ARG and _bwd(gs=(64, 64, 2)) == NF_ERR_ARG
    assert _bwd(dq=None, dk=None, dv=None) == NF_OK
    kept = L.nf_attention_state_bytes(2, 3, 4, 4, 2, 16, 1)
    assert kept >= 2 * 3 * 4 * (4 + 16 * 2)
    assert L.nf_attention_state_bytes(2, 3, 4, 4, 2, 16, 0) < kept  # fp32: nothing left over
    assert _bwd(state=None) == NF_ERR_ARG
    for bad in ((2, 3, 4, 4, 3, 16), (2, 3, 4, 4, 2, 200), (-2, 3, 4, 4, 2, 16)):
        assert L.nf_attention_state_bytes(*bad, 1) == 0
        assert L.nf_attention_fwd_workspace(*bad, 0, 1) == 0
        assert L.nf_attention_bwd_workspace(*bad, 0, 1) == 0


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("ladder", ["axis", "joint"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d, sections", [(16, (8,)), (16, (2, 3, 3)), (13, (1, 0, 2, 2)), (10, (2, 2))])
def test_rotary_eager(d, sections, ladder, interleaved, dtype):
    g = torch.Generator().manual_seed(d)
    q, k = (torch.randn(2, 5, n, d, generator=g).to(dtype).requires_grad_(True) for n in (3, 1))
    pos = torch.randint(-50, 1_000_000, (2, 5, len(sections)), generator=g)
    form = dict(base=500.0, ladder=ladder, interleaved=interleaved)
    out = fused_rotary(q, k, pos, sections, **form)
    ups = [torch.randn(x.shape, generator=g).to(dtype) for x in out]
    grads = torch.autograd.grad(out, [q, k], ups)
    ref = (sections, 500.0, ladder == "joint", interleaved)
    for x, y, up, gr in zip((q, k), out, ups, grads):
        within(y, *rotary64(x, pos, *ref), "turned")
        within(gr, *rotary64(up, pos, *ref, inverse=True), "gradient")
        assert torch.equal(y[..., 2 * sum(sections):], x[..., 2 * sum(sections):])


def test_rotary_equal_coordinates_turn_as_one_position():
    q = torch.randn(1, 6, 2, 16, generator=torch.Generator().manual_seed(0))
    at = torch.tensor([0, 3, 10, 100, 5000, 999999])
    one, _ = fused_rotary(q, None, at[:, None], (8,), ladder="joint")
    three, none = fused_rotary(q, None, at[:, None].expand(6, 3), (2, 3, 3), ladder="joint")
    assert torch.equal(one, three) and none is None
    half, _ = fused_rotary(q, None, at[:, None].float() + 0.5, (8,))
    whole, _ = fused_rotary(q, None, 2 * at[:, None] + 1, (8,))
    turned, _ = fused_rotary(half, None, at[:, None].float() + 0.5, (8,))  # twice a half turn
    near(turned, whole.double(), 0, 0, "half positions", slack=1e-6)


def test_rotary_positions_shared_or_per_sample():
    q = torch.randn(3, 4, 2, 8)
    pos = torch.arange(4)[:, None]
    a = fused_rotary(q, None, pos, (4,))[0]
    for p in (pos[None], pos[None].expand(3, 4, 1), pos.int(), pos.float()):
        assert torch.equal(fused_rotary(q, None, p, (4,))[0], a)
    assert fused_rotary(q[:, :0], None, pos[:0], (4,))[0].shape == (3, 0, 2, 8)


def test_rotary_refusals():
    q, k, pos = torch.randn(2, 3, 4, 8), torch.randn(2, 3, 2, 8), torch.zeros(3, 2, dtype=torch.long)
    for args in ((q[0], k, pos, (2, 2)), (q, k[:, :2], pos, (2, 2)), (q, k[..., :4], pos, (2, 2)),
                 (q, k, pos, (2, 3)), (q, k, pos, (0, 0)), (q, k, pos, (5, -1)), (q, k, pos, ()),
                 (q, k, pos, (1,) * 5), (q, k, pos, (4,)), (q, k, pos[:2], (2, 2)),
                 (q, k, pos[None].expand(5, 3, 2), (2, 2))):
        with pytest.raises(ValueError, match="fused_rotary"):
            fused_rotary(*args)
    with pytest.raises(ValueError, match="ladder"):
        fused_rotary(q, k, pos, (2, 2), ladder="both")
    for base in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="base"):
            fused_rotary(q, k, pos, (2, 2), base=base)
    for args in ((q, k.half(), pos, (2, 2)), (q.double(), None, pos, (2, 2)),
                 (q, k, pos.double(), (2, 2))):
        with pytest.raises(TypeError):
            fused_rotary(*args)
    with pytest.raises(DeviceMismatchError, match="positions is on meta"):
        fused_rotary(q, k, pos.to("meta"), (2, 2))


def test_rotary_c_abi_refusals():
    def call(q=FAKE, qo=FAKE, H=2, k=FAKE, ko=FAKE, Hk=1, pos=FAKE, kind=0, B=1, T=3, D=16,
             sections=(4, 4), base=1e4, dtype=1, axes=None):
        s = (ctypes.c_int32 * max(1, len(sections)))(*sections)
        return _lib.lib().nf_rotary(q, 96, 32, 16, qo, H, k, 48, 16, 16, ko, Hk, pos, 0, kind, B, T,
                                    D, s, len(sections) if axes is None else axes, base, 0, 0, 0,
                                    dtype, None)

    assert call(dtype=9) == NF_ERR_DTYPE and call(kind=3) == NF_ERR_DTYPE
    for over in (dict(B=-1), dict(T=-1), dict(D=0), dict(H=-1), dict(Hk=-1), dict(sections=(5, 4)),
                 dict(sections=(0, 0)), dict(sections=(-1, 4)), dict(sections=()), dict(axes=5),
                 dict(sections=(300,), D=1000), dict(D=1025), dict(base=0.0), dict(base=math.inf),
                 dict(base=math.nan), dict(q=None), dict(qo=None), dict(k=None), dict(ko=None),
                 dict(pos=None), dict(T=1 << 31), dict(H=1 << 20), dict(B=1 << 40)):
        assert call(**over) == NF_ERR_ARG, over
        assert "nf_rotary" in _err()
    assert call(B=0) == NF_OK and call(T=0) == NF_OK and call(H=0, Hk=0) == NF_OK


# ---------------------------------------------------------------------------
# the layouts that the kernels are handed
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, d", [(BF16, 100), (F16, 7), (F32, 90), (F32, 1), (BF16, 64)])
@pytest.mark.parametrize("order", [(0, 1, 2, 3), (0, 2, 3, 1), (0, 3, 2, 1), (3, 2, 0, 1),
                                   (1, 3, 0, 2)])
@pytest.mark.parametrize("b, t, h", [(2, 70, 4), (1, 70, 1), (2, 1, 3), (1, 1, 1)])
def test_attention_rows_are_whole_vectors_whatever_the_layout(b, t, h, order, dtype, d):
    """What the Python entry hands to the kernels holds the values, zeros up to a whole vector, and
    strides that the C entry takes."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(b, t, h, d, generator=g).to(dtype)
    y = x.permute(order).contiguous().permute([order.index(i) for i in range(4)])
    for z in (y, x[:, :1, :1].expand(b, t, h, d), x[..., :1].expand(b, t, h, d)):
        rows = attention._vector_rows(z)
        e = 16 // z.element_size()
        assert rows.shape[:3] == z.shape[:3] and rows.shape[3] == -(-d // e) * e
        assert torch.equal(rows[..., :d], z) and (rows[..., d:] == 0).all()
        sb, st, sh = attention._strides(rows)
        assert rows.stride(3) == 1 or rows.shape[3] == 1
        assert sb % e == 0 and st % e == 0 and sh % e == 0 and rows.data_ptr() % 16 == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("mask", [False, True])
def test_attention_rows_without_a_key_reach_no_gradient_on_the_host(mask, dtype):
    q, k, v = _qkv(2, 7, 4, 2, 1, 6, dtype)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(dtype)
    m = torch.tensor([[False, False, True, True], [False] * 4]) if mask else None
    bare = torch.arange(7)[None].expand(2, 7) < (torch.tensor([[5], [7]]) if mask else 3)

    def run(q, dout):
        x = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = fused_attention(*x, causal=True, key_mask=m)
        return [out, *torch.autograd.grad(out, x, dout)]

    want = run(q, dout)
    assert (want[0][bare] == 0).all() and (want[1][bare] == 0).all()
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max):
        q2, d2 = (torch.where(bare[..., None, None], torch.tensor(bad, dtype=dtype), t)
                  for t in (q, dout))
        assert all(torch.equal(a, b) for a, b in zip(want, run(q2, d2))), bad


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, 2e38, math.nextafter(2.0 ** 127, math.inf)])
def test_attention_scales_beyond_fp32_are_refused(scale):
    """2^127 log2(e) is below fp32's largest number, about 2^128."""
    q, k, v = _qkv(2, 3, 4, 4, 2, 8)
    with pytest.raises(ValueError, match="fused_attention: scale"):
        fused_attention(q, k, v, scale=scale)
    for s in (2.0 ** 127, -2.0 ** 127, 0.0):
        assert fused_attention(q * 0.0, k, v, scale=s).isfinite().all()
    for call in (_fwd, _bwd):
        if abs(scale) < 3.4e38 and ctypes.c_float(scale).value != 2.0 ** 127:
            assert call(scale=scale) == NF_ERR_ARG and "scale" in _err()
