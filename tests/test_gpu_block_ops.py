"""Attention and the rotary positions on the GPU against 64 bits, within the bounds that
block_ops_ref derives: types, head layouts, lengths, masks, strides, streams, graphs, buffers.
"""

from __future__ import annotations

import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from nuvla_forge_amd import _lib
from nuvla_forge_amd.kernels import (
    embedding_lookup,
    fused_attention,
    fused_rotary,
    fused_swiglu,
)

from .block_ops_ref import attention64, near, rotary64, within
from .helpers import assert_graph_replays_match, gen, note, randn
from .test_gpu_token_ops_edges import route  # noqa: F401  (a fixture)
from .token_ops_ref import half_step

pytestmark = pytest.mark.gpu
BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16
NAMES = ("out", "dq", "dk", "dv")


def _qkv(b, tq, tk, h, hk, d, dtype, dev, seed=0, sharp=1.5):
    g = gen(seed)
    q = randn((b, tq, h, d), g, dtype, dev, std=sharp)
    k, v, do = (randn(s, g, dtype, dev) for s in ((b, tk, hk, d), (b, tk, hk, d), (b, tq, h, d)))
    return q, k, v, do


def _mask(kind, b, tk, dev, seed=0):
    if kind is None:
        return None
    m = torch.rand(b, tk, generator=gen(seed)) > 0.3
    if kind == "lengths":
        n = torch.randint(1, tk + 1, (b, 1), generator=gen(seed))
        m = torch.arange(tk)[None] < n
    elif kind == "holes":  # whole tiles without a key
        m = (torch.arange(tk)[None] // 130 % 2 == 1).expand(b, tk).clone()
        m[:, -1] = True
    return m.to(dev)


def _run(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = fused_attention(*leaves, **kw)
    return [out, *torch.autograd.grad(out, leaves, do)]


def _check(q, k, v, do, what="", **kw):
    got = _run(q, k, v, do, **kw)
    with torch.no_grad():
        bare = fused_attention(q, k, v, **kw)
    want = attention64(q, k, v, do, **kw)
    u = 0.0 if q.dtype == F32 else half_step(q.dtype)
    # an fp32 logit z is off by 2^-24 |z| or more whatever is done (its own rounding, its scaling to
    # powers of two, the difference with the row's log-sum-exp, of the same size: four roundings),
    # and P by that times itself
    slack = 2e-5 + 2.0 ** -22 * want["largest"]
    for name, x in zip(NAMES, got):
        assert x.dtype == q.dtype and x.is_contiguous()
        within(x, want[name], want["tol_" + name], f"{what} {name}")
        # over one key dP = delta, so that dq and dk are 0 but for their sums: no size to relate to
        if k.shape[1] > 1 or name in ("out", "dv"):
            near(x, want[name], u, 3, f"{what} {name}", slack=slack)
    within(bare, want["out"], want["tol_out"], f"{what} out without a backward")
    return got


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("mask", [None, "lengths", "random"])
@pytest.mark.parametrize("b, tq, tk, h, hk, d", [
    (2, 17, 17, 2, 2, 64), (1, 130, 130, 2, 1, 128), (2, 65, 300, 6, 2, 80), (1, 33, 64, 3, 3, 16)])
def test_attention_values_and_gradients(cuda, b, tq, tk, h, hk, d, mask, causal, dtype):
    note(f"attention {b} {tq} {tk} {h} {hk} {d} {mask} {causal} {dtype}")
    _check(*_qkv(b, tq, tk, h, hk, d, dtype, cuda), causal=causal,
           key_mask=_mask(mask, b, tk, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 515])
def test_attention_lengths_at_tile_borders(cuda, n, dtype):
    """Rows, keys and both at the borders of the tiles (32, 64, 128)."""
    note(f"attention lengths {n} {dtype}")
    for tq, tk, causal in ((n, n, True), (n, 40, False), (40, n, False)):
        _check(*_qkv(1, tq, tk, 2, 1, 64, dtype, cuda, seed=n), f"{tq} {tk}", causal=causal)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("mask", [None, "lengths", "random"])
@pytest.mark.parametrize("b, tq, tk, h, hk, d", [
    (64, 33, 33, 4, 4, 64), (64, 70, 129, 4, 4, 128), (64, 129, 64, 4, 4, 40),
    (37, 65, 191, 21, 7, 72), (3, 300, 200, 86, 86, 64)])
def test_attention_over_many_heads(cuda, b, tq, tk, h, hk, d, mask, causal, dtype):
    """Blocks enough for every CU: each wavefront has rows, or keys, of its own."""
    note(f"attention many heads {b} {tq} {tk} {h} {hk} {d} {mask} {causal} {dtype}")
    _check(*_qkv(b, tq, tk, h, hk, d, dtype, cuda), causal=causal,
           key_mask=_mask(mask, b, tk, cuda))


@pytest.mark.parametrize("dtype, b, tq, tk, h, hk, d", [
    (BF16, 1, 4100, 4100, 4, 2, 128), (BF16, 1, 200, 30000, 8, 4, 128), (F16, 1, 30000, 200, 8, 4, 64),
    (F16, 2, 1700, 3300, 6, 3, 128), (F32, 1, 2100, 2100, 8, 4, 128), (F32, 1, 5000, 700, 16, 8, 96),
    (BF16, 1, 3000, 3100, 12, 12, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("mask", [None, "holes"])
def test_attention_long_axes_in_parts(cuda, dtype, b, tq, tk, h, hk, d, mask, causal):
    """Few heads over long sequences: the keys of a row, the rows of a key, in parts that are
    joined."""
    note(f"attention parts {b} {tq} {tk} {h} {hk} {d} {mask} {causal} {dtype}")
    _check(*_qkv(b, tq, tk, h, hk, d, dtype, cuda), causal=causal,
           key_mask=_mask(mask, b, tk, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [1, 2, 7, 8, 31, 37, 40, 63, 64, 65, 72, 96, 100, 127, 128])
def test_attention_head_widths(cuda, d, dtype):
    note(f"attention width {d} {dtype}")
    _check(*_qkv(2, 37, 70, 4, 2, d, dtype, cuda, seed=d), causal=True,
           key_mask=_mask("random", 2, 70, cuda))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("h, hk", [(1, 1), (8, 1), (6, 2), (12, 4), (40, 8), (33, 3), (67, 1)])
@pytest.mark.parametrize("tq, tk", [(1, 90), (3, 90), (50, 90)])
def test_attention_head_groups(cuda, tq, tk, h, hk, dtype):
    """Groups that end inside a tile of rows, a tile that ends inside a group."""
    note(f"attention groups {h} {hk} {tq} {dtype}")
    _check(*_qkv(2, tq, tk, h, hk, 64, dtype, cuda, seed=h), causal=True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b, tq, tk, h, hk, d", [
    (1, 1, 1, 1, 1, 64), (3, 1, 5000, 8, 2, 128), (1, 1, 20011, 4, 4, 64), (1, 5, 9001, 4, 1, 40),
    (2, 40, 6007, 2, 2, 128), (1, 6, 1176, 6, 6, 64)])
@pytest.mark.parametrize("mask", [None, "lengths", "holes"])
def test_attention_few_rows_over_many_keys(cuda, b, tq, tk, h, hk, d, mask, dtype):
    """The keys split over wavefronts and blocks, and joined; parts without a key among them."""
    note(f"attention few rows {b} {tq} {tk} {h} {hk} {d} {mask} {dtype}")
    _check(*_qkv(b, tq, tk, h, hk, d, dtype, cuda, seed=tk), causal=True,
           key_mask=_mask(mask, b, tk, cuda))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b, tq, tk, h, hk", [(8, 1, 3000, 16, 4), (2, 700, 900, 4, 2)])
def test_attention_holes_in_the_mask(cuda, b, tq, tk, h, hk, dtype):
    """Tiles that the mask leaves no key of are passed over."""
    note(f"attention holes {b} {tq} {tk} {dtype}")
    _check(*_qkv(b, tq, tk, h, hk, 64, dtype, cuda), causal=True,
           key_mask=_mask("holes", b, tk, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tq, tk", [(1, 70), (20, 9), (200, 150), (4, 3000)])
def test_attention_rows_without_a_key(cuda, tq, tk, dtype):
    """Zeros, and zero gradients, exactly: a sample whose mask leaves nothing, causal rows before
    the first key."""
    note(f"attention empty {tq} {tk} {dtype}")
    q, k, v, do = _qkv(3, tq, tk, 4, 2, 64, dtype, cuda)
    m = torch.ones(3, tk, dtype=torch.bool, device=cuda)
    m[1] = False
    m[2, : tk // 2] = False
    out, dq, dk, dv = _check(q, k, v, do, causal=True, key_mask=m)
    first = max(0, tq - tk)  # rows before it see no key
    for x in (out, dq):
        assert (x[1] == 0).all() and (x[:, :first] == 0).all()
    for x in (dk, dv):
        assert (x[~m] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tq, tk", [(1, 4000), (3, 200), (150, 150)])
def test_attention_masked_places_are_never_read(cuda, tq, tk, dtype):
    """NaN, infinities and the type's largest values in keys and values that the mask drops change
    no bit of any result."""
    note(f"attention masked places {tq} {tk} {dtype}")
    q, k, v, do = _qkv(2, tq, tk, 4, 2, 72, dtype, cuda)
    m = _mask("random", 2, tk, cuda)
    m[0, tk // 2:] = False
    want = _run(q, k, v, do, causal=True, key_mask=m)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min, torch.finfo(dtype).max):
        kb, vb = (torch.where(m[..., None, None], t, torch.tensor(bad, dtype=dtype, device=cuda))
                  for t in (k, v))
        got = _run(q, kb, vb, do, causal=True, key_mask=m)
        assert all(torch.equal(a, b) for a, b in zip(want, got)), bad


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tq, tk, d", [(150, 150, 72), (40, 300, 128), (129, 65, 32)])
def test_attention_masks_over_many_heads(cuda, tq, tk, d, dtype):
    """Blocks enough for every CU: samples and rows without a key give zeros, and what masked
    places hold changes no bit."""
    note(f"attention masks over many heads {tq} {tk} {d} {dtype}")
    q, k, v, do = _qkv(70, tq, tk, 8, 4, d, dtype, cuda)
    m = _mask("random", 70, tk, cuda)
    m[0, tk // 2:] = False
    m[1] = False
    m[2, : tk // 2] = False
    first = max(0, tq - tk)
    want = _check(q, k, v, do, causal=True, key_mask=m)
    for x in (want[0], want[1]):
        assert (x[1] == 0).all() and (x[:, :first] == 0).all()
    for x in (want[2], want[3]):
        assert (x[~m] == 0).all()
    for bad in (math.nan, -math.inf, torch.finfo(dtype).max):
        kb, vb = (torch.where(m[..., None, None], t, torch.tensor(bad, dtype=dtype, device=cuda))
                  for t in (k, v))
        got = _run(q, kb, vb, do, causal=True, key_mask=m)
        assert all(torch.equal(a, b) for a, b in zip(want, got)), bad


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tq", [1, 100])
def test_attention_a_nan_stays_in_its_head_and_sample(cuda, tq, dtype):
    note(f"attention nan {tq} {dtype}")
    q, k, v, do = _qkv(2, tq, 100, 4, 2, 64, dtype, cuda)
    want = _run(q, k, v, do)
    v2 = v.clone()
    v2[1, 50, 1, 3] = math.nan
    out = fused_attention(q, k, v2)
    assert out[1, :, 2:, 3].isnan().all()
    assert torch.equal(out[0], want[0][0]) and torch.equal(out[1, :, :2], want[0][1, :, :2])
    q2 = q.clone()
    q2[0, 0, 3] = math.nan
    out = fused_attention(q2, k, v)
    assert out[0, 0, 3].isnan().all()
    out[0, 0, 3] = want[0][0, 0, 3]
    assert torch.equal(out, want[0])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-3])
@pytest.mark.parametrize("tq", [2, 70])
def test_attention_scales(cuda, tq, scale, dtype):
    note(f"attention scale {scale} {tq} {dtype}")
    _check(*_qkv(2, tq, 90, 4, 2, 64, dtype, cuda), causal=True, scale=scale,
           key_mask=_mask("random", 2, 90, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attention_large_logits(cuda, dtype):
    """Logits of some hundreds: each row attends about one key, the maximum moves by much."""
    note(f"attention large logits {dtype}")
    q, k, v, do = _qkv(1, 150, 300, 2, 1, 64, dtype, cuda, sharp=100.0)
    _check(q, k, v, do)
    order = torch.argsort((k[0, :, 0].float() @ q[0, 0, 0].float()))
    _check(q, k[:, order].contiguous(), v, do)  # row 0's logits rise from key to key


@pytest.mark.parametrize("shift", [-22, -12, 0, 10])
@pytest.mark.parametrize("tq, tk", [(4, 300), (150, 200)])
def test_attention_fp16_gradients_of_any_size(cuda, tq, tk, shift):
    """dout by powers of two: dS keeps its precision, and the gradients are those of the plain
    dout by the same power where fp16 holds them."""
    note(f"attention fp16 range {tq} {tk} {shift}")
    q, k, v, do = _qkv(2, tq, tk, 4, 2, 64, F16, cuda)
    do = (do.float() * 2.0 ** shift).to(F16)
    _check(q, k, v, do, causal=tq == tk)


def test_attention_strided_operands(cuda, route):
    """Parts of one projection, [B, H, T, D] storage, broadcast heads and samples, operands that
    begin between vectors, gradients that are views: as their dense copies."""
    note(f"attention strides {route}")
    b, t, h, hk, d = 2, 70, 4, 2, 64
    g = gen(3)
    qkv = randn((b, t, h + 2 * hk, d), g, BF16, cuda)
    do = randn((b, t, h, d), g, BF16, cuda)
    m = _mask("random", b, t, cuda)
    q, k, v = qkv.split([h, hk, hk], 2)
    wide = randn((b, t, hk, d + 1), g, BF16, cuda)
    forms = [
        (q, k, v, do, m),
        (*(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, do)), m),
        (q, k[:, :, :1].expand(b, t, hk, d), v[:1].expand(b, t, hk, d), do, m),
        (q, k[:, :1].expand(b, t, hk, d), v, do[:1, :1, :1, :1].expand(b, t, h, d), m),
        (q, wide[..., 1:], wide[..., :d], do, m),
        (q.transpose(1, 3).contiguous().transpose(1, 3), k, v, do, m),
        (q, k, v, do, m.t().contiguous().t()),
        (q, k, v, do, m[:1].expand(b, t)),
        (q, k, v, do, torch.cat([m, m], 1)[:, 3:3 + t]),
        (q[:, ::2], k[:, ::2], v[:, 1::2], do[:, 1::2], m[:, ::2]),
        (q.flatten()[1:1 + 70 * 64].view(1, 70, 1, 64), *(x.flatten()[3:3 + 70 * 64].view(
            1, 70, 1, 64) for x in (k, v, do)), m[:1]),
    ]
    for i, (q, k, v, do, m) in enumerate(forms):
        dense = [x.contiguous().clone() for x in (q, k, v, do, m)]
        want = _run(*dense[:4], causal=True, key_mask=dense[4])
        got = _run(q, k, v, do, causal=True, key_mask=m)
        assert all(torch.equal(a, b) for a, b in zip(want, got)), i
    q, k, v = (x.detach().clone().requires_grad_(True) for x in qkv.split([h, hk, hk], 2))
    fused_attention(q, k, v).sum().backward()  # an expanded gradient of stride 0
    want = _run(q, k, v, torch.ones_like(q))
    assert torch.equal(q.grad, want[1]) and torch.equal(v.grad, want[3])


@pytest.mark.parametrize("tq", [1, 40])
def test_attention_cache_beyond_32_bit_offsets(cuda, tq):
    """Keys and values far apart in a buffer of more than 4 GiB, rows of q and dout too."""
    note(f"attention far rows {tq}")
    apart, tk, hk, d = 1 << 20, 2300, 2, 64
    room = torch.empty(tk * apart, dtype=BF16, device=cuda)
    assert room.numel() * 2 > 1 << 32
    q, k, v, do = _qkv(1, tq, tk, 4, hk, d, BF16, cuda)
    kf = room.as_strided((1, tk, hk, d), (room.numel(), apart, d, 1))
    vf = room.as_strided((1, tk, hk, d), (room.numel(), apart, d, 1), hk * d)
    kf.copy_(k)
    vf.copy_(v)
    want = _run(q, k, v, do, causal=True)
    got = _run(q, kf, vf, do, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    qf = room.as_strided(q.shape, (room.numel(), 50 * apart, d, 1), 2 * hk * d)
    df = room.as_strided(q.shape, (room.numel(), 50 * apart, d, 1), 2 * hk * d + 4 * d)
    qf.copy_(q)
    df.copy_(do)
    got = _run(qf, kf, vf, df, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_attention_many_small_samples(cuda):
    note("attention many samples")
    q, k, v, do = _qkv(3001, 3, 5, 2, 1, 16, BF16, cuda)
    _check(q, k, v, do, causal=True)
    _check(*_qkv(7, 2, 2, 3, 3, 8, F32, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tq, tk", [(3, 2000), (150, 150)])
def test_attention_gradients_asked_for_in_part(cuda, route, tq, tk, dtype):
    note(f"attention partial gradients {tq} {dtype} {route}")
    q, k, v, do = _qkv(2, tq, tk, 4, 2, 64, dtype, cuda)
    want = _run(q, k, v, do, causal=True)
    for pick in ((0,), (1,), (2,), (0, 2), (1, 2)):
        x = [t.detach().requires_grad_(i in pick) for i, t in enumerate((q, k, v))]
        out = fused_attention(*x, causal=True)
        got = torch.autograd.grad(out, [x[i] for i in pick], do)
        assert torch.equal(out, want[0])
        assert all(torch.equal(a, want[1 + i]) for a, i in zip(got, pick))
    # one tensor as key and value, and as all three
    x = q[:, :, :2].detach().requires_grad_(True)
    both = torch.autograd.grad(fused_attention(x, x, x), x, do[:, :, :2])[0]
    parts = _run(x, x, x, do[:, :, :2])
    assert torch.equal(both, sum(p for p in parts[1:])) or torch.allclose(
        both.double(), sum(p.double() for p in parts[1:]), rtol=3 * half_step(dtype),
        atol=3 * half_step(dtype) * float(both.abs().max()))


@pytest.mark.parametrize("b, tq, tk, h, hk, d, mask", [
    (2, 100, 100, 4, 2, 64, "random"), (8, 1, 3000, 8, 2, 128, "lengths"),
    (2, 6, 1176, 6, 6, 64, None)])
def test_attention_in_a_graph(cuda, b, tq, tk, h, hk, d, mask):
    """Replays give the eager bits, with eager work between; two graphs share no workspace."""
    note(f"attention graph {tq} {tk}")
    args = _qkv(b, tq, tk, h, hk, d, BF16, cuda)
    m = _mask(mask, b, tk, cuda)

    def make():
        q, k, v, do = (t.clone() for t in args)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]

        def step():
            out = fused_attention(*leaves, causal=True, key_mask=m)
            return [out.detach(), *torch.autograd.grad(out, leaves, do)]

        return step

    assert_graph_replays_match(make)
    assert_graph_replays_match(lambda: lambda: [fused_attention(*args[:3], key_mask=m)])
    graphs = []
    for seed in (1, 2):
        q, k, v, _ = _qkv(b, tq, tk, h, hk, d, BF16, cuda, seed=seed)
        want = fused_attention(q, k, v, key_mask=m)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = fused_attention(q, k, v, key_mask=m)
        graphs.append((graph, out, want, (q, k, v)))
    for _ in range(3):
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want, _ in graphs)


def test_attention_mask_that_changed_before_the_backward_raises(cuda, route):
    note(f"attention changed mask {route}")
    q, k, v, do = _qkv(2, 9, 70, 4, 2, 64, BF16, cuda)
    m = _mask("random", 2, 70, cuda)
    x = q.detach().requires_grad_(True)
    out = fused_attention(x, k, v, key_mask=m)
    m[0, 0] = ~m[0, 0]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, x, do)


def test_attention_same_bits_every_run(cuda):
    note("attention determinism")
    for shape in ((2, 300, 300, 8, 2, 128), (1, 2, 9000, 4, 1, 64), (1, 2000, 2000, 8, 4, 128)):
        args = _qkv(*shape, BF16, cuda)
        want = _run(*args, causal=True)
        for _ in range(4):
            assert all(torch.equal(a, b) for a, b in zip(want, _run(*args, causal=True)))


def test_block_ops_from_two_threads_on_two_streams(cuda):
    note("block ops threads")

    def work(seed):
        q, k, v, do = _qkv(2, 90, 90, 4, 2, 64, BF16, cuda, seed=seed)
        pos = torch.arange(90, device=cuda)[:, None]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        res = []
        with torch.cuda.stream(stream):
            for _ in range(6):
                x = [t.detach().requires_grad_(True) for t in (q, k, v)]
                a, c = fused_rotary(x[0], x[1], pos, (32,))
                out = fused_attention(a, c, x[2], causal=True)
                few = fused_attention(a[:, :1], c, x[2])
                res.append([out, few, *torch.autograd.grad([out, few], x, [do, do[:, :1]])])
            stream.synchronize()
        return res

    torch.cuda.synchronize()
    alone = [work(s)[0] for s in (1, 2)]
    with ThreadPoolExecutor(2) as ex:
        both = list(ex.map(work, (1, 2)))
    for want, got in zip(alone, both):
        for one in got:
            assert all(torch.equal(p, q) for p, q in zip(want, one, strict=True))


@pytest.mark.parametrize("b, tq, tk, h, hk, d, dtype, masked", [
    (2, 100, 130, 4, 2, 64, BF16, True), (1, 1, 5000, 8, 2, 128, BF16, False),
    (3, 33, 65, 3, 1, 40, F16, True), (1, 65, 65, 2, 2, 128, F32, True),
    (2, 5, 9001, 2, 1, 64, F32, False), (1, 4100, 4100, 2, 1, 128, BF16, True),
    (64, 40, 70, 4, 4, 64, BF16, True), (1, 300, 3000, 2, 2, 104, F16, False)])
def test_attention_buffers_of_exactly_the_size_asked_for(cuda, b, tq, tk, h, hk, d, dtype, masked):
    """The C entries with a state and workspaces of the bytes that the size calls name, outputs
    with room behind them: what lies behind stays as it was, and the results are the public
    call's."""
    note(f"attention exact buffers {b} {tq} {tk} {dtype}")
    L = _lib.lib()
    q, k, v, do = _qkv(b, tq, tk, h, hk, d, dtype, cuda)
    m = _mask("random", b, tk, cuda) if masked else None
    want = _run(q, k, v, do, causal=True, key_mask=m)
    dt, st, sizes = _lib.dtype_code(q), _lib.stream_of(q), (b, tq, tk, h, hk, d)

    def room(n):
        return torch.full((n + 4096,), 171, dtype=torch.uint8, device=cuda), n

    state, fw, bw = (room(n) for n in (
        L.nf_attention_state_bytes(*sizes, dt), L.nf_attention_fwd_workspace(*sizes, 1, dt),
        L.nf_attention_bwd_workspace(*sizes, 1, dt)))
    outs = [room(t.numel() * t.element_size()) for t in (q, q, k, v)]
    at = [(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)) for t in (q, k, v, do)]
    mask = (_lib.ptr(m), 0 if m is None else m.stride(0))
    _lib.check(L.nf_attention_fwd(
        *at[0], *at[1], *at[2], *mask, *sizes, 1, d ** -0.5, dt, outs[0][0].data_ptr(),
        state[0].data_ptr(), state[1], fw[0].data_ptr(), fw[1], st), "fwd")
    _lib.check(L.nf_attention_bwd(
        *at[0], *at[1], *at[2], *mask, outs[0][0].data_ptr(), *at[3], *sizes, 1, d ** -0.5, dt,
        state[0].data_ptr(), state[1], *(o[0].data_ptr() for o in outs[1:]), bw[0].data_ptr(), bw[1],
        st), "bwd")
    for x, n in (state, fw, bw, *outs):
        assert (x[n:] == 171).all()
    for (x, n), w in zip(outs, want):
        assert torch.equal(x[:n].view(dtype).view(w.shape), w)


def test_attention_the_eager_formulation_where_the_kernels_end(cuda):
    note("attention eager on the device")
    for d in (129, 192):
        q, k, v, do = _qkv(2, 9, 12, 4, 2, d, F32, cuda)
        got, want = _run(q, k, v, do, causal=True), attention64(q, k, v, do, causal=True)
        for name, x in zip(NAMES, got):
            near(x, want[name], 0, 0, name, slack=1e-5)
    q, k, v, _ = _qkv(2, 9, 12, 4, 2, 64, BF16, cuda)
    assert (fused_attention(q, k[:, :0], v[:, :0]) == 0).all()
    ref = fused_attention(q, k, v, force_reference=True)
    near(fused_attention(q, k, v), ref.double(), half_step(BF16), 3, "against the eager one")


def test_attention_refusals_on_the_device(cuda, route):
    note(f"attention refusals {route}")
    q, k, v, _ = _qkv(2, 3, 4, 4, 2, 64, BF16, cuda)
    m = torch.ones(2, 4, dtype=torch.bool, device=cuda)
    for bad in ((q[0], k, v), (q, k, v[:, :3]), (q[:, :, :3], k, v), (q, k, v.cpu())):
        with pytest.raises(ValueError, match="fused_attention"):
            fused_attention(*bad)
    with pytest.raises(ValueError, match="key_mask"):
        fused_attention(q, k, v, key_mask=m[:, :3])
    with pytest.raises(ValueError, match="key_mask is on cpu"):
        fused_attention(q, k, v, key_mask=m.cpu())
    with pytest.raises(TypeError):
        fused_attention(q, k.float(), v)
    with pytest.raises(ValueError, match="scale"):
        fused_attention(q, k, v, scale=math.inf)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def _turn(q, k, pos, sections, ups, **kw):
    x = [t.detach().requires_grad_(True) for t in (q, k)]
    out = fused_rotary(*x, pos, sections, **kw)
    return [*out, *torch.autograd.grad(out, x, ups)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("ladder", ["axis", "joint"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b, t, h, hk, d, sections", [
    (2, 70, 4, 2, 64, (8, 12, 12)), (8, 1, 16, 4, 128, (64,)), (3, 41, 5, 1, 90, (19, 18)),
    (1, 300, 3, 3, 13, (1, 0, 2, 2)), (2, 9, 1, 1, 2, (1,)), (1, 5, 2, 1, 600, (100, 99, 57)),
    (700, 2, 2, 2, 16, (3, 5))])
def test_rotary_values_and_gradients(cuda, b, t, h, hk, d, sections, ladder, interleaved, dtype):
    note(f"rotary {b} {t} {h} {hk} {d} {sections} {ladder} {interleaved} {dtype}")
    g = gen(t)
    q, k, uq, uk = (randn((b, t, n, d), g, dtype, cuda) for n in (h, hk, h, hk))
    pos = torch.randint(-100, 1_000_000, (b, t, len(sections)), generator=g).to(cuda)
    got = _turn(q, k, pos, sections, [uq, uk], base=7000.0, ladder=ladder, interleaved=interleaved)
    ref = (sections, 7000.0, ladder == "joint", interleaved)
    for i, (x, inverse) in enumerate(((q, False), (k, False), (uq, True), (uk, True))):
        within(got[i], *rotary64(x, pos, *ref, inverse=inverse), f"result {i}")
        assert got[i].is_contiguous() and got[i].dtype == dtype
        assert torch.equal(got[i][..., 2 * sum(sections):], x[..., 2 * sum(sections):])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_widths(cuda, interleaved, dtype):
    """Pairs and elements past them that are no whole pieces, and the widest heads; the same bits
    every run where pieces share elements."""
    for d, p in ((1024, 255), (1024, 256), (1024, 1), (1023, 250), (123, 18), (8, 1), (9, 4), (10, 1),
                 (14, 3), (15, 7), (17, 8), (21, 5), (24, 4), (25, 8), (26, 9), (34, 17), (47, 15),
                 (64, 9)):
        note(f"rotary width {d} {p} {interleaved} {dtype}")
        q, k = (randn((2, 40, n, d), gen(d), dtype, cuda) for n in (3, 1))
        pos = torch.randint(0, 9000, (2, 40, 1), generator=gen(p)).to(cuda)
        got = fused_rotary(q, k, pos, (p,), interleaved=interleaved)
        for x, y in zip((q, k), got):
            within(y, *rotary64(x, pos, (p,), interleaved=interleaved), f"{d} {p}")
            assert torch.equal(y[..., 2 * p:], x[..., 2 * p:])
        again = fused_rotary(q, k, pos, (p,), interleaved=interleaved)
        assert all(torch.equal(x, y) for x, y in zip(got, again))


def test_rotary_strides_positions_and_parts(cuda, route):
    note(f"rotary strides {route}")
    b, t, h, hk, d = 2, 30, 4, 2, 64
    g = gen(5)
    qkv = randn((b, t, h + 2 * hk, d), g, BF16, cuda)
    q, k, _ = qkv.split([h, hk, hk], 2)
    pos = torch.randint(0, 2000, (t, 2), generator=g).to(cuda)
    ups = [torch.ones_like(q), torch.ones_like(k)]
    want = _turn(q.contiguous(), k.contiguous(), pos, (20, 12), ups)
    wide = torch.empty(b, t, h, d + 3, dtype=BF16, device=cuda)
    wide[..., 3:] = q
    for q2, k2, p2, s2 in (
            (q, k, pos, (20, 12)), (q, k, pos[None], [20, 12]),
            (q, k, pos[None].expand(b, t, 2), (20, 12)),
            (q, k, pos.int(), (20, 12)), (q, k, pos.float(), (20, 12)),
            (wide[..., 3:], k.transpose(1, 2).contiguous().transpose(1, 2), pos, (20, 12)),
            (q.transpose(1, 3).contiguous().transpose(1, 3), k, pos.t().contiguous().t(), (20, 12))):
        got = _turn(q2, k2, p2, s2, ups)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    one, none = fused_rotary(q, None, pos, (20, 12))
    assert torch.equal(one, want[0]) and none is None
    for i in (0, 1):  # a gradient of one of the two
        x = [q.detach().requires_grad_(i == 0), k.detach().requires_grad_(i == 1)]
        out = fused_rotary(*x, pos, (20, 12))
        assert torch.equal(torch.autograd.grad(out[i], x[i], ups[i])[0], want[2 + i])
        x = [t.detach().requires_grad_(True) for t in (q, k)]
        out = fused_rotary(*x, pos, (20, 12))
        got = torch.autograd.grad(out[i], x, ups[i], allow_unused=True)
        assert torch.equal(got[i], want[2 + i])
        assert got[1 - i] is None or (got[1 - i] == 0).all()
    x = q.detach().requires_grad_(True)
    y = fused_rotary(x, None, pos, (20, 12))[0]
    assert torch.equal(torch.autograd.grad(y, x, ups[0])[0], want[2])
    same = q[:, :, :2].detach().requires_grad_(True)  # one tensor twice
    a, c = fused_rotary(same, same, pos, (20, 12))
    assert torch.equal(a, c)
    with pytest.raises(RuntimeError):  # positions that changed before the backward
        x = q.detach().requires_grad_(True)
        y = fused_rotary(x, None, p := pos.clone(), (20, 12))[0]
        p += 1
        torch.autograd.grad(y, x, ups[0])


def test_rotary_second_derivatives(cuda, route):
    """Linear: the gradient of the gradient's sum of squares is twice the identity's."""
    note(f"rotary second derivatives {route}")
    g = gen(2)
    q = randn((1, 9, 2, 16), g, F32, cuda).requires_grad_(True)
    k = randn((1, 9, 1, 16), g, F32, cuda).requires_grad_(True)
    pos = torch.arange(9, device=cuda)[:, None]
    out = fused_rotary(q, k, pos, (8,))
    up = [x.detach().clone().requires_grad_(True) for x in out]
    grads = torch.autograd.grad(out, [q, k], up, create_graph=True)
    second = torch.autograd.grad([x * x for x in grads], up, [torch.ones_like(x) for x in grads])
    for s, u in zip(second, up):  # |R^T u|^2 = |u|^2
        near(s, 2 * u.double(), 0, 0, "second", slack=1e-6)


def test_rotary_far_and_fractional_positions(cuda):
    note("rotary far positions")
    q = randn((1, 6, 2, 64), gen(1), F32, cuda)
    far = torch.tensor([[1 << 20], [(1 << 31) - 1], [-(1 << 31)], [1 << 40], [10 ** 9], [0]],
                       device=cuda)
    y, tol = rotary64(q, far, (32,))
    # 64-bit products of frequencies within 2^-52 of themselves: 2 pi 2^40 2^-52 radians at most
    tol = tol + far.abs().double()[None, :, :, None] * 2.0 ** -50 * q.abs().double().amax()
    within(fused_rotary(q, None, far, (32,))[0], y, tol, "far")
    part = torch.linspace(0.25, 77.75, 6, device=cuda)[:, None]
    within(fused_rotary(q, None, part, (32,))[0], *rotary64(q, part, (32,)), "fractions")


def test_rotary_beyond_32_bit_offsets(cuda):
    note("rotary far rows")
    apart, t = 1 << 21, 1100
    room = torch.empty(t * apart, dtype=BF16, device=cuda)
    q = randn((1, t, 2, 64), gen(0), BF16, cuda)
    far = room.as_strided(q.shape, (room.numel(), apart, 64, 1))
    far.copy_(q)
    pos = torch.arange(t, device=cuda)[:, None]
    assert torch.equal(fused_rotary(far, None, pos, (32,))[0], fused_rotary(q, None, pos, (32,))[0])


def test_rotary_outputs_of_exactly_their_size(cuda):
    note("rotary exact buffers")
    import ctypes

    for t, d, p, inter in ((7, 90, 37, 0), (33, 13, 5, 1), (5, 64, 32, 0)):
        q, k = (randn((2, t, n, d), gen(t), BF16, cuda) for n in (3, 1))
        pos = torch.arange(2 * t, device=cuda).view(2, t, 1)
        outs = [torch.full((x.numel() + 64,), 5.0, dtype=BF16, device=cuda) for x in (q, k)]
        _lib.check(_lib.lib().nf_rotary(
            q.data_ptr(), *q.stride()[:3], outs[0].data_ptr(), 3, k.data_ptr(), *k.stride()[:3],
            outs[1].data_ptr(), 1, pos.data_ptr(), t, 0, 2, t, d, (ctypes.c_int32 * 1)(p), 1, 1e4, 0,
            inter, 0, 1, _lib.stream_of(q)), "rotary")
        want = fused_rotary(q, k, pos, (p,), interleaved=bool(inter))
        for x, w in zip(outs, want):
            assert torch.equal(x[:w.numel()].view(w.shape), w) and (x[w.numel():] == 5.0).all()


def test_rotary_in_a_graph_reads_positions_at_replay(cuda):
    note("rotary graph")
    q, k = (randn((2, 40, n, 64), gen(n), BF16, cuda) for n in (4, 2))
    pos = torch.arange(40, device=cuda)[:, None].clone()

    def make():
        x = [t.clone().requires_grad_(True) for t in (q, k)]

        def step():
            out = fused_rotary(*x, pos, (32,))
            return [*(o.detach() for o in out),
                    *torch.autograd.grad(out, x, [torch.ones_like(o) for o in out])]

        return step

    assert_graph_replays_match(make)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, _ = fused_rotary(q, None, pos, (32,))
    for at in (0, 17, 100000):
        pos.copy_(torch.arange(40, device=cuda)[:, None] + at)
        graph.replay()
        assert torch.equal(out, fused_rotary(q, None, pos, (32,))[0])


# ---------------------------------------------------------------------------
# together, and what sees or replaces a call
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_block_of_them_trains(cuda, dtype):
    """Embedded tokens, one projection, turned, attended, a gated unit: values and gradients
    against the eager formulations of the same calls.  Both round at the same places; each
    rounding is off by u, and about a dozen lie between a leaf and the result."""
    note(f"block {dtype}")
    g = gen(8)
    b, t, h, hk, d = 2, 48, 4, 2, 32
    width = h * d
    table = randn((200, width), g, dtype, cuda)
    wqkv = randn((width, (h + 2 * hk) * d), g, dtype, cuda, std=width ** -0.5)
    wo = randn((width, 2 * width), g, dtype, cuda, std=width ** -0.5)
    ids = torch.randint(0, 200, (b, t), generator=g).to(cuda)
    frames = torch.stack([torch.arange(t) // 16, torch.arange(t) // 4 % 4, torch.arange(t) % 4], 1)
    mask = torch.ones(b, t, dtype=torch.bool, device=cuda)
    mask[1, 40:] = False

    def block(eager):
        leaves = [x.detach().clone().requires_grad_(True) for x in (table, wqkv, wo)]
        x = embedding_lookup(ids, leaves[0], force_reference=eager)
        q, k, v = (x.view(b * t, width) @ leaves[1]).view(b, t, h + 2 * hk, d).split([h, hk, hk], 2)
        q, k = fused_rotary(q, k, frames.to(cuda), (4, 6, 6), force_reference=eager)
        y = fused_attention(q, k, v, causal=True, key_mask=mask, force_reference=eager)
        u, w = ((y.reshape(b * t, width) + x.view(b * t, width)) @ leaves[2]).chunk(2, 1)
        out = fused_swiglu(u, w, force_reference=eager)
        return [out, *torch.autograd.grad(out.float().square().mean(), leaves)]

    u = 2.0 ** -22 if dtype == F32 else half_step(dtype)
    for i, (a, c) in enumerate(zip(block(False), block(True))):
        near(a, c.double(), u, 12, f"block result {i}")


def _calls(dev):
    q, k, v, _ = _qkv(2, 40, 40, 4, 2, 64, BF16, dev)
    pos = torch.arange(40, device=dev)[:, None]
    m = _mask("random", 2, 40, dev)
    return {
        "attention": (lambda a, b, c: (fused_attention(a, b, c, causal=True, key_mask=m),),
                      [q, k, v]),
        "few": (lambda a, b, c: (fused_attention(a, b, c),), [q[:, :1].clone(), k, v]),
        "rotary": (lambda a, b: fused_rotary(a, b, pos, (32,)), [q, k]),
    }


def _all(op, args):
    leaves = [v.detach().clone().requires_grad_(True) for v in args]
    outs = op(*leaves)
    ups = [torch.linspace(-1, 1, o.numel(), device=o.device).view(o.shape).to(o.dtype) for o in outs]
    return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, ups)]


@pytest.mark.parametrize("name", ["attention", "few", "rotary"])
def test_block_ops_saved_tensors_go_through_the_hooks(cuda, route, name):
    note(f"block ops hooks {name} {route}")
    op, args = _calls(cuda)[name]
    plain, packed = _all(op, args), []

    def pack(v):
        packed.append(v.shape)
        return v.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v.to(cuda)):
        hooked = _all(op, args)
    assert len(packed) == {"attention": 6, "few": 5, "rotary": 1}[name]
    assert all(torch.equal(a, b) for a, b in zip(plain, hooked, strict=True))


@pytest.mark.parametrize("name", ["attention", "few", "rotary"])
def test_block_ops_hooks_may_change_the_layout(cuda, route, name):
    """Saved tensors that come back with other strides."""
    note(f"block ops hooks that change strides {name} {route}")
    op, args = _calls(cuda)[name]
    plain = _all(op, args)

    def turned(v):  # the same values, the last axis outermost
        return v.movedim(-1, 0).contiguous().movedim(0, -1)

    with torch.autograd.graph.saved_tensors_hooks(lambda v: v, turned):
        hooked = _all(op, args)
    assert all(torch.equal(a, b) for a, b in zip(plain, hooked, strict=True))


@pytest.mark.parametrize("name", ["attention", "few", "rotary"])
def test_block_ops_under_modes_tracing_and_transforms(cuda, name):
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    note(f"block ops modes {name}")
    op, args = _calls(cuda)[name]
    plain, seen = _all(op, args), []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, a=(), kw=None):
            seen.append(str(func))
            return func(*a, **(kw or {}))

    class Functions(TorchFunctionMode):
        def __torch_function__(self, func, types, a=(), kw=None):
            return func(*a, **(kw or {}))

    for mode in (Dispatch, Functions):
        with mode():
            got = _all(op, args)
        assert all(torch.equal(a, b) for a, b in zip(plain, got, strict=True))
    assert any("empty" in f for f in seen)
    traced = torch.jit.trace(op, tuple(args), check_trace=False)
    assert all(torch.equal(a, b) for a, b in zip(op(*args), traced(*args), strict=True))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda *v: op(*v)[0])(*(v[None] for v in args))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises(RuntimeError):
            op(dual, *args[1:])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_second_derivatives_raise(cuda, route, dtype):
    note(f"attention second derivative {dtype} {route}")
    q, k, v, do = _qkv(1, 9, 9, 2, 2, 16, dtype, cuda)
    x = [t.detach().requires_grad_(True) for t in (q, k, v)]
    up = do.clone().requires_grad_(True)
    want = torch.autograd.grad(fused_attention(*x), x, up)
    got = torch.autograd.grad(fused_attention(*x), x, up, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for leaf in (*x, up):
        with pytest.raises(RuntimeError, match="fused_attention: second derivatives"):
            torch.autograd.grad(sum((t.float() ** 2).sum() for t in got), leaf, retain_graph=True,
                                allow_unused=True)
