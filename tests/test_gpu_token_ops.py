"""Token log probabilities, embedding lookup and dropout on the GPU, against 64-bit
restatements (tests/token_ops_ref.py) within bounds derived there.
"""

from __future__ import annotations

import math

import pytest
import torch

from nuvla_forge_amd.kernels import (
    chunked_token_logprobs,
    embedding_lookup,
    fused_dropout,
    fused_gate_up_swiglu,
)
from nuvla_forge_amd.kernels.dropout import dropout_threshold
from nuvla_forge_amd.kernels.reference import dropout_keep

from .helpers import assert_graph_replays_match, gen, note, randn
from .token_ops_ref import half_step, least_step, logprobs64

pytestmark = pytest.mark.gpu
BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
def _dropout_check(x, p, seed, offset, r, dout):
    """Values: a product and a sum, each off by 2^-24 of itself before the store's rounding."""
    x.requires_grad_(True)
    out = fused_dropout(x, p, seed, offset=offset, residual=r)
    (dx,) = torch.autograd.grad(out, x, dout)
    t = dropout_threshold(p)
    s = seed.cpu() if isinstance(seed, torch.Tensor) else seed
    keep = dropout_keep(x.shape, t, s, offset, "cpu").to(x.device)
    f = 65536 / (65536 - t) if t < 65536 else 0.0
    y = torch.where(keep, x.detach().double() * f, 0.0)
    want = y if r is None else y + r.double()
    assert out.dtype == (x.dtype if r is None else r.dtype) and out.shape == x.shape
    tol = (half_step(out.dtype) * want.abs() + least_step(out.dtype)
           + 3 * 2.0 ** -24 * (y.abs() + want.abs()))
    fine = torch.isfinite(want)
    assert ((out.double() - want).abs()[fine] <= tol[fine]).all()
    assert torch.equal(out.double()[~fine].isnan(), want[~fine].isnan())
    gx = torch.where(keep, dout.double() * f, 0.0)
    tol = (half_step(dx.dtype) + 2.0 ** -23) * gx.abs() + least_step(dx.dtype)
    assert ((dx.double() - gx).abs() <= tol).all()
    assert (dx[~keep] == 0).all()
    return out, dx


@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (513,), (48, 384), (33, 1001), (2, 3, 1024)])
@pytest.mark.parametrize("dtype, rtype", [(F32, None), (BF16, None), (F16, None), (BF16, BF16),
                                          (BF16, F32), (F16, F32), (F16, F16), (F32, F32)])
def test_dropout_matches_definition(cuda, shape, dtype, rtype):
    note(f"dropout {shape} {dtype} {rtype}")
    g = gen(1)
    x = randn(shape, g, dtype, cuda)
    r = None if rtype is None else randn(shape, g, rtype, cuda)
    dout = randn(shape, g, dtype if rtype is None else rtype, cuda)
    for p, seed, offset in ((0.1, 3, 0), (0.5, torch.tensor([1 << 61], device=cuda), 5),
                            (0.0, -1, 2), (1.0, 9, 1 << 40), (2.0 ** -17, 4, 1)):
        _dropout_check(x.detach().clone(), p, seed, offset, r, dout)


def test_dropout_views_and_masked_values(cuda):
    note("dropout views")
    g = gen(2)
    base = randn((65, 131), g, BF16, cuda)
    dout = randn((64, 130), g, BF16, cuda)
    _dropout_check(base[1:, 1:].detach(), 0.3, 11, 0, randn((64, 130), g, BF16, cuda), dout)
    flat = randn((1025,), g, BF16, cuda)
    _dropout_check(flat[1:].detach(), 0.3, 11, 0, None, randn((1024,), g, BF16, cuda))
    t = randn((40, 24), g, F32, cuda).t()
    _dropout_check(t.detach(), 0.3, 11, 0, None, randn((40, 24), g, F32, cuda).t())
    # what a dropped place holds does not matter
    x = torch.full((4096,), float("nan"), device=cuda)
    keep = dropout_keep((4096,), 32768, 5, 0, "cpu").to(cuda)
    out = fused_dropout(x, 0.5, 5)
    assert (out[~keep] == 0).all() and out[keep].isnan().all()
    assert fused_dropout(x[:0], 0.5, 5).shape == (0,)


def test_dropout_seed_changed_before_backward_raises(cuda):
    seed = torch.tensor([3], device=cuda)
    x = torch.ones(16, device=cuda, requires_grad=True)
    out = fused_dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_dropout_graph_reads_the_seed_at_replay(cuda):
    note("dropout graph")
    x = randn((48, 384), gen(3), BF16, cuda)
    r = randn((48, 384), gen(4), F32, cuda)
    seed = torch.tensor([100], device=cuda)

    def step():
        leaf = x.detach().requires_grad_(True)
        out = fused_dropout(leaf, 0.2, seed, offset=1, residual=r)
        return [out.detach(), *torch.autograd.grad(out, leaf, torch.ones_like(out))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        seed.fill_(100 + k)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want), k
        torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# embedding lookup
# ---------------------------------------------------------------------------
def _embedding_check(ids, table, scale=1.0, pad=None, out_dtype=None, dout=None):
    """Forward: one fp32 product and one rounding.  Gradient: fp32 sums of the rows, at
    most n additions each off by 2^-24 of the sum of absolute values, the scale's product, and
    the store's rounding."""
    v, d = table.shape
    table.requires_grad_(True)
    out = embedding_lookup(ids, table, scale=scale, padding_idx=pad, out_dtype=out_dtype)
    od = table.dtype if out_dtype is None else out_dtype
    live = (ids >= 0) & (ids < v)
    safe = torch.where(live, ids, 0).long()
    want = torch.where(live[..., None], table.detach()[safe].float() * scale, 0.0).to(od)
    assert out.dtype == od and out.shape == want.shape
    if od == F16:
        # the product may go to fp16 in one rounding (half a step off) or by way of fp32 (2^-24
        # more): 22 of 384000 products next to a tie come out on the other side of it
        exact = torch.where(live[..., None], table.detach()[safe].double()
                            * torch.tensor(scale).double().item(), 0.0)
        tol = (half_step(od) + 2.0 ** -24) * exact.abs() + least_step(od)
        assert ((out.double() - exact).abs() <= tol).all()
    else:
        assert torch.equal(out, want)
    if dout is None:
        dout = torch.randn(out.shape, generator=gen(9)).to(od).to(table.device)
    (dt,) = torch.autograd.grad(out, table, dout)
    use = live if pad is None else live & (ids != pad)
    rows = torch.where(use[..., None], dout.double(), 0.0).reshape(-1, d)
    flat = safe.reshape(-1)
    grad, size = (torch.zeros(v, d, dtype=torch.float64, device=table.device) for _ in "12")
    grad.index_put_((flat,), rows, accumulate=True)
    size.index_put_((flat,), rows.abs(), accumulate=True)
    n = torch.bincount(flat[use.reshape(-1)], minlength=v)[:, None]
    grad, size = grad * scale, size * abs(scale)
    tol = (n + 2) * 2.0 ** -24 * size + (
        half_step(dt.dtype) * (grad.abs() + 2.0 ** -20 * size) + least_step(dt.dtype))
    assert dt.dtype == table.dtype and dt.shape == table.shape
    assert ((dt.double() - grad).abs() <= tol).all()
    assert (dt[(n == 0)[:, 0]] == 0).all()
    (again,) = torch.autograd.grad(embedding_lookup(ids, table, scale, pad, out_dtype), table, dout)
    assert torch.equal(dt, again)  # the same bits every run
    return out, dt


@pytest.mark.parametrize("m, d, v", [(1, 1, 1), (8, 384, 32000), (512, 384, 1000), (33, 7, 5),
                                     (2000, 1001, 77), (300, 2, 9), (4097, 520, 50001),
                                     (100, 2048, 3), (257, 64, 140001)])
@pytest.mark.parametrize("dtype, od", [(F32, None), (BF16, None), (F16, None), (F32, BF16),
                                       (F32, F16)])
def test_embedding_matches_definition(cuda, m, d, v, dtype, od):
    note(f"embedding {m} {d} {v} {dtype} {od}")
    g = gen(m + d + v)
    table = randn((v, d), g, dtype, cuda, std=0.05)
    # crowded ids: squares of a uniform number
    ids = (torch.rand(m, generator=g) ** 2 * v).long().clamp(max=v - 1).to(cuda)
    _embedding_check(ids, table, scale=math.sqrt(d), out_dtype=od)


@pytest.mark.parametrize("count", [1, 2, 31, 32, 33, 63, 64, 65, 1000, 9000])
def test_embedding_gradient_of_one_token_many_times(cuda, count):
    """Runs that end inside a span, at its border and far past it, at every offset of a span."""
    note(f"embedding run {count}")
    g = gen(count)
    for before in (0, 1, 31, 32, 40):
        ids = torch.cat([torch.arange(before) % 3, torch.full((count,), 5), torch.arange(7) + 6])
        ids = ids[torch.randperm(len(ids), generator=g)].to(cuda)
        for d in (8, 72, 1032):
            _embedding_check(ids, randn((20, d), g, BF16, cuda))
        _embedding_check(ids, randn((20, 9), g, F32, cuda), scale=-0.5)


def test_embedding_ids_that_do_not_count(cuda):
    note("embedding ids")
    g = gen(5)
    table = randn((50, 40), g, F32, cuda)
    ids = torch.randint(-20, 70, (600,), generator=g)
    ids[:4] = torch.tensor([1 << 40, -(1 << 40), (1 << 63) - 1, -(1 << 63)])
    _embedding_check(ids.to(cuda), table, pad=7)
    _embedding_check(torch.full((100,), 7, device=cuda), table, pad=7)  # nothing but padding
    _embedding_check(torch.full((100,), -1, device=cuda), table)
    _embedding_check(torch.zeros(0, dtype=torch.int64, device=cuda), table)
    _embedding_check(torch.randint(0, 50, (4, 3, 5), generator=g).int().to(cuda), table, pad=0)


def test_embedding_views(cuda):
    note("embedding views")
    g = gen(6)
    ids = torch.randint(0, 30, (90, 2), generator=g).to(cuda)[:, 0]
    wide = randn((30, 131), g, BF16, cuda)
    _embedding_check(ids, wide[:, 1:129].detach())  # rows that are not whole vectors
    _embedding_check(ids, wide[:, :128].detach())
    _embedding_check(ids, randn((128, 30), g, BF16, cuda).t().detach())
    _embedding_check(ids, randn((1, 16), g, F32, cuda).expand(30, 16).detach())
    one = torch.ones((), device=cuda)
    _embedding_check(ids, randn((30, 64), g, F32, cuda), dout=one.expand(90, 64))


def test_embedding_graph_and_stream(cuda):
    note("embedding graph")
    g = gen(7)
    table = randn((1000, 96), g, BF16, cuda)
    ids = (torch.rand(700, generator=g) ** 3 * 1000).long().to(cuda)
    dout = randn((700, 96), g, BF16, cuda)

    def make():
        leaf = table.detach().clone().requires_grad_(True)

        def step():
            out = embedding_lookup(ids, leaf, scale=2.0, padding_idx=0)
            return [out.detach(), *torch.autograd.grad(out, leaf, dout)]

        return step

    assert_graph_replays_match(make)
    want = make()()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = make()()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------
def _head(m, d, v, dtype, dev, seed=0, grid=False, ignored=0.2, std=None):
    g = gen(seed)
    std = 2.0 / math.sqrt(d) if std is None else std
    h, w = torch.randn(m, d, generator=g), torch.randn(v, d, generator=g) * std
    if grid:  # values on which every logit is exact in fp32: h in 1/16, w in 1/1024
        h, w = (h * 16).round() / 16, (w * 1024).round() / 1024
    t = torch.randint(0, v, (m,), generator=g)
    t[torch.rand(m, generator=g) < ignored] = -100
    up = torch.randn(2, m, generator=g)
    return (h.to(dtype).to(dev), w.to(dtype).to(dev), t.to(dev), up[0].to(dev), up[1].to(dev))


def _logprobs_check(h, w, t, g, gh, k=0, chunk_size=1024, need=(True, True), ids=True):
    h, w = h.detach().requires_grad_(need[0]), w.detach().requires_grad_(need[1])
    out = chunked_token_logprobs(h, w, t, top_k=k, chunk_size=chunk_size)
    ref = logprobs64(h, w, t, g, gh, k)
    for name, tol in (("logprobs", "tol_lp"), ("entropy", "tol_ent")):
        off = (getattr(out, name).double() - ref[name]).abs()
        assert (off <= ref[tol]).all(), (name, (off / ref[tol]).max())
    if k:
        off = (out.top_logprobs.double() - ref["top_logprobs"]).abs()
        assert (off <= ref["tol_lp"][:, None] + 2.0 ** -22 * ref["top_logprobs"].abs()).all()
        if ids:
            assert torch.equal(out.top_ids, ref["top_ids"])
    leaves = [x for x in (h, w) if x.requires_grad]
    if leaves:
        grads = iter(torch.autograd.grad([out.logprobs, out.entropy], leaves, [g, gh]))
        for name, x in (("dh", h), ("dw", w)):
            if x.requires_grad:
                got = next(grads)
                off = (got.double() - ref[name]).abs()
                assert got.dtype == x.dtype
                assert (off <= ref["tol_" + name]).all(), (name, (off / ref["tol_" + name]).max())
    return out, ref


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m, d, v, k", [
    (1, 64, 1000, 5), (2, 384, 32000, 8), (3, 256, 333, 0), (17, 40, 130, 3), (33, 2048, 515, 20),
    (5, 8, 7, 7), (1, 1, 1, 1), (40, 101, 259, 4), (300, 384, 4099, 8), (257, 128, 50001, 20),
    (600, 64, 5000, 32), (65, 520, 2049, 1)])
def test_logprobs_match_definition(cuda, m, d, v, k, dtype):
    note(f"logprobs {m} {d} {v} {k} {dtype}")
    _logprobs_check(*_head(m, d, v, dtype, cuda, seed=m + v, grid=True), k)
    _logprobs_check(*_head(m, d, v, dtype, cuda, seed=m), k, ids=False)


@pytest.mark.parametrize("m", [33, 64])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logprobs_few_rows_of_a_large_vocabulary(cuda, m, dtype):
    note(f"logprobs few rows {m} {dtype}")
    for d, v, k in ((72, 33001, 8), (37, 40000, 20)):
        _logprobs_check(*_head(m, d, v, dtype, cuda, seed=m + d, grid=True), k)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logprobs_in_chunks(cuda, dtype):
    note(f"logprobs chunks {dtype}")
    args = _head(1100, 96, 3001, dtype, cuda, grid=True)
    whole, _ = _logprobs_check(*args, 6, chunk_size=4096)
    part, _ = _logprobs_check(*args, 6, chunk_size=1)
    assert torch.equal(whole.top_ids, part.top_ids)


@pytest.mark.parametrize("m, d, v, chunk_size", [(1100, 1024, 1001, 8), (129, 1024, 100, 1024),
                                                 (700, 384, 3001, 1)])
def test_logprobs_kept_in_one_small_chunk(cuda, m, d, v, chunk_size):
    """The accumulator's share of the memory bound keeps every row's logits at once."""
    note(f"logprobs kept {m} {d} {v} {chunk_size}")
    args = _head(m, d, v, BF16, cuda, grid=True)
    few, _ = _logprobs_check(*args, 20, chunk_size=chunk_size)
    many, _ = _logprobs_check(*args, 20, chunk_size=4096)
    for a, b in zip(few, many):
        assert torch.equal(a, b)


def test_logprobs_ties_go_to_the_lower_token(cuda):
    """Equal rows of the head far apart, and a hidden row of zeros: every logit equal."""
    note("logprobs ties")
    for m, v in ((6, 1000), (300, 5003), (40, 40000)):
        h, w, t, g, gh = _head(m, 64, v, BF16, cuda, seed=v, grid=True, ignored=0.0)
        w[v // 2:] = w[: v - v // 2].clone()
        w[7::13] = w[3]
        h[1] = 0
        h[4] = (w[3].float() * 16).round() / 16 * 4
        _logprobs_check(h, w, t, g, gh, 12)
        h, w = h.float(), w.float()
        out, _ = _logprobs_check(h, w, t, g, gh, 12)
        assert out.top_ids[1].tolist() == list(range(12))
        assert abs(out.entropy[1].item() - math.log(v)) < 1e-5


@pytest.mark.parametrize("k", [1, 4, 8, 32])
@pytest.mark.parametrize("m, v", [(3, 70), (3, 32000), (300, 5000), (300, 130000)])
def test_logprobs_many_equal_logits(cuda, m, v, k):
    """Rows of equal logits, and rows whose best k - 1, k, 65 and 66 logits alone are equal."""
    note(f"logprobs equal {m} {v} {k}")
    h, w = torch.zeros(m, 64, device=cuda), torch.zeros(v, 64, device=cuda)
    places = torch.randperm(v, generator=gen(v + k))
    for c, n in enumerate((k - 1, k, 65, 66)):
        w[places[:min(n, v)], c] = 1.0
        h[c % m, :4] = 0.0
        h[c % m, c] = 2.0
    if m > 4:
        h[4, 0], h[5, 2] = -2.0, -2.0  # the equal ones last
    w[:, 8] = -torch.arange(v, device=cuda) / 2.0 ** 20  # falling: exact in fp32 and its parts
    if m > 6:
        h[6, 8] = 1.0
    t = torch.zeros(m, dtype=torch.int64, device=cuda)
    out = chunked_token_logprobs(h, w, t, top_k=k)
    val, idx = torch.sort(h @ w.T, dim=1, descending=True, stable=True)
    assert torch.equal(out.top_ids, idx[:, :k])
    want = torch.log_softmax((h @ w.T).double(), 1).gather(1, idx[:, :k])
    # logits are exact; log S and the difference: 2^-22 of them, log 130000 < 12, and V / 64 + 64
    # roundings of S
    tol = 2.0 ** -22 * 16 + (v / 64 + 64) * 2.0 ** -24
    assert ((out.top_logprobs.double() - want).abs() <= tol).all()


def test_logprobs_alternatives_crowded_in_one_place(cuda):
    """The most probable tokens next to each other, at every place of the vocabulary's tiles."""
    note("logprobs crowded")
    for m in (9, 280):
        h, w, t, g, gh = _head(m, 64, 2000, BF16, cuda, seed=m, grid=True, ignored=0.0)
        h[:, 0] = 4.0
        for at in (0, 60, 120, 250, 1000, 1980):
            x = w.clone()
            x[at:at + 20, 0] += torch.arange(20, device=cuda) % 7 / 4 + 2
            out, _ = _logprobs_check(h, x, t, g, gh, 16, need=(False, False))
            assert ((out.top_ids >= at) & (out.top_ids < at + 20)).float().mean() > 0.9


def test_logprobs_far_targets_and_large_logits(cuda):
    """Logits of deviation ~100: probabilities of 0 and 1, given tokens hundreds of nats away."""
    note("logprobs far")
    for dtype in (BF16, F32):
        for m in (20, 300):
            _logprobs_check(*_head(m, 64, 3001, dtype, cuda, std=12.0), 3, ids=False)


def test_logprobs_logits_of_minus_infinity(cuda):
    """Tokens that a huge negative weight rules out: no probability, no part in the entropy."""
    note("logprobs -inf")
    for m in (4, 270):
        for dtype in (F32, BF16):
            h, w, t, g, gh = _head(m, 64, 1500, dtype, cuda, grid=True, ignored=0.0)
            h[:, :2] = 8.0
            base = _logprobs_check(h, w[:1400], t % 1400, g, gh, 5)[0]
            w[:, :2] = 0
            w[1400:] = 0
            w[1400:, :2] = -3.0e38  # 8 * -3e38 twice: -inf in fp32
            h, w = h.requires_grad_(True), w.requires_grad_(True)
            out = chunked_token_logprobs(h, w, t % 1400, top_k=5)
            z = h.detach().double() @ w.detach()[:1400].double().T
            lp = z.log_softmax(1)
            want = lp.gather(1, (t % 1400)[:, None])[:, 0]
            assert (out.logprobs.double() - want).abs().max() < 1e-4
            ent = -(lp.exp() * lp).sum(1)
            assert (out.entropy.double() - ent).abs().max() < 1e-4
            assert (out.top_ids < 1400).all() and base.top_ids.shape == out.top_ids.shape
            dh, dw = torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh])
            assert torch.isfinite(dh).all() and torch.isfinite(dw).all()
            assert (dw[1400:] == 0).all()


def test_logprobs_nan_stays_in_its_row(cuda):
    note("logprobs nan")
    for m in (6, 260):
        for dtype in (BF16, F32):
            h, w, t, g, gh = _head(m, 64, 700, dtype, cuda, ignored=0.0)
            clean = chunked_token_logprobs(h, w, t, top_k=3)
            h[2, 5] = float("nan")
            h = h.requires_grad_(True)
            out = chunked_token_logprobs(h, w, t, top_k=3)
            rest = torch.arange(m, device=cuda) != 2
            for a, b in zip(out, clean):
                assert torch.equal(a[rest], b[rest])
            assert out.logprobs[2].isnan() and out.entropy[2].isnan()
            assert out.top_logprobs[2].isnan().all()
            assert ((out.top_ids[2] >= -1) & (out.top_ids[2] < 700)).all()
            (dh,) = torch.autograd.grad(out.logprobs, h, g)
            assert dh[2].isnan().all() and torch.isfinite(dh[rest]).all()


@pytest.mark.parametrize("m", [6, 100, 290])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logprobs_rows_left_out_may_hold_anything(cuda, m, dtype):
    """NaN and infinities in a row that is left out, and in its upstream gradients, reach nothing."""
    note(f"logprobs ignored nan {m} {dtype}")
    h, w, t, g, gh = _head(m, 64, 900, dtype, cuda, ignored=0.0)
    t[2] = -100
    h[2, ::3], h[2, 1] = float("nan"), float("inf")
    g[2], gh[2] = float("nan"), float("inf")
    ref = logprobs64(torch.where(torch.isfinite(h), h, 0.0), w, t, torch.where(t >= 0, g, 0.0),
                     torch.where(t >= 0, gh, 0.0))
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    out = chunked_token_logprobs(h, w, t, top_k=2)
    assert out.logprobs[2] == 0 and out.entropy[2] == 0 and (out.top_ids[2] == -1).all()
    for x, name in zip(torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh]),
                       ("dh", "dw")):
        assert ((x.double() - ref[name]).abs() <= ref["tol_" + name]).all(), name


@pytest.mark.parametrize("m", [6, 100, 290])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logprobs_infinite_weight_and_rows_left_out(cuda, m, dtype):
    """A token that a weight of -inf rules out has probability 0 in every row; the rows left out,
    which the products see as zeros, add no 0 * inf to weight's gradient."""
    note(f"logprobs inf weight {m} {dtype}")
    h, w, t, g, gh = _head(m, 64, 900, dtype, cuda, ignored=0.3)
    h[:, 0] = h[:, 0].abs() + 0.125
    t = torch.where(t == 7, 8, t)
    t[0], t[1] = -100, 8  # both kinds at every size
    w[7, 0] = float("-inf")
    h[0, 0] = 0.0  # 0 * inf where it does not count
    out = chunked_token_logprobs(h, w.requires_grad_(True), t)
    (dw,) = torch.autograd.grad([out.logprobs, out.entropy], [w], [g, gh])
    rest = torch.arange(900, device=cuda) != 7
    ref = logprobs64(h, w.detach()[rest], torch.where(t > 7, t - 1, t), g, gh)
    assert ((out.logprobs.double() - ref["logprobs"]).abs() <= ref["tol_lp"]).all()
    assert ((out.entropy.double() - ref["entropy"]).abs() <= ref["tol_ent"]).all()
    assert (dw[7] == 0).all()
    assert ((dw[rest].double() - ref["dw"]).abs() <= ref["tol_dw"]).all()


def test_logprobs_past_two_gib(cuda):
    """What is kept for the backward takes more than 2 GiB: 32-bit offsets do not reach it."""
    note("logprobs past 2 GiB")
    m, d, v = 16700, 32, 65601
    h, w, t, g, gh = _head(m, d, v, BF16, cuda, grid=True)
    assert 2 * 16896 * 65664 > 1 << 31
    for chunk_size in (m, 1024):
        _logprobs_check(h, w, t, g, gh, 3, chunk_size=chunk_size)


def test_token_ops_from_two_threads_on_two_streams(cuda):
    note("token ops threads")
    from concurrent.futures import ThreadPoolExecutor

    def work(seed):
        h, w, t, g, gh = _head(200, 64, 1500, BF16, cuda, seed=seed)
        table = randn((1500, 64), gen(seed), F32, cuda)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        res = []
        with torch.cuda.stream(stream):
            for _ in range(6):
                a, b, c = (x.detach().requires_grad_(True) for x in (h, w, table))
                lp = chunked_token_logprobs(a, b, t, top_k=3)
                emb = embedding_lookup(t.clamp(min=0), c, out_dtype=BF16)
                out = fused_dropout(emb, 0.2, seed, residual=a)
                res.append([*lp, out, *torch.autograd.grad(
                    [lp.logprobs, lp.entropy, out], [a, b, c], [g, gh, torch.ones_like(out)])])
            stream.synchronize()
        return res

    torch.cuda.synchronize()
    alone = [work(s)[0] for s in (1, 2)]
    with ThreadPoolExecutor(2) as ex:
        both = list(ex.map(work, (1, 2)))
    for want, got in zip(alone, both):
        for one in got:
            assert all(torch.equal(p, q) for p, q in zip(want, one, strict=True))


@pytest.mark.parametrize("m", [5, 290])
def test_logprobs_rows_left_out(cuda, m):
    note(f"logprobs ignored {m}")
    h, w, t, g, gh = _head(m, 64, 900, BF16, cuda, grid=True)
    t[0], t[1], t[3] = -1, 900, 1 << 40
    out, _ = _logprobs_check(h, w, t, g, gh, 4)
    assert (out.top_ids[[0, 1, 3]] == -1).all() and (out.logprobs[[0, 1, 3]] == 0).all()
    t[:] = -100  # none left
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    out = chunked_token_logprobs(h, w, t, top_k=4)
    assert (out.logprobs == 0).all() and (out.entropy == 0).all() and (out.top_ids == -1).all()
    for x in torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh]):
        assert (x == 0).all()
    out = chunked_token_logprobs(h[:0], w, t[:0], top_k=2)
    assert out.top_ids.shape == (0, 2)
    dh, dw = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum(), [h, w])
    assert (dh == 0).all() and (dw == 0).all()


def test_logprobs_one_gradient_at_a_time(cuda):
    note("logprobs single gradients")
    for m, dtype in ((300, BF16), (40, F32)):
        h, w, t, g, gh = _head(m, 128, 1500, dtype, cuda)
        zero = torch.zeros_like(g)
        for need in ((True, False), (False, True)):
            _logprobs_check(h, w, t, g, gh, need=need)
        h, w = h.requires_grad_(True), w.requires_grad_(True)
        for i in range(2):
            out = chunked_token_logprobs(h, w, t)
            got = torch.autograd.grad(out[i], [h, w], (g, gh)[i])
            ref = logprobs64(h, w, t, *((g, zero) if i == 0 else (zero, gh)))
            for x, name in zip(got, ("dh", "dw")):
                assert ((x.double() - ref[name]).abs() <= ref["tol_" + name]).all()


@pytest.mark.parametrize("m, chunk_size", [(3, 1024), (100, 1024), (300, 1024), (300, 1)])
def test_logprobs_backward_twice(cuda, m, chunk_size):
    """What the forward kept serves again: two backward passes of one graph give the same bits."""
    note(f"logprobs twice {m} {chunk_size}")
    h, w, t, g, gh = _head(m, 64, 1500, BF16, cuda)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    out = chunked_token_logprobs(h, w, t, chunk_size=chunk_size)
    first = torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh], retain_graph=True)
    again = torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh])
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_logprobs_gradient_of_few_rows_is_rounded_once(cuda):
    """With few rows dz is held as two bf16 terms (2^-16 of it left), so the gradients are off by
    little more than their own rounding."""
    note("logprobs few rows")
    for m in (1, 2, 9, 65, 128):
        h, w, t, g, gh = _head(m, 128, 2003, BF16, cuda, seed=m, std=0.5)
        h, w = h.requires_grad_(True), w.requires_grad_(True)
        out = chunked_token_logprobs(h, w, t)
        ref = logprobs64(h.float(), w.float(), t, g, gh)  # fp32's bounds, without bf16's
        for x, name in zip(torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh]),
                           ("dh", "dw")):
            off = (x.double() - ref[name]).abs()
            size = torch.zeros_like(off)
            tol = ref["tol_" + name] * 2 + half_step(BF16) * ref[name].abs()
            # 2^-16 of dz, against the sum of |dz||w| or |dz||h|: from the bound of one bf16 term
            one = logprobs64(h, w, t, g, gh)["tol_" + name]
            assert (off <= tol + 2.0 ** -7 * one + size).all(), (m, name, (off / tol).max())


def test_logprobs_types_and_views(cuda):
    note("logprobs types")
    h, w, t, g, gh = _head(50, 64, 700, F32, cuda)
    h2 = torch.cat([h, h], 1)[:, :64]
    w2 = w.t().contiguous().t()
    _logprobs_check(h2, w2, t.int(), g, gh, 3, ids=False)
    # fp16 is widened; under bf16 autocast everything is bf16 and the gradients keep their types
    out = chunked_token_logprobs(h.half(), w.half(), t, top_k=3)
    ref = logprobs64(h.half().float(), w.half().float(), t, g, gh)
    assert ((out.logprobs.double() - ref["logprobs"]).abs() <= ref["tol_lp"]).all()
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    with torch.autocast("cuda", dtype=BF16):
        out = chunked_token_logprobs(h, w, t)
    ref = logprobs64(h.detach().bfloat16(), w.detach().bfloat16(), t, g, gh)
    assert ((out.logprobs.double() - ref["logprobs"]).abs() <= ref["tol_lp"]).all()
    for x, name in zip(torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh]),
                       ("dh", "dw")):
        assert x.dtype == F32
        assert ((x.double() - ref[name]).abs() <= ref["tol_" + name]).all()


@pytest.mark.parametrize("m, dtype, k", [(4, BF16, 5), (300, BF16, 5), (300, BF16, 0), (3, F32, 2),
                                         (300, F32, 2)])
def test_logprobs_graph_stream_and_repeats(cuda, m, dtype, k):
    note(f"logprobs graph {m} {dtype} {k}")
    h, w, t, g, gh = _head(m, 128, 2003, dtype, cuda)

    def make():
        a, b = (x.detach().clone().requires_grad_(True) for x in (h, w))

        def step():
            out = chunked_token_logprobs(a, b, t, top_k=k)
            return [x.detach() for x in out if x is not None] + list(
                torch.autograd.grad([out.logprobs, out.entropy], [a, b], [g, gh]))

        return step

    assert_graph_replays_match(make)
    want = make()()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = make()()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_logprobs_make_no_host_sync(cuda):
    h, w, t, g, gh = _head(300, 64, 900, BF16, cuda)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        out = chunked_token_logprobs(h, w, t, top_k=3)
        torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh])
    finally:
        torch.cuda.set_sync_debug_mode("default")


# ---------------------------------------------------------------------------
# the C++ host side against the Functions in Python
# ---------------------------------------------------------------------------
class _NoNative:
    """Every entry answers None: the call takes its Function in Python."""

    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.parametrize("grad", [True, False])
def test_plain_calls_match_the_functions(cuda, monkeypatch, grad):
    note(f"native token ops grad={grad}")
    h, w, t, g, gh = _head(70, 64, 900, BF16, cuda)
    ids = torch.randint(0, 900, (5, 14), generator=gen(1)).to(cuda)
    table, x = randn((900, 64), gen(2), F32, cuda), randn((70, 64), gen(3), BF16, cuda)
    r, seed = randn((70, 64), gen(4), F32, cuda), torch.tensor([5], device=cuda)

    def calls():
        a, b, c, y, z = (v.detach().clone().requires_grad_(grad) for v in (h, w, table, x, r))
        lp = chunked_token_logprobs(a, b, t, top_k=4)
        emb = embedding_lookup(ids, c, scale=3.0, padding_idx=2, out_dtype=BF16)
        out = fused_dropout(y, 0.3, seed, offset=2, residual=z)
        one = fused_dropout(y, 0.3, 5, offset=2)
        res = [*lp, emb, out, one]
        assert [v.requires_grad for v in res] == [grad, grad, False, False, grad, grad, grad]
        if grad:
            res += torch.autograd.grad([lp.logprobs, lp.entropy, emb, out], [a, b, c, y, z],
                                       [g, gh, torch.ones_like(emb), torch.ones_like(out)])
            res += torch.autograd.grad(one, y, torch.ones_like(one))
        return res

    native = calls()
    from nuvla_forge_amd import _lib

    with monkeypatch.context() as mp:
        mp.setattr(_lib, "native", _NoNative)
        general = calls()
    for p, q in zip(native, general, strict=True):
        assert p.dtype == q.dtype and torch.equal(p, q)


def test_calls_that_are_not_plain_raise_as_documented(cuda):
    note("token ops refusals on the device")
    h, w, t, *_ = _head(10, 64, 900, BF16, cuda)
    with pytest.raises(ValueError, match="top_k"):
        chunked_token_logprobs(h, w, t, top_k=33)
    with pytest.raises(ValueError, match="on cpu"):
        chunked_token_logprobs(h, w, t.cpu())
    with pytest.raises(ValueError, match="padding_idx"):
        embedding_lookup(t, w, padding_idx=900)
    with pytest.raises(TypeError, match="table in"):
        embedding_lookup(t, w, out_dtype=F32)
    with pytest.raises(ValueError, match="shape mismatch"):
        fused_dropout(h, 0.1, 0, residual=h[:5])
    with pytest.raises(TypeError, match="residual"):
        fused_dropout(h.float(), 0.1, 0, residual=h)
    with pytest.raises(ValueError, match="on cpu"):
        fused_dropout(h, 0.1, torch.tensor([1]))


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("b, t, d, v", [(2, 16, 64, 500), (4, 33, 96, 3001)])
def test_policy_gradient_step_of_a_tied_head(cuda, b, t, d, v):
    """Lookup, dropout, a SwiGLU MLP on a residual stream, and the log probabilities under the
    same table: the losses and every gradient of a policy-gradient step in fp32, against 64 bits
    (norm-wise within the framework's 1e-5)."""
    note(f"policy gradient step {b} {t} {d} {v}")
    g = gen(b * t)
    table = randn((v, d), g, F32, cuda, std=0.3).requires_grad_(True)
    wg, wu = (randn((2 * d, d), g, F32, cuda, std=0.1).requires_grad_(True) for _ in "12")
    wd = randn((d, 2 * d), g, F32, cuda, std=0.1).requires_grad_(True)
    ids = torch.randint(0, v, (b, t), generator=g).to(cuda)
    ids[:, t // 2:][ids[:, t // 2:] % 3 == 0] = 0  # padding
    nxt = torch.where(ids.roll(-1, 1) == 0, -100, ids.roll(-1, 1)).view(-1)
    adv = randn((b * t,), g, F32, cuda)
    seed = torch.tensor([77], device=cuda)
    n = (nxt >= 0).sum()

    def run(tb, g1, g2, g3, own):
        if own:
            x = embedding_lookup(ids, tb, scale=2.0, padding_idx=0).view(-1, d)
            x = fused_dropout(x, 0.1, seed, offset=0)
            y = fused_gate_up_swiglu(x, g1, g2) @ g3.t()
            x = fused_dropout(y, 0.1, seed, offset=1, residual=x)
            lp = chunked_token_logprobs(x, tb, nxt)
            return -(adv * lp.logprobs).sum() / n - 0.01 * lp.entropy.sum() / n
        def drop(x, offset):
            keep = dropout_keep(x.shape, dropout_threshold(0.1), 77, offset, "cpu").to(cuda)
            return x * keep * (65536 / (65536 - dropout_threshold(0.1)))
        rows = tb[ids] * 2.0
        x = drop(torch.where((ids == 0)[..., None], rows.detach(), rows).view(-1, d), 0)
        y = (torch.nn.functional.silu(x @ g1.t()) * (x @ g2.t())) @ g3.t()
        x = x + drop(y, 1)
        lp = (x @ tb.t()).log_softmax(1)
        live = nxt >= 0
        own_lp = lp.gather(1, nxt.clamp(min=0)[:, None])[:, 0]
        ent = -(lp.exp() * lp).sum(1)
        return (-(adv.double() * own_lp)[live].sum() - 0.01 * ent[live].sum()) / n

    leaves = [table, wg, wu, wd]
    loss = run(*leaves, True)
    grads = torch.autograd.grad(loss, leaves)
    wide = [x.detach().double().requires_grad_(True) for x in leaves]
    want = run(*wide, False)
    assert abs(loss.item() - want.item()) < 1e-5 * abs(want.item())
    for x, y in zip(grads, torch.autograd.grad(want, wide)):
        assert (x.double() - y).norm() < 1e-5 * y.norm()
