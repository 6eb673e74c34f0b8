"""Token log probabilities, embedding lookup and dropout on the GPU where few calls go: large
logits, very peaked rows, second derivatives, operands that are not aligned, sizes at the borders
between kernels.  Against 64 bits, within bounds derived beside each.
"""

from __future__ import annotations

import math

import pytest
import torch

from nuvla_forge_amd import _lib
from nuvla_forge_amd.kernels import chunked_token_logprobs, embedding_lookup, fused_dropout
from nuvla_forge_amd.kernels.dropout import dropout_threshold
from nuvla_forge_amd.kernels.reference import dropout_keep

from .helpers import assert_graph_replays_match, gen, note, randn
from .test_gpu_token_ops import _embedding_check
from .token_ops_ref import logprobs64

pytestmark = pytest.mark.gpu
BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m", [3, 20, 100, 300])
def test_logprobs_do_not_depend_on_a_shift_of_the_logits(cuda, m, dtype):
    """960 added to every logit changes nothing: the values of sure tokens too, whose log
    probability is far below a step of the logits.

    h in 1/16 and w in 1/1024: every logit is exact (below 2^10 in steps of 2^-14), and so is its
    difference from the largest.  What is left is exp's, log's and their arguments' roundings,
    2^-21 of 1 + |x|, and those of a sum of V terms in 64 or more pieces, (V / 64 + 64) 2^-24."""
    note(f"logprobs shift {m} {dtype}")
    g, d, v, k = gen(m), 16, 3001, 8
    h, w = torch.randn(m, d, generator=g), torch.randn(v, d, generator=g) * 0.25
    t = torch.randint(0, v, (m,), generator=g)
    h[:, 0] = 0.0
    h[:, 1] = torch.where(torch.arange(m) % 3 == 0, 4.0, 0.0)  # a third of the rows: sure of one
    w[:, 1] = 0.0
    sure = torch.arange(v) % 997 == 5
    w[sure, 1] = 3.0 + 2.5 * torch.arange(int(sure.sum()))
    t[::3] = int(sure.nonzero()[-1])
    h, w = ((x * s).round().div(s).to(dtype).to(cuda) for x, s in ((h, 16), (w, 1024)))
    t, up = t.to(cuda), torch.randn(2, m, generator=g).to(cuda)
    ref = logprobs64(h, w, t, *up, k)  # without the shift
    h[:, 0], w[:, 0] = 32.0, 30.0
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    out = chunked_token_logprobs(h, w, t, top_k=k)
    tol = (v / 64 + 64) * 2.0 ** -24
    for x, y in ((out.logprobs, ref["logprobs"]), (out.top_logprobs, ref["top_logprobs"])):
        assert ((x.double() - y).abs() <= tol + 2.0 ** -21 * (1 + y.abs())).all()
    assert torch.equal(out.top_ids, ref["top_ids"])
    assert ((out.entropy.double() - ref["entropy"]).abs() <= ref["tol_ent"]).all()
    # the gradients but for the shift's own column are those without it
    for x, name in zip(torch.autograd.grad([out.logprobs, out.entropy], [h, w], list(up)),
                       ("dh", "dw")):
        off = (x.double() - ref[name]).abs()[:, 1:]
        assert (off <= ref["tol_" + name][:, 1:]).all(), (name, off.max())


@pytest.mark.parametrize("chunk_size", [1024, 1])
@pytest.mark.parametrize("far", [9.0, 13.0, 18.0, 24.0])
def test_logprobs_gradient_of_tokens_far_below_a_sure_one(cuda, far, chunk_size):
    """Every row is sure of one token, and the others are ``far`` nats below: those next to it
    (of its strip) have their gradient in weight like those far away, whether or not what the
    forward kept of the logits (exp(z - strip maximum) in 16 bits) is what the backward reads.

    Every row is alike (h, z), so dw[v] = h sum_m dz[m, v] with no cancellation between the p of
    different rows.  dz of a token is off by p's error, r = 2^-8 for its rounding to bf16, and
    for what was kept 2^-11 of itself or, more than 20 nats below the strip's largest, 2^-40 of that;
    p's by exp's argument, 2^-21 (1 + far), and by the sum's roundings, (V / 64 + 64) 2^-24."""
    note(f"logprobs far below {far} {chunk_size}")
    m, d, v, at = 300, 8, 4099, 1000
    h, w = torch.zeros(m, d), torch.zeros(v, d)
    h[:, 0] = 1.0
    w[at, 0] = far  # exact in bf16
    w[:, 1] = torch.arange(v) % 7 / 8.0  # h[:, 1] is 0: seen by dh alone
    h, w = (x.to(BF16).to(cuda).requires_grad_(True) for x in (h, w))
    t = torch.full((m,), at, device=cuda)
    g = torch.linspace(0.5, 1.5, m, device=cuda)
    out = chunked_token_logprobs(h, w, t, chunk_size=chunk_size)
    (dw,) = torch.autograd.grad(out.logprobs, w, g)
    z = w.detach().double()[:, 0]
    p = (z - torch.logsumexp(z, 0)).exp()
    want = -p * g.double().sum()
    want[at] += g.double().sum()
    size = p * g.double().sum()
    rel = 2.0 ** -8 + 2.0 ** -11 + 2 * ((v / 64 + 64) * 2.0 ** -24 + 2.0 ** -21 * (1 + far))
    tol = rel * size + 2.0 ** -40 * g.double().sum() + (m + 2) * 2.0 ** -24 * size
    tol += 2.0 ** -8 * (want.abs() + tol)  # dw's own rounding
    # the sure token's 1 - p, from its fp32 log probability: 2^-23 and the sum's roundings of 1
    tol[at] += 2 * (v / 64 + 66) * 2.0 ** -24 * g.double().sum()
    off = (dw.double()[:, 0] - want).abs()
    assert (off <= tol).all(), (off / tol).max()
    assert (dw[:, 1:] == 0).all()


def _head(m, d, v, dtype, dev, seed, ignored=0.2):
    """Inputs on which every logit is exact in fp32: h in 1/16, w in 1/1024."""
    g = gen(seed)
    h, w = torch.randn(m, d, generator=g), torch.randn(v, d, generator=g) * 2 / math.sqrt(d)
    h, w = (h * 16).round() / 16, (w * 1024).round() / 1024
    t = torch.randint(0, v, (m,), generator=g)
    t[torch.rand(m, generator=g) < ignored] = -100
    up = torch.randn(2, m, generator=g)
    return h.to(dtype).to(dev), w.to(dtype).to(dev), t.to(dev), up[0].to(dev), up[1].to(dev)


def _holds(h, w, t, g, gh, k, **kw):
    """Values, alternatives and gradients within the bounds of logprobs64."""
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    out = chunked_token_logprobs(h, w, t, top_k=k, **kw)
    ref = logprobs64(h, w, t, g, gh, k)
    got = dict(logprobs=out.logprobs, entropy=out.entropy)
    got["dh"], got["dw"] = torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh])
    for name, tol in (("logprobs", "lp"), ("entropy", "ent"), ("dh", "dh"), ("dw", "dw")):
        off = (got[name].double() - ref[name]).abs()
        assert (off <= ref["tol_" + tol]).all(), (name, (off / ref["tol_" + tol]).max())
    if k:
        assert torch.equal(out.top_ids, ref["top_ids"])
        off = (out.top_logprobs.double() - ref["top_logprobs"]).abs()
        assert (off <= ref["tol_lp"][:, None] + 2.0 ** -22 * ref["top_logprobs"].abs()).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m, d, v", [(5, 64, 1000), (70, 64, 33001), (100, 1024, 2003),
                                     (200, 1024, 2003), (300, 64, 2003), (1100, 1024, 1001)])
@pytest.mark.parametrize("off", [(1, 0), (0, 1), (3, 5)])
def test_logprobs_operands_that_begin_between_vectors(cuda, m, d, v, dtype, off):
    """Contiguous hidden and weight that do not begin on 16 bytes, as views into larger buffers:
    with the state kept and not, weight read as it lies or transposed for aligned ones."""
    note(f"logprobs misaligned {m} {d} {v} {dtype} {off}")
    h, w, t, g, gh = _head(m, d, v, dtype, cuda, m + d)

    def moved(x, by):
        flat = torch.empty(x.numel() + by, dtype=x.dtype, device=cuda)
        return flat[by:].view(x.shape).copy_(x)

    _holds(moved(h, off[0]), moved(w, off[1]), t, g, gh, 5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m", [65, 100, 128, 129, 256, 257])
def test_logprobs_of_middling_rows_over_a_large_vocabulary(cuda, m, dtype):
    """More than 32768 tokens and 65 rows: compacted, also where dz is held in two terms."""
    note(f"logprobs middling {m} {dtype}")
    for d, v, k in ((64, 33001, 8), (37, 40000, 20), (72, 32769, 0)):
        _holds(*_head(m, d, v, dtype, cuda, m + d, ignored=0.3), k)
    h, w, t, g, gh = _head(m, 64, 33001, dtype, cuda, m)
    _holds(h, w, torch.full_like(t, -100), g, gh, 3)  # none left


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m, d, v, chunk_rows", [(5, 72, 1003, 1024), (100, 64, 33001, 1024),
                                                 (200, 1024, 2003, 1024), (300, 64, 2003, 1),
                                                 (1000, 136, 5001, 1024), (700, 37, 999, 300)])
def test_logprobs_buffers_of_exactly_the_size_asked_for(cuda, m, d, v, chunk_rows, dtype):
    """The C entries with a state and workspaces of the bytes that the size calls name: what lies
    behind them stays as it was, and the results are those of the public call."""
    note(f"logprobs exact buffers {m} {d} {v} {chunk_rows} {dtype}")
    L, k = _lib.lib(), 4
    h, w, t, g, gh = _head(m, d, v, dtype, cuda, m)
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = chunked_token_logprobs(a, b, t, top_k=k, chunk_size=chunk_rows)
    want = [*out, *torch.autograd.grad([out.logprobs, out.entropy], [a, b], [g, gh])]
    code, st = _lib.dtype_code(h), _lib.stream_of(h)

    def room(n):
        assert n > 0
        x = torch.full((n + 4096,), 171, dtype=torch.uint8, device=cuda)
        return x, n

    state, fw, bw = (room(n) for n in (
        L.nf_token_logprobs_state_bytes(m, d, v, chunk_rows, 1, code),
        L.nf_token_logprobs_fwd_workspace(m, d, v, chunk_rows, k, code),
        L.nf_token_logprobs_bwd_workspace(m, d, v, chunk_rows, code)))
    lp, ent = torch.empty(m, device=cuda), torch.empty(m, device=cuda)
    top, ids = torch.empty(m, k, device=cuda), torch.empty(m, k, dtype=torch.int64, device=cuda)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    _lib.check(L.nf_token_logprobs_fwd(
        h.data_ptr(), w.data_ptr(), t.data_ptr(), m, d, v, -100, chunk_rows, k, 1, code,
        lp.data_ptr(), ent.data_ptr(), top.data_ptr(), ids.data_ptr(), state[0].data_ptr(),
        state[1], fw[0].data_ptr(), fw[1], st), "fwd")
    _lib.check(L.nf_token_logprobs_bwd(
        w.data_ptr(), m, d, v, chunk_rows, 1, code, state[0].data_ptr(), state[1],
        g.data_ptr(), gh.data_ptr(), dh.data_ptr(), code, dw.data_ptr(), code, bw[0].data_ptr(),
        bw[1], st), "bwd")
    for x, n in (state, fw, bw):
        assert (x[n:] == 171).all()
    assert all(torch.equal(x, y) for x, y in zip((lp, ent, top, ids, dh, dw), want))


class _NoNative:
    """No plain call is taken by the C++ host side: each runs its Function in Python."""

    def __init__(self, module):
        self.first_order_only = module.first_order_only

    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    """Both host sides of a call."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "native", lambda m=_lib.native(): _NoNative(m))
    return request.param


@pytest.mark.parametrize("m, dtype", [(5, BF16), (300, BF16), (40, F32)])
def test_logprobs_second_derivatives_raise(cuda, route, m, dtype):
    """Under create_graph the gradients are those without it; a derivative through them raises
    beside terms that have one, and by the upstream gradient."""
    note(f"logprobs second derivative {m} {dtype} {route}")
    g = gen(m)
    h, w = (randn(s, g, dtype, cuda).requires_grad_(True) for s in ((m, 16), (50, 16)))
    t = torch.randint(0, 50, (m,), generator=g).to(cuda)
    up = randn((m,), g, F32, cuda).requires_grad_(True)
    want = torch.autograd.grad(chunked_token_logprobs(h, w, t).logprobs, [h, w], up)
    got = torch.autograd.grad(chunked_token_logprobs(h, w, t).logprobs, [h, w], up,
                              create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for leaf in (h, w, up):
        with pytest.raises(RuntimeError, match="chunked_token_logprobs: second derivatives"):
            torch.autograd.grad((got[0].float() ** 2).sum() + (h * h).sum(), leaf,
                                retain_graph=True, allow_unused=True)
    loss = chunked_token_logprobs(h, w, t).entropy.sum()
    (dw,) = torch.autograd.grad(loss, w, create_graph=True)
    with pytest.raises(RuntimeError, match="chunked_token_logprobs: second derivatives"):
        (dw.float().sum() + (w * w).sum()).backward()


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("xt, rt", [(F32, None), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("by_tensor", [False, True])
def test_dropout_second_derivatives(cuda, route, xt, rt, by_tensor):
    """sum((r + drop(x))^3) with r = x (or without a residual): first, second and third
    derivatives by x.  With f the factor of an element (0 where dropped) and s = f + 1 (f without
    a residual), y = s x and the k-th derivative is s^k times that of y^3.

    A gradient passes through a handful of fp32 products and sums, each 2^-24 of the terms'
    absolute sum, and (bf16) roundings of the branch's value and of its gradient, 2^-8 each of its
    share."""
    note(f"dropout second derivative {xt} {rt} {by_tensor} {route}")
    g = gen(3)
    x = randn((33, 40), g, xt, cuda).float().requires_grad_(True)
    v = randn((33, 40), g, F32, cuda)
    seed = torch.tensor([21], device=cuda) if by_tensor else 21
    y = fused_dropout(x.to(xt), 0.25, seed, offset=4, residual=None if rt is None else x)
    t = dropout_threshold(0.25)
    f = dropout_keep(x.shape, t, 21, 4, "cpu").to(cuda).double() * (65536 / (65536 - t))
    s = f if rt is None else f + 1
    xd, vd, step = x.detach().double(), v.double(), 2.0 ** -7 if xt == BF16 else 2.0 ** -20
    (d1,) = torch.autograd.grad((y.float() ** 3).sum(), x, create_graph=True)
    (d2,) = torch.autograd.grad((d1 * v).sum(), x, create_graph=True)
    (d3,) = torch.autograd.grad((d2 * v).sum(), x)
    for got, want in ((d1, 3 * s ** 3 * xd ** 2), (d2, 6 * s ** 3 * xd * vd),
                      (d3, 6 * s ** 3 * vd ** 2)):
        assert ((got.double() - want).abs() <= 4 * step * want.abs() + 1e-30).all()
    # the gradient of what was a gradient: dout's own
    up = randn((33, 40), g, y.dtype, cuda).requires_grad_(True)
    y = fused_dropout(x.to(xt), 0.25, seed, offset=4, residual=None if rt is None else x)
    (dx,) = torch.autograd.grad(y, x, up, create_graph=True)
    (du,) = torch.autograd.grad(dx, up, v)
    assert du.dtype == up.dtype
    assert ((du.double() - s * vd).abs() <= 4 * step * (s * vd).abs()).all()


# ---------------------------------------------------------------------------
# embedding lookup
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("m, pad", [(60, None), (60, 3), (1500, 3)])
@pytest.mark.parametrize("dtype, od", [(F32, None), (F32, BF16), (BF16, None)])
def test_embedding_second_derivatives(cuda, route, m, pad, dtype, od):
    """sum(c out^3) of the lookup, and an upstream gradient's own gradient, against the dense
    formulas in 64 bits.  The derivatives by table row v hold sums of n terms each:
    (n + 8) 2^-24 of their absolute sum, and where rows or gradients are bf16 four roundings of
    2^-8 of it."""
    note(f"embedding second derivative {m} {pad} {dtype} {od} {route}")
    g, v, d, scale = gen(m), 40, 24, 2.0
    table = randn((v, d), g, dtype, cuda).requires_grad_(True)
    ids = torch.randint(-2, v + 2, (m,), generator=g).to(cuda)
    c, vt = randn((m, d), g, F32, cuda), randn((v, d), g, dtype, cuda)
    live = (ids >= 0) & (ids < v)
    hot = torch.nn.functional.one_hot(torch.where(live, ids, 0), v).double() * live[:, None]
    back = hot if pad is None else hot * (ids != pad)[:, None]  # what carries a gradient
    out = embedding_lookup(ids, table, scale=scale, padding_idx=pad, out_dtype=od)
    (d1,) = torch.autograd.grad((c * out.float() ** 3).sum(), table, create_graph=True)
    (d2,) = torch.autograd.grad((d1.float() * vt).sum(), table, create_graph=True)
    (d3,) = torch.autograd.grad((d2.float() * vt).sum(), table)
    e, cd, u = hot @ table.detach().double() * scale, c.double(), back @ vt.double() * scale
    step = (m + 8) * 2.0 ** -24 + (2.0 ** -6 if BF16 in (dtype, od) else 0)
    for got, term in ((d1, 3 * cd * e ** 2), (d2, 6 * cd * e * u), (d3, 6 * cd * u * u)):
        want, size = back.T @ term * scale, back.T @ term.abs() * scale
        assert got.dtype == dtype
        assert ((got.double() - want).abs() <= step * size).all()
    up = randn((m, d), g, out.dtype, cuda).requires_grad_(True)
    out = embedding_lookup(ids, table, scale=scale, padding_idx=pad, out_dtype=od)
    (dt,) = torch.autograd.grad(out, table, up, create_graph=True)
    (du,) = torch.autograd.grad(dt, up, vt)
    assert du.dtype == up.dtype and torch.equal(du.double(), u.to(du.dtype).double())


# The gradient of more than 1024 tokens: the sort, the spans' sums and the join of runs that cross
# spans, of 8 sorted positions, or of 16 and 32 from 131072 and 262144 (token, 512 columns) pairs on.
@pytest.mark.parametrize("span, m, d", [(8, 1300, 8), (8, 1300, 7), (8, 1300, 1), (8, 1300, 1032),
                                        (16, 135001, 8), (16, 66001, 520), (32, 270001, 8),
                                        (32, 270003, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_gradient_runs_at_span_borders(cuda, span, m, d, dtype):
    """Runs that end one before, at and one past a border between spans, that take a span exactly,
    and that cross one and several; the tokens of ids below 256 are sorted by id, so the counts
    say where each run lies.  Many tokens of one id on top: more than a wavefront notes."""
    note(f"embedding spans {span} {m} {d} {dtype}")
    counts = [span - 1, 1, span, span + 1, span - 1, 2 * span, 1, 3 * span - 2, 1, span, 9 * span + 1,
              span - 1, 12 * span, 1, 1, span - 2, 70 * span + 3]
    counts = [c for i, c in enumerate(counts) if sum(counts[:i + 1]) < m]
    counts += [m - sum(counts)]
    ids = torch.repeat_interleave(torch.arange(len(counts)) * 3, torch.tensor(counts))
    ids = ids[torch.randperm(m, generator=gen(m))].to(cuda)
    _embedding_check(ids, randn((60, d), gen(d), dtype, cuda), scale=0.5)


@pytest.mark.parametrize("m", [1025, 3000, 20000])
@pytest.mark.parametrize("d", [5, 40, 520])
def test_embedding_gradient_of_many_tokens_that_do_not_count(cuda, m, d):
    note(f"embedding many ids {m} {d}")
    g = gen(m + d)
    table = randn((50, d), g, F32, cuda)
    ids = torch.randint(-20, 70, (m,), generator=g)
    ids[:4] = torch.tensor([1 << 40, -(1 << 40), (1 << 63) - 1, -(1 << 63)])
    _embedding_check(ids.to(cuda), table, pad=7)
    _embedding_check(torch.full((m,), 7, device=cuda), table, pad=7)  # nothing but padding
    _embedding_check(torch.full((m,), -1, device=cuda), table)
    _embedding_check(torch.full((m,), 49, device=cuda), table, pad=0)  # one id, the last
    ids = torch.full((m,), 7)
    ids[m // 2] = 8  # one token that counts
    _embedding_check(ids.to(cuda), table, pad=7)
    _embedding_check(ids.view(-1, 1).to(cuda).expand(m, 2)[:, 1], table.t().contiguous().t())


@pytest.mark.parametrize("v", [131072, 131073, 140001, 300000])
def test_embedding_gradient_over_a_large_vocabulary(cuda, v):
    """More ids than 256 blocks of 512 hold: several share the bits that name a block, the first
    and the last of the table among them."""
    note(f"embedding large vocabulary {v}")
    g = gen(v)
    for m in (3000, 700):
        ids = torch.randint(0, v, (m,), generator=g)
        ids[::3] = torch.randint(0, 40, (len(ids[::3]),), generator=g) * 512 + 3
        ids[:6] = torch.tensor([0, v - 1, v - 1, v, -1, 0])
        _embedding_check(ids.to(cuda), randn((v, 16), g, F32, cuda), pad=3)


def test_embedding_gradient_of_many_tokens_in_a_graph_and_in_threads(cuda):
    note("embedding many tokens: graph, streams, threads")
    from concurrent.futures import ThreadPoolExecutor

    def inputs(seed):
        g = gen(seed)
        ids = (torch.rand(5000, generator=g) ** 3 * 1000).long().to(cuda)
        return ids, randn((1000, 96), g, BF16, cuda), randn((5000, 96), g, BF16, cuda)

    def make(seed=1):
        ids, table, dout = inputs(seed)
        leaf = table.requires_grad_(True)

        def step():
            out = embedding_lookup(ids, leaf, scale=2.0, padding_idx=0)
            return [out.detach(), *torch.autograd.grad(out, leaf, dout)]

        return step

    assert_graph_replays_match(make)
    alone = [make(s)() for s in (1, 2)]
    steps = [make(s) for s in (1, 2)]
    torch.cuda.synchronize()

    def work(step):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            res = [step() for _ in range(8)]
        stream.synchronize()
        return res

    with ThreadPoolExecutor(2) as ex:
        for want, got in zip(alone, ex.map(work, steps)):
            for one in got:
                assert all(torch.equal(a, b) for a, b in zip(want, one, strict=True))


# ---------------------------------------------------------------------------
# what sees or replaces a call
# ---------------------------------------------------------------------------
def _calls(dev):
    """Each operator as a function of its differentiable inputs, and those."""
    g = gen(17)
    h, w, t, *_ = _head(140, 1024, 900, BF16, dev, 17)
    ids = torch.randint(0, 40, (50,), generator=g).to(dev)
    seed = torch.tensor([3], device=dev)
    x, r = randn((20, 24), g, BF16, dev), randn((20, 24), g, F32, dev)
    return {
        "logprobs": (lambda a, b: chunked_token_logprobs(a, b, t, top_k=3)[:2], [h, w]),
        "few": (lambda a, b: chunked_token_logprobs(a, b, t[:6], top_k=3)[:2], [h[:6], w]),
        "embedding": (lambda a: (embedding_lookup(ids, a, padding_idx=1, out_dtype=BF16),),
                      [randn((40, 24), g, F32, dev)]),
        "dropout": (lambda a, b: (fused_dropout(a, 0.3, seed, offset=1, residual=b),), [x, r]),
    }


def _run(op, args):
    leaves = [v.detach().clone().requires_grad_(True) for v in args]
    outs = op(*leaves)
    ups = [torch.linspace(-1, 1, o.numel(), device=o.device).view(o.shape).to(o.dtype) for o in outs]
    return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, ups)]


@pytest.mark.parametrize("name", ["logprobs", "few", "embedding", "dropout"])
def test_token_ops_saved_tensors_go_through_the_hooks(cuda, route, name):
    note(f"token ops saved-tensor hooks {name} {route}")
    op, args = _calls(cuda)[name]
    plain, packed = _run(op, args), []

    def pack(v):
        packed.append(v.shape)
        return v.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v.to(cuda)):
        hooked = _run(op, args)
    assert len(packed) == (2 if name in ("logprobs", "few") else 1)
    assert all(torch.equal(a, b) for a, b in zip(plain, hooked, strict=True))


@pytest.mark.parametrize("name", ["logprobs", "few", "embedding", "dropout"])
def test_token_ops_under_modes_tracing_and_transforms(cuda, name):
    """Dispatch and function modes see the general path, which gives the same; a trace runs it;
    transforms that the Functions have no rule for are refused."""
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    note(f"token ops modes {name}")
    op, args = _calls(cuda)[name]
    plain, seen = _run(op, args), []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, a=(), kw=None):
            seen.append(str(func))
            return func(*a, **(kw or {}))

    class Functions(TorchFunctionMode):
        def __torch_function__(self, func, types, a=(), kw=None):
            return func(*a, **(kw or {}))

    for mode in (Dispatch, Functions):
        with mode():
            got = _run(op, args)
        assert all(torch.equal(a, b) for a, b in zip(plain, got, strict=True))
    assert any("empty" in f for f in seen)
    traced = torch.jit.trace(op, tuple(args), check_trace=False)
    # (what a call without a backward gives: it sums on other tiles)
    assert all(torch.equal(a, b) for a, b in zip(op(*args), traced(*args), strict=True))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda *v: op(*v)[0])(*(v[None] for v in args))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises(RuntimeError):
            op(dual, *args[1:])
