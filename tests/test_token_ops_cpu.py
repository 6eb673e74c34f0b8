"""Token log probabilities, embedding lookup and dropout without a GPU: the eager
formulations that host tensors take, the generator against its published values, the
gradient formulas against differences, the refusals of the Python entries and of the
C ABI.
"""

from __future__ import annotations

import math

import pytest
import torch

from nuvla_forge_amd import _lib
from nuvla_forge_amd.kernels import (
    chunked_token_logprobs,
    embedding_lookup,
    fused_dropout,
)
from nuvla_forge_amd.kernels.reference import _philox_words, dropout_keep
from nuvla_forge_amd.kernels.utils import DeviceMismatchError, first_order_only

from .token_ops_ref import logprobs64

NF_OK, NF_ERR_ARG, NF_ERR_DTYPE, NF_ERR_WORKSPACE = 0, -1, -2, -3
FAKE = 4096  # a non-null pointer value; every call below returns before using it


def _err() -> str:
    return _lib.lib().nf_last_error().decode()


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("counter, key, want", [
    # the known answers that the generator's authors publish (Random123, kat_vectors)
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(counter, key, want):
    def signed(lo, hi):  # 64 bits as int64 holds them
        x = lo | hi << 32
        return x - (1 << 64) if x >> 63 else x

    got = _philox_words(signed(*key), torch.tensor([signed(*counter[:2])]), signed(*counter[2:]))
    assert tuple(int(w) for w in got) == want


def test_dropout_eager_values_and_gradient():
    x = torch.arange(1.0, 41.0).view(5, 8).requires_grad_(True)
    r = torch.full((5, 8), 100.0)
    keep = dropout_keep((5, 8), 16384, 7, 3, "cpu")
    out = fused_dropout(x, 0.25, 7, offset=3, residual=r)
    assert torch.equal(out, torch.where(keep, x.detach() * (4 / 3), 0.0) + r)
    out.sum().backward()
    assert torch.equal(x.grad, keep.float() * (65536 / 49152))
    # the mask goes by the element's place, not by strides or by how the seed is given
    y = fused_dropout(x.detach().t().contiguous().t(), 0.25, torch.tensor([7]), offset=3)
    assert torch.equal(y, torch.where(keep, x.detach() * (4 / 3), 0.0))
    assert not torch.equal(keep, dropout_keep((5, 8), 16384, 7, 4, "cpu"))
    assert not torch.equal(keep, dropout_keep((5, 8), 16384, 8, 3, "cpu"))


def test_dropout_rate():
    """n Bernoulli draws: the kept share is within 6 standard deviations of 1 - p."""
    n = 1 << 20
    for p in (0.02, 0.5, 0.9):
        t = math.floor(p * 65536 + 0.5)
        kept = dropout_keep((n,), t, 12345, 0, "cpu").double().mean().item()
        q = 1 - t / 65536
        assert abs(kept - q) < 6 * math.sqrt(q * (1 - q) / n), (p, kept)


def test_dropout_refusals():
    x = torch.zeros(4, 4)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="p must be"):
            fused_dropout(x, p, 0)
    with pytest.raises(ValueError, match="offset"):
        fused_dropout(x, 0.1, 0, offset=-1)
    with pytest.raises(ValueError, match="seed"):
        fused_dropout(x, 0.1, 1 << 63)
    with pytest.raises(ValueError, match="seed"):
        fused_dropout(x, 0.1, torch.tensor([1, 2]))
    with pytest.raises(ValueError, match="seed"):
        fused_dropout(x, 0.1, torch.tensor([1.0]))
    with pytest.raises(ValueError, match="shape mismatch"):
        fused_dropout(x, 0.1, 0, residual=torch.zeros(4))
    with pytest.raises(TypeError, match="residual"):
        fused_dropout(x, 0.1, 0, residual=torch.zeros(4, 4, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="unsupported dtype"):
        fused_dropout(x.double(), 0.1, 0)
    with pytest.raises(DeviceMismatchError):
        fused_dropout(x, 0.1, 0, residual=torch.zeros(4, 4, device="meta"))


def test_dropout_c_abi_refusals():
    f = _lib.lib().nf_dropout
    ok = [FAKE, None, FAKE, 64, 100, None, 1, 0, 1, 1, None]
    for i, bad, rc in ((3, -1, NF_ERR_ARG), (4, -1, NF_ERR_ARG), (4, 65537, NF_ERR_ARG),
                       (7, -1, NF_ERR_ARG), (0, None, NF_ERR_ARG), (2, None, NF_ERR_ARG),
                       (8, 3, NF_ERR_DTYPE), (9, 2, NF_ERR_DTYPE), (9, -1, NF_ERR_DTYPE),
                       (3, 1 << 50, NF_ERR_ARG)):
        assert f(*(ok[:i] + [bad] + ok[i + 1:])) == rc, (i, bad, _err())
    assert f(None, None, None, 0, 100, None, 1, 0, 1, 1, None) == NF_OK  # empty: no launch


# ---------------------------------------------------------------------------
# embedding lookup
# ---------------------------------------------------------------------------
def test_embedding_eager_values_and_gradient():
    table = torch.randn(6, 3, generator=torch.Generator().manual_seed(0)).requires_grad_(True)
    ids = torch.tensor([[1, 5, 1], [0, -2, 6]], dtype=torch.int32)
    out = embedding_lookup(ids, table, scale=2.0, padding_idx=0)
    want = torch.stack([table[i] * 2 if 0 <= i < 6 else torch.zeros(3)
                        for i in ids.flatten().tolist()]).view(2, 3, 3)
    assert torch.equal(out, want.detach())
    dout = torch.arange(1.0, 19.0).view(2, 3, 3)
    out.backward(dout)
    grad = torch.zeros(6, 3)
    grad[1] = 2 * (dout[0, 0] + dout[0, 2])
    grad[5] = 2 * dout[0, 1]
    assert torch.equal(table.grad, grad)  # none from the padding id or outside the table
    assert embedding_lookup(ids, table, out_dtype=torch.bfloat16).dtype == torch.bfloat16
    assert embedding_lookup(ids[:0], table).shape == (0, 3, 3)


def test_embedding_refusals():
    table, ids = torch.zeros(6, 3), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="table"):
        embedding_lookup(ids, torch.zeros(6))
    with pytest.raises(ValueError, match="table"):
        embedding_lookup(ids, torch.zeros(0, 3))
    with pytest.raises(TypeError, match="ids"):
        embedding_lookup(ids.float(), table)
    with pytest.raises(ValueError, match="padding_idx"):
        embedding_lookup(ids, table, padding_idx=6)
    with pytest.raises(TypeError, match="table in"):
        embedding_lookup(ids, table.bfloat16(), out_dtype=torch.float32)
    with pytest.raises(TypeError, match="unsupported dtype"):
        embedding_lookup(ids, table.double())
    with pytest.raises(DeviceMismatchError):
        embedding_lookup(ids.to("meta"), table)


def test_embedding_c_abi_refusals():
    L = _lib.lib()
    ok = [FAKE, FAKE, 64, 1.0, 16, 64, 100, FAKE, 1, 1, None]
    for i, bad, rc in ((2, 63, NF_ERR_ARG), (4, -1, NF_ERR_ARG), (5, 0, NF_ERR_ARG),
                       (6, 0, NF_ERR_ARG), (0, None, NF_ERR_ARG), (1, None, NF_ERR_ARG),
                       (7, None, NF_ERR_ARG), (8, 2, NF_ERR_DTYPE), (9, 0, NF_ERR_DTYPE),
                       (4, 1 << 31, NF_ERR_ARG)):
        assert L.nf_embedding_fwd(*(ok[:i] + [bad] + ok[i + 1:])) == rc, (i, bad, _err())
    need = L.nf_embedding_bwd_workspace(16, 64, 100)
    assert need > 0 and L.nf_embedding_bwd_workspace(-1, 64, 100) == 0
    assert L.nf_embedding_bwd_workspace(16, 1 << 26, 100) == 0
    ok = [FAKE, FAKE, -1, 1.0, 16, 64, 100, FAKE, 1, 1, FAKE, need, None]
    for i, bad, rc in ((4, -1, NF_ERR_ARG), (5, 0, NF_ERR_ARG), (0, None, NF_ERR_ARG),
                       (1, None, NF_ERR_ARG), (7, None, NF_ERR_ARG), (9, 2, NF_ERR_DTYPE),
                       (8, 0, NF_ERR_DTYPE), (10, None, NF_ERR_WORKSPACE),
                       (10, FAKE + 8, NF_ERR_WORKSPACE), (11, need - 1, NF_ERR_WORKSPACE)):
        assert L.nf_embedding_bwd(*(ok[:i] + [bad] + ok[i + 1:])) == rc, (i, bad, _err())


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------
def _case(m=7, d=5, v=11, seed=0):
    g = torch.Generator().manual_seed(seed)
    h, w = torch.randn(m, d, generator=g), torch.randn(v, d, generator=g)
    t = torch.randint(0, v, (m,), generator=g)
    t[2], t[4], t[5] = -100, v, -1
    return h, w, t, torch.randn(m, generator=g), torch.randn(m, generator=g)


def test_logprobs_formula_against_differences():
    """The 64-bit gradient that the GPU tests hold the kernels to, against central
    differences of its own values: truncation ~ eps^2, rounding ~ 2^-53 / eps."""
    h, w, t, g, gh = (x.double() if x.is_floating_point() else x for x in _case())
    want = logprobs64(h, w, t, g, gh)
    eps = 1e-5
    for name, x in (("dh", h), ("dw", w)):
        num = torch.zeros_like(x)
        for i in range(x.numel()):
            val = []
            for step in (eps, -eps):
                y = x.clone()
                y.view(-1)[i] += step
                r = logprobs64(*((y, w) if name == "dh" else (h, y)), t, g, gh)
                val.append((r["logprobs"] * g + r["entropy"] * gh).sum())
            num.view(-1)[i] = (val[0] - val[1]) / (2 * eps)
        assert (num - want[name]).abs().max() < 1e-8, name


@pytest.mark.parametrize("chunk_size", [3, 1024])
def test_logprobs_eager(chunk_size):
    h, w, t, g, gh = _case()
    h.requires_grad_(True), w.requires_grad_(True)
    out = chunked_token_logprobs(h, w, t, top_k=4, chunk_size=chunk_size)
    want = logprobs64(h, w, t, g, gh, 4)
    dh, dw = torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh])
    for name, x in dict(logprobs=out.logprobs, entropy=out.entropy, dh=dh, dw=dw,
                        top_logprobs=out.top_logprobs).items():
        assert (x.double() - want[name]).abs().max() < 5e-6, name
    assert torch.equal(out.top_ids, want["top_ids"])
    assert not out.top_logprobs.requires_grad
    for row in (2, 4, 5):  # left out
        assert out.logprobs[row] == 0 and out.entropy[row] == 0
        assert (out.top_ids[row] == -1).all() and (dh[row] == 0).all()
    none = chunked_token_logprobs(h, w, t)
    assert none.top_logprobs is None and none.top_ids is None
    assert chunked_token_logprobs(h[:0], w, t[:0], top_k=2).top_ids.shape == (0, 2)


def test_logprobs_eager_rows_left_out_may_hold_anything():
    """NaN and infinities in rows that are left out, and an infinite weight beside them, reach no
    gradient."""
    h, w, t, g, gh = _case()
    clean = logprobs64(h, w, t, g, gh)
    h[2], h[4, 0], h[5, 1] = float("nan"), float("inf"), float("-inf")
    h.requires_grad_(True), w.requires_grad_(True)
    out = chunked_token_logprobs(h, w, t, top_k=2)
    dh, dw = torch.autograd.grad([out.logprobs, out.entropy], [h, w], [g, gh])
    assert (dh[[2, 4, 5]] == 0).all() and (out.entropy[[2, 4, 5]] == 0).all()
    assert (dh.double() - clean["dh"]).abs().max() < 5e-6
    assert (dw.double() - clean["dw"]).abs().max() < 5e-6
    w = w.detach().clone()
    w[3, 0] = float("-inf")
    h = h.detach().abs().nan_to_num(1.0, posinf=1.0)
    h[2, 0] = 0.0  # 0 * inf where it does not count
    (dw,) = torch.autograd.grad(
        sum(x.sum() for x in chunked_token_logprobs(h, w.requires_grad_(True), t)[:2]), w)
    # p of token 3 is 0: dz there is 1 where it is the row's own token, else 0
    assert torch.isfinite(dw).all() and torch.allclose(dw[3], h[t == 3].sum(0), rtol=1e-6)


def test_logprobs_eager_logits_of_minus_infinity_and_nan():
    """A token that an infinite weight rules out has no part in the entropy; alternatives go by
    the logits, which may differ where the log probabilities' fp32 values no longer do; a NaN is
    no alternative."""
    h, w, t, *_ = _case()
    h = h.abs() + 0.125
    t = torch.where(t == 3, 4, t)
    rest = torch.arange(11) != 3
    want = chunked_token_logprobs(h, w[rest], torch.where(t > 3, t - 1, t), top_k=3)
    w[3, 0] = float("-inf")
    out = chunked_token_logprobs(h, w, t, top_k=11)
    live = (t >= 0) & (t < 11)
    assert (out.logprobs[live] - want.logprobs[live]).abs().max() < 1e-5
    assert (out.entropy[live] - want.entropy[live]).abs().max() < 1e-5
    assert (out.top_ids[live, -1] == 3).all() and (out.top_logprobs[live, -1] < -1e30).all()
    tiny = torch.tensor([[1e-9], [3e-9], [2e-9], [3e-9]])
    out = chunked_token_logprobs(torch.ones(1, 1), tiny, torch.tensor([0]), top_k=4)
    assert out.top_ids.tolist() == [[1, 3, 2, 0]] and out.top_logprobs.unique().numel() == 1
    tiny[1] = float("nan")
    out = chunked_token_logprobs(torch.ones(1, 1), tiny, torch.tensor([0]), top_k=4)
    assert out.top_ids.tolist() == [[3, 2, 0, -1]] and out.top_logprobs.isnan().all()


def test_logprobs_refusals():
    h, w, t, *_ = _case()
    with pytest.raises(ValueError, match="expected"):
        chunked_token_logprobs(h[0], w, t)
    with pytest.raises(ValueError, match="expected"):
        chunked_token_logprobs(h, w[:, :4], t)
    with pytest.raises(ValueError, match="targets"):
        chunked_token_logprobs(h, w, t[:3])
    for k in (-1, 12, 33):
        with pytest.raises(ValueError, match="top_k"):
            chunked_token_logprobs(h, w, t, top_k=k)
    with pytest.raises(ValueError, match="chunk_size"):
        chunked_token_logprobs(h, w, t, chunk_size=0)
    with pytest.raises(ValueError, match="empty"):
        chunked_token_logprobs(h, w[:0], t)
    with pytest.raises(DeviceMismatchError):
        chunked_token_logprobs(h, w.to("meta"), t)


def test_logprobs_c_abi_refusals():
    L = _lib.lib()
    st, fw = (L.nf_token_logprobs_state_bytes(16, 64, 100, 1024, 1, 1),
              L.nf_token_logprobs_fwd_workspace(16, 64, 100, 1024, 5, 1))
    bw = L.nf_token_logprobs_bwd_workspace(16, 64, 100, 1024, 1)
    assert st > 0 and fw > 0 and bw > 0
    assert L.nf_token_logprobs_state_bytes(16, 64, 100, 1024, 1, 2) == 0
    assert L.nf_token_logprobs_fwd_workspace(16, 64, 100, 1024, 33, 1) == 0
    assert L.nf_token_logprobs_fwd_workspace(16, 64, 4, 1024, 5, 1) == 0
    assert L.nf_token_logprobs_bwd_workspace(16, 64, 100, 0, 1) == 0
    assert L.nf_token_logprobs_fwd_workspace(16, 1, (1 << 30) + 1, 1024, 0, 1) == 0
    ok = [FAKE, FAKE, FAKE, 16, 64, 100, -100, 1024, 5, 1, 1, FAKE, FAKE, FAKE, FAKE, FAKE, st,
          FAKE, fw, None]
    bad = [(3, 0, NF_ERR_ARG), (4, 0, NF_ERR_ARG), (5, 1 << 32, NF_ERR_ARG), (7, 0, NF_ERR_ARG),
           (8, -1, NF_ERR_ARG), (8, 33, NF_ERR_ARG), (10, 2, NF_ERR_DTYPE),
           (15, FAKE + 8, NF_ERR_WORKSPACE), (16, st - 1, NF_ERR_WORKSPACE),
           (17, None, NF_ERR_WORKSPACE), (18, fw - 1, NF_ERR_WORKSPACE)]
    bad += [(i, None, NF_ERR_ARG) for i in (0, 1, 2, 11, 12, 13, 14, 15)]
    for i, x, rc in bad:
        assert L.nf_token_logprobs_fwd(*(ok[:i] + [x] + ok[i + 1:])) == rc, (i, x, _err())
    ok = [FAKE, 16, 64, 100, 1024, 1, 1, FAKE, st, FAKE, None, FAKE, 1, FAKE, 1, FAKE, bw, None]
    bad = [(1, 0, NF_ERR_ARG), (4, 0, NF_ERR_ARG), (6, 2, NF_ERR_DTYPE), (0, None, NF_ERR_ARG),
           (7, None, NF_ERR_ARG), (8, st - 1, NF_ERR_WORKSPACE), (12, 3, NF_ERR_DTYPE),
           (14, -1, NF_ERR_DTYPE), (15, None, NF_ERR_WORKSPACE), (16, bw - 1, NF_ERR_WORKSPACE)]
    for i, x, rc in bad:
        assert L.nf_token_logprobs_bwd(*(ok[:i] + [x] + ok[i + 1:])) == rc, (i, x, _err())
    nothing = ok[:11] + [None, 1, None, 1] + ok[15:]
    assert L.nf_token_logprobs_bwd(*nothing) == NF_OK  # no gradient wanted: no launch


@pytest.mark.parametrize("m, d, v, chunk_rows", [(1024, 1024, 520, 8), (4096, 2048, 32000, 64),
                                                 (129, 1024, 100, 1024), (256, 1024, 300, 1)])
def test_logprobs_workspace_holds_what_a_kept_forward_writes(m, d, v, chunk_rows):
    """Where the state holds 16 bits of every logit, the forward takes every row at once: whole
    blocks of 256 rows by 256 columns with an 8-byte record per 32 columns, and 4 bytes a row."""
    L = _lib.lib()
    mcap, tiles = -(-m // 256) * 256, -(-v // 256)
    assert L.nf_token_logprobs_state_bytes(m, d, v, chunk_rows, 1, 1) >= 2 * mcap * v
    assert (L.nf_token_logprobs_fwd_workspace(m, d, v, chunk_rows, 5, 1)
            >= mcap * tiles * 8 * 8 + mcap * 4)


# ---------------------------------------------------------------------------
# second derivatives
# ---------------------------------------------------------------------------
class _Cube(torch.autograd.Function):
    """x^3 by code that autograd does not see, as the kernels' gradients are."""

    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return x ** 3

    @staticmethod
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        dx = torch.from_numpy(3 * x.detach().numpy() ** 2 * g.detach().numpy())
        return first_order_only("cube", (g,), (dx,))[0]


@pytest.mark.parametrize("graph", [False, True])
def test_first_order_only(graph):
    """The gradient under create_graph has its value and may be used; a derivative through it
    raises, by the input and by the upstream gradient, beside other terms too."""
    x = torch.tensor([1.0, -2.0], requires_grad=True)
    g = torch.tensor([0.5, 4.0], requires_grad=True)
    y = x + 0  # not a leaf
    out = _Cube.apply(y) + x
    (dx,) = torch.autograd.grad(out, x, g, create_graph=graph)
    assert torch.equal(dx.detach(), g.detach() * (3 * x.detach() ** 2 + 1))
    assert dx.requires_grad == graph
    if graph:
        for leaf in (x, g, y):
            with pytest.raises(RuntimeError, match="cube: second derivatives"):
                torch.autograd.grad((dx + x * y).sum(), leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="cube: second derivatives"):
            (dx ** 2).sum().backward()
        (dx2,) = torch.autograd.grad(out.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="cube: second derivatives"):
            (dx2 * x).sum().backward()
        other = torch.ones(2, requires_grad=True)  # what does not go through it is free
        (d,) = torch.autograd.grad((dx.detach() * other).sum(), other)
        assert torch.equal(d, dx.detach())


def test_sizes_beyond_a_launch_are_refused():
    """A launch has at most 2^32 - 1 threads along an extent: calls that would need more are
    refused before any of their kernels, or take more launches."""
    L = _lib.lib()
    for n in ((1 << 35) + 1, 1 << 36):
        assert L.nf_dropout(FAKE, None, FAKE, n, 100, None, 1, 0, 1, 1, None) == NF_ERR_ARG
    for m, d in ((1 << 26, 512), (1 << 27, 200), (1 << 28, 128), (1 << 29, 64)):
        assert L.nf_embedding_fwd(FAKE, FAKE, d, 1.0, m, d, 9, FAKE, 1, 1, None) == NF_ERR_ARG
    for m, d, v in ((1 << 29, 8, 100), (100, 1, (1 << 30) + 1), ((1 << 31) - 1, 512, 1 << 30)):
        assert L.nf_embedding_bwd_workspace(m, d, v) == 0
        args = [FAKE, FAKE, -1, 1.0, m, d, v, FAKE, 1, 1, FAKE, 1 << 50, None]
        assert L.nf_embedding_bwd(*args) == NF_ERR_ARG
    assert L.nf_embedding_bwd_workspace(1 << 27, 64, 1 << 29) > 0
    # 16 bytes a row and 128 logits; a launch of 2^20 tokens by 2^18 rows, not 2^20
    assert 0 < L.nf_token_logprobs_fwd_workspace(1 << 20, 16, 1 << 20, 1 << 20, 0, 1) < 1 << 36
    assert L.nf_token_logprobs_fwd_workspace(1 << 10, 16, 1 << 30, 1 << 20, 0, 0) > 0
    # exponentials are kept for fewer than 2^24 rows
    few, many = ((1 << 24) - 256, 1 << 24)
    st = [L.nf_token_logprobs_state_bytes(m, 8, 64, 1 << 25, 1, 1) / m for m in (few, many)]
    assert st[0] >= 2 * 64 and st[1] < 64


def test_logprobs_backward_refuses_a_state_without_keep():
    """Without ``keep`` the forward of few rows copies none of them for a backward."""
    L = _lib.lib()
    for m in (16, 4096):
        st = L.nf_token_logprobs_state_bytes(m, 64, 100, 1024, 0, 1)
        bw = L.nf_token_logprobs_bwd_workspace(m, 64, 100, 1024, 1)
        assert L.nf_token_logprobs_bwd(FAKE, m, 64, 100, 1024, 0, 1, FAKE, st, FAKE, None, FAKE, 1,
                                       FAKE, 1, FAKE, bw, None) == NF_ERR_ARG
        assert "keep" in _err()


@pytest.mark.parametrize("m, d, v, kept", [(4096, 2048, 32000, True), (8, 2048, 128256, False),
                                           (200, 1024, 32000, True), (4096, 2048, 128256, True)])
def test_logprobs_backward_asks_for_no_transpose_that_it_does_not_make(m, d, v, kept):
    """Weight's transpose is in the state, or weight is read as it lies: the backward's workspace
    has no room for one, beside dz in bf16 (rows of whole lines of 64) and dh in fp32 where the
    rows are many."""
    L = _lib.lib()
    need = L.nf_token_logprobs_bwd_workspace(m, d, v, 1024, 1)
    many = 2 * (-(-m // 256) * 256) * (v + 64) + 4 * m * d if kept and m > 256 else 0
    assert need < many + 2 * d * v
