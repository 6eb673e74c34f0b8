"""64-bit restatements of attention and the rotary positions, and what results may be off by."""

from __future__ import annotations

import math

import torch

from .token_ops_ref import half_step, least_step

U32 = 2.0 ** -24


def attention64(q, k, v, dout=None, causal=False, key_mask=None, scale=None):
    """out, and dq, dk, dv for ``dout``, from the definition in 64 bits; and ``tol_*``, bounds on
    the error of each element of a result that is computed with fp32 sums, the probabilities and
    dS rounded once to the inputs' type, and rounded once at the end.

    With u the half step of the inputs' type (0 if fp32):
      a logit in powers of two: (d + 4) 2^-24 scale sum |q||k| log2(e), and its exponential's
      argument, a difference of two such with a maximum or a log-sum-exp: 2^-22 of 1 + its size;
      so P is off by ep of itself, with its sum over tk terms;
      out: P's roundings, the sum over tk terms, the last rounding;
      delta = sum dout out takes out's error before its last rounding (out and what the rounding
      left are both there), dP its sum over d terms; dS = P (dP - delta) and its rounding; the
      products their sums over tk or the group's tq rows."""
    b, tq, h, d = q.shape
    tk, hk = k.shape[1:3]
    g = h // hk
    u = 0.0 if q.dtype == torch.float32 else half_step(q.dtype)
    last, floor = half_step(q.dtype), least_step(q.dtype)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if key_mask is not None:
        k, v = (torch.where(key_mask[..., None, None], t, 0.0) for t in (k, v))

    def heads(x):  # [b, t, h, d] -> [b, h, t, d]
        return x.detach().double().transpose(1, 2).contiguous()

    def grouped(x):
        return heads(x).repeat_interleave(g, 1)

    q2, k2, v2 = heads(q), grouped(k), grouped(v)
    t = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    barred = torch.zeros(b, 1, tq, tk, dtype=torch.bool, device=q.device)
    if causal:
        barred = barred | torch.ones(tq, tk, dtype=torch.bool, device=q.device).triu(tk - tq + 1)
    if key_mask is not None:
        barred = barred | ~key_mask[:, None, None]
    z = torch.matmul(q2, t(k2)) * scale
    z = z.masked_fill(barred, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p, v2)
    # bounds
    size = torch.matmul(q2.abs(), t(k2.abs())) * abs(scale)
    size = torch.where(barred, 0.0, size).amax(-1, keepdim=True)  # the row's worst logit
    far = torch.where(p > 0, top - z, 0.0)
    ep = 2 * (d + 4) * U32 * size + 2.0 ** -21 * (1 + far + size) + (tk / 16 + 32) * U32
    # fp16 holds nothing below 2^-24 of what it is scaled to, at least 2^-17 down from the largest
    tiny = {torch.float16: 2.0 ** -30, torch.bfloat16: 2.0 ** -120,
            torch.float32: 2.0 ** -120}[q.dtype]
    live = (~barred).double()
    rough = p * (ep + u) + tiny * live
    mid = torch.matmul(rough, v2.abs()) + (tk / 8 + 32) * U32 * torch.matmul(p, v2.abs())
    tol = mid + last * (o.abs() + mid) + floor

    def flat(x):
        return x.transpose(1, 2)

    def summed(x):  # over a group's heads
        return flat(x.view(b, hk, g, tk, d).sum(2))

    res = {"out": flat(o), "tol_out": flat(tol),
           "largest": float(torch.where(barred, 0.0, z).abs().amax())}
    if dout is None:
        return res
    do = heads(dout)
    delta = (do * o).sum(-1, keepdim=True)
    dp = torch.matmul(do, t(v2))
    ds = p * (dp - delta)
    e_dp = (d + 4) * U32 * torch.matmul(do.abs(), t(v2.abs()))
    e_delta = (do.abs() * (mid + u * u * o.abs())).sum(-1, keepdim=True) + (d + 4) * U32 * (
        do.abs() * o.abs()).sum(-1, keepdim=True)
    e_ds = (ds.abs() * (ep + 2 * U32) + p * (e_dp + e_delta)) * (1 + u) + u * ds.abs()
    if q.dtype == torch.float16:  # dS in fp16: 2^-24 beside a largest of 2^10 at least
        e_ds = e_ds + 2.0 ** -34 * ds.abs().amax((-1, -2), keepdim=True) * live
    n = g * tq
    dq, dk, dv = torch.matmul(ds, k2) * scale, torch.matmul(t(ds), q2) * scale, torch.matmul(t(p), do)
    acc = lambda m: (m / 8 + 32) * U32  # noqa: E731
    e_dq = abs(scale) * (torch.matmul(e_ds, k2.abs()) + acc(tk) * torch.matmul(ds.abs(), k2.abs()))
    e_dk = abs(scale) * (torch.matmul(t(e_ds), q2.abs()) + acc(n) * torch.matmul(t(ds.abs()),
                                                                                   q2.abs()))
    e_dv = torch.matmul(t(rough), do.abs()) + acc(n) * torch.matmul(t(p), do.abs())
    for name, x, e, back in (("dq", dq, e_dq, flat), ("dk", dk, e_dk, summed),
                             ("dv", dv, e_dv, summed)):
        x, e = back(x), back(e)
        res[name], res["tol_" + name] = x, e + last * (x.abs() + e) + floor
    return res


def rotary64(x, positions, sections, base=10000.0, joint=False, interleaved=False, inverse=False):
    """x turned, by complex products in 64 bits, and the bound of each element: sine and cosine
    within 4 2^-24 each, three fp32 operations, one rounding."""
    pairs, freqs, axis = sum(sections), [], []
    for a, n in enumerate(sections):
        for i in range(n):
            freqs.append(math.pow(base, -(len(freqs) / pairs if joint else i / n)))
            axis.append(a)
    f = torch.tensor(freqs, dtype=torch.float64, device=x.device)
    pos = torch.stack([positions[..., a] for a in axis], -1).double()
    turn = torch.polar(torch.ones_like(pos), pos * f * (-1 if inverse else 1))[..., None, :]
    y = x.detach().double().clone()
    at = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved
          else (slice(0, pairs), slice(pairs, 2 * pairs)))
    w = torch.complex(y[..., at[0]].clone(), y[..., at[1]].clone()) * turn
    tol = torch.zeros_like(y)
    size = y[..., at[0]].abs() + y[..., at[1]].abs()
    y[..., at[0]], y[..., at[1]] = w.real, w.imag
    for s in at:
        tol[..., s] = 8 * U32 * size
    last = half_step(x.dtype)
    tol = tol + last * (y.abs() + tol) + least_step(x.dtype)
    tol[..., 2 * pairs:] = 0.0
    return y, tol


def within(got, want, tol, what):
    """Every element of ``got`` within ``tol`` of ``want``; the worst excess in the message."""
    err = (got.detach().double() - want).abs()
    over = err - tol
    bad = ~(over <= 0)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, the worst "
                           f"by {float(over[bad].max()):.3e}, at {bad.nonzero()[0].tolist()}")


def near(got, want, u, roundings, what, slack=1e-6):
    """The norm of the error within ``roundings`` half steps u (plus fp32's part) of the result's:
    independent roundings of relative size u of terms that do not cancel.  Among the type's
    subnormals an element's last rounding is off by up to least_step whatever its size."""
    err = float((got.detach().double() - want).norm())
    size = float(want.norm())
    floor = least_step(got.dtype) * math.sqrt(want.numel()) if got.dtype != torch.float64 else 0.0
    assert err <= (roundings * u + slack) * size + floor, f"{what}: {err / max(size, 1e-300):.3e}"
