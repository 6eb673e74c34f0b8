"""64-bit restatements of the token operators, and what their results may be off by."""

from __future__ import annotations

import torch


def half_step(t: torch.dtype) -> float:
    """The largest relative error of one rounding to ``t``."""
    return torch.finfo(t).eps / 2


def least_step(t: torch.dtype) -> float:
    """The largest absolute error of one rounding to ``t`` among its subnormals, where the spacing
    no longer falls with the value: it is tiny * eps there (2^-14 * 2^-10 in fp16, which has
    values that small among ordinary ones), half of it the error.  half_step alone holds from
    tiny = finfo.tiny on only."""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def logprobs64(h, w, t, g, gh, k=0, ignore=-100, chunk=2048):
    """Values and gradients of the token log probabilities, from the definition; and (``tol_*``)
    bounds on the error of results computed with fp32 sums and the gradients' one rounding of dz
    to the inputs' type and one at the end.

    A logit summed in fp32 in any order is off by at most (d + 2) 2^-24 sum |h||w| (with fp32
    inputs of three bf16 parts the part left out adds 2^-22 of it).  exp, log and their arguments
    add a few 2^-23 of 1 + |z - lse| each, and a sum of v positive terms in 64 or more pieces
    (v / 64 + 64) 2^-24."""
    f32 = w.dtype == torch.float32
    hd, wd = h.detach().double(), w.detach().double()
    (m, d), v = hd.shape, wd.shape[0]
    live = (t != ignore) & (t >= 0) & (t < v)
    out = {n: [] for n in ("logprobs", "entropy", "top_logprobs", "top_ids", "dh", "tol_lp",
                           "tol_ent", "tol_dh")}
    dw, tol_dw = torch.zeros_like(wd), torch.zeros_like(wd)
    r = half_step(h.dtype) if h.dtype != torch.float64 else 0.0
    for a in range(0, m, chunk):
        hs, lv = hd[a:a + chunk], live[a:a + chunk, None]
        z = hs @ wd.T
        lse = torch.logsumexp(z, 1, keepdim=True)
        x = z - lse
        p = x.exp()
        px = torch.where(p > 0, p * x, 0.0)
        ent = -px.sum(1, keepdim=True)
        col = torch.where(live[a:a + chunk], t[a:a + chunk], 0)[:, None]
        out["logprobs"].append(torch.where(lv, x.gather(1, col), 0.0)[:, 0])
        out["entropy"].append(torch.where(lv, ent, 0.0)[:, 0])
        if k:
            val, idx = torch.sort(x, dim=1, descending=True, stable=True)
            out["top_logprobs"].append(torch.where(lv, val[:, :k], 0.0))
            out["top_ids"].append(torch.where(lv, idx[:, :k], -1))
        gs, ghs = (torch.where(lv, u[a:a + chunk, None].double(), 0.0) for u in (g, gh))
        xs = torch.where(p > 0, x, 0.0)
        dz = -p * (gs + ghs * (xs + ent))
        dz.scatter_add_(1, col, gs)
        out["dh"].append(dz @ wd)
        dw += dz.T @ hs
        # bounds
        size = (hs.abs() @ wd.abs().T).amax(1, keepdim=True)  # sum |h||w| of the row's worst logit
        ez = ((d + 2) * 2.0 ** -24 + (2.0 ** -22 if f32 else 0)) * size
        far = 1 + px.abs().sum(1, keepdim=True) + lse.abs()
        es = (v / 64 + 64) * 2.0 ** -24 + 2.0 ** -21 * far
        out["tol_lp"].append((2 * ez + es + 2.0 ** -22 * x.gather(1, col).abs())[:, 0])
        out["tol_ent"].append(((ez + es) * (2 + 2 * far))[:, 0])
        # dz: relative error of p, and of the bracket
        ep = 2 * ez + es + 2.0 ** -21 * (1 + xs.abs())
        # and what is below 2^-126, fp32's and bf16's normal range, may become zero
        bracket = gs.abs() + ghs.abs() * (xs.abs() + ent.abs() + 1)
        edz = (p * ep * 2 + 2.0 ** -126) * bracket + r * dz.abs() + 2.0 ** -126
        if w.dtype == torch.bfloat16 and m > 128:
            # exp(z - strip maximum) may be kept in fp16: off by half a step, 2^-11 of itself,
            # or 2^-25 among its subnormals, of at most the row's largest p; p (z - lse) by that
            # times |z - lse| + 2
            edz += 2 * (2.0 ** -11 * p + 2.0 ** -25 * p.amax(1, keepdim=True)) * (
                bracket + ghs.abs())
        acc = (v + 2) * 2.0 ** -24 if f32 else (v / 16 + 16) * 2.0 ** -24
        out["tol_dh"].append(edz @ wd.abs() + acc * (dz.abs() @ wd.abs()))
        tol_dw += edz.T @ hs.abs() + (m + 2) * 2.0 ** -24 * (dz.abs().T @ hs.abs())
    res = {n: torch.cat(x) for n, x in out.items() if x}
    res["dw"] = dw
    if r:
        res["tol_dh"] = res["tol_dh"] + r * (res["dh"].abs() + res["tol_dh"])
        res["tol_dw"] = tol_dw + r * (dw.abs() + tol_dw)
    return res
