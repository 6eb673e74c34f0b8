"""What a transformer block does between its projections: rotary positions and attention.

Two operators, forward and (with ``train``) backward:

  attention  ``fused_attention`` on q [b, tq, h, d] and k, v [b, tk, hk, d]; the h / hk query heads
             of a group share a key head.  Row i may attend key j where the sample's ``key_mask``
             allows j and, if ``causal``, j <= i + tk - tq.  Over the allowed keys

                 S = scale q k^T     P = softmax(S)     out = P v     (no key allowed: 0)
                 dv = P^T dout       dS = P (dout v^T - rowsum(dout out))
                 dq = scale dS k     dk = scale dS^T q

             with dk and dv summed over a group's query heads.
  rotary     ``fused_rotary`` on q [b, t, h, d] and k [b, t, hk, d]: pair j of a head turns by the
             angle pos[token, axis(j)] * freq(j),

                 (x, y) -> (x cos - y sin, x sin + y cos)

             ``sections`` gives each axis (time, height, width) its number of pairs, in order.
             ladder "axis": freq = base^(-i / n) for the i-th of an axis's n pairs; "joint":
             base^(-j / P) for the j-th of all P pairs, so that equal coordinates turn as one
             position does.  Pair j is (x[j], x[P + j]), or (x[2 j], x[2 j + 1]) if interleaved;
             elements past 2 P stay.  The gradient turns back.

``own`` False: the plain forms, elementary torch operations in 32 bits (angles in 64).  True: the
operators.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    def attention(name, b, tq, tk, h, hk, d, dtype, causal, mask, train):
        return dict(name=name, op="attention", b=b, tq=tq, tk=tk, h=h, hk=hk, d=d, dtype=dtype,
                    causal=causal, mask=mask, train=train)

    def rotary(name, b, t, h, hk, d, axes, pairs, dtype, ladder, interleaved, far, train):
        return dict(name=name, op="rotary", b=b, t=t, h=h, hk=hk, d=d, axes=axes, pairs=pairs,
                    dtype=dtype, ladder=ladder, interleaved=interleaved, far=far, train=train)

    return [
        # one generated token for 8 requests: caches of 4096 places, each filled to its own length
        attention("attn_decode", 8, 1, 4096, 16, 4, 128, "bf16", False, "lengths", False),
        # the trajectory planner's 6 waypoints over the encoder's 1176 tokens, in training
        attention("attn_planner_cross", 8, 6, 1176, 6, 6, 64, "bf16", False, "none", True),
        # the encoder's own attention over its image tokens (8 x 1176 tokens of width 384)
        attention("attn_encoder", 8, 1176, 1176, 6, 6, 64, "bf16", False, "none", True),
        # the reasoning head's 8 x 64 text tokens, padded to the longest
        attention("attn_reasoning", 8, 64, 64, 6, 6, 64, "bf16", True, "lengths", True),
        # a 2048-wide language model's training step, 4 query heads on a key head
        attention("attn_lm_train", 2, 4096, 4096, 16, 4, 128, "bf16", True, "none", True),
        # the same model reading a long prompt
        attention("attn_prefill", 1, 16384, 16384, 16, 4, 128, "bf16", True, "none", False),
        # odd lengths, a head of 80, scattered masked keys, half precision
        attention("attn_odd_fp16", 3, 301, 1003, 6, 2, 80, "fp16", False, "scattered", True),
        # the reasoning head in full precision over longer texts
        attention("attn_fp32_train", 8, 512, 512, 6, 6, 64, "fp32", True, "none", True),
        # the positions of one generated token for 8 requests: latency
        rotary("rotary_decode", 8, 1, 16, 4, 128, 3, 64, "bf16", "joint", False, True, False),
        # the encoder's video tokens, a ladder for each of time, height and width
        rotary("rotary_encoder_train", 8, 1176, 6, 6, 64, 3, 32, "bf16", "axis", False, False,
               True),
        # a language model's long mixed sequences, beyond the caches
        rotary("rotary_lm_train", 16, 4096, 16, 4, 128, 3, 64, "bf16", "joint", False, True, True),
        # odd sizes in full precision: part of a head turned, neighbours paired
        rotary("rotary_odd_fp32", 3, 1361, 5, 1, 90, 2, 37, "fp32", "axis", True, False, True),
    ]


def _log_int(rng, lo, hi, step=1):
    x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(x / step)) * step))


def draw(rng):
    if rng.random() < 0.65:
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        hk, group = rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([1, 1, 2, 3, 4, 8])
        d = rng.choice([64, 128, 8 * rng.randint(2, 16), rng.randint(16, 128)])
        train = rng.random() < 0.6
        b = rng.choice([1, 1, 2, 3, 5, 8])
        # no dearer than the listed: the logits that the plain form holds, and fp32's products
        most = 5e8 if train else 4e9
        if dtype == "fp32":
            most = min(most, 3e10 / d)
        most /= b * hk * group
        shape = rng.choice(["self", "self", "cross", "decode"])
        # a gradient takes some keys to be more than rounding: over one key dq and dk are 0
        least = 16 if train else 1
        if shape == "decode":
            tq, tk = rng.choice([1, 1, 1, 2, 5]), _log_int(rng, 1, int(min(65536, most / 5)))
            train = False
        elif shape == "self":
            tq = tk = _log_int(rng, least, int(min(16384, math.sqrt(most))))
        else:
            tq = _log_int(rng, 1, int(min(8192, math.sqrt(most))))
            tk = _log_int(rng, least, int(min(16384, most / tq)))
        causal = rng.random() < 0.7 if shape != "cross" else tq <= tk and rng.random() < 0.3
        return dict(op="attention", b=b, tq=tq, tk=tk, h=hk * group, hk=hk, d=d, dtype=dtype,
                    causal=causal, mask=rng.choice(["none", "none", "lengths", "scattered"]),
                    train=train)
    hk, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
    d = rng.choice([64, 128, 2 * rng.randint(8, 64), rng.randint(16, 128)])
    most = 1.6e8 / (hk * (group + 1) * d)
    b = rng.choice([1, 2, 3, 8, 16])
    return dict(op="rotary", b=b, t=_log_int(rng, 1, int(max(2, min(16384, most / b)))),
                h=hk * group, hk=hk, d=d, axes=rng.choice([1, 2, 3, 3]),
                pairs=rng.choice([d // 2, d // 2, rng.randint(4, d // 2)]),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                ladder=rng.choice(["axis", "joint"]), interleaved=rng.random() < 0.4,
                far=rng.random() < 0.5, train=rng.random() < 0.7)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _attention_inputs(case, g):
    b, tq, tk, h, hk, d = (case[n] for n in ("b", "tq", "tk", "h", "hk", "d"))
    dt = TYPES[case["dtype"]]

    def randn(*s):
        return torch.randn(*s, device=DEVICE, generator=g)

    if tq == tk:  # one projection's output, its three parts used where they lie
        qkv = randn(b, tq, h + 2 * hk, d)
        qkv[:, :, :h] *= 1.7  # logits of deviation 1.7, as of a trained head
        q, k, v = qkv.to(dt).split([h, hk, hk], 2)
    else:
        q = (randn(b, tq, h, d) * 1.7).to(dt)
        k, v = randn(b, tk, 2 * hk, d).to(dt).split([hk, hk], 2)
    mask = None
    if case["mask"] == "lengths":  # padded batches, caches filled in part
        n = torch.randint((tk + 1) // 2, tk + 1, (b, 1), device=DEVICE, generator=g)
        mask = torch.arange(tk, device=DEVICE)[None] < n
    elif case["mask"] == "scattered":  # a tenth of the keys dropped
        mask = torch.rand(b, tk, device=DEVICE, generator=g) >= 0.1
    dout = randn(b, tq, h, d).to(dt) if case["train"] else None
    return dict(q=q, k=k, v=v, mask=mask, dout=dout, scale=1.0 / math.sqrt(d))


def _sections(case):
    n, p = case["axes"], case["pairs"]
    first = p // n if n < 3 else p // 4  # time takes fewer pairs than height and width
    rest = [(p - first) // (n - 1)] * (n - 1) if n > 1 else []
    return [p - sum(rest)] + rest


def _rotary_inputs(case, g):
    b, t, h, hk, d = (case[n] for n in ("b", "t", "h", "hk", "d"))
    dt = TYPES[case["dtype"]]
    qkv = torch.randn(b, t, h + 2 * hk, d, device=DEVICE, generator=g).to(dt)
    q, k, _ = qkv.split([h, hk, hk], 2)
    # frames of 14 x 12 patches, one after the other; a long conversation before them if ``far``
    i = torch.arange(t, device=DEVICE)
    pos = torch.stack([i // 168, i // 12 % 14, i % 12], 1)[:, :case["axes"]]
    if case["axes"] == 1:
        pos = i[:, None]
    start = torch.randint(0, 1_000_000 if case["far"] else 64, (b, 1, 1), device=DEVICE,
                          generator=g)
    grads = None
    if case["train"]:
        grads = [torch.randn(b, t, n, d, device=DEVICE, generator=g).to(dt) for n in (h, hk)]
    return dict(q=q, k=k, pos=pos + start, sections=_sections(case), base=10000.0, grads=grads)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    make = dict(attention=_attention_inputs, rotary=_rotary_inputs)[case["op"]]
    state = make(case, g)
    state["case"] = case
    for name in ("q", "k", "v"):  # the program's leaves
        if name in state:
            state[name] = state[name].detach().requires_grad_(case["train"])
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_attention(s, causal, train):
    q, k, v, mask = s["q"].detach(), s["k"].detach(), s["v"].detach(), s["mask"]
    b, tq, h, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    g = h // hk

    def rows(x):  # [b, tq, h, d] -> [b * hk, g * tq, d] in 32 bits
        return x.float().view(b, tq, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b * hk, g * tq, d)

    def heads(x):  # and back
        return x.view(b, hk, g, tq, d).permute(0, 3, 1, 2, 4).reshape(b, tq, h, d).to(q.dtype)

    def keys(x):  # [b, tk, hk, d] -> [b * hk, tk, d]
        return x.float().permute(0, 2, 1, 3).reshape(b * hk, tk, d).contiguous()

    def unkeys(x):
        return x.view(b, hk, tk, d).permute(0, 2, 1, 3).to(k.dtype).contiguous()

    q2, k2, v2 = rows(q), keys(k), keys(v)
    p = torch.matmul(q2, k2.transpose(1, 2).contiguous()).mul_(s["scale"])
    p5 = p.view(b, hk, g, tq, tk)
    if causal:
        i = torch.arange(tq, device=q.device)[:, None]
        p5.masked_fill_(torch.arange(tk, device=q.device)[None] > i + (tk - tq), -math.inf)
    if mask is not None:
        p5.masked_fill_(~mask[:, None, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0.0, 1.0, total))
    o = torch.matmul(p, v2)
    out = {"out": heads(o)}
    if train:
        do = rows(s["dout"])
        out["dv"] = unkeys(torch.matmul(p.transpose(1, 2).contiguous(), do))
        ds = torch.matmul(do, v2.transpose(1, 2).contiguous())
        ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
        out["dq"] = heads(torch.matmul(ds, k2))
        out["dk"] = unkeys(torch.matmul(ds.transpose(1, 2).contiguous(), q2))
    return out


def _ladder(case, s):
    """Each pair's axis and frequency, in 64 bits."""
    n = torch.tensor(s["sections"], device=s["pos"].device)
    j = torch.arange(case["pairs"], device=n.device)
    axis = (j[:, None] >= n.cumsum(0)[None]).sum(1)
    if case["ladder"] == "axis":
        x = (j - (n.cumsum(0) - n)[axis]).double() / n[axis]
    else:
        x = j.double() / case["pairs"]
    return axis, torch.exp(-math.log(s["base"]) * x)


def _plain_turn(x, cos, sin, pairs, interleaved):
    y = x.float()
    if interleaved:
        a, b = y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]
    else:
        a, b = y[..., :pairs], y[..., pairs:2 * pairs]
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, y[..., 2 * pairs:]), -1).to(x.dtype)


def _plain_rotary(s, case, train):
    axis, freq = _ladder(case, s)
    angle = (s["pos"][..., axis].double() * freq)[:, :, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    form = (case["pairs"], case["interleaved"])
    out = {"q": _plain_turn(s["q"].detach(), cos, sin, *form),
           "k": _plain_turn(s["k"].detach(), cos, sin, *form)}
    if train:
        out["dq"], out["dk"] = (_plain_turn(x, cos, -sin, *form) for x in s["grads"])
    return out


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def _own_attention(s, causal, train):
    from nuvla_forge_amd.kernels import fused_attention

    y = fused_attention(s["q"], s["k"], s["v"], causal=causal, key_mask=s["mask"],
                        scale=s["scale"])
    out = {"out": y}
    if train:
        out["dq"], out["dk"], out["dv"] = torch.autograd.grad(y, [s["q"], s["k"], s["v"]],
                                                              s["dout"])
    return out


def _own_rotary(s, case, train):
    from nuvla_forge_amd.kernels import fused_rotary

    q, k = fused_rotary(s["q"], s["k"], s["pos"], s["sections"], base=s["base"],
                        ladder=case["ladder"], interleaved=case["interleaved"])
    out = {"q": q, "k": k}
    if train:
        out["dq"], out["dk"] = torch.autograd.grad([q, k], [s["q"], s["k"]], s["grads"])
    return out


def run(state):
    case = state["case"]
    if case["op"] == "attention":
        call = _own_attention if own else _plain_attention
        return call(state, case["causal"], case["train"])
    return (_own_rotary if own else _plain_rotary)(state, case, case["train"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":
        n = case["b"] * case["t"] * (case["h"] + case["hk"]) * case["d"] * (1 + case["train"])
        share = 2.0 * case["pairs"] / case["d"]  # four products and two sums for each pair
        return {"bytes": 2 * n * e + case["b"] * case["t"] * case["axes"] * 8,
                "flops": 3.0 * n * share}
    b, tq, tk, h, hk, d = (case[n] for n in ("b", "tq", "tk", "h", "hk", "d"))
    share = {"none": 1.0, "lengths": 0.75, "scattered": 0.9}[case["mask"]]
    pairs = float(tq * tk)
    if case["causal"]:  # row i sees i + 1 + tk - tq keys, at least none
        first = max(0, tq - tk)
        seen = tq - first
        pairs = seen * (2.0 * tk - seen + 1) / 2
    pairs *= share * b * h
    nq, nk = b * tq * h * d, b * tk * hk * d
    nbytes = 2 * nq * e + 2 * nk * share * e
    flops = 4.0 * d * pairs
    if case["train"]:
        nbytes += 2 * nq * e + 2 * nk * e  # the gradients; q, k and v are read already
        flops += 10.0 * d * pairs  # with the logits, which are formed again
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _exact_attention(s, case):
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    b, tq, h, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    late = None
    if case["causal"]:
        late = torch.ones(tq, tk, dtype=torch.bool, device=q.device).triu(tk - tq + 1)
    out = {"out": torch.zeros_like(q)}
    if case["train"]:
        out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    for n in range(b):
        barred = torch.zeros(tq, tk, dtype=torch.bool, device=q.device) if late is None else late
        if s["mask"] is not None:
            barred = barred | ~s["mask"][n]
        empty = barred.all(1, keepdim=True)
        for i in range(h):  # a head at a time
            j = i * hk // h
            qi, kj, vj = (x.clone() for x in (q[n, :, i], k[n, :, j], v[n, :, j]))
            z = torch.mm(qi, kj.t()) * s["scale"]
            z = torch.softmax(z.masked_fill(barred & ~empty, -math.inf), dim=-1)
            z = z.masked_fill(empty, 0.0)
            o = torch.mm(z, vj)
            out["out"][n, :, i] = o
            if case["train"]:
                do = s["dout"][n, :, i].double()
                out["dv"][n, :, j] += torch.mm(z.t(), do)
                dz = torch.mm(do, vj.t())
                dz = z * (dz - (z * dz).sum(1, keepdim=True)) * s["scale"]
                out["dq"][n, :, i] = torch.mm(dz, kj)
                out["dk"][n, :, j] += torch.mm(dz.t(), qi)
    return out


def _exact_rotary(s, case):
    p, at, freqs, axes = case["pairs"], 0, [], []
    for a, n in enumerate(s["sections"]):
        for i in range(n):
            e = i / n if case["ladder"] == "axis" else (at + i) / p
            freqs.append(math.pow(s["base"], -e))
            axes.append(a)
        at += n
    f = torch.tensor(freqs, dtype=torch.float64, device=DEVICE)
    pos = torch.stack([s["pos"][..., a] for a in axes], -1).double()
    turn = torch.polar(torch.ones_like(pos), pos * f)[:, :, None]

    def by(x, z):
        y = x.detach().double().clone()
        at = ((slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if case["interleaved"]
              else (slice(0, p), slice(p, 2 * p)))
        w = torch.complex(y[..., at[0]].clone(), y[..., at[1]].clone()) * z
        y[..., at[0]], y[..., at[1]] = w.real, w.imag
        return y

    out = {"q": by(s["q"], turn), "k": by(s["k"], turn)}
    if case["train"]:
        out["dq"], out["dk"] = (by(x, turn.conj()) for x in s["grads"])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return (_exact_attention if case["op"] == "attention" else _exact_rotary)(state, case)
