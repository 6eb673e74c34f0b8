"""The operators at the two ends of a language model and between its layers, as they are called.

Three operators, forward and (with ``train``) backward:

  logprobs   ``chunked_token_logprobs`` on hidden [m, d], lm_head [v, d] and one token a row:
             its log probability, the entropy of the row's distribution and the row's ``top_k``
             most probable tokens.  With z = hidden lm_head^T, lse = log sum exp z, p = exp(z - lse):

                 logprob = z[t] - lse            entropy = H = - sum p (z - lse)
                 dz      = g (onehot(t) - p) - gH p (z - lse + H)
                 dhidden = dz lm_head            dlm_head = dz^T hidden

             Rows whose token is ``IGNORE`` give 0 (alternatives: 0 and token -1) and no gradient.
  embedding  ``embedding_lookup``: out = scale * table[ids] and dtable[v] = scale * the sum of dout
             over the positions that hold v, none for the padding token.
  dropout    ``fused_dropout``: out = residual + keep * x / (1 - p), with keep recomputed in the
             backward.  Elements 8 b .. 8 b + 7 take the eight 16-bit parts of Philox4x32-10's
             block (b, offset) under the key ``seed``, lowest first; an element is kept where its
             part is at least T = round(65536 p), and 1 - p stands for (65536 - T) / 65536.

``dtype`` is ``bf16`` or ``fp32`` (every tensor), or ``amp``: for the embedding an fp32 table whose
rows leave in bf16, for the dropout a bf16 branch on an fp32 residual stream.

``own`` False: the plain forms, elementary torch operations in 32 bits.  True: the operators.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
IGNORE = -100


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    def logprobs(name, m, d, v, dtype, top_k, ignored, train):
        return dict(name=name, op="logprobs", m=m, d=d, v=v, dtype=dtype, top_k=top_k,
                    ignored=ignored, train=train)

    def embedding(name, m, d, v, dtype, padded, train):
        return dict(name=name, op="embedding", m=m, d=d, v=v, dtype=dtype, padded=padded,
                    train=train)

    def dropout(name, m, n, dtype, p, residual, train):
        return dict(name=name, op="dropout", m=m, n=n, dtype=dtype, p=p, residual=residual,
                    train=train)

    return [
        # one step of generating for 8 scenes: a row each, the alternatives reported
        logprobs("logprobs_decode", 8, 2048, 32000, "bf16", 8, 0.0, False),
        # policy-gradient training of the reasoning head: 8 x 64 text tokens, the prompt masked
        logprobs("logprobs_head_train", 512, 384, 32000, "bf16", 0, 1 / 7, True),
        # scoring rollouts of a 2048-wide language model with their alternatives
        logprobs("logprobs_score", 4096, 2048, 32000, "bf16", 8, 0.1, False),
        # the same model's policy-gradient step
        logprobs("logprobs_lm_train", 4096, 2048, 32000, "bf16", 0, 0.1, True),
        # a narrow head over many tokens, an odd vocabulary, many alternatives
        logprobs("logprobs_tall_odd", 12289, 384, 50001, "bf16", 20, 0.03, False),
        # the reasoning head trained in full precision
        logprobs("logprobs_fp32_train", 512, 384, 32000, "fp32", 0, 1 / 7, True),
        # the text tokens of one inference call: latency
        embedding("embedding_decode", 8, 384, 32000, "bf16", 0.0, False),
        # the reasoning head's 8 x 64 tokens in training, fp32 table, half of them padding
        embedding("embedding_head_train", 512, 384, 32000, "amp", 0.5, True),
        # a large language model's batch over a large vocabulary, beyond the caches
        embedding("embedding_lm_train", 65536, 2048, 128256, "bf16", 0.0, True),
        # dropout of the trajectory planner's branch: 8 x 6 waypoints of width 384
        dropout("dropout_planner", 48, 384, "amp", 0.1, True, True),
        # an odd width in full precision, no residual (dropout of the embedded tokens)
        dropout("dropout_odd_fp32", 4097, 1001, "fp32", 0.25, False, True),
        # a language model's branch over 65536 tokens, beyond the caches
        dropout("dropout_lm", 65536, 2048, "bf16", 0.1, True, True),
    ]


def _log_int(rng, lo, hi, step=1):
    x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(x / step)) * step))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "embedding", "dropout"])
    if op == "logprobs":
        train = rng.random() < 0.5
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        d = _log_int(rng, 256, 2048, 8)
        v = _log_int(rng, 1000, 128256)
        most = (1e11 if dtype == "fp32" else 1.4e12) / (6.0 * d * v)  # no dearer than the listed
        return dict(op=op, m=_log_int(rng, 1, int(max(2, min(16384, most)))), d=d, v=v,
                    dtype=dtype, top_k=rng.choice([0, 0, 1, 5, 8, 20]),
                    ignored=rng.choice([0.0, round(rng.uniform(0.0, 0.6), 3)]), train=train)
    if op == "embedding":
        d = _log_int(rng, 64, 2048)
        v = _log_int(rng, 1000, 128256)
        return dict(op=op, m=_log_int(rng, 1, 65536), d=d, v=v,
                    dtype=rng.choice(["bf16", "amp", "fp32"]) if d <= 1024 else "bf16",
                    padded=rng.choice([0.0, round(rng.uniform(0.0, 0.9), 3)]),
                    train=rng.random() < 0.75)
    n = _log_int(rng, 64, 4096)
    dtype = rng.choice(["bf16", "bf16", "amp", "fp32"])
    most = (1 << 27 if dtype == "bf16" else 1 << 26) // n
    return dict(op=op, m=_log_int(rng, 1, min(65536, most)), n=n, dtype=dtype,
                p=round(rng.uniform(0.02, 0.6), 3), residual=rng.random() < 0.7,
                train=rng.random() < 0.8)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _logprobs_inputs(case, g):
    m, d, v, dt = case["m"], case["d"], case["v"], _type(case)

    def randn(*s):
        return torch.randn(*s, device=DEVICE, generator=g)

    # logits of deviation ~2.3, as of a trained head, and the given tokens 0 to 8 above the rest:
    # a policy's own samples.  Where alternatives are asked for, the values lie on a grid (1/16 and
    # 1/1024) on which every logit is exact in 32 bits in whatever order it is summed: which token
    # comes first, and every tie between two, is then a fact of the inputs.
    std = 2.3 / math.sqrt(d)
    w = randn(v, d) * std
    t = torch.randint(0, v, (m,), device=DEVICE, generator=g)
    lift = torch.rand(m, 1, device=DEVICE, generator=g) * (8.0 / (d * std * std))
    if case["top_k"]:
        w = (w * 1024).round() / 1024
    w = w.to(dt)
    h = randn(m, d) + lift * w[t].float()
    if case["top_k"]:
        h = (h * 16).round() / 16
    drop = torch.rand(m, device=DEVICE, generator=g) < case["ignored"]
    t = torch.where(drop, IGNORE, t)
    # upstream: minus a normalised advantage, and an entropy bonus, over the tokens' count
    return dict(h=h.to(dt), w=w, t=t, g=randn(m) / m,
                gh=-0.01 * (1.0 + 0.1 * randn(m)) / m)


def _embedding_inputs(case, g):
    m, d, v = case["m"], case["d"], case["v"]
    # Zipf's law: token i with a probability of about 1 / (i ln v); token 0 is the padding
    u = torch.rand(m, device=DEVICE, generator=g, dtype=torch.float64)
    ids = torch.exp(u * math.log(v)).long().clamp_(1, v - 1)
    pad = torch.rand(m, device=DEVICE, generator=g) < case["padded"]
    ids = torch.where(pad, 0, ids)
    table = (torch.randn(v, d, device=DEVICE, generator=g) * 0.02).to(_type(case))
    out = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    dout = torch.randn(m, d, device=DEVICE, generator=g).to(out) if case["train"] else None
    return dict(ids=ids, table=table, dout=dout, out=out, scale=math.sqrt(d),
                pad=0 if case["padded"] else None)


def _dropout_inputs(case, g):
    m, n = case["m"], case["n"]
    branch = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    x = torch.randn(m, n, device=DEVICE, generator=g).to(branch)
    r = torch.randn(m, n, device=DEVICE, generator=g).to(_type(case)) if case["residual"] else None
    dout = (torch.randn(m, n, device=DEVICE, generator=g).to(x.dtype if r is None else r.dtype)
            if case["train"] else None)
    # the program's generator state: a seed on the device and the call's own number
    seed = torch.randint(0, 1 << 62, (1,), device=DEVICE, generator=g)
    return dict(x=x, r=r, dout=dout, seed=seed, offset=11, p=case["p"])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    make = dict(logprobs=_logprobs_inputs, embedding=_embedding_inputs, dropout=_dropout_inputs)
    state = make[case["op"]](case, g)
    state["case"] = case
    if case["train"]:  # the program's leaves
        for name in ("h", "w", "table", "x"):
            if name in state:
                state[name].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_logprobs(s, top_k, train):
    h, w, t = s["h"].detach().float(), s["w"].detach().float(), s["t"]
    v = w.shape[0]
    live = t != IGNORE
    col = torch.where(live, t, 0)[:, None]
    z = h @ w.T + 0.0  # no -0
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    ent = torch.log(total) - ((z - top) * e).sum(1, keepdim=True) / total
    out = {"logprobs": torch.where(live, (z.gather(1, col) - lse)[:, 0], 0.0),
           "entropy": torch.where(live, ent[:, 0], 0.0)}
    if top_k:
        # one whole-numbered key orders by value, then by the lower token
        bits = z.view(torch.int32).long()
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        key = (bits << 32) + (v - 1 - torch.arange(v, device=z.device))
        ids = v - 1 - (torch.topk(key, top_k).values & 0xFFFFFFFF)
        out["top_logprobs"] = torch.where(live[:, None], z.gather(1, ids) - lse, 0.0)
        out["top_ids"] = torch.where(live[:, None], ids, -1)
    if train:
        g, gh = (torch.where(live, s[k], 0.0)[:, None] for k in ("g", "gh"))
        dz = (e / total) * -(g + gh * (z - lse + ent))
        dz.scatter_add_(1, col, g)
        out["dh"] = (dz @ w).to(s["h"].dtype)
        out["dw"] = (dz.T @ h).to(s["w"].dtype)
    return out


def _plain_embedding(s, train):
    ids, table = s["ids"], s["table"].detach()
    out = {"out": (table[ids].float() * s["scale"]).to(s["out"])}
    if train:
        d = s["dout"].float() * s["scale"]
        if s["pad"] is not None:
            d = torch.where((ids != s["pad"])[:, None], d, 0.0)
        grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
        out["dtable"] = grad.index_add_(0, ids, d).to(table.dtype)
    return out


def _philox(seed, block, offset):
    """The four 32-bit words of Philox4x32-10's blocks, as int64."""
    low = 0xFFFFFFFF
    k0, k1 = seed & low, (seed >> 32) & low
    c0, c1 = block & low, (block >> 32) & low
    c2, c3 = torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)
    for r in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits, whose halves are wanted
        c0, c1, c2, c3 = (((b >> 32) & low) ^ c1 ^ ((k0 + r * 0x9E3779B9) & low), b & low,
                          ((a >> 32) & low) ^ c3 ^ ((k1 + r * 0xBB67AE85) & low), a & low)
    return c0, c1, c2, c3


def _plain_dropout(s, train):
    x, r = s["x"].detach(), s["r"]
    t = math.floor(s["p"] * 65536 + 0.5)
    n = x.numel()
    words = torch.stack(_philox(s["seed"], torch.arange((n + 7) // 8, device=x.device),
                                s["offset"]), 1)
    parts = torch.stack((words & 0xFFFF, words >> 16), 2)
    keep = (parts.reshape(-1)[:n] >= t).view(x.shape)
    f = 65536 / (65536 - t)
    y = torch.where(keep, x.float() * f, 0.0)
    out = {"out": (y if r is None else y + r.float()).to(x.dtype if r is None else r.dtype)}
    if train:
        out["dx"] = torch.where(keep, s["dout"].float() * f, 0.0).to(x.dtype)
    return out


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def _own_logprobs(s, top_k, train):
    from nuvla_forge_amd.kernels import chunked_token_logprobs

    r = chunked_token_logprobs(s["h"], s["w"], s["t"], top_k=top_k, ignore_index=IGNORE)
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if top_k:
        out["top_logprobs"], out["top_ids"] = r.top_logprobs, r.top_ids
    if train:
        out["dh"], out["dw"] = torch.autograd.grad([r.logprobs, r.entropy], [s["h"], s["w"]],
                                                   [s["g"], s["gh"]])
    return out


def _own_embedding(s, train):
    from nuvla_forge_amd.kernels import embedding_lookup

    y = embedding_lookup(s["ids"], s["table"], scale=s["scale"], padding_idx=s["pad"],
                         out_dtype=s["out"])
    out = {"out": y}
    if train:
        (out["dtable"],) = torch.autograd.grad(y, s["table"], s["dout"])
    return out


def _own_dropout(s, train):
    from nuvla_forge_amd.kernels import fused_dropout

    y = fused_dropout(s["x"], s["p"], s["seed"], offset=s["offset"], residual=s["r"])
    out = {"out": y}
    if train:
        (out["dx"],) = torch.autograd.grad(y, s["x"], s["dout"])
    return out


def run(state):
    case = state["case"]
    if case["op"] == "logprobs":
        call = _own_logprobs if own else _plain_logprobs
        return call(state, case["top_k"], case["train"])
    if case["op"] == "embedding":
        return (_own_embedding if own else _plain_embedding)(state, case["train"])
    return (_own_dropout if own else _plain_dropout)(state, case["train"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "logprobs":
        m, d, v, k = case["m"], case["d"], case["v"], case["top_k"]
        e = 2 if case["dtype"] == "bf16" else 4
        live = m * (1.0 - case["ignored"])
        nbytes = (m + v) * d * e + m * (8 + 8 + 12 * k)
        flops = 2.0 * live * v * d
        if case["train"]:
            nbytes += (m + v) * d * e + 8 * m
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "embedding":
        m, d, v = case["m"], case["d"], case["v"]
        et, eo = (2 if case["dtype"] == "bf16" else 4), (4 if case["dtype"] == "fp32" else 2)
        rows = v * (1.0 - math.exp(-m / v))  # about as many different rows as are read, at most
        nbytes = 8 * m + min(rows, m) * d * et + m * d * eo
        if case["train"]:
            nbytes += m * d * eo + v * d * et
        return {"bytes": nbytes, "flops": m * d * (2.0 if case["train"] else 1.0)}
    n = case["m"] * case["n"]
    ex = 4 if case["dtype"] == "fp32" else 2
    er = ex if case["dtype"] != "amp" or not case["residual"] else 4
    nbytes = n * (ex + er + (er if case["residual"] else 0))
    if case["train"]:
        nbytes += n * (er + ex)
    # ten rounds of two products, four exclusive ors and two sums for each eight elements
    return {"bytes": nbytes, "flops": n * (10 * 8 / 8 + 2) * (2 if case["train"] else 1)}


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _exact_logprobs(s, case):
    k, train = case["top_k"], case["train"]
    h, w, t = s["h"].detach().double(), s["w"].detach().double(), s["t"]
    m, v = t.numel(), w.shape[0]
    parts, dw = [], torch.zeros_like(w)
    for at in range(0, m, 1024):  # a thousand rows' logits at a time
        hs, ts = h[at:at + 1024], t[at:at + 1024]
        live = (ts != IGNORE).double()[:, None]
        z = torch.mm(hs, w.t())
        lp = torch.log_softmax(z, dim=-1)
        p = lp.exp()
        ent = -(p * lp).sum(-1, keepdim=True)
        one = torch.zeros_like(z)
        one[torch.arange(len(ts), device=z.device), ts.clamp(min=0)] = 1.0
        got = [((one * lp).sum(-1, keepdim=True) * live)[:, 0], (ent * live)[:, 0]]
        if k:
            val, idx = torch.sort(lp, dim=-1, descending=True, stable=True)
            got += [val[:, :k] * live, torch.where(live > 0, idx[:, :k], -1)]
        if train:
            g, gh = (s[n][at:at + 1024].double()[:, None] * live for n in ("g", "gh"))
            dz = g * (one - p) - gh * p * (lp + ent)
            got.append(torch.mm(dz, w))
            dw += torch.mm(dz.t(), hs)
        parts.append(got)
    names = ["logprobs", "entropy"] + (["top_logprobs", "top_ids"] if k else []) + (
        ["dh"] if train else [])
    out = {name: torch.cat([got[i] for got in parts]) for i, name in enumerate(names)}
    if train:
        out["dw"] = dw
    return out


def _exact_embedding(s, case):
    ids, table = s["ids"], s["table"].detach().double()
    out = {"out": torch.index_select(table, 0, ids) * s["scale"]}
    if case["train"]:
        counted = torch.ones_like(ids) if s["pad"] is None else (ids != s["pad"]).long()
        grad = torch.zeros_like(table)
        grad.index_put_((ids,), s["dout"].double() * counted[:, None], accumulate=True)
        out["dtable"] = grad * s["scale"]
    return out


def _exact_dropout(s, case):
    x = s["x"].detach()
    n, seed, offset = x.numel(), int(s["seed"].item()), s["offset"]
    block = torch.arange((n + 7) // 8, device=x.device)

    def times(c, k):  # (high, low) 32 bits of a product, by 16-bit parts
        lo, hi = c * (k & 0xFFFF), c * (k >> 16)
        hi = hi + (lo >> 16)
        return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)

    ctr = [block % (1 << 32), block // (1 << 32), torch.full_like(block, offset % (1 << 32)),
           torch.full_like(block, offset >> 32)]
    key = [seed % (1 << 32), seed >> 32]
    for _ in range(10):
        h0, l0 = times(ctr[0], 0xD2511F53)
        h1, l1 = times(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    t = int(math.floor(65536 * s["p"] + 0.5))
    bits = torch.empty(block.numel(), 8, dtype=torch.bool, device=x.device)
    for j in range(8):
        bits[:, j] = (ctr[j // 2] >> (16 * (j % 2))) % 65536 >= t
    keep = bits.view(-1)[:n].view(x.shape).double() * (65536.0 / (65536.0 - t))
    y = x.double() * keep
    out = {"out": y if s["r"] is None else s["r"].double() + y}
    if case["train"]:
        out["dx"] = s["dout"].double() * keep
    return out


def exact(case, seed):
    state = prepare(case, seed)
    call = dict(logprobs=_exact_logprobs, embedding=_exact_embedding, dropout=_exact_dropout)
    return call[case["op"]](state, case)
