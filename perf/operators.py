"""Performance cases of the encoder operators: what makes and trains the vectors that an index holds.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges. ``prepare`` makes what a
user's program has in hand before the call, ``run`` is one call (the plain form in 32-bit torch
operations, or with ``own`` the framework's operator), ``work`` the bytes and operations the call
cannot do without, ``exact`` the same outputs in 64 bits.

The kinds of call:
  embed           rows of a table by token, scaled; a token outside the table (-1: padding, an empty
                  search result) gives a row of zeros.
  embed_grad      the table's gradient: per row the sum over the tokens that named it.
  linear          y = act(x w^T + b) + residual.
  linear_grad     the gradients of x, w and b from y's gradient and the kept pre-activation.
  orthogonalize   Newton-Schulz steps on a weight's update: X <- a X + (b A + c A A) X, A = X X^T,
                  from X = G / |G|_F, on the side with fewer rows.
"""

from __future__ import annotations

import math

import torch

own = False

_DEVICE = "cuda"
_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
_STEPS, _COEFFICIENTS = 5, (3.4445, -4.7750, 2.0315)


# ---- the cases --------------------------------------------------------------------------------


def _embed(name, kind, dtype, rows, dim, tokens, index="int64", padding=0.0, scale=1.0):
    return dict(name=name, kind=kind, dtype=dtype, rows=rows, dim=dim, tokens=tokens, index=index, padding=padding,
                scale=scale)


def _linear(name, kind, dtype, m, k, n, act="none", bias=False, residual=False, keep=False):
    return dict(name=name, kind=kind, dtype=dtype, m=m, k=k, n=n, act=act, bias=bias, residual=residual, keep=keep)


def _ortho(name, dtype, batch, m, n):
    return dict(name=name, kind="orthogonalize", dtype=dtype, batch=batch, m=m, n=n)


def listed():
    return [
        # One short query's tokens, looked up while a user waits: launch and call latency.
        _embed("embed_query", "embed", "bf16", 32_000, 768, 24, scale=27.7),
        # A batch of padded texts over a word-vector table (the 1,183,514 x 100 collection).
        _embed("embed_words", "embed", "fp32", 1_183_514, 100, 250_007, padding=0.2),
        # A small table's gradient in a small step: sorting and launches count.
        _embed("embed_grad_small", "embed_grad", "fp32", 10_000, 128, 1_000, index="int32"),
        # Fine-tuning on long batches: every row hit, a few of them thousands of times.
        _embed("embed_grad_batch", "embed_grad", "bf16", 32_000, 1_024, 262_144, scale=32.0, padding=0.05),
        # One query through a wide layer: the weight is read once, nothing else matters.
        _linear("linear_query", "linear", "bf16", 1, 1_024, 4_096, "gelu", bias=True),
        # A ragged batch of word-vector width into a narrow layer.
        _linear("linear_ragged", "linear", "fp16", 1_003, 100, 384, "relu", bias=True, residual=True),
        # 10,000 text vectors through a square fp32 layer (the indexes take fp32), with a skip connection.
        _linear("linear_fp32", "linear", "fp32", 10_000, 768, 768, "silu", bias=True, residual=True),
        # A training batch through a wide layer, the pre-activation kept for the backward pass.
        _linear("linear_batch", "linear", "bf16", 16_384, 1_024, 4_096, "gelu", bias=True, keep=True),
        # The backward pass of that layer: long sums over the batch for the weight.
        _linear("linear_grad_batch", "linear_grad", "bf16", 16_384, 1_024, 4_096, "gelu", bias=True),
        # The backward pass of a projection in fp32, a modest batch.
        _linear("linear_grad_fp32", "linear_grad", "fp32", 2_000, 768, 128, "none", bias=True),
        # The update of a small rotation or head: launch latency.
        _ortho("ortho_small", "fp32", 1, 128, 128),
        # The update of the wide layer's weight.
        _ortho("ortho_wide", "bf16", 1, 4_096, 1_024),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "linear", "linear", "linear_grad", "orthogonalize"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if kind in ("embed", "embed_grad"):
        dim = _log_int(rng, 16, 1_024)
        rows = _log_int(rng, 1_000, min(1_183_514, 120_000_000 // dim))
        tokens = _log_int(rng, 1 if kind == "embed" else 64, 262_144)
        case = _embed("", kind, dtype, rows, dim, tokens, rng.choice(["int64", "int32"]), rng.choice([0.0, 0.0, 0.2]),
                      rng.choice([1.0, math.sqrt(dim)]))
    elif kind == "linear":
        # At most 7e10 operations a call (the largest listed one takes 1.4e11), a quarter in fp32.
        k, n = _log_int(rng, 16, 4_096), _log_int(rng, 16, 4_096)
        most = (1.75e10 if dtype == "fp32" else 7e10) / (2.0 * k * n)
        m = _log_int(rng, 1, max(2, min(16_384, int(most))))
        case = _linear("", kind, dtype, m, k, n, rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.7,
                       rng.random() < 0.4, rng.random() < 0.3)
    elif kind == "linear_grad":
        k, n = _log_int(rng, 16, 4_096), _log_int(rng, 16, 4_096)
        most = (2.5e10 if dtype == "fp32" else 1e11) / (4.0 * k * n)
        m = _log_int(rng, 16, max(32, min(16_384, int(most))))
        case = _linear("", kind, dtype, m, k, n, rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.7)
    else:
        m, n = _log_int(rng, 16, 1_024), _log_int(rng, 16, 2_048)
        batch = rng.choice([1, 1, 2, 6])
        if rng.random() < 0.3:
            m, n = n, m
        case = _ortho("", dtype, batch, m, n)
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE)
    g.manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=_DEVICE) * std).to(dt)

    state = dict(case=case)
    if case["kind"] in ("embed", "embed_grad"):
        rows, dim, n = case["rows"], case["dim"], case["tokens"]
        # Words come by rank, their frequency falling as 1 / rank; padding (-1) at random places.
        u = torch.rand(n, generator=g, device=_DEVICE, dtype=torch.float64)
        tok = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
        pad = torch.rand(n, generator=g, device=_DEVICE) < case["padding"]
        state["tokens"] = torch.where(pad, torch.full_like(tok, -1), tok).to(
            torch.int32 if case["index"] == "int32" else torch.int64)
        if case["kind"] == "embed":
            state["table"] = normal(rows, dim, std=0.05)
        else:
            state["grad"] = normal(n, dim, std=0.01)
        return state
    if case["kind"] == "orthogonalize":
        # Momentum of a weight's gradient: a few strong directions over a noise floor.
        b, m, n = case["batch"], case["m"], case["n"]
        r = max(1, min(m, n) // 8)
        left = torch.randn((b, m, r), generator=g, device=_DEVICE)
        right = torch.randn((b, r, n), generator=g, device=_DEVICE)
        noise = torch.randn((b, m, n), generator=g, device=_DEVICE)
        upd = (1e-3 * (left @ right / math.sqrt(r) + 0.5 * noise)).to(dt)
        state["update"] = upd if b > 1 else upd[0]
        return state
    m, k, n = case["m"], case["k"], case["n"]
    state["x"] = normal(m, k)
    state["weight"] = normal(n, k, std=1.0 / math.sqrt(k))
    bias = normal(n, std=0.1) if case["bias"] else None
    if case["kind"] == "linear":
        state["bias"] = bias
        state["residual"] = normal(m, n) if case["residual"] else None
    else:
        state["grad"] = normal(m, n, std=0.01)
        state["pre"] = None
        if case["act"] != "none":  # what the forward pass kept
            z = state["x"].float() @ state["weight"].float().T
            state["pre"] = (z if bias is None else z + bias.float()).to(dt)
    return state


# ---- one pass ---------------------------------------------------------------------------------


def _activate(z, act):
    if act == "relu":
        return z * (z > 0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain(state):
    case = state["case"]
    kind, dt = case["kind"], _TYPES[case["dtype"]]
    if kind == "embed":
        tok, table = state["tokens"], state["table"]
        named = (tok >= 0) & (tok < case["rows"])
        y = table[tok.clamp(0, case["rows"] - 1)].float() * case["scale"]
        return torch.where(named[:, None], y, torch.zeros_like(y)).to(dt)
    if kind == "embed_grad":
        tok = state["tokens"].long()
        named = (tok >= 0) & (tok < case["rows"])
        out = torch.zeros((case["rows"], case["dim"]), device=tok.device)
        out.index_add_(0, tok[named], state["grad"][named].float())
        return (out * case["scale"]).to(dt)
    if kind == "linear":
        z = state["x"].float() @ state["weight"].float().T
        if state["bias"] is not None:
            z = z + state["bias"].float()
        y = _activate(z, case["act"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return (y.to(dt), z.to(dt)) if case["keep"] else y.to(dt)
    if kind == "linear_grad":
        dz = state["grad"].float()
        if state["pre"] is not None:
            dz = dz * _slope(state["pre"].float(), case["act"])
        dx, dw = dz @ state["weight"].float(), dz.T @ state["x"].float()
        return (dx.to(dt), dw.to(dt), dz.sum(0).to(dt)) if case["bias"] else (dx.to(dt), dw.to(dt))
    x = state["update"].float()
    tall = case["m"] > case["n"]
    if tall:
        x = x.transpose(-1, -2).contiguous()
    norm = (x * x).sum((-2, -1), keepdim=True).sqrt()
    x = torch.where(norm > 0, x / norm, torch.zeros_like(x))
    a, b, c = _COEFFICIENTS
    for _ in range(_STEPS):
        s = x @ x.transpose(-1, -2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.transpose(-1, -2) if tall else x).to(dt).contiguous()


def run(state):
    if not own:
        return _plain(state)
    import quiver_amd as quiver

    case = state["case"]
    kind = case["kind"]
    if kind == "embed":
        return quiver.embed(state["table"], state["tokens"], scale=case["scale"])
    if kind == "embed_grad":
        return quiver.embed_grad(state["grad"], state["tokens"], case["rows"], scale=case["scale"])
    if kind == "linear":
        return quiver.linear(state["x"], state["weight"], bias=state["bias"], activation=case["act"],
                             residual=state["residual"], keep_preactivation=case["keep"])
    if kind == "linear_grad":
        dx, dw, db = quiver.linear_grad(state["grad"], state["x"], state["weight"], preactivation=state["pre"],
                                        activation=case["act"], bias=case["bias"])
        return (dx, dw, db) if case["bias"] else (dx, dw)
    return quiver.orthogonalize(state["update"], steps=_STEPS, coefficients=_COEFFICIENTS)


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    kind, e = case["kind"], float(_SIZE[case["dtype"]])
    if kind in ("embed", "embed_grad"):
        t, d = float(case["tokens"]), float(case["dim"])
        index = t * (4.0 if case["index"] == "int32" else 8.0)
        if kind == "embed":  # the rows named, each once, and every output row
            return {"bytes": index + e * d * (t + min(t, float(case["rows"]))), "flops": t * d}
        return {"bytes": index + e * d * (t + case["rows"]), "flops": t * d}
    if kind == "orthogonalize":
        # Two of the three products are symmetric: half of each is enough.
        lo, hi = float(min(case["m"], case["n"])), float(max(case["m"], case["n"]))
        return {"bytes": 2.0 * e * case["batch"] * lo * hi,
                "flops": case["batch"] * _STEPS * (3.0 * lo * lo * hi + lo * lo * lo)}
    m, k, n = float(case["m"]), float(case["k"]), float(case["n"])
    if kind == "linear":
        return {"bytes": e * (m * k + n * k + m * n * (1 + case["residual"] + case["keep"]) + n * case["bias"]),
                "flops": 2.0 * m * n * k}
    return {"bytes": e * (2.0 * (m * k + n * k) + m * n * (2 if case["act"] != "none" else 1) + n * case["bias"]),
            "flops": 4.0 * m * n * k}


# ---- 64-bit results ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.to(torch.float64) for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    kind = case["kind"]
    if kind in ("embed", "embed_grad"):
        tok = s["tokens"].to(torch.int64)
        ok = torch.logical_and(tok.ge(0), tok.lt(case["rows"]))
        if kind == "embed":
            y = torch.zeros((tok.numel(), case["dim"]), dtype=torch.float64, device=tok.device)
            y[ok] = d["table"].index_select(0, tok[ok]).mul(case["scale"])
            return y
        # Runs of equal tokens in sorted order, each a difference of running sums.
        order = torch.argsort(torch.where(ok, tok, torch.full_like(tok, case["rows"])), stable=True)
        count = torch.bincount(tok[ok], minlength=case["rows"])
        end = torch.cumsum(count, 0)
        out = torch.empty((case["rows"], case["dim"]), dtype=torch.float64, device=tok.device)
        for c in range(0, case["dim"], 64):
            run_sum = torch.cumsum(d["grad"][:, c:c + 64][order], 0)
            run_sum = torch.cat([torch.zeros_like(run_sum[:1]), run_sum])
            out[:, c:c + 64] = run_sum[end] - run_sum[end - count]
        return out.mul_(case["scale"])
    if kind == "linear":
        z = torch.mm(d["x"], d["weight"].t().contiguous())
        if "bias" in d:
            z += d["bias"]
        y = {"none": lambda t: t.clone(), "relu": lambda t: t.clamp(min=0),
             "gelu": lambda t: t * torch.special.ndtr(t), "silu": lambda t: t * torch.sigmoid(t)}[case["act"]](z)
        if "residual" in d:
            y += d["residual"]
        return (y, z) if case["keep"] else y
    if kind == "linear_grad":
        dz = d["grad"]
        if "pre" in d:
            z = d["pre"]
            sig = torch.sigmoid(z)
            dz = dz * {"relu": z.gt(0).to(torch.float64), "silu": sig + z * sig * (1 - sig),
                       "gelu": torch.special.ndtr(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)}[case["act"]]
        dx, dw = torch.mm(dz, d["weight"]), torch.mm(dz.t().contiguous(), d["x"])
        return (dx, dw, dz.sum(0)) if case["bias"] else (dx, dw)
    # The same odd polynomial of each singular value, step by step on the whole matrix.
    a, b, c = _COEFFICIENTS
    u = d["update"].reshape(case["batch"], case["m"], case["n"])
    tall = case["m"] > case["n"]
    u = u.transpose(1, 2).contiguous() if tall else u
    u = u / u.flatten(1).norm(dim=1).clamp_min(1e-300)[:, None, None]
    eye = torch.eye(u.shape[1], dtype=torch.float64, device=u.device)
    for _ in range(_STEPS):
        s = torch.bmm(u, u.transpose(1, 2).contiguous())
        u = torch.bmm(a * eye + b * s + c * torch.bmm(s, s), u)
    u = u.transpose(1, 2) if tall else u
    return (u if case["batch"] > 1 else u[0]).contiguous()
