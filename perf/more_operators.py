"""Performance cases of the operators that make a block of an encoder, and of training it.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges. ``prepare`` makes what a
user's program has in hand before the call, ``run`` is one call (the plain form in 32-bit torch
operations, or with ``own`` the framework's operator), ``work`` the bytes and operations the call
cannot do without, ``exact`` the same outputs in 64 bits.

The kinds of call:
  norm            the way from one block to the next: r = x + scale * act(gate) * norm(y) * post and
                  h = norm(r) * weight, norm(x) = x / sqrt(mean(x^2) + eps); or h of x alone.
  norm_grad       the gradients of x, y, gate and of the three vectors.
  attention       linear attention with a decay for each head: S_t = exp(g) S_{t-1} + k_t v_t^T,
                  o_t = scale S_t^T q_t. Whole texts, ragged ones behind padding, or one token with its state.
  attention_grad  the gradients of q, k, v (and of the first state).
  clip            the norm over all gradients of a model, and the gradients scaled down to a limit.
"""

from __future__ import annotations

import math

import torch

own = False

_DEVICE = "cuda"
_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
_EPS = 1e-6


# ---- the cases --------------------------------------------------------------------------------


def _norm(name, kind, dtype, rows, dim, block=True, gate="none", scale=True):
    """gate: none (no gate), plain, sigmoid or silu."""
    return dict(name=name, kind=kind, dtype=dtype, rows=rows, dim=dim, block=block, gate=gate, scale=scale)


def _attention(name, kind, dtype, batch, tokens, heads, kv_heads, dk, dv, state=False, ragged=False, packed=False):
    return dict(name=name, kind=kind, dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv,
                state=state, ragged=ragged, packed=packed)


def _clip(name, dtype, words, dim, layers, limit):
    return dict(name=name, kind="clip", dtype=dtype, words=words, dim=dim, layers=layers, limit=limit)


def listed():
    return [
        # One short query's tokens between two blocks, while a user waits: launch and call latency.
        _norm("norm_query", "norm", "bf16", 24, 768),
        # A training batch between two blocks, the block's output gated.
        _norm("norm_batch", "norm", "bf16", 16_384, 1_024, gate="silu"),
        # Its backward pass: six matrices of gradients and inputs, three vectors' gradients as sums over the batch.
        _norm("norm_grad_batch", "norm_grad", "bf16", 16_384, 1_024, gate="silu"),
        # Fine-tuning at the word vectors' width in fp32, rows that are no multiple of anything.
        _norm("norm_grad_words", "norm_grad", "fp32", 10_007, 100, gate="plain", scale=False),
        # A text that grows by a token: latency.
        _attention("attention_token", "attention", "bf16", 1, 1, 16, 16, 64, 64, state=True),
        # One token for each of many texts: every state is read and written.
        _attention("attention_tokens", "attention", "bf16", 256, 1, 16, 16, 128, 128, state=True),
        # Queries of uneven length behind one padding, heads sharing keys and values.
        _attention("attention_ragged", "attention", "fp16", 37, 131, 12, 4, 64, 64, ragged=True, packed=True),
        # Texts in fp32, the type that the indexes take.
        _attention("attention_fp32", "attention", "fp32", 8, 1_000, 12, 12, 64, 64),
        # One long document: few heads, a long axis, its state kept.
        _attention("attention_document", "attention", "bf16", 1, 32_768, 16, 16, 128, 128, state=True),
        # A training batch backwards, straight from one projection's result.
        _attention("attention_grad_batch", "attention_grad", "bf16", 8, 4_096, 16, 16, 128, 128, packed=True),
        # The gradients of a small encoder: a few tensors, launches count.
        _clip("clip_small", "fp32", 4_096, 64, 1, 1.0),
        # The gradients of 24 layers of 1,024 and a table: 290 tensors, matrices in bf16 and vectors in fp32.
        _clip("clip_model", "bf16", 32_000, 1_024, 24, 1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "attention", "attention", "attention", "attention_grad", "attention_grad", "clip"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if kind in ("norm", "norm_grad"):
        dim = _log_int(rng, 16, 8_192)
        rows = _log_int(rng, 1, (8_000_000 if dtype == "fp32" else 16_000_000) // dim)
        block = rng.random() < 0.8
        case = _norm("", kind, dtype, rows, dim, block, rng.choice(["none", "plain", "sigmoid", "silu"]) if block else "none",
                     block and rng.random() < 0.6)
    elif kind == "clip":
        dim = _log_int(rng, 16, 1_024)
        case = _clip("", dtype, _log_int(rng, 100, 32_000), dim, _log_int(rng, 1, 10 if dtype == "fp32" else 24),
                     rng.choice([0.1, 1.0, 1.0, 100.0]))
    else:
        # At most 1.2e8 elements of q, k, v and the result (the largest listed one has 2.7e8), 6e7 of states.
        dk = rng.choice([32, 64, 64, 128, 128, _log_int(rng, 16, 256)])
        dv = dk if rng.random() < 0.6 else _log_int(rng, 16, 256)
        share = rng.choice([1, 1, 2, 4])
        kv_heads = _log_int(rng, 1, 16)
        heads = kv_heads * share
        one = kind == "attention" and rng.random() < 0.4
        batch = _log_int(rng, 1, min(256, 60_000_000 // (heads * dk * dv)) if one else 32)
        most = int((3e7 if dtype == "fp32" else 6e7) / (batch * heads * (dk + dv)))
        tokens = 1 if one else _log_int(rng, 2, max(3, min(32_768, most)))
        case = _attention("", kind, dtype, batch, tokens, heads, kv_heads, dk, dv, one or rng.random() < 0.3,
                          not one and rng.random() < 0.4, dk == dv and rng.random() < 0.4)
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------------


def _shapes(case):
    """The tensors of a model with so many layers, each a matrix or a vector."""
    d = case["dim"]
    shapes = [(case["words"], d), (d,)]
    for _ in range(case["layers"]):
        shapes += [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,), (d,)]
    return shapes


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE)
    g.manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    kind = case["kind"]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=_DEVICE) * std + mean).to(dt)

    state = dict(case=case)
    if kind == "clip":
        # Backward passes leave gradients of very different sizes; vectors are kept in fp32.
        shapes = _shapes(case)
        size = sum(math.prod(s) for s in shapes)
        grads = []
        for i, s in enumerate(shapes):
            std = 10.0 * 2.0 ** (i % 5 - 2) / math.sqrt(size)
            x = torch.randn(s, generator=g, device=_DEVICE) * std
            grads.append(x.to(dt) if len(s) == 2 else x)
        # The clipped gradients go into two buffers, matrices and vectors, as an optimiser's steps take them.
        flat = [torch.empty(sum(math.prod(s) for s in shapes if len(s) == n), device=_DEVICE, dtype=dt if n == 2 else torch.float32)
                for n in (2, 1)]
        parts = [iter(x.split([math.prod(s) for s in shapes if len(s) == n])) for x, n in zip(flat, (2, 1))]
        return dict(case=case, grads=grads, flat=flat, out=[next(parts[0 if len(s) == 2 else 1]).view(s) for s in shapes])
    if kind in ("norm", "norm_grad"):
        n, d = case["rows"], case["dim"]
        state["weight"] = normal(d, std=0.1, mean=1.0)
        if case["block"]:
            state["y"] = normal(n, d, std=0.7)
            state["post"] = normal(d, std=0.1, mean=1.0)
        if case["gate"] != "none":
            state["gate"] = normal(n, d)
        if case["scale"]:
            state["scale"] = normal(d, std=0.05, mean=0.3)
        if kind == "norm":
            state["x"] = normal(n, d, std=2.0)
        else:  # r is what the forward pass gave
            state["r"] = normal(n, d, std=2.0)
            state["grad_h"] = normal(n, d, std=0.01)
            if case["block"]:
                state["grad_r"] = normal(n, d, std=0.01)
        return state
    b, t, h, hk, dk, dv = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dk", "dv"))
    if case["packed"]:  # views of one projection's result
        p = normal(b, t, (h + 2 * hk) * dk)
        q, k, v = p.split([h * dk, hk * dk, hk * dk], dim=-1)
        state["q"], state["k"], state["v"] = q.unflatten(-1, (h, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hk, dk))
    else:
        state["q"], state["k"], state["v"] = normal(b, t, h, dk), normal(b, t, hk, dk), normal(b, t, hk, dv)
    # Memories from two tokens to a thousand.
    state["log_decay"] = -torch.exp2(-10.0 * torch.rand(h, generator=g, device=_DEVICE))
    state["state"] = torch.randn((b, h, dk, dv), generator=g, device=_DEVICE) if case["state"] else None
    state["lengths"] = None
    if case["ragged"]:
        state["lengths"] = torch.randint(t + 1, (b,), generator=g, device=_DEVICE)
        state["lengths"][0] = t
    if kind == "attention_grad":
        state["grad"] = normal(b, t, h, dv, std=0.01)
        state["grad_state"] = torch.randn((b, h, dk, dv), generator=g, device=_DEVICE) * 0.01 if case["state"] else None
    return state


# ---- one pass ---------------------------------------------------------------------------------


def _inverse(x):
    return 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)


def _open(gate, act):
    """The gate and its slope."""
    if act == "plain":
        return gate, torch.ones_like(gate)
    s = 1.0 / (1.0 + torch.exp(-gate))
    return (s, s * (1.0 - s)) if act == "sigmoid" else (gate * s, s * (1.0 + gate * (1.0 - s)))


def _scan(q, k, v, log_decay, state, valid, first):
    """o = S^T q over the tokens in order, in fp32 [b, h, t, d], by chunks: within one the scores of its pairs, between them
    the state. first: 1 where the state decays ahead of the first token, 0 where behind it."""
    count = torch.cumsum(valid.float(), 1)
    g = log_decay[None, :, None]
    k, v = k * valid[:, None, :, None], v * valid[:, None, :, None]
    out = torch.empty((*q.shape[:3], v.shape[3]), device=q.device)
    base = torch.zeros_like(count[:, :1])
    for c in range(0, q.shape[2], 128):
        part = slice(c, c + 128)
        at = (count[:, part] - base)[:, None, :]
        qc, kc, vc = q[:, :, part], k[:, :, part], v[:, :, part]
        apart = (at[..., :, None] - at[..., None, :]).clamp(min=0.0)
        scores = (qc @ kc.transpose(2, 3).contiguous()) * torch.exp(g[..., None] * apart)
        near = scores.tril() @ vc
        total = at[..., -1:]
        out[:, :, part] = near + (qc @ state) * torch.exp(g * (at - 1.0 + first))[..., None]
        weighed = kc * torch.exp(g * (total - at + (1.0 - first)))[..., None]
        state = state * torch.exp(g * total)[..., None] + weighed.transpose(2, 3).contiguous() @ vc
        base = count[:, part][:, -1:]
    return out * valid[:, None, :, None], state


def _plain_attention(state):
    case = state["case"]
    dt, h, hk, dk, dv = _TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dk"], case["dv"]
    wide = lambda x: x.float().transpose(1, 2).contiguous()  # noqa: E731  [b, h, t, d]
    each = lambda x: wide(x).repeat_interleave(h // hk, 1)  # noqa: E731
    q, k, v, g = wide(state["q"]), each(state["k"]), each(state["v"]), state["log_decay"]
    b, t = q.shape[0], q.shape[2]
    at = torch.arange(t, device=q.device)[None]
    valid = at < (state["lengths"][:, None] if state["lengths"] is not None else t)
    valid = valid.expand(b, t)
    start = state["state"] if state["state"] is not None else torch.zeros((b, h, dk, dv), device=q.device)
    factor = dk ** -0.5
    back = lambda x: x.transpose(1, 2).to(dt).contiguous()  # noqa: E731
    if case["kind"] == "attention":
        o, end = _scan(q, k, v, g, start, valid, 1.0)
        return (back(o * factor), end) if case["state"] else back(o * factor)
    grad = wide(state["grad"])
    dq, _ = _scan(grad, v, k, g, start.transpose(2, 3).contiguous(), valid, 1.0)
    turn = lambda x: x.flip(2)  # noqa: E731
    behind = state["grad_state"] if state["grad_state"] is not None else torch.zeros_like(start)
    late = valid.flip(1)
    q, grad, k, v = turn(q * factor), turn(grad), turn(k), turn(v)
    dv_, dstart = _scan(k, q, grad, g, behind, late, 0.0)
    dk_, _ = _scan(v, grad, q, g, behind.transpose(2, 3).contiguous(), late, 0.0)
    shared = lambda x: x.unflatten(1, (hk, h // hk)).sum(2)  # noqa: E731
    grads = back(dq * factor), back(shared(turn(dk_))), back(shared(turn(dv_)))
    return (*grads, dstart) if case["state"] else grads


def _plain(state):
    case = state["case"]
    kind, dt = case["kind"], _TYPES[case["dtype"]]
    if kind == "clip":
        total = sum((x.double() ** 2).sum() for x in state["grads"])
        norm = torch.sqrt(total)
        factor = (case["limit"] / (norm + _EPS)).clamp(max=1.0).float()
        for x, o in zip(state["grads"], state["out"]):
            o.copy_((x.float() * factor).to(x.dtype))
        return *state["flat"], norm.float()
    if kind in ("attention", "attention_grad"):
        return _plain_attention(state)
    weight = state["weight"].float()
    if kind == "norm":
        r = state["x"].float()
        if case["block"]:
            y = state["y"].float()
            u = y * _inverse(y) * state["post"].float()
            if case["gate"] != "none":
                u = u * _open(state["gate"].float(), case["gate"])[0]
            r = r + (u * state["scale"].float() if case["scale"] else u)
        h = (r * _inverse(r) * weight).to(dt)
        return (r.to(dt), h) if case["block"] else h
    r, dh = state["r"].float(), state["grad_h"].float()
    inv = _inverse(r)
    rn, a = r * inv, dh * weight
    dr = inv * (a - rn * (a * rn).mean(-1, keepdim=True))
    dweight = (dh * rn).sum(0)
    if not case["block"]:
        return dr.to(dt), dweight.to(dt)
    dr = dr + state["grad_r"].float()
    y, post = state["y"].float(), state["post"].float()
    inv = _inverse(y)
    yn = y * inv
    u = yn * post
    gate, slope = _open(state["gate"].float(), case["gate"]) if case["gate"] != "none" else (None, None)
    du = dr * state["scale"].float() if case["scale"] else dr
    out = [dr.to(dt), dweight.to(dt)]
    if gate is not None:
        dgate = (du * u * slope).to(dt)
        dscale = dr * u * gate
        du = du * gate
    else:
        dscale = dr * u
    b = du * post
    out += [(inv * (b - yn * (b * yn).mean(-1, keepdim=True))).to(dt), (du * yn).sum(0).to(dt)]
    if gate is not None:
        out.append(dgate)
    if case["scale"]:
        out.append(dscale.sum(0).to(dt))
    return tuple(out)


def run(state):
    if not own:
        return _plain(state)
    import quiver_amd as quiver

    case = state["case"]
    kind = case["kind"]
    if kind == "clip":
        _, norm = quiver.clip_grad_norm(state["grads"], case["limit"], out=state["out"])
        return *state["flat"], norm
    if kind == "attention":
        return quiver.linear_attention(state["q"], state["k"], state["v"], state["log_decay"], state=state["state"],
                                       lengths=state["lengths"], keep_state=case["state"])
    if kind == "attention_grad":
        grads = quiver.linear_attention_grad(state["grad"], state["q"], state["k"], state["v"], state["log_decay"],
                                             state=state["state"], lengths=state["lengths"], grad_state=state["grad_state"])
        return grads if case["state"] else grads[:3]
    block = dict(y=state.get("y"), post_weight=state.get("post"), gate=state.get("gate"), scale=state.get("scale"),
                 gate_activation=case["gate"] if case["gate"] in ("sigmoid", "silu") else None, eps=_EPS)
    if kind == "norm":
        return quiver.block_norm(state["x"], state["weight"], **block)
    grads = quiver.block_norm_grad(state["grad_h"], state["r"], state["weight"], grad_r=state.get("grad_r"), **block)
    return tuple(x for x in grads if x is not None)


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    kind, e = case["kind"], float(_SIZE[case["dtype"]])
    if kind == "clip":
        sizes = [(math.prod(s), e if len(s) == 2 else 4.0) for s in _shapes(case)]
        return {"bytes": 2.0 * sum(n * b for n, b in sizes), "flops": 3.0 * sum(n for n, _ in sizes)}
    if kind in ("norm", "norm_grad"):
        n, d, gate = float(case["rows"]), float(case["dim"]), case["gate"] != "none"
        if kind == "norm":
            matrices = (4 + gate) if case["block"] else 2
            return {"bytes": e * d * (n * matrices + 3), "flops": n * d * (12 if case["block"] else 5)}
        matrices = (6 + 2 * gate) if case["block"] else 3  # in: dh, dr, r, y, gate; out: dx, dy, dgate
        return {"bytes": e * d * (n * matrices + 6), "flops": n * d * (30 if case["block"] else 10)}
    b, t, h, hk, dk, dv = (float(case[k]) for k in ("batch", "tokens", "heads", "kv_heads", "dk", "dv"))
    states = b * h * dk * dv * (2 if case["state"] else 0)
    q, kv, o = b * t * h * dk, b * t * hk * (dk + dv), b * t * h * dv
    if kind == "attention":  # the state's step and the result, by the recurrence
        return {"bytes": e * (q + kv + o) + 4.0 * states, "flops": 4.0 * b * t * h * dk * dv}
    # In: q, k, v, the result's gradient, both states; out: the gradients of q, k, v and of the first state.
    return {"bytes": e * (2.0 * q + 2.0 * kv + o) + 6.0 * states, "flops": 10.0 * b * t * h * dk * dv}


# ---- 64-bit results ---------------------------------------------------------------------------


def _exact_attention(case, s):
    """Token by token, by the recurrence itself."""
    d = lambda name: s[name].to(torch.float64)  # noqa: E731
    each = case["heads"] // case["kv_heads"]
    q, k, v = d("q"), torch.repeat_interleave(d("k"), each, dim=2), torch.repeat_interleave(d("v"), each, dim=2)
    b, t, h, dk = q.shape
    dv = v.shape[3]
    decay = torch.exp(d("log_decay"))[None, :, None, None]
    mem = d("state").clone() if case["state"] else q.new_zeros((b, h, dk, dv))
    scale = 1.0 / math.sqrt(dk)
    lengths = s["lengths"].tolist() if s["lengths"] is not None else [t] * b
    live = (torch.arange(t)[:, None] < torch.tensor(lengths)[None, :]).to(q.device)  # [t, b]
    whole = [min(lengths) > i for i in range(t)]

    def moved(i, new, old):
        return new if whole[i] else torch.where(live[i][:, None, None, None], new, old)

    def outer(x, y):
        return x[..., :, None] * y[..., None, :]

    if case["kind"] == "attention":
        o = q.new_zeros((b, t, h, dv))
        for i in range(t):
            mem = moved(i, mem * decay + outer(k[:, i], v[:, i]), mem)
            o[:, i] = (q[:, i][..., None, :] @ mem)[..., 0, :]
        o = o * scale * live.t()[:, :, None, None]
        return (o, mem) if case["state"] else o
    grad = d("grad") * scale
    dq, dk_, dv_ = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(t):
        mem = moved(i, mem * decay + outer(k[:, i], v[:, i]), mem)
        dq[:, i] = (mem @ grad[:, i][..., None])[..., 0]
    back = d("grad_state").clone() if case["state"] else torch.zeros_like(mem)
    for i in range(t - 1, -1, -1):
        now = back + outer(q[:, i], grad[:, i])
        dk_[:, i] = (now @ v[:, i][..., None])[..., 0]
        dv_[:, i] = (k[:, i][..., None, :] @ now)[..., 0, :]
        back = moved(i, now * decay, back)
    mask = live.t()[:, :, None, None]
    total = lambda x: torch.where(mask, x, torch.zeros_like(x)).reshape(b, t, -1, each, x.shape[-1]).sum(3)  # noqa: E731
    grads = torch.where(mask, dq, torch.zeros_like(dq)), total(dk_), total(dv_)
    return (*grads, back) if case["state"] else grads


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("attention", "attention_grad"):
        return _exact_attention(case, s)
    if kind == "clip":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(x.to(torch.float64)) for x in s["grads"]]))
        factor = min(1.0, case["limit"] / (norm.item() + _EPS))
        flat = [torch.cat([x.reshape(-1) for x in s["grads"] if x.dim() == n]) for n in (2, 1)]
        return *(x.to(torch.float64) * factor for x in flat), norm
    # The gradients by differentiating the formula itself.
    forward = kind == "norm"
    d = {k: x.to(torch.float64).requires_grad_(not forward) for k, x in s.items() if isinstance(x, torch.Tensor)}

    def normed(x, w):
        return torch.nn.functional.rms_norm(x, (case["dim"],), w, _EPS)

    def step():
        u = normed(d["y"], d["post"])
        if "gate" in d:
            u = u * {"plain": lambda z: z, "sigmoid": torch.sigmoid, "silu": lambda z: z * torch.sigmoid(z)}[case["gate"]](d["gate"])
        return u * d["scale"] if "scale" in d else u

    if forward:
        r = d["x"] + step() if case["block"] else d["x"]
        h = normed(r, d["weight"])
        return (r, h) if case["block"] else h
    dr, dweight = torch.autograd.grad(normed(d["r"], d["weight"]), (d["r"], d["weight"]), d["grad_h"].detach())
    if not case["block"]:
        return dr, dweight
    dr = dr + d["grad_r"].detach()
    wanted = [d[k] for k in ("y", "post", "gate", "scale") if k in d]
    return (dr, dweight, *torch.autograd.grad(step(), wanted, dr))
