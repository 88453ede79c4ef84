"""Norms around a block and the gradients' norm against 64-bit arithmetic.

u is the unit roundoff of the result's type (2^-24, 2^-11, 2^-8). Bounds are of the formulas' terms: a norm's sum of
squares is at most 64 additions deep (32 of a thread, 10 in the wave, 16 waves, the rest), so its inverse root is
off by 34 2^-24 at most, and a value of f such factors by their sum. Those below are rounded up to powers of two.
"""

import math

import pytest

import quiver_amd as quiver

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_encoder_gpu import ROUND, TINY, TYPES, _gpu, _randn, _say, _within  # noqa: E402

E = 2.0**-24


def _inverse(t, eps):
    return 1.0 / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)


def _gate(z, act):
    """Value, slope and the slope's magnitude."""
    if act is None:
        return z, torch.ones_like(z), torch.ones_like(z)
    s, o = torch.sigmoid(z), torch.sigmoid(-z)
    if act == "sigmoid":
        return s, s * o, s * o
    return z * s, s * (1 + z * o), s * (1 + (z * o).abs())


def _forward_64(x, w, y, post, gate, act, scale, eps):
    """r, h and the bounds of fp32's arithmetic on them."""
    r, off = x, torch.zeros_like(x)
    if y is not None:
        u = y * _inverse(y, eps) * post
        if gate is not None:
            u = u * _gate(gate, act)[0]
        if scale is not None:
            u = u * scale
        r = x + u
        off = 64 * E * u.abs() + E * r.abs()
    inv = _inverse(r, eps)
    # An error of r also moves its norm, by at most as large a part of it as of its largest ones.
    along = (off * r.abs()).mean(-1, keepdim=True) * inv * inv
    return r, off, r * inv * w, ((off + r.abs() * (64 * E + along)) * inv * w.abs())


def _block(g, shape, dtype, gate=True, scale=True):
    dim = shape[-1]
    return dict(y=_randn(g, *shape, dtype=dtype, std=0.7), post_weight=1 + _randn(g, dim, dtype=dtype, std=0.2),
                gate=_randn(g, *shape, dtype=dtype, std=2.0) if gate else None,
                scale=_randn(g, dim, dtype=dtype, std=0.5) if scale else None)


def _check_norm(x, w, dtype, act=None, eps=1e-6, **block):
    got = quiver.block_norm(x, w, gate_activation=act, eps=eps, **block)
    wide = {k: v.double() if v is not None else None for k, v in block.items()}
    r, r_off, h, h_off = _forward_64(x.double(), w.double(), wide.get("y"), wide.get("post_weight"), wide.get("gate"), act,
                                     wide.get("scale"), eps)
    if block.get("y") is not None:
        assert got[0].dtype == x.dtype
        _within(got[0], r, r_off + r.abs() * ROUND[dtype] + TINY[dtype], "r")
        got = got[1]
    assert got.dtype == x.dtype
    _within(got, h, h_off + h.abs() * ROUND[dtype] + TINY[dtype], "h")


# Every way of taking a row: parts of a wave, a wave, four waves and sixteen, whole pieces and a last one moved back.
DIMS = [1, 3, 5, 8, 31, 64, 100, 129, 256, 500, 768, 1000, 1024, 1025, 2000, 2051, 4096, 4099, 8192, 8200, 16_384]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", DIMS)
def test_block_norm(dtype, dim):
    g = torch.Generator().manual_seed(dim)
    for rows in (1, 37):
        _say("block_norm", dtype, rows, dim)
        x, w = _randn(g, rows, dim, dtype=dtype, std=2.0), 1 + _randn(g, dim, dtype=dtype, std=0.2)
        _check_norm(x, w, dtype)
        _check_norm(x, w, dtype, **_block(g, (rows, dim), dtype, gate=False))
        for act in (None, "sigmoid", "silu"):
            _check_norm(x, w, dtype, act=act, **_block(g, (rows, dim), dtype, scale=act != "silu"))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim", [(20_011, 24), (4_100, 768), (2_500, 1_500), (1_100, 5_000)])
def test_block_norm_of_more_rows_than_work_groups(dtype, rows, dim):
    g = torch.Generator().manual_seed(rows)
    _say("block_norm", dtype, rows, dim)
    x, w = _randn(g, rows, dim, dtype=dtype), 1 + _randn(g, dim, dtype=dtype, std=0.2)
    _check_norm(x, w, dtype)
    _check_norm(x, w, dtype, act="silu", **_block(g, (rows, dim), dtype))
    _check_grad(g, (rows, dim), dtype, "silu")


def _grad_64(gh, gr, r, w, y, post, gate, act, scale, eps):
    """The gradients by the formula, each with the magnitude of its terms."""
    inv = _inverse(r, eps)
    a, rn = gh * w, r * inv
    dx = inv * (a - rn * (a * rn).mean(-1, keepdim=True))
    mx = inv * (a.abs() + rn.abs() * (a * rn).abs().mean(-1, keepdim=True))
    if gr is not None:
        dx, mx = dx + gr, mx + gr.abs()
    out = [(dx, mx), ((gh * rn).sum(0), (gh * rn).abs().sum(0)), None, None, None, None]
    if y is None:
        return out
    inv = _inverse(y, eps)
    yn = y * inv
    u = yn * post
    opened, slope, mslope = _gate(gate, act) if gate is not None else (torch.ones_like(y),) * 3
    s = scale if scale is not None else torch.ones_like(post)
    du, mu = dx * s * opened, mx * (s * opened).abs()
    b, mb = du * post, mu * post.abs()
    out[2] = (inv * (b - yn * (b * yn).mean(-1, keepdim=True)), inv * (mb + yn.abs() * (mb * yn.abs()).mean(-1, keepdim=True)))
    out[3] = ((du * yn).sum(0), (mu * yn.abs()).sum(0))
    if gate is not None:
        out[4] = (dx * s * u * slope, mx * (s * u).abs() * mslope)
    if scale is not None:
        out[5] = ((dx * opened * u).sum(0), (mx * (opened * u).abs()).sum(0))
    return out


def _check_grad(g, shape, dtype, act=None, eps=1e-6, block=True, gate=True, scale=True, gr=True):
    rows, dim = shape
    r, w = _randn(g, *shape, dtype=dtype, std=2.0), 1 + _randn(g, dim, dtype=dtype, std=0.2)
    gh = _randn(g, *shape, dtype=dtype)
    grad_r = _randn(g, *shape, dtype=dtype) if gr else None
    parts = _block(g, shape, dtype, gate, scale) if block else {}
    got = quiver.block_norm_grad(gh, r, w, grad_r=grad_r, gate_activation=act, eps=eps, **parts)
    wide = {k: v.double() if v is not None else None for k, v in parts.items()}
    want = _grad_64(gh.double(), None if grad_r is None else grad_r.double(), r.double(), w.double(), wide.get("y"),
                    wide.get("post_weight"), wide.get("gate"), act, wide.get("scale"), eps)
    for name, a, b in zip(("x", "weight", "y", "post_weight", "gate", "scale"), got, want):
        assert (a is None) == (b is None), name
        if a is None:
            continue
        assert a.dtype == r.dtype, name
        # Up to six norms and means one after another, 70 2^-24 each; sums over the rows add a term's 2^-23 each.
        count = 0 if a.dim() == 2 else rows
        _within(a, b[0], b[1] * (512 * E + count * 2.0**-23) + b[0].abs() * ROUND[dtype] + TINY[dtype], name)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", DIMS)
def test_block_norm_grad(dtype, dim):
    g = torch.Generator().manual_seed(dim + 1)
    for rows in (1, 41):
        _say("block_norm_grad", dtype, rows, dim)
        _check_grad(g, (rows, dim), dtype, block=False, gr=rows > 1)
        _check_grad(g, (rows, dim), dtype, gate=False, scale=rows > 1)
        for act in (None, "sigmoid", "silu"):
            _check_grad(g, (rows, dim), dtype, act, scale=act != "silu", gr=act != "sigmoid")


def test_block_norm_grad_against_differences():
    """A step along a direction changes the loss by the gradient's part along it (fp32, central differences)."""
    g = torch.Generator().manual_seed(3)
    _say("block_norm differences")
    x, w = _randn(g, 9, 50, dtype="fp32"), 1 + _randn(g, 50, dtype="fp32", std=0.2)
    parts = _block(g, (9, 50), "fp32")
    cr, ch = _randn(g, 9, 50, dtype="fp32"), _randn(g, 9, 50, dtype="fp32")

    def loss(x, w, **parts):
        r, h = quiver.block_norm(x, w, gate_activation="silu", **parts)
        return (cr.double() * r.double()).sum() + (ch.double() * h.double()).sum()

    r, _ = quiver.block_norm(x, w, gate_activation="silu", **parts)
    grads = quiver.block_norm_grad(ch, r, w, grad_r=cr, gate_activation="silu", **parts)
    names = ("x", "w", "y", "post_weight", "gate", "scale")
    values = dict(x=x, w=w, **parts)
    for name, grad in zip(names, grads):
        d = _randn(g, *values[name].shape, dtype="fp32")
        d /= d.norm()
        step = 2.0**-6
        up, down = (loss(**{**values, name: values[name] + s * d}) for s in (step, -step))
        slope = ((up - down) / (2 * step)).item()
        along = (grad.double() * d.double()).sum().item()
        # Third derivatives of order one leave step^2 = 2^-12 of the gradient's size; fp32 results 2^-24 of the loss's terms.
        size = grad.double().norm().item() + 1.0
        assert abs(slope - along) <= size * 2.0**-10 + 900 * 8 * E / step, name


def test_block_norm_strided_misaligned_and_empty():
    dev = _gpu()
    g = torch.Generator().manual_seed(5)
    _say("block_norm strided")
    for dtype in TYPES:
        big = _randn(g, 60, 210, dtype=dtype)
        w, post = 1 + _randn(g, 101, dtype=dtype, std=0.2), 1 + _randn(g, 202, dtype=dtype, std=0.2)[::2]
        for x in (big[:, 1:102], big[::3][:, 7:108], big.t()[:101].t(), big[:50, 3:104].reshape(5, 10, 101)):
            y, gate = x.flip(0), x * 0.5
            got = quiver.block_norm(x, w, y=y, post_weight=post, gate=gate, gate_activation="silu")
            want = quiver.block_norm(x.contiguous(), w, y=y.contiguous(), post_weight=post.contiguous(), gate=gate.contiguous(),
                                     gate_activation="silu")
            assert got[0].shape == x.shape and all(torch.equal(a, b) for a, b in zip(got, want))
            grads = quiver.block_norm_grad(x, y, w, grad_r=gate, y=x, post_weight=post, gate=y)
            plain = quiver.block_norm_grad(x.contiguous(), y.contiguous(), w, grad_r=gate.contiguous(), y=x.contiguous(),
                                           post_weight=post.contiguous(), gate=y.contiguous())
            assert all(torch.equal(a, b) for a, b in zip(grads, plain) if a is not None)
        # A gate that is broadcast has no rows of its own.
        shared = quiver.block_norm(big, torch.ones_like(big[0]), y=big, post_weight=big[1], gate=big[:1].expand_as(big))
        assert torch.equal(shared[0], quiver.block_norm(big, torch.ones_like(big[0]), y=big, post_weight=big[1],
                                                        gate=big[:1].repeat(60, 1))[0])
        none = big[:0]
        assert quiver.block_norm(none, big[0]).shape == (0, 210)
        r, h = quiver.block_norm(none, big[0], y=none, post_weight=big[1], scale=big[2])
        assert r.shape == h.shape == (0, 210)
        grads = quiver.block_norm_grad(none, none, big[0], y=none, post_weight=big[1], gate=none, scale=big[2])
        assert [tuple(t.shape) for t in grads] == [(0, 210), (210,), (0, 210), (210,), (0, 210), (210,)]
        assert not any(t.any() for t in grads)
    assert torch.equal(quiver.block_norm(torch.full((7,), 2.0, device=dev), torch.ones(7, device=dev), eps=0.0), torch.ones(7, device=dev))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [24, 100, 1024, 3000])
def test_block_norm_keeps_rows_apart(dtype, dim):
    """Rows of NaN, infinities and zeros leave the others as they are."""
    g = torch.Generator().manual_seed(dim)
    _say("block_norm special", dtype, dim)
    x, w = _randn(g, 9, dim, dtype=dtype), 1 + _randn(g, dim, dtype=dtype, std=0.2)
    parts = _block(g, (9, dim), dtype)
    want = quiver.block_norm(x, w, gate_activation="silu", **parts)
    y, gate = parts["y"].clone(), parts["gate"].clone()
    x2 = x.clone()
    x2[1], y[3, dim // 2], gate[5, 0], y[7] = float("nan"), float("inf"), float("nan"), 0.0
    got = quiver.block_norm(x2, w, gate_activation="silu", **{**parts, "y": y, "gate": gate})
    others = [0, 2, 4, 6, 8]
    assert all(torch.equal(a[others], b[others]) for a, b in zip(got, want))
    assert torch.isnan(got[1][1]).all() and torch.isnan(got[0][3, dim // 2]) and torch.isnan(got[1][5]).all()
    assert torch.equal(got[0][7], x[7])  # the norm of zeros is zeros
    zero = torch.zeros_like(x)
    assert not quiver.block_norm(zero, w).any()
    dx, dw = quiver.block_norm_grad(x, zero, w)[:2]
    assert torch.isfinite(dx).all() and not dw.any()


def test_block_norm_gates_far_out():
    """Gates at the ends of their range: the logistic function's own values, slopes that go to zero."""
    dev = _gpu()
    _say("block_norm gates")
    z = torch.tensor([-300.0, -80.0, -20.0, -1.27846, 0.0, 20.0, 80.0, 300.0], device=dev)
    one = torch.ones_like(z)
    for act in ("sigmoid", "silu"):
        r, _ = quiver.block_norm(z * 0, one, y=one, post_weight=one, gate=z, gate_activation=act, eps=0.0)
        value, slope, size = _gate(z.double(), act)
        _within(r, value, value.abs() * 16 * E + 2.0**-126, act)
        dgate = quiver.block_norm_grad(one * 0, one, one, grad_r=one, y=one, post_weight=one, gate=z, gate_activation=act, eps=0.0)[4]
        _within(dgate, slope, size * 32 * E + 2.0**-120, act)


# ---- the gradients' norm ----------------------------------------------------------------------


def _model(g, sizes, types):
    return [_randn(g, *(s or (1,)), dtype=t, std=1.0 + i % 3).reshape(s) for i, (s, t) in enumerate(zip(sizes, types))]


SIZES = {"one": [(1,)], "few": [(64, 100), (7,), (), (3, 0), (129, 65), (8193,), (8192,), (5, 3, 11)],
         "many": [(i % 37 + 1, i % 11 + 1) for i in range(700)], "large": [(3_000_001,), (17,), (999, 1001)]}


@pytest.mark.parametrize("dtype", [*TYPES, "mixed"])
@pytest.mark.parametrize("which", list(SIZES))
def test_clip_grad_norm(dtype, which):
    g = torch.Generator().manual_seed(7)
    sizes = SIZES[which]
    types = [dtype if dtype != "mixed" else list(TYPES)[i % 3] for i in range(len(sizes))]
    _say("clip_grad_norm", dtype, which)
    grads = _model(g, sizes, types)
    want = math.sqrt(sum((t.double() ** 2).sum().item() for t in grads))
    norm = quiver.grad_norm(grads)
    assert norm.shape == () and norm.dtype == torch.float32
    # fp64 sums of 4e6 terms at most, one rounding to fp32.
    assert abs(norm.item() - want) <= want * 1.01 * E
    for limit in (want * 0.37, 1.0, want * 1.5):
        clipped, norm = quiver.clip_grad_norm(grads, limit)
        assert abs(norm.item() - want) <= want * 1.01 * E
        factor = min(1.0, limit / (want + 1e-6))
        for a, b, t in zip(clipped, grads, types):
            assert a.dtype == b.dtype and a.shape == b.shape and a.data_ptr() != b.data_ptr() or not b.numel()
            exact = b.double() * factor
            _within(a, exact, exact.abs() * (ROUND[t] + 3 * E) + TINY[t])
            if factor == 1.0:
                assert torch.equal(a, b)
        held = [b.clone() for b in grads]
        same, _ = quiver.clip_grad_norm(held, limit, out=held)
        assert all(a is b for a, b in zip(same, held)) and all(torch.equal(a, b) for a, b in zip(same, clipped))


def test_clip_grad_norm_special():
    dev = _gpu()
    _say("clip_grad_norm special")
    big = torch.full((1000,), 3e38, device=dev)  # squares past fp32's range
    small = torch.full((1000,), 1e-30, device=dev)  # and below it
    want = math.sqrt(1000.0) * 1e-30
    assert abs(quiver.grad_norm([small]).item() / want - 1) <= 4 * E
    clipped, norm = quiver.clip_grad_norm([big, small], 1.0)
    assert torch.isinf(norm) == (math.sqrt(1000.0) * 3e38 > 3.4028e38)
    # The factor follows from the fp64 norm, which fp32 cannot hold here.
    assert abs(clipped[0][0].item() * math.sqrt(1000.0) - 1) <= 16 * E
    x = torch.arange(10.0, device=dev)
    x[3] = float("inf")
    clipped, norm = quiver.clip_grad_norm([x, torch.ones(5, device=dev)], 1.0)
    assert torch.isinf(norm) and torch.isnan(clipped[0][3]) and not clipped[1].any() and not clipped[0][4:].any()
    x[3] = float("nan")
    clipped, norm = quiver.clip_grad_norm([x, torch.ones(5, device=dev)], 1.0)
    assert torch.isnan(norm) and all(torch.isnan(t).all() for t in clipped)
    zeros = [torch.zeros(9, device=dev)]
    clipped, norm = quiver.clip_grad_norm(zeros, 0.0)
    assert norm.item() == 0 and not clipped[0].any()
    clipped, norm = quiver.clip_grad_norm([], 1.0)
    assert clipped == [] and norm.item() == 0 and quiver.grad_norm([]).item() == 0
    assert quiver.grad_norm([torch.zeros(0, device=dev)]).item() == 0
    base = torch.randn(40, 61, generator=torch.Generator().manual_seed(1)).to(dev)
    for view in (base[:, 1:60], base.t(), base[1:, ::2], base.view(-1)[1:]):
        want = view * (1.0 / (view.double().norm().item() + 1e-6))
        for out in (None, [torch.empty_like(view)], [torch.empty(view.shape[::-1], device=dev).t()]):
            clipped, _ = quiver.clip_grad_norm([view], 1.0, out=out)
            _within(clipped[0], want, want.abs().double() * 8 * E)
        copy = base.clone()
        held = copy.as_strided(view.shape, view.stride(), view.storage_offset())
        quiver.clip_grad_norm([held], 1.0, out=[held])
        _within(held, want, want.abs().double() * 8 * E)
        touched = torch.zeros_like(base, dtype=torch.bool)
        touched.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(True)
        assert torch.equal(copy[~touched], base[~touched])


def test_clip_grad_norm_of_zeros_where_nothing_is_added():
    """A norm of 0 and an eps of 0 leave the gradients as they are, whatever the limit; other norms follow the formula."""
    dev = _gpu()
    _say("clip_grad_norm zeros")
    zeros = [torch.zeros(9, device=dev), torch.full((3, 5), -0.0, device=dev, dtype=torch.bfloat16), torch.zeros(0, device=dev)]
    for limit in (0.0, 1.0):
        held = [t.clone() for t in zeros]
        for out in (None, held):
            clipped, norm = quiver.clip_grad_norm(zeros if out is None else held, limit, out=out, eps=0.0)
            assert norm.item() == 0 and all(torch.equal(a, b) for a, b in zip(clipped, zeros))
    one = torch.ones(4, device=dev)
    assert not quiver.clip_grad_norm([one], 0.0, eps=0.0)[0][0].any()
    assert torch.equal(quiver.clip_grad_norm([one], 1.0, eps=0.0)[0][0], one * 0.5)
    one[2] = float("nan")
    assert torch.isnan(quiver.clip_grad_norm([one], 0.0, eps=0.0)[0][0]).all()


@pytest.mark.parametrize("limit", [1e-10, 1e-20, 1e-30, 2.0**-110, 2.0**-126, 2.0**-140, 0.0])
def test_clip_grad_norm_to_limits_far_below_the_norm(limit):
    """Factors that fp32 cannot hold, of gradients as large as it can: results that it holds come out as they are."""
    dev = _gpu()
    _say("clip_grad_norm far", limit)
    for types in (("fp32",), ("bf16",), ("fp32", "bf16")):
        values = torch.tensor([3e38, -1e38, 2.0**100, 1.0, 0.0, 2.0**-140], dtype=torch.float64)
        grads = [values.to(TYPES[t]).repeat(2_000).to(dev) for t in types]  # more than a chunk of a work-group's, and a rest
        norm = math.sqrt(sum((x.double() ** 2).sum().item() for x in grads))
        clipped, _ = quiver.clip_grad_norm(grads, limit)
        for a, x, t in zip(clipped, grads, types):
            want = x.double() * (limit / (norm + 1e-6))
            # The factor, a product and what is left of the fp32 range: half a step each; the limit itself is fp32.
            _within(a, want, want.abs() * (ROUND[t] + 3 * E) + TINY[t] + 2.0**-149)


def test_results_whose_elements_share_memory_are_refused_ahead_of_all_else():
    """A gradient that torch expanded has one element in many places: nothing of the list is scaled in place by halves."""
    dev = _gpu()
    _say("shared elements")
    whole, shared = torch.full((40,), 3.0, device=dev), torch.full((1, 8), 2.0, device=dev).expand(5, 8)
    with pytest.raises(ValueError, match="share memory"):
        quiver.clip_grad_norm([whole, shared], 1.0, out=[whole, shared])
    assert (whole == 3.0).all() and (shared == 2.0).all()
    clipped, norm = quiver.clip_grad_norm([whole, shared], 1.0)  # as inputs they are taken
    assert abs(norm.item() - math.sqrt(360 + 160)) <= 1e-4 and clipped[1].shape == (5, 8)
    q = torch.ones((2, 3, 4, 8), device=dev)
    state = torch.zeros((1, 4, 8, 8), device=dev).expand(2, 4, 8, 8)
    with pytest.raises(ValueError, match="share memory"):
        quiver.linear_attention(q, q, q, torch.zeros(4, device=dev), state=state, state_out=state)
    assert not state.any()


def test_clip_grad_norm_in_place_is_seen_by_autograd():
    dev = _gpu()
    x = torch.ones(4, device=dev, requires_grad=True)
    y = x * 2
    z = y * y  # keeps y
    quiver.clip_grad_norm([y.detach()], 1.0, out=[y.detach()])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


def test_clip_grad_norm_past_32_bit_offsets():
    dev = _gpu()
    n = 2**31 + 5_000
    _say("clip_grad_norm", n)
    x = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    x[0], x[-1], x[2**31] = 3.0, 4.0, 12.0
    (clipped,), norm = quiver.clip_grad_norm([x], 6.5, out=[x])
    assert norm.item() == 13.0
    assert abs(clipped[-1].item() - 2.0) <= 2.0**-7 and abs(clipped[2**31].item() - 6.0) <= 2.0**-6 and abs(clipped[0].item() - 1.5) <= 2.0**-8


# ---- refusals ---------------------------------------------------------------------------------


def test_refusals():
    dev = _gpu()
    _say("refusals")
    f = torch.zeros((8, 16), device=dev)
    w = torch.ones(16, device=dev)
    n = lambda *a, **k: lambda: quiver.block_norm(*a, **k)  # noqa: E731
    c = lambda *a, **k: lambda: quiver.clip_grad_norm(*a, **k)  # noqa: E731
    for call, word in [
            (n(f.double(), w), "float32"), (n(f, w[:8]), "weight must"), (n(f, w.half()), "weight is"), (n(f[0, 0], w), "x must"),
            (n(f.cpu(), w), "GPU memory"), (n(f, w, gate=f), "belongs"), (n(f, w, scale=w), "belongs"), (n(f, w, post_weight=w), "belongs"),
            (n(f, w, y=f), "post_weight"), (n(f, w, y=f[:4], post_weight=w), "y must"), (n(f, w, y=f, post_weight=w, gate=f[:, :8]), "gate must"),
            (n(f, w, y=f, post_weight=w, gate=f, gate_activation="gelu"), "gate_activation"), (n(f, w, eps=-1.0), "eps"),
            (n(f, w, eps=float("nan")), "eps"), (n(f[:, :0], w[:0]), "dim"), (n(torch.zeros((1, 16_385), device=dev), torch.zeros(16_385, device=dev)), "16384"),
            (lambda: quiver.block_norm_grad(f[:4], f, w), "grad_h must"), (lambda: quiver.block_norm_grad(f, f, w, grad_r=f.half()), "grad_r is"),
            (c([f.double()], 1.0), "float32"), (c([f, f.cpu()], 1.0), "others"), (c([f], float("inf")), "max_norm"), (c([f], -1.0), "max_norm"),
            (c([f], float("nan")), "max_norm"), (c([f], 1.0, eps=-1.0), "eps"), (c([f], 1.0, out=[]), "out must"), (c([f], 1.0, out=[f.half()]), "out must"),
            (c([f], 1.0, out=[f[:4]]), "out must"), (c([f, f], 1.0, out=[f, f]), "overlap"), (c([f[:6], f[4:]], 1.0, out=[f[:6], f[4:]]), "overlap"),
            (c([f[:4], f[2:6]], 1.0, out=[f[:4], w.new_empty(4, 16)]), "overlap"), (c([f.to_sparse()], 1.0), "dense")]:
        with pytest.raises(ValueError, match=word):
            call()
    with pytest.raises(TypeError):
        quiver.block_norm([1.0], w)
    with pytest.raises(TypeError):
        quiver.clip_grad_norm([f, None], 1.0)


# ---- together, streams, graphs ----------------------------------------------------------------


def _encoder_state(dtype, texts=5, tokens=70, seed=0):
    """A causal encoder of one block: a table, the norms' and the layers' weights, gates and decays."""
    g = torch.Generator().manual_seed(seed)
    d, h = 48, 3
    w = lambda n, k: _randn(g, n, k, dtype=dtype, std=k ** -0.5)  # noqa: E731
    v = lambda mean, n=d: mean + _randn(g, n, dtype=dtype, std=0.1)  # noqa: E731
    return dict(tok=torch.randint(-1, 300, (texts, tokens), generator=g).to(_gpu()), table=_randn(g, 300, d, dtype=dtype), w_in=v(1.0),
                w_qkv=w(3 * d, d), decay=-torch.exp2(-torch.arange(1.0, h + 1.0)).to(_gpu()), w_gate=w(d, d), w_att=v(1.0), s_att=v(0.4),
                w_mid=v(1.0), w_up=w(2 * d, d), b_up=v(0.0, 2 * d), w_down=w(d, 2 * d), w_out=v(1.0), s_out=v(0.4), w_end=v(1.0),
                lengths=torch.randint(1, tokens + 1, (texts,), generator=g).to(_gpu()), grad=_randn(g, texts, tokens, d, dtype=dtype))


def _step(s, limit=0.5):
    """Forwards, backwards by hand and the clipped gradients: as a program without autograd runs them."""
    b, t, d = s["grad"].shape
    heads = lambda x: x.unflatten(-1, (3, -1))  # noqa: E731
    x0 = quiver.embed(s["table"], s["tok"])
    h0 = quiver.block_norm(x0, s["w_in"])
    qkv = quiver.linear(h0, s["w_qkv"])
    q, k, v = (heads(p) for p in qkv.split(d, -1))
    o = quiver.linear_attention(q, k, v, s["decay"], lengths=s["lengths"])
    gate = quiver.linear(h0, s["w_gate"])
    y0 = o.flatten(2)
    x1, h1 = quiver.block_norm(x0, s["w_mid"], y=y0, post_weight=s["w_att"], gate=gate, gate_activation="silu", scale=s["s_att"])
    u, z = quiver.linear(h1, s["w_up"], bias=s["b_up"], activation="gelu", keep_preactivation=True)
    y1 = quiver.linear(u, s["w_down"])
    x2, h2 = quiver.block_norm(x1, s["w_end"], y=y1, post_weight=s["w_out"], scale=s["s_out"])

    dx2, dw_end, dy1, dw_out, _, ds_out = quiver.block_norm_grad(s["grad"], x2, s["w_end"], y=y1, post_weight=s["w_out"], scale=s["s_out"])
    du, dw_down, _ = quiver.linear_grad(dy1, u, s["w_down"], bias=False)
    dh1, dw_up, db_up = quiver.linear_grad(du, h1, s["w_up"], preactivation=z, activation="gelu")
    dx1, dw_mid, dy0, dw_att, dgate, ds_att = quiver.block_norm_grad(dh1, x1, s["w_mid"], grad_r=dx2, y=y0, post_weight=s["w_att"], gate=gate,
                                                                     gate_activation="silu", scale=s["s_att"])
    dh0, dw_gate, _ = quiver.linear_grad(dgate, h0, s["w_gate"], bias=False)
    dq, dk, dv, _ = quiver.linear_attention_grad(heads(dy0), q, k, v, s["decay"], lengths=s["lengths"])
    dqkv = torch.cat([p.flatten(2) for p in (dq, dk, dv)], -1)
    dh0b, dw_qkv, _ = quiver.linear_grad(dqkv, h0, s["w_qkv"], bias=False)
    dx0, dw_in = quiver.block_norm_grad(dh0 + dh0b, x0, s["w_in"])[:2]
    dtable = quiver.embed_grad(dx0 + dx1, s["tok"], len(s["table"]))
    grads = dict(table=dtable, w_in=dw_in, w_qkv=dw_qkv, w_gate=dw_gate, w_att=dw_att, s_att=ds_att, w_mid=dw_mid, w_up=dw_up, b_up=db_up,
                 w_down=dw_down, w_out=dw_out, s_out=ds_out, w_end=dw_end)
    clipped, norm = quiver.clip_grad_norm(list(grads.values()), limit)
    return h2, grads, clipped, norm


def _plain_encoder(s):
    """The same encoder in elementary operations, for torch's autograd in 64 bits."""
    def norm(x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w

    b, t, d = s["grad"].shape
    named = s["tok"] >= 0
    x0 = torch.where(named[..., None], s["table"][s["tok"].clamp(min=0)], torch.zeros((), dtype=torch.float64, device=named.device))
    h0 = norm(x0, s["w_in"])
    q, k, v = (p.unflatten(-1, (3, -1)).transpose(1, 2) for p in (h0 @ s["w_qkv"].t()).split(d, -1))
    at = torch.arange(t, device=x0.device)
    live = at[None, :] < s["lengths"][:, None]
    apart = (at[:, None] - at[None, :]).clamp(min=0).double()
    scores = (q @ k.transpose(2, 3).contiguous() * torch.exp(s["decay"].double()[:, None, None] * apart)).tril() * live[:, None, None, :]
    o = (scores @ v.contiguous()).transpose(1, 2).flatten(2) * (d // 3) ** -0.5 * live[..., None]
    x1 = x0 + s["s_att"] * torch.nn.functional.silu(h0 @ s["w_gate"].t()) * norm(o, s["w_att"])
    u = torch.nn.functional.gelu(norm(x1, s["w_mid"]) @ s["w_up"].t() + s["b_up"])
    x2 = x1 + s["s_out"] * norm(u @ s["w_down"].t(), s["w_out"])
    return norm(x2, s["w_end"])


def test_an_encoder_block_trains():
    """One step of a whole block in fp32, by hand and under torch's autograd, against autograd in 64 bits."""
    s = _encoder_state("fp32")
    _say("encoder block")
    h2, grads, clipped, norm = _step(s)
    wide = {k: v.double().requires_grad_(k in grads) if v.is_floating_point() else v for k, v in s.items()}
    out = _plain_encoder(wide)
    names = list(grads)
    want = torch.autograd.grad(out, [wide[k] for k in names], wide["grad"])
    # About forty fp32 products, norms and sums of up to 350 terms follow one another, each off by 512 2^-24 of its size at the
    # most and passed on by factors of a few: 2^-10 of a result's largest element covers them with room.
    assert (h2.double() - out).abs().max() <= 2.0**-10 * out.abs().max()
    for name, g, w in zip(names, grads.values(), want):
        assert (g.double() - w).abs().max() <= 2.0**-10 * w.abs().max(), name
    total = math.sqrt(sum((w ** 2).sum().item() for w in want))
    assert abs(norm.item() - total) <= 2.0**-10 * total
    leaves = {k: v.detach().clone().requires_grad_(k in grads) if v.is_floating_point() else v for k, v in s.items()}
    d = 48
    x0 = quiver.embed(leaves["table"], s["tok"])
    h0 = quiver.block_norm(x0, leaves["w_in"])
    q, k, v = (p.unflatten(-1, (3, -1)) for p in quiver.linear(h0, leaves["w_qkv"]).split(d, -1))
    o = quiver.linear_attention(q, k, v, s["decay"], lengths=s["lengths"]).flatten(2)
    x1, h1 = quiver.block_norm(x0, leaves["w_mid"], y=o, post_weight=leaves["w_att"], gate=quiver.linear(h0, leaves["w_gate"]),
                               gate_activation="silu", scale=leaves["s_att"])
    y1 = quiver.linear(quiver.linear(h1, leaves["w_up"], bias=leaves["b_up"], activation="gelu"), leaves["w_down"])
    _, h2 = quiver.block_norm(x1, leaves["w_end"], y=y1, post_weight=leaves["w_out"], scale=leaves["s_out"])
    got = torch.autograd.grad(h2, [leaves[k] for k in names], s["grad"])
    for name, g, w in zip(names, got, want):
        assert (g.double() - w).abs().max() <= 2.0**-10 * w.abs().max(), name


def test_block_norm_under_backward():
    g = torch.Generator().manual_seed(31)
    _say("block_norm autograd")
    x, w = _randn(g, 6, 40, dtype="fp32"), _randn(g, 40, dtype="fp32")
    parts = _block(g, (6, 40), "fp32")
    cr, ch = _randn(g, 6, 40, dtype="fp32"), _randn(g, 6, 40, dtype="fp32")
    leaves = [t.clone().requires_grad_() for t in (x, w, parts["y"], parts["post_weight"], parts["gate"], parts["scale"])]
    call = lambda x, w, y, p, gate, s: quiver.block_norm(x, w, y=y, post_weight=p, gate=gate, scale=s, gate_activation="sigmoid")  # noqa: E731
    r, h = call(*leaves)
    torch.autograd.backward([r, h], [cr, ch])
    plain = quiver.block_norm_grad(ch, r.detach(), w, grad_r=cr, gate_activation="sigmoid", **parts)
    assert all(torch.equal(t.grad, p) for t, p in zip(leaves, plain))
    r, h = call(*leaves)
    only = torch.autograd.grad(r, leaves[2], cr)[0]  # h unused, one input wanted
    assert torch.equal(only, quiver.block_norm_grad(ch * 0, r.detach(), w, grad_r=cr, gate_activation="sigmoid", **parts)[2])
    gate = leaves[4][:1].detach().requires_grad_()
    r, h = call(*leaves[:4], gate.expand(6, 40), leaves[5])
    shared = torch.autograd.grad(h, gate, ch)[0]
    each = quiver.block_norm_grad(ch, r.detach(), w, gate_activation="sigmoid", **{**parts, "gate": gate.detach().expand(6, 40)})[4]
    assert torch.allclose(shared, each.sum(0, keepdim=True), rtol=1e-5, atol=1e-6)
    h = quiver.block_norm(leaves[0], leaves[1])
    first = torch.autograd.grad(h.sum(), leaves[0], create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiated twice"):
        first.sum().backward()
    with torch.no_grad():
        assert not quiver.block_norm(leaves[0], leaves[1]).requires_grad


def _flat(result):
    return [t for part in result for t in (part.values() if isinstance(part, dict) else part if isinstance(part, list) else [part])]


@pytest.mark.parametrize("dtype", list(TYPES))
def test_calls_follow_the_current_stream_and_repeat(dtype):
    _say("blocks streams", dtype)
    want = _flat(_step(_encoder_state(dtype)))
    assert all(torch.equal(a, b) for a, b in zip(_flat(_step(_encoder_state(dtype))), want))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        later = [t.clone() for t in _flat(_step(_encoder_state(dtype)))]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(later, want))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("texts,tokens", [(3, 5), (2, 700)])
def test_calls_in_graphs(dtype, texts, tokens):
    """Two graphs captured from the same calls, replayed by turns on new inputs with eager work between the replays."""
    _say("blocks graph", dtype, texts, tokens)
    states = [_encoder_state(dtype, texts, tokens, seed) for seed in (0, 1)]
    for s in states:
        _step(s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_flat(_step(s)))
    for seed in (2, 3, 4):
        for i in (0, 1):
            fresh = _encoder_state(dtype, texts, tokens, seed + 10 * i)
            for name, t in fresh.items():
                states[i][name].copy_(t)
            want = _flat(_step(fresh))
            torch.cuda.synchronize()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want)), (seed, i)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_backward_pass_in_a_graph(dtype):
    """Forward and backward captured together, with leaves that no eager graph has seen; replays on new inputs, against eager passes
    on leaves of their own."""
    _gpu()
    _say("autograd graph", dtype)

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        made = {name: _randn(g, 2, 70, 3, 32, dtype=dtype) for name in ("q", "k", "v")}
        made |= {name: _randn(g, 2, 70, 96, dtype=dtype) for name in ("x", "gate", "cr", "ch")}
        made |= {name: _randn(g, 96, dtype=dtype) for name in ("weight", "post", "scale")}
        return made

    decay = torch.tensor([-0.01, -0.1, -1.0], device="cuda")

    def run(s):
        o = quiver.linear_attention(s["q"], s["k"], s["v"], decay).flatten(2)
        r, h = quiver.block_norm(s["x"], s["weight"], y=o, post_weight=s["post"], gate=s["gate"], gate_activation="silu", scale=s["scale"])
        torch.autograd.backward([r, h], [s["cr"], s["ch"]])

    def leaves(s):
        return {name: t.detach().clone().requires_grad_(name not in ("cr", "ch")) for name, t in s.items()}

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        run(leaves(inputs(0)))
    torch.cuda.synchronize()
    held = leaves(inputs(1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(held)
    for seed in (2, 3, 4):
        fresh = leaves(inputs(seed))
        run(fresh)
        with torch.no_grad():
            for name, t in held.items():
                t.copy_(fresh[name])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name, t in held.items():
            assert t.grad is None if name in ("cr", "ch") else torch.equal(t.grad, fresh[name].grad), (seed, name)


def test_a_growing_text_in_a_graph():
    """One token a replay, the state in place."""
    dev = _gpu()
    g = torch.Generator().manual_seed(41)
    _say("attention graph")
    q, k, v = (_randn(g, 2, 20, 4, 32, dtype="bf16") for _ in range(3))
    decay = torch.tensor([-0.1, -0.2, -0.5, 0.0], device=dev)
    now = [t[:, :1].clone() for t in (q, k, v)]
    state = torch.zeros((2, 4, 32, 32), device=dev)
    quiver.linear_attention(*now, decay, state=state, state_out=state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = quiver.linear_attention(*now, decay, state=state, state_out=state)
    state.zero_()
    eager = torch.zeros_like(state)
    for t in range(20):
        for a, b in zip(now, (q, k, v)):
            a.copy_(b[:, t:t + 1])
        want, _ = quiver.linear_attention(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], decay, state=eager, state_out=eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, eager)


def test_allocates_nothing_of_its_own():
    import ctypes as C

    from qvh_ctypes import LIB

    lib = C.CDLL(LIB)
    count = C.c_uint64()
    assert lib.qvh_device_allocations(C.byref(count)) == 0
    before = count.value
    _step(_encoder_state("bf16"))
    assert lib.qvh_device_allocations(C.byref(count)) == 0 and count.value == before
