"""The encoder's calls on tensors that require gradients: torch's own backward pass, and what has no derivative says so."""

import math

import pytest

import quiver_amd as quiver
from test_encoder_gpu import TYPES, _act64, _gpu, _randn, _say, _slope64, _within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _leaf(t):
    return t.clone().requires_grad_()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_linear_under_backward(dtype, act):
    """The same bits as linear_grad's, for each input that asks for them."""
    _say("linear backward", dtype, act)
    g = torch.Generator().manual_seed(1)
    x, w, b = _randn(g, 7, 50, 36, dtype=dtype), _randn(g, 72, 36, dtype=dtype, std=0.2), _randn(g, 72, dtype=dtype)
    r, up = _randn(g, 7, 50, 72, dtype=dtype), _randn(g, 7, 50, 72, dtype=dtype)
    plain, pre = quiver.linear(x, w, bias=b, activation=act, residual=r, keep_preactivation=True)
    want = quiver.linear_grad(up, x, w, preactivation=pre, activation=act)
    args = [_leaf(t) for t in (x, w, b, r)]
    y = quiver.linear(args[0], args[1], bias=args[2], activation=act, residual=args[3])
    assert y.requires_grad and torch.equal(y, plain)
    y.backward(up)
    assert all(torch.equal(t.grad, v) for t, v in zip(args, (*want, up)))
    for only in range(4):  # one at a time
        one = [_leaf(t) if i == only else t for i, t in enumerate((x, w, b, r))]
        quiver.linear(one[0], one[1], bias=one[2], activation=act, residual=one[3]).backward(up)
        assert torch.equal(one[only].grad, (*want, up)[only])
    # A broadcast gradient, as of a sum, and a layer without bias.
    args = [_leaf(t) for t in (x, w)]
    quiver.linear(*args, activation=act).sum().backward()
    _, pre = quiver.linear(x, w, activation=act, keep_preactivation=True)
    want = quiver.linear_grad(torch.ones_like(up), x, w, preactivation=pre, activation=act, bias=False)
    assert all(torch.equal(t.grad, v) for t, v in zip(args, want))


@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
def test_linear_under_backward_with_its_preactivation(act):
    """A loss of both results in fp32 against 64 bits: gradient dz = gy act'(z) + gz. The kept z is off by (k + 9) 2^-23 of its
    terms, which moves the slope by 1.2 of that; the slope is good to 2^-19, the sums to (terms + 10) 2^-23 of theirs, two
    of which are added."""
    _say("pre-activation backward", act)
    g = torch.Generator().manual_seed(2)
    m, k, n = 60, 40, 30
    x, w, b = _randn(g, m, k, dtype="fp32"), _randn(g, n, k, dtype="fp32", std=0.3), _randn(g, n, dtype="fp32")
    gy, gz = _randn(g, m, n, dtype="fp32"), _randn(g, m, n, dtype="fp32")
    for use_y, use_z in ((True, True), (False, True), (True, False)):
        args = [_leaf(t) for t in (x, w, b)]
        y, z = quiver.linear(args[0], args[1], bias=args[2], activation=act, keep_preactivation=True)
        assert y.requires_grad and z.requires_grad
        ((y * gy).sum() * use_y + (z * gz).sum() * use_z).backward()
        xd, wd = x.double(), w.double()
        z64 = xd @ wd.t() + b.double()
        zb = (xd.abs() @ wd.abs().t() + b.double().abs()) * (k + 9) * 2.0**-23
        dz = use_y * gy.double() * _slope64(z64, act) + use_z * gz.double()
        ze = use_y * gy.double().abs() * (1.2 * zb + 2.0**-19)
        size = use_y * 1.2 * gy.double().abs() + use_z * gz.double().abs()
        _within(args[0].grad, dz @ wd, ze @ wd.abs() + size @ wd.abs() * (n + 10) * 2.0**-23, "x")
        _within(args[1].grad, dz.t() @ xd, ze.t() @ xd.abs() + size.t() @ xd.abs() * (m + 10) * 2.0**-23, "weight")
        _within(args[2].grad, dz.sum(0), ze.sum(0) + size.sum(0) * (m + 10) * 2.0**-23, "bias")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_embed_under_backward(dtype):
    _say("embed backward", dtype)
    g = torch.Generator().manual_seed(3)
    table, up = _randn(g, 90, 24, dtype=dtype), _randn(g, 40, 5, 24, dtype=dtype)
    tok = torch.randint(-1, 90, (40, 5), generator=g).to(_gpu())
    t = _leaf(table)
    y = quiver.embed(t, tok, scale=3.0)
    assert y.requires_grad and torch.equal(y, quiver.embed(table, tok, scale=3.0))
    y.backward(up)
    assert torch.equal(t.grad, quiver.embed_grad(up, tok, 90, scale=3.0))


def test_a_small_encoder_trains_by_backward():
    """Parameters, an optimiser and a loss of torch's own: table and layers learn to tell two kinds of text apart."""
    _say("training by backward")
    g = torch.Generator().manual_seed(4)
    table, w0, w1 = (torch.nn.Parameter(_randn(g, *s, dtype="fp32", std=0.3)) for s in ((50, 16), (32, 16), (2, 32)))
    tok = torch.randint(0, 50, (256, 6), generator=g).to(_gpu())
    kind = (tok % 2).sum(1) > 3
    best = torch.optim.Adam([table, w0, w1], lr=0.02)
    losses = []
    for _ in range(150):
        h = quiver.linear(quiver.embed(table, tok), w0, activation="gelu").mean(1)
        loss = torch.nn.functional.cross_entropy(quiver.linear(h, w1), kind.long())
        best.zero_grad()
        loss.backward()
        best.step()
        losses.append(loss.item())
    assert losses[-1] < 0.5 * losses[0]


def test_nothing_is_recorded_where_nothing_asks():
    _say("no graph")
    g = torch.Generator().manual_seed(5)
    x, w = _randn(g, 9, 16, dtype="fp32"), _leaf(_randn(g, 8, 16, dtype="fp32"))
    tok = torch.zeros(3, dtype=torch.int64, device=_gpu())
    with torch.no_grad():
        assert not quiver.linear(x, w).requires_grad and not quiver.embed(w, tok).requires_grad
        assert not quiver.orthogonalize(w).requires_grad
    assert not quiver.linear(x, w.detach()).requires_grad and not quiver.embed(w.detach(), tok).requires_grad
    # The gradients' own results are constants, as those of torch's backward pass are.
    assert not any(t.requires_grad for t in quiver.linear_grad(x[:, :8], x, w))


def test_what_has_no_derivative_says_so():
    _say("no derivative")
    g = torch.Generator().manual_seed(6)
    x, w = _leaf(_randn(g, 9, 16, dtype="fp32")), _leaf(_randn(g, 8, 16, dtype="fp32"))
    u = quiver.orthogonalize(w)
    assert u.requires_grad
    with pytest.raises(RuntimeError, match="orthogonalize"):
        u.sum().backward()
    y = quiver.linear(x, w, activation="gelu")
    first, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        first.sum().backward()
    import torch.autograd.forward_ad as fwd

    tok = torch.zeros(3, dtype=torch.int64, device=_gpu())
    with fwd.dual_level():
        dual = fwd.make_dual(w.detach(), torch.ones_like(w))
        for call in (lambda: quiver.linear(x.detach(), dual), lambda: quiver.embed(dual, tok), lambda: quiver.orthogonalize(dual)):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        assert quiver.linear(x.detach(), w.detach()).shape == (9, 8)
