"""The encoder operators where small shapes do not lead: large tiles, operands in parts, long tables.

Which kernels a shape takes is held by tests/test_encoder_launches.py, on the CPU; the bounds and their derivation are
those of test_encoder_gpu.py.
"""

import math

import pytest

import quiver_amd as quiver
from encoder_paths import GRAD, LINEAR, ORTHO
from test_encoder_gpu import MUON, ROUND, TYPES, _check_linear, _check_linear_grad, _gpu, _randn, _say, _slope64, _within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim", [(30, 50), (300_000, 100), (250_000, 128), (1_000_000, 1)])
def test_embed_grad_without_tokens(dtype, rows, dim):
    """All rows become zero, also in memory that held something else before."""
    _say("embed_grad without tokens", dtype, rows, dim)
    dev = _gpu()
    stale = [torch.full((rows, dim), 7.0, dtype=TYPES[dtype], device=dev) for _ in range(2)]
    del stale  # the allocator hands this memory to the result
    for index in (torch.int64, torch.int32):
        got = quiver.embed_grad(torch.empty((0, dim), dtype=TYPES[dtype], device=dev),
                                torch.empty((0,), dtype=index, device=dev), rows)
        assert got.shape == (rows, dim) and not got.any()


@pytest.mark.parametrize("count", [0, 10])
def test_embed_grad_of_more_than_2_30_rows(count):
    """More rows than there are work-groups to clear them."""
    _say("embed_grad of 2^30 rows", count)
    rows = 2**30 + 70
    out = quiver.embed_grad(torch.ones((count, 1), dtype=torch.bfloat16, device=_gpu()),
                            torch.arange(count, device=_gpu()) * (rows // 10) + 69, rows)
    named = torch.arange(count, device=_gpu()) * (rows // 10) + 69
    assert bool((out[named] == 1).all())
    out[named] = 0
    assert not out.any()


def test_embed_of_more_than_one_launch():
    """A result of 2^33 pieces and more."""
    _say("embed of more than one launch")
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 200 << 30:
        pytest.skip("needs 150 GB of GPU memory")
    dim, count = 1024, 2**26 + 2_000_003
    table = _randn(torch.Generator().manual_seed(1), 997, dim, dtype="bf16")
    tok = torch.arange(count, device=_gpu(), dtype=torch.int32) % 997
    got = quiver.embed(table, tok)
    for at in (0, 2**25 - 5, 2**26 - 5, 2**26 + 1_000_000, count - 1000):
        s = slice(at, at + 1000)
        assert torch.equal(got[s], table[tok[s].long()])
    del got
    torch.cuda.empty_cache()


# ---- every tile, every way of reading, whole and in splits --------------------------------------


def _each(shapes):
    return [(dtype, *shape) for dtype in TYPES for shape in shapes["bf16" if dtype == "fp16" else dtype]]


@pytest.mark.parametrize("dtype,m,k,n", _each(LINEAR))
def test_linear_by_every_kernel(dtype, m, k, n):
    g = torch.Generator().manual_seed(m + k + n)
    _say("linear paths", dtype, m, k, n)
    x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype, std=1 / math.sqrt(k))
    _check_linear(dtype, x, w, _randn(g, n, dtype=dtype), "gelu", _randn(g, m, n, dtype=dtype))
    _check_linear(dtype, x, w, None, "none", None)


@pytest.mark.parametrize("dtype,m,k,n", _each(GRAD))
def test_linear_grad_by_every_kernel(dtype, m, k, n):
    g = torch.Generator().manual_seed(m + k + n)
    _say("linear_grad paths", dtype, m, k, n)
    x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype, std=1 / math.sqrt(k))
    gr, pre = _randn(g, m, n, dtype=dtype), _randn(g, m, n, dtype=dtype, std=2.0)
    _check_linear_grad(dtype, gr, x, w, pre, "gelu")
    _check_linear_grad(dtype, gr, x, w, None, "none")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_layers_of_strided_rows(dtype):
    """Views with a stride, at and off 16-byte addresses, of a size that takes large tiles and fp32 parts."""
    g = torch.Generator().manual_seed(12)
    _say("large views", dtype)
    m, k, n = 2100, 520, 2050
    x, w = _randn(g, m, k + 24, dtype=dtype), _randn(g, n, k + 24, dtype=dtype, std=1 / math.sqrt(k))
    gr, pre = _randn(g, m, n + 16, dtype=dtype), _randn(g, m, n + 16, dtype=dtype, std=2.0)
    for at in (0, 8, 3):
        s, t = slice(at, at + k), slice(at, at + n)
        _check_linear(dtype, x[:, s], w[:, s], None, "silu", gr[:, t])
        _check_linear_grad(dtype, gr[:, t], x[:, s], w[:, s], pre[:, t], "silu")


def _ortho64_by_products(u, steps, co):
    """The recurrence itself in 64 bits on the side with fewer rows, and the growth of an error (as _ortho64's, over
    all singular values that occur: from 0 to the largest that the values of [0, 1] can reach)."""
    a, b, c = co
    x = u.double().reshape(-1, *u.shape[-2:])
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    x = x / x.flatten(1).norm(dim=1)[:, None, None]
    grow, top = 1.0, 1.0
    for _ in range(steps):
        t = torch.linspace(0, top, 500, dtype=torch.float64)
        grow *= max(1.0, (a + 3 * b * t**2 + 5 * c * t**4).abs().max().item(), (a + b * t**2 + c * t**4).abs().max().item())
        top = (a * t + b * t**3 + c * t**5).abs().max().item()
        s = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * s + c * torch.bmm(s, s), x)
    return (x.transpose(1, 2) if tall else x).reshape(u.shape), grow


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,batch", ORTHO)
def test_orthogonalize_by_every_kernel(dtype, m, n, batch):
    g = torch.Generator().manual_seed(m + n + batch)
    _say("orthogonalize paths", dtype, m, n, batch)
    u = _randn(g, batch, m, n, dtype=dtype, std=1e-3)
    side, depth = min(m, n), max(m, n)
    for steps in (5, 2):
        got = quiver.orthogonalize(u, steps=steps)
        want, grow = _ortho64_by_products(u, steps, MUON)
        bound = grow * (steps + 1) * 2 * math.sqrt(depth) * 2.0**-22 * math.sqrt(side)  # as in test_orthogonalize
        err = (got.double() - want).flatten(-2).norm(dim=-1)
        size = want.flatten(-2).norm(dim=-1)
        assert bool((err <= bound + ROUND[dtype] * size).all()), (steps, err.max().item(), bound)
        assert torch.equal(got, quiver.orthogonalize(u, steps=steps))


# ---- fp32 operands in three parts ---------------------------------------------------------------

PARTS = (2100, 520, 2050)  # forwards and backwards


def _single_products(g):
    """x, w with one non-zero value in each row of w: every result is one product."""
    m, k, n = PARTS
    x = 1.0 + torch.randint(0, 2**23, (m, k), generator=g).double() * 2.0**-23  # all 24 bits
    w = torch.zeros((n, k), dtype=torch.float64)
    w[torch.arange(n), torch.arange(n) * 7 % k] = 1.0 + torch.randint(0, 2**23, (n,), generator=g).double() * 2.0**-23
    return x.float().to(_gpu()), w.float().to(_gpu())


def test_parts_hold_24_bits():
    """One product per result: what the parts leave out is below 2^-25 of it and its six terms are added with at most
    2^-23 of the sum each, 2^-20 altogether. A third part left out would show: it is up to 2^-18 of a value."""
    _say("parts", *PARTS)
    g = torch.Generator().manual_seed(31)
    x, w = _single_products(g)
    want = x.double() @ w.double().t()
    assert ((quiver.linear(x, w).double() - want).abs() <= 2.0**-20 * want.abs()).all()
    for size in (2.0**-100, 2.0**100):  # the range that the parts hold
        assert ((quiver.linear(x * size, w / size).double() - want).abs() <= 2.0**-20 * want.abs()).all()
    # Backwards: one non-zero value per row of the gradient for grad_x, per column for grad_weight.
    m, k, n = PARTS
    gr = torch.zeros((m, n), device=_gpu())
    gr[torch.arange(m), torch.randperm(n, generator=g)[torch.arange(m) % n]] = x[:, 0]
    dx, dw, _ = quiver.linear_grad(gr, x, w + 1.0)
    want = gr.double() @ (w + 1.0).double()
    assert ((dx.double() - want).abs() <= 2.0**-20 * want.abs()).all()
    # A column of the gradient holds one value, or two where n < m: their products do not cancel.
    want = gr.double().t() @ x.double()
    assert ((dw.double() - want).abs() <= 2.0**-20 * want.abs()).all()


def test_parts_of_small_and_large_values():
    """Rows and columns of very different size, and values whose first part would round up to infinity."""
    _say("parts range")
    m, k, n = PARTS
    g = torch.Generator().manual_seed(8)
    x = _randn(g, m, k, dtype="fp32") * torch.logspace(-15, 15, m, device=_gpu())[:, None]
    w = _randn(g, n, k, dtype="fp32") * torch.logspace(-12, 12, k, device=_gpu())[None, :]
    _check_linear("fp32", x, w, None, "none", None)
    gr = _randn(g, m, n, dtype="fp32") * torch.logspace(-8, 8, n, device=_gpu())[None, :]
    _check_linear_grad("fp32", gr, x, w, None, "none")
    big, half = torch.zeros((m, k), device=_gpu()), torch.zeros((n, k), device=_gpu())
    big[:, 3], half[:, 3] = 3.402e38, 0.5
    assert torch.equal(quiver.linear(big, half), torch.full((m, n), 1.701e38, device=_gpu()))
    gr = torch.zeros((m, n), device=_gpu())
    gr[:, 5] = 3.402e38
    dx, dw, _ = quiver.linear_grad(gr, torch.zeros((m, k), device=_gpu()).index_fill_(0, torch.tensor([9], device=_gpu()), 0.5), half)
    assert torch.equal(dx[:, 3], torch.full((m,), 1.701e38, device=_gpu())) and not dx[:, :3].any() and not dx[:, 4:].any()
    assert torch.equal(dw[5], torch.full((k,), 1.701e38, device=_gpu())) and not dw[:5].any() and not dw[6:].any()


def _same_specials(got, want):
    """NaN and infinities in the same places, of the same sign."""
    want = want.to(got.dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]) and torch.equal(torch.isinf(got), torch.isinf(want))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_layers_of_not_finite_values(dtype):
    """As test_linear_not_finite, at a size that takes parts in fp32, and backwards."""
    _say("large not finite", dtype)
    m, k, n = PARTS
    g = torch.Generator().manual_seed(3)
    x, w = _randn(g, m, k, dtype=dtype), torch.ones((n, k), dtype=TYPES[dtype], device=_gpu())
    x[1, 5], x[2, 7], x[3, 0], x[m - 1, k - 1] = float("inf"), float("nan"), -float("inf"), float("inf")
    w[9] = 0.0
    w[9, 5] = 2.0
    w[11, 3] = float("inf")
    w[n - 1, k - 1] = -1.0
    _same_specials(quiver.linear(x, w), x.double() @ w.double().t())
    gr, pre = _randn(g, m, n, dtype=dtype), _randn(g, m, n, dtype=dtype)
    gr[4, 6], gr[5, n - 1], gr[m - 1, 0] = float("inf"), float("nan"), -float("inf")
    for act in ("none", "silu"):
        dx, dw, db = quiver.linear_grad(gr, x, w, preactivation=pre, activation=act)
        dz = gr.double() * _slope64(pre.double(), act)
        _same_specials(dx, dz @ w.double())
        _same_specials(dw, dz.t() @ x.double())
        _same_specials(db, dz.sum(0))


# ---- activations by themselves ------------------------------------------------------------------


def _through(z, act):
    """act(z) and its slope at z, by a layer and a gradient of one product with 1."""
    one = torch.ones((1, 1), dtype=z.dtype, device=z.device)
    y = quiver.linear(z[:, None], one, activation=act)
    slope, _, _ = quiver.linear_grad(torch.ones_like(z)[:, None], z[:, None], one, preactivation=z[:, None], activation=act)
    return y[:, 0].double(), slope[:, 0].double()


@pytest.mark.parametrize("count", [40, 20_000])
def test_fp32_silu_is_good_to_its_last_bits(count):
    """The exponential, a sum, a quotient and a product: 8 roundings of 2^-24 at most, whatever the size of z, and 16 of the
    slope's terms; below that the smallest normal number times z."""
    _say("silu fp32", count)
    z = torch.cat([torch.linspace(-100, 100, count - 8), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 700.0, -700.0, 3e38, -3e38])]).to(_gpu())
    y, slope = _through(z, "silu")
    zd = z.double()
    s, q = torch.sigmoid(zd), torch.sigmoid(-zd)
    tiny = (1 + zd.abs().clamp(max=1e3)) * 2.0**-126
    _within(y, zd * s, (zd * s).abs() * 2.0**-21 + tiny)
    _within(slope, s * (1 + zd * q), s * (1 + zd.abs() * q) * 2.0**-20 + tiny)


@pytest.mark.parametrize("act", ["gelu", "silu", "relu"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_activations_of_not_finite_values(dtype, act):
    """What the formulas give: infinity and NaN go through; -infinity is 0 for ReLU and infinity times 0 for the others."""
    _say("activations not finite", dtype, act)
    z = torch.tensor([float("inf"), -float("inf"), float("nan")] * 20, dtype=TYPES[dtype], device=_gpu())
    y, _ = _through(z, act)
    assert bool((y[0::3] == float("inf")).all()) and bool(torch.isnan(y[2::3]).all())
    assert bool((y[1::3] == 0).all()) if act == "relu" else bool(torch.isnan(y[1::3]).all())


def test_fp32_gelu_slope():
    """Phi to 2^-23; z phi(z) to 8 roundings and that of z^2 in the exponent, 2^-24 of it."""
    _say("gelu slope fp32")
    z = torch.linspace(-15, 15, 30_001).to(_gpu())
    _, slope = _through(z, "gelu")
    zd = z.double()
    term = zd * torch.exp(-0.5 * zd * zd) / math.sqrt(2 * math.pi)
    _within(slope, torch.special.ndtr(zd) + term, 2.0**-23 + term.abs() * (zd * zd + 8) * 2.0**-24)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_16_bit_gelu_is_rounded_once(dtype):
    """Every number of the type from -9 to 9: half of the spacing of numbers at the result, and what the fp32 evaluation may
    leave before that. It has 1.7e-8 from the fit of the normal tail, and 5 + 3 roundings of values below 0.6, so less
    than 2^-23 for GELU; its slope has two such terms, and Phi's rounding: 2^-22."""
    _say("gelu 16 bit", dtype)
    z = torch.arange(-2**15, 2**15, dtype=torch.int32).to(torch.int16).view(TYPES[dtype])
    z = z[torch.isfinite(z) & (z.abs() <= 9)].to(_gpu())
    bits, least = (11, -24) if dtype == "fp16" else (8, -133)
    half = lambda v: 0.5 * torch.exp2((torch.floor(torch.log2(v.abs().clamp(min=1e-300))) - bits + 1).clamp(min=least))  # noqa: E731
    y, slope = _through(z, "gelu")
    zd = z.double()
    want = zd * torch.special.ndtr(zd)
    assert ((y - want).abs() <= half(want.abs() + 2.0**-23) + 2.0**-23).all(), ((y - want).abs() - half(want)).max().item()
    want = torch.special.ndtr(zd) + zd * torch.exp(-0.5 * zd * zd) / math.sqrt(2 * math.pi)
    assert ((slope - want).abs() <= half(want.abs() + 2.0**-22) + 2.0**-22).all(), ((slope - want).abs() - half(want)).max().item()


def test_parts_that_overflow():
    """Finite values whose products are past fp32: their parts overflow both ways, the results are infinite on the side of the
    true sum, and finite sums of them finite."""
    _say("parts overflow")
    m, k, n = PARTS
    g = torch.Generator().manual_seed(14)
    x, w = _randn(g, m, k, dtype="fp32"), _randn(g, n, k, dtype="fp32")
    x[7] *= 1e30  # with w below: sums of 1e40 and more, of either sign
    w[5] *= 1e10
    x[9], w[3] = 0.0, 0.0
    x[9, 100], x[9, 101], w[3, 100], w[3, 101] = 3.3e38, -3.3e38, 1.25e5, 1.25e5  # 4e43 - 4e43
    x[11], w[1] = 0.0, 0.0
    x[11, 33], w[1, 33] = 3.4e38, -3.3e5
    want = x.double() @ w.double().t()
    got = quiver.linear(x, w)
    assert torch.equal(got[7, 5].double(), want[7, 5].sign() * math.inf) and abs(want[7, 5]) > 1e39
    assert got[11, 1] == -math.inf
    assert got[9, 3] == 0 or torch.isnan(got[9, 3])  # in fp32 arithmetic, infinity minus infinity
    plain = torch.ones(m, dtype=torch.bool, device=_gpu()).index_fill_(0, torch.tensor([7, 9, 11], device=_gpu()), False)
    others = torch.ones(n, dtype=torch.bool, device=_gpu()).index_fill_(0, torch.tensor([5, 3, 1], device=_gpu()), False)
    keep = plain[:, None] & others[None, :]
    bound = (x.double().abs() @ w.double().abs().t()) * (k + 8) * 2.0**-23
    assert (((got.double() - want).abs() <= bound + want.abs() * 2.0**-24) | ~keep).all()


def test_infinities_do_not_stall_a_large_layer():
    """One in each row makes every result of parts NaN at first, to be made again. That may take a second product that waits for
    every load, some twenty times as long as the first; a hundred times would be a loop over single elements."""
    _say("infinities' time")
    m, k, n = 4096, 1024, 1024
    g = torch.Generator().manual_seed(13)
    x, w, gr = _randn(g, m, k, dtype="fp32"), _randn(g, n, k, dtype="fp32"), _randn(g, m, n, dtype="fp32")

    def ms(call):
        best = math.inf
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    layer, grad = lambda: quiver.linear(x, w), lambda: quiver.linear_grad(gr, x, w)  # noqa: E731
    layer(), grad()
    before = ms(layer), ms(grad)
    x[torch.arange(m), torch.randint(0, k, (m,), generator=g)] = float("inf")
    after = ms(layer), ms(grad)
    print("ms without and with infinities:", before, after, flush=True)
    _same_specials(layer(), x.double() @ w.double().t())
    _same_specials(grad()[1], gr.double().t() @ x.double())
    assert after[0] < 40 * before[0] and after[1] < 40 * before[1]
