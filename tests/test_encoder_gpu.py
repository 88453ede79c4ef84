"""The encoder operators (embedding lookup and gradient, linear layers and their gradients, orthogonalised
updates) against 64-bit arithmetic.

Tolerances come from the arithmetic. u is the unit roundoff of the result's type (2^-24, 2^-11, 2^-8);
fp32 sums of K terms are off by at most K 2^-23 of the sum of their magnitudes, whatever the order and the
rounding of the matrix unit; every elementwise bound here is the sum of such terms.
"""

import math

import numpy as np
import pytest

import quiver_amd as quiver

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ROUND = {"fp32": 2.0**-24, "fp16": 2.0**-11, "bf16": 2.0**-8}
TINY = {"fp32": 2.0**-126, "fp16": 2.0**-24, "bf16": 2.0**-126}  # absolute error of the smallest results


def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible to torch")
    return torch.device("cuda", quiver._quiver._device_index())


def _say(*what):
    print("case:", *what, flush=True)


def _randn(g, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(TYPES[dtype]).to(_gpu())


def _within(got, want, bound, what=""):
    """Every element: |got - want| <= bound, NaN and infinities in the same places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)]), what
    over = ((got - want).abs() - bound)[finite]
    assert over.numel() == 0 or over.max().item() <= 0, f"{what}: {over.max().item():.3g} past the bound"


# ---- embedding lookup -------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim,shape", [(100, 768, (24,)), (1000, 100, (3, 7)), (50, 1, (1,)), (333, 33, (1000,)),
                                            (7, 6, (5, 1, 2)), (2000, 1025, (70,)), (70_000, 16, (300_000,)), (10, 32_768, (9,))])
def test_embed(dtype, rows, dim, shape):
    g = torch.Generator().manual_seed(rows + dim)
    _say("embed", dtype, rows, dim, shape)
    table = _randn(g, rows, dim, dtype=dtype)
    table[0] = float("nan")  # padding must not read row 0 into its zeros
    for index in (torch.int64, torch.int32):
        tok = torch.randint(-2, rows + 2, shape, generator=g).to(index).to(_gpu())
        tok.view(-1)[-1] = rows - 1
        got = quiver.embed(table, tok, scale=2.5)
        assert got.shape == shape + (dim,) and got.dtype == table.dtype
        named = (tok >= 0) & (tok < rows)
        want = torch.where(named[..., None], table[tok.clamp(0, rows - 1).long()].double() * 2.5, 0.0)
        # One multiplication in fp32 and one rounding to the type.
        _within(got, want, want.abs() * (ROUND[dtype] + 2.0**-24) + TINY[dtype])
        kept = named & (tok != 0)
        assert torch.equal(quiver.embed(table, tok)[kept], table[tok[kept].long()])  # scale 1 changes nothing


def test_embed_strided_misaligned_and_empty():
    dev = _gpu()
    _say("embed strided")
    big = torch.arange(50 * 41, device=dev, dtype=torch.float32).reshape(50, 41)
    tok = torch.tensor([3, -1, 49, 0], device=dev)
    zero = torch.zeros(1, device=dev)
    for table in (big[:, 1:34], big[:, :33], big[::2][:, 5:8], big.t(), big.half()[:, 1:17]):
        want = torch.where((tok >= 0)[:, None] & (tok < len(table))[:, None], table[tok.clamp(0, len(table) - 1)],
                           zero.to(table.dtype))
        assert torch.equal(quiver.embed(table, tok), want)
    assert torch.equal(quiver.embed(big, tok[::2]), big[tok[::2]])  # strided tokens
    assert quiver.embed(big, tok[:0]).shape == (0, 41)
    assert quiver.embed(big, tok[:0].reshape(2, 0)).shape == (2, 0, 41)
    assert not quiver.embed(big[:0], tok).any()  # a table without rows
    assert torch.equal(quiver.embed(big, torch.tensor(7, device=dev)), big[7])
    far = torch.tensor([2**40, -(2**40), 2**32 + 3, 2**63 - 1, -(2**63)], device=dev)
    assert not quiver.embed(big, far).any()


def test_embed_past_32_bit_offsets():
    dev = _gpu()
    rows, dim = 2_200_001, 1_024  # 4.5e9 bytes
    _say("embed", rows, dim)
    table = torch.empty((rows, dim), dtype=torch.bfloat16, device=dev)
    table.random_(-100, 100)
    tok = torch.tensor([rows - 1, 2_097_152, 2_097_151, 0, rows], device=dev)
    got = quiver.embed(table, tok)
    assert torch.equal(got[:4], table[tok[:4]]) and not got[4].any()


# ---- embedding gradient -----------------------------------------------------------------------


def _embed_grad_64(grad, tok, rows, scale):
    """Value and sum of magnitudes."""
    ok = (tok >= 0) & (tok < rows)
    gd, t = grad[ok].double().reshape(-1, grad.shape[-1]), tok[ok].long()
    out = torch.zeros((2, rows, grad.shape[-1]), dtype=torch.float64, device=grad.device)
    out[0].index_add_(0, t, gd)
    out[1].index_add_(0, t, gd.abs())
    return out[0] * scale, out[1] * abs(scale), torch.bincount(t, minlength=rows)


def _check_embed_grad(grad, tok, rows, dtype, scale=1.0):
    got = quiver.embed_grad(grad, tok, rows, scale=scale)
    want, size, count = _embed_grad_64(grad, tok, rows, scale)
    bound = size * ((count + 2) * 2.0**-23)[:, None] + want.abs() * ROUND[dtype] + TINY[dtype]
    _within(got, want, bound)
    assert not got[count == 0].any()
    assert torch.equal(got, quiver.embed_grad(grad, tok, rows, scale=scale))  # the same bits again
    return got


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim,count", [
    (1000, 128, 1), (1000, 128, 63), (10, 100, 2048), (10_000, 100, 2049), (1, 64, 5000), (5, 33, 4096), (300, 1025, 2500),
    (70_000, 40, 20_000), (100_000, 7, 130_000), (256, 8, 3000), (255, 16, 3000), (65_535, 16, 3000), (65_536, 24, 3000),
    (2_000_000, 12, 70_001), (17, 520, 64 * 64)])
def test_embed_grad(dtype, rows, dim, count):
    g = torch.Generator().manual_seed(rows + dim + count)
    _say("embed_grad", dtype, rows, dim, count)
    grad = _randn(g, count, dim, dtype=dtype)
    tok = torch.randint(-1, rows + 1, (count,), generator=g).to(_gpu())
    _check_embed_grad(grad, tok, rows, dtype, scale=0.5)
    _check_embed_grad(grad, tok.int(), rows, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim,count", [
    (1000, 64, 2048), (3000, 768, 300), (3000, 768, 1000), (32_000, 1024, 512), (300_000, 100, 100), (200, 512, 2047),
    (65_536, 3, 40), (1, 1, 2048), (255, 9, 1900)])
def test_embed_grad_of_small_batches(dtype, rows, dim, count):
    """Either side of the choice between rows that look for their tokens and sorted tokens, frequent tokens first."""
    g = torch.Generator().manual_seed(rows + dim + count)
    _say("embed_grad small", dtype, rows, dim, count)
    grad = _randn(g, count, dim, dtype=dtype)
    tok = (torch.exp(torch.rand(count, generator=g, dtype=torch.float64) * math.log(rows + 1.0)) - 1).long().clamp(0, rows - 1)
    _check_embed_grad(grad, tok.to(_gpu()), rows, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim,count", [(5000, 201, 90_000), (300, 64, 300_001)])
def test_embedding_of_large_batches(dtype, rows, dim, count):
    """More than 32 MB of gradients and of looked-up rows, odd rows among them."""
    test_embed_grad(dtype, rows, dim, count)
    g = torch.Generator().manual_seed(rows)
    table = _randn(g, rows, dim, dtype=dtype)
    tok = torch.randint(-1, rows, (count,), generator=g).to(_gpu())
    want = torch.where(tok[:, None] >= 0, table[tok.clamp(min=0)], torch.zeros((), dtype=TYPES[dtype], device=_gpu()))
    assert torch.equal(quiver.embed(table, tok), want)


@pytest.mark.parametrize("dim", [1, 30, 300])
def test_embed_grad_joins_short_and_long_runs(dim):
    """Runs of 1 to 4,000 tokens, so that some end in their piece, some in the next ones and some far behind."""
    _say("embed_grad joins", dim)
    g = torch.Generator().manual_seed(dim)
    lengths = [1, 4000, 15, 16, 17, 1, 250, 256, 260, 272, 3, 31, 32, 33, 2000, 700, 8, 8, 8]
    tok = torch.repeat_interleave(torch.arange(len(lengths)) * 3, torch.tensor(lengths))
    tok = tok[torch.randperm(len(tok), generator=g)].to(_gpu())
    _check_embed_grad(_randn(g, len(tok), dim, dtype="fp32"), tok, 60, "fp32")


@pytest.mark.parametrize("count", [700, 2048, 6400, 6401, 50_000])
@pytest.mark.parametrize("kind", ["one token", "two tokens", "blocks", "padding", "falling", "last row"])
def test_embed_grad_runs(kind, count):
    """Runs of equal tokens that fill many pieces of the sorted list, end at a piece's edge, or are all there is."""
    _say("embed_grad runs", kind, count)
    g = torch.Generator().manual_seed(count)
    rows, dim = 500, 68
    i = torch.arange(count)
    tok = {"one token": torch.full((count,), 77), "two tokens": torch.where(i % 3 == 0, 12, 11), "blocks": i // 64 % rows,
           "padding": torch.full((count,), -1), "falling": (rows - 1 - i * 7 % rows), "last row": torch.full((count,), rows - 1)}[kind]
    grad = _randn(g, count, dim, dtype="fp32")
    _check_embed_grad(grad, tok.to(_gpu()), rows, "fp32")


def test_embed_grad_shapes_and_strides():
    dev = _gpu()
    _say("embed_grad strided")
    g = torch.Generator().manual_seed(5)
    big = _randn(g, 4000, 50, dtype="bf16")
    tok = torch.randint(0, 30, (4000,), generator=g).to(dev)
    _check_embed_grad(big[:, 3:40], tok, 30, "bf16")
    _check_embed_grad(big.t().contiguous().t(), tok, 30, "bf16")
    assert torch.equal(quiver.embed_grad(big.reshape(40, 100, 50), tok.reshape(40, 100), 30), quiver.embed_grad(big, tok, 30))
    assert quiver.embed_grad(big, tok, 0).shape == (0, 50)
    assert not quiver.embed_grad(big[:0], tok[:0], 30).any()
    wide = torch.full((3000, 8), float("inf"), device=dev)  # what padding carries goes nowhere
    pad = torch.where(torch.arange(3000, device=dev) < 10, 4, -1)
    wide[:10] = 1.0
    assert torch.equal(quiver.embed_grad(wide, pad, 9)[4], torch.full((8,), 10.0, device=dev))


def test_embed_grad_past_32_bit_offsets():
    dev = _gpu()
    rows, dim = 2_200_001, 1_024
    _say("embed_grad", rows, dim)
    tok = torch.tensor([rows - 1, 3, rows - 1, 2_097_152], device=dev).repeat(1000)
    grad = torch.ones((4000, dim), dtype=torch.bfloat16, device=dev)
    got = quiver.embed_grad(grad, tok, rows)
    assert bool((got[rows - 1] == 2000).all()) and bool((got[3] == 1000).all()) and bool((got[2_097_152] == 1000).all())
    assert not got[4:2_097_152].any() and not got[2_097_153:rows - 1].any()


def test_embed_grad_is_the_lookups_derivative():
    """<embed(E + h D) - embed(E - h D), G> / 2h against <embed_grad(G), D>: the lookup is linear, so only
    rounding separates them (4096 products of fp32 results, each off by 2^-24 of values below 6)."""
    _say("embed difference")
    g = torch.Generator().manual_seed(11)
    table, d = _randn(g, 200, 64, dtype="fp32"), _randn(g, 200, 64, dtype="fp32")
    tok = torch.randint(-1, 200, (64,), generator=g).to(_gpu())
    up = _randn(g, 64, 64, dtype="fp32")
    h = 0.25
    diff = ((quiver.embed(table + h * d, tok, 3.0).double() - quiver.embed(table - h * d, tok, 3.0).double()) * up).sum() / (2 * h)
    exact = (quiver.embed_grad(up, tok, 200, 3.0).double() * d).sum()
    bound = 4096 * 6 * 3 * 4 * 2.0**-23 / h
    assert abs(diff - exact).item() <= bound


# ---- linear -----------------------------------------------------------------------------------


def _act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * torch.special.ndtr(z),
            "silu": lambda: z * torch.sigmoid(z)}[act]()


def _slope64(z, act):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(),
            "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi),
            "silu": lambda: s * (1 + z * (1 - s))}[act]()


def _product_bound(a, b, k):
    """fp32 sum of k products (and, for fp32 operands, the parts left out)."""
    return (a.abs() @ b.abs()) * ((k + 8) * 2.0**-23)


def _check_linear(dtype, x, w, b, act, r):
    k = x.shape[-1]
    got, pre = quiver.linear(x, w, bias=b, activation=act, residual=r, keep_preactivation=True)
    xd, wd = x.double().reshape(-1, k), w.double()
    z = xd @ wd.t()
    zb = _product_bound(xd, wd.t(), k)
    if b is not None:
        z = z + b.double()
        zb = zb + b.double().abs() * 2.0**-23
    z, zb = z.reshape(got.shape), zb.reshape(got.shape)
    u = ROUND[dtype]
    _within(pre, z, zb + z.abs() * u + TINY[dtype], "pre-activation")
    y = _act64(z, act)
    # The slopes are below 1.13; the exponential and the error function are good to 2^-20 of what they scale.
    yb = 1.13 * zb + (2.0**-20 * (2 + z.abs()) * z.abs() if act in ("gelu", "silu") else 0.0)
    if r is not None:
        y = y + r.double()
    _within(got, y, yb + y.abs() * u + 2.0**-23 * y.abs() + TINY[dtype], "result")
    assert torch.equal(got, quiver.linear(x, w, bias=b, activation=act, residual=r))  # without keeping, again
    return got


SHAPES = [(1, 1, 1), (1, 1024, 512), (3, 100, 17), (16, 64, 64), (17, 33, 40), (64, 100, 129), (65, 8, 8), (65, 64, 64),
          (100, 128, 130), (129, 16, 257), (1003, 100, 384), (300, 777, 501), (1000, 1000, 256), (257, 72, 1), (130, 2000, 33),
          (4096, 24, 2600), (2100, 520, 2050), (128, 4096, 64)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(dtype, m, k, n):
    g = torch.Generator().manual_seed(m + k + n)
    _say("linear", dtype, m, k, n)
    x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype, std=1 / math.sqrt(k))
    b, r = _randn(g, n, dtype=dtype), _randn(g, m, n, dtype=dtype)
    _check_linear(dtype, x, w, b, "gelu", r)
    _check_linear(dtype, x, w, None, "none", None)
    _check_linear(dtype, x, w, b, "relu", None)
    _check_linear(dtype, x, w, None, "silu", r)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(4111, 72, 4501), (8200, 64, 2056)])
def test_linear_of_large_results(dtype, m, k, n):
    """Results of more than 32 MB, with rows that begin anywhere and a last tile that ends anywhere."""
    test_linear(dtype, m, k, n)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m", [5, 200])
def test_linear_views(dtype, m):
    """Rows with a stride, columns that start off alignment, leading dimensions, transposes."""
    g = torch.Generator().manual_seed(m)
    _say("linear views", dtype, m)
    big, wbig = _randn(g, m, 150, dtype=dtype), _randn(g, 96, 150, dtype=dtype, std=0.1)
    b = _randn(g, 200, dtype=dtype)
    r = _randn(g, m, 200, dtype=dtype)
    for s in (slice(0, 128), slice(1, 129), slice(8, 136), slice(3, 20)):
        _check_linear(dtype, big[:, s], wbig[:, s], b[1:97], "silu", r[:, 7:103])
    _check_linear(dtype, big.t().contiguous().t(), wbig.t().contiguous().t(), None, "none", None)
    x3 = _randn(g, m, 3, 64, dtype=dtype)
    assert _check_linear(dtype, x3, wbig[:, :64], b[:96], "none", None).shape == (m, 3, 96)
    one = quiver.linear(x3[0, 0], wbig[:, :64])
    assert one.shape == (96,)
    wide = big[:1].expand(m, 150)  # rows that all are the same memory
    _check_linear(dtype, wide, wbig, None, "none", None)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_empty(dtype):
    dev, t = _gpu(), TYPES[dtype]
    _say("linear empty", dtype)
    w, b = torch.ones((5, 4), dtype=t, device=dev), torch.arange(5, device=dev).to(t)
    assert quiver.linear(torch.ones((0, 4), dtype=t, device=dev), w).shape == (0, 5)
    assert quiver.linear(torch.ones((3, 4), dtype=t, device=dev), w[:0]).shape == (3, 0)
    for m in (2, 100):  # k = 0: nothing but the bias
        got = quiver.linear(torch.ones((m, 0), dtype=t, device=dev), w[:, :0], bias=b, activation="relu")
        assert torch.equal(got, b.expand(m, 5))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m", [4, 150])
def test_linear_not_finite(dtype, m):
    """Infinities and NaN stay in their own rows and columns, and an infinity stays one, against zeros and
    values without low bits too."""
    dev = _gpu()
    _say("linear not finite", dtype, m)
    g = torch.Generator().manual_seed(3)
    x, w = _randn(g, m, 80, dtype=dtype), torch.ones((70, 80), dtype=TYPES[dtype], device=dev)
    x[1, 5], x[2, 7], x[3, 0] = float("inf"), float("nan"), -float("inf")
    w[9] = 0.0
    w[9, 5] = 2.0
    w[11, 3] = float("inf")
    got = quiver.linear(x, w)
    want = x.float().cpu() @ w.float().cpu().t()
    assert torch.equal(torch.isnan(got).cpu(), torch.isnan(want))
    assert torch.equal(torch.isinf(got).cpu(), torch.isinf(want))
    assert torch.equal(got.cpu()[torch.isinf(want)].float(), want[torch.isinf(want)])


def test_linear_fp32_keeps_small_and_large_values():
    """Rows and columns of very different size: the parts of an fp32 value have no common scale to lose it."""
    g = torch.Generator().manual_seed(8)
    _say("linear fp32 range")
    x = _randn(g, 300, 200, dtype="fp32") * torch.logspace(-15, 15, 300, device=_gpu())[:, None]
    w = _randn(g, 150, 200, dtype="fp32") * torch.logspace(-12, 12, 200, device=_gpu())[None, :]
    _check_linear("fp32", x, w, None, "none", None)
    big = torch.full((100, 1), 3.402e38, device=_gpu())  # the first part would round up to infinity
    assert torch.equal(quiver.linear(big, torch.full((70, 1), 0.5, device=_gpu())), torch.full((100, 70), 1.701e38, device=_gpu()))


def test_linear_past_32_bit_offsets():
    dev = _gpu()
    m, n = 70_001, 65_552  # 9.2e9 bytes of results
    _say("linear", m, n)
    g = torch.Generator().manual_seed(2)
    x, w = _randn(g, m, 16, dtype="bf16"), _randn(g, n, 16, dtype="bf16")
    got = quiver.linear(x, w)
    for rows in (slice(0, 3), slice(m - 3, m), slice(65_535, 65_538), slice(32_767, 32_770)):
        xd, wd = x[rows].double(), w.double()
        want = xd @ wd.t()
        _within(got[rows], want, _product_bound(xd, wd.t(), 16) + want.abs() * ROUND["bf16"])


# ---- the linear layer's gradients -------------------------------------------------------------


def _check_linear_grad(dtype, gr, x, w, pre, act):
    dx, dw, db = quiver.linear_grad(gr, x, w, preactivation=pre, activation=act)
    n, k = w.shape
    gd, xd, wd = gr.double().reshape(-1, n), x.double().reshape(-1, k), w.double()
    dz = gd if act == "none" else gd * _slope64(pre.double().reshape(-1, n), act)
    u = ROUND[dtype]
    # dz: the slope to 2^-19 (its terms are at most 1.2 and cancel), and for 16-bit types one rounding.
    ze = gd.abs() * (0.0 if act in ("none", "relu") else 2.0**-19) + (dz.abs() * u + TINY[dtype] if dtype != "fp32" and act != "none" else 0.0)
    m = gd.shape[0]
    want = dz @ wd
    bound = ze @ wd.abs() + _product_bound(dz, wd, n) + want.abs() * u + TINY[dtype]
    _within(dx.reshape(-1, k), want, bound, "grad_x")
    want = dz.t() @ xd
    _within(dw, want, ze.t() @ xd.abs() + _product_bound(dz.t(), xd, m) + want.abs() * u + TINY[dtype], "grad_weight")
    want = dz.sum(0)
    zs = gd.abs() * (0.0 if act in ("none", "relu") else 2.0**-19)
    _within(db, want, zs.sum(0) + dz.abs().sum(0) * (m + 8) * 2.0**-23 + want.abs() * u + TINY[dtype], "grad_bias")
    again = quiver.linear_grad(gr, x, w, preactivation=pre, activation=act)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dw, db)))
    return dx, dw, db


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 100, 30), (16, 64, 64), (63, 65, 66), (200, 8, 8), (1003, 100, 384),
                                   (300, 777, 501), (5000, 64, 72), (2100, 520, 264), (4097, 33, 17), (129, 2000, 1)])
def test_linear_grad(dtype, m, k, n):
    g = torch.Generator().manual_seed(m + k + n)
    _say("linear_grad", dtype, m, k, n)
    x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype, std=1 / math.sqrt(k))
    gr, pre = _randn(g, m, n, dtype=dtype), _randn(g, m, n, dtype=dtype, std=2.0)
    for act in ("none", "relu", "gelu", "silu"):
        _check_linear_grad(dtype, gr, x, w, pre, act)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(24, 938, 117), (90, 30, 1), (2, 2, 3), (70, 338, 65), (513, 6, 129), (5001, 66, 63), (130, 1644, 515)])
def test_linear_grad_of_even_rows_and_odd_ones(dtype, m, k, n):
    """Rows of x and w that are whole dwords but not whole 16-byte pieces, next to odd rows of the gradient."""
    test_linear_grad(dtype, m, k, n)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(65, 2, 1), (100, 1030, 77), (1000, 4094, 66), (3000, 18, 515), (2049, 514, 1027)])
def test_linear_of_even_rows(dtype, m, k, n):
    g = torch.Generator().manual_seed(m + k)
    _say("linear", dtype, m, k, n)
    x, w, b = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype, std=1 / math.sqrt(k)), _randn(g, n, dtype=dtype)
    _check_linear(dtype, x, w, b, "silu", _randn(g, m, n, dtype=dtype))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(4201, 40, 4101), (20_000, 24, 1000)])
def test_linear_grad_of_large_gradients(dtype, m, k, n):
    test_linear_grad(dtype, m, k, n)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_grad_views_and_parts(dtype):
    g = torch.Generator().manual_seed(4)
    _say("linear_grad views", dtype)
    x, w = _randn(g, 500, 150, dtype=dtype), _randn(g, 96, 150, dtype=dtype)
    gr, pre = _randn(g, 500, 200, dtype=dtype), _randn(g, 500, 200, dtype=dtype)
    for s in (slice(0, 96), slice(1, 97), slice(8, 104)):
        for t in (slice(0, 128), slice(1, 129), slice(16, 144)):
            _check_linear_grad(dtype, gr[:, s], x[:, t], w[:, t], pre[:, s], "silu")
            _check_linear_grad(dtype, gr[:, s], x[:, t], w[:, t], None, "none")
    _check_linear_grad(dtype, gr[:, :1].expand(500, 96), x, w, None, "none")  # the gradient of a broadcast sum
    whole = quiver.linear_grad(gr[:, :96], x, w, preactivation=pre[:, :96], activation="gelu")
    part = quiver.linear_grad(gr[:, :96], x, w, preactivation=pre[:, :96], activation="gelu", bias=False, inputs=False)
    assert part[0] is None and part[2] is None and torch.equal(part[1], whole[1])
    three = quiver.linear_grad(gr[:, :96].reshape(50, 10, 96), x.reshape(50, 10, 150), w, pre[:, :96].reshape(50, 10, 96), "gelu")
    assert three[0].shape == (50, 10, 150) and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(three, whole))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_grad_empty(dtype):
    dev, t = _gpu(), TYPES[dtype]
    _say("linear_grad empty", dtype)
    z = lambda *s: torch.ones(s, dtype=t, device=dev)  # noqa: E731
    dx, dw, db = quiver.linear_grad(z(0, 6), z(0, 4), z(6, 4), z(0, 6), "gelu")
    assert dx.shape == (0, 4) and not dw.any() and not db.any()
    dx, dw, db = quiver.linear_grad(z(3, 0), z(3, 4), z(0, 4))
    assert not dx.any() and dx.shape == (3, 4) and dw.shape == (0, 4) and db.shape == (0,)
    dx, dw, db = quiver.linear_grad(z(3, 6), z(3, 0), z(6, 0))
    assert dx.shape == (3, 0) and dw.shape == (6, 0) and bool((db == 3).all())


@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("m", [40, 90])
def test_linear_grad_is_the_layers_derivative(act, m):
    """Central differences of <linear(..), G> in fp32 along random directions. The loss is a sum of m n terms
    below 20 whose errors are independent of h: rounding gives 40 2^-23 m n / 2h at the very most, the third
    derivative (slopes' second derivatives are below 1.2; directions of size 1 in z) h^2 / 6 * 1.2 * sum |G| d^3."""
    _say("linear difference", act, m)
    g = torch.Generator().manual_seed(m)
    k, n, h = 30, 20, 2.0**-6
    x, w, b = _randn(g, m, k, dtype="fp32"), _randn(g, n, k, dtype="fp32", std=0.2), _randn(g, n, dtype="fp32")
    up = _randn(g, m, n, dtype="fp32")
    dx, dw, db = (_randn(g, *s, dtype="fp32", std=0.2) for s in ((m, k), (n, k), (n,)))
    loss = lambda x, w, b: (quiver.linear(x, w, bias=b, activation=act).double() * up).sum()  # noqa: E731
    _, pre = quiver.linear(x, w, bias=b, activation=act, keep_preactivation=True)
    gx, gw, gb = quiver.linear_grad(up, x, w, preactivation=pre, activation=act)
    for what, grad, d, dz in ((0, gx, dx, dx @ w.t()), (1, gw, dw, x @ dw.t()), (2, gb, db, db.expand(m, n))):
        args = [x, w, b]
        step = lambda s: [a + s * h * d if i == what else a for i, a in enumerate(args)]  # noqa: E731
        diff = (loss(*step(1)) - loss(*step(-1))) / (2 * h)
        bound = 40 * 2.0**-23 * m * n / (2 * h) + h * h / 6 * 1.2 * (up.abs() * dz.abs() ** 3).sum().item()
        assert abs(diff - (grad.double() * d).sum()).item() <= bound, (what, bound)


# ---- orthogonalised updates -------------------------------------------------------------------

MUON = (3.4445, -4.7750, 2.0315)


def _ortho64(u, steps, co):
    """The result by the singular values, and how much a relative change of X at the start can grow: per step
    the largest divided difference of s -> f(s) and the polynomial itself over the values that occur."""
    a, b, c = co
    p, s, qt = torch.linalg.svd(u.double().cpu(), full_matrices=False)
    norm = s.square().sum(-1, keepdim=True).sqrt()
    s = torch.where(norm > 0, s / norm, torch.zeros_like(s))
    grow = 1.0
    for _ in range(steps):
        t = torch.linspace(0, s.max().item(), 500, dtype=torch.float64)
        grow *= max(1.0, (a + 3 * b * t**2 + 5 * c * t**4).abs().max().item(), (a + b * t**2 + c * t**4).abs().max().item())
        s = a * s + b * s**3 + c * s**5
    return ((p * s[..., None, :]) @ qt).to(u.device), grow


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (9, 1), (16, 16), (33, 100), (100, 33), (3, 64, 128), (2, 2, 65, 40), (7, 129, 257),
                                   (300, 77), (260, 520), (513, 200)])
def test_orthogonalize(dtype, shape):
    g = torch.Generator().manual_seed(sum(shape))
    _say("orthogonalize", dtype, shape)
    u = _randn(g, *shape, dtype=dtype, std=1e-3)
    side, depth = min(shape[-2:]), max(shape[-2:])
    for steps, co in ((5, MUON), (0, MUON), (3, (1.875, -1.25, 0.375))):
        got = quiver.orthogonalize(u, steps=steps, coefficients=co)
        want, grow = _ortho64(u.float(), steps, co)
        # Every product leaves sqrt(depth) 2^-22 of its size (random roundings of 22-bit parts and of fp32 sums), twice
        # to be safe; the matrices are of norm sqrt(side) at most, and five steps carry each error on.
        bound = grow * (steps + 1) * 2 * math.sqrt(depth) * 2.0**-22 * math.sqrt(side)
        err = (got.double() - want).flatten(-2).norm(dim=-1)
        size = want.flatten(-2).norm(dim=-1)
        assert bool((err <= bound + ROUND[dtype] * size).all()), (steps, err.max().item(), bound)
        assert torch.equal(got, quiver.orthogonalize(u, steps=steps, coefficients=co))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(128, 128), (64, 512), (512, 64), (32, 1100), (1100, 26), (2, 5, 1100), (64, 200), (79, 1220), (1024, 96),
                                   (128, 1300), (1, 2048), (2049, 2), (640, 640), (3, 384, 300)])
def test_orthogonalize_long_and_large(dtype, shape):
    test_orthogonalize(dtype, shape)


def test_orthogonalize_makes_singular_values_alike():
    g = torch.Generator().manual_seed(1)
    _say("orthogonalize singular values")
    for shape in ((200, 300), (300, 200)):
        s = torch.linalg.svdvals(quiver.orthogonalize(_randn(g, *shape, dtype="fp32")).double())
        assert 0.6 < s.min().item() and s.max().item() < 1.3  # what the default coefficients are made for
        s = torch.linalg.svdvals(quiver.orthogonalize(_randn(g, *shape, dtype="fp32"), 30, (1.5, -0.5, 0.0)).double())
        assert (s - 1).abs().max().item() < 1e-4  # classical steps converge


@pytest.mark.parametrize("dtype", list(TYPES))
def test_orthogonalize_scale_zero_and_not_finite(dtype):
    dev = _gpu()
    _say("orthogonalize special", dtype)
    g = torch.Generator().manual_seed(6)
    u = _randn(g, 4, 40, 56, dtype=dtype)
    u[1] = 0.0
    u[2, 3, 5] = float("inf")
    u[3, 0, 0] = float("nan")
    got = quiver.orthogonalize(u)
    assert not got[1].any() and bool(torch.isnan(got[2]).all()) and bool(torch.isnan(got[3]).all())
    assert torch.equal(got[0], quiver.orthogonalize(u[0]))
    assert torch.equal(got[0], quiver.orthogonalize(u[0] * 2.0))  # a power of two changes nothing
    if dtype != "fp16":  # squares past fp32's range on both sides
        for s in (1e30, 1e-30, 1e-37):
            v = (u[0].float() * s).to(u.dtype)
            want, grow = _ortho64(v.float(), 5, MUON)
            err = (quiver.orthogonalize(v).double() - want).norm().item()
            assert err <= grow * 6 * 2 * math.sqrt(56) * 2.0**-22 * math.sqrt(40) + ROUND[dtype] * want.norm().item()
    assert quiver.orthogonalize(u[:0]).shape == (0, 40, 56)
    assert quiver.orthogonalize(torch.zeros((3, 0), device=dev)).shape == (3, 0)
    assert torch.equal(quiver.orthogonalize(u[0].t().contiguous().t()), got[0])  # another layout


# ---- streams, graphs, refusals ----------------------------------------------------------------


def _all_calls(s):
    h = quiver.embed(s["table"], s["tok"], scale=2.0)
    y, z = quiver.linear(h, s["w"], bias=s["b"], activation="gelu", residual=s["r"], keep_preactivation=True)
    dh, dw, db = quiver.linear_grad(y, h, s["w"], preactivation=z, activation="gelu")
    return y, z, dh, dw, db, quiver.embed_grad(dh, s["tok"], len(s["table"])), quiver.orthogonalize(dw)


def _state(dtype, n=3000, seed=0):
    g = torch.Generator().manual_seed(seed)
    return dict(table=_randn(g, 700, 104, dtype=dtype), tok=torch.randint(-1, 700, (n,), generator=g).to(_gpu()),
                w=_randn(g, 120, 104, dtype=dtype, std=0.1), b=_randn(g, 120, dtype=dtype), r=_randn(g, n, 120, dtype=dtype))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_calls_follow_the_current_stream(dtype):
    _say("streams", dtype)
    want = _all_calls(_state(dtype))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = _all_calls(_state(dtype))  # the uploads and the calls on one side stream
        later = [t.clone() for t in got]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(later, want))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [50, 3000])
def test_calls_in_a_graph(dtype, n):
    """Captured once, replayed on new inputs with eager work between the replays."""
    _say("graph", dtype, n)
    state = _state(dtype, n)
    _all_calls(state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _all_calls(state)
    for seed in (1, 2, 3):
        fresh = _state(dtype, n, seed)
        for name, t in fresh.items():
            state[name].copy_(t)
        want = _all_calls(fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_allocates_nothing_of_its_own():
    import ctypes as C

    from qvh_ctypes import LIB

    lib = C.CDLL(LIB)
    count = C.c_uint64()
    assert lib.qvh_device_allocations(C.byref(count)) == 0
    before = count.value
    _all_calls(_state("bf16"))
    assert lib.qvh_device_allocations(C.byref(count)) == 0 and count.value == before


def test_refusals():
    dev = _gpu()
    _say("refusals")
    f = torch.zeros((8, 16), device=dev)
    t = torch.zeros(8, dtype=torch.int64, device=dev)
    for call, word in [
            (lambda: quiver.embed(f.double(), t), "float32"), (lambda: quiver.embed(f[0], t), "table must be"),
            (lambda: quiver.embed(f, t.float()), "int32 or int64"), (lambda: quiver.embed(f, t.cpu()), "tokens are on"),
            (lambda: quiver.embed_grad(f, t[:3], 5), "grad must have shape"), (lambda: quiver.embed_grad(f, t, -1), "non-negative"),
            (lambda: quiver.linear(f, f[:, :8]), "weight"), (lambda: quiver.linear(f, f.half()), "float16"),
            (lambda: quiver.linear(f, f, bias=f[0]), "bias"), (lambda: quiver.linear(f, f, residual=f), "residual"),
            (lambda: quiver.linear(f, f, activation="tanh"), "activation"), (lambda: quiver.linear(f.long(), f), "float32"),
            (lambda: quiver.linear_grad(f, f, f), "grad must have"),
            (lambda: quiver.linear_grad(f[:, :8], f, f, activation="relu"), "pre-activation"),
            (lambda: quiver.linear_grad(f[:, :8], f, f, f, "relu"), "preactivation must"),
            (lambda: quiver.orthogonalize(f[0]), "update must"), (lambda: quiver.orthogonalize(f, coefficients=(1.0, 2.0)), "three"),
            (lambda: quiver.orthogonalize(f, steps=-1), "steps"), (lambda: quiver.orthogonalize(f, coefficients=(9.0, 0.0, 0.0)), "grow")]:
        with pytest.raises(ValueError, match=word):
            call()
    with pytest.raises(TypeError, match="torch tensor"):
        quiver.embed(np.zeros((3, 3), np.float32), t)
