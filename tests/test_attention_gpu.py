"""Linear attention with decays against 64-bit arithmetic, by blocks of the masked product (not the kernel's recurrence).

Bounds are of the terms' magnitudes: M is the same formula of the inputs' absolute values. fp32 sums of dk and T terms are
off by at most (dk + T + 256) 2^-23 M, where 256 stands for the factors of a term and powers of the decay. 16-bit results
have the scores and the state rounded once each on their way, u M at most, and are rounded themselves. A float16
operand is exact to 2^-36 of the largest one beside it.
"""

import math

import pytest

import quiver_amd as quiver

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_encoder_gpu import ROUND, TINY, TYPES, _gpu, _randn, _say, _within  # noqa: E402


def _scan_64(q, k, v, g, state, ahead=1):
    """[h, t, d] in 64 bits from state [h, dk, dv]: results and the last state. ahead: 1 where the state decays ahead of a token."""
    out = torch.zeros((q.shape[0], q.shape[1], v.shape[2]), dtype=torch.float64, device=q.device)
    g = g[:, None].clamp(min=-1e30)
    for c in range(0, q.shape[1], 512):
        qc, kc, vc = q[:, c:c + 512], k[:, c:c + 512], v[:, c:c + 512]
        n = qc.shape[1]
        at = torch.arange(n, device=q.device, dtype=torch.float64)
        apart = (at[:, None] - at[None, :]).clamp(min=0)
        near = (torch.bmm(qc, kc.transpose(1, 2).contiguous()) * torch.exp(g[:, :, None] * apart)).tril()
        out[:, c:c + 512] = torch.bmm(near, vc) + torch.bmm(qc, state) * torch.exp(g * (at + ahead))[:, :, None]
        weighed = kc * torch.exp(g * (n - ahead - at))[:, :, None]
        state = state * torch.exp(g * n)[:, :, None] + torch.bmm(weighed.transpose(1, 2).contiguous(), vc)
    return out, state


def _texts(fn, lengths, batch, tokens):
    for b in range(batch):
        n = tokens if lengths is None else min(max(int(lengths[b]), 0), tokens)
        fn(b, n)


def _forward_64(q, k, v, g, state, lengths, scale):
    """(out, last state) and their magnitudes."""
    b, t, h, dk = q.shape
    share = h // k.shape[2]
    q, k, v = (x.double().transpose(1, 2) for x in (q, k, v))
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    out = torch.zeros((2, b, t, h, v.shape[3]), dtype=torch.float64, device=q.device)
    last = torch.zeros((2, b, h, dk, v.shape[3]), dtype=torch.float64, device=q.device)

    def text(i, n):
        s = state[i].double() if state is not None else torch.zeros_like(last[0, 0])
        for m, f in ((0, lambda x: x), (1, torch.abs)):
            o, e = _scan_64(f(q[i, :, :n]), f(k[i, :, :n]), f(v[i, :, :n]), g.double(), f(s))
            out[m, i, :n], last[m, i] = o.transpose(0, 1) * (abs(scale) if m else scale), e

    _texts(text, lengths, b, t)
    return out, last


def _grad_64(grad, q, k, v, g, state, lengths, scale, grad_state):
    """Gradients of q, k, v and the first state, each with its magnitude."""
    b, t, h, dk = q.shape
    hk, dv = v.shape[2:]
    share = h // hk
    grad, q, k, v = (x.double().transpose(1, 2) for x in (grad, q, k, v))
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    new = lambda *s: torch.zeros((2, b, *s), dtype=torch.float64, device=q.device)  # noqa: E731
    gq, gk, gv, first = new(t, h, dk), new(t, h, dk), new(t, h, dv), new(h, dk, dv)
    zero = torch.zeros_like(first[0, 0])

    def text(i, n):
        for m, f in ((0, lambda x: x), (1, torch.abs)):
            sc = abs(scale) if m else scale
            s = f(state[i].double()) if state is not None else zero
            e = f(grad_state[i].double()) if grad_state is not None else zero
            qi, ki, vi, oi = (f(x[i, :, :n]) for x in (q, k, v, grad))
            gd = g.double()
            gq[m, i, :n] = _scan_64(oi, vi, ki, gd, s.transpose(1, 2).contiguous())[0].transpose(0, 1) * sc
            rq, rk, rv, ro = (x.flip(1) for x in (qi * sc, ki, vi, oi))
            x, y = _scan_64(rk, rq, ro, gd, e, 0)
            gv[m, i, :n], first[m, i] = x.flip(1).transpose(0, 1), y
            gk[m, i, :n] = _scan_64(rv, ro, rq, gd, e.transpose(1, 2).contiguous(), 0)[0].flip(1).transpose(0, 1)

    _texts(text, lengths, b, t)
    return gq, gk.unflatten(3, (hk, share)).sum(4), gv.unflatten(3, (hk, share)).sum(4), first


def _bound(value, size, dtype, terms):
    own = 0.0 if dtype == "fp32" else ROUND[dtype]
    far = 2.0**-36 * size.max().item() if dtype == "fp16" and size.numel() else 0.0
    return size * (own + terms * 2.0**-23) + value.abs() * ROUND[dtype] + TINY[dtype] + far


def _inputs(g, dtype, batch, tokens, heads, kv_heads, dk, dv, state=False):
    q, k, v = (_randn(g, batch, tokens, h, d, dtype=dtype) for h, d in ((heads, dk), (kv_heads, dk), (kv_heads, dv)))
    log_decay = -torch.exp2(-10.0 * torch.rand(heads, generator=g)).to(_gpu())
    return q, k, v, log_decay, torch.randn(batch, heads, dk, dv, generator=g).to(_gpu()) if state else None


def _check(q, k, v, log_decay, state, lengths=None, scale=None):
    dtype = next(n for n, t in TYPES.items() if t is q.dtype)
    got, last = quiver.linear_attention(q, k, v, log_decay, state=state, lengths=lengths, scale=scale, keep_state=True)
    scale = q.shape[3] ** -0.5 if scale is None else scale
    want, end = _forward_64(q, k, v, log_decay, state, lengths, scale)
    terms = q.shape[3] + q.shape[1] + 256
    assert got.dtype == q.dtype and last.dtype == torch.float32
    _within(got, want[0], _bound(want[0], want[1], dtype, terms), "out")
    _within(last, end[0], end[1] * terms * 2.0**-23 + 2.0**-126, "state")
    return got, last


def _check_grad(g, q, k, v, log_decay, state, lengths=None, scale=None, grad_state=None):
    dtype = next(n for n, t in TYPES.items() if t is q.dtype)
    grad = _randn(g, *q.shape[:3], v.shape[3], dtype=dtype)
    got = quiver.linear_attention_grad(grad, q, k, v, log_decay, state=state, lengths=lengths, scale=scale, grad_state=grad_state)
    scale = q.shape[3] ** -0.5 if scale is None else scale
    want = _grad_64(grad, q, k, v, log_decay, state, lengths, scale, grad_state)
    terms = q.shape[3] + v.shape[3] + q.shape[1] + 256 + q.shape[2]
    for name, a, b in zip(("q", "k", "v"), got, want):
        assert a.dtype == q.dtype
        _within(a, b[0], _bound(b[0], b[1], dtype, terms), name)
    assert (got[3] is None) == (state is None)
    if state is not None:
        _within(got[3], want[3][0], want[3][1] * terms * 2.0**-23 + 2.0**-126, "state")


SHAPES = [(1, 1, 64, 64), (3, 1, 64, 64), (4, 2, 128, 128), (2, 2, 16, 40), (1, 1, 1, 1), (6, 3, 33, 100), (2, 1, 200, 72),
          (1, 1, 256, 256), (2, 2, 72, 130)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_attention(dtype, shape):
    g = torch.Generator().manual_seed(sum(shape))
    for tokens in (1, 2, 8, 9, 16, 17, 63, 64, 65, 129, 200):
        _say("attention", dtype, tokens, *shape)
        _check(*_inputs(g, dtype, 2, tokens, *shape, state=tokens % 2 == 1))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_attention_grad(dtype, shape):
    g = torch.Generator().manual_seed(sum(shape) + 1)
    for tokens in (1, 7, 63, 64, 66, 150):
        _say("attention_grad", dtype, tokens, *shape)
        inputs = _inputs(g, dtype, 2, tokens, *shape, state=tokens % 2 == 1)
        end = torch.randn(2, shape[0], shape[2], shape[3], generator=g).to(_gpu()) if tokens % 3 else None
        _check_grad(g, *inputs, grad_state=end, scale=0.3)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,shape", [(1_100, (1, 1, 64, 64)), (1_537, (2, 1, 128, 100)), (3_000, (1, 1, 40, 200))])
def test_long_texts_in_segments(dtype, tokens, shape):
    g = torch.Generator().manual_seed(tokens)
    _say("attention", dtype, tokens, *shape)
    inputs = _inputs(g, dtype, 2, tokens, *shape, state=True)
    lengths = torch.tensor([tokens, tokens - 600], device=_gpu())
    end = torch.randn(2, shape[0], shape[2], shape[3], generator=g).to(_gpu())
    for n in (None, lengths):
        _check(*inputs, lengths=n)
        _check_grad(g, *inputs, lengths=n, grad_state=end)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (12, 6)])
@pytest.mark.parametrize("dk,dv", [(64, 128), (128, 64), (64, 256)])
def test_gradients_of_which_some_go_in_segments(dtype, heads, kv_heads, dk, dv, monkeypatch):
    """The three passes have dk columns or dv of them, and are cut or not by their number: nothing is written behind the workspace."""
    from quiver_amd import blocks

    g = torch.Generator().manual_seed(dk + dv + heads)
    _say("attention_grad segments of some", dtype, heads, dk, dv)
    held = []

    def workspace(nbytes, device):
        held.append((nbytes, torch.full((nbytes + (8 << 20),), 0xA5, dtype=torch.uint8, device=device)))
        return held[-1][1][:nbytes]

    monkeypatch.setattr(blocks, "_workspace", workspace)
    inputs = _inputs(g, dtype, 4, 1_100, heads, kv_heads, dk, dv, state=True)
    lengths = torch.tensor([1_100, 0, 321, 1_024], device=_gpu())
    end = torch.randn(4, heads, dk, dv, generator=g).to(_gpu())
    _check_grad(g, *inputs[:4], None)
    _check_grad(g, *inputs, grad_state=end)
    _check_grad(g, *inputs, lengths=lengths, grad_state=end)
    grad = _randn(g, 4, 1_100, heads, dv, dtype=dtype)
    calls = [quiver.linear_attention_grad(grad, *inputs[:4], state=inputs[4], grad_state=end) for _ in range(3)]
    assert all(torch.equal(a, b) for c in calls[1:] for a, b in zip(c, calls[0]))
    assert len(held) == 6 and all((t[n:] == 0xA5).all() for n, t in held)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_segments_with_padding_and_the_state_in_place(dtype):
    """Texts that end in any segment, on its ends and before the first; decays of everything and nothing; junk behind the ends."""
    g = torch.Generator().manual_seed(53)
    _say("attention segments", dtype)
    tokens, ends = 1_100, [1_100, 0, 1, 320, 640, 641, 900]
    q, k, v, _, s = _inputs(g, dtype, 7, tokens, 4, 2, 24, 40, state=True)
    decay = torch.tensor([-0.01, 0.0, float("-inf"), -3.0], device=_gpu())
    lengths = torch.tensor(ends, device=_gpu())
    clean = _check(q, k, v, decay, s, lengths=lengths)
    assert torch.equal(clean[1][1], s[1])
    _check_grad(g, q, k, v, decay, s, lengths=lengths, grad_state=s)
    behind = torch.arange(tokens, device=_gpu())[None] >= lengths[:, None]
    for t in (q, k, v):
        t[behind] = float("nan")
    held = s.clone()
    got = quiver.linear_attention(q, k, v, decay, state=held, lengths=lengths, state_out=held)
    assert got[1] is held and all(torch.equal(a, b) for a, b in zip(got, clean))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("at", [0, 300, 1_099])
def test_tokens_that_are_not_finite_in_segments(dtype, at):
    g = torch.Generator().manual_seed(59)
    _say("attention special segments", dtype, at)
    q, k, v, g_, s = _inputs(g, dtype, 1, 1_100, 2, 2, 64, 48, state=True)
    clean = quiver.linear_attention(q, k, v, g_, state=s, keep_state=True)
    want, size = _forward_64(q, k, v, g_, s, None, 0.125)[0]
    off = _bound(want, size, dtype, 64 + 1_100 + 256)
    others = [c for c in range(48) if c != 17]
    for junk in (float("inf"), float("-inf"), float("nan")):
        bad = v.clone()
        bad[0, at, 1, 17] = junk
        got, last = quiver.linear_attention(q, k, bad, g_, state=s, keep_state=True)
        assert torch.equal(got[:, :at], clean[0][:, :at]) and torch.equal(got[:, :, 0], clean[0][:, :, 0])
        _within(got[:, :, 1][:, :, others], want[:, :, 1][:, :, others], off[:, :, 1][:, :, others], "other columns")
        assert not torch.isfinite(got[0, at:, 1, 17]).any() and not torch.isfinite(last[0, 1, :, 17]).any()
        assert torch.isfinite(last[0, 1][:, others]).all()
        bad = k.clone()
        bad[0, at, 1, 5] = junk
        got, last = quiver.linear_attention(q, bad, v, g_, state=s, keep_state=True)
        assert torch.equal(got[:, :at], clean[0][:, :at]) and torch.equal(got[:, :, 0], clean[0][:, :, 0])
        assert not torch.isfinite(last[0, 1, 5]).any() and torch.isfinite(last[0, 1][[i for i in range(64) if i != 5]]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_many_texts_fill_the_device(dtype):
    g = torch.Generator().manual_seed(11)
    _say("attention many", dtype)
    inputs = _inputs(g, dtype, 70, 100, 8, 4, 48, 64)
    lengths = torch.randint(0, 101, (70,), generator=g).to(_gpu())
    _check(*inputs, lengths=lengths)
    _check_grad(g, *inputs, lengths=lengths)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens", [4, 5, 70, 300])
def test_padding(dtype, index, tokens):
    """What lies behind a text's end counts for nothing, NaN and infinities too; lengths past either end are clamped."""
    g = torch.Generator().manual_seed(tokens)
    _say("attention padding", dtype, index, tokens)
    lengths = torch.tensor([tokens, 0, 1, tokens // 2, tokens - 1, tokens + 9, -3], dtype=index, device=_gpu())
    q, k, v, g_, s = _inputs(g, dtype, 7, tokens, 2, 1, 24, 32, state=True)
    clean = _check(q, k, v, g_, s, lengths=lengths)
    assert torch.equal(clean[1][1], s[1]) and torch.equal(clean[1][6], s[6])
    grad, end = _randn(g, 7, tokens, 2, 32, dtype=dtype), torch.randn(7, 2, 24, 32, generator=g).to(_gpu())
    want = quiver.linear_attention_grad(grad, q, k, v, g_, state=s, lengths=lengths, grad_state=end)
    assert torch.equal(want[3][1], end[1])
    _check_grad(g, q, k, v, g_, s, lengths=lengths, grad_state=end)
    behind = torch.arange(tokens, device=_gpu())[None] >= lengths[:, None]
    for junk in (float("nan"), float("inf")):
        for t in (q, k, v, grad):
            t[behind] = junk
        got = quiver.linear_attention(q, k, v, g_, state=s, lengths=lengths, keep_state=True)
        assert all(torch.equal(a, b) for a, b in zip(got, clean)) and not got[0][behind].any()
        got = quiver.linear_attention_grad(grad, q, k, v, g_, state=s, lengths=lengths, grad_state=end)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and not any(t[behind].any() for t in got[:3])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens", [4, 6, 90])
def test_tokens_that_are_not_finite_change_later_ones_only(dtype, tokens):
    g = torch.Generator().manual_seed(tokens + 1)
    _say("attention special", dtype, tokens)
    for dk in (24, 64):
        q, k, v, g_, s = _inputs(g, dtype, 2, tokens, 2, 2, dk, 48, state=True)
        clean = quiver.linear_attention(q, k, v, g_, state=s, keep_state=True)
        want, size = _forward_64(q, k, v, g_, s, None, dk ** -0.5)[0]
        off = _bound(want, size, dtype, dk + tokens + 256)
        for at in (0, 3, tokens - 2):
            for junk in (float("inf"), float("-inf"), float("nan")):
                bad = v.clone()
                bad[0, at, 1, 17] = junk
                got, last = quiver.linear_attention(q, k, bad, g_, state=s, keep_state=True)
                assert torch.equal(got[:, :at], clean[0][:, :at]) and torch.equal(got[1], clean[0][1])
                assert torch.equal(got[0, :, 0], clean[0][0, :, 0]) and torch.equal(last[0, 0], clean[1][0, 0])
                others = [c for c in range(48) if c != 17]
                _within(got[0, :, 1][:, others], want[0, :, 1][:, others], off[0, :, 1][:, others], "other columns")
                assert not torch.isfinite(got[0, at:, 1, 17]).any()
                # The recurrence in 64 bits: an infinity times k's sign, NaN once two of them meet. Padding of dk adds none.
                state = s[0, 1].double() * torch.exp(g_[1].double() * (at + 1))
                kept = bad[0, at, 1, 17].double() * k[0, at, 1].double() + state[:, 17] * 0
                assert torch.equal(last[0, 1, :, 17].double().nan_to_num(7.0), kept.nan_to_num(7.0))
                bad = k.clone()
                bad[0, at, 1, 5] = junk
                got, last = quiver.linear_attention(q, bad, v, g_, state=s, keep_state=True)
                assert torch.equal(got[:, :at], clean[0][:, :at]) and torch.equal(got[0, :, 0], clean[0][0, :, 0])
                assert torch.isfinite(last[0, 1][[i for i in range(dk) if i != 5]]).all()
                kept = junk * v[0, at, 1].double()
                assert torch.equal(last[0, 1, 5].double().nan_to_num(7.0), kept.nan_to_num(7.0))
                bad = q.clone()
                bad[0, at, 1, 5] = junk
                got, last = quiver.linear_attention(bad, k, v, g_, state=s, keep_state=True)
                others = [t for t in range(tokens) if t != at]
                assert torch.equal(got[0, others], clean[0][0, others]) and torch.equal(last, clean[1])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_scores_past_fp32_range_stay_behind_the_mask(dtype):
    """Finite tokens whose products with earlier queries are infinite change nothing before them."""
    g = torch.Generator().manual_seed(47)
    _say("attention masked overflow", dtype)
    q, k, v, g_, _ = _inputs(g, dtype, 1, 80, 2, 2, 32, 32)
    q *= 1e18
    clean = quiver.linear_attention(q, k, v, g_)
    for at in (1, 17, 63, 79):
        bad = k.clone()
        bad[0, at] = 3e38
        got = quiver.linear_attention(q, bad, v, g_)
        assert torch.equal(got[:, :at], clean[:, :at]) and torch.isfinite(got[:, :at]).all(), at


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens", [4, 150, 1_200])
def test_decays_from_nothing_to_everything(dtype, tokens):
    g = torch.Generator().manual_seed(tokens + 2)
    _say("attention decays", dtype, tokens)
    q, k, v, _, s = _inputs(g, dtype, 1, tokens, 6, 6, 32, 32, state=True)
    decay = torch.tensor([0.0, float("-inf"), -60.0, -1e-7, -2.0**-12, -1.0], device=_gpu())
    got, _ = _check(q, k, v, decay, s)
    _check_grad(g, q, k, v, decay, s, grad_state=s)
    # No memory: each token by itself.
    alone = (q[:, :, 1] * k[:, :, 1]).double().sum(-1, keepdim=True) * v[:, :, 1].double() * 32 ** -0.5
    size = (q[:, :, 1].double() * k[:, :, 1].double()).abs().sum(-1, keepdim=True) * v[:, :, 1].double().abs()
    alone = (q[:, :, 1].double() * k[:, :, 1].double()).sum(-1, keepdim=True) * v[:, :, 1].double() * 32 ** -0.5
    _within(got[:, :, 1], alone, _bound(alone, size, dtype, 300))


def test_float16_states_past_its_range():
    """Sums that float16 cannot hold, and values that it nearly cannot, come out as they are."""
    dev = _gpu()
    _say("attention fp16 range")
    one = torch.ones((1, 3_000, 1, 64), dtype=torch.float16, device=dev)
    decay = torch.zeros(1, device=dev)
    big = one * 60.0  # a state of 3,000 * 3,600
    got, last = quiver.linear_attention(one * 2.0**-10, big, big, decay, scale=2.0**-9, keep_state=True)
    t = torch.arange(1, 3_001, device=dev, dtype=torch.float64)
    want = (t * 3600.0 * 64 * 2.0**-19)[None, :, None, None].expand_as(got)
    _within(got, want, want * (2 * 2.0**-11 + 4_000 * 2.0**-23))
    _within(last, torch.full_like(last, 3_000 * 3600.0).double(), torch.full_like(last, 3_000 * 3600.0 * 4_000 * 2.0**-23).double())
    small = one * 2.0**-13
    got, _ = quiver.linear_attention(small, small, one, decay, scale=2.0**16, keep_state=True)
    want = (t * 64 * 2.0**-10)[None, :, None, None].expand_as(got)
    _within(got, want, want * (2 * 2.0**-11 + 4_000 * 2.0**-23))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_text_in_parts(dtype):
    """A text that goes on from its state gives what the whole one does, in parts of any size and token by token."""
    g = torch.Generator().manual_seed(13)
    _say("attention parts", dtype)
    q, k, v, g_, s = _inputs(g, dtype, 2, 210, 4, 2, 64, 48, state=True)
    want, size = _forward_64(q, k, v, g_, s, None, 0.125)[0]
    end = _forward_64(q, k, v, g_, s, None, 0.125)[1]
    for parts in ([100, 110], [1, 64, 9, 63, 73], [1] * 210):
        state, outs, at = s.clone(), [], 0
        for n in parts:
            o, same = quiver.linear_attention(q[:, at:at + n], k[:, at:at + n], v[:, at:at + n], g_, state=state, state_out=state)
            assert same is state
            outs.append(o)
            at += n
        _within(torch.cat(outs, 1), want, _bound(want, size, dtype, 64 + 210 + 256), str(parts[:3]))
        _within(state, end[0], end[1] * (210 + 256) * 2.0**-23)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens", [3, 80])
def test_views(dtype, tokens):
    g = torch.Generator().manual_seed(17)
    _say("attention views", dtype, tokens)
    p = _randn(g, 2, tokens, 3, 2, 41, dtype=dtype)
    decay = torch.tensor([[-0.1, 9.0], [-0.3, 9.0]], device=_gpu())[:, 0]
    odd = _randn(g, 2, tokens + 1, 2, 50, dtype=dtype)
    cases = [(p[:, :, 0], p[:, :, 1], p[:, :, 2]), (p[:, :, 0, :, 1:33], p[:, :, 1, :, 3:35], odd[:, 1:, :, 5:46]),
             tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (p[:, :, 0], p[:, :, 1], p[:, :, 2])),
             (p[:, :, 0], p[:, :1, 1].expand(2, tokens, 2, 41), p[:1, :, 2].expand(2, tokens, 2, 41)),
             (p[:, :, 0, :, ::2], p[:, :, 1, :, ::2], p[:, :, 2].flip(1)), (p[:, :, 0], p[:, :, 1, :1], p[:, :, 2, :1])]
    for q, k, v in cases:
        s = torch.randn(v.shape[3], 2, 2, q.shape[3], generator=g).to(_gpu()).permute(1, 2, 3, 0)
        lengths = torch.tensor([[tokens, 1], [tokens - 1, 1]], device=_gpu())[:, 0]
        plain = [t.contiguous() for t in (q, k, v)]
        a = quiver.linear_attention(q, k, v, decay, state=s, lengths=lengths, keep_state=True)
        b = quiver.linear_attention(*plain, decay.contiguous(), state=s.contiguous(), lengths=lengths.contiguous(), keep_state=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        held = s.clone(memory_format=torch.preserve_format)
        assert torch.equal(quiver.linear_attention(q, k, v, decay, state=held, lengths=lengths, state_out=held)[1], a[1])
        grad = a[0].transpose(1, 2).contiguous().transpose(1, 2)
        a = quiver.linear_attention_grad(grad, q, k, v, decay, state=s, lengths=lengths)
        b = quiver.linear_attention_grad(grad.contiguous(), *plain, decay.contiguous(), state=s.contiguous(), lengths=lengths.contiguous())
        assert all(torch.equal(x, y) and x.is_contiguous() for x, y in zip(a, b))


def test_empty():
    dev = _gpu()
    _say("attention empty")
    decay = torch.zeros(3, device=dev)
    for b, t in ((0, 5), (2, 0), (0, 0)):
        q = torch.zeros((b, t, 3, 8), device=dev)
        s = torch.randn((b, 3, 8, 8), device=dev)
        o, last = quiver.linear_attention(q, q, q, decay, state=s, keep_state=True)
        assert o.shape == q.shape and torch.equal(last, s)
        assert not quiver.linear_attention(q, q, q, decay, keep_state=True)[1].any()
        grads = quiver.linear_attention_grad(q, q, q, q, decay, state=s, grad_state=s)
        assert all(x.shape == q.shape for x in grads[:3]) and torch.equal(grads[3], s)


def test_past_32_bit_offsets():
    dev = _gpu()
    _say("attention offsets")
    far = 2**31 + 64
    buffer = torch.empty(2 * far, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(19)
    q, k, v, g_, _ = _inputs(g, "bf16", 2, 80, 1, 1, 16, 16)
    wide = buffer.as_strided((2, 80, 1, 16), (far, 16 * 1_000_000 // 16 * 16, 16, 1))
    want = quiver.linear_attention(q, k, v, g_)
    for name in ("q", "k", "v"):
        t = dict(q=q, k=k, v=v)
        wide.copy_(t[name])
        t[name] = wide
        assert torch.equal(quiver.linear_attention(t["q"], t["k"], t["v"], g_), want)


@pytest.mark.parametrize("tokens", [4, 5, 100])
def test_grad_against_differences(tokens):
    """A step along a direction changes the loss by the gradient's part along it (fp32, central differences)."""
    g = torch.Generator().manual_seed(23)
    _say("attention differences", tokens)
    q, k, v, g_, s = _inputs(g, "fp32", 2, tokens, 2, 1, 20, 12, state=True)
    lengths = torch.tensor([tokens, tokens - 3], device=_gpu())
    co, cs = _randn(g, 2, tokens, 2, 12, dtype="fp32"), _randn(g, 2, 2, 20, 12, dtype="fp32")

    def loss(q, k, v, s):
        o, end = quiver.linear_attention(q, k, v, g_, state=s, lengths=lengths, keep_state=True)
        return (co.double() * o.double()).sum() + (cs.double() * end.double()).sum()

    grads = quiver.linear_attention_grad(co, q, k, v, g_, state=s, lengths=lengths, grad_state=cs)
    values = dict(q=q, k=k, v=v, s=s)
    terms = (co.abs().sum() * 40 + cs.abs().sum() * 40).item()  # results of a few tens at most
    for name, grad in zip("qkvs", grads):
        d = _randn(g, *values[name].shape, dtype="fp32")
        d /= d.norm()
        up, down = (loss(**{**values, name: values[name] + x * d}) for x in (0.5, -0.5))
        along = (grad.double() * d.double()).sum().item()
        # Each input by itself enters linearly: only rounding is left, of every term by (dk + T) 2^-23.
        assert abs((up - down).item() - along) <= terms * (20 + tokens) * 2.0**-23, name


@pytest.mark.parametrize("dtype", list(TYPES))
def test_under_backward(dtype):
    g = torch.Generator().manual_seed(29)
    _say("attention autograd", dtype)
    q, k, v, g_, s = _inputs(g, dtype, 2, 70, 4, 2, 32, 40, state=True)
    lengths = torch.tensor([70, 31], device=_gpu())
    co, cs = _randn(g, 2, 70, 4, 40, dtype=dtype), torch.randn(2, 4, 32, 40, generator=g).to(_gpu())
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s)]
    o, end = quiver.linear_attention(*leaves[:3], g_, state=leaves[3], lengths=lengths, keep_state=True)
    torch.autograd.backward([o, end], [co, cs])
    want = quiver.linear_attention_grad(co, q, k, v, g_, state=s, lengths=lengths, grad_state=cs)
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    o, end = quiver.linear_attention(*leaves[:3], g_, state=leaves[3], lengths=lengths, keep_state=True)
    only = torch.autograd.grad(end, leaves, cs)
    want = quiver.linear_attention_grad(torch.zeros_like(co), q, k, v, g_, state=s, lengths=lengths, grad_state=cs)
    assert all(torch.equal(a, b) for a, b in zip(only, want))
    o = quiver.linear_attention(*leaves[:3], g_)
    first = torch.autograd.grad(o.float().sum(), leaves[0], create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiated twice"):
        first.float().sum().backward()
    with pytest.raises(ValueError, match="state_out"):
        quiver.linear_attention(*leaves[:3], g_, state=s, state_out=s)
    with torch.no_grad():
        assert not quiver.linear_attention(*leaves[:3], g_).requires_grad


def test_more_heads_than_a_launch_has_rows():
    """70,000 texts of one token, and of nine."""
    g = torch.Generator().manual_seed(37)
    _say("attention 70,000 texts")
    for tokens in (1, 9):
        q, k, v, g_, s = _inputs(g, "bf16", 70_000, tokens, 1, 1, 8, 8, state=True)
        got, last = quiver.linear_attention(q, k, v, g_, state=s, keep_state=True)
        part, end = quiver.linear_attention(q[-30:], k[-30:], v[-30:], g_, state=s[-30:], keep_state=True)
        want, size = _forward_64(q[-30:], k[-30:], v[-30:], g_, s[-30:], None, 8 ** -0.5)[0]
        _within(got[-30:], want, _bound(want, size, "bf16", 300))
        assert torch.equal(got[-30:], part) or tokens > 8  # nine tokens of thirty texts may go by segments
        assert torch.isfinite(got).all() and torch.isfinite(last).all()


def test_many_texts_next_to_one_another_within_a_token():
    """65,536 texts whose tokens lie 1 MB apart, longer than a buffer of 2^31 bytes: more than a launch cuts."""
    dev = _gpu()
    _say("attention 65,536 texts by token")
    g = torch.Generator(device=dev).manual_seed(61)
    q, k, v = (torch.randn((2_100, 65_536, 1, 8), generator=g, device=dev, dtype=torch.bfloat16).transpose(0, 1) for _ in range(3))
    decay = torch.tensor([-0.01], device=dev)
    got, last = quiver.linear_attention(q, k, v, decay, keep_state=True)
    grads = quiver.linear_attention_grad(v, q, k, v, decay)
    for some in (slice(0, 15), slice(-15, None)):
        few = [t[some].contiguous() for t in (q, k, v)]
        want, end = _forward_64(*few, decay, None, None, 8 ** -0.5)
        _within(got[some], want[0], _bound(want[0], want[1], "bf16", 8 + 2_100 + 256))
        _within(last[some], end[0], end[1] * (8 + 2_100 + 256) * 2.0**-23)
        for a, (b, size) in zip(grads[:3], _grad_64(few[2], *few, decay, None, None, 8 ** -0.5, None)):
            _within(a[some], b, _bound(b, size, "bf16", 8 + 8 + 2_100 + 257))


def test_under_inference_mode():
    g = torch.Generator().manual_seed(43)
    _say("attention inference mode")
    q, k, v, g_, s = _inputs(g, "bf16", 1, 2, 2, 1, 16, 16, state=True)
    want = quiver.linear_attention(q, k, v, g_, state=s, keep_state=True)
    with torch.inference_mode():
        state = s.clone()
        got = quiver.linear_attention(q, k, v, g_, state=state, state_out=state)
        assert got[1] is state and all(torch.equal(a, b) for a, b in zip(got, want))
        grads = [torch.ones(9, device=_gpu())]
        assert abs(quiver.clip_grad_norm(grads, 1.0, out=grads)[0][0][0].item() - 1 / 3) < 1e-6


def test_refusals():
    dev = _gpu()
    _say("attention refusals")
    f = torch.zeros((2, 6, 4, 16), device=dev)
    d = torch.zeros(4, device=dev)
    s = torch.zeros((2, 4, 16, 16), device=dev)
    n = torch.zeros(2, dtype=torch.int64, device=dev)
    a = lambda *x, **k: lambda: quiver.linear_attention(*x, **k)  # noqa: E731
    for call, word in [
            (a(f.double(), f, f, d), "float32"), (a(f, f.half(), f, d), "k is"), (a(f[0], f, f, d), "q must be"), (a(f, f[:, :5], f, d), "multiple"),
            (a(f, f[:, :, :3], f[:, :, :3], d), "multiple"), (a(f, f[..., :8], f, d), "multiple"), (a(f, f, f[:, :, :2], d), "multiple"),
            (a(f, f, f, d[:3]), "log_decay"), (a(f, f, f, d.double()), "log_decay"), (a(f, f, f, d.cpu()), "log_decay"),
            (a(f, f, f, d, state=s[:1]), "state must"), (a(f, f, f, d, state=s.half()), "state must"), (a(f, f, f, d, state_out=s[:, :2]), "state_out"),
            (a(f, f, f, d, lengths=n[:1]), "lengths must"), (a(f, f, f, d, lengths=n.float()), "lengths must"), (a(f, f, f, d, lengths=n.cpu()), "lengths are"),
            (a(f, f, f, d, scale=float("inf")), "scale"), (a(f.repeat(1, 1, 1, 17), f.repeat(1, 1, 1, 17), f, d), "256"), (a(f[..., :0], f[..., :0], f, d), "256"),
            (lambda: quiver.linear_attention_grad(f[:, :5], f, f, f, d), "grad must"), (lambda: quiver.linear_attention_grad(f, f, f, f, d, grad_state=s[..., :8]), "grad_state")]:
        with pytest.raises(ValueError, match=word):
            call()
    for call in (a(f, f, f, [0.0] * 4), a(f, f, f, d, lengths=[1, 2]), a(f, f, None, d)):
        with pytest.raises(TypeError):
            call()
