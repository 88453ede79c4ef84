"""The refusals of the blocks' operators, which need no GPU: every argument is checked before any device work.

As tests/test_encoder.py: made-up addresses, so only where no GPU could take a call that is not refused.
"""

import ctypes as C

import pytest

import quiver_amd as quiver
from block_launches import U3, AttentionArgs, AttentionGradArgs, Gradient, NormArgs, NormGradArgs
from test_encoder import BUF, _refused, lib  # noqa: F401  (lib: the fixture)


def _norm(lib, **change):  # noqa: F811
    a = dict(rows=8, dim=16, dtype=2, gate_activation=0, eps=1e-6, x=BUF, x_stride=16, y=BUF, y_stride=16, gate=BUF, gate_stride=16,
             weight=BUF, post_weight=BUF, scale=BUF, r=BUF, h=BUF)
    a.update(change)
    return lib.qvh_block_norm_device(C.byref(NormArgs(**a)), None)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=3), "dtype"), (dict(dim=0), "dim"), (dict(dim=16_385, x_stride=20_000), "dim"), (dict(rows=2**31), "rows"),
    (dict(gate_activation=1), "activation"), (dict(gate_activation=2), "activation"), (dict(gate_activation=5), "activation"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(x=None), "null x"),
    (dict(x_stride=15), "x's stride"), (dict(y_stride=2**22 + 1), "y's stride"), (dict(gate_stride=3), "gate's stride"),
    (dict(weight=None), "null weight"), (dict(post_weight=None), "post_weight"), (dict(r=None), "null r"), (dict(h=None), "null h"),
    (dict(y=None), "belong to y"), (dict(y=None, gate=None, post_weight=None), "belong to y")])
def test_block_norm_refuses(lib, change, word):  # noqa: F811
    _refused(lib, _norm(lib, **change), word)


def test_block_norm_of_no_rows_is_no_work(lib):  # noqa: F811
    assert _norm(lib, rows=0, x=None, y=None, gate=None, r=None, h=None) == 0


def _norm_grad(lib, work=BUF, size=1 << 30, **change):  # noqa: F811
    a = dict(rows=8, dim=16, dtype=2, gate_activation=0, eps=1e-6, grad_h=BUF, grad_h_stride=16, grad_r=BUF, grad_r_stride=16, r=BUF,
             r_stride=16, y=BUF, y_stride=16, gate=BUF, gate_stride=16, weight=BUF, post_weight=BUF, scale=BUF, grad_x=BUF, grad_y=BUF,
             grad_gate=BUF, grad_weight=BUF, grad_post=BUF, grad_scale=BUF)
    a.update(change)
    return lib.qvh_block_norm_grad_device(C.byref(NormGradArgs(**a)), work, C.c_uint64(size), None)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=-1), "dtype"), (dict(grad_h=None), "null grad_h"), (dict(r=None), "null r"), (dict(grad_r_stride=8), "grad_r's stride"),
    (dict(weight=None), "null weight"), (dict(gate=None), "grad_gate without"), (dict(scale=None), "grad_scale without"),
    (dict(y=None), "belong to y"), (dict(size=64), "workspace"), (dict(work=None), "workspace"), (dict(work=C.c_void_p((1 << 20) + 8)), "16-byte")])
def test_block_norm_grad_refuses(lib, change, word):  # noqa: F811
    _refused(lib, _norm_grad(lib, **change), word)


def _attention_args(**change):
    a = dict(batch=2, tokens=100, heads=4, kv_heads=2, dk=32, dv=48, dtype=0, scale=1.0, q=BUF, q_stride=U3(12_800, 128, 32), k=BUF,
             k_stride=U3(6_400, 64, 32), v=BUF, v_stride=U3(9_600, 96, 48), log_decay=BUF, lengths=None, index_bytes=0, state=None,
             state_out=None, out=BUF)
    a.update(change)
    return AttentionArgs(**a)


FAR = U3(2**40, 128, 32)
ATTENTION = [(dict(dtype=7), "dtype"), (dict(heads=0), "heads"), (dict(kv_heads=3), "heads"), (dict(kv_heads=0), "heads"), (dict(dk=0), "dk"),
             (dict(dk=257), "dk"), (dict(dv=257), "dv"), (dict(tokens=2**31), "below 2^31"), (dict(batch=2**31), "below 2^31"),
             (dict(batch=2**20), "2^21"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(log_decay=None), "log_decay"),
             (dict(state=BUF, state_out=C.c_void_p((1 << 20) + 64)), "overlaps"), (dict(lengths=BUF, index_bytes=2), "lengths"), (dict(q=None), "null q"), (dict(k=None), "null k"), (dict(v=None), "null v"),
             (dict(q_stride=FAR), "q's strides"), (dict(v_stride=FAR), "v's strides")]


@pytest.mark.parametrize("change,word", [*ATTENTION, (dict(out=None), "null result")])
def test_attention_refuses(lib, change, word):  # noqa: F811
    _refused(lib, lib.qvh_attention_device(C.byref(_attention_args(**change)), BUF, C.c_uint64(1 << 30), None), word)


def test_attention_wants_its_workspace(lib):  # noqa: F811
    a = _attention_args(tokens=4_096)
    need = C.c_uint64()
    assert lib.qvh_attention_workspace(C.byref(a), C.byref(need)) == 0 and need.value > 0 and need.value % (8 * 32 * 48 * 4) == 0
    _refused(lib, lib.qvh_attention_device(C.byref(a), BUF, C.c_uint64(need.value - 1), None), "workspace")
    _refused(lib, lib.qvh_attention_device(C.byref(a), None, need, None), "workspace")
    _refused(lib, lib.qvh_attention_device(C.byref(a), C.c_void_p((1 << 20) + 4), need, None), "16-byte")
    for few in (0, 1, 4):  # the recurrence itself
        assert lib.qvh_attention_workspace(C.byref(_attention_args(tokens=few)), C.byref(need)) == 0 and need.value == 0
    assert lib.qvh_attention_workspace(C.byref(_attention_args(tokens=4_096, batch=200)), C.byref(need)) == 0 and need.value == 0


def test_attention_of_no_texts_is_no_work(lib):  # noqa: F811
    a = _attention_args(batch=0, q=None, k=None, v=None, log_decay=None, out=None)
    assert lib.qvh_attention_device(C.byref(a), None, C.c_uint64(0), None) == 0
    g = AttentionGradArgs(forward=a)
    assert lib.qvh_attention_grad_device(C.byref(g), None, C.c_uint64(0), None) == 0
    assert lib.qvh_attention_device(C.byref(_attention_args(tokens=0, q=None, k=None, v=None, out=None)), None, C.c_uint64(0), None) == 0


@pytest.mark.parametrize("change,word", [*ATTENTION[:8], (dict(grad=None), "null grad"), (dict(grad_stride=FAR), "grad's strides"),
                                         (dict(grad_q=None), "null result"), (dict(grad_k=None), "null result"), (dict(grad_v=None), "null result")])
def test_attention_grad_refuses(lib, change, word):  # noqa: F811
    own = {k: v for k, v in change.items() if k.startswith("grad")}
    forward = _attention_args(**{k: v for k, v in change.items() if k not in own})
    a = dict(forward=forward, grad=BUF, grad_stride=U3(19_200, 192, 48), grad_q=BUF, grad_k=BUF, grad_v=BUF)
    a.update(own)
    _refused(lib, lib.qvh_attention_grad_device(C.byref(AttentionGradArgs(**a)), BUF, C.c_uint64(1 << 30), None), word)


def _clip(lib, grads, max_norm=1.0, eps=1e-6, work=BUF, size=1 << 20):  # noqa: F811
    array = (Gradient * max(len(grads), 1))(*[Gradient(*g) for g in grads])
    return lib.qvh_clip_grad_norm_device(array, C.c_uint64(len(grads)), C.c_float(max_norm), C.c_float(eps), BUF, work, C.c_uint64(size), None)


A = 1 << 20


@pytest.mark.parametrize("grads,more,word", [
    ([(A, A, 10, 4)], {}, "dtype"), ([(None, A, 10, 0)], {}, "null"), ([(A, None, 10, 0)], {}, "null"), ([(A, A, 2**40 + 1, 0)], {}, "2\\^40"),
    ([(A, A, 10, 0)], dict(max_norm=-1.0), "max_norm"), ([(A, A, 10, 0)], dict(max_norm=float("inf")), "max_norm"),
    ([(A, A, 10, 0)], dict(max_norm=float("nan")), "max_norm"), ([(A, A, 10, 0)], dict(eps=-1.0), "eps"), ([(A, A, 10, 0)], dict(size=0), "workspace"),
    ([(A, A, 10, 0)], dict(work=None), "workspace"), ([(A, A, 10, 0)], dict(work=C.c_void_p(A + 8)), "16-byte"),
    ([(A, A, 10, 0), (A, A, 10, 0)], {}, "overlap"), ([(A, A, 10, 0), (A + 36, A + 36, 10, 0)], {}, "overlap"),
    ([(A, A + 4096, 10, 0), (A + 4096, A + 8192, 3, 1)], {}, "another gradient"), ([(A, A + 8, 10, 0)], {}, "another gradient"),
    ([(A, A + 4096, 2**30, 0), (A + 2**22, A + 2**33, 3, 1)], {}, "another gradient")])
def test_clip_refuses(lib, grads, more, word):  # noqa: F811
    status = _clip(lib, grads, **more)
    assert status == -22
    import re

    assert re.search(word, lib.qvh_last_error().decode())


def test_clip_workspace(lib):  # noqa: F811
    need = C.c_uint64()
    assert lib.qvh_grad_norm_workspace(C.c_uint64(0), C.byref(need)) == 0 and need.value == 0
    assert lib.qvh_grad_norm_workspace(C.c_uint64(10**6), C.byref(need)) == 0 and need.value >= 8 * 10**6 // 120
    _refused(lib, lib.qvh_grad_norm_workspace(C.c_uint64(2**20 + 1), C.byref(need)), "2^20")
    _refused(lib, lib.qvh_grad_norm_workspace(C.c_uint64(1), None), "null")


def test_python_calls_want_device_tensors():
    torch = pytest.importorskip("torch")
    if torch.cuda.device_count() > 0:
        pytest.skip("the library would take them to a device")
    f = torch.zeros(4, 8)
    q = torch.zeros(1, 2, 1, 8)
    for call in (lambda: quiver.block_norm(f, f[0]), lambda: quiver.block_norm_grad(f, f, f[0]),
                 lambda: quiver.linear_attention(q, q, q, torch.zeros(1)), lambda: quiver.linear_attention_grad(q, q, q, q, torch.zeros(1)),
                 lambda: quiver.grad_norm([f]), lambda: quiver.clip_grad_norm([f], 1.0)):
        with pytest.raises(ValueError, match="GPU memory"):
            call()
    for call in (lambda: quiver.block_norm(1.0, f), lambda: quiver.linear_attention(None, q, q, f), lambda: quiver.grad_norm([1.0])):
        with pytest.raises(TypeError):
            call()


def test_a_decay_that_wants_a_gradient_is_refused():
    """It would get none, without a word. Refused ahead of all else, so that CPU tensors do."""
    torch = pytest.importorskip("torch")
    q = torch.zeros(1, 2, 1, 8)
    decay = torch.zeros(1, requires_grad=True)
    for inputs in ((q, q, q), (q.clone().requires_grad_(), q, q)):
        with pytest.raises(ValueError, match="log_decay is a constant"):
            quiver.linear_attention(*inputs, decay)
        with pytest.raises(ValueError, match="log_decay is a constant"):
            quiver.linear_attention(*inputs, decay * 2, keep_state=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.zeros(1), torch.ones(1))
        with pytest.raises(ValueError, match="log_decay is a constant"):
            quiver.linear_attention(q, q, q, dual)


def test_a_decay_is_taken_detached_or_without_autograd():
    torch = pytest.importorskip("torch")
    if torch.cuda.device_count() > 0:
        pytest.skip("the library would take the tensors to a device")
    q = torch.zeros(1, 2, 1, 8)
    decay = torch.zeros(1, requires_grad=True)
    with pytest.raises(ValueError, match="GPU memory"):
        quiver.linear_attention(q, q, q, decay.detach())
    with torch.no_grad(), pytest.raises(ValueError, match="GPU memory"):
        quiver.linear_attention(q, q, q, decay)
