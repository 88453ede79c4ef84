"""The encoder operators' refusals, which need no GPU: every argument is checked before any device work.

The buffers are made-up addresses, so these tests run only where no GPU could take a call that is not
refused; the refusals on the GPU are in test_encoder_gpu.py, with real tensors.
"""

import ctypes as C

import pytest

import quiver_amd as quiver
from qvh_ctypes import LIB

EINVAL = -22


class LinearArgs(C.Structure):
    _fields_ = [("m", C.c_uint64), ("k", C.c_uint32), ("n", C.c_uint32), ("dtype", C.c_int), ("activation", C.c_int),
                ("x", C.c_void_p), ("x_stride", C.c_uint64), ("weight", C.c_void_p), ("weight_stride", C.c_uint64),
                ("bias", C.c_void_p), ("residual", C.c_void_p), ("residual_stride", C.c_uint64), ("out", C.c_void_p),
                ("out_stride", C.c_uint64), ("preactivation", C.c_void_p), ("preactivation_stride", C.c_uint64)]


class LinearGradArgs(C.Structure):
    _fields_ = [("m", C.c_uint64), ("k", C.c_uint32), ("n", C.c_uint32), ("dtype", C.c_int), ("activation", C.c_int),
                ("grad", C.c_void_p), ("grad_stride", C.c_uint64), ("preactivation", C.c_void_p),
                ("preactivation_stride", C.c_uint64), ("x", C.c_void_p), ("x_stride", C.c_uint64),
                ("weight", C.c_void_p), ("weight_stride", C.c_uint64), ("grad_x", C.c_void_p),
                ("grad_x_stride", C.c_uint64), ("grad_weight", C.c_void_p), ("grad_weight_stride", C.c_uint64),
                ("grad_bias", C.c_void_p)]


@pytest.fixture(scope="module")
def lib():
    torch = pytest.importorskip("torch")
    if torch.cuda.device_count() > 0:
        pytest.skip("made-up addresses: not where a GPU could run a call that is not refused")
    lib = C.CDLL(LIB)
    lib.qvh_last_error.restype = C.c_char_p
    return lib


def _refused(lib, status, word):
    assert status == EINVAL
    assert word in lib.qvh_last_error().decode()


BUF = C.c_void_p(1 << 20)  # never read: the calls fail before any device work


def _embed(lib, rows=10, dim=8, stride=8, dtype=0, tokens=BUF, index=8, count=4, out=BUF):
    return lib.qvh_embed_device(BUF, C.c_uint64(rows), C.c_uint32(dim), C.c_uint64(stride), dtype, tokens, index,
                                C.c_uint64(count), C.c_float(1.0), out, None)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(index=2), "int32"), (dict(dim=0), "dim"),
    (dict(dim=32769, stride=40000), "dim"), (dict(stride=7), "stride"), (dict(rows=2**32), "rows"),
    (dict(count=2**31), "tokens"), (dict(tokens=None), "null"), (dict(out=None), "null")])
def test_embed_refuses(lib, change, word):
    _refused(lib, _embed(lib, **change), word)


def test_embed_without_tokens_is_no_work(lib):
    assert _embed(lib, count=0, tokens=None, out=None) == 0


def _embed_grad(lib, rows=100, dim=8, stride=8, dtype=0, index=8, count=5000, grad=BUF, out=BUF, work=BUF, size=1 << 30):
    return lib.qvh_embed_grad_device(grad, C.c_uint64(stride), BUF, index, C.c_uint64(count), C.c_uint64(rows),
                                     C.c_uint32(dim), dtype, C.c_float(1.0), out, work, C.c_uint64(size), None)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=9), "dtype"), (dict(index=1), "int32"), (dict(dim=0), "dim"), (dict(stride=4), "stride"),
    (dict(grad=None), "null"), (dict(out=None), "null"), (dict(size=16), "workspace"), (dict(work=None), "workspace"),
    (dict(work=C.c_void_p((1 << 20) + 4)), "16-byte")])
def test_embed_grad_refuses(lib, change, word):
    _refused(lib, _embed_grad(lib, **change), word)


def test_embed_grad_workspace(lib):
    size = C.c_uint64(1)
    get = lambda rows, dim, count: (lib.qvh_embed_grad_workspace(C.c_uint64(rows), C.c_uint32(dim),  # noqa: E731
                                                                 C.c_uint64(count), C.byref(size)), size.value)
    assert get(100, 8, 10) == (0, 0)  # a small batch needs none
    assert get(100, 8, 100_000)[1] >= 16 * 100_000
    _refused(lib, get(100, 0, 10)[0], "dim")


def _linear(**change):
    a = LinearArgs(m=100, k=32, n=16, dtype=2, activation=0, x=1 << 20, x_stride=32, weight=1 << 20, weight_stride=32,
                   out=1 << 20, out_stride=16, residual_stride=16, preactivation_stride=16)
    for name, v in change.items():
        setattr(a, name, v)
    return a


# A float32 product large enough to be made of 16-bit parts, which lie in a workspace.
SPLIT = dict(m=4096, k=1024, n=1024, x_stride=1024, weight_stride=1024, out_stride=1024)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=4), "dtype"), (dict(activation=7), "activation"), (dict(m=2**31), "m must"), (dict(k=2**20 + 1), "k and n"),
    (dict(n=2**21), "k and n"), (dict(x=None), "x is null"), (dict(weight=None), "weight is null"),
    (dict(out=None), "out is null"), (dict(x_stride=31), "stride"), (dict(x_stride=2**22 + 1), "stride"),
    (dict(out_stride=15), "stride"), (dict(residual=1 << 20, residual_stride=3), "stride"),
    (dict(x=(1 << 20) + 1), "aligned"), (dict(bias=(1 << 20) + 1), "aligned"), (dict(dtype=0, **SPLIT), "workspace")])
def test_linear_refuses(lib, change, word):
    _refused(lib, lib.qvh_linear_device(C.byref(_linear(**change)), None, C.c_uint64(0), None), word)


def test_linear_workspace(lib):
    size = C.c_uint64(1)
    assert lib.qvh_linear_workspace(C.byref(_linear(m=4)), C.byref(size)) == 0 and size.value == 0
    assert lib.qvh_linear_workspace(C.byref(_linear(dtype=0)), C.byref(size)) == 0 and size.value == 0  # read as it is
    assert lib.qvh_linear_workspace(C.byref(_linear(dtype=0, **SPLIT)), C.byref(size)) == 0
    assert size.value >= 6 * (4096 + 1024) * 1024  # three 16-bit parts of both operands
    _refused(lib, lib.qvh_linear_workspace(None, C.byref(size)), "null")
    _refused(lib, lib.qvh_linear_workspace(C.byref(_linear()), None), "null")


def _linear_grad(**change):
    a = LinearGradArgs(m=100, k=32, n=16, dtype=2, activation=0, grad=1 << 20, grad_stride=16, preactivation_stride=16,
                       x=1 << 20, x_stride=32, weight=1 << 20, weight_stride=32, grad_x=1 << 20, grad_x_stride=32,
                       grad_weight=1 << 20, grad_weight_stride=32)
    for name, v in change.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(dtype=-2), "dtype"), (dict(activation=-1), "activation"), (dict(activation=2), "pre-activation"),
    (dict(grad=None), "grad is null"), (dict(grad_stride=15), "stride"), (dict(x=None), "x is null"),
    (dict(weight=None), "weight is null"), (dict(grad_x_stride=31), "stride"), (dict(grad_bias=(1 << 20) + 1), "aligned"),
    (dict(activation=1, preactivation=1 << 20), "workspace")])
def test_linear_grad_refuses(lib, change, word):
    _refused(lib, lib.qvh_linear_grad_device(C.byref(_linear_grad(**change)), None, C.c_uint64(0), None), word)


def _ortho(lib, batch=1, m=8, n=8, dtype=0, steps=5, co=(3.4445, -4.775, 2.0315), update=BUF, work=BUF, size=1 << 30):
    return lib.qvh_orthogonalize_device(update, C.c_uint64(batch), C.c_uint32(m), C.c_uint32(n), dtype, C.c_uint32(steps),
                                        *(C.c_float(c) for c in co), BUF, work, C.c_uint64(size), None)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=5), "dtype"), (dict(m=65537), "65536"), (dict(batch=65536), "65535"), (dict(co=(5.0, 0.0, 0.0)), "grow"),
    (dict(co=(float("nan"), 0.0, 0.0)), "grow"), (dict(co=(1.5, 3.0, 1.0)), "grow"), (dict(co=(1e30, 0.0, 0.0)), "grow"),
    (dict(update=None), "null"), (dict(m=300, n=300, size=100), "workspace"), (dict(n=2500, work=None), "workspace"),
    (dict(update=C.c_void_p((1 << 20) + 2)), "aligned")])
def test_orthogonalize_refuses(lib, change, word):
    _refused(lib, _ortho(lib, **change), word)


def test_orthogonalize_of_nothing_is_no_work(lib):
    assert _ortho(lib, batch=0, update=None, work=None) == 0
    assert _ortho(lib, m=0, update=None, work=None) == 0


def test_python_calls_want_device_tensors():
    torch = pytest.importorskip("torch")
    x = torch.zeros(4, 4)
    with pytest.raises(TypeError, match="torch tensor"):
        quiver.linear([[1.0]], x)
    for call in (lambda: quiver.linear(x, x), lambda: quiver.embed(x, torch.zeros(2, dtype=torch.int64)),
                 lambda: quiver.embed_grad(x, torch.zeros(4, dtype=torch.int64), 10), lambda: quiver.orthogonalize(x),
                 lambda: quiver.linear_grad(x, x, x)):
        with pytest.raises(ValueError, match="GPU memory"):
            call()
