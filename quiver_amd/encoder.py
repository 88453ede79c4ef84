"""The encoder in front of an index, on torch (ROCm) tensors in GPU memory.

    >>> tokens -> rows of a table -> layers -> vectors -> index.search
    >>> h = quiver.embed(table, tokens)                                  # [n, dim]
    >>> y, z = quiver.linear(h, w, bias=b, activation="gelu", keep_preactivation=True)
    >>> dh, dw, db = quiver.linear_grad(dy, h, w, preactivation=z, activation="gelu")
    >>> dtable = quiver.embed_grad(dh, tokens, len(table))
    >>> w -= lr * quiver.orthogonalize(momentum)                         # momentum follows dw

Tensors are float32, float16 or bfloat16, the same for all matrices of a call; sums are fp32 and
results are rounded once. (One thing in between is too: where ``linear_grad`` has an activation and 16-bit
tensors, the gradient behind it is rounded to their type for the products.) Calls run on torch's current stream, return
without waiting, and repeat bit for bit; other shapes, strides, alignments, batches or results asked for may
change the last bits. Workspaces come from torch's allocator. ``embed`` and ``linear`` take part in
torch's autograd where an input requires a gradient; results of ``embed_grad`` and ``linear_grad``, which
are its backward passes, are constants to it. Wrong arguments raise ``ValueError``
(``TypeError`` where something is not a tensor). Rows may be strided; any other layout is copied
first. The reference has no counterpart: its callers bring finished vectors
(python/quiver/__init__.py:166-251).
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

from . import _quiver

_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3}
_MAX_STRIDE = 1 << 22

_torch = None
_tensor = None
_dtypes = {}
_raw_stream = None
_forward_ad = None
_grad_enabled = None


def _load_torch():
    """torch, once it is known to share this library's HIP runtime."""
    global _torch, _tensor, _raw_stream, _forward_ad, _grad_enabled
    if _torch is None:
        import torch

        runtimes = set(_quiver._hip_runtimes())
        if len(runtimes) > 1:
            raise ValueError("torch and quiver_amd run on different HIP runtimes in this process "
                             f"({', '.join(sorted(runtimes))}), so device tensors cannot be shared: "
                             "import torch before quiver_amd")
        _dtypes.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        # The current stream's handle alone; torch.cuda.current_stream makes an object of it, at 2 us a call.
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        _tensor = torch.Tensor
        _forward_ad = torch.autograd.forward_ad
        _grad_enabled = torch.is_grad_enabled
        _torch = torch
    return _torch


def _differentiated(x, weight=None, bias=None, residual=None) -> bool:
    """Whether autograd has to know of a call: an input requires a gradient, or carries a tangent."""
    if _torch is None:
        _load_torch()
    try:
        if (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)
                or (residual is not None and residual.requires_grad)):
            return _grad_enabled() or _forward_ad._current_level >= 0
        if _forward_ad._current_level < 0:
            return False
        return any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in (x, weight, bias, residual))
    except AttributeError:
        return False  # not a tensor, which the call refuses


def _node(name: str, *args):
    from . import autograd

    return getattr(autograd, name).apply(*args)


def _check(name: str, x, device=None, dtype=None):
    """A floating device tensor, on `device` and of `dtype` where those are given."""
    if x.__class__ is _tensor:  # what nearly every call finds, in a third of the time
        if dtype is not None:
            if x.dtype is dtype and x.device == device:
                return
        elif x.is_cuda and x.dtype in _dtypes and x.device.index == _quiver._device_index():
            return
    torch = _load_torch()
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor in GPU memory")
    if not x.is_cuda:
        raise ValueError(f"{name} must be in GPU memory, got a tensor on {x.device}")
    if device is None:
        if x.device.index != _quiver._device_index():
            raise ValueError(f"{name} is on {x.device}, the library on cuda:{_quiver._device_index()}")
    elif x.device != device:
        raise ValueError(f"{name} is on {x.device}, the other tensors on {device}")
    if x.dtype not in _dtypes:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {x.dtype}")
    if dtype is not None and x.dtype != dtype:
        raise ValueError(f"{name} is {x.dtype}, the other tensors {dtype}")


def _rows(x, cols: int):
    """x as rows of `cols` contiguous elements, and the elements between rows."""
    if x.is_contiguous():
        return x, cols
    if x.dim() != 2:
        x = x.reshape(x.numel() // cols if cols else 0, cols)
        if x.is_contiguous():
            return x, cols
    stride = x.stride(0)
    if x.stride(1) != 1 or stride < cols or stride > _MAX_STRIDE:
        return x.contiguous(), cols
    return x, stride


def _tokens(tokens, device):
    torch = _load_torch()
    if not isinstance(tokens, torch.Tensor):
        raise TypeError("tokens must be a torch tensor in GPU memory")
    if tokens.device != device:
        raise ValueError(f"tokens are on {tokens.device}, the other tensors on {device}")
    if tokens.dtype is torch.int64:
        size = 8
    elif tokens.dtype is torch.int32:
        size = 4
    else:
        raise ValueError(f"tokens must be int32 or int64, got {tokens.dtype}")
    return tokens if tokens.is_contiguous() else tokens.contiguous(), size


def _activation(name) -> int:
    try:
        return _ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be none, relu, gelu or silu, got {name!r}") from None


def _stream(device) -> int:
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return _torch.cuda.current_stream(device).cuda_stream


def _workspace(nbytes: int, device):
    return _torch.empty(nbytes, dtype=_torch.uint8, device=device)


def embed(table, tokens, scale: float = 1.0):
    """Rows of a table by token: ``scale * table[tokens]``, of shape ``tokens.shape + (dim,)``.

    A token outside the table gives a row of zeros: -1 is padding, and the label of an empty search
    result. Tokens are int32 or int64; dim is at most 32768.
    """
    return _node("Embed", table, tokens, scale) if _differentiated(table) else _embed(table, tokens, scale)


def _embed(table, tokens, scale):
    _check("table", table)
    if table.dim() != 2:
        raise ValueError(f"table must be [rows, dim], got shape {tuple(table.shape)}")
    device = table.device
    tokens, size = _tokens(tokens, device)
    dim = table.shape[1]
    rows, stride = _rows(table, dim)
    out = table.new_empty(tokens.shape + (dim,))
    _quiver._embed(rows.data_ptr(), table.shape[0], dim, stride, _dtypes[table.dtype], tokens.data_ptr(), size,
                   tokens.numel(), scale, out.data_ptr(), _stream(device))
    return out


def embed_grad(grad, tokens, rows: int, scale: float = 1.0):
    """The table's gradient [rows, dim] from the gradient of ``embed``'s result.

    Each row is ``scale`` times the sum of the gradients of the tokens that name it, in fp32 and in an order
    that depends on the tokens alone; zero where no token does. Tokens outside the table add nothing.
    """
    _check("grad", grad)
    device = grad.device
    tokens, size = _tokens(tokens, device)
    if grad.dim() < 1 or grad.shape[:-1] != tokens.shape:
        raise ValueError(f"grad must have shape tokens.shape + (dim,), got {tuple(grad.shape)} for tokens "
                         f"{tuple(tokens.shape)}")
    rows = int(rows)
    if rows < 0:
        raise ValueError("rows must be non-negative")
    dim = grad.shape[-1]
    g, stride = _rows(grad, dim)
    out = grad.new_empty((rows, dim))
    need = _quiver._embed_grad_workspace(rows, dim, tokens.numel())
    work = _workspace(need, device) if need else None
    _quiver._embed_grad(g.data_ptr(), stride, tokens.data_ptr(), size, tokens.numel(), rows, dim, _dtypes[grad.dtype],
                        scale, out.data_ptr(), work.data_ptr() if need else 0, need, _stream(device))
    return out


def linear(x, weight, bias=None, activation: Optional[str] = None, residual=None, keep_preactivation: bool = False):
    """``act(x @ weight.T + bias) + residual`` in one product.

    x is [..., k], weight [n, k], bias [n], residual of the result's shape [..., n]; activation is none,
    relu, gelu (with the error function) or silu. With keep_preactivation the sum in front of the
    activation, which ``linear_grad`` takes, comes back too: (result, preactivation).
    """
    if _differentiated(x, weight, bias, residual):
        return _node("Linear", x, weight, bias, residual, activation, keep_preactivation)
    return _linear(x, weight, bias, activation, residual, keep_preactivation)


def _linear(x, weight, bias, activation, residual, keep_preactivation):
    _check("x", x)
    device, dtype = x.device, x.dtype
    _check("weight", weight, device, dtype)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., k] and weight [n, k], got shapes {tuple(x.shape)} and {tuple(weight.shape)}")
    n, k = weight.shape
    act = _activation(activation)
    shape = x.shape[:-1] + (n,)
    xr, xs = (x, k) if x.is_contiguous() else _rows(x, k)
    wr, ws = (weight, k) if weight.is_contiguous() else _rows(weight, k)
    br = rr = None
    rs = n
    if bias is not None:
        _check("bias", bias, device, dtype)
        if bias.shape != (n,):
            raise ValueError(f"bias must have shape ({n},), got {tuple(bias.shape)}")
        br = bias if bias.is_contiguous() else bias.contiguous()
    if residual is not None:
        _check("residual", residual, device, dtype)
        if residual.shape != shape:
            raise ValueError(f"residual must have shape {tuple(shape)}, got {tuple(residual.shape)}")
        rr, rs = _rows(residual, n)
    out = x.new_empty(shape)
    pre = x.new_empty(shape) if keep_preactivation else None
    m = out.numel() // n if n else 0
    args = (m, k, n, _dtypes[dtype], act, xr.data_ptr(), xs, wr.data_ptr(), ws, 0 if br is None else br.data_ptr(),
            0 if rr is None else rr.data_ptr(), rs, out.data_ptr(), n, 0 if pre is None else pre.data_ptr(), n)
    stream = _stream(device)
    need = _quiver._linear(*args, 0, 0, stream)  # enqueued where it needs no workspace
    if need:
        work = _workspace(need, device)
        _quiver._linear(*args, work.data_ptr(), need, stream)
    return out if pre is None else (out, pre)


def linear_grad(grad, x, weight, preactivation=None, activation: Optional[str] = None, bias: bool = True,
                inputs: bool = True) -> Tuple:
    """Gradients of ``linear`` from its result's gradient: (grad_x, grad_weight, grad_bias).

    preactivation is what ``linear`` kept; it is needed with an activation only. grad_bias is None without
    ``bias``, grad_x without ``inputs``. The residual's gradient is ``grad`` itself. With an activation and 16-bit
    tensors, ``grad * act'(preactivation)`` enters the products rounded to their type (grad_bias does not use
    the rounded values); in float16 it is infinite past 65,504 and keeps multiples of 2^-24 only.
    """
    return _linear_grad(grad, x, weight, preactivation, activation, bias, inputs, True)


def _linear_grad(grad, x, weight, preactivation, activation, bias, inputs, weights):
    _check("grad", grad)
    device, dtype = grad.device, grad.dtype
    _check("x", x, device, dtype)
    _check("weight", weight, device, dtype)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., k] and weight [n, k], got shapes {tuple(x.shape)} and {tuple(weight.shape)}")
    n, k = weight.shape
    if grad.shape != x.shape[:-1] + (n,):
        raise ValueError(f"grad must have shape {tuple(x.shape[:-1] + (n,))}, got {tuple(grad.shape)}")
    act = _activation(activation)
    pr, ps = None, n
    if act != 0:
        if preactivation is None:
            raise ValueError("an activation's gradient needs the pre-activation that linear kept")
        _check("preactivation", preactivation, device, dtype)
        if preactivation.shape != grad.shape:
            raise ValueError(f"preactivation must have shape {tuple(grad.shape)}, got {tuple(preactivation.shape)}")
        pr, ps = _rows(preactivation, n)
    gr, gs = _rows(grad, n)
    xr, xs = _rows(x, k)
    wr, ws = _rows(weight, k)
    m = grad.numel() // n if n else x.numel() // k if k else 0
    gx = x.new_empty(x.shape) if inputs else None
    gw = weight.new_empty((n, k)) if weights else None
    gb = weight.new_empty((n,)) if bias else None
    args = (m, k, n, _dtypes[dtype], act, gr.data_ptr(), gs, 0 if pr is None else pr.data_ptr(), ps, xr.data_ptr(), xs,
            wr.data_ptr(), ws, 0 if gx is None else gx.data_ptr(), k, 0 if gw is None else gw.data_ptr(), k,
            0 if gb is None else gb.data_ptr())
    stream = _stream(device)
    need = _quiver._linear_grad(*args, 0, 0, stream)
    if need:
        work = _workspace(need, device)
        _quiver._linear_grad(*args, work.data_ptr(), need, stream)
    return gx, gw, gb


def orthogonalize(update, steps: int = 5, coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315)):
    """Newton-Schulz steps on an update [..., m, n], each matrix by itself (as the Muon optimiser does).

    From ``X = G / |G|_F``, ``steps`` times ``X <- a X + (b A + c A A) X`` with ``A = X X^T`` (from the right
    where m > n): the singular vectors stay, every singular value s goes through a s + b s^3 + c s^5.
    The default coefficients bring all but tiny ones near 1 in five steps. A zero matrix stays zero.
    Coefficients that let singular values grow without bound are refused. It makes an optimiser's steps
    and has no derivative: a backward pass through it raises an error.
    """
    if _differentiated(update):
        return _node("Orthogonalize", update, steps, coefficients)
    return _orthogonalize(update, steps, coefficients)


def _orthogonalize(update, steps, coefficients):
    _check("update", update)
    if update.dim() < 2:
        raise ValueError(f"update must be [..., m, n], got shape {tuple(update.shape)}")
    if len(coefficients) != 3:
        raise ValueError("coefficients must be three numbers")
    steps = int(steps)
    if steps < 0 or steps > 1000:
        raise ValueError("steps must be in [0, 1000]")
    a, b, c = (float(v) for v in coefficients)
    g = update.contiguous()
    m, n = g.shape[-2:]
    batch = g.numel() // (m * n) if m and n else 0
    out = g.new_empty(g.shape)
    need = _quiver._orthogonalize_workspace(batch, m, n)
    work = _workspace(need, g.device) if need else None
    _quiver._orthogonalize(g.data_ptr(), batch, m, n, _dtypes[g.dtype], steps, a, b, c, out.data_ptr(),
                           work.data_ptr() if need else 0, need, _stream(g.device))
    return out
