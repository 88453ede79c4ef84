"""Blocks of an encoder, and their training step, on torch (ROCm) tensors in GPU memory.

    >>> x, h = quiver.block_norm(x, w_in, y=y, post_weight=w_out, gate=g, gate_activation="silu", scale=s)
    >>> o, state = quiver.linear_attention(q, k, v, log_decay, lengths=lengths, keep_state=True)
    >>> norm = quiver.clip_grad_norm(grads, 1.0, out=grads)[1]           # in front of the optimiser's step

They follow the rules of quiver_amd/encoder.py, whose layers go between them: types, streams, errors, strided rows,
workspaces, results that repeat bit for bit, torch's autograd where an input requires a gradient.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

from . import _quiver
from . import encoder as _encoder
from .encoder import _check, _dtypes, _node, _rows, _stream, _workspace

_GATES = {None: 0, "none": 0, "silu": 3, "sigmoid": 4}


def _gate_activation(name) -> int:
    try:
        return _GATES[name]
    except (KeyError, TypeError):
        raise ValueError(f"gate_activation must be none, silu or sigmoid, got {name!r}") from None


def _differentiated(*tensors) -> bool:
    """Whether autograd has to know of a call (as encoder._differentiated, of any number of inputs)."""
    if _encoder._torch is None:
        _encoder._load_torch()
    forward = _encoder._forward_ad
    try:
        for t in tensors:
            if t is not None and t.requires_grad:
                return _encoder._grad_enabled() or forward._current_level >= 0
        if forward._current_level < 0:
            return False
        return any(t is not None and forward.unpack_dual(t).tangent is not None for t in tensors)
    except AttributeError:
        return False  # not a tensor, which the call refuses


def _vector(name, v, dim, device, dtype):
    if v.__class__ is not _encoder._tensor or v.dtype is not dtype or v.device != device:
        _check(name, v, device, dtype)
    if v.shape != (dim,):
        raise ValueError(f"{name} must have shape ({dim},), got {tuple(v.shape)}")
    return v if v.is_contiguous() else v.contiguous()


def _matrix(name, m, shape, device, dtype):
    if m.__class__ is not _encoder._tensor or m.dtype is not dtype or m.device != device:
        _check(name, m, device, dtype)
    if m.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(m.shape)}")
    return (m, shape[-1]) if m.is_contiguous() else _rows(m, shape[-1])


def _written(tensors):
    """Tells autograd of tensors that a call has written to."""
    tensors = [t for t in tensors if not t.is_inference()]
    if tensors:
        _encoder._torch.autograd.graph.increment_version(tensors)


def _own_elements(name, t):
    """Refuses a result that could not take what is made aside of it, before anything is written."""
    if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{name} has elements that share memory")


def _pointer(t) -> int:
    return 0 if t is None else t.data_ptr()


# ---- norms around a block ---------------------------------------------------------------------


def block_norm(x, weight, y=None, post_weight=None, gate=None, gate_activation: Optional[str] = None, scale=None, eps: float = 1e-6):
    """From one block to the next: ``(r, h)`` with ``r = x + scale * act(gate) * norm(y) * post_weight`` and
    ``h = norm(r) * weight``, where ``norm(t) = t / sqrt(mean(t^2) + eps)`` over the last dimension.

    x [..., dim] is the residual stream, y of its shape the block's result, weight and post_weight [dim]. gate, a factor for
    each element, has y's shape (gate_activation: none, silu or sigmoid), scale [dim] is one for each column; both may be
    left out. Without y there is no block yet: ``h = norm(x) * weight`` alone. dim is at most 16384.
    """
    if _differentiated(x, weight, y, post_weight, gate, scale):
        return _node("BlockNorm", x, weight, y, post_weight, gate, gate_activation, scale, eps)
    return _block_norm(x, weight, y, post_weight, gate, gate_activation, scale, eps)


def _block_arguments(x, weight, y, post_weight, gate, gate_activation, scale):
    """What both passes check, as the calls take it: (tensors to hold, activation, arguments from y on)."""
    _check("x", x)
    device, dtype = x.device, x.dtype
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., dim], got shape {tuple(x.shape)}")
    dim = x.shape[-1]
    act = _gate_activation(gate_activation)
    w = _vector("weight", weight, dim, device, dtype)
    if y is None:
        for name, t in (("post_weight", post_weight), ("gate", gate), ("scale", scale)):
            if t is not None:
                raise ValueError(f"{name} belongs to a block's result y")
        return (w, None, None, None, None), act, (0, dim, 0, dim, w.data_ptr(), 0, 0)
    yr, ys = _matrix("y", y, x.shape, device, dtype)
    if post_weight is None:
        raise ValueError("y needs post_weight")
    pw = _vector("post_weight", post_weight, dim, device, dtype)
    gr, gs = (None, dim) if gate is None else _matrix("gate", gate, x.shape, device, dtype)
    sc = None if scale is None else _vector("scale", scale, dim, device, dtype)
    return (w, yr, pw, gr, sc), act, (yr.data_ptr(), ys, _pointer(gr), gs, w.data_ptr(), pw.data_ptr(), _pointer(sc))


def _block_norm(x, weight, y, post_weight, gate, gate_activation, scale, eps):
    held, act, args = _block_arguments(x, weight, y, post_weight, gate, gate_activation, scale)
    dim = x.shape[-1]
    xr, xs = _rows(x, dim)
    h = x.new_empty(x.shape)
    r = None if y is None else x.new_empty(x.shape)
    _quiver._block_norm(x.numel() // dim, dim, _dtypes[x.dtype], act, eps, xr.data_ptr(), xs, *args, _pointer(r), h.data_ptr(),
                        _stream(x.device))
    return h if y is None else (r, h)


def block_norm_grad(grad_h, r, weight, grad_r=None, y=None, post_weight=None, gate=None, gate_activation: Optional[str] = None,
                    scale=None, eps: float = 1e-6) -> Tuple:
    """Gradients of ``block_norm`` from its results': (grad_x, grad_weight, grad_y, grad_post_weight, grad_gate, grad_scale).

    r is what ``block_norm`` returned (x itself where there is no y), grad_r its gradient where it was used besides h. Gradients of
    what the block does not have are None.
    """
    return _block_norm_grad(grad_h, r, weight, grad_r, y, post_weight, gate, gate_activation, scale, eps, (True,) * 6)


def _block_norm_grad(grad_h, r, weight, grad_r, y, post_weight, gate, gate_activation, scale, eps, wanted):
    held, act, args = _block_arguments(r, weight, y, post_weight, gate, gate_activation, scale)
    device, dtype, dim = r.device, r.dtype, r.shape[-1]
    rr, rs = _rows(r, dim)
    gh, ghs = _matrix("grad_h", grad_h, r.shape, device, dtype)
    gr, grs = (None, dim) if grad_r is None else _matrix("grad_r", grad_r, r.shape, device, dtype)
    has = (True, True, y is not None, y is not None, gate is not None, scale is not None)
    matrix = (True, False, True, False, True, False)
    out = [r.new_empty(r.shape if m else (dim,)) if h and w else None for h, m, w in zip(has, matrix, wanted)]
    gx, gw, gy, gp, gg, gs = out
    rows, kind = r.numel() // dim, _dtypes[dtype]
    need = _quiver._block_norm_grad_workspace(rows, dim, kind, y is not None)
    work = _workspace(need, device) if need else None
    _quiver._block_norm_grad(rows, dim, kind, act, eps, gh.data_ptr(), ghs, _pointer(gr), grs, rr.data_ptr(), rs, *args, _pointer(gx),
                             _pointer(gy), _pointer(gg), _pointer(gw), _pointer(gp), _pointer(gs), _pointer(work), need, _stream(device))
    return tuple(out)


# ---- linear attention -------------------------------------------------------------------------


def linear_attention(q, k, v, log_decay, state=None, lengths=None, scale: Optional[float] = None, keep_state: bool = False,
                     state_out=None):
    """Attention without a softmax: ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T`` and ``out_t = scale * S_t^T q_t``, token by token.

    q is [batch, tokens, heads, dk], k [batch, tokens, kv_heads, dk], v [batch, tokens, kv_heads, dv], out [batch, tokens, heads, dv];
    kv_heads divides heads, and neighbouring heads share theirs. Views are read as they are where their last dimension is contiguous.
    log_decay, float32 [heads] and at most 0, is a constant: one that requires a gradient is refused where autograd records, and
    is passed detached. scale is ``dk ** -0.5`` where it is left out.
    lengths (int32 or int64 [batch], clamped to [0, tokens]): the tokens of each text in front of its padding, which changes no
    state and gives zeros. dk and dv are at most 256.

    A text can go on where it ended: state, float32 [batch, heads, dk, dv], is what it starts from (zeros where it is
    left out), and with keep_state the last one comes back too: (out, state). state_out takes it where it is given, and may be
    ``state`` itself, for texts that grow by a token at a time.
    """
    if _differentiated(q, k, v, state, log_decay):
        if _differentiated(log_decay):
            raise ValueError("log_decay is a constant and would get no gradient: pass it detached")
        if state_out is not None:
            raise ValueError("state_out is not for calls that autograd records")
        return _node("LinearAttention", q, k, v, log_decay, state, lengths, scale, keep_state)
    return _linear_attention(q, k, v, log_decay, state, lengths, scale, keep_state, state_out)


def _heads(name, t, device, dtype):
    """A [batch, tokens, heads, dim] tensor with contiguous rows of dim, and its strides."""
    if t.__class__ is not _encoder._tensor or t.dtype is not dtype or t.device != device:
        _check(name, t, device, dtype)
    if t.dim() != 4:
        raise ValueError(f"{name} must be [batch, tokens, heads, dim], got shape {tuple(t.shape)}")
    s = t.stride()
    if s[3] != 1 and t.shape[3] > 1:
        t = t.contiguous()
        s = t.stride()
    return t, s[:3]


def _state(name, t, shape, device):
    if not isinstance(t, _encoder._tensor):
        raise TypeError(f"{name} must be a torch tensor in GPU memory")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if t.dtype is not _encoder._torch.float32:
        raise ValueError(f"{name} must be float32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _attention_arguments(q, k, v, log_decay, state, lengths, scale):
    """(tensors to hold, sizes, scale, strides, arguments from log_decay on, shape of a state)."""
    _check("q", q)
    device, dtype = q.device, q.dtype
    q, qs = _heads("q", q, device, dtype)
    k, ks = _heads("k", k, device, dtype)
    v, vs = _heads("v", v, device, dtype)
    batch, tokens, heads, dk = q.shape
    kv_heads, dv = v.shape[2:]
    if k.shape != (batch, tokens, kv_heads, dk) or v.shape[:2] != q.shape[:2] or kv_heads < 1 or heads % kv_heads:
        raise ValueError("q must be [batch, tokens, heads, dk], k [batch, tokens, kv_heads, dk] and v [batch, tokens, kv_heads, dv] with "
                         f"heads a multiple of kv_heads, got shapes {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    log_decay = _state("log_decay", log_decay, (heads,), device)
    if state is not None:
        state = _state("state", state, (batch, heads, dk, dv), device)
    size = 0
    if lengths is not None:
        torch = _encoder._torch
        if not isinstance(lengths, torch.Tensor):
            raise TypeError("lengths must be a torch tensor in GPU memory")
        if lengths.device != device:
            raise ValueError(f"lengths are on {lengths.device}, the other tensors on {device}")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lengths must be int32 or int64, got {lengths.dtype}")
        if lengths.shape != (batch,):
            raise ValueError(f"lengths must have shape ({batch},), got {tuple(lengths.shape)}")
        lengths = lengths if lengths.is_contiguous() else lengths.contiguous()
        size = lengths.element_size()
    sizes = (batch, tokens, heads, kv_heads, dk, dv, _dtypes[dtype])
    if scale is None:
        scale = dk ** -0.5 if dk else 1.0
    return ((q, k, v, log_decay, state, lengths), sizes, scale, (*qs, *ks, *vs),
            (log_decay.data_ptr(), _pointer(lengths), size, _pointer(state)), (batch, heads, dk, dv))


def _linear_attention(q, k, v, log_decay, state, lengths, scale, keep_state, state_out=None):
    (q, k, v, *held), sizes, scale, strides, args, shape = _attention_arguments(q, k, v, log_decay, state, lengths, scale)
    device = q.device
    out = q.new_empty((*q.shape[:3], sizes[5]))
    last = filled = None
    if state_out is not None:
        last, filled = state_out, _state("state_out", state_out, shape, device)
        if filled is not last:
            _own_elements("state_out", last)
    elif keep_state:
        last = filled = held[0].new_empty(shape)  # log_decay's type
    args = (sizes, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, *args, _pointer(filled), out.data_ptr())
    stream = _stream(device)
    need = _quiver._attention(*args, 0, 0, stream)
    if need:
        work = _workspace(need, device)
        _quiver._attention(*args, work.data_ptr(), need, stream)
    if state_out is not None:
        if filled is not last:
            last.copy_(filled)
        else:
            _written([last])
    return out if last is None else (out, last)


def linear_attention_grad(grad, q, k, v, log_decay, state=None, lengths=None, scale: Optional[float] = None, grad_state=None) -> Tuple:
    """Gradients of ``linear_attention`` from its result's: (grad_q, grad_k, grad_v, grad_first).

    grad_state is the last state's gradient where that was used. grad_first is the gradient of ``state``, None where the texts
    started from zeros. Padding has gradients of zero.
    """
    (q, k, v, *held), sizes, scale, strides, args, shape = _attention_arguments(q, k, v, log_decay, state, lengths, scale)
    device = q.device
    grad, gs = _heads("grad", grad, device, q.dtype)
    if grad.shape != (*q.shape[:3], sizes[5]):
        raise ValueError(f"grad must have shape {(*q.shape[:3], sizes[5])}, got {tuple(grad.shape)}")
    if grad_state is not None:
        grad_state = _state("grad_state", grad_state, shape, device)
    contiguous = _encoder._torch.contiguous_format
    gq, gk, gv = (_encoder._torch.empty_like(t, memory_format=contiguous) for t in (q, k, v))
    first = None if state is None else _encoder._torch.empty(shape, dtype=_encoder._torch.float32, device=device)
    args = (sizes, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), (*strides, *gs), *args, grad.data_ptr(), _pointer(grad_state),
            gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), _pointer(first))
    stream = _stream(device)
    need = _quiver._attention_grad(*args, 0, 0, stream)
    if need:
        work = _workspace(need, device)
        _quiver._attention_grad(*args, work.data_ptr(), need, stream)
    return gq, gk, gv, first


# ---- the gradients' norm ----------------------------------------------------------------------


def _gradients(name, tensors):
    """The tensors as contiguous ones, and lists of their addresses, elements and types."""
    torch = _encoder._load_torch()
    tensors = list(tensors)
    held, pointers, counts, types = [], [], [], []
    device = None
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be torch tensors in GPU memory")
        if device is None:
            _check(name, t)
            device = t.device
        elif t.device != device:
            raise ValueError(f"{name}: one is on {t.device}, the others on {device}")
        kind = _dtypes.get(t.dtype)
        if kind is None:
            raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
        if t.layout is not torch.strided:
            raise ValueError(f"{name} must be dense tensors")
        if not t.is_contiguous():
            t = t.contiguous()
        held.append(t)
        pointers.append(t.data_ptr())
        counts.append(t.numel())
        types.append(kind)
    return tensors, held, pointers, counts, types, device


def _run_clip(pointers, outs, counts, types, max_norm, eps, device):
    norm = _encoder._torch.empty((), dtype=_encoder._torch.float32, device=device)
    need = _quiver._clip_grad_norm_most(len(pointers))
    work = _workspace(need, device)
    _quiver._clip_grad_norm(pointers, outs, counts, types, max_norm, eps, norm.data_ptr(), work.data_ptr(), need, _stream(device))
    return norm


def _own_device():
    return _encoder._load_torch().device("cuda", _quiver._device_index())


def grad_norm(grads: Sequence):
    """The norm over all of a list of tensors, ``sqrt`` of the sum of their squares, as a float32 tensor of no dimensions.

    The tensors may be of different types and shapes; sums are fp64. The norm of no tensors is zero.
    """
    _, held, pointers, counts, types, device = _gradients("grads", grads)
    return _run_clip(pointers, [], counts, types, 0.0, 0.0, device or _own_device())


def clip_grad_norm(grads: Sequence, max_norm: float, out: Optional[Sequence] = None, eps: float = 1e-6) -> Tuple:
    """Gradients scaled down to a limit of their common norm: (list of ``grad * min(1, max_norm / (norm + eps))``, norm).

    grads are the tensors of a model, of any of the three types each. out takes the results where it is given: tensors of
    the same shapes and types, or ``out=grads`` to scale them in place. norm is ``grad_norm`` of the gradients as they came
    in, and stays on the device. One that is infinite leaves zeros (NaN in place of infinities), NaN leaves NaN; gradients
    of zeros stay, with an eps of 0 too. The results are constants to autograd.
    """
    grads, held, pointers, counts, types, device = _gradients("grads", grads)
    torch = _encoder._torch
    if out is None:
        results = [torch.empty_like(t, requires_grad=False, memory_format=torch.contiguous_format) for t in held]
        outs = [t.data_ptr() for t in results]
        return results, _run_clip(pointers, outs, counts, types, max_norm, eps, device or _own_device())
    results, filled, outs, out_counts, out_types, _ = _gradients("out", out)
    if len(results) != len(grads) or out_types != types or any(a.shape != b.shape for a, b in zip(results, grads)):
        raise ValueError("out must hold a tensor of each gradient's shape and type")
    if results and results[0].device != device:
        raise ValueError(f"out is on {results[0].device}, the gradients on {device}")
    # A result that is not contiguous is made aside; its gradient, where it is the same tensor, was copied already.
    aside = [(t, f) for t, f in zip(results, filled) if t is not f]
    for t, _ in aside:
        _own_elements("out", t)
    norm = _run_clip(pointers, outs, counts, types, max_norm, eps, device or _own_device())
    with torch.no_grad():
        for t, f in aside:
            t.copy_(f)
    _written([t for t, f in zip(results, filled) if t is f] if aside else results)
    return results, norm
