"""The encoder's calls as nodes of torch's autograd graph (quiver_amd/encoder.py makes them where an input asks for it).

The backward passes are ``embed_grad`` and ``linear_grad``. They are not differentiable themselves, and
nothing here has a forward-mode derivative: either raises an error.
"""

from __future__ import annotations

import torch

from . import encoder


class _Once(torch.autograd.Function):
    """A gradient that a graph is made of (create_graph): one that follows from `sources` and has no derivative. (torch's
    own once_differentiable looks at the incoming gradient alone, and would take it as constant in x and the weight.)"""

    @staticmethod
    def forward(ctx, name, gradient, *sources):
        ctx.name = name
        return gradient()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} cannot be differentiated twice")


def _once(name, gradient, *sources):
    return _Once.apply(name, gradient, *sources) if torch.is_grad_enabled() else gradient()


class Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale):
        rows = encoder._embed(table, tokens, scale)
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.scale = table.shape[0], scale
        return rows

    @staticmethod
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        return _once("embed", lambda: encoder.embed_grad(grad, tokens, ctx.rows, ctx.scale), grad), None, None


class Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, keep):
        layer = any(ctx.needs_input_grad[:3])  # not the residual alone
        slope = layer and encoder._activation(activation) != 0
        y = encoder._linear(x, weight, bias, activation, residual, keep or slope)
        y, pre = y if keep or slope else (y, None)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        if layer:
            ctx.save_for_backward(x, weight, pre if slope else None)
        return (y, pre) if keep else y

    @staticmethod
    def backward(ctx, grad, grad_pre=None):
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        gx = gw = gb = None
        if want_x or want_w or want_b:
            x, weight, pre = ctx.saved_tensors

            def gradient():
                # The pre-activation's own gradient goes round the activation; sums of the two are rounded once more.
                parts = [encoder._linear_grad(g, x, weight, z, act, want_b, want_x, want_w)
                         for g, z, act in ((grad, pre, ctx.activation), (grad_pre, None, None)) if g is not None]
                return parts[0] if len(parts) == 1 else tuple(None if a is None else a + b for a, b in zip(*parts))

            if grad is not None or grad_pre is not None:
                gx, gw, gb = _once("linear", gradient, grad, grad_pre, x, weight, pre)
        return gx, gw, gb, grad if want_r else None, None, None


class Orthogonalize(torch.autograd.Function):
    @staticmethod
    def forward(ctx, update, steps, coefficients):
        return encoder._orthogonalize(update, steps, coefficients)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("orthogonalize has no derivative: it makes an optimiser's steps, of an update that is detached "
                           "or under torch.no_grad()")
