"""The encoder's calls as nodes of torch's autograd graph (quiver_amd/encoder.py makes them where an input asks for it).

The backward passes are ``embed_grad`` and ``linear_grad``. They are not differentiable themselves, and
nothing here has a forward-mode derivative: either raises an error.
"""

from __future__ import annotations

import torch

from . import blocks, encoder


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


class BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, y, post_weight, gate, gate_activation, scale, eps):
        result = blocks._block_norm(x, weight, y, post_weight, gate, gate_activation, scale, eps)
        ctx.settings = gate_activation, eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if y is None else result[0], weight, y, post_weight, gate, scale)
        return result

    @staticmethod
    def backward(ctx, *grads):
        grad_r, grad_h = grads if len(grads) == 2 else (None, grads[0])
        if grad_r is None and grad_h is None:
            return (None,) * 8
        r, weight, y, post, gate, scale = ctx.saved_tensors
        activation, eps = ctx.settings
        need = ctx.needs_input_grad
        wanted = need[0], need[1], need[2], need[3], need[4], need[6]

        def gradient():
            h = grad_h if grad_h is not None else torch.zeros_like(r)
            return blocks._block_norm_grad(h, r, weight, grad_r, y, post, gate, activation, scale, eps, wanted)

        gx, gw, gy, gp, gg, gs = _once("block_norm", gradient, grad_h, grad_r, r, weight, y, post, gate, scale)
        return gx, gw, gy, gp, gg, None, gs, None


class LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale, keep_state):
        result = blocks._linear_attention(q, k, v, log_decay, state, lengths, scale, keep_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        return result

    @staticmethod
    def backward(ctx, grad, grad_state=None):
        if grad is None and grad_state is None:
            return (None,) * 8
        q, k, v, log_decay, state, lengths = ctx.saved_tensors

        def gradient():
            g = grad if grad is not None else q.new_zeros((*q.shape[:3], v.shape[3]))
            return blocks.linear_attention_grad(g, q, k, v, log_decay, state, lengths, ctx.scale, grad_state)

        gq, gk, gv, first = _once("linear_attention", gradient, grad, grad_state, q, k, v, state)
        return gq, gk, gv, None, first, None, None, None


class Orthogonalize(torch.autograd.Function):
    @staticmethod
    def forward(ctx, update, steps, coefficients):
        return encoder._orthogonalize(update, steps, coefficients)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("orthogonalize has no derivative: it makes an optimiser's steps, of an update that is detached "
                           "or under torch.no_grad()")
