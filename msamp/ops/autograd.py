"""Backward passes whose results have no gradient of their own."""
import functools

import torch


class _NoGradientFn(torch.autograd.Function):
    """Passes gradients on; differentiating them is an error."""
    @staticmethod
    def forward(ctx, anchor, name, *grads):
        ctx.name = name
        return grads

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f'{ctx.name}: the gradient is made by a kernel that cannot be differentiated twice')


def once(backward):
    """For the ``backward`` of an autograd function that calls kernels: with ``create_graph`` its gradients belong to a graph that raises an
    error when it is differentiated, where they would have none and their share would be missing from a sum.  (torch's decorator of this
    kind leaves them without a graph when the incoming gradient is a constant.)
    """
    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        out = out if isinstance(out, tuple) else (out, )
        # the anchor asks for a gradient where no incoming one does
        back = iter(_NoGradientFn.apply(torch.empty(0, requires_grad=True), type(ctx).__name__, *(g for g in out if g is not None)))
        return tuple(None if g is None else next(back) for g in out)

    return wrapped
