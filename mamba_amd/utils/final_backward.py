"""Backwards without a derivative of their own."""
import functools

import torch

from .. import _native as nat


def final_backward(what):
    """Decorates an autograd function's backward whose results have no derivative: with
    create_graph they come out of a node that raises when a second backward
    reaches it (plain tensors would drop its terms); their values are of use as they are."""
    def wrap(backward):
        @functools.wraps(backward)
        def run(ctx, *grads):
            if not torch.is_grad_enabled():
                return backward(ctx, *grads)
            with torch.no_grad():
                r = backward(ctx, *grads)
            if isinstance(r, tuple):
                return tuple(nat.host().final_grads(what, list(r)))
            return nat.host().final_grads(what, [r])[0]
        return run
    return wrap
