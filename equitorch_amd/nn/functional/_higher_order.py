"""Gradients of a tensor expression for a backward that runs in gradient mode (forces in the loss): they are differentiable
themselves, and replace what a kernel computes otherwise."""
import torch
from torch import Tensor


def higher_order(expression, inputs, need, g: Tensor, create_graph: bool = True):
    """Gradients of ``expression(*inputs)`` for the inputs ``need`` marks, None for the others and where nothing depends on one.

    Partial derivatives: the expression is evaluated on views of the inputs and differentiated with respect to the views.  The
    inputs come with their history, and one may be another, or computed from another (the features and the harmonics of a
    second layer, queries and keys of one tensor): with respect to the inputs themselves a path through another one would count
    here and once more where the engine walks on from it.

    The expression chooses its types itself: under autocast its products in 32 bits would be taken in 16."""
    with torch.enable_grad(), torch.autocast(g.device.type, enabled=False):
        own = [None if t is None else t.view_as(t) for t in inputs]
        grads = iter(torch.autograd.grad(expression(*own), [t for t, n in zip(own, need) if n], g, create_graph=create_graph,
                                         allow_unused=True))
    return tuple(next(grads) if n else None for n in need)
