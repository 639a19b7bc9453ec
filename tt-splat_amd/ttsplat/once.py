"""Gradients that have no derivative of their own."""
import torch


class _Once(torch.autograd.Function):
    """The first n tensors, as results of all of them whose backward raises."""

    @staticmethod
    def forward(ctx, n, *tensors):
        return tuple(t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("a second derivative through a token operator (attention, layer norm, "
                           "embedding) is not provided")


def once(grads, sources):
    """Gradients (None among them) made from `sources` outside autograd.  Under create_graph they
    keep a path to the sources that raises where a second derivative takes it: cut off, that part would
    be left out of the result without a word.  (torch's once_differentiable raises in backward()
    only: autograd.grad does not visit a node that leads to none of its inputs.)"""
    if not torch.is_grad_enabled():
        return grads
    some = [g for g in grads if g is not None]
    some = iter(_Once.apply(len(some), *some, *(s for s in sources if s is not None)))
    return tuple(None if g is None else next(some) for g in grads)
