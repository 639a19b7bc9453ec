"""Embedding lookup with scaling on the GPU (no counterpart in the reference): codes of gaussians
and of a view's tokens.

`embedding(table, ids, scale)` is differentiable w.r.t. the table.  The gradient sorts the
tokens by id and sums each row's tokens in token order in fp32: it is dense ([V, D], like the
table) and the same bits every time.
"""
import torch

from . import kernels
from .once import once


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.meta = (table.shape[0], scale)
        return kernels.embedding_fwd(table, ids, scale)

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        V, scale = ctx.meta
        dtable = kernels._embedding_bwd(dout.contiguous(), ids, V, scale)
        return (*once((dtable,), (dout,)), None, None)


def embedding(table, ids, scale=1.0):
    """scale * table[ids] [*ids.shape, D] for a table [V, D] of fp32, fp16 or bf16 and int32 or
    int64 ids; an id outside [0, V) stands for no entry: a row of zeros, without gradient."""
    if isinstance(ids, torch.Tensor):
        ids = ids.contiguous()
    if not isinstance(table, torch.Tensor):
        raise TypeError("table must be a torch.Tensor")
    table = table.contiguous()
    if torch.is_grad_enabled() and table.requires_grad:
        return _Embedding.apply(table, ids, float(scale))
    return kernels.embedding_fwd(table, ids, scale)
