"""Layer norm of feature rows on the GPU (no counterpart in the reference).

`layer_norm(x, weight, bias, eps)` is differentiable w.r.t. x, weight and bias.  Rows may be
fp32, fp16 or bf16, weights of the same type or fp32; statistics and sums are fp32, and the
gradients of weight and bias are summed over the rows in a fixed order.
"""
import torch

from . import kernels
from .once import once

F32 = torch.float32


def _rows(x):
    """x [..., D] as [rows, D] with contiguous columns (a view wherever one exists)."""
    D = x.shape[-1]
    r = x if x.dim() == 2 else x.reshape(-1, D)
    return r if D == 1 or r.stride(1) == 1 else r.contiguous()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows = _rows(x)
        stats = torch.empty(rows.shape[0], 2, device=x.device, dtype=F32)
        y = kernels.layer_norm_fwd(rows, weight, bias, eps, stats=stats)
        ctx.save_for_backward(x, weight, stats)
        ctx.w_dtype = (bias.dtype if bias is not None else x.dtype) if weight is None else weight.dtype
        return y if x.dim() == 2 else y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        nx, nw, nb, _ = ctx.needs_input_grad
        dx, dw, db = kernels._layer_norm_bwd(_rows(x), weight, _rows(dy), stats, nx, nw, nb,
                                             ctx.w_dtype)
        dx = dx if dx is None or x.dim() == 2 else dx.view(x.shape)
        return (*once((dx, dw, db), (x, weight, dy)), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x [..., D]."""
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be a tensor [..., D] with D >= 1")
    if torch.is_grad_enabled() and (x.requires_grad
                                    or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    y = kernels.layer_norm_fwd(_rows(x), weight, bias, eps)
    return y if x.dim() == 2 else y.view(x.shape)
