"""Attention on the GPU (no counterpart in the reference): gaussians over a view's tokens, tokens
among themselves.

`attention(q, k, v, key_mask, causal, scale)` is differentiable w.r.t. q, k and v.  The forward
keeps no scores, but each row's log-sum-exp and, in half types, what rounding the output left
behind; the backward recomputes the probabilities.  Types fp32, fp16 and bf16; the softmax and all
sums are fp32.  Results are the same bits every time.
"""
import torch

from . import kernels
from .once import once

F32 = torch.float32


def _last_contiguous(t):
    return t if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[3] < 2 \
        or t.stride(3) == 1 else t.contiguous()


class _Attention(torch.autograd.Function):
    """mask: uint8 or None, checked with the rest by attention()."""

    @staticmethod
    def forward(ctx, q, k, v, mask, causal, scale):
        lse = torch.empty(q.shape[:3], device=q.device, dtype=F32)
        out = kernels._attn_like(q)
        rest = None if q.dtype == F32 else torch.empty_like(out)
        kernels._attention_fwd(q, k, v, mask, causal, scale, out, lse, rest)
        ctx.save_for_backward(q, k, v, mask, out, rest, lse)
        ctx.meta = (causal, scale)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, mask, out, rest, lse = ctx.saved_tensors
        causal, scale = ctx.meta
        nq, nk, nv, _, _, _ = ctx.needs_input_grad
        grads = kernels._attention_bwd(q, k, v, mask, causal, scale, out, rest, lse,
                                       _last_contiguous(dout), nq, nk, nv)
        return (*once(grads, (q, k, v, dout)), None, None, None)


def attention(q, k, v, key_mask=None, causal=False, scale=None):
    """softmax(scale q k^T) v.  q [B, Hq, Nq, D], k and v [B, Hkv, Nk, D]: query head h reads key
    head h / (Hq / Hkv); any strides ([B, N, H, D] memory as a transposed view needs no copy), D up
    to 128, scale 1/sqrt(D) unless given (1e-30 to 1e30).  key_mask [B, Nk] bool or uint8: False
    hides a key (a gaussian out of view, padding), whatever its k and v hold.  causal: row i sees
    keys up to i + Nk - Nq.  A row that sees no key gives zeros and no gradient."""
    q, k, v = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        mask, scale = kernels._attn_check(q, k, v, key_mask, scale, None)
        return _Attention.apply(q, k, v, mask, bool(causal), scale)
    return kernels.attention_fwd(q, k, v, key_mask, causal, scale)
