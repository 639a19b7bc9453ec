"""Colours that follow a view's look: exposure, white balance, time of day (no counterpart in the
reference, whose scenes have one look).

A scene photographed under changing conditions keeps its geometry and a colour for each gaussian;
what a view changes is a colour offset that a small network gives from a code of the gaussian
and a few tokens of the view:

  x = s C[code]                        codes of the gaussians          ttsplat.embedding
  h = norm(x), t = norm(s T[view])     normalised, as are the tokens   ttsplat.norm
  y = x + attention(h Wq, t Wk, t Wv) Wo                               ttsplat.attention
  offset = norm(y) Wc                  added to color_dc (zero at the start: Wc = 0)

Codes are shared by gaussians of a neighbourhood (cell_codes), so their gradient is a sum over many
gaussians; views of a batch may have different numbers of tokens (token_mask).

    app = Appearance(n_codes=4096, n_views=len(cameras), device="cuda")
    ids = cell_codes(model.means3d, 4096, cell=0.1)
    fit_appearance(model, app, ids, cameras, images, iters=200)
    img = binned.render_binned_device(app.dress(model, ids, view), cam, tmap)
"""
import math

import torch

from . import binned, kernels
from .attention import attention
from .embedding import embedding
from .loss import loss_fn
from .norm import layer_norm

F32 = torch.float32


def cell_codes(means, n_codes, cell):
    """Code ids [G] int32 of gaussians by the cube of side `cell` that their mean is in, hashed to
    [0, n_codes); a gaussian whose mean is not finite gets -1 (no code)."""
    if n_codes < 1 or not cell > 0:
        raise ValueError("n_codes must be >= 1 and cell > 0")
    m = means.detach()
    fine = torch.isfinite(m).all(1)
    q = torch.floor(torch.where(fine[:, None], m, torch.zeros_like(m)) / cell).long()
    h = (q[:, 0] * 73856093) ^ (q[:, 1] * 19349663) ^ (q[:, 2] * 83492791)   # primes: spread cells
    return torch.where(fine, h % n_codes, torch.full_like(h, -1)).to(torch.int32)


class _Dressed:
    """A model's parameters in a view's colours, as the renders read a model."""

    def __init__(self, model, params):
        self.params = params
        for name in ("w_b_raw", "c_b", "depth_beta", "depth_tau", "softz_beta", "color_rest"):
            if hasattr(model, name):
                setattr(self, name, getattr(model, name))


class Appearance:
    """Codes, view tokens and weights, as leaves of one fp32 block (`flat`, the optimizer's view of
    them).  width: values a code, a multiple of heads; kv_heads: key heads (heads a multiple of it);
    dtype: the network's type (products and rows between them; leaves and sums are fp32)."""

    def __init__(self, n_codes, n_views, tokens=16, width=32, heads=4, kv_heads=None, dtype=F32,
                 seed=0, device="cuda"):
        kv_heads = heads if kv_heads is None else kv_heads
        if min(n_codes, n_views, tokens, width, heads, kv_heads) < 1:
            raise ValueError("sizes must be positive")
        if width % heads or heads % kv_heads:
            raise ValueError("width must be a multiple of heads, and heads of kv_heads")
        if dtype not in kernels.DTYPE_CODES:
            raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        self.n_views, self.tokens, self.heads, self.kv_heads = n_views, tokens, heads, kv_heads
        self.dtype, self.scale = dtype, math.sqrt(width)
        kv = width // heads * kv_heads
        r = 1.0 / math.sqrt(width)
        shapes = [("codes", (n_codes, width), r), ("views", (n_views * tokens, width), r),
                  ("norm_x", (2, width), None), ("norm_t", (2, width), None),
                  ("norm_y", (2, width), None), ("wq", (width, width), r), ("wk", (width, kv), r),
                  ("wv", (width, kv), r), ("wo", (width, width), r), ("wc", (width, 3), 0.0)]
        gen = torch.Generator().manual_seed(seed)
        parts = []
        for name, shape, std in shapes:
            if std is None:                      # a norm's weight and bias
                parts.append(torch.stack([torch.ones(shape[1]), torch.zeros(shape[1])]))
            else:
                parts.append(torch.randn(shape, generator=gen) * std)
        self.flat = torch.cat([p.reshape(-1) for p in parts]).to(device)
        at = 0
        for (name, shape, _), p in zip(shapes, parts):
            setattr(self, name, self.flat[at:at + p.numel()].view(shape).requires_grad_(True))
            at += p.numel()
        self.names = [s[0] for s in shapes]

    def leaves(self):
        return [getattr(self, n) for n in self.names]

    def _norm(self, x, wb):
        return layer_norm(x, wb[0], wb[1])

    def offsets(self, code_ids, view, token_mask=None):
        """Colour offsets [G, 3] of the gaussians with these codes in view `view`; token_mask
        [tokens] (non-zero: used) leaves tokens of the view out."""
        if not 0 <= int(view) < self.n_views:
            raise ValueError(f"view must be in [0, {self.n_views}), got {view}")
        dev, dt = self.flat.device, self.dtype
        G = code_ids.shape[0]
        first = int(view) * self.tokens
        x = embedding(self.codes.to(dt), code_ids, self.scale)
        t = embedding(self.views.to(dt), torch.arange(first, first + self.tokens, device=dev),
                      self.scale)
        h, t = self._norm(x, self.norm_x), self._norm(t, self.norm_t)

        def heads(y, n):                          # [rows, n * size] -> [1, n, rows, size], a view
            return y.view(1, y.shape[0], n, -1).transpose(1, 2)

        q = heads(h @ self.wq.to(dt), self.heads)
        k = heads(t @ self.wk.to(dt), self.kv_heads)
        v = heads(t @ self.wv.to(dt), self.kv_heads)
        mask = None if token_mask is None else token_mask.reshape(1, -1)
        o = attention(q, k, v, key_mask=mask).transpose(1, 2).reshape(G, -1)
        y = x + o @ self.wo.to(dt)
        return self._norm(y, self.norm_y).float() @ self.wc

    def dress(self, model, code_ids, view, token_mask=None):
        """`model` in view `view`'s colours, for any of the renders; differentiable w.r.t. the
        network and the model."""
        P = binned.params_of(model)
        off = self.offsets(code_ids, view, token_mask)
        return _Dressed(model, torch.cat([P[:, :10], P[:, 10:13] + off, P[:, 13:]], 1))


def fit_appearance(model, app, code_ids, cameras, images, iters=200, lr=5e-3, lambda_ssim=0.2, K=128,
                   views=None):
    """Trains the network on photographs of a scene whose gaussians stay as they are: one binned
    render and photometric loss a camera and iteration, Adam (tts_adam_flat).  views: the view
    number of each camera (its index unless given).  Returns the mean loss of each iteration."""
    views = list(range(len(cameras))) if views is None else list(views)
    dev = app.flat.device
    tmaps = [binned.TileMap(c.H, c.W) for c in cameras]
    gts = [g.to(dev, F32).contiguous() for g in images]
    m, v = torch.zeros_like(app.flat), torch.zeros_like(app.flat)
    step, lr1 = kernels.adam_state(dev), torch.tensor([float(lr)], device=dev)
    leaves, history = app.leaves(), []
    for _ in range(iters):
        total = 0.0
        for cam, tmap, gt, view in zip(cameras, tmaps, gts, views):
            img = binned.render_binned_device(app.dress(model, code_ids, view), cam, tmap, K=K)
            total = total + loss_fn(img, gt, lambda_ssim)
        total = total / len(cameras)
        grads = torch.autograd.grad(total, leaves)
        kernels.adam_advance(step)
        with torch.no_grad():
            kernels.adam_flat(app.flat, m, v, torch.cat([g.reshape(-1) for g in grads]), lr1, step)
        history.append(float(total.detach()))
    return history
