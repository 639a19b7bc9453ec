"""Layer norm of rows of one column: x is its own mean, so y is the bias and dx is zero, both to the last
bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("w32", [False, True])
@pytest.mark.parametrize("R", [1, 77, 30000])
def test_one_column(R, w32, dtype):
    from ttsplat.norm import layer_norm
    print(f"[norm] one column R={R} {dtype} w32={w32}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(R)
    wt = torch.float32 if w32 else dtype
    x, dy = (torch.randn(R, 1, device="cuda", generator=gen).to(dtype) for _ in range(2))
    w, b = (torch.randn(1, device="cuda", generator=gen).to(wt) for _ in range(2))
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.equal(y.detach(), b.detach().to(dtype).expand(R, 1))
    assert bool((dx == 0).all()) and bool((dw == 0).all())
    # db is a sum of R values held in 32 bits, rounded once
    u = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[wt]
    want, size = dy.double().sum(), float(dy.double().abs().sum())
    assert abs(float(db.double() - want)) <= u * abs(float(want)) + 2.0 ** -24 * R ** 0.5 * size
