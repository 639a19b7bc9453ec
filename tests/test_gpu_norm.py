"""Layer norm (ttsplat.norm) against the formula in 64 bits, on the GPU.

Tolerances, from the arithmetic (u the unit roundoff of the result's type, 2^-24, 2^-11, 2^-8 for
fp32, fp16, bf16): y and dx are rounded once, so each is off by u times its size, plus the fp32
sums' error.  A sum of n fp32 terms in any order is off by at most n 2^-24 times the sum of
sizes, a few sqrt(n) 2^-24 in practice: 1e-5 of the largest value covers rows and columns of
up to 1e5 terms; where a row's mean is s standard deviations from zero, x - m carries 2^-24 s more.
dx is a difference of terms of size r |g|, r |mean g| and r |xh mean(g xh)|, which cancel in short
rows (two values: to zero but for eps), so its share of the fp32 error goes by the terms' size."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def formula(x, w, b, dy, eps):
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[-1], dtype=x.dtype, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    m = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - m) * r
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, x.shape[-1]).sum(0)   # noqa: E731
    terms = r * (g.abs() + g.mean(-1, keepdim=True).abs()
                 + (xh * (g * xh).mean(-1, keepdim=True)).abs())
    return xh * w + b, dx, flat(dy * xh), flat(dy), float(terms.max()) if terms.numel() else 0.0


def close(got, want, what, u, slack=1e-5, size=0.0):
    assert got.dtype in U and got.shape == want.shape, what
    if want.numel() == 0:
        return
    err = (got.double() - want).abs()
    top = max(float(want.abs().max()), size)
    bad = err > u * want.abs() * 1.01 + slack * max(top, 1e-30)
    assert not bool(bad.any()), f"{what}: max err {float(err.max()):.3e}, largest value {top:.3e}"


def inputs(shape, dtype, wdtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(shape, device="cuda", generator=g) * 1.5
         + spread * torch.randn((*shape[:-1], 1), device="cuda", generator=g)).to(dtype)
    dy = torch.randn(shape, device="cuda", generator=g).to(dtype)
    w = (1 + 0.2 * torch.randn(shape[-1], device="cuda", generator=g)).to(wdtype)
    b = torch.randn(shape[-1], device="cuda", generator=g).to(wdtype)
    return x, dy, w, b


def check(x, dy, w, b, eps=1e-5, slack=1e-5):
    from ttsplat.norm import layer_norm
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(leaves)
    xl = next(it)
    wl = next(it) if w is not None else None
    bl = next(it) if b is not None else None
    y = layer_norm(xl, wl, bl, eps)
    grads = list(torch.autograd.grad(y, leaves, dy))
    ry, rdx, rdw, rdb, terms = formula(x, w, b, dy, eps)
    close(y.detach(), ry, "y", U[x.dtype], slack)
    close(grads.pop(0), rdx, "dx", U[x.dtype], slack, terms)
    if w is not None:
        close(grads.pop(0), rdw, "dw", U[w.dtype], slack)
    if b is not None:
        close(grads.pop(0), rdb, "db", U[b.dtype], slack)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D", [(1, 1), (1, 2), (3, 3), (5, 7), (64, 8), (65, 9), (33, 17),
                                 (257, 32), (64, 64), (130, 65), (31, 127), (40, 128), (19, 255),
                                 (64, 511), (50, 1003), (9, 1024), (7, 1025), (5, 2048), (4, 2049),
                                 (3, 4096), (37, 5000)])
def test_sizes(R, D, dtype):
    print(f"[norm] {R}x{D} {dtype}", flush=True)
    check(*inputs((R, D), dtype, dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,D", [(300, 64), (77, 1003), (6, 3000)])
def test_weights_in_32_bits(R, D, dtype):
    print(f"[norm] {R}x{D} {dtype} fp32 weights", flush=True)
    check(*inputs((R, D), dtype, torch.float32))


@pytest.mark.parametrize("R,D", [(100000, 32), (20011, 64), (8040, 257), (4000, 4100)])
def test_many_rows(R, D):
    print(f"[norm] {R}x{D}", flush=True)
    check(*inputs((R, D), torch.float32, torch.float32))


@pytest.mark.parametrize("w,b", [(False, False), (True, False), (False, True)])
def test_absent_weights(w, b):
    x, dy, wt, bi = inputs((50, 48), torch.bfloat16, torch.float32)
    check(x, dy, wt if w else None, bi if b else None)


def test_strides_and_shapes():
    """Rows of a wider block, a row repeated by a stride of zero, columns that are not contiguous,
    rows at an odd address, more axes than two, gradients that are expanded."""
    x, dy, w, b = inputs((40, 96), torch.bfloat16, torch.bfloat16)
    check(x[:, :64], dy[:, :64], w[:64], b[:64])
    check(x[:, 5:38], dy[:, 3:36], w[5:38].contiguous(), b[5:38].contiguous())
    check(x[:1].expand(40, 96), dy, w, b)
    check(x.t().contiguous().t(), dy, w, b)
    check(x.view(4, 10, 96), dy.view(4, 10, 96), w, b)
    check(x.view(4, 10, 96).transpose(0, 1), dy.view(10, 4, 96), w, b)
    check(x[0], dy[0], w, b)
    check(x, dy[:1].expand(40, 96), w, b)


def test_offsets_past_32_bits():
    """Rows two million elements apart, the last 8 GB behind the first."""
    wide = torch.empty(2100, 1 << 21, device="cuda", dtype=torch.bfloat16)
    x, dy, w, b = inputs((2100, 40), torch.bfloat16, torch.float32)
    wide[:, :40] = x
    wide[:, 64:104] = dy
    check(wide[:, :40], wide[:, 64:104], w, b)


def test_no_rows():
    from ttsplat.norm import layer_norm
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and torch.equal(dw, torch.zeros(16).cuda())


def test_far_from_zero_mean():
    """Rows 1000 standard deviations from zero: squared deviations, not a difference of squares.
    x - m carries 2^-24 * 1000 of the deviation, so 1e-4 covers a row's values."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = 1000 + torch.randn(64, 200, device="cuda", generator=g)
    _, dy, w, b = inputs((64, 200), torch.float32, torch.float32)
    check(x, dy, w, b, slack=1e-3)


def test_constant_rows():
    """Variance zero: 1 / sqrt(eps), finite."""
    x = torch.full((3, 40), 2.5, device="cuda")
    _, dy, w, b = inputs((3, 40), torch.float32, torch.float32)
    check(x, dy, w, b)


def test_a_row_with_nan_stays_alone():
    from ttsplat.norm import layer_norm
    x, dy, w, b = inputs((64, 24), torch.float32, torch.float32)
    x[7, 3] = float("nan")
    y = layer_norm(x, w, b)
    bad = ~torch.isfinite(y).all(1)
    assert bad.nonzero().flatten().tolist() == [7]


def test_gradients_against_differences():
    """Central differences of the kernel's own forward on fp32: step h = 1e-2, the error h^2 / 6 of the
    third derivative plus 2^-24 |L| / h of rounding, well below 1e-2 of the largest entry."""
    from ttsplat.norm import layer_norm
    x, dy, w, b = inputs((3, 6), torch.float32, torch.float32, seed=5)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    for k, g in enumerate(grads):
        num = torch.zeros_like(g)
        for i in range(g.numel()):
            vals = []
            for s in (1e-2, -1e-2):
                t = [v.clone() for v in (x, w, b)]
                t[k].view(-1)[i] += s
                vals.append((layer_norm(*t).double() * dy.double()).sum())
            num.view(-1)[i] = float(vals[0] - vals[1]) / 2e-2
        assert float((num - g).abs().max()) <= 1e-2 * float(g.abs().max())


def test_same_bits_twice():
    from ttsplat import kernels
    x, dy, w, b = inputs((30011, 96), torch.float32, torch.float32)
    stats = torch.empty(30011, 2, device="cuda")
    kernels.layer_norm_fwd(x, w, b, stats=stats)
    a = kernels.layer_norm_bwd(x, w, dy, stats)
    c = kernels.layer_norm_bwd(x, w, dy, stats)
    assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_parts_of_the_backward():
    from ttsplat import kernels
    x, dy, w, b = inputs((333, 40), torch.float32, torch.float32)
    stats = torch.empty(333, 2, device="cuda")
    kernels.layer_norm_fwd(x, w, b, stats=stats)
    dx, dw, db = kernels.layer_norm_bwd(x, w, dy, stats)
    for fx, fw, fb in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
        p = kernels.layer_norm_bwd(x, w, dy, stats, bool(fx), bool(fw), bool(fb))
        for got, want, f in zip(p, (dx, dw, db), (fx, fw, fb)):
            assert torch.equal(got, want) if f else got is None


def test_another_stream_and_graph():
    """On a stream of the caller's, and replayed from a graph."""
    from ttsplat import kernels
    x, dy, w, b = inputs((500, 72), torch.bfloat16, torch.float32)
    stats = torch.empty(500, 2, device="cuda")
    y0 = kernels.layer_norm_fwd(x, w, b, stats=stats)
    g0 = kernels.layer_norm_bwd(x, w, dy, stats)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y1 = kernels.layer_norm_fwd(x, w, b)
    s.synchronize()
    assert torch.equal(y0, y1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2 = kernels.layer_norm_fwd(x, w, b, stats=stats)
        g2 = kernels.layer_norm_bwd(x, w, dy, stats)
    for _ in range(3):
        y2.zero_()
        [t.zero_() for t in g2]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y0, y2) and all(torch.equal(p, q) for p, q in zip(g0, g2))


def test_refusals():
    from ttsplat import kernels
    from ttsplat.norm import layer_norm
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for bad in (lambda: layer_norm(x.cpu()), lambda: layer_norm(x.double()),
                lambda: layer_norm(x, w[:4]), lambda: layer_norm(x, w.half()),
                lambda: layer_norm(x.half(), w.half(), w), lambda: layer_norm(x[:, :0]),
                lambda: layer_norm(x, w.cpu()),
                lambda: kernels.layer_norm_fwd(x[0]),
                lambda: kernels.layer_norm_fwd(x.t()),
                lambda: kernels.layer_norm_fwd(x, y=torch.zeros(4, 7, device="cuda")),
                lambda: kernels.layer_norm_bwd(x, w, x.half(), torch.zeros(4, 2, device="cuda")),
                lambda: kernels.layer_norm_bwd(x, w, x, torch.zeros(3, 2, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
