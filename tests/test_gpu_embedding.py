"""Embedding lookup and its gradient (ttsplat.embedding) against sums in 64 bits, on the GPU.

Tolerances: a lookup is one product rounded once, u of its size (u = 2^-24, 2^-11, 2^-8); a row
of the gradient is a sum of n fp32 terms, off by at most n 2^-24 times the sum of their sizes
(here through levels of 64, so far less: 1e-5 of that sum), rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def check(table, ids, dy, scale=1.0):
    from ttsplat.embedding import embedding
    V, D = table.shape
    t = table.detach().requires_grad_(True)
    y = embedding(t, ids, scale)
    (g,) = torch.autograd.grad(y, t, dy)
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < V)
    want = torch.zeros(flat.numel(), D, device="cuda", dtype=torch.float64)
    want[ok] = table.double()[flat[ok]] * scale
    u = U[table.dtype]
    assert y.shape == (*ids.shape, D) and y.dtype == table.dtype
    # 1.01 for the fp32 product's rounding before the last one, twice u for fp32 itself; results
    # under the type's normal range are off by half its smallest step
    tiny = 2.0 ** -25 if table.dtype == torch.float16 else 0.0
    err = (y.detach().double().reshape(want.shape) - want).abs()
    assert bool((err <= 2 * u * want.abs() + tiny).all())
    gd = (dy.double().reshape(-1, D)[ok] * scale).cpu()      # on the host: no contended atomics
    ref = torch.zeros(V, D, dtype=torch.float64).index_add_(0, flat[ok].cpu(), gd).cuda()
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, flat[ok].cpu(), gd.abs()).cuda()
    assert g.shape == table.shape and g.dtype == table.dtype
    err = (g.double() - ref).abs()
    assert bool((err <= 2 * u * ref.abs() + 1e-5 * mag + tiny).all()), float(err.max())
    # rows no token names are zeros
    assert bool((g[(mag == 0).all(1)] == 0).all())
    from ttsplat import kernels
    assert torch.equal(kernels.embedding_bwd(dy.contiguous(), ids.contiguous(), V, scale), g)
    return g


def inputs(N, V, D, dtype, draw, itype=torch.int32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.randn(V, D, device="cuda", generator=gen).to(dtype)
    dy = torch.randn(N, D, device="cuda", generator=gen).to(dtype)
    u = torch.rand(N, device="cuda", generator=gen)
    if draw == "uniform":
        ids = (u * V).long().clamp(max=V - 1)
    elif draw == "skewed":
        ids = (u.pow(6) * V).long().clamp(max=V - 1)
    elif draw == "one":
        ids = torch.full((N,), V // 2, device="cuda")
    elif draw == "sorted":
        ids = (torch.arange(N, device="cuda") * V) // max(N, 1)
    else:                                     # some outside the table on both sides
        ids = (u * 2 * V).long() - V // 2
    return table, ids.to(itype), dy


@pytest.mark.parametrize("draw", ["uniform", "skewed", "one", "sorted", "outside"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 5, 3), (63, 2, 8), (64, 1, 4), (65, 3, 5),
                                   (127, 40, 33), (257, 1000, 64), (4095, 7, 17),
                                   (4096, 2047, 32), (4097, 2048, 9), (9000, 2, 40),
                                   (12288, 5000, 2), (20000, 300, 16)])
def test_sizes(N, V, D, draw):
    print(f"[embed] N={N} V={V} D={D} {draw}", flush=True)
    check(*inputs(N, V, D, torch.float32, draw), scale=1.5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (300, 20, 7), (5000, 100, 64), (5000, 9000, 130),
                                   (70000, 4, 513)])
def test_half_types(N, V, D, dtype):
    print(f"[embed] N={N} V={V} D={D} {dtype}", flush=True)
    check(*inputs(N, V, D, dtype, "skewed", torch.int64), scale=0.125)


@pytest.mark.parametrize("N,V,D,draw", [(300001, 5, 8, "skewed"), (1000000, 100003, 16, "skewed"),
                                        (100000, 5000000, 4, "uniform"),
                                        (600000, 64, 24, "one")])
def test_long(N, V, D, draw):
    print(f"[embed] N={N} V={V} D={D} {draw}", flush=True)
    check(*inputs(N, V, D, torch.float32, draw))


def test_token_order_within_a_row():
    """Sums of a row run in token order: with values whose order shows (2^24, 1, -2^24, 1), the row's
    result is that of the order of the tokens, in both sorts."""
    for pad in (0, 5000):
        seq = torch.tensor([2.0 ** 24, 1.0, -2.0 ** 24, 1.0], device="cuda")
        ids = torch.cat([torch.zeros(4), 1 + torch.arange(pad) % 7]).to(torch.int32).cuda()
        perm = torch.randperm(4 + pad, generator=torch.Generator().manual_seed(1)).cuda()
        ids = ids[perm]
        dy = torch.ones(4 + pad, 1, device="cuda")
        dy[(ids == 0).nonzero().flatten(), 0] = seq
        from ttsplat import kernels
        g = kernels.embedding_bwd(dy, ids.contiguous(), 9)
        want = torch.tensor(0.0)
        for s in seq.cpu():
            want = want + s
        assert float(g[0, 0]) == float(want)


def test_shapes_and_strides():
    table, ids, dy = inputs(60, 30, 20, torch.float32, "uniform", torch.int64)
    check(table, ids.view(3, 4, 5), dy.view(3, 4, 5, 20))
    check(table, ids.view(6, 10).t(), dy.view(6, 10, 20).transpose(0, 1))
    check(table, ids[::2], dy[::2])
    check(table, ids, dy[:1].expand(60, 20))
    wide = torch.randn(30, 50, device="cuda")
    check(wide[:, 7:27], ids, dy)
    check(table, ids[0], dy[0])                       # a single id: no axes


def test_nothing():
    from ttsplat.embedding import embedding
    table = torch.randn(4, 6, device="cuda", requires_grad=True)
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    y = embedding(table, ids)
    (g,) = torch.autograd.grad(y, table, torch.empty_like(y))
    assert y.shape == (0, 6) and torch.equal(g, torch.zeros(4, 6, device="cuda"))


def test_offsets_past_32_bits():
    """A table of 5 GB: rows at its end, and their gradient."""
    from ttsplat import kernels
    V, D = 40_000_000, 64
    table = torch.empty(V, D, device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(V - 900, V, (3000,), device="cuda", generator=gen)
    table[V - 900:] = torch.randn(900, D, device="cuda", generator=gen).to(torch.bfloat16)
    dy = torch.randn(3000, D, device="cuda", generator=gen).to(torch.bfloat16)
    assert torch.equal(kernels.embedding_fwd(table, ids), table[ids])
    del table
    g = kernels.embedding_bwd(dy, ids, V)
    ref = torch.zeros(900, D, dtype=torch.float64).index_add_(0, (ids - (V - 900)).cpu(), dy.double().cpu())
    err = (g[V - 900:].double().cpu() - ref).abs()
    assert bool((err <= 2.0 ** -7 * ref.abs() + 1e-5 * 20).all())
    assert int(g[:V - 900].count_nonzero()) == 0


def test_rows_outside_leave_nan_out():
    """A NaN in the gradient of a token without an entry reaches no row."""
    table, ids, dy = inputs(200, 10, 8, torch.float32, "uniform")
    ids[5], ids[77] = -1, 10
    dy[5], dy[77] = float("nan"), float("inf")
    from ttsplat import kernels
    assert bool(torch.isfinite(kernels.embedding_bwd(dy, ids, 10)).all())


def test_graph_replays():
    from ttsplat import kernels
    table, ids, dy = inputs(9001, 700, 24, torch.float32, "skewed")
    want, gwant = kernels.embedding_fwd(table, ids, 2.0), kernels.embedding_bwd(dy, ids, 700, 2.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kernels.embedding_fwd(table, ids, 2.0)
        g = kernels.embedding_bwd(dy, ids, 700, 2.0)
    for _ in range(3):
        y.zero_()
        g.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(g, gwant)


def test_refusals():
    from ttsplat import _lib, kernels
    from ttsplat.embedding import embedding
    table = torch.zeros(4, 8, device="cuda")
    ids = torch.zeros(5, dtype=torch.int32, device="cuda")
    for bad in (lambda: embedding(table.cpu(), ids), lambda: embedding(table, ids.cpu()),
                lambda: embedding(table, ids.float()), lambda: embedding(table.double(), ids),
                lambda: embedding(table[0], ids),
                lambda: kernels.embedding_fwd(table.t(), ids),
                lambda: kernels.embedding_bwd(torch.zeros(4, 8, device="cuda"), ids, 4),
                lambda: kernels.embedding_bwd(torch.zeros(5, 8, device="cuda"), ids, 4,
                                              out=torch.zeros(3, 8, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.TTSError):
        kernels.embedding_bwd(torch.zeros(5, 8, device="cuda"), ids, 4,
                              workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(_lib.TTSError):
        kernels.embedding_bwd(torch.zeros(5, 8, device="cuda"), ids, 0,
                              out=torch.zeros(0, 8, device="cuda"))
